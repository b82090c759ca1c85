"""GPU: the head's kernels at sizes that reach each of them, with remainders in rows, classes and features, and labels and listed classes on both sides
of every 256th class; bounds as in codebook_reference.py."""
import pytest
import torch

import codebook_reference as ref
from codebook_plans import CASES
from rise_sdf_amd.loss import linear_cross_entropy
from test_gpu_codebook import BF16, F16, F32, check_head, gen, head_case, teacher

pytestmark = pytest.mark.gpu


def borders(n, v):
    """Up to n classes at the ends of the head and around the multiples of 256, spread over all of them."""
    at = torch.arange(0, v + 256, 256)
    at = torch.cat([at, at - 1, torch.tensor([v - 1])])
    at = at[(at >= 0) & (at < v)].unique()
    return at[torch.linspace(0, at.numel() - 1, min(n, at.numel())).long()]


@pytest.mark.parametrize("n,v,d,kind", CASES)
def test_every_kernel_of_the_head(dev, n, v, d, kind):
    dtype = (F32, BF16, F16)[kind]
    x, w, y = head_case(dev, n, v, d, dtype, seed=n + d)
    at = borders(n, v).to(dev)
    y[:at.numel()] = at
    y[n // 2] = v - 1
    y[1::7] = -100
    check_head(x, w, y)
    ids, logits = teacher(dev, n, v, 3, seed=v)
    ids[:at.numel(), 0] = at.flip(0)
    check_head(x, w, ids, logits, temperature=2.0, reduction="none", grad=torch.rand(n, device=dev, generator=gen(dev, 5)))


def test_more_rows_than_one_launch_takes_classes_of(dev):
    """2^22 + 5 rows read where they are: the classes come in two launches of z.  Every 4099th row, and the last ones, against 64 bits."""
    n, v, d = (1 << 22) + 5, 8200, 8
    g = gen(dev, 6)
    w = (torch.randn(v, d, device=dev, generator=g) * 0.7).to(BF16)
    x = torch.randn(n, d, device=dev, generator=g).to(BF16)
    y = torch.randint(0, v, (n,), device=dev, generator=g)
    rows = torch.cat([torch.arange(0, n, 4099, device=dev), torch.arange(n - 300, n, device=dev)])
    y[rows[:20]] = torch.tensor([0, 255, 256, 7935, 7936, 7937, 8191, 8192, 8198, 8199] * 2, device=dev)
    loss = linear_cross_entropy(x, w, y, reduction="none")
    want = ref.head(x[rows], w, y[rows][:, None], None, -100, 1.0, "none")
    ref.assert_within("loss", loss[rows], want["loss"], want["e_loss"])
    assert bool(torch.isfinite(loss).all())
