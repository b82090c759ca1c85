"""GPU: the codebook operators at the largest sizes that they take and at the smallest shapes, and torch's transforms that they refuse."""
import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

import codebook_reference as ref
from rise_sdf_amd import _lib, ops
from rise_sdf_amd.loss import linear_cross_entropy, linear_distillation
from test_gpu_codebook import BF16, F16, F32, TYPES, check_head, check_lookup, gen, head_case, lookup_case, teacher

pytestmark = pytest.mark.gpu


def test_lookup_of_two_to_the_30_positions(dev):
    """One number per id; the gradient of ones counts the positions of each id: whole numbers below 2^24, so they are exact."""
    n, v = 1 << 30, 70000
    ids = torch.randint(0, v, (n,), device=dev, generator=gen(dev, 1))
    ids[-3:] = v - 1
    table = torch.randn(v, 1, device=dev, generator=gen(dev, 2)).requires_grad_(True)
    out = ops.embedding(ids, table, 2.0)
    (dt,) = torch.autograd.grad(out, table, torch.ones_like(out))
    for part in range(0, n, 1 << 27):
        assert torch.equal(out[part:part + (1 << 27)], table.detach()[ids[part:part + (1 << 27)]] * 2.0)
    assert torch.equal(dt[:, 0], torch.bincount(ids, minlength=v).float() * 2.0)
    del ids, out
    torch.cuda.empty_cache()


def test_lookup_in_two_to_the_30_rows(dev):
    n, v = 5000, 1 << 30
    ids = torch.randint(0, v, (n,), device=dev, generator=gen(dev, 3))
    ids[:3] = torch.tensor([0, v - 1, v - 1], device=dev)
    rows, at = torch.unique(ids, return_inverse=True)
    small = torch.randn(rows.numel(), 2, device=dev, generator=gen(dev, 4)).to(F16)
    table = torch.zeros(v, 2, dtype=F16, device=dev)
    table[rows] = small
    grad = torch.randn(n, 2, device=dev, generator=gen(dev, 5)).to(F16)
    table.requires_grad_(True)
    out = ops.embedding(ids, table)
    (dt,) = torch.autograd.grad(out, table, grad)
    want, bound, d_want, d_bound = ref.embedding(at, small, 1.0, None, grad)
    ref.assert_within("out", out.detach(), want, bound)
    ref.assert_within("d_table", dt[rows], d_want, d_bound)
    dt[rows] = 0.0
    assert not any(bool(part.any()) for part in dt.split(1 << 27))
    del table, dt
    torch.cuda.empty_cache()


def test_head_of_two_to_the_24_rows(dev):
    """In chunks of 2^20 rows against 64 bits.  The bound of a chunk's part of dw allows for the sums over its rows; over all rows each of its terms
    grows at most 16-fold."""
    n, v, d, step = 1 << 24, 300, 8, 1 << 20
    g = gen(dev, 6)
    w = (torch.randn(v, d, device=dev, generator=g) * 0.7).to(BF16).requires_grad_(True)
    x = torch.randn(n, d, device=dev, generator=g).to(BF16).requires_grad_(True)
    y = torch.randint(0, v, (n,), device=dev, generator=g)
    y[::5] = -100
    loss = linear_cross_entropy(x, w, y)
    dx, dw = torch.autograd.grad(loss, (x, w))
    count = int((y != -100).sum())
    xd, wd = x.detach(), w.detach()
    total, e_total, want_dw, e_dw = 0.0, 0.0, 0.0, 0.0
    weight = torch.full((step,), 1.0 / count, dtype=torch.float64, device=dev)
    for a in range(0, n, step):
        rows = slice(a, a + step)
        want = ref.head(xd[rows], wd, y[rows][:, None], None, -100, 1.0, "none", weight)
        total, e_total = total + float(want["loss"].sum()), e_total + float(want["e_loss"].sum())
        want_dw, e_dw = want_dw + want["dw"], e_dw + 16 * want["e_dw"]
        ref.assert_within("dx", dx[rows], want["dx"], want["e_dx"])
    assert abs(float(loss) - total / count) <= e_total / count + 2 * ref.E32 * total / count
    ref.assert_within("dw", dw, want_dw, e_dw)


@pytest.mark.parametrize("dtype", TYPES)
def test_shapes_without_dimensions(dev, dtype):
    """One id, one row, no batch dimension."""
    ids, table, grad = lookup_case(dev, 1, 9, 12, dtype, seed=7)
    t = table.clone().requires_grad_(True)
    out = ops.embedding(ids[0], t, 0.5)
    assert out.shape == (12,) and torch.equal(out, (table[ids[0]].float() * 0.5).to(dtype))
    (dt,) = torch.autograd.grad(out, t, grad[0])
    assert torch.equal(dt, check_lookup(ids, table, grad, 0.5, None)[1])
    x, w, y = head_case(dev, 1, 40, 24, dtype, seed=8)
    tid, tl = teacher(dev, 1, 40, 3, seed=9, missing=0.0)
    for red in ("none", "mean", "sum"):
        a = linear_cross_entropy(x[0], w, y[0], reduction=red)
        assert a.shape == () and torch.equal(a, linear_cross_entropy(x, w, y, reduction="sum"))
        b = linear_distillation(x[0], w, tid[0], tl[0], reduction=red)
        assert b.shape == () and torch.equal(b, linear_distillation(x, w, tid, tl, reduction="sum"))


@pytest.mark.parametrize("dtype", TYPES)
def test_an_ignored_label_inside_the_head(dev, dtype):
    """The class itself stays in every other row's sum."""
    x, w, y = head_case(dev, 90, 300, 40, dtype, seed=10)
    y[::4] = 0
    check_head(x, w, y, ignore=0)
    y[::4] = 299
    check_head(x, w, y, ignore=299, reduction="none", grad=torch.rand(90, device=dev, generator=gen(dev, 11)))


def test_transforms_are_refused(dev):
    """vmap, torch.func's gradients and forward mode: an error, no wrong number."""
    ids, table, _ = lookup_case(dev, 20, 10, 8, F32, seed=12)
    x, w, y = head_case(dev, 20, 10, 8, F32, seed=13)
    tid, tl = teacher(dev, 20, 10, 2, seed=14)
    calls = ((table, lambda t: ops.embedding(ids, t).sum()), (x, lambda t: linear_cross_entropy(t, w, y)),
             (w, lambda t: linear_cross_entropy(x, t, y)), (x, lambda t: linear_distillation(t, w, tid, tl)))
    for t, fn in calls:
        with pytest.raises(RuntimeError):
            torch.func.grad(fn)(t)
        with pytest.raises(RuntimeError):
            torch.func.vmap(fn)(torch.stack([t, t]))
        with pytest.raises(RuntimeError):
            with fwd_ad.dual_level():
                out = fn(fwd_ad.make_dual(t, torch.ones_like(t)))
                assert fwd_ad.unpack_dual(out).tangent is not None, "a silent zero"
        fn(t)
    _lib.poll_status(dev)
