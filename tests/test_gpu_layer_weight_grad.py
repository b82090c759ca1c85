"""GPU: the per-layer weight gradient (rsdf_linear_bwd_weight) at odd rows, widths and strides against 64 bits."""
import pytest
import torch

from rise_sdf_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("precision", ["fp32", "bf16"])
@pytest.mark.parametrize("n,K,N", [(1, 1, 9), (7, 33, 64), (8, 35, 10), (15, 64, 49), (16, 64, 64), (17, 96, 33), (1009, 35, 64), (4099, 128, 128),
                                   (40000, 84, 97), (5000, 128, 31)])
def test_weight_gradient(dev, n, K, N, precision):
    """Rows with gaps behind them: neither the gaps nor what lies behind the last row is read (it is NaN)."""
    g = torch.Generator(device=dev).manual_seed(n + K + N)
    lddz, ldx = N + 3, K + 5
    dz, x = (torch.full(((n + 20) * ld,), float("nan"), device=dev) for ld in (lddz, ldx))
    dzv, xv = dz[:n * lddz].view(n, lddz)[:, :N], x[:n * ldx].view(n, ldx)[:, :K]
    dzv.copy_(torch.randn(n, N, device=dev, generator=g))
    xv.copy_(torch.randn(n, K, device=dev, generator=g))
    dw, db = torch.zeros(N, K, device=dev), torch.zeros(N, device=dev)
    _lib.check(_lib.mlp_fn("rsdf_linear_bwd_weight", precision)(_lib.ptr(dz), lddz, _lib.ptr(x), ldx, n, K, N, _lib.ptr(dw), _lib.ptr(db),
                                                                _lib.stream_ptr()), "linear_bwd_weight")
    want, size = dzv.double().t() @ xv.double(), dzv.double().abs().t() @ xv.double().abs()
    # n products and as many sums in 32 bits, in any order (a matrix instruction: 16 at a time); six of nine partial products of the split
    # operands: 8 steps; one rounding of each operand to bf16: 2^-8 each
    e = (n + 64 + 8) * 2.0 ** -24 + (2.0 ** -7 + 2.0 ** -16 if precision == "bf16" else 0.0)
    assert bool(((dw.double() - want).abs() <= e * size).all())
    assert bool(((db.double() - dzv.double().sum(0)).abs() <= (n + 64) * 2.0 ** -24 * dzv.double().abs().sum(0)).all())
