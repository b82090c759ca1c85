"""CPU: the sizes of codebook_plans reach every kernel of a head in every type, by what the library itself says of them."""
import ctypes

import pytest

from codebook_plans import CASES, plan
from rise_sdf_amd import _lib


@pytest.mark.parametrize("kind", [0, 1, 2])
def test_the_sizes_reach_every_kernel(kind):
    plans = [plan(*c) for c in CASES if c[3] == kind]
    seen = {(k, p[k]) for p in plans for k in ("fwd", "bwd", "products")}
    assert seen >= {("fwd", 32), ("fwd", 128), ("fwd", 256), ("bwd", 128), ("bwd", 256), ("products", 128), ("products", 256)}

    def some(**want):
        return any(all(p[k] >= v if k.endswith("pieces") or k.startswith("split") else p[k] == v for k, v in want.items()) for p in plans)
    # several pieces of the classes: behind each forward tile, and each pair of tiles of the backward
    for tile in (32, 128, 256):
        assert some(fwd=tile, fwd_pieces=2)
    assert some(bwd=256, products=256, bwd_pieces=2) and some(bwd=128, products=128, bwd_pieces=2)
    # products of large tiles that are cut over k and joined, and that are not
    assert some(products=256, split_dw=2, split_dx=2) and any(p["products"] == 256 and p["split_dw"] == 1 for p in plans)
    assert some(direct=0, products=256)
    if kind != 0:
        assert some(direct=1, fwd=256, bwd=256, products=256) and some(direct=1, bwd=256, products=256, bwd_pieces=2)


def test_plan_refusals():
    lib, out = _lib.lib(), (ctypes.c_int32 * 8)()
    for size in ((0, 8, 8, 0), (4, 0, 8, 0), (4, 8, 0, 0), (4, 8, 8, 3)):
        assert lib.rsdf_class_head_plan(*size, out) == 10001
    assert lib.rsdf_class_head_plan(4, 8, 8, 0, None) == 10001


@pytest.mark.parametrize("n,v,d", [(4096, 131072, 512), (4096, 32768, 512), (8192, 131072, 64), (256, 1 << 22, 64), (65536, 65536, 512), (1 << 18, 8192, 64),
                                   (1 << 20, 1000, 48), (1 << 24, 256, 64), (1, 53163, 697), (4096, 1000, 48)])
@pytest.mark.parametrize("kind", [0, 1, 2])
def test_workspace_is_the_sum_of_its_stated_terms(n, v, d, kind):
    size = _lib.lib().rsdf_class_head_workspace_bytes
    p, s = plan(n, v, d, kind), 6 if kind == 0 else 2
    rows, dp = -(-n // 256) * 256, -(-d // 64) * 64
    packed, mb = not p["direct"], 1 << 20
    x, w = rows * dp * s, max(128 * mb, 256 * dp * s)
    forward = 8 * n * -(-v // 128) + 4 * n + packed * (x + w) + 2048
    assert int(size(n, v, d, kind, 0)) <= forward
    piece = max(128 * mb, 256 * rows * s)
    classes = piece // (rows * s)
    dx = 4 * p["split_dx"] * n * dp
    dw = 4 * p["split_dw"] * classes * dp if p["split_dw"] > 1 else 0
    for which in (1, 2, 3):
        bound = piece + x + packed * w + (which & 1) * dx + (which >> 1) * dw + 4 * n + 2048
        assert int(size(n, v, d, kind, which)) <= bound
    # no logits: where they would be much, the backward's space is a part of them alone in 16 bits
    if n * v * 2 >= 1 << 30 and n <= 1 << 16:
        assert int(size(n, v, d, kind, 3)) < n * v * 2 // 4
