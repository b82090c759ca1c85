"""Sizes at which a head of many classes takes each of its kernels, and what of its plan a size stands for (rsdf_class_head_plan)."""
import ctypes

from rise_sdf_amd import _lib

# rows, classes, features
FP32 = [(1025, 5003, 512), (1025, 10007, 200), (1300, 20011, 200), (2500, 10007, 512), (200, 10007, 515), (3001, 8193, 40), (257, 90001, 200),
        (513, 40001, 515), (300, 90001, 512), (5, 1300, 20000), (20, 50000, 1000)]
HALF = [(700, 40001, 200), (1025, 10007, 515), (2500, 33003, 333), (2500, 33003, 328), (6007, 10007, 200), (513, 16411, 512), (200, 10007, 1000),
        (1025, 12345, 40), (2049, 5003, 101), (3001, 40001, 200), (20, 66001, 1001), (40, 66001, 1001), (700, 66001, 1001)]
CASES = [(*s, 0) for s in FP32] + [(*s, t) for s in HALF for t in (1, 2)]


def plan(n, v, d, kind):
    out = (ctypes.c_int32 * 8)()
    assert _lib.lib().rsdf_class_head_plan(n, v, d, kind, out) == 0
    return dict(zip(("fwd", "bwd", "products", "fwd_pieces", "bwd_pieces", "split_dw", "split_dx", "direct"), out))
