"""CPU: every refusal of the codebook operators' C entries by its code and message.  The pointers are not ones that a kernel could use, so nothing
here may reach a launch: a launch error has another code."""
import ctypes

import pytest

from rise_sdf_amd import _lib

EINVAL = 10001
P = ctypes.c_void_p(1 << 20)          # (never dereferenced)
BIG = 1 << 40

FWD = dict(ids=P, n=2000, table=P, v=8, d=8, dtype=0, scale=1.0, padding=-1, out=P, bad=None, stream=None)
BWD = dict(ids=P, n=2000, grad=P, v=8, d=8, dtype=0, scale=1.0, padding=-1, d_table=P, ws=P, ws_bytes=BIG, stream=None)
HEAD_FWD = dict(x=P, w=P, n=4, v=8, d=8, dtype=0, ids=P, logits=None, k=1, ignore=-100, temperature=1.0, reduction=1, loss=P, lse=P, count=P,
                q=None, z=None, bad=None, ws=P, ws_bytes=BIG, stream=None)
HEAD_BWD = dict(x=P, w=P, n=4, v=8, d=8, dtype=0, ids=P, q=None, z=None, k=1, temperature=1.0, lse=P, count=P, grad=P, per_row=0, dx=P, dw=P, ws=P,
                ws_bytes=BIG, stream=None)


def refused(name, base, message, **change):
    assert set(change) <= set(base)
    lib = _lib.lib()
    rc = getattr(lib, name)(*{**base, **change}.values())
    assert rc == EINVAL, (name, change, rc, lib.rsdf_last_error())
    assert message in lib.rsdf_last_error().decode(), (name, change, lib.rsdf_last_error())


@pytest.mark.parametrize("change,message", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(v=0), "rows in"), (dict(n=-1), "positions"), (dict(n=(1 << 30) + 1), "positions"),
    (dict(v=(1 << 30) + 1), "rows in"), (dict(d=0), "row length"), (dict(d=(1 << 16) + 1), "row length")])
def test_lookup_sizes(change, message):
    refused("rsdf_embedding_fwd", FWD, message, **change)
    refused("rsdf_embedding_bwd", BWD, message, **change)


def test_lookup_pointers():
    for name in ("ids", "table", "out"):
        refused("rsdf_embedding_fwd", FWD, "NULL", **{name: None})
    for n in (1, 1000, 2000):               # (few positions need no workspace, many do)
        for name in ("ids", "grad", "d_table"):
            refused("rsdf_embedding_bwd", BWD, "NULL", n=n, **{name: None})
    refused("rsdf_embedding_bwd", BWD, "NULL", n=0, d_table=None)
    need = _lib.lib().rsdf_embedding_bwd_workspace_bytes(2000, 8, 8)
    refused("rsdf_embedding_bwd", BWD, "workspace", ws_bytes=need - 1)
    refused("rsdf_embedding_bwd", BWD, "workspace", ws=None)
    refused("rsdf_embedding_bwd", BWD, "workspace", n=1000, v=20000, ws_bytes=100)
    assert _lib.lib().rsdf_embedding_fwd(None, 0, P, 8, 8, 0, 1.0, -1, None, None, None) == 0          # nothing to do


@pytest.mark.parametrize("change,message", [
    (dict(dtype=3), "dtype"), (dict(n=0), "rows must"), (dict(n=(1 << 24) + 1), "rows must"), (dict(v=0), "classes in"),
    (dict(v=(1 << 28) + 1), "classes in"), (dict(d=0), "features"), (dict(d=(1 << 15) + 1), "features"),
    (dict(x=ctypes.c_void_p((1 << 20) + 8)), "16-byte"), (dict(w=ctypes.c_void_p((1 << 20) + 2)), "16-byte"),
    (dict(ws_bytes=10), "workspace"), (dict(ws=None), "workspace")])
def test_head_sizes(change, message):
    refused("rsdf_class_head_fwd", HEAD_FWD, message, **change)
    refused("rsdf_class_head_bwd", HEAD_BWD, message, **change)


def test_head_pointers_and_options():
    for name in ("x", "w", "ids", "loss", "lse", "count"):
        refused("rsdf_class_head_fwd", HEAD_FWD, "NULL", **{name: None})
    for name in ("x", "w", "ids", "lse", "grad"):
        refused("rsdf_class_head_bwd", HEAD_BWD, "NULL", **{name: None})
    refused("rsdf_class_head_fwd", HEAD_FWD, "labels need k = 1", k=2)
    refused("rsdf_class_head_fwd", HEAD_FWD, "listed classes", k=0)
    refused("rsdf_class_head_fwd", HEAD_FWD, "listed classes", k=4097, logits=P, q=P, z=P)
    refused("rsdf_class_head_fwd", HEAD_FWD, "a teacher needs", logits=P, q=P)
    refused("rsdf_class_head_fwd", HEAD_FWD, "reduction", reduction=3)
    for t in (0.0, -1.0, 1e-7, 2e6, float("inf"), float("nan")):
        refused("rsdf_class_head_fwd", HEAD_FWD, "temperature", temperature=t)
    refused("rsdf_class_head_bwd", HEAD_BWD, "a teacher needs", q=P)
    refused("rsdf_class_head_bwd", HEAD_BWD, "labels need k = 1", k=2)
    refused("rsdf_class_head_bwd", HEAD_BWD, "dx and dw", dx=ctypes.c_void_p((1 << 20) + 4))
    refused("rsdf_class_head_bwd", HEAD_BWD, "dx and dw", dw=ctypes.c_void_p((1 << 20) + 8))
    lib = _lib.lib()
    assert lib.rsdf_class_head_bwd(*{**HEAD_BWD, "dx": None, "dw": None, "ws": None}.values()) == 0      # nothing to do
    for size in ((0, 8, 8, 0, 0), (4, 8, 1 << 20, 0, 0), (4, 8, 8, 5, 3)):
        assert lib.rsdf_class_head_workspace_bytes(*size) == -1
    for size in ((-1, 8, 8), (4, 0, 8), (4, 8, 0)):
        assert lib.rsdf_embedding_bwd_workspace_bytes(*size) == -1
