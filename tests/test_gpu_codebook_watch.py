"""GPU: the timer and the debug log of the entry points see the calls of the C++ nodes too."""
import pytest
import torch

from rise_sdf_amd import _lib, ops
from rise_sdf_amd.loss import linear_cross_entropy, linear_distillation
from test_gpu_codebook import F32, head_case, lookup_case, teacher

pytestmark = pytest.mark.gpu


def passes(dev):
    ids, table, grad = lookup_case(dev, 300, 50, 48, F32, seed=1)
    x, w, y = head_case(dev, 70, 300, 48, F32, seed=2)
    tid, tl = teacher(dev, 70, 300, 3, seed=3)
    t, xr = table.requires_grad_(True), x.requires_grad_(True)
    out = [torch.autograd.grad(ops.embedding(ids, t), t, grad)[0]]
    for loss in (linear_cross_entropy(xr, w, y), linear_distillation(xr, w, tid, tl)):
        out += [loss.detach(), torch.autograd.grad(loss, xr)[0]]
    return out


NAMES = ["embedding_fwd", "embedding_bwd", "class_head_fwd", "class_head_fwd", "class_head_bwd", "class_head_bwd"]


def test_timer(dev):
    want = passes(dev)
    timer = _lib.KernelTimer()
    _lib.set_timer(timer)
    try:
        got = passes(dev)
    finally:
        _lib.set_timer(None)
    passes(dev)
    torch.cuda.synchronize()
    assert sorted(r[0] for r in timer.records) == sorted("rsdf_" + n for n in NAMES)
    s = timer.summary()
    assert all(s["rsdf_" + n]["ms"] > 0.0 for n in NAMES)
    assert s["rsdf_embedding_fwd"]["args"] == [(300, 50, 48, 0)] and s["rsdf_class_head_bwd"]["args"] == [(70, 300, 48, 0, 1), (70, 300, 48, 0, 3)]
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_debug_log(dev, tmp_path, monkeypatch):
    want = passes(dev)
    monkeypatch.setattr(_lib, "_DEBUG_SYNC", str(tmp_path / "log"))
    _lib._watch_nodes()
    try:
        got = passes(dev)
        with pytest.raises(_lib.RiseSdfHipError, match="row length"):
            ops.embedding(torch.zeros(1, dtype=torch.int64, device=dev), torch.zeros(1, (1 << 16) + 1, device=dev))
    finally:
        monkeypatch.setattr(_lib, "_DEBUG_SYNC", "")
        _lib._watch_nodes()
    passes(dev)
    assert sorted((tmp_path / "log").read_text().split()) == sorted(NAMES + ["embedding_fwd"])
    assert all(torch.equal(p, q) for p, q in zip(got, want))
