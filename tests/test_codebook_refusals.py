"""CPU: what the codebook operators refuse, and the limits their C entries check before any launch."""
import ctypes

import pytest
import torch

from rise_sdf_amd import Config, _lib, ops
from rise_sdf_amd.loss import linear_cross_entropy, linear_distillation

ERR = _lib.RiseSdfHipError


def test_lookup_refusals():
    ids, table = torch.zeros(4, dtype=torch.int64), torch.zeros(5, 3)
    with pytest.raises(ERR, match="device"):
        ops.embedding(ids, table)
    with pytest.raises(ERR, match="integer ids"):
        ops.embedding(ids.float(), table)
    with pytest.raises(ERR, match="float32"):
        ops.embedding(ids, table.double())
    with pytest.raises(ERR, match="padding_idx"):
        ops.embedding(ids, table, padding_idx=5)
    with pytest.raises(ERR, match="padding_idx"):
        ops.embedding(ids, table, padding_idx=-1)
    for bad in (torch.zeros(3), torch.zeros(0, 3), torch.zeros(3, 0), torch.zeros(2, 2, 2)):
        with pytest.raises(ERR, match="table"):
            ops.embedding(ids, bad)


def test_head_refusals():
    x, w, y = torch.zeros(4, 8), torch.zeros(10, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ERR, match="device"):
        linear_cross_entropy(x, w, y)
    with pytest.raises(ERR, match="one type"):
        linear_cross_entropy(x, w.half(), y)
    with pytest.raises(ERR, match="float32"):
        linear_cross_entropy(x.double(), w.double(), y)
    with pytest.raises(ERR, match="one target per row"):
        linear_cross_entropy(x, w, y[:3])
    with pytest.raises(ERR, match="features"):
        linear_cross_entropy(x, torch.zeros(10, 7), y)
    with pytest.raises(ERR, match="at least one"):
        linear_cross_entropy(x, torch.zeros(0, 8), y)
    with pytest.raises(ERR, match="reduction"):
        linear_cross_entropy(x, w, y, reduction="batchmean")
    with pytest.raises(ERR, match="integer ids"):
        linear_cross_entropy(x, w, y.float())
    ids, lg = torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3)
    with pytest.raises(ERR, match="device"):
        linear_distillation(x, w, ids, lg)
    with pytest.raises(ERR, match="ids and logits"):
        linear_distillation(x, w, ids, lg[:, :2])
    with pytest.raises(ERR, match="ids and logits"):
        linear_distillation(x, w, ids[:3], lg[:3])
    with pytest.raises(ERR, match="listed"):
        linear_distillation(x, w, ids[:, :0], lg[:, :0])
    with pytest.raises(ERR, match="floating"):
        linear_distillation(x, w, ids, ids)
    for t in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ERR, match="temperature"):
            linear_distillation(x, w, ids, lg, temperature=t)


def test_entry_points_check_before_they_launch():
    """Error codes and messages, no device needed: every call below is refused on the host."""
    l = _lib.lib()
    bad = [l.rsdf_embedding_fwd(None, 4, None, 0, 8, 0, 1.0, -1, None, None, None),
           l.rsdf_embedding_fwd(None, 4, None, 8, 8, 3, 1.0, -1, None, None, None),
           l.rsdf_embedding_bwd(None, 4, None, 8, 0, 0, 1.0, -1, None, None, 0, None),
           l.rsdf_embedding_bwd(None, 1000, None, 8, 8, 0, 1.0, -1, None, None, 100, None),        # workspace
           l.rsdf_class_head_fwd(None, None, 4, 8, 8, 0, None, None, 2, -100, 1.0, 0, None, None, None, None, None, None, None, 1 << 30, None),
           l.rsdf_class_head_fwd(None, None, 4, 8, 8, 0, None, None, 1, -100, 0.0, 0, None, None, None, None, None, None, None, 1 << 30, None),
           l.rsdf_class_head_fwd(None, None, 4, 8, 8, 0, None, None, 1, -100, 1.0, 3, None, None, None, None, None, None, None, 1 << 30, None),
           l.rsdf_class_head_fwd(None, None, 4, 8, 8, 0, None, None, 1, -100, 1.0, 0, None, None, None, None, None, None, None, 10, None),
           l.rsdf_class_head_fwd(ctypes.c_void_p(8), None, 4, 8, 8, 0, None, None, 1, -100, 1.0, 0, None, None, None, None, None, None, None, 1 << 30, None)]
    assert all(rc != 0 for rc in bad)
    assert l.rsdf_class_head_bwd(None, None, 4, 8, 8, 0, None, None, None, 1, 1.0, None, None, None, 0, ctypes.c_void_p(16), None, None, 10, None) != 0
    assert l.rsdf_class_head_workspace_bytes(0, 8, 8, 0, 0) == -1 and l.rsdf_class_head_workspace_bytes(4, 8, 1 << 20, 0, 0) == -1
    assert l.rsdf_embedding_bwd_workspace_bytes(-1, 8, 8) == -1


def test_workspace_does_not_grow_with_the_logits():
    size = _lib.lib().rsdf_class_head_workspace_bytes
    for dtype in (0, 1, 2):
        for n, v, d in ((4096, 131072, 512), (8192, 131072, 64), (256, 1 << 22, 64)):
            for p in (0, 3):
                b = int(size(n, v, d, dtype, p))
                # one piece (256 MiB) + packed codes (128 MiB) + split sums and statistics
                assert 0 < b < (1 << 30) + 64 * n * d * 4 + 64 * (32768 + 256) * d * 4, (n, v, d, dtype, p, b)


def test_embedding_encoding_on_the_cpu():
    from rise_sdf_amd.network_utils import get_encoding
    e = get_encoding(1, Config({"otype": "Embedding", "n_embeddings": 7, "n_features": 5, "padding_idx": 2}))
    assert e.n_output_dims == 5 and tuple(e.params.shape) == (7, 5) and not bool(e.params[2].any())
    assert list(e.state_dict()) == ["params"]
    with pytest.raises(NotImplementedError, match="Embedding"):
        get_encoding(3, Config({"otype": "Embedding", "n_embeddings": 7, "n_features": 5}))


def test_missing_nodes_fail_loudly(tmp_path, monkeypatch):
    monkeypatch.setattr(_lib, "_nodes", None)
    monkeypatch.setattr(_lib, "NODES_PATH", str(tmp_path / "nope.so"))
    with pytest.raises(ERR, match="missing"):
        _lib.nodes()


def test_nodes_load_and_report_errors_as_the_library_does():
    """Without a device: the nodes bind to the loaded library, and a refused size comes back as the framework's error."""
    n = _lib.nodes()
    ids, table = torch.zeros(2, dtype=torch.int64), torch.zeros(3, (1 << 16) + 1)
    with pytest.raises((ERR, RuntimeError)):
        n.embedding(ids, table, 1.0, -1, 0)


def test_temperatures_out_of_range():
    """T^2 and 1 / T have to stay far inside fp32."""
    x, w = torch.zeros(4, 8), torch.zeros(10, 8)
    ids, lg = torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3)
    for t in (1e-7, 2e6, 1e30):
        with pytest.raises(ERR, match="temperature"):
            linear_distillation(x, w, ids, lg, temperature=t)
    l = _lib.lib()
    for t in (0.0, 1e-7, 2e6, float("nan")):
        assert l.rsdf_class_head_fwd(None, None, 4, 8, 8, 0, None, None, 1, -100, t, 0, None, None, None, None, None, None, None, 1 << 30, None) != 0
