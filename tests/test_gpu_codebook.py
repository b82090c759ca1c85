"""GPU tests of the codebook operators (ops.embedding, loss.linear_cross_entropy, loss.linear_distillation) against plain 64-bit
forms; the bounds are derived in codebook_reference.py."""
import pytest
import torch

import codebook_reference as ref
from rise_sdf_amd import _lib, ops
from rise_sdf_amd.loss import linear_cross_entropy, linear_distillation

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


# ---- embedding ----------------------------------------------------------------------------------------------------------------
def lookup_case(dev, n, v, d, dtype, kind="uniform", seed=0):
    g = gen(dev, seed)
    if kind == "same":
        ids = torch.full((n,), v // 2, dtype=torch.int64, device=dev)
    elif kind == "zipf":
        u = torch.rand(n, device=dev, generator=g, dtype=torch.float64)
        ids = ((v + 1.0) ** u - 1.0).long().clamp_(0, v - 1)
    else:
        ids = torch.randint(0, v, (n,), device=dev, generator=g)
    table = (torch.randn(v, d, device=dev, generator=g) * 0.5).to(dtype)
    grad = torch.randn(n, d, device=dev, generator=g).to(dtype)
    return ids, table, grad


def check_lookup(ids, table, grad, scale, padding):
    t = table.clone().requires_grad_(True)
    out = ops.embedding(ids, t, scale=scale, padding_idx=padding)
    (dt,) = torch.autograd.grad(out, t, grad.reshape(out.shape))
    want, bound, d_want, d_bound = ref.embedding(ids, table, scale, padding, grad)
    assert out.dtype == table.dtype and dt.dtype == table.dtype and out.shape == (*ids.shape, table.shape[1])
    ref.assert_within("out", out.detach().reshape(-1, table.shape[1]), want, bound)
    ref.assert_within("d_table", dt, d_want, d_bound)
    return out.detach(), dt


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,d,kind", [
    (1, 1, 1, "uniform"), (1, 1000, 48, "uniform"), (2, 3, 3, "same"), (63, 255, 64, "uniform"), (64, 256, 100, "uniform"),
    (65, 257, 7, "zipf"), (257, 70000, 33, "uniform"), (1025, 5, 256, "uniform"), (4097, 1000, 48, "zipf"),
    (5000, 300, 520, "zipf"), (3000, 77, 1030, "same"), (40001, 4999, 96, "zipf"), (70001, 66000, 12, "uniform"),
    (100000, 2, 16, "same")])
def test_lookup_and_gradient(dev, n, v, d, kind, dtype):
    ids, table, grad = lookup_case(dev, n, v, d, dtype, kind, seed=n + v)
    check_lookup(ids, table, grad, d ** 0.5, None)
    if v > 2:
        check_lookup(ids, table, grad, 1.0, v // 2)


@pytest.mark.parametrize("dtype", TYPES)
def test_lookup_of_nothing(dev, dtype):
    ids, table, grad = lookup_case(dev, 0, 300, 20, dtype)
    out, dt = check_lookup(ids, table, grad, 1.0, None)
    assert out.shape == (0, 20) and not bool(dt.any())


@pytest.mark.parametrize("id_type", [torch.int32, torch.int16, torch.uint8])
def test_lookup_shapes_strides_and_id_types(dev, id_type):
    ids, table, grad = lookup_case(dev, 600, 250, 24, F32, seed=3)
    ids2 = ids.reshape(20, 30).to(id_type).t()                                # a transposed view
    wide = torch.zeros(250, 50, device=dev)
    wide[:, 1:25] = table
    check_lookup(ids2, wide[:, 1:25], grad, 0.25, 0)                          # rows with gaps, off 16-byte alignment
    t = table.clone().requires_grad_(True)
    one = torch.ones(24, device=dev)
    (dt,) = torch.autograd.grad(ops.embedding(ids, t), t, one.expand(600, 24))   # a broadcast gradient
    assert torch.equal(dt, torch.bincount(ids, minlength=250).float()[:, None].expand(250, 24))


def test_lookup_unaligned_table(dev):
    """A contiguous table that starts anywhere: every vector width."""
    for off in (1, 2, 3, 4, 8):
        for dtype in TYPES:
            flat = torch.randn(40 * 16 + 16, device=dev, generator=gen(dev, off)).to(dtype)
            table = flat[off:off + 40 * 16].view(40, 16)
            ids, _, grad = lookup_case(dev, 100, 40, 16, dtype, seed=off)
            check_lookup(ids, table, grad, 2.0, None)


def test_lookup_outside_ids(dev):
    _lib.poll_status(dev)
    ids, table, grad = lookup_case(dev, 500, 100, 40, F32, seed=9)
    ids[[3, 77, 78, 400]] = torch.tensor([-1, 100, 1 << 40, -(1 << 63)], device=dev)
    out, dt = check_lookup(ids, table, grad, 1.0, 5)
    assert bool(torch.isnan(out[[3, 77, 78, 400]]).all()) and bool(torch.isfinite(dt).all())
    with pytest.raises(_lib.RiseSdfHipError, match="outside"):
        _lib.poll_status(dev)
    _lib.poll_status(dev)                                                     # reported once


def test_lookup_nonfinite_rows_stay_where_they_are(dev):
    ids, table, grad = lookup_case(dev, 300, 50, 8, F32, seed=1)
    grad[ids == 7] = float("inf")
    grad[ids == 0] = float("nan")                                             # padding: masked
    table[9] = float("-inf")
    out, dt = check_lookup(ids, table, grad, 1.0, 0)
    assert not bool(out[ids == 0].any()) and not bool(dt[0].any()) and bool(torch.isinf(dt[7]).all())


def test_lookup_repeats_bit_for_bit(dev):
    ids, table, grad = lookup_case(dev, 50000, 300, 64, F32, "zipf", seed=4)
    a, b = check_lookup(ids, table, grad, 1.0, None), check_lookup(ids, table, grad, 1.0, None)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_lookup_gradient_against_differences(dev):
    """The lookup is linear in the table: a difference quotient is exact up to rounding."""
    ids, table, grad = lookup_case(dev, 400, 60, 16, F32, "zipf", seed=5)
    _, dt = check_lookup(ids, table, grad, 1.5, 2)
    step = torch.randn(60, 16, device=dev, generator=gen(dev, 6))
    hi = (ops.embedding(ids, table + step, 1.5, 2).double() * grad.double()).sum()
    lo = (ops.embedding(ids, table - step, 1.5, 2).double() * grad.double()).sum()
    got, want = float((dt.double() * step.double()).sum()), float(hi - lo) / 2
    size = float((ops.embedding(ids, table.abs() + step.abs(), 1.5, 2).double() * grad.double().abs()).sum())
    assert abs(got - want) <= 100 * ref.E32 * size        # up to ~60 positions per id, four roundings each way


# ---- losses ---------------------------------------------------------------------------------------------------------------------
def head_case(dev, n, v, d, dtype, seed=0, lean=2.0):
    g = gen(dev, seed)
    w = torch.randn(v, d, device=dev, generator=g) * (2.0 / d ** 0.5)
    target = torch.randint(0, v, (n,), device=dev, generator=g)
    x = torch.randn(n, d, device=dev, generator=g) + lean * torch.rand(n, 1, device=dev, generator=g) * w[target]
    return x.to(dtype), w.to(dtype), target


def teacher(dev, n, v, k, seed=0, missing=0.2):
    g = gen(dev, seed + 1000)
    ids = torch.randint(0, v, (n, k), device=dev, generator=g)               # a class may be listed twice
    logits = torch.randn(n, k, device=dev, generator=g) * 2
    drop = torch.rand(n, k, device=dev, generator=g) < missing
    drop |= torch.rand(n, 1, device=dev, generator=g) < missing
    return torch.where(drop, torch.full_like(ids, -1), ids), logits


def check_head(x, w, ids, logits=None, *, ignore=-100, temperature=1.0, reduction="mean", grad=None, what=(True, True)):
    xr, wr = x.detach().clone().requires_grad_(what[0]), w.detach().clone().requires_grad_(what[1])
    if logits is None:
        loss = linear_cross_entropy(xr, wr, ids, ignore_index=ignore, reduction=reduction)
        rid = ids[:, None]
    else:
        loss = linear_distillation(xr, wr, ids, logits, temperature=temperature, reduction=reduction)
        rid = ids
    if grad is None:
        grad = torch.ones_like(loss)
    leaves = [t for t in (xr, wr) if t.requires_grad]
    grads = list(torch.autograd.grad(loss, leaves, grad)) if leaves else []
    want = ref.head(x, w, rid, logits, ignore, temperature, reduction, grad)
    assert loss.dtype == F32
    ref.assert_within("loss", loss.detach(), want["loss"], want["e_loss"])
    dx = dw = None
    if what[0]:
        dx = grads.pop(0)
        assert dx.dtype == x.dtype
        ref.assert_within("dx", dx, want["dx"], want["e_dx"])
        assert not bool(dx[~want["alive"]].any())
    if what[1]:
        dw = grads.pop(0)
        assert dw.dtype == w.dtype
        ref.assert_within("dw", dw, want["dw"], want["e_dw"])
    return loss.detach(), dx, dw


SIZES = [(1, 1, 1), (1, 2, 3), (3, 5, 7), (1, 1000, 48), (2, 300, 512), (31, 257, 64), (32, 256, 32), (33, 255, 96),
         (64, 1000, 33), (127, 129, 128), (128, 256, 160), (129, 1003, 100), (257, 513, 520), (300, 2000, 256),
         (1000, 40, 17), (5000, 10, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,d", SIZES)
def test_cross_entropy(dev, n, v, d, dtype):
    x, w, y = head_case(dev, n, v, d, dtype, seed=n + v + d)
    check_head(x, w, y)
    y[::3] = -100
    check_head(x, w, y, reduction="sum")
    y[:] = torch.where(y == -100, torch.full_like(y, v + 5), y)               # an ignored label may lie anywhere
    g = torch.randn(n, device=dev, generator=gen(dev, 2))
    g[n // 2:n // 2 + 1] = 0.0
    check_head(x, w, y, ignore=v + 5, reduction="none", grad=g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,d", SIZES)
def test_distillation(dev, n, v, d, dtype):
    x, w, _ = head_case(dev, n, v, d, dtype, seed=n + v + d)
    for k, t, red in ((1, 1.0, "mean"), (5, 2.0, "none"), (33, 0.5, "sum")):
        ids, logits = teacher(dev, n, v, k, seed=n + k)
        g = torch.rand(n, device=dev, generator=gen(dev, 3)) if red == "none" else None
        check_head(x, w, ids, logits, temperature=t, reduction=red, grad=g)


@pytest.mark.parametrize("n,v,d,dtype", [(2100, 60100, 64, BF16), (1000, 44003, 40, F32), (4096, 33000, 32, F16)])
def test_more_than_one_piece_of_classes(dev, n, v, d, dtype):
    x, w, y = head_case(dev, n, v, d, dtype, seed=7)
    y[5:50] = -100
    y[:4] = torch.tensor([0, v - 1, v - 2, 32768], device=dev)
    check_head(x, w, y)
    ids, logits = teacher(dev, n, v, 3, seed=8)
    check_head(x, w, ids, logits, temperature=2.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("need", [(True, False), (False, True), (False, False)])
def test_only_what_is_asked_for(dev, dtype, need):
    x, w, y = head_case(dev, 70, 300, 40, dtype, seed=1)
    check_head(x, w, y, what=need)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_take_part_in_nothing(dev, dtype):
    x, w, y = head_case(dev, 150, 500, 64, dtype, seed=2)
    dead = torch.arange(0, 150, 4, device=dev)
    y[dead] = -100
    a = check_head(x, w, y)
    x2 = x.clone()
    x2[dead] = torch.tensor([float("nan"), float("inf")] * 32, device=dev).to(dtype)
    xr, wr = x2.requires_grad_(True), w.clone().requires_grad_(True)
    loss = linear_cross_entropy(xr, wr, y)
    dx, dw = torch.autograd.grad(loss, (xr, wr))
    assert torch.equal(loss.detach(), a[0]) and torch.equal(dx, a[1]) and torch.equal(dw, a[2])
    # nobody takes part
    for red, shape in (("mean", ()), ("sum", ()), ("none", (150,))):
        xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = linear_cross_entropy(xr, wr, torch.full_like(y, -100), reduction=red)
        dx, dw = torch.autograd.grad(loss.sum(), (xr, wr))
        assert loss.shape == shape and not bool(loss.any()) and not bool(dx.any()) and not bool(dw.any())
    ids, logits = teacher(dev, 150, 500, 4, seed=3)
    ids[::2] = -1
    logits[ids < 0] = float("nan")                                            # masked places hold anything
    logits[1] = float("-inf")                                                 # listed, but without weight
    ids[1] = 3
    xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = linear_distillation(xr, wr, ids, logits, temperature=2.0, reduction="none")
    dx, dw = torch.autograd.grad(loss.sum(), (xr, wr))
    assert bool(torch.isfinite(loss).all()) and not bool(loss[::2].any()) and not bool(dx[::2].any()) and not bool(loss[1])
    assert bool(torch.isfinite(dw).all())


def test_teacher_logits_at_the_ends_of_their_type(dev):
    x, w, _ = head_case(dev, 6, 300, 32, F32, seed=4)
    ids, _ = teacher(dev, 6, 300, 4, missing=0.0)
    low, high = torch.finfo(F32).min, torch.finfo(F32).max
    logits = torch.tensor([[low] * 4, [low, 0, 0, 1], [high] * 4, [high, low, 0, 0], [float("-inf"), 0, 1, 2], [5, 5, low, low]],
                          device=dev)
    check_head(x, w, ids, logits, reduction="none", grad=torch.ones(6, device=dev))
    check_head(x, w, ids, logits, temperature=0.5, reduction="none", grad=torch.ones(6, device=dev))


@pytest.mark.parametrize("dtype", TYPES)
def test_large_logits(dev, dtype):
    """Logits of some hundreds: the softmax is a maximum, exponentials of their differences underflow."""
    x, w, y = head_case(dev, 64, 700, 64, dtype, seed=5)
    check_head((x.float() * 60).to(dtype), w, y)
    check_head((x.float() * 60).to(dtype), w, y, reduction="none", grad=torch.rand(64, device=dev, generator=gen(dev, 1)))


def test_infinite_and_nan_rows_stay_in_their_loss(dev):
    x, w, y = head_case(dev, 40, 300, 32, F32, seed=6)
    x[3, 5], x[7, 0] = float("nan"), float("inf")
    loss = linear_cross_entropy(x, w, y, reduction="none")
    bad = torch.isnan(loss)
    assert bad.nonzero().reshape(-1).tolist() == [3, 7]
    keep = ~bad
    want = ref.head(x[keep], w, y[keep][:, None], None, -100, 1.0, "none")
    ref.assert_within("loss", loss[keep], want["loss"], want["e_loss"])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_classes_of_minus_infinity(dev, dtype):
    """A class whose every logit is -inf has probability 0; whole tiles of them too.  (fp32 operands are split: finite ones only.)"""
    x, w, y = head_case(dev, 20, 1200, 32, dtype, seed=8)
    x = x.abs() + 0.1
    w[256:600] = float("-inf")
    y = y % 256
    loss = linear_cross_entropy(x, w, y, reduction="none")
    keep = torch.cat([w[:256], w[600:]])
    want = ref.head(x, keep, y[:, None], None, -100, 1.0, "none")
    ref.assert_within("loss", loss, want["loss"], want["e_loss"])


@pytest.mark.parametrize("dtype", TYPES)
def test_labels_outside_the_head(dev, dtype):
    _lib.poll_status(dev)
    x, w, y = head_case(dev, 50, 200, 48, dtype, seed=9)
    ok = y.clone()
    y[[4, 9, 30]] = torch.tensor([200, -1, 1 << 50], device=dev)
    xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = linear_cross_entropy(xr, wr, y, reduction="none")
    dx, dw = torch.autograd.grad(loss, (xr, wr), torch.ones(50, device=dev))
    assert torch.isnan(loss).nonzero().reshape(-1).tolist() == [4, 9, 30]
    ok[[4, 9, 30]] = -100
    a = check_head(x, w, ok, reduction="none", grad=torch.ones(50, device=dev))
    assert torch.equal(dx, a[1]) and torch.equal(dw, a[2])
    with pytest.raises(_lib.RiseSdfHipError, match="outside"):
        _lib.poll_status(dev)
    ids, logits = teacher(dev, 50, 200, 4, missing=0.0)
    ids[7, 2] = 200
    loss = linear_distillation(x, w, ids, logits, reduction="none")
    assert torch.isnan(loss).nonzero().reshape(-1).tolist() == [7]
    with pytest.raises(_lib.RiseSdfHipError, match="outside"):
        _lib.poll_status(dev)


@pytest.mark.parametrize("dtype", TYPES)
def test_head_shapes_strides_alignment(dev, dtype):
    x, w, y = head_case(dev, 60, 130, 64, dtype, seed=10)
    a = check_head(x, w, y)
    xt, wt = x.t().contiguous().t(), w.t().contiguous().t()                   # column-major
    b = linear_cross_entropy(xt, wt, y)
    flat = torch.zeros(60 * 64 + 3, dtype=dtype, device=dev)
    flat[3:] = x.reshape(-1)
    c = linear_cross_entropy(flat[3:].view(60, 64), w, y.to(torch.int32))     # off 16-byte alignment
    e = linear_cross_entropy(x.view(3, 20, 64), w, y.view(3, 20))
    per = linear_cross_entropy(x.view(3, 20, 64), w, y.view(3, 20), reduction="none")
    assert per.shape == (3, 20)
    for other in (b, c, e):
        assert torch.equal(a[0], other)
    big = torch.zeros(60, 100, dtype=dtype, device=dev)
    big[:, 10:74] = x
    assert torch.equal(a[0], linear_cross_entropy(big[:, 10:74], w, y))
    xr = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(linear_cross_entropy(xr[:1].expand(60, 64), w, y), xr)   # a broadcast input: its rows' sum
    want = ref.head(x[:1].expand(60, 64), w, y[:, None], None, -100, 1.0, "mean", torch.ones((), device=dev))
    bound = want["e_dx"].sum(0) + 60 * ref.half_step(dtype) * want["dx"].abs().sum(0)     # torch's own sum in the input's type
    ref.assert_within("dx", dx[0], want["dx"].sum(0), bound)


def test_head_without_rows(dev):
    w = torch.randn(30, 16, device=dev, requires_grad=True)
    x = torch.randn(0, 16, device=dev, requires_grad=True)
    y = torch.zeros(0, dtype=torch.int64, device=dev)
    for red in ("mean", "sum", "none"):
        loss = linear_cross_entropy(x, w, y, reduction=red)
        assert loss.shape == ((0,) if red == "none" else ()) and not bool(loss.any())
        dx, dw = torch.autograd.grad(loss.sum(), (x, w))
        assert dx.shape == (0, 16) and not bool(dw.any())
    loss = linear_distillation(x, w, torch.zeros(0, 3, dtype=torch.int64, device=dev), torch.zeros(0, 3, device=dev))
    assert float(loss) == 0.0


@pytest.mark.parametrize("dtype", TYPES)
def test_losses_repeat_bit_for_bit(dev, dtype):
    x, w, y = head_case(dev, 700, 3000 + 11, 96, dtype, seed=11)
    ids, logits = teacher(dev, 700, 3011, 7)
    for args in ((y, None), (ids, logits)):
        runs = [check_head(x, w, *args) for _ in range(2)]
        assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_gradients_against_differences(dev):
    """Central differences of the loss itself along one direction: an error of h^2 / 6 times the third derivative (|d^3| <=
    the third central moment of the logits' change, below 8 max|change|^3) and the loss's own error over h."""
    x, w, y = head_case(dev, 24, 90, 32, F32, seed=12)
    y[3] = -100
    ids, logits = teacher(dev, 24, 90, 5)
    h = 1.0 / 64
    for args in ((y, None), (ids, logits)):
        _, dx, dw = check_head(x, w, *args, reduction="sum")
        sx, sw = (torch.randn(t.shape, device=dev, generator=gen(dev, 13)) * 0.1 for t in (x, w))

        def loss(s):
            a, b = (x + s * sx), (w + s * sw)
            out = linear_cross_entropy(a, b, y, reduction="sum") if args[1] is None else \
                linear_distillation(a, b, ids, logits, reduction="sum")
            rid = y[:, None] if args[1] is None else ids
            return float(out), float(ref.head(a, b, rid, args[1], -100, 1.0, "sum")["e_loss"])
        (hi, e1), (lo, e2) = loss(h), loss(-h)
        got = float((dx.double() * sx.double()).sum() + (dw.double() * sw.double()).sum())
        change = float((sx.double() @ w.double().t()).abs().max() + (x.double() @ sw.double().t()).abs().max()) + 0.1
        bound = (e1 + e2) / (2 * h) + 24 * h * h * 8 * (change ** 3 + change) + 1e-5
        assert abs((hi - lo) / (2 * h) - got) <= bound, (args[1] is None, got, (hi - lo) / (2 * h), bound)


# ---- streams and graphs ----------------------------------------------------------------------------------------------------------
def test_on_another_stream(dev):
    ids, table, grad = lookup_case(dev, 3000, 200, 32, F32, "zipf", seed=20)
    x, w, y = head_case(dev, 300, 900, 48, BF16, seed=21)
    a, b = check_lookup(ids, table, grad, 1.0, None), check_head(x, w, y)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c, e = check_lookup(ids, table, grad, 1.0, None), check_head(x, w, y)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a + b, c + e))


def test_captured_training_passes(dev):
    """Two graphs, forward and backward, replayed with new inputs between eager work; each replay against the eager result."""
    ids, table, grad = lookup_case(dev, 4000, 300, 48, F32, "zipf", seed=22)
    x, w, y = head_case(dev, 300, 1100, 64, BF16, seed=23)
    tid, tl = teacher(dev, 300, 1100, 6)

    def lookup():
        t = table.detach().requires_grad_(True)
        out = ops.embedding(ids, t, 1.5, 0)
        return out.detach(), torch.autograd.grad(out, t, grad)[0]

    def head():
        xr, wr = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        a = linear_cross_entropy(xr, wr, y)
        b = linear_distillation(xr, wr, tid, tl, temperature=2.0, reduction="sum")
        return (a.detach(), b.detach(), *torch.autograd.grad(a + b, (xr, wr)))

    graphs = []
    for fn in (lookup, head):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fn()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = fn()
        graphs.append((g, out, fn))
    for k in range(4):
        gk = gen(dev, 30 + k)
        ids.copy_(torch.randint(0, 300, (4000,), device=dev, generator=gk))
        grad.copy_(torch.randn(grad.shape, device=dev, generator=gk))
        x.copy_(torch.randn(x.shape, device=dev, generator=gk))
        y.copy_(torch.randint(0, 1100, (300,), device=dev, generator=gk))
        y[k::5] = -100
        for g, out, fn in graphs:
            want = fn()
            torch.cuda.synchronize()
            g.replay()
            assert all(torch.equal(p, q) for p, q in zip(out, want)), k
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, want)), k


# ---- together --------------------------------------------------------------------------------------------------------------------
def test_codes_through_a_network_into_both_losses(dev):
    """A tied codebook as a label field uses it: codes looked up, a VanillaMLP on top of them, the result scored against the
    same codes with labels and a teacher; every gradient against the same chain in 64 bits."""
    from rise_sdf_amd.network_utils import get_encoding_with_network
    from rise_sdf_amd import Config
    torch.manual_seed(0)
    V, D, n = 211, 48, 400
    field = get_encoding_with_network(
        1, D, Config({"otype": "Embedding", "n_embeddings": V, "n_features": D, "scale": 2.0, "padding_idx": 0}),
        Config({"otype": "VanillaMLP", "n_neurons": 64, "n_hidden_layers": 2, "activation": "ReLU"})).to(dev)
    codes = field.encoding.params
    with torch.no_grad():
        codes.copy_(torch.randn(V, D, device=dev, generator=gen(dev, 1)) * 0.3)
    ids = torch.randint(0, V, (n,), device=dev, generator=gen(dev, 2))
    y = torch.randint(0, V, (n,), device=dev, generator=gen(dev, 3))
    y[::7] = -100
    tid, tl = teacher(dev, n, V, 5)
    feats = field(ids)
    loss = linear_cross_entropy(feats, codes, y) + 0.5 * linear_distillation(feats, codes, tid, tl, temperature=2.0)
    loss.backward()
    # the chain in 64 bits
    cd = codes.detach().double().requires_grad_(True)
    wb = [(w.detach().double(), b.detach().double().requires_grad_(True)) for w, b in field.network.effective_weights()]
    h = cd[ids] * 2.0 * (ids != 0)[:, None]
    for i, (w, b) in enumerate(wb):
        w.requires_grad_(True)
        h = h @ w.t() + b
        if i < len(wb) - 1:
            h = torch.relu(h)
    logits = h @ cd.t()
    want = torch.nn.functional.cross_entropy(logits, y, ignore_index=-100)
    alive = (tid >= 0).any(1)
    q = torch.where(tid >= 0, tl.double() / 2.0, torch.full_like(tl, float("-inf"), dtype=torch.float64))[alive].softmax(1)
    lp = torch.gather(torch.log_softmax(logits[alive] / 2.0, 1), 1, tid[alive].clamp(min=0))
    kd = torch.where(q > 0, torch.special.xlogy(q, q) - q * lp, torch.zeros_like(q)).sum() * 4.0 / alive.sum()
    want = want + 0.5 * kd
    want.backward()
    # three fp32-equivalent layers of at most 64 terms, then the bounds of the losses: 1e-5 of the largest entry is
    # (3 * 64 + 4 * 40 + V / 16) e, with e = 2^-24, rounded up
    def close(got, exact, tol=1e-5 * 4):
        assert float((got.double() - exact).abs().max()) <= tol * float(exact.abs().max())
    close(loss.detach(), want.detach())
    close(codes.grad, cd.grad)
    for m, (w, b) in zip([m for m in field.network.layers if isinstance(m, torch.nn.Linear)], wb):
        close(m.weight.grad, w.grad)
        close(m.bias.grad, b.grad)


def test_second_derivatives_are_refused(dev):
    ids, table, _ = lookup_case(dev, 20, 10, 4, F32)
    x, w, y = head_case(dev, 20, 30, 8, F32)
    for out, leaf in ((ops.embedding(ids, table.requires_grad_(True)).square().sum(), table),
                      (linear_cross_entropy(x.requires_grad_(True), w, y), x)):
        (g,) = torch.autograd.grad(out, leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated twice"):
            g.square().sum().backward()


def test_saved_tensors_changed_in_place_are_noticed(dev):
    x, w, y = head_case(dev, 20, 30, 8, F32)
    w.requires_grad_(True)
    loss = linear_cross_entropy(x, w, y)
    with torch.no_grad():
        w.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
