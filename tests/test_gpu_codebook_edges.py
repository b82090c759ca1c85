"""GPU tests of the codebook operators where their documentation allows more than a usual call makes: long rows, many rows, many
listed classes, tables beyond 2^32 elements, weights that are not finite, gradients of any layout, several host threads, passes
captured from real leaves, and the memory around every result.  Bounds as in codebook_reference.py."""
import threading

import pytest
import torch

import codebook_reference as ref
from rise_sdf_amd import _lib, ops
from rise_sdf_amd.loss import linear_cross_entropy, linear_distillation
from test_gpu_codebook import BF16, F16, F32, TYPES, check_head, check_lookup, gen, head_case, lookup_case, teacher

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,v,d,dtype", [
    (2100, 30000, 200, BF16), (1030, 66000, 328, F16), (1500, 50000, 77, F16), (1025, 40000, 45, F32),      # alternating groups
    (20001, 50, 24, BF16), (20001, 50, 23, F32), (70001, 3, 8, F16),                                         # many rows
    (5, 70, 5001, BF16), (300, 520, 2104, F16), (40, 300, 2047, F32), (3, 40, 32768, BF16)])                 # long rows
def test_head_sizes(dev, n, v, d, dtype):
    x, w, y = head_case(dev, n, v, d, dtype, seed=40)
    y[::9] = -100
    check_head(x, w, y)
    ids, logits = teacher(dev, n, v, 9, seed=41)
    check_head(x, w, ids, logits, temperature=2.0, reduction="none", grad=torch.rand(n, device=dev, generator=gen(dev, 42)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,k", [(3, 40, 4096), (700, 90, 130), (4100, 33, 64), (5000, 200, 20)])
def test_many_listed_classes(dev, n, v, k, dtype):
    """More entries than classes: every class listed many times."""
    x, w, _ = head_case(dev, n, v, 37, dtype, seed=43)
    ids, logits = teacher(dev, n, v, k, seed=44)
    check_head(x, w, ids, logits, temperature=2.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [1, 2, 3, 5, 9, 15, 17, 31, 101, 250])
def test_lookup_of_odd_rows(dev, d, dtype):
    for n, v in ((300, 50), (3000, 700), (60000, 300)):
        ids, table, grad = lookup_case(dev, n, v, d, dtype, "zipf", seed=d)
        check_lookup(ids, table, grad, 0.75, 1)


def test_table_beyond_32_bit_offsets(dev):
    """2^26 + 5 codes of 72 fp16: 9.7 GB, more than 2^32 elements."""
    v, d, n = (1 << 26) + 5, 72, 1000
    table = torch.zeros(v, d, dtype=F16, device=dev)
    ids = torch.randint(0, v, (n,), device=dev, generator=gen(dev, 45))
    ids[:4] = torch.tensor([0, v - 1, v - 2, v - 1], device=dev)
    rows, at = torch.unique(ids, return_inverse=True)
    small = torch.randn(rows.numel(), d, device=dev, generator=gen(dev, 46)).to(F16)
    table[rows] = small
    grad = torch.randn(n, d, device=dev, generator=gen(dev, 47)).to(F16)
    table.requires_grad_(True)
    out = ops.embedding(ids, table, scale=2.0)
    (dt,) = torch.autograd.grad(out, table, grad)
    want, bound, d_want, d_bound = ref.embedding(at, small, 2.0, None, grad)
    ref.assert_within("out", out.detach(), want, bound)
    ref.assert_within("d_table", dt[rows], d_want, d_bound)
    dt[rows] = 0.0
    assert not any(bool(part.any()) for part in dt.split(1 << 23))


def test_head_beyond_32_bit_offsets(dev):
    """2^23 + 2^20 + 3 classes of 512 bf16: more than 2^32 elements.  All but the last three codes are zero, so their logits are 0 and the
    sums are known in closed form."""
    v, d, n = (1 << 23) + (1 << 20) + 3, 512, 4
    x = torch.randn(n, d, device=dev, generator=gen(dev, 48)).to(BF16).requires_grad_(True)
    w = torch.zeros(v, d, dtype=BF16, device=dev)
    w[-3:] = (torch.randn(3, d, device=dev, generator=gen(dev, 49)) * 0.3).to(BF16)
    w.requires_grad_(True)
    y = torch.tensor([v - 1, v - 2, 0, -100], device=dev)
    loss = linear_cross_entropy(x, w, y, reduction="sum")
    dx, dw = torch.autograd.grad(loss, (x, w))
    xd, wd = x.detach().double(), w[-3:].detach().double()
    z = torch.cat([torch.zeros(n, 1, device=dev, dtype=torch.float64), xd @ wd.t()], 1)       # class 0 for all the zero codes
    many = torch.tensor([float(v - 3), 1.0, 1.0, 1.0], device=dev, dtype=torch.float64)
    lse = torch.logsumexp(z + many.log(), 1)
    p = torch.exp(z - lse[:, None])                                                           # of one class
    at = torch.tensor([3, 2, 0], device=dev)
    want = (lse[:3] - z[:3].gather(1, at[:, None])[:, 0]).sum()
    mag = (xd.abs() @ wd.abs().t()).max()
    # a logit: (2 (D / 32 + 40) + D) steps of its terms; the sums over 36868 tiles: (300 + V / 8192) steps
    e_z = (2 * (d / 32 + 40) + d) * ref.E32 * mag
    e_l = e_z + (300 + v / 8192 + 8 * float(z.abs().max()) + 64) * ref.E32
    # three rows; the logarithm, the product with ln 2 and the difference of numbers near 16: 8 (1 + 16) steps < 1e-5
    assert abs(float(loss) - float(want)) <= 3 * (float(e_z + e_l) + 1e-5)
    dz = p[:3].clone()
    dz[torch.arange(3), at] -= 1.0
    u = ref.half_step(BF16)
    for row, col in ((-1, 3), (-2, 2), (-3, 1), (1, 0), (1 << 23, 0)):
        c = p[:3, col] if col == 0 else dz[:, col]
        want = c @ xd[:3]
        bound = (c.abs() * (u + float(e_z + e_l)) + 2.0 ** -126) @ xd[:3].abs() + (u + 100 * ref.E32) * want.abs() + float(e_z + e_l) * \
            (xd[:3].abs().sum(0) * p[:3, col].max())
        ref.assert_within(f"dw {row}", dw[row], want, bound)
    want = dz[:, 1:] @ wd
    bound = (dz[:, 1:].abs() * (u + float(e_z + e_l))) @ wd.abs() + (u + 100 * ref.E32) * want.abs() + float(e_z + e_l) * wd.abs().sum(0)
    ref.assert_within("dx", dx[:3], want, bound)
    assert not bool(dx[3].any())


def test_weights_of_rows_that_are_not_finite(dev):
    """An infinite or NaN gradient of one row's loss spoils that row's dx (and dw, a sum over the rows), no other row's."""
    for dtype in TYPES:
        x, w, y = head_case(dev, 40, 300, 64, dtype, seed=50)
        g = torch.rand(40, device=dev, generator=gen(dev, 51)) + 0.5
        _, want, _ = check_head(x, w, y, reduction="none", grad=g)
        g[[3, 8]] = torch.tensor([float("inf"), float("nan")], device=dev)
        top = g[torch.isfinite(g)].max()
        assert bool(top == g.nan_to_num(0.0, 0.0).max())
        xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        dx, dw = torch.autograd.grad(linear_cross_entropy(xr, wr, y, reduction="none"), (xr, wr), g)
        assert not bool(torch.isfinite(dx[[3, 8]]).all(1).any()) and not bool(torch.isfinite(dw).all())
        rest = [i for i in range(40) if i not in (3, 8)]
        exact = ref.head(x[rest], w, y[rest][:, None], None, -100, 1.0, "none", g[rest])
        ref.assert_within("dx", dx[rest], exact["dx"], exact["e_dx"])


@pytest.mark.parametrize("dtype", TYPES)
def test_a_spoilt_row_leaves_the_others_gradients(dev, dtype):
    x, w, y = head_case(dev, 300, 700, 64, dtype, seed=52)
    x[5, 3], x[200, 0] = float("nan"), float("inf")
    xr = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(linear_cross_entropy(xr, w, y, reduction="sum"), xr)
    rest = [i for i in range(300) if i not in (5, 200)]
    exact = ref.head(x[rest], w, y[rest][:, None], None, -100, 1.0, "sum", torch.ones((), device=dev))
    ref.assert_within("dx", dx[rest], exact["dx"], exact["e_dx"])
    assert bool(torch.isnan(dx[[5, 200]]).all())


def test_gradients_of_any_layout(dev):
    ids, table, grad = lookup_case(dev, 700, 90, 24, BF16, "zipf", seed=53)
    a = check_lookup(ids, table, grad.t().contiguous().t(), 1.0, None)                      # column-major
    b = check_lookup(ids, table, grad, 1.0, None)
    assert torch.equal(a[1], b[1])
    check_lookup(ids, table, torch.ones((), dtype=BF16, device=dev).expand(700, 24), 1.0, None)
    # a view of other codes as the table, ids with strides and repeated ones
    wide = torch.randn(90, 50, device=dev, generator=gen(dev, 54)).requires_grad_(True)
    out = ops.embedding(ids.view(70, 10)[:, ::2], wide[:, 3:20], 2.0)
    assert torch.equal(out, wide[:, 3:20][ids.view(70, 10)[:, ::2]] * 2.0)
    (dw,) = torch.autograd.grad(out.sum(), wide)
    count = torch.zeros(90, device=dev).index_add_(0, ids.view(70, 10)[:, ::2].reshape(-1), torch.ones(350, device=dev)) * 2.0
    assert torch.equal(dw[:, 3:20], count[:, None].expand(90, 17)) and not bool(dw[:, :3].any()) and not bool(dw[:, 20:].any())
    # the head: column-major operands, a gradient expanded from one number, the same graph twice
    x, w, y = head_case(dev, 60, 130, 40, F16, seed=55)
    xr, wr = x.t().contiguous().t().requires_grad_(True), w.t().contiguous().t().requires_grad_(True)
    loss = linear_cross_entropy(xr, wr, y, reduction="none")
    one = torch.full((), -2.0, device=dev).expand(60)
    first = torch.autograd.grad(loss, (xr, wr), one, retain_graph=True)
    again = torch.autograd.grad(loss, (xr, wr), one)
    _, dx, dw = check_head(x, w, y, reduction="none", grad=torch.full((60,), -2.0, device=dev))
    for p, q, r in zip(first, again, (dx, dw)):
        assert torch.equal(p, q) and torch.equal(p, r)


def test_from_several_threads(dev):
    """Each thread on a stream of its own, all at once: the results of one after another."""
    cases = [head_case(dev, 200 + 50 * i, 900, 48 + 8 * i, TYPES[i % 3], seed=60 + i) for i in range(4)]
    looks = [lookup_case(dev, 3000 + i, 200, 40 + i, TYPES[i % 3], "zipf", seed=70 + i) for i in range(4)]

    def work(i):
        return [*check_head(*cases[i]), *check_lookup(*looks[i], 1.5, 0)]
    want = [work(i) for i in range(4)]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(3):
                    got[i] = work(i)
                torch.cuda.current_stream().synchronize()
        except BaseException as e:      # noqa: BLE001 (reported by the test's own thread)
            errors.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert all(torch.equal(p, q) for a, b in zip(want, got) for p, q in zip(a, b))


def test_capture_with_real_leaves(dev):
    """Parameters as leaves: captured after the warm-up's graph is gone; refused while a graph that used them elsewhere lives."""
    ids, codes, _ = lookup_case(dev, 600, 150, 32, F32, "zipf", seed=80)
    y = torch.randint(0, 150, (600,), device=dev, generator=gen(dev, 81))
    codes.requires_grad_(True)

    def passes():
        loss = linear_cross_entropy(ops.embedding(ids, codes, 2.0), codes, y)
        return loss.detach(), torch.autograd.grad(loss, codes)[0]
    want = passes()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = passes()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    alive = ops.embedding(ids, codes, 2.0)                  # an eager graph of the same leaf, on this stream
    other = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(other):
            _ = y + 1
            ops.embedding(ids, codes, 2.0)
    other = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(other):
            _ = y + 1
            linear_cross_entropy(alive.detach(), codes, y)
    with torch.no_grad():                                   # nothing is recorded: nothing to refuse
        other = torch.cuda.CUDAGraph()
        with torch.cuda.graph(other):
            again = ops.embedding(ids, codes, 2.0)
    other.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, alive)


def margin(dev, shape, dtype, fill):
    """A contiguous tensor with 64 elements of a sentinel on both sides of it."""
    n = 1
    for s in shape:
        n *= s
    whole = torch.full((n + 128,), fill, dtype=dtype, device=dev)
    return whole, whole[64:64 + n].view(shape)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (33, 257, 77), (129, 130, 200), (700, 3011, 45), (1025, 66001, 36), (3, 5, 13)])
def test_nothing_is_written_around_the_results(dev, n, v, d, dtype):
    lib, st = _lib.lib(), torch.cuda.current_stream().cuda_stream
    kind = ops.DTYPE_IDS[dtype]
    x, w, y = head_case(dev, n, v, d, dtype, seed=90)
    a = check_head(x, w, y)
    pair = {}
    for name, shape, t in (("loss", (1,), F32), ("lse", (2, n), F32), ("count", (1,), F32), ("dx", (n, d), dtype), ("dw", (v, d), dtype),
                           ("out", (n, d), dtype), ("dt", (v, d), dtype)):
        pair[name] = margin(dev, shape, t, 7.0)
    p = {k: t[1].data_ptr() for k, t in pair.items()}

    def ws(size):
        t = torch.full((size + 256,), 77, dtype=torch.uint8, device=dev)
        return t, size
    f, fn = ws(lib.rsdf_class_head_workspace_bytes(n, v, d, kind, 0))
    b, bn = ws(lib.rsdf_class_head_workspace_bytes(n, v, d, kind, 3))
    e, en = ws(lib.rsdf_embedding_bwd_workspace_bytes(n, v, d))
    one = torch.ones(1, device=dev)
    grad = torch.ones(n, d, dtype=dtype, device=dev)
    assert lib.rsdf_class_head_fwd(x.data_ptr(), w.data_ptr(), n, v, d, kind, y.data_ptr(), None, 1, -100, 1.0, 1, p["loss"], p["lse"],
                                   p["count"], None, None, None, f.data_ptr(), fn, st) == 0
    assert lib.rsdf_class_head_bwd(x.data_ptr(), w.data_ptr(), n, v, d, kind, y.data_ptr(), None, None, 1, 1.0, p["lse"], p["count"],
                                   one.data_ptr(), 0, p["dx"], p["dw"], b.data_ptr(), bn, st) == 0
    assert lib.rsdf_embedding_fwd(y.data_ptr(), n, w.data_ptr(), v, d, kind, 1.0, -1, p["out"], None, st) == 0
    assert lib.rsdf_embedding_bwd(y.data_ptr(), n, grad.data_ptr(), v, d, kind, 1.0, -1, p["dt"], e.data_ptr(), en, st) == 0
    torch.cuda.synchronize()
    for name, (whole, view) in pair.items():
        assert bool((whole[:64] == 7.0).all()) and bool((whole[64 + view.numel():] == 7.0).all()), name
    for t, size in ((f, fn), (b, bn), (e, en)):
        assert bool((t[size:] == 77).all())
    assert torch.equal(pair["loss"][1][0], a[0]) and torch.equal(pair["dx"][1], a[1]) and torch.equal(pair["dw"][1], a[2])
    assert torch.equal(pair["out"][1], w[y])


def test_other_modes_of_torch(dev):
    """Inference mode, autocast, checkpointing, accumulated .grad; a teacher's logits of any floating type, which take no gradient."""
    from torch.utils.checkpoint import checkpoint
    x, w, y = head_case(dev, 130, 300, 48, F32, seed=100)
    ids, table, _ = lookup_case(dev, 130, 90, 48, F32, seed=101)
    tid, tl = teacher(dev, 130, 300, 6, seed=102)
    loss, dx, dw = check_head(x, w, y)
    with torch.inference_mode():
        assert torch.equal(linear_cross_entropy(x, w, y), loss)
        assert torch.equal(ops.embedding(ids, table), table[ids])
    with torch.autocast("cuda", dtype=BF16):
        assert torch.equal(linear_cross_entropy(x, w, y), loss)
    xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    for _ in range(2):
        checkpoint(lambda a, b: linear_cross_entropy(a, b, y), xr, wr, use_reentrant=False).backward()
    assert torch.equal(xr.grad, dx + dx) and torch.equal(wr.grad, dw + dw)
    half = tl.to(BF16)
    a = linear_distillation(x, w, tid, half, temperature=2.0)
    assert torch.equal(a, linear_distillation(x, w, tid, half.double(), temperature=2.0))
    soft = tl.clone().requires_grad_(True)
    assert not linear_distillation(x, w, tid, soft).requires_grad
    both = linear_distillation(x.clone().requires_grad_(True), w, tid.t().contiguous().t(), soft)
    both.backward()
    assert soft.grad is None


def test_temperatures_at_the_ends(dev):
    """1 / T of the logits' spread: at 1e-6 the teacher is its largest logit, at 1e6 uniform; what is left of the loss (T^2 times a divergence
    near 1 / T^2) is rounding, so only the gradient, T times a difference of probabilities, is compared: within T e."""
    x, w, _ = head_case(dev, 40, 200, 32, F32, seed=103)
    tid, tl = teacher(dev, 40, 200, 5, seed=104, missing=0.0)
    for t in (1e-6, 1e6):
        xr = x.clone().requires_grad_(True)
        loss = linear_distillation(xr, w, tid, tl, temperature=t, reduction="sum")
        (dx,) = torch.autograd.grad(loss, xr)
        want = ref.head(x, w, tid, tl, -100, t, "sum", torch.ones((), device=dev))
        assert not bool(torch.isnan(loss)) and bool(torch.isfinite(dx).all())
        ref.assert_within("dx", dx, want["dx"], want["e_dx"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,d", [(65, 4, 48), (64, 1, 5), (1024, 9, 48), (1024, 16384, 20), (1024, 5, 2100), (700, 3, 512), (1023, 2, 1),
                                   (1025, 5, 48), (512, 16385, 8)])
def test_lookup_of_one_batch_with_few_ids(dev, n, v, d, dtype):
    """A batch whose positions name one id, two ids, or an id and the padding: as one view's rays do.  Also around the sizes from
    which the positions are sorted."""
    ids, table, grad = lookup_case(dev, n, v, d, dtype, "same", seed=n)
    check_lookup(ids, table, grad, 1.0, None)
    ids[::3] = 0
    check_lookup(ids, table, grad, 0.5, None)
    if v > 1:
        check_lookup(ids, table, grad, 0.5, 0)
    ids[5:60] = torch.randint(0, v, (55,), device=dev, generator=gen(dev, 110))
    ids[7] = v                                              # outside: no part in the gradient
    t = table.clone().requires_grad_(True)
    (dt,) = torch.autograd.grad(ops.embedding(ids, t), t, grad)
    _, _, want, bound = ref.embedding(ids, table, 1.0, None, grad)
    ref.assert_within("d_table", dt, want, bound)
    with pytest.raises(_lib.RiseSdfHipError, match="outside"):
        _lib.poll_status(dev)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,d", [(2, 183, 80), (3, 1000, 64), (40, 300, 48), (33, 5000, 200), (300, 70000, 64)])
def test_sure_rows_keep_their_digits(dev, n, v, d, dtype):
    """Features along their own class: logits of 24 to 30, probabilities within 1e-3 to 1e-11 of 1.  The loss and the label's entry of dz are as small,
    and have to be right relative to themselves: with R the sum over the other classes, relative to the label, the loss is log(1 + R) and
    1 - p = R / (1 + R); R's relative error is that of the differences of logits, 2 ez, and of its sum, (300 + V / 8192) e."""
    g = gen(dev, 120)
    w = (torch.randn(v, d, device=dev, generator=g) * (3.0 / d ** 0.5)).to(dtype)
    y = torch.randint(0, v, (n,), device=dev, generator=g)
    own = w[y].float()
    x = (own * ((24.0 + 6.0 * torch.rand(n, 1, device=dev, generator=g)) / own.square().sum(1, keepdim=True))).to(dtype)
    z = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    rest = torch.exp(z - z.gather(1, y[:, None])).scatter(1, y[:, None], 0.0)
    R = rest.sum(1)
    ez = (2 * (d / 32 + 40) + (8 if dtype == F32 else 0)) * ref.E32 * mag
    rel = 2 * ez.max(1).values + (d + 4) * ref.E32 * mag.gather(1, y[:, None])[:, 0] + (300 + v / 8192) * ref.E32 + \
        16 * ref.E32 * (z.abs().max(1).values + 1)
    assert float(R.max()) < 0.3 and float(rel.max()) < 1e-3
    tid = torch.stack([y, (y + 1) % v], 1)
    sure = torch.tensor([[40.0, -80.0]], device=dev).expand(n, 2)             # q of the second: exp(-120) = 0 in 32 bits
    for args in ((linear_cross_entropy, (y,)), (linear_distillation, (y[:, None], sure[:, :1])), (linear_distillation, (tid, sure))):
        xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = args[0](xr, wr, *args[1], reduction="none")
        want = torch.log1p(R)
        ref.assert_within("loss", loss.detach(), want, want * (rel + 8 * ref.E32) + 2.0 ** -126)
        dx, _ = torch.autograd.grad(loss, (xr, wr), torch.ones(n, device=dev))
        dz = (rest / (1 + R)[:, None]).scatter(1, y[:, None], (-R / (1 + R))[:, None])
        u = ref.half_step(dtype)
        # entries: their relative error, the rounding to the operands' type (fp16: the smallest numbers), the tail of three parts
        e_dz = dz.abs() * (rel[:, None] + ez + u + 8 * ref.E32) + 4 * 2.0 ** -126 + (2.0 ** -25 / 4096 if dtype == F16 else 0.0)
        exact = dz @ w.double()
        bound = e_dz @ w.double().abs() + (2 * (v / 32 + 40) + 72) * ref.E32 * ((dz.abs() + e_dz) @ w.double().abs()) + u * exact.abs() + \
            ref.floor_of(dtype)
        ref.assert_within("dx", dx, exact, bound)
