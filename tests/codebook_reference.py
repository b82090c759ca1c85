"""Plain 64-bit forms of the codebook operators and the error bounds their tests use.

Bounds.  u = half a step of the result's type (torch.finfo(t).eps / 2), e = 2^-24 (half a step of fp32).
  sum of m fp32 terms, any order                        m e sum|terms|; the matrix unit adds 32 products at a time, so a
                                                        product over K costs at most (K / 32 + 40) steps of 2 e each
  logit z = sum_k x_k w_k                               ez = (2 (D / 32 + 40) + 8 [fp32: the split operands and the three
                                                        dropped products]) e sum_k |x_k w_k|
  lse                                                   max_j ez / T + (300 + tiles / 32) e + 8 e max_j |z_j| / T: the sums in a
                                                        lane, over lanes, over tiles; the exponent's own rounding
  p = exp(z / T - lse)                                  p (ez / T + e_lse)
  dz = p - q, held in the operands' type                + u |dz| (fp16: + 2^-25 / 4096 of the largest row weight for its smallest numbers)
                                                        + 4 * 2^-126: the exponential and each of up to three parts of dz may
                                                        lose what lies below the normal range
  dx, dw: products of dz                                sum |error of dz| |other| + their own sums + u |result|
"""
import torch

E32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def floor_of(dtype):
    """Half the smallest positive number: what rounding may lose below the normal range."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def embedding(ids, table, scale, padding, grad=None):
    """-> (out, bound, d_table, bound) in float64; ids outside the table give NaN rows and no gradient."""
    V, D = table.shape
    t = table.double()
    flat = ids.reshape(-1).long()
    ok = (flat >= 0) & (flat < V)
    live = ok if padding is None else ok & (flat != padding)
    out = torch.zeros(flat.numel(), D, dtype=torch.float64, device=table.device)
    out[live] = t[flat[live]] * scale
    out[~ok] = float("nan")
    u = half_step(table.dtype)
    bound = (u + 2 * E32) * out.abs() + floor_of(table.dtype)
    if grad is None:
        return out, bound
    g = grad.reshape(-1, D).double() * scale
    dt, mag, cnt = torch.zeros_like(t), torch.zeros_like(t), torch.zeros(V, dtype=torch.float64, device=t.device)
    dt.index_add_(0, flat[live], g[live])
    mag.index_add_(0, flat[live], g[live].abs())
    cnt.index_add_(0, flat[live], torch.ones_like(flat[live], dtype=torch.float64))
    return out, bound, dt, (cnt[:, None] + 2) * E32 * mag + u * dt.abs() + floor_of(table.dtype)


def head(x, w, ids, logits, ignore, temperature, reduction, grad=None, lowered=None):
    """x [N, D], w [V, D], ids [N, K]; logits None = labels.  ``grad``: d(loss) ([N] for "none").  -> dict with loss, dx, dw
    and their bounds (float64)."""
    dt = x.dtype
    xd, wd, T = x.double(), w.double(), float(temperature)
    N, V, D = x.shape[0], w.shape[0], x.shape[1]
    if logits is None:
        has = ids != ignore
        q = has.double()
    else:
        has = (ids >= 0) & ~torch.isneginf(logits)
        t = torch.where(has, logits.double(), torch.full_like(logits, float("-inf"), dtype=torch.float64))
        top = t.max(1, keepdim=True).values
        top = torch.where(torch.isneginf(top), torch.zeros_like(top), top)
        ex = torch.where(has, torch.exp((t - top) / T), torch.zeros_like(t))
        q = ex / ex.sum(1, keepdim=True).clamp(min=1e-300)
    alive = has.any(1)
    xs = torch.where(alive[:, None], xd, torch.zeros_like(xd))        # rows that take part in nothing
    z = xs @ wd.t()
    mag = xs.abs() @ wd.abs().t()
    split = 8 if dt == torch.float32 else 0
    ez = (2 * (D / 32 + 40) + split) * E32 * mag / T
    lse = torch.logsumexp(z / T, 1)
    e_lse = ez.max(1).values + (300 + V / 8192) * E32 + 8 * E32 * (z.abs().max(1).values / T + 1)
    at = ids.clamp(0, V - 1)                                          # (an ignored label may lie anywhere)
    logp = torch.gather(z, 1, at) / T - lse[:, None]
    per_row = torch.where(q > 0, torch.special.xlogy(q, q) - q * logp, torch.zeros_like(q)).sum(1) * T * T
    per_row = torch.where(alive, per_row, torch.zeros_like(per_row))
    # the listed logits are dot products of their own: D fp32 steps
    e_row = (e_lse + (q * (torch.gather(ez, 1, at) + (D + 4) * E32 * torch.gather(mag, 1, at) / T)).sum(1)
             + 16 * E32 * (q * (torch.log(q.clamp(min=1e-300)).abs() + logp.abs())).sum(1)
             + 8 * E32 * (1 + lse.abs())) * T * T
    e_row = torch.where(alive, e_row + ids.shape[1] * 4 * E32 * per_row.abs(), torch.zeros_like(e_row))
    count = alive.sum().clamp(min=1).double()
    if reduction == "none":
        loss, e_loss = per_row, e_row
    elif reduction == "sum":
        loss, e_loss = per_row.sum(), e_row.sum()
    else:
        loss, e_loss = per_row.sum() / count, e_row.sum() / count
    res = dict(loss=loss, e_loss=e_loss + 2 * E32 * loss.abs(), alive=alive)
    if grad is None:
        return res
    g = grad.double() * torch.ones_like(per_row) / (count if reduction == "mean" else 1.0)
    weight = torch.where(alive, g * T, torch.zeros_like(g))
    u = half_step(dt)
    p = torch.exp(z / T - lse[:, None])
    e_p = p * (ez + e_lse[:, None] + 4 * E32)
    dz = p.clone()
    dz.scatter_add_(1, at, -q)
    # a listed entry is taken from its own dot product
    e_p.scatter_add_(1, at, torch.where(q > 0, torch.gather(p, 1, at) * (D + 8) * E32 * torch.gather(mag, 1, at) / T
                                        + 8 * E32 * q, torch.zeros_like(q)))
    wa = weight.abs()[:, None]
    # the products of the entry with its row's weight: + 4 roundings
    e_dz = (e_p + (u + 4 * E32) * dz.abs()) * wa + (4 * 2.0 ** -126 + (2.0 ** -25 / 4096 if dt == torch.float16 else 0.0)) * wa.max()
    wz = dz * weight[:, None]
    a_dz = wz.abs() + e_dz
    steps_v, steps_n = 2 * (V / 32 + 40) + 64, 2 * (N / 32 + 40) + 64
    dx, dw = wz @ wd, wz.t() @ xs
    e_dx = e_dz @ wd.abs() + (steps_v + split) * E32 * (a_dz @ wd.abs())
    e_dw = e_dz.t() @ xs.abs() + (steps_n + split) * E32 * (a_dz.t() @ xs.abs())
    res.update(dx=dx, e_dx=e_dx + (u + 4 * E32) * dx.abs() + floor_of(dt),
               dw=dw, e_dw=e_dw + (u + 4 * E32) * dw.abs() + floor_of(dt))
    return res


def assert_within(name, got, want, bound):
    got = got.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{name}: NaN in other places"
    excess = torch.where(nan, torch.zeros_like(want), (got - want).abs() - bound)
    worst = float(excess.max()) if excess.numel() else 0.0
    if worst > 0:
        i = int(excess.reshape(-1).argmax())
        raise AssertionError(f"{name}: off by {float((got - want).abs().reshape(-1)[i]):.3e} where {float(bound.reshape(-1)[i] if bound.numel() > 1 else bound):.3e} "
                             f"is allowed (value {float(want.reshape(-1)[i]):.6e}, element {i} of {want.numel()})")
