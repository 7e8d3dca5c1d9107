"""Plain 64-bit forms of the operators around the experts, and the error bounds of their tests.

U is the unit roundoff of fp32. A result rounded to type t from an fp32 value with error e is off
by at most e + half a step of t at that value; ``tol`` adds the two (and the half step at the
smallest subnormal of fp16, below which steps no longer shrink).
"""
import torch

U = 2.0 ** -24


def tol(ref, err, dtype):
    half = torch.finfo(dtype).eps / 2
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134,
            torch.float32: 2.0 ** -150}[dtype]
    return err + half * (ref.abs() + err) + tiny


def check(got, ref, err, what):
    """Every value of ``got`` within the bound of its 64-bit reference."""
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    d = (got.double() - ref).abs()
    t = tol(ref, err, got.dtype)
    bad = ~(d <= t)
    assert not bool(bad.any()), (what, int(bad.sum()), float((d / t).nan_to_num(9e9).max()))


def order(ids, lo, E, align):
    """Tables of the stable sort, with Python lists. Returns base, row_pick, pick_row."""
    T, K = ids.shape
    flat = ids.reshape(-1).tolist()
    base, rows = [0], []
    pick_row = [-1] * (T * K)
    for e in range(E):
        picks = [p for p, i in enumerate(flat) if i == lo + e]
        for p in picks:
            pick_row[p] = len(rows)
            rows.append(p)
        rows += [-1] * (-len(rows) % align)
        base.append(len(rows))
    R = T * K + min(T * K, E) * (align - 1)
    assert len(rows) <= R
    rows += [-1] * (R - len(rows))
    return base, rows, torch.tensor(pick_row, dtype=torch.int32).view(T, K)


def rows_of(x, row_pick, K):
    """[R, H] float64: the token row of each pick, zero without one."""
    pick = torch.tensor(row_pick, device=x.device)
    out = torch.zeros(len(row_pick), x.shape[1], dtype=torch.float64, device=x.device)
    live = pick >= 0
    out[live] = x.double()[pick[live] // K]
    return out


def unsort(rows, pick_row, w):
    """y and the sum of the terms' magnitudes."""
    has = (pick_row >= 0)[:, :, None]
    picked = torch.where(has, rows.double()[pick_row.clamp(min=0).long()], 0.0)
    terms = torch.where(has, picked * (1.0 if w is None else w.double()[:, :, None]), 0.0)
    return terms.sum(1), terms.abs().sum(1)


def quantize(x):
    amax = x.double().abs().amax(1).clamp(min=float(torch.tensor(1e-30)))
    return torch.round(127 * x.double() / amax[:, None]), amax / 127


def product(a, w, a_scale, w_scale, bias=None):
    """y and the bound of the fp32 scaling: int32 to fp32, two products, one sum."""
    y = (a.double() @ w.double().t()) * a_scale.double()[:, None] * w_scale.double()
    mag = y.abs()
    if bias is not None:
        y = y + bias.double()
        mag = mag + bias.double().abs()
    return y, 4 * U * mag


def norm_leaves(branch, residual, wp, gate, wq):
    return [None if t is None else t.detach().double().requires_grad_()
            for t in (branch, residual, wp, gate, wq)]


def block_norm(f, x, wp, gate, wq, s, eps):
    """hidden and normed in the arguments' type (float64), as the definition reads."""
    h = s * x
    if f is not None:
        n = f if wp is None else f / torch.sqrt(f.square().mean(1, keepdim=True) + eps) * wp
        h = h + (n if gate is None else gate * n)
    y = None if wq is None else h / torch.sqrt(h.square().mean(1, keepdim=True) + eps) * wq
    return h, y


def block_norm_bounds(f, x, wp, gate, wq, s, eps):
    """Error bounds of hidden and normed before their rounding, and of the gradients' factors.

    A thread adds at most 64 squares, then come ten shuffle levels, the mean and eps: fewer than 80
    roundings of positive terms, so a mean of squares is off by 80 U relative and its rsqrt by
    40 U + 4 U (rsqrtf: two units in the last place). With three products that puts n within 48 U,
    g n + s x within 50 U (|g n| + |s x|). The second rsqrt moves by at most the error of h over its
    norm on top: (44 + 50 rho) U with rho = |(|g n| + |s x|)| / |h| (2-norms of the row).
    """
    with torch.no_grad():
        gn = torch.zeros_like(x)
        if f is not None:
            n = f if wp is None else f / torch.sqrt(f.square().mean(1, keepdim=True) + eps) * wp
            gn = n if gate is None else gate * n
        mag = gn.abs() + (s * x).abs()
        h = gn + s * x
        r2 = 1 / torch.sqrt(h.square().mean(1, keepdim=True) + eps)
        # eps keeps the row's size away from zero, in the norm as in the ratio
        rho = torch.sqrt(mag.square().mean(1, keepdim=True) + eps) * r2
        eh = 50 * U * mag
        ey = None
        if wq is not None:
            ey = (h * r2 * wq).abs() * (47 + 50 * rho) * U + (r2 * wq).abs() * eh
        return eh, ey, mag, rho, r2


def block_norm_grad_bounds(leaves, s, eps, da, dy):
    """Bounds of the gradients: 640 U rho^2 of the sum of their terms' magnitudes.

    r2 enters as a cube (3 (44 + 50 rho) U), h with 50 U of its magnitude in two places, the row
    sums add 80 U each, and the products around them fewer than 20 U: under 600 rho^2 U in all for
    dh, and at most 40 U more for what is computed from it.
    """
    f, x, wp, gate, wq = (None if t is None else t.detach() for t in leaves)
    _, _, hm, rho, r2 = block_norm_bounds(f, x, wp, gate, wq, s, eps)
    H = x.shape[1]
    rho = rho.clamp(min=1.0)
    zero = torch.zeros_like(x)
    u = zero if dy is None else (dy.double() * wq).abs()
    m_dh = (zero if da is None else da.double().abs()) + r2 * u
    m_dh = m_dh + hm * r2 ** 3 / H * (u * hm).sum(1, keepdim=True)
    k = 640 * U * rho.square()
    out = {"residual": k * abs(s) * m_dh}
    if wq is not None:
        out["pre_w"] = (k * r2 * hm * (zero if dy is None else dy.double().abs())).sum(0)
    if f is not None:
        r1 = torch.ones_like(r2) if wp is None else \
            1 / torch.sqrt(f.square().mean(1, keepdim=True) + eps)
        g = torch.ones_like(x) if gate is None else gate.abs() * torch.ones_like(x)
        w = torch.ones_like(x[0]) if wp is None else wp.abs()
        v = g * w * m_dh
        out["branch"] = k * (r1 * v)
        if wp is not None:
            fa = f.abs()
            out["branch"] = k * (r1 * v + fa * r1 ** 3 / H * (v * fa).sum(1, keepdim=True))
            out["post_w"] = (k * g * m_dh * fa * r1).sum(0)
        if gate is not None:
            out["gate"] = (k * m_dh * f.abs() * r1 * w).sum_to_size(gate.shape)
    # sums over T tokens add up to T roundings more; far below 640 for the tests' T
    assert x.shape[0] <= 600
    for n in ("pre_w", "post_w"):
        if n in out:
            out[n] = 2 * out[n]
    if "gate" in out and gate.shape != x.shape:
        out["gate"] = 2 * out["gate"]
    return out
