"""The operators of kaldi_decoder.frames in 64 bits, from their definition, and how far f32 sums may
be from them.  Rows are handled one list at a time, on the CPU.

Error bounds.  u = 2^-24 is half a step of f32.  With d_j = x_j - m, e_j = exp(d_j / t):
 * d_j carries u |d_j|, its product with log2(e) / t twice u |d_j / t| more (product and constant),
   exp2 one step (2 u): e_j is off by u (3 |d_j| / t + 2) of itself.
 * a sum of e_j: a lane adds at most 128 of them one by one (64, but for loss and gradient of many rows
   of 128 to 256 KiB), then 6 levels join lanes, at most 16 waves follow one by one and at most
   8 + 6 + 4 steps join segments: CHAIN = 168 roundings cover it, and s is off by
   S = u (CHAIN + E[3 |d| / t + 2]) of itself, with E over p.
 * log s: S, and 2 u |log s| of its own (the library's logarithm is within one step).
"""
import torch

U = 2.0 ** -24
CHAIN = 168
TINY = 1e-37  # f32 results below 2^-126 may be flushed


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _parts(x, t=1.0):
    x = x.double()
    m = x.max()
    base = 0.0 if m == float("-inf") else m
    d = (x - base) / t
    e = torch.exp(d)
    s = e.sum()
    p = e / s if s != 0 else e
    fin = torch.where(p > 0, d, torch.zeros_like(d)).abs()
    tol_s = U * (CHAIN + float((p * (3 * fin + 2)).sum()))
    ls = torch.log(s) if s != 0 else s
    return m, d, s, ls, p, tol_s


def row_scores(x, token, top):
    """(logp, entropy, (m, s), [(column, log p)]) and the bounds (logp, entropy, s, [log p])."""
    v = x.shape[0]
    m, d, s, ls, p, tol_s = _parts(x)
    nan = bool(torch.isnan(s))
    tol_ls = tol_s + 2 * U * abs(float(ls))
    plogp = torch.where(p > 0, p * (d - ls), torch.zeros_like(p))
    h = -plogp.sum() if not nan else s
    absd = torch.where(p > 0, d, torch.zeros_like(d)).abs()
    mean, sq = float((p * absd).sum()), float((p * absd * absd).sum())
    # s1 / s: terms e d off by u (3 |d| + 4) of themselves, CHAIN additions, the quotient
    tol_h = tol_ls + mean * (tol_s + (CHAIN + 6) * U) + 3 * U * sq
    logp, tol_logp = 0.0, 0.0
    if 0 <= token < v:
        logp = float(d[token] - ls) if not nan else float("nan")
        tol_logp = tol_ls + U * (abs(float(d[token])) + abs(logp)) if abs(logp) != float("inf") else 0.0
    xs = x.double()
    order = torch.sort(xs, descending=True, stable=True).indices[:top].tolist()
    alts, tols = [], []
    for k in range(top):
        if nan:
            alts.append((-1, float("nan")))
        elif k < len(order) and xs[order[k]] > float("-inf"):
            alts.append((order[k], float(d[order[k]] - ls)))
        else:
            alts.append((-1, float("-inf")))
        a = alts[-1][1]
        tols.append(tol_ls + U * (abs(a) + abs(a + float(ls))) if abs(a) < float("inf") else 0.0)
    return (logp, float(h), (float(m), float(s)), alts), (tol_logp, tol_h, float(s) * tol_s, tols)


def row_scores_grad(x, token, g_logp, g_entropy):
    """(gradient, bound before the last rounding) of g_logp * logp + g_entropy * entropy."""
    m, d, s, ls, p, tol_s = _parts(x)
    if s == 0:
        return torch.zeros_like(d), torch.zeros_like(d)
    lp = torch.where(p > 0, d - ls, torch.zeros_like(d))
    h = -(p * lp).sum()
    on = 0 <= token < x.shape[0]
    gl = g_logp if on else 0.0
    g = -gl * p - g_entropy * p * (lp + h)
    absd = torch.where(p > 0, d, torch.zeros_like(d)).abs()
    rel = tol_s + U * (3 * absd + 8)
    terms = abs(gl) + abs(g_entropy) * (lp.abs() + abs(float(h)) + 1)
    tol = p * terms * (rel + 8 * U) + p * abs(g_entropy) * (4 * tol_s * (1 + float((p * absd).sum())) + 4 * U * abs(float(ls)))
    tol = tol + p * abs(g_entropy) * 3 * U * float((p * absd * absd).sum())
    if on:
        g[token] += gl
        tol[token] += U * abs(gl)
    return g, tol + TINY * (1 + abs(gl) + abs(g_entropy))


def row_distill(x, ids, teacher, weight, t, upstream=1.0):
    """(loss, gradient) and their bounds."""
    v = x.shape[0]
    zero = torch.zeros(v, dtype=torch.float64)
    keep = [k for k, i in enumerate(ids) if 0 <= i < v and not teacher[k] == float("-inf")]
    if weight == 0 or not keep:
        return (0.0, zero), (0.0, zero)
    m, d, s, ls, p, tol_s = _parts(x, t)
    um, ud, us, uls, q, tol_u = _parts(torch.tensor([teacher[k] for k in keep], dtype=torch.float64), t)
    tol_ls = tol_s + 2 * U * abs(float(ls))
    loss, tol = 0.0, 0.0
    dx = p.clone()
    tol_dx = p * (tol_s + U * (3 * torch.where(p > 0, d, zero).abs() + 10))
    for n, k in enumerate(keep):
        i, qk = ids[k], float(q[n])
        tol_q = tol_u + U * (3 * abs(float(ud[n])) + 8)
        if qk > 0 or qk != qk:
            each = float((ud[n] - uls) - (d[i] - ls))
            loss += qk * each
            if each < float("inf"):
                tol += qk * (abs(each) * (tol_q + (len(keep) + 4) * U) + tol_u + tol_ls
                             + U * (4 * abs(float(ud[n])) + 4 * abs(float(uls)) + 4 * abs(float(d[i])) + 4 * abs(float(ls))))
        dx[i] -= qk
        tol_dx[i] += qk * (tol_q + (len(keep) + 6) * U)
    c = abs(weight * upstream / t)
    return (weight * loss, dx * (weight * upstream / t)), (abs(weight) * tol, tol_dx * c + TINY * (1 + c))
