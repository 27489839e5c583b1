"""The language-model operators written out in float64 on the host, and what float32 costs them.

U is half a step of float32.  A sum over a row is a chain of at most 64 additions in a lane and
a tree of 18 over lanes, waves and parts (82 U), with at most 22 changes of the running maximum
(an exponential of 2 U, a product of 1 U each, and arguments that telescope: 28 U), each term an
exponential (2 U) of an argument with two roundings (1.4 U per nat of it, 18 U on average over a
softmax of 2^19 columns): together under SUM = 200 half steps.
"""
import math

import torch

U = 2.0 ** -24
SUM = 200


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half the spacing of the type's subnormal numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def softmax64(x, temperature):
    """log p, p of every row; a row with nothing left has log p = -inf, one with NaN or +inf has NaN."""
    z = x.double() / temperature
    dead = torch.isneginf(z).all(1, keepdim=True)
    # by the maximum first: next to the type's lowest value even float64 has no room for log n
    d = z - torch.where(dead, 0.0, z.amax(1, keepdim=True))
    logp = d - torch.where(dead, 0.0, d.exp().sum(1, keepdim=True).log())
    bad = (torch.isnan(z) | torch.isposinf(z)).any(1, keepdim=True)
    return torch.where(bad, math.nan, logp), dead[:, 0], bad[:, 0]


def scores64(x, t, top, temperature):
    n, v = x.shape
    logp, dead, bad = softmax64(x, temperature)
    p = logp.exp()
    counts = (t >= 0) & (t < v)
    at = t.clamp(0, v - 1).long()[:, None]
    xf = x.double()
    xt = xf.gather(1, at)
    before = torch.arange(v)[None, :] < at
    ahead = ((xf > xt) | ((xf == xt) & before)).sum(1)
    rank = torch.where(counts & ~bad, ahead, -1)
    err = counts & (bad | (ahead > 0) | torch.isneginf(xt[:, 0]))
    lp = torch.where(counts, logp.gather(1, at)[:, 0], 0.0)
    entropy = torch.where(bad, math.nan, -torch.special.xlogy(p, p).sum(1))
    out = {"logprob": lp, "entropy": entropy, "rank": rank.int(), "err": err.to(torch.uint8)}
    if top:
        # a stable sort of the negated values puts the lower column of equal ones first
        k = min(top, v)
        order = (-torch.where(torch.isnan(xf), -math.inf, xf)).sort(dim=1, stable=True).indices[:, :k]
        value = logp.gather(1, order)
        keep = ~torch.isneginf(xf.gather(1, order)) & ~bad[:, None]
        value = torch.where(bad[:, None], math.nan, torch.where(keep, value, -math.inf))
        index = torch.where(keep, order, -1)
        pad = (0, top - k)
        fill = torch.where(bad, math.nan, -math.inf)[:, None].expand(n, top - k)
        out["top_logprob"] = torch.cat([value, fill], 1)
        out["top_index"] = torch.nn.functional.pad(index, pad, value=-1).int()
    return out


def scores_tolerance(x, ref, temperature):
    """Bounds on |logprob - exact| (also of the alternatives) and |entropy - exact|, float32."""
    v = x.shape[1]
    log_v = math.log(v) + 1.0
    lp = lambda r: U * (SUM + 3 * log_v + 4 * torch.nan_to_num(r.abs(), posinf=0.0))  # noqa: E731
    # H = log S - U/S: the first as above, the second a quotient of two sums of size <= log_v + H
    h = U * (SUM + 3 * log_v + (2 * SUM + 10) * 2 * log_v)
    return lp, h


def scores_grad64(x, t, ref, temperature, d_logprob=None, d_entropy=None, d_top=None):
    n, v = x.shape
    logp, dead, bad = softmax64(x, temperature)
    p = logp.exp()
    counts = (t >= 0) & (t < v)
    zero = torch.zeros(n, dtype=torch.float64)
    g_lp = torch.where(counts, d_logprob.double(), 0.0) if d_logprob is not None else zero
    g_h = d_entropy.double() if d_entropy is not None else zero
    rows = torch.arange(n)
    direct = torch.zeros(n, v, dtype=torch.float64)
    direct[rows, t.clamp(0, v - 1).long()] += g_lp
    a = g_lp.clone()
    if d_top is not None:
        listed = ref["top_index"] >= 0
        g_top = torch.where(listed, d_top.double(), 0.0)
        direct.scatter_add_(1, ref["top_index"].clamp(min=0).long(), g_top)
        a = a + g_top.sum(1)
    plogp = torch.special.xlogy(p, p)
    dx = (direct - a[:, None] * p - g_h[:, None] * (plogp + p * ref["entropy"][:, None])) / temperature
    dx = torch.where(bad[:, None], math.nan, torch.where(dead[:, None], 0.0, dx))
    # float32: p to SUM + 8 per nat of its logarithm, the bracket to a few half steps of its parts
    size = p * (a.abs()[:, None] + g_h.abs()[:, None] * (torch.nan_to_num(ref["entropy"].abs())[:, None] + 1))
    size = size + g_h.abs()[:, None] * plogp.abs()
    if d_top is not None:
        size = size + p * g_top.abs().sum(1)[:, None]
    nats = 1.0 + torch.nan_to_num(logp.abs(), posinf=0.0).clamp(max=100.0)
    tol = U * ((3 * SUM + 8 * nats) * size + 4 * direct.abs()) / temperature
    # the entropy that enters the bracket is float32's
    tol = tol + p * g_h.abs()[:, None] * scores_tolerance(x, ref, temperature)[1] / temperature
    return dx, torch.nan_to_num(tol)


def close(got, want, tol, dtype=torch.float32):
    """|got - want| <= tol + one rounding to `dtype`; infinities and NaN in the same places."""
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, (got.shape, want.shape)
    beyond = want.abs() > torch.finfo(dtype).max          # the lowest value over a temperature below one
    want = torch.where(beyond & torch.isfinite(want), want.sign() * math.inf, want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in other places"
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)]), "infinities differ"
    bound = torch.as_tensor(tol, dtype=torch.float64).expand(want.shape) * (1 + half_step(dtype))
    bound = bound + half_step(dtype) * want.abs() + smallest(dtype)
    off = ((got - want).abs() - bound)[fin]
    assert off.numel() == 0 or off.max() <= 0, (float(off.max()), float((got - want).abs()[fin].max()))


def first_of_each(index, v):
    """Which entries count: inside the row, and no repeat of an earlier one."""
    inside = (index >= 0) & (index < v)
    same = (index[:, :, None] == index[:, None, :]).tril(-1).any(2)
    return inside & ~same


def distill64(x, index, logprob, tail, temperature, weight=None):
    """(loss, its bound, gradient, its bound) in float64."""
    n, v = x.shape
    logp, dead, bad = softmax64(x, temperature)
    keep = first_of_each(index, v)
    head = torch.zeros(n, v, dtype=torch.bool)
    logq = torch.full((n, v), -math.inf, dtype=torch.float64)
    for r in range(n):
        cols = index[r][keep[r]].long()
        head[r, cols] = True
        logq[r, cols] = logprob[r][keep[r]].double()
    given = logq.clone()
    if tail == "renorm":
        logq = logq / temperature
        top = logq.amax(1, keepdim=True)
        some = top > -math.inf
        logq = torch.where(some, logq - top, -math.inf)
        logq = logq - torch.where(some, logq.exp().sum(1, keepdim=True).log(), 0.0)
        rest = torch.zeros(n, 1, dtype=torch.float64)
    else:
        rest = 1.0 - logq.exp().sum(1, keepdim=True)
        rest = torch.where((rest < 2.0 ** -20) | (head.sum(1, keepdim=True) == v), 0.0, rest)
    q = logq.exp()
    log_rest = torch.logsumexp(torch.where(head, -math.inf, logp), 1, keepdim=True)
    gap = torch.where(q > 0, logq - logp, 0.0)
    last = torch.where(rest > 0, rest.log() - log_rest, 0.0)
    loss = (torch.where(q > 0, q * gap, 0.0).sum(1, keepdim=True) + torch.where(rest > 0, rest * last, 0.0))[:, 0]
    loss = torch.where(bad, math.nan, loss)
    calm = lambda t: torch.nan_to_num(t, nan=0.0, posinf=0.0, neginf=0.0).abs()  # noqa: E731
    log_v = math.log(v) + 1.0
    # log p: a sum and two nats' roundings; q: its exponential and normalisation; the remainder:
    # a difference with 12 half steps of 1
    tol = (q * (SUM + 20 + 3 * log_v + 4 * calm(logp) + 16 * calm(gap) + 4 * calm(given / temperature))).sum(1)
    tol = tol + 12 * (calm(last)[:, 0] + 1) + (rest * (2 * SUM + 6 * log_v + 4 * calm(log_rest)))[:, 0]
    p = logp.exp()
    share = torch.where(head | torch.isneginf(log_rest), 0.0, (logp - log_rest).exp())
    w = torch.ones(n, 1, dtype=torch.float64) if weight is None else weight.double()[:, None]
    whole = q.sum(1, keepdim=True) + rest
    dx = torch.where(head, p * whole - q, p * whole - rest * share)
    nats = 1.0 + calm(logp).clamp(max=100.0)
    p_rest = log_rest.exp()
    head_tol = p * (2 * SUM + 8 * nats + 24) + q * (24 + 8 * calm(given / temperature) + 8 * calm(logq))
    if tail == "rest":
        bulk_tol = share * ((SUM + 8 * nats + 8 * calm(log_rest)) * (p_rest * whole - rest).abs()
                            + p_rest * (2 * SUM + 8 * calm(log_rest) + 24) + 16)
    else:
        bulk_tol = p * (2 * SUM + 8 * nats + 24)
    none = dead[:, None] | (w == 0)
    dx = torch.where(none, 0.0, torch.where(bad[:, None], math.nan, dx)) * w / temperature
    dx = torch.where(none, 0.0, dx)
    dx_tol = U * torch.nan_to_num(torch.where(head, head_tol, bulk_tol)) * w.abs() / temperature
    return loss, U * torch.nan_to_num(tol), dx, dx_tol


def gated64(x, log_a, offsets, state, scale, h_given=None, d_h=None, d_state=None):
    """The recurrence a row at a time in float64, with bounds of what float32 may differ by.

    A step costs an exponential, the factor, a product and a sum, and their regrouping as much
    again: under STEP = 10 half steps of the majorant H_t = a H_{t-1} + |b_t|, which also bounds
    what any grouping of the steps adds up on the way.  Returns dicts of (value, bound)."""
    import numpy as np
    step = 10 * U
    rows, d = x.shape
    g = log_a.shape[1]
    xd, lam = x.double().numpy(), np.repeat(log_a.double().numpy(), d // g, 1)
    a = np.exp(lam)
    with np.errstate(all="ignore"):
        if scale == "none":
            f, df = np.ones_like(a), np.zeros_like(a)
        elif scale == "ewma":
            f, df = -np.expm1(lam), -a
        else:
            f = np.sqrt(np.maximum(-np.expm1(2 * lam), 0))
            df = np.where(f > 0, -a * a / np.where(f > 0, f, 1), 0.0)
    off = [0, rows] if offsets is None else offsets.tolist()
    n = len(off) - 1
    h0 = np.zeros((n, d)) if state is None else state.double().numpy()
    h, ht = np.zeros((rows, d)), np.zeros((rows, d))
    s, st = h0.copy(), np.zeros((n, d))
    b = f * xd
    ab = np.abs(b)
    for q in range(n):
        c, m, t = h0[q], np.abs(h0[q]), np.zeros(d)
        for r in range(off[q], off[q + 1]):
            c = a[r] * c + b[r]
            m = a[r] * m + ab[r]
            t = a[r] * t + step * m
            h[r], ht[r] = c, t
        s[q], st[q] = c, t
    pair = lambda v, t: (torch.from_numpy(v), torch.from_numpy(t))  # noqa: E731
    out = {"h": pair(h, ht), "state": pair(s, st)}
    if d_h is None:
        return out
    hg, dh = h_given.double().numpy(), d_h.double().numpy()
    ds = np.zeros((n, d)) if d_state is None else d_state.double().numpy()
    dx, dxt, dl, dlt = (np.zeros((rows, d)) for _ in range(4))
    d0, d0t = ds.copy(), np.zeros((n, d))
    for q in range(n):
        c, m, t = ds[q], np.abs(ds[q]), np.zeros(d)
        for r in range(off[q + 1] - 1, off[q] - 1, -1):
            c, m = c + dh[r], m + np.abs(dh[r])
            t = t + step * m
            before = hg[r - 1] if r > off[q] else h0[q]
            dx[r], dxt[r] = c * f[r], (t + step * m) * f[r]
            parts = np.abs(a[r] * before) + np.abs(df[r] * xd[r])
            dl[r], dlt[r] = c * (a[r] * before + df[r] * xd[r]), (t + 2 * step * m) * parts
            c, m, t = a[r] * c, a[r] * m, a[r] * t + step * a[r] * m
        d0[q], d0t[q] = c, t
    share = d // g
    if share > 1:                               # one gate's sum, in any order
        size = np.abs(dl).reshape(rows, g, share).sum(2)
        dl = dl.reshape(rows, g, share).sum(2)
        dlt = dlt.reshape(rows, g, share).sum(2) + U * share * size
    out.update(d_x=pair(dx, dxt), d_log_a=pair(dl, dlt), d_state=pair(d0, d0t))
    return out
