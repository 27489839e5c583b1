"""gated_scan, its gradient and its step against a row-by-row recurrence in float64: every
layout of lanes, tiles and groups, ragged and empty sequences, shared gates, strides, and the
charts of a monitored model's scores."""
import math

import pytest
import torch

from lm_reference import close, gated64

pytestmark = pytest.mark.gpu
F, B, H = torch.float32, torch.bfloat16, torch.float16


def make(rows, d, g, dtype, gate_dtype, seed, seqs=None, state=True):
    """Inputs on the host; seqs None: one sequence without offsets, else ragged ones with rows before, behind
    and between... nothing, one empty, one of a single row."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, d, generator=gen).to(dtype)
    lam = -torch.exp(torch.rand(rows, g, generator=gen) * -7)
    lam[torch.rand(rows, g, generator=gen) < 0.02] = -math.inf if seed % 2 else -50.0
    lam[torch.rand(rows, g, generator=gen) < 0.02] = 0.0
    lam = lam.to(gate_dtype)
    off, n = None, 1
    if seqs is not None:
        n = seqs
        lo, hi = (rows // 10, rows - rows // 7) if rows > 20 else (0, rows)
        cuts = torch.randint(lo, hi + 1, (n + 1,), generator=gen).sort().values
        cuts[0], cuts[-1] = lo, hi
        if n > 3:
            cuts[2] = cuts[1]
            cuts[3] = min(int(cuts[2]) + 1, hi)
            cuts = cuts.sort().values
        off = cuts
    return x, lam, off, torch.randn(n, d, generator=gen) if state else None


def on(*ts):
    return [None if t is None else t.cuda() for t in ts]


def check(x, lam, off, state, scale, grad, seed=0):
    import ddm_amd
    xc, lc, oc, sc = on(x, lam, off, state)
    h, after = ddm_amd.gated_scan(xc, lc, offsets=oc, state=sc, scale=scale)
    gen = torch.Generator().manual_seed(seed)
    d_h = torch.randn(x.shape, generator=gen).to(x.dtype)
    d_state = torch.randn(after.shape, generator=gen) if seed % 2 == 0 else None
    ref = gated64(x, lam, off, state, scale, *((h.cpu(), d_h, d_state) if grad else ()))
    close(h, *ref["h"], x.dtype)
    close(after, *ref["state"])
    if grad:
        d_x, d_a, d_0 = ddm_amd.gated_scan_grad(xc, lc, h, d_h.cuda(), offsets=oc, state=sc,
                                                d_state=None if d_state is None else d_state.cuda(), scale=scale)
        close(d_x, *ref["d_x"], x.dtype)
        close(d_a, *ref["d_log_a"], lam.dtype)
        close(d_0, *ref["d_state"])
    return h, after


@pytest.mark.parametrize("dtype,gate_dtype", [(F, F), (B, B), (B, F), (H, H), (H, F)])
@pytest.mark.parametrize("rows,d,g,seqs", [(1, 1, 1, None), (1, 7, 7, 1), (2, 2, 1, 2), (31, 3, 3, None), (500, 1, 1, 9),
                                           (700, 4, 1, 5), (333, 5, 1, 4), (300, 8, 2, 5), (257, 12, 4, 3), (400, 64, 64, 6),
                                           (3000, 256, 256, 11), (900, 257, 257, 3), (1000, 260, 65, 4),
                                           (600, 768, 12, 5), (400, 1000, 1, 3), (300, 513, 27, 4), (9, 2048, 2048, 40)])
def test_scan_and_gradient(dtype, gate_dtype, rows, d, g, seqs):
    for k, scale in enumerate(("none", "ewma", "unit")):
        check(*make(rows, d, g, dtype, gate_dtype, rows + d + k, seqs, state=k != 1), scale, True, seed=k)


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("rows,d,g,seqs", [(70001, 256, 256, 3), (9001, 2048, 32, 5), (8200, 2050, 1, None)])
def test_many_tiles(dtype, rows, d, g, seqs):
    """Sizes at which a lane takes its larger number of rows, and groups of tiles follow each other."""
    check(*make(rows, d, g, dtype, dtype, 3, seqs), "unit", True)


def test_a_long_stream():
    check(*make(300001, 1, 1, F, F, 4, 3), "ewma", False)
    check(*make(40001, 2, 1, F, F, 4, 2), "ewma", True)


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("rows,d,g,seqs", [(3000, 40, 40, 513), (5000, 3, 1, 5000), (900, 64, 64, 9000), (20, 70, 7, 2000),
                                           (40001, 12, 12, 600)])
def test_many_sequences(dtype, rows, d, g, seqs):
    """More sequences than a workgroup has threads, most of them empty or of a row; narrow rows of many tiles."""
    check(*make(rows, d, g, dtype, dtype, 7, seqs), "ewma", True)


def test_the_same_every_time():
    import ddm_amd
    x, lam, off, state = on(*make(20000, 512, 512, B, B, 5, 6))
    d_h = torch.randn_like(x)
    first = None
    for _ in range(5):
        h, s = ddm_amd.gated_scan(x, lam, offsets=off, state=state, scale="unit")
        got = (h, s) + ddm_amd.gated_scan_grad(x, lam, h, d_h, offsets=off, state=state, scale="unit")
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("shift,pad", [(0, 4), (1, 3), (2, 6)])
def test_strides(dtype, shift, pad):
    import ddm_amd
    x, lam, off, state = make(600, 64, 64, dtype, dtype, 6, 5)
    wide = torch.full((600, shift + 64 + pad), math.nan, dtype=dtype, device="cuda")
    lwide, owide = wide.clone(), torch.full_like(wide, 7.0)
    for w, t in ((wide, x), (lwide, lam)):
        w[:, shift:shift + 64] = t.cuda()
    xv, lv, ov = (w[:, shift:shift + 64] for w in (wide, lwide, owide))
    h, after = ddm_amd.gated_scan(xv, lv, offsets=off.cuda(), state=state.cuda(), scale="ewma", out=ov)
    assert h is ov
    d_h = torch.randn(600, 64, device="cuda").to(dtype)
    ref = gated64(x, lam, off, state, "ewma", h.cpu(), d_h.cpu())
    a, b = int(off[0]), int(off[-1])
    close(h[a:b], *(t[a:b] for t in ref["h"]), dtype)
    close(after, *ref["state"])
    # rows of no sequence, and what lies between the rows, are left as they were
    assert (owide[:, :shift] == 7).all() and (owide[:, shift + 64:] == 7).all()
    assert (h[:a] == 7).all() and (h[b:] == 7).all()
    d_x, d_a, d_0 = ddm_amd.gated_scan_grad(xv, lv, h, d_h, offsets=off.cuda(), state=state.cuda(), scale="ewma")
    for got, name in ((d_x, "d_x"), (d_a, "d_log_a"), (d_0, "d_state")):
        close(got, *ref[name], got.dtype)
    # over x itself
    same, after2 = ddm_amd.gated_scan(xv, lv, offsets=off.cuda(), state=state.cuda(), scale="ewma", out=xv)
    assert torch.equal(same[a:b], h[a:b]) and torch.equal(after2, after)


@pytest.mark.parametrize("dtype,d,g", [(F, 40, 40), (B, 64, 64), (B, 30, 6)])
def test_inputs_and_gates_in_one_buffer(dtype, d, g):
    """As a projection gives them; the result over the inputs, the gates as they were."""
    import ddm_amd
    x, lam, off, state = make(2500, d, g, dtype, dtype, 11, 5)
    both = torch.cat([x, lam], 1).cuda()
    h, after = ddm_amd.gated_scan(both[:, :d], both[:, d:], off.cuda(), state.cuda(), scale="unit", out=both[:, :d])
    ref = gated64(x, lam, off, state, "unit")
    a, b = int(off[0]), int(off[-1])
    close(h[a:b], *(t[a:b] for t in ref["h"]), dtype)
    close(after, *ref["state"])
    assert torch.equal(both[:, d:].cpu(), lam) and torch.equal(both[:a, :d].cpu(), x[:a])


def test_one_row_of_gates_for_all_rows():
    import ddm_amd
    x, lam, off, state = make(900, 96, 12, F, F, 8, 4)
    one = lam[:1].expand(900, 12)
    ref = gated64(x, one.contiguous(), off, state, "ewma")
    h, after = ddm_amd.gated_scan(x.cuda(), lam[:1].cuda().expand(900, 12), offsets=off.cuda(), state=state.cuda(),
                                  scale="ewma")
    close(h, *ref["h"])
    close(after, *ref["state"])


@pytest.mark.parametrize("dtype", [F, B])
def test_broken_sequences_stay_apart(dtype):
    """NaN and infinities in one sequence, in its state, behind the last one: not in the others."""
    import ddm_amd
    x, lam, off, state = make(3000, 256, 256, dtype, dtype, 9, 8)
    d_h = torch.randn(x.shape).to(dtype)
    clean = ddm_amd.gated_scan(*on(x, lam, off, state))
    cleang = ddm_amd.gated_scan_grad(*on(x, lam), clean[0], d_h.cuda(), offsets=off.cuda(), state=state.cuda())
    a, b = int(off[4]), int(off[5])
    assert b - a > 2
    x2, s2, l2, dh2 = x.clone(), state.clone(), lam.clone(), d_h.clone()
    x2[a + 1] = math.inf
    x2[b - 1] = math.nan
    dh2[a] = dh2[b - 1] = math.nan
    s2[5] = math.nan
    for t in (x2, l2, dh2):
        t[:int(off[0])] = math.nan
        t[int(off[-1]):] = math.nan
    h, after = ddm_amd.gated_scan(*on(x2, l2, off, s2))
    got = ddm_amd.gated_scan_grad(*on(x2, l2), h, dh2.cuda(), offsets=off.cuda(), state=s2.cuda())
    ok = torch.ones(3000, dtype=torch.bool)
    ok[a:int(off[6])] = False
    for u, v in ((h, clean[0]), (got[0], cleang[0]), (got[1], cleang[1])):
        assert torch.equal(u.cpu()[ok], v.cpu()[ok])
    assert h.cpu()[b - 1].isnan().all() and h.cpu()[a + 1].isinf().all()
    keep = [0, 1, 2, 3, 6, 7]
    assert torch.equal(after.cpu()[keep], clean[1].cpu()[keep]) and torch.equal(got[2].cpu()[keep], cleang[2].cpu()[keep])


def test_no_rows():
    import ddm_amd
    state = torch.randn(3, 8, device="cuda")
    x = torch.empty(0, 8, device="cuda")
    off = torch.zeros(4, dtype=torch.int64, device="cuda")
    h, after = ddm_amd.gated_scan(x, x, offsets=off, state=state)
    assert h.shape == (0, 8) and torch.equal(after, state)
    d = ddm_amd.gated_scan_grad(x, x, h, h, offsets=off, state=state, d_state=state)
    assert torch.equal(d[2], state) and d[0].shape == (0, 8)
    h, after = ddm_amd.gated_scan(x, x)
    assert (after == 0).all() and after.shape == (1, 8)
    x = torch.randn(5, 8, device="cuda")
    h, after = ddm_amd.gated_scan(x, x, offsets=off, state=state)           # rows, but none in a sequence
    assert (h == 0).all() and torch.equal(after, state)
    h, after = ddm_amd.gated_scan(x, x, offsets=off[:1])                     # no sequence at all
    assert (h == 0).all() and after.shape == (0, 8)


@pytest.mark.parametrize("dtype,gate_dtype", [(F, F), (B, B), (B, F), (H, H)])
@pytest.mark.parametrize("n,d,g", [(1, 1, 1), (3, 7, 7), (256, 2048, 2048), (17, 100, 25), (5, 1024, 1), (33, 6, 2)])
def test_step(dtype, gate_dtype, n, d, g):
    import ddm_amd
    x, lam, _, _ = make(n, d, g, dtype, gate_dtype, n + d)
    state = torch.randn(n, d)
    off = torch.arange(n + 1)
    for scale in ("none", "ewma", "unit"):
        ref = gated64(x, lam, off, state, scale)
        own = state.cuda()
        h, after = ddm_amd.gated_step(*on(x, lam), own, scale=scale)
        close(h, *ref["h"], dtype)
        close(after, *ref["state"])
        h2, same = ddm_amd.gated_step(*on(x, lam), own, scale=scale, out_state=own)
        assert same is own and torch.equal(own, after) and torch.equal(h2, h)
        ref = gated64(x, lam, off, None, scale)
        close(ddm_amd.gated_step(*on(x, lam), scale=scale)[1], *ref["state"])


def test_prompt_then_tokens():
    """A prompt by the scan, then tokens by the step: the scan of all of it."""
    import ddm_amd
    x, lam, _, state = make(700, 128, 128, F, F, 12)
    xc, lc, sc = on(x, lam, state)
    _, s = ddm_amd.gated_scan(xc[:690], lc[:690], state=sc, scale="unit")
    rows = []
    for r in range(690, 700):
        h, s = ddm_amd.gated_step(xc[r:r + 1], lc[r:r + 1], s, scale="unit", out_state=s)
        rows.append(h)
    ref = gated64(x, lam, None, state, "unit")
    close(torch.cat(rows), ref["h"][0][690:], ref["h"][1][690:])
    close(s, *ref["state"])


def test_streams_and_captures():
    import ddm_amd
    sets = [on(*make(6000, 256, 16, B, B, s, 5)) for s in (20, 22, 24)]
    torch.cuda.synchronize()
    want = [ddm_amd.gated_scan(*s, scale="unit") for s in sets]
    d_h = torch.randn(6000, 256, device="cuda").to(B)
    wantg = [ddm_amd.gated_scan_grad(s[0], s[1], w[0], d_h, offsets=s[2], state=s[3], scale="unit")
             for s, w in zip(sets, want)]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    at_once = [ddm_amd.gated_scan(*sets[0], scale="unit", stream=st) for st in side]
    torch.cuda.synchronize()
    for got in at_once:
        assert torch.equal(got[0], want[0][0]) and torch.equal(got[1], want[0][1])
    bufs = [t.clone() for t in sets[0]]

    def both():
        h, s = ddm_amd.gated_scan(*bufs, scale="unit")
        return (h, s) + ddm_amd.gated_scan_grad(bufs[0], bufs[1], h, d_h, offsets=bufs[2], state=bufs[3], scale="unit")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = both()
        graphs.append((g, held))
    for k in range(6):
        for to, of in zip(bufs, sets[k % 3]):
            to.copy_(of)
        for g, held in graphs:
            g.replay()
        both()
        torch.cuda.synchronize()
        for _, held in graphs:
            for a, b in zip(held, want[k % 3] + wantg[k % 3]):
                assert torch.equal(a, b)


def test_charts_of_a_models_scores():
    """Scores of two streams of answers, then their exponentially weighted charts, carried over two calls."""
    import ddm_amd
    gen = torch.Generator().manual_seed(2)
    n, v = 4000, 300
    x = (torch.randn(n, v, generator=gen) * 2).to(B).cuda()
    t = torch.randint(0, v, (n,), generator=gen).cuda()
    r = ddm_amd.token_scores(x, t)
    signal = torch.stack([r.logprob, r.entropy], 1)
    lam = torch.full((1, 1), math.log(0.99), device="cuda")
    off = torch.tensor([0, 1500, 4000], device="cuda")
    h, _ = ddm_amd.gated_scan(signal, lam.expand(n, 1), offsets=off, scale="ewma")
    ref = gated64(signal.cpu(), lam.cpu().expand(n, 1).contiguous(), off.cpu(), None, "ewma")
    close(h, *ref["h"])
    # the same in two calls of half the rows each, the second stream cut in its middle
    _, s1 = ddm_amd.gated_scan(signal[:2000], lam.expand(2000, 1), offsets=torch.tensor([0, 1500, 2000], device="cuda"),
                               scale="ewma")
    h2, _ = ddm_amd.gated_scan(signal[2000:], lam.expand(2000, 1), state=s1[1:], scale="ewma")
    close(h2, *(q[2000:] for q in ref["h"]))


def test_a_stream_of_millions():
    """Over 64 groups of 64 tiles of one channel; the reference's steps composed by doubling, in float64."""
    import ddm_amd
    rows = 8_600_007
    gen = torch.Generator().manual_seed(6)
    x = torch.rand(rows, 1, generator=gen)
    lam = -torch.exp(torch.rand(rows, 1, generator=gen) * -7)
    off = torch.tensor([0, 4_000_000, rows])
    state = torch.tensor([[0.5], [0.25]])
    h, after = ddm_amd.gated_scan(*on(x, lam, off, state), scale="ewma")
    a, f = lam.double().exp().cuda(), (-torch.expm1(lam.double())).cuda()
    b = f * x.double().cuda()
    b[0] += a[0] * 0.5
    b[4_000_000] += a[4_000_000] * 0.25
    a[0] = a[4_000_000] = 0.0

    def compose(a, b):
        step = 1
        while step < rows:
            b = torch.cat([b[:step], b[step:] + a[step:] * b[:-step]])
            a = torch.cat([a[:step], a[step:] * a[:-step]])
            step *= 2
        return b
    want = compose(a, b).cpu()                      # everything is positive: the majorant is the state itself
    tol = compose(a, 10 * 2.0 ** -24 * want.cuda()).cpu()
    close(h, want, tol)
    last = [3_999_999, rows - 1]
    close(after, want[last], tol[last])


def test_beyond_four_gigabytes():
    """Rows whose bytes lie past 2^32, forward and backward: a sequence there is what it is by itself."""
    import ddm_amd
    rows, d, first = 1_100_000, 2048, 1_090_000
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(rows, d, dtype=B, device="cuda")
    for r in range(0, rows, 110_000):
        x[r:r + 110_000] = torch.randn(110_000, d, generator=gen, device="cuda")
    lam = -torch.rand(rows, 16, generator=gen, device="cuda").to(B)
    off = torch.tensor([0, first, rows], device="cuda")
    h, s = ddm_amd.gated_scan(x, lam, offsets=off, scale="ewma")
    few, fs = ddm_amd.gated_scan(x[first:], lam[first:], scale="ewma")
    # tiles begin at other rows, so steps are composed in another order: float32's, then bf16's rounding
    assert (s[1] - fs[0]).abs().max() < 1e-5
    assert (h[first:].float() - few.float()).abs().max() < 2.0 ** -6
    dx, dl, ds = ddm_amd.gated_scan_grad(x, lam, h, x, offsets=off, scale="ewma")
    fx, fl, fd = ddm_amd.gated_scan_grad(x[first:], lam[first:], h[first:], x[first:], scale="ewma")
    assert (ds[1] - fd[0]).abs().max() < 1e-4
    assert (dx[first:].float() - fx.float()).abs().max() < 2.0 ** -4
    assert (dl[first:].float() - fl.float()).abs().max() / fl.float().abs().max() < 2.0 ** -7



def nan_gates(x, lam, off, rows, channels):
    """The inputs with NaN for the gates of `rows`, and what float64 makes of them."""
    lam = lam.clone()
    for r in rows:
        lam[r, channels] = math.nan
    return x, lam, off


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("d,g", [(64, 64), (5, 5), (96, 6)])
@pytest.mark.parametrize("scale", ["none", "ewma", "unit"])
@pytest.mark.parametrize("where", [1, 40, -1])
def test_a_nan_gate_shows_wherever_it_counts(dtype, d, g, scale, where):
    """One in a sequence's second row, further on, and in its last: in h from there on, in the state after, in the
    gradients that it enters, and in nothing else."""
    x, lam, off, state = make(900, d, g, dtype, dtype, 21, 4)
    a, b = int(off[3]), int(off[4])
    assert b - a > 45
    x, lam, off = nan_gates(x, lam, off, [a + where if where > 0 else b - 1], slice(0, g, 2))
    check(x, lam, off, state, scale, True)


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("scale", ["ewma", "unit"])
def test_a_nan_gates_factor_without_a_state(dtype, scale):
    """The first row has no state that a NaN gate could meet; the input's factor is NaN all the same."""
    import ddm_amd
    x, lam, off, _ = make(300, 32, 32, dtype, dtype, 22, 4, state=False)
    lam[int(off[3]), ::3] = math.nan
    gen = torch.Generator().manual_seed(0)
    d_h, d_state = torch.randn(x.shape, generator=gen).to(dtype), torch.randn(4, 32, generator=gen)
    xc, lc, oc = on(x, lam, off)
    h, after = ddm_amd.gated_scan(xc, lc, offsets=oc, scale=scale)
    got = ddm_amd.gated_scan_grad(xc, lc, h, d_h.cuda(), offsets=oc, d_state=d_state.cuda(), scale=scale)
    ref = gated64(x, lam, off, None, scale, h.cpu(), d_h, d_state)
    close(h, *ref["h"], dtype)
    close(after, *ref["state"])
    close(got[0], *ref["d_x"], dtype)
    close(got[2], *ref["d_state"])
    # At a log gate of -50, a^2 = e^-100 lies under float32's normal numbers: rounding it is off by 2^-150 and not by a
    # share of it, so is rounding its product with x, and both are multiplied by the gradient (f = 1 there: d_x).
    want, tol = ref["d_log_a"]
    close(got[1], want, tol + 2.0 ** -150 * (x.double().abs() + 1) * ref["d_x"][0].abs(), dtype)
    h, after = ddm_amd.gated_step(*on(x, lam), scale=scale)
    ref = gated64(x, lam, torch.arange(301), None, scale)
    close(h, *ref["h"], dtype)
    close(after, *ref["state"])


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("seqs", [None, 4])
def test_a_nan_gate_in_a_first_row_without_a_state(dtype, seqs):
    """NaN times a state of 0 is NaN, in the scan as in the step, though nothing but the gate says so."""
    import ddm_amd
    x, lam, off, _ = make(300, 40, 20, dtype, dtype, 23, seqs, state=False)
    first = 0 if off is None else int(off[3])
    lam[first, 1::4] = math.nan
    check(x, lam, off, None, "none", True)
    h, after = ddm_amd.gated_step(*on(x, lam))
    assert torch.equal(h[first].isnan().cpu(), lam[first].isnan().repeat_interleave(2))
    one, state = ddm_amd.gated_scan(*on(x[first:first + 1], lam[first:first + 1]))
    assert torch.equal(one[0].isnan(), h[first].isnan()) and torch.equal(state[0].isnan(), after[first].isnan())


@pytest.mark.parametrize("dtype", [F, B, H])
@pytest.mark.parametrize("scale", ["none", "ewma", "unit"])
@pytest.mark.parametrize("value", [2.0 ** -22, 0.5, 60.0, math.inf])
def test_a_gate_over_one_counts_as_nan(dtype, scale, value):
    """Products of gates over 1 can overflow where the recurrence is finite (a state of 0), so there are none."""
    import ddm_amd
    x, lam, off, state = make(4000, 24, 12, dtype, dtype, 25, 5)
    at = [0, int(off[3]), int(off[4]) + 70, int(off[4]) + 71, 3999]
    x[int(off[4]):] = 0.0
    above, nan = lam.clone(), lam.clone()
    above[at, 1::3] = value
    nan[at, 1::3] = math.nan
    assert (above[at, 1::3] > 0).all()
    d_h = torch.randn(4000, 24, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    xc, oc, sc = on(x, off, state)

    def both(gates):
        h, after = ddm_amd.gated_scan(xc, gates, offsets=oc, state=sc, scale=scale)
        few = [0, int(off[3]), 3999]
        step = ddm_amd.gated_step(xc[few], gates[few], scale=scale)
        return (h, after) + ddm_amd.gated_scan_grad(xc, gates, h, d_h, offsets=oc, state=sc, scale=scale) + step
    for a, b in zip(both(above.cuda()), both(nan.cuda())):
        assert torch.equal(a.isnan(), b.isnan()) and a.isnan().any()
        assert torch.equal(a.nan_to_num(), b.nan_to_num())
    assert both(torch.zeros_like(lam).cuda())[0].isfinite().all()           # 0 itself is a gate of 1


def test_no_wait_gives_up():
    """Hundreds of tiles that wait for each other, forwards and backwards, on two streams."""
    import ddm_amd
    x, lam, _, state = make(40000, 128, 128, B, B, 30)
    args = on(x, lam, None, state)
    h, _ = ddm_amd.gated_scan(*args)
    torch.cuda.synchronize()
    for stream in (None, torch.cuda.Stream()):
        ddm_amd.gated_scan(*args, stream=stream)
        ddm_amd.gated_scan_grad(args[0], args[1], h, h, state=args[3], stream=stream)
    assert ddm_amd.wait_gave_up() is False and ddm_amd.wait_gave_up(0) is False


@pytest.mark.parametrize("dtype,gate_dtype", [(B, B), (B, F), (H, H), (H, F)])
@pytest.mark.parametrize("rows,d,g,seqs", [(1, 3, 1, None), (500, 64, 64, 6), (900, 257, 257, 3), (1000, 260, 65, 4), (600, 768, 12, 5),
                                           (9001, 2048, 32, 5), (70001, 256, 256, 3)])
def test_float32_h(dtype, gate_dtype, rows, d, g, seqs):
    """h as it was computed: no rounding of the state in it, nor in the gates' gradients."""
    import ddm_amd
    for k, scale in enumerate(("none", "ewma", "unit")):
        x, lam, off, state = make(rows, d, g, dtype, gate_dtype, rows + d + 2 * k + 1, seqs)
        xc, lc, oc, sc = on(x, lam, off, state)
        h, after = ddm_amd.gated_scan(xc, lc, offsets=oc, state=sc, scale=scale, dtype=F)
        assert h.dtype == F
        d_h = torch.randn(x.shape, generator=torch.Generator().manual_seed(k)).to(dtype)
        got = ddm_amd.gated_scan_grad(xc, lc, h, d_h.cuda(), offsets=oc, state=sc, scale=scale)
        ref = gated64(x, lam, off, state, scale, h.cpu(), d_h)
        close(h, *ref["h"])
        close(after, *ref["state"])
        close(got[0], *ref["d_x"], dtype)
        close(got[1], *ref["d_log_a"], gate_dtype)
        close(got[2], *ref["d_state"])
        short, same = ddm_amd.gated_scan(xc, lc, offsets=oc, state=sc, scale=scale)
        # not h.to(dtype) bit by bit: one instruction rounds a fused product to float16 at once, two round it twice;
        # either is within the bound of h and half a step of the type
        close(short, *ref["h"], dtype)
        assert torch.equal(same, after)


@pytest.mark.parametrize("dtype", [B, H])
def test_a_gates_gradient_without_a_rounded_state(dtype):
    """Float32 gates and h: d_log_a against the recurrence that is float64 throughout."""
    import ddm_amd
    x, lam, off, state = make(700, 96, 96, dtype, F, 41, 4)
    d_h = torch.randn(x.shape, generator=torch.Generator().manual_seed(3)).to(dtype)
    xc, lc, oc, sc = on(x, lam, off, state)
    h, _ = ddm_amd.gated_scan(xc, lc, offsets=oc, state=sc, dtype=F)
    _, d_a, _ = ddm_amd.gated_scan_grad(xc, lc, h, d_h.cuda(), offsets=oc, state=sc)
    exact, bound = gated64(x, lam, off, state, "none")["h"]
    ref = gated64(x, lam, off, state, "none", exact, d_h)
    # d_log_a = grad a h_{t-1}, and grad is d_x here: h_{t-1} is off by its bound and half a step of float32
    off_by = torch.zeros_like(bound)
    off_by[1:] = (bound + 2.0 ** -24 * exact.abs())[:-1]
    want, tol = ref["d_log_a"]
    close(d_a, want, tol + ref["d_x"][0].abs() * lam.double().exp() * off_by)


def test_float32_out_and_strides():
    import ddm_amd
    x, lam, off, state = make(600, 64, 64, B, B, 43, 5)
    args = on(x, lam, off, state)
    want, _ = ddm_amd.gated_scan(*args, scale="ewma", dtype=F)
    a, b = int(off[0]), int(off[-1])
    d_h = torch.randn(600, 64, device="cuda").to(B)
    grads = ddm_amd.gated_scan_grad(args[0], args[1], want, d_h, offsets=args[2], state=args[3], scale="ewma")
    for shift in (0, 1, 2):                              # a shift by one: no aligned pair of h
        wide = torch.full((600, 70), 7.0, device="cuda")
        out = wide[:, shift:shift + 64]
        h, _ = ddm_amd.gated_scan(*args, scale="ewma", out=out)
        assert h is out and (wide[:, :shift] == 7).all() and (wide[:, shift + 64:] == 7).all()
        assert (h[:a] == 7).all() and (h[b:] == 7).all()
        ref = gated64(x, lam, off, state, "ewma", h.cpu(), d_h.cpu())
        close(h[a:b], *(t[a:b] for t in ref["h"]))
        got = ddm_amd.gated_scan_grad(args[0], args[1], h, d_h, offsets=args[2], state=args[3], scale="ewma")
        for t, name in zip(got, ("d_x", "d_log_a", "d_state")):
            close(t, *ref[name], t.dtype)
        if shift == 0:
            assert all(torch.equal(t, u) for t, u in zip(got, grads))
