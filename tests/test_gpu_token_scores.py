"""token_scores and its gradient against float64 on the host: sizes around every launch shape,
masks, ties, rows with nothing left or with NaN, strides, streams, captures, and the run of
scores into the DDM scan."""
import math

import numpy as np
import pytest
import torch

from conftest import oracle_scan_c
from lm_reference import close, scores64, scores_grad64, scores_tolerance

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(n, v, dtype, seed, special=True):
    """Logits on the host with every kind of row, and targets on every kind of place."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, v, generator=g) * 3).to(dtype)
    t = torch.randint(0, v, (n,), generator=g)
    low = torch.finfo(dtype).min
    if special:
        for r in range(n):
            kind = r % 12
            if kind == 1:
                x[r] = -math.inf
            elif kind == 2:
                x[r] = low
            elif kind == 3:
                x[r, torch.rand(v, generator=g) < 0.5] = low
                x[r, t[r]] = 1.0
            elif kind == 4:
                x[r, torch.rand(v, generator=g) < 0.7] = -math.inf
            elif kind == 5:
                x[r] = -math.inf
                x[r, torch.randint(0, v, (1,), generator=g)] = 2.5
            elif kind == 6:
                x[r] = 0.75                                     # all equal
            elif kind == 7:
                x[r] = torch.randint(-1, 2, (v,), generator=g).to(dtype) * 0.0   # +0 and -0
            elif kind == 8:
                x[r] = torch.randint(0, 3, (v,), generator=g).to(dtype)          # many ties
            elif kind == 9:
                t[r] = -100
            elif kind == 10:
                t[r] = v
            elif kind == 11:
                t[r] = v - 1 if r % 2 else 0
    return x, t


def check_scores(x, t, top, temperature, r):
    ref = scores64(x, t, top, temperature)
    lp_tol, h_tol = scores_tolerance(x, ref, temperature)
    n = x.shape[0]
    assert torch.equal(r.rank.cpu(), ref["rank"])
    assert torch.equal(r.err.cpu()[:n], ref["err"]) and not r.err.cpu()[n:].any()
    if top:
        assert torch.equal(r.top_index.cpu(), ref["top_index"])
        close(r.top_logprob, ref["top_logprob"], lp_tol(ref["top_logprob"]))
    else:
        assert r.top_index is None and r.top_logprob is None
    close(r.logprob, ref["logprob"], lp_tol(ref["logprob"]))
    close(r.entropy, ref["entropy"], h_tol)
    return ref


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,top", [(13, 1, 1), (13, 2, 0), (30, 7, 5), (25, 8, 64), (25, 9, 2), (24, 64, 64),
                                     (13, 513, 20), (26, 1000, 33), (13, 2049, 7), (13, 4096, 64), (13, 4099, 1),
                                     (13, 20001, 20), (1, 70001, 64), (3, 131072, 20), (12, 262147, 5)])
def test_scores(dtype, n, v, top):
    import ddm_amd
    x, t = make(n, v, dtype, n * 1000 + v)
    r = ddm_amd.token_scores(x.cuda(), t.cuda(), top=top)
    check_scores(x, t, top, 1.0, r)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,top", [(13, 3, 2), (25, 129, 16), (13, 2047, 0), (13, 9001, 64), (2, 50021, 20)])
@pytest.mark.parametrize("temperature", [0.3, 1.7])
def test_gradient(dtype, n, v, top, temperature):
    import ddm_amd
    x, t = make(n, v, dtype, n + v)
    g = torch.Generator().manual_seed(v)
    d = {"d_logprob": torch.randn(n, generator=g), "d_entropy": torch.randn(n, generator=g)}
    if top:
        d["d_top"] = torch.randn(n, top, generator=g)
    xc, tc = x.cuda(), t.int().cuda()
    r = ddm_amd.token_scores(xc, tc, top=top, temperature=temperature)
    ref = check_scores(x, t, top, temperature, r)
    for use in (["d_logprob"], ["d_entropy"], list(d)):
        given = {k: d[k] for k in use}
        want, tol = scores_grad64(x, t, ref, temperature, **given)
        got = ddm_amd.token_scores_grad(xc, tc, r, **{k: a.cuda() for k, a in given.items()})
        close(got, want, tol, dtype)
    assert torch.equal(xc.cpu().view(torch.uint8), x.view(torch.uint8))     # read only
    own = ddm_amd.token_scores_grad(xc, tc, r, **{k: a.cuda() for k, a in d.items()}, out=xc)
    assert own is xc and torch.equal(own.view(torch.uint8), got.view(torch.uint8))


def test_gradient_against_differences():
    """The reference's own gradient: central differences of its scores in float64."""
    x, t = make(9, 40, torch.float32, 5, special=False)
    g = torch.Generator().manual_seed(1)
    d = {"d_logprob": torch.randn(9, generator=g), "d_entropy": torch.randn(9, generator=g),
         "d_top": torch.randn(9, 6, generator=g)}

    def total(z):
        r = scores64(z, t, 6, 0.8)
        return (d["d_logprob"] * r["logprob"] + d["d_entropy"] * r["entropy"] + (d["d_top"] * r["top_logprob"]).sum(1))
    z = x.double()
    want, _ = scores_grad64(z, t, scores64(z, t, 6, 0.8), 0.8, **d)
    h = 1e-6
    for c in range(40):
        e = torch.zeros_like(z)
        e[:, c] = h
        diff = (total(z + e) - total(z - e)) / (2 * h)
        # second order h^2 ~ 1e-12, cancellation 1e-16 * 10 / h = 1e-9
        assert (diff - want[:, c]).abs().max() < 1e-7


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift,pad", [(0, 8), (1, 5), (3, 0), (7, 9)])
def test_strides_and_alignment(dtype, shift, pad):
    import ddm_amd
    for n, v in ((13, 777), (3, 30011)):
        x, t = make(n, v, dtype, shift)
        wide = torch.full((n, shift + v + pad), math.nan, dtype=dtype, device="cuda")
        view = wide[:, shift:shift + v]
        view.copy_(x)
        r = ddm_amd.token_scores(view, t.cuda(), top=9)
        ref = check_scores(x, t, 9, 1.0, r)
        out = torch.full((n, v + 3), 7.0, dtype=dtype, device="cuda")
        d = torch.randn(n, generator=torch.Generator().manual_seed(2))
        got = ddm_amd.token_scores_grad(view, t.cuda(), r, d_logprob=d.cuda(), out=out[:, 1:v + 1])
        want, tol = scores_grad64(x, t, ref, 1.0, d_logprob=d)
        close(got, want, tol, dtype)
        assert (out[:, 0] == 7).all() and (out[:, v + 1:] == 7).all()
        assert wide[:, :shift].isnan().all() and wide[:, shift + v:].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("where", [0, 511, 12345])
def test_rows_with_nan_and_infinity(dtype, where):
    import ddm_amd
    v = 16385
    x, t = make(12, v, dtype, 3, special=False)
    x[1, where] = math.nan
    x[3, where] = math.inf
    x[5] = math.nan
    x[7] = math.inf
    t[9] = -1
    x[9, where] = math.nan
    r = ddm_amd.token_scores(x.cuda(), t.cuda(), top=12)
    ref = check_scores(x, t, 12, 1.0, r)
    d = torch.ones(12)
    want, tol = scores_grad64(x, t, ref, 1.0, d_logprob=d, d_entropy=d)
    got = ddm_amd.token_scores_grad(x.cuda(), t.cuda(), r, d_logprob=d.cuda(), d_entropy=d.cuda())
    close(got, want, tol, dtype)


def test_no_rows():
    import ddm_amd
    x = torch.empty(0, 100, device="cuda")
    t = torch.empty(0, dtype=torch.int64, device="cuda")
    r = ddm_amd.token_scores(x, t, top=3)
    assert r.logprob.shape == (0,) and r.top_index.shape == (0, 3) and r.err.shape == (0,)
    assert ddm_amd.token_scores_grad(x, t, r, d_logprob=r.logprob).shape == (0, 100)


def test_another_stream_and_two_calls_at_once():
    import ddm_amd
    x, t = make(40, 33000, torch.bfloat16, 8)
    xc, tc = x.cuda(), t.cuda()
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    rs = [ddm_amd.token_scores(xc, tc, top=20, stream=s) for s in side]
    torch.cuda.synchronize()
    for r in rs:
        check_scores(x, t, 20, 1.0, r)


def test_captured_and_replayed():
    import ddm_amd
    xs = [make(5, 40000, torch.bfloat16, k)[0].cuda() for k in range(3)]
    t = make(5, 40000, torch.bfloat16, 0)[1].cuda()
    d = torch.randn(5, device="cuda")
    buf = xs[0].clone()

    def both():
        r = ddm_amd.token_scores(buf, t, top=8)
        return r, ddm_amd.token_scores_grad(buf, t, r, d_logprob=d, d_entropy=d)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both()
    torch.cuda.current_stream().wait_stream(s)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        r1, dx1 = both()
    with torch.cuda.graph(g2):
        r2, dx2 = both()
    for k in range(6):
        buf.copy_(xs[k % 3])
        r, dx = both()
        for g, rg, dg in ((g1, r1, dx1), (g2, r2, dx2)):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(dg.view(torch.int16), dx.view(torch.int16))
            for a, b in zip(rg[:6], r[:6]):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_scores_into_the_drift_scan(oracle_lib):
    """A monitored run: the answers get worse half way, the flags go to the scan on the device."""
    import ddm_amd
    from ddm_amd import kernels
    n, v = 3000, 1000
    g = torch.Generator().manual_seed(4)
    x = torch.randn(n, v, generator=g)
    t = torch.randint(0, v, (n,), generator=g)
    right = torch.rand(n, generator=g) < torch.where(torch.arange(n) < n // 2, 0.97, 0.55)
    x[right, t[right]] += 20.0
    r = ddm_amd.token_scores(x.to(torch.bfloat16).cuda(), t.cuda())
    ref = scores64(x.to(torch.bfloat16), t, 0, 1.0)
    off = torch.tensor([0, n], device="cuda")
    nb = -(-n // 100)
    ev = torch.empty(nb, 2, dtype=torch.int32, device="cuda")
    state = torch.from_numpy(kernels.fresh_states(1).view(np.uint8)).cuda()
    nev = torch.empty(1, dtype=torch.int64, device="cuda")
    kernels.scan_streams(r.err, off, kernels.params_struct(), state, torch.zeros(1, dtype=torch.int64, device="cuda"),
                         nb, ev, nev=nev, mode=1)
    want, _, _, _ = oracle_scan_c(oracle_lib, ref["err"].numpy(), np.array([0, n]), mode=1)
    assert np.array_equal(ev.cpu().numpy(), want) and (want[:, 1] >= 0).any()


def test_beyond_four_gigabytes():
    """Rows whose bytes lie past 2^32 score as the same rows by themselves."""
    import ddm_amd
    n, v = 33000, 70000
    x = torch.empty(n, v, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    for r in range(0, n, 11000):
        x[r:r + 11000] = torch.randn(11000, v, generator=g, device="cuda") * 3
    t = torch.randint(0, v, (n,), generator=g, device="cuda")
    d = torch.randn(n, generator=g, device="cuda")
    r = ddm_amd.token_scores(x, t, top=5)
    dx = ddm_amd.token_scores_grad(x, t, r, d_logprob=d)
    for a in (0, 15000, n - 40):
        part, pt = x[a:a + 40], t[a:a + 40]
        few = ddm_amd.token_scores(part, pt, top=5)
        assert torch.equal(few.rank, r.rank[a:a + 40]) and torch.equal(few.top_index, r.top_index[a:a + 40])
        # parts of another size sum in another order
        assert (few.logprob - r.logprob[a:a + 40]).abs().max() < 1e-4
        few_dx = ddm_amd.token_scores_grad(part, pt, few, d_logprob=d[a:a + 40])
        assert (few_dx.float() - dx[a:a + 40].float()).abs().max() < 2.0 ** -7
    ref = scores64(x[n - 3:].cpu(), t[n - 3:].cpu(), 5, 1.0)
    assert torch.equal(r.rank[n - 3:].cpu(), ref["rank"])
    close(r.logprob[n - 3:], ref["logprob"], scores_tolerance(x[:1].cpu(), ref, 1.0)[0](ref["logprob"]))


def test_timer():
    import ddm_amd
    from ddm_amd.kernels import LaunchTimer
    x, t = make(30, 50000, torch.bfloat16, 1)
    timer = LaunchTimer()
    ddm_amd.token_scores(x.cuda(), t.cuda(), top=3, timer=timer)
    torch.cuda.synchronize()
    assert 0.0 < timer.elapsed_ms() < 1000.0


def test_tiny_and_huge_temperatures():
    import ddm_amd
    x, t = make(12, 3000, torch.float32, 4, special=False)
    for temperature in (1e-3, 1e-30, 1e5, 1e30):
        r = ddm_amd.token_scores(x.cuda(), t.cuda(), top=4, temperature=temperature)
        check_scores(x, t, 4, temperature, r)


def test_alternatives_beyond_the_row_are_none():
    import ddm_amd
    x, t = make(13, 1000, torch.bfloat16, 5)
    xc, tc = x.cuda(), t.cuda()
    r = ddm_amd.token_scores(xc, tc, top=4)
    d = torch.randn(13, 4, generator=torch.Generator().manual_seed(6)).cuda()
    none, beyond = r.top_index.clone(), r.top_index.clone()
    none[:, 1::2] = -1
    beyond[:, 1] = 1000
    beyond[:, 3] = 2**31 - 1
    want = ddm_amd.token_scores_grad(xc, tc, r._replace(top_index=none), d_top=d)
    got = ddm_amd.token_scores_grad(xc, tc, r._replace(top_index=beyond), d_top=d)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v", [(13, 517), (12, 9001)])
def test_gradient_beside_the_logits(dtype, n, v):
    """Two halves of one buffer; the logits stay as they were."""
    import ddm_amd
    x, t = make(n, v, dtype, 9)
    both = torch.zeros(n, 2 * v, dtype=dtype, device="cuda")
    both[:, :v] = x.cuda()
    r = ddm_amd.token_scores(both[:, :v], t.cuda())
    d = torch.randn(n, generator=torch.Generator().manual_seed(1)).cuda()
    want = ddm_amd.token_scores_grad(x.cuda(), t.cuda(), r, d_logprob=d)
    got = ddm_amd.token_scores_grad(both[:, :v], t.cuda(), r, d_logprob=d, out=both[:, v:])
    # the same numbers; a product that is -0 may come as +0, by the instruction that rounds it to float16
    assert ((got == want) | (got.isnan() & want.isnan())).all()
    assert torch.equal(both[:, :v].cpu().view(torch.uint8), x.view(torch.uint8))


@pytest.mark.parametrize("v,shift", [(524285, 0), (524286, 0), (524287, 0), (524288, 0), (524288, 1), (524286, 3), (524287, 2)])
@pytest.mark.parametrize("top", [0, 20])
def test_the_longest_rows_to_their_end(v, shift, top):
    """Float32 rows of most columns, aligned or not: what counts lies in their last three columns."""
    import ddm_amd
    n = 3
    g = torch.Generator().manual_seed(v + shift)
    x = torch.randn(n, v, generator=g)
    x[:, -3:] += torch.tensor([12.0, 14.0, 13.0])
    x[1, -1] = 20.0
    t = torch.tensor([v - 1, v - 2, v - 3])
    flat = torch.zeros(shift + n * v, device="cuda")
    view = flat[shift:].view(n, v)
    view.copy_(x)
    r = ddm_amd.token_scores(view, t.cuda(), top=top)
    ref = check_scores(x, t, top, 1.0, r)
    d = torch.randn(n, generator=g)
    want, tol = scores_grad64(x, t, ref, 1.0, d_logprob=d, d_entropy=d)
    close(ddm_amd.token_scores_grad(view, t.cuda(), r, d_logprob=d.cuda(), d_entropy=d.cuda()), want, tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [1.0, 3e37, 6e37, 3e38])
@pytest.mark.parametrize("v", [2000, 4001, 40000])
def test_rows_with_infinity_at_huge_temperatures(dtype, temperature, v):
    """+inf behind finite entries of its lane, and before them: NaN, rank and indexes -1, error 1."""
    import ddm_amd
    x, t = make(12, v, dtype, 7, special=False)
    x[1, v - 1] = x[3, 0] = x[5, v // 2] = math.inf
    x[7, v - 1000] = math.nan
    for n in (12, 8):
        r = ddm_amd.token_scores(x[:n].cuda(), t[:n].cuda(), top=6, temperature=temperature)
        check_scores(x[:n], t[:n], 6, temperature, r)


def saved(make_buffer, write):
    """Whether autograd refuses a backward pass whose saved tensor `write` has overwritten."""
    leaf = make_buffer().requires_grad_()
    buf = leaf * 1.0
    total = buf.pow(2).sum()                            # keeps buf
    write(buf.detach())
    try:
        total.backward()
    except RuntimeError as e:
        return "inplace" in str(e)
    return False


def test_results_over_saved_tensors():
    import ddm_amd
    n, v = 5, 300
    t = torch.zeros(n, dtype=torch.int64, device="cuda")
    x = torch.randn(n, v, device="cuda")
    r = ddm_amd.token_scores(x, t, top=4)
    d = torch.ones(n, device="cuda")
    assert saved(x.clone, lambda b: ddm_amd.token_scores_grad(b, t, r, d_logprob=d, out=b))
    assert saved(x.clone, lambda b: ddm_amd.token_scores_grad(x, t, r, d_logprob=d, out=b))
    assert saved(x.clone, lambda b: ddm_amd.topk_distill(b, r.top_index, r.top_logprob, out=b))
    assert saved(x.clone, lambda b: ddm_amd.gated_scan(b, -x.abs(), out=b))
    assert saved(x.clone, lambda b: ddm_amd.gated_step(x, -x.abs(), b, out_state=b))
    assert not saved(x.clone, lambda b: ddm_amd.token_scores_grad(b, t, r, d_logprob=d))
    assert not saved(x.clone, lambda b: ddm_amd.gated_scan(b, -x.abs()))
    with torch.inference_mode():
        y = x.clone()
        ddm_amd.token_scores_grad(y, t, r, d_logprob=d, out=y)


def test_timers_of_calls_without_rows():
    import ddm_amd
    from ddm_amd.kernels import LaunchTimer
    x, t = torch.empty(0, 100, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda")
    r = ddm_amd.token_scores(x, t, top=2)
    for call in (lambda timer: ddm_amd.token_scores(x, t, timer=timer),
                 lambda timer: ddm_amd.token_scores_grad(x, t, r, timer=timer),
                 lambda timer: ddm_amd.topk_distill(x, r.top_index, r.top_logprob, grad=True, timer=timer),
                 lambda timer: ddm_amd.gated_step(x, x, timer=timer),
                 lambda timer: ddm_amd.gated_scan(x, x, timer=timer),
                 lambda timer: ddm_amd.gated_scan_grad(x, x, x, x, timer=timer)):
        timer = LaunchTimer()
        call(timer)
        torch.cuda.synchronize()
        assert 0.0 <= timer.elapsed_ms() < 1000.0
