"""topk_distill against float64 on the host: both tails, every launch shape, teachers with
repeats, gaps and indexes that are none, students with masks, and a refit run from one model's
token_scores."""
import math

import pytest
import torch

from lm_reference import close, distill64

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(n, v, k, dtype, seed, full=False):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, v, generator=g) * 3).to(dtype)
    index = torch.stack([torch.randperm(v, generator=g)[:k] if k <= v else torch.randint(0, v, (k,), generator=g)
                         for _ in range(n)])
    mass = 1.0 if full else 0.5 + 0.45 * torch.rand(n, 1, generator=g).double()
    logprob = torch.log_softmax(torch.randn(n, k, generator=g).double() * 2, 1) + torch.tensor(1.0).double().mul(mass).log()
    logprob = logprob.float()
    for r in range(n):
        kind = r % 11
        if kind == 1 and k > 2:
            index[r, k - 1] = index[r, 0]                  # a repeat
            index[r, k // 2] = index[r, 0]
        elif kind == 2:
            index[r, k // 2] = -1
            index[r, 0] = v if k > 1 else index[r, 0]
        elif kind == 3:
            index[r] = -1                                   # nothing given
        elif kind == 4:
            x[r, torch.rand(v, generator=g) < 0.5] = -math.inf
            x[r, index[r]] = 1.0                            # the student excludes others
        elif kind == 5:
            x[r, index[r, 0]] = -math.inf                   # ... and what the teacher expects
        elif kind == 6:
            logprob[r, k // 2] = -math.inf
        elif kind == 7:
            x[r] = -math.inf
        elif kind == 8:
            keep = x[r, index[r]].clone()
            x[r] = -math.inf                                # nothing outside what is given
            x[r, index[r]] = keep
        elif kind == 9:
            x[r, index[r]] += 30.0                          # the others' share far below float32's step of 1
    return x, index, logprob


def check(x, index, logprob, tail, temperature, weight, got_loss, got_grad):
    loss, tol, dx, dx_tol = distill64(x, index, logprob, tail, temperature, weight)
    close(got_loss, loss, tol)
    if got_grad is not None:
        close(got_grad, dx, dx_tol, x.dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail,temperature", [("rest", 1.0), ("renorm", 1.0), ("renorm", 2.5)])
@pytest.mark.parametrize("n,v,k", [(22, 1, 1), (22, 5, 3), (22, 40, 64), (22, 64, 64), (22, 513, 16), (33, 3000, 33),
                                   (22, 4100, 1), (12, 20001, 64), (300, 5000, 7), (280, 30000, 20), (257, 70001, 64),
                                   (1, 131072, 64), (5, 200003, 17)])
def test_distill(dtype, tail, temperature, n, v, k):
    import ddm_amd
    x, index, logprob = make(n, v, k, dtype, n + v + k)
    g = torch.Generator().manual_seed(n)
    weight = torch.rand(n, generator=g) * (64.0 if dtype == torch.float16 else 1.0)
    weight[::5] = 0.0
    args = [t.cuda() for t in (x, index, logprob)]
    loss, none = ddm_amd.topk_distill(*args, tail=tail, temperature=temperature)
    assert none is None
    both, grad = ddm_amd.topk_distill(*args, tail=tail, temperature=temperature, weight=weight.cuda(), grad=True)
    check(x, index, logprob, tail, temperature, weight, loss, grad)
    check(x, index, logprob, tail, temperature, None, both, None)
    # over the logits themselves
    own, over = ddm_amd.topk_distill(args[0], args[1].int(), args[2], tail=tail, temperature=temperature,
                                     weight=weight.cuda(), out=args[0])
    assert over is args[0] and torch.equal(over.view(torch.uint8), grad.view(torch.uint8))
    assert torch.equal(own.view(torch.int32), both.view(torch.int32))


@pytest.mark.parametrize("dtype", TYPES)
def test_complete_teacher(dtype):
    """All of the vocabulary is given: no remainder, whatever float32 makes of the sum."""
    import ddm_amd
    x, index, logprob = make(22, 50, 50, dtype, 1, full=True)
    rows = [r for r in range(22) if r % 11 not in (1, 2, 3, 6)]
    x, index, logprob = x[rows], index[rows], logprob[rows]
    loss, grad = ddm_amd.topk_distill(x.cuda(), index.cuda(), logprob.cuda(), grad=True)
    check(x, index, logprob, "rest", 1.0, None, loss, grad)


@pytest.mark.parametrize("tail,temperature", [("rest", 1.0), ("renorm", 1.7)])
def test_reference_gradient_against_differences(tail, temperature):
    x, index, logprob = make(1, 30, 6, torch.float32, 3)
    x = x.double()
    want = distill64(x, index, logprob, tail, temperature)[2]
    h = 1e-6
    for c in range(30):
        e = torch.zeros_like(x)
        e[:, c] = h
        up, down = (distill64(z, index, logprob, tail, temperature)[0] for z in (x + e, x - e))
        # second order h^2, cancellation 1e-16 * 10 / h = 1e-9
        assert ((up - down) / (2 * h) - want[:, c]).abs().max() < 1e-7


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v", [(11, 300), (300, 9001), (11, 40001)])
@pytest.mark.parametrize("shift", [0, 1, 5])
def test_strides_and_broken_rows(dtype, n, v, shift):
    import ddm_amd
    x, index, logprob = make(n, v, 9, dtype, shift)
    x[0, index[0, 2]] = math.nan
    x[6, (index[6].max() + 1) % v] = math.inf
    logprob[10 % n, 0] = math.nan
    wide = torch.full((n, shift + v + 3), math.nan, dtype=dtype, device="cuda")
    wide[:, shift:shift + v] = x.cuda()
    out = torch.full((n, v + 5), 7.0, dtype=dtype, device="cuda")
    for tail in ("rest", "renorm"):
        loss, grad = ddm_amd.topk_distill(wide[:, shift:shift + v], index.cuda(), logprob.cuda(), tail=tail,
                                          out=out[:, 2:2 + v])
        want = list(distill64(x, index, logprob, tail, 1.0))
        assert loss[[0, 6, 10 % n]].isnan().all() and grad[[0, 6, 10 % n]].isnan().all()
        sound = [r for r in range(n) if r not in (0, 6, 10 % n)]
        close(loss[sound], want[0][sound], want[1][sound])
        close(grad[sound], want[2][sound], want[3][sound], dtype)
        assert (out[:, :2] == 7).all() and (out[:, 2 + v:] == 7).all()


def test_nothing_to_do():
    import ddm_amd
    x = torch.randn(0, 50, device="cuda")
    i, lp = torch.zeros(0, 4, dtype=torch.int32, device="cuda"), torch.zeros(0, 4, device="cuda")
    loss, grad = ddm_amd.topk_distill(x, i, lp, grad=True)
    assert loss.shape == (0,) and grad.shape == (0, 50)
    x = torch.randn(3, 50, device="cuda")
    i, lp = torch.zeros(3, 0, dtype=torch.int32, device="cuda"), torch.zeros(3, 0, device="cuda")
    for tail in ("rest", "renorm"):
        loss, grad = ddm_amd.topk_distill(x, i, lp, tail=tail, grad=True)
        assert (loss == 0).all() and grad.abs().max() <= 2.0 ** -20    # p * (1 - q_rest / p_rest) of rounded ones


def test_captured_and_replayed():
    import ddm_amd
    sets = [make(300, 20000, 32, torch.bfloat16, s) for s in range(3)]
    x, index, logprob = (t.cuda().clone() for t in sets[0])
    few = x[:3]

    def both():
        a = ddm_amd.topk_distill(x, index, logprob, grad=True)
        return a + ddm_amd.topk_distill(few, index[:3], logprob[:3], grad=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for r in range(6):
        for to, of in zip((x, index, logprob), sets[r % 3]):
            to.copy_(of)
        want = both()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_refit_on_a_teachers_answers():
    """token_scores gives a teacher's alternatives; a student's logits descend on their loss."""
    import ddm_amd
    g = torch.Generator().manual_seed(0)
    n, v = 64, 3000
    teacher = (torch.randn(n, v, generator=g) * 3).to(torch.bfloat16).cuda()
    student = torch.randn(n, v, generator=g).cuda()
    t = torch.zeros(n, dtype=torch.int32, device="cuda")
    kept = ddm_amd.token_scores(teacher, t, top=48)
    loss, grad = ddm_amd.topk_distill(student, kept.top_index, kept.top_logprob, grad=True)
    check(student.cpu(), kept.top_index.cpu(), kept.top_logprob.cpu(), "rest", 1.0, None, loss, grad)
    # a teacher distilled into itself: loss and gradient are the rounding of the kept log probabilities
    same, flat = ddm_amd.topk_distill(teacher.float(), kept.top_index, kept.top_logprob, grad=True)
    want = distill64(teacher.float().cpu(), kept.top_index.cpu(), kept.top_logprob.cpu(), "rest", 1.0)
    close(same, want[0], want[1])
    close(flat, want[2], want[3])


def test_calls_on_several_streams_at_once():
    """Launches whose workgroups wait for each other, several in flight: each finishes, and is right."""
    import ddm_amd
    x, index, logprob = (t.cuda() for t in make(600, 60001, 20, torch.bfloat16, 9))
    lam = -torch.rand(9000, 1024, device="cuda").bfloat16()
    h_in = torch.randn(9000, 1024, device="cuda").bfloat16()
    want = ddm_amd.topk_distill(x, index, logprob, grad=True)
    want_h = ddm_amd.gated_scan(h_in, lam, scale="unit")
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for _ in range(3):
        for k, s in enumerate(streams):
            got.append(ddm_amd.gated_scan(h_in, lam, scale="unit", stream=s) if k % 2 else
                       ddm_amd.topk_distill(x, index, logprob, grad=True, stream=s))
    torch.cuda.synchronize()
    for k, g in enumerate(got):
        for a, b in zip(g, want_h if k % 2 else want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("tail,temperature", [("rest", 1.0), ("renorm", 1.0), ("renorm", 1.5)])
@pytest.mark.parametrize("v,shift", [(524285, 0), (524286, 0), (524287, 0), (524288, 0), (524288, 1), (524286, 3), (524287, 2)])
def test_the_longest_rows_to_their_end(v, shift, tail, temperature):
    """Float32 rows of most columns, aligned or not: the student's mass lies in their last three columns, one of
    which the teacher names."""
    import ddm_amd
    n, k = 3, 17
    x, index, logprob = make(n, v, k, torch.float32, v + shift)
    index[:] = torch.randint(0, v - 3, (n, k), generator=torch.Generator().manual_seed(v))
    index[:, 3] = v - 1 - torch.arange(n)
    x[:, -3:] = torch.tensor([12.0, 14.0, 13.0])
    flat = torch.zeros(shift + n * v, device="cuda")
    view = flat[shift:].view(n, v)
    view.copy_(x)
    args = (view, index.cuda(), logprob.cuda())
    loss, _ = ddm_amd.topk_distill(*args, tail=tail, temperature=temperature)
    both, grad = ddm_amd.topk_distill(*args, tail=tail, temperature=temperature, grad=True)
    check(x, index, logprob, tail, temperature, None, loss, None)
    check(x, index, logprob, tail, temperature, None, both, grad)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [2.0, 6e37, 3e38])
@pytest.mark.parametrize("v", [2000, 4001, 40000])
def test_students_with_infinity_at_huge_temperatures(dtype, temperature, v):
    import ddm_amd
    x, index, logprob = make(11, v, 9, dtype, 5)
    x[0, v - 1] = x[2, v // 2] = math.inf
    loss, grad = ddm_amd.topk_distill(x.cuda(), index.cuda(), logprob.cuda(), tail="renorm", temperature=temperature,
                                      grad=True)
    alone, _ = ddm_amd.topk_distill(x.cuda(), index.cuda(), logprob.cuda(), tail="renorm", temperature=temperature)
    want = distill64(x, index, logprob, "renorm", temperature)
    assert loss[[0, 2]].isnan().all() and alone[[0, 2]].isnan().all() and grad[[0, 2]].isnan().all()
    sound = [r for r in range(11) if r not in (0, 2)]
    close(loss[sound], want[0][sound], want[1][sound])
    close(alone[sound], want[0][sound], want[1][sound])


def test_a_wait_that_gives_up_says_so():
    import ddm_amd
    from ddm_amd import _capi
    args = [t.cuda() for t in make(64, 60000, 16, torch.float32, 3)]
    want = ddm_amd.topk_distill(*args, grad=True)
    assert not ddm_amd.wait_gave_up()
    _capi.check(_capi.lib.ddm_wait_limit(0), "limit")
    try:
        _, grad = ddm_amd.topk_distill(*args, grad=True)
        assert ddm_amd.wait_gave_up() and (grad.isnan() & ~want[1].isnan()).any()
    finally:
        _capi.check(_capi.lib.ddm_wait_limit(1 << 22), "limit")
    again = ddm_amd.topk_distill(*args, grad=True)
    assert all(torch.equal(a.view(torch.int32), b.view(torch.int32)) for a, b in zip(again, want))
    assert not ddm_amd.wait_gave_up()
