"""What the language-model calls refuse, on the host: nothing is launched."""
import ctypes

import pytest
import torch

from ddm_amd import _capi, gated, tokens

X = torch.zeros(4, 10)
T = torch.zeros(4, dtype=torch.int64)


def scores(n=4, top=0):
    return tokens.TokenScores(torch.zeros(n), torch.zeros(n), torch.zeros(n, dtype=torch.int32),
                              torch.zeros(16, dtype=torch.uint8), torch.zeros(n, top) if top else None,
                              torch.zeros(n, top, dtype=torch.int32) if top else None, torch.zeros(n, 2), 1.0)


@pytest.mark.parametrize("args,kw,error", [
    ((X, T), {}, "on the GPU"),
    ((X[0], T), {}, "two dimensions"),
    ((X.double(), T), {}, "type"),
    ((X.t(), T), {}, "contiguous"),
    ((X.expand(4, 10)[:1].expand(4, 10), T), {}, "overlap"),
    ((torch.zeros(4, 0), T), {}, "columns"),
    ((torch.zeros(1, tokens.MAX_COLUMNS + 1), T[:1]), {}, "columns"),
    ((X, T[:3]), {}, "targets"),
    ((X, T.float()), {}, "targets"),
    ((X, T), {"top": 65}, "top"),
    ((X, T), {"top": -1}, "top"),
    ((X, T), {"temperature": 0.0}, "temperature"),
    ((X, T), {"temperature": float("nan")}, "temperature"),
    ((X, T), {"temperature": float("inf")}, "temperature"),
])
def test_token_scores(args, kw, error):
    with pytest.raises((ValueError, TypeError), match=error):
        tokens.token_scores(*args, **kw)


@pytest.mark.parametrize("args,kw,error", [
    ((X, T, scores()), {}, "on the GPU"),
    ((X, T, scores(3)), {}, "stats"),
    ((X, T, scores()), {"d_logprob": torch.zeros(3)}, "d_logprob"),
    ((X, T, scores()), {"d_entropy": torch.zeros(4, dtype=torch.float64)}, "d_entropy"),
    ((X, T, scores()), {"d_top": torch.zeros(4, 2)}, "no alternatives"),
    ((X, T, scores(top=3)), {"d_top": torch.zeros(4, 2)}, "d_top"),
    ((X, T, scores()), {"out": torch.zeros(4, 9)}, "out"),
    ((X, T, scores()), {"out": torch.zeros(4, 10, dtype=torch.bfloat16)}, "out"),
    ((torch.zeros(50).as_strided((4, 10), (10, 1), 0), T, scores()), {}, "on the GPU"),
])
def test_token_scores_grad(args, kw, error):
    with pytest.raises((ValueError, TypeError), match=error):
        tokens.token_scores_grad(*args, **kw)


def test_gradient_over_a_shifted_view_of_the_logits():
    base = torch.zeros(5, 10)
    with pytest.raises(ValueError, match="overlaps"):
        tokens.token_scores_grad(base[:4], T, scores(), out=base[1:])


def last_error():
    return _capi.lib.ddm_last_error().decode()


def test_entry_points_check_before_they_launch():
    one = ctypes.c_void_p(256)          # never read: every call below is refused
    score = lambda dtype=0, n=4, v=10, ld=10, tb=8, temp=1.0, top=0, x=one: _capi.lib.ddm_token_scores(  # noqa: E731
        x, dtype, n, v, ld, one, tb, temp, top, one, one, one, one, one, None, None, None, None, None, None)
    for kw, text in (({"dtype": 3}, "type"), ({"v": 0}, "columns"), ({"v": 1 << 20, "ld": 1 << 20}, "columns"),
                     ({"ld": 9}, "stride"), ({"n": -1}, "rows"), ({"n": 1 << 40}, "rows"), ({"tb": 2}, "targets"),
                     ({"temp": 0.0}, "temperature"), ({"temp": 1e-40}, "temperature"), ({"temp": float("inf")}, "temperature"), ({"top": 65}, "alternatives"),
                     ({"top": 2}, "null"), ({"x": None}, "null"), ({"v": 100000, "ld": 100000}, "null")):
        assert score(**kw) == _capi.DDM_E_ARG and text in last_error(), (kw, last_error())
    assert score(n=0) == 0
    assert _capi.lib.ddm_token_scores_grad(one, 0, 4, 10, 10, one, 8, 1.0, 0, one, one, None, None, None, None, one, 9,
                                           None, None, None) == _capi.DDM_E_ARG and "stride" in last_error()
    assert _capi.lib.ddm_token_scores_scratch_bytes(4, 100, 0, 3) == 0
    assert _capi.lib.ddm_token_scores_scratch_bytes(4, 100000, 0, 3) > 0


I, LP = torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4, 3)


@pytest.mark.parametrize("args,kw,error", [
    ((X, I, LP), {}, "on the GPU"),
    ((X, I, LP), {"tail": "head"}, "tail"),
    ((X, I, LP), {"temperature": 2.0}, "temperature 1"),
    ((X, I, LP), {"tail": "renorm", "temperature": -1.0}, "temperature"),
    ((X, I[0], LP), {}, "index"),
    ((X, I[:3], LP), {}, "index"),
    ((X, I.float(), LP), {}, "index"),
    ((X, torch.zeros(4, 65, dtype=torch.int32), torch.zeros(4, 65)), {}, "index"),
    ((X, I, LP[:, :2]), {}, "logprob"),
    ((X, I, LP.double()), {}, "logprob"),
    ((X, I, LP), {"weight": torch.zeros(3)}, "weight"),
    ((X, I, LP), {"out": torch.zeros(4, 11)}, "out"),
])
def test_topk_distill(args, kw, error):
    with pytest.raises((ValueError, TypeError), match=error):
        tokens.topk_distill(*args, **kw)


def test_distill_entry_point_checks_before_it_launches():
    one = ctypes.c_void_p(256)

    def distill(k=3, tail=0, temp=1.0, index=one, grad=None, grad_ld=10, v=10, ld=10):
        return _capi.lib.ddm_topk_distill(one, 0, 4, v, ld, index, 4, one, k, tail, temp, None, one, grad, grad_ld,
                                          None, None, None, None)
    for kw, text in (({"k": 65}, "alternatives"), ({"tail": 2}, "tail"), ({"tail": 1, "temp": 2.0}, "temperature 1"),
                     ({"index": None}, "null"), ({"grad": one, "grad_ld": 9}, "gradient stride"),
                     ({"v": 100000, "ld": 100000}, "null")):
        assert distill(**kw) == _capi.DDM_E_ARG and text in last_error(), (kw, last_error())
    assert _capi.lib.ddm_topk_distill_scratch_bytes(4, 100, 0) == 0
    assert _capi.lib.ddm_topk_distill_scratch_bytes(4, 100000, 0) > 0


G = torch.zeros(4, 5)
OFF = torch.zeros(3, dtype=torch.int64)
S = torch.zeros(2, 10)


@pytest.mark.parametrize("args,kw,error", [
    ((X, G), {}, "on the GPU"),
    ((X, G[:1].expand(4, 5)), {}, "on the GPU"),
    ((X, torch.zeros(4, 3)), {}, "dividing"),
    ((X, torch.zeros(3, 5)), {}, "log_a"),
    ((X, torch.zeros(4, 0)), {}, "log_a"),
    ((X, G.to(torch.bfloat16)), {}, "log_a"),
    ((X.to(torch.bfloat16), G.to(torch.float16)), {}, "log_a"),
    ((X.double(), G), {}, "type"),
    ((X.t(), torch.zeros(10, 4)), {}, "contiguous"),
    ((torch.zeros(4, 0), G), {}, "channels"),
    ((X, G), {"scale": "max"}, "scale"),
    ((X, G), {"offsets": OFF.int()}, "offsets"),
    ((X, G), {"offsets": [0, 4]}, "offsets"),
    ((X, G), {"offsets": OFF[:0]}, "offsets"),
    ((X, G), {"offsets": OFF, "state": S[:1]}, "state"),
    ((X, G), {"state": S}, "state"),
    ((X, G), {"offsets": OFF, "state": S.double()}, "state"),
    ((X, G), {"out": torch.zeros(4, 9)}, "out"),
    ((X, torch.zeros(4, 10)), {"out": "log_a"}, "overlaps"),
])
def test_gated_scan(args, kw, error):
    if kw.get("out") == "log_a":
        kw = {"out": args[1]}
    with pytest.raises((ValueError, TypeError), match=error):
        gated.gated_scan(*args, **kw)


@pytest.mark.parametrize("args,kw,error", [
    ((X, G, X, X), {}, "on the GPU"),
    ((X, G, X[:3], X), {}, "h must"),
    ((X, G, X, X.double()), {}, "d_h"),
    ((X, G, X, X), {"d_state": S}, "d_state"),
    ((X, G, X, X), {"offsets": OFF, "d_state": S, "state": S[:1]}, "state"),
])
def test_gated_scan_grad(args, kw, error):
    with pytest.raises((ValueError, TypeError), match=error):
        gated.gated_scan_grad(*args, **kw)


@pytest.mark.parametrize("args,kw,error", [
    ((X, G), {}, "on the GPU"),
    ((X, G, X), {}, "on the GPU"),
    ((X, G, X[:3]), {}, "state"),
    ((X, G), {"out_state": X.to(torch.bfloat16)}, "out_state"),
    ((X, G, torch.zeros(10, 4).t()), {}, "contiguous"),
    ((X, G), {"scale": None}, "scale"),
])
def test_gated_step(args, kw, error):
    with pytest.raises((ValueError, TypeError), match=error):
        gated.gated_step(*args, **kw)


def test_step_into_a_shifted_view_of_the_state():
    base = torch.zeros(5, 10)
    with pytest.raises(ValueError, match="overlaps"):
        gated.gated_step(X, G, base[:4], out_state=base[1:])


def test_gated_entry_points_check_before_they_launch():
    one, two = ctypes.c_void_p(256), ctypes.c_void_p(512)
    lib = _capi.lib

    def scan(dtype=0, gd=0, ld=10, la=5, rows=4, d=10, g=5, off=one, n=2, scale=0, s_in=None, s_out=one, out=one, lo=10):
        return lib.ddm_gated_scan(one, dtype, ld, one, gd, la, rows, d, g, off, n, scale, s_in, s_out, out, lo, 1, None,
                                  None, None, None)

    def grad(h=one, ldh=10, lda=5, s0=two, ds=None):
        return lib.ddm_gated_scan_grad(one, 0, 10, one, 0, 5, h, ldh, one, 10, 4, 10, 5, one, 2, 0, None, ds, s0, one, 10,
                                       one, lda, 1, None, None, None, None)

    def step(out=one, lo=10, d=10):
        return lib.ddm_gated_step(one, 0, 10, one, 0, 5, 4, d, 5, 0, None, two, out, lo, None, None, None)
    for call, cases in ((scan, (({"dtype": 5}, "types"), ({"dtype": 0, "gd": 1}, "types"), ({"dtype": 1, "gd": 2}, "types"),
                                ({"g": 3}, "gates"), ({"g": 0}, "gates"), ({"ld": 9}, "strides"), ({"la": 4}, "strides"),
                                ({"rows": -1}, "rows"), ({"n": -1}, "rows"), ({"scale": 3}, "scale"), ({"out": None}, "null"),
                                ({"lo": 9}, "stride"), ({"off": None}, "one sequence"), ({"s_out": None}, "null"),
                                ({"s_in": one}, "one buffer"), ({"rows": 1 << 39, "d": 1 << 20, "g": 1 << 20, "ld": 1 << 20,
                                                                 "la": 1 << 20, "lo": 1 << 20}, "tiles"),
                                ({"rows": 100000}, "scratch"), ({"ld": 1 << 23}, "row stride"))),
                        (grad, (({"h": None}, "null"), ({"ldh": 9}, "stride"), ({"lda": 4}, "stride"),
                                ({"s0": None}, "null"), ({"ds": two}, "one buffer"))),
                        (step, (({"out": None}, "null"), ({"lo": 9}, "stride"), ({"d": 11}, "gates")))):
        for kw, text in cases:
            assert call(**kw) == _capi.DDM_E_ARG and text in last_error(), (kw, last_error())
    assert lib.ddm_gated_scan_scratch_bytes(0, 8, 8, 0, 0) == 0
    assert lib.ddm_gated_scan_scratch_bytes(100000, 8, 8, 0, 0) > 0


def test_results_over_other_arguments():
    base = torch.zeros(44)
    out = base[:40].view(4, 10)
    for kw in ({"d_logprob": base[39:43]}, {"d_entropy": base[:4]}):
        with pytest.raises(ValueError, match="overlaps another"):
            tokens.token_scores_grad(X, T, scores(), out=out, **kw)
    index = torch.zeros(4, 1, dtype=torch.int64)
    with pytest.raises(ValueError, match="overlaps another"):
        tokens.topk_distill(X, index, base[38:42].view(4, 1), out=out)
    with pytest.raises(ValueError, match="overlaps another"):
        tokens.topk_distill(X, index, torch.zeros(4, 1), weight=base[::11], out=out)
    with pytest.raises(ValueError, match="overlaps an input"):
        gated.gated_scan(X, G, state=base[20:30].view(1, 10), out=out)
    x, log_a = 1 << 20, 1 << 21         # 4 rows of 10 and of 5 float32: 160 and 80 bytes
    for state in (x + 156, x - 156, log_a + 76, log_a - 156):
        rc = _capi.lib.ddm_gated_step(x, 0, 10, log_a, 0, 5, 4, 10, 5, 0, None, state, 1 << 22, 10, None, None, None)
        assert rc == _capi.DDM_E_ARG and "overlaps" in last_error(), last_error()


def test_launches_have_room():
    one, two, lib = ctypes.c_void_p(256), ctypes.c_void_p(512), _capi.lib
    n = (1 << 24) + 5                   # rows of 4100 bfloat16: a workgroup of 256 each
    for rc in (lib.ddm_token_scores(one, 1, n, 4100, 4100, one, 8, 1.0, 0, one, one, one, one, one, None, None, one, None,
                                    None, None),
               lib.ddm_token_scores_grad(one, 1, n, 4100, 4100, one, 8, 1.0, 0, one, one, None, None, None, None, one,
                                         4100, None, None, None),
               lib.ddm_topk_distill(one, 1, n, 4100, 4100, one, 8, one, 1, 0, 1.0, None, one, one, 4100, one, None, None,
                                    None),
               lib.ddm_gated_step(one, 0, 1 << 20, one, 0, 1, 4096, 1 << 20, 1, 0, None, two, one, 1 << 20, None, None,
                                  None),
               lib.ddm_gated_scan_grad(one, 1, 2049, one, 1, 3, one, 2049, one, 2049, (1 << 32) // 3 + 1, 2049, 3, one, 2,
                                       0, None, None, two, one, 2049, one, 3, 1, one, None, None, None)):
        assert rc == _capi.DDM_E_ARG and "work-items" in last_error(), last_error()


def test_columns_of_one_buffer_lie_apart():
    from ddm_amd._launch import overlap
    base = torch.zeros(6, 30)
    cut = lambda a, b, r=slice(0, 6): base[r, a:b]  # noqa: E731
    for a, b, want in ((cut(0, 10), cut(10, 25), False), (cut(0, 10), cut(9, 25), True), (cut(10, 25), cut(0, 10), False),
                       (cut(10, 25), cut(0, 11), True), (cut(20, 30), cut(0, 20, slice(1, 6)), False),
                       (cut(0, 10, slice(0, 3)), cut(0, 10, slice(3, 6)), False), (cut(0, 10), cut(0, 10), True),
                       (cut(0, 10, slice(0, 4)), cut(5, 8, slice(2, 6)), True), (cut(0, 30), cut(29, 30), True),
                       (base.view(12, 15)[:, :5], cut(5, 15), True), (base[0], cut(3, 5), True)):
        assert overlap(a, b) == want and overlap(b, a) == want, (a.shape, b.shape, want)
    # a projection's inputs and gates side by side, the result over the inputs
    with pytest.raises(ValueError, match="on the GPU"):
        gated.gated_scan(cut(0, 20), cut(20, 30), out=cut(0, 20))
    with pytest.raises(ValueError, match="on the GPU"):
        tokens.token_scores_grad(cut(0, 10, slice(0, 4)), T, scores(), out=cut(10, 20, slice(0, 4)))


def test_the_guards_state_needs_a_place():
    assert _capi.lib.ddm_wait_gave_up(None) == _capi.DDM_E_ARG and "null" in last_error()


def test_types_of_h():
    x, g, f = X.to(torch.bfloat16), G.to(torch.bfloat16), torch.float32
    for kw, error in (({"dtype": torch.float16}, "h has type"), ({"dtype": torch.float64}, "h has type"),
                      ({"out": torch.zeros(4, 10, dtype=torch.float16)}, "h has type"),
                      ({"out": X.clone(), "dtype": torch.bfloat16}, "out must be"), ({"out": X.clone()}, "on the GPU"),
                      ({"dtype": f}, "on the GPU"), ({"dtype": f, "out": x}, "out must be")):
        with pytest.raises((ValueError, TypeError), match=error):
            gated.gated_scan(x, g, **kw)
    base = torch.zeros(4, 20, dtype=torch.bfloat16)     # float32 results over the 16-bit inputs
    with pytest.raises(ValueError, match="overlaps"):
        gated.gated_scan(base[:, :10], g, out=base.view(f))
    with pytest.raises(ValueError, match="on the GPU"):
        gated.gated_scan_grad(x, g, X, x)
    with pytest.raises(ValueError, match="h must"):
        gated.gated_scan_grad(x, g, x.half(), x)
    with pytest.raises(ValueError, match="d_h must"):
        gated.gated_scan_grad(x, g, X, X)
    one, two = ctypes.c_void_p(256), ctypes.c_void_p(512)
    for flags in (4, -1):
        assert _capi.lib.ddm_gated_scan(one, 1, 10, one, 1, 5, 4, 10, 5, one, 2, 0, None, two, one, 10, flags, None, None,
                                        None, None) == _capi.DDM_E_ARG and "flags" in last_error()


def test_what_was_written_counts_as_changed():
    from ddm_amd._launch import written
    x = torch.ones(3, requires_grad=True)
    y = x * 2
    z = y.pow(2).sum()                                  # keeps y
    written(y.detach())
    with pytest.raises(RuntimeError, match="inplace"):
        z.backward()
    written(None)
    with torch.inference_mode():
        written(torch.ones(3))
