"""What the language-model calls refuse, on the host: nothing is launched."""
import ctypes

import pytest
import torch

from ddm_amd import _capi, tokens

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
                     ({"temp": 0.0}, "temperature"), ({"temp": float("inf")}, "temperature"), ({"top": 65}, "alternatives"),
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
    assert _capi.lib.ddm_topk_distill_scratch_bytes(4, 100, 0, 3, 1) == 0
    assert _capi.lib.ddm_topk_distill_scratch_bytes(4, 100000, 0, 3, 1) > 0
