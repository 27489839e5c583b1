"""A language model in the place of the forest: what its answers say, and what a refit trains it on.

`token_scores` is predict_rf's part (DDM_Process.py:110-128) for rows of logits: per answer
the error flag the DDM scans read (`kernels.scan_streams` and its relatives), and next to it
log probability, entropy, rank and the top alternatives; `token_scores_grad` is its backward
pass.  `topk_distill` is the loss (and gradient) of train_rf's part (:98-105): a model
refitted on the alternatives another one gave.

The calls are asynchronous on `stream` (default: the current stream of the logits' device),
read nothing back and can be captured.  Results belong to that stream.  They carry no autograd history, whether
the logits require a gradient or not: the gradients are calls of their own (`logits.backward(gradient)`
goes on from there).
"""
import collections

import torch

from ._capi import check, lib
from ._launch import DTYPES, dense, launch_on, overlap, rows_of, scratch_for, shaped, written
from .kernels import _evs, _ptr

MAX_COLUMNS = 1 << 19
MAX_TOP = 64

TokenScores = collections.namedtuple("TokenScores", ["logprob", "entropy", "rank", "err", "top_logprob", "top_index",
                                                     "stats", "temperature"])
TokenScores.__doc__ = """What token_scores returns: logprob, entropy float32 [n]; rank int32 [n]; err uint8
[n rounded up to 16] (the scans' layout, zeros behind row n-1); top_logprob float32 and top_index int32 [n, top]
(None for top 0); stats float32 [n, 2] and the temperature, for token_scores_grad."""


def _temperature(t):
    t = float(t)
    if not torch.finfo(torch.float32).tiny <= t < float("inf"):
        raise ValueError(f"temperature must be positive (a normal float32) and finite, got {t}")
    return t


def _logits(logits):
    ld = rows_of("logits", logits)
    n, v = logits.shape
    if not 1 <= v <= MAX_COLUMNS:
        raise ValueError(f"logits have {v} columns (1..{MAX_COLUMNS})")
    return n, v, ld


def _check_out(out, logits, *others):
    if out is None:
        return
    rows_of("out", out)
    if out.shape != logits.shape or out.dtype != logits.dtype:
        raise ValueError(f"out must be {logits.dtype} {list(logits.shape)}, got {out.dtype} {list(out.shape)}")
    same = out.data_ptr() == logits.data_ptr() and out.stride() == logits.stride()
    if not same and overlap(out, logits):
        raise ValueError("out overlaps the logits without being them")
    if any(t is not None and overlap(out, t) for t in others):
        raise ValueError("out overlaps another argument")


def _new_like(out, logits):
    return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device) if out is None else out


def token_scores(logits, targets, top=0, temperature=1.0, stream=None, timer=None):
    """Scores of every row of logits [n, v] (float32, bfloat16 or float16; rows contiguous, any
    row stride) against targets [n] (int32 or int64): see TokenScores.

    A target outside [0, v) is not scored (logprob 0, rank -1, err 0).  -inf logits are masked:
    probability 0, never an alternative; index -1 and -inf stand behind the last alternative.  A
    row with nothing left has logprob -inf, entropy 0, err 1.  A row with NaN or +inf has NaN
    scores, rank and indexes -1, err 1.  Equal logits rank by the lower column."""
    n, v, ld = _logits(logits)
    shaped("targets", targets, (n,), torch.int32, torch.int64)
    top, temperature = int(top), _temperature(temperature)
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"top must be 0..{MAX_TOP}, got {top}")
    dev, code = logits.device, DTYPES[logits.dtype]
    context, s = launch_on(logits, stream, (logits, targets))
    with context:
        targets = dense(targets)
        logprob = torch.empty(n, dtype=torch.float32, device=dev)
        entropy = torch.empty_like(logprob)
        stats = logprob.new_empty((n, 2))
        rank = torch.empty(n, dtype=torch.int32, device=dev)
        err = torch.empty((n + 15) // 16 * 16, dtype=torch.uint8, device=dev)
        top_lp = logprob.new_empty((n, top)) if top else None
        top_ix = rank.new_empty((n, top)) if top else None
        scratch = scratch_for(dev, "ddm_token_scores_scratch_bytes", n, v, code, top)
        check(lib.ddm_token_scores(logits.data_ptr(), code, n, v, ld, targets.data_ptr(), targets.element_size(),
                                   temperature, top, logprob.data_ptr(), entropy.data_ptr(), stats.data_ptr(),
                                   rank.data_ptr(), err.data_ptr(), _ptr(top_lp), _ptr(top_ix), _ptr(scratch), s,
                                   *_evs(timer)), "ddm_token_scores")
    return TokenScores(logprob, entropy, rank, err, top_lp, top_ix, stats, temperature)


def token_scores_grad(logits, targets, scores, d_logprob=None, d_entropy=None, d_top=None, out=None, stream=None,
                      timer=None):
    """Gradient by the logits of  d_logprob . logprob + d_entropy . entropy + d_top . top_logprob
    (float32 [n], [n], [n, top]; None: zero), in the logits' type.  `scores` is what
    token_scores returned for the same logits and targets.  out: None, the logits themselves
    (overwritten), or a tensor of their shape apart from every argument."""
    n, v, ld = _logits(logits)
    shaped("targets", targets, (n,), torch.int32, torch.int64)
    shaped("scores.stats", scores.stats, (n, 2), torch.float32)
    shaped("scores.entropy", scores.entropy, (n,), torch.float32)
    for name, g in (("d_logprob", d_logprob), ("d_entropy", d_entropy)):
        if g is not None:
            shaped(name, g, (n,), torch.float32)
    top, index = 0, None
    if d_top is not None:
        if scores.top_index is None:
            raise ValueError("d_top given, but the scores have no alternatives")
        index, top = scores.top_index, scores.top_index.shape[1]
        shaped("scores.top_index", index, (n, top), torch.int32)
        shaped("d_top", d_top, (n, top), torch.float32)
    _check_out(out, logits, targets, scores.stats, scores.entropy, index, d_logprob, d_entropy, d_top)
    into = out
    given = (logits, targets, scores.stats, scores.entropy, index, d_logprob, d_entropy, d_top, out)
    context, s = launch_on(logits, stream, given)
    with context:
        targets, stats, entropy, index, d_logprob, d_entropy, d_top = map(dense, given[1:8])
        out = _new_like(out, logits)
        out_ld = out.stride(0) if n > 1 else v
        check(lib.ddm_token_scores_grad(logits.data_ptr(), DTYPES[logits.dtype], n, v, ld, targets.data_ptr(),
                                        targets.element_size(), scores.temperature, top, stats.data_ptr(),
                                        entropy.data_ptr(), _ptr(index), _ptr(d_logprob), _ptr(d_entropy),
                                        _ptr(d_top), out.data_ptr(), out_ld, s, *_evs(timer)),
              "ddm_token_scores_grad")
    written(into)
    return out


TAILS = {"renorm": 0, "rest": 1}


def topk_distill(logits, index, logprob, tail="rest", temperature=1.0, weight=None, grad=False, out=None, stream=None,
                 timer=None):
    """Loss [n] (float32) of a student's logits [n, v] against a teacher's alternatives: index
    [n, k] (int32 or int64) with their log probabilities [n, k] (float32), k at most 64, as
    token_scores gives them.  Indexes outside [0, v) are none, and repeats of an earlier one too.

    tail "rest": what the alternatives leave of the teacher's probability is one more outcome,
    "none of these" (temperature 1); "renorm": the alternatives alone, softened by the
    temperature.  grad (or out, a tensor like token_scores_grad's): also the gradient of
    weight . loss (float32 [n], None: ones) by the logits, from the same reading.  Returns (loss,
    gradient or None)."""
    n, v, ld = _logits(logits)
    if tail not in TAILS:
        raise ValueError(f"tail must be one of {', '.join(TAILS)}, got {tail!r}")
    temperature = _temperature(temperature)
    if tail == "rest" and temperature != 1.0:
        raise ValueError("tail 'rest' is known at temperature 1 only")
    if not isinstance(index, torch.Tensor) or index.dim() != 2 or index.shape[1] > MAX_TOP:
        raise ValueError(f"index must be a tensor [n, k] with k at most {MAX_TOP}")
    k = index.shape[1]
    shaped("index", index, (n, k), torch.int32, torch.int64)
    shaped("logprob", logprob, (n, k), torch.float32)
    if weight is not None:
        shaped("weight", weight, (n,), torch.float32)
    _check_out(out, logits, index, logprob, weight)
    into, code = out, DTYPES[logits.dtype]
    context, s = launch_on(logits, stream, (logits, index, logprob, weight, out))
    with context:
        index, logprob, weight = dense(index), dense(logprob), dense(weight)
        loss = torch.empty(n, dtype=torch.float32, device=logits.device)
        out = _new_like(out, logits) if grad or out is not None else None
        scratch = scratch_for(logits.device, "ddm_topk_distill_scratch_bytes", n, v, code)
        out_ld = v if out is None or n <= 1 else out.stride(0)
        check(lib.ddm_topk_distill(logits.data_ptr(), code, n, v, ld, index.data_ptr(), index.element_size(),
                                   logprob.data_ptr(), k, TAILS[tail], temperature, _ptr(weight), loss.data_ptr(),
                                   _ptr(out), out_ld, _ptr(scratch), s, *_evs(timer)), "ddm_topk_distill")
    written(into)
    return loss, out
