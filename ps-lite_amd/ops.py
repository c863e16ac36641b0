"""Operators on rows: what a worker does with rows between its pull and its push. Tokens sorted by expert and back, the
learned relative position bias, dropout, and their gradients (pskv_route_*, pskv_relbias*, pskv_dropout of
include/pskv/capi.h).

Arguments are torch tensors on one GPU; a call fills the tensors that it is given for its answers. Rows are float32, float16
or bfloat16, the elements of a row lie side by side, rows may be any number of elements apart. A call is enqueued on torch's
current stream of that GPU, or on `stream` (the address of a hipStream_t), waits for nothing and may be captured into a
graph (after a first call outside any capture). What a call writes may share no memory with what it reads, but where an answer may be
its own input. With a `stream` of one's own, tensors have to be complete on it and to be
kept until it has run the call.

These are calls, not nodes of autograd: a gradient is the call that is named as such. Tensors that do not fit raise TypeError
or ValueError, what the library refuses raises PskvError.
"""
from . import capi
from .capi import _check

MAX_EXPERTS = 2048
MAX_BUCKETS = 256


def _native():
    if capi._native is None:
        capi.load()
    return capi._native


def _room(nbytes, like, stream):
    """Working memory of a call that was not given any. It belongs to the stream that the call runs on: it may have been used
    there before, and is used again there behind the call at the earliest."""
    import torch
    if stream is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=like.device)
    with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=like.device)):
        return torch.empty(nbytes, dtype=torch.uint8, device=like.device)


def route_room(n, num_experts):
    """Bytes of working memory that a sort of n choices takes (0: none)."""
    return capi.load().pskv_route_room(n, num_experts)


def route_sort(experts, num_experts, order, place, offsets, work=None, stream=None):
    """Sorts the choices `experts` ([tokens, choices], int32 or int64) by expert, stably. place (int32, as many) gets where
    each choice went, order (int32, as many) the choice at each place, offsets (int32, num_experts + 1) where each expert's
    begin. Numbers outside 0 .. num_experts - 1 are choices that are not here: their place is -1, and order is -1 behind the
    last expert's. work: at least route_room() bytes, for a program that keeps them; else they are allocated."""
    rc = _native().route_sort(experts, num_experts, order, place, offsets, work, stream, _room)
    if rc:
        _check(rc)


def route_rows(x, place, rows, stream=None):
    """rows[place[t, j]] = x[t]: every token's row ([tokens, k]) goes to the places of its choices, which name a row once at most.
    Rows that no place names are left as they are: those behind the last expert's hold what an earlier call wrote there. The gradient
    of x is route_sum(grad of rows, place, grad of x)."""
    rc = _native().route_rows(x, place, rows, stream)
    if rc:
        _check(rc)


def route_sum(rows, place, out, weights=None, stream=None):
    """out[t] = sum over j of weights[t, j] * rows[place[t, j]], in the order of j, in float. A choice that is not here adds
    nothing. weights: float32 [tokens, choices]; None: all are 1."""
    rc = _native().route_sum(rows, place, out, weights, stream)
    if rc:
        _check(rc)


def route_sum_grad(grad, rows, place, weights, grad_rows, grad_weights, stream=None):
    """The gradient of route_sum: grad_rows[place[t, j]] = weights[t, j] * grad[t] and grad_weights[t, j] = <grad[t],
    rows[place[t, j]]> (float32, 0 for a choice that is not here). Rows that no place names are left as they are. A row that
    several choices name gets the gradient of one of them: places are those of route_sort, which name a row once at most."""
    rc = _native().route_sum_grad(grad, rows, place, weights, grad_rows, grad_weights, stream)
    if rc:
        _check(rc)


def relbias_bucket(rel, buckets, max_distance, two_sided=True):
    """The bucket of a relative position (key position less query position)."""
    rc = capi.load().pskv_relbias_bucket(rel, buckets, max_distance, 1 if two_sided else 0)
    if rc < 0:
        _check(rc)
    return rc


def relbias(table, out, max_distance, two_sided=True, scores=None, q_first=0, k_first=0, q_at=None, stream=None):
    """out[b, h, i, j] = scores[b, h, i, j] + table[bucket(rel), h], rel = (k_first + j) - (q_first + q_at[b] + i). table
    (float32, [buckets, heads]) is what a pull of a table of rows with a key per bucket answers. out is [batch, heads,
    queries, keys] or [heads, queries, keys]; scores has its type and shape, may be out itself and may be expanded over the
    batch; None: the bias alone. q_at (int64, [batch]): where the sequences of a batch stand, as single tokens of several do."""
    rc = _native().relbias(table, out, max_distance, two_sided, scores, q_first, k_first, q_at, stream)
    if rc:
        _check(rc)


def relbias_grad_room(buckets, batch, heads, queries, keys, own_positions=False):
    """Bytes of working memory that a gradient of [batch, heads, queries, keys] takes (0: none); own_positions: with q_at."""
    return capi.load().pskv_relbias_grad_room(buckets, heads, batch, queries, keys, 1 if own_positions else 0)


def relbias_grad(grad, grad_table, max_distance, two_sided=True, q_first=0, k_first=0, q_at=None, work=None, stream=None):
    """The gradient of the table: grad_table[u, h] (float32, all of it is written) = the sum of grad over what bucket u was
    added to, the values of a push to the table of rows. work: at least relbias_grad_room() bytes, for a program that keeps
    them; else they are allocated."""
    rc = _native().relbias_grad(grad, grad_table, max_distance, two_sided, q_first, k_first, q_at, work, stream, _room)
    if rc:
        _check(rc)


def dropout(x, out, p, seed, keys=None, first=0, step=None, stream=None):
    """out = x * scale where an element is kept, 0 where it is dropped, with probability p (to 16 bits). Whether an element is
    kept depends on seed (0 .. 2^64 - 1), on its row's key (keys: int64, [rows]; else first, first + 1, ...) and its column
    alone, so the gradient is the same call on the gradient's rows, in any order. step (one int64 on the GPU) is added to the
    seed, for graphs that draw anew at every replay: seeds that share a step lie further apart than there are steps (random ones do),
    or one draws what the other drew some steps before. out may be x."""
    rc = _native().dropout(x, out, p, seed, step, keys, first, stream)
    if rc:
        _check(rc)
