"""The operators on rows on the GPU at the sizes from which on they take other paths: wavefronts that serve several choices of a
token in turn, rows of two and four vectors to a lane and longer ones, two wavefronts to a row, calls that go past the caches. Against
64 bits, with the tolerances of test_gpu_ops.py."""
import numpy as np
import pytest

from conftest import announce
from test_gpu_ops import F, TYPES, laid, near, normal, ops, places, plain_bits, plain_bucket, rounded, seeded  # noqa: F401

pytestmark = pytest.mark.gpu

SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
PAST = 256 << 20  # bytes from which on a call goes past the caches


def share(T, K, k, type):
    """How many choices of a token a wavefront of the sum's gradient takes (pskv_route_sum_grad)."""
    vectors, lanes = -(-k * SIZE[type] // 16), 1
    while lanes < 64 and lanes < vectors:
        lanes *= 2
    s = K
    while s > 1 and T * -(-K // s) * lanes < 64 * 4096:
        s = (s + 1) // 2
    return s


def routed(ops, T, K, k, R, gap, type, lost):
    import torch
    g, rng = seeded(T + k), np.random.default_rng(T * k)
    place = places(rng, T, K, R, lost)
    at = place.long()
    here = (at >= 0) & (at < R)
    weights = torch.rand(T, K, generator=g, device="cuda:0") - 0.2

    # out: rows that no place names, and what lies between rows, keep what they hold
    _, x = laid(g, T, k, type, gap)
    whole, rows = laid(None, R, k, type, gap)
    between = whole.clone()
    mark = between.as_strided(rows.shape, rows.stride(), rows.storage_offset())
    for j in range(K):
        some = here[:, j]
        mark[at[some, j]] = x[some]
    ops.route_rows(x, place, rows)
    assert torch.equal(whole, between)
    del whole, between, mark, rows

    # back: rows that no choice has do not matter
    _, answers = laid(g, R, k, type, gap)
    named = torch.zeros(R, dtype=torch.bool, device="cuda:0")
    named[at[here]] = True
    answers[~named] = float("nan")
    outs = [laid(None, T, k, type, gap) for _ in range(2)]
    ops.route_sum(answers, place, outs[0][1], weights=weights)
    ops.route_sum(answers, place, outs[1][1])
    for (whole, out), w in zip(outs, (weights.double(), torch.ones(T, K, dtype=torch.float64, device="cuda:0"))):
        value, size = (torch.zeros(T, k, dtype=torch.float64, device="cuda:0") for _ in range(2))
        for j in range(K):
            term = torch.where(here[:, j, None], answers[at[:, j].clamp(0, R - 1)].double(), 0.0) * w[:, j, None]
            value += term
            size += term.abs()
        near(out, value, rounded(value, K * F * size, type), "route_sum")
        if gap:
            out.fill_(99.0)
            assert bool((whole == 99.0).all())

    # the gradient of back
    _, grad = laid(g, T, k, type, gap)
    whole, grad_rows = laid(None, R, k, type, gap)
    grad_weights = torch.full((T, K), 5.0, device="cuda:0")
    ops.route_sum_grad(grad, answers, place, weights, grad_rows, grad_weights)
    assert bool((grad_weights[~here] == 0).all())
    for j in range(K):
        some = here[:, j]
        product = answers[at[some, j]].double() * grad[some].double()
        near(grad_weights[some, j], product.sum(1), (k + 1) * F * product.abs().sum(1) + 2.0 ** -149, "weights")
        value = weights[some, j, None].double() * grad[some].double()
        near(grad_rows[at[some, j]], value, rounded(value, F * value.abs() + 2.0 ** -150, type), "grad_rows")
        grad_rows[at[some, j]] = 99.0
    assert bool((whole == 99.0).all())


# (the choices divided among wavefronts evenly and unevenly; vectors to a lane: 1, 2, 4, more; whole vectors and odd elements)
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("T,K,k,gap", [(5003, 7, 300, 0), (4099, 5, 777, 3), (4099, 3, 1500, 0), (4097, 6, 2056, 0), (4100, 2, 2100, 1),
                                       (3001, 5, 1031, 0), (9001, 8, 130, 0), (40001, 3, 40, 0), (33000, 9, 21, 5)])
@pytest.mark.parametrize("lost", [0.0, 0.4])
def test_many_tokens(ops, dev, type, T, K, k, gap, lost):
    announce("route_rows, route_sum, route_sum_grad, many tokens", type, T, K, k, gap, lost)
    assert share(T, K, k, type) > 1
    routed(ops, T, K, k, T * K + 17 if lost else T * K - 5, gap, type, lost)


@pytest.mark.parametrize("type,T,K,k,gap", [("bfloat16", 9001, 5, 2504, 0), ("float16", 9001, 5, 2501, 0), ("bfloat16", 20011, 6, 961, 2),
                                            ("float32", 9001, 5, 1253, 0), ("float32", 150001, 2, 151, 0), ("float16", 700001, 3, 49, 0)])
def test_past_the_caches(ops, dev, type, T, K, k, gap):
    announce("route_rows, route_sum, route_sum_grad, past the caches", type, T, K, k, gap)
    assert (1 + K) * T * k * SIZE[type] > PAST
    routed(ops, T, K, k, T * K - 5, gap, type, 0.3)


@pytest.mark.parametrize("type,H,Q,K", [("bfloat16", 9, 2047, 1901), ("float16", 9, 2047, 1904), ("float32", 5, 2041, 1903)])
@pytest.mark.parametrize("own", [False, True])
def test_bias_past_the_caches(ops, dev, type, H, Q, K, own):
    import torch
    announce("relbias past the caches", type, H, Q, K, own)
    B, far = 4, 128
    assert B * H * Q * K * SIZE[type] > PAST
    g = seeded(K)
    table = normal(g, 32, H)
    at = torch.tensor([0, 700, -40, 5], device=dev) if own else None
    reach = Q + K + 800
    bucket = torch.tensor([plain_bucket(r, 32, far, True) for r in range(-reach, reach + 1)], device=dev)
    rel = torch.arange(K, device=dev)[None, :] - torch.arange(Q, device=dev)[:, None] + reach
    scores, out = normal(g, B, H, Q, K, type=type), torch.empty(B, H, Q, K, dtype=getattr(torch, type), device=dev)

    def check(got, before):
        for b in range(B):
            u = bucket[rel - (int(at[b]) if own else 0)]
            for h in range(H):
                want = table[:, h].double()[u]
                if before is None:
                    near(got[b, h], want, rounded(want, 0.0, type), "bias")
                else:
                    want = before[b, h].double() + want
                    near(got[b, h], want, rounded(want, F * want.abs(), type), "scores")

    ops.relbias(table, out, far, q_at=at)
    check(out, None)
    ops.relbias(table, out, far, q_at=at, scores=scores)
    check(out, scores)
    inside = scores.clone()
    ops.relbias(table, inside, far, q_at=at, scores=inside)
    assert torch.equal(inside, out)
    # rows that begin at odd elements
    wide = torch.full((B, H, Q, K + 1), 9.0, device=dev).to(out.dtype)
    ops.relbias(table, wide[..., 1:], far, q_at=at, scores=scores)
    assert torch.equal(wide[..., 1:], out) and bool((wide[..., 0] == 9).all())


@pytest.mark.parametrize("type,n,k", [("bfloat16", 70001, 1003), ("float16", 1100003, 64), ("float32", 35001, 1003), ("float32", 600001, 61)])
def test_dropout_past_the_caches(ops, dev, type, n, k):
    import torch
    announce("dropout past the caches", type, n, k)
    assert 2 * n * k * SIZE[type] > PAST
    g = seeded(k)
    x = normal(g, n, k, type=type)
    keys = torch.randint(-(1 << 63), (1 << 63) - 1, (n,), generator=g, device=dev)
    out, pieces = torch.empty_like(x), torch.full_like(x, 7.0)
    ops.dropout(x, out, 0.25, 987654321, keys=keys)
    step = n // 7
    for a in range(0, n, step):
        ops.dropout(x[a:a + step], pieces[a:a + step], 0.25, 987654321, keys=keys[a:a + step])
    assert torch.equal(out, pieces)
    some = torch.randperm(n, generator=g, device=dev)[:500]
    keep = torch.from_numpy(plain_bits(keys[some].cpu().numpy().view(np.uint64), k, 987654321) >= 16384).to(dev)
    want = torch.where(keep, x[some].double() * (4 / 3), 0.0)
    near(out[some], want, rounded(want, 2 * F * want.abs() + 2.0 ** -149, type), "dropout")
