"""The operators on rows (ps-lite_amd/ops.py) on the GPU against plain implementations in 64 bits.

Tolerances are counted: U is half a step of the type that an answer is rounded to, F half a step of float32, in which sums are
taken. A sum of n terms, in any order, is off by at most n F times the sum of its terms' magnitudes (the product of a fused
multiply-add is exact); its rounding adds U of the value, and half of the least subnormal number where float16 underflows.
"""
import numpy as np
import pytest

from conftest import announce

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]
F = 2.0 ** -24
U = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
LEAST = {"float32": 2.0 ** -149, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -133}


@pytest.fixture(scope="module")
def ops(capi):
    import __graft_entry__ as graft
    return graft.load_package().ops


def rounded(value, slack, type):
    """How far a float32 sum that is off by `slack` may be from `value` once it is rounded to `type`."""
    return slack + U[type] * (value.abs() + slack) + LEAST[type] / 2


def near(got, want, tolerance, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    bad = ~(off <= tolerance)
    if bool(bad.any()):
        i = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError("%s: %d of %d are off, first at %s: got %r want %r" % (
            what, int(bad.sum()), bad.numel(), i, float(got[i]), float(want[i])))


def normal(g, *shape, type="float32", dev="cuda:0", scale=1.0):
    import torch
    return (torch.randn(*shape, generator=g, device=dev) * scale).to(getattr(torch, type))


def seeded(seed, dev="cuda:0"):
    import torch
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


# --- tokens sorted by expert -------------------------------------------------------------------------------------

def plain_sort(experts, E):
    flat = experts.reshape(-1).astype(np.int64)
    here = (flat >= 0) & (flat < E)
    mine = np.flatnonzero(here)
    mine = mine[np.argsort(flat[mine], kind="stable")]
    order = np.full(flat.size, -1, np.int32)
    order[:mine.size] = mine
    place = np.full(flat.size, -1, np.int32)
    place[mine] = np.arange(mine.size)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[here], minlength=E))]).astype(np.int32)
    return order, place.reshape(experts.shape), offsets


def sort(ops, experts, E, **more):
    import torch
    n, dev = experts.numel(), experts.device
    order = torch.full((n + 3,), -7, dtype=torch.int32, device=dev)  # (three that no call owns)
    place = torch.full((n + 3,), -7, dtype=torch.int32, device=dev)
    offsets = torch.full((E + 4,), -7, dtype=torch.int32, device=dev)
    ops.route_sort(experts, E, order[:n], place[:n].view(experts.shape), offsets[:E + 1], **more)
    torch.cuda.synchronize()
    for x in (order[n:], place[n:], offsets[E + 1:]):
        assert bool((x == -7).all())
    return order[:n], place[:n].view(experts.shape), offsets[:E + 1]


@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("T,K,E", [(0, 2, 5), (1, 1, 1), (1, 2, 2048), (7, 3, 2), (64, 1, 7), (65, 8, 63), (1000, 3, 64), (513, 5, 65),
                                   (1024, 8, 256), (8193, 1, 8), (1025, 1, 8), (4096, 1, 9), (4097, 1, 300), (4099, 6, 1000), (2731, 3, 2048), (100003, 3, 60),
                                   (2048, 1, 20), (131072, 1, 33), (131073, 1, 70), (524289, 1, 3), (262145, 1, 1), (600007, 1, 2047)])
@pytest.mark.parametrize("lost", [0.0, 0.3, 1.0])
def test_sort(ops, dev, bits, T, K, E, lost):
    import torch
    announce("route_sort", bits, T, K, E, lost)
    rng = np.random.default_rng(T * 7 + E)
    # skewed: a tenth of the choices fall on one expert
    experts = np.where(rng.random((T, K)) < 0.1, E // 2, rng.integers(0, E, (T, K)))
    far = [-1, E, -E - 1, 2 ** 31 - 1, -2 ** 31] + ([2 ** 32, 2 ** 32 + E // 2, -2 ** 63, 2 ** 63 - 1] if bits == 64 else [])
    experts = np.where(rng.random((T, K)) < lost, rng.choice(np.array(far, np.int64), (T, K)), experts)
    t = torch.from_numpy(experts.astype(np.int64 if bits == 64 else np.int32)).to(dev)
    for got, want in zip(sort(ops, t, E), plain_sort(experts, E)):
        assert np.array_equal(got.cpu().numpy(), want)


def test_sort_with_working_memory(ops, dev):
    import torch
    announce("route_sort, working memory")
    rng = np.random.default_rng(1)
    experts = rng.integers(0, 33, (20000, 2))
    t = torch.from_numpy(experts).to(dev)
    work = torch.full((ops.route_room(40000, 33) // 4 + 2,), 77, dtype=torch.int32, device=dev)
    for _ in range(2):  # as it was left
        for got, want in zip(sort(ops, t, 33, work=work[:-2]), plain_sort(experts, 33)):
            assert np.array_equal(got.cpu().numpy(), want)
    assert work[-2:].tolist() == [77, 77]


# --- rows out and back -------------------------------------------------------------------------------------------

def places(rng, T, K, R, lost):
    """Places of T x K choices among R rows, each at most once; some are not here, in more than one way."""
    import torch
    n = T * K
    p = rng.permutation(max(R, n))[:n]
    p = np.where((p >= R) | (rng.random(n) < lost), rng.choice(np.array([-1, R, R + 5, -2 ** 31, 2 ** 31 - 1]), n), p)
    return torch.from_numpy(p.reshape(T, K).astype(np.int32)).cuda()


def laid(g, n, k, type, gap):
    """[n, k] with `gap` elements between rows, beginning at an odd element where there is a gap."""
    import torch
    whole = torch.full((n * (k + gap) + gap + 1,), 99.0, device="cuda:0").to(getattr(torch, type))
    view = whole[gap and 1:].as_strided((n, k), (k + gap, 1))
    if g is not None:
        view.copy_(normal(g, n, k, type=type))
    return whole, view


SHAPES = [(1, 1, 1, 1, 0), (1, 2, 64, 2, 0), (3, 2, 8, 9, 5), (7, 8, 9, 60, 0), (64, 1, 1001, 64, 1), (33, 3, 4, 99, 0),
          (100, 6, 777, 600, 3), (16, 2, 1024, 40, 0), (257, 4, 130, 1100, 0), (5, 9, 4099, 45, 0), (2, 2, 20000, 4, 0),
          (1000, 8, 16, 8000, 16), (3, 65, 24, 200, 0)]


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("T,K,k,R,gap", SHAPES)
@pytest.mark.parametrize("lost", [0.0, 0.4])
def test_rows_out_and_back(ops, dev, type, T, K, k, R, gap, lost):
    import torch
    announce("route_rows, route_sum, route_sum_grad", type, T, K, k, R, gap, lost)
    g, rng = seeded(T + k), np.random.default_rng(T * k)
    place = places(rng, T, K, R, lost)
    at = place.long()
    here = (at >= 0) & (at < R)
    weights = torch.rand(T, K, generator=g, device=dev) - 0.2
    u = lambda x, s: rounded(x, s, type)

    # out: rows that no place names keep what they hold
    _, x = laid(g, T, k, type, gap)
    whole, rows = laid(None, R, k, type, gap)
    want = rows.clone()
    want[at[here]] = x[:, None, :].expand(T, K, k)[here]
    between = whole.clone()
    between.as_strided(rows.shape, rows.stride(), rows.storage_offset()).copy_(want)
    ops.route_rows(x, place, rows)
    torch.cuda.synchronize()
    assert torch.equal(whole, between)

    # back: what lies in rows that no choice has does not matter
    _, answers = laid(g, R, k, type, gap)
    named = torch.zeros(R, dtype=torch.bool, device=dev)
    named[at[here]] = True
    answers[~named] = float("nan")
    terms = torch.where(here[:, :, None], answers.double()[at.clamp(0, R - 1)], 0.0)
    for w in (weights, None):
        scaled = terms if w is None else terms * w.double()[:, :, None]
        whole, out = laid(None, T, k, type, gap)
        mark = whole.clone()
        ops.route_sum(answers, place, out, weights=w)
        torch.cuda.synchronize()
        value = scaled.sum(1)
        near(out, value, u(value, K * F * scaled.abs().sum(1)), "route_sum")
        mark.as_strided(out.shape, out.stride(), out.storage_offset()).copy_(out)
        assert torch.equal(whole, mark)

    # the gradient of back
    _, grad = laid(g, T, k, type, gap)
    whole, grad_rows = laid(None, R, k, type, gap)
    mark = whole.clone()
    grad_weights = torch.full((T, K), 5.0, device=dev)
    ops.route_sum_grad(grad, answers, place, weights, grad_rows, grad_weights)
    torch.cuda.synchronize()
    product = terms * grad.double()[:, None, :]
    near(grad_weights, product.sum(2), (k + 1) * F * product.abs().sum(2) + 2.0 ** -149, "weights")
    assert bool((grad_weights[~here] == 0).all())
    value = (weights.double()[:, :, None] * grad.double()[:, None, :])[here]
    near(grad_rows[at[here]], value, u(value, F * value.abs() + 2.0 ** -150), "grad_rows")
    mark.as_strided(grad_rows.shape, grad_rows.stride(), grad_rows.storage_offset())[at[here]] = grad_rows[at[here]]
    assert torch.equal(whole, mark)


@pytest.mark.parametrize("type", TYPES)
def test_sum_rounds_once_and_keeps_infinities(ops, dev, type):
    import torch
    announce("route_sum, special values", type)
    dt = getattr(torch, type)
    eps = torch.finfo(dt).eps
    # each of the small terms alone would be lost in the type, together they round up (in float32, the sum's own type, they are lost)
    rows = torch.tensor([[1.0], [eps / 4], [eps / 2], [float("inf")], [float("nan")], [0.0]], device=dev).to(dt)
    place = torch.tensor([[0, 1, 2], [0, 3, -1], [4, -1, -1], [-1, -1, -1], [3, 3, 5]], dtype=torch.int32, device=dev)
    weights = torch.tensor([[1, 1, 1], [1, -1, float("nan")], [1, float("inf"), 1], [float("nan")] * 3, [1, -1, 1]], device=dev)
    out = torch.full((5, 1), 7.0, device=dev).to(dt)
    ops.route_sum(rows, place, out, weights=weights)
    got = out.float().view(-1).tolist()
    assert got[0] == (1.0 if type == "float32" else 1.0 + eps)
    assert got[1] == float("-inf") and got[3] == 0.0
    assert np.isnan(got[2]) and np.isnan(got[4])


def test_gradients_against_differences(ops, dev):
    """route_sum is linear in its rows and in its weights: a difference over any step is the gradient, but for roundings."""
    import torch
    announce("route_sum_grad, differences")
    T, K, k, R = 37, 3, 21, 130
    g, rng = seeded(5), np.random.default_rng(5)
    place = places(rng, T, K, R, 0.2)
    rows, weights, c = normal(g, R, k), normal(g, T, K), normal(g, T, k)

    def loss(r, w):
        out = torch.empty(T, k, device=dev)
        ops.route_sum(r, place, out, weights=w)
        return out

    grad_rows, grad_weights = torch.zeros(R, k, device=dev), torch.empty(T, K, device=dev)
    ops.route_sum_grad(c, rows, place, weights, grad_rows, grad_weights)
    step = 0.5
    for r0, w0, r1, w1, along in [(rows, weights, rows, weights + step, grad_weights.double().sum()),
                                  (rows, weights, rows + step, weights, grad_rows.double().sum())]:
        a, b = loss(r0, w0), loss(r1, w1)
        got = ((b.double() - a.double()) * c.double()).sum() / step
        # rows + step and weights + step are off by F of themselves, every output by (K + 1) F of its terms' magnitudes
        most = float((weights.abs().max() + step) * (rows.abs().max() + step)) * K
        assert abs(float(got - along)) <= float(c.abs().double().sum()) * (2 * (K + 1) + 2) * F * most / step \
            + 2 * F * (k + 1) * T * K * k * float(c.abs().max() * (rows.abs().max() + weights.abs().max()))


def test_no_tokens_and_no_rows(ops, dev):
    import torch
    announce("route, nothing there")
    i32 = dict(dtype=torch.int32, device=dev)
    rows = torch.full((4, 6), 7.0, device=dev)
    empty, none = torch.empty(0, 6, device=dev), torch.empty(0, 2, **i32)
    ops.route_rows(empty, none, rows)
    ops.route_sum(rows, none, empty, weights=torch.empty(0, 2, device=dev))
    ops.route_sum_grad(empty, rows, none, torch.empty(0, 2, device=dev), rows.clone(), torch.empty(0, 2, device=dev))
    assert bool((rows == 7).all())
    # tokens without any row: nothing is here
    x, place = torch.ones(3, 6, device=dev), torch.tensor([[0, 1], [-1, 5], [0, 0]], **i32)
    weights, grad_weights = torch.full((3, 2), float("nan"), device=dev), torch.full((3, 2), 7.0, device=dev)
    out = torch.full((3, 6), 7.0, device=dev)
    ops.route_rows(x, place, empty)
    ops.route_sum(empty, place, out, weights=weights)
    ops.route_sum_grad(x, empty, place, weights, torch.empty_like(empty), grad_weights)
    assert bool((out == 0).all()) and bool((grad_weights == 0).all())
    y = torch.empty(0, 6, device=dev)
    ops.dropout(y, y, 0.5, 1)


def test_choices_of_one_expert_twice(ops, dev):
    """A token may name an expert twice: it has two rows there. Its row's gradient takes both."""
    import torch
    announce("route, the same expert twice")
    experts = torch.tensor([[1, 1], [0, 1], [1, 0]], device=dev)
    order, place, offsets = sort(ops, experts, 2)
    assert place.tolist() == [[2, 3], [0, 4], [5, 1]] and order.tolist() == [2, 5, 0, 1, 3, 4] and offsets.tolist() == [0, 2, 6]
    g = seeded(1)
    x, grad = normal(g, 3, 5), normal(g, 6, 5)
    rows, back = torch.zeros(6, 5, device=dev), torch.zeros(3, 5, device=dev)
    ops.route_rows(x, place, rows)
    assert torch.equal(rows, x[order.long() // 2])
    ops.route_sum(grad, place, back)
    assert torch.equal(back, grad[place.long()[:, 0]] + grad[place.long()[:, 1]])


# --- the relative position bias ----------------------------------------------------------------------------------

def plain_bucket(rel, buckets, far, two_sided):
    side = buckets // 2 if two_sided else buckets
    d = abs(rel) if two_sided else max(-rel, 0)
    near_, n = side // 2, side - side // 2
    row = d
    if d >= near_:
        row = near_
        while row < side - 1 and d ** n >= near_ ** (n - (row + 1 - near_)) * far ** (row + 1 - near_):
            row += 1
    return side + row if two_sided and rel > 0 else row


def plain_buckets(B, Q, K, buckets, far, two_sided, q_first, k_first, q_at):
    """[B, Q, K]"""
    import torch
    at = [0] * B if q_at is None else q_at.tolist()
    known = {}

    def row(q):
        lo = k_first - q
        for r in range(lo, lo + K):
            if r not in known:
                known[r] = plain_bucket(max(-far - 1, min(r, far + 1)), buckets, far, two_sided)
        return [known[r] for r in range(lo, lo + K)]
    one = {}
    for b in range(B):
        if at[b] not in one:
            one[at[b]] = torch.tensor([row(q_first + at[b] + i) for i in range(Q)]).view(Q, K)
    return torch.stack([one[at[b]] for b in range(B)]).cuda()


BIAS = [  # B, H, Q, K, buckets, far, two_sided, q_first, k_first, own positions
    (1, 1, 1, 1, 2, 2, False, 0, 0, False),
    (1, 3, 5, 7, 32, 128, True, 0, 0, False),
    (2, 4, 33, 65, 32, 128, True, 0, 0, False),
    (1, 2, 129, 1025, 32, 128, False, 0, 0, False),
    (3, 2, 300, 77, 8, 20, True, 1000, 990, False),
    (2, 1, 64, 2048, 64, 500, True, 0, 700, False),
    (5, 7, 1, 1500, 32, 128, False, 0, 0, True),
    (4, 3, 17, 300, 16, 60, True, 3, 1, True),
    (1, 2, 3, 5, 256, 2000, True, 0, 0, False),
    (1, 40, 70, 70, 255, 128, False, 0, 0, False),
    (1, 1, 40, 40, 32, 128, True, (1 << 60), (1 << 60) - 20, False),
    (1, 1, 9, 9, 32, 128, False, -(1 << 60), 1 << 60, False),
    (2, 2, 513, 511, 128, 1000, True, 0, 0, False),
    (70, 1000, 1, 3, 4, 5, True, 0, 0, False),
    (64, 13, 1, 5000, 32, 128, False, 0, 0, True),
    (3, 2, 8, 513, 32, 128, True, 0, 0, True),
    # few columns: planes of 2,048 elements, and what is behind the last of them; many batches to a workgroup; either side of 63, 80, 112 and 127
    (9, 2, 2049, 1, 32, 128, True, 0, 0, False),
    (6, 3, 1030, 2, 16, 300, False, 5, 0, True),
    (1, 2, 2000, 17, 64, 1500, False, 0, 1990, False),
    (130, 4, 49, 49, 32, 128, True, 0, 0, False),
    (200, 70, 50, 31, 32, 40, True, 0, 0, False),
    (2, 3, 17, 127, 256, 2000, True, 3, 1, True),
    (3, 5, 33, 128, 32, 128, True, 0, 0, False),
    (3, 5, 33, 129, 32, 128, True, 0, 0, False),
    (7, 3, 1, 100, 32, 128, False, 90, 0, False),
    (9, 2, 65, 63, 32, 128, True, 40, 0, True),
    (3, 2, 65, 64, 32, 128, True, 40, 0, True),
    (9, 2, 64, 63, 32, 128, True, 40, 0, True),
    (5, 2, 27, 20, 32, 128, True, 40, 0, True),
    (5, 2, 28, 20, 32, 128, True, 40, 0, True),
    (5, 3, 26, 80, 32, 128, True, 0, 0, False),
    (5, 3, 26, 81, 32, 128, True, 0, 0, False),
    (5, 3, 21, 112, 32, 128, True, 0, 0, False),
    (5, 3, 21, 113, 32, 128, True, 0, 0, False),
    (11, 3, 33, 127, 64, 128, False, 100, 0, False),
]


def spread(g, B, H, Q, K, type, how):
    """A tensor of this shape: dense, with gaps and an odd beginning, or [B, Q, H, K] in memory."""
    import torch
    if how == "dense":
        t = torch.full((B, H, Q, K), 9.0, device="cuda:0").to(getattr(torch, type))
    elif how == "gaps":
        whole = torch.full((1 + B * (H * (Q * (K + 3) + 2) + 1),), 9.0, device="cuda:0").to(getattr(torch, type))
        row, head = K + 3, Q * (K + 3) + 2
        t = whole[1:].as_strided((B, H, Q, K), (H * head + 1, head, row, 1))
    else:
        t = torch.full((B, Q, H, K), 9.0, device="cuda:0").to(getattr(torch, type)).transpose(1, 2)
    if g is not None:
        t.copy_(normal(g, B, H, Q, K, type=type))
    return t


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("case", BIAS)
@pytest.mark.parametrize("how", ["dense", "gaps", "queries first"])
def test_bias_and_gradient(ops, dev, type, case, how):
    import torch
    B, H, Q, K, buckets, far, two_sided, q_first, k_first, own = case
    announce("relbias, relbias_grad", type, case, how)
    g = seeded(B * 100 + K)
    at = torch.randint(0, 2 * K, (B,), generator=g, device=dev) if own else None
    if own:
        at[0] = 0
    bucket = plain_buckets(B, Q, K, buckets, far, two_sided, q_first, k_first, at)
    table = normal(g, buckets, H)
    more = dict(two_sided=two_sided, q_first=q_first, k_first=k_first, q_at=at)
    bias = table.double()[bucket].permute(0, 3, 1, 2)

    out = spread(None, B, H, Q, K, type, how)
    store = out.untyped_storage()
    mark = torch.tensor([], dtype=out.dtype, device=dev).set_(store).clone()
    ops.relbias(table, out, far, **more)
    torch.cuda.synchronize()
    near(out, bias, rounded(bias, 0.0, type), "bias")
    after = torch.tensor([], dtype=out.dtype, device=dev).set_(store).clone()
    mark.as_strided(out.shape, out.stride(), out.storage_offset()).copy_(out)
    assert torch.equal(after, mark)  # nothing between the rows

    scores = spread(g, B, H, Q, K, type, how)
    want = scores.double() + bias
    tolerance = rounded(want, F * want.abs(), type)
    ops.relbias(table, out, far, scores=scores, **more)
    near(out, want, tolerance, "scores")
    shared = scores[:1, :, :, :].expand(B, H, Q, K)
    want = shared.double() + bias
    ops.relbias(table, out, far, scores=shared, **more)
    near(out, want, rounded(want, F * want.abs(), type), "shared scores")
    before = scores.double()
    ops.relbias(table, scores, far, scores=scores, **more)
    near(scores, before + bias, tolerance, "in place")

    grad = spread(g, B, H, Q, K, type, how)
    grad_table = torch.full((buckets, H), 9.0, device=dev)
    ops.relbias_grad(grad, grad_table, far, **more)
    hot = torch.zeros(buckets, H, dtype=torch.float64, device=dev)
    size = hot.clone()
    for h in range(H):
        flat = grad[:, h].double().reshape(-1)
        hot[:, h].index_add_(0, bucket.reshape(-1), flat)
        size[:, h].index_add_(0, bucket.reshape(-1), flat.abs())
    # no chain of additions is longer than 1,024 and the batch (and no longer than its terms)
    near(grad_table, hot, (1024 + B) * F * size, "gradient")


def test_gradient_of_bias_against_differences(ops, dev):
    """The bias is linear in its table: the difference over a step is the gradient, but for roundings."""
    import torch
    announce("relbias_grad, differences")
    g = seeded(11)
    H, Q, K, buckets = 3, 50, 61, 32
    table, c = normal(g, buckets, H), normal(g, 1, H, Q, K)
    grad = torch.empty(buckets, H, device=dev)
    ops.relbias_grad(c, grad, 128)
    step = torch.zeros_like(table)
    for u in (0, 1, 7, 8, 15, 17, 31):
        step.zero_()[u] = 0.5
        a, b = torch.empty_like(c), torch.empty_like(c)
        ops.relbias(table, a, 128)
        ops.relbias(table + step, b, 128)
        got = ((b.double() - a.double()) * c.double()).sum() / 0.5
        # table + step is off by F of itself, at each of Q * K * H places at most
        slack = float(c.abs().double().sum()) * 2 * F * (float(table.abs().max()) + 0.5) / 0.5 + Q * K * F * float(c.abs().sum())
        assert abs(float(got - grad[u].double().sum())) <= slack


@pytest.mark.parametrize("type,B,H,Q,K", [("bfloat16", 2, 64, 1021, 2100), ("float32", 3, 30, 700, 1000), ("float16", 9, 16, 300, 520)])
def test_gradient_of_many_rows(ops, dev, type, B, H, Q, K):
    """Sizes at which a wavefront takes 128 rows, or several batches."""
    import torch
    announce("relbias_grad, large", type, B, H, Q, K)
    grad = normal(seeded(3), B, H, Q, K, type=type)
    got = torch.empty(32, H, device=dev)
    ops.relbias_grad(grad, got, 128)
    far = max(Q, K)
    bucket = torch.tensor([plain_bucket(r, 32, 128, True) for r in range(-far, far + 1)], device=dev)
    at = bucket[torch.arange(K, device=dev)[None, :] - torch.arange(Q, device=dev)[:, None] + far]
    total, size = grad.sum(0, dtype=torch.float64), grad.abs().sum(0, dtype=torch.float64)
    for u in range(32):
        here = at == u
        near(got[u], torch.where(here, total, 0.0).sum((1, 2)), (1024 + B) * F * torch.where(here, size, 0.0).sum((1, 2)), "bucket %d" % u)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("narrow", [False, True])
def test_infinities_stay_in_their_bucket(ops, dev, type, narrow):
    import torch
    announce("relbias_grad, special values", type, narrow)
    H, Q, K = (3, 613, 70) if narrow else (3, 70, 613)
    grad = normal(seeded(4), 2, H, Q, K, type=type)
    clean = torch.empty(32, H, device=dev)
    ops.relbias_grad(grad, clean, 128)
    want = clean.clone()
    for h, i, j, value in [(0, 5, 5, float("inf")), (1, 69, 612, float("nan")), (2, 69, 0, float("-inf")), (2, 0, 3, float("inf")),
                           (0, 33, 610, float("nan"))]:
        if narrow:
            i, j = j, i
        grad[1, h, i, j] = value
        u = plain_bucket(j - i, 32, 128, True)
        want[u, h] = float("nan") if not np.isinf(value) or not torch.isfinite(want[u, h]) else value
    got = torch.empty(32, H, device=dev)
    ops.relbias_grad(grad, got, 128)
    assert torch.equal(torch.nan_to_num(got, nan=1e30), torch.nan_to_num(want, nan=1e30))


def test_bias_without_batch_and_empty(ops, dev):
    import torch
    announce("relbias, three dimensions and none")
    g = seeded(2)
    table = normal(g, 32, 4)
    a, b = torch.empty(4, 9, 11, device=dev), torch.empty(1, 4, 9, 11, device=dev)
    ops.relbias(table, a, 128)
    ops.relbias(table, b, 128)
    assert torch.equal(a, b[0])
    for shape in [(0, 4, 3, 3), (2, 4, 0, 3), (2, 4, 3, 0)]:
        ops.relbias(table, torch.empty(shape, device=dev), 128)
        grad = torch.full((32, 4), 3.0, device=dev)
        ops.relbias_grad(torch.empty(shape, device=dev), grad, 128)
        assert bool((grad == 0).all())


def test_bias_keeps_masked_scores(ops, dev):
    import torch
    announce("relbias, masked scores")
    for type in TYPES:
        dt = getattr(torch, type)
        scores = torch.zeros(1, 2, 5, 40, device=dev).to(dt)
        scores[..., 1::3] = float("-inf")
        scores[..., 2::3] = torch.finfo(dt).min
        scores[0, 1, 3] = float("nan")
        table = torch.ones(32, 2, device=dev)
        out = torch.empty_like(scores)
        ops.relbias(table, out, 128, scores=scores)
        want = (scores.float() + 1.0).to(dt)
        assert torch.equal(torch.nan_to_num(out.float(), nan=123.0), torch.nan_to_num(want.float(), nan=123.0))


# --- dropout -----------------------------------------------------------------------------------------------------

def plain_bits(keys, k, seed):
    """[n, k]: the 16 bits of every element, from the generator's definition."""
    n, blocks = keys.size, -(-k // 8)
    M = 0xFFFFFFFF
    c = [np.repeat(keys & np.uint64(M), blocks), np.repeat(keys >> np.uint64(32), blocks),
         np.tile(np.arange(blocks, dtype=np.uint64), n), np.zeros(n * blocks, np.uint64)]
    k0, k1 = seed & M, seed >> 32
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & np.uint64(M), (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & np.uint64(M)]
        k0, k1 = (k0 + 0x9E3779B9) & M, (k1 + 0xBB67AE85) & M
    out = np.empty((n * blocks, 8), np.int64)
    for w in range(4):
        out[:, 2 * w], out[:, 2 * w + 1] = c[w] & np.uint64(0xFFFF), c[w] >> np.uint64(16)
    return out.reshape(n, blocks * 8)[:, :k]


DROPS = [(1, 1, 0), (1, 8, 0), (3, 7, 2), (5, 9, 0), (17, 64, 0), (33, 100, 4), (4, 1001, 0), (1000, 24, 0), (2, 4099, 5), (257, 3, 0)]


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("n,k,gap", DROPS)
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.999, 1.0])
def test_dropout(ops, dev, type, n, k, gap, p):
    import torch
    announce("dropout", type, n, k, gap, p)
    g, rng = seeded(n * k), np.random.default_rng(n + k)
    _, x = laid(g, n, k, type, gap)
    x[0, 0] = float("nan")
    x[-1, -1] = float("inf")
    seed = int(rng.integers(0, 1 << 64, dtype=np.uint64))
    keys = rng.integers(0, 1 << 64, n, dtype=np.uint64)
    least = int(np.floor(p * 65536 + 0.5))
    scale = 65536.0 / (65536 - least) if least < 65536 else 0.0
    d_keys = torch.from_numpy(keys.view(np.int64)).to(dev)
    first = int(keys[0]) >> 1
    counted = (np.arange(n, dtype=np.uint64) + np.uint64(first))
    step = torch.tensor([41], device=dev)
    for which, more in [(keys, dict(keys=d_keys)), (counted, dict(first=first)), (keys, dict(keys=d_keys, step=step))]:
        bits = plain_bits(which, k, seed + (41 if "step" in more else 0) & ((1 << 64) - 1))
        keep = torch.from_numpy(bits >= least).to(dev)
        want = torch.where(keep, x.double() * scale, 0.0)
        whole, out = laid(None, n, k, type, gap)
        mark = whole.clone()
        ops.dropout(x, out, p, seed, **more)
        torch.cuda.synchronize()
        assert bool((out[~keep] == 0).all())
        fine = torch.isfinite(want)
        near(out[fine], want[fine], rounded(want[fine], 2 * F * want[fine].abs() + 2.0 ** -149, type), "dropout")
        assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(torch.isinf(out) & ~torch.isinf(x), torch.zeros_like(keep))
        mark.as_strided(out.shape, out.stride(), out.storage_offset()).copy_(out)
        assert torch.equal(torch.nan_to_num(whole), torch.nan_to_num(mark))
    inside = x.clone()
    ops.dropout(x, out, p, seed, keys=d_keys)
    ops.dropout(inside, inside, p, seed, keys=d_keys)
    assert torch.equal(torch.nan_to_num(inside), torch.nan_to_num(out))


def test_dropout_goes_by_keys(ops, dev):
    """The gradient's rows may come in another order and in pieces; their keys bring the same mask back."""
    import torch
    announce("dropout, order and pieces")
    g = seeded(9)
    n, k = 500, 37
    keys = torch.randint(-(1 << 63), (1 << 63) - 1, (n,), generator=g, device=dev)
    ones = torch.ones(n, k, device=dev)
    out, other = torch.empty_like(ones), torch.empty_like(ones)
    ops.dropout(ones, out, 0.3, 12345, keys=keys)
    perm = torch.randperm(n, generator=g, device=dev)
    for a, b in [(0, 1), (1, 200), (200, 500)]:
        ops.dropout(ones[a:b], other[a:b], 0.3, 12345, keys=keys[perm[a:b]])
    assert torch.equal(other, out[perm])
    ops.dropout(ones, out, 0.3, 7, first=100)
    ops.dropout(ones[20:], other[20:], 0.3, 7, first=120)
    assert torch.equal(other[20:], out[20:])
    # how many stay: 18,500 draws of 0.7, five standard deviations
    kept = float((out != 0).double().mean())
    assert abs(kept - 0.7) < 5 * (0.21 / (n * k)) ** 0.5


# --- how they are called -----------------------------------------------------------------------------------------

def test_shapes_and_types_are_refused(ops, capi, dev):
    import torch
    announce("ops, refusals")
    i32 = dict(dtype=torch.int32, device=dev)
    x, rows = torch.zeros(4, 8, device=dev), torch.zeros(8, 8, device=dev)
    place, w = torch.zeros(4, 2, **i32), torch.zeros(4, 2, device=dev)
    order, offsets, table, s = torch.zeros(8, **i32), torch.zeros(5, **i32), torch.zeros(32, 2, device=dev), torch.zeros(2, 2, 4, 4, device=dev)
    wide = torch.zeros(8, 16, device=dev)
    bad = [
        (TypeError, lambda: ops.route_sort(w, 4, order, place, offsets)), (TypeError, lambda: ops.route_sort(place, 4, order.long(), place, offsets)),
        (ValueError, lambda: ops.route_sort(place, 4, order[:7], place, offsets)), (ValueError, lambda: ops.route_sort(place, 5, order, place, offsets)),
        (ValueError, lambda: ops.route_sort(place.t(), 4, order, place, offsets)), (ValueError, lambda: ops.route_sort(place, 4, order, place[:3], offsets)),
        (TypeError, lambda: ops.route_rows(x.double(), place, rows)), (TypeError, lambda: ops.route_rows(x.half(), place, rows)),
        (ValueError, lambda: ops.route_rows(x[:3], place, rows)), (ValueError, lambda: ops.route_rows(x, place, rows[:, :7])),
        (ValueError, lambda: ops.route_rows(rows.t()[:4], place, rows)), (ValueError, lambda: ops.route_rows(x[0], place, rows)),
        (TypeError, lambda: ops.route_rows(x, place.long(), rows)), (ValueError, lambda: ops.route_rows(x, place.view(-1), rows)),
        (capi.PskvError, lambda: ops.route_rows(rows[:4], place, rows)), (capi.PskvError, lambda: ops.route_rows(x, place, x[:1].expand(8, 8))),
        (ValueError, lambda: ops.route_sum(rows, place, x, weights=w[:, :1])), (TypeError, lambda: ops.route_sum(rows, place, x, weights=w.half())),
        (ValueError, lambda: ops.route_sum(rows, place, x[:3])), (capi.PskvError, lambda: ops.route_sum(rows, place, rows[2:6])),
        (ValueError, lambda: ops.route_sum_grad(x, rows, place, w, rows[:7].clone(), w.clone())),
        (ValueError, lambda: ops.route_sum_grad(x[:3], rows, place, w, rows.clone(), w.clone())),
        (capi.PskvError, lambda: ops.route_sum_grad(x, rows, place, w, rows, w.clone())),
        (ValueError, lambda: ops.relbias(table, s[0, 0], 128)), (ValueError, lambda: ops.relbias(table[:, :1], s, 128)),
        (TypeError, lambda: ops.relbias(table.half(), s, 128)), (ValueError, lambda: ops.relbias(table, s, 128, scores=s[:1])),
        (TypeError, lambda: ops.relbias(table, s, 128, scores=s.half())), (ValueError, lambda: ops.relbias(table, s.transpose(2, 3), 128)),
        (TypeError, lambda: ops.relbias(table, s, 128, q_at=place[:2, 0])), (ValueError, lambda: ops.relbias(table, s, 128, q_at=torch.zeros(3, dtype=torch.int64, device=dev))),
        (capi.PskvError, lambda: ops.relbias(table, s, 8)), (capi.PskvError, lambda: ops.relbias(table, s[:, :1].expand(2, 2, 4, 4), 128)),
        (ValueError, lambda: ops.relbias_grad(s, table[:, :1], 128)), (TypeError, lambda: ops.relbias_grad(s, table.double(), 128)),
        (capi.PskvError, lambda: ops.relbias_grad(torch.zeros(2, 2, 100, 100, device=dev), table, 128, work=order)),
        (ValueError, lambda: ops.dropout(x, rows, 0.5, 1)), (capi.PskvError, lambda: ops.dropout(x, x, 1.5, 1)),
        (ValueError, lambda: ops.dropout(x, x, 0.5, 1, keys=order.long())), (TypeError, lambda: ops.dropout(x, x, 0.5, 1, keys=order[:4])),
        (OverflowError, lambda: ops.dropout(x, x, 0.5, 1 << 64)), (TypeError, lambda: ops.dropout(x, x, 0.5, 1, step=order[:1])),
        (capi.PskvError, lambda: ops.dropout(wide[:, :8], wide[:, 1:9], 0.5, 1)),
        (ValueError, lambda: ops.dropout(x, x.cpu(), 0.5, 1)),
    ]
    for i, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            pytest.fail("refusal %d" % i)
    ops.dropout(wide[:, :8], wide[:, 8:], 0.5, 1)  # columns beside each other are fine
    ops.route_rows(x[:1].expand(4, 8), place[:, :1].contiguous(), rows)  # so is one row read four times
    torch.cuda.synchronize()


def test_numbers_and_working_memory_of_other_types(ops, dev):
    import torch
    announce("ops, numpy numbers, bytes as working memory")
    experts = torch.randint(0, 9, (5000, 1), device=dev)
    work = torch.empty(ops.route_room(5000, 9), dtype=torch.uint8, device=dev)
    a, b = sort(ops, experts, 9), sort(ops, experts, np.int64(9), work=work)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    x = torch.ones(4, 9, device=dev)
    y, z = torch.empty_like(x), torch.empty_like(x)
    ops.dropout(x, y, 0.5, 77)
    ops.dropout(x, z, np.float64(0.5), np.uint64(77))
    assert torch.equal(y, z)
    with pytest.raises(ValueError):
        ops.route_sort(experts, 9, a[0], a[1], a[2], work=work[::2])
    with pytest.raises(ValueError):
        ops.route_sort(experts, 9, a[0], a[1], a[2], work=work.cpu())


def test_many_choices(ops, dev):
    import torch
    announce("route_sort, 20,000,001 choices")
    g = seeded(8)
    experts = torch.randint(-1, 300, (20000001, 1), generator=g, device=dev, dtype=torch.int32)
    order, place, offsets = sort(ops, experts, 300)
    key = torch.where(experts.view(-1) < 0, 300, experts.view(-1))
    held = torch.sort(key, stable=True)
    n = int((held.values < 300).sum())
    assert torch.equal(order[:n], held.indices[:n].to(torch.int32)) and bool((order[n:] == -1).all())
    assert torch.equal(offsets, torch.searchsorted(held.values, torch.arange(301, device=dev, dtype=torch.int32)).to(torch.int32))
    assert torch.equal(place.view(-1)[held.indices[:n]], torch.arange(n, device=dev, dtype=torch.int32))
    assert bool((place.view(-1)[held.indices[n:]] == -1).all())


def test_rows_beyond_32_bits(ops, dev):
    """Rows that lie 2^32 elements and more into their memory."""
    import torch
    announce("route, 70,001 rows of 65,536")
    R, k = 70001, 65536
    g = seeded(6)
    rows = torch.zeros(R, k, dtype=torch.bfloat16, device=dev)
    x, grad = normal(g, 3, k, type="bfloat16"), normal(g, 3, k, type="bfloat16")
    place = torch.tensor([[0, R - 1], [65537, -1], [R - 2, 32769]], dtype=torch.int32, device=dev)
    ops.route_rows(x, place, rows)
    named = torch.tensor([0, R - 1, 65537, R - 2, 32769], device=dev)
    assert torch.equal(rows[named], x[torch.tensor([0, 0, 1, 2, 2], device=dev)])
    rows[named] = 0
    assert not bool(rows.view(torch.int32).any())
    answers = normal(g, 5, k, type="bfloat16")
    rows[named] = answers
    out = torch.empty_like(x)
    ops.route_sum(rows, place, out)
    want = torch.stack([answers[0].double() + answers[1].double(), answers[2].double(), answers[3].double() + answers[4].double()])
    near(out, want, rounded(want, 2 * F * want.abs(), "bfloat16"), "sum")
    weights, grad_weights = torch.ones(3, 2, device=dev), torch.empty(3, 2, device=dev)
    grad_rows = torch.zeros_like(rows)
    ops.route_sum_grad(grad, rows, place, weights, grad_rows, grad_weights)
    assert torch.equal(grad_rows[named], grad[torch.tensor([0, 0, 1, 2, 2], device=dev)])
    grad_rows[named] = 0
    assert not bool(grad_rows.view(torch.int32).any())


@pytest.mark.parametrize("K", [601, 60])
def test_scores_beyond_32_bits(ops, dev, K):
    import torch
    announce("relbias, a batch 2^31 elements apart", K)
    B, H, Q, apart = 3, 2, 9, (1 << 31) + 24
    whole = torch.zeros((B - 1) * apart + H * Q * K, dtype=torch.bfloat16, device=dev)
    out = whole.as_strided((B, H, Q, K), (apart, Q * K, K, 1))
    g = seeded(7)
    table, scores = normal(g, 32, H), normal(g, B, H, Q, K, type="bfloat16")
    plain, sums, more = torch.empty_like(scores), torch.empty_like(table), torch.empty_like(table)
    ops.relbias(table, plain, 128, scores=scores)
    ops.relbias(table, out, 128, scores=scores)
    assert torch.equal(out, plain)
    ops.relbias(table, out, 128, scores=out)
    ops.relbias(table, plain, 128, scores=plain)
    assert torch.equal(out, plain)
    ops.relbias_grad(out, sums, 128)
    ops.relbias_grad(plain, more, 128)
    assert torch.equal(sums, more)


@pytest.mark.parametrize("type", ["bfloat16", "float32"])
def test_dropout_in_pieces(ops, dev, type):
    """More rows than one launch counts."""
    import torch
    announce("dropout, 2^31 + 1000 rows", type)
    n = (1 << 31) + 1000
    x = torch.full((1, 1), 2.0, device=dev).to(getattr(torch, type)).expand(n, 1)
    out = torch.empty(n, 1, dtype=getattr(torch, type), device=dev)
    ops.dropout(x, out, 0.5, 1234, first=5)
    for at in (0, (1 << 31) - 600, (1 << 31) - 512, (1 << 31) - 300, (1 << 31) - 10, n - 100):
        keep = plain_bits(np.arange(at + 5, at + 105, dtype=np.uint64), 1, 1234) >= 32768
        assert np.array_equal(out[at:at + 100].float().cpu().numpy(), np.where(keep, 4.0, 0.0)), at


def test_two_threads(ops, capi, dev):
    """Calls share no state: two threads, each on a stream of its own."""
    import threading
    import torch
    announce("ops, two threads")
    plain = chain_state(ops, capi, dev, 3)
    chain(ops, plain)
    states, sides = [chain_state(ops, capi, dev, 3) for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()

    def work(s, side):
        with torch.cuda.stream(side):
            for _ in range(20):
                chain(ops, s)

    threads = [threading.Thread(target=work, args=a) for a in zip(states, sides)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for s in states:
        for name in ANSWERS:
            assert torch.equal(s[name], plain[name]), name


def chain(ops, s):
    """A worker's step with everything in it."""
    import torch
    ops.route_sort(s["experts"], 40, s["order"], s["place"], s["offsets"], work=s["work"])
    ops.dropout(s["x"], s["dropped"], 0.2, 99, keys=s["keys"], step=s["step"])
    ops.route_rows(s["dropped"], s["place"], s["rows"])
    ops.route_sum(s["rows"], s["place"], s["out"], weights=s["weights"])
    ops.route_sum_grad(s["out"], s["rows"], s["place"], s["weights"], s["grad_rows"], s["grad_weights"])
    ops.route_sum(s["grad_rows"], s["place"], s["grad_x"])
    ops.dropout(s["grad_x"], s["grad_x"], 0.2, 99, keys=s["keys"], step=s["step"])
    ops.relbias(s["table"], s["scores_out"], 128, scores=s["scores"], q_at=s["at"])
    ops.relbias_grad(s["scores_out"], s["grad_table"], 128, q_at=s["at"], work=s["bias_work"])


ANSWERS = ["order", "place", "offsets", "dropped", "rows", "out", "grad_rows", "grad_weights", "grad_x", "scores_out", "grad_table"]


def chain_state(ops, capi, dev, seed, type="bfloat16"):
    import torch
    g = seeded(seed)
    T, K, k, dt = 6000, 3, 40, getattr(torch, type)
    n = T * K
    i32 = dict(dtype=torch.int32, device=dev)
    room = ops.relbias_grad_room(32, 2, 3, 20, 300, own_positions=True)
    return {"experts": torch.randint(-2, 40, (T, K), generator=g, device=dev), "x": normal(g, T, k, type=type),
            "keys": torch.randint(-(1 << 63), (1 << 63) - 1, (T,), generator=g, device=dev), "step": torch.zeros(1, dtype=torch.int64, device=dev),
            "weights": torch.rand(T, K, generator=g, device=dev), "table": normal(g, 32, 3), "scores": normal(g, 2, 3, 20, 300, type=type),
            "at": torch.randint(0, 300, (2,), generator=g, device=dev),
            "order": torch.zeros(n, **i32), "place": torch.zeros(T, K, **i32), "offsets": torch.zeros(41, **i32),
            "dropped": torch.zeros(T, k, dtype=dt, device=dev), "rows": torch.zeros(n, k, dtype=dt, device=dev),
            "out": torch.zeros(T, k, dtype=dt, device=dev), "grad_rows": torch.zeros(n, k, dtype=dt, device=dev),
            "grad_weights": torch.zeros(T, K, device=dev), "grad_x": torch.zeros(T, k, dtype=dt, device=dev),
            "scores_out": torch.zeros(2, 3, 20, 300, dtype=dt, device=dev), "grad_table": torch.zeros(32, 3, device=dev),
            "work": torch.zeros(ops.route_room(n, 40) // 4, **i32), "bias_work": torch.zeros(room // 4, **i32)}


def fresh(s, g):
    """Other inputs, in place."""
    import torch
    s["experts"].copy_(torch.randint(-2, 40, s["experts"].shape, generator=g, device=s["x"].device))
    s["x"].copy_(torch.randn(s["x"].shape, generator=g, device=s["x"].device))
    s["scores"].copy_(torch.randn(s["scores"].shape, generator=g, device=s["x"].device))
    s["at"].copy_(torch.randint(0, 300, (2,), generator=g, device=s["x"].device))
    s["step"].add_(1)
    for name in ("rows", "grad_rows"):
        s[name].zero_()


def test_captured_and_replayed(ops, capi, dev):
    """Two graphs of the same calls, each with working memory of its own, replayed in turn with eager work between."""
    import torch
    announce("ops, captured")
    states = [chain_state(ops, capi, dev, seed) for seed in (1, 2)]
    eager = [{k: v.clone() for k, v in s.items()} for s in states]
    for s in states:
        chain(ops, s)  # (the first call, outside any capture)
    torch.cuda.synchronize()
    graphs = []
    for s in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            chain(ops, s)
        graphs.append(graph)
    g = seeded(77)
    for round_ in range(4):
        for s, e in zip(states, eager):
            fresh(s, g)
            for name in ("experts", "x", "scores", "at", "step"):
                e[name].copy_(s[name])
            for name in ("rows", "grad_rows"):
                e[name].zero_()
        graphs[0].replay()
        if round_ % 2:
            torch.cuda.synchronize()
            chain(ops, eager[0])
        graphs[1].replay()
        for e in eager:
            chain(ops, e)
        torch.cuda.synchronize()
        for s, e in zip(states, eager):
            for name in ANSWERS:
                assert torch.equal(s[name], e[name]), (round_, name)


def test_on_another_stream(ops, capi, dev):
    """On torch's current stream, whichever it is, and on a stream that is named; two streams at once; the same bits every time."""
    import torch
    announce("ops, streams")
    plain = chain_state(ops, capi, dev, 3)
    chain(ops, plain)
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    others = [chain_state(ops, capi, dev, 3) for _ in sides]
    torch.cuda.synchronize()
    for _ in range(3):
        for side, s in zip(sides, others):
            with torch.cuda.stream(side):
                chain(ops, s)
    torch.cuda.synchronize()
    for s in others:
        for name in ANSWERS:
            assert torch.equal(s[name], plain[name]), name
    # a named stream, working memory by itself
    s = chain_state(ops, capi, dev, 3)
    at = sides[0].cuda_stream
    torch.cuda.synchronize()
    ops.route_sort(s["experts"], 40, s["order"], s["place"], s["offsets"], stream=at)
    ops.relbias(s["table"], s["scores_out"], 128, scores=s["scores"], q_at=s["at"], stream=at)
    ops.relbias_grad(s["scores_out"], s["grad_table"], 128, q_at=s["at"], stream=at)
    sides[0].synchronize()
    for name in ("order", "place", "offsets", "scores_out", "grad_table"):
        assert torch.equal(s[name], plain[name]), name


def test_between_pull_and_push(ops, capi, dev):
    """A worker's step next to the store: rows of the biases and of the tokens are pulled, used, and their gradients pushed."""
    import torch
    announce("ops with tables")
    g = seeded(21)
    H, buckets, T, K, E, k = 4, 32, 300, 2, 6, 24
    bias_keys = torch.arange(100, 100 + buckets, device=dev)
    token_keys = torch.sort(torch.randperm(10000, generator=g, device=dev)[:T]).values
    biases, tokens = capi.Table(capi.MODE_FIXED, row_len=H), capi.Table(capi.MODE_FIXED, row_len=k)
    b0, t0 = normal(g, buckets, H), normal(g, T, k)
    biases.push(bias_keys, b0.view(-1))
    tokens.push(token_keys, t0.view(-1))
    table, x = torch.empty(buckets, H, device=dev), torch.empty(T, k, device=dev)
    biases.pull(bias_keys, table.view(-1))
    tokens.pull(token_keys, x.view(-1))
    biases.sync()
    tokens.sync()
    assert torch.equal(table, b0) and torch.equal(x, t0)

    scores = normal(g, 2, H, 30, 50)
    biased, grad_table = torch.empty_like(scores), torch.empty(buckets, H, device=dev)
    ops.relbias(table, biased, 128, scores=scores)
    ops.relbias_grad(biased, grad_table, 128)

    experts = torch.randint(0, E, (T, K), generator=g, device=dev)
    weights = torch.rand(T, K, generator=g, device=dev)
    _, place, offsets = sort(ops, experts, E)
    dropped, rows = torch.empty_like(x), torch.zeros(T * K, k, device=dev)
    ops.dropout(x, dropped, 0.25, 5, keys=token_keys)
    ops.route_rows(dropped, place, rows)
    products = normal(g, E, k, k)
    answers = torch.empty_like(rows)
    bounds = offsets.tolist()
    for e in range(E):
        answers[bounds[e]:bounds[e + 1]] = rows[bounds[e]:bounds[e + 1]] @ products[e]
    out = torch.empty_like(x)
    ops.route_sum(answers, place, out, weights=weights)
    dy = normal(g, T, k)
    grad_answers, grad_weights = torch.zeros_like(answers), torch.empty_like(weights)
    ops.route_sum_grad(dy, answers, place, weights, grad_answers, grad_weights)
    grad_rows = torch.zeros_like(rows)
    for e in range(E):
        grad_rows[bounds[e]:bounds[e + 1]] = grad_answers[bounds[e]:bounds[e + 1]] @ products[e].t().contiguous()
    grad_x = torch.empty_like(x)
    ops.route_sum(grad_rows, place, grad_x)
    ops.dropout(grad_x, grad_x, 0.25, 5, keys=token_keys)

    # the same in 64 bits
    keep = torch.from_numpy(plain_bits(token_keys.cpu().numpy().view(np.uint64), k, 5) >= 16384).to(dev)
    dx = torch.where(keep, x.double() * (4 / 3), 0.0)
    per = products.double()[experts]  # [T, K, k, k]
    ans = (dx[:, None, None, :] * per.transpose(2, 3)).sum(3)
    want = (weights.double()[:, :, None] * ans).sum(1)
    # k-term products, then a sum of K: magnitudes first
    size = (dx.abs()[:, None, None, :] * per.abs().transpose(2, 3)).sum(3)
    near(out, want, (k + K + 6) * F * (weights.double()[:, :, None] * size).sum(1) + 2.0 ** -120, "out")
    back = weights.double()[:, :, None] * dy.double()[:, None, :]
    through, reach = (back[:, :, None, :] * per).sum(3), (back.abs()[:, :, None, :] * per.abs()).sum(3)
    near(grad_x, torch.where(keep, through.sum(1) * (4 / 3), 0.0), (k + K + 6) * F * reach.sum(1) * (4 / 3) + 2.0 ** -120, "grad_x")
    near(grad_weights, (ans * dy.double()[:, None, :]).sum(2), (2 * k + 6) * F * (size * dy.double().abs()[:, None, :]).sum(2) + 2.0 ** -120,
         "grad_weights")

    biases.push(bias_keys, grad_table.view(-1))
    tokens.push(token_keys, grad_x.view(-1))
    biases.pull(bias_keys, table.view(-1))
    tokens.pull(token_keys, x.view(-1))
    biases.sync()
    tokens.sync()
    assert torch.equal(table, b0 + grad_table) and torch.equal(x, t0 + grad_x)
