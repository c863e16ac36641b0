"""Calls of the operators on rows that their documentation allows and that no other test makes."""
import pytest

from conftest import announce
from test_gpu_ops import ANSWERS, chain, chain_state, normal, ops, seeded  # noqa: F401

pytestmark = pytest.mark.gpu


def test_on_the_null_stream(ops, capi, dev):
    """`stream` is an address: 0 is the null stream, and working memory that a call takes by itself belongs to it."""
    import torch
    announce("ops, the null stream by its address")
    plain, s = (chain_state(ops, capi, dev, 3) for _ in range(2))
    chain(ops, plain)
    torch.cuda.synchronize()
    for _ in range(3):
        ops.route_sort(s["experts"], 40, s["order"], s["place"], s["offsets"], stream=0)
        ops.relbias(s["table"], s["scores_out"], 128, scores=s["scores"], q_at=s["at"], stream=0)
        ops.relbias_grad(s["scores_out"], s["grad_table"], 128, q_at=s["at"], stream=0)
    torch.cuda.synchronize()
    for name in ("order", "place", "offsets", "scores_out", "grad_table"):
        assert torch.equal(s[name], plain[name]), name


def test_captured_with_working_memory_of_their_own(ops, capi, dev):
    """Two graphs whose calls take working memory by themselves, replayed at once on two streams."""
    import torch
    announce("ops, captured, working memory by themselves")
    states = [chain_state(ops, capi, dev, seed) for seed in (1, 2)]
    plain = [chain_state(ops, capi, dev, seed) for seed in (1, 2)]

    def calls(s):
        ops.route_sort(s["experts"], 40, s["order"], s["place"], s["offsets"])
        ops.relbias_grad(s["scores"], s["grad_table"], 128, q_at=s["at"])

    for s in plain + states:
        calls(s)
    torch.cuda.synchronize()
    graphs = []
    for s in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            calls(s)
        graphs.append(graph)
    sides = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for s in states:
            for name in ("order", "place", "offsets", "grad_table"):
                s[name].fill_(7)
        torch.cuda.synchronize()
        for graph, side in zip(graphs, sides):
            with torch.cuda.stream(side):
                graph.replay()
        torch.empty(1 << 20, device=dev).fill_(3.0)  # (eager work beside them)
        torch.cuda.synchronize()
        for s, p in zip(states, plain):
            for name in ("order", "place", "offsets", "grad_table"):
                assert torch.equal(s[name], p[name]), name


def test_unsigned_keys_and_experts(ops, dev):
    import torch
    announce("ops, uint64")
    g = seeded(4)
    experts = torch.randint(-2, 9, (700, 2), generator=g, device=dev)
    answers = []
    for e in (experts, experts.view(torch.uint64)):
        order, place = (torch.empty(1400, dtype=torch.int32, device=dev) for _ in range(2))
        offsets = torch.empty(10, dtype=torch.int32, device=dev)
        ops.route_sort(e, 9, order, place, offsets)
        answers.append((order, place, offsets))
    assert all(torch.equal(a, b) for a, b in zip(*answers))
    x = normal(g, 30, 21)
    keys = torch.randint(-(1 << 63), (1 << 63) - 1, (30,), generator=g, device=dev)
    a, b = torch.empty_like(x), torch.empty_like(x)
    ops.dropout(x, a, 0.5, 3, keys=keys)
    ops.dropout(x, b, 0.5, 3, keys=keys.view(torch.uint64))
    assert torch.equal(a, b)


def test_a_seed_and_a_step_are_one_number(ops, dev):
    """What the documentation says of seeds that share a step: d apart, they draw the same d steps later."""
    import torch
    announce("dropout, seeds and steps")
    x = torch.ones(50, 40, device=dev)
    out = [torch.empty_like(x) for _ in range(3)]
    ops.dropout(x, out[0], 0.5, 100, step=torch.tensor([7], device=dev))
    ops.dropout(x, out[1], 0.5, 107)
    ops.dropout(x, out[2], 0.5, (1 << 64) - 1, step=torch.tensor([108], device=dev))
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])


def test_what_lies_upon_each_other_is_refused(ops, capi, dev):
    """From Python, with tensors; nothing is launched, so they keep what they hold."""
    import torch
    announce("ops, aliases")
    i32 = torch.int32
    x, rows, w = torch.ones(4, 8, device=dev), torch.ones(8, 8, device=dev), torch.ones(4, 2, device=dev)
    place = torch.arange(8, dtype=i32, device=dev).view(4, 2)
    scores, keys = torch.ones(1, 2, 16, 16, device=dev), torch.ones(16, dtype=torch.int64, device=dev)
    calls = [lambda: ops.route_rows(x, rows.view(-1)[:8].view(i32).view(4, 2), rows), lambda: ops.route_sum(rows, place, x, weights=x.view(-1)[8:16].view(4, 2)),
             lambda: ops.route_sum(rows, x.view(-1)[:8].view(i32).view(4, 2), x), lambda: ops.route_sum_grad(x, rows, place, w, rows.clone(), x.view(-1)[:8].view(4, 2)),
             lambda: ops.route_sum_grad(x, rows, place, rows[0].view(4, 2), rows, w.clone()),
             lambda: ops.relbias_grad(scores, scores.view(-1)[:64].view(32, 2), 128),
             lambda: ops.dropout(keys.view(torch.float32).view(16, 2), keys.view(torch.float32).view(16, 2), 0.5, 1, keys=keys),
             lambda: ops.dropout(x, x, 0.5, 1, step=x[1].view(torch.int64)[:1])]
    for i, call in enumerate(calls):
        with pytest.raises(capi.PskvError) as e:
            call()
            pytest.fail("refusal %d" % i)
        assert e.value.code == capi.EINVAL
    torch.cuda.synchronize()
    for t in (x, rows, w, scores):
        assert bool((t == 1).all())
    assert bool((keys == 1).all())
