"""The position bias where a sequence's own position is any 64-bit number: positions are whole numbers, and do not wrap."""
import pytest

from conftest import announce
from test_gpu_ops import F, TYPES, near, normal, ops, plain_bucket, rounded, seeded  # noqa: F401

pytestmark = pytest.mark.gpu

FAR = [(1 << 63) - 1, -(1 << 63), (1 << 63) - 40, -(1 << 63) + 40, (1 << 62) + 5, -(1 << 62) - 5, 1 << 60, 0, 3]


# single queries, tiles and planes of both directions
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("Q,K", [(1, 700), (9, 130), (65, 20), (3, 600)])
@pytest.mark.parametrize("q_first,k_first", [(0, 0), (1 << 60, -(1 << 60)), (-(1 << 60), 1 << 60)])
@pytest.mark.parametrize("two_sided", [True, False])
def test_far_positions_of_their_own(ops, dev, type, Q, K, q_first, k_first, two_sided):
    import torch
    announce("relbias, relbias_grad, far positions", type, Q, K, q_first, k_first, two_sided)
    g = seeded(Q + K)
    B, H, buckets, far = len(FAR), 3, 32, 128
    table, at = normal(g, buckets, H), torch.tensor(FAR, device=dev)
    row = [[[plain_bucket(max(-far - 1, min(far + 1, k_first + j - q_first - own - i)), buckets, far, two_sided) for j in range(K)]
            for i in range(Q)] for own in FAR]
    bucket = torch.tensor(row, device=dev)
    bias = table.double()[bucket].permute(0, 3, 1, 2)
    out = torch.empty(B, H, Q, K, dtype=getattr(torch, type), device=dev)
    more = dict(two_sided=two_sided, q_first=q_first, k_first=k_first, q_at=at)
    ops.relbias(table, out, far, **more)
    near(out, bias, rounded(bias, 0.0, type), "bias")
    grad, grad_table = normal(g, B, H, Q, K, type=type), torch.empty(buckets, H, device=dev)
    ops.relbias_grad(grad, grad_table, far, **more)
    want, size = (torch.zeros(buckets, H, dtype=torch.float64, device=dev) for _ in range(2))
    for h in range(H):
        flat = grad[:, h].double().reshape(-1)
        want[:, h].index_add_(0, bucket.reshape(-1), flat)
        size[:, h].index_add_(0, bucket.reshape(-1), flat.abs())
    # no chain of additions is longer than 1,024 and the batch
    near(grad_table, want, (1024 + B) * F * size, "gradient")
