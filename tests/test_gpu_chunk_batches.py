"""Chunk attention over batches of which most requests bring no token."""

import math

import pytest

torch = pytest.importorskip("torch")

from decodebench_b200 import ops  # noqa: E402
from tests.test_gpu_paged import D, check_attention, i32, make  # noqa: E402

pytestmark = pytest.mark.gpu


def spread(batch, at, new, lens, table):
    """The requests of a small batch put at places `at` of a large one."""
    n, full = torch.zeros(batch, dtype=torch.int32), torch.full((batch,), 33, dtype=torch.int32)
    many = torch.full((batch, table.shape[1]), -1, dtype=torch.int32, device="cuda")
    for i, b in enumerate(at):
        n[b], full[b], many[b] = new[i], lens[i], table[i]
    cu = torch.cat([torch.zeros(1, dtype=torch.int32), n.cumsum(0).int()])
    return cu.cuda(), full.cuda(), many


@pytest.mark.parametrize("at", [(0, 1, 2), (0, 31, 32), (33, 65, 97), (0, 40000, 65535), (65533, 65534, 65535), (5, 6, 65000)])
@pytest.mark.parametrize("ctx,new", [([300, 20, 700], [5, 1, 140]), ([0, 9000, 3], [1, 2, 1]), ([2000, 2500, 100], [300, 1, 900])])
def test_largest_batch_mostly_empty(at, ctx, new):
    dt, batch = torch.float16, 65536
    q, k, v, _, _, table = make(ctx, new, 8, 2, 16, dt, seed=at[1])
    lens = [c + n for c, n in zip(ctx, new)]
    cu, full, many = spread(batch, at, new, lens, table)
    out = torch.full_like(q, 9.0)
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    ops.chunk_attention(q, k, v, cu, full, page_table=many, out=out)
    a.record()
    ops.chunk_attention(q, k, v, cu, full, page_table=many, out=out)
    b.record()
    torch.cuda.synchronize()
    check_attention(out, q, k, v, ctx, new, table, 1 / math.sqrt(D))
    assert ops.take_device_error() == 0
    # walked one by one, 65,536 requests take about 7 ms, while the other warps wait
    assert a.elapsed_time(b) < 4


def test_runs_of_empty_requests_between_many_live_ones():
    """Cuts of the line fall next to empty requests of every run length."""
    dt = torch.bfloat16
    g = torch.Generator().manual_seed(4)
    live = 60
    ctx = torch.randint(0, 900, (live,), generator=g).tolist()
    new = torch.randint(1, 90, (live,), generator=g).tolist()
    q, k, v, cu0, lens0, table = make(ctx, new, 8, 2, 16, dt)
    want = ops.chunk_attention(q, k, v, cu0, lens0, page_table=table)
    at, b = [], 0
    for i in range(live):
        b += int(torch.randint(1, 80, (1,), generator=g)) if i % 3 else 1
        at.append(b)
    cu, full, many = spread(b + 70, at, new, lens0.tolist(), table)
    out = ops.chunk_attention(q, k, v, cu, full, page_table=many)
    assert torch.equal(out, want)                       # empty requests cost nothing on the line: the same cuts
    check_attention(out, q, k, v, ctx, new, table, 1 / math.sqrt(D))
