"""Softmax weights of chunk attention: their range in fp16, and what is left of them for the
tensor cores."""

import math

import pytest

torch = pytest.importorskip("torch")

from decodebench_b200 import ops  # noqa: E402
from tests.test_gpu_paged import D, check_attention, i32  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nats", [14, 16, 17])
@pytest.mark.parametrize("length,new", [(131072, 1), (131072, 40), (30000, 200)])
def test_fp16_body_far_below_a_sink(nats, length, new):
    """A first key that takes nearly all weight and has v = 0: the result is what the others give,
    each of whose weights is far below 2^-14 of the largest (2^-20 to 2^-24.5: fp16 has 11 bits for them
    once they are scaled, so half a step of the weighted |v|, as for any weights)."""
    hq, hkv, page = 8, 1, 64
    g = torch.Generator(device="cuda").manual_seed(nats)
    q = torch.zeros(new, hq, D, dtype=torch.float16, device="cuda")
    q[..., 0] = 8
    shape = (length // page + 1, hkv, page, D)
    k = torch.zeros(shape, dtype=torch.float16, device="cuda")
    v = (torch.randn(shape, generator=g, device="cuda") + 1).to(torch.float16)
    k[0, 0, 0, 0] = nats * math.sqrt(D) / 8
    v[0, 0, 0] = 0
    table = torch.arange(shape[0], dtype=torch.int32, device="cuda")[None]
    out = ops.chunk_attention(q, k, v, i32([0, new]), i32([length]), page_table=table)
    check_attention(out, q, k, v, [length - new], [new], table, 1 / math.sqrt(D))
