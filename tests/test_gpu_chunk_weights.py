"""Softmax weights of chunk attention: their range in fp16, and what is left of them for the
tensor cores."""

import math

import pytest

torch = pytest.importorskip("torch")

from decodebench_b200 import ops  # noqa: E402
from tests.test_gpu_paged import ATTEND, D, DTYPES, attend64, check_attention, i32, make  # noqa: E402

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


# ------------------------------------------------------------------------ two parts
PART = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -22}     # what two parts leave of a weight


def check_two_parts(out, q, k, v, ctx, new, table, scale):
    """As check_attention, without a rounding of the weights: the result's own half step; a weight
    in two parts (PART, and 2^-36 in fp16); scores of 128 products and their exponential, the fp32
    sums."""
    u = torch.finfo(q.dtype).eps / 2
    t0 = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        if n == 0:
            continue
        length = c + n
        ids = table[b, :-(-length // k.shape[2])].long()
        kb, vb = (t[ids].transpose(0, 1).reshape(t.shape[1], -1, D)[:, :length] for t in (k, v))
        want, weight, big = attend64(q[t0:t0 + n], kb, vb, length, n, scale)
        delta = 2.0 ** -23 * (128 * big + 64) + (length / 128 + 128) * 2.0 ** -24
        tol = u * want.abs() + (PART[q.dtype] + 2 * delta)[..., None] * weight * 1.01 + 2.0 ** -24
        err = (out[t0:t0 + n].double() - want).abs()
        bad = ~(err <= tol)
        assert not bad.any(), (f"sequence {b}: {int(bad.sum())} of {bad.numel()} off, worst "
                               f"{float((err / tol).nan_to_num(1e9).max())} of tolerance")
        t0 += n


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_two_parts(dt, case):
    ctx, new, hq, hkv, page = ATTEND[case]
    q, k, v, cu, lens, table = make(ctx, new, hq, hkv, page, dt, seed=case)
    out = ops.chunk_attention(q, k, v, cu, lens, page_table=table)
    check_two_parts(out, q, k, v, ctx, new, table, 1 / math.sqrt(D))
    assert ops.take_device_error() == 0


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("parts", [1, 2])
def test_growing_scores(dt, parts):
    """The running maximum jumps between blocks by more than weights can: O is rescaled, and the
    first half of a block's weights formed again."""
    q, k, v, cu, lens, table = make([700, 3], [100, 1], 4, 1, 16, dt, garbage=False)
    k *= torch.linspace(0.1, 6, k.shape[0], device="cuda").to(dt)[:, None, None, None]
    out = ops.chunk_attention(q, k, v, cu, lens, page_table=table, scale=0.5, weight_parts=parts)
    (check_two_parts if parts == 2 else check_attention)(out, q, k, v, [700, 3], [100, 1], table, 0.5)


@pytest.mark.parametrize("dt", DTYPES)
def test_one_part(dt):
    q, k, v, cu, lens, table = make([2000, 900, 0, 64], [1, 513, 1, 200], 16, 4, 32, dt)
    out = ops.chunk_attention(q, k, v, cu, lens, page_table=table, weight_parts=1)
    check_attention(out, q, k, v, [2000, 900, 0, 64], [1, 513, 1, 200], table, 1 / math.sqrt(D))


@pytest.mark.parametrize("dt", DTYPES)
def test_decoding_is_as_exact_as_flashdecode(dt):
    """The same requests through both calls: root-mean-square error against 64 bits. Each rounds its
    result once; what else chunk attention rounds is 2^-16 of a weight and below, which adds
    far less than the 1 % allowed to it."""
    ctx, hq, hkv = [500, 1000, 2000, 4000, 100, 3000] * 4, 32, 8
    q, k, v, cu, lens, table = make(ctx, [1] * 24, hq, hkv, 64, dt, garbage=False)
    table = table.clamp(min=0)
    a = ops.chunk_attention(q, k, v, cu, lens, page_table=table)
    b = ops.flashdecode(q, k, v, seq_lens=lens, page_table=table)
    err = []
    for out in (a, b):
        sq = 0.0
        for i, c in enumerate(ctx):
            ids = table[i, :-(-(c + 1) // 64)].long()
            kb, vb = (t[ids].transpose(0, 1).reshape(hkv, -1, D)[:, :c + 1] for t in (k, v))
            want = attend64(q[i:i + 1], kb, vb, c + 1, 1, 1 / math.sqrt(D))[0]
            sq += float((out[i:i + 1].double() - want).square().sum())
        err.append(math.sqrt(sq))
    assert err[0] <= 1.01 * err[1], err


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("parts", [1, 2])
def test_an_infinite_value_that_all_rows_see(dt, parts):
    """The key that takes most of the weight, exactly 1 of the maximum for some rows, has an infinite V."""
    q, k, v, cu, lens, table = make([700], [60], 8, 2, 16, dt, garbage=False)
    page, off = int(table[0, 0]), 5
    for value in (float("inf"), -float("inf")):
        v2, k2, q2 = v.clone(), k.clone(), q.clone()
        q2[..., 0] = 4
        k2[page, 0, off, 0] = 8                      # about 2.8 nats above the others
        v2[page, 0, off, 9] = value
        out = ops.chunk_attention(q2, k2, v2, cu, lens, page_table=table, weight_parts=parts)
        assert (out[:, :4, 9] == value).all()
        out[:, :4, 9] = 0
        assert out.isfinite().all()


def test_refuses_other_parts():
    q, k, v, cu, lens, table = make([20], [3], 2, 1, 16, torch.bfloat16)
    for bad in (0, 3, None, "two"):
        with pytest.raises(ValueError, match="weight_parts"):
            ops.chunk_attention(q, k, v, cu, lens, page_table=table, weight_parts=bad)


def test_refuses_a_workspace_whose_bytes_are_not_there():
    """An expanded tensor has as many elements as asked for and one byte of memory."""
    q, k, v, cu, lens, table = make([20], [3], 2, 1, 16, torch.bfloat16)
    for bad in (torch.zeros(1, dtype=torch.uint8, device="cuda").expand(1 << 26),
                torch.zeros(1 << 26, dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(ValueError, match="workspace"):
            ops.chunk_attention(q, k, v, cu, lens, page_table=table, workspace=bad)
