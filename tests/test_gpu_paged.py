"""Paged-serving operators on the GPU against 64-bit restatements: page plan, RoPE + append of
a packed chunk, attention of chunks over the cache, and a step that runs them together."""

import math

import pytest

torch = pytest.importorskip("torch")

from decodebench_b200 import _native as N  # noqa: E402
from decodebench_b200 import ops  # noqa: E402

pytestmark = pytest.mark.gpu
D = 128
DTYPES = [torch.float16, torch.bfloat16]


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------ page plan
def plan_oracle(ctx, new, free, table, page, n_tokens):
    table = [list(r) for r in table]
    width = len(table[0])
    lens, cu, pos, slots, at = [], [0], [], [], 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        for j in range(-(-c // page), min(-(-(c + n) // page), width)):
            table[b][j] = free[at] if at < len(free) else -1
            at += 1
        for p in range(c, c + n):
            pg = table[b][p // page] if p // page < width else -1
            pos.append(p)
            slots.append(pg * page + p % page if pg >= 0 else -1)
        lens.append(c + n)
        cu.append(cu[-1] + n)
    pad = max(0, n_tokens - len(pos))
    return (table, lens, cu, (pos + [0] * pad)[:n_tokens], (slots + [-1] * pad)[:n_tokens], at)


PLANS = {
    "one": ([0], [1], 16, 4, 10, 0),
    "none-new": ([5, 0], [0, 0], 16, 4, 10, 0),
    "edges": ([15, 16, 17, 0, 31], [1, 1, 16, 33, 0], 16, 6, 20, 0),
    "padded": ([3, 100], [7, 29], 8, 40, 30, 13),
    "page-1": ([2, 0, 7], [3, 5, 1], 1, 12, 20, 0),
    "odd-page": ([2, 48, 7], [60, 5, 100], 24, 12, 20, 2),
    "list-too-short": ([5, 30, 2], [40, 40, 40], 16, 8, 4, 0),
    "empty-list": ([5, 30], [4, 40], 16, 8, 0, 0),
    "table-too-narrow": ([5, 30, 200], [200, 3, 20], 16, 5, 30, 0),
    "negative": ([-3, 4], [5, -2], 16, 4, 10, 1),
    "truncated": ([10, 10], [50, 50], 16, 8, 20, -30),
}


@pytest.mark.parametrize("name", sorted(PLANS))
def test_page_plan_against_lists(name):
    ctx, new, page, width, n_free, pad = PLANS[name]
    g = torch.Generator().manual_seed(3)
    ids = torch.randperm(2000, generator=g).tolist()
    free, ids = ids[:n_free], ids[n_free:]
    table = [[ids[b * width + j] if j < -(-max(c, 0) // page) else -7 for j in range(width)]
             for b, c in enumerate(ctx)]
    n_tokens = sum(max(n, 0) for n in new) + pad
    want = plan_oracle(ctx, new, free, table, page, n_tokens)
    dev_table = i32(table)
    p = ops.page_plan(i32(ctx), i32(new), i32(free), dev_table, page, n_tokens)
    got = (dev_table.tolist(), p.seq_lens.tolist(), p.cu_seqlens.tolist(), p.positions.tolist(),
           p.slots.tolist(), p.used.tolist()[0])
    assert got == want


@pytest.mark.parametrize("batch,page", [(1000, 16), (700, 64), (16384, 32)])
def test_page_plan_large_batch(batch, page):
    g = torch.Generator().manual_seed(batch)
    ctx = torch.randint(0, 300, (batch,), generator=g).tolist()
    new = (torch.randint(0, 6, (batch,), generator=g) * torch.randint(0, 2, (batch,), generator=g)).tolist()
    width, total = 20, sum(new)
    table = torch.arange(batch * width).reshape(batch, width).tolist()
    free = torch.randperm(batch * 2, generator=g).tolist()
    want = plan_oracle(ctx, new, free, table, page, total)
    dev_table = i32(table)
    p = ops.page_plan(i32(ctx), i32(new), i32(free), dev_table, page, total)
    assert (dev_table.tolist(), p.seq_lens.tolist(), p.cu_seqlens.tolist(), p.positions.tolist(),
            p.slots.tolist(), p.used.tolist()[0]) == want


def test_page_plan_slots_past_32_bits():
    table = i32([[2_000_000, 0]])
    p = ops.page_plan(i32([4095]), i32([2]), i32([1_999_999]), table, 4096, 2)
    assert p.slots.tolist() == [2_000_000 * 4096 + 4095, 1_999_999 * 4096]


# ------------------------------------------------------------------------ RoPE + append
def rope64(x, pos, inv):
    """x [n, heads, 128] -> float64, rotate-half pairs."""
    ang = (pos.double()[:, None] * inv.double()[None])[:, None]
    lo, hi = x.double()[..., :64], x.double()[..., 64:]
    return torch.cat([lo * ang.cos() - hi * ang.sin(), hi * ang.cos() + lo * ang.sin()], -1)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n,hq,hkv,page,first", [
    (1, 1, 1, 16, 0), (1, 32, 8, 64, 131071), (5, 7, 1, 24, 1000), (77, 32, 8, 64, 4000),
    (300, 8, 8, 16, 1_000_000), (2500, 5, 3, 1, 17)])
def test_rope_append(dt, n, hq, hkv, page, first):
    g = torch.Generator(device="cuda").manual_seed(n)
    qkv = torch.randn(n, (hq + 2 * hkv) * D, generator=g, device="cuda").to(dt)
    pages = -(-n // page) + 2
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:n].clone()
    if n > 2:
        slots[1] = -1                                  # padded row
        slots[2] = pages * page                        # outside the cache
    pos = torch.arange(first, first + n, dtype=torch.int32, device="cuda")
    inv = ops.rope_inv_freq(D, 500000.0, device="cuda")
    k = torch.full((pages, hkv, page, D), 7.0, dtype=dt, device="cuda")
    v = torch.full_like(k, -3.0)
    q = ops.rope_append(qkv, pos, slots, inv, k, v, hq, hkv)
    x = qkv.view(n, hq + 2 * hkv, D)
    want = rope64(x[:, :hq + hkv], pos, inv)
    # one rounding of the result; sine, cosine (2^-22 each after the 64-bit reduction to 2^-24 *
    # pi) and two products and a sum in 32 bits: 8 * 2^-24 of |lo| + |hi|
    size = x[:, :hq + hkv].double().abs()
    size = size[..., :64] + size[..., 64:]
    tol = torch.finfo(dt).eps / 2 * want.abs() + 8 * 2.0 ** -24 * torch.cat([size, size], -1)
    tol = tol * 1.001 + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    assert ((q.double() - want[:, :hq]).abs() <= tol[:, :hq]).all()
    ek, ev, et = (torch.full((pages * page, hkv, D), c, dtype=torch.float64, device="cuda")
                  for c in (7.0, -3.0, 0.0))
    ok = (slots >= 0) & (slots < pages * page)
    ek[slots[ok]] = want[ok][:, hq:]
    et[slots[ok]] = tol[ok][:, hq:]
    ev[slots[ok]] = x[ok][:, hq + hkv:].double()
    flat = lambda c: c.transpose(1, 2).reshape(pages * page, hkv, D).double()  # noqa: E731
    assert ((flat(k) - ek).abs() <= et).all()
    assert torch.equal(flat(v), ev)


def test_rope_append_matches_the_one_token_projection():
    """The one-token call (projection, RoPE, append) and the chunk call agree on the same token;
    near positions only: the one-token call forms its angle in 32 bits."""
    g = torch.Generator(device="cuda").manual_seed(2)
    hq, hkv, page, d = 8, 2, 16, 256
    dt = torch.float16
    W = (torch.randn((hq + 2 * hkv) * D, d, generator=g, device="cuda") / 16).to(dt)
    x = torch.randn(2, d, generator=g, device="cuda").to(dt)
    inv = ops.rope_inv_freq(D, device="cuda")
    table = i32([[3, 1], [0, 2]])
    pos = i32([20, 3])
    ka, va, kb, vb = (torch.zeros(4, hkv, page, D, dtype=dt, device="cuda") for _ in range(4))
    qa = ops.qkv_rope_append(x, ops.interleave_rope_rows(W, hq, hkv), pos, inv, ka, va, hq, hkv,
                             page_table=table)
    slots = torch.tensor([1 * 16 + 4, 0 * 16 + 3], device="cuda")
    qb = ops.rope_append(ops.gemv(x, W), pos, slots, inv, kb, vb, hq, hkv)
    # values below 8 in size; the chunk call starts from a projection rounded to 16 bits:
    # 2 roundings of 2^-11 on sums of two products
    for a, b in ((qa, qb), (ka, kb), (va, vb)):
        assert ((a.float() - b.float()).abs() <= 3 * 2.0 ** -11 * 8).all()


# ------------------------------------------------------------------------ chunk attention
def attend64(q, keys, vals, length, n, scale):
    """One sequence in 64 bits: q [n, Hq, D], keys / vals [Hkv, length, D] -> (out, weighted |v|,
    largest weighted |q||k| of a row)."""
    hq, hkv = q.shape[1], keys.shape[0]
    kk = keys.double().repeat_interleave(hq // hkv, 0)
    vv = vals.double().repeat_interleave(hq // hkv, 0)
    qq = q.double().transpose(0, 1)
    sc = qq @ kk.transpose(1, 2) * scale
    size = (qq.abs() @ kk.abs().transpose(1, 2) * scale)
    p = torch.arange(length - n, length, device="cuda")
    dead = torch.arange(length, device="cuda")[None] > p[:, None]
    sc = sc.masked_fill(dead, -math.inf)
    top = sc.amax(-1, keepdim=True) if length else torch.zeros_like(sc[..., :1])
    w = (sc - top.clamp(min=-1e300)).exp()
    tot = w.sum(-1, keepdim=True)
    w = torch.where(tot > 0, w / tot.clamp(min=1e-300), 0.0)
    big = size.masked_fill(dead, 0).amax(-1) if length else torch.zeros_like(sc[..., 0])
    return (w @ vv).transpose(0, 1), (w @ vv.abs()).transpose(0, 1), big.transpose(0, 1)


def check_attention(out, q, k, v, ctx, new, table, scale):
    """Weights rounded to the type (half a step), the result rounded once; scores: 128 products in
    32 bits (2^-23 each, accumulators may truncate), their exponential twice that, the fp32 sum
    over `length` weights."""
    u = torch.finfo(q.dtype).eps / 2
    t0 = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        if n == 0:
            continue
        length = c + n
        if table is None:
            kb, vb = k[b, :, :length], v[b, :, :length]
        else:
            page = k.shape[2]
            ids = table[b, :-(-length // page)].long()
            kb, vb = (t[ids].transpose(0, 1).reshape(t.shape[1], -1, D)[:, :length] for t in (k, v))
        want, weight, big = attend64(q[t0:t0 + n], kb, vb, length, n, scale)
        delta = 2.0 ** -23 * (128 * big + 64) + (length / 128 + 128) * 2.0 ** -24
        tol = u * want.abs() + (u + 2 * delta)[..., None] * weight * 1.01 + 2.0 ** -24
        err = (out[t0:t0 + n].double() - want).abs()
        bad = ~(err <= tol)
        assert not bad.any(), (f"sequence {b}: {int(bad.sum())} of {bad.numel()} off, first at "
                               f"{bad.nonzero()[0].tolist()}, worst {float((err / tol).nan_to_num(1e9).max())} of tolerance")
        t0 += n
    return t0


def make(ctx, new, hq, hkv, page, dt, seed=0, pad=0, contiguous=0, garbage=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens = [c + n for c, n in zip(ctx, new)]
    total = sum(new) + pad
    q = torch.randn(total, hq, D, generator=g, device="cuda").to(dt)
    if contiguous:
        shape, table = (len(lens), hkv, contiguous, D), None
    else:
        used = [-(-n // page) for n in lens]
        pages = sum(used) + 3
        shape = (pages, hkv, page, D)
        perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((len(lens), max(max(used), 1) + 1), -5, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(used):
            table[b, :n] = perm[at:at + n]
            at += n
    k = torch.randn(shape, generator=g, device="cuda").to(dt)
    v = torch.randn(shape, generator=g, device="cuda").to(dt)
    if garbage:            # slots that hold no token of the batch: NaN and infinities
        live = torch.zeros(shape[0] * shape[2], dtype=torch.bool, device="cuda")
        for b, n in enumerate(lens):
            tok = torch.arange(n, device="cuda")
            if table is None:
                live[b * shape[2] + tok] = True
            else:
                live[table[b].long()[tok // page] * page + tok % page] = True
        dead = ~live.view(shape[0], 1, shape[2], 1).expand(shape)
        k[dead] = float("nan")
        v[dead] = float("nan")
        v[dead & (torch.rand(shape, generator=g, device="cuda") < 0.5)] = float("inf")
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return q, k, v, i32(cu), i32(lens), table


ATTEND = [
    # ctx, new, hq, hkv, page
    ([0], [1], 1, 1, 16),
    ([0], [2], 4, 1, 64),
    ([127], [1], 8, 1, 16),
    ([128], [1], 4, 4, 64),
    ([0], [128], 1, 1, 128),
    ([0], [129], 2, 2, 64),
    ([0], [257], 2, 1, 8),
    ([1000], [300], 8, 2, 64),
    ([5, 0, 700, 33], [0, 3, 65, 1], 8, 2, 16),
    ([100, 2000], [77, 130], 6, 2, 24),            # 3 heads a group: 42 tokens a tile
    ([100, 300], [90, 1], 35, 5, 48),              # 7 heads a group
    ([40], [9], 128, 1, 32),                       # one token a tile
    ([513], [40], 65, 1, 256),                     # 65 heads a group: half the tile idle
    ([4000], [5], 16, 2, 64),                      # few rows, a long axis: split
    ([30000, 10], [3, 2], 8, 1, 64),
    ([3000] * 9, [1] * 9, 64, 8, 64),              # decoding requests only
    ([0, 512, 1500], [1500, 700, 300], 32, 8, 64),
    ([2000, 900, 0, 64, 127], [1, 513, 1, 200, 1], 16, 4, 32),
]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_chunk_attention(dt, case):
    ctx, new, hq, hkv, page = ATTEND[case]
    q, k, v, cu, lens, table = make(ctx, new, hq, hkv, page, dt, seed=case)
    out = ops.chunk_attention(q, k, v, cu, lens, page_table=table)
    torch.cuda.synchronize()
    assert ops.take_device_error() == 0
    check_attention(out, q, k, v, ctx, new, table, 1 / math.sqrt(D))


@pytest.mark.parametrize("max_len", [1, 7, 130, 1001])
def test_chunk_attention_contiguous_cache(max_len):
    new = [min(max_len, n) for n in (1, 60, 300)]
    ctx = [max_len - new[0], (max_len - new[1]) // 2, max_len - new[2]]
    q, k, v, cu, lens, _ = make(ctx, new, 8, 4, 0, torch.bfloat16, contiguous=max_len)
    out = ops.chunk_attention(q, k, v, cu, lens)
    check_attention(out, q, k, v, ctx, new, None, 1 / math.sqrt(D))


def test_chunk_attention_rows_that_see_nothing_and_rows_behind():
    """seq_len below the number of new tokens: the first rows have negative positions and give
    zeros; rows behind the last sequence stay as they were; lengths past the table are clipped."""
    dt = torch.bfloat16
    q, k, v, cu, lens, table = make([0, 50], [40, 20], 8, 2, 16, dt, pad=11)
    lens = i32([25, 70])
    out = torch.full_like(q, 9.0)
    ops.chunk_attention(q, k, v, cu, lens, page_table=table, out=out)
    assert (out[:15] == 0).all()
    assert (out[60:] == 9.0).all()
    check_attention(out[15:40], q[15:40], k, v, [0], [25], table[:1], 1 / math.sqrt(D))
    check_attention(out[40:60], q[40:60], k, v, [50], [20], table[1:], 1 / math.sqrt(D))
    ops.chunk_attention(q, k, v, cu, i32([0, -4]), page_table=table, out=out)
    assert (out[:60] == 0).all() and (out[60:] == 9.0).all()


def test_chunk_attention_batches_that_are_mostly_empty():
    dt = torch.float16
    q, k, v, _, _, table = make([300, 20, 700], [5, 0, 140], 8, 2, 16, dt)
    clean = ops.chunk_attention(q, k, v, i32([0, 5, 5, 145]), i32([305, 20, 840]), page_table=table)
    batch, at = 20000, (7, 12000, 19998)                   # the three among many without a new token
    new, lens = torch.zeros(batch, dtype=torch.int32), torch.full((batch,), 33, dtype=torch.int32)
    many = torch.full((batch, table.shape[1]), -1, dtype=torch.int32, device="cuda")
    for i, b in enumerate(at):
        new[b], lens[b], many[b] = (5, 0, 140)[i], (305, 20, 840)[i], table[i]
    cu = torch.cat([torch.zeros(1, dtype=torch.int32), new.cumsum(0).int()])
    out = ops.chunk_attention(q, k, v, cu.cuda(), lens.cuda(), page_table=many)
    check_attention(out[:5], q[:5], k, v, [300], [5], table[:1], 1 / math.sqrt(D))
    check_attention(out[5:], q[5:], k, v, [700], [140], table[2:], 1 / math.sqrt(D))
    check_attention(clean[5:], q[5:], k, v, [700], [140], table[2:], 1 / math.sqrt(D))
    out = torch.full_like(q, 9.0)                           # and none at all
    ops.chunk_attention(q, k, v, torch.zeros_like(cu, device="cuda"), lens.cuda(), page_table=many, out=out)
    assert (out == 9.0).all() and ops.take_device_error() == 0


def test_chunk_attention_bad_pages_read_as_zeros():
    dt = torch.float16
    q, k, v, cu, lens, table = make([100], [30], 4, 2, 16, dt)
    bad = table.clone()
    bad[0, 2], bad[0, 5] = -1, 2 ** 31 - 1
    out = ops.chunk_attention(q, k, v, cu, lens, page_table=bad)
    k2 = torch.cat([k, torch.zeros_like(k[:1])])
    v2 = torch.cat([v, torch.zeros_like(v[:1])])
    bad[0, 2] = bad[0, 5] = k.shape[0]
    check_attention(out, q, k2, v2, [100], [30], bad, 1 / math.sqrt(D))


def test_chunk_attention_scale_and_large_scores():
    """Scores of hundreds: the running maximum jumps between blocks."""
    dt = torch.float16
    q, k, v, cu, lens, table = make([700], [100], 4, 1, 16, dt, garbage=False)
    k *= torch.linspace(0.1, 6, k.shape[0], device="cuda").to(dt)[:, None, None, None]
    out = ops.chunk_attention(q, k, v, cu, lens, page_table=table, scale=0.5)
    check_attention(out, q, k, v, [700], [100], table, 0.5)


def test_chunk_attention_nan_stays_in_its_rows():
    dt = torch.bfloat16
    q, k, v, cu, lens, table = make([300, 200], [50, 60], 8, 2, 64, dt)
    clean = ops.chunk_attention(q, k, v, cu, lens, page_table=table)
    q2 = q.clone()
    q2[7, 3] = float("nan")
    k2 = k.clone()
    k2[table[1, 0], 1, 5] = float("nan")          # sequence 1, kv head 1, position 5
    out = ops.chunk_attention(q2, k2, v, cu, lens, page_table=table)
    want_nan = torch.zeros(110, 8, dtype=torch.bool, device="cuda")
    want_nan[7, 3] = True
    want_nan[50:, 4:] = True
    assert torch.equal(out.isnan().all(-1), want_nan)
    assert torch.equal(out[~want_nan], clean[~want_nan])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("ctx,new,hq,hkv", [(0, 40, 8, 2), (300, 200, 4, 4), (5000, 30, 16, 2), (90, 300, 2, 1)])
def test_chunk_attention_later_tokens_that_are_not_finite(dt, ctx, new, hq, hkv):
    """A V (and K) of a later token of the chunk that is not finite reaches only the rows that see it."""
    q, k, v, cu, lens, table = make([ctx], [new], hq, hkv, 16, dt)
    clean = ops.chunk_attention(q, k, v, cu, lens, page_table=table)
    at = ctx + new - 7                                   # position of the seventh token from the end
    page, off = int(table[0, at // 16]), at % 16
    for value in (float("nan"), float("inf"), -float("inf")):
        v2, k2 = v.clone(), k.clone()
        v2[page, 0, off, 5] = value
        out = ops.chunk_attention(q, k, v2, cu, lens, page_table=table)
        group = hq // hkv
        sees = torch.zeros(new, hq, D, dtype=torch.bool, device="cuda")
        sees[new - 7:, :group, 5] = True
        want = torch.full_like(out, value)
        assert torch.equal(out[sees].isnan(), want[sees].isnan())
        if value == value:
            assert (out[sees] == value).all()
        assert out[~sees].isfinite().all()
        # the rows done one by one agree with the clean ones as two results within tolerance of one
        check_attention(torch.where(sees, clean, out), q, k, v, [ctx], [new], table, 1 / math.sqrt(D))
        k2[page, 0, off] = value
        out = ops.chunk_attention(q, k2, v2, cu, lens, page_table=table)
        assert out[:new - 7].isfinite().all()
        check_attention(torch.cat([out[:new - 7], clean[new - 7:]]), q, k, v, [ctx], [new], table,
                        1 / math.sqrt(D))


def test_chunk_attention_all_values_not_finite_in_a_long_cache():
    """Every V is NaN, or one of a long sequence's last ones: no wait runs out, all rows are right."""
    dt = torch.bfloat16
    q, k, v, cu, lens, table = make([40000], [700], 8, 1, 64, dt)
    v2 = torch.full_like(v, float("nan"))
    assert ops.chunk_attention(q, k, v2, cu, lens, page_table=table).isnan().all()
    v2 = v.clone()
    page = int(table[0, 40650 // 64])
    v2[page, 0, 40650 % 64] = float("inf")
    out = ops.chunk_attention(q, k, v2, cu, lens, page_table=table)
    clean = ops.chunk_attention(q, k, v, cu, lens, page_table=table)
    assert torch.equal(out[:650], clean[:650])
    assert (out[650:] == float("inf")).all()
    assert ops.take_device_error() == 0


def test_chunk_attention_decoding_equals_flashdecode():
    dt = torch.bfloat16
    ctx = [1, 64, 1000, 5000]
    q, k, v, cu, lens, table = make(ctx, [1] * 4, 32, 8, 64, dt, garbage=False)
    a = ops.chunk_attention(q, k, v, cu, lens, page_table=table)
    table = table.clamp(min=0)
    b = ops.flashdecode(q, k, v, seq_lens=lens, page_table=table)
    # both are within the one-kernel tolerance of the 64-bit result
    check_attention(a, q, k, v, ctx, [1] * 4, table, 1 / math.sqrt(D))
    assert (a.float() - b.float()).abs().max() <= 2 ** -7 * b.float().abs().max()


def test_chunk_attention_repeats_exactly_and_in_a_graph():
    dt = torch.float16
    q, k, v, cu, lens, table = make([9000, 100], [70, 300], 16, 2, 64, dt)
    first = ops.chunk_attention(q, k, v, cu, lens, page_table=table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [ops.chunk_attention(q, k, v, cu, lens, page_table=table) for _ in range(4)]
    torch.cuda.current_stream().wait_stream(side)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.chunk_attention(q, k, v, cu, lens, page_table=table, out=out)
    for _ in range(3):
        out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
    assert all(torch.equal(t, first) for t in again)
    lens.copy_(i32([200, 350]))                     # other lengths in the same graph
    graph.replay()
    check_attention(out, q, k, v, [130, 50], [70, 300], table, 1 / math.sqrt(D))


def test_two_streams_at_once():
    dt = torch.bfloat16
    a = make([5000], [64], 16, 2, 64, dt, seed=1)
    b = make([3000, 70], [40, 500], 16, 2, 64, dt, seed=2)
    call = lambda t: ops.chunk_attention(*t[:5], page_table=t[5])  # noqa: E731
    want = [call(a), call(b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(5):
        for s, t in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(call(t))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 2]) for i, g in enumerate(got))


def test_other_current_stream_and_workspace():
    dt = torch.bfloat16
    q, k, v, cu, lens, table = make([900], [33], 8, 2, 64, dt)
    nb = N.load().dbk_chunk_attention_workspace_bytes(33, 8, 2)
    ws = torch.full((nb,), 255, dtype=torch.uint8, device="cuda")
    out = ops.chunk_attention(q, k, v, cu, lens, page_table=table, workspace=ws)
    check_attention(out, q, k, v, [900], [33], table, 1 / math.sqrt(D))
    with pytest.raises(ValueError, match="workspace"):
        ops.chunk_attention(q, k, v, cu, lens, page_table=table, workspace=ws[:100])


# ------------------------------------------------------------------------ together
def test_serving_steps_together():
    """Three scheduler steps of three requests: plan, projection, append, attention; the cache is
    fed only through the operators, and every step's attention is checked in 64 bits."""
    dt = torch.bfloat16
    hq, hkv, page, d = 8, 2, 16, 256
    g = torch.Generator(device="cuda").manual_seed(5)
    W = (torch.randn((hq + 2 * hkv) * D, d, generator=g, device="cuda") / 16).to(dt)
    inv = ops.rope_inv_freq(D, device="cuda")
    pages = 40
    k = torch.full((pages, hkv, page, D), float("nan"), dtype=dt, device="cuda")
    v = torch.full_like(k, float("nan"))
    free = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((3, 12), -1, dtype=torch.int32, device="cuda")
    ctx = i32([0, 0, 0])
    keys = [[] for _ in range(3)]
    vals = [[] for _ in range(3)]
    for new in ([33, 0, 100], [1, 64, 1], [1, 1, 17]):
        n = sum(new)
        x = torch.randn(n + 5, d, generator=g, device="cuda").to(dt)      # five padded rows
        p = ops.page_plan(ctx, i32(new), free, table, page, n + 5)
        qkv = torch.cat([ops.gemv(c, W) for c in x.split(64)])
        q = ops.rope_append(qkv, p.positions, p.slots, inv, k, v, hq, hkv)
        out = ops.chunk_attention(q, k, v, p.cu_seqlens, p.seq_lens, page_table=table)
        free = free[int(p.used):].contiguous()
        check_attention(out, q, k, v, ctx.tolist(), new, table, 1 / math.sqrt(D))
        t0 = 0
        for b, nb in enumerate(new):
            # the cache holds this request's projections of all its steps, k rotated
            qkv_b = qkv[t0:t0 + nb].view(nb, hq + 2 * hkv, D)
            keys[b].append(rope64(qkv_b[:, hq:hq + hkv], p.positions[t0:t0 + nb], inv))
            vals[b].append(qkv_b[:, hq + hkv:])
            kb, vb = torch.cat(keys[b]), torch.cat(vals[b])
            length = kb.shape[0]
            assert length == int(p.seq_lens[b])
            ids = table[b, :-(-length // page)].long()
            ck, cv = (c[ids].transpose(1, 2).reshape(-1, hkv, D)[:length] for c in (k, v))
            assert torch.equal(cv, vb)
            assert ((ck.double() - kb).abs() <= 2.0 ** -8 * kb.abs() + 8 * 2.0 ** -24 * 16).all()
            t0 += nb
        ctx = p.seq_lens
    assert ops.take_device_error() == 0
