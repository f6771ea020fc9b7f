"""What is measured of the serving step's operators: cases, inputs, the plain forms.

Four operators carry a scheduler step of paged serving from the requests' lengths to the
next tokens, and each case below is one pass through one of them:

* ``plan``    page tables, slot map and positions from the requests' lengths;
* ``append``  rotary positions and the cache append for a packed chunk of new tokens;
* ``attend``  attention of the new tokens over the paged cache, causal from the end;
* ``sample``  temperature, top-k, top-p and min-p sampling from given random numbers.

``own`` chooses between the plain forms (elementary torch operations) and the framework's
kernels (:mod:`decodebench_b200.ops`).
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

HEAD_DIM = 128
_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------- cases
def listed():
    return [
        # One decode step of the paged batch of 8 long sequences: every request adds a token,
        # now and then one of them needs a page. Latency is all there is.
        dict(name="plan-decode-8", op="plan", batch=8, new="ones", tokens=8, ctx_hi=32768,
             page=64, shape_seed=1),
        # A scheduler step of 512 requests with a budget of 16,384 new tokens and small pages.
        dict(name="plan-mixed-512", op="plan", batch=512, new="mixed", tokens=16384,
             ctx_hi=32768, page=16, shape_seed=2),
        # The chunk of one short prompt.
        dict(name="append-77", op="append", tokens=77, hq=32, hkv=8, page=64, dtype="fp16",
             pos_hi=4096),
        # A full token budget with wide heads, far positions.
        dict(name="append-8192", op="append", tokens=8192, hq=64, hkv=8, page=64, dtype="bf16",
             pos_hi=131072),
        # The next 512 tokens of one prompt, 4,096 tokens in.
        dict(name="attend-512-at-4096", op="attend", batch=1, new="even", tokens=512, ctx_hi=4096,
             ctx="top", hq=32, hkv=8, page=64, dtype="bf16", shape_seed=3),
        # Decoding requests beside two prompts' chunks, long contexts, odd lengths.
        dict(name="attend-mixed-40", op="attend", batch=40, new="mixed", tokens=1100,
             ctx_hi=16384, ctx="spread", hq=64, hkv=8, page=64, dtype="bf16", shape_seed=4),
        # Many short ragged prompts, no heads shared, small pages.
        dict(name="attend-ragged-24", op="attend", batch=24, new="spread", tokens=9001,
             ctx_hi=700, ctx="spread", hq=32, hkv=32, page=16, dtype="fp16", shape_seed=5),
        # One whole long prompt.
        dict(name="attend-prompt-16384", op="attend", batch=1, new="even", tokens=16384, ctx_hi=0,
             ctx="top", hq=32, hkv=8, page=64, dtype="bf16", shape_seed=6),
        # A short chunk far into a long document: few rows, a long axis.
        dict(name="attend-24-at-131072", op="attend", batch=1, new="even", tokens=24,
             ctx_hi=131072, ctx="top", hq=64, hkv=8, page=64, dtype="fp16", shape_seed=7),
        # One request's next token from a large vocabulary.
        dict(name="sample-1", op="sample", batch=1, vocab=128000, dtype="fp32", filt="kp",
             shape_seed=8),
        # A batch whose requests all ask for something else, of an odd vocabulary.
        dict(name="sample-mixed-61", op="sample", batch=61, vocab=32003, dtype="bf16",
             filt="mixed", shape_seed=9),
        # A large batch, nucleus sampling over the whole vocabulary.
        dict(name="sample-256", op="sample", batch=256, vocab=128000, dtype="fp32", filt="p",
             shape_seed=10),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "sample", "sample"])
    seed = rng.randrange(1 << 20)
    if op == "plan":
        batch = _log(rng, 1, 512)
        new = rng.choice(["ones", "mixed", "spread"])
        tokens = batch if new == "ones" else _log(rng, batch + 1, 16384)
        return dict(op=op, batch=batch, new=new, tokens=tokens, ctx_hi=_log(rng, 16, 32768),
                    page=rng.choice([16, 32, 64, 128, 24]), shape_seed=seed)
    if op == "append":
        hkv = rng.choice([1, 2, 4, 8])
        return dict(op=op, tokens=_log(rng, 1, 8192), hq=hkv * rng.choice([1, 2, 4, 7, 8]),
                    hkv=hkv, page=rng.choice([16, 32, 64, 128, 24]),
                    dtype=rng.choice(["fp16", "bf16"]), pos_hi=_log(rng, 64, 131072))
    if op == "attend":
        hkv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 5, 8])
        batch = _log(rng, 1, 48)
        new = rng.choice(["ones", "even", "spread", "mixed"])
        tokens = batch if new == "ones" else _log(rng, batch + 1, 8192)
        budget = 16384 * 8192 * 32                 # (new token, cached token, head) triples
        ctx_hi = min(_log(rng, 1, 65536), max(1, budget // (tokens * hkv * group)),
                     max(64, 400000 // batch))
        return dict(op=op, batch=batch, new=new, tokens=tokens, ctx_hi=ctx_hi,
                    ctx=rng.choice(["top", "spread"]), hq=hkv * group, hkv=hkv,
                    page=rng.choice([16, 32, 64, 128, 24]), dtype=rng.choice(["fp16", "bf16"]),
                    shape_seed=seed)
    return dict(op=op, batch=_log(rng, 1, 256), vocab=_log(rng, 1000, 128000),
                dtype=rng.choice(["fp32", "fp16", "bf16"]),
                filt=rng.choice(["none", "k", "p", "kp", "min", "mixed"]), shape_seed=seed)


def _lengths(case):
    """(cached lengths, new lengths) of the case's requests, on the host."""
    rng = random.Random(case["shape_seed"])
    batch, tokens, hi = case["batch"], case["tokens"], case["ctx_hi"]
    kind = case["new"]
    if kind == "ones":
        new = [1] * batch
    elif kind == "even":
        new = [tokens * (i + 1) // batch - tokens * i // batch for i in range(batch)]
    elif kind == "spread":
        cuts = sorted(rng.randint(0, tokens) for _ in range(batch - 1))
        new = [b - a for a, b in zip([0] + cuts, cuts + [tokens])]
    else:                       # "mixed": most requests decode, a few bring the rest in chunks
        chunks = max(1, batch // 20)
        new = [1] * batch
        rest = max(0, tokens - batch)
        for i in range(chunks):
            new[rng.randrange(batch)] += rest * (i + 1) // chunks - rest * i // chunks
    if case.get("ctx", "spread") == "top":
        ctx = [hi] * batch
    else:
        ctx = [rng.randint(min(hi, hi // 16), hi) for _ in range(batch)]
    return ctx, new


def _pages(n, page):
    return -(-n // page)


# ------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    return {"plan": _prepare_plan, "append": _prepare_append, "attend": _prepare_attend,
            "sample": _prepare_sample}[case["op"]](case, gen)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_plan(case, gen):
    ctx, new = _lengths(case)
    page = case["page"]
    # the seed moves each request's length a little: another step of the same batch
    move = torch.randint(0, page, (len(ctx),), generator=gen, device="cuda").tolist()
    ctx = [c + m for c, m in zip(ctx, move)]
    have = [_pages(c, page) for c in ctx]
    most = [_pages(c + page + n, page) for c, n in zip(_lengths(case)[0], new)]
    width, spare = max(most) + 8, sum(_pages(n, page) + 1 for n in new) + 64
    ids = torch.randperm(sum(most) + spare, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(ctx), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, h in enumerate(have):
        table[b, :h] = ids[at:at + h]
        at += h
    return dict(op="plan", ctx=_i32(ctx), new=_i32(new), free=ids[at:at + spare].clone(), table=table,
                page=page, tokens=case["tokens"])


def _prepare_append(case, gen):
    n, hq, hkv, page = case["tokens"], case["hq"], case["hkv"], case["page"]
    dt = _TYPES[case["dtype"]]
    qkv = torch.randn(n, (hq + 2 * hkv) * HEAD_DIM, generator=gen, device="cuda").to(dt)
    pages = _pages(n, page) + 3
    # consecutive positions of one chunk; its pages lie anywhere in the pool
    first = int(torch.randint(0, case["pos_hi"], (1,), generator=gen, device="cuda"))
    pos = torch.arange(n, device="cuda") + first
    perm = torch.randperm(pages, generator=gen, device="cuda")
    rel = torch.arange(n, device="cuda") + first % page
    slots = perm[torch.div(rel, page, rounding_mode="floor")] * page + rel % page
    inv = 1.0 / (500000.0 ** (torch.arange(0, HEAD_DIM, 2, device="cuda").float() / HEAD_DIM))
    shape = (pages, hkv, page, HEAD_DIM)
    return dict(op="append", qkv=qkv, pos=pos.to(torch.int32), slots=slots, inv=inv,
                k=torch.zeros(shape, dtype=dt, device="cuda"),
                v=torch.zeros(shape, dtype=dt, device="cuda"), hq=hq, hkv=hkv)


def _prepare_attend(case, gen):
    ctx, new = _lengths(case)
    hq, hkv, page = case["hq"], case["hkv"], case["page"]
    dt = _TYPES[case["dtype"]]
    lens = [c + n for c, n in zip(ctx, new)]
    used = [_pages(n, page) for n in lens]
    pages = sum(used) + 5
    ids = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(max(used), 1), dtype=torch.int32, device="cuda")
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = ids[at:at + u]
        at += u
    shape = (pages, hkv, page, HEAD_DIM)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return dict(op="attend",
                q=torch.randn(case["tokens"], hq, HEAD_DIM, generator=gen, device="cuda").to(dt),
                k=torch.randn(shape, generator=gen, device="cuda", dtype=dt),
                v=torch.randn(shape, generator=gen, device="cuda", dtype=dt),
                table=table, cu=_i32(cu), lens=_i32(lens), host_cu=cu, host_lens=lens)


def _prepare_sample(case, gen):
    batch, vocab, filt = case["batch"], case["vocab"], case["filt"]
    rng = random.Random(case["shape_seed"])
    # a peaked head over a broad body, as a language model's logits are
    logits = torch.randn(batch, vocab, generator=gen, device="cuda") * 2.5
    hot = torch.randint(0, vocab, (batch, 24), generator=gen, device="cuda")
    logits.scatter_add_(1, hot, torch.rand(batch, 24, generator=gen, device="cuda") * 9)
    f = dict(temperature=[], top_k=[], top_p=[], min_p=[])
    for i in range(batch):
        kind = filt if filt != "mixed" else rng.choice(["none", "k", "p", "kp", "min", "greedy"])
        f["temperature"].append(0.0 if kind == "greedy" else rng.choice([0.6, 0.8, 1.0, 1.3]))
        f["top_k"].append(rng.choice([1, 20, 50, 1000]) if kind in ("k", "kp") else 0)
        f["top_p"].append(rng.choice([0.5, 0.9, 0.95, 0.99]) if kind in ("p", "kp") else 1.0)
        f["min_p"].append(rng.choice([0.02, 0.1]) if kind == "min" else 0.0)
    filters = dict(
        temperature=torch.tensor(f["temperature"], dtype=torch.float32, device="cuda"),
        top_k=_i32(f["top_k"]) if any(f["top_k"]) else None,
        top_p=torch.tensor(f["top_p"], device="cuda") if min(f["top_p"]) < 1 else None,
        min_p=torch.tensor(f["min_p"], device="cuda") if any(f["min_p"]) else None)
    return dict(op="sample", logits=logits.to(_TYPES[case["dtype"]]),
                u=torch.rand(batch, generator=gen, device="cuda"), filters=filters)


# ------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend,
            "sample": _plain_sample}[state["op"]](state)


def _run_own(s):
    from decodebench_b200 import ops

    if s["op"] == "plan":
        p = ops.page_plan(s["ctx"], s["new"], s["free"], s["table"], s["page"], s["tokens"])
        return [s["table"], p.seq_lens, p.cu_seqlens, p.positions, p.slots, p.used]
    if s["op"] == "append":
        q = ops.rope_append(s["qkv"], s["pos"], s["slots"], s["inv"], s["k"], s["v"], s["hq"],
                            s["hkv"])
        return [q, s["k"], s["v"]]
    if s["op"] == "attend":
        return [ops.chunk_attention(s["q"], s["k"], s["v"], s["cu"], s["lens"],
                                    page_table=s["table"])]
    return [ops.sample(s["logits"], s["u"], **s["filters"])]


def _plain_plan(s):
    page, n = s["page"], s["tokens"]
    table, free = s["table"], s["free"]
    ctx, new = s["ctx"].long(), s["new"].long()
    batch, width = table.shape
    ends = torch.cumsum(new, 0)
    cu = torch.cat([torch.zeros_like(ends[:1]), ends])
    have = torch.div(ctx + page - 1, page, rounding_mode="floor")
    need = torch.div(ctx + new + page - 1, page, rounding_mode="floor").clamp(max=width)
    count = (need - have).clamp(min=0)
    first = torch.cumsum(count, 0) - count
    col = torch.arange(width, device=table.device)[None]
    src = first[:, None] + col - have[:, None]
    fresh = (col >= have[:, None]) & (col < need[:, None])
    given = torch.where(src < free.numel(), free[src.clamp(0, free.numel() - 1)].long(), -1)
    table.copy_(torch.where(fresh, given, table.long()))
    tok = torch.arange(n, device=table.device)
    seq = torch.searchsorted(ends, tok, right=True)
    live = seq < batch
    seq = seq.clamp(max=batch - 1)
    pos = torch.where(live, ctx[seq] + tok - cu[seq], 0)
    logical = torch.div(pos, page, rounding_mode="floor")
    phys = table[seq, logical.clamp(max=width - 1)].long()
    ok = live & (logical < width) & (phys >= 0)
    slots = torch.where(ok, phys * page + pos % page, -1)
    used = count.sum(0, keepdim=True)
    return [table, (ctx + new).int(), cu.int(), pos.int(), slots, used.int()]


def _plain_append(s):
    hq, hkv = s["hq"], s["hkv"]
    k_cache, v_cache = s["k"], s["v"]
    n, page = s["qkv"].shape[0], k_cache.shape[2]
    x = s["qkv"].float().view(n, hq + 2 * hkv, HEAD_DIM)
    ang = s["pos"].double()[:, None] * s["inv"].double()[None]
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
    lo, hi = x[:, :hq + hkv, :HEAD_DIM // 2], x[:, :hq + hkv, HEAD_DIM // 2:]
    rot = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).to(s["qkv"].dtype)
    where = torch.div(s["slots"], page, rounding_mode="floor")
    k_cache[where, :, s["slots"] % page] = rot[:, hq:]
    v_cache[where, :, s["slots"] % page] = x[:, hq + hkv:].to(v_cache.dtype)
    return [rot[:, :hq].contiguous(), k_cache, v_cache]


def _plain_attend(s):
    q, k, v, table = s["q"], s["k"], s["v"], s["table"]
    hq, hkv, page = q.shape[1], k.shape[1], k.shape[2]
    group, scale = hq // hkv, 1.0 / math.sqrt(HEAD_DIM)
    out = torch.zeros_like(q)
    for b, length in enumerate(s["host_lens"]):
        t0, t1 = s["host_cu"][b], s["host_cu"][b + 1]
        n = t1 - t0
        if n == 0:
            continue
        rows = table[b, :_pages(length, page)].long()
        step = max(1, (1 << 28) // max(1, group * length))         # query tokens at a time
        cols = torch.arange(length, device=q.device)
        for h in range(hkv):
            kb = k[rows, h].reshape(-1, HEAD_DIM)[:length].float()
            vb = v[rows, h].reshape(-1, HEAD_DIM)[:length].float()
            for a in range(0, n, step):
                e = min(n, a + step)
                qb = q[t0 + a:t0 + e, h * group:(h + 1) * group].float()
                sc = torch.matmul(qb, kb.t()) * scale                # [tokens, group, length]
                last = torch.arange(a, e, device=q.device) + (length - n)
                sc.masked_fill_((cols[None] > last[:, None])[:, None], -math.inf)
                p = (sc - sc.amax(-1, keepdim=True)).exp_()
                o = torch.matmul(p, vb) / p.sum(-1, keepdim=True)
                out[t0 + a:t0 + e, h * group:(h + 1) * group] = o.to(q.dtype)
    return [out]


def _plain_sample(s):
    f = s["filters"]
    x = s["logits"].double()
    batch, vocab = x.shape
    vals, order = torch.sort(x, dim=1, descending=True, stable=True)
    top = vals[:, :1]
    temp = f["temperature"].double()[:, None]
    greedy = temp <= 0
    w = ((vals - top) / torch.where(greedy, 1.0, temp)).exp()        # 64 bits: cuts fall on sums
    if f["top_k"] is not None:
        k = f["top_k"].long()[:, None]
        k = torch.where((k <= 0) | (k > vocab), vocab, k)
        w = torch.where(torch.arange(vocab, device=x.device)[None] < k, w, 0.0)
    if f["top_p"] is not None:
        p = f["top_p"].double()[:, None]
        cum = torch.cumsum(w, 1)
        before = torch.cat([torch.zeros_like(cum[:, :1]), cum[:, :-1]], 1)
        w = torch.where((p >= 1) | (before < p * cum[:, -1:]), w, 0.0)
    if f["min_p"] is not None:
        w = torch.where(w >= f["min_p"].double()[:, None], w, 0.0)
    by_index = torch.zeros_like(w).scatter_(1, order, w)
    cum = torch.cumsum(by_index, 1)
    hit = cum > s["u"].double()[:, None] * cum[:, -1:]
    first = torch.where(hit, torch.arange(vocab, device=x.device)[None], vocab).amin(1)
    return [torch.where(greedy[:, 0], order[:, 0], first)]


# ------------------------------------------------------------------------- floors
def work(case):
    op = case["op"]
    if op == "plan":
        ctx, new = _lengths(case)
        fresh = sum(_pages(c + n, case["page"]) - _pages(c, case["page"])
                    for c, n in zip(ctx, new))
        n = case["tokens"]
        # lengths in, lengths and offsets out, free pages in and table entries out,
        # position (4 bytes) and slot (8 bytes) of each token
        return {"bytes": 16 * case["batch"] + 8 + 8 * fresh + 12 * n, "flops": 4 * n}
    if op == "append":
        n, heads = case["tokens"], case["hq"] + 2 * case["hkv"]
        return {"bytes": n * (2 * heads * HEAD_DIM * 2 + 12) + 256,
                "flops": n * (case["hq"] + case["hkv"]) * HEAD_DIM * 3}
    if op == "attend":
        ctx, new = _lengths(case)
        seen = sum(n * c + n * (n + 1) // 2 for c, n in zip(ctx, new))
        cached = sum(c + n for c, n in zip(ctx, new) if n)
        return {"bytes": 4 * HEAD_DIM * (case["tokens"] * case["hq"] + cached * case["hkv"]),
                "flops": 4 * HEAD_DIM * case["hq"] * seen}
    size = 4 if case["dtype"] == "fp32" else 2
    return {"bytes": case["batch"] * (case["vocab"] * size + 28),
            "flops": 8 * case["batch"] * case["vocab"]}


# ------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "append": _exact_append, "attend": _exact_attend,
            "sample": _exact_sample}[case["op"]](s)


def _exact_plan(s):
    page, free = s["page"], s["free"].tolist()
    table = s["table"].cpu().numpy().copy()
    lens, cu, pos, slots, at = [], [0], [], [], 0
    for b, (c, n) in enumerate(zip(s["ctx"].tolist(), s["new"].tolist())):
        for j in range(_pages(c, page), _pages(c + n, page)):
            table[b, j] = free[at]
            at += 1
        for p in range(c, c + n):
            pos.append(p)
            slots.append(int(table[b, p // page]) * page + p % page)
        lens.append(c + n)
        cu.append(cu[-1] + n)
    pad = s["tokens"] - len(pos)
    make = lambda v, t: torch.tensor(v, dtype=t, device="cuda")  # noqa: E731
    return [torch.from_numpy(table).cuda(), make(lens, torch.int32), make(cu, torch.int32),
            make(pos + [0] * pad, torch.int32), make(slots + [-1] * pad, torch.int64),
            make([at], torch.int32)]


def _exact_append(s):
    hq, hkv, page = s["hq"], s["hkv"], s["k"].shape[2]
    n = s["qkv"].shape[0]
    half = HEAD_DIM // 2
    x = s["qkv"].double().reshape(n, -1, 2, half)
    z = torch.complex(x[:, :hq + hkv, 0], x[:, :hq + hkv, 1])
    turn = torch.polar(torch.ones(n, 1, half, dtype=torch.float64, device="cuda"),
                       (s["pos"].double()[:, None] * s["inv"].double())[:, None])
    z = z * turn
    rot = torch.cat([z.real, z.imag], -1)
    k, v = s["k"].double(), s["v"].double()
    kf, vf = k.transpose(1, 2).reshape(-1, hkv, HEAD_DIM), v.transpose(1, 2).reshape(-1, hkv, HEAD_DIM)
    kf[s["slots"]] = rot[:, hq:]
    vf[s["slots"]] = s["qkv"].double().reshape(n, -1, HEAD_DIM)[:, hq + hkv:]
    back = lambda t: t.reshape(-1, page, hkv, HEAD_DIM).transpose(1, 2).contiguous()  # noqa: E731
    return [rot[:, :hq].contiguous(), back(kf), back(vf)]


def _exact_attend(s):
    q, page, group = s["q"], s["k"].shape[2], s["q"].shape[1] // s["k"].shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b, length in enumerate(s["host_lens"]):
        t0, n = s["host_cu"][b], s["host_cu"][b + 1] - s["host_cu"][b]
        if n == 0:
            continue
        ids = s["table"][b, :_pages(length, page)].long()
        for head in range(q.shape[1]):
            keys = s["k"][ids, head // group].reshape(-1, HEAD_DIM)[:length].double()
            vals = s["v"][ids, head // group].reshape(-1, HEAD_DIM)[:length].double()
            for a in range(0, n, 2048):
                e = min(n, a + 2048)
                vis = length - n + e                              # nothing past it is seen
                sc = q[t0 + a:t0 + e, head].double() @ keys[:vis].t() / math.sqrt(HEAD_DIM)
                sc = sc + torch.full_like(sc, -math.inf).triu(length - n + a + 1)
                out[t0 + a:t0 + e, head] = torch.softmax(sc, -1) @ vals[:vis]
    return [out]


def _exact_sample(s):
    f = {k: None if v is None else v.double().cpu().numpy() for k, v in s["filters"].items()}
    x, u = s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy()
    tokens = []
    for b in range(x.shape[0]):
        row, t = x[b], f["temperature"][b]
        order = np.argsort(-row, kind="stable")
        if t <= 0:
            tokens.append(int(order[0]))
            continue
        if f["top_k"] is not None and 0 < f["top_k"][b] < len(order):
            order = order[:int(f["top_k"][b])]
        w = np.exp((row[order] - row[order[0]]) / t)
        if f["top_p"] is not None and f["top_p"][b] < 1:
            cum = np.cumsum(w)
            keep = int(np.searchsorted(cum, f["top_p"][b] * cum[-1])) + 1
            order, w = order[:keep], w[:keep]
        if f["min_p"] is not None:
            keep = int((w >= f["min_p"][b]).sum())
            order, w = order[:keep], w[:keep]
        by = np.argsort(order)
        cum = np.cumsum(w[by])
        at = int(np.searchsorted(cum, u[b] * cum[-1], side="right"))
        tokens.append(int(order[by[min(at, len(by) - 1)]]))
    return [torch.tensor(tokens, dtype=torch.int64, device="cuda")]
