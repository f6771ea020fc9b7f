"""dbk_sample where far logits decide: heavy tails, cuts among them, draws of 0. The restatement
sums 80-bit floats (2^-64 a step: 2^-44 over 2^20 of them)."""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from decodebench_b200 import ops  # noqa: E402

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
LD = np.longdouble


def picks(row, us, t=1.0, k=0, p=1.0):
    """[(token, how near the draw or a cut comes to another answer, in parts of the sum)] of one row for
    several random numbers."""
    x = row.double().numpy()
    order = np.argsort(-x, kind="stable")
    t = float(np.float32(t))
    if 0 < k < len(order):
        order = order[:k]
    w = np.exp((x[order].astype(LD) - LD(x[order[0]])) / LD(t))
    w = np.where(w > np.exp2(LD(-1075)), w, LD(0))       # 80 bits have exponents that 64 do not
    near = 1.0
    if p < 1:
        cum = np.cumsum(w)
        need = LD(np.float32(p)) * cum[-1]
        keep = int(np.searchsorted(cum, need)) + 1
        near = float(np.abs(cum - need).min() / cum[-1])
        order, w = order[:keep], w[:keep]
    by = np.argsort(order)
    cum = np.cumsum(w[by])
    out = []
    for u in us:
        target = LD(float(u)) * cum[-1]
        at = int(np.searchsorted(cum, target, side="right"))
        gap = float(np.abs(cum[max(at - 2, 0):at + 2] - target).min() / cum[-1]) if target > 0 else 1.0
        out.append((int(order[by[min(at, len(by) - 1)]]), min(near, gap)))
    return out


def check_rows(x, us, within, **f):
    """x [vocab], us [n]: n rows alike. Only a draw or cut within `within` of a border may fall on its
    other side."""
    rows = x.cuda()[None].expand(len(us), -1).contiguous()
    names = {"temperature": "t", "top_k": "k", "top_p": "p"}
    got = ops.sample(rows, us.cuda(), **f).tolist()
    want = picks(x, us.tolist(), **{names[n]: v for n, v in f.items()})
    bad = [(i, g, w) for i, (g, (w, near)) in enumerate(zip(got, want)) if g != w and near >= within]
    assert not bad, f"{len(bad)} of {len(us)} with {f}, first {bad[0]}"


def tail(vocab, kind, seed, dt=F32):
    """One logit at 0 (anywhere), the others 12 to 18 below it."""
    g = torch.Generator().manual_seed(seed)
    if kind == "flat":
        x = torch.full((vocab,), -14.37)
    elif kind == "spread":
        x = -15.0 + 0.3 * torch.randn(vocab, generator=g)
    else:
        x = -12.0 - 6.0 * torch.rand(vocab, generator=g)
    x[int(torch.randint(0, vocab, (1,), generator=g))] = 0.0
    return x.to(dt), torch.rand(48, generator=g)


# What the general path's rounding comes to: weights by 64-bit exp() of a rounded argument of at most 32
# (2^-47), sums of doubles in trees and runs of 32 (2^-47), cuts in units of which 2^20 roundings are
# 2^-42 of the row's sum: below 2^-41 together.
GENERAL = 2.0 ** -41


@pytest.mark.parametrize("vocab", [300001, 1 << 20])
@pytest.mark.parametrize("kind", ["flat", "spread", "even"])
@pytest.mark.parametrize("t", [0.6, 1.0, 1.3])
def test_tails_that_carry_weight(vocab, kind, t):
    x, u = tail(vocab, kind, seed=vocab % 97)
    check_rows(x, u, GENERAL, temperature=t)
    check_rows(x, u, GENERAL, temperature=t, top_p=0.9)
    check_rows(x, u[:16], GENERAL, temperature=t, top_k=vocab // 3, top_p=0.999)


@pytest.mark.parametrize("dt", [F16, BF16])
def test_tails_of_16_bit_logits(dt):
    x, u = tail(262147, "even", 3, dt)
    check_rows(x, u, GENERAL, temperature=1.1)
    check_rows(x, u, GENERAL, temperature=1.1, top_p=0.97)


def test_crowded_rows_of_a_common_vocabulary():
    """Rows that overflow the common path's lists: many equal logits at the cut, far below the largest."""
    x, u = tail(120000, "flat", 5)
    check_rows(x, u, GENERAL, top_p=0.97)
    check_rows(x, u, GENERAL, temperature=0.8, top_k=70000)


def test_top_k_among_logits_that_weigh_next_to_nothing():
    """The k-th logit lies more than 2^-46 below the largest: the first k are kept all the same, and a
    draw of 0 takes the first of them."""
    vocab = 300001
    g = torch.Generator().manual_seed(8)
    x = -40.0 - 20.0 * torch.rand(vocab, generator=g)
    x[200000:200040] = 0.5 * torch.rand(40, generator=g)
    for k in (1000, 41, 250000, vocab - 1):
        for t in (1.0, 0.5):
            check_rows(x, torch.tensor([0.0, 0.25, 1 - 2.0 ** -24]), GENERAL, top_k=k, temperature=t)
    x[::2] = -math.inf
    check_rows(x, torch.tensor([0.0, 0.5]), GENERAL, top_k=149999)
    check_rows(x, torch.tensor([0.0, 0.5]), GENERAL, top_k=200000)


def test_a_draw_of_zero_takes_the_first_that_weighs_anything():
    vocab = 300001
    x = torch.full((vocab,), -math.inf)
    x[7:] = -800.0                                # exp() of it is 0 in 64 bits
    x[1000:] = -60.0
    x[150000] = 0.0
    check_rows(x, torch.tensor([0.0]), GENERAL)
    check_rows(x, torch.tensor([0.0]), GENERAL, temperature=2.0)


def test_infinite_logits_and_a_cut_behind_them():
    x = torch.linspace(-3, 3, 300001)
    x[5], x[77], x[299999] = math.inf, math.inf, math.inf
    got = ops.sample(x.cuda()[None].expand(5, -1).contiguous(), torch.tensor([0.0, 0.4, 0.9, 0.5, 0.999]).cuda(),
                     top_k=torch.tensor([0, 3, 2, 1, 1000], dtype=torch.int32, device="cuda"))
    assert got.tolist() == [5, 77, 77, 5, 299999]


def test_a_logit_that_rounds_onto_a_bin_border():
    """Distances whose product with the bins per logit lies just below the border of two bins and rounds
    onto it: every pass has to put the logit into the same bin. The cut falls into the second of
    the two, behind more logits than the lists hold; the last kept one has the highest index."""
    vocab, front = 32003, 6000
    scale = np.float32(np.float32(1.4426950408889634) * np.float32(8 * np.float32(np.float32(512) / np.float32(46))))
    rows, last = [], []
    for b in range(2, 40):
        edge = 8 * b - 0.5
        d = np.float32(edge / float(scale))
        near = [d, np.nextafter(d, np.float32(0)), np.nextafter(d, np.float32(9))]
        hit = [v for v in near if np.float32(v * scale) == np.float32(edge) and float(v) * float(scale) < edge]
        if not hit:
            continue
        x = torch.full((vocab,), -31.0)
        x[0] = 0.0
        x[1:1 + front] = -(8 * (b - 1) + 3) / float(scale)
        x[front + 50] = -float(hit[0])
        x[20000:20300] = -(8 * b + 0.2 + torch.arange(300) * 0.02) / float(scale)
        rows.append(x)
        last.append(20000 + 149)
    assert len(rows) > 10
    x, u = torch.stack(rows[:8]).cuda(), torch.full((8,), 1 - 2.0 ** -24, device="cuda")
    assert ops.sample(x, u, top_k=front + 2 + 150).tolist() == last[:8]
    x, u = torch.stack(rows[8:]).cuda(), torch.full((len(rows) - 8,), 1 - 2.0 ** -24, device="cuda")
    assert ops.sample(x, u, top_k=front + 2 + 150).tolist() == last[8:]


@pytest.mark.parametrize("dt,vocab", [(F32, 9), (F16, 1000), (BF16, 32003), (F32, 128000)])
def test_draws_among_the_smallest_weights(dt, vocab):
    """Draws of 0, and below the step of 24-bit random numbers, in rows of the common path: the first
    index that is kept and weighs anything, however little."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(vocab, generator=g)
    x[0], x[1], x[2] = -math.inf, -900.0, -60.0
    x = x.to(dt)
    u = torch.tensor([0.0, 1e-44, 1e-30, 2.0 ** -40, 2.0 ** -25, 2.0 ** -24, 2.0 ** -20])
    check_rows(x, u[:6], GENERAL)
    assert ops.sample(x.cuda()[None], u[:1].cuda()).tolist() == [2]
    check_rows(x, u, 2.0 ** -25, temperature=0.5)
    for f in (dict(top_k=vocab - 2), dict(top_k=5), dict(top_p=0.99), dict(top_k=40, top_p=0.9)):
        check_rows(x, u, 2.0 ** -25, **f)


def test_parameters_that_are_not_numbers():
    """NaN among the rows' parameters: top-p and min-p are off, temperature takes the largest logit."""
    x = torch.randn(4, 5000, generator=torch.Generator().manual_seed(1)).cuda()
    u = torch.tensor([0.3, 0.7, 0.9, 0.5]).cuda()
    nan = torch.full((4,), math.nan, device="cuda")
    plain = ops.sample(x, u)
    assert torch.equal(ops.sample(x, u, min_p=nan), plain)
    assert torch.equal(ops.sample(x, u, top_p=nan), plain)
    assert torch.equal(ops.sample(x, u, temperature=nan), x.argmax(1))
    big = torch.randn(2, 300001, generator=torch.Generator().manual_seed(2)).cuda()
    assert torch.equal(ops.sample(big, u[:2], min_p=nan[:2]), ops.sample(big, u[:2]))
