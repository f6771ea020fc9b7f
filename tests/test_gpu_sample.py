"""dbk_sample against a 64-bit restatement that sorts: the same token, row by row."""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from decodebench_b200 import ops  # noqa: E402

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def pick(row, u, t=1.0, k=0, p=1.0, mp=0.0):
    """(token, how near the draw or a cut comes to another answer, in parts of the sum)."""
    x = row.double().numpy()
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.argsort(-x, kind="stable")
    top = x[order[0]]
    if top == -np.inf:
        return -1, 1.0
    if not t > 0:
        return int(order[0]), 1.0
    if 0 < k < len(order):
        order = order[:k]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / t))
    near = 1.0
    if p < 1:
        cum = np.cumsum(w)
        need = np.float64(np.float32(p)) * cum[-1]
        keep = int(np.searchsorted(cum, need)) + 1
        # an exact hit is an exact sum of equal weights: no doubt about it
        gaps = np.abs(cum / need - 1) if need > 0 else np.ones(1)
        near = min([near] + [g for g in gaps if g > 0])
        order, w = order[:keep], w[:keep]
    keep = int((w >= min(np.float64(np.float32(mp)), 1.0)).sum())
    order, w = order[:keep], w[:keep]
    by = np.argsort(order)
    cum = np.cumsum(w[by])
    target = np.float64(u) * cum[-1]
    at = int(np.searchsorted(cum, target, side="right"))
    if target > 0:
        near = min([near] + [g for g in np.abs(cum / target - 1) if g > 0])
    return int(order[by[min(at, len(by) - 1)]]), near


def check(logits, u, **f):
    got = ops.sample(logits.cuda(), u.cuda(), **{
        n: (v.cuda() if isinstance(v, torch.Tensor) else v) for n, v in f.items()}).tolist()
    names = {"temperature": ("t", 1.0), "top_k": ("k", 0), "top_p": ("p", 1.0), "min_p": ("mp", 0.0)}
    for b in range(logits.shape[0]):
        kw = {}
        for n, (short, off) in names.items():
            v = f.get(n)
            kw[short] = off if v is None else (v[b].item() if isinstance(v, torch.Tensor) else v)
        want, near = pick(logits[b], u[b].item(), **kw)
        # weights below 2^-14 are 32-bit (2^-21 each): sums are right to 2^-34, so only a draw
        # within 2^-30 of a border may fall on its other side
        assert got[b] == want or near < 2.0 ** -30, f"row {b}: {got[b]} for {want} with {kw}"


def rows(batch, vocab, dt, seed, spread=2.5, hot=9.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(batch, vocab, generator=g) * spread
    idx = torch.randint(0, vocab, (batch, 12), generator=g)
    x.scatter_add_(1, idx, torch.rand(batch, 12, generator=g) * hot)
    return x.to(dt), torch.rand(batch, generator=g)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("batch,vocab", [(1, 1), (3, 2), (5, 7), (2, 1000), (7, 4097), (3, 32003),
                                         (1, 128000), (300, 501), (2, 200001)])
def test_filters(dt, batch, vocab):
    x, u = rows(batch, vocab, dt, seed=vocab + batch)
    check(x, u)
    check(x, u, temperature=0.0)
    check(x, u, temperature=0.7, top_k=5)
    check(x, u, temperature=1.3, top_p=0.9)
    check(x, u, temperature=0.8, top_k=50, top_p=0.95)
    check(x, u, min_p=0.05)
    check(x, u, temperature=1.1, top_k=40, top_p=0.8, min_p=0.1)


def test_small_min_p():
    x, u = rows(6, 20000, F32, seed=3, spread=1.5)
    for mp in (1e-9, 1e-5, 2.0 ** -14, 1.1e-4, 2.0 ** -13, 1e-3):
        check(x, u, min_p=mp, temperature=1.7)
        check(x, u, min_p=mp, top_p=0.9)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_flat_and_long_tails(dt):
    """Flat rows (every weight counts), cuts deep in the tail, sharp temperatures."""
    x, u = rows(4, 30000, dt, seed=1, spread=0.3, hot=0.0)
    for f in (dict(), dict(top_p=0.5), dict(top_p=0.999), dict(top_k=20000), dict(top_k=29999),
              dict(temperature=5.0, top_p=0.99), dict(temperature=0.01, top_k=10)):
        check(x, u, **f)
    x, u = rows(4, 50000, dt, seed=2, spread=6.0, hot=0.0)
    for f in (dict(top_p=0.99999), dict(top_k=30000), dict(top_k=49000, top_p=0.9999),
              dict(temperature=0.05, top_p=0.9999), dict(temperature=3.0, top_k=1000)):
        check(x, u, **f)


@pytest.mark.parametrize("dt,vocab", [(F32, 32768), (F32, 32771), (BF16, 32768), (F16, 32761)])
def test_many_rows_with_the_largest_slices(dt, vocab):
    """More rows than SMs: a CTA has up to 32,768 logits, here also all in one bin of its histogram."""
    batch = 160
    x, u = rows(batch, vocab, dt, 11)
    for b in range(0, batch, 8):               # all but one alike, at several places of a bin
        x[b] = 0.0
        x[b, (b * 977) % vocab] = 1.0 + b / 64
    for b in range(1, batch, 8):               # a few values, many of each
        x[b] = torch.randint(-3, 4, (vocab,), generator=torch.Generator().manual_seed(b)).to(dt)
    check(x, u, top_p=0.9, temperature=0.7)
    check(x, u, top_k=1000, top_p=0.95)
    k = torch.tensor([1, 40, 5000, vocab - 1], dtype=torch.int32).repeat(batch // 4)
    check(x, u, top_k=k)
    check(x, u, min_p=0.05)


@pytest.mark.parametrize("dt,batch,vocab", [(F32, 2, 300001), (BF16, 3, 262145), (F16, 1, 1 << 20), (F32, 150, 262148)])
def test_vocabularies_past_a_cluster_of_slices(dt, batch, vocab):
    x, u = rows(batch, vocab, dt, 12)
    check(x, u, top_p=0.9, temperature=0.7)
    if batch < 10:
        check(x, u, top_k=1000, top_p=0.95)
        check(x, u, top_k=50)
        check(x, u, min_p=0.05)
        check(x, u)


def test_ties():
    """Equal logits: the lower index comes first in every cut."""
    u = torch.tensor([0.0, 0.3, 0.6, 0.999999])
    x = torch.zeros(4, 9001)
    for f in (dict(), dict(top_k=1), dict(top_k=17), dict(top_p=0.5), dict(top_p=0.25, top_k=4000),
              dict(min_p=1.0), dict(temperature=0.0)):
        check(x, u, **f)
    g = torch.Generator().manual_seed(0)
    x = torch.randint(0, 4, (4, 9001), generator=g).float()
    for f in (dict(top_k=3000), dict(top_p=0.6), dict(top_p=0.97, temperature=2.0), dict(top_k=1),
              dict(top_k=7000, top_p=0.9), dict(min_p=0.3)):
        check(x, u, **f)
    x = torch.randint(-1, 2, (4, 9001), generator=g).float() * 0.0        # +0 and -0
    check(x, u, top_k=5000)


def test_masked_rows():
    """-inf, the type's lowest value, NaN and +inf among the logits; rows with nothing left."""
    for dt in (F32, F16, BF16):
        x, u = rows(8, 3001, dt, seed=5)
        low = torch.finfo(dt).min
        x[0, 5:] = -math.inf
        x[1] = -math.inf
        x[2, ::2] = low
        x[3] = low
        x[4, 7:] = float("nan")
        x[5] = float("nan")
        x[6, 100] = math.inf
        x[7, 100:200] = math.inf
        for f in (dict(), dict(top_k=3), dict(top_p=0.7), dict(min_p=0.2), dict(temperature=0.0),
                  dict(top_k=1000, top_p=0.99)):
            check(x, u, **f)
        assert ops.sample(x.cuda(), u.cuda())[1].item() == -1


def test_parameters_per_row_and_extremes():
    x, _ = rows(12, 6000, F32, seed=9)
    u = torch.tensor([0.0, 1 - 2.0 ** -24] * 6)
    f = dict(temperature=torch.tensor([0.0, -1, 1e-30, 1e-3, 1e6, 1.0, 1, 1, 1, 1, 2, 0.5]),
             top_k=torch.tensor([0, 3, 0, 6000, 7000, -5, 1, 5999, 50, 0, 10, 2], dtype=torch.int32),
             top_p=torch.tensor([1.0, 0.5, 2.0, 0.9, 0.9, 0.0, -1.0, 1.0, 1e-9, 0.5, 0.99, 0.999]),
             min_p=torch.tensor([0.0, 0.5, 0, 0, 0.5, 0, 0, 0, 0, 1.0, 3.0, -1.0]))
    check(x, u, **f)


def test_many_draws_follow_the_weights():
    """Equally spaced numbers hit each token as often as its share of the weight says."""
    x = torch.tensor([[0.0, 1.0, 2.0, -math.inf, 0.5]])
    n = 4096
    u = (torch.arange(n) + 0.5) / n
    got = ops.sample(x.expand(n, 5).contiguous().cuda(), u.cuda()).cpu()
    share = torch.bincount(got, minlength=5).double() / n
    assert ((share - torch.softmax(x[0].double(), 0)).abs() <= 1.5 / n).all()


def test_graph_and_streams():
    x, u = rows(33, 20000, BF16, seed=4)
    x, u = x.cuda(), u.cuda()
    f = dict(temperature=0.9, top_k=100, top_p=0.9)
    want = ops.sample(x, u, **f)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample(x, u, out=out, **f)
    out.fill_(-7)
    graph.replay()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(ops.sample(x, u, **f))
    torch.cuda.synchronize()
    assert torch.equal(out, want) and all(torch.equal(g, want) for g in got)


def test_refuses_wrong_tensors():
    x, u = torch.zeros(2, 10, device="cuda"), torch.zeros(2, device="cuda")
    for bad in (dict(top_k=torch.zeros(2, device="cuda")), dict(top_p=torch.zeros(3, device="cuda")),
                dict(temperature=float("nan")), dict(out=torch.zeros(2, device="cuda"))):
        with pytest.raises(ValueError):
            ops.sample(x, u, **bad)
    with pytest.raises(TypeError):
        ops.sample(x.double(), u)
    with pytest.raises(ValueError, match="contiguous"):
        ops.sample(torch.zeros(10, 2, device="cuda").t(), u)
