"""Refusals of the paged-serving entry points, decided before any device work."""

import pytest

torch = pytest.importorskip("torch")

from decodebench_b200 import _native as N  # noqa: E402
from decodebench_b200 import ops  # noqa: E402

ENULL, ESHAPE, EALIGN, EDTYPE = -1, -2, -3, -5


def plan(**kw):
    a = dict(ctx=16, new=16, free=16, table=16, lens=16, cu=16, pos=16, slots=16, used=16, batch=2,
             n_free=4, page=16, width=8, tokens=5)
    a.update(kw)
    return N.load().dbk_page_plan(*[a[k] for k in ("ctx", "new", "free", "table", "lens", "cu", "pos",
                                                   "slots", "used", "batch", "n_free", "page",
                                                   "width", "tokens")], None)


@pytest.mark.parametrize("kw,want", [
    (dict(ctx=None), ENULL), (dict(table=None), ENULL), (dict(used=None), ENULL),
    (dict(free=None), ENULL), (dict(pos=None), ENULL), (dict(batch=0), ESHAPE),
    (dict(batch=16385), ESHAPE), (dict(page=0), ESHAPE), (dict(width=0), ESHAPE),
    (dict(tokens=-1), ESHAPE), (dict(n_free=-1), ESHAPE),
    (dict(batch=16384, width=131073), ESHAPE)])
def test_page_plan_refusals(kw, want):
    assert plan(**kw) == want


def append(**kw):
    a = dict(qkv=16, pos=16, slots=16, inv=16, q=16, k=16, v=16, n=3, hq=4, hkv=2, d=128, pages=4,
             page=16, dt=0)
    a.update(kw)
    return N.load().dbk_rope_append(*[a[k] for k in ("qkv", "pos", "slots", "inv", "q", "k", "v", "n",
                                                     "hq", "hkv", "d", "pages", "page", "dt")], None)


@pytest.mark.parametrize("kw,want", [
    (dict(qkv=None), ENULL), (dict(inv=None), ENULL), (dict(k=None), ENULL), (dict(d=64), ESHAPE),
    (dict(n=-1), ESHAPE), (dict(hq=0), ESHAPE), (dict(page=0), ESHAPE), (dict(dt=2), EDTYPE),
    (dict(q=24), EALIGN), (dict(v=8), EALIGN), (dict(q=16), ESHAPE), (dict(q=16 + 3 * 8 * 256 - 16), ESHAPE), (dict(n=0, qkv=None, q=None), 0)])
def test_rope_append_refusals(kw, want):
    assert append(**kw) == want


def attend(**kw):
    a = dict(q=16, k=16, v=16, cu=16, lens=16, table=16, out=32, n=3, batch=2, hq=4, hkv=2, d=128,
             pages=4, page=16, width=8, scale=0.1, dt=0)
    a.update(kw)
    return N.load().dbk_chunk_attention(*[a[k] for k in (
        "q", "k", "v", "cu", "lens", "table", "out", "n", "batch", "hq", "hkv", "d", "pages", "page",
        "width", "scale", "dt")], None, 0, None)


@pytest.mark.parametrize("kw,want", [
    (dict(q=None), ENULL), (dict(cu=None), ENULL), (dict(lens=None), ENULL), (dict(d=64), ESHAPE),
    (dict(hq=5), ESHAPE), (dict(hq=258), ESHAPE), (dict(hq=1), ESHAPE), (dict(n=-1), ESHAPE),
    (dict(batch=0), ESHAPE), (dict(page=20), ESHAPE), (dict(page=4), ESHAPE), (dict(width=0), ESHAPE),
    (dict(table=None, page=100), ESHAPE),                         # contiguous: pages != batch
    (dict(scale=0.0), ESHAPE), (dict(scale=-1.0), ESHAPE), (dict(scale=float("nan")), ESHAPE),
    (dict(scale=float("inf")), ESHAPE), (dict(scale=2e38), ESHAPE),
    (dict(out=16), ESHAPE), (dict(out=16 + 3 * 4 * 256 - 16), ESHAPE), (dict(batch=65537), ESHAPE), (dict(pages=1 << 24, page=128), ESHAPE),
    (dict(dt=3), EDTYPE), (dict(out=8), EALIGN), (dict(k=20), EALIGN),
    (dict(n=0, q=None, out=None), 0)])
def test_chunk_attention_refusals(kw, want):
    assert attend(**kw) == want


def test_chunk_attention_workspace_stops_growing():
    f = N.load().dbk_chunk_attention_workspace_bytes
    assert f(0, 8, 2) == 0 and f(5, 8, 3) == 0
    assert 0 < f(1, 8, 2) < f(32, 8, 2) < f(33, 8, 2) == f(129, 8, 2) == f(1 << 20, 8, 2)
    assert f(129, 1, 1) == f(5000, 1, 1)


def test_ops_refuse_cpu_tensors():
    z = lambda *s: torch.zeros(*s, dtype=torch.float16)  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.page_plan(i(2), i(2), i(4), i(2, 3), 16, 4)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.rope_append(z(3, 4 * 128), i(3), i(3).long(), torch.zeros(64), z(2, 1, 16, 128),
                        z(2, 1, 16, 128), 2, 1)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.chunk_attention(z(3, 2, 128), z(2, 1, 16, 128), z(2, 1, 16, 128), i(2), i(1), i(1, 2))


def sample(**kw):
    a = dict(x=16, u=16, t=None, k=None, p=None, mp=None, out=16, batch=2, vocab=100, temp=1.0,
             top_k=0, top_p=1.0, min_p=0.0, dt=2)
    a.update(kw)
    return N.load().dbk_sample(*[a[k] for k in ("x", "u", "t", "k", "p", "mp", "out", "batch", "vocab",
                                                "temp", "top_k", "top_p", "min_p", "dt")], None)


@pytest.mark.parametrize("kw,want", [
    (dict(x=None), ENULL), (dict(u=None), ENULL), (dict(out=None), ENULL), (dict(vocab=0), ESHAPE),
    (dict(vocab=(1 << 20) + 1), ESHAPE), (dict(batch=-1), ESHAPE), (dict(dt=5), EDTYPE),
    (dict(x=4), EALIGN), (dict(temp=float("nan")), ESHAPE), (dict(top_p=float("nan")), ESHAPE),
    (dict(batch=0, x=None), 0)])
def test_sample_refusals(kw, want):
    assert sample(**kw) == want
