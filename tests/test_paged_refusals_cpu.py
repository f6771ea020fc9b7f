"""More refusals of the paged-serving entry points, decided before any device work."""

import pytest

pytest.importorskip("torch")

from decodebench_b200 import _native as N  # noqa: E402
from tests.test_paged_cpu import EDTYPE, ENULL, ESHAPE, append, attend, plan, sample  # noqa: E402


@pytest.mark.parametrize("dt,want", [
    (N.DBK_F32 | N.DBK_WEIGHTS_ONE, EDTYPE), (N.DBK_BF16 | 0x400, EDTYPE), (N.DBK_BF16 | N.DBK_WEIGHTS_ONE, ENULL),
    (N.DBK_F16 | N.DBK_WEIGHTS_ONE, ENULL)])
def test_chunk_attention_weight_parts(dt, want):
    assert attend(dt=dt, q=None) == want


# Addresses that nothing is read from: every call here is refused. 3 tokens, 4 / 2 heads, 4 pages of 16:
# q 3,072 bytes, qkv 6,144, a cache 32,768.
APART = dict(qkv=0x100000, q=0x200000, k=0x300000, v=0x400000, pos=0x500000, slots=0x600000, inv=0x700000)


@pytest.mark.parametrize("kw", [
    dict(q=0x300000 + 32768 - 16), dict(q=0x300000 - 3072 + 16), dict(q=0x400000), dict(k=0x400000 + 16),
    dict(v=0x300000), dict(qkv=0x300000 + 16), dict(qkv=0x400000 - 6144 + 16), dict(qkv=0x200000 + 3072 - 16),
    dict(pos=0x200000), dict(slots=0x300000 + 64), dict(inv=0x400000 + 32768 - 4)])
def test_rope_append_outputs_that_overlap(kw):
    assert append(**{**APART, **kw}) == ESHAPE


def attend_apart(ws=0x500000, ws_bytes=1 << 16, **kw):
    a = dict(q=0x100000, out=0x200000, k=0x300000, v=0x400000, cu=0x600000, lens=0x610000, table=0x620000,
             n=3, batch=2, hq=4, hkv=2, d=128, pages=4, page=16, width=8, scale=0.1, dt=0)
    a.update(kw)
    return N.load().dbk_chunk_attention(*[a[k] for k in (
        "q", "k", "v", "cu", "lens", "table", "out", "n", "batch", "hq", "hkv", "d", "pages", "page",
        "width", "scale", "dt")], ws, ws_bytes, None)


@pytest.mark.parametrize("kw", [
    dict(out=0x300000), dict(out=0x300000 + 32768 - 16), dict(out=0x400000 - 16), dict(cu=0x200000 + 3068),
    dict(lens=0x200000), dict(table=0x200000 - 60), dict(ws=0x200000 + 3072 - 16), dict(ws=0x400000 - (1 << 16) + 16),
    dict(ws=0x100000), dict(ws=0x610000 - 256, ws_bytes=512)])
def test_chunk_attention_outputs_that_overlap(kw):
    assert attend_apart(**kw) == ESHAPE


@pytest.mark.parametrize("kw", [
    dict(lens=0x1000), dict(lens=0x2000 + 4), dict(cu=0x1000 - 8), dict(table=0x3000 + 12), dict(table=0x1000 - 60),
    dict(pos=0x8000), dict(slots=0x7000 + 16), dict(used=0x5000 + 4), dict(used=0x3000), dict(used=0x8000 + 36)])
def test_page_plan_outputs_that_overlap(kw):
    """2 requests of 8 pages, 4 free pages, 5 tokens; seq_lens written over ctx_lens would be read by
    other blocks."""
    apart = dict(ctx=0x1000, new=0x2000, free=0x3000, table=0x4000, lens=0x5000, cu=0x6000, pos=0x7000,
                 slots=0x8000, used=0x9000)
    apart.update(kw)
    assert plan(**apart) == ESHAPE


@pytest.mark.parametrize("kw", [
    dict(out=0x1000 + 792), dict(out=0x2000 - 8), dict(t=0x7000 + 12), dict(k=0x7000), dict(p=0x7000 + 8),
    dict(mp=0x7000 - 4)])
def test_sample_outputs_that_overlap(kw):
    """2 rows of 100 fp32 logits; 16 bytes of tokens."""
    assert sample(**{**dict(x=0x1000, u=0x2000, out=0x7000), **kw}) == ESHAPE


def test_the_status_of_an_overlap_says_so():
    assert "overlap" in N.status_string(ESHAPE)
