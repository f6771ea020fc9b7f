"""More refusals of the paged-serving entry points, decided before any device work."""

import pytest

pytest.importorskip("torch")

from decodebench_b200 import _native as N  # noqa: E402
from tests.test_paged_cpu import EDTYPE, ENULL, attend  # noqa: E402


@pytest.mark.parametrize("dt,want", [
    (N.DBK_F32 | N.DBK_WEIGHTS_ONE, EDTYPE), (N.DBK_BF16 | 0x400, EDTYPE), (N.DBK_BF16 | N.DBK_WEIGHTS_ONE, ENULL),
    (N.DBK_F16 | N.DBK_WEIGHTS_ONE, ENULL)])
def test_chunk_attention_weight_parts(dt, want):
    assert attend(dt=dt, q=None) == want
