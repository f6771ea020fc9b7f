"""Bounded waits of chunk attention's file, which has an error flag and a poll budget of its own: they
run out, are reported by the library's calls, and leave the context usable."""

import math

import pytest

torch = pytest.importorskip("torch")

from decodebench_b200 import _native as N  # noqa: E402
from decodebench_b200 import ops  # noqa: E402
from tests.test_gpu_paged import D, check_attention, make  # noqa: E402

pytestmark = pytest.mark.gpu
K_TIMEOUT_EMPTY, K_TIMEOUT_MMA = 2, 3


@pytest.fixture()
def lib():
    L = N.load()
    assert ops.take_device_error() == 0
    yield L
    N.check("set_spin_limit", L.dbk_set_spin_limit(0))
    assert ops.take_device_error() == 0


@pytest.mark.parametrize("which,code", [(2, K_TIMEOUT_EMPTY), (3, K_TIMEOUT_MMA)])
def test_wait_runs_out_and_reports(lib, which, code):
    s = torch.cuda.current_stream().cuda_stream
    N.check("set_spin_limit", lib.dbk_set_spin_limit(2000))
    N.check("test_bounded_wait", lib.dbk_test_bounded_wait(which, s))
    assert lib.dbk_take_device_error() == code
    assert lib.dbk_take_device_error() == 0                # taking it cleared it
    N.check("test_bounded_wait", lib.dbk_test_bounded_wait(which, s))
    with pytest.raises(RuntimeError, match="bounded wait"):
        ops.check_device_error()
    N.check("set_spin_limit", lib.dbk_set_spin_limit(0))
    q, k, v, cu, lens, table = make([700, 3], [40, 1], 8, 2, 16, torch.bfloat16)
    out = ops.chunk_attention(q, k, v, cu, lens, page_table=table)
    check_attention(out, q, k, v, [700, 3], [40, 1], table, 1 / math.sqrt(D))
    assert lib.dbk_take_device_error() == 0


def test_the_budget_is_this_files_too(lib):
    """The smaller the budget the sooner a wait gives up: with 16 times the polls it takes several times
    as long."""
    s = torch.cuda.current_stream().cuda_stream
    times = []
    for polls in (2000, 2000, 32000):                      # (the first launch loads the kernel)
        N.check("set_spin_limit", lib.dbk_set_spin_limit(polls))
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        N.check("test_bounded_wait", lib.dbk_test_bounded_wait(3, s))
        b.record()
        assert lib.dbk_take_device_error() == K_TIMEOUT_MMA
        times.append(a.elapsed_time(b))
    assert times[2] > 4 * times[1]


def test_refuses_other_waits(lib):
    assert lib.dbk_test_bounded_wait(4, None) == N.DBK_ESHAPE
    assert lib.dbk_test_bounded_wait(-1, None) == N.DBK_ESHAPE
