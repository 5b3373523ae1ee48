"""What the block-scaled operators report, and how they end when a wait of theirs runs out.  No test here faults or hangs a GPU: bad layouts
are found by the kernels' own checks, and every wait has its limit."""
import ctypes

import pytest
import torch

import block128_ref as ref

pytestmark = pytest.mark.gpu

BAD_GROUP_LAYOUT, PIPE_TIMEOUT = 5, 2


@pytest.fixture(scope="module", autouse=True)
def _need_gpu(built_lib):
    if not torch.cuda.is_available():
        pytest.fail("needs a CUDA device")


def _read(lib, stream):
    from deepgemm_b200 import _lib
    out = (ctypes.c_int32 * 5)()
    _lib.check(lib.mm_block128_read_status(stream.cuda_stream, out))
    return list(out)


def test_a_read_on_another_stream_takes_each_report_whole(built_lib):
    """A kernel reports a mixed block while another stream reads: the report comes with one of the reads (or with several: each warp that sees
    the block reports it), with all its words."""
    import megamoe
    zeros = lambda *s: torch.zeros(s, dtype=torch.uint8, device="cuda").view(ref.E4M3)   # noqa: E731
    index = torch.zeros(256, dtype=torch.int32, device="cuda")
    index[200] = 1
    a, w = (zeros(256, 128), torch.ones((256, 1), device="cuda")), (zeros(2, 128, 128), torch.ones((2, 1, 1), device="cuda"))
    d = torch.zeros((256, 128), dtype=torch.bfloat16, device="cuda")
    here, there = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    _read(built_lib, here)
    for turn in range(1000):
        with torch.cuda.stream(there):
            torch.cuda._sleep(1000 + turn % 100 * 400)               # up to 20 us, so that reads come before, within and behind the report
            megamoe.m_grouped_fp8_gemm_nt_contiguous_block128(a, w, d, index)
        got = [_read(built_lib, here) for _ in range(6)]
        there.synchronize()
        got.append(_read(built_lib, here))
        reports = [r for r in got if r[0]]
        assert reports and all(r == [BAD_GROUP_LAYOUT, 0, 1, 0, 1] for r in reports), (turn, reports)
