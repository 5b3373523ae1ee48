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


@pytest.fixture
def waits(built_lib):
    """Sets how the waits of the calls that follow end; as ever afterwards."""
    yield lambda given_up=-1, limit_ns=0: built_lib.mm_block128_test_waits(given_up, limit_ns)
    built_lib.mm_block128_test_waits(-1, 0)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (77, 300, 2048)])
@pytest.mark.parametrize("cta", [0, 1, 5])
def test_a_split_tile_is_not_written_when_one_of_its_ctas_gave_up(built_lib, waits, m, n, k, cta):
    """The CTAs that share a tile add up what each has left in its shared memory, and one that gave up has left operands there."""
    import megamoe
    g = torch.Generator().manual_seed(5)
    a, sa = ref.random_operand(g, m, k).cuda(), ref.random_scales(g, m, ref.blocks(k)).cuda()
    b, sb = ref.random_operand(g, n, k).cuda(), ref.random_scales(g, ref.blocks(n), ref.blocks(k)).cuda()
    want = megamoe.fp8_gemm_nt_block128((a, sa), (b, sb), out_dtype=torch.float32)
    megamoe.check_block128_status()
    out = torch.full((m, n), 5.0, device="cuda")
    waits(given_up=cta)
    megamoe.fp8_gemm_nt_block128((a, sa), (b, sb), out=out)
    status = _read(built_lib, torch.cuda.current_stream())
    assert status[:3] == [PIPE_TIMEOUT, 20, cta], status
    assert not bool((want == 5).any())
    left = (out == 5).all(0).view(-1).cpu()
    tiles = [left[i:i + 128] for i in range(0, n, 128)]
    assert sum(bool(t.all()) for t in tiles) == 1 and not any(bool(t.any()) for t in tiles if not bool(t.all())), "one whole tile and nothing else"
    assert torch.equal(out.cpu()[:, ~left], want.cpu()[:, ~left])
    waits()
    assert torch.equal(megamoe.fp8_gemm_nt_block128((a, sa), (b, sb), out=out), want)
    megamoe.check_block128_status()


def _layer(t, e, k, h, i):
    import megamoe
    from test_gpu_few_tokens import make
    g = torch.Generator().manual_seed(6)
    x, w1, w2 = make(g, t, e, h, i)
    l1, l2 = (megamoe.pack_weights_tiled(w1[0].cuda(), "l1"), w1[1].cuda()), (megamoe.pack_weights_tiled(w2[0].cuda(), "l2"), w2[1].cuda())
    x, logits = x.cuda(), torch.randn((t, e), generator=g).cuda()
    return lambda out=None: megamoe.fp8_moe_few_tokens(x, l1, l2, router_logits=logits, num_topk=k, out=out)


@pytest.mark.parametrize("t,e,k,h,i", [(1, 16, 6, 4096, 2048), (33, 16, 4, 2048, 1024), (130, 8, 2, 1024, 512)])
def test_a_layer_whose_waits_run_out_reports_it_and_ends(built_lib, waits, t, e, k, h, i):
    """With a limit of a nanosecond the wait for the activations of the first product runs out in every CTA, and all other waits end by
    that: the call returns, leaves the output as it was, and the next one is as ever."""
    import megamoe
    call = _layer(t, e, k, h, i)
    want = call()
    megamoe.check_block128_status()
    out = torch.full((t, h), 3.0, dtype=torch.bfloat16, device="cuda")
    for _ in range(3):
        waits(limit_ns=1)
        call(out)
        status = _read(built_lib, torch.cuda.current_stream())
        assert status[:2] == [PIPE_TIMEOUT, 30], status
        assert bool((out == 3.0).all())
        waits()
        assert torch.equal(call(), want)
        megamoe.check_block128_status()


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (2000, 3000, 4096), (600, 1500, 1024)])
def test_a_product_with_a_limit_that_may_run_out_is_right_or_reports_it(built_lib, waits, m, n, k):
    import megamoe
    g = torch.Generator().manual_seed(5)
    a, sa = ref.random_operand(g, m, k).cuda(), ref.random_scales(g, m, ref.blocks(k)).cuda()
    b, sb = ref.random_operand(g, n, k).cuda(), ref.random_scales(g, ref.blocks(n), ref.blocks(k)).cuda()
    want = megamoe.fp8_gemm_nt_block128((a, sa), (b, sb))
    for _ in range(3):
        waits(limit_ns=1)
        got = megamoe.fp8_gemm_nt_block128((a, sa), (b, sb))
        status = _read(built_lib, torch.cuda.current_stream())
        assert torch.equal(got, want) if status[0] == 0 else status[:2] == [PIPE_TIMEOUT, 20], status
        waits()
        assert torch.equal(megamoe.fp8_gemm_nt_block128((a, sa), (b, sb)), want)
        megamoe.check_block128_status()


def test_a_read_does_not_wait_for_reads_of_other_streams(built_lib):
    """While a read waits for its busy stream, another thread's read of an idle one returns."""
    import threading
    busy, idle = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    _read(built_lib, idle)
    with torch.cuda.stream(busy):
        torch.cuda._sleep(1_000_000_000)                             # half a second or more
    first = threading.Thread(target=_read, args=(built_lib, busy))
    first.start()
    others = [threading.Thread(target=_read, args=(built_lib, idle)) for _ in range(8)]
    for t in others:
        t.start()
    for t in others:
        t.join()
    assert first.is_alive() and not busy.query(), "the reads of the idle stream came back only with the busy one's"
    first.join()
