"""The block-scaled products and norms where a block of threads does several tiles or rows, each against its definition in 64 bits:
grouped tiles of 256 columns and of 128, with padding and bad blocks between them, and every kernel of the norm by the types that pick it."""
import pytest
import torch

import block128_ref as ref
from test_gpu_block128 import _assert_product, _norm_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu(built_lib):
    if not torch.cuda.is_available():
        pytest.fail("needs a CUDA device")


@pytest.fixture
def g():
    return torch.Generator().manual_seed(41)


def _turns(m_tiles, n):
    """Turns of the SMs with tiles of 128 and of 256 columns."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return -(-m_tiles * ref.blocks(n) // sms), -(-m_tiles * (-(-n // 256)) // sms)


def _mixed_layout(m_tiles, experts, g, bad=()):
    """Blocks of 128 rows of sorted experts, most full, some with few rows; every seventh is padding, those of `bad` have an expert that
    does not exist."""
    index = torch.full((m_tiles, 128), -1, dtype=torch.int32)
    for b in range(m_tiles):
        if b % 7 == 5:
            continue
        rows = 128 if b % 3 else int(torch.randint(1, 129, (1,), generator=g))
        index[b, :rows] = experts + 5 if b in bad else b * experts // m_tiles
    return index.view(-1)


def _check_grouped(g, m_tiles, n, k, experts, tiled, dtype, bad):
    import megamoe
    from deepgemm_b200 import _lib
    rows = 128 * m_tiles
    index = _mixed_layout(m_tiles, experts, g, bad)
    a, sa = ref.random_operand(g, rows, k).cuda(), ref.random_scales(g, rows, ref.blocks(k)).cuda()
    b, sb = ref.random_operand(g, experts, n, k).cuda(), ref.random_scales(g, experts, ref.blocks(n), ref.blocks(k)).cuda()
    d = torch.full((rows, n), 3.0, dtype=dtype, device="cuda")
    w = megamoe.pack_weights_tiled(b, "l2") if tiled else b
    megamoe.m_grouped_fp8_gemm_nt_contiguous_block128((a, sa), (w, sb), d, index.cuda())
    if bad:
        with pytest.raises(_lib.MegaMoeError, match="mixes experts"):
            megamoe.check_block128_status()
    else:
        megamoe.check_block128_status()
    valid = ((index >= 0) & (index < experts)).cuda()
    assert bool((d[~valid] == 3.0).all()), "padding and bad rows must be left as they were"
    for e in range(experts):
        m = index.cuda() == e
        want, bound = ref.product_and_bound(ref.by_row(a[m], sa[m]), ref.by_block(b[e], sb[e]))
        _assert_product(d[m], want, bound, f"expert {e}")


@pytest.mark.parametrize("m_tiles,n,k,tiled,dtype", [(40, 1920, 2048, True, torch.bfloat16), (40, 2050, 2064, False, torch.float32),
                                                     (75, 1024, 2176, True, torch.float32), (47, 1800, 2048, False, torch.bfloat16)])
@pytest.mark.parametrize("bad", [(), (11, 12, 30)])
def test_grouped_tiles_of_256_columns(g, m_tiles, n, k, tiled, dtype, bad):
    """Several tiles for each CTA: the rings of operands and scales go on from one expert's tile to the next, over blocks without work."""
    turns128, turns256 = _turns(m_tiles, n)
    assert turns128 * 7 >= turns256 * 10 and turns256 >= 2, "sizes that take the wide tile"
    _check_grouped(g, m_tiles, n, k, 6, tiled, dtype, bad)


@pytest.mark.parametrize("n,k,tiled", [(128, 1024, True), (100, 528, False)])
def test_grouped_tiles_of_128_columns_in_turns(g, n, k, tiled):
    m_tiles = 400
    turns128, turns256 = _turns(m_tiles, n)
    assert turns128 * 7 < turns256 * 10 and turns128 >= 2
    _check_grouped(g, m_tiles, n, k, 5, tiled, torch.bfloat16, (3, 200))


def test_product_of_a_prompt(g):
    """More than one turn of 256-wide tiles in the dense product, with a K that ends inside a block and columns inside a tile."""
    import megamoe
    m, n, k = 4000, 3400, 2000
    turns128, turns256 = _turns(ref.blocks(m), n)
    assert turns128 * 7 >= turns256 * 10 and turns256 >= 2
    a, sa = ref.random_operand(g, m, k).cuda(), ref.random_scales(g, m, ref.blocks(k)).cuda()
    b, sb = ref.random_operand(g, n, k).cuda(), ref.random_scales(g, ref.blocks(n), ref.blocks(k)).cuda()
    want, bound = ref.product_and_bound(ref.by_row(a, sa), ref.by_block(b, sb))
    for dtype in (torch.bfloat16, torch.float32):
        _assert_product(megamoe.fp8_gemm_nt_block128((a, sa), (b, sb), out_dtype=dtype), want, bound)


def check_norm(g, t, h, quant, yt, rt, wt, gt, gate):
    """norm_gate_residual of these types against 64 bits: gate None, "channel", "token" or "full" of type gt."""
    import megamoe
    y = (torch.randn((t, h), generator=g) * torch.exp(torch.randn((t, 1), generator=g))).to(yt).cuda()
    r = (torch.randn((t, h), generator=g) * 2).to(rt).cuda()
    post, pre = (1 + 0.3 * torch.randn(h, generator=g)).to(wt).cuda(), (0.3 * torch.randn(h, generator=g)).to(wt).cuda()
    shape = {"channel": (h,), "token": (t, 1), "full": (t, h), None: None}[gate]
    gate_t = None if shape is None else torch.randn(shape, generator=g).to(gt).cuda()
    alpha, eps, offset = 0.75, 1e-5, 1.0
    out = megamoe.norm_gate_residual(y, r, post_weight=post, gate=gate_t, residual_scale=alpha, pre_weight=pre, eps=eps, weight_offset=offset, quant=quant)
    want_r, mag, want_x, xmag = _norm_ref(y, r, post, gate_t, alpha, pre, eps, offset)
    # each value passes about ten roundings of 2^-24, the sums of squares 16 additions per thread and 10 levels across the block,
    # rsqrt is 2 units of the last place: 64 roundings cover them
    slack = 64 * 2.0 ** -24
    assert out.residual.dtype == rt and out.normed.dtype == (torch.float32 if rt == torch.float16 else torch.bfloat16)
    # (fp16 steps do not shrink below 2^-24: half of one is 2^-25)
    assert bool(((out.residual.double() - want_r).abs() <= slack * mag + ref.half_step(rt) * (want_r.abs() + slack * mag) + 2.0 ** -25).all())
    assert bool(((out.normed.double() - want_x).abs() <= slack * xmag + ref.half_step(out.normed.dtype) * (want_x.abs() + slack * xmag)).all())
    if quant is None:
        assert out.codes is None and out.scales is None
        return
    group = 128 if quant == "block128" else h
    u, top = ref.cast(want_x, group)
    xerr = slack * xmag
    group_err = torch.stack([xerr[:, j * group:(j + 1) * group].amax(1) for j in range(top.shape[1])], 1)
    assert bool(((out.scales.reshape(t, -1).double() * 448.0 - top).abs() <= group_err + 2.0 ** -22 * top).all())
    wide = lambda v: v.repeat_interleave(group, 1)[:, :h]   # noqa: E731
    u_err = (xerr + wide(group_err) * (u.abs() / 448.0)) * wide(448.0 / top) + 2.0 ** -22 * u.abs()
    assert bool(((out.codes.double() - u).abs() <= 0.5 * ref.e4m3_step(u.abs() + u_err) + u_err).all())


B, H, F = torch.bfloat16, torch.float16, torch.float32


# one row for each block of threads; several without, and with, the weights in shared memory; one and two vectors a thread; rows that fill
# no whole warp, and the longest ones
@pytest.mark.parametrize("t,h", [(1, 4096), (200, 4096), (700, 4096), (1300, 4096), (330, 1032), (5000, 1032), (9000, 264), (200, 16384), (400, 12296)])
@pytest.mark.parametrize("rt", [B, F])
@pytest.mark.parametrize("gate", [None, "channel", "token", "full"])
@pytest.mark.parametrize("quant", [None, "block128", "channelwise"])
def test_norm_with_fp32_weights_and_gate(g, t, h, rt, gate, quant):
    """y in bf16, weights and gate in fp32: the kernels whose types are known when they are compiled."""
    check_norm(g, t, h, quant, B, rt, F, F, gate)


@pytest.mark.parametrize("t,h", [(1, 4096), (700, 4096), (1300, 4096), (5000, 264), (301, 16384)])
@pytest.mark.parametrize("quant", [None, "block128", "channelwise"])
@pytest.mark.parametrize("yt,rt,wt,gt,gate", [(B, B, B, B, "channel"), (B, F, B, F, "full"), (B, H, F, F, "channel"), (H, H, H, H, "token"),
                                              (B, B, F, B, "channel"), (F, B, F, F, "token"), (B, B, B, B, None)])
def test_norm_of_many_rows_of_any_types(g, t, h, quant, yt, rt, wt, gt, gate):
    """Other types, which one kernel serves; several rows for each block of threads but in the first size."""
    check_norm(g, t, h, quant, yt, rt, wt, gt, gate)
