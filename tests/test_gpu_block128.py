"""Casts, products and norms with block scales on a B200, against their definitions in 64 bits."""
import math

import pytest
import torch

import block128_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module", autouse=True)
def _need_gpu(built_lib):
    if not torch.cuda.is_available():
        pytest.fail("needs a CUDA device")


@pytest.fixture
def g():
    return torch.Generator().manual_seed(7)


def _check_codes(q, u, exact):
    """Codes against the unrounded 448 x / top: half a step away at most, and equal to the nearest (ties to even) where the quotient
    is exact; otherwise the quotient itself is one rounding (2^-24) and one correction off, 2^-22 covers both."""
    err = (q.double() - u).abs()
    assert bool((err <= 0.5 * ref.e4m3_step(u) + 2.0 ** -22 * u.abs()).all()), float((err - 0.5 * ref.e4m3_step(u)).max())
    if exact:
        assert torch.equal(q.double(), ref.e4m3_of(u))


# ------------------------------------------------------------------------------------------------ casts
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 8), (1, 128), (3, 136), (5, 200), (2, 1024), (37, 4096), (300, 264)])
def test_cast_rows(g, dtype, rows, k):
    import megamoe
    x = (torch.randn((rows, k), generator=g) * torch.exp(2 * torch.randn((rows, 1), generator=g))).to(dtype)
    x[0, : min(k, 128)] *= 0.0                                    # a block of zeros: the smallest scale
    q, sf = megamoe.cast_to_fp8_block128(x.cuda())
    assert q.dtype == ref.E4M3 and q.shape == x.shape and sf.shape == (rows, ref.blocks(k))
    u, top = ref.cast(x.double(), 128)
    _check_codes(q.cpu(), u, exact=dtype != torch.float32)
    assert bool(((sf.cpu().double() * 448.0 / top - 1).abs() <= 2.0 ** -23).all())


def test_cast_ties_go_to_the_even_code():
    """16-bit values that lie exactly half way between two codes: the quotient has to be exact there."""
    import megamoe
    x = torch.zeros((4, 128), dtype=torch.bfloat16)
    for r, top in enumerate([448.0, 7.0, 1.75, 224.0]):           # scales that are powers of two
        x[r, 0] = top
        x[r, 1:65] = torch.arange(64).bfloat16() * (top / 448.0) * 0.5
        x[r, 65:97] = -(torch.arange(32).bfloat16() + 0.5) * (top / 448.0)
    g = torch.Generator().manual_seed(0)
    y = torch.randint(-127, 128, (512, 128), generator=g).bfloat16()   # small integers over small integers
    x = torch.cat([x, y])
    q, _ = megamoe.cast_to_fp8_block128(x.cuda())
    u, _ = ref.cast(x.double(), 128)
    assert torch.equal(q.cpu().double(), ref.e4m3_of(u))


def test_cast_extreme_values():
    import megamoe
    x = torch.zeros((6, 256), dtype=torch.float32)
    x[0, 0] = 3.0e38; x[0, 1] = -1.5e38
    x[1, 0] = 1e-45; x[1, 200] = 1e-5
    x[2, 3] = math.inf
    x[3, 4] = math.nan
    x[4, 130] = -math.inf
    x[5] = 65504.0
    q, sf = (t.cpu() for t in megamoe.cast_to_fp8_block128(x.cuda()))
    assert q[0, 0].item() == 448.0 and q[0, 1].item() == -224.0 and math.isfinite(sf[0, 0].item())
    assert bool((q[1].double() == ref.e4m3_of(ref.cast(x[1:2].double(), 128)[0])[0]).all())
    for row, block in ((2, 0), (3, 0), (4, 1)):                    # a value that is not finite shows in its block and only there
        own = slice(128 * block, 128 * block + 128)
        assert not math.isfinite(sf[row, block].item()) and bool(torch.isnan(q[row, own].float()).all())
        other = slice(128 * (1 - block), 128 * (1 - block) + 128)
        assert math.isfinite(sf[row, 1 - block].item()) and bool((q[row, other].float() == 0).all())
    assert bool((q[5].float() == 448.0).all())


def test_cast_strides_shapes_and_empty(g):
    import megamoe
    base = torch.randn((9, 1000), generator=g).bfloat16().cuda()
    for x in (base[:, 8:520], base[:, 3:515], base[::2, :512], base.t()[:512].t(), base[:, :512].reshape(3, 3, 512)):
        q, sf = megamoe.cast_to_fp8_block128(x)
        want, wsf = megamoe.cast_to_fp8_block128(x.contiguous().clone())
        assert q.shape == x.shape and torch.equal(q.view(torch.uint8), want.view(torch.uint8)) and torch.equal(sf, wsf)
    q, sf = megamoe.cast_to_fp8_block128(base[:0])
    assert q.shape == (0, 1000) and sf.shape == (0, 8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 8), (128, 128), (130, 136), (3, 300, 264), (2, 256, 512)])
def test_cast_weights(g, dtype, shape):
    import megamoe
    w = torch.randn(shape, generator=g).to(dtype)
    q, sf = megamoe.cast_weight_to_fp8_block128(w.cuda())
    n, k = shape[-2:]
    assert sf.shape == (*shape[:-2], ref.blocks(n), ref.blocks(k))
    q, sf, w = q.cpu().reshape(-1, n, k), sf.cpu().reshape(-1, ref.blocks(n), ref.blocks(k)), w.reshape(-1, n, k)
    for e in range(w.shape[0]):
        for i in range(ref.blocks(n)):
            for j in range(ref.blocks(k)):
                part = w[e, 128 * i:128 * i + 128, 128 * j:128 * j + 128].double()
                u, top = ref.cast(part.reshape(1, -1), part.numel())
                _check_codes(q[e, 128 * i:128 * i + 128, 128 * j:128 * j + 128].reshape(1, -1), u, exact=dtype != torch.float32)
                assert abs(sf[e, i, j].item() * 448.0 / top.item() - 1) <= 2.0 ** -23


# ------------------------------------------------------------------------------------------------ products
def _assert_product(out, want, bound, label=""):
    tol = bound + ref.half_step(out.dtype) * (want.abs() + bound)
    err = (out.double() - want).abs()
    assert bool((err <= tol).all()), f"{label}: off by {float((err - tol).max())} more than allowed"


def _operands(g, m, n, k, e=None):
    a, sa = ref.random_operand(g, m, k), ref.random_scales(g, m, ref.blocks(k))
    lead = () if e is None else (e,)
    b, sb = ref.random_operand(g, *lead, n, k), ref.random_scales(g, *lead, ref.blocks(n), ref.blocks(k))
    return (a, sa), (b, sb)


def _cuda(pair):
    return tuple(t.cuda() for t in pair)


@pytest.mark.parametrize("m,n,k", [
    (1, 1, 16), (1, 128, 128), (7, 8, 144), (128, 128, 256), (129, 130, 512), (300, 257, 1040), (1, 4096, 4096), (77, 256, 2048),
    (33, 1000, 640), (600, 1500, 96), (2500, 2050, 272), (130, 127, 4096), (2049, 2304, 128),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_dense_product(g, m, n, k, dtype):
    import megamoe
    a, b = _operands(g, m, n, k)
    out = megamoe.fp8_gemm_nt_block128(_cuda(a), _cuda(b), out_dtype=dtype)
    assert out.dtype == dtype and out.shape == (m, n)
    want, bound = ref.product_and_bound(ref.by_row(*_cuda(a)), ref.by_block(*_cuda(b)))
    _assert_product(out, want, bound)
    megamoe.check_block128_status()


def test_dense_product_strided_and_in_place(g):
    """Rows of a and of the output as slices of wider tensors; what lies between the output's rows stays as it was."""
    import megamoe
    m, n, k = 150, 300, 384
    (a, sa), (b, sb) = _operands(g, m, n, k)
    wide_a = torch.zeros((m, k + 64), dtype=torch.uint8, device="cuda").view(ref.E4M3)
    wide_a[:, 16:16 + k] = a.cuda()
    wide_sa = torch.zeros((m, ref.blocks(k) + 3), device="cuda")
    wide_sa[:, 2:2 + ref.blocks(k)] = sa.cuda()
    want, bound = ref.product_and_bound(ref.by_row(a, sa), ref.by_block(b, sb))
    for dtype, offset, pitch in ((torch.bfloat16, 0, n), (torch.bfloat16, 3, n + 13), (torch.float32, 16, n + 20), (torch.bfloat16, 16, 512)):
        wide = torch.full((m, pitch + 16), 5.0, dtype=dtype, device="cuda")
        out = wide[:, offset:offset + n]
        got = megamoe.fp8_gemm_nt_block128((wide_a[:, 16:16 + k], wide_sa[:, 2:2 + ref.blocks(k)]), _cuda((b, sb)), out=out)
        assert got.data_ptr() == out.data_ptr()
        _assert_product(out.cpu(), want, bound)
        assert bool((wide[:, :offset] == 5).all()) and bool((wide[:, offset + n:] == 5).all())


def test_dense_product_empty_and_repeatable(g):
    import megamoe
    a, b = _operands(g, 5, 700, 2048)
    assert megamoe.fp8_gemm_nt_block128((a[0][:0].cuda(), a[1][:0].cuda()), _cuda(b)).shape == (0, 700)
    outs = [megamoe.fp8_gemm_nt_block128(_cuda(a), _cuda(b), out_dtype=torch.float32) for _ in range(4)]
    assert all(torch.equal(o, outs[0]) for o in outs)


def test_product_passes_nan_and_infinity_on(g):
    """A scale that is not finite (the cast's mark for a bad block) reaches its rows, and no others."""
    import megamoe
    (a, sa), (b, sb) = _operands(g, 40, 256, 512)
    sa[3, 1] = math.nan
    sa[17, 2] = math.inf
    out = megamoe.fp8_gemm_nt_block128(_cuda((a, sa)), _cuda((b, sb))).cpu()
    bad = ~torch.isfinite(out).all(1)
    assert bad.nonzero()[:, 0].tolist() == [3, 17]


def _layout(counts):
    index = []
    for e, c in enumerate(counts):
        index += [e] * c + [-1] * (-c % 128)
    return torch.tensor(index + [-1] * 128, dtype=torch.int32)


@pytest.mark.parametrize("n,k,tiled", [(512, 256, False), (384, 512, True), (130, 144, False), (1000, 640, False), (2048, 1024, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_grouped_product(g, n, k, tiled, dtype):
    import megamoe
    counts = [200, 0, 128, 1, 77, 300]
    index = _layout(counts)
    rows = index.numel()
    (a, sa), (b, sb) = _operands(g, rows, n, k, e=len(counts))
    d = torch.full((rows, n), 3.0, dtype=dtype, device="cuda")
    w = megamoe.pack_weights_tiled(b.cuda(), "l2") if tiled else b.cuda()
    megamoe.m_grouped_fp8_gemm_nt_contiguous_block128(_cuda((a, sa)), (w, sb.cuda()), d, index.cuda(), check=True)
    d = d.cpu()
    assert bool((d[index < 0] == 3.0).all()), "padding rows must be left as they were"
    for e in range(len(counts)):
        m = index == e
        want, bound = ref.product_and_bound(ref.by_row(a[m], sa[m]), ref.by_block(b[e], sb[e]))
        _assert_product(d[m], want, bound, f"expert {e}")


def test_grouped_product_reports_a_mixed_block(g):
    import megamoe
    from deepgemm_b200 import _lib
    index = torch.full((256,), 0, dtype=torch.int32)
    index[128:] = 1
    index[200] = 0
    a, b = _operands(g, 256, 128, 128, e=2)
    d = torch.full((256, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(_lib.MegaMoeError, match="mixes experts"):
        megamoe.m_grouped_fp8_gemm_nt_contiguous_block128(_cuda(a), _cuda(b), d, index.cuda(), check=True)
    assert bool((d[200] == 3.0).all()) and bool((d[199] != 3.0).any())
    megamoe.check_block128_status()                                  # reported once
    index[200] = 7                                                    # an expert that does not exist, inside a block and as a block's first
    index[:128] = 9
    with pytest.raises(_lib.MegaMoeError, match="mixes experts"):
        megamoe.m_grouped_fp8_gemm_nt_contiguous_block128(_cuda(a), _cuda(b), d.fill_(3.0), index.cuda(), check=True)
    assert bool((d[:128] == 3.0).all()) and bool((d[200] == 3.0).all())


# ------------------------------------------------------------------------------------------------ norms
def _norm_ref(y, r, post, gate, alpha, pre, eps, offset):
    """64-bit values, and magnitudes that the 32-bit errors are relative to."""
    r = r.double()
    mag = r.abs()
    if y is not None:
        y = y.double()
        if post is not None:
            y = y / torch.sqrt(y.square().mean(1, keepdim=True) + eps) * (post.double() + offset)
        if gate is not None:
            y = y * gate.double()
        mag = abs(alpha) * mag + y.abs()
        r = alpha * r + y
    if pre is None:
        return r, mag, None, None
    n = 1 / torch.sqrt(r.square().mean(1, keepdim=True) + eps)
    # r' is off by a few roundings of its terms; n by half of that of the mean of squares, which the largest terms dominate
    xmag = mag * n * (pre.double() + offset).abs() + (r * n * (pre.double() + offset)).abs() * (mag.square().sum(1, keepdim=True) / r.square().sum(1, keepdim=True).clamp(min=1e-300)).sqrt()
    return r, mag, r * n * (pre.double() + offset), xmag


@pytest.mark.parametrize("t,h", [(1, 8), (3, 136), (1, 4096), (5, 1000), (700, 512), (2, 8200), (3, 16384)])
@pytest.mark.parametrize("quant", [None, "block128", "channelwise"])
@pytest.mark.parametrize("yt,rt,wt,gate", [(torch.bfloat16, torch.bfloat16, torch.float32, "channel"), (torch.float32, torch.float32, torch.bfloat16, "token"),
                                           (torch.float16, torch.float32, torch.float32, "full"), (torch.bfloat16, torch.float16, torch.float16, None)])
def test_norm(g, t, h, quant, yt, rt, wt, gate):
    import megamoe
    y = (torch.randn((t, h), generator=g) * torch.exp(torch.randn((t, 1), generator=g))).to(yt)
    r = (torch.randn((t, h), generator=g) * 2).to(rt)
    post, pre = (1 + 0.3 * torch.randn(h, generator=g)).to(wt), (0.3 * torch.randn(h, generator=g)).to(wt)
    shape = {"channel": (h,), "token": (t, 1), "full": (t, h), None: None}[gate]
    gate_t = None if shape is None else torch.randn(shape, generator=g).to(rt)
    alpha, eps, offset = 0.75, 1e-5, 1.0
    out = megamoe.norm_gate_residual(y.cuda(), r.cuda(), post_weight=post.cuda(), gate=None if gate_t is None else gate_t.cuda(), residual_scale=alpha,
                                     pre_weight=pre.cuda(), eps=eps, weight_offset=offset, quant=quant)
    want_r, mag, want_x, xmag = _norm_ref(y, r, post, gate_t, alpha, pre, eps, offset)
    # each value passes about ten roundings of 2^-24, the sums of squares 16 additions per thread and 10 levels across the block,
    # rsqrt is 2 units of the last place: 64 roundings cover them
    slack = 64 * 2.0 ** -24
    got_r, got_x = out.residual.cpu(), out.normed.cpu()
    assert got_r.dtype == rt and got_x.dtype == (torch.float32 if rt == torch.float16 else torch.bfloat16)
    assert bool(((got_r.double() - want_r).abs() <= slack * mag + ref.half_step(rt) * (want_r.abs() + slack * mag) + 2.0 ** -25).all())
    assert bool(((got_x.double() - want_x).abs() <= slack * xmag + ref.half_step(got_x.dtype) * (want_x.abs() + slack * xmag)).all())
    if quant is None:
        assert out.codes is None and out.scales is None
        return
    group = 128 if quant == "block128" else h
    u, top = ref.cast(want_x, group)
    sf = out.scales.cpu().reshape(t, -1)
    xerr = slack * xmag
    group_err = torch.stack([xerr[:, j * group:(j + 1) * group].amax(1) for j in range(top.shape[1])], 1)
    assert bool(((sf.double() * 448.0 - top).abs() <= group_err + 2.0 ** -22 * top).all())
    rel = (448.0 / top).repeat_interleave(group, 1)[:, :h]
    u_err = (xerr + group_err.repeat_interleave(group, 1)[:, :h] * (u.abs() / 448.0)) * rel + 2.0 ** -22 * u.abs()
    assert bool(((out.codes.cpu().double() - u).abs() <= 0.5 * ref.e4m3_step(u.abs() + u_err) + u_err).all())


def test_norm_optional_parts(g):
    import megamoe
    t, h = 9, 640
    y, r = torch.randn((t, h), generator=g).cuda().bfloat16(), torch.randn((t, h), generator=g).cuda()
    pre = torch.rand(h, generator=g).cuda() + 0.5
    # before the first block: only the norm, the residual comes back as it is
    out = megamoe.norm_gate_residual(None, r, pre_weight=pre)
    assert out.residual is r and torch.allclose(out.normed.float(), (r * torch.rsqrt(r.square().mean(1, keepdim=True) + 1e-6) * pre), rtol=2 ** -7, atol=1e-6)
    # after the last one: only the sum
    out = megamoe.norm_gate_residual(y, r, residual_scale=0.5)
    assert out.normed is None and torch.equal(out.residual, torch.add(y.float(), r, alpha=0.5))
    # codes without the values
    out = megamoe.norm_gate_residual(y, r, pre_weight=pre, quant="block128", out_normed=False)
    full = megamoe.norm_gate_residual(y, r, pre_weight=pre, quant="block128")
    assert out.normed is None and torch.equal(out.codes.view(torch.uint8), full.codes.view(torch.uint8)) and torch.equal(out.scales, full.scales)
    # rows of zeros: eps alone under the root
    out = megamoe.norm_gate_residual(torch.zeros_like(y), torch.zeros_like(r), post_weight=pre, pre_weight=pre, quant="channelwise")
    assert bool((out.residual == 0).all()) and bool((out.normed == 0).all()) and bool((out.codes.float() == 0).all())
    # no tokens
    out = megamoe.norm_gate_residual(y[:0], r[:0], pre_weight=pre, quant="block128")
    assert out.codes.shape == (0, h) and out.scales.shape == (0, 5)


def test_norm_strides(g):
    import megamoe
    t, h = 6, 256
    wide = torch.randn((t, 3 * h + 8), generator=g).cuda().bfloat16()
    pre = torch.ones(h, device="cuda")
    gate = torch.randn((t, 2 * h), generator=g).cuda()
    for y, r, ga in ((wide[:, :h], wide[:, h:2 * h], gate[:, :h]), (wide[:, 1:h + 1], wide[:, h + 3:2 * h + 3], gate[:, 5:5 + h]),
                     (wide[:, :2 * h:2], wide[:, 8:h + 8], gate[:, h:h + 1]), (wide[:, :h], wide[:, h:2 * h], gate[0, 1:h + 1])):
        a = megamoe.norm_gate_residual(y, r, post_weight=pre, gate=ga, pre_weight=pre, quant="block128")
        b = megamoe.norm_gate_residual(y.contiguous().clone(), r.contiguous().clone(), post_weight=pre, gate=ga.contiguous().clone(), pre_weight=pre, quant="block128")
        for u, v in zip(a, b):
            assert torch.equal(u.view(torch.uint8) if u.dtype == ref.E4M3 else u, v.view(torch.uint8) if v.dtype == ref.E4M3 else v)


def test_norm_feeds_the_channelwise_layer(g):
    """Codes and scales written into the layer's input views equal the layer's own cast of the same values."""
    import megamoe
    t, h = 40, 512
    sb = megamoe.get_symm_buffer_for_mega_moe(None, 8, 64, 2, h, 256)
    y, r = torch.randn((t, h), generator=g).cuda().bfloat16(), torch.randn((t, h), generator=g).cuda().bfloat16()
    pre = torch.rand(h, generator=g).cuda() + 0.5
    out = megamoe.norm_gate_residual(y, r, post_weight=pre, pre_weight=pre, quant="channelwise", out_codes=sb.x[:t], out_scales=sb.x_sf[:t])
    assert out.codes.data_ptr() == sb.x.data_ptr()
    # the layer's cast takes bf16: its scale differs by the rounding of the largest value
    q, s = megamoe.cast_to_fp8_channelwise(out.normed)
    assert bool(((sb.x_sf[:t] / s - 1).abs() <= 2.0 ** -7).all())
    # the codes are of the unrounded x: |code s - x| <= 2^-4 |x| + 2^-10 s (half a step, at least half of the smallest one), the bf16 output
    # is within 2^-8 |x| of x, so |x| <= |normed| (1 + 2^-7) and together (2^-4 + 2^-8)(1 + 2^-7) |normed| + 2^-10 s
    v = out.normed.float()
    err = (sb.x[:t].float() * sb.x_sf[:t, None] - v).abs()
    assert bool((err <= (2.0 ** -4 + 2.0 ** -8) * (1 + 2.0 ** -7) * v.abs() + 2.0 ** -10 * (1 + 2.0 ** -7) * s[:, None]).all())
    sb.destroy()
