"""The block-scaled operators as a program uses them: one after the other, captured and replayed, on several streams, on tensors
whose rows lie more than 2^31 elements apart."""
import pytest
import torch

import block128_ref as ref
from test_gpu_block128 import _assert_product, _norm_ref, test_norm as _check_norm
from test_gpu_few_tokens import assert_layer, choose, layer64, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu(built_lib):
    if not torch.cuda.is_available():
        pytest.fail("needs a CUDA device")


@pytest.fixture
def g():
    return torch.Generator().manual_seed(23)


def _bits(t):
    return t.view(torch.uint8) if t.dtype == ref.E4M3 else t


class Block:
    """Norm, experts beside a shared projection, norm: what a decoder layer runs behind its attention."""

    def __init__(self, g, h=512, i=256, e=8, k=2):
        import megamoe
        _, self.w1, self.w2 = make(g, 1, e, h, i)
        self.l1 = (megamoe.pack_weights_tiled(self.w1[0].cuda(), "l1"), self.w1[1].cuda())
        self.l2 = (megamoe.pack_weights_tiled(self.w2[0].cuda(), "l2"), self.w2[1].cuda())
        self.shared = tuple(t.cuda() for t in megamoe.cast_weight_to_fp8_block128((torch.randn((h, h), generator=g) / h ** 0.5).cuda()))
        self.router = torch.randn((h, e), generator=g).cuda() / h ** 0.5
        self.pre, self.post = (torch.rand(h, generator=g).cuda() + 0.5 for _ in range(2))
        self.k = k

    def __call__(self, r):
        import megamoe
        first = megamoe.norm_gate_residual(None, r, pre_weight=self.pre, quant="block128")
        logits = first.normed.float() @ self.router
        x = (first.codes, first.scales)
        routed = megamoe.fp8_moe_few_tokens(x, self.l1, self.l2, router_logits=logits, num_topk=self.k)
        both = megamoe.fp8_gemm_nt_block128(x, self.shared)
        last = megamoe.norm_gate_residual(routed, r, post_weight=self.post, residual_scale=0.5, pre_weight=self.pre, quant="block128")
        dense = megamoe.cast_to_fp8_block128(last.normed)
        return dict(codes=first.codes, scales=first.scales, normed=first.normed, logits=logits, routed=routed, both=both, residual=last.residual,
                    normed2=last.normed, codes2=last.codes, dense=dense[0], dense_scales=dense[1])


@pytest.mark.parametrize("t", [1, 9, 150])
def test_one_after_the_other(g, t):
    """Every operator against its formula, on what the one before it gave."""
    import megamoe
    block = Block(g)
    r = torch.randn((t, 512), generator=g).cuda()
    out = {n: v.cpu() for n, v in block(r).items()}
    megamoe.check_block128_status()
    xv = ref.by_row(out["codes"], out["scales"])
    idx, w = choose(out["logits"], 2)
    y, bound = layer64_of_codes(out["codes"], out["scales"], block.w1, block.w2, idx, w)
    assert_layer(out["routed"], y, bound)
    want, bound = ref.product_and_bound(xv, ref.by_block(block.shared[0].cpu(), block.shared[1].cpu()))
    _assert_product(out["both"], want, bound)
    want_r, mag, want_x, xmag = _norm_ref(out["routed"], r.cpu(), block.post.cpu(), None, 0.5, block.pre.cpu(), 1e-6, 0.0)
    slack = 64 * 2.0 ** -24
    assert bool(((out["residual"].double() - want_r).abs() <= slack * mag + 2.0 ** -24 * want_r.abs() * 2).all())
    assert bool(((out["normed2"].double() - want_x).abs() <= slack * xmag + 2.0 ** -8 * (want_x.abs() + slack * xmag)).all())
    u, _ = ref.cast(out["normed2"].double(), 128)
    assert bool(((out["dense"].double() - u).abs() <= 0.5 * ref.e4m3_step(u) + 2.0 ** -22 * u.abs()).all())


def layer64_of_codes(q, sf, w1, w2, idx, w):
    """layer64 on rows that are codes already: a bf16 row whose cast gives these codes does not always exist, so the cast is stepped over."""
    cast, first = ref.cast, []

    def once(x, group):
        if not first:
            first.append(1)
            return q.double(), sf.double() * 448
        return cast(x, group)
    ref.cast = once
    try:
        return layer64(q.double(), w1, w2, idx, w)
    finally:
        ref.cast = cast


def test_captured_and_replayed(g):
    """Two graphs of the same operators, replayed on new inputs and beside one another, give the bits of plain calls."""
    block = Block(g)
    graphs = []
    for t in (3, 70):
        r = torch.randn((t, 512), generator=g).cuda()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block(r)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block(r)
        graphs.append((graph, r, out, torch.cuda.Stream()))
    for turn in range(4):
        want = []
        for graph, r, out, _ in graphs:
            r.copy_(torch.randn(r.shape, generator=g))
            want.append({n: v.clone() for n, v in block(r).items()})
        torch.cuda.synchronize()
        for graph, r, out, stream in graphs:
            with torch.cuda.stream(stream):
                for _ in range(5):
                    graph.replay()
        torch.cuda.synchronize()
        for (graph, r, out, _), w in zip(graphs, want):
            for name in w:
                assert torch.equal(_bits(out[name]), _bits(w[name])), (turn, name)


def test_calls_on_several_streams_at_once(g):
    """Layers, split products and casts of three streams share the SMs; each gives what it gives alone."""
    import megamoe
    block = Block(g, h=1024, i=512, e=16, k=4)
    inputs = [torch.randn((t, 1024), generator=g).cuda() for t in (1, 20, 130)]
    want = [{n: v.clone() for n, v in block(r).items()} for r in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    got = [[] for _ in inputs]
    for _ in range(20):
        for k, (r, s) in enumerate(zip(inputs, streams)):
            with torch.cuda.stream(s):
                got[k].append(block(r))
    torch.cuda.synchronize()
    megamoe.check_block128_status()
    for k, w in enumerate(want):
        for out in got[k]:
            for name in w:
                assert torch.equal(_bits(out[name]), _bits(w[name])), (k, name)


COUNTS = [3, 60, 128, 1, 0, 33, 200, 49, 97, 5]


@pytest.mark.parametrize("h,i", [(512, 256), (128, 640), (1280, 128)])
def test_layer_with_experts_of_every_size(g, h, i):
    """Blocks of a row, of a few and of 128 behind one another, so that warps without rows stand beside warps that have some."""
    import megamoe
    t, e = sum(COUNTS), len(COUNTS)
    x, w1, w2 = make(g, t, e, h, i)
    idx = torch.repeat_interleave(torch.arange(e), torch.tensor(COUNTS))[torch.randperm(t, generator=g)][:, None]
    w = torch.rand((t, 1), generator=g) + 0.5
    out = megamoe.fp8_moe_few_tokens(x.cuda(), (w1[0].cuda(), w1[1].cuda()), (w2[0].cuda(), w2[1].cuda()), topk_idx=idx.cuda(), topk_weights=w.cuda())
    megamoe.check_block128_status()
    assert_layer(out, *layer64(x, w1, w2, idx, w))


@pytest.mark.parametrize("layout", ["native", "tiled"])
@pytest.mark.parametrize("h,i", [(128, 640), (1280, 128), (640, 640)])
def test_layer_with_more_tiles_than_shares(g, h, i, layout):
    """512 experts, so many tiles that a chunk is a tile in one product, in the other one or in both; four weights stand for all."""
    import megamoe
    t, e = 512, 512
    x, w1, w2 = make(g, t, 4, h, i)
    idx = torch.stack([torch.randperm(e, generator=g), torch.full((t,), 7)], 1)
    idx[::3, 1] = torch.arange(0, t, 3) // 5
    w = torch.rand((t, 2), generator=g) + 0.5
    many = [v.cuda().repeat(e // 4, 1, 1) for v in (w1[0].view(torch.uint8), w1[1], w2[0].view(torch.uint8), w2[1])]
    q1, q2 = many[0].view(ref.E4M3), many[2].view(ref.E4M3)
    if layout == "tiled":
        q1, q2 = megamoe.pack_weights_tiled(q1, "l1"), megamoe.pack_weights_tiled(q2, "l2")
    out = megamoe.fp8_moe_few_tokens(x.cuda(), (q1, many[1]), (q2, many[3]), topk_idx=idx.cuda(), topk_weights=w.cuda())
    megamoe.check_block128_status()
    assert_layer(out, *layer64(x, w1, w2, idx % 4, w))


def test_rows_behind_2_31_elements(g):
    import megamoe
    far = 2 ** 31 + 2 ** 20                                        # elements from one row to the next, a multiple of 32
    h = 256
    # casts and norms
    wide = torch.empty(far + h, dtype=torch.bfloat16, device="cuda")
    x = wide.as_strided((2, h), (far, 1))
    x.copy_(torch.randn((2, h), generator=g))
    near = x.clone()
    for a, b in zip(megamoe.cast_to_fp8_block128(x), megamoe.cast_to_fp8_block128(near)):
        assert torch.equal(_bits(a), _bits(b))
    pre = torch.ones(h, device="cuda")
    for a, b in zip(megamoe.norm_gate_residual(x, x, gate=x, pre_weight=pre, quant="block128"),
                    megamoe.norm_gate_residual(near, near, gate=near, pre_weight=pre, quant="block128")):
        assert torch.equal(_bits(a), _bits(b))
    # the layer's x
    _, w1, w2 = make(g, 1, 2, h, 128)
    l1, l2 = (w1[0].cuda(), w1[1].cuda()), (w2[0].cuda(), w2[1].cuda())
    logits = torch.zeros((2, 2), device="cuda")
    assert torch.equal(megamoe.fp8_moe_few_tokens(x, l1, l2, router_logits=logits, num_topk=2), megamoe.fp8_moe_few_tokens(near, l1, l2, router_logits=logits, num_topk=2))
    # operand and output of a product: rows of a far apart as bytes, of the output as elements
    a, sa = megamoe.cast_to_fp8_block128(near)
    b = megamoe.cast_weight_to_fp8_block128(torch.randn((136, h), generator=g).cuda())
    want = megamoe.fp8_gemm_nt_block128((a, sa), b)
    far_a = wide.view(torch.uint8).view(ref.E4M3).as_strided((2, h), (far, 1))
    far_a.view(torch.uint8).copy_(a.view(torch.uint8))
    assert torch.equal(megamoe.fp8_gemm_nt_block128((far_a, sa), b), want)
    out = wide.as_strided((2, 136), (far, 1))
    assert torch.equal(megamoe.fp8_gemm_nt_block128((a, sa), b, out=out), want)


def test_more_than_2_31_elements(g):
    """The last rows of a cast and of a product whose operands or outputs hold more than 2^31 elements."""
    import megamoe
    k, rows = 2048, 2 ** 20 + 130
    x = torch.empty((rows, k), dtype=torch.bfloat16, device="cuda")
    x[:100].normal_()
    x[-100:].normal_()
    q, sf = megamoe.cast_to_fp8_block128(x)
    for part in (slice(0, 100), slice(rows - 100, rows)):
        q1, sf1 = megamoe.cast_to_fp8_block128(x[part])
        assert torch.equal(_bits(q[part]), _bits(q1)) and torch.equal(sf[part], sf1)
    del x
    b = megamoe.cast_weight_to_fp8_block128(torch.randn((2064, k), generator=g).cuda())
    out = megamoe.fp8_gemm_nt_block128((q, sf), b)
    assert out.numel() > 2 ** 31
    want, bound = ref.product_and_bound(ref.by_row(q[-100:], sf[-100:]), ref.by_block(*b))
    _assert_product(out[-100:], want, bound)


def test_fp32_rows_that_begin_at_any_16_bytes(g):
    """Rows of four more values than a multiple of eight: aligned for 16-byte loads, so they are read where they are."""
    import megamoe
    wide = torch.randn((7, 5 * 64 + 4), generator=g).cuda()
    x, near = wide[:, 4:4 + 64], wide[:, 4:4 + 64].contiguous()
    for a, b in zip(megamoe.cast_to_fp8_block128(x), megamoe.cast_to_fp8_block128(near)):
        assert torch.equal(_bits(a), _bits(b))
    y, r, gate, pre = wide[:, 68:132], x, wide[:, 200:264], torch.ones(64, device="cuda")
    for a, b in zip(megamoe.norm_gate_residual(y, r, gate=gate, pre_weight=pre, quant="channelwise"),
                    megamoe.norm_gate_residual(y.contiguous(), near, gate=gate.contiguous(), pre_weight=pre, quant="channelwise")):
        assert torch.equal(_bits(a), _bits(b))


@pytest.mark.parametrize("t,h", [(1300, 4096), (1250, 4104), (301, 16384), (2500, 2056)])
@pytest.mark.parametrize("rt,gate,quant", [(torch.bfloat16, "channel", "block128"), (torch.float32, "channel", "channelwise"), (torch.bfloat16, "token", None),
                                           (torch.bfloat16, None, "channelwise"), (torch.float32, "full", "block128")])
def test_norm_of_many_rows(g, t, h, rt, gate, quant):
    """Several rows for each block of threads: weights are worked out once, with the gate if it is the same for all rows."""
    _check_norm(g, t, h, quant, torch.bfloat16, rt, torch.float32, gate)


def test_norm_of_many_rows_without_its_parts(g):
    import megamoe
    t, h = 1300, 4096
    y, r = torch.randn((t, h), generator=g).cuda().bfloat16(), torch.randn((t, h), generator=g).cuda().bfloat16()
    pre, gate = torch.rand(h, generator=g).cuda() + 0.5, torch.randn(h, generator=g).cuda()
    # (rows alone take the other path: one row for each block of threads)
    for kw in (dict(pre_weight=pre), dict(gate=gate), dict(gate=gate, pre_weight=pre, weight_offset=1.0), dict(post_weight=pre)):
        many, few = megamoe.norm_gate_residual(y, r, **kw), megamoe.norm_gate_residual(y[:9], r[:9], **kw)
        for a, b in zip(many, few):
            assert (a is None) == (b is None)
            if a is not None:           # the same roundings but for the order of the sum of squares and of weight and gate
                assert bool(((a[:9].float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 2.0 ** -8 * r[:9].float().abs()).all())
    first = megamoe.norm_gate_residual(None, r, pre_weight=pre)
    want, _, x, xmag = _norm_ref(None, r.cpu(), None, None, 1.0, pre.cpu(), 1e-6, 0.0)
    assert first.residual is r and bool(((first.normed.cpu().double() - x).abs() <= 64 * 2.0 ** -24 * xmag + 2.0 ** -8 * (x.abs() + 64 * 2.0 ** -24 * xmag)).all())


def test_captured_behind_copies_and_other_streams(g):
    """First kernel of a graph, or behind a copy, a memset or an event of another stream: every kind of edge before a call."""
    import megamoe
    block = Block(g)
    host = torch.randn((6, 512), generator=g).pin_memory()
    r, other = torch.zeros((6, 512), device="cuda"), torch.zeros((6, 512), device="cuda")
    raw = torch.zeros((6, 512), dtype=torch.uint8, device="cuda").view(ref.E4M3)
    block(r)
    q0, s0 = megamoe.cast_to_fp8_block128(r)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        first = megamoe.cast_to_fp8_block128(r)                     # the graph's first node
        other.copy_(r)                                              # device to device
        second = megamoe.cast_to_fp8_block128(other)
        r.copy_(host, non_blocking=True)                            # host to device
        out = block(r)
        raw.view(torch.uint8).zero_()
        product = megamoe.fp8_gemm_nt_block128((raw, s0), block.shared)
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            beside = megamoe.norm_gate_residual(out["routed"], r, pre_weight=block.pre, quant="block128")
        main.wait_stream(side)
        joined = megamoe.fp8_gemm_nt_block128((beside.codes, beside.scales), block.shared)
    for _ in range(3):
        before = torch.randn((6, 512), generator=g)
        r.copy_(before)
        host.copy_(torch.randn((6, 512), generator=g))
        raw.view(torch.uint8).fill_(0x38)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        q, s = megamoe.cast_to_fp8_block128(before.cuda())
        for a in (first, second):
            assert torch.equal(_bits(a[0]), _bits(q)) and torch.equal(a[1], s)
        want = block(host.cuda())
        for name in want:
            assert torch.equal(_bits(out[name]), _bits(want[name])), name
        assert bool((product == 0).all())
        n = megamoe.norm_gate_residual(want["routed"], host.cuda(), pre_weight=block.pre, quant="block128")
        assert torch.equal(_bits(beside.codes), _bits(n.codes))
        assert torch.equal(joined, megamoe.fp8_gemm_nt_block128((n.codes, n.scales), block.shared))
    megamoe.check_block128_status()
