"""The mixture-of-experts layer for a few tokens on a B200, against its definition in 64 bits."""
import math

import pytest
import torch

import block128_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu(built_lib):
    if not torch.cuda.is_available():
        pytest.fail("needs a CUDA device")


@pytest.fixture
def g():
    return torch.Generator().manual_seed(11)


def make(g, t, e, h, i):
    """Weights in the native layout, with the popular spread of scales; x with a row of zeros if there is room for one."""
    w1, s1 = ref.random_operand(g, e, 2 * i, h), ref.random_scales(g, e, 2 * i // 128, h // 128) * (1.2 / h ** 0.5)
    w2, s2 = ref.random_operand(g, e, h, i), ref.random_scales(g, e, h // 128, i // 128) * (1.2 / i ** 0.5)
    x = (torch.randn((t, h), generator=g) * torch.exp(0.5 * torch.randn((t, 1), generator=g))).bfloat16()
    if t > 4:
        x[3] = 0
    return x, (w1, s1), (w2, s2)


def layer64(x, w1, w2, idx, w, clamp=None):
    """(y, bound): the layer in 64 bits, and how far 32-bit arithmetic may be from it before the last rounding.

    The first product is off by product_and_bound; silu has slope 1.1 at most, __expf is off by 2 + 1.16 |g| units of the last place
    and the quotient by 2 more.  Where the quotient 448 a / top comes that near to the middle between two codes, the code may be the other
    one: a whole step.  The rest is linear: those steps and the sums of the second product, weighted."""
    (w1, s1), (w2, s2) = w1, w2
    t, h = x.shape
    i = w2.shape[-1]
    u, top = ref.cast(x.double(), 128)
    xv = ref.e4m3_of(u) * (top / 448).repeat_interleave(128, 1)
    y = torch.zeros((t, h), dtype=torch.float64)
    bound = torch.zeros_like(y)
    for e in range(w1.shape[0]):
        tok, slot = ((idx == e) & (w != 0)).nonzero(as_tuple=True)
        if tok.numel() == 0:
            continue
        gu, gu_err = ref.product_and_bound(xv[tok], ref.by_block(w1[e], s1[e]))
        gate, up = gu[:, :i], gu[:, i:]
        if clamp is not None:
            gate, up = gate.clamp(-clamp, clamp), up.clamp(-clamp, clamp)
        silu = gate * torch.sigmoid(gate)
        act = silu * up
        err = 1.1 * gu_err[:, :i] * up.abs() + silu.abs() * gu_err[:, i:] + 2.0 ** -23 * (8 + 1.2 * gate.abs()) * act.abs()
        u, top = ref.cast(act, 128)
        top_err = torch.stack([err[:, 128 * j:128 * j + 128].amax(1) for j in range(i // 128)], 1)
        wide = lambda v: v.repeat_interleave(128, 1)   # noqa: E731
        near = (err / wide(top) + u.abs() / 448 * wide(top_err / top)) * 448 + 2.0 ** -22 * u.abs()
        codes = ref.e4m3_of(u)
        step = ref.e4m3_step(u.abs() + near)
        flip = ((codes - u).abs() + near >= 0.5 * ref.e4m3_step((u.abs() - near).clamp(min=0))).double() * (step + near)
        act_err = (flip + codes.abs() * wide(top_err / top)) * wide(top / 448)
        w2v = ref.by_block(w2[e], s2[e])
        out, out_err = ref.product_and_bound(codes * wide(top / 448), w2v)
        weight = w[tok, slot].double()[:, None]
        y.index_add_(0, tok, out * weight)
        bound.index_add_(0, tok, (out_err + act_err @ w2v.abs().t() + 2.0 ** -20 * out.abs()) * weight.abs())
    return y, bound


def assert_layer(out, y, bound):
    out = out.cpu().double()
    tol = bound + 2.0 ** -8 * (y.abs() + bound)
    assert bool(((out - y).abs() <= tol).all()), float(((out - y).abs() - tol).max())
    # rounding to bf16 alone is 2^-8 / sqrt(3) of the norm; the bound above is for the worst case, this for the whole
    assert float((out - y).norm()) <= 2.0 ** -8 * float(y.norm())


def choose(logits, k):
    top, idx = torch.sort(logits.double(), dim=1, descending=True, stable=True)
    top, idx = top[:, :k], idx[:, :k].clone()
    closed = top == -math.inf
    p = torch.exp(torch.where(closed, -math.inf, top - top[:, :1].clamp(min=-1e300)))
    p = torch.where(closed, 0.0, p)
    p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
    idx[closed] = -1
    return idx, p


def run(x, w1, w2, layout="native", **kw):
    import megamoe
    (w1, s1), (w2, s2) = w1, w2
    w1, w2 = w1.cuda(), w2.cuda()
    if layout == "tiled":
        w1, w2 = megamoe.pack_weights_tiled(w1, "l1"), megamoe.pack_weights_tiled(w2, "l2")
    kw = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    x = tuple(v.cuda() for v in x) if isinstance(x, tuple) else x.cuda()
    out = megamoe.fp8_moe_few_tokens(x, (w1, s1.cuda()), (w2, s2.cuda()), **kw)
    megamoe.check_block128_status()
    return out


SHAPES = [(1, 8, 2, 512, 256), (1, 4, 4, 128, 128), (2, 8, 1, 640, 384), (5, 16, 3, 384, 128), (33, 8, 2, 512, 256), (130, 4, 2, 256, 128), (64, 40, 6, 1024, 512),
          (300, 2, 2, 128, 256)]


@pytest.mark.parametrize("layout", ["native", "tiled"])
@pytest.mark.parametrize("t,e,k,h,i", SHAPES)
def test_layer_from_router_logits(g, t, e, k, h, i, layout):
    x, w1, w2 = make(g, t, e, h, i)
    logits = torch.randn((t, e), generator=g)
    out = run(x, w1, w2, layout, router_logits=logits, num_topk=k)
    idx, w = choose(logits, k)
    assert_layer(out, *layer64(x, w1, w2, idx, w))


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_layer_from_chosen_experts(g, dtype):
    """Indexes that are no expert, weights of zero and of either sign, the same expert twice, tokens without any route."""
    t, e, k, h, i = 12, 6, 3, 384, 256
    x, w1, w2 = make(g, t, e, h, i)
    idx = torch.randint(0, e, (t, k), generator=g)
    w = torch.randn((t, k), generator=g)
    idx[0] = torch.tensor([2, 2, 2])
    idx[1] = torch.tensor([-1, e, 4])
    idx[2] = -1
    w[5] = 0
    w[6, 1] = 0
    out = run(x, w1, w2, topk_idx=idx.to(dtype), topk_weights=w)
    keep = (idx >= 0) & (idx < e)
    y, bound = layer64(x, w1, w2, torch.where(keep, idx, -1), w)
    assert_layer(out, y, bound)
    assert bool((out[2] == 0).all()) and bool((out[5] == 0).all())


def test_no_route_at_all(g):
    x, w1, w2 = make(g, 7, 4, 256, 128)
    out = torch.full((7, 256), 3.0, dtype=torch.bfloat16)
    got = run(x, w1, w2, topk_idx=torch.full((7, 2), -1, dtype=torch.int32), topk_weights=torch.ones((7, 2)), out=out)
    assert bool((got == 0).all())
    got = run(x, w1, w2, router_logits=torch.full((7, 4), -math.inf), num_topk=2)
    assert bool((got == 0).all())


def test_closed_experts_and_odd_logits(g):
    """-inf, NaN and the type's lowest value as masks; infinities share; a token with fewer open experts than slots; ties."""
    t, e, k, h, i = 9, 12, 4, 256, 128
    x, w1, w2 = make(g, t, e, h, i)
    logits = torch.randn((t, e), generator=g)
    logits[0, 3:] = -math.inf                  # three open
    logits[1] = -math.inf                      # none
    logits[2, ::2] = torch.finfo(torch.float32).min
    logits[4, 5] = math.inf
    logits[5, [1, 7]] = math.inf
    logits[6] = 1.0                            # all equal: the first four
    logits[7, [0, 4]] = math.nan
    logits[8] = torch.finfo(torch.float32).min
    out = run(x, w1, w2, router_logits=logits, num_topk=k)
    ref_logits = logits.clone()
    ref_logits[torch.isnan(ref_logits)] = -math.inf
    idx, w = choose(ref_logits, k)
    for row, at in ((4, [5]), (5, [1, 7])):    # exp(inf - inf) is not a number: the infinities alone, in equal parts
        idx[row] = -1
        idx[row, :len(at)] = torch.tensor(at)
        w[row] = 0
        w[row, :len(at)] = 1.0 / len(at)
    assert idx[6].tolist() == [0, 1, 2, 3] and idx[8].tolist() == [0, 1, 2, 3]
    assert_layer(out, *layer64(x, w1, w2, idx, w))
    assert bool((out[1] == 0).all())


def test_activation_clamp(g):
    x, w1, w2 = make(g, 6, 4, 256, 128)
    logits = torch.randn((6, 4), generator=g)
    idx, w = choose(logits, 2)
    y0, _ = layer64(x, w1, w2, idx, w)
    y, bound = layer64(x, w1, w2, idx, w, clamp=0.5)
    assert float((y - y0).norm()) > 0.05 * float(y0.norm())
    assert_layer(run(x, w1, w2, router_logits=logits, num_topk=2, activation_clamp=0.5), y, bound)


def test_cast_input_equals_plain_input(g):
    """Codes and scales from the cast, or from the norm before the layer, give the very same output as the layer's own cast."""
    import megamoe
    x, w1, w2 = make(g, 21, 8, 512, 256)
    logits = torch.randn((21, 8), generator=g)
    a = run(x, w1, w2, router_logits=logits, num_topk=2)
    q, s = megamoe.cast_to_fp8_block128(x.cuda())
    b = run((q, s), w1, w2, router_logits=logits, num_topk=2)
    assert torch.equal(a, b)


def test_one_popular_expert(g):
    """More than 128 routes on one expert, none on most: several blocks of routes, the last of one row."""
    t, e, k, h, i = 257, 16, 1, 256, 256
    x, w1, w2 = make(g, t, e, h, i)
    idx = torch.full((t, k), 5)
    w = torch.rand((t, k), generator=g) + 0.5
    assert_layer(run(x, w1, w2, topk_idx=idx, topk_weights=w), *layer64(x, w1, w2, idx, w))


def test_bad_rows_stay_in_their_rows(g):
    """A token with NaN or infinity spoils its own output only, even among routes to the same expert."""
    x, w1, w2 = make(g, 10, 3, 256, 128)
    x[2, 7] = math.nan
    x[8, 100] = math.inf
    logits = torch.randn((10, 3), generator=g)
    out = run(x, w1, w2, router_logits=logits, num_topk=2).cpu()
    assert (~torch.isfinite(out).all(1)).nonzero()[:, 0].tolist() == [2, 8]
    ok = [r for r in range(10) if r not in (2, 8)]
    idx, w = choose(logits, 2)
    y, bound = layer64(x[ok], w1, w2, idx[ok], w[ok])
    assert_layer(out[ok], y, bound)


def test_repeatable_and_after_larger_calls(g):
    """The same bits whatever the work memory held before and whichever CTA came last."""
    x, w1, w2 = make(g, 40, 8, 1024, 512)
    logits = torch.randn((40, 8), generator=g)
    first = run(x, w1, w2, "tiled", router_logits=logits, num_topk=3)
    for n in (40, 1, 17, 40):
        out = run(x[:n], w1, w2, "tiled", router_logits=logits[:n], num_topk=3)
        if n == 40:
            assert torch.equal(out, first)
