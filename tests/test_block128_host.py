"""Refusals of the block-scaled operators that need no GPU: the C entry points before any CUDA call, the Python checks on CPU tensors."""
import pytest
import torch

P = 0x1000            # an aligned address that nothing reads


def _refused(lib, rc, words):
    assert rc != 0 and words in lib.mm_last_error().decode(), lib.mm_last_error()


def test_cast_entry_points_refuse(built_lib):
    f = built_lib.mm_cast_block128
    _refused(built_lib, f(P, 3, 4, 128, 128, P, P, None), "unknown type")
    _refused(built_lib, f(P, 0, 4, 12, 16, P, P, None), "multiples of 8")
    _refused(built_lib, f(P, 0, 4, 128, 120, P, P, None), "multiples of 8")
    _refused(built_lib, f(P, 0, 4, 128, 132, P, P, None), "16 bytes")
    _refused(built_lib, f(P, 2, 4, 128, 130, P, P, None), "16 bytes")
    _refused(built_lib, f(P, 0, -1, 128, 128, P, P, None), "multiples of 8")
    _refused(built_lib, f(None, 0, 4, 128, 128, P, P, None), "null")
    _refused(built_lib, f(P + 8, 0, 4, 128, 128, P, P, None), "aligned")
    _refused(built_lib, f(P, 0, 1 << 33, 128, 128, P, P, None), "too many")
    assert f(None, 0, 0, 128, 128, None, None, None) == 0
    f = built_lib.mm_cast_weight_block128
    _refused(built_lib, f(P, 0, 1, 4, 12, P, P, None), "multiple of 8")
    _refused(built_lib, f(P, 9, 1, 4, 16, P, P, None), "unknown type")
    _refused(built_lib, f(P, 0, 1, 4, 16, None, P, None), "null")
    assert f(None, 0, 0, 4, 16, None, None, None) == 0


def test_product_entry_point_refuses(built_lib):
    def call(a=P, a_stride=256, sa=P, sa_stride=2, b=P, sb=P, experts=1, tiled=0, mi=None, out=P, out_stride=128, fp32=0, m=8, n=128, k=256):
        return built_lib.mm_fp8_gemm_block128(a, a_stride, sa, sa_stride, b, sb, experts, tiled, mi, out, out_stride, fp32, m, n, k, None)
    _refused(built_lib, call(k=200), "multiple of 16")
    _refused(built_lib, call(m=-1), "multiple of 16")
    _refused(built_lib, call(experts=2), "m_indices")
    _refused(built_lib, call(experts=0), "m_indices")
    _refused(built_lib, call(mi=P, m=100), "multiple of 128")
    _refused(built_lib, call(tiled=1, n=100), "tiled")
    _refused(built_lib, call(b=None), "null")
    _refused(built_lib, call(a=P + 8), "aligned")
    _refused(built_lib, call(a_stride=264), "aligned")
    _refused(built_lib, call(sa_stride=1), "strides")
    _refused(built_lib, call(out_stride=100), "strides")
    assert call(m=0) == 0 and call(n=0) == 0


def test_norm_entry_point_refuses(built_lib):
    def call(y=P, ys=64, r=P, rs=64, post=P, gate=None, grs=0, gcs=0, pre=P, ro=P, xo=P, xt=0, q=None, sf=None, quant=0, t=2, h=64, yt=0):
        return built_lib.mm_norm_gate_residual(y, yt, ys, r, 0, rs, post, 2, gate, 2, grs, gcs, pre, 2, ro, xo, xt, q, sf, quant, t, h, 1.0, 1e-6, 0.0, None)
    _refused(built_lib, call(h=60), "multiple of 8")
    _refused(built_lib, call(h=16392, ys=16392, rs=16392), "at most")
    _refused(built_lib, call(quant=3), "unknown cast")
    _refused(built_lib, call(yt=5), "unknown type")
    _refused(built_lib, call(y=None), "null")
    _refused(built_lib, call(ro=None), "null")
    _refused(built_lib, call(pre=None), "weight")
    _refused(built_lib, call(quant=1), "null")
    _refused(built_lib, call(ys=56), "strides")
    _refused(built_lib, call(gate=P, gcs=2), "strides")
    _refused(built_lib, call(y=P + 4), "aligned")
    assert call(t=0) == 0


def test_python_checks_on_cpu_tensors():
    import megamoe
    x = torch.zeros((4, 128), dtype=torch.bfloat16)
    q, s = torch.zeros((4, 128), dtype=torch.uint8).view(torch.float8_e4m3fn), torch.ones((4, 1))
    for call in (lambda: megamoe.cast_to_fp8_block128(x), lambda: megamoe.cast_weight_to_fp8_block128(x),
                 lambda: megamoe.fp8_gemm_nt_block128((q, s), (q, s[:1])), lambda: megamoe.norm_gate_residual(x, x)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(ValueError):
        megamoe.cast_to_fp8_block128(x[:, :100])
    with pytest.raises(TypeError):
        megamoe.cast_to_fp8_block128(x.double())
    with pytest.raises(TypeError):
        megamoe.cast_weight_to_fp8_block128(x[0])


def test_layer_entry_point_refuses(built_lib):
    def call(x=P, fp8=0, xs=256, xsf=None, logits=P, ls=8, idx=None, w=None, w1=P, work=P, y=P, t=4, e=8, k=2, h=256, i=128, clamp=float("inf")):
        return built_lib.mm_moe_few_tokens(x, fp8, xs, xsf, logits, ls, idx, 0, w, w1, P, P, P, 0, t, e, k, h, i, clamp, work, 1 << 40, y, None)
    _refused(built_lib, call(k=9), "topk")
    _refused(built_lib, call(k=0), "topk")
    _refused(built_lib, call(e=64, k=33), "topk")
    _refused(built_lib, call(e=2000), "experts")
    _refused(built_lib, call(h=200), "multiples of 128")
    _refused(built_lib, call(i=100), "multiples of 128")
    _refused(built_lib, call(h=65536, xs=65536), "at most")
    _refused(built_lib, call(t=2049), "routes")
    _refused(built_lib, call(clamp=0.0), "clamp")
    _refused(built_lib, call(clamp=float("nan")), "clamp")
    _refused(built_lib, call(w1=None), "null")
    _refused(built_lib, call(fp8=1), "null")
    _refused(built_lib, call(fp8=1, xsf=P, xs=512), "contiguous")
    _refused(built_lib, call(idx=P, w=P), "either")
    _refused(built_lib, call(logits=None), "either")
    _refused(built_lib, call(logits=None, idx=P), "either")
    _refused(built_lib, call(x=P + 8), "aligned")
    _refused(built_lib, call(xs=248), "aligned")
    _refused(built_lib, call(work=P + 16), "aligned")
    _refused(built_lib, call(ls=7), "stride")
    assert call(t=0) == 0
    _refused(built_lib, built_lib.mm_moe_few_tokens_workspace(4, 8, 2, 256, 128, None), "null")
    _refused(built_lib, built_lib.mm_block128_read_status(None, None), "null")


def test_layer_python_checks(monkeypatch):
    """What the layer's Python entry refuses, on CPU tensors that it is told to take for a GPU's."""
    import megamoe
    from deepgemm_b200.megamoe import block128
    monkeypatch.setattr(block128, "_device_index", lambda *a: 0)
    e, k, h, i, t = 4, 2, 256, 128, 3
    codes = lambda *s: torch.zeros(s, dtype=torch.uint8).view(torch.float8_e4m3fn)   # noqa: E731
    good = dict(x=torch.zeros((t, h), dtype=torch.bfloat16), l1_weights=(codes(e, 2 * i, h), torch.ones((e, 2, 2))), l2_weights=(codes(e, h, i), torch.ones((e, 2, 1))),
                router_logits=torch.zeros((t, e)), num_topk=k)
    chosen = dict(router_logits=None, num_topk=None, topk_idx=torch.zeros((t, k), dtype=torch.int32), topk_weights=torch.ones((t, k)))
    bad = [
        (dict(x=torch.zeros((t, h))), "bfloat16"),
        (dict(x=(codes(t, h), torch.ones((t, 1)))), "scales of x"),
        (dict(x=torch.zeros((t, 128), dtype=torch.bfloat16)), "do not match"),
        (dict(l1_weights=(codes(e, i, h), good["l1_weights"][1])), "do not match"),
        (dict(l1_weights=(codes(e, 2 * i, 2 * h)[:, :, ::2], good["l1_weights"][1])), "contiguous"),
        (dict(l2_weights=(good["l2_weights"][0], torch.ones((e, 2, 2)))), "do not match"),
        (dict(l2_weights=(torch.zeros((e, h, i)), good["l2_weights"][1])), "e4m3"),
        (dict(router_logits=None), "either"),
        (dict(topk_idx=chosen["topk_idx"]), "either"),
        (dict(num_topk=None), "num_topk"),
        (dict(num_topk=e + 1), "topk must be"),
        (dict(router_logits=torch.zeros((t, e), dtype=torch.bfloat16)), "fp32"),
        (dict(chosen, topk_weights=None), "both be"),
        (dict(chosen, topk_idx=torch.zeros((t, k), dtype=torch.int16)), "int32 or int64"),
        (dict(chosen, num_topk=1), "does not match"),
        (dict(activation_clamp=-1.0), "positive"),
        (dict(out=torch.zeros((t, h))), "out must be"),
        (dict(x=torch.zeros((2049, h), dtype=torch.bfloat16), router_logits=torch.zeros((2049, e))), "4096 routes"),
    ]
    for change, words in bad:
        with pytest.raises((RuntimeError, ValueError), match=words):
            megamoe.fp8_moe_few_tokens(**{**good, **change})


def test_product_python_checks(monkeypatch):
    import megamoe
    from deepgemm_b200.megamoe import block128
    monkeypatch.setattr(block128, "_device_index", lambda *a: 0)
    codes = lambda *s: torch.zeros(s, dtype=torch.uint8).view(torch.float8_e4m3fn)   # noqa: E731
    a, b, w = (codes(128, 256), torch.ones((128, 2))), (codes(64, 256), torch.ones((1, 2))), (codes(3, 64, 256), torch.ones((3, 1, 2)))
    for args, kw, words in (((a, (b[0], torch.ones((2, 2)))), {}, "weight scales"), (((a[0], torch.ones((128, 1))), b), {}, "with scales"),
                            ((a, b), dict(out_dtype=torch.float16), "bfloat16 or float32"), ((a, b), dict(out=torch.zeros((128, 65))), "out must be"),
                            (((a[0][:, :200], a[1]), (b[0][:, :200], b[1])), {}, "multiple of 16"), (((a[0].float(), a[1]), b), {}, "e4m3"), ((a, w), {}, "2D")):
        with pytest.raises(RuntimeError, match=words):
            megamoe.fp8_gemm_nt_block128(*args, **kw)
    d, idx = torch.zeros((128, 64), dtype=torch.bfloat16), torch.zeros(128, dtype=torch.int32)
    for args, words in (((a, w, d.half(), idx), "contiguous bfloat16"), ((a, w, d, idx.long()), "int32"), ((a, b, d, idx), "expects weights"),
                        ((a, w, d[:, :48].contiguous(), idx), "do not match"), (((a[0][:100], a[1][:100]), w, d[:100], idx[:100]), "multiple of 128")):
        with pytest.raises(RuntimeError, match=words):
            megamoe.m_grouped_fp8_gemm_nt_contiguous_block128(*args)
