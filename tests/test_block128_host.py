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
