"""Sizes that do not fit the C entry points' 32-bit arguments are refused, not cut off, and so are the test hook's.  No GPU: tensors without
memory that the checks are told to take for a GPU's."""
import pytest
import torch


@pytest.fixture
def block128(monkeypatch, built_lib):
    from deepgemm_b200.megamoe import block128
    monkeypatch.setattr(block128, "_device_index", lambda *a: 0)

    def call(index, fn, *args):
        raise AssertionError(f"the library was called with {args}")
    monkeypatch.setattr(block128, "_call", call)
    return block128


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


FAR = 2 ** 32 + 128                     # cut off to 32 bits: 128


def test_rows_longer_than_31_bits_are_refused(block128):
    for k in (2 ** 31, FAR):
        with pytest.raises(ValueError, match="2\\^31"):
            block128.cast_to_fp8_block128(_meta(k))
        with pytest.raises(ValueError, match="2\\^31"):
            block128.cast_weight_to_fp8_block128(_meta(1, k))
        with pytest.raises(ValueError, match="2\\^31"):
            block128.cast_weight_to_fp8_block128(_meta(k, 8))
        with pytest.raises(ValueError, match="2\\^31"):
            block128.cast_weight_to_fp8_block128(_meta(k, 8, 8))


def test_norms_of_more_than_31_bits_of_rows_are_refused(block128):
    for t in (2 ** 31, FAR):
        with pytest.raises(ValueError, match="2\\^31"):
            block128.norm_gate_residual(None, _meta(t, 8), pre_weight=_meta(8, dtype=torch.float32))


def test_products_of_more_than_31_bits_are_refused(block128):
    codes = lambda *s: _meta(*s, dtype=torch.float8_e4m3fn)   # noqa: E731
    ones = lambda *s: _meta(*s, dtype=torch.float32)   # noqa: E731
    for n in (2 ** 31, FAR):
        with pytest.raises(RuntimeError, match="2\\^31"):
            block128.fp8_gemm_nt_block128((codes(1, 16), ones(1, 1)), (codes(n, 16), ones(n // 128, 1)))
        with pytest.raises(RuntimeError, match="2\\^31"):
            block128.fp8_gemm_nt_block128((codes(1, n), ones(1, n // 128)), (codes(1, n), ones(1, n // 128)))
        with pytest.raises(RuntimeError, match="2\\^31"):
            block128.m_grouped_fp8_gemm_nt_contiguous_block128((codes(128, 16), ones(128, 1)), (codes(1, n, 16), ones(1, n // 128, 1)), _meta(128, n),
                                                               _meta(128, dtype=torch.int32))
        with pytest.raises(RuntimeError, match="2\\^31"):
            block128.m_grouped_fp8_gemm_nt_contiguous_block128((codes(128, 16), ones(128, 1)), (codes(n, 1, 16), ones(n, 1, 1)), _meta(128, 1),
                                                               _meta(128, dtype=torch.int32))


def test_layers_of_more_experts_than_31_bits_are_refused(block128):
    e = FAR
    with pytest.raises((RuntimeError, ValueError), match="experts"):
        block128.fp8_moe_few_tokens(_meta(1, 128), (_meta(e, 256, 128, dtype=torch.float8_e4m3fn), _meta(e, 2, 1, dtype=torch.float32)),
                                    (_meta(e, 128, 128, dtype=torch.float8_e4m3fn), _meta(e, 1, 1, dtype=torch.float32)),
                                    topk_idx=_meta(1, 2, dtype=torch.int32), topk_weights=_meta(1, 2, dtype=torch.float32))


def test_the_hook_of_the_waits_refuses(built_lib):
    for args in ((-2, 0), (-1, -1)):
        assert built_lib.mm_block128_test_waits(*args) != 0 and b"no such" in built_lib.mm_last_error()
    assert built_lib.mm_block128_test_waits(-1, 0) == 0
