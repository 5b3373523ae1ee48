"""Operators in FP8 e4m3 with one fp32 scale for each block of 128 values, and the norms that feed them.

Activations carry a scale for each 128 values of a row ([rows, ceil(K/128)]), weights one for each 128 x 128 block
([.., ceil(N/128), ceil(K/128)]).  The channelwise layer (`fp8_mega_moe`) has one scale per row and per output channel instead; a
checkpoint quantised by blocks cannot be converted to that without a second rounding, so it is served by these:

  cast_to_fp8_block128, cast_weight_to_fp8_block128      bf16 / fp16 / fp32 -> codes and scales
  fp8_gemm_nt_block128                                   dense product
  m_grouped_fp8_gemm_nt_contiguous_block128              product of rows grouped by expert
  fp8_moe_few_tokens                                     a whole mixture-of-experts layer for a few tokens, on one GPU
  norm_gate_residual                                     norms around a block with its gate, scaled residual and either cast

Calls are asynchronous on the current stream of the tensors' device, keep nothing between calls and may be captured into a CUDA
graph.  `check_block128_status()` reports what a kernel could not (a bounded wait that expired, a grouped layout that mixes experts).
"""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import NamedTuple, Optional, Tuple

import torch

from .. import _lib

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_E4M3 = torch.float8_e4m3fn
_DIM = 2 ** 31      # sizes pass through the library's 32-bit arguments, where ctypes would cut off a larger one without a word


def _blocks(n: int) -> int:
    return (n + 127) // 128


# The stream's handle without building a Stream object around it: 0.1 us instead of 3, and a call for one token takes about ten.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(index: int, fn, *args) -> None:
    """Run a library call (its last argument, the stream, is added here) with device `index` current."""
    if index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc != 0:
        _lib.check(rc)


def _device_index(name: str, *tensors: Optional[torch.Tensor]) -> int:
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != index:
            index = -1
    if index < 0:
        if any(t is not None and not t.is_cuda for t in tensors):
            raise RuntimeError(f"{name} needs CUDA tensors (this package has no CPU path)")
        raise RuntimeError(f"{name}: tensors are on different devices")
    return index


def _rows_of(t: torch.Tensor, align: int) -> Tuple[torch.Tensor, int]:
    """`t` [rows, k] as it is if its rows are dense and start on `align`-byte boundaries, else a contiguous copy; and the elements from
    a row to the next (the stride of a single row says nothing)."""
    rows, k = t.shape
    pitch, step = t.stride()
    if rows <= 1:
        pitch = k
    if step == 1 and pitch >= k and t.data_ptr() % align == 0 and (pitch * t.element_size()) % align == 0:
        return t, pitch
    return _dense(t, align), k


def _dense(t: torch.Tensor, align: int) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % align == 0 else t.clone()


def _pitch(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def cast_to_fp8_block128(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows [.., K] of bf16, fp16 or fp32 (K a multiple of 8) -> (e4m3 [.., K], fp32 scales [.., ceil(K/128)]).

    For each 128 values of a row: top = max(amax, 1e-4), scale = top / 448, code = e4m3(448 x / top), ties to even.  A block that
    holds an infinity or a NaN gets NaN codes and a scale that is not finite."""
    kind = _TYPES.get(x.dtype)
    if kind is None or x.dim() < 1:
        raise TypeError("cast_to_fp8_block128 expects a bfloat16, float16 or float32 tensor with at least one dimension")
    shape = x.shape
    k = shape[-1]
    if k == 0 or k % 8 != 0 or k >= _DIM:
        raise ValueError("the row length must be a positive multiple of 8" if k < _DIM else "the row length must be below 2^31")
    index = _device_index("cast_to_fp8_block128", x)
    q = torch.empty_like(x, dtype=_E4M3, memory_format=torch.contiguous_format)      # (half of new_empty's time)
    sf = x.new_empty((*shape[:-1], (k + 127) // 128), dtype=torch.float32)
    rows = x.numel() // k
    if rows:
        stride = k
        if not x.is_contiguous() or x.data_ptr() % 16 != 0:
            x, stride = _rows_of(x if x.dim() == 2 else x.reshape(-1, k), 16)
        _call(index, _lib.lib().mm_cast_block128, x.data_ptr(), kind, rows, k, stride, q.data_ptr(), sf.data_ptr())
    return q, sf


def cast_weight_to_fp8_block128(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Weights [N, K] or [E, N, K] (K a multiple of 8) -> (e4m3 of the same shape, fp32 scales [.., ceil(N/128), ceil(K/128)]):
    the cast of `cast_to_fp8_block128` with one scale for each 128 x 128 block."""
    if w.dim() not in (2, 3) or w.dtype not in _TYPES:
        raise TypeError("cast_weight_to_fp8_block128 expects a 2D or 3D bfloat16, float16 or float32 tensor")
    n, k = w.shape[-2:]
    if k == 0 or k % 8 != 0:
        raise ValueError("the row length must be a positive multiple of 8")
    if max(w.shape) >= _DIM:
        raise ValueError("each size of a weight must be below 2^31")
    index = _device_index("cast_weight_to_fp8_block128", w)
    w = w.contiguous()
    if w.data_ptr() % 16 != 0:
        w = w.clone()
    q = w.new_empty(w.shape, dtype=_E4M3)
    sf = w.new_empty((*w.shape[:-2], _blocks(n), _blocks(k)), dtype=torch.float32)
    if w.numel():
        _call(index, _lib.lib().mm_cast_weight_block128, w.data_ptr(), _TYPES[w.dtype], w.shape[0] if w.dim() == 3 else 1, n, k, q.data_ptr(), sf.data_ptr())
    return q, sf


def _check_operands(name, a, a_sf, b, b_sf, n, k):
    if a.dtype != _E4M3 or b.dtype != _E4M3:
        raise RuntimeError(f"{name} expects e4m3 operands")
    if a_sf.dtype != torch.float32 or b_sf.dtype != torch.float32:
        raise RuntimeError(f"{name} expects fp32 scales")
    if k == 0 or k % 16 != 0:
        raise RuntimeError(f"{name}: K must be a positive multiple of 16")
    if k >= _DIM or n >= _DIM or b.shape[0] >= _DIM:
        raise RuntimeError(f"{name}: N, K and the number of experts must be below 2^31")
    kb = (k + 127) // 128
    if a.dim() != 2 or a.shape[1] != k or a_sf.shape != (a.shape[0], kb):
        raise RuntimeError(f"{name} expects a [M, K] with scales [M, ceil(K/128)], got {tuple(a.shape)} and {tuple(a_sf.shape)}")
    if b_sf.shape[-2:] != ((n + 127) // 128, kb):
        raise RuntimeError(f"{name} expects weight scales [.., ceil(N/128), ceil(K/128)], got {tuple(b_sf.shape)}")


def _scale_rows(sf: torch.Tensor) -> torch.Tensor:
    return sf if sf.is_contiguous() or (sf.stride(1) == 1 and sf.stride(0) >= sf.shape[1]) else sf.contiguous()


def fp8_gemm_nt_block128(a: Tuple[torch.Tensor, torch.Tensor], b: Tuple[torch.Tensor, torch.Tensor], out: Optional[torch.Tensor] = None,
                         out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """out[M, N] = a [M, K] . b [N, K]^T with a = (e4m3, scales [M, ceil(K/128)]), b = (e4m3, scales [ceil(N/128), ceil(K/128)]).

    K is a multiple of 16 and may end inside a block; M and N are any.  Rows of `a` and of `out` may be strided.  The sums are fp32;
    the output is bf16 or fp32 (`out`'s type, else `out_dtype`, else bf16)."""
    (a_q, a_sf), (b_q, b_sf) = a, b
    name = "fp8_gemm_nt_block128"
    index = _device_index(name, a_q, a_sf, b_q, b_sf, out)
    if b_q.dim() != 2 or b_sf.dim() != 2:
        raise RuntimeError(f"{name} expects b [N, K] with 2D scales")
    n, k = b_q.shape
    _check_operands(name, a_q, a_sf, b_q, b_sf, n, k)
    m = a_q.shape[0]
    if out is None:
        out = a_q.new_empty((m, n), dtype=torch.bfloat16 if out_dtype is None else out_dtype)
        pitch = n
    else:
        if tuple(out.shape) != (m, n) or (n > 1 and out.stride(1) != 1) or (m > 1 and out.stride(0) < n) or (out_dtype is not None and out.dtype != out_dtype):
            raise RuntimeError(f"{name}: out must be [{m}, {n}] with dense rows (and of out_dtype, if that is given)")
        pitch = _pitch(out)
    if out.dtype not in (torch.bfloat16, torch.float32):
        raise RuntimeError(f"{name}: the output is bfloat16 or float32")
    if m == 0 or n == 0:
        return out
    (a_q, a_pitch), b_q, a_sf, b_sf = _rows_of(a_q, 16), _dense(b_q, 16), _scale_rows(a_sf), b_sf.contiguous()
    _call(index, _lib.lib().mm_fp8_gemm_block128, a_q.data_ptr(), a_pitch, a_sf.data_ptr(), _pitch(a_sf), b_q.data_ptr(),
          b_sf.data_ptr(), 1, 0, None, out.data_ptr(), pitch, out.dtype == torch.float32, m, n, k)
    return out


def m_grouped_fp8_gemm_nt_contiguous_block128(a: Tuple[torch.Tensor, torch.Tensor], b: Tuple[torch.Tensor, torch.Tensor], d: torch.Tensor,
                                              m_indices: torch.Tensor, check: bool = False) -> torch.Tensor:
    """d[row] = a[row] . b[e]^T with e = m_indices[row], as `m_grouped_fp8_gemm_nt_contiguous` with scales by blocks.

    a = (e4m3 [rows, K], scales [rows, ceil(K/128)]), b = (e4m3 [E, N, K] or tiled (`pack_weights_tiled(w, "l2")`), scales
    [E, ceil(N/128), ceil(K/128)]), d bf16 or fp32.  Rows are grouped by expert, groups padded to 128 rows; rows with m_indices -1 are
    left as they were.  check=True synchronises and raises if a 128-row block mixed experts (such rows are not written)."""
    (a_q, a_sf), (w, w_sf) = a, b
    name = "m_grouped_fp8_gemm_nt_contiguous_block128"
    index = _device_index(name, a_q, a_sf, w, w_sf, d, m_indices)
    if w_sf.dim() != 3 or w.dim() not in (3, 5) or w.shape[0] != w_sf.shape[0]:
        raise RuntimeError(f"{name} expects weights [E, N, K] (or tiled) with scales [E, ceil(N/128), ceil(K/128)]")
    k = a_q.shape[-1]
    n = d.shape[-1]
    tiled = w.dim() == 5
    if tiled and (n % 128 != 0 or k % 128 != 0 or tuple(w.shape[1:]) != ((n + 255) // 256, k // 128, 256, 128)):
        raise RuntimeError(f"{name}: tiled weights of shape {tuple(w.shape)} do not match N = {n}, K = {k}")
    if not tiled and tuple(w.shape[1:]) != (n, k):
        raise RuntimeError(f"{name}: weights of shape {tuple(w.shape)} do not match N = {n}, K = {k}")
    _check_operands(name, a_q, a_sf, w, w_sf, n, k)
    rows = a_q.shape[0]
    if tuple(d.shape) != (rows, n) or not d.is_contiguous() or d.dtype not in (torch.bfloat16, torch.float32):
        raise RuntimeError(f"{name}: d must be a contiguous bfloat16 or float32 [{rows}, {n}]")
    if m_indices.dtype != torch.int32 or tuple(m_indices.shape) != (rows,):
        raise RuntimeError(f"{name} expects int32 m_indices [{rows}]")
    if rows % _lib.BLOCK_M != 0:
        raise RuntimeError(f"{name}: rows must be a multiple of {_lib.BLOCK_M} (groups padded to it)")
    if rows and n and w.shape[0] == 0:
        raise RuntimeError(f"{name}: no experts")
    if rows and n:
        (a_q, a_pitch), w, a_sf, w_sf, m_indices = _rows_of(a_q, 16), _dense(w, 16), _scale_rows(a_sf), w_sf.contiguous(), m_indices.contiguous()
        _call(index, _lib.lib().mm_fp8_gemm_block128, a_q.data_ptr(), a_pitch, a_sf.data_ptr(), _pitch(a_sf), w.data_ptr(),
              w_sf.data_ptr(), w.shape[0], tiled, m_indices.data_ptr(), d.data_ptr(), n, d.dtype == torch.float32, rows, n, k)
    if check:
        check_block128_status(index)
    return d


def transform_fp8_weights_for_few_tokens(l1_weights: torch.Tensor, l2_weights: torch.Tensor, layout: str = "tiled"):
    """bf16, fp16 or fp32 [E, 2I, H] (gate rows, then up rows) and [E, H, I] -> ((w1, s1 [E, 2I/128, H/128]), (w2, s2 [E, H/128, I/128])).
    layout="tiled" packs the codes in the order the kernel streams them (`pack_weights_tiled`), "native" keeps [E, rows, K]."""
    if layout not in ("tiled", "native"):
        raise ValueError("layout must be 'tiled' or 'native'")
    if l1_weights.dim() != 3 or l2_weights.dim() != 3:
        raise ValueError("MoE weights must be 3D tensors")
    (w1, s1), (w2, s2) = cast_weight_to_fp8_block128(l1_weights), cast_weight_to_fp8_block128(l2_weights)
    if layout == "tiled":
        from . import pack_weights_tiled
        w1, w2 = pack_weights_tiled(w1, "l1"), pack_weights_tiled(w2, "l2")
    return (w1, s1), (w2, s2)


@lru_cache(maxsize=256)
def _moe_work_bytes(device: int, t: int, e: int, k: int, h: int, i: int) -> int:
    out = ctypes.c_int64()
    with torch.cuda.device(device):
        _lib.check(_lib.lib().mm_moe_few_tokens_workspace(t, e, k, h, i, ctypes.byref(out)))
    return out.value


def fp8_moe_few_tokens(x, l1_weights: Tuple[torch.Tensor, torch.Tensor], l2_weights: Tuple[torch.Tensor, torch.Tensor], *,
                       router_logits: Optional[torch.Tensor] = None, num_topk: Optional[int] = None, topk_idx: Optional[torch.Tensor] = None,
                       topk_weights: Optional[torch.Tensor] = None, activation_clamp: Optional[float] = None,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """A whole mixture-of-experts layer for a few tokens (T * topk <= 4096 routes), in two launches on one GPU:

        y[t] = sum over slots of weight * W2[e] . cast(silu(g) * u),    (g, u) = W1[e] . cast(x[t])

    x: bf16 [T, H], or (codes [T, H], scales [T, H/128]) as the casts of this module give them.  Routing: router_logits fp32 [T, E] with
    num_topk -- the largest logits, ties to the lower index, softmax over the chosen ones, as `fill_inputs_from_router`; NaN and -inf
    (closed experts) are never chosen -- or topk_idx (int32 or int64) and topk_weights fp32, both [T, topk]; an index outside 0 .. E-1 or a
    weight of 0 is no route.  A token without any route gets zeros.  Weights: `transform_fp8_weights_for_few_tokens`, tiled or native.
    activation_clamp bounds gate and up to +-clamp, as in `fp8_mega_moe`.

    Sums, SwiGLU and the combine are fp32; the output bf16 [T, H] is rounded once.  Each call takes its work memory from torch's
    allocator.  For many tokens per expert use the grouped product, for channelwise weights or several GPUs `fp8_mega_moe`."""
    name = "fp8_moe_few_tokens"
    x_sf = None
    if isinstance(x, (tuple, list)):
        x, x_sf = x
    (w1, s1), (w2, s2) = l1_weights, l2_weights
    index = _device_index(name, x, x_sf, w1, s1, w2, s2, router_logits, topk_idx, topk_weights, out)
    if x.dim() != 2 or x.dtype != (torch.bfloat16 if x_sf is None else _E4M3):
        raise RuntimeError(f"{name} expects x as bfloat16 [T, H] or as e4m3 codes with their scales")
    if w1.dtype != _E4M3 or w2.dtype != _E4M3 or s1.dtype != torch.float32 or s2.dtype != torch.float32:
        raise RuntimeError(f"{name} expects e4m3 weights with fp32 scales")
    t, h = x.shape
    if s1.dim() != 3 or s2.dim() != 3 or s1.shape[1] % 2 != 0:
        raise RuntimeError(f"{name} expects weight scales [E, 2I/128, H/128] and [E, H/128, I/128]")
    e, i = s1.shape[0], s1.shape[1] * 64
    if h == 0 or i == 0 or h % 128 != 0 or tuple(s1.shape) != (e, i // 64, h // 128) or tuple(s2.shape) != (e, h // 128, i // 128):
        raise RuntimeError(f"{name}: weight scales {tuple(s1.shape)} and {tuple(s2.shape)} do not match H = {h}")
    tiled = w1.dim() == 5
    if tiled:
        ok = tuple(w1.shape) == (e, i // 128, h // 128, 256, 128) and tuple(w2.shape) == (e, (h + 255) // 256, i // 128, 256, 128)
    else:
        ok = tuple(w1.shape) == (e, 2 * i, h) and tuple(w2.shape) == (e, h, i)
    if not ok:
        raise RuntimeError(f"{name}: weights {tuple(w1.shape)} and {tuple(w2.shape)} do not match their scales (both native or both tiled)")
    for v in (w1, w2):
        if not v.is_contiguous() or v.data_ptr() % 16 != 0:
            raise RuntimeError(f"{name}: weights must be contiguous and 16-byte aligned")
    if (router_logits is None) == (topk_idx is None):
        raise ValueError(f"{name}: pass either router_logits with num_topk, or topk_idx with topk_weights")
    if router_logits is not None:
        if num_topk is None or topk_weights is not None:
            raise ValueError(f"{name}: router_logits need num_topk and no topk_weights")
        if router_logits.dtype != torch.float32 or tuple(router_logits.shape) != (t, e):
            raise RuntimeError(f"{name}: router_logits must be fp32 [{t}, {e}]")
        k = int(num_topk)
        router_logits = _scale_rows(router_logits)
    else:
        if topk_weights is None or topk_idx.dim() != 2 or topk_idx.shape[0] != t or topk_idx.shape != topk_weights.shape:
            raise RuntimeError(f"{name}: topk_idx and topk_weights must both be [{t}, topk]")
        if topk_idx.dtype not in (torch.int32, torch.int64) or topk_weights.dtype != torch.float32:
            raise RuntimeError(f"{name}: topk_idx must be int32 or int64, topk_weights fp32")
        k = topk_idx.shape[1]
        if num_topk is not None and num_topk != k:
            raise ValueError(f"{name}: num_topk does not match topk_idx")
        topk_idx, topk_weights = topk_idx.contiguous(), topk_weights.contiguous()
    if e >= _DIM:
        raise ValueError(f"{name}: too many experts")
    if not 0 < k <= min(e, 32):
        raise ValueError(f"{name}: topk must be in 1..{min(e, 32)}")
    if t * k > 4096:
        raise ValueError(f"{name}: {t} tokens x {k} experts are more than 4096 routes; use the grouped product")
    if x_sf is not None and (x_sf.dtype != torch.float32 or tuple(x_sf.shape) != (t, h // 128)):
        raise RuntimeError(f"{name}: scales of x must be fp32 [{t}, {h // 128}]")
    clamp = float("inf") if activation_clamp is None else float(activation_clamp)
    if not clamp > 0:
        raise ValueError(f"{name}: activation_clamp must be positive")
    if out is None:
        out = x.new_empty((t, h), dtype=torch.bfloat16)
    elif out.dtype != torch.bfloat16 or tuple(out.shape) != (t, h) or not out.is_contiguous() or out.data_ptr() % 16 != 0:
        raise RuntimeError(f"{name}: out must be a contiguous bfloat16 [{t}, {h}], 16-byte aligned")
    if t == 0:
        return out
    if x_sf is None:
        x, stride = _rows_of(x, 32)      # 16 values
    else:
        x, x_sf, stride = x.contiguous(), x_sf.contiguous(), h
        if x.data_ptr() % 16 != 0:
            x = x.clone()
    s1, s2 = s1.contiguous(), s2.contiguous()
    nbytes = _moe_work_bytes(index, t, e, k, h, i)
    work = x.new_empty((nbytes,), dtype=torch.uint8)
    logits = router_logits
    _call(index, _lib.lib().mm_moe_few_tokens, x.data_ptr(), x_sf is not None, stride, None if x_sf is None else x_sf.data_ptr(),
          None if logits is None else logits.data_ptr(), 0 if logits is None else _pitch(logits), None if topk_idx is None else topk_idx.data_ptr(),
          topk_idx is not None and topk_idx.dtype == torch.int64, None if topk_weights is None else topk_weights.data_ptr(), w1.data_ptr(), s1.data_ptr(),
          w2.data_ptr(), s2.data_ptr(), tiled, t, e, k, h, i, clamp, work.data_ptr(), nbytes, out.data_ptr())
    return out


def check_block128_status(device=None) -> None:
    """Synchronise the current stream and raise if a kernel of this module has reported a failure on `device` since the last call."""
    out = (ctypes.c_int32 * 5)()
    with torch.cuda.device(device):
        _lib.check(_lib.lib().mm_block128_read_status(torch.cuda.current_stream().cuda_stream, out))
    if out[0] != 0:
        raise _lib.MegaMoeError(f"device status {out[0]} ({_lib.STATUS_NAMES.get(out[0], '?')}): phase={out[1]} block={out[2]} "
                                f"expected={out[3]} observed={out[4]}")


class NormOutputs(NamedTuple):
    """Outputs of norm_gate_residual; None where nothing was asked for."""
    residual: torch.Tensor
    normed: Optional[torch.Tensor]
    codes: Optional[torch.Tensor]
    scales: Optional[torch.Tensor]


def norm_gate_residual(y: Optional[torch.Tensor], residual: torch.Tensor, *, post_weight: Optional[torch.Tensor] = None,
                       gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0, pre_weight: Optional[torch.Tensor] = None,
                       eps: float = 1e-6, weight_offset: float = 0.0, quant: Optional[str] = None, out_normed: bool = True,
                       out_codes: Optional[torch.Tensor] = None, out_scales: Optional[torch.Tensor] = None) -> NormOutputs:
    """What stands between two blocks of a model, in one pass over [T, H]:

        residual' = residual_scale * residual + gate * RMSNorm(y; post_weight)
        normed    = RMSNorm(residual'; pre_weight)          (and its e4m3 codes)

    with RMSNorm(v; w) = v * rsqrt(mean v^2 + eps) * (w + weight_offset).  y is the block's output; without it (before the first block)
    the residual is only normed and returned as it is.  Without post_weight y is not normed, without gate it is not gated, without
    pre_weight (after the last block) nothing but residual' comes back.  gate is [H], [T, 1] or [T, H].  quant: None, "block128" (scales
    [T, ceil(H/128)], for the products of this module) or "channelwise" (scales [T], as `fp8_mega_moe` reads them; out_codes and
    out_scales may be views of a SymmBuffer, `sb.x[:T]` and `sb.x_sf[:T]`).

    y, residual, weights and gate are bf16, fp16 or fp32, each in its own type; residual' has residual's type, normed is bf16 (fp32 where
    residual is fp16, never narrower than the range of the stream).  Arithmetic is fp32 throughout and each output is rounded once.  H is a
    multiple of 8, at most 16384."""
    name = "norm_gate_residual"
    index = _device_index(name, residual, y, post_weight, gate, pre_weight, out_codes, out_scales)
    if residual.dim() != 2:
        raise ValueError(f"{name} expects a residual [T, H]")
    t, h = residual.shape
    if h == 0 or h % 8 != 0 or h > 16384:
        raise ValueError(f"{name}: H must be a multiple of 8, at most 16384")
    if t >= _DIM:
        raise ValueError(f"{name}: at most 2^31 - 1 tokens")
    if y is None:
        if post_weight is not None or gate is not None or residual_scale != 1.0:
            raise ValueError(f"{name}: post_weight, gate and residual_scale need y")
    elif y.shape != (t, h):
        raise ValueError(f"{name}: y must be [{t}, {h}]")
    quant_kind = _QUANT.get(quant)
    if quant_kind is None:
        raise ValueError(f"{name}: quant must be None, 'block128' or 'channelwise'")
    if quant_kind == 0:
        if out_codes is not None or out_scales is not None:
            raise ValueError(f"{name}: out_codes and out_scales need quant")
    elif pre_weight is None:
        raise ValueError(f"{name}: codes need pre_weight")
    r_kind = _type_of(name, residual)
    y_kind = gate_kind = post_kind = pre_kind = normed_kind = gate_rows = gate_cols = 0
    y_ptr = post_ptr = gate_ptr = pre_ptr = normed_ptr = codes_ptr = scales_ptr = new_ptr = None
    y_stride = h
    r, r_stride = _rows_of(residual, 16)
    residual_out = residual
    if y is not None:
        y_kind = _type_of(name, y)
        y, y_stride = _rows_of(y, 16)
        y_ptr = y.data_ptr()
        residual_out = torch.empty_like(residual, memory_format=torch.contiguous_format)
        new_ptr = residual_out.data_ptr()
        if post_weight is not None:
            post_weight, post_kind = _norm_weight(name, post_weight, h)
            post_ptr = post_weight.data_ptr()
        if gate is not None:
            gate_kind = _type_of(name, gate)
            shape = gate.shape
            if gate.dim() == 1 and shape[0] == h:                    # (as it is: a view would take a microsecond)
                gate, gate_cols = _dense(gate, 16), 1
            elif gate.dim() == 2 and shape[0] in (1, t) and shape[1] in (1, h):
                if shape[1] == h:
                    (gate, gate_rows), gate_cols = _rows_of(gate, 16), 1
                else:
                    gate_rows = gate.stride(0)
                if shape[0] == 1:
                    gate_rows = 0
            elif gate.dim() != 1 or shape[0] != 1:                   # [1]: one number for all
                raise ValueError(f"{name}: gate must be [{h}], [{t}, 1] or [{t}, {h}]")
            gate_ptr = gate.data_ptr()
    normed = codes = scales = None
    if pre_weight is not None:
        pre_weight, pre_kind = _norm_weight(name, pre_weight, h)
        pre_ptr = pre_weight.data_ptr()
        if out_normed:
            normed = torch.empty_like(residual, dtype=torch.float32 if r_kind == 1 else torch.bfloat16, memory_format=torch.contiguous_format)
            normed_ptr, normed_kind = normed.data_ptr(), 2 if r_kind == 1 else 0
        if quant_kind:
            sf_shape = (t, (h + 127) // 128) if quant_kind == 1 else (t,)
            if out_codes is None:
                codes = torch.empty_like(residual, dtype=_E4M3, memory_format=torch.contiguous_format)
            else:
                codes = out_codes
                if codes.dtype != _E4M3 or codes.shape != (t, h) or not codes.is_contiguous() or codes.data_ptr() % 8 != 0:
                    raise ValueError(f"{name}: out_codes must be a contiguous e4m3 [{t}, {h}], 8-byte aligned")
            if out_scales is None:
                scales = residual.new_empty(sf_shape, dtype=torch.float32)
            else:
                scales = out_scales
                if scales.dtype != torch.float32 or scales.shape != sf_shape or not scales.is_contiguous():
                    raise ValueError(f"{name}: out_scales must be a contiguous float32 {list(sf_shape)}")
            codes_ptr, scales_ptr = codes.data_ptr(), scales.data_ptr()
        if normed is None and codes is None:
            pre_ptr = None
    if t and (y is not None or pre_ptr is not None):
        _call(index, _lib.lib().mm_norm_gate_residual, y_ptr, y_kind, y_stride, r.data_ptr(), r_kind, r_stride, post_ptr, post_kind, gate_ptr,
              gate_kind, gate_rows, gate_cols, pre_ptr, pre_kind, new_ptr, normed_ptr, normed_kind, codes_ptr, scales_ptr, quant_kind, t, h,
              residual_scale, eps, weight_offset)
    return NormOutputs(residual_out, normed, codes, scales)


_QUANT = {None: 0, "block128": 1, "channelwise": 2}


def _type_of(name: str, t: torch.Tensor) -> int:
    kind = _TYPES.get(t.dtype)
    if kind is None:
        raise TypeError(f"{name} expects bfloat16, float16 or float32 tensors")
    return kind


def _norm_weight(name: str, w: torch.Tensor, h: int) -> Tuple[torch.Tensor, int]:
    if w.shape != (h,):
        raise ValueError(f"{name}: norm weights must be [{h}]")
    return _dense(w, 16), _type_of(name, w)
