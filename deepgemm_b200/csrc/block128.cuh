// Casts to e4m3 with one fp32 scale for each block of 128 values, and the fused norms between two blocks of a model.
//
// Cast:  top = max(max |x|, 1e-4) over the 128 values of a row (weights: over 128 x 128),  sf = top / 448,
//        q = e4m3_rne(448 x / top).
// The quotient is the correctly rounded one wherever it matters: 16-bit values lie exactly half way between two codes often
// (x and top have 8-bit mantissas), and a quotient that is one rounding off takes the wrong code there, one code step
// (2^-3) of error.  x * (1 / top) alone is not enough; one residual step makes it so (Markstein, "Computation of elementary
// functions on the IBM RISC System/6000 processor", 1990): r = fma(-q0, top, a) is exact, q1 = fma(r, 1 / top, q0).  The
// numerator is taken as 7/8 x, exact for 16-bit inputs and free of overflow, and the missing 512 is a power of two.
// A group that holds an infinity or a NaN gets NaN codes and a scale that is not finite, so that it cannot pass unseen.
//
// All of this is bound by HBM: one read of the inputs, one write of the outputs, everything between in registers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include "pack.cuh"

namespace mm {

enum { B128_BF16 = 0, B128_FP16 = 1, B128_FP32 = 2 };

// |x| as an integer orders like |x| and puts NaN above infinity, so an integer maximum keeps both.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ float group_top(uint32_t amax_bits) {
    return __uint_as_float(max(amax_bits, __float_as_uint(1.0e-4f)));
}

// 448 x / top for several x of one group
struct GroupQuotient {
    float top, inv;
    __device__ __forceinline__ explicit GroupQuotient(float t) : top(t), inv(1.0f / t) {}
    __device__ __forceinline__ float operator()(float x) const {
        const float a = 0.875f * x;
        const float q0 = a * inv;
        const float q1 = fmaf(fmaf(-q0, top, a), inv, q0);
        return q1 * 512.0f;
    }
};

__device__ __forceinline__ uint2 quantise8(const float (&v)[8], const GroupQuotient& g) {
    return make_uint2(pack4_e4m3(g(v[0]), g(v[1]), g(v[2]), g(v[3])), pack4_e4m3(g(v[4]), g(v[5]), g(v[6]), g(v[7])));
}
__device__ __forceinline__ uint32_t amax8(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[i]));
    return m;
}
__device__ __forceinline__ uint32_t half_warp_max(uint32_t m) {   // over the 16 lanes that hold one group
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}

// eight neighbouring elements (16-byte aligned) as floats; the type is the same for a whole launch
__device__ __forceinline__ void load8(const void* p, int64_t i, int type, float (&v)[8]) {
    if (type == B128_FP32) {
        const float4 a = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i)[0];
        const float4 b = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        return;
    }
    const uint4 d = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    const uint32_t w[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (type == B128_BF16) {
            v[2 * j] = bf16_lo(w[j]); v[2 * j + 1] = bf16_hi(w[j]);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
            v[2 * j] = f.x; v[2 * j + 1] = f.y;
        }
    }
}
__device__ __forceinline__ float load1(const void* p, int64_t i, int type) {
    if (type == B128_FP32) return static_cast<const float*>(p)[i];
    if (type == B128_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store8(void* p, int64_t i, int type, const float (&v)[8]) {
    if (type == B128_FP32) {
        float4* o = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
        o[0] = make_float4(v[0], v[1], v[2], v[3]);
        o[1] = make_float4(v[4], v[5], v[6], v[7]);
        return;
    }
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (type == B128_BF16) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&b);
        } else {
            const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Rows of activations: 16 lanes hold one group of 128 values, 8 each.
template <int kType>
__global__ void __launch_bounds__(256) cast_block128_kernel(const void* __restrict__ x, int64_t row_stride, uint32_t groups,
                                                            uint32_t groups_per_row, int k, uint8_t* __restrict__ q, float* __restrict__ sf) {
    const uint32_t lane16 = threadIdx.x & 15;
    const uint32_t first = (blockIdx.x * blockDim.x + threadIdx.x) >> 4;
    const uint32_t step = (gridDim.x * blockDim.x) >> 4;
    const uint32_t rounds = (groups + step - 1) / step;          // the same for every lane: the shuffles need whole warps
    for (uint32_t it = 0; it < rounds; ++it) {
        const uint32_t g = first + it * step;
        const uint32_t row = g / groups_per_row;
        const int col = static_cast<int>(g - row * groups_per_row) * 128 + static_cast<int>(lane16) * 8;
        const bool ok = g < groups && col < k;
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (ok) load8(x, static_cast<int64_t>(row) * row_stride + col, kType, v);
        const float top = group_top(half_warp_max(amax8(v)));
        if (ok) *reinterpret_cast<uint2*>(q + static_cast<int64_t>(row) * k + col) = quantise8(v, GroupQuotient(top));
        if (lane16 == 0 && g < groups) sf[g] = __fdiv_rn(top, 448.0f);
    }
}

// Weights: one block of 128 x 128 for each thread block, held in registers between the maximum and the codes.
template <int kType>
__global__ void __launch_bounds__(256) cast_weight_block128_kernel(const void* __restrict__ w, int rows, int k, int row_blocks, int k_blocks,
                                                                   uint8_t* __restrict__ q, float* __restrict__ sf) {
    __shared__ uint32_t s_max[8];
    const int warp = threadIdx.x >> 5, lane16 = threadIdx.x & 15;
    const int64_t b = blockIdx.x;                                // [expert][row block][k block]
    const int kb = static_cast<int>(b % k_blocks);
    const int64_t rest = b / k_blocks;
    const int rb = static_cast<int>(rest % row_blocks);
    const int64_t base = (rest / row_blocks) * rows * static_cast<int64_t>(k);
    const int col = kb * 128 + lane16 * 8;
    float v[8][8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = rb * 128 + i * 16 + (threadIdx.x >> 4);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
        if (row < rows && col < k) load8(w, base + static_cast<int64_t>(row) * k + col, kType, v[i]);
        m = max(m, amax8(v[i]));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) s_max[warp] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, s_max[i]);
    const float top = group_top(m);
    const GroupQuotient g(top);
    if (threadIdx.x == 0) sf[b] = __fdiv_rn(top, 448.0f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = rb * 128 + i * 16 + (threadIdx.x >> 4);
        if (row < rows && col < k) *reinterpret_cast<uint2*>(q + base + static_cast<int64_t>(row) * k + col) = quantise8(v[i], g);
    }
}

// Between two blocks of a model, one pass over the row:
//   r' = alpha r + gate * (y * rsqrt(mean y^2 + eps) * (w_post + offset)),   x = r' * rsqrt(mean r'^2 + eps) * (w_pre + offset),
//   codes of x with a scale for each 128 values or for the row.
// Every part is optional; all arithmetic is fp32 and every output is rounded once, from the unrounded r' and x.
struct NormParams {
    const void* y; const void* r; const void* post; const void* pre; const void* gate;      // y, post, pre, gate may be null
    void* r_out; void* x_out; uint8_t* q; float* sf;                                        // each may be null
    int y_type, r_type, w_post_type, w_pre_type, gate_type, x_type;
    int64_t y_stride, r_stride, gate_row_stride;
    int gate_col_stride;                                                                    // 0 or 1
    int tokens, hidden, quant;                                                              // quant: 0 none, 1 by 128, 2 by row
    float alpha, eps, offset;
};

// maximum or sum over the block; s: one word for each warp, reused behind the second barrier
template <typename T, typename Op>
__device__ __forceinline__ T block_reduce(T v, T* s, Op op) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (warps == 1) return v;
    if (lane == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    T out = lane < warps ? s[lane] : T(0);       // 0 is neutral: sums, and maxima of unsigned numbers
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) out = op(out, __shfl_xor_sync(0xffffffffu, out, o));
    return out;
}

// One row per block, kVec vectors of 8 values per thread (vector i of a thread is number i * blockDim + threadIdx of the row).
template <int kVec>
__global__ void __launch_bounds__(1024) norm_gate_residual_kernel(NormParams p) {
    __shared__ float s_sum[3][32];
    const int vecs = p.hidden >> 3;
    const float inv_h = 1.0f / static_cast<float>(p.hidden);
    const auto add = [](float a, float b) { return a + b; };
    const auto umax = [](uint32_t a, uint32_t b) { return max(a, b); };
    for (int row = blockIdx.x; row < p.tokens; row += gridDim.x) {
        float r[kVec][8];
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const int v = i * blockDim.x + threadIdx.x;
#pragma unroll
            for (int j = 0; j < 8; ++j) r[i][j] = 0.0f;
            if (v < vecs) load8(p.r, static_cast<int64_t>(row) * p.r_stride + v * 8, p.r_type, r[i]);
        }
        if (p.y != nullptr) {
            float y[kVec][8];
            float sq = 0.0f;
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                const int v = i * blockDim.x + threadIdx.x;
#pragma unroll
                for (int j = 0; j < 8; ++j) y[i][j] = 0.0f;
                if (v < vecs) load8(p.y, static_cast<int64_t>(row) * p.y_stride + v * 8, p.y_type, y[i]);
#pragma unroll
                for (int j = 0; j < 8; ++j) sq = fmaf(y[i][j], y[i][j], sq);
            }
            if (p.post != nullptr) {
                sq = block_reduce(sq, s_sum[0], add);
                const float n = rsqrtf(fmaf(sq, inv_h, p.eps));
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    const int v = i * blockDim.x + threadIdx.x;
                    if (v >= vecs) continue;
                    float w[8];
                    load8(p.post, v * 8, p.w_post_type, w);
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[i][j] = y[i][j] * n * (w[j] + p.offset);
                }
            }
            if (p.gate != nullptr) {
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    const int v = i * blockDim.x + threadIdx.x;
                    if (v >= vecs) continue;
                    float g[8];
                    if (p.gate_col_stride) {
                        load8(p.gate, row * p.gate_row_stride + v * 8, p.gate_type, g);
                    } else {
                        const float one = load1(p.gate, row * p.gate_row_stride, p.gate_type);
#pragma unroll
                        for (int j = 0; j < 8; ++j) g[j] = one;
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[i][j] *= g[j];
                }
            }
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                const int v = i * blockDim.x + threadIdx.x;
#pragma unroll
                for (int j = 0; j < 8; ++j) r[i][j] = fmaf(p.alpha, r[i][j], y[i][j]);
                if (v < vecs && p.r_out != nullptr) store8(p.r_out, static_cast<int64_t>(row) * p.hidden + v * 8, p.r_type, r[i]);
            }
        }
        if (p.pre != nullptr) {
            float sq = 0.0f;
#pragma unroll
            for (int i = 0; i < kVec; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) sq = fmaf(r[i][j], r[i][j], sq);
            sq = block_reduce(sq, s_sum[1], add);
            const float n = rsqrtf(fmaf(sq, inv_h, p.eps));
            uint32_t row_max = 0;
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                const int v = i * blockDim.x + threadIdx.x;
                if (v < vecs) {
                    float w[8];
                    load8(p.pre, v * 8, p.w_pre_type, w);
#pragma unroll
                    for (int j = 0; j < 8; ++j) r[i][j] = r[i][j] * n * (w[j] + p.offset);
                    if (p.x_out != nullptr) store8(p.x_out, static_cast<int64_t>(row) * p.hidden + v * 8, p.x_type, r[i]);
                }
                if (p.quant == 1) {                  // 16 neighbouring threads hold one group
                    const float top = group_top(half_warp_max(amax8(r[i])));
                    if (v < vecs) {
                        *reinterpret_cast<uint2*>(p.q + static_cast<int64_t>(row) * p.hidden + v * 8) = quantise8(r[i], GroupQuotient(top));
                        if ((threadIdx.x & 15) == 0) p.sf[static_cast<int64_t>(row) * ((p.hidden + 127) / 128) + v / 16] = __fdiv_rn(top, 448.0f);
                    }
                } else if (p.quant == 2) {
                    row_max = max(row_max, amax8(r[i]));
                }
            }
            if (p.quant == 2) {
                row_max = block_reduce(row_max, reinterpret_cast<uint32_t*>(s_sum[2]), umax);
                const float top = group_top(row_max);
                const GroupQuotient g(top);
                if (threadIdx.x == 0) p.sf[row] = __fdiv_rn(top, 448.0f);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    const int v = i * blockDim.x + threadIdx.x;
                    if (v < vecs) *reinterpret_cast<uint2*>(p.q + static_cast<int64_t>(row) * p.hidden + v * 8) = quantise8(r[i], g);
                }
            }
        }
        __syncthreads();                             // the next row's first reduction writes s_sum[0] again
    }
}

}  // namespace mm
