// Casts to e4m3 with one fp32 scale for each block of 128 values, and the fused norms between two blocks of a model.
//
// Cast:  top = max(max |x|, 1e-4) over the 128 values of a row (weights: over 128 x 128),  sf = top / 448,
//        q = e4m3_rne(448 x / top).
// The quotient is the correctly rounded one wherever it matters: 16-bit values lie exactly half way between two codes often
// (x and top have 8-bit mantissas), and a quotient that is one rounding off takes the wrong code there, one code step
// (2^-3) of error.  x * (448 / top) alone is not enough; one residual step makes it so (Markstein, "Computation of elementary
// functions on the IBM RISC System/6000 processor", 1990): with a = 448 x and q0 near a / top, the residual r = fma(-q0, top, a)
// is exact and fma(r, 1 / top, q0) rounds a value that is off by (a / top - q0) times the reciprocal's error only.
// A group that holds an infinity or a NaN gets NaN codes and a scale that is not finite, so that it cannot pass unseen.  (Where the codes are
// of values that were computed here, quantise_computed, a group with an infinity has the NaN code for that value alone and 0 for its
// finite ones; the scale is infinite, so products with the group are NaN all the same.)
//
// All of this is bound by HBM: one read of the inputs, one write of the outputs, everything between in registers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include "pack.cuh"

namespace mm {

enum { B128_BF16 = 0, B128_FP16 = 1, B128_FP32 = 2 };

// Eight neighbouring values of a row, as four pairs for the two-wide fp32 instructions: these kernels have a budget of some ten
// instructions per value before they are bound by them and not by HBM.
struct F8 { uint64_t v[4]; };

__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) { uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) { uint64_t r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
// maximum that is NaN if either operand is
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

__device__ __forceinline__ float amax8(const F8& x) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpair(x.v[i]);
        m = max_nan(m, max_nan(fabsf(f.x), fabsf(f.y)));
    }
    return m;
}
__device__ __forceinline__ float half_warp_max(float m) {   // over the 16 lanes that hold one group
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}
__device__ __forceinline__ float group_top(float amax) { return max_nan(amax, 1.0e-4f); }
// top / 448, correctly rounded: the quotient by the reciprocal and one residual step, as below
__device__ __forceinline__ float group_scale(float top) {
    constexpr float inv = 1.0f / 448.0f;
    const float s = top * inv;
    return top < INFINITY ? fmaf(fmaf(-s, 448.0f, top), inv, s) : top;
}
__device__ __forceinline__ float rcp_approx(float x) { float r; asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

__device__ __forceinline__ uint2 to_e4m3(const F8& x) {
    const float2 a = unpair(x.v[0]), b = unpair(x.v[1]), c = unpair(x.v[2]), d = unpair(x.v[3]);
    return make_uint2(pack4_e4m3(a.x, a.y, b.x, b.y), pack4_e4m3(c.x, c.y, d.x, d.y));
}
// Codes of values as they were given: 448 x / top, the correctly rounded quotient (see above).  448 x = 512 (7/8 x), and top / 512 is exact.
__device__ __forceinline__ uint2 quantise_exact(const F8& x, float top) {
    const float divisor = top * (1.0f / 512.0f), inv = rcp_approx(divisor), first = 0.875f * inv;
    const uint64_t d2 = pair(-divisor, -divisor), i2 = pair(inv, inv), f2 = pair(first, first), e2 = pair(0.875f, 0.875f);
    F8 q;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint64_t q0 = mul2(x.v[i], f2);
        q.v[i] = fma2(fma2(q0, d2, mul2(x.v[i], e2)), i2, q0);
    }
    return to_e4m3(q);
}
// Codes of values that were computed in fp32: none of them lies half way between two codes but by chance, so one multiplication by
// 448 / top does (2^-23 off, which moves one code in a million).
__device__ __forceinline__ uint2 quantise_computed(const F8& x, float mul) {
    const uint64_t m2 = pair(mul, mul);
    F8 q;
#pragma unroll
    for (int i = 0; i < 4; ++i) q.v[i] = mul2(x.v[i], m2);
    return to_e4m3(q);
}

// eight neighbouring elements (16-byte aligned); the type is known when the kernel is compiled, or (kAny) the same for a whole launch
constexpr int kAny = -1;
struct Raw8 { uint4 a, b; };                 // as they were loaded (b: fp32 only)
template <int kType>
__device__ __forceinline__ Raw8 fetch8(const void* p, int64_t i, int type) {
    Raw8 r;
    r.b = make_uint4(0, 0, 0, 0);
    if (kType == B128_FP32 || (kType == kAny && type == B128_FP32)) {
        r.a = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i)[0];
        r.b = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i)[1];
    } else {
        r.a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    }
    return r;
}
template <int kType>
__device__ __forceinline__ F8 values8(const Raw8& r, int type) {
    F8 x;
    const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
    if (kType == B128_FP32 || (kType == kAny && type == B128_FP32)) {
        x.v[0] = pair(__uint_as_float(r.a.x), __uint_as_float(r.a.y)); x.v[1] = pair(__uint_as_float(r.a.z), __uint_as_float(r.a.w));
        x.v[2] = pair(__uint_as_float(r.b.x), __uint_as_float(r.b.y)); x.v[3] = pair(__uint_as_float(r.b.z), __uint_as_float(r.b.w));
        return x;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (kType == B128_BF16 || (kType == kAny && type == B128_BF16)) {
            x.v[j] = pair(bf16_lo(w[j]), bf16_hi(w[j]));
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
            x.v[j] = pair(f.x, f.y);
        }
    }
    return x;
}
template <int kType>
__device__ __forceinline__ F8 load8(const void* p, int64_t i, int type) { return values8<kType>(fetch8<kType>(p, i, type), type); }
__device__ __forceinline__ float load1(const void* p, int64_t i, int type) {
    if (type == B128_FP32) return static_cast<const float*>(p)[i];
    if (type == B128_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}
template <int kType>
__device__ __forceinline__ void store8(void* p, int64_t i, int type, const F8& x) {
    if (kType == B128_FP32 || (kType == kAny && type == B128_FP32)) {
        float4* o = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
        const float2 a = unpair(x.v[0]), b = unpair(x.v[1]), c = unpair(x.v[2]), d = unpair(x.v[3]);
        o[0] = make_float4(a.x, a.y, b.x, b.y);
        o[1] = make_float4(c.x, c.y, d.x, d.y);
        return;
    }
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 f = unpair(x.v[j]);
        if (kType == B128_BF16 || (kType == kAny && type == B128_BF16)) {
            w[j] = pack_bf16x2(f.x, f.y);
        } else {
            const __half2 h = __floats2half2_rn(f.x, f.y);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ F8 zero8() { return F8{{0ull, 0ull, 0ull, 0ull}}; }

// Rows of activations: 16 lanes hold one group of 128 values, 8 each, and each lane has kCastGroups groups in flight.  kFlat: whole groups
// and dense rows, so that a group's place is its number (the division by groups per row costs as much as the rest of a group's addresses).
constexpr int kCastGroups = 4;

template <int kType, bool kFlat>
__global__ void __launch_bounds__(256) cast_block128_kernel(const void* x, int64_t row_stride, uint32_t groups, uint32_t groups_per_row,
                                                            int k, uint8_t* q, float* sf) {      // (no __restrict__: a load that counts as invariant could pass pdl_wait)
    pdl_launch();
    pdl_wait();
    const uint32_t lane16 = threadIdx.x & 15;
    const uint32_t first = blockIdx.x * (16 * kCastGroups) + (threadIdx.x >> 4);
    F8 v[kCastGroups];
    int64_t out[kCastGroups];
#pragma unroll
    for (int i = 0; i < kCastGroups; ++i) {
        const uint32_t g = first + i * 16;
        int64_t in;
        if (kFlat) {
            in = static_cast<int64_t>(g) * 128 + lane16 * 8;
            out[i] = g < groups ? in : -1;
        } else {
            const uint32_t row = g / groups_per_row;
            const int col = static_cast<int>(g - row * groups_per_row) * 128 + static_cast<int>(lane16) * 8;
            in = row * row_stride + col;
            out[i] = g < groups && col < k ? static_cast<int64_t>(row) * k + col : -1;
        }
        v[i] = zero8();
        if (out[i] >= 0) v[i] = load8<kType>(x, in, kType);
    }
#pragma unroll
    for (int i = 0; i < kCastGroups; ++i) {
        const uint32_t g = first + i * 16;
        const float top = group_top(half_warp_max(amax8(v[i])));
        if (out[i] >= 0) *reinterpret_cast<uint2*>(q + out[i]) = quantise_exact(v[i], top);
        if (lane16 == 0 && g < groups) sf[g] = group_scale(top);
    }
}

// Weights: one block of 128 x 128 for each thread block, held in registers between the maximum and the codes.
template <int kType>
__global__ void __launch_bounds__(256) cast_weight_block128_kernel(const void* __restrict__ w, int rows, int k, int row_blocks, int k_blocks,
                                                                   uint8_t* __restrict__ q, float* __restrict__ sf) {
    __shared__ float s_max[8];
    const int warp = threadIdx.x >> 5, lane16 = threadIdx.x & 15;
    const int64_t b = blockIdx.x;                                // [expert][row block][k block]
    const int kb = static_cast<int>(b % k_blocks);
    const int64_t rest = b / k_blocks;
    const int rb = static_cast<int>(rest % row_blocks);
    const int64_t base = (rest / row_blocks) * rows * static_cast<int64_t>(k);
    const int col = kb * 128 + lane16 * 8;
    F8 v[8];
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = rb * 128 + i * 16 + (threadIdx.x >> 4);
        v[i] = zero8();
        if (row < rows && col < k) v[i] = load8<kType>(w, base + static_cast<int64_t>(row) * k + col, kType);
        m = max_nan(m, amax8(v[i]));
    }
    m = half_warp_max(m);
    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 16));
    if ((threadIdx.x & 31) == 0) s_max[warp] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max_nan(m, s_max[i]);
    const float top = group_top(m);
    if (threadIdx.x == 0) sf[b] = group_scale(top);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = rb * 128 + i * 16 + (threadIdx.x >> 4);
        if (row < rows && col < k) *reinterpret_cast<uint2*>(q + base + static_cast<int64_t>(row) * k + col) = quantise_exact(v[i], top);
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

// Sum or maximum over the block; s: 32 words, zero behind the block's warps (which changes neither a sum nor a maximum of magnitudes),
// written again only behind another barrier.
template <typename Op>
__device__ __forceinline__ float block_reduce(float v, float* s, Op op) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (warps == 1) return v;
    if (lane == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
    for (int w = 0; w < warps; w += 4) {                         // broadcast reads, the same order in every thread
        const float4 f = *reinterpret_cast<const float4*>(s + w);
        v = op(v, op(op(f.x, f.y), op(f.z, f.w)));
    }
    return v;
}
__device__ __forceinline__ float squares(const F8& x, float before) {
    uint64_t a = pair(before, 0.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) a = fma2(x.v[i], x.v[i], a);
    const float2 f = unpair(a);
    return f.x + f.y;
}

constexpr int kNormMaxHidden = 16384;

// One row per block at a time, kVec vectors of 8 values per thread (vector i of a thread is number i * blockDim + threadIdx of the row).
// The next row's values are loaded while this one is reduced.  kY, kR and kWeight: the types of y, of the residual, and of the weights
// and the gate, or kAny; with types of its own the normed output is bf16.
// kStaged: the weights of y (with a gate that is the same for all rows) and of r' are worked out once into shared memory.
// Measured at 8192 x 4096 in bf16 with codes by blocks: 55 us, 5.5 TB/s of the bytes it must move (a plain copy: 6.5); instructions and the
// three waits of a row share what is left.  With weights read and added up in every row 61; the first form, without the prefetch and the
// two-wide arithmetic either, took 107; one vector per thread 68, four 69, two rows at a time 60 to 76 (all three before staging).
// The same size with an fp32 stream: 86 us (436 MB, 5.0 TB/s).  With weights and gate in bf16, or any other types, kAny: 86 with a bf16 stream
// and weights, 88 with an fp32 stream, 102 in fp16; its two vectors a thread do not fit the 64 registers (488 bytes of spill stores), and
// neither do those of an fp32 stream above H = 8192 (2400 x 16384: 154 us against 79 in bf16).
template <int kVec, int kY, int kR, int kWeight, bool kStaged>
__global__ void __launch_bounds__(1024) norm_gate_residual_kernel(const __grid_constant__ NormParams p) {
    pdl_launch();
    __shared__ __align__(16) float s_sum[3][32];
    extern __shared__ __align__(16) float s_weight[];                // kStaged: [2][hidden], of y and of r'
    const int vecs = p.hidden >> 3;
    const float inv_h = 1.0f / static_cast<float>(p.hidden);
    const auto add = [](float a, float b) { return a + b; };
    const uint64_t offset2 = pair(p.offset, p.offset), alpha2 = pair(p.alpha, p.alpha);
    for (int i = threadIdx.x; i < 3 * 32; i += blockDim.x) (&s_sum[0][0])[i] = 0.0f;
    pdl_wait();
    const bool channel_gate = p.gate != nullptr && p.gate_col_stride && p.gate_row_stride == 0;
    const bool staged_y = kStaged && (p.post != nullptr || channel_gate);
    if (kStaged) {
        for (int v = threadIdx.x; v < vecs; v += blockDim.x) {
            F8 w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w.v[j] = pair(1.0f, 1.0f);
            if (p.post != nullptr) {
                w = load8<kWeight>(p.post, v * 8, p.w_post_type);
#pragma unroll
                for (int j = 0; j < 4; ++j) w.v[j] = add2(w.v[j], offset2);
            }
            if (channel_gate) {
                const F8 g = load8<kWeight>(p.gate, v * 8, p.gate_type);
#pragma unroll
                for (int j = 0; j < 4; ++j) w.v[j] = mul2(w.v[j], g.v[j]);
            }
            store8<B128_FP32>(s_weight, v * 8, B128_FP32, w);
            if (p.pre != nullptr) {
                w = load8<kWeight>(p.pre, v * 8, p.w_pre_type);
#pragma unroll
                for (int j = 0; j < 4; ++j) w.v[j] = add2(w.v[j], offset2);
                store8<B128_FP32>(s_weight, p.hidden + v * 8, B128_FP32, w);
            }
        }
    }
    __syncthreads();
    Raw8 y_next[kVec], r_next[kVec];
    auto fetch = [&](int row) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const int v = i * blockDim.x + threadIdx.x;
            r_next[i].a = r_next[i].b = y_next[i].a = y_next[i].b = make_uint4(0, 0, 0, 0);
            if (row >= p.tokens || v >= vecs) continue;
            r_next[i] = fetch8<kR>(p.r, row * p.r_stride + v * 8, p.r_type);
            if (p.y != nullptr) y_next[i] = fetch8<kY>(p.y, row * p.y_stride + v * 8, p.y_type);
        }
    };
    fetch(blockIdx.x);
    for (int64_t row = blockIdx.x; row < p.tokens; row += gridDim.x) {
        F8 r[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) r[i] = values8<kR>(r_next[i], p.r_type);
        if (p.y != nullptr) {
            F8 y[kVec];
#pragma unroll
            for (int i = 0; i < kVec; ++i) y[i] = values8<kY>(y_next[i], p.y_type);
            fetch(static_cast<int>(min(row + gridDim.x, static_cast<int64_t>(p.tokens))));
            float n = 1.0f;
            if (p.post != nullptr) {
                float sq = 0.0f;
#pragma unroll
                for (int i = 0; i < kVec; ++i) sq = squares(y[i], sq);
                n = rsqrtf(fmaf(block_reduce(sq, s_sum[0], add), inv_h, p.eps));
            }
            if (p.gate != nullptr && !p.gate_col_stride) n *= load1(p.gate, row * p.gate_row_stride, p.gate_type);
            const uint64_t n2 = pair(n, n);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                const int v = i * blockDim.x + threadIdx.x;
                if (v >= vecs) continue;
                if (staged_y) {
                    const F8 w = load8<B128_FP32>(s_weight, v * 8, B128_FP32);
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[i].v[j] = mul2(y[i].v[j], w.v[j]);
                }
                if (!kStaged && p.post != nullptr) {
                    const F8 w = load8<kWeight>(p.post, v * 8, p.w_post_type);
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[i].v[j] = mul2(y[i].v[j], add2(w.v[j], offset2));
                }
                if (p.gate != nullptr && p.gate_col_stride && !(kStaged && channel_gate)) {
                    const F8 g = load8<kWeight>(p.gate, row * p.gate_row_stride + v * 8, p.gate_type);
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[i].v[j] = mul2(y[i].v[j], g.v[j]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) r[i].v[j] = fma2(y[i].v[j], n2, mul2(r[i].v[j], alpha2));
                store8<kR>(p.r_out, row * p.hidden + v * 8, p.r_type, r[i]);
            }
        } else {
            fetch(static_cast<int>(min(row + gridDim.x, static_cast<int64_t>(p.tokens))));
        }
        if (p.pre != nullptr) {
            float sq = 0.0f;
#pragma unroll
            for (int i = 0; i < kVec; ++i) sq = squares(r[i], sq);
            const float n = rsqrtf(fmaf(block_reduce(sq, s_sum[1], add), inv_h, p.eps));
            const uint64_t n2 = pair(n, n);
            float row_max = 0.0f;
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                const int v = i * blockDim.x + threadIdx.x;
                const int64_t at = row * p.hidden + v * 8;
                if (v < vecs) {
                    F8 w;
                    if (kStaged) {
                        w = load8<B128_FP32>(s_weight, p.hidden + v * 8, B128_FP32);
                    } else {
                        w = load8<kWeight>(p.pre, v * 8, p.w_pre_type);
#pragma unroll
                        for (int j = 0; j < 4; ++j) w.v[j] = add2(w.v[j], offset2);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) r[i].v[j] = mul2(mul2(r[i].v[j], n2), w.v[j]);
                    if (p.x_out != nullptr) store8<kY == kAny ? kAny : B128_BF16>(p.x_out, at, p.x_type, r[i]);
                }
                if (p.quant == 1) {                  // 16 neighbouring threads hold one group
                    const float top = group_top(half_warp_max(amax8(r[i])));
                    if (v < vecs) {
                        *reinterpret_cast<uint2*>(p.q + at) = quantise_computed(r[i], 448.0f * rcp_approx(top));
                        if ((threadIdx.x & 15) == 0) p.sf[row * ((p.hidden + 127) / 128) + v / 16] = group_scale(top);
                    }
                } else if (p.quant == 2) {
                    row_max = max_nan(row_max, amax8(r[i]));
                }
            }
            if (p.quant == 2) {
                const float top = group_top(block_reduce(row_max, s_sum[2], max_nan)), mul = 448.0f * rcp_approx(top);
                if (threadIdx.x == 0) p.sf[row] = group_scale(top);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    const int v = i * blockDim.x + threadIdx.x;
                    if (v < vecs) *reinterpret_cast<uint2*>(p.q + row * p.hidden + v * 8) = quantise_computed(r[i], mul);
                }
            }
        }
        __syncthreads();                             // the next row's first reduction writes s_sum[0] again
    }
}

}  // namespace mm
