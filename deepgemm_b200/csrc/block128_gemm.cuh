// Products of e4m3 operands with a scale for each block of 128 (tcgen05, accumulators in TMEM, operands by TMA).
//
//   d[m, n] = sum over kb of ( sum over k in block kb of a[m, k] b[e][n, k] ) * sa[m, kb] * sb[e][n / 128, kb]
//
// The tensor core sums one block of 128 k exactly as it would any product; the scales change from block to block, so each
// block's accumulator is read back from TMEM, multiplied and added to fp32 sums in registers, while the tensor core works on
// the next block in another TMEM buffer.  For a 128 x 256 tile that is 32768 values for each 512 cycles of MMA at the e4m3
// rate: 8 epilogue warps hold 128 sums per thread.
//
// One CTA per SM, 384 threads: warp 0 = TMA, warp 1 = MMA, warps 2-3 = scales, warps 4-11 = epilogue (registers moved to them).  The
// scales of a k block travel with its operands, copied to a ring of their own in shared memory: read from global memory by the epilogue
// they cost it an L2 latency now and then, and every cycle of the epilogue counts.
// What bounds it (8192 x 4096 x 4096: 137 us, 2.0 PFLOP/s, at the 1.54 GHz that the power cap leaves): 800 cycles for each of a CTA's 224 k
// blocks and 4200 for each of its seven tiles (K = 1024 to 8192 lie on that line).  An accumulator goes round through its MMAs (512), the
// promotion (520 to 600 of a warp) and two hand-overs (300); two accumulators share the way, so a block takes 690 to 790, above the 512 of the
// MMAs and the 675 of moving 48 KiB into and out of shared memory.  A tile's own 4200 are its beginning and its end: the warps that
// sum also store, 32 bytes a lane, and meanwhile the MMA warp is at most two blocks ahead.
// kSplit: the CTAs of a cluster share one tile and divide its k blocks; the fp32 parts meet in distributed shared memory
// and are added in rank order, so the result does not depend on timing.
#pragma once
#include <cuda_bf16.h>
#include "layout.h"
#include "pack.cuh"
#include "ptx.cuh"

namespace mm {

constexpr int kB128Threads = 384;
constexpr int kB128MaxSplit = 8;           // CTAs that share a tile: the largest portable cluster

struct B128GemmParams {
    int m, n, k_blocks;
    int m_tiles, n_tiles;              // of 128 rows and BN columns
    int a_box_rows;
    int n_sf;                          // 128-blocks of weight rows for each expert
    int experts;
    int tiled;                         // weights as [expert][n block][k block][256 rows][128]: a 2-D map, else [expert][n][k]: a 3-D map
    int tiled_n_blocks;
    const float* sa; int64_t sa_stride;        // [m][k_blocks]
    const float* sb;                           // [experts][n_sf][k_blocks]
    const int* m_indices;                      // grouped: expert of each row (-1: padding, not written), else null
    void* out; int64_t out_stride;             // elements
    int out_fp32;
    int out_vec32;                             // rows and base are multiples of 32 bytes
    int* status;
    uint64_t timeout_ns;
    int given_up;                              // CTA that counts as one whose wait has run out (mm_block128_test_waits), else -1
};

__device__ __forceinline__ void tma_load_3d(uint32_t smem_dst, const CUtensorMap* map, int32_t c0, int32_t c1, int32_t c2, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
}
__device__ __forceinline__ int ld_shared_volatile(uint32_t addr) {
    int v;
    asm volatile("ld.volatile.shared.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void st_shared_volatile(uint32_t addr, int v) { asm volatile("st.volatile.shared.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
// Bounded wait of one thread like mbar_wait, for hand-overs that follow one another every few hundred cycles: the clock is not read before
// the wait has failed a thousand times, because reading it costs more than such a hand-over.
__device__ __forceinline__ bool mbar_wait_often(uint32_t bar, uint32_t parity, uint32_t abort_flag, uint64_t timeout_ns) {
    uint64_t t0 = 0;
    for (uint32_t it = 1;; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 1023u) != 0u) continue;
        if (ld_shared_volatile(abort_flag) != 0) return false;
        const uint64_t t = global_timer_ns();
        if (t0 == 0) t0 = t;
        else if (t - t0 > timeout_ns) { st_shared_volatile(abort_flag, 1); return false; }
    }
}
// The same for a converged warp, with one answer for all of its lanes.  If each lane decided for itself, one could give up while another still
// sees the barrier complete, and what follows such a wait (tcgen05.ld, elect, votes, __syncwarp) needs all of them.  (A vote for "any failed",
// behind the loop: written as "all came", or inside the loop, it made 644 us of the layer's 128 tokens into 735 and 47 of one token into 54.)
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, uint32_t abort_flag, uint64_t timeout_ns) {
    const bool came = mbar_wait_often(bar, parity, abort_flag, timeout_ns);
    return !__any_sync(0xffffffffu, !came);
}
__device__ __forceinline__ float ld_shared_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
// threadIdx.x, read anew each time: what is kept beside the epilogue's 128 sums and 64 staged values makes it spill, and what can be worked
// out again is therefore not kept.
__device__ __forceinline__ int tid_again() {
    int t;
    asm volatile("mov.u32 %0, %%tid.x;" : "=r"(t));
    return t;
}
__device__ __forceinline__ bool elect_lane() {                        // one lane of a converged warp
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void mbar_arrive_n(uint32_t bar, uint32_t n) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(bar), "r"(n) : "memory");
}
template <int kRegs> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }

// Two fp32 sums at a time.
__device__ __forceinline__ uint64_t pack_f32x2(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ float2 unpack_f32x2(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
__device__ __forceinline__ float4 unpack_f32x4(uint64_t a, uint64_t b) {
    const float2 x = unpack_f32x2(a), y = unpack_f32x2(b);
    return make_float4(x.x, x.y, y.x, y.y);
}
__device__ __forceinline__ void fma_f32x2(uint64_t& acc, uint64_t a, uint64_t b) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(a), "l"(b));
}
__device__ __forceinline__ void st_global_32b(void* p, const uint32_t (&v)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
__device__ __forceinline__ float4 ld_shared_cluster_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ int ld_shared_cluster_s32(uint32_t addr) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

template <int kBN> struct B128Shape {
    static constexpr int kStages = kBN == 256 ? 4 : 6;
    static constexpr int kAccs = 512 / kBN;                          // TMEM accumulators in turn
    static constexpr int kABytes = 128 * 128;
    static constexpr int kBBytes = kBN * 128;
    static constexpr int kStageBytes = kABytes + kBBytes;
    // Scales of a k block: 128 rows, then two of the weights.  A stage is filled when the MMA that read it last is done; the epilogue
    // may be as many blocks behind that as there are accumulators, and one more.
    static constexpr int kScaleSlots = 16;
    static_assert(kScaleSlots >= kStages + kAccs + 1, "scale ring");
    static constexpr int kScaleBytes = 544;
    static constexpr int kStagingBytes = 8 * 32 * 17 * 4;            // a 32 x 16 fp32 piece for each epilogue warp
    static constexpr int kBarBytes = 256;
    static constexpr int kSmemBytes = kStages * kStageBytes + kScaleSlots * kScaleBytes + kStagingBytes + kBarBytes;
    static_assert(kSmemBytes <= 232448, "exceeds the 227 KiB of shared memory a CTA can have");
    static_assert(128 * (kBN + 4) * 4 <= kStages * kStageBytes, "the fp32 part of a split tile fits in the operand ring");
};

// Tile number -> (m tile, n tile): eight m tiles at a time run through all n tiles, so that the operands that CTAs of one wave
// read stay few.
__device__ __forceinline__ void b128_tile(const B128GemmParams& p, int tile, int& mt, int& nt) {
    const int per_group = 8 * p.n_tiles;
    const int g = tile / per_group, r = tile - g * per_group;
    const int gm = min(8, p.m_tiles - g * 8);
    nt = r / gm;
    mt = g * 8 + r - nt * gm;
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

// 32 lanes x 16 consecutive columns of 32-bit
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

// Adds one k block's accumulator (kCols columns of this warp's 32 lanes from `taddr` on) to the sums, times row_scale * weight_scale of its
// place in the ring of scales; then the tensor core may have the buffer back (`free_bar`).  16 columns are on their way from TMEM while
// the 16 before them are added (with 32, the sums and what is staged do not fit the registers any more, and a spilled word in this loop costs
// a fifth of the rate).  Two sums with each fma: plain fma is as fast by itself, but
// takes twice the issue slots, and the thread that issues the MMAs sits on one of the same four schedulers: beside plain fma four MMAs took
// 955 cycles, beside fma.rn.f32x2 512, their own rate.
template <int kCols>
__device__ __forceinline__ void b128_promote(uint64_t* sum, uint32_t taddr, uint32_t row_scale, uint32_t weight_scale, uint32_t free_bar) {
    constexpr int kStep = 16;
    uint32_t v[2][kStep];
    tmem_ld_32x16(taddr, v[0]);
    const float s = ld_shared_f32(row_scale) * ld_shared_f32(weight_scale);
    const uint64_t s2 = pack_f32x2(s, s);
    tmem_ld_wait();
#pragma unroll
    for (int c = 0; c < kCols; c += kStep) {
        uint32_t (&now)[kStep] = v[(c / kStep) & 1];
        if (c + kStep < kCols) {
            tmem_ld_32x16(taddr + c + kStep, v[((c / kStep) & 1) ^ 1]);
        } else {
            tc_fence_before();
            __syncwarp();
            if (elect_lane()) mbar_arrive(free_bar);
        }
#pragma unroll
        for (int j = 0; j < kStep / 2; ++j) fma_f32x2(sum[c / 2 + j], pack_f32x2(__uint_as_float(now[2 * j]), __uint_as_float(now[2 * j + 1])), s2);
        if (c + kStep < kCols) tmem_ld_wait();
    }
}

// Rounds and stores this warp's part of a tile: rows row0 + lane, columns col0 .. col0 + kCols - 1.
template <int kCols>
__device__ __forceinline__ void b128_store(const B128GemmParams& p, const uint64_t* sum, int row0, int col0, bool row_ok, int lane, float* my_staging) {
    if (p.out_vec32 && col0 + kCols <= p.n) {
        if (row_ok) {
            if (p.out_fp32) {
                float* o = static_cast<float*>(p.out) + static_cast<int64_t>(row0 + lane) * p.out_stride + col0;
#pragma unroll
                for (int j = 0; j < kCols; j += 8) {
                    uint32_t v[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) { const float2 f = unpack_f32x2(sum[j / 2 + i]); v[2 * i] = __float_as_uint(f.x); v[2 * i + 1] = __float_as_uint(f.y); }
                    st_global_32b(o + j, v);
                }
            } else {
                __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + static_cast<int64_t>(row0 + lane) * p.out_stride + col0;
#pragma unroll
                for (int j = 0; j < kCols; j += 16) {
                    uint32_t v[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) { const float2 f = unpack_f32x2(sum[j / 2 + i]); v[i] = pack_bf16x2(f.x, f.y); }
                    st_global_32b(o + j, v);
                }
            }
        }
    } else {
        // any number of columns and any alignment: 16 columns at a time through shared memory, so that half a warp writes
        // neighbouring columns of one row
        const unsigned rows_ok = __ballot_sync(0xffffffffu, row_ok);
#pragma unroll
        for (int c = 0; c < kCols; c += 16) {
#pragma unroll
            for (int j = 0; j < 8; ++j) { const float2 f = unpack_f32x2(sum[c / 2 + j]); my_staging[lane * 17 + 2 * j] = f.x; my_staging[lane * 17 + 2 * j + 1] = f.y; }
            __syncwarp();
            const int col = col0 + c + (lane & 15);
            for (int r = lane >> 4; r < 32; r += 2) {
                if (!((rows_ok >> r) & 1u) || col >= p.n) continue;
                const int64_t at = static_cast<int64_t>(row0 + r) * p.out_stride + col;
                if (p.out_fp32) static_cast<float*>(p.out)[at] = my_staging[r * 17 + (lane & 15)];
                else static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16(my_staging[r * 17 + (lane & 15)]);
            }
            __syncwarp();
        }
    }
}

// Status words of a device: [0] code of the first failure since the last read, [1 .. 4] its details, [5] whether a failure has been claimed.
// The claim comes first and the code last, so that a reader on another stream finds either nothing yet or all of it.
__device__ __forceinline__ void b128_report(int* status, int code, int phase, int block, int expected, int observed) {
    if (atomicCAS(status + 5, 0, 1) != 0) return;
    volatile int* s = status;
    s[1] = phase; s[2] = block; s[3] = expected; s[4] = observed;
    __threadfence();
    atomicExch(status, code);
}
// Hands the report over, if there is one, and makes room for the next.  Copying and clearing as two operations of a stream lost what another
// stream's kernel reported between them (one of eight reports in a loop of reads), or saw its code without its details.
__global__ void b128_take_status_kernel(int* status, int* taken) {
    const int code = ld_acquire_gpu(status);
    volatile const int* s = status;
    taken[0] = code;
    for (int i = 1; i < 5; ++i) taken[i] = code != 0 ? s[i] : 0;
    if (code == 0) return;
    __threadfence();
    atomicExch(status, 0);
    __threadfence();
    atomicExch(status + 5, 0);
}

// A 128-row block of a grouped layout: rows of another expert than its first one, or behind padding, are a mistake, reported and not written.
__device__ __forceinline__ void b128_check_group(const B128GemmParams& p, int mt, int et) {
    const int first = p.m_indices[mt * 128];
    const int own = p.m_indices[mt * 128 + et];
    if (first >= p.experts || (own >= 0 && own != first)) b128_report(p.status, MM_ERR_BAD_GROUP_LAYOUT, 0, mt, first, own);
}

template <int kBN, bool kSplit>
__global__ void __launch_bounds__(kB128Threads, 1)
block128_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const B128GemmParams p) {
    using S = B128Shape<kBN>;
    constexpr int kStages = S::kStages, kAccs = S::kAccs;
    constexpr int kCols = kBN / 2;                               // columns of a tile that one epilogue thread sums
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t smem_base = smem_u32(smem);
    uint8_t* scales = smem + kStages * S::kStageBytes;
    uint8_t* staging = scales + S::kScaleSlots * S::kScaleBytes;
    const uint32_t bars = smem_u32(staging) + S::kStagingBytes;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (kStages + s); };
    auto tfull_bar = [&](int a) { return bars + 8u * (2 * kStages + a); };
    auto tempty_bar = [&](int a) { return bars + 8u * (2 * kStages + kAccs + a); };
    constexpr int kTail = 8 * (2 * kStages + 2 * kAccs);
    static_assert(kTail + 16 <= S::kBarBytes, "barriers");
    const uint32_t abort_flag = bars + kTail;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(staging + S::kStagingBytes + kTail + 8);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int split = 1, part = 0;
    if (kSplit) {
        asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(split));
        part = static_cast<int>(cluster_ctarank());
    }
    const int num_tiles = p.m_tiles * p.n_tiles;
    const int first_tile = blockIdx.x / split, tile_step = gridDim.x / split;
    // the k blocks of this CTA
    const int kb0 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * part / split);
    const int kb1 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * (part + 1) / split);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) { mbar_init(full_bar(s), 3); mbar_init(empty_bar(s), 1); }
        for (int a = 0; a < kAccs; ++a) { mbar_init(tfull_bar(a), 1); mbar_init(tempty_bar(a), 8); }
        st_shared_volatile(abort_flag, static_cast<int>(blockIdx.x) == p.given_up ? 1 : 0);
        fence_barrier_init();
        prefetch_tensormap(&tm_a);
        prefetch_tensormap(&tm_b);
    }
    pdl_launch();
    pdl_wait();
    __syncthreads();
    // TMEM is allocated while the first copies are on their way; the MMA warp and the epilogue meet behind it
    auto tmem_ready = [&]() {
        tc_fence_before();
        named_bar_sync(1, kB128Threads - 96);
        tc_fence_after();
        return *static_cast<volatile uint32_t*>(tmem_slot);
    };

    // expert of an m tile (grouped: of its first row), or -1 when there is nothing to do; every role asks and skips alike
    auto tile_expert = [&](int mt) {
        if (p.m_indices == nullptr) return 0;
        const int e = p.m_indices[mt * 128];
        return e < p.experts ? e : -1;
    };

    if (warp < 4) {
        regs_dec<88>();
        if (warp == 0 && lane == 0) {
            // ------------------------------------------------------------------ TMA
            int stage = 0; uint32_t phase = 0;
            bool alive = true;
            const uint32_t bytes = static_cast<uint32_t>(p.a_box_rows) * 128 + S::kBBytes;
            for (int tile = first_tile; tile < num_tiles && alive; tile += tile_step) {
                int mt, nt;
                b128_tile(p, tile, mt, nt);
                const int e = tile_expert(mt);
                if (e < 0) continue;
                const int64_t tiled0 = (static_cast<int64_t>(e) * p.tiled_n_blocks + (nt * kBN) / 256) * p.k_blocks;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!mbar_wait_often(empty_bar(stage), phase ^ 1u, abort_flag, p.timeout_ns)) { alive = false; break; }
                    const uint32_t a_dst = smem_base + stage * S::kStageBytes;
                    mbar_arrive_expect_tx(full_bar(stage), bytes);
                    if (p.tiled) tma_load_2d(a_dst + S::kABytes, &tm_b, 0, static_cast<int32_t>((tiled0 + kb) * 256 + (nt * kBN) % 256), full_bar(stage));
                    else tma_load_3d(a_dst + S::kABytes, &tm_b, kb * 128, nt * kBN, e, full_bar(stage));
                    tma_load_2d(a_dst, &tm_a, kb * 128, mt * 128, full_bar(stage));
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                }
            }
        } else if (warp == 1) {
            // ------------------------------------------------------------------ MMA
            constexpr uint32_t idesc = umma_idesc_f8(128, kBN);
            tmem_alloc(smem_u32(tmem_slot), 512);
            tmem_relinquish();
            const uint32_t tmem_base = tmem_ready();
            int stage = 0; uint32_t phase = 0;
            int acc = 0; uint32_t acc_phase = 0;
            bool alive = lane == 0;
            for (int tile = first_tile; tile < num_tiles && alive; tile += tile_step) {
                int mt, nt;
                b128_tile(p, tile, mt, nt);
                if (tile_expert(mt) < 0) continue;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!mbar_wait_often(tempty_bar(acc), acc_phase ^ 1u, abort_flag, p.timeout_ns)) { alive = false; break; }
                    if (!mbar_wait_often(full_bar(stage), phase, abort_flag, p.timeout_ns)) { alive = false; break; }
                    tc_fence_after();
                    const uint64_t da = umma_desc_k_sw128(smem_base + stage * S::kStageBytes);
                    const uint64_t db = umma_desc_k_sw128(smem_base + stage * S::kStageBytes + S::kABytes);
#pragma unroll
                    for (int k = 0; k < 4; ++k) umma_f8(tmem_base + acc * kBN, da + 2u * k, db + 2u * k, idesc, k != 0 ? 1u : 0u);
                    umma_commit(tfull_bar(acc));             // first: the epilogue is what the loop waits for
                    umma_commit(empty_bar(stage));
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                    if (++acc == kAccs) { acc = 0; acc_phase ^= 1u; }
                }
            }
        } else if (warp >= 2) {
            // ------------------------------------------------------------------ scales, two rows a lane
            constexpr int kAhead = 2;                        // copies in flight before the oldest is handed over
            int stage = 0; uint32_t phase = 0;
            int slot = 0, hand = 0, pending = 0;
            bool alive = true;
            const int l64 = threadIdx.x - 64;
            auto hand_over = [&]() {
                __syncwarp();
                if (lane == 0) mbar_arrive(full_bar(hand));
                if (++hand == kStages) hand = 0;
                --pending;
            };
            for (int tile = first_tile; tile < num_tiles && alive; tile += tile_step) {
                int mt, nt;
                b128_tile(p, tile, mt, nt);
                const int e = tile_expert(mt);
                if (e < 0) continue;
                const float* sa0 = p.sa + static_cast<int64_t>(min(mt * 128 + l64, p.m - 1)) * p.sa_stride;
                const float* sa1 = p.sa + static_cast<int64_t>(min(mt * 128 + 64 + l64, p.m - 1)) * p.sa_stride;
                const float* sb = p.sb + (static_cast<int64_t>(e) * p.n_sf + min(nt * (kBN / 128) + (l64 & 1), p.n_sf - 1)) * p.k_blocks;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!mbar_wait_warp(empty_bar(stage), phase ^ 1u, abort_flag, p.timeout_ns)) { alive = false; break; }
                    const uint32_t dst = smem_u32(scales) + slot * S::kScaleBytes + l64 * 4;
                    cp_async_4(dst, sa0 + kb);
                    cp_async_4(dst + 256, sa1 + kb);
                    if (l64 < 2) cp_async_4(dst + 512, sb + kb);
                    cp_async_commit();
                    ++pending;
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                    if (++slot == S::kScaleSlots) slot = 0;
                    if (pending > kAhead) { cp_async_wait<kAhead>(); hand_over(); }
                }
            }
            cp_async_wait<0>();
            while (pending > 0) hand_over();
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------------------- epilogue
        regs_inc<208>();                                         // 2 x 208 + 88 = 3 x 168, the registers of the launch
        const uint32_t tmem_base = tmem_ready();
        // row et of the tile is lane et % 32 of TMEM's quarter et / 32; warps 4-7 take the first half of the columns, 8-11 the second
        const uint32_t my_tmem = tmem_base + (static_cast<uint32_t>(warp & 3) << 21) + ((warp - 4) >> 2) * kCols;
        const uint32_t my_scale = smem_u32(scales) + (threadIdx.x & 127) * 4;
        const uint32_t my_weight_scale = smem_u32(scales) + 512 + (kBN == 256 ? ((warp - 4) >> 2) * 4 : 0);
        uint32_t n = 0;                                      // k blocks so far: accumulator n % kAccs, place in the ring of scales n % 16
        bool alive = true;
#pragma unroll 1
        for (int tile = first_tile; tile < num_tiles && alive; tile += tile_step) {
            if (p.m_indices != nullptr) {
                int mt, nt;
                b128_tile(p, tile, mt, nt);
                b128_check_group(p, mt, threadIdx.x & 127);
                if (tile_expert(mt) < 0) continue;
            }
            // A split tile has few rows, as a rule; warps without any only hand the accumulators back.
            bool idle = false;
            if (kSplit) {
                int mt, nt;
                b128_tile(p, tile, mt, nt);
                idle = mt * 128 + (warp & 3) * 32 >= p.m;
            }
            uint64_t sum[kCols / 2];
#pragma unroll
            for (int j = 0; j < kCols / 2; ++j) sum[j] = 0ull;
#pragma unroll 1
            for (int left = kb1 - kb0; left > 0; --left, ++n) {
                const uint32_t acc = n % kAccs;
                if (!mbar_wait_warp(tfull_bar(acc), (n / kAccs) & 1u, abort_flag, p.timeout_ns)) { alive = false; break; }
                if (kSplit && idle) {
                    if (elect_lane()) mbar_arrive(tempty_bar(acc));
                    continue;
                }
                tc_fence_after();
                const uint32_t slot = (n % S::kScaleSlots) * S::kScaleBytes;
                b128_promote<kCols>(sum, my_tmem + acc * kBN, my_scale + slot, my_weight_scale + slot, tempty_bar(acc));
            }
            if (!alive) break;
            if (kSplit && idle) continue;
            if (kSplit) {
                // this CTA's part of the tile, for the cluster to add up: the operand ring is idle now (the last accumulator
                // was complete, so every copy and every MMA of this CTA is done)
                float* mine = reinterpret_cast<float*>(smem) + (threadIdx.x & 127) * (kBN + 4) + ((warp - 4) >> 2) * kCols;
#pragma unroll
                for (int j = 0; j < kCols; j += 4) *reinterpret_cast<float4*>(mine + j) = unpack_f32x4(sum[j / 2], sum[j / 2 + 1]);
                continue;
            }
            int mt, nt;
            b128_tile(p, tile, mt, nt);
            const int t = tid_again() - 128, row = mt * 128 + (t & 127);
            bool row_ok = row < p.m;
            if (row_ok && p.m_indices != nullptr) row_ok = p.m_indices[row] == tile_expert(mt);
            b128_store<kCols>(p, sum, row & ~31, nt * kBN + (t >> 7) * kCols, row_ok, t & 31, reinterpret_cast<float*>(staging) + (t >> 5) * 32 * 17);
        }
    }

    if (kSplit) {
        __syncwarp();
        cluster_sync_all();                                  // every part of the tile is in shared memory
        if (warp >= 4 && first_tile < num_tiles) {
            int mt, nt;
            b128_tile(p, first_tile, mt, nt);
            // rows part, part + split, .. of the tile are this CTA's: a warp to a row, four columns a lane
            static_assert(!kSplit || kBN == 128, "a warp holds a row of a split tile");
            const int rows = min(128, p.m - mt * 128), col = nt * kBN + lane * 4;
            int r = part + (warp - 4) * split;
            float4 v[kB128MaxSplit];
            auto fetch = [&]() {                                         // all on their way before the first is added
                const uint32_t at = smem_base + static_cast<uint32_t>(r * (kBN + 4) + lane * 4) * 4;
#pragma unroll
                for (int i = 0; i < kB128MaxSplit; ++i)
                    if (i < split) v[i] = ld_shared_cluster_f4(mapa_shared(at, i));
            };
            // A CTA that has given up has no part there, but operands: then no CTA of the cluster writes anything of the tile.  (Asked
            // together with the first row's parts: before them it cost 0.2 us.)
            const int failed = lane < split ? ld_shared_cluster_s32(mapa_shared(abort_flag, lane)) : 0;
            if (r < rows) fetch();
            if (__any_sync(0xffffffffu, failed != 0)) r = rows;
            while (r < rows) {
                float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int i = 0; i < kB128MaxSplit; ++i)
                    if (i < split) { t.x += v[i].x; t.y += v[i].y; t.z += v[i].z; t.w += v[i].w; }
                const float f[4] = {t.x, t.y, t.z, t.w};
                const int64_t o = (mt * 128 + r) * p.out_stride + col;
                r += 8 * split;
                if (r < rows) fetch();
                if (p.out_vec32 && col + 4 <= p.n) {
                    if (p.out_fp32) *reinterpret_cast<float4*>(static_cast<float*>(p.out) + o) = t;
                    else *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + o) = make_uint2(pack_bf16x2(t.x, t.y), pack_bf16x2(t.z, t.w));
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (col + j >= p.n) continue;
                        if (p.out_fp32) static_cast<float*>(p.out)[o + j] = f[j];
                        else static_cast<__nv_bfloat16*>(p.out)[o + j] = __float2bfloat16(f[j]);
                    }
                }
            }
        }
        __syncwarp();
        cluster_sync_all();                                  // nobody leaves while its part may still be read
    }

    if (ld_shared_volatile(abort_flag) != 0) {
        // a bounded wait expired: give copies that may still be in flight time to land, then report
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 1000000ull) __nanosleep(1000);
        if (threadIdx.x == 0) b128_report(p.status, MM_ERR_PIPE_TIMEOUT, 20, blockIdx.x, num_tiles, 0);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(*tmem_slot, 512);
    }
}

}  // namespace mm
