// The products of block128_gemm.cuh on CTA pairs (cluster of two, tcgen05 cta_group::2), for many rows: a pair takes 256 rows x 256 columns.
//
// Each CTA brings its own 128 rows of a and half of the 256 weight rows, 32 KiB for a k block instead of 48, and an MMA of one leader
// thread reads both CTAs' shared memory and writes each one's 128 rows into its own TMEM.  One CTA by itself cannot keep the pipe fed: an
// MMA of 128 x 256 reads 48 KiB of shared memory for a k block while the copies write the next 48, 750 cycles at 128 bytes a cycle for
// 512 cycles of MMA; the pair reads 32 and writes 32.
// Everything behind the MMA is as in block128_gemm.cuh, in each CTA for its own rows.
//
// Grouped rows: a pair takes two neighbouring blocks of one expert.  Which ones is worked out by every CTA for itself; an expert with an odd
// number of blocks leaves the second CTA of its last pair without rows, and it brings its half of the weights all the same.
#pragma once
#include "block128_gemm.cuh"

namespace mm {

constexpr int kB128PairStages = 6;
constexpr int kB128PairStageBytes = 2 * 128 * 128;                   // own rows of a, own half of the weight rows
constexpr int kB128PairMaxPairs = 4096;                              // of grouped blocks
constexpr int kB128PairMaxTiles = 256;                               // of one pair of CTAs
constexpr int kB128PairScaleSlots = 16;
constexpr int kB128PairScaleBytes = 544;
constexpr int kB128PairStagingBytes = 8 * 32 * 17 * 4;
constexpr int kB128PairSmemBytes = kB128PairStages * kB128PairStageBytes + kB128PairScaleSlots * kB128PairScaleBytes + kB128PairStagingBytes +
                                   kB128PairMaxTiles * 16 + 512;
static_assert(kB128PairSmemBytes <= 232448, "exceeds the 227 KiB of shared memory a CTA can have");
static_assert(kB128PairScaleSlots >= kB128PairStages + 2 + 1, "scale ring");

__device__ __forceinline__ void tma_load_3d_pair(uint32_t smem_dst, const CUtensorMap* map, int32_t c0, int32_t c1, int32_t c2, uint32_t bar_cluster) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar_cluster)
        : "memory");
}

// Pairs of grouped blocks, by one warp: list[i] = first block | second one there << 15.  s_expert: of each block, -1 for none, and one -1 more.
__device__ __forceinline__ int b128_list_pairs(const int* s_expert, int blocks, uint16_t* list, int lane) {
    int count = 0, run = 0, before = -1;                             // start of the run that reaches into this chunk, and its expert
    for (int b0 = 0; b0 < blocks; b0 += 32) {
        const int b = b0 + lane;
        const int e = b < blocks ? s_expert[b] : -1;
        const int up = __shfl_up_sync(0xffffffffu, e, 1);
        int start = e != (lane == 0 ? before : up) ? b : (lane == 0 ? run : -1);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int s = __shfl_up_sync(0xffffffffu, start, o);
            if (lane >= o) start = max(start, s);
        }
        const bool first = e >= 0 && ((b - start) & 1) == 0;
        const bool second = first && s_expert[b + 1] == e;
        const unsigned mask = __ballot_sync(0xffffffffu, first);
        if (first) list[count + __popc(mask & ((1u << lane) - 1u))] = static_cast<uint16_t>(b | (second ? 0x8000 : 0));
        count += __popc(mask);
        run = __shfl_sync(0xffffffffu, start, 31);
        before = __shfl_sync(0xffffffffu, e, 31);
    }
    return count;
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kB128Threads, 1)
block128_gemm_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b_half, const B128GemmParams p) {
    constexpr int kStages = kB128PairStages, kCols = 128;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t smem_base = smem_u32(smem);
    uint8_t* scales = smem + kStages * kB128PairStageBytes;
    uint8_t* staging = scales + kB128PairScaleSlots * kB128PairScaleBytes;
    int4* s_tiles = reinterpret_cast<int4*>(staging + kB128PairStagingBytes);               // block of rows (-1 - block: not this CTA's own), output tile, expert
    uint8_t* tail = reinterpret_cast<uint8_t*>(s_tiles + kB128PairMaxTiles);
    const uint32_t bars = smem_u32(tail);
    auto full_bar = [&](int s) { return bars + 8u * s; };                                   // used in the leader only
    auto empty_bar = [&](int s) { return bars + 8u * (kStages + s); };                      // in each CTA
    auto tfull_bar = [&](int a) { return bars + 8u * (2 * kStages + a); };                  // in each CTA
    auto tempty_bar = [&](int a) { return bars + 8u * (2 * kStages + 2 + a); };             // used in the leader only
    auto scale_bar = [&](int s) { return bars + 8u * (2 * kStages + 4 + s); };              // in each CTA
    constexpr int kTail = 8 * (2 * kStages + 4 + kB128PairScaleSlots);
    static_assert(kTail + 16 <= 512, "barriers");
    const uint32_t abort_flag = bars + kTail;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + kTail + 4);
    int* s_pairs = reinterpret_cast<int*>(tail + kTail + 8);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cta = static_cast<int>(cluster_ctarank());
    const bool leader = cta == 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(tfull_bar(a), 1); mbar_init(tempty_bar(a), 16); }
        for (int s = 0; s < kB128PairScaleSlots; ++s) mbar_init(scale_bar(s), 2);
        st_shared_volatile(abort_flag, 0);
        *s_pairs = (p.m_tiles + 1) / 2;
        fence_barrier_init();
        prefetch_tensormap(&tm_a);
        prefetch_tensormap(&tm_b_half);
    }
    // The tiles of this pair, worked out once and for all roles (the operand ring is not in use yet)
    uint16_t* list = reinterpret_cast<uint16_t*>(smem + 65536);
    if (p.m_indices != nullptr) {
        int* s_expert = reinterpret_cast<int*>(smem);
        for (int b = threadIdx.x; b <= p.m_tiles; b += blockDim.x) {
            const int e = b < p.m_tiles ? p.m_indices[b * 128] : -1;
            s_expert[b] = e < p.experts ? e : -1;
        }
        __syncthreads();
        if (warp == 0) {
            const int n = b128_list_pairs(s_expert, p.m_tiles, list, lane);
            if (lane == 0) *s_pairs = n;
        }
    }
    __syncthreads();
    const int tiles = (max(0, *s_pairs * p.n_tiles - static_cast<int>(blockIdx.x >> 1)) + static_cast<int>(gridDim.x >> 1) - 1) / static_cast<int>(gridDim.x >> 1);
    for (int i = threadIdx.x; i < tiles; i += blockDim.x) {
        // eight pairs at a time run through all output tiles
        const int tile = (blockIdx.x >> 1) + i * (gridDim.x >> 1), pairs = *s_pairs;
        const int per_group = 8 * p.n_tiles;
        const int g = tile / per_group, r = tile - g * per_group;
        const int gm = min(8, pairs - g * 8);
        const int nt = r / gm, pt = g * 8 + r - nt * gm;
        int first = 2 * pt, e = 0;
        bool own = leader || first + 1 < p.m_tiles;
        if (p.m_indices != nullptr) {
            first = list[pt] & 0x7fff;
            own = leader || (list[pt] & 0x8000) != 0;
            e = p.m_indices[first * 128];
        }
        s_tiles[i] = make_int4(own ? first + cta : -1 - first, nt, e, 0);
    }
    fence_proxy_async_smem();
    __syncthreads();
    cluster_sync_all();                                              // both CTAs' barriers exist before anyone arrives remotely
    if (warp == 2) {
        tmem_alloc_pair(smem_u32(tmem_slot), 512);                   // the same warp in both CTAs
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp < 4) {
        regs_dec<88>();
        if (warp == 0 && lane == 0) {
            // ------------------------------------------------------------------ TMA, in each CTA
            int stage = 0; uint32_t phase = 0;
            bool alive = true;
            for (int i = 0; i < tiles && alive; ++i) {
                const int4 t = s_tiles[i];
                const int a_row = (t.x < 0 ? -1 - t.x : t.x) * 128, nt = t.y, e = t.z;
                const int tiled0 = (e * p.tiled_n_blocks + nt) * p.k_blocks * 256 + cta * 128;
                for (int kb = 0; kb < p.k_blocks; ++kb) {
                    if (!mbar_wait_often(empty_bar(stage), phase ^ 1u, abort_flag, p.timeout_ns)) { alive = false; break; }
                    const uint32_t a_dst = smem_base + stage * kB128PairStageBytes, b_dst = a_dst + 128 * 128;
                    const uint32_t lead_full = mapa_shared(full_bar(stage), 0);
                    // Only the leader arrives, for the bytes of both; the other CTA's copies count on its barrier as they land.  They cannot
                    // be a phase ahead: a stage is filled again only after the commit that follows the leader's wait on this barrier.
                    if (leader) mbar_arrive_expect_tx(full_bar(stage), 2 * kB128PairStageBytes);
                    if (p.tiled) tma_load_2d_pair(b_dst, &tm_b_half, 0, tiled0 + kb * 256, lead_full);
                    else tma_load_3d_pair(b_dst, &tm_b_half, kb * 128, nt * 256 + cta * 128, e, lead_full);
                    tma_load_2d_pair(a_dst, &tm_a, kb * 128, a_row, lead_full);
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                }
            }
        } else if (warp == 1 && lane == 0 && leader) {
            // ------------------------------------------------------------------ MMA, in the leader
            constexpr uint32_t idesc = umma_idesc_f8(256, 256);
            int stage = 0; uint32_t phase = 0;
            int acc = 0; uint32_t acc_phase = 0;
            bool alive = true;
            for (int i = 0; i < tiles && alive; ++i) {
                for (int kb = 0; kb < p.k_blocks; ++kb) {
                    if (!mbar_wait_often(tempty_bar(acc), acc_phase ^ 1u, abort_flag, p.timeout_ns)) { alive = false; break; }
                    if (!mbar_wait_often(full_bar(stage), phase, abort_flag, p.timeout_ns)) { alive = false; break; }
                    tc_fence_after();
                    const uint64_t da = umma_desc_k_sw128(smem_base + stage * kB128PairStageBytes);
                    const uint64_t db = umma_desc_k_sw128(smem_base + stage * kB128PairStageBytes + 128 * 128);
#pragma unroll
                    for (int k = 0; k < 4; ++k) umma_f8_pair(tmem_base + acc * 256, da + 2u * k, db + 2u * k, idesc, k != 0 ? 1u : 0u);
                    umma_commit_pair(tfull_bar(acc));
                    umma_commit_pair(empty_bar(stage));
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                    if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
                }
            }
        } else if (warp >= 2) {
            // ------------------------------------------------------------------ scales of this CTA's rows, two rows a lane
            constexpr int kAhead = 2;                                // copies in flight before the oldest is handed over
            int stage = 0; uint32_t phase = 0;
            int slot = 0, hand = 0, pending = 0;
            bool alive = true;
            const int l64 = threadIdx.x - 64;
            auto hand_over = [&]() {
                __syncwarp();
                if (lane == 0) mbar_arrive(scale_bar(hand));
                if (++hand == kB128PairScaleSlots) hand = 0;
                --pending;
            };
            for (int i = 0; i < tiles && alive; ++i) {
                const int4 t = s_tiles[i];
                const int mt = t.x < 0 ? -1 - t.x : t.x, nt = t.y, e = t.z;
                const float* sa0 = p.sa + static_cast<int64_t>(min(mt * 128 + l64, p.m - 1)) * p.sa_stride;
                const float* sa1 = p.sa + static_cast<int64_t>(min(mt * 128 + 64 + l64, p.m - 1)) * p.sa_stride;
                const float* sb = p.sb + (static_cast<int64_t>(e) * p.n_sf + min(nt * 2 + (l64 & 1), p.n_sf - 1)) * p.k_blocks;
                for (int kb = 0; kb < p.k_blocks; ++kb) {
                    if (!mbar_wait_often(empty_bar(stage), phase ^ 1u, abort_flag, p.timeout_ns)) { alive = false; break; }
                    const uint32_t dst = smem_u32(scales) + slot * kB128PairScaleBytes + l64 * 4;
                    cp_async_4(dst, sa0 + kb);
                    cp_async_4(dst + 256, sa1 + kb);
                    if (l64 < 2) cp_async_4(dst + 512, sb + kb);
                    cp_async_commit();
                    ++pending;
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                    if (++slot == kB128PairScaleSlots) slot = 0;
                    if (pending > kAhead) { cp_async_wait<kAhead>(); hand_over(); }
                }
            }
            cp_async_wait<0>();
            while (pending > 0) hand_over();
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------------------- epilogue, in each CTA
        regs_inc<208>();
        const uint32_t my_tmem = tmem_base + (static_cast<uint32_t>(warp & 3) << 21) + ((warp - 4) >> 2) * kCols;
        const uint32_t my_scale = smem_u32(scales) + (threadIdx.x & 127) * 4;
        const uint32_t my_weight_scale = smem_u32(scales) + 512 + ((warp - 4) >> 2) * 4;
        const uint32_t lead_tempty = mapa_shared(tempty_bar(0), 0);
        uint32_t n = 0;                                              // k blocks so far: accumulator n % 2, place in the ring of scales n % 16
        bool alive = true;
#pragma unroll 1
        for (int i = 0; i < tiles && alive; ++i) {
            uint64_t sum[kCols / 2];
#pragma unroll
            for (int j = 0; j < kCols / 2; ++j) sum[j] = 0ull;
#pragma unroll 1
            for (int left = p.k_blocks; left > 0; --left, ++n) {
                const uint32_t acc = n & 1u, slot = n % kB128PairScaleSlots;
                if (!mbar_wait_often(scale_bar(slot), (n / kB128PairScaleSlots) & 1u, abort_flag, p.timeout_ns)) { alive = false; break; }
                if (!mbar_wait_often(tfull_bar(acc), (n >> 1) & 1u, abort_flag, p.timeout_ns)) { alive = false; break; }
                tc_fence_after();
                b128_promote<kCols, true>(sum, my_tmem + acc * 256, my_scale + slot * kB128PairScaleBytes, my_weight_scale + slot * kB128PairScaleBytes,
                                          lead_tempty + acc * 8);
            }
            if (!alive) break;
            const int4 at = s_tiles[i];
            if (at.x < 0) continue;
            const int t = tid_again() - 128, row = at.x * 128 + (t & 127);
            if (p.m_indices != nullptr) b128_check_group(p, at.x, t & 127);
            bool row_ok = row < p.m;
            if (row_ok && p.m_indices != nullptr) row_ok = p.m_indices[row] == at.z;
            b128_store<kCols>(p, sum, row & ~31, at.y * 256 + (t >> 7) * kCols, row_ok, t & 31, reinterpret_cast<float*>(staging) + (t >> 5) * 32 * 17);
        }
    }

    if (p.m_indices != nullptr && blockIdx.x < 2 && leader && warp == 4) {
        // blocks that are in no pair because their first row names no expert: padding, or a mistake
        for (int b = 0; b < p.m_tiles; ++b) {
            const int first = p.m_indices[b * 128];
            if (first >= 0 && first < p.experts) continue;
            for (int r = lane; r < 128; r += 32) b128_check_group(p, b, r);
        }
    }
    if (ld_shared_volatile(abort_flag) != 0) {
        // a bounded wait expired: give copies that may still be in flight time to land, then report
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 1000000ull) __nanosleep(1000);
        if (threadIdx.x == 0 && atomicCAS(p.status, 0, MM_ERR_PIPE_TIMEOUT) == 0) {
            p.status[1] = 21; p.status[2] = blockIdx.x; p.status[3] = tiles; p.status[4] = 0;
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                                              // the other CTA may still arrive here, or read this shared memory
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

}  // namespace mm
