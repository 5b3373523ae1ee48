// A whole mixture-of-experts layer for a few tokens, in two launches:
//
//   y[t] = sum over slots s of  w[t, s] * W2[e] . cast( silu(g) * u ),   (g, u) = W1[e] . cast(x[t]),   e = topk[t, s]
//
// e4m3 weights with a scale for each 128 x 128 block, activations cast with one for each 128 values, fp32 everywhere else.
//
//   1. moe_route_kernel: a block per token: the k largest router logits and their softmax (or the caller's choice, checked), the
//      cast of x, and the zeroes that the second launch counts from.
//   2. moe_experts_kernel: both products and the combine, one CTA per SM.
//
// With few tokens all that counts is reading each chosen expert's weights once at the rate of HBM, so the work is the list of weight
// blocks (256 rows x 128 k, 32 KiB), not of outputs: all k blocks of all tiles of the first product, then of the second, cut into
// chunks that CTAs claim from one counter.  While tiles are few (under 16 per SM), a chunk is an equal share of the whole list, cut
// wherever the share ends, and the parts of a tile meet in memory: of the first product, whoever brings the last part adds them up in order,
// of the second, the combine does.  Else a chunk is a tile.  Weights need nothing but the routes, so the TMA warp runs ahead into the
// second product, up to the depth of its ring, while the activations of the first are still being finished; only the token operand waits
// for them.  (Prefetching more of them to L2 meanwhile took bandwidth from CTAs that were still at the first product: 8 blocks for each CTA
// made 48 us of T = 1 into 51, 24 made 87 us of T = 33 into 93.)
//
// A chunk of the second product is claimed only after every chunk of the first one has been, and by a CTA that runs; so what a CTA waits
// for is always being worked on, however many of the CTAs are resident, and two such launches may share a GPU.
//
// Measured: 1 token, 256 experts, top-6, 4096 / 2048: 47 us (151 MB; 3.2 TB/s over the whole call, the streams themselves run at 6); 33 tokens,
// 64 experts, top-8, 2048 / 1024: 88 us (58 experts have a token: 365 MB, 4.1 TB/s); 128 tokens, else as the first, with 170 to 190 popular
// experts (4.3 to 4.7 GB): 640 to 680 us alone (HBM's own rate), 730 to 800 in a loop, where the power cap sets the clock.  With native
// weights, two copies of 16 KiB for each block: 49, 89 and 663.  What bounds it at one token are the latencies around the streams: 8 us until the first
// copy, 8 from the last sums of the first product to its activations being known everywhere, 4 for the combine.
//
// Tile = up to 128 routes of one expert x 256 weight rows (first product: 128 gate rows and their 128 up rows, so that a tile holds
// one whole block of the activations' cast).  Warp 0 = TMA (weights), 1 = MMA, 2-3 = token operand and scales (cp.async: rows are gathered
// by route), 8-15 = sums: the promotion by block scales of block128_gemm.cuh, 4-7 = what becomes of the sums of a tile (joining parts,
// SwiGLU and cast, the counts that other CTAs wait for, the combine) while the next tile is being summed.
#pragma once
#include "block128.cuh"
#include "block128_gemm.cuh"

namespace mm {

constexpr int kMoeMaxRoutes = 4096;
constexpr int kMoeMaxBlocks = MM_MAX_EXPERTS + kMoeMaxRoutes / 128;      // of up to 128 routes of one expert
constexpr int kMoeBBytes = 256 * 128;
// The operand ring: four stages with room for 128 token rows, or five with room for 48 where no expert has more.  (An MMA reads 64
// or 128 rows either way; those behind the last route are zeroes, or what follows in the ring, and their sums are not looked at.)
constexpr int kMoeMaxStages = 5, kMoeFewRows = 48;
constexpr int kMoeRingBytes = 4 * (128 * 128 + kMoeBBytes);
static_assert(kMoeMaxStages * (kMoeFewRows * 128 + kMoeBBytes) <= kMoeRingBytes, "the ring of few rows");
constexpr int kMoePlanBytes = kMoeMaxRoutes * 2 + kMoeMaxBlocks * 8 + kMoeMaxRoutes / 8;
constexpr int kMoeTurnRows = 6, kMoeTurnPitch = 260;    // fp32 rows that go from the summing to the finishing warps, in two buffers
constexpr int kMoeThreads = 512;
constexpr int kMoeSegments = 8;
constexpr int kMoeCtrRows1 = 8, kMoeCtrUnits2 = 16;
constexpr int kMoeTailBytes = 768;        // barriers and MoeWords
// Scales of a unit: 128 rows, then two of the weights.  As in block128_gemm.cuh: stages + accumulators + 1 units may be on their way.
constexpr int kMoeScaleSlots = 8, kMoeScaleBytes = 544;
static_assert(kMoeScaleSlots >= kMoeMaxStages + 2 + 1, "scale ring");
constexpr int kMoeSmemBytes = kMoeRingBytes + kMoePlanBytes + 2 * kMoeTurnRows * kMoeTurnPitch * 4 + kMoeScaleSlots * kMoeScaleBytes + kMoeTailBytes;
static_assert(kMoeSmemBytes <= 232448, "exceeds the 227 KiB of shared memory a CTA can have");
constexpr int kMoeStreamTiles = 16;        // tiles per SM below which chunks are equal shares

struct MoeParams {
    int tokens, experts, topk, hidden, inter;
    // routing: either logits or the caller's choice
    const float* logits; int64_t logits_stride;
    const void* topk_idx; int idx_i64; const float* topk_w;
    // x: bf16 to be cast, or already codes and scales
    const void* x; int64_t x_stride;
    const uint8_t* xq; const float* xsf;
    uint8_t* xq_out; float* xsf_out;
    int* route_expert; float* route_w;       // [tokens * topk], -1 = none
    int* counters; int num_counters;
    // counters: [0] claims, [kMoeCtrRows1] finished tiles of the first product (times the warps that finish their rows), [ctr_done1 ..) the
    // same by block of routes, [ctr_tile1 ..) k blocks that have arrived for each of its tiles that was cut, by warp, [kMoeCtrUnits2] k
    // blocks of the second product whose sums are written
    int ctr_done1, ctr_tile1;
    const float* s1; const float* s2;
    int tiled;
    // [routes][inter] and [routes][inter / 128], by place in the sorted list.  A row of scales has 128-byte lines of its own: they are
    // read through L1, which must not hold a line that another expert's tiles are still writing to
    uint8_t* act_q; float* act_sf; int act_sf_pitch;
    float* rows_out;                         // [routes][hidden]: weighted rows of the second product, by route, where a tile is whole
    float* parts; int part_rows;             // [2 products][chunks][2][part_rows][256], then [CTAs][2][part_rows][256] for tiles that are whole
    __nv_bfloat16* y;
    float clamp;
    int* status;
    uint64_t timeout_ns;
};

// kPer: experts per lane.  Ties go to the lower index; NaN and -inf logits are never chosen.
template <int kPer>
__device__ __forceinline__ void moe_topk(const MoeParams& p, int t, int lane) {
    // Floats as integers of the same order, 0 for what cannot be chosen: two warp reductions find a maximum and its lowest index, where
    // comparing pairs of floats and indexes took ten shuffles.
    uint32_t v[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = lane + 32 * i;
        const float l = e < p.experts ? p.logits[t * p.logits_stride + e] : -INFINITY;
        const uint32_t bits = __float_as_uint(l == 0.0f ? 0.0f : l);                     // -0 and 0 are a tie
        v[i] = l > -INFINITY ? (bits >> 31 ? ~bits : bits | 0x80000000u) : 0u;
    }
    float sel = 0.0f, sum = 0.0f, top = 0.0f;
    int sel_e = -1;
    for (int k = 0; k < p.topk; ++k) {
        uint32_t best = 0;
        int best_i = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (v[i] > best) { best = v[i]; best_i = i; }
        const uint32_t most = __reduce_max_sync(0xffffffffu, best);
        if (most == 0) break;                                        // nothing left to choose from
        const int best_e = static_cast<int>(__reduce_min_sync(0xffffffffu, best == most ? static_cast<uint32_t>(lane + 32 * best_i) : 0xffffffffu));
        const float value = __uint_as_float(most >> 31 ? most & 0x7fffffffu : ~most);
        if (k == 0) top = value;
        const float w = value == top ? 1.0f : expf(value - top);     // equal infinities share alike
        sum += w;
        if (lane == k) { sel = w; sel_e = best_e; }
        if ((best_e & 31) == lane) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) if (i == (best_e >> 5)) v[i] = 0u;
        }
    }
    if (lane < p.topk) {
        const float w = sel_e >= 0 ? __fdiv_rn(sel, sum) : 0.0f;
        p.route_expert[t * p.topk + lane] = w != 0.0f ? sel_e : -1;
        p.route_w[t * p.topk + lane] = w;
    }
}

__global__ void __launch_bounds__(256) moe_route_kernel(const MoeParams p) {
    pdl_launch();
    pdl_wait();
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < p.num_counters; i += gridDim.x * blockDim.x) p.counters[i] = 0;
    if (warp == 0) {
        if (p.logits != nullptr) {
            if (p.experts <= 256) moe_topk<8>(p, t, lane);
            else moe_topk<MM_MAX_EXPERTS / 32>(p, t, lane);
        } else if (lane < p.topk) {
            const int r = t * p.topk + lane;
            const int64_t e = p.idx_i64 ? static_cast<const int64_t*>(p.topk_idx)[r] : static_cast<const int32_t*>(p.topk_idx)[r];
            const float w = p.topk_w[r];
            p.route_expert[r] = e >= 0 && e < p.experts && w != 0.0f ? static_cast<int>(e) : -1;
            p.route_w[r] = w;
        }
    } else if (p.x != nullptr) {
        const int groups = p.hidden / 128;                          // 16 lanes hold one
        for (int g0 = (warp - 1) * 2; g0 < groups; g0 += 14) {
            const int g = g0 + (lane >> 4);
            const int col = g * 128 + (lane & 15) * 8;
            F8 v = zero8();
            if (g < groups) v = load8<B128_BF16>(p.x, t * p.x_stride + col, B128_BF16);
            const float top = group_top(half_warp_max(amax8(v)));
            if (g < groups) {
                *reinterpret_cast<uint2*>(p.xq_out + static_cast<int64_t>(t) * p.hidden + col) = quantise_exact(v, top);
                if ((lane & 15) == 0) p.xsf_out[t * groups + g] = group_scale(top);
            }
        }
    }
}

// The list of weight blocks of one product: tiles * kb units, cut into chunks.
struct MoeList {
    int tiles, kb, chunks;
    int shares;                                                     // chunks are equal shares, else tiles
    // shares: tiles < 16 CTAs and kb <= 256 keep the products below 2^31
    __device__ __forceinline__ int start(int c) const { return shares ? static_cast<int>(static_cast<uint32_t>(tiles * kb) * c / chunks) : c * kb; }
    __device__ __forceinline__ int chunk_of(int unit) const {        // the chunk c with start(c) <= unit < start(c + 1)
        return shares ? static_cast<int>((static_cast<uint32_t>(unit + 1) * chunks - 1) / static_cast<uint32_t>(tiles * kb)) : unit / kb;
    }
};
__device__ __forceinline__ MoeList moe_list(int tiles, int kb, int ctas) {
    MoeList l;
    l.tiles = tiles; l.kb = kb;
    l.shares = tiles < kMoeStreamTiles * ctas;
    l.chunks = l.shares ? min(ctas, tiles * kb) : tiles;
    return l;
}

// A run of k blocks of one tile, as the TMA thread walks through its chunks and the other warps follow it.  They read it from shared memory
// whenever they want something of it: held in registers beside the epilogue's 128 sums it made them spill in the innermost loop.
struct MoeSegment {
    int kind;                                            // 0, 1: first or second product; -1: no more
    int chunk, tile, block, out;                         // chunk and tile of its product; block of routes and output tile
    int k0, k1;
    int rows, first;                                     // of the block of routes
    int expert;
};

// Shared memory behind the operand ring
struct MoeWords {
    int abort;
    uint32_t tmem;
    int blocks, most, finishers;                         // blocks of routes, routes of the most popular expert, sum of moe_finishers
    int ready;                                           // blocks of routes whose activations this CTA knows to be finished
    MoeList list[2];                                     // of either product
    MoeSegment segment[kMoeSegments];
};
struct MoeSmem {
    float* turn;                                         // [2][kMoeTurnRows][kMoeTurnPitch]
    uint2* block;                                        // blocks of routes: expert | rows << 16, first place
    uint32_t* valid;                                     // a bit for each route
    uint16_t* route;                                     // routes sorted by expert
    float* scale;                                        // [slots][128 rows, 2 of the weights, 6 unused]
    uint32_t bars;
    MoeWords* words;
    static constexpr int kBars = 2 * kMoeMaxStages + 9 + 2 * kMoeSegments;
    static_assert(8 * kBars + sizeof(MoeWords) <= kMoeTailBytes, "barriers");
    __device__ __forceinline__ explicit MoeSmem(uint8_t* smem) {
        turn = reinterpret_cast<float*>(smem + kMoeRingBytes);
        block = reinterpret_cast<uint2*>(turn + 2 * kMoeTurnRows * kMoeTurnPitch);
        valid = reinterpret_cast<uint32_t*>(block + kMoeMaxBlocks);
        route = reinterpret_cast<uint16_t*>(valid + kMoeMaxRoutes / 32);
        scale = reinterpret_cast<float*>(route + kMoeMaxRoutes);
        uint8_t* tail = reinterpret_cast<uint8_t*>(scale) + kMoeScaleSlots * kMoeScaleBytes;
        bars = smem_u32(tail);
        words = reinterpret_cast<MoeWords*>(tail + 8 * kBars);
    }
    __device__ __forceinline__ uint32_t turn_full(int b) const { return bars + 8u * (kBars - 5 + b); }
    __device__ __forceinline__ uint32_t turn_empty(int b) const { return bars + 8u * (kBars - 3 + b); }
    __device__ __forceinline__ uint32_t finish_bar() const { return bars + 8u * (kBars - 1); }
};

// silu(gate) * up of one row's block of 128, four columns a lane, and its cast
__device__ __forceinline__ void moe_finish_row(const MoeParams& p, float4 g4, float4 u4, bool do_clamp, int64_t place, int nt, int lane) {
    const float g[4] = {g4.x, g4.y, g4.z, g4.w}, u[4] = {u4.x, u4.y, u4.z, u4.w};
    float v[4];
    float top = 1.0e-4f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a = g[i], b = u[i];
        if (do_clamp) {                                              // NaN stays NaN
            a = a < -p.clamp ? -p.clamp : (a > p.clamp ? p.clamp : a);
            b = b < -p.clamp ? -p.clamp : (b > p.clamp ? p.clamp : b);
        }
        v[i] = silu_f(a) * b;
        top = max_nan(top, fabsf(v[i]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float mul = 448.0f * rcp_approx(top);
    *reinterpret_cast<uint32_t*>(p.act_q + place * p.inter + nt * 128 + lane * 4) = pack4_e4m3(v[0] * mul, v[1] * mul, v[2] * mul, v[3] * mul);
    if (lane == 0) p.act_sf[place * p.act_sf_pitch + nt] = group_scale(top);
}
__device__ __forceinline__ void add4(float4& a, const float4& b) { a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w; }

// Bounded wait until *p (written by other CTAs, released) has reached `want`.  One thread of a CTA asks, and not without pause: with every
// warp of every CTA asking (1480 pollers), the counts themselves got through so slowly that a single token took 80 to 150 us.
__device__ __forceinline__ bool moe_wait_count(const int* p, int want, uint32_t abort_flag, uint64_t timeout_ns) {
    const uint64_t t0 = global_timer_ns();
    while (ld_acquire_gpu(p) < want) {
        if (ld_shared_volatile(abort_flag) != 0) return false;
        if (global_timer_ns() - t0 > timeout_ns) { st_shared_volatile(abort_flag, 1); return false; }
        __nanosleep(100);
    }
    return true;
}
// b128_promote for 64 columns, without its overlap: these tiles wait for HBM, not for their sums.  `arrivals` of the eight that the barrier
// of the accumulator counts, if kLast.
template <bool kLast>
__device__ __forceinline__ void moe_promote(uint64_t* sum, uint32_t taddr, float s, uint32_t free_bar, uint32_t arrivals) {
    const uint64_t s2 = pack_f32x2(s, s);
#pragma unroll
    for (int c = 0; c < 64; c += 32) {
        uint32_t v[32];
        tmem_ld_32x32(taddr + c, v);
        tmem_ld_wait();
        if (kLast && c == 32) {
            tc_fence_before();
            __syncwarp();
            if (elect_lane()) mbar_arrive_n(free_bar, arrivals);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) fma_f32x2(sum[c / 2 + j], pack_f32x2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), s2);
    }
}
// Whether a phase is complete, without the pause that try_wait may make
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Bounded wait of a converged warp, as mbar_wait_warp, for something that takes a tile's time
__device__ __forceinline__ bool mbar_wait_asleep(uint32_t bar, uint32_t parity, uint32_t abort_flag, uint64_t timeout_ns) {
    const auto wait = [&]() {
        uint64_t t0 = 0;
        while (!mbar_try_wait(bar, parity)) {
            if (ld_shared_volatile(abort_flag) != 0) return false;
            const uint64_t t = global_timer_ns();
            if (t0 == 0) t0 = t;
            else if (t - t0 > timeout_ns) { st_shared_volatile(abort_flag, 1); return false; }
            __nanosleep(40);
        }
        return true;
    };
    const bool came = wait();
    return !__any_sync(0xffffffffu, !came);
}
__device__ __forceinline__ void st_release_cta(uint32_t addr, int v) { asm volatile("st.release.cta.shared::cta.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ int ld_acquire_cta(uint32_t addr) {
    int v;
    asm volatile("ld.acquire.cta.shared::cta.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
// Bounded wait, a warp at a time, until this CTA knows that the activations of block of routes `rb` are finished; returns how many are, or 0.
__device__ __forceinline__ int moe_wait_ready(uint32_t ready, int rb, int lane, uint32_t abort_flag, uint64_t timeout_ns) {
    int n = 0;
    if (lane == 0) {
        const uint64_t t0 = global_timer_ns();
        while ((n = ld_acquire_cta(ready)) <= rb) {
            n = 0;
            if (ld_shared_volatile(abort_flag) != 0) break;
            if (global_timer_ns() - t0 > timeout_ns) { st_shared_volatile(abort_flag, 1); break; }
        }
    }
    n = __shfl_sync(0xffffffffu, n, 0);
    __syncwarp();
    return n;
}
__device__ __forceinline__ int atomic_add_acq_rel(int* p, int v) {
    int old;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
    return old;
}

// Rows of a tile in each quarter of TMEM.  Up to 64 of them take an MMA with M = 64 (16 lanes of each quarter): the same time, half of the
// tensor core's power (128 tokens in a loop: 780 us instead of 880).
__device__ __forceinline__ int moe_lanes(int rows) { return rows <= 64 ? 16 : 32; }

__device__ __forceinline__ void st_shared_zero16(uint32_t addr) { asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(addr), "r"(0) : "memory"); }

// Work memory for the sums of a tile, [part_rows][256]: of a part, by the chunk that brought it (a chunk holds two at most, one that its
// beginning cuts off and one its end), or of a whole tile, two for each CTA in turn.
__device__ __forceinline__ float* moe_part(const MoeParams& p, const MoeList& l, int kind, int ch, int tile, bool whole, int buffer) {
    const int64_t at = whole ? static_cast<int64_t>(gridDim.x) * 4 + blockIdx.x * 2 + buffer
                             : (static_cast<int64_t>(kind) * gridDim.x + ch) * 2 + (l.start(ch) > tile * l.kb ? 0 : 1);
    return p.parts + at * p.part_rows * 256;
}

// Warps that finish rows of a tile: row r belongs to warp r % 4
__device__ __forceinline__ int moe_finishers(int rows) { return min(4, rows); }

// What a finishing warp does with a tile, or a part of one, once its sums have been written down (buffer `buffer` full in `phase`).  Each of
// the four counts for itself and its own rows: counting for all of them took two barriers of the four in every tile.  False if a wait
// has run out.
__device__ __forceinline__ bool moe_finish_tile(const MoeParams& p, const MoeSmem& sm, const MoeSegment& g, int buffer, uint32_t phase) {
    const int kind = g.kind, tile = g.tile, units = g.k1 - g.k0, rows = g.rows;
    const MoeList& l = sm.words->list[kind];
    const int fw = (threadIdx.x >> 5) - 4, lane = threadIdx.x & 31;
    const bool whole = units == l.kb;
    const bool mine = fw < moe_finishers(rows);
    // where the sums are (the divisions while others still work)
    const float* src = nullptr;
    int n = 1;
    if (kind == 0 && mine) {
        int c0 = g.chunk;
        if (!whole) {
            c0 = l.chunk_of(tile * l.kb);
            n = l.chunk_of(tile * l.kb + l.kb - 1) - c0 + 1;
        }
        src = moe_part(p, l, 0, c0, tile, whole, buffer);
    }
    if (!mbar_wait_asleep(sm.turn_full(buffer), phase, smem_u32(&sm.words->abort), p.timeout_ns)) return false;
    auto release = [&]() {                               // the buffer's values have been read
        __syncwarp();
        if (lane == 0) mbar_arrive(sm.turn_empty(buffer));
    };
    if (kind) {
        // rows of a whole tile are in their place already, parts are added up by the combine
        release();
        if (fw == 0 && lane == 0) {
            __threadfence();
            atomicAdd(p.counters + kMoeCtrUnits2, units);
        }
        return true;
    }
    if (!whole || !mine) release();                      // parts have memory of their own
    if (!mine) return true;
    if (!whole) {
        // the parts are added up by whoever brings the last one, in the order of the chunks (read from L2: other SMs wrote them)
        int have = 0;
        if (lane == 0) have = atomic_add_acq_rel(p.counters + p.ctr_tile1 + tile * 4 + fw, units) + units;
        if (__shfl_sync(0xffffffffu, have, 0) != l.kb) return true;
    }
    const bool turn = whole && rows <= kMoeTurnRows;
    const float* my_turn = sm.turn + buffer * kMoeTurnRows * kMoeTurnPitch;
    const int64_t step = static_cast<int64_t>(p.part_rows) * 256;        // from the first part to the second; two of these to each one after (moe_part)
    const bool do_clamp = p.clamp < 3.0e38f;
    // A row at a time, four columns each of gate and up in a lane (with one thread to a row, as the sums were held, a tile of few rows would
    // keep eight warps waiting for the few threads that have any); two rows' loads and two parts' in flight.
    for (int r = fw; r < rows; r += 8) {
        const bool two = r + 4 < rows;
        float4 v[2][2];                                  // [row][gate, up]
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i >> 1][i & 1] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (turn) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < 2 || two) v[i >> 1][i & 1] = *reinterpret_cast<const float4*>(my_turn + (r + (i & 2) * 2) * kMoeTurnPitch + (i & 1) * 128 + lane * 4);
        } else {
            const float* in = src + r * 256 + lane * 4;
#pragma unroll 1
            for (int c = 0; c < n; c += 2) {
                float4 f[2][4];
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (c + k < n && (i < 2 || two))
                            f[k][i] = __ldcg(reinterpret_cast<const float4*>(in + (c + k == 0 ? 0 : 2 * (c + k) - 1) * step + (i & 2) * 512 + (i & 1) * 128));
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (c + k < n && (i < 2 || two)) add4(v[i >> 1][i & 1], f[k][i]);
            }
        }
#pragma unroll 1
        for (int i = 0; i < (two ? 2 : 1); ++i)
            moe_finish_row(p, i ? v[1][0] : v[0][0], i ? v[1][1] : v[0][1], do_clamp, static_cast<int64_t>(g.first) + r + 4 * i, g.out, lane);
    }
    if (whole) release();
    __syncwarp();
    if (lane == 0) {
        __threadfence();
        atomicAdd(p.counters + p.ctr_done1 + g.block, 1);
        atomicAdd(p.counters + kMoeCtrRows1, 1);
    }
    return true;
}

// The combine, by the finishing warps of every CTA once the sums of all `units` of the second product are written: each token's rows, in the
// order of its slots, four columns a thread.  A tile that was cut is read as its parts, in the order of the chunks: adding them up
// first, by whoever brings the last one, and reading the sum then made the end of a call for one token 7 us long instead of 4.
__device__ __forceinline__ void moe_combine(const MoeParams& p, const MoeSmem& sm, uint8_t* ring, int units) {
    const int tid = threadIdx.x - 128, lane = threadIdx.x & 31;
    const MoeList& l = sm.words->list[1];
    const int nt2 = (p.hidden + 255) / 256;
    // The operand ring has done its work.  Of each route: first tile of its block | row << 16; of each tile: place of its first part | parts
    // << 16, or 0 parts if it is whole.
    uint32_t* place = reinterpret_cast<uint32_t*>(ring);
    uint32_t* parts_of = place + kMoeMaxRoutes;
    const bool cut = l.shares;                                       // (fewer tiles than 16 for each CTA, and a GPU has fewer than 1024 SMs)
    static_assert(kMoeMaxRoutes * 4 + kMoeStreamTiles * 1024 * 4 <= kMoeRingBytes && kMoeStreamTiles * 1024 <= 65536, "places and parts");
    const int64_t step = static_cast<int64_t>(p.part_rows) * 256;    // from a tile's first part to its second; two of these to each one after (moe_part)
    const float* parts2 = p.parts + static_cast<int64_t>(gridDim.x) * 2 * step;      // of the second product
    if (cut) {
        const int blocks = sm.words->blocks;
        for (int b = tid >> 5; b < blocks; b += 4) {
            const uint2 blk = sm.block[b];
            for (uint32_t r = lane; r < blk.x >> 16; r += 32) place[sm.route[blk.y + r]] = static_cast<uint32_t>(b * nt2) | r << 16;
        }
        // (the divisions of chunk_of here, once for each tile and while others still work: 24 of them in a thread's way to its loads took 6 us)
        for (int t = tid; t < l.tiles; t += 128) {
            const int c0 = l.chunk_of(t * l.kb), n = l.chunk_of(t * l.kb + l.kb - 1) - c0 + 1;
            parts_of[t] = static_cast<uint32_t>(c0 * 2 + 1) | static_cast<uint32_t>(n == 1 ? 0 : n) << 16;
        }
    }
    const bool ok = tid != 0 || moe_wait_count(p.counters + kMoeCtrUnits2, units, smem_u32(&sm.words->abort), p.timeout_ns);
    if (!__all_sync(0xffffffffu, ok)) return;
    if (lane == 0) mbar_arrive(sm.finish_bar());
    if (!mbar_wait_warp(sm.finish_bar(), 0, smem_u32(&sm.words->abort), p.timeout_ns)) return;
    // A warp takes 64 columns of a token: `group` slots side by side, 32 / group lanes to each, then a sum over the slots in a fixed order.
    // (Eight slots one after the other in each thread, unrolled, were code that every SM ran once: fetching it took 4 us.)
    int group = 1;
    while (group < 8 && group < p.topk) group *= 2;
    const int lanes = 32 / group, my_slot = lane / lanes, my_col = lane % lanes * 4;
    const int strips = p.hidden / 64;
#pragma unroll 1
    for (int i = (tid >> 5) * gridDim.x + blockIdx.x; i < p.tokens * strips; i += gridDim.x * 4) {
        const int t = i / strips, col0 = (i - t * strips) * 64;
#pragma unroll 1
        for (int c0 = 0; c0 < 64; c0 += lanes * 16) {                // up to four runs of four columns a lane; with one slot half the lanes have none
            const int c = c0 + my_col, col = col0 + c;
            float4 a[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
            for (int s = my_slot; s < p.topk; s += group) {
                const int r = t * p.topk + s;
                if (c >= 64 || !((sm.valid[r >> 5] >> (r & 31)) & 1u)) continue;
                const float* src = p.rows_out + static_cast<int64_t>(r) * p.hidden + col;
                float w = 1.0f;
                int n = 1;                                           // parts
                if (cut) {
                    const uint32_t at = place[r], parts = parts_of[(at & 0xffff) + (col >> 8)];
                    if (parts >> 16) {
                        n = static_cast<int>(parts >> 16);
                        src = parts2 + (parts & 0xffff) * step + (at >> 16) * 256 + (col & 255);
                        w = p.route_w[r];
                    }
                }
                float4 f[2][4];
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        f[k][j] = k < n && c + j * lanes * 4 < 64 ? __ldcg(reinterpret_cast<const float4*>(src + k * step + j * lanes * 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int j = 0; j < 4; ++j) add4(f[0][j], f[1][j]);
#pragma unroll 1
                for (int k = 2; k < n; ++k)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (c + j * lanes * 4 < 64) add4(f[0][j], __ldcg(reinterpret_cast<const float4*>(src + (2 * k - 1) * step + j * lanes * 4)));
#pragma unroll
                for (int j = 0; j < 4; ++j) { a[j].x = fmaf(f[0][j].x, w, a[j].x); a[j].y = fmaf(f[0][j].y, w, a[j].y); a[j].z = fmaf(f[0][j].z, w, a[j].z); a[j].w = fmaf(f[0][j].w, w, a[j].w); }
            }
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll 1
                for (int o = lanes; o < 32; o *= 2) {
                    a[j].x += __shfl_xor_sync(0xffffffffu, a[j].x, o); a[j].y += __shfl_xor_sync(0xffffffffu, a[j].y, o);
                    a[j].z += __shfl_xor_sync(0xffffffffu, a[j].z, o); a[j].w += __shfl_xor_sync(0xffffffffu, a[j].w, o);
                }
                if (my_slot == 0 && c + j * lanes * 4 < 64)
                    *reinterpret_cast<uint2*>(p.y + static_cast<int64_t>(t) * p.hidden + col + j * lanes * 4) = make_uint2(pack_bf16x2(a[j].x, a[j].y), pack_bf16x2(a[j].z, a[j].w));
            }
        }
    }
}

__global__ void __launch_bounds__(kMoeThreads, 1)
moe_experts_kernel(const __grid_constant__ CUtensorMap tm_w1, const __grid_constant__ CUtensorMap tm_w2, const __grid_constant__ MoeParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t smem_base = smem_u32(smem);
    const MoeSmem sm(smem);
    pdl_launch();
    auto full_bar = [&](int s) { return sm.bars + 8u * s; };
    auto empty_bar = [&](int s) { return sm.bars + 8u * (kMoeMaxStages + s); };
    auto tfull_bar = [&](int a) { return sm.bars + 8u * (2 * kMoeMaxStages + a); };
    auto tempty_bar = [&](int a) { return sm.bars + 8u * (2 * kMoeMaxStages + 2 + a); };
    auto sfull_bar = [&](int c) { return sm.bars + 8u * (2 * kMoeMaxStages + 4 + c); };
    auto sempty_bar = [&](int c) { return sm.bars + 8u * (2 * kMoeMaxStages + 4 + kMoeSegments + c); };
    const uint32_t abort_flag = smem_u32(&sm.words->abort);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kMoeMaxStages; ++s) { mbar_init(full_bar(s), 3); mbar_init(empty_bar(s), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(tfull_bar(a), 1); mbar_init(tempty_bar(a), 8); }
        for (int c = 0; c < kMoeSegments; ++c) { mbar_init(sfull_bar(c), 1); mbar_init(sempty_bar(c), 15); }
        for (int b = 0; b < 2; ++b) { mbar_init(sm.turn_full(b), 8); mbar_init(sm.turn_empty(b), 4); }
        mbar_init(sm.finish_bar(), 4);
        st_shared_volatile(abort_flag, 0);
        st_release_cta(smem_u32(&sm.words->ready), 0);
        fence_barrier_init();
        prefetch_tensormap(&tm_w1);
        prefetch_tensormap(&tm_w2);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&sm.words->tmem), 512);
        tmem_relinquish();
    }
    // ---- the plan, by every CTA for itself: routes sorted by expert (stable), blocks of up to 128 routes.  Each warp counts and later
    // places a run of the routes; between the two the counts become places, by warp for each expert and by expert.
    const int routes = p.tokens * p.topk;
    int first_claim = 0;                                             // its answer is not needed before the plan
    {
        constexpr int kWarps = kMoeThreads / 32;
        uint32_t* s_first = reinterpret_cast<uint32_t*>(smem);       // [experts]; the operand ring is not in use yet
        uint16_t* s_id = reinterpret_cast<uint16_t*>(s_first + MM_MAX_EXPERTS);
        uint16_t* s_hist = s_id + kMoeMaxRoutes;                     // [warps][experts, even]
        const int pitch = (p.experts + 1) & ~1;
        static_assert(MM_MAX_EXPERTS * 4 + kMoeMaxRoutes * 2 + kWarps * MM_MAX_EXPERTS * 2 <= kMoeRingBytes, "the plan");
        uint16_t* hist = s_hist + warp * pitch;
        const int run = (routes + 32 * kWarps - 1) / (32 * kWarps) * 32, run0 = warp * run, run1 = min(routes, run0 + run);
        const int runs = (routes + run - 1) / run;                   // warps that have one
        if (warp < runs)
            for (int e = lane * 2; e < pitch; e += 64) *reinterpret_cast<uint32_t*>(hist + e) = 0;
        __syncwarp();
        pdl_wait();                                                  // routes, cast x and zeroed counters of the first launch
        if (threadIdx.x == 0) first_claim = atomicAdd(p.counters, 1);
        for (int r0 = run0; r0 < run1; r0 += 32) {
            const int r = r0 + lane;
            const int e = r < run1 ? p.route_expert[r] : -1;
            const uint32_t same = __match_any_sync(0xffffffffu, e);
            const uint32_t valid = __ballot_sync(0xffffffffu, e >= 0);
            if (r < run1) s_id[r] = static_cast<uint16_t>(e);        // -1: 0xffff
            if (e >= 0 && (same >> lane) == 1u) hist[e] += __popc(same);                 // the group's last lane
            if (lane == 0) sm.valid[r0 / 32] = valid;
            __syncwarp();
        }
        __syncthreads();
        for (int e = threadIdx.x; e < p.experts; e += kMoeThreads) {
            uint32_t n = 0;
#pragma unroll 4
            for (int w = 0; w < runs; ++w) {
                const uint32_t c = s_hist[w * pitch + e];
                s_hist[w * pitch + e] = static_cast<uint16_t>(n);
                n += c;
            }
            s_first[e] = n;
        }
        __syncthreads();
        if (warp == 0) {
            // counts -> first places, and the blocks of each expert; a lane takes neighbouring experts
            const int per = (p.experts + 31) / 32, e0 = lane * per, e1 = min(p.experts, e0 + per);
            uint32_t n_own = 0, b_own = 0, most = 0, fin = 0;
            for (int e = e0; e < e1; ++e) {
                const uint32_t n = s_first[e];
                n_own += n; b_own += (n + 127) >> 7; most = max(most, n);
                fin += 4 * (n >> 7) + min(4u, n & 127u);
            }
            uint32_t n_scan = n_own, b_scan = b_own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t a = __shfl_up_sync(0xffffffffu, n_scan, o), c = __shfl_up_sync(0xffffffffu, b_scan, o);
                if (lane >= o) { n_scan += a; b_scan += c; }
            }
            const int blocks = static_cast<int>(__shfl_sync(0xffffffffu, b_scan, 31));
            uint32_t at = n_scan - n_own, b = b_scan - b_own;
            for (int e = e0; e < e1; ++e) {
                const uint32_t n = s_first[e];
                s_first[e] = at;
                for (uint32_t i = 0; i < n; i += 128) sm.block[b++] = make_uint2(static_cast<uint32_t>(e) | min(128u, n - i) << 16, at + i);
                at += n;
            }
            most = __reduce_max_sync(0xffffffffu, most);
            fin = __reduce_add_sync(0xffffffffu, fin);
            if (lane == 0) {
                sm.words->blocks = blocks;
                sm.words->most = static_cast<int>(most);
                sm.words->finishers = static_cast<int>(fin);
                sm.words->list[0] = moe_list(blocks * (p.inter / 128), p.hidden / 128, gridDim.x);
                sm.words->list[1] = moe_list(blocks * ((p.hidden + 255) / 256), p.inter / 128, gridDim.x);
            }
        }
        __syncthreads();
        for (int r0 = run0; r0 < run1; r0 += 32) {
            const int r = r0 + lane;
            const uint32_t e = r < run1 ? s_id[r] : 0xffffu;
            const uint32_t same = __match_any_sync(0xffffffffu, e);
            uint32_t before = 0;
            if (e != 0xffffu) {
                before = hist[e];
                sm.route[s_first[e] + before + __popc(same & ((1u << lane) - 1u))] = static_cast<uint16_t>(r);
            }
            __syncwarp();
            if (e != 0xffffu && (same >> lane) == 1u) hist[e] = static_cast<uint16_t>(before + __popc(same));
            __syncwarp();
        }
        fence_proxy_async_smem();                                    // these words become TMA destinations
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = sm.words->tmem;

    const int n_blocks = sm.words->blocks;                                  // blocks of routes
    const bool few_rows = sm.words->most <= kMoeFewRows;
    const int stages = few_rows ? kMoeMaxStages : 4;
    const uint32_t a_bytes = few_rows ? kMoeFewRows * 128 : 128 * 128, stage_bytes = a_bytes + kMoeBBytes;
    const uint32_t topk_magic = 0xffffffffu / static_cast<uint32_t>(p.topk) + 1u;        // r / topk, exact for r < 2^16; topk 1 apart
    auto token_of = [&](uint32_t r) { return p.topk == 1 ? r : __umulhi(r, topk_magic); };
    const int kb1 = p.hidden / 128, kb2 = p.inter / 128;
    const int nt1 = p.inter / 128, nt2 = (p.hidden + 255) / 256;
    const int chunks1 = sm.words->list[0].chunks, chunks = n_blocks == 0 ? 0 : chunks1 + sm.words->list[1].chunks;

    struct Place { int slot = 0; uint32_t phase = 0; };              // in the ring of segments
    auto segment_came = [&](const Place& at) { return mbar_wait_warp(sfull_bar(at.slot), at.phase, abort_flag, p.timeout_ns); };
    auto segment_done = [&](Place& at) {                             // one thread of a warp, or the MMA thread
        mbar_arrive(sempty_bar(at.slot));
    };
    auto step = [&](Place& at) { if (++at.slot == kMoeSegments) { at.slot = 0; at.phase ^= 1u; } };
    if (warp < 4) {
        regs_dec<56>();
        if (warp == 0) {
            // ------------------------------------------------------------------ claims and weights
            if (lane == 0) {
                int stage = 0; uint32_t phase = 0;
                Place at;
                bool alive = true, first = true;
                auto publish = [&](const MoeSegment& g) {
                    if (!mbar_wait_often(sempty_bar(at.slot), at.phase ^ 1u, abort_flag, p.timeout_ns)) return false;
                    sm.words->segment[at.slot] = g;
                    mbar_arrive(sfull_bar(at.slot));
                    step(at);
                    return true;
                };
                while (alive) {
                    // Not before the copies of the last chunk are under way: whoever claims ahead takes a second share while others have
                    // none.  The ring holds more work than the claim takes.
                    const int id = first ? first_claim : atomicAdd(p.counters, 1);
                    first = false;
                    if (id >= chunks) break;
                    MoeSegment g;
                    g.kind = id >= chunks1 ? 1 : 0;
                    g.chunk = id - (g.kind ? chunks1 : 0);
                    const MoeList l = sm.words->list[g.kind];
                    const CUtensorMap* map = g.kind ? &tm_w2 : &tm_w1;
                    const int per_block = g.kind ? nt2 : nt1;        // tiles go block by block: the second product begins with what was finished first
                    int u = l.start(g.chunk);
                    const int end = l.start(g.chunk + 1);
                    while (u < end && alive) {
                        g.tile = u / l.kb;
                        g.k0 = u - g.tile * l.kb;
                        g.k1 = min(l.kb, g.k0 + end - u);
                        g.block = g.tile / per_block;
                        g.out = g.tile - g.block * per_block;
                        const uint2 blk = sm.block[g.block];
                        g.expert = blk.x & 0xffff;
                        g.rows = blk.x >> 16;
                        g.first = blk.y;
                        if (!publish(g)) { alive = false; break; }
                        const int64_t tiled0 = (static_cast<int64_t>(g.expert) * per_block + g.out) * l.kb;
                        const int row_a = g.kind ? g.expert * p.hidden + g.out * 256 : g.expert * 2 * p.inter + g.out * 128;
                        const int row_b = g.kind ? row_a + 128 : row_a + p.inter;
                        for (int k = g.k0; k < g.k1; ++k) {
                            if (!mbar_wait_often(empty_bar(stage), phase ^ 1u, abort_flag, p.timeout_ns)) { alive = false; break; }
                            const uint32_t dst = smem_base + stage * stage_bytes + a_bytes;
                            mbar_arrive_expect_tx(full_bar(stage), 256 * 128);
                            if (p.tiled) {
                                tma_load_2d(dst, map, 0, static_cast<int32_t>((tiled0 + k) * 256), full_bar(stage));
                            } else {
                                tma_load_2d(dst, map, k * 128, row_a, full_bar(stage));
                                tma_load_2d(dst + 128 * 128, map, k * 128, row_b, full_bar(stage));
                            }
                            if (++stage == stages) { stage = 0; phase ^= 1u; }
                        }
                        u += g.k1 - g.k0;
                    }
                }
                MoeSegment none;
                none.kind = -1;
                if (alive) publish(none);
            }
        } else if (warp == 1) {
            // ------------------------------------------------------------------ MMA
            if (lane == 0) {
                int stage = 0; uint32_t phase = 0;
                int acc = 0; uint32_t acc_phase = 0;
                Place at;
                bool alive = true;
                while (alive) {
                    if (!mbar_wait_often(sfull_bar(at.slot), at.phase, abort_flag, p.timeout_ns)) break;
                    const MoeSegment* g = &sm.words->segment[at.slot];
                    if (g->kind < 0) break;
                    const int units = g->k1 - g->k0;
                    const uint32_t idesc = moe_lanes(g->rows) == 16 ? umma_idesc_f8(64, 256) : umma_idesc_f8(128, 256);
                    segment_done(at);
                    step(at);
                    for (int u = 0; u < units; ++u) {
                        if (!mbar_wait_often(tempty_bar(acc), acc_phase ^ 1u, abort_flag, p.timeout_ns)) { alive = false; break; }
                        if (!mbar_wait_often(full_bar(stage), phase, abort_flag, p.timeout_ns)) { alive = false; break; }
                        tc_fence_after();
                        const uint64_t da = umma_desc_k_sw128(smem_base + stage * stage_bytes);
                        const uint64_t db = umma_desc_k_sw128(smem_base + stage * stage_bytes + a_bytes);
#pragma unroll
                        for (int k = 0; k < 4; ++k) umma_f8(tmem_base + acc * 256, da + 2u * k, db + 2u * k, idesc, k != 0 ? 1u : 0u);
                        umma_commit(tfull_bar(acc));
                        umma_commit(empty_bar(stage));
                        if (++stage == stages) { stage = 0; phase ^= 1u; }
                        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
                    }
                }
            }
        } else {
            // ------------------------------------------------------------------ token operand: rows gathered by route, 16 bytes a lane
            constexpr int kAhead = 2;                                // copies in flight before the oldest is handed over
            int stage = 0; uint32_t phase = 0;                       // next stage to fill
            int slot = 0;                                            // next place in the ring of scales
            int hand = 0, pending = 0;                               // next stage to hand over, stages filled but not handed over
            const int l64 = threadIdx.x - 64;
            const int piece = l64 & 7;
            int ready_blocks = 0;                                    // this CTA's chunks of the second product go up in blocks of routes
            Place at;
            bool alive = true;
            // Rows behind a tile's last one are read by its MMAs all the same; zeroes there cost the least power (128 tokens in a loop: 737
            // us instead of 761).  Rows that a stage may hold, a byte for each stage.
            uint64_t filled = 0x0101010101010101ull * (few_rows ? kMoeFewRows : 128u);
            auto hand_over = [&]() {
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(full_bar(hand));
                if (++hand == stages) hand = 0;
                --pending;
            };
            auto drain = [&]() {
                cp_async_wait<0>();
                while (pending > 0) hand_over();
            };
            while (alive) {
                if (!__all_sync(0xffffffffu, mbar_test(sfull_bar(at.slot), at.phase))) drain();          // nothing to go on with yet
                if (!segment_came(at)) break;
                const MoeSegment g = sm.words->segment[at.slot];
                if (g.kind < 0) break;
                __syncwarp();
                if (lane == 0) segment_done(at);
                step(at);
                const int kind = g.kind, rb = g.block, rows = g.rows, first = g.first;
                const int pitch = kind ? p.inter : p.hidden;
                const uint8_t* src = kind ? p.act_q : p.xq;
                const float* src_sf = kind ? p.act_sf : p.xsf;
                const int sf_pitch = kind ? p.act_sf_pitch : kb1;
                {
                    // the last two lanes bring the weights' scales: gate and up, or two blocks of outputs (the last tile may have one)
                    const int n_block = kind ? min(2 * g.out + (l64 & 1), kb1 - 1) : g.out + (l64 & 1) * nt1;
                    const float* sb = kind ? p.s2 + (static_cast<int64_t>(g.expert) * kb1 + n_block) * kb2
                                           : p.s1 + (static_cast<int64_t>(g.expert) * 2 * nt1 + n_block) * kb1;
                    if (kind && rb >= ready_blocks) {
                        if (l64 >= 62) asm volatile("prefetch.global.L2 [%0];" ::"l"(sb + g.k0));        // (a line, 32 k blocks, of what comes from HBM)
                        // The rows this product reads.  One warp asks for both, and if it has to wait, everything filled so far is handed
                        // over first, because the tiles that finish those rows may be this CTA's own.
                        if (warp == 2) {
                            auto look = [&]() {                      // lane 0: all tiles of the first product, or at least this block's
                                const int all = ld_acquire_gpu(p.counters + kMoeCtrRows1), own = ld_acquire_gpu(p.counters + p.ctr_done1 + rb);
                                return all >= sm.words->finishers * nt1 ? n_blocks : own >= moe_finishers(rows) * nt1 ? rb + 1 : 0;
                            };
                            ready_blocks = __shfl_sync(0xffffffffu, lane == 0 ? look() : 0, 0);
                            if (ready_blocks == 0) {
                                drain();
                                int n = 0;
                                if (lane == 0 && moe_wait_count(p.counters + p.ctr_done1 + rb, moe_finishers(rows) * nt1, abort_flag, p.timeout_ns)) n = rb + 1;
                                ready_blocks = __shfl_sync(0xffffffffu, n, 0);
                            }
                            if (ready_blocks == 0) { alive = false; break; }
                            if (lane == 0) st_release_cta(smem_u32(&sm.words->ready), ready_blocks);
                            __syncwarp();                            // what lane 0 has acquired, the others may read
                        } else {
                            if (!__all_sync(0xffffffffu, ld_acquire_cta(smem_u32(&sm.words->ready)) > rb)) drain();
                            ready_blocks = moe_wait_ready(smem_u32(&sm.words->ready), rb, lane, abort_flag, p.timeout_ns);
                            if (ready_blocks == 0) { alive = false; break; }
                        }
                    }
                    for (int k = g.k0; k < g.k1; ++k) {
                        if (!mbar_wait_warp(empty_bar(stage), phase ^ 1u, abort_flag, p.timeout_ns)) { alive = false; break; }
                        const uint32_t sdst = smem_u32(sm.scale) + slot * kMoeScaleBytes;
                        for (int r = l64; r < rows; r += 64) {
                            const uint32_t row = kind ? first + r : token_of(sm.route[first + r]);
                            cp_async_4(sdst + r * 4, src_sf + static_cast<int64_t>(row) * sf_pitch + k);
                        }
                        if (l64 >= 62) cp_async_4(sdst + 512 + (l64 - 62) * 4, sb + k);
                        if (++slot == kMoeScaleSlots) slot = 0;
                        const uint32_t dst = smem_base + stage * stage_bytes;
                        for (int r = l64 >> 3; r < rows; r += 8) {
                            const uint32_t row = kind ? first + r : token_of(sm.route[first + r]);
                            cp_async_16(dst + r * 128 + ((piece ^ (r & 7)) << 4), src + static_cast<int64_t>(row) * pitch + k * 128 + piece * 16);
                        }
                        cp_async_commit();
                        const int before = static_cast<int>(filled >> (8 * stage)) & 255;
                        if (before != rows) {
                            for (int r = rows + (l64 >> 3); r < before; r += 8) st_shared_zero16(dst + r * 128 + piece * 16);
                            filled ^= static_cast<uint64_t>(before ^ rows) << (8 * stage);
                        }
                        ++pending;
                        if (++stage == stages) { stage = 0; phase ^= 1u; }
                        if (pending > kAhead) {
                            cp_async_wait<kAhead>();
                            hand_over();
                        }
                    }
                }
            }
            drain();
        }
        __syncwarp();
    } else if (warp < 8) {
        // ---------------------------------------------------------------------- finishing
        regs_dec<104>();
        if (n_blocks == 0) {                                         // no route at all: the sum is empty
            for (int64_t i = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x - 128; i < static_cast<int64_t>(p.tokens) * p.hidden / 8;
                 i += static_cast<int64_t>(gridDim.x) * 128)
                reinterpret_cast<uint4*>(p.y)[i] = make_uint4(0, 0, 0, 0);
        }
        int buffer = 0; uint32_t buffer_phase = 0;
        Place at;
        while (true) {
            if (!segment_came(at)) break;
            const MoeSegment* g = &sm.words->segment[at.slot];
            if (g->kind < 0) {
                if (n_blocks > 0) moe_combine(p, sm, smem, n_blocks * nt2 * kb2);
                break;
            }
            if (!moe_finish_tile(p, sm, *g, buffer, buffer_phase)) break;
            __syncwarp();
            if (lane == 0) segment_done(at);
            step(at);
            buffer ^= 1;
            if (buffer == 0) buffer_phase ^= 1u;
        }
    } else {
        // ---------------------------------------------------------------------- sums
        regs_inc<176>();
        const int q = warp & 3, half = (warp - 8) >> 2;
        int acc = 0; uint32_t acc_phase = 0;
        int slot = 0;                                                // place of the next unit in the ring of scales
        int buffer = 0; uint32_t buffer_phase = 0;
        Place at;
        bool alive = true;
        while (alive) {
            if (!segment_came(at)) break;
            const MoeSegment* g = &sm.words->segment[at.slot];
            if (g->kind < 0) break;
            const int units = g->k1 - g->k0;
            const int lanes = moe_lanes(g->rows), et = lane < lanes ? q * lanes + lane : 127;                            // row of the tile; 127: none
            if (q * lanes < g->rows) {
                // column parts A and B of this thread: gate and up, or two neighbouring runs of 64 outputs
                const int col_a = g->kind ? half * 128 : half * 64, col_b = g->kind ? col_a + 64 : col_a + 128;
                const int sb_a = g->kind ? 128 + half : 128, sb_b = g->kind ? 128 + half : 129;
                // Warps without a row of the tile take no part in this: waiting beside the others they slow them down.  The barrier
                // that gives the accumulator back counts all eight, so the warps of the first rows arrive for the idle ones.
                const uint32_t arrivals = q == 0 ? 5u - static_cast<uint32_t>((g->rows + lanes - 1) / lanes) : 1u;
                uint64_t sum[64];                                    // pairs: 64 columns of part A, 64 of part B
#pragma unroll
                for (int j = 0; j < 64; ++j) sum[j] = 0ull;
#pragma unroll 1
                for (int u = 0; u < units; ++u) {
                    if (!mbar_wait_warp(tfull_bar(acc), acc_phase, abort_flag, p.timeout_ns)) { alive = false; break; }
                    tc_fence_after();
                    const float* sc = sm.scale + slot * (kMoeScaleBytes / 4);
                    const float s_row = sc[et];
                    const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * 256;
                    moe_promote<false>(sum, t_addr + col_a, s_row * sc[sb_a], 0, 0);
                    moe_promote<true>(sum + 32, t_addr + col_b, s_row * sc[sb_b], tempty_bar(acc), arrivals);
                    if (++slot == kMoeScaleSlots) slot = 0;
                    if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
                }
                if (!alive || !mbar_wait_warp(sm.turn_empty(buffer), buffer_phase ^ 1u, abort_flag, p.timeout_ns)) break;
                // Where the sums go next: rows of activations that are finished here to shared memory if they fit; else, and parts of a
                // tile, to work memory; whole rows of outputs straight to their place.
                if (lane < lanes && et < g->rows) {
                    const MoeList& l = sm.words->list[g->kind];
                    const bool whole = g->k1 - g->k0 == l.kb;
                    if (g->kind && whole) {
                        if (half * 128 < p.hidden - g->out * 256) {
                            const uint32_t route = sm.route[g->first + et];
                            const float w = p.route_w[route];
                            float* o = p.rows_out + static_cast<int64_t>(route) * p.hidden + g->out * 256 + half * 128;
#pragma unroll
                            for (int j = 0; j < 128; j += 4) {
                                const float4 f = unpack_f32x4(sum[j / 2], sum[j / 2 + 1]);
                                *reinterpret_cast<float4*>(o + j) = make_float4(f.x * w, f.y * w, f.z * w, f.w * w);
                            }
                        }
                    } else {
                        const bool turn = whole && g->rows <= kMoeTurnRows;
                        float* o = turn ? sm.turn + (buffer * kMoeTurnRows + et) * kMoeTurnPitch : moe_part(p, l, g->kind, g->chunk, g->tile, whole, buffer) + et * 256;
#pragma unroll
                        for (int j = 0; j < 128; j += 4)
                            *reinterpret_cast<float4*>(o + (j < 64 ? col_a + j : col_b + j - 64)) = unpack_f32x4(sum[j / 2], sum[j / 2 + 1]);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(sm.turn_full(buffer));
            } else {
                // Not ahead of the others, though: a barrier tells a phase from the one after the next by nothing.  So an idle warp is
                // counted where the sums are handed on, and waits there, mostly asleep, until the others have come.
                if (!mbar_wait_warp(sm.turn_empty(buffer), buffer_phase ^ 1u, abort_flag, p.timeout_ns)) break;
                if (lane == 0) mbar_arrive(sm.turn_full(buffer));
                if (!mbar_wait_asleep(sm.turn_full(buffer), buffer_phase, abort_flag, p.timeout_ns)) break;
                slot = (slot + units) % kMoeScaleSlots;
                acc += units;
                acc_phase ^= static_cast<uint32_t>(acc >> 1) & 1u;
                acc &= 1;
            }
            buffer ^= 1;
            if (buffer == 0) buffer_phase ^= 1u;
            __syncwarp();
            if (lane == 0) segment_done(at);
            step(at);
        }
    }

    if (ld_shared_volatile(abort_flag) != 0) {
        // a bounded wait expired: give copies that may still be in flight time to land, then report
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 1000000ull) __nanosleep(1000);
        if (threadIdx.x == 0) b128_report(p.status, MM_ERR_PIPE_TIMEOUT, 30, blockIdx.x, chunks, 0);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

}  // namespace mm
