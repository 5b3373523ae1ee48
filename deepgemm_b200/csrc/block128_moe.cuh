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
// wherever the share ends, and the parts of a tile meet in memory: whoever brings the last part adds them up in order.  Else a chunk is
// a tile.  Weights need nothing but the routes, so the TMA warp runs ahead into the second product, up to the depth of its ring, while the
// activations of the first are still being finished; only the token operand waits for them.
//
// A chunk of the second product is claimed only after every chunk of the first one has been, and by a CTA that runs; so what a CTA waits
// for is always being worked on, however many of the CTAs are resident, and two such launches may share a GPU.
//
// Tile = up to 128 routes of one expert x 256 weight rows (first product: 128 gate rows and their 128 up rows, so that a tile holds
// one whole block of the activations' cast).  Warp 0 = TMA (weights), 1 = MMA, 2-3 = token operand (cp.async: rows are gathered by
// route), 4-11 = epilogue, with the promotion by block scales of block128_gemm.cuh.
#pragma once
#include "block128.cuh"
#include "block128_gemm.cuh"

namespace mm {

constexpr int kMoeMaxRoutes = 4096;
constexpr int kMoeMaxBlocks = MM_MAX_EXPERTS + kMoeMaxRoutes / 128;      // of up to 128 routes of one expert
constexpr int kMoeStages = 4;
constexpr int kMoeABytes = 128 * 128;
constexpr int kMoeStageBytes = kMoeABytes + 256 * 128;
constexpr int kMoePlanBytes = kMoeMaxRoutes * 4 + kMoeMaxBlocks * 8;
constexpr int kMoeSmemBytes = kMoeStages * kMoeStageBytes + kMoePlanBytes + 1024 /* row maxima */ + 512 /* barriers */;
static_assert(kMoeSmemBytes <= 232448, "exceeds the 227 KiB of shared memory a CTA can have");
constexpr int kMoeClaims = 4;
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
    // counters: [0] claims, [32 ..) finished tiles of the first product by block of routes, then of the second by output tile, then
    // k blocks that have arrived for each tile that was cut, of either product
    int ctr_done1, ctr_done2, ctr_tile1, ctr_tile2;
    const float* s1; const float* s2;
    int tiled;
    uint8_t* act_q; float* act_sf;           // [routes][inter], [routes][inter / 128], by place in the sorted list
    float* rows_out;                         // [routes][hidden]: weighted rows of the second product, by route
    float* parts; int part_rows;             // [2 products][chunks][2][part_rows][256]
    __nv_bfloat16* y;
    float clamp;
    int* status;
    uint64_t timeout_ns;
};

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// kPer: experts per lane.  Ties go to the lower index; NaN and -inf logits are never chosen.
template <int kPer>
__device__ __forceinline__ void moe_topk(const MoeParams& p, int t, int lane) {
    float v[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = lane + 32 * i;
        const float l = e < p.experts ? p.logits[t * p.logits_stride + e] : -INFINITY;
        v[i] = l == l ? l : -INFINITY;
    }
    float sel = 0.0f, sum = 0.0f, top = 0.0f;
    int sel_e = -1;
    for (int k = 0; k < p.topk; ++k) {
        float best = -INFINITY;
        int best_e = -1;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (v[i] > best) { best = v[i]; best_e = lane + 32 * i; }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float ob = __shfl_xor_sync(0xffffffffu, best, o);
            const int oe = __shfl_xor_sync(0xffffffffu, best_e, o);
            if (ob > best || (ob == best && oe >= 0 && oe < best_e)) { best = ob; best_e = oe; }
        }
        if (best_e < 0) break;                                       // nothing left to choose from
        if (k == 0) top = best;
        const float w = best == top ? 1.0f : expf(best - top);       // equal infinities share alike
        sum += w;
        if (lane == k) { sel = w; sel_e = best_e; }
        if ((best_e & 31) == lane) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) if (i == (best_e >> 5)) v[i] = -INFINITY;
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
            float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (g < groups) load8(p.x, t * p.x_stride + col, B128_BF16, v);
            const float top = group_top(half_warp_max(amax8(v)));
            if (g < groups) {
                *reinterpret_cast<uint2*>(p.xq_out + static_cast<int64_t>(t) * p.hidden + col) = quantise8(v, GroupQuotient(top));
                if ((lane & 15) == 0) p.xsf_out[t * groups + g] = __fdiv_rn(top, 448.0f);
            }
        }
    }
}

// The list of weight blocks of one product: tiles * kb units, cut into chunks.
struct MoeList {
    int tiles, kb, chunks;
    bool shares;                                                     // chunks are equal shares, else tiles
    __device__ __forceinline__ int start(int c) const {
        return shares ? static_cast<int>(static_cast<int64_t>(tiles) * kb * c / chunks) : c * kb;
    }
    __device__ __forceinline__ int chunk_of(int unit) const {        // the chunk c with start(c) <= unit < start(c + 1)
        return shares ? static_cast<int>(((static_cast<int64_t>(unit) + 1) * chunks - 1) / (static_cast<int64_t>(tiles) * kb)) : unit / kb;
    }
};
__device__ __forceinline__ MoeList moe_list(int tiles, int kb, int ctas) {
    MoeList l;
    l.tiles = tiles; l.kb = kb;
    l.shares = tiles < kMoeStreamTiles * ctas;
    l.chunks = l.shares ? min(ctas, tiles * kb) : tiles;
    return l;
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

// 64 columns of one accumulator
template <bool kLast>
__device__ __forceinline__ void moe_promote64(uint64_t* acc, uint32_t taddr, float s, uint32_t free_bar, int lane) {
    const uint64_t s2 = pack_f32x2(__float_as_uint(s), __float_as_uint(s));
    uint32_t v0[32], v1[32];
    tmem_ld_32x32(taddr, v0);
    tmem_ld_32x32(taddr + 32, v1);
    tmem_ld_wait();
    if (kLast) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(free_bar);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) fma_f32x2(acc[j], pack_f32x2(v0[2 * j], v0[2 * j + 1]), s2);
#pragma unroll
    for (int j = 0; j < 16; ++j) fma_f32x2(acc[16 + j], pack_f32x2(v1[2 * j], v1[2 * j + 1]), s2);
}

// Bounded wait until *p (written by other CTAs, released) has reached `want`.
__device__ __forceinline__ bool moe_wait_count(const int* p, int want, volatile int* abort_flag, uint64_t timeout_ns) {
    if (ld_acquire_gpu(p) >= want) return true;
    const uint64_t t0 = global_timer_ns();
    while (ld_acquire_gpu(p) < want) {
        if (*abort_flag != 0) return false;
        if (global_timer_ns() - t0 > timeout_ns) { *abort_flag = 1; return false; }
    }
    return true;
}

__global__ void __launch_bounds__(kB128Threads, 1)
moe_experts_kernel(const __grid_constant__ CUtensorMap tm_w1, const __grid_constant__ CUtensorMap tm_w2, const MoeParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t smem_base = smem_u32(smem);
    uint8_t* plan_gen = smem + kMoeStages * kMoeStageBytes;
    uint32_t* s_route = reinterpret_cast<uint32_t*>(plan_gen);                       // sorted by expert: token << 16 | route
    uint2* s_block = reinterpret_cast<uint2*>(plan_gen + kMoeMaxRoutes * 4);         // blocks of routes: expert | rows << 16, first place
    float* s_max = reinterpret_cast<float*>(plan_gen + kMoePlanBytes);               // [2 halves][128 rows]
    uint8_t* tail = plan_gen + kMoePlanBytes + 1024;
    const uint32_t bars = smem_u32(tail);
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (kMoeStages + s); };
    auto tfull_bar = [&](int a) { return bars + 8u * (2 * kMoeStages + a); };
    auto tempty_bar = [&](int a) { return bars + 8u * (2 * kMoeStages + 2 + a); };
    auto cfull_bar = [&](int c) { return bars + 8u * (2 * kMoeStages + 4 + c); };
    auto cempty_bar = [&](int c) { return bars + 8u * (2 * kMoeStages + 4 + kMoeClaims + c); };
    const uint32_t esync_bar = bars + 8u * (2 * kMoeStages + 4 + 2 * kMoeClaims);
    constexpr int kTail = 8 * (2 * kMoeStages + 5 + 2 * kMoeClaims);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + kTail);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + kTail + 8);
    volatile int* s_claim = reinterpret_cast<volatile int*>(tail + kTail + 16);      // [kMoeClaims]
    volatile int* s_last = s_claim + kMoeClaims;
    int* s_blocks = reinterpret_cast<int*>(tail + kTail + 16) + kMoeClaims + 1;
    static_assert(kTail + 16 + 4 * (kMoeClaims + 2) <= 512, "barriers");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kMoeStages; ++s) { mbar_init(full_bar(s), 3); mbar_init(empty_bar(s), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(tfull_bar(a), 1); mbar_init(tempty_bar(a), 8); }
        for (int c = 0; c < kMoeClaims; ++c) { mbar_init(cfull_bar(c), 1); mbar_init(cempty_bar(c), 11); }
        mbar_init(esync_bar, 8);
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tensormap(&tm_w1);
        prefetch_tensormap(&tm_w2);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    }
    pdl_wait();                                          // routes, cast x and zeroed counters of the first launch

    // ---- the plan, by every CTA for itself: routes sorted by expert (stable), blocks of up to 128 routes
    const int routes = p.tokens * p.topk;
    {
        int* s_off = reinterpret_cast<int*>(smem);                   // the operand ring is not in use yet
        uint16_t* s_id = reinterpret_cast<uint16_t*>(smem + (MM_MAX_EXPERTS + 32) * 4);
        for (int e = threadIdx.x; e < p.experts; e += blockDim.x) s_off[e] = 0;
        __syncthreads();
        for (int r = threadIdx.x; r < routes; r += blockDim.x) {
            const int e = p.route_expert[r];
            s_id[r] = static_cast<uint16_t>(e < 0 ? 0xffff : e);
            if (e >= 0) atomicAdd(&s_off[e], 1);
        }
        __syncthreads();
        if (warp == 0) {
            int off = 0, blocks = 0;
            for (int e0 = 0; e0 < p.experts; e0 += 32) {             // counts -> first places, and the blocks of each expert
                const int e = e0 + lane;
                const int n = e < p.experts ? s_off[e] : 0;
                const int b = (n + 127) >> 7;
                int n_scan = n, b_scan = b;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int a = __shfl_up_sync(0xffffffffu, n_scan, o), c = __shfl_up_sync(0xffffffffu, b_scan, o);
                    if (lane >= o) { n_scan += a; b_scan += c; }
                }
                const int first = off + n_scan - n;
                for (int i = 0; i < b; ++i)
                    s_block[blocks + b_scan - b + i] = make_uint2(static_cast<uint32_t>(e) | static_cast<uint32_t>(min(128, n - 128 * i)) << 16, first + 128 * i);
                if (e < p.experts) s_off[e] = first;
                off += __shfl_sync(0xffffffffu, n_scan, 31);
                blocks += __shfl_sync(0xffffffffu, b_scan, 31);
            }
            if (lane == 0) *s_blocks = blocks;
            __syncwarp();
            for (int r0 = 0; r0 < routes; r0 += 32) {                // place every route, 32 at a time
                const int r = r0 + lane;
                const uint32_t e = r < routes ? s_id[r] : 0xffffu;
                const uint32_t same = __match_any_sync(0xffffffffu, e);
                if (e != 0xffffu) {
                    const int at = s_off[e] + __popc(same & ((1u << lane) - 1u));
                    s_route[at] = static_cast<uint32_t>(r / p.topk) << 16 | static_cast<uint32_t>(r);
                }
                __syncwarp();
                if (e != 0xffffu && (same >> lane) == 1u) s_off[e] += __popc(same);      // the group's last lane
                __syncwarp();
            }
        }
        fence_proxy_async_smem();                                    // these words become TMA destinations
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    const int n_blocks = *s_blocks;                                  // blocks of routes
    const int kb1 = p.hidden / 128, kb2 = p.inter / 128;
    const int nt1 = p.inter / 128, nt2 = (p.hidden + 255) / 256;
    const MoeList list1 = moe_list(n_blocks * nt1, kb1, gridDim.x), list2 = moe_list(n_blocks * nt2, kb2, gridDim.x);
    const int chunks1 = list1.chunks, chunks = n_blocks == 0 ? 0 : chunks1 + list2.chunks;

    // The chunk of claim number i of this CTA, as its consumers read it (a warp at a time; -1 = no more)
    struct Claims { int slot = 0; uint32_t phase = 0; };
    auto next_claim = [&](Claims& c, bool one_thread) {
        int id = -1;
        if (!mbar_wait(cfull_bar(c.slot), c.phase, abort_flag, p.timeout_ns)) return -1;
        id = s_claim[c.slot];
        if (!one_thread) __syncwarp();
        if (one_thread || lane == 0) mbar_arrive(cempty_bar(c.slot));
        if (++c.slot == kMoeClaims) { c.slot = 0; c.phase ^= 1u; }
        return id;
    };
    // tile number -> (block of routes, output tile): the first product block by block, the second output tile by output tile
    auto split_tile = [&](int kind, int tile, int& rb, int& nt) {
        if (kind == 0) { rb = tile / nt1; nt = tile - rb * nt1; }
        else { nt = tile / n_blocks; rb = tile - nt * n_blocks; }
    };

    if (warp < 4) {
        regs_dec<88>();
        if (warp == 0) {
            // ------------------------------------------------------------------ claims and weights
            if (lane == 0) {
                int stage = 0; uint32_t phase = 0;
                int slot = 0; uint32_t cphase = 0;
                int id = chunks > 0 ? atomicAdd(p.counters, 1) : 0;
                bool alive = true;
                while (alive) {
                    if (!mbar_wait(cempty_bar(slot), cphase ^ 1u, abort_flag, p.timeout_ns)) break;
                    const int chunk = id < chunks ? id : -1;
                    s_claim[slot] = chunk;
                    mbar_arrive(cfull_bar(slot));
                    if (++slot == kMoeClaims) { slot = 0; cphase ^= 1u; }
                    if (chunk < 0) break;
                    id = atomicAdd(p.counters, 1);                   // the next one, wanted only after this one's copies
                    const int kind = chunk >= chunks1 ? 1 : 0;
                    const MoeList& l = kind ? list2 : list1;
                    const int c = chunk - (kind ? chunks1 : 0);
                    const CUtensorMap* map = kind ? &tm_w2 : &tm_w1;
                    int u = l.start(c);
                    const int end = l.start(c + 1);
                    while (u < end && alive) {
                        const int tile = u / l.kb, k0 = u - tile * l.kb, k1 = min(l.kb, k0 + end - u);
                        int rb, nt;
                        split_tile(kind, tile, rb, nt);
                        const int e = s_block[rb].x & 0xffff;
                        const int64_t tiled0 = (static_cast<int64_t>(e) * (kind ? nt2 : nt1) + nt) * l.kb;
                        const int row_a = kind ? e * p.hidden + nt * 256 : e * 2 * p.inter + nt * 128;
                        const int row_b = kind ? row_a + 128 : row_a + p.inter;
                        for (int k = k0; k < k1; ++k) {
                            if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.timeout_ns)) { alive = false; break; }
                            const uint32_t dst = smem_base + stage * kMoeStageBytes + kMoeABytes;
                            mbar_arrive_expect_tx(full_bar(stage), 256 * 128);
                            if (p.tiled) {
                                tma_load_2d(dst, map, 0, static_cast<int32_t>((tiled0 + k) * 256), full_bar(stage));
                            } else {
                                tma_load_2d(dst, map, k * 128, row_a, full_bar(stage));
                                tma_load_2d(dst + 128 * 128, map, k * 128, row_b, full_bar(stage));
                            }
                            if (++stage == kMoeStages) { stage = 0; phase ^= 1u; }
                        }
                        u += k1 - k0;
                    }
                }
            }
        } else if (warp == 1) {
            // ------------------------------------------------------------------ MMA
            if (lane == 0) {
                constexpr uint32_t idesc = umma_idesc_f8(128, 256);
                int stage = 0; uint32_t phase = 0;
                int acc = 0; uint32_t acc_phase = 0;
                Claims claims;
                bool alive = true;
                while (alive) {
                    const int chunk = next_claim(claims, true);
                    if (chunk < 0) break;
                    const int units = chunk >= chunks1 ? list2.start(chunk - chunks1 + 1) - list2.start(chunk - chunks1) : list1.start(chunk + 1) - list1.start(chunk);
                    for (int u = 0; u < units; ++u) {
                        if (!mbar_wait(tempty_bar(acc), acc_phase ^ 1u, abort_flag, p.timeout_ns)) { alive = false; break; }
                        if (!mbar_wait(full_bar(stage), phase, abort_flag, p.timeout_ns)) { alive = false; break; }
                        tc_fence_after();
                        const uint64_t da = umma_desc_k_sw128(smem_base + stage * kMoeStageBytes);
                        const uint64_t db = umma_desc_k_sw128(smem_base + stage * kMoeStageBytes + kMoeABytes);
#pragma unroll
                        for (int k = 0; k < 4; ++k) umma_f8(tmem_base + acc * 256, da + 2u * k, db + 2u * k, idesc, k != 0 ? 1u : 0u);
                        umma_commit(empty_bar(stage));
                        umma_commit(tfull_bar(acc));
                        if (++stage == kMoeStages) { stage = 0; phase ^= 1u; }
                        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
                    }
                }
            }
        } else {
            // ------------------------------------------------------------------ token operand: rows gathered by route, 16 bytes a lane
            constexpr int kAhead = 2;                                // copies in flight before the oldest is handed over
            int stage = 0; uint32_t phase = 0;                       // next stage to fill
            int hand = 0, pending = 0;                               // next stage to hand over, stages filled but not handed over
            const int l64 = threadIdx.x - 64;
            const int piece = l64 & 7;
            Claims claims;
            bool alive = true;
            auto hand_over = [&]() {
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(full_bar(hand));
                if (++hand == kMoeStages) hand = 0;
                --pending;
            };
            auto drain = [&]() {
                cp_async_wait<0>();
                while (pending > 0) hand_over();
            };
            while (alive) {
                if (!mbar_try_wait(cfull_bar(claims.slot), claims.phase)) drain();       // no chunk to go on with yet
                const int chunk = next_claim(claims, false);
                if (chunk < 0) break;
                const int kind = chunk >= chunks1 ? 1 : 0;
                const MoeList& l = kind ? list2 : list1;
                const int c = chunk - (kind ? chunks1 : 0);
                const int pitch = kind ? p.inter : p.hidden;
                const uint8_t* src = kind ? p.act_q : p.xq;
                int u = l.start(c);
                const int end = l.start(c + 1);
                while (u < end && alive) {
                    const int tile = u / l.kb, k0 = u - tile * l.kb, k1 = min(l.kb, k0 + end - u);
                    int rb, nt;
                    split_tile(kind, tile, rb, nt);
                    const uint2 blk = s_block[rb];
                    const int rows = blk.x >> 16, first = blk.y;
                    if (kind) {
                        // the rows this product reads: everything filled so far is handed over first, because the tiles that finish
                        // them may be this CTA's own
                        bool ready = false;
                        if (lane == 0) ready = ld_acquire_gpu(p.counters + p.ctr_done1 + rb) >= nt1;
                        ready = __shfl_sync(0xffffffffu, ready, 0);
                        if (!ready) {
                            drain();
                            if (lane == 0) ready = moe_wait_count(p.counters + p.ctr_done1 + rb, nt1, abort_flag, p.timeout_ns);
                            ready = __shfl_sync(0xffffffffu, ready, 0);
                            if (!ready) { alive = false; break; }
                        }
                        __syncwarp();                                // what lane 0 has acquired, the others may read
                    }
                    for (int k = k0; k < k1; ++k) {
                        if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.timeout_ns)) { alive = false; break; }
                        const uint32_t dst = smem_base + stage * kMoeStageBytes;
                        for (int r = l64 >> 3; r < rows; r += 8) {
                            const int row = kind ? first + r : static_cast<int>(s_route[first + r] >> 16);
                            cp_async_16(dst + r * 128 + ((piece ^ (r & 7)) << 4), src + static_cast<int64_t>(row) * pitch + k * 128 + piece * 16);
                        }
                        cp_async_commit();
                        ++pending;
                        if (++stage == kMoeStages) { stage = 0; phase ^= 1u; }
                        if (pending > kAhead) {
                            cp_async_wait<kAhead>();
                            hand_over();
                        }
                    }
                    u += k1 - k0;
                }
            }
            drain();
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------------------- epilogue
        regs_inc<208>();
        const int q = warp & 3, half = (warp - 4) >> 2;
        const int et = q * 32 + lane;
        const bool boss = threadIdx.x == 128;
        const bool do_clamp = p.clamp < 3.0e38f;
        int acc = 0; uint32_t acc_phase = 0;
        uint32_t sync_phase = 0;
        Claims claims;
        bool alive = true;
        // barrier of the eight epilogue warps, bounded like every other wait: a warp that has given up does not hold the others
        auto epi_sync = [&]() {
            __syncwarp();
            if (lane == 0) mbar_arrive(esync_bar);
            if (!mbar_wait(esync_bar, sync_phase, abort_flag, p.timeout_ns)) alive = false;
            sync_phase ^= 1u;
            return alive;
        };
        if (n_blocks == 0) {                                         // no route at all: the sum is empty
            for (int64_t i = static_cast<int64_t>(blockIdx.x) * kB128EpiThreads + threadIdx.x - 128; i < static_cast<int64_t>(p.tokens) * p.hidden / 8;
                 i += static_cast<int64_t>(gridDim.x) * kB128EpiThreads)
                reinterpret_cast<uint4*>(p.y)[i] = make_uint4(0, 0, 0, 0);
        }
        while (alive) {
            const int chunk = next_claim(claims, false);
            if (chunk < 0) break;
            const int kind = chunk >= chunks1 ? 1 : 0;
            const MoeList& l = kind ? list2 : list1;
            const int c = chunk - (kind ? chunks1 : 0);
            int u = l.start(c);
            const int end = l.start(c + 1);
            while (u < end && alive) {
                const int tile = u / l.kb, k0 = u - tile * l.kb, k1 = min(l.kb, k0 + end - u);
                u += k1 - k0;
                int rb, nt;
                split_tile(kind, tile, rb, nt);
                const uint2 blk = s_block[rb];
                const int e = blk.x & 0xffff, rows = blk.x >> 16, place = static_cast<int>(blk.y) + et;
                const bool row_ok = et < rows, warp_ok = q * 32 < rows;
                const uint32_t route = row_ok ? s_route[place] : 0u;
                if (kind && warp_ok) {                               // scales of the activations: written by other CTAs
                    bool ready = true;
                    if (lane == 0) ready = moe_wait_count(p.counters + p.ctr_done1 + rb, nt1, abort_flag, p.timeout_ns);
                    if (!__shfl_sync(0xffffffffu, ready, 0)) { alive = false; break; }
                    __syncwarp();
                }
                const float* sa = kind ? p.act_sf + static_cast<int64_t>(row_ok ? place : 0) * kb2 : p.xsf + static_cast<int64_t>(route >> 16) * kb1;
                // column parts A and B of this thread: gate and up, or two neighbouring runs of 64 outputs
                const int col_a = kind ? half * 128 : half * 64, col_b = kind ? col_a + 64 : col_a + 128;
                const float* sb_a;
                const float* sb_b;
                if (kind) {
                    sb_a = p.s2 + (static_cast<int64_t>(e) * (p.hidden / 128) + min(2 * nt + half, p.hidden / 128 - 1)) * kb2;
                    sb_b = sb_a;
                } else {
                    sb_a = p.s1 + (static_cast<int64_t>(e) * 2 * nt1 + nt) * kb1;
                    sb_b = sb_a + static_cast<int64_t>(nt1) * kb1;
                }
                uint64_t sum[64];
#pragma unroll
                for (int j = 0; j < 64; ++j) sum[j] = 0ull;
                float lane_a = 0.0f, lane_b = 0.0f, s_next = 0.0f;       // weight scales of 32 k blocks, one a lane
                if (warp_ok) s_next = kind ? __ldcg(sa + k0) : sa[k0];
                for (int k = k0; k < k1; ++k) {
                    const int i = (k - k0) & 31;
                    if (i == 0 && warp_ok && k + lane < k1) { lane_a = sb_a[k + lane]; lane_b = sb_b[k + lane]; }
                    const float s_row = s_next;
                    if (warp_ok && k + 1 < k1) s_next = kind ? __ldcg(sa + k + 1) : sa[k + 1];
                    const float w_a = __shfl_sync(0xffffffffu, lane_a, i), w_b = __shfl_sync(0xffffffffu, lane_b, i);
                    if (!mbar_wait(tfull_bar(acc), acc_phase, abort_flag, p.timeout_ns)) { alive = false; break; }
                    tc_fence_after();
                    if (warp_ok) {
                        const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * 256;
                        moe_promote64<false>(sum, t_addr + col_a, s_row * w_a, 0, lane);
                        moe_promote64<true>(sum + 32, t_addr + col_b, s_row * w_b, tempty_bar(acc), lane);
                    } else {
                        __syncwarp();
                        if (lane == 0) mbar_arrive(tempty_bar(acc));
                    }
                    if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
                }
                if (!alive) break;
                if (k1 - k0 < l.kb) {
                    // a part of the tile: written down, and added up by whoever brings the last one, in the order of the chunks
                    const int64_t part_size = static_cast<int64_t>(p.part_rows) * 256;
                    auto part_of = [&](int ch) {      // a chunk holds two parts at most: one that its beginning cuts off, one its end
                        const int which = l.start(ch) > tile * l.kb ? 0 : 1;
                        return p.parts + ((static_cast<int64_t>(kind) * gridDim.x + ch) * 2 + which) * part_size + static_cast<int64_t>(et) * 256 + half * 128;
                    };
                    if (row_ok) {
                        float* o = part_of(c);
#pragma unroll
                        for (int j = 0; j < 64; j += 4) {
                            uint32_t v[8];
#pragma unroll
                            for (int i = 0; i < 4; ++i) { float a, b; unpack_f32x2(sum[j + i], a, b); v[2 * i] = __float_as_uint(a); v[2 * i + 1] = __float_as_uint(b); }
                            st_global_32b(o + 2 * j, v);
                        }
                    }
                    __threadfence();
                    if (!epi_sync()) break;
                    if (boss) *s_last = atomicAdd(p.counters + (kind ? p.ctr_tile2 : p.ctr_tile1) + tile, k1 - k0) + (k1 - k0) == l.kb;
                    if (!epi_sync()) break;
                    if (*s_last == 0) continue;
                    __threadfence();
                    if (row_ok) {
                        const int c0 = l.chunk_of(tile * l.kb), c1 = l.chunk_of(tile * l.kb + l.kb - 1);
#pragma unroll
                        for (int j0 = 0; j0 < 64; j0 += 16) {
                            float t[32];
#pragma unroll
                            for (int j = 0; j < 32; ++j) t[j] = 0.0f;
                            for (int ch = c0; ch <= c1; ++ch) {
                                const float4* in = reinterpret_cast<const float4*>(part_of(ch) + 2 * j0);
#pragma unroll
                                for (int j = 0; j < 8; ++j) {
                                    const float4 f = __ldcg(in + j);
                                    t[4 * j] += f.x; t[4 * j + 1] += f.y; t[4 * j + 2] += f.z; t[4 * j + 3] += f.w;
                                }
                            }
#pragma unroll
                            for (int j = 0; j < 16; ++j) sum[j0 + j] = pack_f32x2(__float_as_uint(t[2 * j]), __float_as_uint(t[2 * j + 1]));
                        }
                    }
                }
                if (kind == 0) {
                    // silu(gate) * up, and the cast: this thread has half of the block of 128, its partner in the other half the rest
                    uint32_t top_bits = 0;
                    if (row_ok) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            float g[2], v[2];
                            unpack_f32x2(sum[j], g[0], g[1]);
                            unpack_f32x2(sum[32 + j], v[0], v[1]);
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                if (do_clamp) {                      // NaN stays NaN
                                    g[i] = g[i] < -p.clamp ? -p.clamp : (g[i] > p.clamp ? p.clamp : g[i]);
                                    v[i] = v[i] < -p.clamp ? -p.clamp : (v[i] > p.clamp ? p.clamp : v[i]);
                                }
                                v[i] *= silu_f(g[i]);
                                top_bits = max(top_bits, abs_bits(v[i]));
                            }
                            sum[j] = pack_f32x2(__float_as_uint(v[0]), __float_as_uint(v[1]));
                        }
                        s_max[half * 128 + et] = __uint_as_float(top_bits);
                    }
                    if (!epi_sync()) break;
                    if (row_ok) {
                        top_bits = max(top_bits, __float_as_uint(s_max[(half ^ 1) * 128 + et]));
                        const float top = group_top(top_bits);
                        const GroupQuotient quot(top);
                        uint4* o = reinterpret_cast<uint4*>(p.act_q + static_cast<int64_t>(place) * p.inter + nt * 128 + half * 64);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t w[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float a, b, d, f;
                                unpack_f32x2(sum[j * 8 + 2 * i], a, b);
                                unpack_f32x2(sum[j * 8 + 2 * i + 1], d, f);
                                w[i] = pack4_e4m3(quot(a), quot(b), quot(d), quot(f));
                            }
                            o[j] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                        if (half == 0) p.act_sf[static_cast<int64_t>(place) * kb2 + nt] = __fdiv_rn(top, 448.0f);
                    }
                    __threadfence();
                    if (!epi_sync()) break;
                    if (boss) red_release_gpu_add(p.counters + p.ctr_done1 + rb, 1);
                } else {
                    const int col0 = nt * 256 + half * 128;
                    if (row_ok && col0 < p.hidden) {
                        const int r = static_cast<int>(route & 0xffffu);
                        const float w = p.route_w[r];
                        float* o = p.rows_out + static_cast<int64_t>(r) * p.hidden + col0;
#pragma unroll
                        for (int j = 0; j < 64; j += 4) {
                            uint32_t v[8];
#pragma unroll
                            for (int i = 0; i < 4; ++i) { float a, b; unpack_f32x2(sum[j + i], a, b); v[2 * i] = __float_as_uint(a * w); v[2 * i + 1] = __float_as_uint(b * w); }
                            st_global_32b(o + 2 * j, v);
                        }
                    }
                    __threadfence();
                    if (!epi_sync()) break;
                    if (boss) *s_last = atomicAdd(p.counters + p.ctr_done2 + nt, 1) == n_blocks - 1;
                    if (!epi_sync()) break;
                    if (*s_last != 0) {
                        // every expert's rows of these 256 outputs are there: add each token's up, in the order of its slots
                        __threadfence();
                        const int cols4 = min(256, p.hidden - nt * 256) / 4;
                        for (int i = threadIdx.x - 128; i < p.tokens * cols4; i += kB128EpiThreads) {
                            const int t = i / cols4, col = nt * 256 + (i - t * cols4) * 4;
                            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
                            for (int s = 0; s < p.topk; ++s) {
                                const int r = t * p.topk + s;
                                if (p.route_expert[r] < 0) continue;
                                const float4 f = __ldcg(reinterpret_cast<const float4*>(p.rows_out + static_cast<int64_t>(r) * p.hidden + col));
                                a.x += f.x; a.y += f.y; a.z += f.z; a.w += f.w;
                            }
                            *reinterpret_cast<uint2*>(p.y + static_cast<int64_t>(t) * p.hidden + col) = make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
                        }
                    }
                }
            }
        }
    }

    if (*abort_flag != 0) {
        // a bounded wait expired: give copies that may still be in flight time to land, then report
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 1000000ull) __nanosleep(1000);
        if (threadIdx.x == 0 && atomicCAS(p.status, 0, MM_ERR_PIPE_TIMEOUT) == 0) {
            p.status[1] = 30; p.status[2] = blockIdx.x; p.status[3] = chunks; p.status[4] = 0;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

}  // namespace mm
