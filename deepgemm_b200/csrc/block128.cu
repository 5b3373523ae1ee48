// extern "C" entry points of the block-scaled FP8 operators (declared in include/megamoe_b200.h).
#include <cuda.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <atomic>
#include <mutex>

#include "../../include/megamoe_b200.h"
#include "block128.cuh"
#include "block128_gemm.cuh"
#include "block128_moe.cuh"
#include "layout.h"

// abi.cu: error message, launch counter and wait limit of the library
void mm_detail_set_error(const char* msg);
void mm_detail_count_launch();
uint64_t mm_detail_pipe_timeout_ns();

// First failed wait or bad layout of any of these operators on a device since it was last read (b128_report); written by kernels only then.
// Behind its eight words, eight for each read that may be under way: what it took.
constexpr int kStatusReads = 64;
__device__ int g_b128_status[8 + 8 * kStatusReads];

namespace {

int fail(int code, const char* fmt, ...) {
    char msg[384];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof(msg), fmt, ap);
    va_end(ap);
    mm_detail_set_error(msg);
    return code;
}

#define B_CUDA(expr)                                                                                            \
    do {                                                                                                        \
        cudaError_t _e = (expr);                                                                                \
        if (_e != cudaSuccess) return fail(100 + (int)_e, "%s failed: %s", #expr, cudaGetErrorString(_e));      \
    } while (0)
#define B_REQUIRE(cond, ...)                      \
    do {                                          \
        if (!(cond)) return fail(1, __VA_ARGS__); \
    } while (0)
#define B_LAUNCHED()                  \
    do {                              \
        mm_detail_count_launch();     \
        B_CUDA(cudaGetLastError());   \
    } while (0)

// mm_block128_test_waits
std::atomic<int> g_given_up{-1};
std::atomic<int64_t> g_limit_ns{0};
uint64_t wait_limit_ns() {
    const int64_t test = g_limit_ns.load();
    return test > 0 ? (uint64_t)test : mm_detail_pipe_timeout_ns();
}

constexpr int kMaxDevices = 64;
constexpr int64_t kMaxDim = (int64_t)1 << 31;

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// What a launch needs to know about the current device, looked up once per device.
struct Device {
    bool ready = false;
    int sms = 0;
    int clusters[4] = {0, 0, 0, 0};      // of 1, 2, 4 and 8 CTAs of the split product that are resident at once
    int* status = nullptr;
};

// A launch that may begin while the kernel before it in the stream drains (pdl_wait): 0.2 to 0.5 us less for each of a chain of small
// kernels, 1 us for a cast of 24576 x 2048, none for large products.
struct Launch {
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attrs[2];
    Launch(int64_t grid, int threads, size_t smem, cudaStream_t st, int cluster = 1) {
        memset(this, 0, sizeof(*this));
        cfg.gridDim = dim3((unsigned)grid);
        cfg.blockDim = dim3((unsigned)threads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attrs[0].val.programmaticStreamSerializationAllowed = 1;
        attrs[1].id = cudaLaunchAttributeClusterDimension;
        attrs[1].val.clusterDim.x = (unsigned)cluster; attrs[1].val.clusterDim.y = 1; attrs[1].val.clusterDim.z = 1;
        cfg.attrs = attrs;
        cfg.numAttrs = cluster > 1 ? 2 : 1;
    }
    Launch(const Launch&) = delete;
    template <typename... P, typename... A> cudaError_t operator()(void (*kernel)(P...), A... args) const {
        return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    }
};
Launch split_launch(int64_t tiles, int split, cudaStream_t st) { return Launch(tiles * split, mm::kB128Threads, mm::B128Shape<128>::kSmemBytes, st, split); }

int device_of(Device** out) {
    static Device devices[kMaxDevices];
    static std::mutex mu;
    int dev = 0;
    B_CUDA(cudaGetDevice(&dev));
    B_REQUIRE(dev < kMaxDevices, "device number above %d", kMaxDevices - 1);
    Device& d = devices[dev];
    std::lock_guard<std::mutex> lk(mu);
    if (!d.ready) {
        B_CUDA(cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev));
        void* p = nullptr;
        B_CUDA(cudaGetSymbolAddress(&p, g_b128_status));
        d.status = static_cast<int*>(p);
        B_CUDA(cudaFuncSetAttribute(mm::block128_gemm_kernel<256, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, mm::B128Shape<256>::kSmemBytes));
        B_CUDA(cudaFuncSetAttribute(mm::block128_gemm_kernel<128, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, mm::B128Shape<128>::kSmemBytes));
        B_CUDA(cudaFuncSetAttribute(mm::block128_gemm_kernel<128, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, mm::B128Shape<128>::kSmemBytes));
        B_CUDA(cudaFuncSetAttribute(mm::moe_experts_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, mm::kMoeSmemBytes));
#define B_STAGED(V, R) B_CUDA(cudaFuncSetAttribute(mm::norm_gate_residual_kernel<V, mm::B128_BF16, R, mm::B128_FP32, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * mm::kNormMaxHidden))
        B_STAGED(1, mm::B128_BF16);
        B_STAGED(1, mm::B128_FP32);
        B_STAGED(2, mm::B128_BF16);
        B_STAGED(2, mm::B128_FP32);
#undef B_STAGED
        d.clusters[0] = d.sms;
        for (int i = 1; i < 4; ++i) {
            const Launch launch = split_launch(d.sms, 1 << i, nullptr);
            B_CUDA(cudaOccupancyMaxActiveClusters(&d.clusters[i], mm::block128_gemm_kernel<128, true>, &launch.cfg));
        }
        d.ready = true;
    }
    *out = &d;
    return 0;
}

int encode_fn(EncodeFn* out) {
    static EncodeFn fn = nullptr;
    static std::mutex mu;
    std::lock_guard<std::mutex> lk(mu);
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult qres;
        B_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qres));
        B_REQUIRE(p != nullptr && qres == cudaDriverEntryPointSuccess, "cuTensorMapEncodeTiled is not available in this driver");
        fn = reinterpret_cast<EncodeFn>(p);
    }
    *out = fn;
    return 0;
}

// byte tensor [d2][rows][inner] (d2 = 0: two dimensions), boxes of box_rows x 128 bytes, 128-byte swizzle, zero outside
int byte_map(const void* ptr, uint64_t inner, uint64_t rows, uint64_t row_stride, uint64_t d2, uint64_t d2_stride, uint32_t box_rows, CUtensorMap* out) {
    EncodeFn enc;
    if (int rc = encode_fn(&enc)) return rc;
    cuuint64_t dims[3] = {inner, rows, d2};
    cuuint64_t strides[2] = {row_stride, d2_stride};
    cuuint32_t box[3] = {128, box_rows, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, d2 ? 3 : 2, const_cast<void*>(ptr), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    B_REQUIRE(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    return 0;
}

// Work memory of mm_moe_few_tokens, in bytes from its start
struct MoeWork {
    int64_t counters, route_expert, route_w, xq, xsf, act_q, act_sf, rows_out, parts, total;
    int num_counters, ctr_done1, ctr_tile1, part_rows, act_sf_pitch;
};

MoeWork moe_work(int T, int E, int K, int H, int I, int ctas) {
    MoeWork w;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t o = at; at = (at + bytes + 255) / 256 * 256; return o; };
    const int64_t routes = (int64_t)T * K;
    const int64_t blocks = (routes < E ? routes : E) + routes / 128;
    const int64_t nt1 = I / 128;
    w.ctr_done1 = 32;
    w.ctr_tile1 = w.ctr_done1 + (int)blocks;
    w.num_counters = w.ctr_tile1 + (int)(blocks * nt1 * 4);
    w.part_rows = (int)(routes < 128 ? routes : 128);
    w.counters = take((int64_t)w.num_counters * 4);
    w.route_expert = take(routes * 4);
    w.route_w = take(routes * 4);
    w.xq = take((int64_t)T * H);
    w.xsf = take((int64_t)T * (H / 128) * 4);
    w.act_q = take(routes * I);
    w.act_sf_pitch = (I / 128 + 31) / 32 * 32;
    w.act_sf = take(routes * w.act_sf_pitch * 4);
    w.rows_out = take(routes * H * 4);
    w.parts = take((int64_t)6 * ctas * w.part_rows * 256 * 4);
    w.total = at;
    return w;
}

int moe_check_shape(int T, int E, int K, int H, int I) {
    B_REQUIRE(T >= 0 && E > 0 && E <= MM_MAX_EXPERTS && K > 0 && K <= MM_MAX_TOPK && K <= E, "mm_moe_few_tokens: need 0 < topk <= min(experts, %d), experts <= %d",
              MM_MAX_TOPK, MM_MAX_EXPERTS);
    B_REQUIRE(H > 0 && I > 0 && H % 128 == 0 && I % 128 == 0 && H <= 32768 && I <= 32768, "mm_moe_few_tokens: hidden sizes must be multiples of 128, at most 32768");
    B_REQUIRE((int64_t)T * K <= mm::kMoeMaxRoutes, "mm_moe_few_tokens: at most %d routes (tokens x topk)", mm::kMoeMaxRoutes);
    return 0;
}

// rows that are read 16 bytes at a time
bool row_aligned(int64_t stride, int type) { return stride % (type == mm::B128_FP32 ? 4 : 8) == 0; }
bool known_type(int t) { return t == mm::B128_BF16 || t == mm::B128_FP16 || t == mm::B128_FP32; }

}  // namespace

extern "C" {

int mm_cast_block128(const void* x, int type, int64_t rows, int k, int64_t row_stride, void* q, float* sf, void* stream_) {
    B_REQUIRE(known_type(type), "mm_cast_block128: unknown type");
    B_REQUIRE(rows >= 0 && k > 0 && k % 8 == 0 && row_stride >= k && row_aligned(row_stride, type), "mm_cast_block128: k must come in multiples of 8, the row stride in multiples of 16 bytes");
    if (rows == 0) return 0;
    B_REQUIRE(x && q && sf, "mm_cast_block128: null pointer");
    B_REQUIRE(aligned(x, 16) && aligned(q, 8) && aligned(sf, 4), "mm_cast_block128: x must be 16-byte, q 8-byte aligned");
    const int64_t per_row = (k + 127) / 128, groups = rows * per_row;
    B_REQUIRE(rows < kMaxDim && groups < kMaxDim, "mm_cast_block128: too many groups");
    Device* d;
    if (int rc = device_of(&d)) return rc;
    const int64_t blocks = (groups + 16 * mm::kCastGroups - 1) / (16 * mm::kCastGroups);
    cudaStream_t st = static_cast<cudaStream_t>(stream_);
    uint8_t* o = static_cast<uint8_t*>(q);
    const bool flat = k % 128 == 0 && row_stride == k;
    const Launch launch(blocks, 256, 0, st);
#define B_CAST(T) B_CUDA(launch(flat ? mm::cast_block128_kernel<T, true> : mm::cast_block128_kernel<T, false>, x, row_stride, groups, per_row, k, o, sf))
    if (type == mm::B128_BF16) B_CAST(mm::B128_BF16);
    else if (type == mm::B128_FP16) B_CAST(mm::B128_FP16);
    else B_CAST(mm::B128_FP32);
#undef B_CAST
    B_LAUNCHED();
    return 0;
}

int mm_cast_weight_block128(const void* w, int type, int experts, int rows, int k, void* q, float* sf, void* stream_) {
    B_REQUIRE(known_type(type), "mm_cast_weight_block128: unknown type");
    B_REQUIRE(experts >= 0 && rows >= 0 && k > 0 && k % 8 == 0, "mm_cast_weight_block128: k must be a positive multiple of 8");
    if (experts == 0 || rows == 0) return 0;
    B_REQUIRE(w && q && sf, "mm_cast_weight_block128: null pointer");
    B_REQUIRE(aligned(w, 16) && aligned(q, 8) && aligned(sf, 4), "mm_cast_weight_block128: w must be 16-byte, q 8-byte aligned");
    const int rb = (rows + 127) / 128, kb = (k + 127) / 128;
    const int64_t blocks = (int64_t)experts * rb * kb;
    B_REQUIRE(blocks < kMaxDim, "mm_cast_weight_block128: too many blocks");
    cudaStream_t st = static_cast<cudaStream_t>(stream_);
    uint8_t* o = static_cast<uint8_t*>(q);
    if (type == mm::B128_BF16) mm::cast_weight_block128_kernel<mm::B128_BF16><<<(unsigned)blocks, 256, 0, st>>>(w, rows, k, rb, kb, o, sf);
    else if (type == mm::B128_FP16) mm::cast_weight_block128_kernel<mm::B128_FP16><<<(unsigned)blocks, 256, 0, st>>>(w, rows, k, rb, kb, o, sf);
    else mm::cast_weight_block128_kernel<mm::B128_FP32><<<(unsigned)blocks, 256, 0, st>>>(w, rows, k, rb, kb, o, sf);
    B_LAUNCHED();
    return 0;
}

int mm_norm_gate_residual(const void* y, int y_type, int64_t y_stride, const void* r, int r_type, int64_t r_stride, const void* post, int post_type,
                          const void* gate, int gate_type, int64_t gate_row_stride, int gate_col_stride, const void* pre, int pre_type,
                          void* r_out, void* x_out, int x_type, void* q, float* sf, int quant, int tokens, int hidden, float alpha, float eps,
                          float offset, void* stream_) {
    B_REQUIRE(tokens >= 0 && hidden > 0 && hidden % 8 == 0 && hidden <= mm::kNormMaxHidden, "mm_norm_gate_residual: hidden must be a multiple of 8, at most 16384");
    B_REQUIRE(quant >= 0 && quant <= 2, "mm_norm_gate_residual: unknown cast");
    B_REQUIRE(known_type(y_type) && known_type(r_type) && known_type(post_type) && known_type(gate_type) && known_type(pre_type) && known_type(x_type),
              "mm_norm_gate_residual: unknown type");
    if (tokens == 0) return 0;
    B_REQUIRE(r && (y ? r_out != nullptr : !post && !gate && !r_out), "mm_norm_gate_residual: null pointer (a norm or gate needs y, y needs a new residual)");
    B_REQUIRE(pre || (!x_out && quant == 0), "mm_norm_gate_residual: outputs of the second norm need its weight");
    B_REQUIRE(quant == 0 || (q && sf), "mm_norm_gate_residual: null pointer");
    B_REQUIRE(r_stride >= hidden && (!y || y_stride >= hidden) && row_aligned(r_stride, r_type) && row_aligned(y_stride, y_type) && (gate_col_stride == 0 || gate_col_stride == 1) &&
              gate_row_stride >= 0 && (gate_col_stride == 0 || row_aligned(gate_row_stride, gate_type)), "mm_norm_gate_residual: bad strides");
    B_REQUIRE(aligned(y, 16) && aligned(r, 16) && aligned(post, 16) && aligned(pre, 16) && (gate_col_stride == 0 || aligned(gate, 16)) && aligned(r_out, 16) &&
              aligned(x_out, 16) && aligned(q, 8) && aligned(sf, 4), "mm_norm_gate_residual: pointers must be 16-byte aligned (codes 8)");
    Device* d;
    if (int rc = device_of(&d)) return rc;
    mm::NormParams p;
    p.y = y; p.r = r; p.post = post; p.pre = pre; p.gate = gate;
    p.r_out = r_out; p.x_out = x_out; p.q = static_cast<uint8_t*>(q); p.sf = sf;
    p.y_type = y_type; p.r_type = r_type; p.w_post_type = post_type; p.w_pre_type = pre_type; p.gate_type = gate_type; p.x_type = x_type;
    p.y_stride = y_stride; p.r_stride = r_stride; p.gate_row_stride = gate_row_stride; p.gate_col_stride = gate_col_stride;
    p.tokens = tokens; p.hidden = hidden; p.quant = quant; p.alpha = alpha; p.eps = eps; p.offset = offset;
    const int vecs = hidden / 8;
    // One vector of 8 values per thread while a row has an SM to itself (one row of 4096: 3.9 us against 4.7) and for an fp32 residual, whose
    // two would not fit the registers (4000 x 4096: 45 us against 56), else two (see the kernel).  64 registers a thread, so 1024 threads
    // are resident on an SM; a block more than those waits a whole turn (74 us instead of 62).
    const bool two = vecs > 1024 || (tokens > 2 * d->sms && r_type != mm::B128_FP32);
    const int threads = ((two ? (vecs + 1) / 2 : vecs) + 31) / 32 * 32;
    int64_t blocks = (int64_t)d->sms * (threads < 1024 ? 1024 / threads : 1);
    if (blocks > tokens) blocks = tokens;
    cudaStream_t st = static_cast<cudaStream_t>(stream_);
    const bool usual = (!y || y_type == mm::B128_BF16) && (!x_out || x_type == mm::B128_BF16) && (!post || post_type == mm::B128_FP32) &&
                       (!pre || pre_type == mm::B128_FP32) && (!gate || gate_type == mm::B128_FP32);
    // Weights in shared memory, already with their offset and a gate that is the same for all rows, where a block does two rows or more
    // (of 4096: 8192 rows 55 us instead of 61, 1200 14.3 instead of 14.8; 700, which make 592 blocks, 9.9 instead of 8.3).
    const bool staged = tokens >= 2 * blocks;
    const bool typed = usual && r_type != mm::B128_FP16;
    const Launch launch(blocks, threads, staged && typed ? 8 * (size_t)hidden : 0, st);
#define B_NORM(V, R)                                                                                                                       \
    B_CUDA(launch(staged ? mm::norm_gate_residual_kernel<V, mm::B128_BF16, R, mm::B128_FP32, true> : mm::norm_gate_residual_kernel<V, mm::B128_BF16, R, mm::B128_FP32, false>, p))
#define B_NORM_TYPES(V)                                                                                                                               \
    do {                                                                                                                                              \
        if (typed && r_type == mm::B128_BF16) B_NORM(V, mm::B128_BF16);                                                                               \
        else if (typed) B_NORM(V, mm::B128_FP32);                                                                                                     \
        else B_CUDA(launch(mm::norm_gate_residual_kernel<V, mm::kAny, mm::kAny, mm::kAny, false>, p));                                                \
    } while (0)
    if (two) B_NORM_TYPES(2);
    else B_NORM_TYPES(1);
#undef B_NORM_TYPES
#undef B_NORM
    B_LAUNCHED();
    return 0;
}

int mm_fp8_gemm_block128(const void* a, int64_t a_stride, const float* sa, int64_t sa_stride, const void* b, const float* sb, int experts,
                         int weights_tiled, const int* m_indices, void* out, int64_t out_stride, int out_fp32, int64_t m64, int n, int k, void* stream_) {
    B_REQUIRE(m64 >= 0 && m64 < kMaxDim - 256 && n >= 0 && k > 0 && k % 16 == 0, "mm_fp8_gemm_block128: k must be a positive multiple of 16");
    B_REQUIRE(experts > 0 && (experts == 1 || m_indices), "mm_fp8_gemm_block128: several experts need m_indices");
    B_REQUIRE(!m_indices || m64 % 128 == 0, "mm_fp8_gemm_block128: grouped rows must be a multiple of 128");
    B_REQUIRE(!weights_tiled || (k % 128 == 0 && n % 128 == 0), "mm_fp8_gemm_block128: tiled weights need n and k to be multiples of 128");
    if (m64 == 0 || n == 0) return 0;
    B_REQUIRE(a && sa && b && sb && out, "mm_fp8_gemm_block128: null pointer");
    B_REQUIRE(aligned(a, 16) && aligned(b, 16) && a_stride % 16 == 0 && a_stride >= k, "mm_fp8_gemm_block128: operands must be 16-byte aligned, rows of a too");
    const int m = (int)m64, kb = (k + 127) / 128, n_sf = (n + 127) / 128;
    B_REQUIRE(sa_stride >= kb && out_stride >= n, "mm_fp8_gemm_block128: bad strides");
    Device* d;
    if (int rc = device_of(&d)) return rc;
    mm::B128GemmParams p;
    memset(&p, 0, sizeof(p));
    p.m = m; p.n = n; p.k_blocks = kb; p.n_sf = n_sf; p.experts = experts;
    p.tiled = weights_tiled ? 1 : 0;
    p.tiled_n_blocks = (n + 255) / 256;
    p.sa = sa; p.sa_stride = sa_stride; p.sb = sb; p.m_indices = m_indices;
    p.out = out; p.out_stride = out_stride; p.out_fp32 = out_fp32 ? 1 : 0;
    const int esz = out_fp32 ? 4 : 2;
    p.out_vec32 = aligned(out, 32) && (out_stride * esz) % 32 == 0;
    p.status = d->status;
    p.timeout_ns = wait_limit_ns();
    p.given_up = g_given_up.load();
    p.m_tiles = (m + 127) / 128;
    p.a_box_rows = m >= 128 ? 128 : (m + 7) / 8 * 8;
    // Tile width and split of K.  A turn of the SMs with tiles of 128 columns takes 0.7 of the time of one with 256 (1024 x 4096 x 4096: 29 us in
    // two turns of 128, 21 in one of 256), so 128 is taken where that makes less.  The k blocks of a tile are then divided among up to
    // eight CTAs, as long as all clusters are resident at once (1 x 4096 x 4096: 8.2 us with four CTAs to a tile, 11.0 with two, 15.0 with
    // one, before the parts were read side by side) and each CTA keeps a few blocks.
    const int64_t tiles256 = (int64_t)p.m_tiles * ((n + 255) / 256), tiles128 = (int64_t)p.m_tiles * n_sf;
    const int64_t turns256 = (tiles256 + d->sms - 1) / d->sms, turns128 = (tiles128 + d->sms - 1) / d->sms;
    const int bn = turns128 * 7 < turns256 * 10 ? 128 : 256;
    const int64_t tiles = bn == 256 ? tiles256 : tiles128;
    B_REQUIRE(tiles < kMaxDim, "mm_fp8_gemm_block128: too many tiles");
    p.n_tiles = bn == 256 ? (n + 255) / 256 : n_sf;
    int log_split = 0;
    while (bn == 128 && !m_indices && (2 << log_split) <= mm::kB128MaxSplit && tiles <= d->clusters[log_split + 1] && kb >= (4 << log_split)) ++log_split;
    const int split = 1 << log_split;
    CUtensorMap tm_a, tm_b;
    if (int rc = byte_map(a, (uint64_t)k, (uint64_t)m, (uint64_t)a_stride, 0, 0, (uint32_t)p.a_box_rows, &tm_a)) return rc;
    if (p.tiled) {
        if (int rc = byte_map(b, 128, (uint64_t)experts * p.tiled_n_blocks * kb * 256, 128, 0, 0, (uint32_t)bn, &tm_b)) return rc;
    } else {
        if (int rc = byte_map(b, (uint64_t)k, (uint64_t)n, (uint64_t)k, (uint64_t)experts, (uint64_t)n * k, (uint32_t)bn, &tm_b)) return rc;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream_);
    if (split > 1) {
        B_CUDA(split_launch(tiles, split, st)(mm::block128_gemm_kernel<128, true>, tm_a, tm_b, p));
    } else {
        const int64_t grid = tiles < d->sms ? tiles : d->sms;
        if (bn == 256) B_CUDA(Launch(grid, mm::kB128Threads, mm::B128Shape<256>::kSmemBytes, st)(mm::block128_gemm_kernel<256, false>, tm_a, tm_b, p));
        else B_CUDA(Launch(grid, mm::kB128Threads, mm::B128Shape<128>::kSmemBytes, st)(mm::block128_gemm_kernel<128, false>, tm_a, tm_b, p));
    }
    B_LAUNCHED();
    return 0;
}

int mm_moe_few_tokens_workspace(int T, int E, int K, int H, int I, int64_t* bytes) {
    B_REQUIRE(bytes, "mm_moe_few_tokens_workspace: null pointer");
    if (int rc = moe_check_shape(T, E, K, H, I)) return rc;
    Device* d;
    if (int rc = device_of(&d)) return rc;
    *bytes = moe_work(T, E, K, H, I, d->sms).total;
    return 0;
}

int mm_moe_few_tokens(const void* x, int x_is_fp8, int64_t x_stride, const float* x_sf, const float* logits, int64_t logits_stride, const void* topk_idx,
                      int idx_i64, const float* topk_w, const void* w1, const float* s1, const void* w2, const float* s2, int tiled, int T, int E, int K,
                      int H, int I, float clamp, void* work, int64_t work_bytes, void* y, void* stream_) {
    if (int rc = moe_check_shape(T, E, K, H, I)) return rc;
    B_REQUIRE(!isnan(clamp) && clamp > 0.0f, "mm_moe_few_tokens: the clamp must be positive (+inf for none)");
    if (T == 0) return 0;
    B_REQUIRE(x && w1 && s1 && w2 && s2 && work && y && (!x_is_fp8 || x_sf), "mm_moe_few_tokens: null pointer");
    B_REQUIRE((logits != nullptr) != (topk_idx != nullptr) && (!topk_idx || topk_w), "mm_moe_few_tokens: either logits or topk_idx with topk_w");
    B_REQUIRE(aligned(x, 16) && aligned(w1, 16) && aligned(w2, 16) && aligned(work, 256) && aligned(y, 16) && x_stride % 16 == 0 && x_stride >= H,
              "mm_moe_few_tokens: x, weights and y must be 16-byte, the work memory 256-byte aligned");
    B_REQUIRE(!x_is_fp8 || x_stride == H, "mm_moe_few_tokens: codes must be contiguous");
    B_REQUIRE(!logits || logits_stride >= E, "mm_moe_few_tokens: bad logits stride");
    Device* d;
    if (int rc = device_of(&d)) return rc;
    const MoeWork w = moe_work(T, E, K, H, I, d->sms);
    B_REQUIRE(work_bytes >= w.total, "mm_moe_few_tokens: needs %lld bytes of work memory, has %lld", (long long)w.total, (long long)work_bytes);
    uint8_t* base = static_cast<uint8_t*>(work);
    mm::MoeParams p;
    memset(&p, 0, sizeof(p));
    p.tokens = T; p.experts = E; p.topk = K; p.hidden = H; p.inter = I;
    p.logits = logits; p.logits_stride = logits_stride;
    p.topk_idx = topk_idx; p.idx_i64 = idx_i64; p.topk_w = topk_w;
    if (x_is_fp8) {
        p.xq = static_cast<const uint8_t*>(x);
        p.xsf = x_sf;
    } else {
        p.x = x; p.x_stride = x_stride;
        p.xq_out = base + w.xq; p.xsf_out = reinterpret_cast<float*>(base + w.xsf);
        p.xq = p.xq_out; p.xsf = p.xsf_out;
    }
    p.route_expert = reinterpret_cast<int*>(base + w.route_expert);
    p.route_w = reinterpret_cast<float*>(base + w.route_w);
    p.counters = reinterpret_cast<int*>(base + w.counters);
    p.num_counters = w.num_counters;
    p.ctr_done1 = w.ctr_done1; p.ctr_tile1 = w.ctr_tile1;
    p.s1 = s1; p.s2 = s2; p.tiled = tiled ? 1 : 0;
    p.act_q = base + w.act_q; p.act_sf = reinterpret_cast<float*>(base + w.act_sf); p.act_sf_pitch = w.act_sf_pitch;
    p.rows_out = reinterpret_cast<float*>(base + w.rows_out);
    p.parts = reinterpret_cast<float*>(base + w.parts); p.part_rows = w.part_rows;
    p.y = static_cast<__nv_bfloat16*>(y);
    p.clamp = clamp;
    p.status = d->status;
    p.timeout_ns = wait_limit_ns();
    CUtensorMap tm1, tm2;
    if (tiled) {
        if (int rc = byte_map(w1, 128, (uint64_t)E * (I / 128) * (H / 128) * 256, 128, 0, 0, 256, &tm1)) return rc;
        if (int rc = byte_map(w2, 128, (uint64_t)E * ((H + 255) / 256) * (I / 128) * 256, 128, 0, 0, 256, &tm2)) return rc;
    } else {
        if (int rc = byte_map(w1, (uint64_t)H, (uint64_t)E * 2 * I, (uint64_t)H, 0, 0, 128, &tm1)) return rc;
        if (int rc = byte_map(w2, (uint64_t)I, (uint64_t)E * H, (uint64_t)I, 0, 0, 128, &tm2)) return rc;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream_);
    B_CUDA(Launch(T, 256, 0, st)(mm::moe_route_kernel, p));
    B_LAUNCHED();
    // starts while the first one runs: its barriers, TMEM and tensor maps need nothing of it
    B_CUDA(Launch(d->sms, mm::kMoeThreads, mm::kMoeSmemBytes, st)(mm::moe_experts_kernel, tm1, tm2, p));
    B_LAUNCHED();
    return 0;
}

int mm_block128_test_waits(int given_up_cta, int64_t limit_ns) {
    B_REQUIRE(given_up_cta >= -1 && limit_ns >= 0, "mm_block128_test_waits: no such CTA or limit");
    g_given_up.store(given_up_cta);
    g_limit_ns.store(limit_ns);
    return 0;
}

int mm_block128_read_status(void* stream_, int32_t* out5) {
    B_REQUIRE(out5, "mm_block128_read_status: null pointer");
    Device* d;
    if (int rc = device_of(&d)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream_);
    // Words of its own for each read, not a lock: what this stream waits for may be the work of a thread that reads its own status first.
    struct Place {
        std::atomic<bool>* at = nullptr;
        int index = 0;
        Place() {
            static std::atomic<bool> taken[kStatusReads];
            for (index = 0; index < kStatusReads; ++index)
                if (!taken[index].exchange(true)) { at = &taken[index]; return; }
        }
        ~Place() { if (at) at->store(false); }
    } place;
    B_REQUIRE(place.at, "mm_block128_read_status: %d reads are under way already", kStatusReads);
    int* taken = d->status + 8 + 8 * place.index;
    mm::b128_take_status_kernel<<<1, 1, 0, st>>>(d->status, taken);
    B_LAUNCHED();
    B_CUDA(cudaMemcpyAsync(out5, taken, 5 * sizeof(int32_t), cudaMemcpyDeviceToHost, st));
    B_CUDA(cudaStreamSynchronize(st));
    return 0;
}

}  // extern "C"
