// extern "C" entry points of the block-scaled FP8 operators (declared in include/megamoe_b200.h).
#include <cuda.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <mutex>

#include "../../include/megamoe_b200.h"
#include "block128.cuh"
#include "block128_gemm.cuh"
#include "layout.h"

// abi.cu: error message, launch counter and wait limit of the library
void mm_detail_set_error(const char* msg);
void mm_detail_count_launch();
uint64_t mm_detail_pipe_timeout_ns();

// First failed wait or bad layout of any of these operators on a device since it was last read; written by kernels only then.
__device__ int g_b128_status[8];

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

constexpr int kMaxDevices = 64;
constexpr int64_t kMaxDim = (int64_t)1 << 31;

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// What a launch needs to know about the current device, looked up once per device.
struct Device {
    bool ready = false;
    int sms = 0;
    int* status = nullptr;
};

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

bool known_type(int t) { return t == mm::B128_BF16 || t == mm::B128_FP16 || t == mm::B128_FP32; }

}  // namespace

extern "C" {

int mm_cast_block128(const void* x, int type, int64_t rows, int k, int64_t row_stride, void* q, float* sf, void* stream_) {
    B_REQUIRE(known_type(type), "mm_cast_block128: unknown type");
    B_REQUIRE(rows >= 0 && k > 0 && k % 8 == 0 && row_stride >= k && row_stride % 8 == 0, "mm_cast_block128: k and the row stride must be multiples of 8");
    if (rows == 0) return 0;
    B_REQUIRE(x && q && sf, "mm_cast_block128: null pointer");
    B_REQUIRE(aligned(x, 16) && aligned(q, 8) && aligned(sf, 4), "mm_cast_block128: x must be 16-byte, q 8-byte aligned");
    const int64_t per_row = (k + 127) / 128, groups = rows * per_row;
    B_REQUIRE(rows < kMaxDim && groups < kMaxDim, "mm_cast_block128: too many groups");
    Device* d;
    if (int rc = device_of(&d)) return rc;
    int64_t blocks = (groups + 15) / 16;
    if (blocks > (int64_t)d->sms * 16) blocks = (int64_t)d->sms * 16;
    cudaStream_t st = static_cast<cudaStream_t>(stream_);
    uint8_t* o = static_cast<uint8_t*>(q);
    if (type == mm::B128_BF16) mm::cast_block128_kernel<mm::B128_BF16><<<(unsigned)blocks, 256, 0, st>>>(x, row_stride, (uint32_t)groups, (uint32_t)per_row, k, o, sf);
    else if (type == mm::B128_FP16) mm::cast_block128_kernel<mm::B128_FP16><<<(unsigned)blocks, 256, 0, st>>>(x, row_stride, (uint32_t)groups, (uint32_t)per_row, k, o, sf);
    else mm::cast_block128_kernel<mm::B128_FP32><<<(unsigned)blocks, 256, 0, st>>>(x, row_stride, (uint32_t)groups, (uint32_t)per_row, k, o, sf);
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
    B_REQUIRE(tokens >= 0 && hidden > 0 && hidden % 8 == 0 && hidden <= 16384, "mm_norm_gate_residual: hidden must be a multiple of 8, at most 16384");
    B_REQUIRE(quant >= 0 && quant <= 2, "mm_norm_gate_residual: unknown cast");
    B_REQUIRE(known_type(y_type) && known_type(r_type) && known_type(post_type) && known_type(gate_type) && known_type(pre_type) && known_type(x_type),
              "mm_norm_gate_residual: unknown type");
    if (tokens == 0) return 0;
    B_REQUIRE(r && (y ? r_out != nullptr : !post && !gate && !r_out), "mm_norm_gate_residual: null pointer (a norm or gate needs y, y needs a new residual)");
    B_REQUIRE(pre || (!x_out && quant == 0), "mm_norm_gate_residual: outputs of the second norm need its weight");
    B_REQUIRE(quant == 0 || (q && sf), "mm_norm_gate_residual: null pointer");
    B_REQUIRE(r_stride >= hidden && (!y || y_stride >= hidden) && r_stride % 8 == 0 && y_stride % 8 == 0 && (gate_col_stride == 0 || gate_col_stride == 1) &&
              gate_row_stride >= 0 && (gate_col_stride == 0 || gate_row_stride % 8 == 0), "mm_norm_gate_residual: bad strides");
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
    const int per = vecs <= 1024 ? 1 : 2;
    const int threads = ((vecs + per - 1) / per + 31) / 32 * 32;
    const int resident = 2048 / threads;
    int64_t blocks = (int64_t)d->sms * (resident < 1 ? 1 : resident);
    if (blocks > tokens) blocks = tokens;
    cudaStream_t st = static_cast<cudaStream_t>(stream_);
    if (per == 1) mm::norm_gate_residual_kernel<1><<<(unsigned)blocks, threads, 0, st>>>(p);
    else mm::norm_gate_residual_kernel<2><<<(unsigned)blocks, threads, 0, st>>>(p);
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
    p.timeout_ns = mm_detail_pipe_timeout_ns();
    p.m_tiles = (m + 127) / 128;
    p.a_box_rows = m >= 128 ? 128 : (m + 7) / 8 * 8;
    // Tile width and split of K: 256 columns when that fills the SMs, else 128 columns, and as long as that leaves SMs
    // idle the k blocks of a tile are divided among up to eight CTAs.
    const int64_t tiles256 = (int64_t)p.m_tiles * ((n + 255) / 256), tiles128 = (int64_t)p.m_tiles * n_sf;
    const int bn = tiles256 >= d->sms ? 256 : 128;
    const int64_t tiles = bn == 256 ? tiles256 : tiles128;
    B_REQUIRE(tiles < kMaxDim, "mm_fp8_gemm_block128: too many tiles");
    p.n_tiles = bn == 256 ? (n + 255) / 256 : n_sf;
    int split = 1;
    while (bn == 128 && !m_indices && split < 8 && tiles * split * 2 <= d->sms && kb >= split * 4) split *= 2;
    CUtensorMap tm_a, tm_b;
    if (int rc = byte_map(a, (uint64_t)k, (uint64_t)m, (uint64_t)a_stride, 0, 0, (uint32_t)p.a_box_rows, &tm_a)) return rc;
    if (p.tiled) {
        if (int rc = byte_map(b, 128, (uint64_t)experts * p.tiled_n_blocks * kb * 256, 128, 0, 0, (uint32_t)bn, &tm_b)) return rc;
    } else {
        if (int rc = byte_map(b, (uint64_t)k, (uint64_t)n, (uint64_t)k, (uint64_t)experts, (uint64_t)n * k, (uint32_t)bn, &tm_b)) return rc;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream_);
    if (split > 1) {
        cudaLaunchConfig_t cfg;
        memset(&cfg, 0, sizeof(cfg));
        cfg.gridDim = dim3((unsigned)(tiles * split));
        cfg.blockDim = dim3(mm::kB128Threads);
        cfg.dynamicSmemBytes = mm::B128Shape<128>::kSmemBytes;
        cfg.stream = st;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = (unsigned)split; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        B_CUDA(cudaLaunchKernelEx(&cfg, mm::block128_gemm_kernel<128, true>, tm_a, tm_b, p));
    } else {
        const unsigned grid = (unsigned)(tiles < d->sms ? tiles : d->sms);
        if (bn == 256) mm::block128_gemm_kernel<256, false><<<grid, mm::kB128Threads, mm::B128Shape<256>::kSmemBytes, st>>>(tm_a, tm_b, p);
        else mm::block128_gemm_kernel<128, false><<<grid, mm::kB128Threads, mm::B128Shape<128>::kSmemBytes, st>>>(tm_a, tm_b, p);
    }
    B_LAUNCHED();
    return 0;
}

int mm_block128_read_status(void* stream_, int32_t* out5) {
    B_REQUIRE(out5, "mm_block128_read_status: null pointer");
    Device* d;
    if (int rc = device_of(&d)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream_);
    B_CUDA(cudaMemcpyAsync(out5, d->status, 5 * sizeof(int32_t), cudaMemcpyDeviceToHost, st));
    B_CUDA(cudaMemsetAsync(d->status, 0, 8 * sizeof(int), st));
    B_CUDA(cudaStreamSynchronize(st));
    return 0;
}

}  // extern "C"
