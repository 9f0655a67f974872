// extern "C" entry points: argument checks, then the launches on the caller's
// stream.  Nothing here allocates device memory or synchronises.
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <mutex>

#include "common.h"

namespace fni8h {

static thread_local char g_detail[512];

void set_error_detail(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_detail, sizeof g_detail, fmt, ap);
    va_end(ap);
}

}  // namespace fni8h

namespace {

using fni8h::set_error_detail;

constexpr int64_t kMaxDim = (int64_t)1 << 31;
constexpr int kMaxDevices = 64;
// 0 = unknown, 1 = gfx950, -1 = other.  Written once per device; a repeated
// write of the same value from two threads is harmless.
int g_device_ok[kMaxDevices];

int scratch_address(int8_t** out);

int check_device() {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0) {
        set_error_detail("no current HIP device");
        return FNI8_ERR_DEVICE;
    }
    if (dev < kMaxDevices && g_device_ok[dev] == 1) return FNI8_OK;
    hipDeviceProp_t prop;
    if (hipGetDeviceProperties(&prop, dev) != hipSuccess) {
        set_error_detail("hipGetDeviceProperties failed on device %d", dev);
        return FNI8_ERR_DEVICE;
    }
    const bool ok = strncmp(prop.gcnArchName, "gfx950", 6) == 0;
    if (!ok) {
        if (dev < kMaxDevices) g_device_ok[dev] = -1;
        set_error_detail("device %d is %s; these kernels are built for gfx950", dev,
                         prop.gcnArchName);
        return FNI8_ERR_DEVICE;
    }
    // The first call on a device also looks up the no-allocation entry point's
    // scratch address, so that a later call of that entry point under graph
    // capture makes no runtime query.
    int8_t* sp = nullptr;
    const int rc = scratch_address(&sp);
    if (rc) return rc;
    if (dev < kMaxDevices) g_device_ok[dev] = 1;
    return FNI8_OK;
}

// ---- scratch of fni8_linear_w8a8_f16_noalloc ---------------------------------
// The quantized activations (int8 [M, K], row stride K) and their scales
// (fp32 [M]) of the entry point that allocates nothing live in this array: one
// copy per GPU, resident from the library's load on that GPU until the process
// ends.  Every call on a GPU shares its copy (overlapping calls race).
constexpr int64_t kNoAllocQBytes = (int64_t)48 << 20;  // M * K (every Qwen3-8B linear to M = 4096)
constexpr int64_t kNoAllocRows = 65536;                // M
static __device__ __align__(256) int8_t scratch[kNoAllocQBytes + kNoAllocRows * 4];

// Device address of `scratch` on the current device, looked up once per device
// with that device current (in host code `scratch` names a host-side stand-in,
// not device memory).
void* g_scratch_dev[kMaxDevices];
std::mutex g_scratch_mu;

int scratch_address(int8_t** out) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) {
        set_error_detail("no usable current device for the scratch lookup");
        return FNI8_ERR_DEVICE;
    }
    void* p = __atomic_load_n(&g_scratch_dev[dev], __ATOMIC_ACQUIRE);
    if (p == nullptr) {
        std::lock_guard<std::mutex> lock(g_scratch_mu);
        p = g_scratch_dev[dev];
        if (p == nullptr) {
            const hipError_t e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
            if (e != hipSuccess || p == nullptr) {
                set_error_detail("scratch lookup on device %d: %s", dev, hipGetErrorString(e));
                return FNI8_ERR_LAUNCH;
            }
            __atomic_store_n(&g_scratch_dev[dev], p, __ATOMIC_RELEASE);
        }
    }
    *out = static_cast<int8_t*>(p);
    return FNI8_OK;
}

bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }

#define REQUIRE(cond, code, ...)          \
    do {                                  \
        if (!(cond)) {                    \
            set_error_detail(__VA_ARGS__); \
            return (code);                \
        }                                 \
    } while (0)

int check_gemm_shape(int64_t M, int64_t K, int64_t N) {
    REQUIRE(M >= 0 && M < kMaxDim, FNI8_ERR_SHAPE, "M=%lld out of range", (long long)M);
    REQUIRE(N > 0 && N < kMaxDim, FNI8_ERR_SHAPE, "N=%lld out of range", (long long)N);
    REQUIRE(K > 0 && K < kMaxDim, FNI8_ERR_SHAPE, "K=%lld out of range", (long long)K);
    REQUIRE(K % 4 == 0, FNI8_ERR_SHAPE, "K=%lld is not a multiple of 4", (long long)K);
    return FNI8_OK;
}

int check_w4a8(int64_t M, int64_t K, int64_t N, int64_t G, const uint8_t* w, const float* ws,
               const void* bias, const void* y, int64_t ldy) {
    REQUIRE(w && ws && y, FNI8_ERR_NULL, "w, ws and y are required");
    REQUIRE(M >= 0 && M < kMaxDim && N > 0 && N < kMaxDim && K > 0 && K < kMaxDim,
            FNI8_ERR_SHAPE, "M=%lld N=%lld K=%lld out of range", (long long)M, (long long)N,
            (long long)K);
    REQUIRE(G == 32 || G == 64 || G == 128 || G == 256, FNI8_ERR_SHAPE,
            "group size %lld not supported (32, 64, 128, 256)", (long long)G);
    REQUIRE(K % 32 == 0 && K % G == 0, FNI8_ERR_SHAPE,
            "K=%lld must be a multiple of 32 and of the group size %lld", (long long)K,
            (long long)G);
    REQUIRE(ldy >= N, FNI8_ERR_STRIDE, "ldy=%lld < N=%lld", (long long)ldy, (long long)N);
    REQUIRE(aligned(w, 16) && aligned(ws, 4) && aligned(bias, 2) && aligned(y, 2),
            FNI8_ERR_ALIGN, "w must be 16-byte aligned; ws, bias, y element-aligned");
    return FNI8_OK;
}

int check_rmsnorm(const void* x, int64_t ldx, const void* residual, int64_t ldr,
                  const void* weight, float eps, int64_t M, int64_t K, int64_t ldo,
                  const void* residual_out, int64_t ldro) {
    REQUIRE(x && weight, FNI8_ERR_NULL, "x and weight are required");
    REQUIRE(M >= 0 && M < kMaxDim && K > 0 && K < kMaxDim, FNI8_ERR_SHAPE,
            "M=%lld K=%lld out of range", (long long)M, (long long)K);
    REQUIRE(eps >= 0.0f && eps < __builtin_inff(), FNI8_ERR_SHAPE, "eps must be finite and >= 0");
    REQUIRE(ldx >= K && ldo >= K, FNI8_ERR_STRIDE, "ldx=%lld or output stride %lld < K=%lld",
            (long long)ldx, (long long)ldo, (long long)K);
    REQUIRE(!residual || ldr >= K, FNI8_ERR_STRIDE, "ldr=%lld < K", (long long)ldr);
    REQUIRE(!residual || !residual_out || ldro >= K, FNI8_ERR_STRIDE, "ldro=%lld < K",
            (long long)ldro);
    REQUIRE(aligned(x, 2) && aligned(residual, 2) && aligned(weight, 2) &&
                aligned(residual_out, 2),
            FNI8_ERR_ALIGN, "fp16 operands misaligned");
    return FNI8_OK;
}

int linear_launch(const void* x, int64_t ldx, int64_t M, int64_t K, const int8_t* w,
                  const float* ws, int64_t N, const void* bias, void* y, int64_t ldy, int8_t* xq,
                  float* xs, int32_t* acc_out, int8_t* work, int64_t work_bytes, hipStream_t st);

int check_linear(const void* x, int64_t ldx, int64_t M, int64_t K, const int8_t* w,
                 const float* ws, int64_t N, const void* bias, const void* y, int64_t ldy,
                 const int8_t* xq, const float* xs, const int32_t* acc_out) {
    REQUIRE(x && w && ws && y && xq && xs, FNI8_ERR_NULL,
            "x, w, ws, y, xq and xs are required");
    int rc = check_gemm_shape(M, K, N);
    if (rc) return rc;
    REQUIRE(ldx >= K && ldy >= N, FNI8_ERR_STRIDE, "ldx=%lld < K or ldy=%lld < N",
            (long long)ldx, (long long)ldy);
    REQUIRE(aligned(x, 2) && aligned(xq, 4) && aligned(w, 4), FNI8_ERR_ALIGN,
            "x, xq or w misaligned");
    REQUIRE(aligned(xs, 4) && aligned(ws, 4) && aligned(y, 2) && aligned(bias, 2) &&
                aligned(acc_out, 4),
            FNI8_ERR_ALIGN, "scale/output pointers misaligned");
    return FNI8_OK;
}

// One of the q, k, v operands of the rows between QKV and attention.
int check_heads(const char* name, const void* x, int64_t ld, int64_t hs, int64_t H, int64_t D) {
    if (H == 0) return FNI8_OK;
    REQUIRE(x, FNI8_ERR_NULL, "%s is required", name);
    REQUIRE(hs >= D && ld >= D, FNI8_ERR_STRIDE, "%s: token or head stride < D=%lld", name,
            (long long)D);
    REQUIRE(hs < (int64_t)1 << 32, FNI8_ERR_STRIDE, "%s: head stride %lld >= 2^32", name,
            (long long)hs);
    REQUIRE(aligned(x, 16) && ld % 8 == 0 && hs % 8 == 0, FNI8_ERR_ALIGN,
            "%s must be 16-byte aligned with strides that are multiples of 8", name);
    return FNI8_OK;
}

constexpr int64_t kMaxTokens = (int64_t)1 << 23;  // a workgroup a token and 2^32 threads a grid
constexpr int64_t kMaxHeads = 4096;
constexpr int64_t kMaxHeadDim = 256;

int check_rows(const fni8h::QkvRows& r) {
    REQUIRE(r.T >= 0 && r.T <= kMaxTokens, FNI8_ERR_SHAPE, "T=%lld out of range (2^23 at most)",
            (long long)r.T);
    REQUIRE(r.Hq >= 0 && r.Hk >= 0 && r.Hq <= kMaxHeads && r.Hk <= kMaxHeads, FNI8_ERR_SHAPE,
            "Hq=%lld Hk=%lld out of range", (long long)r.Hq, (long long)r.Hk);
    REQUIRE(r.D > 0 && r.D <= kMaxHeadDim && r.D % 8 == 0, FNI8_ERR_SHAPE,
            "D=%lld must be a multiple of 8, at most 256", (long long)r.D);
    REQUIRE(r.R >= 0 && r.R <= r.D && r.R % 2 == 0, FNI8_ERR_SHAPE,
            "R=%lld must be even, from 0 to D=%lld", (long long)r.R, (long long)r.D);
    REQUIRE(r.eps >= 0.0f && r.eps < __builtin_inff(), FNI8_ERR_SHAPE, "eps must be finite and >= 0");
    int rc = check_heads("q", r.q, r.ldq, r.hsq, r.Hq, r.D);
    if (rc) return rc;
    rc = check_heads("k", r.k, r.ldk, r.hsk, r.Hk, r.D);
    if (rc) return rc;
    REQUIRE(r.Hq == 0 || r.q_out, FNI8_ERR_NULL, "q_out is required");
    REQUIRE(aligned(r.q_weight, 16) && aligned(r.k_weight, 16) && aligned(r.q_out, 16) &&
                aligned(r.k_out, 16),
            FNI8_ERR_ALIGN, "weights and outputs must be 16-byte aligned");
    if (r.R) {
        REQUIRE(r.positions && r.cos_sin, FNI8_ERR_NULL, "positions and cos_sin are required");
        REQUIRE(r.P > 0 && r.P < kMaxDim, FNI8_ERR_SHAPE, "P=%lld out of range", (long long)r.P);
        REQUIRE(aligned(r.positions, 4) && aligned(r.cos_sin, 16), FNI8_ERR_ALIGN,
                "cos_sin must be 16-byte aligned, positions element-aligned");
    }
    return FNI8_OK;
}

int check_cache(const void* k_cache, const void* v_cache, const float* k_scale,
                const float* v_scale, int64_t num_pages, int64_t page_size, int64_t Hk, int64_t D) {
    REQUIRE(k_cache && v_cache, FNI8_ERR_NULL, "k_cache and v_cache are required");
    REQUIRE((k_scale == nullptr) == (v_scale == nullptr), FNI8_ERR_NULL,
            "k_scale and v_scale go together");
    REQUIRE(Hk > 0 && Hk <= kMaxHeads, FNI8_ERR_SHAPE, "Hk=%lld out of range", (long long)Hk);
    REQUIRE(D > 0 && D <= kMaxHeadDim && D % 16 == 0, FNI8_ERR_SHAPE,
            "D=%lld must be a multiple of 16, at most 256, with a cache", (long long)D);
    REQUIRE(page_size >= 16 && page_size <= 65536 && (page_size & (page_size - 1)) == 0,
            FNI8_ERR_SHAPE, "page_size=%lld must be a power of two from 16 to 65536",
            (long long)page_size);
    REQUIRE(num_pages > 0 && num_pages < kMaxDim / page_size, FNI8_ERR_SHAPE,
            "num_pages=%lld out of range (num_pages * page_size < 2^31)", (long long)num_pages);
    REQUIRE(aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(k_scale, 16) &&
                aligned(v_scale, 16),
            FNI8_ERR_ALIGN, "caches and scales must be 16-byte aligned");
    return FNI8_OK;
}

constexpr int64_t kMaxWidth = (int64_t)1 << 23;

bool lora_in_range(int64_t T, int64_t K, int64_t S, int64_t all_rank) {
    return T >= 0 && T <= kMaxTokens && K > 0 && K < (int64_t)1 << 24 && S > 0 && S <= 65534 &&
           all_rank > 0 && all_rank <= 256 * FNI8_LORA_MAX_PARTS;
}

// Whether T rows of `wide` bytes at p, ldp bytes apart, and as many at q, ldq apart, share any.
bool rows_meet(const void* p, int64_t ldp, const void* q, int64_t ldq, int64_t T, int64_t wide) {
    const int64_t d = (int64_t)((uintptr_t)q - (uintptr_t)p);
    if (T == 0 || d >= (T - 1) * ldp + wide || -d >= (T - 1) * ldq + wide) return false;
    // rows at s of p's are met by q's at or before s, or by the next
    auto met = [&](int64_t s, int64_t first, int64_t last) {
        const int64_t j = s >= 0 ? s / ldq : -((-s + ldq - 1) / ldq);
        return (j >= first && j <= last && s - j * ldq < wide) ||
               (j + 1 >= first && j + 1 <= last && (j + 1) * ldq - s < wide);
    };
    if (ldp == ldq) return met(-d, 1 - T, T - 1);  // rows i of p and i + j of q
    for (int64_t i = 0; i < T; i++)
        if (met(i * ldp - d, 0, T - 1)) return true;
    return false;
}

bool sample_in_range(int64_t B, int64_t V) {
    return B >= 0 && B <= (int64_t)1 << 20 && V > 0 && V <= (int64_t)1 << 22;
}

}  // namespace

extern "C" {

const char* fni8_strerror(int code) {
    switch (code) {
        case FNI8_OK: return "ok";
        case FNI8_ERR_NULL: return "required pointer is NULL";
        case FNI8_ERR_SHAPE: return "shape out of range";
        case FNI8_ERR_ALIGN: return "pointer or stride misaligned";
        case FNI8_ERR_STRIDE: return "leading dimension smaller than the row";
        case FNI8_ERR_LAUNCH: return "HIP launch error";
        case FNI8_ERR_DEVICE: return "unsupported or missing device";
        default: return "unknown error";
    }
}

const char* fni8_last_error(void) { return fni8h::g_detail; }

const char* fni8_version(void) { return "fni8amd 0.1.0 gfx950"; }

int fni8_init(void) {
    fni8h::g_detail[0] = 0;
    int count = 0, cur = 0;
    if (hipGetDeviceCount(&count) != hipSuccess || count <= 0) {
        set_error_detail("no HIP device");
        return FNI8_ERR_DEVICE;
    }
    if (hipGetDevice(&cur) != hipSuccess) cur = 0;
    int rc = FNI8_OK;
    for (int d = 0; d < count && d < kMaxDevices; d++) {
        hipDeviceProp_t prop;
        if (hipGetDeviceProperties(&prop, d) != hipSuccess ||
            strncmp(prop.gcnArchName, "gfx950", 6) != 0)
            continue;  // other devices are left alone
        if (hipSetDevice(d) != hipSuccess) {
            set_error_detail("hipSetDevice(%d) failed", d);
            rc = FNI8_ERR_DEVICE;
            break;
        }
        rc = check_device();
        if (rc) break;
    }
    (void)hipSetDevice(cur);
    return rc;
}

int fni8_quantize_rowwise_f16(const void* x, int64_t M, int64_t K, int64_t ldx, int8_t* xq,
                              int64_t ldq, float* xs, void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(x && xq && xs, FNI8_ERR_NULL, "x, xq and xs are required");
    REQUIRE(M >= 0 && M < kMaxDim, FNI8_ERR_SHAPE, "M=%lld out of range", (long long)M);
    REQUIRE(K > 0 && K < kMaxDim && K % 4 == 0, FNI8_ERR_SHAPE,
            "K=%lld must be positive and a multiple of 4", (long long)K);
    REQUIRE(ldx >= K && ldq >= K, FNI8_ERR_STRIDE, "ldx=%lld ldq=%lld < K=%lld",
            (long long)ldx, (long long)ldq, (long long)K);
    REQUIRE(aligned(x, 2) && aligned(xs, 4), FNI8_ERR_ALIGN, "x or xs misaligned");
    int rc = check_device();
    if (rc) return rc;
    return fni8h::launch_quant_rowwise((const uint16_t*)x, M, K, ldx, xq, ldq, xs,
                                       (hipStream_t)stream);
}

int fni8_gemm_w8a8(const int8_t* xq, int64_t ldq, const float* xs, int64_t M, int64_t K,
                   const int8_t* w, const float* ws, int64_t N, const void* bias, void* y,
                   int64_t ldy, int32_t* acc_out, void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(xq && xs && w && ws && y, FNI8_ERR_NULL, "xq, xs, w, ws and y are required");
    int rc = check_gemm_shape(M, K, N);
    if (rc) return rc;
    REQUIRE(ldq >= K && ldy >= N, FNI8_ERR_STRIDE, "ldq=%lld < K or ldy=%lld < N",
            (long long)ldq, (long long)ldy);
    REQUIRE(ldq % 4 == 0 && aligned(xq, 4) && aligned(w, 4), FNI8_ERR_ALIGN,
            "int8 operands need 4-byte aligned rows");
    REQUIRE(aligned(xs, 4) && aligned(ws, 4) && aligned(y, 2) && aligned(bias, 2) &&
                aligned(acc_out, 4),
            FNI8_ERR_ALIGN, "scale/output pointers misaligned");
    rc = check_device();
    if (rc) return rc;
    return fni8h::launch_gemm(xq, ldq, xs, nullptr, M, K, w, ws, N, 0, nullptr,
                              (const uint16_t*)bias, (uint16_t*)y, ldy, acc_out,
                              (hipStream_t)stream);
}

int fni8_linear_w8a8_f16(const void* x, int64_t ldx, int64_t M, int64_t K, const int8_t* w,
                         const float* ws, int64_t N, const void* bias, void* y, int64_t ldy,
                         int8_t* xq, float* xs, int32_t* acc_out, void* stream) {
    fni8h::g_detail[0] = 0;
    int rc = check_linear(x, ldx, M, K, w, ws, N, bias, y, ldy, xq, xs, acc_out);
    if (rc) return rc;
    rc = check_device();
    if (rc) return rc;
    return linear_launch(x, ldx, M, K, w, ws, N, bias, y, ldy, xq, xs, acc_out, nullptr, 0,
                         (hipStream_t)stream);
}

int fni8_linear_w8a8_f16_ws(const void* x, int64_t ldx, int64_t M, int64_t K, const int8_t* w,
                            const float* ws, int64_t N, const void* bias, void* y, int64_t ldy,
                            int8_t* xq, float* xs, int32_t* acc_out, void* workspace,
                            int64_t workspace_bytes, void* stream) {
    fni8h::g_detail[0] = 0;
    int rc = check_linear(x, ldx, M, K, w, ws, N, bias, y, ldy, xq, xs, acc_out);
    if (rc) return rc;
    REQUIRE(workspace_bytes >= 0 && (!workspace || aligned(workspace, 256)), FNI8_ERR_ALIGN,
            "workspace must be 256-byte aligned with a size >= 0");
    rc = check_device();
    if (rc) return rc;
    return linear_launch(x, ldx, M, K, w, ws, N, bias, y, ldy, xq, xs, acc_out,
                         static_cast<int8_t*>(workspace), workspace ? workspace_bytes : 0,
                         (hipStream_t)stream);
}

int64_t fni8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M < 0 || N <= 0 || K <= 0 || M >= kMaxDim || N >= kMaxDim || K >= kMaxDim) return 0;
    if (M <= 16) return fni8h::coop_workspace_bytes(M, N, K);
    return fni8h::pp_workspace_bytes(M, N, K);
}

int fni8_gemm_w8a8_ws(const int8_t* xq, int64_t ldq, const float* xs, int64_t M, int64_t K,
                      const int8_t* w, const float* ws, int64_t N, const void* bias, void* y,
                      int64_t ldy, int32_t* acc_out, void* workspace, int64_t workspace_bytes,
                      void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(xq && xs && w && ws && y, FNI8_ERR_NULL, "xq, xs, w, ws and y are required");
    int rc = check_gemm_shape(M, K, N);
    if (rc) return rc;
    REQUIRE(ldq >= K && ldy >= N, FNI8_ERR_STRIDE, "ldq=%lld < K or ldy=%lld < N",
            (long long)ldq, (long long)ldy);
    REQUIRE(ldq % 4 == 0 && aligned(xq, 4) && aligned(w, 4), FNI8_ERR_ALIGN,
            "int8 operands need 4-byte aligned rows");
    REQUIRE(aligned(xs, 4) && aligned(ws, 4) && aligned(y, 2) && aligned(bias, 2) &&
                aligned(acc_out, 4),
            FNI8_ERR_ALIGN, "scale/output pointers misaligned");
    REQUIRE(workspace_bytes >= 0 && (!workspace || aligned(workspace, 256)), FNI8_ERR_ALIGN,
            "workspace must be 256-byte aligned with a size >= 0");
    rc = check_device();
    if (rc) return rc;
    return fni8h::launch_gemm(xq, ldq, xs, nullptr, M, K, w, ws, N, 0, nullptr,
                              (const uint16_t*)bias, (uint16_t*)y, ldy, acc_out,
                              (hipStream_t)stream, static_cast<int8_t*>(workspace),
                              workspace ? workspace_bytes : 0);
}

void fni8_debug_coop_wait_ticks(int64_t ticks) { fni8h::set_coop_wait_ticks(ticks); }

void fni8_debug_gemm_plan(int64_t bm, int64_t bn, int64_t split) {
    fni8h::set_gemm_plan(bm, bn, split);
}

int fni8_linear_w8a8_f16_noalloc(const void* x, int64_t ldx, int64_t M, int64_t K,
                                 const int8_t* w, const float* ws, int64_t N, const void* bias,
                                 void* y, int64_t ldy, void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(x && w && ws && y, FNI8_ERR_NULL, "x, w, ws and y are required");
    int rc = check_gemm_shape(M, K, N);
    if (rc) return rc;
    REQUIRE(M <= kNoAllocRows && M * K <= kNoAllocQBytes, FNI8_ERR_SHAPE,
            "M=%lld K=%lld exceeds the no-allocation scratch (M <= %lld and M*K <= %lld bytes)",
            (long long)M, (long long)K, (long long)kNoAllocRows, (long long)kNoAllocQBytes);
    REQUIRE(ldx >= K && ldy >= N, FNI8_ERR_STRIDE, "ldx=%lld < K or ldy=%lld < N",
            (long long)ldx, (long long)ldy);
    REQUIRE(aligned(x, 2) && aligned(w, 4) && aligned(ws, 4) && aligned(y, 2) && aligned(bias, 2),
            FNI8_ERR_ALIGN, "x, w, ws, y or bias misaligned");
    rc = check_device();
    if (rc) return rc;
    int8_t* sp = nullptr;
    rc = scratch_address(&sp);
    if (rc) return rc;
    // xq: M rows of K bytes at the start; xs: M floats after the xq area; the
    // rest of the xq area (past M * K, 256-aligned) is the workspace of the
    // one-launch decode path and of the split-K prefill GEMM (where its plan
    // fits).  Every byte the GEMM reads is written by this call's quantization
    // first, and the workspace needs no clearing, so nothing is cleared between
    // calls.
    const int64_t work_off = (M * K + 255) & ~(int64_t)255;
    return linear_launch(x, ldx, M, K, w, ws, N, bias, y, ldy, sp,
                         reinterpret_cast<float*>(sp + kNoAllocQBytes), nullptr, sp + work_off,
                         kNoAllocQBytes - work_off, (hipStream_t)stream);
}

}  // extern "C"

namespace {

// The launches of the whole W8A8 linear on caller-checked arguments.
int linear_launch(const void* x, int64_t ldx, int64_t M, int64_t K, const int8_t* w,
                  const float* ws, int64_t N, const void* bias, void* y, int64_t ldy, int8_t* xq,
                  float* xs, int32_t* acc_out, int8_t* work, int64_t work_bytes, hipStream_t st) {
    int rc;
    // 5..16 tokens with a workspace: one launch, the quantization shared per XCD
    if (M >= 5 && work != nullptr) {
        rc = fni8h::launch_decode_coop((const uint16_t*)x, ldx, M, K, w, ws, N,
                                       (const uint16_t*)bias, (uint16_t*)y, ldy, xq, xs, acc_out,
                                       work, work_bytes, st);
        if (rc != 1) return rc;
    }
    // Decode sizes: one launch, the quantization fused into the GEMM -- on MFMA
    // for 3..4 tokens, as a dot4 GEMV for 1..2 (and shapes the MFMA kernel does
    // not take), where the streaming loop without an LDS pass is faster.
    if (M >= 3) {
        rc = fni8h::launch_decode_mfma_fused((const uint16_t*)x, ldx, M, K, w, ws, N,
                                             (const uint16_t*)bias, (uint16_t*)y, ldy, xq, xs,
                                             acc_out, st);
        if (rc != 1) return rc;
    }
    rc = fni8h::launch_decode_fused((const uint16_t*)x, ldx, M, K, w, ws, N, (const uint16_t*)bias,
                                    (uint16_t*)y, ldy, xq, xs, acc_out, st);
    if (rc != 1) return rc;
    rc = fni8h::launch_quant_rowwise((const uint16_t*)x, M, K, ldx, xq, K, xs, st);
    if (rc) return rc;
    return fni8h::launch_gemm(xq, K, xs, nullptr, M, K, w, ws, N, 0, nullptr,
                              (const uint16_t*)bias, (uint16_t*)y, ldy, acc_out, st, work,
                              work_bytes);
}

}  // namespace

extern "C" {

int fni8_moe_sort(const int32_t* topi, int64_t T, int64_t k, int64_t E, int32_t* seg_off,
                  int32_t* row_token, int32_t* pos, void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(topi && seg_off && row_token && pos, FNI8_ERR_NULL,
            "topi, seg_off, row_token and pos are required");
    REQUIRE(T >= 0 && k > 0 && k <= 32 && E > 0 && E < 65536 && T * k < kMaxDim,
            FNI8_ERR_SHAPE, "T=%lld k=%lld E=%lld out of range (k <= 32)", (long long)T,
            (long long)k, (long long)E);
    REQUIRE(aligned(topi, 4) && aligned(seg_off, 4) && aligned(row_token, 4) && aligned(pos, 4),
            FNI8_ERR_ALIGN, "int32 arrays misaligned");
    int rc = check_device();
    if (rc) return rc;
    return fni8h::launch_moe_sort(topi, T, k, E, seg_off, row_token, pos, (hipStream_t)stream);
}

int fni8_gemm_w8a8_grouped(const int8_t* aq, const float* as, const int32_t* row_index,
                           int64_t R_max, int64_t K, const int8_t* w, const float* ws,
                           int64_t E, int64_t N, const int32_t* seg_off, const void* bias,
                           void* y, int32_t* acc_out, void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(aq && as && w && ws && seg_off && y, FNI8_ERR_NULL,
            "aq, as, w, ws, seg_off and y are required");
    int rc = check_gemm_shape(R_max, K, N);
    if (rc) return rc;
    REQUIRE(E > 0 && E < 65536, FNI8_ERR_SHAPE, "E=%lld out of range", (long long)E);
    REQUIRE(aligned(aq, 4) && aligned(w, 4) && aligned(as, 4) && aligned(ws, 4) &&
                aligned(row_index, 4) && aligned(seg_off, 4) && aligned(y, 2) &&
                aligned(bias, 2) && aligned(acc_out, 4),
            FNI8_ERR_ALIGN, "grouped operands misaligned");
    rc = check_device();
    if (rc) return rc;
    return fni8h::launch_gemm(aq, K, as, row_index, R_max, K, w, ws, N, E, seg_off,
                              (const uint16_t*)bias, (uint16_t*)y, N, acc_out,
                              (hipStream_t)stream);
}

int fni8_gemm_w4a8_grouped(const int8_t* aq, const float* as, const int32_t* row_index,
                           int64_t R_max, int64_t K, const uint8_t* w, const float* ws,
                           int64_t E, int64_t N, int64_t G, const int32_t* seg_off,
                           const void* bias, void* y, void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(aq && as && w && ws && seg_off && y, FNI8_ERR_NULL,
            "aq, as, w, ws, seg_off and y are required");
    int rc = check_w4a8(R_max, K, N, G, w, ws, bias, y, N);
    if (rc) return rc;
    REQUIRE(E > 0 && E < 65536, FNI8_ERR_SHAPE, "E=%lld out of range", (long long)E);
    REQUIRE(G >= 64 && K % 256 == 0 && N < (1 << 21), FNI8_ERR_SHAPE,
            "grouped W4A8 needs G in {64, 128, 256}, K a multiple of 256 and N < 2^21 "
            "(G=%lld K=%lld N=%lld)", (long long)G, (long long)K, (long long)N);
    REQUIRE(aligned(aq, 16) && aligned(as, 4) && aligned(row_index, 4) && aligned(seg_off, 4),
            FNI8_ERR_ALIGN, "aq must be 16-byte aligned; as, row_index, seg_off 4-byte aligned");
    rc = check_device();
    if (rc) return rc;
    return fni8h::launch_gemm_w4a8_grouped(aq, as, row_index, R_max, K, w, ws, E, N, G, seg_off,
                                           (const uint16_t*)bias, (uint16_t*)y,
                                           (hipStream_t)stream);
}

int fni8_moe_combine_f16(const void* y_sorted, int64_t H, const int32_t* topi,
                         const void* topw, const int32_t* pos, int64_t T, int64_t k,
                         void* out, void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(y_sorted && topi && topw && pos && out, FNI8_ERR_NULL,
            "y_sorted, topi, topw, pos and out are required");
    REQUIRE(H > 0 && H < kMaxDim && T >= 0 && T < kMaxDim && k > 0 && k <= 32 &&
                T * k < kMaxDim,
            FNI8_ERR_SHAPE, "H=%lld T=%lld k=%lld out of range (k <= 32)", (long long)H,
            (long long)T, (long long)k);
    REQUIRE(aligned(y_sorted, 2) && aligned(topw, 2) && aligned(out, 2) && aligned(topi, 4) &&
                aligned(pos, 4),
            FNI8_ERR_ALIGN, "combine operands misaligned");
    int rc = check_device();
    if (rc) return rc;
    return fni8h::launch_moe_combine((const uint16_t*)y_sorted, H, topi, (const uint16_t*)topw,
                                     pos, T, k, (uint16_t*)out, (hipStream_t)stream);
}

int fni8_gemm_w4a8(const int8_t* xq, int64_t ldq, const float* xs, int64_t M, int64_t K,
                   const uint8_t* w, const float* ws, int64_t N, int64_t G, const void* bias,
                   void* y, int64_t ldy, void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(xq && xs, FNI8_ERR_NULL, "xq and xs are required");
    int rc = check_w4a8(M, K, N, G, w, ws, bias, y, ldy);
    if (rc) return rc;
    REQUIRE(ldq >= K, FNI8_ERR_STRIDE, "ldq=%lld < K=%lld", (long long)ldq, (long long)K);
    REQUIRE(ldq % 16 == 0 && aligned(xq, 16) && aligned(xs, 4), FNI8_ERR_ALIGN,
            "xq rows must be 16-byte aligned");
    rc = check_device();
    if (rc) return rc;
    return fni8h::launch_gemm_w4a8(xq, ldq, xs, M, K, w, ws, N, G, (const uint16_t*)bias,
                                   (uint16_t*)y, ldy, (hipStream_t)stream);
}

int fni8_linear_w4a8_f16(const void* x, int64_t ldx, int64_t M, int64_t K, const uint8_t* w,
                         const float* ws, int64_t N, int64_t G, const void* bias, void* y,
                         int64_t ldy, int8_t* xq, float* xs, void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(x && xq && xs, FNI8_ERR_NULL, "x, xq and xs are required");
    int rc = check_w4a8(M, K, N, G, w, ws, bias, y, ldy);
    if (rc) return rc;
    REQUIRE(ldx >= K, FNI8_ERR_STRIDE, "ldx=%lld < K=%lld", (long long)ldx, (long long)K);
    REQUIRE(aligned(x, 2) && aligned(xq, 16) && aligned(xs, 4), FNI8_ERR_ALIGN,
            "x, xq or xs misaligned");
    rc = check_device();
    if (rc) return rc;
    hipStream_t st = (hipStream_t)stream;
    // decode sizes: one launch, the quantization fused into the stream kernel
    rc = fni8h::launch_linear_w4a8_fused((const uint16_t*)x, ldx, M, K, w, ws, N, G,
                                         (const uint16_t*)bias, (uint16_t*)y, ldy, xq, xs, st);
    if (rc != 1) return rc;
    rc = fni8h::launch_quant_rowwise((const uint16_t*)x, M, K, ldx, xq, K, xs, st);
    if (rc) return rc;
    return fni8h::launch_gemm_w4a8(xq, K, xs, M, K, w, ws, N, G, (const uint16_t*)bias,
                                   (uint16_t*)y, ldy, st);
}

int fni8_moe_route(const float* logits, int64_t T, int64_t E, int64_t ldl, int scoring,
                   const float* bias, int64_t groups, int64_t topk_group, int64_t k, int renorm,
                   float scale, void* topw, int32_t* topi, void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(logits && topw && topi, FNI8_ERR_NULL, "logits, topw and topi are required");
    REQUIRE(T >= 0 && T < kMaxDim && E >= 1 && E <= 1024, FNI8_ERR_SHAPE,
            "T=%lld E=%lld out of range (E <= 1024)", (long long)T, (long long)E);
    REQUIRE(k >= 1 && k <= 32 && k <= E, FNI8_ERR_SHAPE, "k=%lld out of range (1..min(32, E))",
            (long long)k);
    REQUIRE(scoring == FNI8_SCORE_SOFTMAX || scoring == FNI8_SCORE_SIGMOID, FNI8_ERR_SHAPE,
            "unknown scoring function %d", scoring);
    REQUIRE(groups == 0 || (groups >= 1 && groups <= 64 && E % groups == 0 && topk_group >= 1 &&
                            topk_group <= groups),
            FNI8_ERR_SHAPE, "groups=%lld topk_group=%lld invalid for E=%lld", (long long)groups,
            (long long)topk_group, (long long)E);
    REQUIRE(scale == scale && scale > -__builtin_inff() && scale < __builtin_inff(),
            FNI8_ERR_SHAPE, "scale must be finite");
    REQUIRE(ldl >= E, FNI8_ERR_STRIDE, "ldl=%lld < E=%lld", (long long)ldl, (long long)E);
    REQUIRE(aligned(logits, 4) && aligned(bias, 4) && aligned(topw, 2) && aligned(topi, 4),
            FNI8_ERR_ALIGN, "router operands misaligned");
    int rc = check_device();
    if (rc) return rc;
    return fni8h::launch_moe_route(logits, ldl, T, E, scoring, bias, groups, topk_group, k,
                                   renorm ? 1 : 0, scale, (uint16_t*)topw, topi,
                                   (hipStream_t)stream);
}

int fni8_act_and_mul_f16(const void* x, int64_t ldx, int64_t M, int64_t I, int act, void* out,
                         int64_t ldo, void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(x && out, FNI8_ERR_NULL, "x and out are required");
    REQUIRE(M >= 0 && M < kMaxDim && I > 0 && I < kMaxDim / 2, FNI8_ERR_SHAPE,
            "M=%lld I=%lld out of range", (long long)M, (long long)I);
    REQUIRE(act == FNI8_ACT_SILU || act == FNI8_ACT_GELU_TANH, FNI8_ERR_SHAPE,
            "unknown activation %d", act);
    REQUIRE(ldx >= 2 * I && ldo >= I, FNI8_ERR_STRIDE, "ldx=%lld < 2I or ldo=%lld < I",
            (long long)ldx, (long long)ldo);
    REQUIRE(aligned(x, 2) && aligned(out, 2), FNI8_ERR_ALIGN, "x or out misaligned");
    int rc = check_device();
    if (rc) return rc;
    return fni8h::launch_act_and_mul((const uint16_t*)x, ldx, M, I, act, (uint16_t*)out, ldo,
                                     (hipStream_t)stream);
}

int fni8_act_and_mul_quant_f16(const void* x, int64_t ldx, int64_t M, int64_t I, int act,
                               int8_t* xq, int64_t ldq, float* xs, void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(x && xq && xs, FNI8_ERR_NULL, "x, xq and xs are required");
    REQUIRE(M >= 0 && M < kMaxDim && I > 0 && I < kMaxDim / 2 && I % 4 == 0, FNI8_ERR_SHAPE,
            "M=%lld I=%lld out of range (I a multiple of 4)", (long long)M, (long long)I);
    REQUIRE(act == FNI8_ACT_SILU || act == FNI8_ACT_GELU_TANH, FNI8_ERR_SHAPE,
            "unknown activation %d", act);
    REQUIRE(ldx >= 2 * I && ldq >= I, FNI8_ERR_STRIDE, "ldx=%lld < 2I or ldq=%lld < I",
            (long long)ldx, (long long)ldq);
    REQUIRE(aligned(x, 2) && aligned(xs, 4), FNI8_ERR_ALIGN, "x or xs misaligned");
    int rc = check_device();
    if (rc) return rc;
    return fni8h::launch_act_and_mul_quant((const uint16_t*)x, ldx, M, I, act, xq, ldq, xs,
                                           nullptr, 0, (hipStream_t)stream);
}

int fni8_act_and_mul_quant_f16_ws(const void* x, int64_t ldx, int64_t M, int64_t I, int act,
                                  int8_t* xq, int64_t ldq, float* xs, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(x && xq && xs, FNI8_ERR_NULL, "x, xq and xs are required");
    REQUIRE(M >= 0 && M < kMaxDim && I > 0 && I < kMaxDim / 2 && I % 4 == 0, FNI8_ERR_SHAPE,
            "M=%lld I=%lld out of range (I a multiple of 4)", (long long)M, (long long)I);
    REQUIRE(act == FNI8_ACT_SILU || act == FNI8_ACT_GELU_TANH, FNI8_ERR_SHAPE,
            "unknown activation %d", act);
    REQUIRE(ldx >= 2 * I && ldq >= I, FNI8_ERR_STRIDE, "ldx=%lld < 2I or ldq=%lld < I",
            (long long)ldx, (long long)ldq);
    REQUIRE(aligned(x, 2) && aligned(xs, 4), FNI8_ERR_ALIGN, "x or xs misaligned");
    REQUIRE(workspace_bytes >= 0 && (!workspace || aligned(workspace, 256)), FNI8_ERR_ALIGN,
            "workspace must be 256-byte aligned with a size >= 0");
    int rc = check_device();
    if (rc) return rc;
    return fni8h::launch_act_and_mul_quant((const uint16_t*)x, ldx, M, I, act, xq, ldq, xs,
                                           static_cast<int8_t*>(workspace),
                                           workspace ? workspace_bytes : 0, (hipStream_t)stream);
}

int64_t fni8_act_and_mul_quant_workspace_bytes(int64_t M, int64_t I) {
    if (M < 0 || I <= 0 || M >= kMaxDim || I >= kMaxDim / 2) return 0;
    return fni8h::act_quant_workspace_bytes(M, I);
}

int fni8_rmsnorm_f16(const void* x, int64_t ldx, const void* residual, int64_t ldr,
                     const void* weight, float eps, int unit_offset, int64_t M, int64_t K,
                     void* out, int64_t ldo, void* residual_out, int64_t ldro, void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(out, FNI8_ERR_NULL, "out is required");
    int rc = check_rmsnorm(x, ldx, residual, ldr, weight, eps, M, K, ldo, residual_out, ldro);
    if (rc) return rc;
    REQUIRE(aligned(out, 2), FNI8_ERR_ALIGN, "out misaligned");
    rc = check_device();
    if (rc) return rc;
    return fni8h::launch_rmsnorm((const uint16_t*)x, ldx, (const uint16_t*)residual, ldr,
                                 (const uint16_t*)weight, eps, unit_offset ? 1 : 0, M, K,
                                 (uint16_t*)out, ldo,
                                 residual ? (uint16_t*)residual_out : nullptr, ldro, nullptr, 0,
                                 nullptr, (hipStream_t)stream);
}

int fni8_rmsnorm_quant_f16(const void* x, int64_t ldx, const void* residual, int64_t ldr,
                           const void* weight, float eps, int unit_offset, int64_t M, int64_t K,
                           int8_t* xq, int64_t ldq, float* xs, void* residual_out,
                           int64_t ldro, void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(xq && xs, FNI8_ERR_NULL, "xq and xs are required");
    int rc = check_rmsnorm(x, ldx, residual, ldr, weight, eps, M, K, ldq, residual_out, ldro);
    if (rc) return rc;
    REQUIRE(K % 4 == 0, FNI8_ERR_SHAPE, "K=%lld is not a multiple of 4", (long long)K);
    REQUIRE(aligned(xs, 4), FNI8_ERR_ALIGN, "xs misaligned");
    rc = check_device();
    if (rc) return rc;
    return fni8h::launch_rmsnorm((const uint16_t*)x, ldx, (const uint16_t*)residual, ldr,
                                 (const uint16_t*)weight, eps, unit_offset ? 1 : 0, M, K, nullptr,
                                 0, residual ? (uint16_t*)residual_out : nullptr, ldro, xq, ldq,
                                 xs, (hipStream_t)stream);
}

int fni8_qk_norm_rope_f16(const void* q, int64_t ldq, int64_t hsq, int64_t Hq, const void* k,
                          int64_t ldk, int64_t hsk, int64_t Hk, int64_t T, int64_t D,
                          const void* q_weight, const void* k_weight, float eps, int unit_offset,
                          const int32_t* positions, const float* cos_sin, int64_t P, int64_t R,
                          int interleaved, void* q_out, void* k_out, void* stream) {
    fni8h::g_detail[0] = 0;
    fni8h::QkvRows r{};
    r.q = (const uint16_t*)q; r.ldq = ldq; r.hsq = hsq; r.Hq = Hq;
    r.k = (const uint16_t*)k; r.ldk = ldk; r.hsk = hsk; r.Hk = Hk;
    r.T = T; r.D = D;
    r.q_weight = (const uint16_t*)q_weight; r.k_weight = (const uint16_t*)k_weight;
    r.eps = eps; r.unit_offset = unit_offset;
    r.positions = positions; r.cos_sin = cos_sin; r.P = P; r.R = R; r.interleaved = interleaved;
    r.q_out = (uint16_t*)q_out; r.k_out = (uint16_t*)k_out;
    int rc = check_rows(r);
    if (rc) return rc;
    REQUIRE(Hk == 0 || k_out, FNI8_ERR_NULL, "k_out is required");
    rc = check_device();
    if (rc) return rc;
    return fni8h::launch_qkv_rows(r, (hipStream_t)stream);
}

int fni8_rope_append_f16(const void* q, int64_t ldq, int64_t hsq, int64_t Hq, const void* k,
                         int64_t ldk, int64_t hsk, int64_t Hk, const void* v, int64_t ldv,
                         int64_t hsv, int64_t T, int64_t D, const void* q_weight,
                         const void* k_weight, float eps, int unit_offset,
                         const int32_t* positions, const float* cos_sin, int64_t P, int64_t R,
                         int interleaved, void* q_out, void* k_cache, void* v_cache,
                         float* k_scale, float* v_scale, int64_t num_pages, int64_t page_size,
                         const int32_t* slots, void* stream) {
    fni8h::g_detail[0] = 0;
    fni8h::QkvRows r{};
    r.q = (const uint16_t*)q; r.ldq = ldq; r.hsq = hsq; r.Hq = Hq;
    r.k = (const uint16_t*)k; r.ldk = ldk; r.hsk = hsk; r.Hk = Hk;
    r.v = (const uint16_t*)v; r.ldv = ldv; r.hsv = hsv;
    r.T = T; r.D = D;
    r.q_weight = (const uint16_t*)q_weight; r.k_weight = (const uint16_t*)k_weight;
    r.eps = eps; r.unit_offset = unit_offset;
    r.positions = positions; r.cos_sin = cos_sin; r.P = P; r.R = R; r.interleaved = interleaved;
    r.q_out = (uint16_t*)q_out;
    r.k_cache = k_cache; r.v_cache = v_cache; r.k_scale = k_scale; r.v_scale = v_scale;
    r.num_pages = num_pages; r.page_size = page_size; r.slots = slots;
    int rc = check_rows(r);
    if (rc) return rc;
    rc = check_cache(k_cache, v_cache, k_scale, v_scale, num_pages, page_size, Hk, D);
    if (rc) return rc;
    rc = check_heads("v", v, ldv, hsv, Hk, D);
    if (rc) return rc;
    REQUIRE(slots, FNI8_ERR_NULL, "slots is required");
    REQUIRE(aligned(slots, 4), FNI8_ERR_ALIGN, "slots misaligned");
    rc = check_device();
    if (rc) return rc;
    return fni8h::launch_qkv_rows(r, (hipStream_t)stream);
}

int fni8_paged_attention_f16(const void* q, int64_t ldq, int64_t hsq, int64_t T, int64_t Hq,
                             int64_t Hk, int64_t D, const void* k_cache, const void* v_cache,
                             const float* k_scale, const float* v_scale, int64_t num_pages,
                             int64_t page_size, const int32_t* block_tables, int64_t ldt,
                             int64_t max_pages, const int32_t* context_lens,
                             const int32_t* cu_seqlens, int64_t B, int64_t max_seqlen, float scale,
                             int64_t window, void* out, void* workspace, int64_t workspace_bytes,
                             void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(out && block_tables && context_lens, FNI8_ERR_NULL,
            "out, block_tables and context_lens are required");
    REQUIRE(T >= 0 && T <= kMaxTokens, FNI8_ERR_SHAPE, "T=%lld out of range (2^23 at most)",
            (long long)T);
    REQUIRE(B > 0 && B <= 65536, FNI8_ERR_SHAPE, "B=%lld out of range (1 to 65536)", (long long)B);
    REQUIRE(cu_seqlens || T == B, FNI8_ERR_SHAPE, "without cu_seqlens, T=%lld must equal B=%lld",
            (long long)T, (long long)B);
    REQUIRE(max_seqlen >= 0, FNI8_ERR_SHAPE, "max_seqlen=%lld is negative", (long long)max_seqlen);
    int rc = check_cache(k_cache, v_cache, k_scale, v_scale, num_pages, page_size, Hk, D);
    if (rc) return rc;
    REQUIRE(Hq > 0 && Hq <= kMaxHeads && Hq % Hk == 0, FNI8_ERR_SHAPE,
            "Hq=%lld must be a multiple of Hk=%lld", (long long)Hq, (long long)Hk);
    rc = check_heads("q", q, ldq, hsq, Hq, D);
    if (rc) return rc;
    REQUIRE(max_pages > 0 && max_pages <= ((int64_t)1 << 30) / page_size, FNI8_ERR_SHAPE,
            "max_pages=%lld out of range (max_pages * page_size <= 2^30)", (long long)max_pages);
    REQUIRE(ldt >= max_pages, FNI8_ERR_STRIDE, "ldt=%lld < max_pages=%lld", (long long)ldt,
            (long long)max_pages);
    REQUIRE(window >= 0, FNI8_ERR_SHAPE, "window=%lld is negative", (long long)window);
    REQUIRE(scale == scale && scale > -__builtin_inff() && scale < __builtin_inff(),
            FNI8_ERR_SHAPE, "scale must be finite");
    REQUIRE(aligned(out, 16) && aligned(block_tables, 4) && aligned(context_lens, 4) &&
                aligned(cu_seqlens, 4),
            FNI8_ERR_ALIGN, "out must be 16-byte aligned, the int32 arrays element-aligned");
    REQUIRE(workspace_bytes >= 0 && (!workspace || aligned(workspace, 256)), FNI8_ERR_ALIGN,
            "workspace must be 256-byte aligned with a size >= 0");
    rc = check_device();
    if (rc) return rc;
    fni8h::PagedAttention a{};
    a.q = (const uint16_t*)q; a.ldq = ldq; a.hsq = hsq; a.T = T; a.Hq = Hq; a.Hk = Hk; a.D = D;
    a.k_cache = k_cache; a.v_cache = v_cache; a.k_scale = k_scale; a.v_scale = v_scale;
    a.num_pages = num_pages; a.page_size = page_size;
    a.block_tables = block_tables; a.ldt = ldt; a.max_pages = max_pages;
    a.context_lens = context_lens; a.cu_seqlens = cu_seqlens; a.B = B;
    // one token a sequence without cu_seqlens; a bound beyond T says no more than T
    a.max_seqlen = cu_seqlens ? (max_seqlen < T ? max_seqlen : T) : 1;
    a.scale = scale; a.window = window; a.out = (uint16_t*)out;
    a.work = static_cast<int8_t*>(workspace);
    a.work_bytes = workspace ? workspace_bytes : 0;
    return fni8h::launch_paged_attention(a, (hipStream_t)stream);
}

int64_t fni8_paged_attention_workspace_bytes(int64_t T, int64_t Hq, int64_t Hk, int64_t D,
                                             int64_t B, int64_t max_seqlen, int64_t max_context) {
    if (T <= 0 || T > kMaxTokens || Hk <= 0 || Hk > kMaxHeads || Hq <= 0 || Hq > kMaxHeads ||
        Hq % Hk || D <= 0 || D > kMaxHeadDim || B <= 0 || B > 65536 || max_seqlen < 0 ||
        max_context <= 0 || max_context > (int64_t)1 << 30)
        return 0;
    return fni8h::paged_attention_workspace_bytes(T, Hq, Hk, D, B, max_seqlen < T ? max_seqlen : T,
                                                  max_context);
}

int fni8_lora_add_f16(const void* x, int64_t ldx, int64_t T, int64_t K, const void* a,
                      const void* b, int64_t S, int64_t rank, const int64_t* splits,
                      int64_t parts, const float* scaling, const int32_t* seg_off,
                      const int32_t* rows, const void* y, int64_t ldy, void* out, int64_t ldo,
                      void* workspace, int64_t workspace_bytes, void* stream) {
    return fni8_lora_add_ranks_f16(x, ldx, T, K, a, b, S, rank, splits, parts, scaling, nullptr,
                                   seg_off, rows, y, ldy, out, ldo, workspace, workspace_bytes,
                                   stream);
}

int fni8_lora_add_ranks_f16(const void* x, int64_t ldx, int64_t T, int64_t K, const void* a,
                            const void* b, int64_t S, int64_t rank, const int64_t* splits,
                            int64_t parts, const float* scaling, const int32_t* ranks,
                            const int32_t* seg_off, const int32_t* rows, const void* y,
                            int64_t ldy, void* out, int64_t ldo, void* workspace,
                            int64_t workspace_bytes, void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(x && a && b && splits && seg_off && rows && y && out, FNI8_ERR_NULL,
            "x, a, b, splits, seg_off, rows, y and out are required");
    REQUIRE(rank > 0 && rank <= 256 && rank % 8 == 0, FNI8_ERR_SHAPE,
            "rank=%lld must be a multiple of 8, at most 256", (long long)rank);
    REQUIRE(parts > 0 && parts <= FNI8_LORA_MAX_PARTS, FNI8_ERR_SHAPE, "parts=%lld (1 to %d)",
            (long long)parts, FNI8_LORA_MAX_PARTS);
    REQUIRE(lora_in_range(T, K, S, parts * rank), FNI8_ERR_SHAPE,
            "T=%lld K=%lld S=%lld out of range (T <= 2^23, K < 2^24, S <= 65534)", (long long)T,
            (long long)K, (long long)S);
    int64_t N = 0;
    for (int64_t i = 0; i < parts; i++) {
        REQUIRE(splits[i] > 0 && splits[i] < kMaxWidth, FNI8_ERR_SHAPE,
                "splits[%lld]=%lld out of range", (long long)i, (long long)splits[i]);
        N += splits[i];
    }
    REQUIRE(N < kMaxWidth, FNI8_ERR_SHAPE, "N=%lld out of range (< 2^23)", (long long)N);
    REQUIRE(ldx >= K && ldy >= N && ldo >= N, FNI8_ERR_STRIDE,
            "ldx=%lld < K=%lld, or ldy=%lld or ldo=%lld < N=%lld", (long long)ldx, (long long)K,
            (long long)ldy, (long long)ldo, (long long)N);
    REQUIRE(out != y || ldo == ldy, FNI8_ERR_STRIDE, "out is y, with ldo=%lld and ldy=%lld",
            (long long)ldo, (long long)ldy);
    REQUIRE(aligned(x, 2) && aligned(y, 2) && aligned(out, 2) && aligned(a, 16) &&
                aligned(b, 16) && aligned(scaling, 4) && aligned(seg_off, 4) && aligned(rows, 4) &&
                aligned(ranks, 4),
            FNI8_ERR_ALIGN, "a and b must be 16-byte aligned, the others element-aligned");
    REQUIRE(out == y || !rows_meet(y, 2 * ldy, out, 2 * ldo, T, 2 * N), FNI8_ERR_STRIDE,
            "out overlaps y without being y");
    const int64_t need = fni8h::lora_workspace_bytes(T, K, S, parts * rank);
    REQUIRE(!need || (workspace && aligned(workspace, 256)), FNI8_ERR_ALIGN,
            "a 256-byte aligned workspace is required");
    REQUIRE(workspace_bytes >= need, FNI8_ERR_SHAPE, "workspace of %lld bytes, %lld needed",
            (long long)workspace_bytes, (long long)need);
    int rc = check_device();
    if (rc) return rc;
    fni8h::LoraAdd l{};
    l.x = (const uint16_t*)x; l.ldx = ldx; l.T = T; l.K = K;
    l.a = (const uint16_t*)a; l.b = (const uint16_t*)b; l.S = S; l.rank = rank;
    l.splits = splits; l.parts = parts; l.scaling = scaling; l.seg_off = seg_off; l.rows = rows;
    l.ranks = ranks;
    l.y = (const uint16_t*)y; l.ldy = ldy; l.out = (uint16_t*)out; l.ldo = ldo;
    l.work = static_cast<float*>(workspace);
    return fni8h::launch_lora_add(l, (hipStream_t)stream);
}

int64_t fni8_lora_workspace_bytes(int64_t T, int64_t K, int64_t S, int64_t all_rank) {
    return lora_in_range(T, K, S, all_rank) ? fni8h::lora_workspace_bytes(T, K, S, all_rank) : 0;
}

int fni8_sample(const void* logits, int fp32, int64_t B, int64_t V, int64_t ldl, const float* u,
                const float* temperature, float temperature_all, const int32_t* top_k,
                int64_t top_k_all, const float* top_p, float top_p_all, const float* min_p,
                float min_p_all, int64_t* tokens, float* logprobs, void* workspace,
                int64_t workspace_bytes, void* stream) {
    fni8h::g_detail[0] = 0;
    REQUIRE(logits && tokens, FNI8_ERR_NULL, "logits and tokens are required");
    REQUIRE(sample_in_range(B, V), FNI8_ERR_SHAPE,
            "B=%lld V=%lld out of range (B <= 2^20, 1 <= V <= 2^22)", (long long)B, (long long)V);
    REQUIRE(ldl >= V, FNI8_ERR_STRIDE, "ldl=%lld < V=%lld", (long long)ldl, (long long)V);
    REQUIRE(aligned(logits, fp32 ? 4 : 2) && aligned(u, 4) && aligned(temperature, 4) &&
                aligned(top_k, 4) && aligned(top_p, 4) && aligned(min_p, 4) &&
                aligned(tokens, 8) && aligned(logprobs, 4),
            FNI8_ERR_ALIGN, "a tensor is not aligned to its elements");
    const int64_t need = fni8h::sample_workspace_bytes(B, V);
    REQUIRE(!need || (workspace && aligned(workspace, 256)), FNI8_ERR_ALIGN,
            "a 256-byte aligned workspace is required");
    REQUIRE(workspace_bytes >= need, FNI8_ERR_SHAPE, "workspace of %lld bytes, %lld needed",
            (long long)workspace_bytes, (long long)need);
    int rc = check_device();
    if (rc) return rc;
    fni8h::Sample a{};
    a.logits = logits; a.fp32 = fp32 != 0; a.B = B; a.V = V; a.ld = ldl; a.u = u;
    a.temperature = temperature; a.temperature1 = temperature_all;
    a.top_k = top_k;
    a.top_k1 = (int32_t)(top_k_all < 0 ? 0 : top_k_all > V ? 0 : top_k_all);
    a.top_p = top_p; a.top_p1 = top_p_all; a.min_p = min_p; a.min_p1 = min_p_all;
    a.tokens = tokens; a.logprobs = logprobs;
    a.work = static_cast<int8_t*>(workspace);
    return fni8h::launch_sample(a, (hipStream_t)stream);
}

int64_t fni8_sample_workspace_bytes(int64_t B, int64_t V) {
    return sample_in_range(B, V) ? fni8h::sample_workspace_bytes(B, V) : 0;
}

}  // extern "C"
