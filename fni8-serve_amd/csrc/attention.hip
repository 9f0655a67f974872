// Attention of new tokens over the paged cache (gfx950).
//
// Query token i of the n new ones of a sequence of L tokens (the new ones among them)
// stands at p = L - n + i and sees the keys j, 0 <= j <= p, j > p - window:
//   out = sum_j softmax_j(scale * q . k_j) v_j
// with an online softmax: running maximum m, sum l and unnormalised output o in fp32.  A
// row that sees no key (p < 0, or no tokens) is 0.
//
// The simple form: one wave a (token, query head), a lane holds 4 elements of the head,
// keys one after another.
#include "common.h"

namespace {

using fni8::f2h;
using fni8::h2f;
using fni8h::PagedAttention;

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

__device__ __forceinline__ int seq_start(const PagedAttention& a, int64_t s) {
    if (s > a.B) return (int)a.T;
    int c = a.cu_seqlens ? a.cu_seqlens[s] : (int)s;
    c = c < 0 ? 0 : c;
    return c > a.T ? (int)a.T : c;
}

__global__ __launch_bounds__(64) void simple_kernel(PagedAttention a) {
    const int64_t t = blockIdx.x;
    const int head = blockIdx.y, lane = threadIdx.x;
    const int group = (int)(a.Hq / a.Hk), h = head / group;
    const int plog = __builtin_ctzll((uint64_t)a.page_size);
    float q[4] = {}, o[4] = {}, m = -__builtin_inff(), l = 0.0f;
    const bool mine = lane * 4 < a.D;
    if (mine)
        for (int i = 0; i < 4; i++) q[i] = h2f(a.q[t * a.ldq + head * a.hsq + lane * 4 + i]);
    int64_t s = 0;
    while (s < a.B && seq_start(a, s + 1) <= t) s++;
    if (s < a.B && t >= seq_start(a, s)) {
        const int64_t n = seq_start(a, s + 1) - seq_start(a, s), L0 = a.context_lens[s],
                      W = a.max_pages << plog, L = L0 > W + 1 ? W + 1 : L0;
        const int64_t p = L - n + (t - seq_start(a, s));
        int64_t j = a.window && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
        for (; j <= p; j++) {
            const int64_t col = j >> plog;
            int64_t page = col < a.max_pages ? a.block_tables[s * a.ldt + col] : -1;
            const bool bad = page < 0 || page >= a.num_pages;
            const int64_t at = (((bad ? 0 : page) * a.Hk + h) << plog) + (j & (a.page_size - 1));
            float dot = 0.0f, v[4] = {};
            if (mine && !bad)
                for (int i = 0; i < 4; i++) {
                    const int64_t e = at * a.D + lane * 4 + i;
                    if (a.k_scale) {
                        dot += q[i] * ((float)static_cast<const int8_t*>(a.k_cache)[e] * a.k_scale[at]);
                        v[i] = (float)static_cast<const int8_t*>(a.v_cache)[e] * a.v_scale[at];
                    } else {
                        dot += q[i] * h2f(static_cast<const uint16_t*>(a.k_cache)[e]);
                        v[i] = h2f(static_cast<const uint16_t*>(a.v_cache)[e]);
                    }
                }
            const float z = bad ? __builtin_nanf("") : wave_sum(dot) * a.scale;
            const float top = z > m || z != z ? z : m;
            const float w = __builtin_expf(z - top), keep = m == top ? 1.0f : __builtin_expf(m - top);
            l = l * keep + w;
            for (int i = 0; i < 4; i++) o[i] = o[i] * keep + w * v[i];
            m = top;
        }
    }
    if (mine)
        for (int i = 0; i < 4; i++)
            a.out[(t * a.Hq + head) * a.D + lane * 4 + i] = f2h(l == 0.0f ? 0.0f : o[i] / l);
}

}  // namespace

namespace fni8h {

int64_t paged_attention_workspace_bytes(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t,
                                        int64_t) {
    return 0;
}

int launch_paged_attention(const PagedAttention& a, hipStream_t st) {
    if (a.T == 0) return FNI8_OK;
    simple_kernel<<<dim3((uint32_t)a.T, (uint32_t)a.Hq), 64, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        set_error_detail("paged_attention launch: %s", hipGetErrorString(e));
        return FNI8_ERR_LAUNCH;
    }
    return FNI8_OK;
}

}  // namespace fni8h
