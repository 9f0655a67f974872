// The rows between the QKV projection and attention (gfx950): an RMS norm of every query
// and key head, rotary positions, and the append of keys and values to the paged cache,
// in one pass over the rows.
//
// A row is one head of one token, D elements x.  With n = x, or
// n = x * (1 / sqrt(sum(x^2) / D + eps)) * w with a weight (w = weight, or 1 + weight),
// and the token's table row cos[0..R/2), sin[0..R/2):
//   halves (a, b) = (n[i], n[i + R/2]), pairs (a, b) = (n[2i], n[2i + 1]),  i < R/2
//   (a, b) <- (a cos[i] - b sin[i], b cos[i] + a sin[i]);  n[R..D) stays.
// All of it in fp32 from the fp16 input to one rounding to fp16: the normed row is not
// rounded in between.  A position outside the table gives NaN in the rotated elements.
// A key or value row goes to its token's slot of the cache as it is (fp16), or in the
// per-token quantization of the linears (common.h), one scale a row.  A slot outside the
// cache (negative: padding) drops the row.
//
// Memory bounds it: 4 bytes an element (fp16 in and out), R * 4 a token for its table
// row.  The vector instructions come next, so a row has one form whatever its pairs, its
// weight and its R: (x c w + x' s w') m with the other element x' of the pair, c = 1 and
// s = -0 where nothing turns (x + 0 * -0 is x, its sign included), and w = m = 1 without a
// weight.  A row is held by LPR = 8, 16 or 32 lanes of 8 elements (16-byte accesses).  The
// other half of a rotated pair is read a second time from the input (the L1 has it)
// rather than exchanged between lanes: both loads are in flight together, and any R that
// is a multiple of 16 works the same way.
#include "common.h"

namespace {

using fni8::f2h;
using fni8::h2f;

struct RowArgs {
    const uint16_t *q, *k, *v;
    int64_t ldq, ldk, ldv;
    uint32_t hsq, hsk, hsv;
    int Hq, Hk, Hv, D, R, pairs, unit;
    const uint16_t *qw, *kw;
    float eps, inv_d;
    const int32_t* pos;
    const float* table;
    int64_t P;
    uint16_t *q_out, *k_out;
    // append: caches of `slots_n` slots in pages of 1 << page_log2; NULL slot = no cache
    const int32_t* slot;
    int64_t slots_n;
    int page_log2;
    void *kc, *vc;
    float *ks, *vs;
};

// Sum over the LPR lanes of a row, in every one of them.
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
    auto add = [](float a, int b) { return a + __builtin_bit_cast(float, b); };
    v = add(v, fni8::dpp<fni8::kDppXor1>(__builtin_bit_cast(int, v)));
    v = add(v, fni8::dpp<fni8::kDppXor2>(__builtin_bit_cast(int, v)));
    v = add(v, fni8::dpp<fni8::kDppHalfMirror>(__builtin_bit_cast(int, v)));
    if (LPR >= 16) v = add(v, fni8::dpp<fni8::kDppMirror>(__builtin_bit_cast(int, v)));
    if (LPR >= 32) v += __shfl_xor(v, 16, 64);
    return v;
}

template <int LPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    auto up = [](uint32_t a, int b) { return a > (uint32_t)b ? a : (uint32_t)b; };
    v = up(v, fni8::dpp<fni8::kDppXor1>((int)v));
    v = up(v, fni8::dpp<fni8::kDppXor2>((int)v));
    v = up(v, fni8::dpp<fni8::kDppHalfMirror>((int)v));
    if (LPR >= 16) v = up(v, fni8::dpp<fni8::kDppMirror>((int)v));
    if (LPR >= 32) v = up(v, __shfl_xor((int)v, 16, 64));
    return v;
}

__device__ __forceinline__ float half_of(uint4 v, int i) {
    const uint32_t w = (i >> 1) == 0 ? v.x : (i >> 1) == 1 ? v.y : (i >> 1) == 2 ? v.z : v.w;
    return h2f((uint16_t)(i & 1 ? w >> 16 : w & 0xffffu));
}

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h2));  // to nearest even
}

// The other elements of the pairs of the 8 elements from e on, `self`, of the row at src; 0
// where nothing turns.
template <bool ALIGNED>
__device__ __forceinline__ uint4 others(const uint16_t* src, uint4 self, int e, int R, int pairs) {
    const int half = R >> 1;
    auto turned = [](uint32_t w) { return w >> 16 | w << 16; };
    uint4 o = make_uint4(0, 0, 0, 0);
    if (ALIGNED) {
        if (e >= R) return o;
        if (pairs)
            return make_uint4(turned(self.x), turned(self.y), turned(self.z), turned(self.w));
        return *reinterpret_cast<const uint4*>(src + (e < half ? e + half : e - half));
    }
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        h[i] = 0;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int d = e + 2 * i + k;
            if (d >= R) continue;
            const int at = pairs ? d ^ 1 : d < half ? d + half : d - half;
            h[i] |= (uint32_t)src[at] << 16 * k;
        }
    }
    return make_uint4(h[0], h[1], h[2], h[3]);
}

// A block takes NR rows per group of LPR lanes of one token (blockIdx.x): rows 0..Hq are
// query heads, then key heads, then value heads.  ALIGNED: every chunk of 8 elements is
// rotated as a whole or not at all and its table entries are 16-byte aligned (R a multiple
// of 16 for halves, of 8 for pairs); otherwise element by element.
// NORM: some row has a weight.
template <int LPR, int NR, bool ALIGNED, bool NORM>
__global__ __launch_bounds__(256) void row_kernel(RowArgs a) {
    constexpr int GROUPS = 256 / LPR;
    const int64_t t = blockIdx.x;
    const int lane = threadIdx.x & (LPR - 1), group = threadIdx.x / LPR;
    const int e = lane * 8;
    const bool mine = e < a.D;
    const int rows = a.Hq + a.Hk + a.Hv;
    const int row0 = blockIdx.y * (GROUPS * NR) + group;

    // the lane's 8 elements of the token's angles, the same for every head
    float c[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        c[i] = 1.0f;
        s[i] = -0.0f;
    }
    int64_t p = 0;
    bool outside = false;
    if (a.R) {
        p = a.pos[t];
        outside = p < 0 || p >= a.P;
        if (outside) p = 0;
    }
    const int half = a.R >> 1;
    const float* row = a.table + p * a.R;
    if (ALIGNED) {
        if (e < a.R) {
            if (a.pairs) {
                const float4 c4 = *reinterpret_cast<const float4*>(row + e / 2);
                const float4 s4 = *reinterpret_cast<const float4*>(row + half + e / 2);
                const float cc[4] = {c4.x, c4.y, c4.z, c4.w}, ss[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    c[i] = cc[i / 2];
                    s[i] = i & 1 ? ss[i / 2] : -ss[i / 2];
                }
            } else {
                const float* at = row + (e < half ? e : e - half);
                const float4 c0 = *reinterpret_cast<const float4*>(at);
                const float4 c1 = *reinterpret_cast<const float4*>(at + 4);
                const float4 s0 = *reinterpret_cast<const float4*>(at + half);
                const float4 s1 = *reinterpret_cast<const float4*>(at + half + 4);
                const float cc[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
                const float ss[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    c[i] = cc[i];
                    s[i] = e < half ? -ss[i] : ss[i];
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int d = e + i;
            if (d < a.R) {
                const int n = a.pairs ? d >> 1 : d < half ? d : d - half;
                const float sn = row[half + n];
                c[i] = row[n];
                s[i] = (a.pairs ? d & 1 : d >= half) ? sn : -sn;
            }
        }
    }
    if (outside)
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (e + i < a.R) c[i] = s[i] = __builtin_nanf("");

    const uint16_t *q = a.q + t * a.ldq, *k = a.k + t * a.ldk, *v = a.v + t * a.ldv;
    uint4 x[NR], o[NR];
#pragma unroll
    for (int j = 0; j < NR; j++) {
        const int r = row0 + j * GROUPS;
        x[j] = o[j] = make_uint4(0, 0, 0, 0);
        if (r >= rows || !mine) continue;
        const bool is_q = r < a.Hq, turns = r < a.Hq + a.Hk;
        const uint32_t h = is_q ? r : turns ? r - a.Hq : r - a.Hq - a.Hk;
        const uint32_t hs = is_q ? a.hsq : turns ? a.hsk : a.hsv;
        const uint16_t* src = (is_q ? q : turns ? k : v) + (uint64_t)h * hs;
        x[j] = *reinterpret_cast<const uint4*>(src + e);
        if (turns) o[j] = others<ALIGNED>(src, x[j], e, a.R, a.pairs);
    }
    int64_t slot = -1;
    if (a.slot) {
        slot = a.slot[t];
        if (slot >= a.slots_n) slot = -1;
    }

#pragma unroll
    for (int j = 0; j < NR; j++) {
        const int r = row0 + j * GROUPS;
        const bool is_q = r < a.Hq, is_k = !is_q && r < a.Hq + a.Hk;
        if (r >= rows) continue;
        uint4 y = x[j];
        if (is_q || is_k) {
            float f[8], g[8], z[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                f[i] = half_of(x[j], i);
                g[i] = half_of(o[j], i);
            }
            if (NORM) {
                const uint16_t* w = is_q ? a.qw : a.kw;
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) ss = __builtin_fmaf(f[i], f[i], ss);
                const float m = __builtin_amdgcn_rsqf(__builtin_fmaf(row_sum<LPR>(ss), a.inv_d, a.eps));
                const uint32_t one = a.unit ? 0 : 0x3c003c00u;
                uint4 w4 = make_uint4(one, one, one, one), o4 = w4;
                if (w && mine) {
                    w4 = *reinterpret_cast<const uint4*>(w + e);
                    o4 = others<ALIGNED>(w, w4, e, a.R, a.pairs);
                }
                const float scale = w ? m : 1.0f, unit = a.unit ? 1.0f : 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float wc = (unit + half_of(w4, i)) * c[i], ws = (unit + half_of(o4, i)) * s[i];
                    z[i] = __builtin_fmaf(f[i], wc, g[i] * ws) * scale;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) z[i] = __builtin_fmaf(f[i], c[i], g[i] * s[i]);
            }
            y = make_uint4(pack2(z[0], z[1]), pack2(z[2], z[3]), pack2(z[4], z[5]),
                           pack2(z[6], z[7]));
        }
        if (is_q || (is_k && !a.slot)) {
            uint16_t* dst = is_q ? a.q_out + (t * a.Hq + r) * a.D
                                 : a.k_out + (t * a.Hk + r - a.Hq) * a.D;
            if (mine) *reinterpret_cast<uint4*>(dst + e) = y;
            continue;
        }
        if (slot < 0) continue;
        const int h = is_k ? r - a.Hq : r - a.Hq - a.Hk;
        const int64_t page = slot >> a.page_log2, in = slot & ((1 << a.page_log2) - 1);
        const int64_t at = ((page * a.Hk + h) << a.page_log2) + in;
        void* cache = is_k ? a.kc : a.vc;
        float* scale = is_k ? a.ks : a.vs;
        if (!scale) {
            if (mine) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(cache) + at * a.D + e) = y;
            continue;
        }
        const uint32_t top = row_max<LPR>(fni8::amax_fold(mine ? fni8::amax_chunk(0, y) : 0));
        const float step = fni8::row_scale_from_bits(top);
        // a row with an infinity or NaN: codes 0 under a scale that is not finite
        const bool live = top < 0x7c00u;
        if (mine)
            *reinterpret_cast<uint2*>(static_cast<int8_t*>(cache) + at * a.D + e) =
                fni8::quant_chunk(y, step, 1.0f / step, live);
        if (lane == 0) scale[at] = step;
    }
}

template <int LPR, int NR>
void launch_rows(const RowArgs& a, int64_t T, bool aligned, hipStream_t st) {
    const int rows = a.Hq + a.Hk + a.Hv, per = 256 / LPR * NR;
    const dim3 grid((uint32_t)T, (uint32_t)((rows + per - 1) / per));
    const bool norm = a.qw || a.kw;
    const auto kernel = aligned ? norm ? row_kernel<LPR, NR, true, true> : row_kernel<LPR, NR, true, false>
                                : norm ? row_kernel<LPR, NR, false, true> : row_kernel<LPR, NR, false, false>;
    kernel<<<grid, 256, 0, st>>>(a);
}

}  // namespace

namespace fni8h {

int launch_qkv_rows(const QkvRows& r, hipStream_t st) {
    if (r.T == 0 || r.Hq + r.Hk == 0) return FNI8_OK;
    RowArgs a;
    a.q = r.q; a.ldq = r.ldq; a.hsq = (uint32_t)r.hsq; a.Hq = (int)r.Hq;
    a.k = r.k; a.ldk = r.ldk; a.hsk = (uint32_t)r.hsk; a.Hk = (int)r.Hk;
    a.v = r.v; a.ldv = r.ldv; a.hsv = (uint32_t)r.hsv; a.Hv = r.slots ? (int)r.Hk : 0;
    a.D = (int)r.D; a.R = (int)r.R; a.pairs = r.interleaved != 0; a.unit = r.unit_offset != 0;
    a.qw = r.q_weight; a.kw = r.k_weight; a.eps = r.eps; a.inv_d = 1.0f / (float)r.D;
    a.pos = r.positions; a.table = r.cos_sin; a.P = r.P;
    a.q_out = r.q_out; a.k_out = r.k_out;
    a.slot = r.slots; a.slots_n = r.num_pages * r.page_size;
    a.page_log2 = r.slots ? __builtin_ctzll((uint64_t)r.page_size) : 0;
    a.kc = r.k_cache; a.vc = r.v_cache; a.ks = r.k_scale; a.vs = r.v_scale;
    const bool aligned = a.R % (a.pairs ? 8 : 16) == 0;
    // three rows a lane group share the angles and keep more loads in flight: 40 rows of 128 a
    // token, one against three, take 5.3 and 5.5 us at 64 tokens, 7.3 and 6.9 at 1024, 11.0
    // and 9.7 at 2048, 18.0 and 16.9 at 4096, 35 and 28 (6.1 TB/s) at 8192
    const bool many = r.T * (a.Hq + a.Hk + a.Hv) >= 32768;
    if (r.D <= 64)
        many ? launch_rows<8, 3>(a, r.T, aligned, st) : launch_rows<8, 1>(a, r.T, aligned, st);
    else if (r.D <= 128)
        many ? launch_rows<16, 3>(a, r.T, aligned, st) : launch_rows<16, 1>(a, r.T, aligned, st);
    else
        many ? launch_rows<32, 3>(a, r.T, aligned, st) : launch_rows<32, 1>(a, r.T, aligned, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        set_error_detail("qkv rows launch: %s", hipGetErrorString(e));
        return FNI8_ERR_LAUNCH;
    }
    return FNI8_OK;
}

}  // namespace fni8h
