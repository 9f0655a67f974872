// Low-rank adapters of many requests beside one projection (gfx950):
//
//   out[t, n] = fp16(y[t, n] + s_e * sum_j B_e[n, j] h[t, p(n) r + j]),   h[t] = A_e x[t]
//
// e is token t's adapter, p(n) the part of a merged projection (Q, K, V; gate, up) that column
// n belongs to.  Tokens come sorted by adapter (seg_off, rows); a tile is a run of one
// adapter's tokens.  Two launches:
//
//   shrink  h = A x, a tile's tokens by a group of 16-row blocks of A by a part of K.  Waves
//           split the part and add up in LDS; the parts' sums go to the workspace in fp32.
//   expand  adds the parts, then B h on the matrix cores, 16 tokens by a strip of columns a
//           wave, and y in the same pass.
//
// h enters the second product as two fp16 numbers, h * 2^k = hi + lo with one k a token that
// brings the largest |h| to 2^8: the pair keeps 2^-22 of the largest h, so nothing overflows or
// is rounded on the way but in fp32, and out is rounded once.
#include "common.h"

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kWaves = 4;

struct Args {
    const uint16_t *x, *y, *a, *b;
    uint16_t* out;
    int64_t ldx, ldy, ldo;
    const float* scaling;
    const int32_t *seg_off, *rows;
    float* h;            // [kparts][T][R]
    int T, K, S, rank, R, kparts;
    int copy;            // out is not y: tokens without an adapter are copied
    int parts, cols;     // parts of the projection; columns of a workgroup
    int start[FNI8_LORA_MAX_PARTS + 1];  // first column of each part
};

// 8 fp16 at p, of which `n` are there (the others 0); WIDE: all of them or none, aligned.
template <bool WIDE>
__device__ __forceinline__ h8 load8(const uint16_t* p, int64_t n) {
    h8 v = {0, 0, 0, 0, 0, 0, 0, 0};
    if constexpr (WIDE) {
        if (n > 0) v = *reinterpret_cast<const h8*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            v[i] = i < n ? __builtin_bit_cast(_Float16, p[i]) : (_Float16)0.0f;
    }
    return v;
}

template <int JT, int NT, bool WIDE>
__global__ __launch_bounds__(kThreads) void shrink_kernel(const Args a) {
    __shared__ f32x4 red[kWaves][JT * NT][64];
    int e, r0, r1;
    if (!fni8::find_group_tile(a.seg_off, a.S, 16 * NT, blockIdx.x, a.T, e, r0, r1)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int j0 = blockIdx.y * 16 * JT, count = r1 - r0;

    const uint16_t *xr[NT], *ar[JT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int i = t * 16 + (lane & 15);
        int row = a.rows[r0 + (i < count ? i : count - 1)];
        row = row < 0 ? 0 : row < a.T ? row : a.T - 1;
        xr[t] = a.x + (int64_t)row * a.ldx;
    }
#pragma unroll
    for (int j = 0; j < JT; j++) {
        const int i = j0 + j * 16 + (lane & 15);
        ar[j] = a.a + ((int64_t)e * a.R + (i < a.R ? i : a.R - 1)) * a.K;
    }
    f32x4 acc[JT][NT];
#pragma unroll
    for (int j = 0; j < JT; j++)
#pragma unroll
        for (int t = 0; t < NT; t++) acc[j][t] = f32x4{0, 0, 0, 0};

    // steps of 32 elements of K, a run of them for each wave of each part
    const int steps = (a.K + 31) / 32, ways = a.kparts * kWaves;
    const int per = (steps + ways - 1) / ways;
    const int s0 = (blockIdx.z * kWaves + wave) * per;
    const int s1 = s0 + per < steps ? s0 + per : steps;
#pragma unroll WIDE ? 2 : 1
    for (int s = s0; s < s1; s++) {
        const int k = s * 32 + 8 * (lane >> 4);
        h8 xf[NT], af[JT];
#pragma unroll
        for (int t = 0; t < NT; t++) xf[t] = load8<WIDE>(xr[t] + k, a.K - k);
#pragma unroll
        for (int j = 0; j < JT; j++) af[j] = load8<WIDE>(ar[j] + k, a.K - k);
#pragma unroll
        for (int j = 0; j < JT; j++)
#pragma unroll
            for (int t = 0; t < NT; t++)
                acc[j][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(af[j], xf[t], acc[j][t], 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < JT; j++)
#pragma unroll
        for (int t = 0; t < NT; t++) red[wave][j * NT + t][lane] = acc[j][t];
    __syncthreads();
    for (int i = threadIdx.x; i < JT * NT * 64; i += kThreads) {
        const int tile = i >> 6, l = i & 63, t = (tile % NT) * 16 + (l & 15);
        const int j = j0 + (tile / NT) * 16 + 4 * (l >> 4);
        f32x4 v = red[0][tile][l];
#pragma unroll
        for (int w = 1; w < kWaves; w++) v += red[w][tile][l];
        if (t < count && j < a.R)
            *reinterpret_cast<f32x4*>(a.h + ((int64_t)blockIdx.z * a.T + r0 + t) * a.R + j) = v;
    }
}

// KS: 32-element steps of the rank.  A strip is 16 * QT columns; lane (t, g) of a wave ends up
// with the 4 * QT consecutive columns 4 * QT * g .. of token t, one to two 16-byte accesses.
template <int KS, int NT>
__global__ __launch_bounds__(kThreads) void expand_kernel(const Args a) {
    constexpr int TM = 16 * NT, QT = KS <= 4 ? 4 : 2, UNITS = (TM * KS * 4 + kThreads - 1) / kThreads;
    __shared__ h8 hs[NT * KS * 2][64];
    __shared__ uint32_t top[TM];
    __shared__ float back[TM];
    __shared__ int token[TM];
    int e, r0, r1;
    if (!fni8::find_group_tile(a.seg_off, a.S + 1, TM, blockIdx.x, a.T, e, r0, r1)) return;
    const bool bare = e == a.S;
    if (bare && !a.copy) return;
    const int count = r1 - r0, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // the part that this workgroup's columns are of
    int part = 0, n0 = 0, block = blockIdx.y;
    for (; part < a.parts; part++) {
        const int width = a.start[part + 1] - a.start[part], blocks = (width + a.cols - 1) / a.cols;
        if (block < blocks) break;
        block -= blocks;
    }
    if (part == a.parts) return;
    n0 = a.start[part] + block * a.cols;
    const int end = a.start[part + 1];
    const int n1 = n0 + a.cols < end ? n0 + a.cols : end;

    for (int t = threadIdx.x; t < TM; t += kThreads) {
        const int row = t < count ? a.rows[r0 + t] : -1;
        token[t] = row < a.T ? row : -1;
        top[t] = 0;
    }
    __syncthreads();
    if (bare) {
        for (int t = wave; t < count; t += kWaves) {
            if (token[t] < 0) continue;
            const uint16_t* y = a.y + (int64_t)token[t] * a.ldy;
            uint16_t* o = a.out + (int64_t)token[t] * a.ldo;
            for (int n = n0 + lane; n < n1; n += 64) o[n] = y[n];
        }
        return;
    }
    float v[UNITS][8];
#pragma unroll
    for (int i = 0; i < UNITS; i++) {
        const int u = threadIdx.x + i * kThreads, t = u / (KS * 4), g = u % (KS * 4);
#pragma unroll
        for (int j = 0; j < 8; j++) v[i][j] = 0.0f;
        if (t >= count || g * 8 >= a.rank) continue;
        const float* h = a.h + (int64_t)(r0 + t) * a.R + part * a.rank + g * 8;
        for (int p = 0; p < a.kparts; p++, h += (int64_t)a.T * a.R) {
            const f32x4 lo = *reinterpret_cast<const f32x4*>(h);
            const f32x4 hi = *reinterpret_cast<const f32x4*>(h + 4);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[i][j] += lo[j];
                v[i][j + 4] += hi[j];
            }
        }
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t w = __builtin_bit_cast(uint32_t, v[i][j]) & 0x7fffffffu;
            m = w > m ? w : m;
        }
        atomicMax(&top[t], m);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < UNITS; i++) {
        const int u = threadIdx.x + i * kThreads, t = u / (KS * 4), g = u % (KS * 4);
        if (t >= TM) continue;
        const uint32_t m = top[t];
        const bool finite = m < 0x7f800000u;
        int up = 135 - (int)(m >> 23);  // brings the largest to 2^8
        up = !finite || m == 0 ? 0 : up > 120 ? 120 : up;
        h8 hi, lo;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float w = __builtin_ldexpf(v[i][j], up);
            hi[j] = (_Float16)w;
            lo[j] = finite ? (_Float16)(w - (float)hi[j]) : (_Float16)0.0f;
        }
        const int at = ((t >> 4) * KS + (g >> 2)) * 2, l = (t & 15) + 16 * (g & 3);
        hs[at][l] = hi;
        hs[at + 1][l] = lo;
        if (g == 0) back[t] = __builtin_ldexpf(1.0f, -up);
    }
    __syncthreads();

    const float scale = a.scaling ? a.scaling[e] : 1.0f;
    const int g = lane >> 4;
    const bool wide = (a.ldy | a.ldo | n0) % 8 == 0 &&
                      (((uintptr_t)a.y | (uintptr_t)a.out) & 15) == 0;
    for (int n = n0 + wave * 16 * QT; n < n1; n += kWaves * 16 * QT) {
        h8 bf[QT][KS];
        const int i = lane & 15;
#pragma unroll
        for (int q = 0; q < QT; q++) {
            // row i of the q-th product: the column that brings lane (t, g) its runs
            int c = n + 4 * QT * (i >> 2) + 4 * q + (i & 3);
            c = c < n1 ? c : n1 - 1;
            const uint16_t* b = a.b + ((int64_t)e * a.start[a.parts] + c) * a.rank;
#pragma unroll
            for (int s = 0; s < KS; s++) bf[q][s] = load8<true>(b + s * 32 + 8 * g, a.rank - s * 32 - 8 * g);
        }
        const int c0 = n + 4 * QT * g;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if (t * 16 >= count) break;
            const int row = token[t * 16 + i];
            const bool live = row >= 0;
            const uint16_t* y = a.y + (int64_t)(live ? row : 0) * a.ldy + c0;
            uint16_t* o = a.out + (int64_t)(live ? row : 0) * a.ldo + c0;
            const bool whole = wide && n + 16 * QT <= n1;
            h8 in[QT / 2];
#pragma unroll
            for (int q = 0; q < QT / 2; q++)
                in[q] = whole ? load8<true>(y + 8 * q, live ? 8 : 0)
                              : load8<false>(y + 8 * q, live ? n1 - c0 - 8 * q : 0);
            f32x4 acc[QT];
#pragma unroll
            for (int q = 0; q < QT; q++) acc[q] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const h8 hi = hs[(t * KS + s) * 2][lane], lo = hs[(t * KS + s) * 2 + 1][lane];
#pragma unroll
                for (int q = 0; q < QT; q++) {
                    acc[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bf[q][s], lo, acc[q], 0, 0, 0);
                    acc[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bf[q][s], hi, acc[q], 0, 0, 0);
                }
            }
            const float down = back[t * 16 + i];
#pragma unroll
            for (int q = 0; q < QT; q++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float d = acc[q][r] * down * scale;
                    const int z = (q & 1) * 4 + r;
                    in[q >> 1][z] = __builtin_bit_cast(_Float16, fni8::f2h((float)in[q >> 1][z] + d));
                }
            if (!live) continue;
#pragma unroll
            for (int q = 0; q < QT / 2; q++) {
                if (whole) {
                    *reinterpret_cast<h8*>(o + 8 * q) = in[q];
                } else {
#pragma unroll
                    for (int r = 0; r < 8; r++) {
                        const _Float16 z = in[q][r];  // an element is no lvalue to bit_cast
                        if (c0 + 8 * q + r < n1) o[8 * q + r] = __builtin_bit_cast(uint16_t, z);
                    }
                }
            }
        }
    }
}

// Tiles of 16 tokens, or of 64 where an adapter has that many on average.
bool big_tiles(int64_t T, int64_t S) { return T >= 64 * (S < 16 ? S : 16) && T >= 256; }

int64_t tiles_of(int64_t T, int64_t groups, int64_t bm) {
    return T / bm + (groups < T ? groups : T);
}

struct Plan {
    bool big;
    int jt;
    int64_t jgroups, tiles, kparts;
};
Plan plan_of(int64_t T, int64_t K, int64_t S, int64_t R) {
    Plan p{};
    p.big = big_tiles(T, S);
    p.jt = R <= 16 ? 1 : R <= 32 ? 2 : 3;
    p.jgroups = (R + 16 * p.jt - 1) / (16 * p.jt);
    p.tiles = tiles_of(T, S, p.big ? 64 : 16);
    // enough workgroups for two on each CU, no wave with less than two steps of K
    const int64_t want = 512 / (p.tiles * p.jgroups) + 1, most = (K + 255) / 256;
    p.kparts = want < most ? want : most;
    if (p.kparts > 16) p.kparts = 16;
    return p;
}

template <int NT, bool WIDE>
void shrink(const Args& a, const Plan& p, hipStream_t st) {
    const dim3 grid((uint32_t)p.tiles, (uint32_t)p.jgroups, (uint32_t)p.kparts);
    if (p.jt == 1) shrink_kernel<1, NT, WIDE><<<grid, kThreads, 0, st>>>(a);
    else if (p.jt == 2) shrink_kernel<2, NT, WIDE><<<grid, kThreads, 0, st>>>(a);
    else shrink_kernel<3, NT, WIDE><<<grid, kThreads, 0, st>>>(a);
}

template <int NT>
void expand(const Args& a, dim3 grid, hipStream_t st) {
    if (a.rank <= 32) expand_kernel<1, NT><<<grid, kThreads, 0, st>>>(a);
    else if (a.rank <= 64) expand_kernel<2, NT><<<grid, kThreads, 0, st>>>(a);
    else if (a.rank <= 128) expand_kernel<4, NT><<<grid, kThreads, 0, st>>>(a);
    else expand_kernel<8, NT < 2 ? NT : 2><<<grid, kThreads, 0, st>>>(a);
}

}  // namespace

namespace fni8h {

int64_t lora_workspace_bytes(int64_t T, int64_t K, int64_t S, int64_t R) {
    return T ? plan_of(T, K, S, R).kparts * T * R * 4 : 0;
}

int launch_lora_add(const LoraAdd& l, hipStream_t st) {
    if (l.T == 0) return FNI8_OK;
    const int64_t R = l.parts * l.rank;
    const Plan p = plan_of(l.T, l.K, l.S, R);
    Args a{};
    a.x = l.x; a.ldx = l.ldx; a.y = l.y; a.ldy = l.ldy; a.out = l.out; a.ldo = l.ldo;
    a.a = l.a; a.b = l.b; a.scaling = l.scaling; a.seg_off = l.seg_off; a.rows = l.rows;
    a.h = l.work;
    a.T = (int)l.T; a.K = (int)l.K; a.S = (int)l.S; a.rank = (int)l.rank; a.R = (int)R;
    a.kparts = (int)p.kparts;
    a.copy = l.out != l.y;
    a.parts = (int)l.parts;
    for (int i = 0; i < l.parts; i++) a.start[i + 1] = a.start[i] + (int)l.splits[i];

    const bool wide = l.K % 8 == 0 && l.ldx % 8 == 0 && (((uintptr_t)l.x | (uintptr_t)l.a) & 15) == 0;
    if (p.big) wide ? shrink<4, true>(a, p, st) : shrink<4, false>(a, p, st);
    else wide ? shrink<1, true>(a, p, st) : shrink<1, false>(a, p, st);

    const int nt = !p.big ? 1 : l.rank > 128 ? 2 : 4;
    const int64_t tiles = tiles_of(l.T, l.S + 1, 16 * nt);
    // columns of a workgroup: four waves' strips, more where that leaves plenty of workgroups
    const int64_t N = a.start[l.parts];
    int64_t cols = 256;
    while (cols < 1024 && tiles * (N / (2 * cols)) >= 1024) cols *= 2;
    a.cols = (int)cols;
    int64_t blocks = 0;
    for (int i = 0; i < l.parts; i++) blocks += (l.splits[i] + cols - 1) / cols;
    const dim3 grid((uint32_t)tiles, (uint32_t)blocks);
    if (p.big) expand<4>(a, grid, st);
    else expand<1>(a, grid, st);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) {
        set_error_detail("lora launch: %s", hipGetErrorString(err));
        return FNI8_ERR_LAUNCH;
    }
    return FNI8_OK;
}

}  // namespace fni8h
