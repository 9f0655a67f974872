// Low-rank adapters of many requests beside one projection (gfx950):
//
//   out[t, n] = fp16(y[t, n] + s_e * sum_j B_e[n, j] h[t, p(n) r + j]),   h[t] = A_e x[t]
//
// e is token t's adapter, p(n) the part of a merged projection (Q, K, V; gate, up) that column
// n belongs to.  Tokens come sorted by adapter (seg_off, rows); a tile is a run of one
// adapter's tokens.  Two launches:
//
//   shrink  h = A x: 16 or 64 tokens by up to 96 rows of A; K split over the eight waves of a
//           tile of 16, and over workgroups where there are few tiles; fp32 sums to the workspace
//   expand  adds the parts, then B h on the matrix cores, 16 tokens by a strip of columns a
//           wave, and y in the same pass
//
// Both wait for memory only.  A call of few tokens is a chain of dependent loads (which tile,
// which rows, their data), so each wave finds its tile by itself, without a barrier, and
// everything that depends on the tile alone is on its way at once.
//
// h enters the second product as two fp16 numbers, h * 2^k = hi + lo with one k a token that
// brings the largest |h| to 2^8: the pair keeps 2^-22 of the largest h, so nothing overflows or
// is rounded on the way but in fp32, and out is rounded once.
#include "common.h"

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef h8 h8_anywhere __attribute__((aligned(2)));  // loads and stores are as wide at any address
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kShrinkWaves = 8;            // of a workgroup
constexpr int kThreads = 256, kWaves = 4;  // expand

struct Args {
    const uint16_t *x, *y, *a, *b;
    uint16_t* out;
    int64_t ldx, ldy, ldo;
    const float* scaling;
    const int32_t *seg_off, *rows, *ranks;
    float* h;            // [kparts][T][R]
    int T, K, S, rank, R, kparts;
    int copy;            // out is not y: tokens without an adapter are copied
    int parts, cols, blocks;  // parts of the projection; columns of a workgroup, their number
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

// Inclusive sum over the lanes, by data movement within the vector unit.
__device__ __forceinline__ int lane_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
    return v;
}

// Tile `slot` of the segments 0 .. E - 1, cut into tiles of BM tokens: its adapter and its tokens
// r0 .. r1, or false past the last.  Bounded by T whatever seg_off holds.  64 segments a step, each
// of which waits for the last: up to 64 adapters cost nothing, 512 three to four us a call, 4096
// 37, 65534 600 (one token, and 48).
template <int BM>
__device__ __forceinline__ bool find_tile(const Args& a, int E, int slot, int& e, int& r0, int& r1) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int c = 0; c < E; c += 64) {
        const int i = c + lane;
        const int lo = i < E ? a.seg_off[i] : 0, hi = i < E ? a.seg_off[i + 1] : 0;
        const int tiles = hi > lo ? (hi - lo + BM - 1) / BM : 0, end = base + lane_scan(tiles);
        const uint64_t who = __ballot(slot < end && slot >= end - tiles);
        if (who) {
            const int l = __builtin_ctzll(who);
            const int first = __builtin_amdgcn_readlane(end - tiles, l);
            const int from = __builtin_amdgcn_readlane(lo, l), to = __builtin_amdgcn_readlane(hi, l);
            e = c + l;
            r0 = from + (slot - first) * BM;
            r1 = r0 + BM < to ? r0 + BM : to;
            r1 = r1 < a.T ? r1 : a.T;
            return r0 >= 0 && r0 < r1;
        }
        base = __builtin_amdgcn_readlane(end, 63);
    }
    return false;
}

// The token at position r0 + i (i below count; else the last one's), -1 where rows holds none.
// `ahead` is lane l's rows[l], loaded with the segments: enough for 64 tokens.
__device__ __forceinline__ int token_at(const Args& a, int ahead, int r0, int i, int count) {
    const int p = r0 + (i < count ? i : count - 1);
    const int row = a.T <= 64 ? __shfl(ahead, p, 64) : a.rows[p];
    return (unsigned)row < (unsigned)a.T ? row : -1;
}
__device__ __forceinline__ int rows_ahead(const Args& a) {
    const int lane = threadIdx.x & 63;
    return a.rows[lane < a.T ? lane : a.T - 1];
}

// 16 tokens by 16 * JT rows of A, fragments straight from memory: each value is used once, and
// K is split over the waves, so that all of a tile's loads are on their way in a few steps of
// the matrix cores.  Bound by the latency of tile, rows, data, sums: 3.7 us for one token of
// K = 4096, 5.8 for 48 tokens with 48 adapters of 32 rows (12.6 MB of A), 7.0 where K = 12288.
template <int JT, bool WIDE>
__global__ __launch_bounds__(kShrinkWaves * 64) void shrink_kernel(const Args a) {
    constexpr int HALF = kShrinkWaves / 2;
    __shared__ f32x4 red[HALF][JT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ahead = rows_ahead(a);
    int e, r0, r1;
    if (!find_tile<16>(a, a.S, blockIdx.x, e, r0, r1)) return;
    const int j0 = blockIdx.y * 16 * JT, count = r1 - r0;

    const int row = token_at(a, ahead, r0, lane & 15, count);
    const uint16_t *xr = a.x + (int64_t)(row < 0 ? 0 : row) * a.ldx, *ar[JT];
#pragma unroll
    for (int j = 0; j < JT; j++) {
        const int i = j0 + j * 16 + (lane & 15);
        ar[j] = a.a + ((int64_t)e * a.R + (i < a.R ? i : a.R - 1)) * a.K;
    }
    f32x4 acc[JT];
#pragma unroll
    for (int j = 0; j < JT; j++) acc[j] = f32x4{0, 0, 0, 0};

    // steps of 32 elements of K, a run of them for each wave of each part
    const int steps = (a.K + 31) / 32, ways = a.kparts * kShrinkWaves;
    const int per = (steps + ways - 1) / ways;
    const int s0 = (blockIdx.z * kShrinkWaves + wave) * per;
    const int s1 = s0 + per < steps ? s0 + per : steps;
    constexpr int AHEAD = !WIDE ? 1 : JT > 4 ? 2 : 4;  // steps whose loads are on their way
    h8 xf[AHEAD], af[AHEAD][JT];
    auto fetch = [&](int s, h8& xs, h8 (&as)[JT]) {
        const h8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
        if (s >= s1) {
            xs = zero;
#pragma unroll
            for (int j = 0; j < JT; j++) as[j] = zero;
            return;
        }
        const int k = s * 32 + 8 * (lane >> 4);
        if (WIDE && s * 32 + 32 <= a.K) {
            xs = *reinterpret_cast<const h8*>(xr + k);
#pragma unroll
            for (int j = 0; j < JT; j++) as[j] = *reinterpret_cast<const h8*>(ar[j] + k);
        } else {
            xs = load8<WIDE>(xr + k, a.K - k);
#pragma unroll
            for (int j = 0; j < JT; j++) as[j] = load8<WIDE>(ar[j] + k, a.K - k);
        }
    };
#pragma unroll
    for (int i = 0; i < AHEAD; i++) fetch(s0 + i, xf[i], af[i]);
    for (int s = s0; s < s1; s += AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
#pragma unroll
            for (int j = 0; j < JT; j++)
                acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(af[i][j], xf[i], acc[j], 0, 0, 0);
            fetch(s + AHEAD + i, xf[i], af[i]);
        }
    }
    // half of the waves' sums go through LDS to the other half, then those by all threads
    auto keep = [&](int w) {
#pragma unroll
        for (int j = 0; j < JT; j++) red[w][j][lane] = acc[j];
    };
    if (wave >= HALF) keep(wave - HALF);
    __syncthreads();
    if (wave < HALF) {
#pragma unroll
        for (int j = 0; j < JT; j++) acc[j] += red[wave][j][lane];
        keep(wave);  // its own slots
    }
    __syncthreads();
    for (int i = threadIdx.x; i < JT * 64; i += kShrinkWaves * 64) {
        const int tile = i >> 6, l = i & 63, t = l & 15, j = j0 + tile * 16 + 4 * (l >> 4);
        f32x4 v = red[0][tile][l];
#pragma unroll
        for (int w = 1; w < HALF; w++) v += red[w][tile][l];
        if (t < count && j < a.R)
            *reinterpret_cast<f32x4*>(a.h + ((int64_t)blockIdx.z * a.T + r0 + t) * a.R + j) = v;
    }
}

// 64 tokens by up to 32 * JW rows of A, for whole vectors: chunks of 128 elements of K go through
// LDS, the next one's loads on their way.  A row's 256 bytes are read by 16 lanes side by side;
// fragments loaded straight from memory take 64 bytes from each of 16 rows, which lie a power of
// two apart and so in one channel of the cache (8192 tokens, K = 4096, 96 rows: 49 us that way).
// Wave w has token group w % 4 and the rows' half w / 4, so no sums are added up.
template <int JW>
__global__ __launch_bounds__(512) void shrink_tile_kernel(const Args a) {
    constexpr int TM = 64, JR = 32 * JW, CK = 128, ROW = 2 * CK + 16;  // bytes of a padded row
    constexpr int LOADS = (TM + JR) * 16 / 512;                       // 16 bytes each, a thread
    __shared__ __align__(16) uint8_t lds[(TM + JR) * ROW];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ahead = rows_ahead(a);
    int e, r0, r1;
    if (!find_tile<TM>(a, a.S, blockIdx.x, e, r0, r1)) return;
    const int j0 = blockIdx.y * JR, count = r1 - r0;
    // a thread's loads: 16 bytes (tid % 16) of rows tid / 16 + 32 i, tokens first
    const uint16_t* src[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
        const int r = (tid >> 4) + 32 * i;
        if (r < TM) {
            const int row = token_at(a, ahead, r0, r, count);
            src[i] = a.x + (int64_t)(row < 0 ? 0 : row) * a.ldx;
        } else {
            const int j = j0 + r - TM;
            src[i] = a.a + ((int64_t)e * a.R + (j < a.R ? j : a.R - 1)) * a.K;
        }
        src[i] += 8 * (tid & 15);
    }
    const int chunks = (a.K + CK - 1) / CK, per = (chunks + a.kparts - 1) / a.kparts;
    const int c0 = blockIdx.z * per, c1 = c0 + per < chunks ? c0 + per : chunks;
    h8 next[LOADS];
    auto fetch = [&](int c) {
        if (c >= c1) return;
        const int k = c * CK;
        if (k + CK <= a.K) {
#pragma unroll
            for (int i = 0; i < LOADS; i++) next[i] = *reinterpret_cast<const h8*>(src[i] + k);
        } else {
#pragma unroll
            for (int i = 0; i < LOADS; i++) next[i] = load8<true>(src[i] + k, a.K - k - 8 * (tid & 15));
        }
    };
    f32x4 acc[JW];
#pragma unroll
    for (int j = 0; j < JW; j++) acc[j] = f32x4{0, 0, 0, 0};
    fetch(c0);
    const uint8_t* xs = lds + ((wave & 3) * 16 + (lane & 15)) * ROW + 16 * (lane >> 4);
    const uint8_t* as = lds + (TM + (wave >> 2) * 16 * JW + (lane & 15)) * ROW + 16 * (lane >> 4);
    for (int c = c0; c < c1; c++) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < LOADS; i++)
            *reinterpret_cast<h8*>(lds + ((tid >> 4) + 32 * i) * ROW + 16 * (tid & 15)) = next[i];
        __syncthreads();
        fetch(c + 1);
#pragma unroll
        for (int s = 0; s < CK / 32; s++) {
            const h8 x = *reinterpret_cast<const h8*>(xs + 64 * s);
#pragma unroll
            for (int j = 0; j < JW; j++)
                acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    *reinterpret_cast<const h8*>(as + j * 16 * ROW + 64 * s), x, acc[j], 0, 0, 0);
        }
    }
    const int t = (wave & 3) * 16 + (lane & 15);
#pragma unroll
    for (int j = 0; j < JW; j++) {
        const int i = j0 + ((wave >> 2) * JW + j) * 16 + 4 * (lane >> 4);
        if (t < count && i < a.R)
            *reinterpret_cast<f32x4*>(a.h + ((int64_t)blockIdx.z * a.T + r0 + t) * a.R + i) = acc[j];
    }
}

// What a workgroup's column block is of: the part, and the columns n0 .. n1 of it.
__device__ __forceinline__ bool find_block(const Args& a, int block, int& part, int& n0, int& n1) {
    for (part = 0; part < a.parts; part++) {
        const int width = a.start[part + 1] - a.start[part], blocks = (width + a.cols - 1) / a.cols;
        if (block < blocks) break;
        block -= blocks;
    }
    if (part == a.parts) return false;
    n0 = a.start[part] + block * a.cols;
    const int end = a.start[part + 1];
    n1 = n0 + a.cols < end ? n0 + a.cols : end;
    return true;
}

// How many rows of the part are the adapter's: what the others (filled up) make of x is not
// looked at, since 0 times an infinity is not 0.
__device__ __forceinline__ int own_rank(const Args& a, int e, int part) {
    int own = a.rank;
    if (a.ranks) own = __builtin_amdgcn_readfirstlane(a.ranks[e * a.parts + part]);  // of the wave
    return own;
}

// Eight consecutive values of a token's low-rank row, the parts added in order (MANY of them on
// their way at once), scaled; 0 from `left` on.
template <int MANY>
__device__ __forceinline__ void low_rank(const Args& a, int pos, int part, int j, int left,
                                         float scale, float (&v)[8]) {
    const float* h = a.h + (int64_t)pos * a.R + part * a.rank + j;
    const int64_t step = (int64_t)a.T * a.R;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = 0.0f;
    for (int p = 0; p < a.kparts; p += MANY) {
        f32x4 lo[MANY], hi[MANY];
#pragma unroll
        for (int i = 0; i < MANY; i++) {
            const bool has = p + i < a.kparts;
            const float* q = h + (has ? i * step : 0);
            lo[i] = *reinterpret_cast<const f32x4*>(q);
            hi[i] = *reinterpret_cast<const f32x4*>(q + 4);
            if (!has) lo[i] = hi[i] = f32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < MANY; i++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                v[k] += lo[i][k];
                v[k + 4] += hi[i][k];
            }
        h += MANY * step;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = i < left ? v[i] * scale : 0.0f;
}

__device__ __forceinline__ uint32_t top_of(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const uint32_t w = __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu;
        m = w > m ? w : m;
    }
    return m;
}

// The power of two that brings a token's largest |h| (its bits) to 2^8; 0 for a row of zeros.
// Beside infinities and NaN, which decide the row, whatever is finite stays so in fp16.
__device__ __forceinline__ int shift_of(uint32_t top) {
    const int up = 135 - (int)(top >> 23);
    return top >= 0x7f800000u ? -113 : top == 0 ? 0 : up > 120 ? 120 : up;
}

__device__ __forceinline__ void split8(const float (&v)[8], uint32_t top, h8& hi, h8& lo) {
    const int up = shift_of(top);
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float w = __builtin_ldexpf(v[j], up);
        const _Float16 h = (_Float16)w;
        hi[j] = h;
        lo[j] = top < 0x7f800000u ? (_Float16)(w - (float)h) : (_Float16)0.0f;
    }
}

// A strip of a wave: 16 * QT columns from n on, the rows of B for it.  Row i of the q-th product
// is column 32 (q / 2) + 8 (i / 4) + 4 (q & 1) + i % 4, which leaves lane (t, g) with columns
// 8 g .. 8 g + 7 of every 32: a load of 16 bytes a lane takes 64 in a row of each token.
// b: B of the adapter; whole: the strip ends before n1.
template <int KS, int QT>
__device__ __forceinline__ void load_b(const Args& a, const uint16_t* b, int n, int n1, bool whole,
                                       int lane, h8 (&bf)[QT][KS]) {
    const int i = lane & 15, g = lane >> 4, mine = 8 * (i >> 2) + (i & 3);
    const uint16_t* base = b + (int64_t)n * a.rank;  // the same for the wave
#pragma unroll
    for (int q = 0; q < QT; q++) {
        const int c = 32 * (q >> 1) + 4 * (q & 1);
        const uint16_t* from = base + c * a.rank;
        int off = mine * a.rank + 8 * g;
        if (!whole) off = ((n + c + mine < n1 ? c + mine : n1 - 1 - n) - c) * a.rank + 8 * g;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            // past the rank: the row's first values, then zeros
            const bool has = 32 * s + 8 * g < a.rank;
            bf[q][s] = *reinterpret_cast<const h8*>(from + off + (has ? 32 * s : -8 * g));
            if (a.rank < 32 * (s + 1) && !has) bf[q][s] = h8{0, 0, 0, 0, 0, 0, 0, 0};
        }
    }
}

// y: the lane's first column of the strip, `left` columns before the end; whole (the same for
// the wave): all of the strip is there.
template <int QT>
__device__ __forceinline__ void load_y(const uint16_t* y, int left, bool whole, h8 (&in)[QT / 2]) {
    if (whole) {
#pragma unroll
        for (int q = 0; q < QT / 2; q++) in[q] = *reinterpret_cast<const h8_anywhere*>(y + 32 * q);
    } else {
#pragma unroll
        for (int q = 0; q < QT / 2; q++) in[q] = load8<false>(y + 32 * q, left - 32 * q);
    }
}

// down is a power of two: the product is exact, the sum rounded once to 32 bits, then to 16.
template <int QT>
__device__ __forceinline__ void store_y(uint16_t* o, int left, bool whole, const h8 (&in)[QT / 2],
                                        const f32x4 (&acc)[QT], float down) {
#pragma unroll
    for (int q = 0; q < QT / 2; q++) {
        h8 z;
#pragma unroll
        for (int r = 0; r < 8; r++)
            z[r] = (_Float16)__builtin_fmaf(acc[2 * q + r / 4][r & 3], down, (float)in[q][r]);
        if (whole) {
            *reinterpret_cast<h8_anywhere*>(o + 32 * q) = z;
        } else {
#pragma unroll
            for (int r = 0; r < 8; r++) {
                const _Float16 f = z[r];  // an element is no lvalue to bit_cast
                if (32 * q + r < left) o[32 * q + r] = __builtin_bit_cast(uint16_t, f);
            }
        }
    }
}

// Tokens without an adapter: out is y.  MANY of a wave's rows are on their way at once (3323
// tokens, 6144 columns, rank 64, half of them without: 32.0 us, 34.0 with one).
template <int MANY>
__device__ __forceinline__ void copy_rows(const Args& a, int ahead, int r0, int count, int n0, int n1) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int whole = n0 + (n1 - n0) / 8 * 8;
    for (int t0 = wave; t0 < count; t0 += kWaves * MANY) {
        int row[MANY];
#pragma unroll
        for (int i = 0; i < MANY; i++) {
            const int t = t0 + kWaves * i, r = token_at(a, ahead, r0, t, count);
            row[i] = t < count ? r : -1;
        }
        for (int n = n0 + lane * 8; n < whole; n += 512) {
            h8 v[MANY];
#pragma unroll
            for (int i = 0; i < MANY; i++)
                if (row[i] >= 0)
                    v[i] = *reinterpret_cast<const h8_anywhere*>(a.y + (int64_t)row[i] * a.ldy + n);
#pragma unroll
            for (int i = 0; i < MANY; i++)
                if (row[i] >= 0)
                    *reinterpret_cast<h8_anywhere*>(a.out + (int64_t)row[i] * a.ldo + n) = v[i];
        }
        if (whole + lane < n1) {
#pragma unroll
            for (int i = 0; i < MANY; i++)
                if (row[i] >= 0)
                    a.out[(int64_t)row[i] * a.ldo + whole + lane] =
                        a.y[(int64_t)row[i] * a.ldy + whole + lane];
        }
    }
}

// KS: 32-element steps of the rank.  Tiles of 16 tokens; a wave keeps the low-rank rows in
// registers and goes through its strips, the loads of the next on their way.  48 tokens of 48
// adapters, rank 16, 24576 columns: 12.4 us for 42 MB; 16 tokens, 151936 columns: 11.0 us.  At
// ranks above 32 the waves share the sums of the low-rank rows (9 tokens, rank 128, 32000
// columns: 10.8 us; 17.7 with all sums in each wave).
template <int KS>
__global__ __launch_bounds__(kThreads, KS <= 2 ? 4 : KS == 4 ? 2 : 1) void expand_few_kernel(const Args a) {
    constexpr int QT = KS == 1 ? 4 : 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ahead = rows_ahead(a);
    int e, r0, r1, part, n0, n1;
    if (!find_tile<16>(a, a.S + 1, blockIdx.x, e, r0, r1)) return;
    if (!find_block(a, blockIdx.y, part, n0, n1)) return;
    const int count = r1 - r0, t = lane & 15, g = lane >> 4;
    if (e == a.S) {
        if (a.copy) copy_rows<4>(a, ahead, r0, count, n0, n1);
        return;
    }
    const int row = token_at(a, ahead, r0, t, count);
    const bool live = t < count && row >= 0;
    // lanes without a token load another's row, and store nothing
    const uint16_t* y = a.y + (int64_t)(row < 0 ? 0 : row) * a.ldy + 8 * g;
    uint16_t* o = a.out + (int64_t)(row < 0 ? 0 : row) * a.ldo + 8 * g;
    const uint16_t* rows_b = a.b + (int64_t)e * a.start[a.parts] * a.rank;
    constexpr int STEP = kWaves * 16 * QT;
    h8 bf[2][QT][KS], in[2][QT / 2];
    auto fetch = [&](int n, h8 (&b)[QT][KS], h8 (&z)[QT / 2]) {
        if (n >= n1) return;
        load_b<KS, QT>(a, rows_b, n, n1, n + 16 * QT <= n1, lane, b);
        load_y<QT>(y + n, n1 - n - 8 * g, n + 16 * QT <= n1, z);
    };
    int n = n0 + wave * 16 * QT;
    fetch(n, bf[0], in[0]);  // comes from memory, the low-rank rows from a cache
    const float scale = a.scaling ? a.scaling[e] : 1.0f;
    const int own = own_rank(a, e, part);
    float v[KS][8];
    uint32_t top = 0;
    auto sum = [&](int s, float (&to)[8]) {
        const int j = s * 32 + 8 * g;
        if (t < count && j < a.rank) {
            low_rank<8>(a, r0 + t, part, j, own - j, scale, to);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) to[i] = 0.0f;
        }
    };
    if constexpr (KS == 1) {
        sum(0, v[0]);
    } else {  // a step or two of the rank for each wave, so that all parts are on their way at once
        __shared__ f32x4 sums[KS][2][64];
        for (int s = wave; s < KS; s += kWaves) {
            float w[8];
            sum(s, w);
            sums[s][0][lane] = f32x4{w[0], w[1], w[2], w[3]};
            sums[s][1][lane] = f32x4{w[4], w[5], w[6], w[7]};
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int i = 0; i < 8; i++) v[s][i] = sums[s][i / 4][lane][i % 4];
    }
#pragma unroll
    for (int s = 0; s < KS; s++) {
        const uint32_t m = top_of(v[s]);
        top = m > top ? m : top;
    }
#pragma unroll
    for (int d = 16; d < 64; d *= 2) {
        const uint32_t m = (uint32_t)__shfl_xor((int)top, d, 64);
        top = m > top ? m : top;
    }
    h8 hi[KS], lo[KS];
#pragma unroll
    for (int s = 0; s < KS; s++) split8(v[s], top, hi[s], lo[s]);
    const float down = __builtin_ldexpf(1.0f, -shift_of(top));
    fetch(n + STEP, bf[1], in[1]);
    auto strip = [&](int n, h8 (&b)[QT][KS], h8 (&z)[QT / 2]) {
        if (n >= n1) return;
        f32x4 acc[QT];
#pragma unroll
        for (int q = 0; q < QT; q++) acc[q] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int q = 0; q < QT; q++) {
                acc[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[q][s], lo[s], acc[q], 0, 0, 0);
                acc[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[q][s], hi[s], acc[q], 0, 0, 0);
            }
        h8 was[QT / 2];
#pragma unroll
        for (int q = 0; q < QT / 2; q++) was[q] = z[q];
        fetch(n + 2 * STEP, b, z);
        if (live)
            store_y<QT>(o + n, n1 - n - 8 * g, n + 16 * QT <= n1, was, acc, down);
    };
    for (; n < n1; n += 2 * STEP) {
        strip(n, bf[0], in[0]);
        strip(n + STEP, bf[1], in[1]);
    }
}

// The same for tiles of 16 * NT tokens: the low-rank rows lie in LDS, a strip's rows of B serve
// all NT groups of 16.  WHOLE: every strip is there to its end.  8192 tokens, 6144 columns, rank
// 32 (201 MB of y in and out): 50 us, 4.0 TB/s; a copy in the same order of addresses alone takes
// 39 us, one straight through 32.
template <int KS, int NT, bool WHOLE>
__global__ __launch_bounds__(kThreads) void expand_kernel(const Args a) {
    constexpr int TM = 16 * NT, QT = KS <= 2 ? 4 : 2;
    constexpr int UNITS = (TM * KS * 4 + kThreads - 1) / kThreads;
    __shared__ h8 hs[NT * KS * 2][64];
    __shared__ uint32_t top[TM];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ahead = rows_ahead(a);
    int e, r0, r1, part, n0, n1;
    // the column blocks of a tile side by side
    const int tile = blockIdx.x / (uint32_t)a.blocks;
    if (!find_tile<TM>(a, a.S + 1, tile, e, r0, r1)) return;
    if (!find_block(a, blockIdx.x - tile * a.blocks, part, n0, n1)) return;
    const int count = r1 - r0, g = lane >> 4;
    if (e == a.S) {
        if (a.copy) copy_rows<8>(a, ahead, r0, count, n0, n1);
        return;
    }
    int row[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int i = t * 16 + (lane & 15), r = token_at(a, ahead, r0, i, count);
        row[t] = i < count ? r : -1;  // -1: loads row 0, stores nothing
    }
    const uint16_t* rows_b = a.b + (int64_t)e * a.start[a.parts] * a.rank;
    h8 bf[QT][KS], in[NT][QT / 2];
    auto fetch = [&](int n) {
        const bool whole = WHOLE || n + 16 * QT <= n1;
        load_b<KS, QT>(a, rows_b, n, n1, WHOLE || n + 16 * QT <= n1, lane, bf);
#pragma unroll
        for (int t = 0; t < NT; t++)
            load_y<QT>(a.y + (int64_t)(row[t] < 0 ? 0 : row[t]) * a.ldy + n + 8 * g, n1 - n - 8 * g,
                       whole, in[t]);
    };
    // the low-rank rows before y: loads come back in order, and these come from the cache
    const float scale = a.scaling ? a.scaling[e] : 1.0f;
    const int own = own_rank(a, e, part);
    float v[UNITS][8];
#pragma unroll
    for (int i = 0; i < UNITS; i++) {
        const int u = threadIdx.x + i * kThreads, t = u / (KS * 4), j = u % (KS * 4) * 8;
        if (t < count && j < a.rank) {
            low_rank<4>(a, r0 + t, part, j, own - j, scale, v[i]);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) v[i][k] = 0.0f;
        }
    }
    int n = n0 + wave * 16 * QT;
    if (n < n1) fetch(n);
    for (int t = threadIdx.x; t < TM; t += kThreads) top[t] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < UNITS; i++) {
        const int t = (threadIdx.x + i * kThreads) / (KS * 4);
        if (t < count) atomicMax(&top[t], top_of(v[i]));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < UNITS; i++) {
        const int u = threadIdx.x + i * kThreads, t = u / (KS * 4), k = u % (KS * 4);
        if (t >= TM) continue;
        const int at = ((t >> 4) * KS + (k >> 2)) * 2, l = (t & 15) + 16 * (k & 3);
        split8(v[i], top[t], hs[at][l], hs[at + 1][l]);
    }
    __syncthreads();
    float down[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) down[t] = __builtin_ldexpf(1.0f, -shift_of(top[t * 16 + (lane & 15)]));
    while (n < n1) {
        const bool whole = WHOLE || n + 16 * QT <= n1;
#pragma unroll
        for (int t = 0; t < NT; t++) {
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
            if (row[t] >= 0)
                store_y<QT>(a.out + (int64_t)row[t] * a.ldo + n + 8 * g, n1 - n - 8 * g, whole, in[t],
                            acc, down[t]);
        }
        n += kWaves * 16 * QT;
        if (n < n1) fetch(n);
    }
}

// Tiles of 16 tokens, or of 64 from 1024 tokens on.  How many adapters share these the host does
// not know: S counts slots, of which a step may use a few.  Tiles of 16 and of 64, calls with
// K = 4096: 6144 columns, rank 32, 16 adapters, 1024 tokens 33.4 us, 21.5, 8192 tokens 128, 80;
// 64 adapters, 1024 tokens 44, 31.5; 4096 columns, rank 16, 16 adapters, 1024 tokens 17.6, 15.5,
// 8192 tokens 61, 53.  Tiles of 64 lose where an adapter has fewer than about 16 tokens: 1024
// tokens of 128 adapters 19.8, 26.2, of 1024 adapters 77, 180; and on small projections (K = 2048,
// 1024 columns, rank 8, 1024 tokens 10.5, 11.0).
bool big_tiles(int64_t T) { return T >= 1024; }

int64_t tiles_of(int64_t T, int64_t groups, int64_t bm) {
    return T / bm + (groups < T ? groups : T);
}

struct Plan {
    bool big;
    int jt;  // blocks of 16 rows of A in a workgroup: x is read once for each group of them
    int64_t jgroups, tiles, kparts;
};
Plan plan_of(int64_t T, int64_t K, int64_t S, int64_t R) {
    Plan p{};
    p.big = big_tiles(T);
    const int64_t blocks = (R + 15) / 16;
    p.tiles = tiles_of(T, S, p.big ? 64 : 16);
    if (p.big) {
        p.jt = blocks <= 2 ? 2 : blocks <= 4 || blocks == 7 || blocks == 8 ? 4 : 6;
        p.jgroups = (blocks + p.jt - 1) / p.jt;
        // parts of K that leave the 256 CUs evenly loaded; each costs its share of the sums' way
        // through memory
        double best = 1e30;
        for (int64_t k = 1; k <= 8 && (k == 1 || k * 256 <= K); k++) {
            const int64_t rounds = (p.tiles * p.jgroups * k + 255) / 256;
            const double cost = (double)rounds / k + 0.05 * k;
            if (cost < best) {
                best = cost;
                p.kparts = k;
            }
        }
        return p;
    }
    // as many blocks in a workgroup as leave 192 with eight parts of K, and parts for one on each
    // CU; more than eight cost the expansion a round trip
    for (int jt : {6, 4, 3, 2, 1}) {
        p.jt = jt;
        p.jgroups = (blocks + jt - 1) / jt;
        if (jt == 1 || (blocks % jt == 0 && p.tiles * p.jgroups * 8 >= 192)) break;
    }
    const int64_t want = 256 / (p.tiles * p.jgroups) + 1, most = (K + 511) / 512;
    p.kparts = want < most ? want : most;
    if (p.kparts > 8) p.kparts = 8;
    return p;
}

template <bool WIDE>
void shrink(const Args& a, const Plan& p, hipStream_t st) {
    dim3 grid((uint32_t)p.tiles, (uint32_t)p.jgroups, (uint32_t)p.kparts);
    constexpr int threads = kShrinkWaves * 64;
    if (p.big && WIDE) {
        if (p.jt == 2) shrink_tile_kernel<1><<<grid, 512, 0, st>>>(a);
        else if (p.jt == 4) shrink_tile_kernel<2><<<grid, 512, 0, st>>>(a);
        else shrink_tile_kernel<3><<<grid, 512, 0, st>>>(a);
        return;
    }
    if (p.big) grid.x = (uint32_t)tiles_of(a.T, a.S, 16);
    if (p.jt == 1) shrink_kernel<1, WIDE><<<grid, threads, 0, st>>>(a);
    else if (p.jt == 2) shrink_kernel<2, WIDE><<<grid, threads, 0, st>>>(a);
    else if (p.jt == 3) shrink_kernel<3, WIDE><<<grid, threads, 0, st>>>(a);
    else if (p.jt == 4) shrink_kernel<4, WIDE><<<grid, threads, 0, st>>>(a);
    else shrink_kernel<6, WIDE><<<grid, threads, 0, st>>>(a);
}

void expand_few(const Args& a, dim3 grid, hipStream_t st) {
    if (a.rank <= 32) expand_few_kernel<1><<<grid, kThreads, 0, st>>>(a);
    else if (a.rank <= 64) expand_few_kernel<2><<<grid, kThreads, 0, st>>>(a);
    else if (a.rank <= 128) expand_few_kernel<4><<<grid, kThreads, 0, st>>>(a);
    else expand_few_kernel<8><<<grid, kThreads, 0, st>>>(a);
}

template <bool WHOLE>
void expand(const Args& a, dim3 grid, hipStream_t st) {
    if (a.rank <= 32) expand_kernel<1, 4, WHOLE><<<grid, kThreads, 0, st>>>(a);
    else if (a.rank <= 64) expand_kernel<2, 4, WHOLE><<<grid, kThreads, 0, st>>>(a);
    else if (a.rank <= 128) expand_kernel<4, 4, WHOLE><<<grid, kThreads, 0, st>>>(a);
    else expand_kernel<8, 2, WHOLE><<<grid, kThreads, 0, st>>>(a);
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
    a.ranks = l.ranks;
    a.h = l.work;
    a.T = (int)l.T; a.K = (int)l.K; a.S = (int)l.S; a.rank = (int)l.rank; a.R = (int)R;
    a.kparts = (int)p.kparts;
    a.copy = l.out != l.y;
    a.parts = (int)l.parts;
    for (int i = 0; i < l.parts; i++) a.start[i + 1] = a.start[i] + (int)l.splits[i];

    const bool wide = l.K % 8 == 0 && l.ldx % 8 == 0 && (((uintptr_t)l.x | (uintptr_t)l.a) & 15) == 0;
    if (wide) shrink<true>(a, p, st);
    else shrink<false>(a, p, st);

    const int nt = !p.big ? 1 : l.rank > 128 ? 2 : 4;
    const int64_t tiles = tiles_of(l.T, l.S + 1, 16 * nt);
    // Columns of a workgroup, whole strips of its four waves.  Tiles of 64: two strips where that
    // leaves 320 workgroups or more, else one (calls with K = 2048, rank 16, four adapters; one
    // strip, two: 8192 tokens, 6144 columns 64.0 us, 61.0; 4096 tokens, 4096 columns 23.8, 22.1;
    // 4096 tokens, 2048 columns 17.1, 19.7; 2048 tokens, 2048 columns 13.7, 15.7; 1024 tokens,
    // 1024 columns 11.2, 12.7; between 320 and 550 they differ by less than 1).  Of 16: the
    // fewest rounds of the four that a CU holds at once, each as long as the columns and a start
    // that takes about as long as 1024 of them.
    const int64_t strips = kWaves * 64;
    int64_t cols = 0, blocks = 0, best = 0;
    for (int64_t c = strips; c <= (p.big ? 512 : 4096); c += strips) {
        int64_t n = 0;
        for (int i = 0; i < l.parts; i++) n += (l.splits[i] + c - 1) / c;
        const int64_t cost = p.big ? (tiles * n >= 320 ? -c : c)
                                   : (tiles * n + 1023) / 1024 * (c + 1024);
        if (!cols || cost < best) {
            cols = c;
            blocks = n;
            best = cost;
        }
    }
    while (p.big && tiles * blocks >= 1 << 24) {  // a launch has fewer than 2^32 threads
        cols *= 2;
        blocks = 0;
        for (int i = 0; i < l.parts; i++) blocks += (l.splits[i] + cols - 1) / cols;
    }
    a.cols = (int)cols;
    a.blocks = (int)blocks;
    // Where all strips are whole the large tiles take code without the branches for others (a call
    // of 8192 tokens, K = 4096, 6144 columns, rank 32: 75.4 us, 78.0 with them; the small tiles are
    // as fast either way).
    bool whole = true;
    for (int i = 0; i < l.parts; i++) whole = whole && l.splits[i] % 64 == 0;
    const uint32_t all = (uint32_t)(tiles * blocks);
    if (!p.big) expand_few(a, dim3((uint32_t)tiles, (uint32_t)blocks), st);
    else if (whole) expand<true>(a, dim3(all), st);
    else expand<false>(a, dim3(all), st);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) {
        set_error_detail("lora launch: %s", hipGetErrorString(err));
        return FNI8_ERR_LAUNCH;
    }
    return FNI8_OK;
}

}  // namespace fni8h
