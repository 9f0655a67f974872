// One token a row of logits, from given random numbers (gfx950).
//
// Order: logit descending, ties by the lower index.  w_i = exp((x_i - max) / T).  Three
// filters, each of which keeps a prefix of that order:
//   top-k  the first k tokens (mass Wk)
//   top-p  a token while the mass before it is less than p * Wk
//   min-p  a token with w_i >= min_p
// The shortest prefix is kept; the first token is in it always.  The drawn token is the first
// kept one, in index order, at which the running mass exceeds u * (kept mass).
//
// Masses are integers, w_i * 2^s rounded, with s such that a row's sum stays below 2^62: their
// sums do not depend on an order, so a histogram filled by atomics gives the same token every
// time.  At 151936 tokens s is 44; 24 bits of a float sum would put about one draw in thirty on
// a neighbour of the token that the sums mean.  A rank, a mass and a place among equal logits
// are all the same search: the first key at which a running sum of integers reaches a number.
//
// Launches:
//   scan    reads the logits once, 8192 to an item: the largest logit of each thread's 32 and,
//           where a row needs its whole mass, the sum of the part's weights in 64 bits
//   draw    one workgroup a row: the threads' maxima bound the kept prefix from below (k of
//           them are k tokens, and have a mass), so only the few groups of 32 that reach over
//           that bound are read again, and all searches run over a short list
// and, unless the host knows that every prefix is short, for rows where it is not:
//   gather  all workgroups: the parts' masses above the place where top-p ends, as far as
//           samples tell, and a list of the tokens around that place (min-p: the kept mass)
//   finish  one workgroup a row: top-p's end in the list, the part that the draw falls into, and
//           the token in it
// A row whose list does not fit is searched whole by its workgroup: a histogram of its mass in 2048
// steps of weight, then the list of one step, 120 to 200 us for up to 64 rows of 151936.  These
// are thousands of equal logits at an end (1.2 ms where all are equal), top-k of thousands, and
// top-p beside min-p where the threads' maxima down to min-p's end fall short of top-p's mass.
// Nothing depends on the number of rows: a row's token is the same in every batch.
#include <type_traits>

#include "common.h"

namespace {

typedef unsigned long long u64;

constexpr int kVec = 8, kPart = 8192, kScanThreads = 256;  // logits: of a load, of a part
constexpr int kSteps = kPart / (kScanThreads * kVec);      // loads of a scan thread
constexpr int kThreads = 512, kWaves = 8;                  // draw
constexpr int kBins = 2048;    // steps of weight; the last one: weights that round to 0
constexpr int kList = 2048;    // candidates in LDS
constexpr int kMini = 64;      // candidates that one wave compares with each other
constexpr int kHits = 4096;    // groups that are read again
constexpr int kShort = 256;    // thread maxima that a bound is taken from (of kThreads)
constexpr int kKeep = 10;      // groups of a draw thread in registers
constexpr int kAround = 8192;  // tokens around a row's end of top-p, in the workspace

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// 2^(d rate + s) for -1000 <= d rate <= 0.  d rate = n + f, |f| <= 1/2, by the addition that
// leaves n + s in the low bits; 2^f = 1 + f q(f), q the polynomial of degree 7 through
// (2^f - 1) / f at the Chebyshev nodes (exactly 1 at 0, else off by 2.2e-12 of the value at
// most; a row of 151936 equal shares has 6.6e-6 for each); n + s goes into the exponent.
__device__ __forceinline__ double exp2_at(double d, double rate, int s) {
    const double magic = 0x1.8p52 + s, tn = __builtin_fma(d, rate, magic);
    const double f = __builtin_fma(d, rate, -(tn - magic));
    double q = 1.325080551750225e-06;
    q = __builtin_fma(q, f, 1.5303700711365693e-05);
    q = __builtin_fma(q, f, 1.5403475186530786e-04);
    q = __builtin_fma(q, f, 1.3333478473685416e-03);
    q = __builtin_fma(q, f, 9.61812913523614e-03);
    q = __builtin_fma(q, f, 5.5504109063258665e-02);
    q = __builtin_fma(q, f, 0.24022650695888503);
    q = __builtin_fma(q, f, 0.6931471805568324);
    q = __builtin_fma(q, f, 1.0);
    u32x2 b = __builtin_bit_cast(u32x2, q);
    const u32x2 n = __builtin_bit_cast(u32x2, tn);
    b.y += n.x << 20;
    return __builtin_bit_cast(double, b);
}

// Order of floats as unsigned numbers; -0 counts as +0, NaN above everything.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return x != x ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __builtin_bit_cast(float, (key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

template <class E>
__device__ __forceinline__ float value(E e) {
    if constexpr (sizeof(E) == 2) return fni8::h2f(e);
    else return e;
}

template <class E>
__device__ __forceinline__ E lowest_of() {  // minus infinity
    if constexpr (sizeof(E) == 2) return (E)0xfc00;
    else return -__builtin_inff();
}

template <class E>
__device__ __forceinline__ E element(float v) {  // of a value that has one
    if constexpr (sizeof(E) == 2) return fni8::f2h(v);
    else return v;
}

// Eight logits from index i on, -inf past the row's end.  Rows need no more than their
// elements' alignment: the loads are as wide at any address.
template <class E>
__device__ __forceinline__ void load8(const E* x, int i, int V, float (&v)[kVec]) {
    typedef E vec __attribute__((ext_vector_type(8), aligned(sizeof(E))));
    if (i + kVec <= V) {
        const vec q = *reinterpret_cast<const vec*>(x + i);
#pragma unroll
        for (int j = 0; j < kVec; j++) {
            const E e = q[j];
            v[j] = value(e);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kVec; j++) v[j] = i + j < V ? value(x[i + j]) : -__builtin_inff();
    }
}

// A row's settings, and weights relative to a largest logit.
struct Row {
    float T, p, least, u, top;
    int k, s;
    double rate, base, step;
    uint32_t low;
    bool by_k, by_p, by_m, inf;

    __device__ __forceinline__ Row(const fni8h::Sample& a, int64_t row, int V) {
        T = a.temperature ? a.temperature[row] : a.temperature1;
        k = a.top_k ? a.top_k[row] : a.top_k1;
        p = a.top_p ? a.top_p[row] : a.top_p1;
        const float m = a.min_p ? a.min_p[row] : a.min_p1;
        least = m > 0.0f ? m < 1.0f ? m : 1.0f : 0.0f;
        u = a.u ? a.u[row] : 0.0f;
        by_k = k > 0 && k < V;
        by_p = p < 1.0f;
        by_m = least > 0.0f;
        // bits of a weight's fraction: V weights of at most 1 add up to less than 2^62
        s = 30 + __builtin_clz(V);
        s = s < 50 ? s : 50;
        step = (kBins - 2) / (double)(s + 2);
    }
    // Every weight of the row is summed: for top-p without top-k, and without any filter.
    __device__ __forceinline__ bool summed() const { return T > 0.0f && !by_k && (by_p || !by_m); }
    __device__ __forceinline__ void largest(float x) {
        inf = x == __builtin_inff();
        top = inf ? 0.0f : x;
        base = top == -__builtin_inff() ? 0.0 : (double)top;
        rate = 1.4426950408889634 / (double)T;
        rate = rate > 1e-280 ? rate : 1e-280;
        low = __builtin_bit_cast(u32x2, -1000.0 / rate).y;
    }
    // Beside plus infinity nothing else has weight: it counts as 0, the rest as minus infinity.
    __device__ __forceinline__ float seen(float v) const {
        return !inf ? v : v == __builtin_inff() ? 0.0f : -__builtin_inff();
    }
    // A seen logit's distance from the largest, down to that of weight 2^-1000 (minus infinity
    // too): of two negative numbers the lower has the larger upper word.
    __device__ __forceinline__ double away(float v) const {
        u32x2 d = __builtin_bit_cast(u32x2, (double)v - base);
        d.y = d.y < low ? d.y : low;
        return __builtin_bit_cast(double, d);
    }
    // log2 of its weight; the weight; the weight as an integer, rounded: adding 2^52 leaves it in
    // the low bits of the sum.
    __device__ __forceinline__ double power(float v) const { return away(v) * rate; }
    __device__ __forceinline__ double weight(float v) const { return exp2_at(away(v), rate, 0); }
    __device__ __forceinline__ u64 mass(float v) const {
        u32x2 m = __builtin_bit_cast(u32x2, exp2_at(away(v), rate, s) + 0x1p52);
        m.y &= 0xfffffu;
        return __builtin_bit_cast(u64, m);
    }
    // What a mass has to be for min-p.
    __device__ __forceinline__ u64 floor() const {
        return (u64)__builtin_rint((double)least * __builtin_ldexp(1.0, s));
    }
    // Step of a weight, rising as it falls; kBins - 1 for weights that round to 0.
    __device__ __forceinline__ int bin(double power) const {
        const double d = -power * step;
        return d < (double)(kBins - 1) ? (int)d : kBins - 1;
    }
};

// Eight seen logits.
template <class E>
__device__ __forceinline__ void load8(const E* x, int i, int V, const Row& r, float (&v)[kVec]) {
    load8(x, i, V, v);
    if (r.inf) {
#pragma unroll
        for (int j = 0; j < kVec; j++) v[j] = r.seen(v[j]);
    }
}

// A row in the workspace.  scan fills top, part, sum and pick; draw the long prefix's state;
// gather its above and around.
enum { kDone, kTopP, kMinP, kWhole };  // what is left to do
struct Long {
    u64 need;        // top-p: the mass to reach
    float high, low; // logits that the end of top-p lies between
    int kind, around;
    uint32_t top;    // key of the row's largest logit
};
struct Work {
    double* sum;     // [parts] masses, relative to the part's largest logit
    u64 *above;      // [parts] masses of what is kept for certain
    u64* around;     // [kAround] orders of the tokens from low up to high
    uint32_t* top;   // [parts][256] keys of the threads' largest logits
    uint32_t* pick;  // [parts][256] two of the 32, as bfloat16
    uint32_t* part;  // [parts] keys of the parts' largest
    Long* more;
};
__host__ __device__ inline int64_t parts_of(int64_t V) { return (V + kPart - 1) / kPart; }
// Tokens around an end that a row has room for.  None for rows of up to kList tokens, which fit a
// list whole; a flat one for which none is tried is searched whole.
__host__ __device__ inline int64_t around_of(int64_t V) {
    return V <= kList ? 0 : V < kAround ? V : kAround;
}
__host__ __device__ inline int64_t row_bytes(int64_t V) {
    return (parts_of(V) * (8 + 8 + 8 * kScanThreads + 4) + around_of(V) * 8 + (int64_t)sizeof(Long) +
            15) / 16 * 16;
}
// Rows that 1 GiB of workspace holds; more take turns in it, a set of launches each (fewer than
// 2^19 parts of rows at once).
inline int64_t rows_at_once(int64_t V) { return ((int64_t)1 << 30) / row_bytes(V); }
__device__ __forceinline__ Work work_of(int8_t* w, int64_t row, int64_t V) {
    const int64_t parts = parts_of(V);
    w += row * row_bytes(V);
    Work r;
    r.sum = reinterpret_cast<double*>(w);
    r.above = reinterpret_cast<u64*>(w + parts * 8);
    r.around = r.above + parts;
    r.more = reinterpret_cast<Long*>(r.around + around_of(V));
    r.top = reinterpret_cast<uint32_t*>(r.more + 1);
    r.pick = r.top + parts * kScanThreads;
    r.part = r.pick + parts * kScanThreads;
    return r;
}

__device__ __forceinline__ uint32_t key_max(uint32_t key) {
    return fni8::wave_max_uniform(key ^ 0x80000000u) ^ 0x80000000u;  // of signed numbers
}

// The value of the lane that a step of a running sum over the lanes adds (0 where there is none),
// by data movement within the vector unit: a round trip through LDS takes ten times as long.
template <int CTRL, int ROWS, class N>
__device__ __forceinline__ N moved(N v) {
    if constexpr (sizeof(N) == 8) {
        u32x2 w = __builtin_bit_cast(u32x2, v);
        w.x = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w.x, CTRL, ROWS, 0xf, false);
        w.y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w.y, CTRL, ROWS, 0xf, false);
        return __builtin_bit_cast(N, w);
    } else {
        return __builtin_bit_cast(
            N, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
    }
}
template <class N>
__device__ __forceinline__ N wave_scan(N v) {
    v += moved<0x111, 0xf>(v);  // row_shr:1, within rows of 16 lanes
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);  // row_bcast:15, a row's end to the next
    v += moved<0x143, 0xc>(v);  // row_bcast:31
    return v;
}
template <class N>
__device__ __forceinline__ N last_lane(N v) {
    if constexpr (sizeof(N) == 8) {
        u32x2 w = __builtin_bit_cast(u32x2, v);
        w.x = (uint32_t)__builtin_amdgcn_readlane((int)w.x, 63);
        w.y = (uint32_t)__builtin_amdgcn_readlane((int)w.y, 63);
        return __builtin_bit_cast(N, w);
    } else {
        return __builtin_bit_cast(N, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
    }
}
template <class N>
__device__ __forceinline__ N wave_sum(N v) {
    return last_lane(wave_scan(v));
}

// A workgroup has a part of a row.  256 rows of 151936 fp16 (77.8 MB): 14.1 us without sums (5.5
// TB/s; a read alone reaches 6.1), 30.9 with them and 32.5 with top-p's samples too, where the
// vector unit bounds it: 18 operations a logit and its sum, 15 of them of 64 bits.
template <class E>
__global__ __launch_bounds__(kScanThreads) void scan_kernel(const fni8h::Sample a, int parts) {
    typedef E vec __attribute__((ext_vector_type(8), aligned(sizeof(E))));
    // maxima keep a NaN, and take two or three 16-bit numbers an operation
    typedef std::conditional_t<sizeof(E) == 2, _Float16, float> number
        __attribute__((ext_vector_type(8)));
    __shared__ uint32_t tops[4];
    __shared__ double sums[4];
    const int V = (int)a.V, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = blockIdx.x / (uint32_t)parts, part = blockIdx.x - row * parts;
    const Work w = work_of(a.work, row, V);
    const E* x = (const E*)a.logits + row * a.ld;
    const int i0 = part * kPart + tid * kVec;
    vec q[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
        const int at = i0 + i * kScanThreads * kVec;
        if (at + kVec <= V) {
            q[i] = *reinterpret_cast<const vec*>(x + at);
        } else {
#pragma unroll
            for (int j = 0; j < kVec; j++) {
                E e = lowest_of<E>();
                if (at + j < V) e = x[at + j];
                q[i][j] = e;
            }
        }
    }
    float v[kSteps][kVec];
    number many = __builtin_bit_cast(number, q[0]);
#pragma unroll
    for (int i = 1; i < kSteps; i++)
        many = __builtin_elementwise_maximum(many, __builtin_bit_cast(number, q[i]));
#pragma unroll
    for (int i = 0; i < kSteps; i++)
#pragma unroll
        for (int j = 0; j < kVec; j++) {
            const E e = q[i][j];
            v[i][j] = value(e);
        }
    auto most = many[0];
#pragma unroll
    for (int j = 1; j < kVec; j++) most = __builtin_elementwise_maximum(most, many[j]);
    uint32_t best = key_of((float)most);
    w.top[part * kScanThreads + tid] = best;
    best = key_max(best);
    if (lane == 0) tops[wave] = best;
    Row r(a, row, V);
    __syncthreads();
    for (int i = 0; i < 4; i++) best = tops[i] > best ? tops[i] : best;
    if (tid == 0) w.part[part] = best;
    if (!r.summed()) return;
    r.largest(value_of(best));
    if (r.inf) {
#pragma unroll
        for (int i = 0; i < kSteps; i++)
#pragma unroll
            for (int j = 0; j < kVec; j++) v[i][j] = r.seen(v[i][j]);
    }
    if (r.by_p) {  // samples, of loads that differ from wave to wave
        float p = 0.0f, q = 0.0f;
#pragma unroll
        for (int i = 0; i < kSteps; i++)
            if (i == (wave & (kSteps - 1))) {
                p = v[i][1];
                q = v[(i + kSteps / 2) % kSteps][6];
            }
        w.pick[part * kScanThreads + tid] =
            (__builtin_bit_cast(uint32_t, p) + 0x8000u) >> 16 |
            ((__builtin_bit_cast(uint32_t, q) + 0x8000u) & 0xffff0000u);
    }
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kSteps; i++)
#pragma unroll
        for (int j = 0; j < kVec; j++) sum += r.weight(v[i][j]);
    sum = wave_sum(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (tid == 0) w.sum[part] = sums[0] + sums[1] + sums[2] + sums[3];
}

struct Candidate {
    u64 order;  // key << 32 | ~index: larger ones come first
    u64 mass;
};
__device__ __forceinline__ uint32_t key_at(const Candidate& c) { return (uint32_t)(c.order >> 32); }
__device__ __forceinline__ uint32_t place_at(const Candidate& c) { return (uint32_t)c.order; }

struct Shared {
    union {
        struct {
            u64 mass[kBins];
            union {
                uint32_t count[kBins];
                u64 hist[256];
            };
        } h;
        uint32_t hits[kHits];
        int bins[kThreads];
        u64 above[kThreads];
    };
    Candidate list[kList], mini[kMini];
    u64 part[2][kWaves], range[kWaves];
    double sums[2][kWaves], before;
    float floats[2][kWaves];
    int ints[2][kWaves], counts[kWaves], highs[kWaves];
    u64 need, all, found;
    uint32_t key;
    int index, n, hits_n, bin, bin2;
};

// Sums over the workgroup take turns with two rows of LDS, so that none has to wait before it
// writes: who writes a row again has passed the barrier of the sum between.
struct Turn {
    int t = 0;
    __device__ __forceinline__ int next() { return t ^= 1; }
};

__device__ __forceinline__ u64 block_sum(Shared& sh, Turn& turn, u64 v) {
    const int row = turn.next();
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) sh.part[row][threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) v += sh.part[row][w];
    return v;
}

// Running sum over the threads, this one's among it, and the sum of all.
template <class N>
__device__ __forceinline__ N block_scan(N (&rows)[2][kWaves], Turn& turn, N v, N& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = turn.next();
    v = wave_scan(v);
    if (lane == 63) rows[row][wave] = v;
    __syncthreads();
    N before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
        const N p = rows[row][w];
        before += w < wave ? p : 0;
        all += p;
    }
    return before + v;
}

// The largest key such that the sum of f over keys no smaller reaches `need` (at least 1; no
// more than the sum of all, or it is lowered to that); `need` is then what the items of that
// key have to bring.  Four passes over the items, eight bits of the key each: for lists that
// are too long otherwise (thousands of equal logits).
template <class K, class F>
__device__ __forceinline__ uint32_t find_key(Shared& sh, int n, u64& need, K key, F f) {
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (threadIdx.x < 256) sh.h.hist[threadIdx.x] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const uint32_t k = key(i);
            if (shift < 24 && (k ^ prefix) >> (shift + 8)) continue;
            const u64 w = f(i);
            if (w) atomicAdd(&sh.h.hist[(k >> shift) & 255], w);
        }
        __syncthreads();
        if (threadIdx.x < 64) {
            const int b = 255 - 4 * (int)threadIdx.x;
            const u64 h0 = sh.h.hist[b], h1 = sh.h.hist[b - 1], h2 = sh.h.hist[b - 2], h3 = sh.h.hist[b - 3];
            u64 run = wave_scan(h0 + h1 + h2 + h3);
            const u64 all = last_lane(run);
            if (need > all) need = all;
            const u64 r3 = run - h3, r2 = r3 - h2, r1 = r2 - h1, r0 = r1 - h0;
            if (r0 < need && run >= need) {
                const int j = r1 >= need ? 0 : r2 >= need ? 1 : r3 >= need ? 2 : 3;
                sh.key = prefix | (uint32_t)(b - j) << shift;
                sh.need = need - (j == 0 ? r0 : j == 1 ? r1 : j == 2 ? r2 : r3);
            }
        }
        __syncthreads();
        prefix = sh.key;
        need = sh.need;
    }
    return prefix;
}

// Finds the first bin of the histogram h.mass at which the running sum reaches `need`, lowered
// to the sum of all (left in `all`); `need` is then what that bin has to bring.
__device__ __forceinline__ int find_bin(Shared& sh, Turn& turn, u64& need) {
    constexpr int B = kBins / kThreads;
    u64 h[B], own = 0, all;
#pragma unroll
    for (int j = 0; j < B; j++) own += h[j] = sh.h.mass[threadIdx.x * B + j];
    u64 run = block_scan(sh.part, turn, own, all) - own;
    if (threadIdx.x == 0) sh.all = all;
    if (need > all) need = all;
#pragma unroll
    for (int j = 0; j < B; j++) {
        if (run < need && run + h[j] >= need) {
            sh.bin = threadIdx.x * B + j;
            sh.need = need - run;
        }
        run += h[j];
    }
    __syncthreads();
    need = sh.need;
    return sh.bin;
}

__device__ __forceinline__ void clear_bins(Shared& sh) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.h.mass[i] = 0;
    __syncthreads();
}

// The candidate of list[0 .. n), weighed by h.mass, at which the running sum reaches `need`, in
// their order or by index; its order goes to `found`.  Not inlined: for buckets with more
// than 64 candidates, mostly equal logits.
__device__ __attribute__((noinline)) void radix_item(Shared* sh, int n, u64 need, bool by_value) {
    __syncthreads();
    auto mass = [&](int i) { return sh->h.mass[i]; };
    uint32_t hi = 0;
    if (by_value) hi = find_key(*sh, n, need, [&](int i) { return key_at(sh->list[i]); }, mass);
    const uint32_t lo = find_key(
        *sh, n, need, [&](int i) { return place_at(sh->list[i]); },
        [&](int i) { return !by_value || key_at(sh->list[i]) == hi ? mass(i) : 0; });
    for (int i = threadIdx.x; i < n; i += kThreads)
        if (place_at(sh->list[i]) == lo && (!by_value || key_at(sh->list[i]) == hi))
            sh->found = sh->list[i].order;
}

// The candidate of list[0 .. n) at which the running sum of f, in the order of `rank` (larger
// ones first, all different), reaches `need`: by buckets (rising in that order), then one wave
// for those of the bucket.  Returns its order.
template <class B, class R, class F>
__device__ __forceinline__ u64 find_item(Shared& sh, Turn& turn, int n, u64 need, B bucket, R rank, F f) {
    const int tid = threadIdx.x;
    __syncthreads();
    clear_bins(sh);
    for (int i = tid; i < n; i += kThreads) {
        const u64 w = f(sh.list[i]);
        if (w) atomicAdd(&sh.h.mass[bucket(sh.list[i])], w);
    }
    if (tid == 0) sh.n = 0;
    __syncthreads();
    const int bin = find_bin(sh, turn, need);
    for (int i = tid; i < n; i += kThreads) {
        const Candidate c = sh.list[i];
        const u64 w = f(c);
        if (!w || bucket(c) != bin) continue;
        const int at = atomicAdd(&sh.n, 1);
        if (at < kMini) sh.mini[at] = {c.order, w};
    }
    __syncthreads();
    const int m = sh.n;
    if (m > kMini) {
        for (int i = tid; i < n; i += kThreads)
            sh.h.mass[i] = bucket(sh.list[i]) == bin ? f(sh.list[i]) : 0;
        radix_item(&sh, n, need, rank(~0ull) >> 32 != 0);
    } else if (tid < m) {
        const Candidate me = sh.mini[tid];
        u64 before = 0;
        for (int j = 0; j < m; j++)
            before += rank(sh.mini[j].order) > rank(me.order) ? sh.mini[j].mass : 0;
        if (before < need && before + me.mass >= need) sh.found = me.order;
    }
    __syncthreads();
    return sh.found;
}

// A place in the order: all keys above `key`, and those equal to it up to index `last`.
struct Cut {
    uint32_t key = 0;
    int last = 0x7fffffff;
    __device__ __forceinline__ bool keeps(uint32_t k, int i) const {
        return k > key || (k == key && i <= last);
    }
};
__device__ __forceinline__ Cut cut_at(u64 order) {
    Cut c;
    c.key = (uint32_t)(order >> 32);
    c.last = (int)~(uint32_t)order;
    return c;
}

// Calls fn(index, logit) for the row's logits i0 .. i1, eight a lane; i0 a multiple of 8.
template <class E, class F>
__device__ __forceinline__ void each(const E* x, int V, const Row& r, int i0, int i1, int who,
                                     int threads, F fn) {
    float next[kVec];
    int i = i0 + who * kVec;
    if (i < i1) load8(x, i, V, r, next);
    while (i < i1) {
        float v[kVec];
#pragma unroll
        for (int j = 0; j < kVec; j++) v[j] = next[j];
        const int at = i;
        i += threads * kVec;
        if (i < i1) load8(x, i, V, r, next);
#pragma unroll
        for (int j = 0; j < kVec; j++) fn(at + j, v[j]);
    }
}

// A wave's run of the row's [lo, hi), in whole loads of a wave.
__device__ __forceinline__ int run_of(int lo, int hi) {
    constexpr int W = 64 * kVec;
    return ((hi - lo + kWaves - 1) / kWaves + W - 1) / W * W;
}

// The first index at which the running sum of f(index, logit) over the row reaches `need` (at
// most the sum of all), the sums of the waves' runs being in sh.range.
template <class E, class F>
__device__ __forceinline__ int find_index(Shared& sh, Turn& turn, const E* x, int V, const Row& r,
                                          u64 need, F f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int lo = 0, hi = V;
    for (;;) {
        const int per = run_of(lo, hi);
        int w = 0;
        for (; w < kWaves - 1 && lo + (w + 1) * per < hi && sh.range[w] < need; w++)
            need -= sh.range[w];
        lo += w * per;
        hi = lo + per < hi ? lo + per : hi;
        if (hi - lo <= kThreads * kVec) break;
        const int next = run_of(lo, hi), i0 = lo + wave * next;
        u64 s = 0;
        each(x, V, r, i0, i0 + next < hi ? i0 + next : hi, lane, 64,
             [&](int i, float v) { s += f(i, v); });
        s = wave_sum(s);
        __syncthreads();
        if (lane == 0) sh.range[wave] = s;
        __syncthreads();
    }
    u64 m[kVec], own = 0, all;
    const int i0 = lo + (int)threadIdx.x * kVec;
    float v[kVec];
    if (i0 < hi) load8(x, i0, V, r, v);
#pragma unroll
    for (int j = 0; j < kVec; j++) own += m[j] = i0 + j < hi ? f(i0 + j, v[j]) : 0;
    u64 run = block_scan(sh.part, turn, own, all) - own;
    if (need > all) need = all;
#pragma unroll
    for (int j = 0; j < kVec; j++) {
        if (run < need && run + m[j] >= need) sh.index = i0 + j;
        run += m[j];
    }
    __syncthreads();
    return sh.index;
}

// The place in the order of the whole row at which the running sum of f(index, logit) reaches
// `need`: a histogram over the steps of weight, then the tokens of one step as a list; over
// the row again where that list is too long.
template <class E, class F>
__device__ __forceinline__ Cut cut_row(Shared& sh, Turn& turn, const E* x, int V, const Row& r, u64 need, F f) {
    __syncthreads();
    clear_bins(sh);
    each(x, V, r, 0, V, threadIdx.x, kThreads, [&](int i, float v) {
        const u64 w = f(i, v);
        if (w) atomicAdd(&sh.h.mass[r.bin(r.power(v))], w);
    });
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    const int bin = find_bin(sh, turn, need);
    each(x, V, r, 0, V, threadIdx.x, kThreads, [&](int i, float v) {
        if (r.bin(r.power(v)) != bin) return;
        const u64 w = f(i, v);
        if (!w) return;
        const int at = atomicAdd(&sh.n, 1);
        if (at < kList) sh.list[at] = {(u64)key_of(v) << 32 | (uint32_t)~i, w};
    });
    __syncthreads();
    const int n = sh.n;
    if (n <= kList)
        return cut_at(find_item(
            sh, turn, n, need,
            [&](const Candidate& c) {
                const double d = -r.power(value_of(key_at(c))) * r.step - bin;
                return (int)(d * (kBins - 1));
            },
            [](u64 order) { return order; }, [](const Candidate& c) { return c.mass; }));
    auto in = [&](int i) {
        const float v = r.seen(value(x[i]));
        return r.bin(r.power(v)) == bin ? f(i, v) : 0;
    };
    auto key = [&](int i) { return key_of(r.seen(value(x[i]))); };
    Cut c;
    c.key = find_key(sh, V, need, key, in);
    c.last = (int)~find_key(sh, V, need, [](int i) { return ~(uint32_t)i; },
                            [&](int i) { return key(i) == c.key ? in(i) : 0; });
    return c;
}

// What a running mass has to reach: the place p of `all`, for top-p; the place of u, for a draw.
__device__ __forceinline__ u64 top_need(float p, double all) {
    const u64 need = p > 0.0f ? (u64)__builtin_ceil((double)p * all) : 1;
    return need ? need : 1;
}
__device__ __forceinline__ u64 draw_need(float u, u64 all) {
    const u64 need = u > 0.0f ? (u64)((double)(u < 1.0f ? u : 1.0f) * (double)all) + 1 : 1;
    return need < all ? need : all;
}

// The token of a row that is searched whole, and the kept mass.
template <class E>
__device__ __forceinline__ int search_row(Shared& sh, Turn& turn, const E* x, int V, const Row& r,
                                          u64 need_p, u64& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const u64 floor = r.floor();
    const bool whole = r.by_p && !r.by_k;
    Cut c;
    auto kept = [&](int i, float v) { return c.keeps(key_of(v), i) ? r.mass(v) : 0; };
    auto drawn = [&](int i, float v) {
        const u64 m = kept(i, v);
        return m >= floor ? m : 0;
    };
    auto sum_of = [&](auto f) {  // and the sums of the waves' runs
        const int per = run_of(0, V), i0 = wave * per;
        u64 s = 0;
        each(x, V, r, i0, i0 + per < V ? i0 + per : V, lane, 64,
             [&](int i, float v) { s += f(i, v); });
        s = wave_sum(s);
        __syncthreads();
        if (lane == 0) sh.range[wave] = s;
        __syncthreads();
        s = 0;
#pragma unroll
        for (int i = 0; i < kWaves; i++) s += sh.range[i];
        return s;
    };
    if (r.by_k)
        c = cut_row(sh, turn, x, V, r, r.k,
                    [&](int, float v) { return (u64)(r.power(v) > -(double)(r.s + 1)); });
    if (r.by_p)
        c = cut_row(sh, turn, x, V, r, whole ? need_p : top_need(r.p, (double)sum_of(kept)), kept);
    all = sum_of(drawn);
    return find_index(sh, turn, x, V, r, draw_need(r.u, all), drawn);
}

// The logits that the end of top-p lies between, as far as the samples tell: two of each
// group of 32, so the mass below a logit is 16 times that of the samples below it, counted in
// steps of weight.  Of `tail`, the mass that top-p leaves out (in units of the largest weight),
// the estimate is off by sqrt(16 w tail) at most (one standard deviation; w the weight at the
// end, the largest of the tail): four of them on either side, and a step for their rounding.
__device__ __forceinline__ void find_ends(Shared& sh, Turn& turn, const Work& w, int groups,
                                          const Row& r, double tail, Long& more) {
    constexpr int B = kBins / kThreads;
    constexpr float f = 16.0f;
    __syncthreads();  // where no list was tried, waves may still have to read the bound in sh.bin
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.h.count[i] = 0;
    if (threadIdx.x == 0) sh.bin = kBins - 2;
    __syncthreads();
    const float rate = (float)(r.rate * r.step);
    auto count = [&](uint32_t bits) {
        const float d = (r.top - __builtin_bit_cast(float, bits)) * rate;
        if (d < (float)(kBins - 1)) atomicAdd(&sh.h.count[d > 0.0f ? (int)d : 0], 1u);
    };
    for (int i0 = threadIdx.x; i0 < groups; i0 += kKeep * kThreads) {
        uint32_t two[kKeep];  // all on their way at once
#pragma unroll
        for (int j = 0; j < kKeep; j++) {
            const int i = i0 + j * kThreads;
            two[j] = i < groups ? w.pick[i] : 0xff80ff80u;  // minus infinity
        }
#pragma unroll
        for (int j = 0; j < kKeep; j++) {
            count(two[j] << 16);
            count(two[j] & 0xffff0000u);
        }
    }
    __syncthreads();
    // from the bottom: a thread's steps are last - j
    const int last = kBins - 1 - (int)threadIdx.x * B;
    const float unit = 1.0f / (float)r.step, goal = (float)tail;
    float m[B], own = 0.0f, all;
#pragma unroll
    for (int j = 0; j < B; j++) {
        const int b = last - j;
        own += m[j] = f * (float)sh.h.count[b] * __builtin_amdgcn_exp2f(-((float)b + 0.5f) * unit);
    }
    const float before = block_scan(sh.floats, turn, own, all) - own;
    // the step in which the mass from the bottom reaches x
    auto reach = [&](float x, int& where) {
        float to = before;
#pragma unroll
        for (int j = 0; j < B; j++) {
            if (to < x && to + m[j] >= x) where = last - j;
            to += m[j];
        }
    };
    reach(goal, sh.bin);
    __syncthreads();
    const int end = sh.bin;
    const float dev = 4.0f * __builtin_sqrtf(f * __builtin_amdgcn_exp2f(-(float)end * unit) * goal);
    __syncthreads();
    if (threadIdx.x == 0) {
        sh.bin = kBins - 3;  // the lowest step with weight, where the tail is too thin to tell
        sh.bin2 = 0;
    }
    __syncthreads();
    reach(goal - dev, sh.bin);
    reach(goal + dev, sh.bin2);
    __syncthreads();
    more.low = r.top - (float)(sh.bin + 2) / rate;
    more.high = sh.bin2 > 0 ? r.top - (float)(sh.bin2 - 1) / rate : r.top;
}

static_assert(kThreads * 2 * kVec == kPart && kPart == kSteps * kScanThreads * kVec, "parts");

// One workgroup a row: a chain of searches, each a few round trips to LDS and the cache, so it is
// bound by their latency, not by bytes (a list of 50 of 151936: 10.1 us for one row; of hundreds,
// 64 rows: 17 us; no filter, 256 rows: 6.7 us; the largest logit, 256 rows: 4.0 us).
// ALONE: no other launch follows, and a row whose list does not fit is searched whole.
template <class E, bool ALONE>
__global__ __launch_bounds__(kThreads) void draw_kernel(const fni8h::Sample a, int parts) {
    __shared__ Shared sh;
    Turn turn;
    const int64_t row = blockIdx.x;
    const E* x = (const E*)a.logits + row * a.ld;
    const int V = (int)a.V, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Work w = work_of(a.work, row, V);

    // parts <= kThreads: a thread each
    if (!ALONE && tid == 0) w.more->kind = kDone;
    const uint32_t own = tid < parts ? w.part[tid] : 0;
    const double own_sum = tid < parts ? w.sum[tid] : 0.0;  // used where the row is summed
    Row r(a, row, V);
    uint32_t best = key_max(own);
    if (lane == 0) sh.counts[wave] = (int)best;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; i++) best = (uint32_t)sh.counts[i] > best ? (uint32_t)sh.counts[i] : best;
    const float top = value_of(best);
    if (best == 0xffffffffu || r.T != r.T || top == -__builtin_inff()) {
        if (tid == 0) {  // a NaN, or nothing to draw
            a.tokens[row] = -1;
            if (a.logprobs) a.logprobs[row] = __builtin_nanf("");
        }
        return;
    }
    r.largest(top);
    auto answer = [&](int token, double share) {  // one thread; the mass in units of the largest
        a.tokens[row] = token;
        if (a.logprobs)
            a.logprobs[row] = (float)(r.power(r.seen(value(x[token]))) * 0.69314718055994531 - log(share));
    };
    // The lowest of the threads' numbers (rising with the thread) that have `first`; where none
    // has, the highest that has `any`.
    auto pick = [&](bool first, bool any, int number) {
        const u64 f = __ballot(first), g = __ballot(any);
        const int lo = __shfl(number, f ? __builtin_ctzll(f) : 0, 64);
        const int hi = __shfl(number, g ? 63 - __builtin_clzll(g) : 0, 64);
        __syncthreads();
        if (lane == 0) {
            sh.counts[wave] = f ? lo : 0x7fffffff;
            sh.highs[wave] = g ? hi : -1;
        }
        __syncthreads();
        int l = 0x7fffffff, h = -1;
#pragma unroll
        for (int i = 0; i < kWaves; i++) {
            l = sh.counts[i] < l ? sh.counts[i] : l;
            h = sh.highs[i] > h ? sh.highs[i] : h;
        }
        return l != 0x7fffffff ? l : h;
    };
    auto load16 = [&](int i0, float (&v)[2 * kVec]) {
        float lo[kVec], hi[kVec];
        load8(x, i0, V, r, lo);
        load8(x, i0 + kVec, V, r, hi);
#pragma unroll
        for (int j = 0; j < kVec; j++) {
            v[j] = lo[j];
            v[j + kVec] = hi[j];
        }
    };
    if (!(r.T > 0.0f)) {  // the first of the largest, in the first part that holds one
        const int i0 = pick(own == best, false, tid) * kPart + tid * 2 * kVec;
        float v[2 * kVec];
        load16(i0, v);
        int at = -1;
#pragma unroll
        for (int j = 2 * kVec - 1; j >= 0; j--)
            if (v[j] == r.top) at = i0 + j;
        at = pick(at >= 0, false, at);
        if (tid == 0) {
            a.tokens[row] = at;
            if (a.logprobs) a.logprobs[row] = 0.0f;
        }
        return;
    }
    double mass = 0.0, part = 0.0, run = 0.0;  // of the row, of this thread's part, up to it
    if (r.summed()) {
        if (tid < parts) part = own_sum * r.weight(r.seen(value_of(own)));
        run = block_scan(sh.sums, turn, part, mass);
    }
    if (!r.by_k && !r.by_p && !r.by_m) {  // no filter: the part, then the token in it
        // the first whose end passes `want`; where rounding leaves none, the last with mass
        const double want = (double)(r.u > 0.0f ? r.u < 1.0f ? r.u : 1.0f : 0.0f) * mass;
        const bool live = part > 0x1p-900;
        const int p = pick(live && run > want, live, tid);
        if (tid == p) sh.before = run - part;
        const int i0 = p * kPart + tid * 2 * kVec;
        float v[2 * kVec];
        load16(i0, v);
        double m[2 * kVec], sum = 0.0, all;
#pragma unroll
        for (int j = 0; j < 2 * kVec; j++) sum += m[j] = r.weight(v[j]);
        run = block_scan(sh.sums, turn, sum, all);
        run = sh.before + (run - sum);
        int at = -1, last = -1;
#pragma unroll
        for (int j = 0; j < 2 * kVec; j++) {
            run += m[j];
            if (m[j] > 0x1p-900) {
                last = i0 + j;
                at = at < 0 && run > want ? last : at;
            }
        }
        const int token = pick(at >= 0, last >= 0, at >= 0 ? at : last);
        if (tid == 0) answer(token, mass);
        return;
    }

    // ---- a bound on the kept prefix, from the threads' maxima
    const double unit = __builtin_ldexp(1.0, r.s);
    const int groups = parts * kScanThreads;
    const bool whole = r.by_p && !r.by_k;  // top-p of the whole mass
    const u64 need_p = whole ? top_need(r.p, mass * unit) : 0;
    const u64 floor = r.floor();
    // The step in which min-p ends, and one more for log2's own rounding: no token further down
    // has a mass that rounds to `floor`.  Top-p after top-k needs the whole mass of top-k.
    int bound = kBins - 2, least = kBins - 2;
    if (floor && !(r.by_k && r.by_p)) {
        least = r.bin(log2((double)floor - 0.5) - r.s) + 1;
        bound = least = least < bound ? least : bound;
    }
    uint32_t keep[kKeep], most = 0;
#pragma unroll
    for (int j = 0; j < kKeep; j++) {
        const int i = tid + j * kThreads;
        keep[j] = i < groups ? w.top[i] : 0;
        most = keep[j] > most ? keep[j] : most;
    }
    for (int i = tid + kKeep * kThreads; i < groups; i += kThreads) {
        const uint32_t key = w.top[i];
        most = key > most ? key : most;
    }
    auto bin_of = [&](uint32_t key) { return r.bin(r.power(r.seen(value_of(key)))); };
    const int mine = most ? bin_of(most) : kBins - 1;
    if (r.by_k && r.k > kShort) {  // the groups' maxima, counted in steps
        for (int i = tid; i < kBins; i += kThreads) sh.h.count[i] = 0;
        if (tid == 0) sh.bin = kBins;
        __syncthreads();
        if (mine <= bound)
            for (int i = tid; i < groups; i += kThreads) {
                const int b = bin_of(w.top[i]);
                if (b <= bound) atomicAdd(&sh.h.count[b], 1u);
            }
        __syncthreads();
        constexpr int B = kBins / kThreads;
        int c[B], some = 0, total;
#pragma unroll
        for (int j = 0; j < B; j++) some += c[j] = (int)sh.h.count[tid * B + j];
        int rank = block_scan(sh.ints, turn, some, total) - some;
#pragma unroll
        for (int j = 0; j < B; j++) {
            if (rank < r.k && rank + c[j] >= r.k) sh.bin = tid * B + j;
            rank += c[j];
        }
        __syncthreads();
        bound = sh.bin < bound ? sh.bin : bound;
    } else if (r.by_k || whole) {
        // One wave, the maxima of the threads' groups: by bisection the first step down to which
        // they are k, or bring top-p's mass (in 32 bits, with room for its error: that only
        // moves the bound), or are kShort.
        sh.bins[tid] = mine;
        __syncthreads();
        if (wave == 0) {
            constexpr int B = kThreads / 64;
            int b[B];
            float m[B];
#pragma unroll
            for (int j = 0; j < B; j++) {
                b[j] = sh.bins[lane + 64 * j];
                m[j] = whole && b[j] < kBins - 1
                           ? __builtin_amdgcn_exp2f(-(float)(b[j] + 1) / (float)r.step) : 0.0f;
            }
            const int want = whole ? kShort : r.k;
            const float goal = (float)((double)need_p / unit) * 1.0001f;
            int lo = 0, hi = bound;  // the answer, if there is one, is in [lo, hi]
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                int count = 0;
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < B; j++) {
                    count += __builtin_popcountll(__ballot(b[j] <= mid));
                    sum += b[j] <= mid ? m[j] : 0.0f;
                }
                bool there = count >= want;
                if (whole && !there) there = wave_sum(sum) >= goal;
                if (there) hi = mid;
                else lo = mid + 1;
            }
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < B; j++) sum += b[j] <= lo ? m[j] : 0.0f;
            sum = wave_sum(sum);
            // The list has more than these maxima (of logits in no order, about 355 tokens where
            // they are 256 of 512): it is tried unless half as much again does not reach the
            // mass (5 us for a list in vain).
            if (lane == 0) sh.bin = whole && lo < least && 1.5f * sum < goal ? -1 : lo;
        }
        __syncthreads();
        bound = sh.bin;
    }
    // ---- the tokens down to the bound, from the groups whose maximum reaches it
    int n = kList + 1;
    if (bound >= 0) {
        // as a logit, a little lower: the list is a first run of the order, at least to the bound
        const double down = r.base - (double)(bound + 1) / (r.step * r.rate);
        const float edge = __builtin_fmaxf((float)(down - __builtin_fabs(down) * 0x1p-22), -0x1.fffffep127f);
        const uint32_t least_key = key_of(r.inf ? __builtin_inff() : edge);
        if (tid == 0) sh.n = sh.hits_n = 0;
        __syncthreads();
        auto hit = [&](uint32_t key, int i) {
            if (key < least_key) return;
            const int at = atomicAdd(&sh.hits_n, 1);
            if (at < kHits) sh.hits[at] = i;
        };
        if (most >= least_key) {
#pragma unroll
            for (int j = 0; j < kKeep; j++)
                if (tid + j * kThreads < groups) hit(keep[j], tid + j * kThreads);
            for (int i = tid + kKeep * kThreads; i < groups; i += kThreads) hit(w.top[i], i);
        }
        __syncthreads();
        const int hits = sh.hits_n;
        if (hits <= kHits) {
            auto first_of = [&](int q) {
                const int group = sh.hits[q / kSteps];
                return group / kScanThreads * kPart +
                       (q % kSteps * kScanThreads + group % kScanThreads) * kVec;
            };
            auto list = [&](int i0, const float (&v)[kVec]) {
#pragma unroll
                for (int j = 0; j < kVec; j++) {
                    if (v[j] < edge) continue;
                    const int at = atomicAdd(&sh.n, 1);
                    if (at < kList) sh.list[at].order = (u64)key_of(v[j]) << 32 | (uint32_t)~(i0 + j);
                }
            };
            for (int q = tid; q < hits * kSteps; q += 2 * kThreads) {  // two loads on their way
                float v[2][kVec];
                const int q1 = q + kThreads, i0 = first_of(q), i1 = first_of(q1 < hits * kSteps ? q1 : q);
                load8(x, i0, V, r, v[0]);
                load8(x, i1, V, r, v[1]);
                list(i0, v[0]);
                if (q1 < hits * kSteps) list(i1, v[1]);
            }
        }
        __syncthreads();
        n = hits <= kHits ? sh.n : kList + 1;
        if (n <= kList) {
            u64 listed = 0;
            for (int i = tid; i < n; i += kThreads)
                listed += sh.list[i].mass = r.mass(value_of(key_at(sh.list[i])));
            // top-p may end below the bound, and does unless the list has the mass
            if (whole && bound < least) {
                if (block_sum(sh, turn, listed) < need_p) n = kList + 1;
            } else {
                __syncthreads();
            }
        }
    }
    if (n <= kMini) {
        // one wave, every pair: a token's rank and the mass before it, then its mass by index
        if (wave) return;
        const Candidate me = lane < n ? sh.list[lane] : Candidate{0, 0};
        const int key = (int)key_at(me), place = (int)place_at(me);
        auto other = [&](u64 v, int j) {
            return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), j) << 32 |
                   (uint32_t)__builtin_amdgcn_readlane((int)v, j);
        };
        int rank = 0;
        u64 before = 0;
        for (int j = 0; j < n; j++) {
            const uint32_t k = (uint32_t)__builtin_amdgcn_readlane(key, j);
            const uint32_t p = (uint32_t)__builtin_amdgcn_readlane(place, j);
            const bool first = k > (uint32_t)key || (k == (uint32_t)key && p > (uint32_t)place);
            rank += first;
            before += first ? other(me.mass, j) : 0;
        }
        bool keep = lane < n && (!r.by_k || rank < r.k);
        const u64 ranked = wave_sum(keep ? me.mass : 0);
        if (r.by_p) keep = keep && before < (whole ? need_p : top_need(r.p, (double)ranked));
        keep = keep && me.mass >= floor;
        const u64 mine = keep ? me.mass : 0, all = wave_sum(mine), need = draw_need(r.u, all);
        u64 to = 0;
        for (int j = 0; j < n; j++) {
            const uint32_t p = (uint32_t)__builtin_amdgcn_readlane(place, j);
            to += p >= (uint32_t)place ? other(mine, j) : 0;
        }
        if (keep && to >= need && to - mine < need) answer((int)~place_at(me), (double)all / unit);
        return;
    }
    u64 all;
    int token;
    if (n <= kList) {
        Cut c;
        auto bucket = [&](const Candidate& i) { return r.bin(r.power(value_of(key_at(i)))); };
        auto order = [](u64 o) { return o; };
        auto kept = [&](const Candidate& i) {
            return c.keeps(key_at(i), (int)~place_at(i)) ? i.mass : 0;
        };
        if (r.by_k)
            c = cut_at(find_item(sh, turn, n, r.k, bucket, order, [](const Candidate&) { return 1ull; }));
        auto sum_of = [&](u64 least) {
            u64 s = 0;
            for (int i = tid; i < n; i += kThreads) {
                const u64 m = kept(sh.list[i]);
                s += m >= least ? m : 0;
            }
            return block_sum(sh, turn, s);
        };
        if (r.by_p) {
            const u64 need = whole ? need_p : top_need(r.p, (double)sum_of(0));
            c = cut_at(find_item(sh, turn, n, need, bucket, order, kept));
        }
        all = sum_of(floor);
        const int shift = 32 - __builtin_clz(V) > 11 ? 32 - __builtin_clz(V) - 11 : 0;
        token = (int)~(uint32_t)find_item(
            sh, turn, n, draw_need(r.u, all),
            [&](const Candidate& i) { return (int)(~place_at(i) >> shift); },
            [](u64 o) { return (u64)(uint32_t)o; },
            [&](const Candidate& i) {
                const u64 m = kept(i);
                return m >= floor ? m : 0;
            });
    } else if constexpr (ALONE) {
        token = search_row(sh, turn, x, V, r, need_p, all);
    } else {  // the long way
        Long more{need_p, 0.0f, 0.0f, kWhole, 0, best};
        if (!r.by_k && !r.by_p) {
            more.kind = kMinP;
            more.low = (float)(r.base - (double)(bound + 2) / (r.step * r.rate));
        }
        if (whole && !r.by_m) {
            more.kind = kTopP;
            find_ends(sh, turn, w, groups, r, mass - (double)need_p / unit, more);
        }
        if (tid == 0) *w.more = more;
        return;
    }
    if (tid == 0) answer(token, (double)all / unit);
}

// One part of a row with a long prefix: the mass of what is kept for certain, and the tokens
// around the end of top-p.  Each wave first moves the logits of its 2048 that are certain next to
// each other in LDS, so that their exponentials, 18 operations, are not computed for the others;
// the few around the end are read again.  256 rows of 151936 fp16 with top-p 0.95, a fifth of
// the logits kept: 30.6 us.  While a workgroup went through several parts it was 36, 56 with the
// exponentials of all, and 43 with the logits loaded only once the row is known to need them and
// the row's largest found again by each workgroup (two changes at once).  The early loads are
// in vain for rows whose prefix is short: 256 of them, 12.2 us.
template <class E>
__global__ __launch_bounds__(kScanThreads) void gather_kernel(const fni8h::Sample a, int parts) {
    constexpr int W = 64 * kVec * kSteps;  // logits of a wave
    typedef E vec __attribute__((ext_vector_type(8), aligned(sizeof(E))));
    __shared__ E logit[4][W];
    __shared__ u64 sums[4];
    const int V = (int)a.V;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row = blockIdx.x / (uint32_t)parts, part = blockIdx.x - row * parts;
    Row r(a, row, V);
    if (!(r.T > 0.0f) || r.by_k || !(r.by_p || r.by_m)) return;
    const Work w = work_of(a.work, row, V);
    // with top-p, the logits are on their way before it is known that the row needs them
    if (!r.by_p && w.more->kind != kMinP) return;
    const E* x = (const E*)a.logits + (int64_t)row * a.ld;
    const int i0 = part * kPart + wave * 64 * kVec;  // of the wave's first load
    vec v[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
        const int at = i0 + (i * kScanThreads + lane) * kVec;
        if (at + kVec <= V) {
            v[i] = *reinterpret_cast<const vec*>(x + at);
        } else {
#pragma unroll
            for (int j = 0; j < kVec; j++) {
                E e = lowest_of<E>();
                if (at + j < V) e = x[at + j];
                v[i][j] = e;
            }
        }
    }
    const Long more = *w.more;
    if (more.kind != kTopP && more.kind != kMinP) return;
    r.largest(value_of(more.top));
    if (r.inf) {
#pragma unroll
        for (int i = 0; i < kSteps; i++)
#pragma unroll
            for (int j = 0; j < kVec; j++) {
                const E e = v[i][j];
                v[i][j] = element<E>(r.seen(value(e)));
            }
    }
    const u64 floor = more.kind == kMinP ? r.floor() : 0;
    const float low = __builtin_fmaxf(more.low, -0x1.fffffep127f);
    const float high = more.kind == kMinP ? low : __builtin_fmaxf(more.high, low);
    int n = 0;
    uint32_t near = 0;  // this lane's around the end
#pragma unroll
    for (int i = 0; i < kSteps; i++)
#pragma unroll
        for (int j = 0; j < kVec; j++) {
            const E e = v[i][j];
            const float q = value(e);
            const bool sure = q >= high;
            const u64 has = __ballot(sure);
            if (sure)
                logit[wave][__builtin_amdgcn_mbcnt_hi(
                    (uint32_t)(has >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)has, n))] = e;
            n += __builtin_popcountll(has);
            near |= (uint32_t)(q >= low && !sure) << (i * kVec + j);
        }
    const int some = __builtin_popcount(near), upto = wave_scan(some), around = last_lane(upto);
    // where there is no room for them the count tells finish, which searches the whole row
    int first = 0;  // on its way while the sums are made
    if (around && lane == 0) first = atomicAdd(&w.more->around, around);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    u64 sum = 0;
    for (int t = lane; t < n; t += 64) {
        const u64 m = r.mass(value(logit[wave][t]));
        sum += m >= floor ? m : 0;
    }
    sum = wave_sum(sum);
    if (around) {
        const int room = around_of(V);
        int to = __builtin_amdgcn_readfirstlane(first) + upto - some;
        for (; near; near &= near - 1, to++) {
            const int b = __builtin_ctz(near);
            const int index = i0 + (b / kVec * kScanThreads + lane) * kVec + b % kVec;
            if (to < room)
                w.around[to] = (u64)key_of(r.seen(value(x[index]))) << 32 | (uint32_t)~index;
        }
    }
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (tid == 0) w.above[part] = sums[0] + sums[1] + sums[2] + sums[3];
}

// One workgroup a row with a long prefix: the list that gather left, in registers, gives the end
// of top-p; the masses of the parts, with what the list brings to each, the part that the draw
// falls into; its 8192 logits the token.  Bound by the latency of these steps, as draw is: 12 us
// for 5 rows of 50257, 20 for 256 of 151936 (23 with the list's neighbours in different threads,
// whose sums then have to be joined by the wave).
template <class E>
__global__ __launch_bounds__(kThreads) void finish_kernel(const fni8h::Sample a, int parts) {
    __shared__ Shared sh;
    Turn turn;
    const int64_t row = blockIdx.x;
    const int V = (int)a.V;
    const Work w = work_of(a.work, row, V);
    const Long more = *w.more;
    if (more.kind == kDone) return;
    const E* x = (const E*)a.logits + row * a.ld;
    const int tid = threadIdx.x;
    Row r(a, row, V);
    r.largest(value_of(more.top));
    const u64 floor = r.floor();
    u64 all = 0;
    int token = -1;
    bool found = false;
    if (more.kind != kWhole) {
        u64 mine = tid < parts ? w.above[tid] : 0;
        Cut c;
        found = true;
        if (more.kind == kTopP) {
            // the end of top-p in the list: a step of weight, then the tokens of that step
            constexpr int HELD = kAround / kThreads;
            const u64 certain = block_sum(sh, turn, mine);
            const int n = more.around;
            found = certain < more.need && n <= around_of(V);
            if (found) {
                const double p0 = r.power(more.high);
                // no token of the list weighs less than 2^-(s + 2)
                const double p1 = r.power(more.low), deep = -(double)(r.s + 2);
                const double steps = (kBins - 1) / (p0 - (p1 > deep ? p1 : deep));
                auto bin = [&](double t) {
                    const double d = (p0 - t) * steps;
                    return d < (double)(kBins - 1) ? (int)d : kBins - 1;
                };
                auto logit = [](u64 order) { return value_of((uint32_t)(order >> 32)); };
                // the list: read once, weighed once, neighbours to a thread
                u64 order[HELD], m[HELD];
                const int per = (n + kThreads - 1) / kThreads;
#pragma unroll
                for (int j = 0; j < HELD; j++)
                    if (j < per) order[j] = tid * per + j < n ? w.around[tid * per + j] : 0;
                clear_bins(sh);
#pragma unroll
                for (int j = 0; j < HELD; j++)
                    if (j < per) {
                        const float v = logit(order[j]);
                        m[j] = order[j] ? r.mass(v) : 0;
                        if (m[j]) atomicAdd(&sh.h.mass[bin(r.power(v))], m[j]);
                    }
                if (tid == 0) sh.n = 0;
                __syncthreads();
                u64 need = more.need - certain;
                const u64 wanted = need;
                const int b = find_bin(sh, turn, need);
#pragma unroll
                for (int j = 0; j < HELD; j++)
                    if (j < per && m[j] && bin(r.power(logit(order[j]))) == b) {
                        const int at = atomicAdd(&sh.n, 1);
                        if (at < kList) sh.list[at] = {order[j], m[j]};
                    }
                __syncthreads();
                const int few = sh.n;
                found = few <= kList && sh.all >= wanted;
                if (found)
                    c = cut_at(find_item(
                        sh, turn, few, need,
                        [&](const Candidate& i) {
                            const double d = (p0 - r.power(logit(i.order))) * steps - b;
                            return d < 1.0 ? (int)(d * (kBins - 1)) : kBins - 1;
                        },
                        [](u64 o) { return o; }, [](const Candidate& i) { return i.mass; }));
                // what the list brings to each part
                __syncthreads();
                sh.above[tid] = mine;
                __syncthreads();
                if (found) {  // neighbours are of one part, or of a few: a sum for each
                    u64 some = 0;
                    int at = 0;
#pragma unroll
                    for (int j = 0; j < HELD; j++)
                        if (j < per && m[j]) {
                            const int index = (int)~(uint32_t)order[j];
                            if (index / kPart != at) {
                                if (some) atomicAdd(&sh.above[at], some);
                                some = 0;
                                at = index / kPart;
                            }
                            some += c.keeps((uint32_t)(order[j] >> 32), index) ? m[j] : 0;
                        }
                    if (some) atomicAdd(&sh.above[at], some);
                }
                __syncthreads();
                mine = sh.above[tid];
            }
        }
        if (found) {  // the part, then the token in it
            u64 run = block_scan(sh.part, turn, mine, all);
            u64 need = draw_need(r.u, all);
            if (run >= need && run - mine < need) {
                sh.bin = tid;
                sh.need = need - (run - mine);
            }
            __syncthreads();
            need = sh.need;
            const int i0 = sh.bin * kPart + tid * 2 * kVec;
            u64 m[2 * kVec], some = 0, total;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float v[kVec];
                load8(x, i0 + h * kVec, V, r, v);
#pragma unroll
                for (int j = 0; j < kVec; j++) {
                    const u64 q = c.keeps(key_of(v[j]), i0 + h * kVec + j) ? r.mass(v[j]) : 0;
                    some += m[h * kVec + j] = q >= floor ? q : 0;
                }
            }
            run = block_scan(sh.part, turn, some, total) - some;
#pragma unroll
            for (int j = 0; j < 2 * kVec; j++) {
                if (run < need && run + m[j] >= need) sh.index = i0 + j;
                run += m[j];
            }
            __syncthreads();
            token = sh.index;
        }
    }
    if (!found) token = search_row(sh, turn, x, V, r, more.need, all);
    if (tid == 0) {
        a.tokens[row] = token;
        if (a.logprobs)
            a.logprobs[row] = (float)(r.power(r.seen(value(x[token]))) * 0.69314718055994531 -
                                      log((double)all * __builtin_ldexp(1.0, -r.s)));
    }
}

template <class E>
void launch(const fni8h::Sample& a, hipStream_t st) {
    const int parts = (int)parts_of(a.V);
    const uint32_t grid = (uint32_t)(a.B * parts);
    scan_kernel<E><<<grid, kScanThreads, 0, st>>>(a, parts);
    // no filter, the largest logit, or top-k of a few: no prefix is long but for equal logits
    const bool alone = (!a.temperature && !(a.temperature1 > 0.0f)) ||
                       (!a.top_k && a.top_k1 > 0 && a.top_k1 <= kShort) ||
                       (!a.top_k && !a.top_p && !a.min_p && a.top_k1 <= 0 && !(a.top_p1 < 1.0f) &&
                        !(a.min_p1 > 0.0f));
    if (alone) {
        draw_kernel<E, true><<<(uint32_t)a.B, kThreads, 0, st>>>(a, parts);
        return;
    }
    draw_kernel<E, false><<<(uint32_t)a.B, kThreads, 0, st>>>(a, parts);
    gather_kernel<E><<<grid, kScanThreads, 0, st>>>(a, parts);
    finish_kernel<E><<<(uint32_t)a.B, kThreads, 0, st>>>(a, parts);
}

}  // namespace

namespace fni8h {

int64_t sample_workspace_bytes(int64_t B, int64_t V) {
    const int64_t most = rows_at_once(V);
    return (B < most ? B : most) * row_bytes(V);
}

int launch_sample(const Sample& a, hipStream_t st) {
    if (a.B == 0) return FNI8_OK;
    const int64_t most = rows_at_once(a.V);
    for (int64_t row = 0; row < a.B; row += most) {
        Sample some = a;
        some.B = a.B - row < most ? a.B - row : most;
        some.logits = (const int8_t*)a.logits + row * a.ld * (a.fp32 ? 4 : 2);
        if (a.u) some.u = a.u + row;
        if (a.temperature) some.temperature = a.temperature + row;
        if (a.top_k) some.top_k = a.top_k + row;
        if (a.top_p) some.top_p = a.top_p + row;
        if (a.min_p) some.min_p = a.min_p + row;
        some.tokens = a.tokens + row;
        if (a.logprobs) some.logprobs = a.logprobs + row;
        if (a.fp32) launch<float>(some, st);
        else launch<uint16_t>(some, st);
    }
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) {
        set_error_detail("sample launch: %s", hipGetErrorString(err));
        return FNI8_ERR_LAUNCH;
    }
    return FNI8_OK;
}

}  // namespace fni8h
