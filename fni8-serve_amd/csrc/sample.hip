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
// Two launches:
//   scan  reads the logits once, 8192 to a workgroup: the largest logit of each thread's 32
//         and, where a row needs its whole mass, the sum of the part's weights in 64 bits
//   draw  one workgroup a row: the threads' maxima bound the kept prefix from below (k of them
//         are k tokens; those down to some logit have a mass), so only the few groups of 32
//         that reach over that bound are read again, and all searches run over a short list
// A row whose prefix is long (thousands of tokens) is searched whole: a histogram of its mass
// in steps of 1/40 bit of weight, then the list of one step.
// Nothing depends on the number of rows: a row's token is the same in every batch.
#include "common.h"

namespace {

typedef unsigned long long u64;

constexpr int kPart = 8192, kScanThreads = 256, kVec = 8;   // logits of a part; a thread's vectors
constexpr int kSteps = kPart / (kScanThreads * kVec);       // vectors of a thread
constexpr int kThreads = 1024, kWaves = 16;                 // draw
constexpr int kBins = 2048;   // steps of weight; the last one: weights that round to 0
constexpr int kList = 2048;   // candidates in LDS
constexpr int kPairs = 512;   // up to here every pair of candidates is compared
constexpr int kHits = 4096;   // groups that are read again
constexpr int kEnough = 1024; // maxima that a top-p bound may take before the list is tried

// 2^t for t <= 0: t = n + f, |f| <= 1/2; 2^f by its Taylor polynomial in f ln 2, degree 11 (the
// first term left out is below 2^-47).
__device__ __forceinline__ double exp2_part(double t, int& n) {
    const double r = __builtin_rint(t), f = t - r;
    n = (int)r;
    double p = 4.4455382718708101e-10;               // ln2^11 / 11!
    p = __builtin_fma(p, f, 7.0549116208011209e-9);  // ln2^10 / 10!
    p = __builtin_fma(p, f, 1.0178086009239696e-7);
    p = __builtin_fma(p, f, 1.3215486790144305e-6);
    p = __builtin_fma(p, f, 1.5252733804059838e-5);
    p = __builtin_fma(p, f, 1.5403530393381606e-4);
    p = __builtin_fma(p, f, 1.3333558146428441e-3);
    p = __builtin_fma(p, f, 9.6181291076284769e-3);
    p = __builtin_fma(p, f, 5.5504108664821576e-2);
    p = __builtin_fma(p, f, 0.24022650695910070);
    p = __builtin_fma(p, f, 0.69314718055994531);
    return __builtin_fma(p, f, 1.0);
}

__device__ __forceinline__ double exp2_neg(double t) {
    if (!(t > -256.0)) return 0.0;  // nothing beside a largest weight of 1
    int n;
    const double p = exp2_part(t, n);
    return __builtin_ldexp(p, n);
}

// 2^t * 2^s as an integer, rounded, for s <= 50: adding 2^52 leaves it in the sum's low bits.
__device__ __forceinline__ u64 exp2_fixed(double t, int s) {
    if (!(t > -(double)(s + 2))) return 0;
    int n;
    const double p = exp2_part(t, n);
    return __builtin_bit_cast(u64, __builtin_ldexp(p, n + s) + 0x1p52) & 0xfffffffffffffull;
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
    double rate;
    bool inf, by_k, by_p, by_m;

    __device__ Row(const fni8h::Sample& a, int64_t row, int V) {
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
    }
    // Every weight of the row is summed: for top-p without top-k, and without any filter.
    __device__ bool summed() const { return T > 0.0f && !by_k && (by_p || !by_m); }
    __device__ void largest(float x) {
        top = x;
        inf = x == __builtin_inff();
        rate = 1.4426950408889634 / (double)T;
    }
    // log2 of a logit's weight
    __device__ __forceinline__ double power(float v) const {
        if (inf) return v == top ? 0.0 : -__builtin_inf();
        if (v == -__builtin_inff()) return -__builtin_inf();
        return ((double)v - (double)top) * rate;
    }
    // Step of a weight, rising as it falls; kBins - 1 for weights that round to 0.
    __device__ __forceinline__ int bin(double power) const {
        const double d = -power * ((kBins - 2) / (double)(s + 2));
        return d < (double)(kBins - 1) ? (int)d : kBins - 1;
    }
};

// What scan leaves of a row, in the workspace.
struct Work {
    uint32_t* top;   // [parts][256] keys of the threads' largest logits
    uint32_t* part;  // [parts] keys of the parts' largest
    double* sum;     // [parts] masses, relative to the part's largest logit
};
__host__ __device__ inline int64_t parts_of(int64_t V) { return (V + kPart - 1) / kPart; }
__host__ __device__ inline int64_t row_bytes(int64_t parts) {
    return (parts * (8 + 4 + 4 * kScanThreads) + 15) / 16 * 16;
}
__device__ inline Work work_of(int8_t* w, int64_t row, int64_t parts) {
    w += row * row_bytes(parts);
    Work r;
    r.sum = reinterpret_cast<double*>(w);
    r.top = reinterpret_cast<uint32_t*>(w + parts * 8);
    r.part = r.top + parts * kScanThreads;
    return r;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}
__device__ __forceinline__ u64 wave_sum(u64 v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}
template <class N>
__device__ __forceinline__ N wave_scan(N v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const N o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    return v;
}

template <class E>
__global__ __launch_bounds__(kScanThreads) void scan_kernel(const fni8h::Sample a, int parts) {
    __shared__ uint32_t tops[4];
    __shared__ double sums[4];
    const int part = blockIdx.x, V = (int)a.V, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.y + (int64_t)blockIdx.z * 32768;
    if (row >= a.B) return;
    const E* x = (const E*)a.logits + row * a.ld;
    const Work w = work_of(a.work, row, parts);
    float v[kSteps][kVec];
#pragma unroll
    for (int i = 0; i < kSteps; i++)
        load8(x, part * kPart + (i * kScanThreads + (int)threadIdx.x) * kVec, V, v[i]);
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < kSteps; i++)
#pragma unroll
        for (int j = 0; j < kVec; j++) {
            const uint32_t key = key_of(v[i][j]);
            best = key > best ? key : best;
        }
    w.top[part * kScanThreads + threadIdx.x] = best;
    best = fni8::wave_max_u32(best);
    if (lane == 0) tops[wave] = best;
    Row r(a, row, V);
    __syncthreads();
    for (int i = 0; i < 4; i++) best = tops[i] > best ? tops[i] : best;
    if (threadIdx.x == 0) w.part[part] = best;
    if (!r.summed()) return;
    r.largest(value_of(best));
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kSteps; i++)
#pragma unroll
        for (int j = 0; j < kVec; j++) sum += exp2_neg(r.power(v[i][j]));
    sum = wave_sum(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) w.sum[part] = sums[0] + sums[1] + sums[2] + sums[3];
}

struct Candidate {
    u64 order;  // key << 32 | ~index: larger ones come first
    u64 mass;
};

struct Shared {
    union {
        struct {
            u64 mass[kBins];
            uint32_t count[kBins];
        } h;
        uint32_t hits[kHits];
        struct {
            u64 before[kPairs];
            uint32_t rank[kPairs];
        } pair;
    };
    Candidate list[kList];
    u64 hist[256];
    u64 part[kWaves];
    double sums[kWaves];
    u64 need, total, kept, all;
    uint32_t key;
    int index, n, hits_n, bin;
};

// The sum over the workgroup, the same in every thread, added in one order.
template <class N>
__device__ N block_sum(N* part, N v) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < kWaves; w++) v += part[w];
    return v;
}

template <class F>
__device__ u64 sum_of(Shared& sh, int n, F f) {
    u64 s = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) s += f(i);
    return block_sum(sh.part, s);
}

// The first index at which the running sum of f reaches `need` (1 to the sum of all).
template <class F>
__device__ int find_index(Shared& sh, int n, u64 need, F f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int lo = 0, hi = n;
    while (hi - lo > kThreads) {
        const int per = ((hi - lo + kWaves - 1) / kWaves + 63) & ~63;
        const int i0 = lo + wave * per, i1 = i0 + per < hi ? i0 + per : hi;
        u64 s = 0;
        for (int i = i0 + lane; i < i1; i += 64) s += f(i);
        s = wave_sum(s);
        __syncthreads();
        if (lane == 0) sh.part[wave] = s;
        __syncthreads();
        int w = 0;
        for (; w < kWaves - 1 && lo + (w + 1) * per < hi && sh.part[w] < need; w++)
            need -= sh.part[w];
        lo += w * per;
        hi = lo + per < hi ? lo + per : hi;
    }
    const int i = lo + threadIdx.x;
    const u64 own = i < hi ? f(i) : 0;
    u64 run = wave_scan(own, lane);
    __syncthreads();
    if (lane == 63) sh.part[wave] = run;
    if (threadIdx.x == 0) sh.index = hi - 1;
    __syncthreads();
    for (int w = 0; w < wave; w++) run += sh.part[w];
    if (run >= need && run - own < need) sh.index = i;
    __syncthreads();
    return sh.index;
}

// The largest key such that the sum of f over keys no smaller reaches `need` (at least 1; no
// more than the sum of all, or it is lowered to that); `need` is then what the items of that
// key have to bring, `total` what they hold.
template <class K, class F>
__device__ uint32_t find_key(Shared& sh, int n, u64& need, u64& total, K key, F f) {
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (threadIdx.x < 256) sh.hist[threadIdx.x] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const uint32_t k = key(i);
            if (shift < 24 && (k ^ prefix) >> (shift + 8)) continue;
            const u64 w = f(i);
            if (w) atomicAdd(&sh.hist[(k >> shift) & 255], w);
        }
        __syncthreads();
        if (threadIdx.x < 64) {
            const int lane = threadIdx.x;
            u64 h[4], own = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) own += h[j] = sh.hist[255 - 4 * lane - j];
            u64 run = wave_scan(own, lane);
            const u64 all = __shfl(run, 63, 64);
            if (need > all) need = all;
            run -= own;
            if (run < need && run + own >= need) {
                for (int j = 0; j < 4; j++) {
                    if (run + h[j] >= need) {
                        sh.key = prefix | (uint32_t)(255 - 4 * lane - j) << shift;
                        sh.need = need - run;
                        sh.total = h[j];
                        break;
                    }
                    run += h[j];
                }
            }
        }
        __syncthreads();
        prefix = sh.key;
        need = sh.need;
    }
    total = sh.total;
    return prefix;
}

// A place in the order: all keys above `key`, and those equal to it up to index `last`.
struct Cut {
    uint32_t key;
    int last;
    __device__ __forceinline__ bool keeps(uint32_t k, int i) const {
        return k > key || (k == key && i <= last);
    }
};

// The place in the order of the whole row at which the running sum of f(index, key, power)
// reaches `need`: a histogram over the steps of weight, then the tokens of one step as a list;
// over the row again where that list is too long (many equal logits).
template <class E, class F>
__device__ Cut cut_row(Shared& sh, const E* x, int V, const Row& r, u64 need, F f) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.h.mass[i] = 0;
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < V; i += kThreads) {
        const float v = value(x[i]);
        const double t = r.power(v);
        const u64 w = f(i, key_of(v), t);
        if (w) atomicAdd(&sh.h.mass[r.bin(t)], w);
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x, b0 = lane * (kBins / 64);
        u64 own = 0;
        for (int b = 0; b < kBins / 64; b++) own += sh.h.mass[b0 + b];
        u64 run = wave_scan(own, lane);
        const u64 all = __shfl(run, 63, 64);
        if (need > all) need = all;
        run -= own;
        if (run < need && run + own >= need) {
            int b = b0;
            for (; run + sh.h.mass[b] < need; b++) run += sh.h.mass[b];
            sh.bin = b;
            sh.need = need - run;
        }
    }
    __syncthreads();
    const int bin = sh.bin;
    need = sh.need;
    for (int i = threadIdx.x; i < V; i += kThreads) {
        const float v = value(x[i]);
        const double t = r.power(v);
        if (r.bin(t) != bin) continue;
        const uint32_t key = key_of(v);
        const u64 w = f(i, key, t);
        if (!w) continue;
        const int at = atomicAdd(&sh.n, 1);
        if (at < kList) sh.list[at] = {(u64)key << 32 | (uint32_t)~i, w};
    }
    __syncthreads();
    const int n = sh.n;
    Cut c;
    u64 total;
    if (n > kList) {
        auto key = [&](int i) { return key_of(value(x[i])); };
        auto in = [&](int i) {
            const float v = value(x[i]);
            const double t = r.power(v);
            return r.bin(t) == bin ? f(i, key_of(v), t) : 0;
        };
        c.key = find_key(sh, V, need, total, key, in);
        c.last = find_index(sh, V, need, [&](int i) { return key(i) == c.key ? in(i) : 0; });
    } else {
        c.key = find_key(sh, n, need, total, [&](int i) { return (uint32_t)(sh.list[i].order >> 32); },
                         [&](int i) { return sh.list[i].mass; });
        c.last = (int)~find_key(
            sh, n, need, total, [&](int i) { return (uint32_t)sh.list[i].order; },
            [&](int i) { return (uint32_t)(sh.list[i].order >> 32) == c.key ? sh.list[i].mass : 0; });
    }
    __syncthreads();
    return c;
}

// What a running mass has to reach for u of `all`.
__device__ __forceinline__ u64 drawn_need(float u, u64 all) {
    const u64 need = u > 0.0f ? (u64)((double)(u < 1.0f ? u : 1.0f) * (double)all) + 1 : 1;
    return need < all ? need : all;
}

static_assert(kThreads * kVec == kPart && kPart == kSteps * kScanThreads * kVec, "parts");

template <class E>
__global__ __launch_bounds__(kThreads) void draw_kernel(const fni8h::Sample a, int parts) {
    __shared__ Shared sh;
    const int64_t row = blockIdx.x;
    const E* x = (const E*)a.logits + row * a.ld;
    const int V = (int)a.V, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Work w = work_of(a.work, row, parts);
    Row r(a, row, V);

    const uint32_t own = (int)threadIdx.x < parts ? w.part[threadIdx.x] : 0;
    uint32_t best = fni8::wave_max_u32(own);
    if (lane == 0) sh.part[wave] = best;
    __syncthreads();
    for (int i = 0; i < kWaves; i++) best = sh.part[i] > best ? (uint32_t)sh.part[i] : best;
    const float top = value_of(best);
    auto answer = [&](int token, u64 all, double mass) {
        // one thread: the token, and the logarithm of its share of the mass
        a.tokens[row] = token;
        if (a.logprobs)
            a.logprobs[row] = (float)(r.power(value(x[token])) * 0.69314718055994531 -
                                      log(all ? (double)all * __builtin_ldexp(1.0, -r.s) : mass));
    };
    if (best == 0xffffffffu || r.T != r.T || top == -__builtin_inff()) {
        if (threadIdx.x == 0) {  // a NaN, or nothing to draw
            a.tokens[row] = -1;
            if (a.logprobs) a.logprobs[row] = __builtin_nanf("");
        }
        return;
    }
    r.largest(top);
    if (!(r.T > 0.0f)) {  // the first of the largest, in the first part that holds one
        if (threadIdx.x == 0) sh.index = V;
        __syncthreads();
        if (own == best) atomicMin(&sh.index, (int)threadIdx.x);
        __syncthreads();
        const int first = sh.index * kPart;
        float v[kVec];
        load8(x, first + (int)threadIdx.x * kVec, V, v);
        __syncthreads();
        if (threadIdx.x == 0) sh.index = V;
        __syncthreads();
        int at = V;
        for (int j = kVec - 1; j >= 0; j--)
            if (key_of(v[j]) == best) at = first + (int)threadIdx.x * kVec + j;
        if (at < V) atomicMin(&sh.index, at);
        __syncthreads();
        if (threadIdx.x == 0) {
            a.tokens[row] = sh.index;
            if (a.logprobs) a.logprobs[row] = 0.0f;
        }
        return;
    }
    double mass = 0.0, part = 0.0;  // of the row, of this thread's part; relative to the largest
    if (r.summed()) {
        if ((int)threadIdx.x < parts)
            part = w.sum[threadIdx.x] * exp2_neg(r.power(value_of(own)));
        mass = block_sum(sh.sums, part);
    }
    if (!r.by_k && !r.by_p && !r.by_m) {  // no filter: the part, then the token in it
        const double want = (double)(r.u > 0.0f ? r.u < 1.0f ? r.u : 1.0f : 0.0f) * mass;
        double run = wave_scan(part, lane);
        __syncthreads();
        if (lane == 63) sh.sums[wave] = run;
        if (threadIdx.x == 0) sh.index = -1;
        __syncthreads();
        for (int i = 0; i < wave; i++) run += sh.sums[i];
        // the first part whose end passes `want`; rounding may leave none: the last with mass
        const bool past = run > want && part > 0.0;
        if (threadIdx.x == 0) sh.bin = parts;
        __syncthreads();
        if (past) atomicMin(&sh.bin, (int)threadIdx.x);
        if (part > 0.0) atomicMax(&sh.index, (int)threadIdx.x);
        __syncthreads();
        const int p = sh.bin < parts ? sh.bin : sh.index;
        if ((int)threadIdx.x == p) sh.sums[0] = run - part;
        __syncthreads();
        const double before = sh.sums[0];
        float v[kVec];
        double m[kVec], sum = 0.0;
        const int i0 = p * kPart + (int)threadIdx.x * kVec;
        load8(x, i0, V, v);
#pragma unroll
        for (int j = 0; j < kVec; j++) sum += m[j] = exp2_neg(r.power(v[j]));
        run = wave_scan(sum, lane);
        __syncthreads();
        if (lane == 63) sh.sums[wave] = run;
        if (threadIdx.x == 0) {
            sh.index = -1;
            sh.bin = V;
        }
        __syncthreads();
        double base = before;
        for (int i = 0; i < wave; i++) base += sh.sums[i];
        run = base + (run - sum);
        int at = V, last = -1;
#pragma unroll
        for (int j = 0; j < kVec; j++) {
            run += m[j];
            if (m[j] > 0.0) {
                last = i0 + j;
                if (run > want && at == V) at = i0 + j;
            }
        }
        if (at < V) atomicMin(&sh.bin, at);
        if (last >= 0) atomicMax(&sh.index, last);
        __syncthreads();
        if (threadIdx.x == 0) answer(sh.bin < V ? sh.bin : sh.index, 0, mass);
        return;
    }

    // ---- a bound on the kept prefix, from the threads' maxima
    const double unit = __builtin_ldexp(1.0, r.s);
    const int groups = parts * kScanThreads;
    u64 need_p = 0;
    if (r.by_p && !r.by_k) {
        need_p = r.p > 0.0f ? (u64)__builtin_ceil((double)r.p * (mass * unit)) : 1;
        need_p = need_p ? need_p : 1;
    }
    const u64 floor = (u64)__builtin_rint((double)r.least * unit);
    // The step in which min-p ends, and one more for log2's own rounding: no token further down
    // has a mass that rounds to `floor`.  Top-p after top-k needs the whole mass of top-k.
    int bound = kBins - 2, least = kBins - 2;
    if (floor && !(r.by_k && r.by_p)) {
        least = r.bin(log2((double)floor - 0.5) - r.s) + 1;
        bound = least = least < bound ? least : bound;
    }
    if (r.by_k || r.by_p) {
        for (int i = threadIdx.x; i < kBins; i += kThreads) {
            sh.h.mass[i] = 0;
            sh.h.count[i] = 0;
        }
        if (threadIdx.x == 0) sh.bin = kBins;
        __syncthreads();
        for (int i = threadIdx.x; i < groups; i += kThreads) {
            const double t = r.power(value_of(w.top[i]));
            const int b = r.bin(t);
            if (b > bound) continue;
            atomicAdd(&sh.h.count[b], 1u);
            if (!r.by_k) atomicAdd(&sh.h.mass[b], exp2_fixed(t, r.s));
        }
        __syncthreads();
        // two steps a thread; the first at which the count or the mass is there
        const uint32_t want = r.by_k ? (uint32_t)r.k : kEnough;
        const int b = 2 * threadIdx.x;
        const uint32_t c0 = sh.h.count[b], c1 = sh.h.count[b + 1];
        const u64 m0 = sh.h.mass[b], m1 = sh.h.mass[b + 1];
        int runc = fni8::wave_incl_scan_i32((int)(c0 + c1), lane);
        u64 runm = wave_scan(m0 + m1, lane);
        __shared__ int counts[kWaves];
        if (lane == 63) {
            counts[wave] = runc;
            sh.part[wave] = runm;
        }
        __syncthreads();
        for (int i = 0; i < wave; i++) {
            runc += counts[i];
            runm += sh.part[i];
        }
        auto there = [&](uint32_t c, u64 m) { return c >= want || (!r.by_k && m >= need_p); };
        if (there((uint32_t)runc - c1, runm - m1)) atomicMin(&sh.bin, b);
        else if (there((uint32_t)runc, runm)) atomicMin(&sh.bin, b + 1);
        __syncthreads();
        bound = sh.bin < bound ? sh.bin : bound;
    }
    // ---- the tokens down to the bound, from the groups whose maximum reaches it
    __syncthreads();
    if (threadIdx.x == 0) sh.n = sh.hits_n = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < groups; i += kThreads) {
        if (r.bin(r.power(value_of(w.top[i]))) > bound) continue;
        const int at = atomicAdd(&sh.hits_n, 1);
        if (at < kHits) sh.hits[at] = i;
    }
    __syncthreads();
    const int hits = sh.hits_n;
    if (hits <= kHits) {
        for (int q = threadIdx.x; q < hits * kSteps; q += kThreads) {
            const int group = sh.hits[q / kSteps];
            const int i0 = group / kScanThreads * kPart +
                           (q % kSteps * kScanThreads + group % kScanThreads) * kVec;
            float v[kVec];
            load8(x, i0, V, v);
#pragma unroll
            for (int j = 0; j < kVec; j++) {
                const double t = r.power(v[j]);
                if (r.bin(t) > bound) continue;
                const u64 m = exp2_fixed(t, r.s);
                if (!m) continue;
                const int at = atomicAdd(&sh.n, 1);
                if (at < kList) sh.list[at] = {(u64)key_of(v[j]) << 32 | (uint32_t)~(i0 + j), m};
            }
        }
        __syncthreads();
    }
    int n = hits <= kHits ? sh.n : kList + 1;
    if (n <= kList && r.by_p && !r.by_k && bound < least) {
        // top-p may end below the bound, and does unless the list has the mass
        const u64 listed = sum_of(sh, n, [&](int i) { return sh.list[i].mass; });
        if (listed < need_p) n = kList + 1;
    }
    u64 all;
    int token;
    if (n <= kPairs) {
        // every pair: a token's rank and the mass before it; then its mass up to it by index
        int wide = 64;
        while (wide < n) wide *= 2;
        const int i = (threadIdx.x & (wide - 1)), ways = kThreads / wide, way = threadIdx.x / wide;
        if ((int)threadIdx.x < kPairs) {
            sh.pair.before[threadIdx.x] = 0;
            sh.pair.rank[threadIdx.x] = 0;
        }
        if (threadIdx.x == 0) sh.kept = sh.all = 0;
        __syncthreads();
        Candidate me{0, 0};
        if (i < n) {
            me = sh.list[i];
            uint32_t rank = 0;
            u64 before = 0;
            for (int j = way; j < n; j += ways) {
                const Candidate c = sh.list[j];
                if (c.order > me.order) {
                    rank++;
                    before += c.mass;
                }
            }
            atomicAdd(&sh.pair.rank[i], rank);
            atomicAdd(&sh.pair.before[i], before);
        }
        __syncthreads();
        bool keep = i < n;
        if (keep && r.by_k) {
            keep = (int)sh.pair.rank[i] < r.k;
            if (r.by_p && keep && way == 0) atomicAdd(&sh.kept, me.mass);
        }
        __syncthreads();
        if (keep && r.by_p) {
            u64 need = need_p;
            if (r.by_k) {
                need = r.p > 0.0f ? (u64)__builtin_ceil((double)r.p * (double)sh.kept) : 1;
                need = need ? need : 1;
            }
            keep = sh.pair.before[i] < need;
        }
        keep = keep && me.mass >= floor;
        __syncthreads();
        if (way == 0 && i < n) {
            if (keep) atomicAdd(&sh.all, me.mass);
            else sh.list[i].mass = 0;
            sh.pair.before[i] = 0;
        }
        __syncthreads();
        all = sh.all;
        const u64 need = drawn_need(r.u, all);
        if (keep) {
            u64 run = 0;
            for (int j = way; j < n; j += ways) {
                const Candidate c = sh.list[j];
                if ((uint32_t)c.order >= (uint32_t)me.order) run += c.mass;
            }
            atomicAdd(&sh.pair.before[i], run);
        }
        __syncthreads();
        if (keep && way == 0) {
            const u64 run = sh.pair.before[i];
            if (run >= need && run - me.mass < need) sh.index = (int)~(uint32_t)me.order;
        }
        __syncthreads();
        token = sh.index;
    } else if (n <= kList) {
        auto key = [&](int i) { return (uint32_t)(sh.list[i].order >> 32); };
        auto place = [&](int i) { return (uint32_t)sh.list[i].order; };
        Cut c{0, V - 1};
        auto kept = [&](int i) {
            return c.keeps(key(i), (int)~place(i)) ? sh.list[i].mass : 0;
        };
        u64 total;
        if (r.by_k && r.k < n) {
            u64 need = r.k;
            const uint32_t k = find_key(sh, n, need, total, key, [](int) { return 1ull; });
            const uint32_t l = find_key(sh, n, need, total, place,
                                        [&](int i) { return (u64)(key(i) == k); });
            c = {k, (int)~l};
        }
        if (r.by_p) {
            u64 need = need_p;
            if (r.by_k) {
                const u64 sum = sum_of(sh, n, kept);
                need = r.p > 0.0f ? (u64)__builtin_ceil((double)r.p * (double)sum) : 1;
                need = need ? need : 1;
            }
            const uint32_t k = find_key(sh, n, need, total, key, kept);
            const uint32_t l = find_key(sh, n, need, total, place,
                                        [&](int i) { return key(i) == k ? kept(i) : 0; });
            c = {k, (int)~l};
        }
        auto drawn = [&](int i) {
            const u64 m = kept(i);
            return m >= floor ? m : 0;
        };
        all = sum_of(sh, n, drawn);
        u64 need = drawn_need(r.u, all);
        token = (int)~find_key(sh, n, need, total, place, drawn);
    } else {
        Cut c{0, V - 1};
        auto kept = [&](int i, uint32_t key, double t) {
            return c.keeps(key, i) ? exp2_fixed(t, r.s) : 0;
        };
        if (r.by_k) {
            auto some = [&](int, uint32_t, double t) { return (u64)(exp2_fixed(t, r.s) != 0); };
            auto at = [&](int i) { return some(i, 0, r.power(value(x[i]))); };
            if (sum_of(sh, V, at) > (u64)r.k) c = cut_row(sh, x, V, r, r.k, some);
        }
        if (r.by_p) {
            u64 need = need_p;
            if (r.by_k) {
                const u64 sum = sum_of(sh, V, [&](int i) {
                    const float v = value(x[i]);
                    return kept(i, key_of(v), r.power(v));
                });
                need = r.p > 0.0f ? (u64)__builtin_ceil((double)r.p * (double)sum) : 1;
                need = need ? need : 1;
            }
            c = cut_row(sh, x, V, r, need, kept);
        }
        auto drawn = [&](int i) {
            const float v = value(x[i]);
            const u64 m = kept(i, key_of(v), r.power(v));
            return m >= floor ? m : 0;
        };
        all = sum_of(sh, V, drawn);
        token = find_index(sh, V, drawn_need(r.u, all), drawn);
    }
    if (threadIdx.x == 0) answer(token, all, 0.0);
}

template <class E>
void launch(const fni8h::Sample& a, hipStream_t st) {
    const int64_t parts = parts_of(a.V), deep = (a.B + 32767) / 32768;
    const dim3 grid((uint32_t)parts, (uint32_t)(a.B < 32768 ? a.B : 32768), (uint32_t)deep);
    scan_kernel<E><<<grid, kScanThreads, 0, st>>>(a, (int)parts);
    draw_kernel<E><<<(uint32_t)a.B, kThreads, 0, st>>>(a, (int)parts);
}

}  // namespace

namespace fni8h {

int64_t sample_workspace_bytes(int64_t B, int64_t V) { return B * row_bytes(parts_of(V)); }

int launch_sample(const Sample& a, hipStream_t st) {
    if (a.B == 0) return FNI8_OK;
    if (a.fp32) launch<float>(a, st);
    else launch<uint16_t>(a, st);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) {
        set_error_detail("sample launch: %s", hipGetErrorString(err));
        return FNI8_ERR_LAUNCH;
    }
    return FNI8_OK;
}

}  // namespace fni8h
