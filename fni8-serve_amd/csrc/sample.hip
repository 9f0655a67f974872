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
// time, and a kept mass is the very sum that the draw runs through.  At 151936 tokens s is 44: a
// running sum is off by some 2^-36 of the largest weight at worst, where 24 bits of a float
// sum would put about one draw in thirty on a neighbour of the token that the sums meant.
// A rank, a mass and a place among equal logits are all the same search: the first key (or
// index) at which a running sum of integers reaches a number.
#include "common.h"

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024, kWaves = 16;

// 2^t * 2^s as an integer, rounded, for t <= 0 and s <= 50.  t = n + f, |f| <= 1/2; 2^f by its
// Taylor polynomial in f ln 2, degree 11 (the first term left out is below 2^-47); adding
// 2^52 leaves the integer in the low bits of the sum.
__device__ __forceinline__ u64 exp2_fixed(double t, int s) {
    if (!(t > -(double)(s + 2))) return 0;
    const double n = __builtin_rint(t), f = t - n;
    double p = 4.4455382718708115e-10;                      // ln2^11 / 11!
    p = __builtin_fma(p, f, 7.0549116208011233e-9);  // ln2^10 / 10!
    p = __builtin_fma(p, f, 1.0178086009239699e-7);
    p = __builtin_fma(p, f, 1.3215486790144309e-6);
    p = __builtin_fma(p, f, 1.5252733804059840e-5);
    p = __builtin_fma(p, f, 1.5403530393381609e-4);
    p = __builtin_fma(p, f, 1.3333558146428443e-3);
    p = __builtin_fma(p, f, 9.6181291076284772e-3);
    p = __builtin_fma(p, f, 5.5504108664821580e-2);
    p = __builtin_fma(p, f, 0.24022650695910071);
    p = __builtin_fma(p, f, 0.69314718055994531);
    p = __builtin_fma(p, f, 1.0);
    const double v = __builtin_ldexp(p, (int)n + s) + 0x1p52;
    return __builtin_bit_cast(u64, v) & 0xfffffffffffffull;
}

// Order of floats as unsigned numbers; -0 counts as +0.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

template <class E>
__device__ __forceinline__ float value(E e) {
    if constexpr (sizeof(E) == 2) return fni8::h2f(e);
    else return e;
}

__device__ __forceinline__ u64 wave_sum(u64 v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

__device__ __forceinline__ u64 wave_scan(u64 v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const u64 o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    return v;
}

struct Shared {
    u64 part[kWaves];
    u64 hist[256];
    u64 need, total;
    uint32_t key;
    int index;
};

// Sum of f(i) over the row, the same in every thread.
template <class F>
__device__ u64 sum_of(Shared& sh, int V, F f) {
    u64 s = 0;
    for (int i = threadIdx.x; i < V; i += kThreads) s += f(i);
    s = wave_sum(s);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.part[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0;
    for (int w = 0; w < kWaves; w++) s += sh.part[w];
    return s;
}

// The first index at which the running sum of f reaches `need` (1 to the sum of all).
template <class F>
__device__ int find_index(Shared& sh, int V, u64 need, F f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int lo = 0, hi = V;
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
        for (; w < kWaves - 1 && sh.part[w] < need; w++) need -= sh.part[w];
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

// The largest key such that the sum of f(i) over keys no smaller reaches `need`; `need` is
// then what the tokens of that key have to bring, `total` what they hold.
template <class K, class F>
__device__ uint32_t find_key(Shared& sh, int V, u64& need, u64& total, K key, F f) {
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (threadIdx.x < 256) sh.hist[threadIdx.x] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < V; i += kThreads) {
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
            u64 run = wave_scan(own, lane) - own;
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

template <class E>
__global__ __launch_bounds__(kThreads) void sample_kernel(const fni8h::Sample a) {
    __shared__ Shared sh;
    const int64_t row = blockIdx.x;
    const E* x = (const E*)a.logits + row * a.ld;
    const int V = (int)a.V, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float T = a.temperature ? a.temperature[row] : a.temperature1;
    const int k = a.top_k ? a.top_k[row] : a.top_k1;
    const float p = a.top_p ? a.top_p[row] : a.top_p1;
    float least = a.min_p ? a.min_p[row] : a.min_p1;
    least = least > 0.0f ? least < 1.0f ? least : 1.0f : 0.0f;
    const float u = a.u ? a.u[row] : 0.0f;

    uint32_t best = 0;
    bool nan = T != T;
    for (int i = threadIdx.x; i < V; i += kThreads) {
        const float v = value(x[i]);
        const uint32_t key = key_of(v);
        nan |= v != v;
        best = key > best ? key : best;
    }
    best = nan ? 0xffffffffu : best;
    best = fni8::wave_max_u32(best);
    if (lane == 0) sh.part[wave] = best;
    __syncthreads();
    for (int w = 0; w < kWaves; w++) best = sh.part[w] > best ? (uint32_t)sh.part[w] : best;
    const float top = __builtin_bit_cast(float, (best & 0x80000000u) ? best ^ 0x80000000u : ~best);
    if (best == 0xffffffffu || top == -__builtin_inff()) {  // a NaN, or nothing to draw
        if (threadIdx.x == 0) {
            a.tokens[row] = -1;
            if (a.logprobs) a.logprobs[row] = __builtin_nanf("");
        }
        return;
    }
    auto key = [&](int i) { return key_of(value(x[i])); };
    if (!(T > 0.0f)) {
        const int i = find_index(sh, V, 1, [&](int i) { return (u64)(key(i) == best); });
        if (threadIdx.x == 0) {
            a.tokens[row] = i;
            if (a.logprobs) a.logprobs[row] = 0.0f;
        }
        return;
    }
    // bits of the fraction, so that V weights of at most 1 add up to less than 2^62
    const int s = 62 - (32 - __builtin_clz(V)) < 50 ? 62 - (32 - __builtin_clz(V)) : 50;
    const double rate = 1.4426950408889634 / (double)T;
    const bool inf = top == __builtin_inff();
    auto power = [&](float v) {
        if (inf) return v == top ? 0.0 : -__builtin_inf();
        if (v == -__builtin_inff()) return -__builtin_inf();
        return ((double)v - (double)top) * rate;
    };
    uint32_t cut = 0;
    int last = V - 1;
    auto kept = [&](int i, uint32_t key) { return key > cut || (key == cut && i <= last); };
    auto mass = [&](int i) {
        const float v = value(x[i]);
        return kept(i, key_of(v)) ? exp2_fixed(power(v), s) : 0;
    };
    if (k > 0 && k < V) {
        u64 need = k, total;
        const uint32_t c = find_key(sh, V, need, total, key, [](int) { return 1ull; });
        const int l = need == total ? V - 1
                    : find_index(sh, V, need, [&](int i) { return (u64)(key(i) == c); });
        cut = c;
        last = l;
    }
    if (p < 1.0f) {
        const u64 all = sum_of(sh, V, mass);
        u64 need = p > 0.0f ? (u64)__builtin_ceil((double)p * (double)all) : 1, total;
        need = need < 1 ? 1 : need < all ? need : all;
        const uint32_t c = find_key(sh, V, need, total, key, mass);
        const int l = find_index(sh, V, need, [&](int i) { return key(i) == c ? mass(i) : 0; });
        cut = c;
        last = l;
    }
    const u64 floor = (u64)__builtin_rint((double)least * __builtin_ldexp(1.0, s));
    auto drawn = [&](int i) {
        const u64 w = mass(i);
        return w >= floor ? w : 0;
    };
    const u64 all = sum_of(sh, V, drawn);
    u64 need = u > 0.0f ? (u64)((double)(u < 1.0f ? u : 1.0f) * (double)all) + 1 : 1;
    need = need < all ? need : all;
    const int i = find_index(sh, V, need, drawn);
    if (threadIdx.x == 0) {
        a.tokens[row] = i;
        if (a.logprobs)
            a.logprobs[row] = (float)(power(value(x[i])) * 0.69314718055994531 -
                                      log((double)all * __builtin_ldexp(1.0, -s)));
    }
}

}  // namespace

namespace fni8h {

int64_t sample_workspace_bytes(int64_t B, int64_t V) { return 0; }

int launch_sample(const Sample& a, hipStream_t st) {
    if (a.B == 0) return FNI8_OK;
    if (a.fp32) sample_kernel<float><<<(uint32_t)a.B, kThreads, 0, st>>>(a);
    else sample_kernel<uint16_t><<<(uint32_t)a.B, kThreads, 0, st>>>(a);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) {
        set_error_detail("sample launch: %s", hipGetErrorString(err));
        return FNI8_ERR_LAUNCH;
    }
    return FNI8_OK;
}

}  // namespace fni8h
