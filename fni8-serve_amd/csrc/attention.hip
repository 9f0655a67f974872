// Attention of new tokens over the paged cache (gfx950).
//
// Query token i of the n new ones of a sequence of L tokens (the new ones among them)
// stands at p = L - n + i and sees the keys j, 0 <= j <= p, j > p - window:
//   out = sum_j softmax_j(scale * q . k_j) v_j
// with an online softmax: running maximum m, sum l and unnormalised output o in fp32, all
// in powers of two (scores times scale * log2 e).  A row that sees no key (p < 0: it always
// sees its own) is 0; one whose scores are all -inf has the sum 0 and gives 0 / 0, NaN.
//
// The query heads that share a key head are packed with the tokens into rows
// r = i * group + head, so that one read of a key serves all of them.  Both kernels compute
// S^T = K Q^T (the keys as the MFMA's rows): a lane then holds several keys of ONE query
// row, so a row's maximum and sum need one or two lane swaps, and the weights P^T are
// already laid out as the second operand of O^T = V^T P^T.  The MFMA's k order is free as
// long as both operands agree, so the keys of P stay where S^T left them, and V^T is read
// from row-major V in LDS with transposing reads (4 keys x 16 elements) in the same order.
//
// The weights P are rounded to fp16 before their product with V, the one rounding below fp32
// between the inputs and the result: that product's MFMA takes 16-bit operands, and P in two
// halves would double its count, half of all products.  l adds the weights unrounded.  Each
// is off by 2^-11 of itself at most (2^-25 of 1 where it is small); the measured cases are
// 2.3e-4 to 2.9e-4 from 64 bits in their norm, of which the result's own rounding to fp16
// makes 2.1e-4.
//
// 8 bits: the codes go through the matrix cores as fp16 integers (exact).  A key's scale
// multiplies its column of S.  A value's scale v_s joins the exponent instead of P:
// P' = 2^(s + log2 v_s - m) with m the maximum of s + log2 v_s (or up to kLag below it), so P'
// rounds to fp16 like P does whatever the scale's size, and l adds P' / v_s.
//
// few_work takes sequences with few rows (decode, drafted tokens): memory bounds it, each
// cached row is read once.  The keys of all sequences are one list of units of 128 keys,
// cut into equal runs, one a workgroup, whatever the lengths; parts of an item that two
// workgroups share are joined by join_kernel.  tile_kernel takes the others: 128 rows a
// workgroup share K and V tiles of 64 keys in LDS; the MFMAs (49% of the busy cycles of a chunk
// of 2048 tokens over 14336) and the vector instructions of the softmax (41%) bound it, at the
// clock that the card's power leaves them.  A batch of both kinds is one launch, so that the reads of the one pass
// beside the products of the other.
#include <atomic>

#include "common.h"

namespace {

using fni8::f2h;
using fni8::h2f;

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef __fp16 tr4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kInf = __builtin_inff();
constexpr int kUnit = 128;      // keys of a unit of few_work: 32 for each of 4 waves
constexpr int kTileRows = 128;  // of a workgroup of tile_kernel: 32 a wave
constexpr int kTileKeys = 64;
constexpr float kLag = 8.0f;
// Block tables of so few units: an item is one workgroup's, and no join is launched.  One
// decoded token a sequence, 8 key heads of 128, whole against split (us): 1 sequence of 100,
// 250, 380, 500 keys 8.1, 10.1, 11.1, 12.1 against 9.6, 11.5, 11.5, 11.6 (8 bits 7.7, 9.6,
// 11.4, 13.1 against 9.1, 10.9, 11.0, 11.0); 64 of 380 21.4 against 23.1.
constexpr int kWholeUnits = 3;
constexpr int kWorkers = 768;  // of few_work at most: three a CU
// Beside tiles: one a CU, the tiles have the rest of it.  Decoded tokens beside one chunk, in
// two launches, one with 512 workers and one with 256 (us): 120 of 2000 to 16000 keys beside
// 2000 tokens 1060, 1020, 969; 63 of up to 8500 beside 512 229, 216, 231, of 8 bits 247, 242,
// 226; 15 of up to 2000 beside 384 58, 51, 51.  Only chunks, 8 bits, 64 of 450 tokens: 2059,
// 2134, 2143.
constexpr int kMixedWorkers = 256;

// What join_kernel does: part p of an item, o [rows][DP], m, l [rows], lies in slot `first`
// (p = 0) or next + (p - 1) * step.
struct Join {
    int parts;  // 0: nothing to do
    int first, next, step;
    int start, row0, nrows, h;
    int p0;  // position of the sequence's first new token
};

// Division of 0 <= n < 2^31 by a divisor d that the host knows (Granlund and Montgomery,
// 1994): with 2^shift the next power of two from d on and mul = floor(2^(32 + shift) / d) -
// 2^32 + 1, n / d = (hi32(n mul) + n) >> shift.  Eight divisions stand before the first load
// of a workgroup.
struct Div {
    uint32_t mul, shift;
};
__device__ __forceinline__ int over(int n, Div d) {
    return (int)((__umulhi((uint32_t)n, d.mul) + (uint32_t)n) >> d.shift);
}

struct Attn {
    const uint16_t* q;
    int64_t ldq, hsq;
    const void *kc, *vc;
    const float *ks, *vs;
    const int32_t *tables, *lens, *cu;
    int64_t ldt;
    uint16_t* out;
    Join *joins, *tile_joins;
    float *part, *tile_part;
    int T, Hq, Hk, D, group, num_pages, plog, max_pages, B, nseq, window, cap;
    float c;       // |scale| * log2 e, not 0
    uint32_t flip; // sign bits of two fp16 where the scale is negative: the queries' signs
    Div by_group, by_heads, by_splits, by_quads;  // group, Hk, splits, D / 4
    int few;       // few_work takes sequences of at most so many new tokens, tiles the others
    int workers;   // workgroups of few_work
    int whole;     // few_work: no parts, an item is one unit
    int splits;    // tile_kernel: parts of an item at most
};

struct Seq {
    int start, n, L;
};
// Where a token stands as a query: its own position, but past the block table (a.cap - 1
// tokens) that of the first token there.  That one is a key of NaN, which such a query sees
// whatever its window; the queries before it keep their positions and never see it.
__device__ __forceinline__ int position(const Attn& a, const Seq& q, int i) {
    const int p = q.L - q.n + i;
    return p < a.cap - 1 ? p : a.cap - 1;
}
// The keys that any of its queries can see, from 0 on.
__device__ __forceinline__ int keys_of(const Attn& a, const Seq& q) {
    return q.L < a.cap ? q.L : a.cap;
}

__device__ __forceinline__ int bound_of(const Attn& a, int s) {
    if (s > a.B) return a.T;
    const int c = a.cu ? a.cu[s] : s;
    return c < 0 ? 0 : c < a.T ? c : a.T;
}

// Sequence s; the tokens past the last one are a sequence of no keys.
__device__ __forceinline__ Seq sequence(const Attn& a, int s) {
    Seq q;
    q.start = bound_of(a, s);
    q.n = bound_of(a, s + 1) - q.start;
    q.n = q.n > 0 ? q.n : 0;
    q.L = 0;
    if (s < a.B) {
        const int L = a.lens[s];
        q.L = L < 0 ? 0 : L;
    }
    return q;
}

// ---- the list of items -----------------------------------------------------------

__device__ __forceinline__ int block_scan(int v, int* sh, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int incl = fni8::wave_incl_scan_i32(v, lane);
    __syncthreads();
    if (lane == 63) sh[wave] = incl;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        if (w < wave) incl += sh[w];
        total += sh[w];
    }
    return incl;
}

// The sequence that holds unit `target(U)` of the list of all U = sum units(s), and the
// number of units before it.  Every thread of the block gets the same answer, in scalar
// registers; false where the target is not in the list.  sh: 16 words of LDS.
template <class Units, class Target>
__device__ __forceinline__ bool find(int nseq, int* sh, Units units, Target target, int& s_out,
                                     int& base_out, int& goal, Seq& q_out) {
    const int tid = threadIdx.x;
    int U = 0, mine = 0, incl = 0, total = 0;
    Seq q{0, 0, 0};
    if (nseq <= 64) {  // every wave by itself
        const int lane = tid & 63;
        if (lane < nseq) mine = units(lane, q);
        incl = fni8::wave_incl_scan_i32(mine, lane);
        U = __builtin_amdgcn_readlane(incl, 63);
        goal = target(U);
        if (goal < 0 || goal >= U) return false;
        const uint64_t at = __ballot(incl >= mine && goal >= incl - mine && goal < incl);
        if (!at) return false;
        s_out = __builtin_ctzll(at);
        base_out = __builtin_amdgcn_readlane(incl - mine, s_out);
        q_out.start = __builtin_amdgcn_readlane(q.start, s_out);
        q_out.n = __builtin_amdgcn_readlane(q.n, s_out);
        q_out.L = __builtin_amdgcn_readlane(q.L, s_out);
        return true;
    }
    if (tid == 0) sh[8] = -1;
    for (int c = 0; c < nseq; c += 256) {
        mine = c + tid < nseq ? units(c + tid, q) : 0;
        incl = block_scan(mine, sh, total);
        U += total;
    }
    U = __builtin_amdgcn_readfirstlane(U);  // wave-uniform from here on, in scalar registers
    goal = target(U);
    if (goal < 0 || goal >= U) return false;
    int base = 0;
    for (int c = 0; c < nseq; c += 256) {
        if (nseq > 256) {
            mine = c + tid < nseq ? units(c + tid, q) : 0;
            incl = block_scan(mine, sh, total);
        }
        const int before = base + incl - mine;
        // (sums that overflow, from a cu_seqlens that is not one, are no place)
        if (before >= 0 && goal >= before && goal - before < mine) {
            sh[8] = c + tid;
            sh[9] = before;
            sh[10] = q.start;
            sh[11] = q.n;
            sh[12] = q.L;
        }
        base += total;
    }
    __syncthreads();
    s_out = __builtin_amdgcn_readfirstlane(sh[8]);
    base_out = __builtin_amdgcn_readfirstlane(sh[9]);
    q_out.start = __builtin_amdgcn_readfirstlane(sh[10]);
    q_out.n = __builtin_amdgcn_readfirstlane(sh[11]);
    q_out.L = __builtin_amdgcn_readfirstlane(sh[12]);
    __syncthreads();
    return s_out >= 0;
}

// ---- small pieces ------------------------------------------------------------------

__device__ __forceinline__ float max_xor32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v),
                                                    __builtin_bit_cast(uint32_t, v), false, false);
    return __builtin_fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]),
                           __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float max_xor16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v),
                                                    __builtin_bit_cast(uint32_t, v), false, false);
    return __builtin_fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]),
                           __builtin_bit_cast(float, (uint32_t)r[1]));
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h2));  // to nearest even
}

// Four int8 codes -> four fp16 (exact): the byte, made unsigned, is the low mantissa of
// 1024 + b; subtracting 1024 + 128 leaves the code.
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
    const uint32_t x = w ^ 0x80808080u;
    const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(
                                          0x64646464u, x, 0x04010400u)) - off);
    hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(
                                          0x64646464u, x, 0x04030402u)) - off);
}

// 16 codes -> two chunks of 8 fp16
__device__ __forceinline__ void codes16(u32x4 w, u32x4& a, u32x4& b) {
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 4; i++) codes_to_half(w[i], o[2 * i], o[2 * i + 1]);
    a = u32x4{o[0], o[1], o[2], o[3]};
    b = u32x4{o[4], o[5], o[6], o[7]};
}

// log2 and reciprocal of a value's scale; a scale of 0 (a row of zeros) counts as 2^-64,
// so that its key keeps its weight in l while its codes add nothing that shows.
__device__ __forceinline__ void value_scale(float v, float& lv, float& rv) {
    v = v < 0x1p-64f ? 0x1p-64f : v;
    lv = __builtin_amdgcn_logf(v);
    rv = __builtin_amdgcn_rcpf(v);
}

// 16 bytes of LDS at a byte offset, and a value fragment: 4 keys at `off`, 4 at `off2`
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) tr4 lds_tr4;
__device__ __forceinline__ h8 lds_read16(uint32_t off) {
    return __builtin_bit_cast(h8, *reinterpret_cast<lds_u32x4*>(off));
}
__device__ __forceinline__ h8 lds_read_tr(uint32_t off, uint32_t off2) {
    const tr4 a = __builtin_amdgcn_ds_read_tr16_b64_v4f16(reinterpret_cast<lds_tr4*>(off));
    const tr4 b = __builtin_amdgcn_ds_read_tr16_b64_v4f16(reinterpret_cast<lds_tr4*>(off2));
    const uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, b);
    const u32x4 v = {x.x, x.y, y.x, y.y};
    return __builtin_bit_cast(h8, v);
}

// Whether any of 8 fp16 is an infinity or NaN (exponent all ones).
__device__ __forceinline__ uint32_t odd_bits(u32x4 v) {
    uint32_t o = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) o |= ((v[i] & 0x7fff7fffu) + 0x04000400u) & 0x80008000u;
    return o;
}

// 8 fp16 with 0 in the place of infinities and NaN.
__device__ __forceinline__ u32x4 finite_part(u32x4 v) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if ((v[i] & 0x7c00u) == 0x7c00u) v[i] &= 0xffff0000u;
        if ((v[i] & 0x7c000000u) == 0x7c000000u) v[i] &= 0xffffu;
    }
    return v;
}

// The fp16 in half `hi` of w where it is an infinity or NaN, else 0.
__device__ __forceinline__ float odd_part(uint32_t w, int hi) {
    const uint32_t b = hi ? w >> 16 : w & 0xffffu;
    return (b & 0x7c00u) == 0x7c00u ? h2f((uint16_t)b) : 0.0f;
}

// Masks and values that are not finite: the weight of a key that a row does not see is 0,
// but 0 times an infinity or NaN is NaN.  Where a tile that some row sees in part only holds
// such a value, the tile's values are made finite before the product, and the rows that see
// the key get the value added afterwards, read once more from the cache.

// A block of 16 keys of a sequence: its page, or why there is none.
constexpr int kNone = -1, kBad = -2;
__device__ __forceinline__ int page_of(const Attn& a, int s, int token, int lo, int hi) {
    if (token >= hi || token + 16 <= lo) return kNone;
    const int col = token >> a.plog;
    if (col >= a.max_pages) return kBad;
    const int page = a.tables[(int64_t)s * a.ldt + col];
    return page < 0 || page >= a.num_pages ? kBad : page;
}

// 16 bytes that are read once.  Past the caches where ONCE: 64 sequences, 1 GB of 16 bits,
// 189 -> 175 us; codes of 8 bits, whose lines two loads share, 49 -> 56.
template <bool ONCE>
__device__ __forceinline__ u32x4 stream(const char* p) {
    const u32x4* q = reinterpret_cast<const u32x4*>(p);
    return ONCE ? __builtin_nontemporal_load(q) : *q;
}

// ---- few rows ----------------------------------------------------------------------

// LDS bytes of a wave: its V tile (32 keys), or its rows of o when they are joined
template <int DP, int RB>
constexpr int few_region() {
    return 32 * DP * 2 > 16 * RB * DP * 4 ? 32 * DP * 2 : 16 * RB * DP * 4;
}
template <int DP, int RB>
constexpr int few_lds() {
    return 4 * few_region<DP, RB>() + 4 * 2 * 16 * RB * 4 + 64;
}
// floats of a part: o [16 RB][DP], m, l [16 RB]
template <int DP, int RB>
constexpr int few_part() {
    return 16 * RB * (DP + 2);
}

// Workgroups a CU, by the registers
constexpr int few_waves(int dp, int rb) {
    return dp > 128 ? 1 : rb == 1 && dp == 64 ? 3 : 2;
}

// What few_work makes of a sequence: its range of keys and its units.
struct FewSeq {
    Seq q;
    int rows, blocks, lo, tiles, units;
};
template <int RB>
__device__ __forceinline__ FewSeq few_seq(const Attn& a, const Seq& q) {
    FewSeq f;
    f.q = q;
    f.rows = f.q.n > a.few ? 0 : f.q.n * a.group;
    f.blocks = (f.rows + 16 * RB - 1) / (16 * RB);
    const int first = position(a, f.q, 0);
    f.lo = a.window && first - a.window + 1 > 0 ? (first - a.window + 1) & ~31 : 0;
    f.tiles = (keys_of(a, f.q) - f.lo + kUnit - 1) / kUnit;
    f.tiles = f.tiles > 1 ? f.tiles : 1;
    f.units = f.blocks * a.Hk * (a.whole ? 1 : f.tiles + 1);
    return f;
}

// The work of one of a.workers workgroups.
template <int DP, bool I8, int RB>
__device__ __forceinline__ void few_work(const Attn& a, const int worker, char* smem) {
    constexpr int KS = DP / 32, DB = DP / 16;
    constexpr int KL = I8 ? DP / 64 : DP / 32, VL = KL;  // loads of 16 keys
    constexpr int CH = DP / 8;                           // chunks of a row in LDS
    constexpr int ES = I8 ? 1 : 2, RC = DP * ES / 16;    // 16-byte pieces of a cached row
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, G = lane >> 4;
    const uint32_t k_off = col * a.D * ES + 16 * G;
    uint16_t* vt = reinterpret_cast<uint16_t*>(smem + wave * few_region<DP, RB>());
    float* ot = reinterpret_cast<float*>(vt);
    float* ml = reinterpret_cast<float*>(smem + 4 * few_region<DP, RB>());  // [4][2][16 RB]
    int* sh = reinterpret_cast<int*>(ml + 4 * 2 * 16 * RB);

    if (!a.whole && threadIdx.x == 0) a.joins[worker].parts = 0;
    int s, base, u, upw = 0;
    Seq sq;
    if (!find(
            a.nseq, sh,
            [&](int i, Seq& q) {
                q = sequence(a, i);
                return few_seq<RB>(a, q).units;
            },
            [&](int U) {
                upw = (U + a.workers - 1) / a.workers;
                return upw * worker;
            },
            s, base, u, sq))
        return;
    const int first_unit = u;
    FewSeq f = few_seq<RB>(a, sq);
    int per_item = a.whole ? 1 : f.tiles + 1;
    int item = (u - base) / per_item, tile = (u - base) - item * per_item;
    int left = upw;

    while (true) {
        // an item's last unit has no keys: it stands for the time of its beginning and end
        int nt = per_item - tile;
        nt = nt < left ? nt : left;
        const int real = a.whole || nt < f.tiles - tile ? nt : f.tiles - tile;
        const bool full = a.whole || real == f.tiles;
        if (real > 0) {
        const int rb = over(item, a.by_heads), h = item - rb * a.Hk;
        const int steps = a.whole ? f.tiles : real;
        const int row0 = rb * 16 * RB;
        const int nrows = f.rows - row0 < 16 * RB ? f.rows - row0 : 16 * RB;
        const int first = position(a, f.q, 0);
        const int lo = a.window && first - a.window + 1 > 0 ? first - a.window + 1 : 0;
        const int hi = keys_of(a, f.q);
        const int pmin = position(a, f.q, over(row0, a.by_group));
        const int pmax = position(a, f.q, over(row0 + nrows - 1, a.by_group));
        const int t_first = f.lo + tile * kUnit + wave * 32;

        // queries: row col of each block; the elements' order is the keys' (8 bits: two
        // k-steps of a 16-byte load)
        h8 q[RB][KS];
        int prow[RB];
        uint32_t span[RB], seen0[RB];
#pragma unroll
        for (int b = 0; b < RB; b++) {
            const int r = row0 + 16 * b + col;
            const int i = over(r, a.by_group), head = h * a.group + r - i * a.group;
            prow[b] = r < f.rows ? position(a, f.q, i) : -1;
            // it sees the keys j with prow - span < j <= prow: one unsigned comparison
            span[b] = prow[b] < 0 ? 0 : a.window ? a.window : prow[b] + 1;
            seen0[b] = 4 * G - (prow[b] + 1 - (int)span[b]);
#pragma unroll
            for (int k = 0; k < KS; k++) {
                const int d = I8 ? 64 * (k >> 1) + 16 * G + 8 * (k & 1) : 32 * k + 8 * G;
                u32x4 v = {0, 0, 0, 0};
                if (r < f.rows && d < a.D)
                    v = *reinterpret_cast<const u32x4*>(a.q + (f.q.start + i) * a.ldq +
                                                        head * a.hsq + d);
                v ^= a.flip;
                q[b][k] = __builtin_bit_cast(h8, v);
            }
        }

        float m[RB], l[RB];
        f32x4 o[RB][DB];
#pragma unroll
        for (int b = 0; b < RB; b++) {
            m[b] = -kInf;
            l[b] = 0.0f;
#pragma unroll
            for (int d = 0; d < DB; d++) o[b][d] = f32x4{0, 0, 0, 0};
        }

        struct Step {  // a wave's 32 keys on their way
            u32x4 kr[2][KL], vr[2][VL];
            f32x4 ksr[2], vsr[2];
            int page[2];
        };
        int pages = 0;  // lane j: block j & 1 of step (j >> 1) of the 32 ahead
        auto load = [&](int i, Step& n) {
            auto &kr = n.kr, &vr = n.vr;
            auto &ksr = n.ksr, &vsr = n.vsr;
            auto& page = n.page;
            if ((i & 31) == 0)
                pages = i + (lane >> 1) < steps
                            ? page_of(a, s, t_first + (i + (lane >> 1)) * kUnit + 16 * (lane & 1),
                                      lo, hi)
                            : kNone;
            const int t0 = t_first + i * kUnit;
#pragma unroll
            for (int tb = 0; tb < 2; tb++) {
                page[tb] = __builtin_amdgcn_readlane(pages, 2 * (i & 31) + tb);
#pragma unroll
                for (int j = 0; j < KL; j++) kr[tb][j] = vr[tb][j] = u32x4{0, 0, 0, 0};
                ksr[tb] = vsr[tb] = f32x4{0, 0, 0, 0};
                if (page[tb] < 0) continue;
                const int tok = t0 + 16 * tb, in = tok & ((1 << a.plog) - 1);
                const int64_t row = (((int64_t)page[tb] * a.Hk + h) << a.plog) + in;
                const char* kp = static_cast<const char*>(a.kc) + row * a.D * ES;
                const char* vp = static_cast<const char*>(a.vc) + row * a.D * ES;
                if constexpr (I8) {
                    ksr[tb] = *reinterpret_cast<const f32x4*>(a.ks + row + 4 * G);
                    vsr[tb] = *reinterpret_cast<const f32x4*>(a.vs + row + 4 * G);
                }
                if (a.D == DP && (I8 || (tok >= lo && tok + 16 <= hi))) {
#pragma unroll
                    for (int j = 0; j < KL; j++) kr[tb][j] = stream<!I8>(kp + k_off + 64 * j);
#pragma unroll
                    for (int j = 0; j < VL; j++) vr[tb][j] = stream<!I8>(vp + 16 * lane + 1024 * j);
                } else {
#pragma unroll
                    for (int j = 0; j < KL; j++)
                        if (64 * j + 16 * G < a.D * ES)
                            kr[tb][j] = *reinterpret_cast<const u32x4*>(kp + k_off + 64 * j);
#pragma unroll
                    for (int j = 0; j < VL; j++) {
                        const int c = j * 64 + lane, t = c / RC, d = 16 * (c % RC);
                        // what lies outside the range may be anything, and 0 * NaN is NaN
                        if (d < a.D * ES && (I8 || (tok + t < hi && tok + t >= lo)))
                            vr[tb][j] = *reinterpret_cast<const u32x4*>(
                                vp + (uint32_t)(t * a.D * ES + d));
                    }
                }
            }
        };
        // The V tile: chunk ch of key t lies at chunk ch ^ f(t), f = 2 (t & 7), or
        // 2 ((t >> 1) & 3) for rows of 128 bytes: the 8 keys of a half wave's transposing
        // read lie on different banks.  Seen from a lane the permutation is an exclusive or
        // with constants on its first address.
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)vt;
        auto f_of = [](int t) { return DP == 64 ? ((t >> 1) & 3) << 1 : (t & 7) << 1; };
        const int wt = I8 ? lane / (DP / 16) : lane / CH, wc = I8 ? 2 * (lane % (DP / 16)) : lane % CH;
        const uint32_t w_addr = lds0 + wt * DP * 2 + 16 * (wc ^ f_of(wt));
        const int rt = 4 * G + (col >> 2);
        const uint32_t r_addr = lds0 + rt * DP * 2 + 16 * (((col & 3) >> 1) ^ f_of(rt)) + 8 * (col & 1);
        auto step = [&](int i, Step& n) {
            auto &kr = n.kr, &vr = n.vr;
            auto &ksr = n.ksr, &vsr = n.vsr;
            auto& page = n.page;
            const int t0 = t_first + i * kUnit;
            const bool bad[2] = {page[0] == kBad, page[1] == kBad};
            const bool none = page[0] == kNone && page[1] == kNone;
            const bool edge = t0 + 31 > pmin || (a.window && t0 <= pmax - a.window);
            bool odd = false;
            const int held[2] = {page[0], page[1]};
            if constexpr (!I8)
                if (edge) {
                    uint32_t bits = 0;
#pragma unroll
                    for (int tb = 0; tb < 2; tb++)
#pragma unroll
                        for (int j = 0; j < VL; j++) bits |= odd_bits(vr[tb][j]);
                    odd = __any(bits != 0);
                    if (odd)
#pragma unroll
                        for (int tb = 0; tb < 2; tb++)
#pragma unroll
                            for (int j = 0; j < VL; j++) vr[tb][j] = finite_part(vr[tb][j]);
                }
            uint32_t wa = w_addr, ra = r_addr;
            asm volatile("" : "+v"(wa), "+v"(ra));  // computed here, not kept in registers
#pragma unroll
            for (int tb = 0; tb < 2; tb++)
#pragma unroll
                for (int j = 0; j < VL; j++) {
                    constexpr int rows = I8 ? 64 / (DP / 16) : 64 / CH;  // of one load
                    const int t = 16 * tb + j * rows;
                    const uint32_t at = (wa ^ (16 * f_of(t))) + t * DP * 2;
                    if constexpr (I8) {
                        u32x4 x, y;
                        codes16(vr[tb][j], x, y);
                        *reinterpret_cast<lds_u32x4*>(at) = x;
                        *reinterpret_cast<lds_u32x4*>(at ^ 16) = y;
                    } else {
                        *reinterpret_cast<lds_u32x4*>(at) = vr[tb][j];
                    }
                }
            f32x4 sc[RB][2];
#pragma unroll
            for (int tb = 0; tb < 2; tb++) {
                h8 kf[KS];
#pragma unroll
                for (int j = 0; j < KL; j++) {
                    if constexpr (I8) {
                        u32x4 x, y;
                        codes16(kr[tb][j], x, y);
                        kf[2 * j] = __builtin_bit_cast(h8, x);
                        kf[2 * j + 1] = __builtin_bit_cast(h8, y);
                    } else {
                        kf[j] = __builtin_bit_cast(h8, kr[tb][j]);
                    }
                }
#pragma unroll
                for (int b = 0; b < RB; b++) {
                    f32x4 acc = {0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < KS; k++)
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[k], q[b][k], acc, 0, 0, 0);
                    sc[b][tb] = acc;
                }
            }
            f32x4 kx[2], lv[2], rv[2];
            if constexpr (I8)
#pragma unroll
                for (int tb = 0; tb < 2; tb++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        float x, y;
                        value_scale(vsr[tb][r], x, y);
                        lv[tb][r] = x;
                        rv[tb][r] = y;
                        kx[tb][r] = ksr[tb][r] * a.c;
                    }
            if (i + 1 < steps) load(i + 1, n);  // its registers are free from here on
            if (none) return;

            h8 p[RB];
#pragma unroll
            for (int b = 0; b < RB; b++) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int tb = e >> 2, r = e & 3;
                    if constexpr (I8)
                        x[e] = __builtin_fmaf(sc[b][tb][r], kx[tb][r], lv[tb][r]);
                    else
                        x[e] = sc[b][tb][r] * a.c;
                    if (bad[tb]) x[e] = __builtin_nanf("");
                }
                if (edge)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        if (seen0[b] + t0 + 16 * (e >> 2) + (e & 3) >= span[b]) x[e] = -kInf;
                    }
                float top = x[0];
#pragma unroll
                for (int e = 1; e < 8; e++) top = __builtin_fmaxf(top, x[e]);
                top = max_xor32(max_xor16(top));
                // m may lag behind the maximum by kLag: weights are at most 2^kLag
                if (__any(top > m[b] + kLag)) {
                    top = __builtin_fmaxf(top, m[b]);
                    const float keep = exp2_(m[b] - (top == -kInf ? 0.0f : top));
                    l[b] *= keep;
#pragma unroll
                    for (int d = 0; d < DB; d++) o[b][d] *= keep;
                    m[b] = top;
                }
                const float at = m[b] == -kInf ? 0.0f : m[b];
                float w[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    w[e] = exp2_(x[e] - at);
                    if constexpr (I8)
                        l[b] += w[e] == 0.0f ? 0.0f : w[e] * rv[e >> 2][e & 3];
                    else
                        l[b] += w[e];
                }
                const u32x4 pk = {pack2(w[0], w[1]), pack2(w[2], w[3]), pack2(w[4], w[5]),
                                  pack2(w[6], w[7])};
                p[b] = __builtin_bit_cast(h8, pk);
            }
#pragma unroll
            for (int d = 0; d < DB; d++) {
                const uint32_t at = (ra ^ (d % 8 * 32)) + d / 8 * 256;
                const h8 v = lds_read_tr(at, at + 16 * DP * 2);
#pragma unroll
                for (int b = 0; b < RB; b++)
                    o[b][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[b], o[b][d], 0, 0, 0);
            }
            if (odd)
#pragma unroll 1
                for (int t = 0; t < 32; t++) {
                    const int pg = t < 16 ? held[0] : held[1], j = t0 + t;
                    if (pg < 0) continue;
                    const int64_t row = (((int64_t)pg * a.Hk + h) << a.plog) + (j & ((1 << a.plog) - 1));
                    const uint16_t* vp = static_cast<const uint16_t*>(a.vc) + row * a.D + 4 * G;
#pragma unroll
                    for (int d = 0; d < DB; d++) {
                        if (16 * d >= a.D) continue;
                        const uint2 w = *reinterpret_cast<const uint2*>(vp + 16 * d);
#pragma unroll
                        for (int b = 0; b < RB; b++) {
                            if (j - (prow[b] + 1 - (int)span[b]) >= span[b]) continue;
#pragma unroll
                            for (int r = 0; r < 4; r++)
                                o[b][d][r] += odd_part(r < 2 ? w.x : w.y, r & 1);
                        }
                    }
                }
        };
        Step on_way;
        load(0, on_way);
        for (int i = 0; i < steps; i++) step(i, on_way);

        // join the four waves: o rows in LDS (16-byte pieces permuted against bank conflicts)
#pragma unroll
        for (int b = 0; b < RB; b++) {
            l[b] += __shfl_xor(l[b], 16, 64);
            l[b] += __shfl_xor(l[b], 32, 64);
            if (G == 0) {
                ml[(wave * 2) * 16 * RB + 16 * b + col] = m[b];
                ml[(wave * 2 + 1) * 16 * RB + 16 * b + col] = l[b];
            }
#pragma unroll
            for (int d = 0; d < DB; d++) {
                const int c4 = (4 * d + G) ^ (col & 7);
                *reinterpret_cast<f32x4*>(ot + (16 * b + col) * DP + 4 * c4) = o[b][d];
            }
        }
        __syncthreads();
        const int D4 = a.D >> 2;
        float* part = a.part + (int64_t)(2 * worker + (first_unit == u ? 0 : 1)) * few_part<DP, RB>();
        for (int e = threadIdx.x; e < nrows * D4; e += 256) {
            const int r = over(e, a.by_quads), d4 = e - r * D4;
            float top = -kInf, wm[4];
#pragma unroll
            for (int w = 0; w < 4; w++) {
                wm[w] = ml[(w * 2) * 16 * RB + r];
                top = __builtin_fmaxf(top, wm[w]);
            }
            const float at = top == -kInf ? 0.0f : top;
            float sum = 0.0f;
            f32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float k = exp2_(wm[w] - at);
                sum += k * ml[(w * 2 + 1) * 16 * RB + r];
                acc += k * *reinterpret_cast<const f32x4*>(
                               smem + w * few_region<DP, RB>() + (r * DP + 4 * (d4 ^ (r & 7))) * 4);
            }
            if (full) {
                const float inv = 1.0f / sum;
                const int rr = row0 + r, i = over(rr, a.by_group), head = h * a.group + rr - i * a.group;
                uint2 y = {pack2(acc[0] * inv, acc[1] * inv), pack2(acc[2] * inv, acc[3] * inv)};
                if (position(a, f.q, i) < 0) y = uint2{0, 0};
                *reinterpret_cast<uint2*>(a.out + ((int64_t)(f.q.start + i) * a.Hq + head) * a.D +
                                          4 * d4) = y;
            } else {
                *reinterpret_cast<f32x4*>(part + r * DP + 4 * d4) = acc;
                if (d4 == 0) {
                    part[16 * RB * DP + r] = top;
                    part[16 * RB * DP + 16 * RB + r] = sum;
                }
            }
        }
        if (!full && tile == 0 && threadIdx.x == 0) {  // this run begins an item, others end it
            // (a cu_seqlens that is not one can have more units than the list's 32-bit sum says:
            // the join reads no part behind the last workgroup's)
            int w1 = (u + f.tiles - 1) / upw;
            w1 = w1 < a.workers ? w1 : a.workers - 1;
            const int w0 = worker;
            a.joins[w0] = Join{w1 - w0 + 1, 2 * w0 + (first_unit == u ? 0 : 1), 2 * w0 + 2, 2,
                               f.q.start, row0, nrows, h, f.q.L - f.q.n};
        }
        }
        left -= nt;
        u += nt;
        if (left <= 0) return;
        tile = 0;
        if (++item >= f.blocks * a.Hk) {
            do {
                if (++s >= a.nseq) return;
                f = few_seq<RB>(a, sequence(a, s));
            } while (f.units == 0);
            item = 0;
            per_item = a.whole ? 1 : f.tiles + 1;
        }
        __syncthreads();  // the rows of o have been read
    }
}

template <int DP, bool I8, int RB>
__global__ __launch_bounds__(256, few_waves(DP, RB)) void few_kernel(Attn a) {
    extern __shared__ __align__(16) char smem[];
    few_work<DP, I8, RB>(a, blockIdx.x, smem);
}

// Joins an item's parts, a wave a row: 64 parts' weights at a time, one a lane, then the
// parts of o, DP / 4 lanes each, several in flight.
template <int DP>
__device__ __forceinline__ void join_few(const Attn& a, int worker, int part_rows) {
    constexpr int LP = DP / 4, NG = 64 / LP;  // lanes of a part, parts at a time
    const Join j = a.joins[worker];
    if (j.parts == 0) return;
    const int lane = threadIdx.x & 63;
    const int64_t size = (int64_t)part_rows * (DP + 2);
    const int d4 = lane % LP, grp = lane / LP;
    auto slot = [&](int p) {
        return a.part + size * (p == 0 ? j.first : j.next + (p - 1) * j.step);
    };
    for (int r = blockIdx.y * 4 + (threadIdx.x >> 6); r < j.nrows; r += 4 * gridDim.y) {
        float top = -kInf, sum = 0.0f;
        f32x4 acc = {0, 0, 0, 0};
        for (int c = 0; c < j.parts; c += 64) {
            const int n = j.parts - c < 64 ? j.parts - c : 64;
            float m = -kInf, l = 0.0f;
            if (lane < n) {
                const float* p = slot(c + lane) + part_rows * DP;
                m = p[r];
                l = p[part_rows + r];
            }
            // the first parts of o are on their way while the weights are made
            constexpr int U = 8;
            f32x4 v[U];
            auto fetch = [&](int i) {
#pragma unroll
                for (int k = 0; k < U; k++) {
                    const int p = i + k * NG + grp;
                    v[k] = f32x4{0, 0, 0, 0};
                    if (p < n) v[k] = *reinterpret_cast<const f32x4*>(slot(c + p) + r * DP + 4 * d4);
                }
            };
            fetch(0);
            float t = __builtin_fmaxf(top, m);
            t = max_xor32(max_xor16(t));
#pragma unroll
            for (int x = 8; x > 0; x >>= 1) t = __builtin_fmaxf(t, __shfl_xor(t, x, 64));
            const float at = t == -kInf ? 0.0f : t;
            const float keep = exp2_(top - at), w = exp2_(m - at);
            acc *= keep;
            float wl = w * l;
#pragma unroll
            for (int x = 32; x > 0; x >>= 1) wl += __shfl_xor(wl, x, 64);
            sum = sum * keep + wl;
            top = t;
            for (int i = 0; i < n; i += U * NG) {
                if (i > 0) fetch(i);
#pragma unroll
                for (int k = 0; k < U; k++) acc += __shfl(w, (i + k * NG + grp) & 63, 64) * v[k];
            }
        }
#pragma unroll
        for (int x = 32; x >= LP; x >>= 1)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[e] += __shfl_xor(acc[e], x, 64);
        if (grp != 0 || 4 * d4 >= a.D) continue;
        const float inv = 1.0f / sum;
        const int rr = j.row0 + r, i = over(rr, a.by_group), head = j.h * a.group + rr - i * a.group;
        uint2 y = {pack2(acc[0] * inv, acc[1] * inv), pack2(acc[2] * inv, acc[3] * inv)};
        if (j.p0 + i < 0) y = uint2{0, 0};
        *reinterpret_cast<uint2*>(a.out + ((int64_t)(j.start + i) * a.Hq + head) * a.D + 4 * d4) = y;
    }
}

// The same for the many rows and few parts of tile_kernel's items: DP / 4 lanes a row, 32
// rows a workgroup.  (A wave a row spends its time on the exchange of the weights: 45 us of
// 76 for 480 items of two parts.)
template <int DP>
__device__ __forceinline__ void join_tile(const Attn& a, int item) {
    constexpr int LP = DP / 4, RP = 256 / LP;  // lanes of a row, rows at a time
    const Join j = a.tile_joins[item];
    if (j.parts == 0) return;
    const int d4 = threadIdx.x % LP;
    if (4 * d4 >= a.D) return;
    const float* parts = a.tile_part + (int64_t)j.first * (kTileRows * (DP + 2));
    for (int r = blockIdx.y * 32 + threadIdx.x / LP; r < (int)blockIdx.y * 32 + 32 && r < j.nrows;
         r += RP) {
        float top = -kInf, sum = 0.0f;
        f32x4 acc = {0, 0, 0, 0};
#pragma unroll 4
        for (int p = 0; p < j.parts; p++)
            top = __builtin_fmaxf(top, parts[p * (kTileRows * (DP + 2)) + kTileRows * DP + r]);
        const float at = top == -kInf ? 0.0f : top;
#pragma unroll 4
        for (int p = 0; p < j.parts; p++) {
            const float* part = parts + p * (kTileRows * (DP + 2));
            const float k = exp2_(part[kTileRows * DP + r] - at);
            sum += k * part[kTileRows * (DP + 1) + r];
            acc += k * *reinterpret_cast<const f32x4*>(part + r * DP + 4 * d4);
        }
        const float inv = 1.0f / sum;
        const int rr = j.row0 + r, i = over(rr, a.by_group), head = j.h * a.group + rr - i * a.group;
        uint2 y = {pack2(acc[0] * inv, acc[1] * inv), pack2(acc[2] * inv, acc[3] * inv)};
        if (j.p0 + i < 0) y = uint2{0, 0};
        *reinterpret_cast<uint2*>(a.out + ((int64_t)(j.start + i) * a.Hq + head) * a.D + 4 * d4) = y;
    }
}

// grid.x: few_work's workers, then the tiles' items
template <int DP>
__global__ __launch_bounds__(256) void join_kernel(Attn a, int part_rows) {
    if ((int)blockIdx.x < a.workers)
        join_few<DP>(a, blockIdx.x, part_rows);
    else
        join_tile<DP>(a, blockIdx.x - a.workers);
}

// ---- tiles of 128 rows -------------------------------------------------------------

// 16 bytes a lane, global -> LDS at `lds` + lane * 16.  The wait is the caller's.
__device__ __forceinline__ void copy16(uint32_t lds, const void* src) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :: "s"(lds), "v"(src) : "memory", "m0");
}

// Waits until at most N of the wave's copies (and other loads) are on their way.
template <int N>
__device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
}

// A workgroup barrier that leaves copies on their way (__syncthreads waits for all of
// them); LDS reads of the stage that is copied into next have returned by then.
__device__ __forceinline__ void barrier_all() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// A wave-uniform address in scalar registers, wherever it was computed.
__device__ __forceinline__ const void* scalar(const void* p) {
    const uint64_t u = (uint64_t)(uintptr_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
    return reinterpret_cast<const void*>((uintptr_t)((uint64_t)hi << 32 | lo));
}

// The same with a wave-uniform base and a byte offset a lane.
__device__ __forceinline__ void copy16_s(uint32_t lds, const void* base, uint32_t voff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :: "s"(lds), "v"(voff), "s"(base) : "memory", "m0");
}

__device__ const uint4 kZeros = {0, 0, 0, 0};
__device__ const uint4 kNaNs = {0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u};

// Stages of K and V tiles: two workgroups a CU share its LDS at 128 elements, three at 64
constexpr int tile_stages(int dp, bool i8) { return dp == 64 && !i8 ? 3 : 2; }
template <int DP, bool I8>
constexpr int tile_lds() {
    return tile_stages(DP, I8) * 2 * kTileKeys * DP * 2 + (I8 ? 2 * 3 * kTileKeys * 4 : 0) + 64;
}

// Workgroups a CU, by the registers
constexpr int tile_waves(int dp, bool mixed) { return mixed ? few_waves(dp, 1) : dp > 128 ? 1 : 2; }

// The item of a workgroup of tile_kernel.
struct TileItem {
    Seq q;
    int s, rows, tile, h, lo, hi, kt0, kt1, per, parts;
};

// The longest items begin first: a sequence's tiles from the last (a causal tile's keys grow
// with its rows), and up to 64 sequences by the keys that their last tile sees, which each
// wave ranks by itself; more of them from the last to the first.  (12 sequences of 98 to 5600
// tokens, a window of 1024: 41.6 us in the order of the batch, 36.4 ranked.)
__device__ __forceinline__ bool tile_item(const Attn& a, int id, int h, int* sh, TileItem& t) {
    auto tiles = [&](int s, Seq& q) {
        q = sequence(a, s);
        return q.n > a.few
                   ? (int)(((int64_t)q.n * a.group + kTileRows - 1) / kTileRows) : 0;
    };
    if (a.nseq <= 64) {
        const int lane = threadIdx.x & 63;
        Seq q{0, 0, 0};
        const int mine = lane < a.nseq ? tiles(lane, q) : 0;
        const int keys = a.window && a.window < q.L ? a.window : q.L;
        int before = 0;
        for (int s = 0; s < a.nseq; s++) {
            const int k = __builtin_amdgcn_readlane(keys, s), n = __builtin_amdgcn_readlane(mine, s);
            before += k > keys || (k == keys && s < lane) ? n : 0;
        }
        // (sums that overflow, from a cu_seqlens that is not one, are no place)
        const uint64_t at = __ballot(before >= 0 && id >= before && id - before < mine);
        if (!at) return false;
        t.s = __builtin_ctzll(at);
        t.tile = __builtin_amdgcn_readlane(mine, t.s) - 1 - (id - __builtin_amdgcn_readlane(before, t.s));
        t.q.start = __builtin_amdgcn_readlane(q.start, t.s);
        t.q.n = __builtin_amdgcn_readlane(q.n, t.s);
        t.q.L = __builtin_amdgcn_readlane(q.L, t.s);
    } else {
        int base, goal;
        if (!find(a.nseq, sh, tiles, [&](int N) { return N - 1 - id; }, t.s, base, goal, t.q))
            return false;
        t.tile = goal - base;
    }
    t.rows = t.q.n * a.group;
    t.h = h;
    const int i0 = over(t.tile * kTileRows, a.by_group);
    int i1 = over(t.tile * kTileRows + kTileRows - 1, a.by_group);
    i1 = i1 < t.q.n ? i1 : t.q.n - 1;
    const int p0 = position(a, t.q, i0), p1 = position(a, t.q, i1);
    t.hi = p1 + 1 > 0 ? p1 + 1 : 0;
    t.lo = a.window && p0 - a.window + 1 > 0 ? p0 - a.window + 1 : 0;
    t.kt0 = t.lo / kTileKeys;
    t.kt1 = (t.hi + kTileKeys - 1) / kTileKeys;
    const int n = t.kt1 > t.kt0 ? t.kt1 - t.kt0 : 0;
    // a part has four tiles of keys at least
    t.parts = n / 4 < a.splits ? (n / 4 > 1 ? n / 4 : 1) : a.splits;
    t.per = (n + t.parts - 1) / t.parts;
    return true;
}

// MIXED: the first a.workers workgroups take the sequences of few rows, whose reads pass
// beside the products of the others.
template <int DP, bool I8, bool MIXED>
__global__ __launch_bounds__(256, tile_waves(DP, MIXED)) void tile_kernel(Attn a) {
    constexpr int KW = kTileKeys / 4;  // keys that a wave copies
    constexpr int S = tile_stages(DP, I8);
    constexpr int KS = DP / 16, DB = DP / 32, CH = DP / 8;
    constexpr int TB = kTileKeys * DP * 2;  // bytes of a K or V tile
    constexpr int NL = KW * DP * (I8 ? 1 : 2) / 1024;  // copies of a wave and tile, K or V
    extern __shared__ __align__(16) char smem[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, H = lane >> 5;
    float* scales = reinterpret_cast<float*>(smem + 2 * S * TB);  // [2][3][64]
    int* sh = reinterpret_cast<int*>(smem + tile_lds<DP, I8>() - 64);

    if constexpr (MIXED)
        if ((int)blockIdx.x < a.workers) {
            few_work<DP, I8, 1>(a, blockIdx.x, smem);
            return;
        }
    const int id = blockIdx.x - (MIXED ? a.workers : 0);
    // a key head's items are neighbours modulo the heads: with the round-robin dispatch
    // over the 8 XCDs they share an L2 where the heads divide 8
    const int rest = over(id, a.by_heads), h = id - rest * a.Hk;
    const int item = over(rest, a.by_splits), split = rest - item * a.splits;
    TileItem t{};
    const bool found = tile_item(a, item, h, sh, t);
    const int index = item * a.Hk + h;
    if (a.splits > 1 && split == 0 && threadIdx.x == 0) {
        const int tile_row0 = t.tile * kTileRows;
        Join j{};
        if (found && t.parts > 1)
            j = Join{t.parts, index * a.splits, index * a.splits + 1, 1, t.q.start, tile_row0,
                     t.rows - tile_row0 < kTileRows ? t.rows - tile_row0 : kTileRows, h,
                     t.q.L - t.q.n};
        a.tile_joins[index] = j;
    }
    if (!found || split >= t.parts) return;
    const int first = t.kt0 + split * t.per;
    const int last = first + t.per < t.kt1 ? first + t.per : t.kt1;

    const int row0 = t.tile * kTileRows + wave * 32;
    const int nrows = t.rows - row0 < 32 ? t.rows - row0 : 32;  // may be 0 or less
    const int pmin = position(a, t.q, over(row0, a.by_group));
    const int pmax = nrows > 0 ? position(a, t.q, over(row0 + nrows - 1, a.by_group)) : -1;
    int prow = -1;
    h8 q[KS];
    const int r = row0 + col, qi = over(r, a.by_group), head = h * a.group + r - qi * a.group;
    if (r < t.rows) prow = position(a, t.q, qi);
#pragma unroll
    for (int k = 0; k < KS; k++) {
        u32x4 v = {0, 0, 0, 0};
        if (r < t.rows && 16 * k + 8 * H < a.D)
            v = *reinterpret_cast<const u32x4*>(a.q + (t.q.start + qi) * a.ldq + head * a.hsq +
                                                16 * k + 8 * H);
        v ^= a.flip;
        q[k] = __builtin_bit_cast(h8, v);
    }
    // the queries, asked for before the first copies, waited for behind them and not in the
    // loop, where a wait for a load is one for every copy
    auto queries_landed = [&] {
#pragma unroll
        for (int k = 0; k < KS; k++) {
            u32x4 v = __builtin_bit_cast(u32x4, q[k]);
            asm volatile("" : "+v"(v));
            q[k] = __builtin_bit_cast(h8, v);
        }
    };

    // the row sees the keys j with prow - span < j <= prow: one unsigned comparison
    const uint32_t span = prow < 0 ? 0 : a.window ? a.window : prow + 1;
    const uint32_t seen0 = 4 * H - (prow + 1 - (int)span);

    // chunk ch of key t: K rows are read by 32 keys at one chunk, V rows by 4 keys at 4
    // chunks (transposing); both permutations put those on different banks
    auto k_swz = [](int t) { return DP == 64 ? (t >> 1) & 7 : t & 15; };
    auto v_swz = [](int t) { return DP == 64 ? ((t >> 1) & 1) << 2 : (t & 3) << 2; };

    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)smem;
    // The permutations split into a part of the lane and one of the fragment, so a fragment's
    // address is one of a few registers and a constant.
    constexpr int KA = KS < 8 ? KS : 8, VA = DB < 4 ? DB : 4;
    uint32_t k_addr[KA], v_addr[VA];
#pragma unroll
    for (int i = 0; i < KA; i++) k_addr[i] = lds0 + col * DP * 2 + 16 * ((2 * i + H) ^ k_swz(col));
#pragma unroll
    for (int d = 0; d < VA; d++) {
        const int tk = 4 * H + ((lane & 15) >> 2);
        const int dd = 32 * d + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        v_addr[d] = lds0 + TB + tk * DP * 2 + 16 * ((dd >> 3) ^ v_swz(tk)) + 2 * (dd & 7);
    }
    // Byte offsets of the wave's copies (16 bits) from its first row; elements past the head's
    // are zeros in K, and in V, where they only reach sums that nobody reads, the row's first.
    uint32_t k_off[I8 ? 1 : NL], v_off[I8 ? 1 : NL], k_pad = 0;
    if constexpr (!I8)
#pragma unroll
        for (int j = 0; j < NL; j++) {
            const int c = j * 64 + lane, k = c / CH;
            const int dk = 8 * (c % CH ^ k_swz(KW * wave + k)), dv = 8 * (c % CH ^ v_swz(KW * wave + k));
            k_off[j] = (k * a.D + dk) * 2;
            v_off[j] = (k * a.D + (dv < a.D ? dv : 0)) * 2;
            if (dk >= a.D) k_pad |= 1u << j;
        }

    // Lane j: where the wave's rows of tile j of the 64 ahead begin in the caches (elements).
    // whole: the tiles whose rows all lie in the range and on a page of the cache.
    int64_t rows_ahead = 0;
    uint64_t whole = 0;
    struct Rows {
        int64_t row;
        bool whole;
    };
    auto rows_of = [&](int kt) {
        const int i = kt - first;
        if ((i & 63) == 0) {
            const int tok = (kt + lane) * kTileKeys + KW * wave;
            const int page = kt + lane < last ? page_of(a, t.s, tok & ~15, t.lo, t.hi) : kNone;
            rows_ahead = (((int64_t)(page < 0 ? 0 : page) * a.Hk + h) << a.plog) +
                         (tok & ((1 << a.plog) - 1));
            whole = __ballot(page >= 0 && tok >= t.lo && tok + KW <= t.hi);
        }
        Rows r;
        const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)rows_ahead, i & 63);
        const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(rows_ahead >> 32), i & 63);
        r.row = (int64_t)((uint64_t)hi << 32 | lo);
        r.whole = whole >> (i & 63) & 1;
        return r;
    };
    u32x4 kr[I8 ? NL : 1], vr[I8 ? NL : 1];
    float ksr = 0.0f, vsr = 1.0f;
    // Begins the copies of the wave's rows of a K or V tile (16 bits).
    auto copy_keys = [&](int kt, int stage, Rows r) {
        const uint32_t to = lds0 + stage * 2 * TB + KW * wave * DP * 2;
        const char* p = static_cast<const char*>(scalar(static_cast<const uint16_t*>(a.kc) + r.row * a.D));
        if (r.whole && a.D == DP) {
#pragma unroll
            for (int j = 0; j < NL; j++) copy16_s(to + j * 1024, p, k_off[j]);
            return;
        }
        const int page = r.whole ? 0 : page_of(a, t.s, (kt * kTileKeys + KW * wave) & ~15, t.lo, t.hi);
#pragma unroll
        for (int j = 0; j < NL; j++) {
            const bool pad = k_pad >> j & 1;
            const void* src = p + k_off[j];
            if (pad || page < 0) src = page == kBad && !pad ? &kNaNs : &kZeros;
            copy16(to + j * 1024, src);
        }
    };
    auto copy_values = [&](int kt, int stage, Rows r) {
        const uint32_t to = lds0 + stage * 2 * TB + TB + KW * wave * DP * 2;
        const char* p = static_cast<const char*>(scalar(static_cast<const uint16_t*>(a.vc) + r.row * a.D));
        if (r.whole) {
#pragma unroll
            for (int j = 0; j < NL; j++) copy16_s(to + j * 1024, p, v_off[j]);
            return;
        }
        const int tok = kt * kTileKeys + KW * wave;
        const int page = page_of(a, t.s, tok & ~15, t.lo, t.hi);
#pragma unroll
        for (int j = 0; j < NL; j++) {
            const int k = (j * 64 + lane) / CH;
            const void* src = p + v_off[j];
            // what lies outside the range may be anything, and 0 * NaN is NaN
            if (page < 0 || tok + k >= t.hi || tok + k < t.lo) src = &kZeros;
            copy16(to + j * 1024, src);
        }
    };
    auto begin = [&](int kt, int stage) {
        const Rows rw = rows_of(kt);
        if constexpr (I8) {
            const int64_t row = rw.row;
            const int page = rw.whole ? 0 : page_of(a, t.s, (kt * kTileKeys + KW * wave) & ~15, t.lo, t.hi);
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const int c = j * 64 + lane, k = c / (DP / 16), d = 16 * (c % (DP / 16));
                kr[j] = vr[j] = u32x4{0, 0, 0, 0};
                if (page >= 0 && d < a.D) {
                    const int64_t at = (row + k) * a.D + d;
                    kr[j] = *reinterpret_cast<const u32x4*>(static_cast<const int8_t*>(a.kc) + at);
                    vr[j] = *reinterpret_cast<const u32x4*>(static_cast<const int8_t*>(a.vc) + at);
                }
            }
            ksr = page == kBad ? __builtin_nanf("") : 0.0f;
            vsr = 1.0f;
            if (page >= 0) {
                ksr = a.ks[row + lane % KW];
                vsr = a.vs[row + lane % KW];
            }
        } else {
            copy_keys(kt, stage, rw);
            copy_values(kt, stage, rw);
        }
    };
    auto finish = [&](int buf) {
        if constexpr (I8) {
            char* kt = smem + buf * 2 * TB;
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const int c = j * 64 + lane, k = KW * wave + c / (DP / 16), ch = 2 * (c % (DP / 16));
                u32x4 x, y;
                codes16(kr[j], x, y);
                char* at = kt + k * DP * 2;
                *reinterpret_cast<u32x4*>(at + 16 * (ch ^ k_swz(k))) = x;
                *reinterpret_cast<u32x4*>(at + 16 * ((ch + 1) ^ k_swz(k))) = y;
                codes16(vr[j], x, y);
                *reinterpret_cast<u32x4*>(at + TB + 16 * (ch ^ v_swz(k))) = x;
                *reinterpret_cast<u32x4*>(at + TB + 16 * ((ch + 1) ^ v_swz(k))) = y;
            }
            if (lane < KW) {
                float lv, rv;
                value_scale(vsr, lv, rv);
                float* sc = scales + buf * 3 * kTileKeys + KW * wave + lane;
                sc[0] = ksr * a.c;
                sc[kTileKeys] = lv;
                sc[2 * kTileKeys] = rv;
            }
        }
    };

    // m counts once a key was seen: limit, of the exponents over it, is -inf before
    float m = 0.0f, l = 0.0f, limit = -kInf;
    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[d][e] = 0.0f;

    // A tile is computed in three steps: the products S^T = K Q^T, the weights, and the
    // products with the values.  A wave skips tiles that none of its rows sees.
    f32x16 s[2];
    h8 p[4];
    auto active = [&](int kt) {
        const int t0 = kt * kTileKeys;
        return t0 <= pmax && !(a.window && t0 + kTileKeys - 1 <= pmin - a.window);
    };
    constexpr int kArithmetic = 0x6;  // what passes a scheduling barrier: reads and products do not
    uint32_t ka[KA], va[VA];
    auto at_stage = [&](int stage, uint32_t (&out)[KA], const uint32_t (&from)[KA]) {
#pragma unroll
        for (int i = 0; i < KA; i++) {
            out[i] = from[i] + stage * 2 * TB;
            asm volatile("" : "+v"(out[i]));  // what follows is in the reads' constants
        }
    };
    auto v_at_stage = [&](int stage) {
#pragma unroll
        for (int d = 0; d < VA; d++) {
            va[d] = v_addr[d] + stage * 2 * TB;
            asm volatile("" : "+v"(va[d]));
        }
    };
    // Fragment i of 2 KS: 16 elements of 32 keys.  Four are read ahead of their products.
    h8 kf[4];
    auto key_fragment = [&](int i) {
        return lds_read16(ka[(i >> 1) % KA] + 32 * (i & 1) * DP * 2 + (i >> 1) / KA * 256);
    };
    auto first_keys = [&] {
#pragma unroll
        for (int i = 0; i < 4; i++) kf[i] = key_fragment(i);
    };
    auto scores = [&] {
#pragma unroll
        for (int tb = 0; tb < 2; tb++)
#pragma unroll
            for (int e = 0; e < 16; e++) s[tb][e] = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * KS; i++) {
            s[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i & 3], q[i >> 1], s[i & 1], 0, 0, 0);
            if (i + 4 < 2 * KS) kf[i & 3] = key_fragment(i + 4);
            __builtin_amdgcn_sched_barrier(kArithmetic);
        }
    };
    auto weights = [&](int kt, int buf) {
        const int t0 = kt * kTileKeys;
        const float* sc = scales + buf * 3 * kTileKeys;
        // element e of block tb is key 32 tb + 8 (e / 4) + 4 H + e % 4: its exponent
#pragma unroll
        for (int tb = 0; tb < 2; tb++)
#pragma unroll
            for (int e4 = 0; e4 < 4; e4++) {
                if constexpr (I8) {
                    const int at = 32 * tb + 8 * e4 + 4 * H;
                    const f32x4 kx = *reinterpret_cast<const f32x4*>(sc + at);
                    const f32x4 lv = *reinterpret_cast<const f32x4*>(sc + kTileKeys + at);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        s[tb][4 * e4 + e] = __builtin_fmaf(s[tb][4 * e4 + e], kx[e], lv[e]) - m;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        s[tb][4 * e4 + e] = __builtin_fmaf(s[tb][4 * e4 + e], a.c, -m);
                }
            }
        const bool edge = t0 + kTileKeys - 1 > pmin || (a.window && t0 <= pmax - a.window);
        if (edge)
#pragma unroll
            for (int tb = 0; tb < 2; tb++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    if (seen0 + t0 + 32 * tb + 8 * (e >> 2) + (e & 3) >= span) s[tb][e] = -kInf;
                }
        float top = s[0][0];
#pragma unroll
        for (int tb = 0; tb < 2; tb++)
#pragma unroll
            for (int e = 0; e < 16; e++) top = __builtin_fmaxf(top, s[tb][e]);
        top = max_xor32(top);
        // m need not be the maximum: it may lag by kLag, weights are at most 2^kLag then
        if (__any(top > limit)) {
            const float up = top > limit ? top : 0.0f;
            const float keep = limit < 0.0f ? 1.0f : exp2_(-up);  // nothing summed yet: 1
            l *= keep;
#pragma unroll
            for (int d = 0; d < DB; d++) o[d] *= keep;
#pragma unroll
            for (int tb = 0; tb < 2; tb++)
#pragma unroll
                for (int e = 0; e < 16; e++) s[tb][e] -= up;
            m += up;
            if (top > limit) limit = kLag;
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                w[e] = exp2_(s[k >> 1][8 * (k & 1) + e]);
                if constexpr (!I8) l += w[e];
            }
            if constexpr (I8) {
#pragma unroll
                for (int e4 = 0; e4 < 2; e4++) {
                    const f32x4 rv = *reinterpret_cast<const f32x4*>(
                        sc + 2 * kTileKeys + 32 * (k >> 1) + 16 * (k & 1) + 8 * e4 + 4 * H);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        l += w[4 * e4 + e] == 0.0f ? 0.0f : w[4 * e4 + e] * rv[e];
                }
            }
            const u32x4 pk = {pack2(w[0], w[1]), pack2(w[2], w[3]), pack2(w[4], w[5]),
                              pack2(w[6], w[7])};
            p[k] = __builtin_bit_cast(h8, pk);
        }
    };
    // Fragments of V: block d of 32 elements, keys 16 k + {4 H .., 8 + 4 H ..}, in groups of
    // up to four blocks.  Two groups are read ahead of their products.
    constexpr int GD = DB < 4 ? DB : 4, GK = DB / GD;  // blocks of a group, groups of 16 keys
    h8 vf[2][GD];
    auto value_group = [&](int g) {
#pragma unroll
        for (int i = 0; i < GD; i++) {
            const uint32_t at = va[i] + 16 * (g / GK) * DP * 2 + g % GK * 256;
            vf[g & 1][i] = lds_read_tr(at, at + 8 * DP * 2);
        }
    };
    auto first_values = [&](int stage) {
        v_at_stage(stage);
        value_group(0);
        value_group(1);
    };
    auto values = [&](auto ahead) {
#pragma unroll
        for (int g = 0; g < 4 * GK; g++) {
#pragma unroll
            for (int i = 0; i < GD; i++) {
                f32x16& acc = o[g % GK * GD + i];
                acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[g & 1][i], p[g / GK], acc, 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(kArithmetic);
            if (g + 2 < 4 * GK) value_group(g + 2);
            if (g + 2 == 4 * GK) ahead();
            __builtin_amdgcn_sched_barrier(kArithmetic);
        }
    };
    auto compute = [&](int kt, int stage) {
        if (!active(kt)) return;
        at_stage(stage, ka, k_addr);
        first_keys();
        scores();
        // (where the registers allow it, on their way while the weights are computed)
        constexpr bool early = !I8 && DP <= 128;
        if constexpr (early) first_values(stage);
        weights(kt, stage);
        if constexpr (!early) first_values(stage);
        values([] {});
    };

    // What lies at the edge of some row of the workgroup (the same for its four waves).
    const int wg_pmin = position(a, t.q, over(t.tile * kTileRows, a.by_group)), wg_pmax = t.hi - 1;
    auto at_edge = [&](int kt) {
        return kt * kTileKeys + kTileKeys - 1 > wg_pmin ||
               (a.window && kt * kTileKeys <= wg_pmax - a.window);
    };
    // Makes the V rows that the wave copied finite; whether it changed any.
    auto clean = [&](int buf) {
        constexpr int N = KW * DP * 2 / 1024;
        u32x4 v[N];
        uint32_t bits = 0;
        const uint32_t at = lds0 + buf * 2 * TB + TB + KW * wave * DP * 2 + lane * 16;
#pragma unroll
        for (int j = 0; j < N; j++) {
            v[j] = __builtin_bit_cast(u32x4, lds_read16(at + j * 1024));
            bits |= odd_bits(v[j]);
        }
        if (!__any(bits != 0)) return 0;
#pragma unroll
        for (int j = 0; j < N; j++)
            *reinterpret_cast<lds_u32x4*>(at + j * 1024) = finite_part(v[j]);
        return 1;
    };
    auto restore = [&](int kt) {
#pragma unroll 1
        for (int i = 0; i < kTileKeys; i++) {
            const int j = kt * kTileKeys + i;
            if (j > pmax || j < t.lo) continue;
            const int page = __builtin_amdgcn_readfirstlane(page_of(a, t.s, j & ~15, t.lo, t.hi));
            if (page < 0) continue;
            const int64_t row = (((int64_t)page * a.Hk + h) << a.plog) + (j & ((1 << a.plog) - 1));
            const uint16_t* vp = static_cast<const uint16_t*>(a.vc) + row * a.D + 4 * H;
            const bool sees = j - (prow + 1 - (int)span) < span;
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
                for (int e4 = 0; e4 < 4; e4++) {
                    uint2 w = {0, 0};
                    if (sees && 32 * d + 8 * e4 < a.D)
                        w = *reinterpret_cast<const uint2*>(vp + 32 * d + 8 * e4);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        o[d][4 * e4 + e] += odd_part(e < 2 ? w.x : w.y, e & 1);
                }
        }
    };

    if constexpr (I8) {  // one tile ahead in registers
        if (first < last) {
            begin(first, 0);
            finish(0);
            queries_landed();
            __syncthreads();
        }
        for (int kt = first; kt < last; kt++) {
            const int buf = (kt - first) & 1;
            if (kt + 1 < last) begin(kt + 1, 0);
            compute(kt, buf);
            if (kt + 1 < last) finish(buf ^ 1);
            __syncthreads();
        }
    } else {  // S - 1 tiles on their way
        for (int i = 0; i < S - 1; i++)
            if (first + i < last) begin(first + i, i);
        queries_landed();
        int stage = 0, into = S - 1;
        for (int kt = first; kt < last; kt++) {
            // every wave's copies of this tile have landed, and the stage that the next
            // copies go to has been read
            if (kt + S - 1 <= last)
                wait_copies<2 * NL * (S - 2)>();
            else
                wait_copies<0>();
            barrier_all();
            if (kt + S - 1 < last) begin(kt + S - 1, into);
            bool odd = false;
            if (at_edge(kt)) {
                const int mine = clean(stage);
                if (lane == 0) sh[wave] = mine;
                __syncthreads();
                for (int w = 0; w < 4; w++) odd |= sh[w] != 0;
            }
            compute(kt, stage);
            if (odd) restore(kt);
            stage = stage + 1 == S ? 0 : stage + 1;
            into = into + 1 == S ? 0 : into + 1;
        }
    }

    l += __shfl_xor(l, 32, 64);
    if (r >= t.rows) return;
    if (t.parts > 1) {
        float* part = a.tile_part + ((int64_t)index * a.splits + split) * (kTileRows * (DP + 2));
        const int pr = wave * 32 + col;
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int e4 = 0; e4 < 4; e4++) {
                const f32x4 v = {o[d][4 * e4], o[d][4 * e4 + 1], o[d][4 * e4 + 2], o[d][4 * e4 + 3]};
                *reinterpret_cast<f32x4*>(part + pr * DP + 32 * d + 8 * e4 + 4 * H) = v;
            }
        if (H == 0) {
            part[kTileRows * DP + pr] = limit < 0.0f ? -kInf : m;
            part[kTileRows * DP + kTileRows + pr] = l;
        }
        return;
    }
    const float inv = 1.0f / l;
    uint16_t* dst = a.out + ((int64_t)(t.q.start + qi) * a.Hq + head) * a.D;
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int e4 = 0; e4 < 4; e4++) {
            const int at = 32 * d + 8 * e4 + 4 * H;
            uint2 y = {pack2(o[d][4 * e4] * inv, o[d][4 * e4 + 1] * inv),
                       pack2(o[d][4 * e4 + 2] * inv, o[d][4 * e4 + 3] * inv)};
            if (prow < 0) y = uint2{0, 0};
            if (at < a.D) *reinterpret_cast<uint2*>(dst + at) = y;
        }
}

// ---- host --------------------------------------------------------------------------

// How a call is cut up, from what the host knows.
struct Plan {
    int rb;               // 16-row blocks of few_work's rows
    int64_t few;          // new tokens of a sequence that few_work takes at most
    bool use_few, use_tile;
    int64_t most_rows;    // of a sequence in few_work that keeps to the bound
    bool whole;           // few_work splits no item
    int64_t workers;      // of few_work
    int64_t tiles;        // of kTileRows rows, at most
    int splits;
    // of the workspace: Join records and parts of few_work, the same of the tiles
    int64_t joins, part, tile_joins, tile_part, bytes;
};

Div div_by(int64_t d) {
    uint32_t shift = 0;
    while (((int64_t)1 << shift) < d) shift++;
    return {(uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - (uint64_t)d)) / (uint64_t)d + 1), shift};
}

int padded_dim(int64_t D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

Plan plan_of(int64_t T, int64_t Hq, int64_t Hk, int64_t D, int64_t B, int64_t most,
             int64_t max_context, int64_t window = 0) {
    const int64_t group = Hq / Hk, rows = most * group, DP = padded_dim(D);
    Plan p{};
    // two blocks of 16 rows keep their sums in registers up to 128 elements
    p.rb = DP <= 128 && rows <= 32 && rows > 16 ? 2 : 1;
    p.use_tile = rows > 16 * p.rb;
    p.most_rows = rows < 1 ? 1 : rows < 16 * p.rb ? rows : 16 * p.rb;
    // one sequence of many rows: nothing is left for few_work but padding, which the
    // tiles take too
    p.use_few = !p.use_tile || B > 1;
    p.few = !p.use_tile ? 1 << 30 : p.use_few ? 16 * p.rb / group : 0;
    const int64_t units = (max_context + 1 + kUnit - 1) / kUnit;
    p.whole = units <= kWholeUnits;
    p.workers = (B + 1 + T * group / (16 * p.rb)) * Hk * units;
    const int64_t most_workers = p.use_tile ? kMixedWorkers : kWorkers;
    p.workers = !p.use_few ? 0 : p.workers < most_workers ? p.workers : most_workers;
    p.tiles = T * group / kTileRows + B + 1;
    const int64_t items = p.tiles * Hk;
    // Parts of an item so that the items fill the CUs' 512 places once; 2048 keys and more of
    // sequences of their own length, twice, so that the long ones do not end last (8
    // sequences of up to 8500 tokens 277 -> 230 us, 16 of few tokens 139 -> 80; a window
    // makes the lengths equal: 41.5 us, in two parts 54).
    const int64_t full = ((T * group + kTileRows - 1) / kTileRows + B / 2) * Hk;
    const int64_t reach = window && window < max_context ? window : max_context;
    p.splits = (int)(B > 1 && !window ? (1024 + full - 1) / full : 512 / full);
    const int64_t most_parts = reach / (4 * kTileKeys);  // of four tiles of keys at least
    if (p.splits > most_parts) p.splits = (int)most_parts;
    if (p.splits > 16) p.splits = 16;
    if (p.splits < 1) p.splits = 1;
    // in this order, each a multiple of 256 bytes
    const auto round = [](int64_t n) { return (n + 255) & ~(int64_t)255; };
    if (!p.whole) {
        p.joins = round(p.workers * (int64_t)sizeof(Join));
        p.part = round(p.workers * 2 * 16 * p.rb * (DP + 2) * 4);
    }
    if (p.use_tile && p.splits > 1) {
        p.tile_joins = round(items * (int64_t)sizeof(Join));
        p.tile_part = round(items * p.splits * kTileRows * (DP + 2) * 4);
    }
    p.bytes = p.joins + p.part + p.tile_joins + p.tile_part;
    return p;
}

// The LDS limit is an attribute of a kernel on a device: a flag for each pair.
template <auto kernel>
int allow_lds(int bytes) {
    static std::atomic<bool> done[64];
    int dev = 0;
    (void)hipGetDevice(&dev);
    if (dev >= 0 && dev < 64 && done[dev].load(std::memory_order_relaxed)) return FNI8_OK;
    const hipError_t e = hipFuncSetAttribute((const void*)kernel,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) {
        fni8h::set_error_detail("LDS attribute (%d bytes): %s", bytes, hipGetErrorString(e));
        return FNI8_ERR_LAUNCH;
    }
    if (dev >= 0 && dev < 64) done[dev].store(true, std::memory_order_relaxed);
    return FNI8_OK;
}

template <auto kernel>
int run(const Attn& a, int64_t grid, int lds, hipStream_t st) {
    const int rc = allow_lds<kernel>(lds);
    if (rc == FNI8_OK) kernel<<<dim3((uint32_t)grid), 256, lds, st>>>(a);
    return rc;
}

template <int DP, bool I8, int RB>
int run_few(Attn& a, hipStream_t st) {
    if (!a.whole && a.workers > 256 * few_waves(DP, RB)) a.workers = 256 * few_waves(DP, RB);
    return run<few_kernel<DP, I8, RB>>(a, a.workers, few_lds<DP, RB>(), st);
}

template <int DP, bool I8>
int run_all(Attn a, const Plan& p, hipStream_t st) {
    const bool parts = a.joins != nullptr;  // there is a workspace
    a.whole = p.whole || !parts;
    a.workers = (int)p.workers;
    if (a.whole && p.use_few)
        a.workers = (int)((a.nseq + (p.use_tile ? 0 : (int64_t)a.T * a.group / (16 * p.rb))) * a.Hk);
    a.splits = parts ? p.splits : 1;
    a.by_splits = div_by(a.splits);
    const int64_t items = p.tiles * a.Hk;
    int rc;
    if (!p.use_tile) {
        if constexpr (DP <= 128)
            rc = p.rb == 1 ? run_few<DP, I8, 1>(a, st) : run_few<DP, I8, 2>(a, st);
        else
            rc = run_few<DP, I8, 1>(a, st);
    } else if (p.use_few) {
        rc = run<tile_kernel<DP, I8, true>>(a, a.workers + items * a.splits, tile_lds<DP, I8>(), st);
    } else {
        rc = run<tile_kernel<DP, I8, false>>(a, items * a.splits, tile_lds<DP, I8>(), st);
    }
    if (rc) return rc;
    if (a.whole) a.workers = 0;  // none that leaves parts
    const bool few_parts = a.workers > 1, tile_parts = p.use_tile && a.splits > 1;
    if (!few_parts && !tile_parts) return FNI8_OK;
    // four of few_work's rows or 32 of a tile's a workgroup
    const int64_t y = tile_parts ? kTileRows / 32 : (p.most_rows + 3) / 4;
    join_kernel<DP><<<dim3((uint32_t)(a.workers + (tile_parts ? items : 0)), (uint32_t)y), 256, 0, st>>>(
        a, 16 * p.rb);
    return FNI8_OK;
}

}  // namespace

namespace fni8h {

int64_t paged_attention_workspace_bytes(int64_t T, int64_t Hq, int64_t Hk, int64_t D, int64_t B,
                                        int64_t max_seqlen, int64_t max_context) {
    return (plan_of(T, Hq, Hk, D, B, max_seqlen, max_context).bytes + 255) & ~(int64_t)255;
}

int launch_paged_attention(const PagedAttention& p, hipStream_t st) {
    if (p.T == 0) return FNI8_OK;
    const int64_t context = p.max_pages * p.page_size;
    const Plan plan = plan_of(p.T, p.Hq, p.Hk, p.D, p.B, p.max_seqlen, context, p.window);
    const int64_t group = p.Hq / p.Hk;
    // the units' sums, rounded up to the workers', are 32 bits, a grid has 2^32 threads
    const int64_t items = (p.B + 1 + (plan.use_tile ? 0 : p.T * group / (16 * plan.rb))) * p.Hk;
    const int64_t blocks = items + (plan.use_tile ? plan.tiles * p.Hk * plan.splits : 0);
    if (items * ((context + kUnit) / kUnit + 1) + kWorkers > (int64_t)1 << 31 || blocks >= (int64_t)1 << 24) {
        set_error_detail("T=%lld tokens of %lld sequences and %lld keys are too many for one call",
                         (long long)p.T, (long long)p.B, (long long)context);
        return FNI8_ERR_SHAPE;
    }
    Attn a{};
    a.q = p.q; a.ldq = p.ldq; a.hsq = p.hsq;
    a.kc = p.k_cache; a.vc = p.v_cache; a.ks = p.k_scale; a.vs = p.v_scale;
    a.tables = p.block_tables; a.lens = p.context_lens; a.cu = p.cu_seqlens; a.ldt = p.ldt;
    a.out = p.out;
    a.T = (int)p.T; a.Hq = (int)p.Hq; a.Hk = (int)p.Hk; a.D = (int)p.D; a.group = (int)group;
    a.by_group = div_by(group); a.by_heads = div_by(p.Hk); a.by_quads = div_by(p.D / 4);
    a.num_pages = (int)p.num_pages;
    a.plog = __builtin_ctzll((uint64_t)p.page_size);
    a.max_pages = (int)p.max_pages;
    a.B = (int)p.B;
    a.nseq = p.cu_seqlens ? a.B + 1 : a.B;
    // a window that reaches past every key is none
    a.window = p.window > context ? 0 : (int)p.window;
    a.cap = (int)context + 1;
    // a positive factor, so that the largest product is the largest exponent; a scale of 0
    // stays one that makes every exponent 0, but 0 * -inf
    a.c = __builtin_fabsf(p.scale) * 1.44269504088896340736f;
    a.c = a.c > 1e-30f ? a.c : 1e-30f;
    a.flip = p.scale < 0.0f ? 0x80008000u : 0;
    a.few = (int)plan.few;
    if (plan.bytes && p.work_bytes >= plan.bytes) {
        int8_t* at = p.work;
        a.joins = reinterpret_cast<Join*>(at);
        a.part = reinterpret_cast<float*>(at += plan.joins);
        a.tile_joins = reinterpret_cast<Join*>(at += plan.part);
        a.tile_part = reinterpret_cast<float*>(at += plan.tile_joins);
    }
    int rc;
    switch (padded_dim(p.D)) {
        case 64: rc = p.k_scale ? run_all<64, true>(a, plan, st) : run_all<64, false>(a, plan, st); break;
        case 128: rc = p.k_scale ? run_all<128, true>(a, plan, st) : run_all<128, false>(a, plan, st); break;
        default: rc = p.k_scale ? run_all<256, true>(a, plan, st) : run_all<256, false>(a, plan, st);
    }
    if (rc) return rc;
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        set_error_detail("paged_attention launch: %s", hipGetErrorString(e));
        return FNI8_ERR_LAUNCH;
    }
    return FNI8_OK;
}

}  // namespace fni8h
