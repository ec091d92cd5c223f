// nnrh_kvattn.hip -- attention over the quantized key/value cache.
//
// A query row (sequence, token, head) sees a prefix that the whole batch
// shares and its own sequence's tokens. Rows of one key/value head are put
// side by side (all of the batch's for the prefix, a sequence's for its own
// tokens), so that every key is read once for 16 or more rows:
//   S^T = K Q^T   (keys x rows),   O^T = V^T P^T   (elements x rows)
// by 16x16x32 fp16 MFMAs. In this orientation a lane of S^T holds the scores
// of one row, and its eight keys of a 32-key tile are the ones that it needs
// as an operand of the second product, since values lie in that order.
//
// Codes are exact in fp16. A query row is scaled by a power of two to below
// 2^15, where fp16 and bf16 elements are exact (those under 2^-38 of the
// row's largest lose their last bits); an fp32 row is the sum of two fp16
// pieces, 22 bits and more. Weights p = exp(s - max) enter as 2^11 p, where
// max may be one that up to 2^4 outgrow, or for fp32 tensors as 2^15 p in two
// pieces; with them, at 8 bits, the values' scales over their largest power of
// two so far. That rounds a weight to 11 bits (22): a 16-bit result is rounded to as
// many or fewer, and a second piece would be a second product. At 4 bits scale
// (8 bits) times code (3 bits) is formed in the operand, over the largest power of
// two so far as well (eu for values, ek for keys: the units, which sums and scores
// follow when they move). Sums, maxima and the running total are fp32.
//
// A unit serves all of a block's rows, tokens and groups, so what is far below it
// would lose its bits, though a row may see nothing else. Such rows are computed
// again in fp32 (slow_rows): at 4 bits all of a block's where a scale is under
// 2^-17 of the unit, beyond which it and its products are no longer exact; at 8
// bits those whose largest weight times scale is under 2^-12 of it (2^-16 in two
// pieces), where fp16's least step would count for more than an fp32 sum's.
//
// Up to 16 rows (few): the block's waves take tiles in turn, operands go from
// memory to registers, and a tile's registers are asked for again as soon as
// they are used; bound by memory: 48 sequences of up to 8192 tokens, 32 heads
// over 8 of 128, 8 bits, 409 MB in 82 us and 5 of joining, the two back to back 84
// to 86 (a copy's rate: 79).
// More rows (many): the waves take rows, and a tile's codes are turned into
// operands once, in LDS. Bound by the instructions between the products: 128
// sequences after a prefix of 32768, 4 bits, 69 GFLOP in 125 us, the join with it (a
// large library product's rate: 57): matrix units 25 % busy, vector units 50 with
// weights and conversion, the rest waits for LDS and at the tile's barrier.
//
// Keys are split over blocks; each leaves (max, total, mean) of its rows, which
// a second kernel joins in a fixed order. One block that sees everything
// writes the result itself.
#include "nnrh_decode.h"

#include <algorithm>

namespace nnrh {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int AW = 4;              // waves of a block
// Weights are kept as 2^15 p where p <= 1. With one fp16 piece a weight, the
// maximum may lag behind by 2^4, and weights are 2^11 p where p <= 2^4: rescaling
// the sums of 32 rows is then rare instead of usual.
constexpr float kTop = 15.0f, kSlack = 4.0f;
constexpr int kNoUnit = -126;      // the least unit of scales (they are 0 or normal)
// What the products carry; rows beyond it are computed again (slow_rows). A 4-bit
// scale has 8 bits: it and its products with codes are fp16 numbers down to 2^-17
// of the unit. A weight of 8 bits has an fp16 step of 2^-24 whatever its size,
// half of which is 2^-24 of the row's largest where that is 2^-1, an fp32 sum's
// rounding. Raw scores of 8 bits fit fp32 up to scales of 2^64, with room for the
// least factor below.
constexpr int kFarScale = 17;
constexpr float kFarWeight = 0.5f;
constexpr uint32_t kLargeScale = (127 + 64) << 7;   // as bf16
constexpr float kLeast = 1e-37f;   // a factor of 0 would make NaN of a masked score, -inf
constexpr float kNegInf = -__builtin_inff();

struct AttnArgs {
    KvCache c;
    KvAttention a;
    int G;                         // query heads a key/value head
    int rows;                      // batch * seq * q_heads
    int slots, pre_slots;          // partial results a row: prefix ones first
    int pre_chunk, own_chunk;      // tiles of a split
    int pre_groups, own_groups;    // row groups: of 16 rows, or of a block's with many
    int page_shift;                // log2(page_size / 32)
    float* part_o;                 // [rows][slots][hd]: means over a split's keys
    float2* part_ml;               // [rows][slots]: maximum and total of its weights
};

// Tables and lengths are read through the scalar cache: a wait for a vector
// load would wait for every code that was asked for before it.
typedef const __attribute__((address_space(4))) int32_t* scalar_ints;
__device__ __forceinline__ int scalar_load(const int32_t* p, long long i) {
    return ((scalar_ints)(uintptr_t)p)[i];
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// maximum and sum over the lanes that differ in bits 4 and 5 (the four lane
// groups of a row), without a trip through LDS
__device__ __forceinline__ float swap_max(float m, bool wide) {
    const uint32_t u = __builtin_bit_cast(uint32_t, m);
    const auto r = wide ? __builtin_amdgcn_permlane32_swap(u, u, false, false)
                        : __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float max16_32(float m) { return swap_max(swap_max(m, false), true); }
// maximum over 16 neighbouring lanes
template <int CTRL>
__device__ __forceinline__ float dpp_max(float m) {
    const int u = __builtin_bit_cast(int, m);
    return fmaxf(m, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(u, u, CTRL, 0xf, 0xf, false)));
}
__device__ __forceinline__ float max_16(float m) {
    return dpp_max<0x140>(dpp_max<0x141>(dpp_max<0x4e>(dpp_max<0xb1>(m))));   // quads, halves and rows of 16 mirrored
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
// the same on whole numbers (bf16 scales, which are not negative, compare as such)
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t swap_umax(uint32_t u, bool wide) {
    const auto r = wide ? __builtin_amdgcn_permlane32_swap(u, u, false, false)
                        : __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return umax((uint32_t)r[0], (uint32_t)r[1]);
}
__device__ __forceinline__ uint32_t umax16_32(uint32_t u) { return swap_umax(swap_umax(u, false), true); }
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_umax(uint32_t u) {
    return umax(u, (uint32_t)__builtin_amdgcn_update_dpp((int)u, (int)u, CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ uint32_t umax_16(uint32_t u) {
    return dpp_umax<0x140>(dpp_umax<0x141>(dpp_umax<0x4e>(dpp_umax<0xb1>(u))));
}
// exponent e of the least 2^e >= the bf16 number of these bits; none for 0
__device__ __forceinline__ int ceil_exp(uint32_t bf16, int none) {
    return bf16 ? (int)((bf16 + 0x7fu) >> 7) - 127 : none;
}
typedef uint16_t us2 __attribute__((ext_vector_type(2)));
typedef int16_t ss2 __attribute__((ext_vector_type(2)));
// the larger of two pairs of bf16 scales, as bits
__device__ __forceinline__ uint32_t pair_max(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, a), __builtin_bit_cast(us2, b)));
}
__device__ __forceinline__ uint32_t half_max(uint32_t a) { return umax(a & 0xffffu, a >> 16); }

// What is kept of the scales that a wave has seen, to know whether the products
// carried them: at 4 bits the least of keys and values (0 aside), at 8 the
// largest of keys, pairs a lane. (As signed numbers: memory that no token was
// written to may hold a sign.)
template <int BITS> struct Seen;
template <> struct Seen<8> {
    uint32_t k = 0;
    __device__ __forceinline__ void add(u4 w) {
        const auto m = [](uint32_t a, uint32_t b) {
            return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ss2, a), __builtin_bit_cast(ss2, b)));
        };
        k = m(k, m(m(w[0], w[1]), m(w[2], w[3])));
    }
    __device__ __forceinline__ bool far(int, int) const { return half_max(k) >= kLargeScale; }
};
template <> struct Seen<4> {
    uint32_t k = 0xffffffffu, v = 0xffffffffu;   // of bits less 1, where 0 is the largest
    __device__ __forceinline__ static uint32_t least(uint32_t a, uint32_t w) {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(us2, a), __builtin_bit_cast(us2, w) - us2{1, 1}));
    }
    __device__ __forceinline__ void add_k(uint32_t w) { k = least(k, w); }
    __device__ __forceinline__ void add_v(u2 w) { v = least(least(v, w[0]), w[1]); }
    __device__ __forceinline__ void add(u2 wk, u2 wv) {
        add_k(wk[0]);
        add_k(wk[1]);
        add_v(wv);
    }
    __device__ __forceinline__ static bool below(uint32_t a, int unit) {
        return min(a & 0xffffu, a >> 16) < (uint32_t)(max(unit - kFarScale + 127, 1) << 7) - 1;
    }
    __device__ __forceinline__ bool far(int ek, int eu) const { return below(k, ek) || below(v, eu); }
};
// keeps the compiler from computing both sides of a branch that a tile hardly ever takes
__device__ __forceinline__ void stay_a_branch() { asm volatile(""); }

// eight 8-bit codes (code + 128) as fp16
__device__ __forceinline__ h8 codes8(uint32_t lo, uint32_t hi) {
    const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    u4 r;
    r[0] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u);
    r[1] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u);
    r[2] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u);
    r[3] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, (uint32_t)r[i]) - off);
    return __builtin_bit_cast(h8, r);
}
// Eight 4-bit codes (code + 8) times scales s[0..3], a pair each: a nibble q
// under the exponent of 16 is 16 + q, and (16 + q) s - 24 s = code s, where 24 s
// has 10 bits and the result 11.
struct Scale4 {
    h2 s, s24;
    __device__ __forceinline__ void set(_Float16 a, _Float16 b) {
        s = h2{a, b};
        s24 = s * h2{(_Float16)-24.0f, (_Float16)-24.0f};
    }
};
__device__ __forceinline__ h2 pair4(uint32_t w, uint32_t magic, const Scale4& s) {
    return __builtin_elementwise_fma(__builtin_bit_cast(h2, (w & 0x03c003c0u) | magic), s.s, s.s24);
}
__device__ __forceinline__ h8 codes4(uint32_t w, const Scale4& a, const Scale4& b, const Scale4& c, const Scale4& d) {
    // (in a vector register: mask, or and word are then one instruction)
    uint32_t magic;
    asm("v_mov_b32 %0, 0x4c004c00" : "=v"(magic));
    const h2 r[4] = {pair4(w << 4, magic, a), pair4(w, magic, b), pair4(w >> 4, magic, c),
                     pair4(__builtin_amdgcn_alignbit(w, w, 8), magic, d)};
    return h8{r[0][0], r[0][1], r[1][0], r[1][1], r[2][0], r[2][1], r[3][0], r[3][1]};
}

__device__ __forceinline__ void load_q8(const KvAttention& a, long long at, float* v) {
    if (a.type == FT_F32) {
        const f4 x = *(const f4*)((const float*)a.q + at), y = *(const f4*)((const float*)a.q + at + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] = x[j]; v[4 + j] = y[j]; }
        return;
    }
    const u4 x = *(const u4*)((const uint16_t*)a.q + at);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t h = (x[j >> 1] >> (16 * (j & 1))) & 0xffffu;
        v[j] = a.type == FT_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h) : __builtin_bit_cast(float, h << 16);
    }
}
__device__ __forceinline__ void store_y4(const KvAttention& a, long long at, f4 v) {
    if (a.type == FT_F32) {
        *(f4*)((float*)a.y + at) = v;
    } else if (a.type == FT_F16) {
        *(h4*)((_Float16*)a.y + at) = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    } else {
        typedef __bf16 b4 __attribute__((ext_vector_type(4)));
        *(b4*)((__bf16*)a.y + at) = b4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
    }
}

// ---- a wave's rows and what it has found so far ------------------------------
template <int HD, int NP, int NR> struct Rows {
    static constexpr int NC = HD / 32, ND = HD / 16;
    h8 q[NP][NR][NC];
    // A raw score is a product of operands (times the key's scale at 8 bits);
    // the score, in powers of two, is rf 2^ek times as much. rf > 0.
    float rf[NR], rk[NR];   // rk: rf 2^ek
    int ek;             // unit of the keys' operands (4 bits)
    float m[NR];        // raw score that weights refer to: the largest, or less by no more than kSlack (in scores)
    // the total of kTop p: this lane's part (8 bits), or, summed by an MFMA whose
    // other operand is all ones, the whole in every element (4 bits)
    f4 l[NR];
    f4 o[NR][ND];       // sums of kTop p v in units of 2^eu
    int eu;
    float x[NR];        // 8 bits: the largest weight with its value's scale so far, this lane's
    int lim[NR];        // keys that the row sees
    int at[NR];         // its place among all rows
    int lo, hi;         // least and largest limit of the wave's rows
};

// what a block works on
struct Job {
    bool pre;
    int head, b, split, slot;
    int row0;                    // first of the block's rows of this head
    int nrows;                   // rows that the source has for this head
    long long len;               // tokens that the source holds
    int t0, t1;                  // tiles
    const int32_t* table;
};

template <int HD, int NP, int NR>
__device__ __forceinline__ void set_rows(const AttnArgs& p, const Job& job, int row0, Rows<HD, NP, NR>& w) {
    const KvAttention& a = p.a;
    const int col = threadIdx.x & 15;
    w.lo = 0x7fffffff;
    w.hi = 0;
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        int r = row0 + 16 * t + col;
        r = r < job.nrows ? r : job.nrows - 1;
        const int tok = r / p.G, hq = job.head * p.G + (r - tok * p.G);   // tok counts over the batch in the prefix's rows
        w.at[t] = (job.pre ? tok : job.b * a.seq + tok) * a.q_heads + hq;
        long long l = job.len;
        if (!job.pre) {
            const long long last = (long long)scalar_load(a.lens, job.b) - a.seq + tok + 1;
            l = last < l ? last : l;
        }
        w.lim[t] = l > 0 ? (int)l : 0;
        w.lo = min(w.lo, w.lim[t]);
        w.hi = max(w.hi, w.lim[t]);
    }
#pragma unroll
    for (int o = 1; o < 16; o *= 2) {
        w.lo = min(w.lo, __shfl_xor(w.lo, o));
        w.hi = max(w.hi, __shfl_xor(w.hi, o));
    }
    w.lo = __builtin_amdgcn_readfirstlane(w.lo);
    w.hi = __builtin_amdgcn_readfirstlane(w.hi);
}

template <int BITS, int HD, int NP, int NR>
__device__ __forceinline__ void clear_rows(Rows<HD, NP, NR>& w) {
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        w.m[t] = kNegInf;
        w.l[t] = f4{0, 0, 0, 0};
        w.x[t] = 0.0f;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) w.o[t][d] = f4{0, 0, 0, 0};
    }
    w.eu = kNoUnit;
    w.ek = BITS == 8 ? 0 : kNoUnit;
}
template <int BITS, int HD, int NP, int NR>
__device__ __forceinline__ void load_rows(const AttnArgs& p, Rows<HD, NP, NR>& w) {
    constexpr int NC = HD / 32;
    const KvAttention& a = p.a;
    const int g = (threadIdx.x & 63) >> 4;
    const bool neg = a.scale < 0.0f;   // the sign goes into the row, so that rf is positive
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        const int bt = w.at[t] / a.q_heads, hq = w.at[t] - bt * a.q_heads;
        const int bq = bt / a.seq;
        const long long at = (long long)bq * a.q_bstride + (long long)(bt - bq * a.seq) * a.q_tstride + (long long)hq * HD + 8 * g;
        float v[NC][8], top = 0.0f;
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            load_q8(a, at + 32 * k, v[k]);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[k][j]));
        }
        top = max16_32(top);
        int e = 0;
        if (top > 0.0f && top < __builtin_inff()) e = 15 - __builtin_amdgcn_frexp_expf(top);
        w.rf[t] = ldexpf(fabsf(a.scale) * 1.44269504088896341f, -e);
        w.rk[t] = fmaxf(w.rf[t], kLeast);
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float s = ldexpf(neg ? -v[k][j] : v[k][j], e);
                if constexpr (NP == 2) asm("" : "+v"(s));   // (both pieces are of this, as below)
                const _Float16 h = (_Float16)s;
                w.q[0][t][k][j] = h;
                if constexpr (NP == 2) w.q[1][t][k][j] = (_Float16)(s - (float)h);
            }
    }
    clear_rows<BITS>(w);
}

// element j of 8 bf16 numbers
__device__ __forceinline__ float bf16_at(u4 w, int j) { return j & 1 ? bf16_hi(w[j >> 1]) : bf16_lo(w[j >> 1]); }

// KT tiles from key `key0` on against a wave's rows. key(z, 2 c + i): elements
// 32 c .. of keys 16 i .. of tile z as an operand; value(z, 2 c + i): elements
// 32 c + 16 i .. of its keys. They are asked for a tile before they are used.
// ks, vs: scales of this lane's 8 keys (8 bits; vs are 0 where there is no token;
// at 4 bits scales are in the operands, keys' over 2^ek, values' over 2^en). ek,
// en: the units from here on. held: tokens in each tile; some: not all have 32.
// after_keys, after_values: what can be done while the first are on their way.
template <int HD, int BITS, int NP, int NR, int KT, class Key, class Value, class AfterKeys, class AfterValues>
__device__ __forceinline__ void tile_step(Rows<HD, NP, NR>& w, int key0, const int* held, bool some, const u4* ks,
                                          const u4* vs, int ek, int en, Key key, Value value, AfterKeys after_keys,
                                          AfterValues after_values) {
    constexpr int NC = HD / 32, ND = HD / 16;
    constexpr float slack = NP == 1 ? kSlack : 0.0f, top = NP == 1 ? kTop - kSlack : kTop;
    const int g = (threadIdx.x & 63) >> 4;
    h8 kf[2 * NC];
#pragma unroll
    for (int j = 0; j < 2 * NC; ++j) kf[j] = key(0, j);
    __builtin_amdgcn_sched_barrier(0);
    after_keys();
    f4 acc[NR][KT][2];
#pragma unroll
    for (int t = 0; t < NR; ++t)
#pragma unroll
        for (int z = 0; z < KT; ++z) acc[t][z][0] = acc[t][z][1] = f4{0, 0, 0, 0};
#pragma unroll
    for (int z = 0; z < KT; ++z)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int t = 0; t < NR; ++t)
#pragma unroll
                    for (int q = 0; q < NP; ++q)
                        acc[t][z][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[2 * c + i], w.q[q][t][c], acc[t][z][i], 0, 0, 0);
                if (z + 1 < KT) kf[2 * c + i] = key(z + 1, 2 * c + i);
            }
    h8 vf[2 * NC];
#pragma unroll
    for (int j = 0; j < 2 * NC; ++j) vf[j] = value(0, j);
    __builtin_amdgcn_sched_barrier(0);
    after_values();
    if (BITS == 4 && ek != w.ek) {
        stay_a_branch();
#pragma unroll
        for (int t = 0; t < NR; ++t) {
            w.m[t] = ldexpf(w.m[t], w.ek - ek);
            w.rk[t] = fmaxf(ldexpf(w.rf[t], ek), kLeast);
        }
        w.ek = ek;
    }
    // raw scores of 2 x 4 keys a tile and row: key 16 i + 4 g + r in element 4 i + r
    float s[NR][KT][8];
#pragma unroll
    for (int t = 0; t < NR; ++t)
#pragma unroll
        for (int z = 0; z < KT; ++z)
#pragma unroll
            for (int j = 0; j < 8; ++j) s[t][z][j] = BITS == 8 ? acc[t][z][j >> 2][j & 3] * bf16_at(ks[z], j) : acc[t][z][j >> 2][j & 3];
    if (key0 + 32 * KT > w.lo || some) {
        stay_a_branch();
#pragma unroll
        for (int t = 0; t < NR; ++t)
#pragma unroll
            for (int z = 0; z < KT; ++z) {
                const int end = min(w.lim[t] - key0 - 32 * z, held[z]) - 4 * g;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (16 * (j >> 2) + (j & 3) >= end) s[t][z][j] = kNegInf;
            }
    }
    // running maximum: moved on only where a score outgrows it by more than the slack
    float mx[NR];
    bool moved = false;
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        mx[t] = s[t][0][0];
#pragma unroll
        for (int z = 0; z < KT; ++z)
#pragma unroll
            for (int j = 0; j < 8; ++j) mx[t] = fmaxf(mx[t], s[t][z][j]);
        mx[t] = max16_32(mx[t]);
        moved |= slack == 0.0f ? mx[t] > w.m[t] : mx[t] * w.rk[t] > __builtin_fmaf(w.m[t], w.rk[t], slack);
    }
    if (__any(moved) || en != w.eu) {
        stay_a_branch();
#pragma unroll
        for (int t = 0; t < NR; ++t) {
            const float m = fmaxf(w.m[t], mx[t]);
            const float al = m == w.m[t] ? 1.0f : exp2_((w.m[t] - m) * w.rk[t]);
            w.m[t] = m;
            w.l[t] *= al;
            const float f = ldexpf(al, w.eu - en);
            if constexpr (BITS == 8) w.x[t] *= f;
#pragma unroll
            for (int d = 0; d < ND; ++d) w.o[t][d] *= f;
        }
        w.eu = en;
    }
    // weights kTop p
    const float fv = ldexpf(1.0f, -en);
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        const float base = w.m[t] == kNegInf ? 0.0f : w.m[t] * w.rk[t];
        const float off = top - base;
#pragma unroll
        for (int z = 0; z < KT; ++z)
#pragma unroll
            for (int j = 0; j < 8; ++j) s[t][z][j] = exp2_(__builtin_fmaf(s[t][z][j], w.rk[t], off));
        if constexpr (BITS == 8) {
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int z = 0; z < KT; ++z)
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[j & 1] += s[t][z][j];
            w.l[t][0] += sum[0] + sum[1];
        }
    }
#pragma unroll
    for (int z = 0; z < KT; ++z) {
        h8 pf[NP][NR];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float vu = BITS == 8 ? bf16_at(vs[z], j) * fv : 1.0f;
#pragma unroll
            for (int t = 0; t < NR; ++t) {
                float x = BITS == 8 ? s[t][z][j] * vu : s[t][z][j];
                // Both pieces are of x as fp32 holds it. Left to itself the compiler takes
                // the second from an fp16 of the product, rounded once, and next to a tie
                // that is not the first.
                if constexpr (NP == 2) asm("" : "+v"(x));
                if constexpr (BITS == 8) w.x[t] = fmaxf(w.x[t], x);
                const _Float16 h = (_Float16)x;
                pf[0][t][j] = h;
                if constexpr (NP == 2) pf[1][t][j] = (_Float16)(x - (float)h);
            }
        }
        if constexpr (BITS == 4) {
            h8 ones;
#pragma unroll
            for (int j = 0; j < 8; ++j) ones[j] = (_Float16)1.0f;
#pragma unroll
            for (int t = 0; t < NR; ++t)
#pragma unroll
                for (int q = 0; q < NP; ++q)
                    w.l[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pf[q][t], w.l[t], 0, 0, 0);
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
#pragma unroll
            for (int t = 0; t < NR; ++t)
#pragma unroll
                for (int q = 0; q < NP; ++q)
                    w.o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[d], pf[q][t], w.o[t][d], 0, 0, 0);
            if (z + 1 < KT) vf[d] = value(z + 1, d);
        }
    }
}

template <int BITS>
__device__ __forceinline__ float row_total(f4 l) {
    if (BITS == 4) return l[0];
    float x = l[0] + __shfl_xor(l[0], 16);
    return x + __shfl_xor(x, 32);
}

// ---- a tile in memory ---------------------------------------------------------
struct TilePtr {
    const uint8_t* codes;        // keys' blocks; values' vcodes further
    const uint16_t* scales;      // keys'; values' vscales further
    bool ok;                     // the page exists (else this is page 0, of which no token counts)
};
template <int HD, int BITS>
__device__ __forceinline__ TilePtr tile_ptr(const AttnArgs& p, int head, int id, int tile) {
    constexpr int BB = BITS == 8 ? 1024 : 512;
    const KvCache& c = p.c;
    TilePtr r;
    r.ok = id >= 0 && id < c.num_pages;
    const int in_page = tile & ((1 << p.page_shift) - 1);
    const uint8_t* base = c.data + ((long long)(r.ok ? id : 0) * c.heads + head) * kv_head_bytes(c.page_size, HD, BITS);
    r.codes = base + (long long)in_page * (HD / 32) * BB;
    r.scales = (const uint16_t*)(base + 2 * kv_codes_bytes(c.page_size, HD, BITS)) + in_page * 32;
    return r;
}
// 8 scales of a lane's keys; those past `held` become 0
__device__ __forceinline__ u4 held_scales(u4 w, int held) {
    if (held < 32) {
        stay_a_branch();
        const int end = held - 4 * (int)((threadIdx.x & 63) >> 4);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (16 * (j >> 2) + (j & 3) >= end) w[j >> 1] &= j & 1 ? 0xffffu : 0xffff0000u;
    }
    return w;
}
// the largest of a lane's 8 scales, as bits of bf16
__device__ __forceinline__ uint32_t top8(u4 w) { return half_max(pair_max(pair_max(w[0], w[1]), pair_max(w[2], w[3]))); }
// Scales of a tile, all groups', 4 a lane (4 bits): those of keys or of values
__device__ __forceinline__ u2 all_scales(const uint16_t* first, int page, int groups) {
    const int lane = threadIdx.x & 63, grp = lane >> 3 < groups ? lane >> 3 : 0;
    return *(const u2*)(first + grp * page + (lane & 7) * 4);
}
// without what the tile's tokens do not hold
__device__ __forceinline__ u2 of_tokens(u2 w, int held, bool key) {
    if (held < 32) {
        stay_a_branch();
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int slot = (lane & 7) * 4 + q;
            const int tok = key ? (slot >> 1) + 16 * (slot & 1) : 16 * ((slot >> 2) & 1) + 4 * (slot >> 3) + (slot & 3);
            if (tok >= held) w[q >> 1] &= q & 1 ? 0xffffu : 0xffff0000u;
        }
    }
    return w;
}
// the unit of a tile's scales, at least `unit`
__device__ __forceinline__ int unit_of(uint32_t pairs, int unit) {
    return max(unit, ceil_exp(__builtin_amdgcn_readfirstlane(umax16_32(umax_16(half_max(pairs)))), kNoUnit));
}
// the pair of scales of keys col and col + 16 (4 bits); 0 past `held`
__device__ __forceinline__ uint32_t held_pair(uint32_t w, int held) {
    if (held < 32) {
        stay_a_branch();
        const int col = threadIdx.x & 15;
        if (col >= held) w &= 0xffff0000u;
        if (col + 16 >= held) w &= 0xffffu;
    }
    return w;
}
__device__ __forceinline__ h8 key4(uint32_t codes, float scale, float unit) {
    const _Float16 x = (_Float16)(scale * unit);
    Scale4 s;
    s.set(x, x);
    return codes4(codes, s, s, s, s);
}
__device__ __forceinline__ void value_scales(u4 w, float unit, Scale4* s) {
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j].set((_Float16)(bf16_lo(w[j]) * unit), (_Float16)(bf16_hi(w[j]) * unit));
}

__device__ __forceinline__ int page_id(const Job& job, const AttnArgs& p, int tile) {
    return scalar_load(job.table, tile >> p.page_shift);
}

// ---- few rows: the block's waves split its keys -------------------------------
// A wave has the codes of one tile on their way: as soon as its keys are turned
// into operands, the next tile's are asked for, and so the values.
template <int HD, int BITS> struct RawTile {
    static constexpr int NC = HD / 32;
    typedef uint32_t vec __attribute__((ext_vector_type(BITS == 8 ? 4 : 2)));
    vec k[NC], v[NC];
    u4 vs[BITS == 8 ? 1 : NC];
    u4 ks;                        // 8 bits
    uint32_t ks4[NC];             // 4 bits
    u2 all_v;                     // 4 bits: the values', 4 a lane
    __device__ __forceinline__ void load_keys(const AttnArgs& p, const TilePtr& t) {
        constexpr int BB = BITS == 8 ? 1024 : 512;
        const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
        if constexpr (BITS == 8) {
            ks = *(const u4*)(t.scales + 8 * g);
        } else {
#pragma unroll
            for (int c = 0; c < NC; ++c) ks4[c] = *(const uint32_t*)(t.scales + c * p.c.page_size + 2 * col);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) k[c] = *(const vec*)(t.codes + c * BB + lane * sizeof(vec));
    }
    __device__ __forceinline__ void load_values(const AttnArgs& p, const TilePtr& t) {
        constexpr int BB = BITS == 8 ? 1024 : 512;
        const int lane = threadIdx.x & 63, g = lane >> 4;
        const uint8_t* vc = t.codes + kv_codes_bytes(p.c.page_size, HD, BITS);
        const uint16_t* vsp = t.scales + (long long)p.c.page_size * kv_groups(HD, BITS);
        if constexpr (BITS == 4) all_v = all_scales(vsp, p.c.page_size, NC);
#pragma unroll
        for (int c = 0; c < (BITS == 8 ? 1 : NC); ++c) vs[c] = *(const u4*)(vsp + c * p.c.page_size + 8 * g);
#pragma unroll
        for (int c = 0; c < NC; ++c) v[c] = *(const vec*)(vc + c * BB + lane * sizeof(vec));
    }
};

// next: the tile to load meanwhile
template <int HD, int BITS, int NP>
__device__ __forceinline__ void few_tile(const AttnArgs& p, Rows<HD, NP, 1>& w, Seen<BITS>& scales, RawTile<HD, BITS>& r,
                                         int tile, int held, const TilePtr& next) {
    constexpr int NC = HD / 32;
    u4 vs[BITS == 8 ? 1 : NC];
#pragma unroll
    for (int c = 0; c < (BITS == 8 ? 1 : NC); ++c) vs[c] = held_scales(r.vs[c], held);
    int ek = 0, en;
    const u4 ks = r.ks;
    uint32_t kb[NC];
    if constexpr (BITS == 4) {
        const u2 v = of_tokens(r.all_v, held, false);
        scales.add_v(v);
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            kb[c] = held_pair(r.ks4[c], held);
            scales.add_k(kb[c]);
            top = pair_max(top, kb[c]);
        }
        ek = max(w.ek, ceil_exp(__builtin_amdgcn_readfirstlane(umax_16(half_max(top))), kNoUnit));
        en = unit_of(pair_max(v[0], v[1]), w.eu);
    } else {
        scales.add(ks);
        en = max(w.eu, ceil_exp(__builtin_amdgcn_readfirstlane(umax16_32(top8(vs[0]))), kNoUnit));
    }
    const float fk = ldexpf(1.0f, -ek), fv = ldexpf(1.0f, -en);
    tile_step<HD, BITS, NP, 1, 1>(
        w, tile * 32, &held, held < 32, &ks, vs, ek, en,
        [&](int, int j) {
            if constexpr (BITS == 8) return codes8(r.k[j >> 1][2 * (j & 1)], r.k[j >> 1][2 * (j & 1) + 1]);
            else return key4(r.k[j >> 1][j & 1], j & 1 ? bf16_hi(kb[j >> 1]) : bf16_lo(kb[j >> 1]), fk);
        },
        [&](int, int j) {
            if constexpr (BITS == 8) {
                return codes8(r.v[j >> 1][2 * (j & 1)], r.v[j >> 1][2 * (j & 1) + 1]);
            } else {
                Scale4 s[4];
                value_scales(vs[j >> 1], fv, s);
                return codes4(r.v[j >> 1][j & 1], s[0], s[1], s[2], s[3]);
            }
        },
        [&] {
            r.load_keys(p, next);
            __builtin_amdgcn_sched_barrier(0);
        },
        [&] {
            r.load_values(p, next);
            __builtin_amdgcn_sched_barrier(0);
        });
}

// The results of a wave's rows, sums in units of 2^unit: into the call's result,
// or among the parts. Divided by the total first: a sum of values and weights of
// up to 2^15 may pass the largest number where their mean does not. Not those
// that are computed again.
template <int HD, int NP, int NR>
__device__ __forceinline__ void put_rows(const AttnArgs& p, const Job& job, int row0, const Rows<HD, NP, NR>& w, int unit,
                                         const float* m, const float* l, const bool* again) {
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        if (row0 + 16 * t + col >= job.nrows || again[t]) continue;
        const bool none = m[t] == kNegInf && l[t] == 0.0f;
        const float inv = none ? 0.0f : 1.0f / l[t];
        const auto mean = [&](int d) {
            const f4 o = w.o[t][d] * inv;
            return f4{ldexpf(o[0], unit), ldexpf(o[1], unit), ldexpf(o[2], unit), ldexpf(o[3], unit)};
        };
        if (p.slots > 1) {
            const long long at = (long long)w.at[t] * p.slots + job.slot;
            if (g == 0) p.part_ml[at] = float2{m[t], l[t]};
            if (none) continue;
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) *(f4*)(p.part_o + at * HD + 16 * d + 4 * g) = mean(d);
        } else {
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) store_y4(p.a, (long long)w.at[t] * HD + 16 * d + 4 * g, mean(d));
        }
    }
}

// ---- rows that the products do not carry --------------------------------------
// One row by one wave in fp32, from the codes: a lane scores half of a key's
// elements, and holds elements 64 apart of the result, the mean so far. As near
// to a sum in fp32 as that comes whatever the sizes of queries, keys and values,
// and some 50 times as slow as the products.
template <int HD, int BITS, int NP>
__device__ __forceinline__ void slow_row(const AttnArgs& p, const Job& job, int row, int lim) {
    constexpr int NC = HD / 32, BB = BITS == 8 ? 1024 : 512, NE = (HD + 63) / 64;
    const KvAttention& a = p.a;
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));   // nothing of this path in registers before it
    const int tok = lane & 31, half = lane >> 5;
    const int bt = row / a.q_heads, hq = row - bt * a.q_heads, bq = bt / a.seq;
    const long long q0 = (long long)bq * a.q_bstride + (long long)(bt - bq * a.seq) * a.q_tstride + (long long)hq * HD;
    const long long vcodes = kv_codes_bytes(p.c.page_size, HD, BITS), vscales = (long long)p.c.page_size * kv_groups(HD, BITS);
    float m = kNegInf, l = 0.0f, y[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) y[i] = 0.0f;
    const int t1 = min(job.t1, (lim + 31) / 32);
    for (int tile = job.t0; tile < t1; ++tile) {
        const TilePtr t = tile_ptr<HD, BITS>(p, job.head, page_id(job, p, tile), tile);
        if (!t.ok) continue;
        const int seen = min(lim - 32 * tile, 32);   // (a row's limit is within what the source holds)
        float s = 0.0f;
#pragma unroll 1
        for (int c = 0; c < NC; ++c) {
            const uint32_t sb = t.scales[BITS == 8 ? kv_slot(tok) : c * p.c.page_size + kv_pair(tok)];
            const float scale = bf16_lo(sb);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int oct = 2 * half + i;
                const uint8_t* from = t.codes + c * BB + ((tok & 15) + 16 * oct) * (BITS == 8 ? 16 : 8) + (tok >> 4) * (BITS == 8 ? 8 : 4);
                float q[8];
                load_q8(a, q0 + 32 * c + 8 * oct, q);
                u2 w = {0, 0};
                if constexpr (BITS == 8) w = *(const u2*)from;
                else w[0] = kv_unturn(*(const uint32_t*)from);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int code = BITS == 8 ? (int)((w[j >> 2] >> (8 * (j & 3))) & 255u) - 128
                                               : (int)((w[0] >> (4 * ((j >> 1) + 4 * (j & 1)))) & 15u) - 8;
                    s = __builtin_fmaf(q[j] * a.scale, (float)code * scale, s);
                }
            }
        }
        s = (s + __shfl_xor(s, 32)) * 1.44269504088896341f;
        if (tok >= seen) s = kNegInf;
        const float top = fmaxf(m, max16_32(max_16(s)));
        const float base = top == kNegInf ? 0.0f : top;
        const float w = exp2_(s - base);
        float sum = tok >= seen || half ? 0.0f : w;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) sum += __shfl_xor(sum, o);
        const float old = l * exp2_(m - base);
        l = old + sum;
        m = top;
        const float inv = 1.0f / l;
#pragma unroll
        for (int i = 0; i < NE; ++i) y[i] *= old * inv;
#pragma unroll 1
        for (int k = 0; k < seen; ++k) {
            const float wk = __shfl(w, k) * inv;
            const int slot = kv_slot(k);
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const int e = min(lane + 64 * i, HD - 1), c = e >> 5;
                const float scale = bf16_lo(t.scales[vscales + (BITS == 8 ? 0 : c * p.c.page_size) + slot]);
                const uint8_t* from = t.codes + vcodes + c * BB + ((e & 15) + 16 * (slot >> 3)) * (BITS == 8 ? 16 : 8) +
                                      ((e >> 4) & 1) * (BITS == 8 ? 8 : 4);
                int code;
                if constexpr (BITS == 8) code = (int)from[slot & 7] - 128;
                else code = (int)((kv_unturn(*(const uint32_t*)from) >> (4 * (((slot & 7) >> 1) + 4 * (slot & 1)))) & 15u) - 8;
                y[i] = __builtin_fmaf(wk, (float)code * scale, y[i]);
            }
        }
    }
    // as the products leave it: totals are of weights with their largest at 2^top
    constexpr float unit = NP == 1 ? kTop - kSlack : kTop;
    const long long part = (long long)row * p.slots + job.slot;
    if (p.slots > 1 && lane == 0) p.part_ml[part] = float2{m, ldexpf(l, (int)unit)};
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        const int e = lane + 64 * i;
        if (HD % 64 && e >= HD) break;
        if (p.slots > 1) p.part_o[part * HD + e] = y[i];
        else if (a.type == FT_F32) ((float*)a.y)[(long long)row * HD + e] = y[i];
        else if (a.type == FT_F16) ((_Float16*)a.y)[(long long)row * HD + e] = (_Float16)y[i];
        else ((__bf16*)a.y)[(long long)row * HD + e] = (__bf16)y[i];
    }
}
// of 16 rows (one a lane of the first group) those that are asked for, every `of`th from `first` on
template <int HD, int BITS, int NP>
__device__ __forceinline__ void slow_rows(const Job& job, int at, int lim, bool again, int first, int of) {
    const uint32_t todo = (uint32_t)__ballot(again) & 0xffffu;
    if (!todo) return;
    // (read anew from the kernel's arguments, its only ones, so that none of them stay in registers for this path)
    uintptr_t args = (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(args));
    const AttnArgs& p = *(const AttnArgs*)args;
#pragma unroll 1
    for (int i = first; i < 16; i += of)
        if (todo >> i & 1) slow_row<HD, BITS, NP>(p, job, __builtin_amdgcn_readlane(at, i), __builtin_amdgcn_readlane(lim, i));
}

template <int HD, int BITS, int NP>
__device__ __forceinline__ void few(const AttnArgs& p, Job& job, char* lds) {
    constexpr int ND = HD / 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    Rows<HD, NP, 1> w;
    set_rows(p, job, job.row0, w);
    job.t1 = min(job.t1, (w.hi + 31) / 32);
    int tile = job.t0 + wave;
    Seen<BITS> scales;
    RawTile<HD, BITS> raw;
    // (past the last tile its own are loaded again, for nothing)
    const auto at = [&](int x) {
        const int y = min(x, job.t1 - 1);
        return tile_ptr<HD, BITS>(p, job.head, page_id(job, p, y), y);
    };
    if (tile < job.t1) {
        TilePtr cur = at(tile), next = at(tile + AW);
        raw.load_keys(p, cur);
        raw.load_values(p, cur);
        load_rows<BITS>(p, w);
        for (; tile < job.t1; tile += AW) {
            const TilePtr after = at(tile + 2 * AW);
            few_tile<HD, BITS, NP>(p, w, scales, raw, tile, cur.ok ? (int)min(job.len - (long long)tile * 32, 32ll) : 0, next);
            cur = next;
            next = after;
        }
    } else {
        clear_rows<BITS>(w);
    }
    // join the waves: first everyone's maximum and unit, then sums in these
    f4(*buf)[ND][64] = (f4(*)[ND][64])lds;                       // [2]
    float(*sm)[16] = (float(*)[16])(lds + 2 * sizeof(*buf));     // [AW]
    float(*sl)[16] = sm + AW;
    float(*sx)[16] = sl + AW;
    float(*sf)[16] = sx + AW;
    int* su = (int*)(sf + AW);                                   // [AW]
    int* sfar = su + AW;
    const float lw = row_total<BITS>(w.l[0]);
    const float top = w.m[0] == kNegInf ? kNegInf : w.m[0] * w.rk[0];   // (rk is not set where there was no tile)
    if (g == 0) {
        sm[wave][col] = top;
        sl[wave][col] = lw;
    }
    const bool wave_far = __any(scales.far(w.ek, w.eu));
    if (lane == 0) {
        su[wave] = w.eu;
        sfar[wave] = wave_far;
    }
    __syncthreads();
    float mall = kNegInf, lall = 0.0f;
#pragma unroll
    for (int v = 0; v < AW; ++v) mall = fmaxf(mall, sm[v][col]);
    const float base = mall == kNegInf ? 0.0f : mall;
#pragma unroll
    for (int v = 0; v < AW; ++v) lall += sl[v][col] * exp2_(sm[v][col] - base);
    int unit = kNoUnit;
    bool again = false;
#pragma unroll
    for (int v = 0; v < AW; ++v) {
        unit = max(unit, su[v]);
        again |= sfar[v] != 0;
    }
    const float f = ldexpf(exp2_(top - base), w.eu - unit);
    if constexpr (BITS == 8) {
        const float x = max16_32(w.x[0]) * f;
        if (g == 0) {
            sx[wave][col] = x;
            sf[wave][col] = f;
        }
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) w.o[0][d] *= f;
    if (wave >= 2) {
#pragma unroll
        for (int d = 0; d < ND; ++d) buf[wave - 2][d][lane] = w.o[0][d];
    }
    __syncthreads();
    if constexpr (BITS == 8) {   // of all waves: the largest weight against the largest step
        float x = 0.0f, step = 0.0f;
#pragma unroll
        for (int v = 0; v < AW; ++v) {
            x = fmaxf(x, sx[v][col]);
            step = fmaxf(step, sf[v][col]);
        }
        again |= x < kFarWeight * step && unit != kNoUnit && lall > 0.0f;
    }
    if (wave < 2) {
#pragma unroll
        for (int d = 0; d < ND; ++d) w.o[0][d] += buf[wave][d][lane];
    }
    __syncthreads();
    if (wave == 1) {
#pragma unroll
        for (int d = 0; d < ND; ++d) buf[0][d][lane] = w.o[0][d];
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int d = 0; d < ND; ++d) w.o[0][d] += buf[0][d][lane];
        put_rows(p, job, job.row0, w, unit, &mall, &lall, &again);
    }
    slow_rows<HD, BITS, NP>(job, w.at[0], w.lim[0], again && job.row0 + col < job.nrows, wave, AW);
}
template <int HD> constexpr int kFewLds = 2 * (HD / 16) * 1024 + 4 * AW * 64 + 2 * AW * 4;

// ---- many rows: the block's waves split its rows ------------------------------
// Tiles between two barriers: two, or one where two would not leave enough
// registers (32 sequences after a prefix of 8192: 26.8 us, with two 30.1).
template <int HD, int BITS> constexpr int kManyTiles = HD == 128 && BITS == 8 ? 1 : 2;

// A tile is turned into operands once, a part by each wave, and lies in LDS
// for all of them; the next tile is written beside it meanwhile, and the codes
// of the one after are on their way.
template <int HD, int BITS> struct Parts {
    static constexpr int NC = HD / 32, NU = (2 * NC + AW - 1) / AW;   // a wave's blocks (NC of keys, then NC of values)
    typedef uint32_t vec __attribute__((ext_vector_type(BITS == 8 ? 4 : 2)));
    // block of round u; is it one of keys (known at compile time where the waves divide them)
    __device__ __forceinline__ static int block(int u, int wave) { return wave + u * AW; }
    __device__ __forceinline__ static bool keys(int u, int b) { return NC % AW == 0 ? u < NC / AW : b < NC; }
    __device__ __forceinline__ static bool none(int b) { return 2 * NC % AW != 0 && b >= 2 * NC; }
    vec code[NU];
    u4 sc[NU];                    // 4 bits: a value block's scales; a key block's pair in the first word
    u4 ks, vs;                    // 8 bits
    u2 all_k, all_v;              // 4 bits: the tile's scales, 4 a lane, for its units
    bool ok;
    __device__ __forceinline__ void load(const AttnArgs& p, int head, int id, int tile, int wave) {
        constexpr int BB = BITS == 8 ? 1024 : 512;
        const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
        const TilePtr t = tile_ptr<HD, BITS>(p, head, id, tile);
        ok = t.ok;
        const uint8_t* vc = t.codes + kv_codes_bytes(p.c.page_size, HD, BITS);
        const uint16_t* vsp = t.scales + (long long)p.c.page_size * kv_groups(HD, BITS);
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int b = block(u, wave);
            if (none(b)) break;
            const bool is_key = keys(u, b);
            const int c = is_key ? b : b - NC;
            code[u] = *(const vec*)((is_key ? t.codes : vc) + c * BB + lane * sizeof(vec));
            if constexpr (BITS == 4) {
                if (is_key) {
                    const uint16_t* s = t.scales + c * p.c.page_size;
                    sc[u][0] = *(const uint32_t*)(s + 2 * col);
                } else {
                    sc[u] = *(const u4*)(vsp + c * p.c.page_size + 8 * g);
                }
            }
        }
        if constexpr (BITS == 8) {
            ks = *(const u4*)(t.scales + 8 * g);
            vs = *(const u4*)(vsp + 8 * g);
        } else {
            all_k = all_scales(t.scales, p.c.page_size, NC);
            all_v = all_scales(vsp, p.c.page_size, NC);
        }
    }
};

template <int HD, int BITS, int NP, int NR>
__device__ __forceinline__ void many(const AttnArgs& p, Job& job, char* lds) {
    constexpr int NC = HD / 32, NU = Parts<HD, BITS>::NU, KT = kManyTiles<HD, BITS>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15;
    h8(*frag)[KT][4 * NC][64] = (h8(*)[KT][4 * NC][64])lds;   // [2]: a tile's keys (c, i), then its values (c, i)
    Rows<HD, NP, NR> w;
    const int row0 = job.row0 + wave * 16 * NR;
    // the block's tiles: the last of its rows sees most
    {
        const int last = min(job.row0 + AW * 16 * NR, job.nrows) - 1;
        long long hi = job.len;
        if (!job.pre) {
            const long long seen = (long long)scalar_load(p.a.lens, job.b) - p.a.seq + last / p.G + 1;
            hi = seen < hi ? seen : hi;
        }
        job.t1 = min(job.t1, hi > 0 ? (int)((hi + 31) / 32) : 0);
    }
    set_rows(p, job, row0, w);   // (a wave past the rows repeats the last one)

    Parts<HD, BITS> raw[KT] = {};
    int id[KT], held[KT], held_next[KT], ek = kNoUnit, ek_next = kNoUnit, en = kNoUnit, en_next = kNoUnit;
    u4 ks_next[KT], vs_next[KT];   // 8 bits
    Seen<BITS> scales;
    auto ids = [&](int tile) {
#pragma unroll
        for (int z = 0; z < KT; ++z) id[z] = tile + z < job.t1 ? page_id(job, p, tile + z) : -1;
    };
    auto load = [&](int tile) {
#pragma unroll
        for (int z = 0; z < KT; ++z) raw[z].load(p, job.head, id[z], tile + z, wave);
    };
    // raw tiles -> operands in frag[at]; tokens past the source's end have scale 0
    auto convert = [&](int tile, int at) {
        float fk = 1.0f, fv = 1.0f;
#pragma unroll
        for (int z = 0; z < KT; ++z) {
            held_next[z] = raw[z].ok ? (int)min(job.len - (long long)(tile + z) * 32, 32ll) : 0;
            ks_next[z] = raw[z].ks;
            vs_next[z] = raw[z].vs;
        }
        if constexpr (BITS == 4) {
            uint32_t tk = 0, tv = 0;
            u2 k[KT], v[KT];
#pragma unroll
            for (int z = 0; z < KT; ++z) {
                k[z] = of_tokens(raw[z].all_k, held_next[z], true);
                v[z] = of_tokens(raw[z].all_v, held_next[z], false);
                tk = pair_max(tk, pair_max(k[z][0], k[z][1]));
                tv = pair_max(tv, pair_max(v[z][0], v[z][1]));
            }
            ek_next = unit_of(tk, ek_next);
            en_next = unit_of(tv, en_next);
            if ((tile / KT) % AW == wave) {   // (one wave of the block is enough)
                stay_a_branch();
#pragma unroll
                for (int z = 0; z < KT; ++z) scales.add(k[z], v[z]);
            }
            fk = ldexpf(1.0f, -ek_next);
            fv = ldexpf(1.0f, -en_next);
        }
#pragma unroll
        for (int z = 0; z < KT; ++z)
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                const int b = Parts<HD, BITS>::block(u, wave);
                if (Parts<HD, BITS>::none(b)) break;
                h8* to = &frag[at][z][2 * b][lane];
                if constexpr (BITS == 8) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) to[64 * i] = codes8(raw[z].code[u][2 * i], raw[z].code[u][2 * i + 1]);
                } else if (Parts<HD, BITS>::keys(u, b)) {
                    const uint32_t s = held_pair(raw[z].sc[u][0], held_next[z]);
                    to[0] = key4(raw[z].code[u][0], bf16_lo(s), fk);
                    to[64] = key4(raw[z].code[u][1], bf16_hi(s), fk);
                } else {
                    Scale4 s[4];
                    value_scales(held_scales(raw[z].sc[u], held_next[z]), fv, s);
#pragma unroll
                    for (int i = 0; i < 2; ++i) to[64 * i] = codes4(raw[z].code[u][i], s[0], s[1], s[2], s[3]);
                }
            }
    };
    if (job.t0 < job.t1) {
        ids(job.t0);
        load(job.t0);
        ids(job.t0 + KT);
    }
    load_rows<BITS>(p, w);
    if (job.t0 < job.t1) {
        convert(job.t0, 0);
        load(job.t0 + KT);
        ids(job.t0 + 2 * KT);
    }
    __syncthreads();
    int at = 0;
    for (int tile = job.t0; tile < job.t1; tile += KT, at ^= 1) {
        u4 ks_raw[KT], vs_raw[KT];
#pragma unroll
        for (int z = 0; z < KT; ++z) {
            held[z] = held_next[z];
            ks_raw[z] = ks_next[z];
            vs_raw[z] = vs_next[z];
        }
        ek = ek_next;
        en = en_next;
        bool some = false;
#pragma unroll
        for (int z = 0; z < KT; ++z) some |= held[z] < 32;
        if constexpr (BITS == 8) {
            uint32_t vtop = 0;
#pragma unroll
            for (int z = 0; z < KT; ++z) {
                vs_raw[z] = held_scales(vs_raw[z], held[z]);
                vtop = umax(vtop, top8(vs_raw[z]));
            }
            if ((tile / KT) % AW == wave) {
                stay_a_branch();
#pragma unroll
                for (int z = 0; z < KT; ++z) scales.add(ks_raw[z]);
            }
            ek = 0;
            en = max(w.eu, ceil_exp(__builtin_amdgcn_readfirstlane(umax16_32(vtop)), kNoUnit));
        }
        const h8(*f)[4 * NC][64] = frag[at];
        tile_step<HD, BITS, NP, NR, KT>(
            w, tile * 32, held, some, ks_raw, vs_raw, ek, en,
            [&](int z, int j) { return f[z][j][lane]; }, [&](int z, int j) { return f[z][2 * NC + j][lane]; },
            [&] {   // past the last tile for nothing: without a branch
                convert(tile + KT, at ^ 1);
                __builtin_amdgcn_sched_barrier(0);
                load(tile + 2 * KT);
                ids(tile + 3 * KT);
                __builtin_amdgcn_sched_barrier(0);
            },
            [] {});
        __syncthreads();
    }
    int* sfar = (int*)lds;   // (past the loop's last barrier)
    const bool wave_far = __any(scales.far(w.ek, w.eu));
    if (lane == 0) sfar[wave] = wave_far;
    __syncthreads();
    bool any_far = false;
#pragma unroll
    for (int v = 0; v < AW; ++v) any_far |= sfar[v] != 0;
    if (row0 >= job.nrows) return;
    float m[NR], l[NR];
    bool again[NR];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        l[t] = row_total<BITS>(w.l[t]);
        m[t] = w.m[t] == kNegInf ? kNegInf : w.m[t] * w.rk[t];
        again[t] = any_far || (BITS == 8 && max16_32(w.x[t]) < kFarWeight && w.eu != kNoUnit && l[t] > 0.0f);
    }
    put_rows(p, job, row0, w, w.eu, m, l, again);
#pragma unroll
    for (int t = 0; t < NR; ++t)
        slow_rows<HD, BITS, NP>(job, w.at[t], w.lim[t], again[t] && row0 + 16 * t + col < job.nrows, 0, 1);
}
template <int HD, int BITS> constexpr int kManyLds = 2 * kManyTiles<HD, BITS> * 4 * (HD / 32) * 1024;

// row tiles of a wave with many rows: two where they fit beside the rest
template <int HD, int NP> constexpr int kManyRows = HD <= 128 && NP == 1 ? 2 : 1;

// One block: rows of one key/value head against one split of the prefix or of
// a sequence's tokens. PM, OM: the prefix's and the sequences' blocks have
// many rows.
template <int HD, int BITS, int NP, bool PM, bool OM>
__global__ __launch_bounds__(AW * 64, HD <= 128 ? (!PM && !OM && NP == 1 ? 3 : 2) : 1) void kv_attn_kernel(AttnArgs p) {
    constexpr int few_lds = PM && OM ? 0 : kFewLds<HD>, many_lds = PM || OM ? kManyLds<HD, BITS> : 0;
    __shared__ __attribute__((aligned(16))) char lds[few_lds > many_lds ? few_lds : many_lds];
    constexpr int NR = kManyRows<HD, NP>;
    const KvAttention& a = p.a;
    const int H = p.c.heads;
    const int npre = p.pre_groups * H * p.pre_slots;
    Job job;
    job.pre = (int)blockIdx.x < npre;
    int x = job.pre ? blockIdx.x : blockIdx.x - npre;
    const int ns = job.pre ? p.pre_slots : p.slots - p.pre_slots;
    // Blocks go to the 8 XCDs in turn. The prefix's: splits first, then heads, so
    // that row groups which read the same keys are a multiple of 8 apart where
    // heads times splits is one. The sequences': heads first and splits last, as
    // late splits of short sequences are empty and would leave an XCD idle.
    job.b = 0;
    int group;
    if (job.pre) {
        job.split = x % ns;
        x /= ns;
        job.head = x % H;
        group = x / H;
    } else {
        job.head = x % H;
        x /= H;
        group = x % p.own_groups;
        x /= p.own_groups;
        job.b = x % a.batch;
        job.split = x / a.batch;
    }
    job.slot = job.pre ? job.split : p.pre_slots + job.split;
    job.nrows = (job.pre ? a.batch : 1) * a.seq * p.G;
    job.table = job.pre ? a.prefix_table : a.table + (long long)job.b * a.max_pages;
    job.len = a.prefix_len;
    if (!job.pre) {
        const long long cap = (long long)a.max_pages * p.c.page_size, len = scalar_load(a.lens, job.b);
        job.len = len < cap ? len : cap;
    }
    const int chunk = job.pre ? p.pre_chunk : p.own_chunk;
    job.t0 = job.split * chunk;
    job.t1 = job.t0 + chunk;   // cut to what the rows see further on
    const bool is_many = job.pre ? PM : OM;
    job.row0 = group * (is_many ? AW * 16 * NR : 16);
    if (is_many) {
        if constexpr (PM || OM) many<HD, BITS, NP, NR>(p, job, lds);
    } else {
        if constexpr (!(PM && OM)) few<HD, BITS, NP>(p, job, lds);
    }
}

// One wave a row: the mean of its partial results, by their totals, in a fixed
// order, several slots side by side where a row is shorter than the wave.
template <int HD>
__global__ __launch_bounds__(256) void kv_join_kernel(AttnArgs p) {
    constexpr int L = HD / 4, W = 64 / L;   // lanes of a row, slots at a time
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= p.rows) return;
    const float2* ml = p.part_ml + (long long)row * p.slots;
    float mx = kNegInf;
    for (int i = lane; i < p.slots; i += 64) mx = fmaxf(mx, ml[i].x);
    mx = max16_32(max_16(mx));
    const float base = mx == kNegInf ? 0.0f : mx;
    // what a slot counts for; of an empty one (whose mean is not written) nothing
    const auto weight = [&](float2 v) { return v.x == kNegInf && v.y == 0.0f ? 0.0f : exp2_(v.x - base) * v.y; };
    float total = 0.0f;
    for (int i = lane; i < p.slots; i += 64) total += weight(ml[i]);
#pragma unroll
    for (int o = 1; o < 64; o *= 2) total += __shfl_xor(total, o);
    const bool none = mx == kNegInf && total == 0.0f;
    const float inv = none ? 0.0f : 1.0f / total;
    const int part = lane / L, at = (lane - part * L) * 4;
    f4 o = {0, 0, 0, 0};
    if (part < W) {
        const float* src = p.part_o + (long long)row * p.slots * HD + at;
#pragma unroll 4
        for (int i = part; i < p.slots; i += W) {
            const float2 v = ml[i];
            const f4 x = *(const f4*)(src + (long long)i * HD);
            const bool some = !(v.x == kNegInf && v.y == 0.0f);
            const float w = weight(v) * inv;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] += some ? x[j] * w : 0.0f;
        }
    }
    const f4 o1 = o;
#pragma unroll
    for (int s = 1; s < W; ++s) {   // into the first lanes, in order
        const int from = (lane % L) + s * L;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] += __shfl(o1[j], from);
    }
    if (part != 0) return;
    store_y4(p.a, (long long)row * HD + at, none ? f4{0, 0, 0, 0} : o);
}

// How a call is cut up; of shapes alone, so that the workspace is known before
struct Plan {
    bool pre_many, own_many;
    int pre_groups, own_groups, pre_slots, own_slots, pre_chunk, own_chunk;
};
int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }
Plan plan(const KvCache& c, const KvAttention& a) {
    Plan p;
    const int G = a.q_heads / c.heads;
    const long long own_rows = (long long)a.seq * G, pre_rows = own_rows * a.batch;
    const int np = a.type == FT_F32 ? 2 : 1, many = AW * 16 * (c.hd <= 128 && np == 1 ? 2 : 1);
    p.own_many = own_rows > 16;
    p.pre_many = a.prefix_len && pre_rows > 16;
    p.own_groups = ceil_div(own_rows, p.own_many ? many : 16);
    p.pre_groups = a.prefix_len ? ceil_div(pre_rows, p.pre_many ? many : 16) : 0;
    const long long pre_items = (long long)p.pre_groups * c.heads, own_items = (long long)p.own_groups * c.heads * a.batch;
    const long long pre_tiles = (a.prefix_len + 31) / 32, own_tiles = (long long)a.max_pages * c.page_size / 32;
    // Blocks with few rows: 32 tiles or more, and short ones whole. (Splits of 8
    // tiles, and their join: 48 sequences of 8192 120 us instead of 86, 16 of 1000
    // 13.6 instead of 12.8, 4 of 8192 21 instead of 16.5, one of 700 13.6 instead of
    // 10.4.)
    const auto few = [](long long items, long long tiles) {
        return tiles <= 32 ? std::max(tiles, 1ll) : std::max(items * tiles / 1024, 32ll);
    };
    // Those with many: no more than run at once, of 8 tiles or more. (128 sequences
    // after a prefix of 32768: 512 blocks 134 us, 384 150, 768 141.) Of 4 where that
    // is a block a CU, and two with the rest: such a block waits for most of a tile's
    // 0.8 us. (32 sequences after a prefix of 1024: 20.0 us, of 8 tiles 23.5; 4096:
    // 22.8 and 24.9. Beyond: 8192 35.6 and 27.2, 128 sequences after 512 31.8 and 30.2.)
    const long long at_once = c.hd <= 128 ? 512 : 256;
    const auto many_blocks = [&](long long chunk) {
        return (p.pre_many ? pre_items * ceil_div(pre_tiles, chunk) : 0) + (p.own_many ? own_items * ceil_div(own_tiles, chunk) : 0);
    };
    const long long rest = (p.pre_many ? 0 : pre_items * ceil_div(pre_tiles, few(pre_items, pre_tiles))) +
                           (p.own_many ? 0 : own_items * ceil_div(own_tiles, few(own_items, own_tiles)));
    long long chunk = many_blocks(4) <= 256 && many_blocks(4) + rest <= 512 ? 4 : 8;
    while (many_blocks(chunk) > at_once && chunk < std::max(pre_tiles, own_tiles)) chunk += 2 + chunk / 16 * 2;
    const long long pre_c = p.pre_many ? chunk : few(pre_items, pre_tiles), own_c = p.own_many ? chunk : few(own_items, own_tiles);
    p.pre_slots = p.pre_groups ? ceil_div(pre_tiles, pre_c) : 0;
    p.own_slots = own_tiles ? ceil_div(own_tiles, own_c) : 1;
    p.pre_chunk = p.pre_slots ? ceil_div(pre_tiles, p.pre_slots) : 0;
    p.own_chunk = ceil_div(own_tiles, p.own_slots);
    return p;
}

template <int HD, int BITS, int NP>
hipError_t go(const AttnArgs& p, const Plan& pl, unsigned blocks, hipStream_t s) {
    if (pl.own_many) kv_attn_kernel<HD, BITS, NP, true, true><<<blocks, AW * 64, 0, s>>>(p);
    else if (pl.pre_many) kv_attn_kernel<HD, BITS, NP, true, false><<<blocks, AW * 64, 0, s>>>(p);
    else kv_attn_kernel<HD, BITS, NP, false, false><<<blocks, AW * 64, 0, s>>>(p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.slots == 1) return e;
    kv_join_kernel<HD><<<(unsigned)ceil_div(p.rows, 4), 256, 0, s>>>(p);
    return hipGetLastError();
}
template <int HD>
hipError_t by_type(const AttnArgs& p, const Plan& pl, unsigned blocks, hipStream_t s) {
    const bool f32 = p.a.type == FT_F32;
    if (p.c.bits == 8) return f32 ? go<HD, 8, 2>(p, pl, blocks, s) : go<HD, 8, 1>(p, pl, blocks, s);
    return f32 ? go<HD, 4, 2>(p, pl, blocks, s) : go<HD, 4, 1>(p, pl, blocks, s);
}

}  // namespace

size_t kv_attention_workspace(const KvCache& c, const KvAttention& a) {
    const Plan pl = plan(c, a);
    const long long slots = pl.pre_slots + pl.own_slots;
    if (slots == 1) return 0;
    const long long rows = (long long)a.batch * a.seq * a.q_heads;
    return (size_t)(rows * slots * (c.hd * 4LL + 8));
}

hipError_t launch_kv_attention(const KvCache& c, const KvAttention& a, void* workspace, hipStream_t s) {
    if (a.batch == 0 || a.seq == 0) return hipSuccess;
    const Plan pl = plan(c, a);
    AttnArgs p;
    p.c = c;
    p.a = a;
    if (c.num_pages == 0) {   // no keys, and no page 0 to read in place of one that does not exist
        p.a.prefix_len = 0;
        p.a.max_pages = 0;
    }
    p.G = a.q_heads / c.heads;
    p.rows = a.batch * a.seq * a.q_heads;
    p.pre_slots = pl.pre_slots;
    p.slots = pl.pre_slots + pl.own_slots;
    p.pre_chunk = pl.pre_chunk;
    p.own_chunk = pl.own_chunk;
    p.pre_groups = pl.pre_groups;
    p.own_groups = pl.own_groups;
    p.page_shift = __builtin_ctz((unsigned)c.page_size) - 5;
    p.part_o = (float*)workspace;
    p.part_ml = (float2*)(p.part_o + (size_t)p.rows * p.slots * c.hd);
    const unsigned blocks = (unsigned)(p.pre_groups * c.heads * p.pre_slots + a.batch * p.own_groups * c.heads * pl.own_slots);
    switch (c.hd) {
    case 64: return by_type<64>(p, pl, blocks, s);
    case 96: return by_type<96>(p, pl, blocks, s);
    case 128: return by_type<128>(p, pl, blocks, s);
    case 256: return by_type<256>(p, pl, blocks, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace nnrh
