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
// pieces, 22 bits and more. Weights p = exp(s - max) enter as p * 2^15, and
// with them, at 8 bits, the values' scales divided by their largest power of
// two so far: 11 significant bits (two pieces, 22, for fp32 tensors) over 39
// binary orders. At 4 bits scale (8 bits) times code (3 bits) is exact in
// fp16 and is formed in the operand. Sums, maxima and the running total are
// fp32.
//
// Keys are split over blocks; each leaves (max, total, O) of its rows, which
// a second kernel joins in a fixed order. One block that sees everything
// writes the result itself.
#include "nnrh_decode.h"

namespace nnrh {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int AW = 4;              // waves of a block
constexpr float kNegInf = -__builtin_inff();

struct AttnArgs {
    KvCache c;
    KvAttention a;
    int G;                         // query heads a key/value head
    int rows;                      // batch * seq * q_heads
    int slots, pre_slots;          // partial results a row: prefix ones first
    int pre_chunk, own_chunk;      // tiles of a split
    int pre_groups, own_groups;    // row groups (of 16 NR rows)
    int page_shift;                // log2(page_size / 32)
    float* part_o;                 // [rows][slots][hd]
    float2* part_ml;               // [rows][slots]
};

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
// exponent e of the least 2^e >= x > 0 (x a normal float)
__device__ __forceinline__ int ceil_exp(float x) {
    return (int)((__builtin_bit_cast(uint32_t, x) + 0x7fffffu) >> 23) - 127;
}

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
// eight 4-bit codes (code + 8) times scales s[0..3], a pair each
__device__ __forceinline__ h8 codes4(uint32_t w, const h2* s) {
    const h2 off = {(_Float16)1032.0f, (_Float16)1032.0f};
    u4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const h2 v = __builtin_bit_cast(h2, ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u) - off;
        r[i] = __builtin_bit_cast(uint32_t, v * s[i]);
    }
    return __builtin_bit_cast(h8, r);
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
    float rf[NR];       // a row's score is rf times its raw score (codes times scaled query), rf > 0
    float m[NR];        // largest raw score
    float l[NR];        // this lane's part of the total of 2^15 p
    f4 o[NR][ND];       // sums of 2^15 p v in units of 2^eu
    int eu;
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
            const long long last = (long long)a.lens[job.b] - a.seq + tok + 1;
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

template <int HD, int NP, int NR>
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
        // (0 would make 0 * -inf of a masked score)
        w.rf[t] = fmaxf(ldexpf(fabsf(a.scale) * 1.44269504088896341f, -e), 1e-37f);
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float s = ldexpf(neg ? -v[k][j] : v[k][j], e);
                const _Float16 h = (_Float16)s;
                w.q[0][t][k][j] = h;
                if constexpr (NP == 2) w.q[1][t][k][j] = (_Float16)(s - (float)h);
            }
        w.m[t] = kNegInf;
        w.l[t] = 0.0f;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) w.o[t][d] = f4{0, 0, 0, 0};
    }
    w.eu = -126;
}

// A tile against a wave's rows. key(c, i): elements 32 c .. of keys 16 i .. as
// an operand, value(c, i): elements 32 c + 16 i .. of the tile's keys. ks, vs:
// scales of this lane's 8 keys (8 bits; at 4 bits they are in the operands,
// keys over 2^ek, values over 2^en). en: the values' unit from here on.
template <int HD, int BITS, int NP, int NR, class Key, class Value>
__device__ __forceinline__ void tile_step(Rows<HD, NP, NR>& w, int tile, const float* ks, const float* vs, int ek, int en,
                                          Key key, Value value) {
    constexpr int NC = HD / 32, ND = HD / 16;
    const int g = (threadIdx.x & 63) >> 4;
    f4 acc[NR][2];
#pragma unroll
    for (int t = 0; t < NR; ++t) acc[t][0] = acc[t][1] = f4{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const h8 kf = key(c, i);
#pragma unroll
            for (int t = 0; t < NR; ++t)
#pragma unroll
                for (int q = 0; q < NP; ++q)
                    acc[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, w.q[q][t][c], acc[t][i], 0, 0, 0);
        }
    // raw scores of 2 x 4 keys a row: key 16 i + 4 g + r in element 4 i + r
    float s[NR][8];
    const float kunit = BITS == 8 ? 1.0f : ldexpf(1.0f, ek);
#pragma unroll
    for (int t = 0; t < NR; ++t)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[t][j] = acc[t][j >> 2][j & 3] * (BITS == 8 ? ks[j] : kunit);
    if (tile * 32 + 32 > w.lo) {
#pragma unroll
        for (int t = 0; t < NR; ++t)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (tile * 32 + 16 * (j >> 2) + 4 * g + (j & 3) >= w.lim[t]) s[t][j] = kNegInf;
    }
    // running maximum; weights 2^15 p
    bool moved = en != w.eu;
    float al[NR];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        float mx = w.m[t];
#pragma unroll
        for (int j = 0; j < 8; ++j) mx = fmaxf(mx, s[t][j]);
        mx = max16_32(mx);
        const float base = mx == kNegInf ? 0.0f : mx * w.rf[t];
        al[t] = exp2_(__builtin_fmaf(w.m[t], w.rf[t], -base));
        moved |= mx != w.m[t];
        w.m[t] = mx;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            s[t][j] = exp2_(__builtin_fmaf(s[t][j], w.rf[t], 15.0f - base));
            sum += s[t][j];
        }
        w.l[t] = __builtin_fmaf(w.l[t], al[t], sum);
    }
    if (__any(moved)) {
#pragma unroll
        for (int t = 0; t < NR; ++t) {
            const float f = ldexpf(al[t], w.eu - en);
#pragma unroll
            for (int d = 0; d < ND; ++d) w.o[t][d] *= f;
        }
    }
    w.eu = en;
    h8 pf[NP][NR];
    float vu[8];
    if constexpr (BITS == 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) vu[j] = ldexpf(vs[j], -en);
    }
#pragma unroll
    for (int t = 0; t < NR; ++t)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = BITS == 8 ? s[t][j] * vu[j] : s[t][j];
            const _Float16 h = (_Float16)x;
            pf[0][t][j] = h;
            if constexpr (NP == 2) pf[1][t][j] = (_Float16)(x - (float)h);
        }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const h8 v = value(c, i);
#pragma unroll
            for (int t = 0; t < NR; ++t)
#pragma unroll
                for (int q = 0; q < NP; ++q)
                    w.o[t][2 * c + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pf[q][t], w.o[t][2 * c + i], 0, 0, 0);
        }
}

// ---- a tile in memory ---------------------------------------------------------
struct TilePtr {
    const uint8_t* codes;        // keys' blocks; values' vcodes further
    const uint16_t* scales;      // keys'; values' vscales further
    bool ok;                     // the page exists
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
// 8 scales of a lane's keys; those past `held` are 0
__device__ __forceinline__ void scales8(u4 w, int held, float* s) {
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = j & 1 ? bf16_hi(w[j >> 1]) : bf16_lo(w[j >> 1]);
    if (held < 32) {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (16 * (j >> 2) + 4 * g + (j & 3) >= held) s[j] = 0.0f;
    }
}
__device__ __forceinline__ h2 scale_pair(float a, float b) { return h2{(_Float16)a, (_Float16)b}; }
__device__ __forceinline__ int unit_of(float top, int none) { return top > 0.0f ? ceil_exp(top) : none; }

__device__ __forceinline__ int page_id(const Job& job, const AttnArgs& p, int tile) {
    return __builtin_amdgcn_readfirstlane(job.table[tile >> p.page_shift]);
}

// ---- few rows: the block's waves split its keys -------------------------------
// Each wave loads a tile's codes into registers one tile ahead.
template <int HD, int BITS> struct RawTile {
    static constexpr int NC = HD / 32;
    typedef uint32_t vec __attribute__((ext_vector_type(BITS == 8 ? 4 : 2)));
    vec k[NC], v[NC];
    u4 vs[BITS == 8 ? 1 : NC];
    u4 ks;                        // 8 bits
    uint16_t ks4[NC][2];          // 4 bits
    bool ok;
    __device__ __forceinline__ void load(const AttnArgs& p, const Job& job, int tile) {
        constexpr int BB = BITS == 8 ? 1024 : 512;
        const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
        const TilePtr t = tile_ptr<HD, BITS>(p, job.head, page_id(job, p, tile), tile);
        ok = t.ok;
        if (!ok) return;
        const uint8_t* vc = t.codes + kv_codes_bytes(p.c.page_size, HD, BITS);
        const uint16_t* vsp = t.scales + (long long)p.c.page_size * kv_groups(HD, BITS);
#pragma unroll
        for (int c = 0; c < NC; ++c) k[c] = *(const vec*)(t.codes + c * BB + lane * sizeof(vec));
        if constexpr (BITS == 8) ks = *(const u4*)(t.scales + 8 * g);
        else
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < 2; ++i) ks4[c][i] = t.scales[c * p.c.page_size + kv_slot(col + 16 * i)];
#pragma unroll
        for (int c = 0; c < (BITS == 8 ? 1 : NC); ++c) vs[c] = *(const u4*)(vsp + c * p.c.page_size + 8 * g);
#pragma unroll
        for (int c = 0; c < NC; ++c) v[c] = *(const vec*)(vc + c * BB + lane * sizeof(vec));
    }
};

template <int HD, int BITS, int NP>
__device__ __forceinline__ void few_tile(Rows<HD, NP, 1>& w, const RawTile<HD, BITS>& r, int tile, int held) {
    constexpr int NC = HD / 32;
    const int col = threadIdx.x & 15;
    float vtop = 0.0f;
    float vs[BITS == 8 ? 1 : NC][8];
#pragma unroll
    for (int c = 0; c < (BITS == 8 ? 1 : NC); ++c) {
        scales8(r.vs[c], held, vs[c]);
#pragma unroll
        for (int j = 0; j < 8; ++j) vtop = fmaxf(vtop, vs[c][j]);
    }
    vtop = max16_32(vtop);
    const int en = max(w.eu, unit_of(vtop, w.eu));
    if constexpr (BITS == 8) {
        float ks[8];
        scales8(r.ks, held, ks);
        tile_step<HD, 8, NP, 1>(
            w, tile, ks, vs[0], 0, en, [&](int c, int i) { return codes8(r.k[c][2 * i], r.k[c][2 * i + 1]); },
            [&](int c, int i) { return codes8(r.v[c][2 * i], r.v[c][2 * i + 1]); });
    } else {
        float ks[NC][2], top = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                ks[c][i] = col + 16 * i < held ? bf16_lo(r.ks4[c][i]) : 0.0f;
                top = fmaxf(top, ks[c][i]);
            }
        top = max_16(top);
        const int ek = unit_of(top, 0);
        const float fk = ldexpf(1.0f, -ek), fv = ldexpf(1.0f, -en);   // (-126 only where all scales are 0)
        tile_step<HD, 4, NP, 1>(
            w, tile, nullptr, nullptr, ek, en,
            [&](int c, int i) {
                const h2 f = scale_pair(ks[c][i] * fk, ks[c][i] * fk);
                const h2 f4_[4] = {f, f, f, f};
                return codes4(r.k[c][i], f4_);
            },
            [&](int c, int i) {
                h2 f[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) f[j] = scale_pair(vs[c][2 * j] * fv, vs[c][2 * j + 1] * fv);
                return codes4(r.v[c][i], f);
            });
    }
}

// the results of a wave's rows: into the call's result, or among the parts
template <int HD, int NP, int NR>
__device__ __forceinline__ void put_rows(const AttnArgs& p, const Job& job, int row0, const Rows<HD, NP, NR>& w,
                                         const float* m, const float* l) {
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        if (row0 + 16 * t + col >= job.nrows) continue;
        const bool none = m[t] == kNegInf && l[t] == 0.0f;
        if (p.slots > 1) {
            const long long at = (long long)w.at[t] * p.slots + job.slot;
            if (g == 0) p.part_ml[at] = float2{m[t], l[t]};
            if (none) continue;
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) *(f4*)(p.part_o + at * HD + 16 * d + 4 * g) = w.o[t][d];
        } else {
            const float inv = none ? 0.0f : 1.0f / l[t];
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) store_y4(p.a, (long long)w.at[t] * HD + 16 * d + 4 * g, w.o[t][d] * inv);
        }
    }
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
    RawTile<HD, BITS> cur, nxt;
    if (tile < job.t1) cur.load(p, job, tile);
    load_rows(p, w);
    for (; tile < job.t1; tile += AW) {
        if (tile + AW < job.t1) nxt.load(p, job, tile + AW);
        if (cur.ok) few_tile<HD, BITS, NP>(w, cur, tile, (int)min(job.len - (long long)tile * 32, 32ll));
        cur = nxt;
    }
    // join the waves: first everyone's maximum, then sums in the units of it
    f4(*buf)[ND][64] = (f4(*)[ND][64])lds;                       // [2]
    float(*sm)[16] = (float(*)[16])(lds + 2 * sizeof(*buf));     // [AW]
    float(*sl)[16] = sm + AW;
    w.l[0] += __shfl_xor(w.l[0], 16);
    w.l[0] += __shfl_xor(w.l[0], 32);
    const float top = w.m[0] == kNegInf ? kNegInf : w.m[0] * w.rf[0];
    if (g == 0) {
        sm[wave][col] = top;
        sl[wave][col] = w.l[0];
    }
    __syncthreads();
    float mall = kNegInf, lall = 0.0f;
#pragma unroll
    for (int v = 0; v < AW; ++v) mall = fmaxf(mall, sm[v][col]);
    const float base = mall == kNegInf ? 0.0f : mall;
#pragma unroll
    for (int v = 0; v < AW; ++v) lall += sl[v][col] * exp2_(sm[v][col] - base);
    const float f = ldexpf(exp2_(top - base), w.eu);
#pragma unroll
    for (int d = 0; d < ND; ++d) w.o[0][d] *= f;
    if (wave >= 2) {
#pragma unroll
        for (int d = 0; d < ND; ++d) buf[wave - 2][d][lane] = w.o[0][d];
    }
    __syncthreads();
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
    if (wave != 0) return;
#pragma unroll
    for (int d = 0; d < ND; ++d) w.o[0][d] += buf[0][d][lane];
    put_rows(p, job, job.row0, w, &mall, &lall);
}
template <int HD> constexpr int kFewLds = 2 * (HD / 16) * 1024 + 2 * AW * 64;

// ---- many rows: the block's waves split its rows ------------------------------
// A tile is turned into operands once, a part by each wave, and lies in LDS
// for all of them; the next tile is written beside it meanwhile, and the codes
// of the one after are on their way.
template <int HD, int BITS> struct Parts {
    static constexpr int NC = HD / 32, NU = (2 * NC + AW - 1) / AW;   // a wave's blocks (NC of keys, then NC of values)
    typedef uint32_t vec __attribute__((ext_vector_type(BITS == 8 ? 4 : 2)));
    vec code[NU];
    u4 sc[NU];                    // 4 bits: a value block's scales; a key block's two in the first word
    u4 ks, vs;                    // 8 bits
    u2 all_k, all_v;              // 4 bits: the tile's scales, 4 a lane, for its units
    bool ok;
    __device__ __forceinline__ void load(const AttnArgs& p, int head, int id, int tile, int wave) {
        constexpr int BB = BITS == 8 ? 1024 : 512;
        const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
        const TilePtr t = tile_ptr<HD, BITS>(p, head, id, tile);
        ok = t.ok;
        if (!ok) return;
        const uint8_t* vc = t.codes + kv_codes_bytes(p.c.page_size, HD, BITS);
        const uint16_t* vsp = t.scales + (long long)p.c.page_size * kv_groups(HD, BITS);
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int b = wave + u * AW;
            if (b >= 2 * NC) break;
            const int c = b < NC ? b : b - NC;
            code[u] = *(const vec*)((b < NC ? t.codes : vc) + c * BB + lane * sizeof(vec));
            if constexpr (BITS == 4) {
                if (b < NC) {
                    const uint16_t* s = t.scales + c * p.c.page_size;
                    sc[u][0] = s[kv_slot(col)] | (uint32_t)s[kv_slot(col + 16)] << 16;
                } else {
                    sc[u] = *(const u4*)(vsp + c * p.c.page_size + 8 * g);
                }
            }
        }
        if constexpr (BITS == 8) {
            ks = *(const u4*)(t.scales + 8 * g);
            vs = *(const u4*)(vsp + 8 * g);
        } else {
            const int grp = lane >> 3 < NC ? lane >> 3 : 0;
            all_k = *(const u2*)(t.scales + grp * p.c.page_size + (lane & 7) * 4);
            all_v = *(const u2*)(vsp + grp * p.c.page_size + (lane & 7) * 4);
        }
    }
    // largest scale of a tile, from all_k or all_v
    __device__ __forceinline__ static float top(u2 w, int held) {
        const int lane = threadIdx.x & 63;
        float m = 0.0f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int slot = (lane & 7) * 4 + q, tok = 16 * ((slot >> 2) & 1) + 4 * (slot >> 3) + (slot & 3);
            const float f = q & 1 ? bf16_hi(w[q >> 1]) : bf16_lo(w[q >> 1]);
            m = fmaxf(m, tok < held ? f : 0.0f);
        }
        m = max16_32(max_16(m));
        return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, m)));
    }
};

template <int HD, int BITS, int NP, int NR>
__device__ __forceinline__ void many(const AttnArgs& p, Job& job, char* lds) {
    constexpr int NC = HD / 32, NU = Parts<HD, BITS>::NU;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    h8(*frag)[4 * NC][64] = (h8(*)[4 * NC][64])lds;   // [2]: keys (c, i) then values (c, i)
    Rows<HD, NP, NR> w;
    const int row0 = job.row0 + wave * 16 * NR;
    // the block's tiles: the last of its rows sees most
    {
        const int last = min(job.row0 + AW * 16 * NR, job.nrows) - 1;
        long long hi = job.len;
        if (!job.pre) {
            const long long seen = (long long)p.a.lens[job.b] - p.a.seq + last / p.G + 1;
            hi = seen < hi ? seen : hi;
        }
        job.t1 = min(job.t1, hi > 0 ? (int)((hi + 31) / 32) : 0);
    }
    const bool rows = row0 < job.nrows;   // this wave has some
    set_rows(p, job, row0, w);

    Parts<HD, BITS> raw;
    int id = 0, ek = 0, ek_next = 0, en = -126, en_next = -126;
    float ks[8], vs[8];
    bool ok = false;
    u4 ks_raw = {0, 0, 0, 0}, vs_raw = {0, 0, 0, 0};
    if (job.t0 < job.t1) raw.load(p, job.head, page_id(job, p, job.t0), job.t0, wave);
    if (job.t0 + 1 < job.t1) id = page_id(job, p, job.t0 + 1);
    load_rows(p, w);

    // raw tile -> operands in frag[at]
    auto convert = [&](int tile, int at) {
        const int held = (int)min(job.len - (long long)tile * 32, 32ll);
        float fk = 1.0f, fv = 1.0f;
        if constexpr (BITS == 4) {
            ek_next = unit_of(raw.top(raw.all_k, held), 0);
            en_next = max(en_next, unit_of(raw.top(raw.all_v, held), -126));
            fk = ldexpf(1.0f, -ek_next);
            fv = ldexpf(1.0f, -en_next);
        }
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int b = wave + u * AW;
            if (b >= 2 * NC) break;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                h8 x;
                if constexpr (BITS == 8) {
                    x = codes8(raw.code[u][2 * i], raw.code[u][2 * i + 1]);
                } else if (b < NC) {
                    float s = i ? bf16_hi(raw.sc[u][0]) : bf16_lo(raw.sc[u][0]);
                    s = col + 16 * i < held ? s * fk : 0.0f;
                    const h2 f = scale_pair(s, s);
                    const h2 f4_[4] = {f, f, f, f};
                    x = codes4(raw.code[u][i], f4_);
                } else {
                    float s[8];
                    scales8(raw.sc[u], held, s);
                    h2 f[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) f[j] = scale_pair(s[2 * j] * fv, s[2 * j + 1] * fv);
                    x = codes4(raw.code[u][i], f);
                }
                frag[at][2 * b + i][lane] = x;
            }
        }
    };
    if (job.t0 < job.t1) {
        ok = raw.ok;
        if (ok) convert(job.t0, 0);
        ks_raw = raw.ks;
        vs_raw = raw.vs;
        ek = ek_next;
        en = en_next;
        if (job.t0 + 1 < job.t1) raw.load(p, job.head, id, job.t0 + 1, wave);
        if (job.t0 + 2 < job.t1) id = page_id(job, p, job.t0 + 2);
    }
    __syncthreads();
    int at = 0;
    for (int tile = job.t0; tile < job.t1; ++tile, at ^= 1) {
        const u4 ks_cur = ks_raw, vs_cur = vs_raw;
        const int ek_cur = ek, en_cur = en;
        const bool ok_cur = ok;
        if (tile + 1 < job.t1) {
            ok = raw.ok;
            if (ok) convert(tile + 1, at ^ 1);
            ks_raw = raw.ks;
            vs_raw = raw.vs;
            ek = ek_next;
            en = en_next;
            if (tile + 2 < job.t1) raw.load(p, job.head, id, tile + 2, wave);
            if (tile + 3 < job.t1) id = page_id(job, p, tile + 3);
        }
        if (rows && ok_cur) {
            int unit = en_cur;
            if constexpr (BITS == 8) {
                const int held = (int)min(job.len - (long long)tile * 32, 32ll);
                scales8(ks_cur, held, ks);
                scales8(vs_cur, held, vs);
                float vtop = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) vtop = fmaxf(vtop, vs[j]);
                unit = max(w.eu, unit_of(max16_32(vtop), w.eu));
            }
            const h8(*f)[64] = frag[at];
            tile_step<HD, BITS, NP, NR>(
                w, tile, ks, vs, ek_cur, unit, [&](int c, int i) { return f[2 * c + i][lane]; },
                [&](int c, int i) { return f[2 * NC + 2 * c + i][lane]; });
        }
        __syncthreads();
    }
    if (!rows) return;
    float m[NR], l[NR];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        l[t] = w.l[t] + __shfl_xor(w.l[t], 16);
        l[t] += __shfl_xor(l[t], 32);
        m[t] = w.m[t] == kNegInf ? kNegInf : w.m[t] * w.rf[t];
        const float f = ldexpf(1.0f, w.eu);
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) w.o[t][d] *= f;
    }
    put_rows(p, job, row0, w, m, l);
}
template <int HD> constexpr int kManyLds = 2 * 4 * (HD / 32) * 1024;

// row tiles of a wave with many rows: two where they fit beside the rest
template <int HD, int NP> constexpr int kManyRows = HD <= 128 && NP == 1 ? 2 : 1;

// One block: rows of one key/value head against one split of the prefix or of
// a sequence's tokens. PM, OM: the prefix's and the sequences' blocks have
// many rows.
template <int HD, int BITS, int NP, bool PM, bool OM>
__global__ __launch_bounds__(AW * 64, HD <= 128 ? 2 : 1) void kv_attn_kernel(AttnArgs p) {
    constexpr int few_lds = PM && OM ? 0 : kFewLds<HD>, many_lds = PM || OM ? kManyLds<HD> : 0;
    __shared__ __attribute__((aligned(16))) char lds[few_lds > many_lds ? few_lds : many_lds];
    constexpr int NR = kManyRows<HD, NP>;
    const KvAttention& a = p.a;
    const int H = p.c.heads;
    const int npre = p.pre_groups * H * p.pre_slots;
    Job job;
    job.pre = (int)blockIdx.x < npre;
    int x = job.pre ? blockIdx.x : blockIdx.x - npre;
    const int ns = job.pre ? p.pre_slots : p.slots - p.pre_slots;
    job.split = x % ns;
    x /= ns;
    job.head = x % H;
    x /= H;
    job.b = 0;
    int group = x;
    if (!job.pre) {
        job.b = x / p.own_groups;
        group = x - job.b * p.own_groups;
    }
    job.slot = job.pre ? job.split : p.pre_slots + job.split;
    job.nrows = (job.pre ? a.batch : 1) * a.seq * p.G;
    job.table = job.pre ? a.prefix_table : a.table + (long long)job.b * a.max_pages;
    job.len = a.prefix_len;
    if (!job.pre) {
        const long long cap = (long long)a.max_pages * p.c.page_size, len = a.lens[job.b];
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

// One wave a row: its partial results joined in a fixed order, several slots
// side by side where a row is shorter than the wave.
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
    const int part = lane / L, at = (lane - part * L) * 4;
    float total = 0.0f;
    f4 o = {0, 0, 0, 0};
    if (part < W) {
        const float* src = p.part_o + (long long)row * p.slots * HD + at;
#pragma unroll 4
        for (int i = part; i < p.slots; i += W) {
            const float2 v = ml[i];
            const f4 x = *(const f4*)(src + (long long)i * HD);   // (not written where the slot is empty)
            const bool some = !(v.x == kNegInf && v.y == 0.0f);
            const float w = some ? exp2_(v.x - base) : 0.0f;
            total += some ? w * v.y : 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] += some ? x[j] * w : 0.0f;
        }
    }
    const float total1 = total;
    const f4 o1 = o;
#pragma unroll
    for (int s = 1; s < W; ++s) {   // into the first lanes, in order
        const int from = (lane % L) + s * L;
        total += __shfl(total1, from);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] += __shfl(o1[j], from);
    }
    if (part != 0) return;
    const bool none = mx == kNegInf && total == 0.0f;
    o *= 1.0f / total;
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
    const long long total = pre_items * pre_tiles + own_items * own_tiles;
    long long chunk = (total + 2047) / 2048;
    chunk = chunk < 8 ? 8 : chunk;
    p.pre_slots = p.pre_groups ? ceil_div(pre_tiles, chunk) : 0;
    p.own_slots = own_tiles ? ceil_div(own_tiles, chunk) : 1;
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
