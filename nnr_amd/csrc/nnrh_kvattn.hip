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
__device__ __forceinline__ float max16_32(float m) {
    m = fmaxf(m, __shfl_xor(m, 16));
    return fmaxf(m, __shfl_xor(m, 32));
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

// One block: 16 NR rows of one key/value head against one split of the prefix
// or of a sequence's tokens. Its waves take 32-key tiles in turn, each with
// its own running maximum, and join their results through LDS.
template <int HD, int BITS, int NP, int NR>
__global__ __launch_bounds__(AW * 64) void kv_attn_kernel(AttnArgs p) {
    constexpr int NC = HD / 32, ND = HD / 16;
    __shared__ f4 buf[2][NR * ND][64];
    __shared__ float sm[AW][NR * 16], sl[AW][NR * 16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const KvAttention& a = p.a;
    const KvCache& c = p.c;

    // what this block is
    const int H = c.heads;
    const int npre = p.pre_groups * H * p.pre_slots;
    const bool pre = (int)blockIdx.x < npre;
    int x = pre ? blockIdx.x : blockIdx.x - npre;
    const int own_slots = p.slots - p.pre_slots;
    const int ns = pre ? p.pre_slots : own_slots;
    const int split = x % ns;
    x /= ns;
    const int head = x % H;
    x /= H;
    int group = x, b = 0;
    if (!pre) {
        b = x / p.own_groups;
        group = x - b * p.own_groups;
    }
    const int nrows = (pre ? a.batch : 1) * a.seq * p.G;
    const int32_t* table = pre ? a.prefix_table : a.table + (long long)b * a.max_pages;

    // rows of this lane: key limit, place among all rows
    long long len = a.prefix_len;
    if (!pre) {
        const long long cap = (long long)a.max_pages * c.page_size;
        len = a.lens[b];
        len = len < cap ? len : cap;
    }
    int rowat[NR], lim[NR];
    int lo = 0x7fffffff, hi = 0;   // least and largest limit of the block's rows
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        int r = group * 16 * NR + 16 * t + col;
        r = r < nrows ? r : nrows - 1;
        const int tok = r / p.G, hq = head * p.G + r % p.G;   // tok counts over the batch in the prefix's rows
        const int bt = pre ? tok : b * a.seq + tok;
        rowat[t] = bt * a.q_heads + hq;
        long long l = len;
        if (!pre) {
            const long long last = (long long)a.lens[b] - a.seq + tok + 1;
            l = last < l ? last : l;
        }
        lim[t] = l > 0 ? (int)l : 0;
        lo = lim[t] < lo ? lim[t] : lo;
        hi = lim[t] > hi ? lim[t] : hi;
    }
#pragma unroll
    for (int o = 1; o < 16; o *= 2) {
        lo = min(lo, __shfl_xor(lo, o));
        hi = max(hi, __shfl_xor(hi, o));
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    const int chunk = pre ? p.pre_chunk : p.own_chunk;
    const int t0 = split * chunk;
    int t1 = (hi + 31) / 32;
    t1 = t1 < t0 + chunk ? t1 : t0 + chunk;
    const int slot = pre ? split : p.pre_slots + split;
    if (t0 >= t1) {   // nothing here
        if (p.slots > 1) {
            if (wave == 0 && g == 0)
#pragma unroll
                for (int t = 0; t < NR; ++t) p.part_ml[(long long)rowat[t] * p.slots + slot] = float2{kNegInf, 0.0f};
        } else if (wave == 0) {
#pragma unroll
            for (int t = 0; t < NR; ++t)
#pragma unroll
                for (int d = 0; d < ND; ++d)
                    store_y4(a, (long long)rowat[t] * HD + 16 * d + 4 * g, f4{0, 0, 0, 0});
        }
        return;
    }

    // query rows
    h8 qf[NP][NR][NC];
    float rf[NR];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        const int bt = rowat[t] / a.q_heads, hq = rowat[t] - bt * a.q_heads;
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
        rf[t] = ldexpf(a.scale * 1.44269504088896341f, -e);
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float s = ldexpf(v[k][j], e);
                const _Float16 h = (_Float16)s;
                qf[0][t][k][j] = h;
                if constexpr (NP == 2) qf[1][t][k][j] = (_Float16)(s - (float)h);
            }
    }

    f4 o[NR][ND];
    float m[NR], l[NR];
    int eu = -200;                 // exponent of the values' unit
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        m[t] = kNegInf;
        l[t] = 0.0f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[t][d] = f4{0, 0, 0, 0};
    }
    constexpr int BB = BITS == 8 ? 1024 : 512;
    const long long cb = kv_codes_bytes(c.page_size, HD, BITS), part = kv_head_bytes(c.page_size, HD, BITS);

    for (int tile = t0 + wave; tile < t1; tile += AW) {
        const int id = __builtin_amdgcn_readfirstlane(table[tile >> p.page_shift]);
        if (id < 0 || id >= c.num_pages) continue;
        const int in_page = tile & ((1 << p.page_shift) - 1);
        const uint8_t* base = c.data + ((long long)id * H + head) * part;
        const uint8_t* kc = base + (long long)in_page * NC * BB;
        const uint8_t* vc = kc + cb;
        const uint16_t* ks = (const uint16_t*)(base + 2 * cb) + in_page * 32;
        const uint16_t* vs = ks + (long long)c.page_size * kv_groups(HD, BITS);
        const int held = (int)(len - (long long)tile * 32);   // keys of this tile that the source holds

        // scores of 2 x 4 keys a row: key 16 i + 4 g + j in element 4 i + j
        float s[NR][8];
        if constexpr (BITS == 8) {
            u4 kr[NC];
#pragma unroll
            for (int k = 0; k < NC; ++k) kr[k] = *(const u4*)(kc + k * BB + lane * 16);
            const u4 sw = *(const u4*)(ks + 8 * g);
            f4 acc[NR][2];
#pragma unroll
            for (int t = 0; t < NR; ++t) acc[t][0] = acc[t][1] = f4{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < NC; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const h8 kf = codes8(kr[k][2 * i], kr[k][2 * i + 1]);
#pragma unroll
                    for (int t = 0; t < NR; ++t)
#pragma unroll
                        for (int q = 0; q < NP; ++q)
                            acc[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[q][t][k], acc[t][i], 0, 0, 0);
                }
#pragma unroll
            for (int t = 0; t < NR; ++t)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float f = j & 1 ? bf16_hi(sw[j >> 1]) : bf16_lo(sw[j >> 1]);
                    s[t][j] = acc[t][j >> 2][j & 3] * rf[t] * f;
                }
        } else {
            float sc[NC][2], top = 0.0f;
#pragma unroll
            for (int k = 0; k < NC; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float f = bf16_lo(ks[(long long)k * c.page_size + kv_slot(col + 16 * i)]);
                    sc[k][i] = col + 16 * i < held ? f : 0.0f;
                    top = fmaxf(top, sc[k][i]);
                }
#pragma unroll
            for (int d = 1; d < 16; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
            const int ek = top > 0.0f ? ceil_exp(top) : 0;
            f4 acc[NR][2];
#pragma unroll
            for (int t = 0; t < NR; ++t) acc[t][0] = acc[t][1] = f4{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < NC; ++k) {
                const u2 kr = *(const u2*)(kc + k * BB + lane * 8);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const _Float16 f = (_Float16)ldexpf(sc[k][i], -ek);
                    const h2 f2[4] = {{f, f}, {f, f}, {f, f}, {f, f}};
                    const h8 kf = codes4(kr[i], f2);
#pragma unroll
                    for (int t = 0; t < NR; ++t)
#pragma unroll
                        for (int q = 0; q < NP; ++q)
                            acc[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[q][t][k], acc[t][i], 0, 0, 0);
                }
            }
#pragma unroll
            for (int t = 0; t < NR; ++t) {
                const float f = ldexpf(rf[t], ek);
#pragma unroll
                for (int j = 0; j < 8; ++j) s[t][j] = acc[t][j >> 2][j & 3] * f;
            }
        }
        if (tile * 32 + 32 > lo) {
#pragma unroll
            for (int t = 0; t < NR; ++t)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (tile * 32 + 16 * (j >> 2) + 4 * g + (j & 3) >= lim[t]) s[t][j] = kNegInf;
        }

        // values' scales; their unit
        float vf[BITS == 8 ? 1 : NC][8], vtop = 0.0f;
#pragma unroll
        for (int k = 0; k < (BITS == 8 ? 1 : NC); ++k) {
            const u4 w = *(const u4*)(vs + (long long)k * c.page_size + 8 * g);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float f = j & 1 ? bf16_hi(w[j >> 1]) : bf16_lo(w[j >> 1]);
                vf[k][j] = 16 * (j >> 2) + 4 * g + (j & 3) < held ? f : 0.0f;
                vtop = fmaxf(vtop, vf[k][j]);
            }
        }
        vtop = max16_32(vtop);
        int en = eu;
        if (vtop > 0.0f) en = max(eu, ceil_exp(vtop));

        // running maximum; weights 2^15 p
        bool moved = en != eu;
        float al[NR];
#pragma unroll
        for (int t = 0; t < NR; ++t) {
            float mx = m[t];
#pragma unroll
            for (int j = 0; j < 8; ++j) mx = fmaxf(mx, s[t][j]);
            mx = max16_32(mx);
            const float base_m = mx == kNegInf ? 0.0f : mx;
            al[t] = exp2_(m[t] - base_m);
            moved |= mx != m[t];
            m[t] = mx;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                s[t][j] = exp2_(s[t][j] - base_m + 15.0f);
                sum += s[t][j];
            }
            l[t] = l[t] * al[t] + sum;
        }
        if (__any(moved)) {
#pragma unroll
            for (int t = 0; t < NR; ++t) {
                const float f = ldexpf(al[t], eu - en);
#pragma unroll
                for (int d = 0; d < ND; ++d) o[t][d] *= f;
            }
        }
        eu = en;
        h8 pf[NP][NR];
#pragma unroll
        for (int t = 0; t < NR; ++t)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float w = s[t][j];
                if constexpr (BITS == 8) w *= ldexpf(vf[0][j], -eu);
                const _Float16 h = (_Float16)w;
                pf[0][t][j] = h;
                if constexpr (NP == 2) pf[1][t][j] = (_Float16)(w - (float)h);
            }
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            h8 v[2];
            if constexpr (BITS == 8) {
                const u4 vr = *(const u4*)(vc + k * BB + lane * 16);
                v[0] = codes8(vr[0], vr[1]);
                v[1] = codes8(vr[2], vr[3]);
            } else {
                const u2 vr = *(const u2*)(vc + k * BB + lane * 8);
                h2 f2[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    f2[i] = h2{(_Float16)ldexpf(vf[k][2 * i], -eu), (_Float16)ldexpf(vf[k][2 * i + 1], -eu)};
                v[0] = codes4(vr[0], f2);
                v[1] = codes4(vr[1], f2);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int t = 0; t < NR; ++t)
#pragma unroll
                    for (int q = 0; q < NP; ++q)
                        o[t][2 * k + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[i], pf[q][t], o[t][2 * k + i], 0, 0, 0);
        }
    }

    // join the waves: first everyone's maximum, then sums in the units of it
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        l[t] += __shfl_xor(l[t], 16);
        l[t] += __shfl_xor(l[t], 32);
        if (g == 0) {
            sm[wave][16 * t + col] = m[t];
            sl[wave][16 * t + col] = l[t];
        }
    }
    __syncthreads();
    float mall[NR], lall[NR];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        float mx = kNegInf;
#pragma unroll
        for (int w = 0; w < AW; ++w) mx = fmaxf(mx, sm[w][16 * t + col]);
        const float base_m = mx == kNegInf ? 0.0f : mx;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < AW; ++w) sum += sl[w][16 * t + col] * exp2_(sm[w][16 * t + col] - base_m);
        mall[t] = mx;
        lall[t] = sum;
        const float f = ldexpf(exp2_(m[t] - base_m), eu);
#pragma unroll
        for (int d = 0; d < ND; ++d) o[t][d] *= f;
    }
    if (wave >= 2) {
#pragma unroll
        for (int t = 0; t < NR; ++t)
#pragma unroll
            for (int d = 0; d < ND; ++d) buf[wave - 2][t * ND + d][lane] = o[t][d];
    }
    __syncthreads();
    if (wave < 2) {
#pragma unroll
        for (int t = 0; t < NR; ++t)
#pragma unroll
            for (int d = 0; d < ND; ++d) o[t][d] += buf[wave][t * ND + d][lane];
    }
    __syncthreads();
    if (wave == 1) {
#pragma unroll
        for (int t = 0; t < NR; ++t)
#pragma unroll
            for (int d = 0; d < ND; ++d) buf[0][t * ND + d][lane] = o[t][d];
    }
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        if (group * 16 * NR + 16 * t + col >= nrows) continue;
        const float inv = 1.0f / lall[t];
        const bool none = mall[t] == kNegInf && lall[t] == 0.0f;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            f4 v = o[t][d] + buf[0][t * ND + d][lane];
            if (p.slots > 1) {
                *(f4*)(p.part_o + ((long long)rowat[t] * p.slots + slot) * HD + 16 * d + 4 * g) = v;
            } else {
                v *= inv;
                if (none) v = f4{0, 0, 0, 0};
                store_y4(a, (long long)rowat[t] * HD + 16 * d + 4 * g, v);
            }
        }
        if (p.slots > 1 && g == 0) p.part_ml[(long long)rowat[t] * p.slots + slot] = float2{mall[t], lall[t]};
    }
}

// One wave a row: its partial results joined in order of their slots.
template <int HD>
__global__ __launch_bounds__(256) void kv_join_kernel(AttnArgs p) {
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= p.rows) return;
    const float2* ml = p.part_ml + (long long)row * p.slots;
    float mx = kNegInf;
    for (int i = 0; i < p.slots; ++i) mx = fmaxf(mx, ml[i].x);
    const float base = mx == kNegInf ? 0.0f : mx;
    const int at = lane * 4;
    float total = 0.0f;
    f4 o = {0, 0, 0, 0};
    for (int i = 0; i < p.slots; ++i) {
        const float2 v = ml[i];
        if (v.x == kNegInf && v.y == 0.0f) continue;   // its O was not written
        const float w = exp2_(v.x - base);
        total += w * v.y;
        if (at < HD) o += *(const f4*)(p.part_o + ((long long)row * p.slots + i) * HD + at) * w;
    }
    if (at >= HD) return;
    const bool none = mx == kNegInf && total == 0.0f;
    o *= 1.0f / total;
    store_y4(p.a, (long long)row * HD + at, none ? f4{0, 0, 0, 0} : o);
}

// How a call is cut up; of shapes alone, so that the workspace is known before
struct Plan {
    int nr, pre_groups, own_groups, pre_slots, own_slots, pre_chunk, own_chunk;
};
int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }
Plan plan(const KvCache& c, const KvAttention& a) {
    Plan p;
    const int G = a.q_heads / c.heads;
    const long long own_rows = (long long)a.seq * G, pre_rows = own_rows * a.batch;
    p.nr = own_rows > 16 || (a.prefix_len && pre_rows > 16) ? 2 : 1;
    p.own_groups = ceil_div(own_rows, 16 * p.nr);
    p.pre_groups = a.prefix_len ? ceil_div(pre_rows, 16 * p.nr) : 0;
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
hipError_t go(const AttnArgs& p, int nr, unsigned blocks, hipStream_t s) {
    if (nr == 1) kv_attn_kernel<HD, BITS, NP, 1><<<blocks, AW * 64, 0, s>>>(p);
    else kv_attn_kernel<HD, BITS, NP, 2><<<blocks, AW * 64, 0, s>>>(p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.slots == 1) return e;
    kv_join_kernel<HD><<<(unsigned)ceil_div(p.rows, 4), 256, 0, s>>>(p);
    return hipGetLastError();
}
template <int HD>
hipError_t by_type(const AttnArgs& p, int nr, unsigned blocks, hipStream_t s) {
    const bool f32 = p.a.type == FT_F32;
    if (p.c.bits == 8) return f32 ? go<HD, 8, 2>(p, nr, blocks, s) : go<HD, 8, 1>(p, nr, blocks, s);
    return f32 ? go<HD, 4, 2>(p, nr, blocks, s) : go<HD, 4, 1>(p, nr, blocks, s);
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
    case 64: return by_type<64>(p, pl.nr, blocks, s);
    case 96: return by_type<96>(p, pl.nr, blocks, s);
    case 128: return by_type<128>(p, pl.nr, blocks, s);
    case 256: return by_type<256>(p, pl.nr, blocks, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace nnrh
