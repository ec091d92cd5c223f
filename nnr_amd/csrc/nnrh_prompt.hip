// nnrh_prompt.hip -- attention of packed prompts to themselves, before their keys
// and values go into a cache: row (token i, head) of a sequence of n tokens sees
// tokens 0 .. i (or all n):
//   y = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale (q k_j - m)).
// One pass over the keys with a running maximum m and total (sums are rescaled when
// m moves).
//
// The rows of one key/value head are its tokens' query heads side by side (token
// major), so that a tile of keys serves all heads of a group, and a block's rows
// see almost the same keys. A block has 4 waves of 32 rows; 64 keys (fp32: 32) are
// brought into LDS by direct loads while the tile before is worked on.
//   S^T = K Q^T (keys x rows),   O^T = V^T P^T (elements x rows)
// by 32x32 MFMAs: a lane of S^T holds 16 scores of one row, 4 neighbouring keys at
// a time, which are its part of the second product's operand as they are. V^T comes
// out of LDS by transposing reads (16 bits) or one element a lane (fp32).
//
// fp32 tensors meet in fp32 MFMAs. 16-bit ones in 16-bit MFMAs with fp32 sums: the
// weights p are rounded to the tensors' type (11 or 8 bits), which is as far off
// as rounding the result is, and would cost a second product to avoid. They are
// held as 2^top p: fp16 has no small numbers (p <= 2^15 there, and weights down to
// 2^-35 of the largest keep a bit); in bf16 and fp32 a sum of largest numbers must
// not pass them (2^20 equal weights of such values still do not), for which sums of results
// under 2^-96 are no normal fp32 numbers: their steps, 2^-149, are 2^-119 of a result.
//
// Bound by the order of a wave's own work (products, maximum, weights, products), which
// two waves a SIMD hide in part, at heads of 256 one cannot: 8192 tokens, 32 heads over
// 8 of 128, bf16, 550 GFLOP in 540 us (a large library product's rate: 407), matrix units
// 57 % busy, vector units 60; 3 sequences to 2001, 8 heads over one of 256, 27 GFLOP in
// 64 us (20), 21 % and 27 %. fp32 by its products: heads of 256, 32 over 4 of 2000
// tokens 576 us, 73 % of a library product's rate.
#include "nnrh_decode.h"


namespace nnrh {
namespace {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef uint16_t us2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
#define NNRH_LDS __attribute__((address_space(3)))

constexpr int PW = 4, PR = 32;              // waves of a block, rows of a wave
// A block's waves are KG groups: waves of different groups take different keys of a
// tile for the same rows, and are joined at the end.
template <int KG> constexpr int kBlockRows = PW / KG * PR;
template <int TY, int KG> constexpr int kWaveKeys = TY != FT_F32 && KG == 1 ? 64 : 32;   // of a tile
constexpr float kNegInf = -__builtin_inff();
constexpr float kLeast = 1e-37f;            // a factor of 0 would make NaN of a masked score, -inf

// slack: powers of two by which scores may outgrow the maximum that they refer to.
// (3 sequences to 2001, heads of 256, bf16, scores of a deviation of 1.4: with 4 in
// place of 10 70 us, 64 so; others 1-2 %. In fp16 it would be small weights' bits.)
template <int TY> struct Type;
template <> struct Type<FT_F32> {
    static constexpr int size = 4;
    static constexpr float top = -30.0f, slack = 10.0f;
};
template <> struct Type<FT_F16> {
    typedef h4 v4;
    typedef h8 v8;
    static constexpr int size = 2;
    static constexpr float top = 11.0f, slack = 4.0f;
    static constexpr uint32_t inf = 0x7c00;
    __device__ static __forceinline__ f16v mfma(u4 a, u4 b, f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
};
template <> struct Type<FT_BF16> {
    typedef b4 v4;
    typedef b8 v8;
    static constexpr int size = 2;
    static constexpr float top = -30.0f, slack = 10.0f;
    static constexpr uint32_t inf = 0x7f80;
    __device__ static __forceinline__ f16v mfma(u4 a, u4 b, f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    }
};

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float max_halves(float m) {   // over lanes 32 apart
    const uint32_t u = __builtin_bit_cast(uint32_t, m);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
// keeps the compiler from computing both sides of a branch that is hardly ever taken
__device__ __forceinline__ void stay_a_branch() { asm volatile(""); }
// no load or store moves past it
__device__ __forceinline__ void in_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// the lane, for what is rarely done: nothing that follows from it is kept in registers before
__device__ __forceinline__ int lane_here() {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    return lane;
}

// ---- which rows a block has -------------------------------------------------------
struct Job {
    int s, len;        // first token, tokens
    int row0, nrows;   // the block's first row, rows of the sequence
};
// blocks of BM rows that tokens s .. e - 1 have
template <int BM>
__device__ __forceinline__ int blocks_of(const PromptAttention& a, int G, int s, int e) {
    s = min(max(s, 0), a.tokens);
    return (int)(((long long)(min(max(e, s), a.tokens) - s) * G + BM - 1) / BM);
}
template <int CTRL> __device__ __forceinline__ int dpp(int x) { return __builtin_amdgcn_update_dpp(x, x, CTRL, 0xf, 0xf, false); }
// fn over all 64 lanes, in all of them: quads, halves and rows of 16 mirrored, then rows and halves exchanged
template <class F> __device__ __forceinline__ int over_lanes(int x, F fn) {
    x = fn(x, dpp<0xb1>(x));
    x = fn(x, dpp<0x4e>(x));
    x = fn(x, dpp<0x141>(x));
    x = fn(x, dpp<0x140>(x));
    const auto r = __builtin_amdgcn_permlane16_swap((uint32_t)x, (uint32_t)x, false, false);
    x = fn((int)r[0], (int)r[1]);
    const auto q = __builtin_amdgcn_permlane32_swap((uint32_t)x, (uint32_t)x, false, false);
    return __builtin_amdgcn_readfirstlane(fn((int)q[0], (int)q[1]));
}
__device__ __forceinline__ int sum_lanes(int x) {
    return over_lanes(x, [](int a, int b) { return a + b; });
}
template <int BM>
__device__ __forceinline__ long long first_number(const PromptAttention& a, int G, int b) {
    return (long long)min(max(a.starts[b], 0), a.tokens) * G / BM + b;
}
// Block `number` of a launch: sequence b and its block. Up to 64 sequences (a lane
// each): all sequences' blocks by their place, the last places first, so that long
// ones begin first wherever they are. More: sequence by sequence from the last one on;
// one's blocks begin at number starts[b] G / BM + b, as rounding up adds at most one
// each. Numbers that no rows are left for do nothing.
template <int BM>
__device__ __forceinline__ bool find_job(const PromptAttention& a, int G, int number, int numbers, Job& job) {
    const int lane = threadIdx.x & 63;
    int b, block;
    if (a.seqs <= 64) {
        const int n = lane < a.seqs ? blocks_of<BM>(a, G, a.starts[lane], a.starts[lane + 1]) : 0;
        // the place p with C(p + 1) <= number < C(p), C(p) = blocks at places p and up
        int p = 0, above = 0;
        if (a.seqs == 1) {
            p = __builtin_amdgcn_readfirstlane(n) - 1 - number;
            if (p < 0) return false;
            above = number;
        } else {
            if (number >= sum_lanes(n)) return false;
            int hi = over_lanes(n, [](int a, int b) { return max(a, b); });
            while (hi - p > 1) {   // C(p) > number >= C(hi)
                const int mid = (p + hi) >> 1, c = sum_lanes(max(n - mid, 0));
                if (c > number) p = mid;
                else hi = mid;
            }
            above = sum_lanes(max(n - p - 1, 0));
        }
        const unsigned long long have = __ballot(n > p);
        const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(have >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)have, 0));
        const unsigned long long mine = __ballot(n > p && rank == number - above);
        if (!mine) return false;   // (not reached: lanes past the sequences have no blocks)
        b = __builtin_ctzll(mine);
        block = p;
    } else {
        number = numbers - 1 - number;
        // the last sequence that does not begin after it: 64 looked at at once
        int lo = 0, n = a.seqs;
        while (true) {
            const int step = (n + 63) / 64;
            const bool le = lane * step < n && first_number<BM>(a, G, lo + lane * step) <= number;
            const int count = __popcll(__ballot(le));
            if (!count) return false;
            lo += (count - 1) * step;
            n = min(step, n - (count - 1) * step);
            if (n <= 1) break;
        }
        b = lo;
        block = (int)(number - first_number<BM>(a, G, b));
    }
    b = __builtin_amdgcn_readfirstlane(b);
    const int s = min(max(a.starts[b], 0), a.tokens), e = min(max(a.starts[b + 1], s), a.tokens);
    job.s = __builtin_amdgcn_readfirstlane(s);
    job.len = __builtin_amdgcn_readfirstlane(e - s);
    const long long row0 = (long long)block * BM, nrows = (long long)job.len * G;
    if (row0 >= nrows) return false;
    job.row0 = __builtin_amdgcn_readfirstlane((int)row0);
    job.nrows = (int)nrows;
    return true;
}

// ---- tiles of keys and values in LDS -------------------------------------------------
// A row of 16-byte chunks a token, at a place that is the chunk's number with some
// bits turned by the token's, so that neither product's reads meet in a bank.
template <int TY, int HD, int KG> struct Lds {
    static constexpr int NW = kWaveKeys<TY, KG>, N = KG * NW;     // tokens of a tile: a wave's, all
    static constexpr int real = HD * Type<TY>::size / 16;         // chunks of a row
    static constexpr int CH = HD == 96 ? real * 4 / 3 : real;     // held, a power of two
    static constexpr int tile = N * CH * 16, part = NW * CH * 16;
    static constexpr int loads = N * CH / (PW * 64);              // of a thread
    // the keys' reads: 32 rows, one chunk
    static __device__ __forceinline__ int key(int row) { return CH == 8 ? row >> 1 & 7 : row & 15; }
    // the values': 16 bits: rows r .. r + 3 (and 4 further), 64 bytes of each; fp32:
    // rows r and r + 4, 128 bytes of each
    static __device__ __forceinline__ int value(int row) {
        if (TY == FT_F32) return (row >> 2 & 1) << 3;
        return CH == 8 ? (row >> 1 & 1) << 2 : (row & 3) << 2 | (row >> 2 & 3);
    }
};
// A thread's loads of a tile: bytes from the tile's first row
template <int TY, int HD, int KG> struct Loads {
    typedef Lds<TY, HD, KG> L;
    uint32_t at[L::loads];
    static __device__ __forceinline__ uint32_t place(int i, int thread, uint32_t stride, bool values) {
        const int id = i * PW * 64 + thread, row = id / L::CH;
        const int chunk = id % L::CH ^ (values ? L::value(row) : L::key(row));
        return chunk < L::real ? row * stride + chunk * 16 : 0xfffffff0u;   // (none: nothing is read there)
    }
    __device__ __forceinline__ void set(uint32_t stride, bool values) {
#pragma unroll
        for (int i = 0; i < L::loads; ++i) at[i] = place(i, threadIdx.x, stride, values);
    }
    // rows: those that are left from the tile's first on; what is past them reads as 0.
    // fn(i): the bytes of load i
    template <class F> static __device__ __forceinline__ void start(const uint8_t* first, uint32_t stride, int rows, uint8_t* lds, F fn) {
        const uint32_t bytes = (uint32_t)(min(rows, L::N) - 1) * stride + HD * Type<TY>::size;
        const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)first, (short)0, (int)bytes, 0x00020000);
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int i = 0; i < L::loads; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (NNRH_LDS void*)(lds + (i * PW + wave) * 1024), 16, (int)fn(i), 0, 0, 0);
    }
    __device__ __forceinline__ void load(const uint8_t* first, uint32_t stride, int rows, uint8_t* lds) const {
        start(first, stride, rows, lds, [&](int i) { return at[i]; });
    }
    // with places found anew, for want of registers
    static __device__ __forceinline__ void load_anew(const uint8_t* first, uint32_t stride, int rows, uint8_t* lds, bool values) {
        const int thread = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 64 + lane_here();
        start(first, stride, rows, lds, [&](int i) { return place(i, thread, stride, values); });
    }
};

// ---- a wave's rows ---------------------------------------------------------------------
template <int TY, int HD> struct Rows {
    static constexpr int ND = HD / 32;
    static constexpr int NQ = TY == FT_F32 ? HD / 8 : HD / 16;
    u4 q[NQ];          // 16 bits: elements 16 i + 8 half ..; fp32: 8 i + 4 half ..
    f16v o[ND];        // sums of 2^top p v: elements 32 d + 8 (r / 4) + 4 half + r % 4
    float m, l;        // the raw score that weights refer to; the lane's total of 2^top p
    float rk;          // scale log2 e > 0
    int lim;           // keys that the row sees
};

// The sums of wide heads lie in the accumulator half of the register file, which
// products read and write but no other instruction does. Left to itself the compiler
// takes all of them to the other half and back at every tile for this one that hardly
// ever runs. (The waits are for a product's result, and before the next one; all sums
// are their operands, so that no product moves past them.)
__device__ __forceinline__ void acc_wait(f16v* o) {
    asm volatile("s_nop 15\n\ts_nop 15" : "+a"(o[0]), "+a"(o[1]), "+a"(o[2]), "+a"(o[3]), "+a"(o[4]), "+a"(o[5]), "+a"(o[6]), "+a"(o[7]));
}
__device__ __forceinline__ void acc_stay(f16v* o) {
    asm volatile("" : "+a"(o[0]), "+a"(o[1]), "+a"(o[2]), "+a"(o[3]), "+a"(o[4]), "+a"(o[5]), "+a"(o[6]), "+a"(o[7]));
}
template <int HD> __device__ __forceinline__ void scale_acc(f16v* o, float al) {
    static_assert(HD == 256);
    acc_wait(o);
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float x = o[d][r], y;
            asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %1, %2\n\tv_accvgpr_write_b32 %0, %1"
                         : "+a"(x), "=&v"(y) : "v"(al));
            o[d][r] = x;
        }
    acc_wait(o);
}
__device__ __forceinline__ float add_acc(float o, float x) {
    float y;
    asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_add_f32 %1, %1, %2\n\tv_accvgpr_write_b32 %0, %1"
                 : "+a"(o), "=&v"(y) : "v"(x));
    return o;
}

// Scores of NB x 16 keys a lane, raw, to weights 2^top p. key0: of the tile;
// masked: some row does not see all of it.
template <int TY, int HD, int KG, int NB>
__device__ __forceinline__ void weigh(Rows<TY, HD>& w, f16v* s, int key0, bool masked) {
    const int half = (threadIdx.x & 63) >> 5;
    if (masked) {
        stay_a_branch();
        const int end = w.lim - key0 - 4 * half;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (32 * b + 8 * (r >> 2) + (r & 3) >= end) s[b][r] = kNegInf;
    }
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[b][r]);
    mx = max_halves(mx);
    // the maximum moves on only where a score outgrows it by more than the slack (a row's
    // by itself: what other rows see has no part in its rounding)
    const bool up = mx * w.rk > __builtin_fmaf(w.m, w.rk, Type<TY>::slack);
    if (__builtin_expect(__any(up), 0)) {
        stay_a_branch();
        const float al = up ? exp2_((w.m - mx) * w.rk) : 1.0f;
        w.m = up ? mx : w.m;
        w.l *= al;
        if constexpr (HD > 128) {
            if (key0 >= NB * 32 * KG) scale_acc<HD>(w.o, al);   // (before a wave's first tile the sums are zeros)
        } else {
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) w.o[d] *= al;
        }
    }
    const float base = w.m == kNegInf ? 0.0f : w.m;
    constexpr float top = Type<TY>::top;
    float sum[2] = {0.0f, 0.0f};
    const float off = top - base * w.rk;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            // (the difference first in fp32: of large scores' products little would be left;
            // nor of an exponent's last bits beside 2^top)
            if constexpr (TY == FT_F32) s[b][r] = exp2_((s[b][r] - base) * w.rk) * ldexpf(1.0f, (int)top);
            else s[b][r] = exp2_(__builtin_fmaf(s[b][r], w.rk, off));
            sum[r & 1] += s[b][r];
        }
    w.l += sum[0] + sum[1];
}

// V^T of a 16-bit tile: elements 32 d .. of keys 16 m + 8 (j / 4) + 4 half + j % 4
template <int TY, int HD, int KG>
__device__ __forceinline__ u4 value_operand(const uint8_t* v, int lane, int m, int d) {
    typedef Lds<TY, HD, KG> L;
    const int half = lane >> 5, in = lane & 15;
    u2 x[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        // 16 lanes read 4 rows of 16 elements, and get an element of 4 rows each
        const int row = 16 * m + 8 * i + 4 * half + (in >> 2), e = 32 * d + (lane & 16) + 4 * (in & 3);
        const uint8_t* at = v + row * L::CH * 16 + ((e >> 3 ^ L::value(row)) << 4) + (e & 4) * 2;
        x[i] = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((NNRH_LDS s4*)at));
    }
    return u4{x[0][0], x[0][1], x[1][0], x[1][1]};
}

// Are there infinities or NaNs among the values of a wave's part of the tile?
template <int TY, int HD, int KG>
__device__ __forceinline__ bool any_bad(const uint8_t* v) {
    typedef Lds<TY, HD, KG> L;
    const uint8_t* at = v + lane_here() * 16;
    us2 top = {0, 0};
    bool bad = false;
#pragma unroll 8
    for (int i = 0; i < L::NW * L::CH / 64; ++i) {   // (in any order; what is held and not a row's is zeros)
        const u4 x = *(const u4*)(at + i * 1024);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (TY == FT_F32) bad |= (x[j] & 0x7fffffffu) >= 0x7f800000u;
            else top = __builtin_elementwise_max(top, __builtin_bit_cast(us2, x[j] & 0x7fff7fffu));
        }
    }
    if constexpr (TY != FT_F32) bad = top[0] >= Type<TY>::inf || top[1] >= Type<TY>::inf;
    return __any(bad);
}

// O^T += V^T P^T over a tile. FINITE: of its finite values alone.
template <int TY, int HD, int KG, bool FINITE>
__device__ __forceinline__ void add_values(Rows<TY, HD>& w, const f16v* s, const uint8_t* v, int lane) {
    const int half = lane >> 5;
    if constexpr (TY == FT_F32) {
        typedef Lds<TY, HD, KG> L;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int row = 8 * (r >> 2) + 4 * half + (r & 3);
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) {
                const int e = 32 * d + (lane & 31);
                float x = *(const float*)(v + (row * L::CH + (e >> 2 ^ L::value(row))) * 16 + (e & 3) * 4);
                if (FINITE) x = fabsf(x) < __builtin_inff() ? x : 0.0f;
                w.o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, s[0][r], w.o[d], 0, 0, 0);
            }
        }
    } else {
        typedef typename Type<TY>::v8 v8;
#pragma unroll
        for (int m = 0; m < kWaveKeys<TY, KG> / 16; ++m) {
            v8 p;
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = s[m >> 1][8 * (m & 1) + j];
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) {
                u4 x = value_operand<TY, HD, KG>(v, lane, m, d);
                if (FINITE) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {   // (an exponent of ones carries into the sign's place)
                        const uint32_t bad = ((x[j] & 0x7fff7fffu) + (0x8000u - Type<TY>::inf) * 0x10001u) >> 15 & 0x10001u;
                        x[j] &= ~(bad * 0xffffu);
                    }
                }
                w.o[d] = Type<TY>::mfma(x, __builtin_bit_cast(u4, p), w.o[d]);
            }
        }
    }
}
// What a row sees of a tile's infinities and NaNs
template <int TY, int HD, int KG>
__device__ __forceinline__ void add_others(Rows<TY, HD>& w, const uint8_t* v, int key0) {
    typedef Lds<TY, HD, KG> L;
    const int half = lane_here() >> 5;
    // (what is not finite of elements 32 d .. in a row that the lane's row sees)
    const auto of_row = [&](int row, int d, auto add) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = 32 * d + 8 * i + 4 * half, c = e * Type<TY>::size / 16;
            const uint8_t* at = v + (row * L::CH + (c ^ L::value(row))) * 16 + e * Type<TY>::size % 16;
            float x[4];
            if constexpr (TY == FT_F32) {
                const f4 y = *(const f4*)at;
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = y[r];
            } else {
                const typename Type<TY>::v4 y = *(const typename Type<TY>::v4*)at;
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = (float)y[r];
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (!(fabsf(x[r]) < __builtin_inff()) && key0 + row < w.lim) add(4 * i + r, x[r]);
        }
    };
    if constexpr (HD > 128) {   // 32 elements at a time in registers that additions reach
        acc_wait(w.o);
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) {
            float sum[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) sum[r] = -0.0f;
#pragma unroll 1
            for (int row = 0; row < L::NW; ++row) {
                if (!__any(key0 + row < w.lim)) break;
                of_row(row, d, [&](int r, float x) { sum[r] += x; });
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) w.o[d][r] = add_acc(w.o[d][r], sum[r]);
        }
        acc_wait(w.o);
    } else {
#pragma unroll 1
        for (int row = 0; row < L::NW; ++row) {
            if (!__any(key0 + row < w.lim)) break;
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) of_row(row, d, [&](int r, float x) { w.o[d][r] += x; });
        }
    }
}

template <int TY, int HD, int KG>
__device__ __forceinline__ void raw_scores(const Rows<TY, HD>& w, f16v* s, const uint8_t* k, int lane) {
    typedef Lds<TY, HD, KG> L;
    const int half = lane >> 5;
#pragma unroll
    for (int b = 0; b < L::NW / 32; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] = 0.0f;
#pragma unroll
    for (int i = 0; i < Rows<TY, HD>::NQ; ++i)
#pragma unroll
        for (int b = 0; b < L::NW / 32; ++b) {
            const int row = 32 * b + (lane & 31);
            const u4 x = *(const u4*)(k + (row * L::CH + (2 * i + half ^ L::key(row))) * 16);
            if constexpr (TY == FT_F32) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    s[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(__builtin_bit_cast(float, (uint32_t)x[j]),
                                                                __builtin_bit_cast(float, (uint32_t)w.q[i][j]), s[b], 0, 0, 0);
            } else {
                s[b] = Type<TY>::mfma(x, w.q[i], s[b]);
            }
        }
    if constexpr (TY != FT_F32 && HD > 64) {
        // four reads on their way before the product that needs the first (of its own the
        // compiler takes one; heads of 256, 32 over 8 of 4096 tokens: 342 us, so 324)
        constexpr int ahead = 4, all = Rows<TY, HD>::NQ * (L::NW / 32);
        __builtin_amdgcn_sched_group_barrier(0x100, ahead, 0);
#pragma unroll
        for (int i = 0; i < all - ahead; ++i) {
            __builtin_amdgcn_sched_group_barrier(8, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(8, ahead, 0);
    }
}

// Waves that have seen other keys for the same rows: sums and totals by the rows'
// common maximum, in the order of the groups. A wave ends up with the elements
// 32 d .. where d % KG is its group's number. parts: [PW], of a wave.
template <int TY, int HD, int KG>
__device__ __forceinline__ void join(Rows<TY, HD>& w, int wave, uint8_t* lds) {
    constexpr int ND = HD / 32;
    const int lane = threadIdx.x & 63, col = lane & 31, group = wave % KG, first = wave - group;
    float2(*ml)[PR] = (float2(*)[PR])lds;                                   // [PW]
    f4(*sums)[ND][4][64] = (f4(*)[ND][4][64])(lds + sizeof(float2) * PW * PR);   // [PW]
    w.l += __shfl_xor(w.l, 32);
    __syncthreads();
    if (lane < PR) ml[wave][col] = float2{w.m, w.l};
    __syncthreads();
    float m = kNegInf;
#pragma unroll
    for (int j = 0; j < KG; ++j) m = fmaxf(m, ml[first + j][col].x);
    const auto factor = [&](float x) { return x == kNegInf ? 0.0f : exp2_((x - m) * w.rk); };
    const float f = factor(w.m);
    w.l = 0.0f;
#pragma unroll
    for (int j = 0; j < KG; ++j) {
        const float2 v = ml[first + j][col];
        w.l += v.y * factor(v.x);
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        w.o[d] *= f;
        if (d % KG == group) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[wave][d][i][lane] = f4{w.o[d][4 * i], w.o[d][4 * i + 1], w.o[d][4 * i + 2], w.o[d][4 * i + 3]};
    }
    __syncthreads();
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        if (d % KG != group) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f4 x = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < KG; ++j)
                x += j == group ? f4{w.o[d][4 * i], w.o[d][4 * i + 1], w.o[d][4 * i + 2], w.o[d][4 * i + 3]} : sums[first + j][d][i][lane];
#pragma unroll
            for (int r = 0; r < 4; ++r) w.o[d][4 * i + r] = x[r];
        }
    }
}
template <int HD> constexpr int kJoinLds = PW * PR * 8 + PW * HD * PR * 4;

// Two tiles of wide fp32 heads do not fit twice: there is a place for keys and one for
// values, and each is loaded as soon as all waves have read it, while they work on the
// other.
template <int TY, int HD, int KG> constexpr bool kOnce = 4 * Lds<TY, HD, KG>::tile > 160 * 1024;

template <int TY, int HD, int KG>
__global__ __launch_bounds__(PW * 64, HD <= 128 ? 2 : 1) void prompt_kernel(PromptAttention a, int G, int blocks) {
    typedef Lds<TY, HD, KG> L;
    constexpr int ES = Type<TY>::size, BM = kBlockRows<KG>, NB = L::NW / 32;
    constexpr bool once = kOnce<TY, HD, KG>;
    constexpr int held = (once ? 2 : 4) * L::tile, bytes = KG > 1 && kJoinLds<HD> > held ? kJoinLds<HD> : held;
    __shared__ __attribute__((aligned(16))) uint8_t lds_[bytes];
    uint8_t(*lds)[2][L::tile] = (uint8_t(*)[2][L::tile])lds_;   // [2]: keys, values
    // Heads first, so that a head's blocks stay on an XCD where heads are a multiple of 8.
    const int head = blockIdx.x % a.kv_heads;
    Job job;
    if (!find_job<BM>(a, G, (int)(blockIdx.x / a.kv_heads), blocks, job)) return;
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part = wave % KG, row0 = job.row0 + wave / KG * PR;
    Rows<TY, HD> w;
    const int row = min(row0 + col, job.nrows - 1);
    const int tok = row / G, hq = head * G + row - tok * G;
    w.lim = a.causal ? tok + 1 : job.len;
    // keys that some row of the block sees, that all of them do, that some row of the wave does
    const int block_hi = a.causal ? (min(job.row0 + BM, job.nrows) - 1) / G + 1 : job.len;
    const int block_lo = a.causal ? job.row0 / G + 1 : job.len;
    const int hi = __builtin_amdgcn_readlane(w.lim, 31);

    Loads<TY, HD, KG> kl, vl;
    const uint32_t ks = (uint32_t)(a.ks * ES), vs = (uint32_t)(a.vs * ES);
    kl.set(ks, false);
    vl.set(vs, true);
    const uint8_t* k = (const uint8_t*)a.k + (job.s * a.ks + (long long)head * HD) * ES;
    const uint8_t* v = (const uint8_t*)a.v + (job.s * a.vs + (long long)head * HD) * ES;
    const auto load = [&](int key0, int at) {
        kl.load(k + (long long)key0 * ks, ks, job.len - key0, lds[at][0]);
        if constexpr (once) in_order();   // (the first wait there counts values behind keys)
        vl.load(v + (long long)key0 * vs, vs, job.len - key0, lds[at][1]);
    };
    load(0, 0);
    {
        const uint8_t* q = (const uint8_t*)a.q + ((job.s + (long long)tok) * a.qs + (long long)hq * HD) * ES + 16 * half;
        const uint32_t sign = a.scale < 0.0f ? (TY == FT_F32 ? 0x80000000u : 0x80008000u) : 0u;   // (so that rk is positive)
#pragma unroll
        for (int i = 0; i < Rows<TY, HD>::NQ; ++i) w.q[i] = *(const u4*)(q + 32 * i) ^ u4{sign, sign, sign, sign};
    }
    w.rk = fmaxf(fabsf(a.scale) * 1.44269504088896341f, kLeast);
    w.m = kNegInf;
    w.l = 0.0f;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) w.o[d][r] = 0.0f;

    int at = 0, key0 = 0;
    f16v s[NB];
    // a wave's part of the tile, with some rows that do not see all of it
    const auto add_masked = [&](const uint8_t* v, int first) {
        if (__builtin_expect(any_bad<TY, HD, KG>(v), 0)) {
            stay_a_branch();
            add_values<TY, HD, KG, true>(w, s, v, lane_here());
            add_others<TY, HD, KG>(w, v, first);
        } else {
            add_values<TY, HD, KG, false>(w, s, v, lane_here());
        }
        if constexpr (HD > 128) acc_stay(w.o);
    };
    if constexpr (once) {
        static_assert(L::loads == 16);   // what the waits count
        for (; key0 < block_hi; key0 += L::N) {
            const int first = key0 + part * L::NW;
            const bool sees = first < hi, more = key0 + L::N < block_hi, masked = key0 + L::N > block_lo;
            asm volatile("s_waitcnt vmcnt(16) lgkmcnt(0)\n\ts_barrier" ::: "memory");   // the keys; the values are on their way
            if (sees) raw_scores<TY, HD, KG>(w, s, lds[0][0] + part * L::part, lane_here());
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (more) kl.load_anew(k + (long long)(key0 + L::N) * ks, ks, job.len - key0 - L::N, lds[0][0], false);
            if (sees) weigh<TY, HD, KG, NB>(w, s, first, masked);
            if (more) asm volatile("s_waitcnt vmcnt(16)\n\ts_barrier" ::: "memory");    // the values; the next keys are on their way
            else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
            const uint8_t* v_ = lds[0][1] + part * L::part;
            if (sees) {
                if (masked) add_masked(v_, first);
                else add_values<TY, HD, KG, false>(w, s, v_, lane_here());
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (more) vl.load_anew(v + (long long)(key0 + L::N) * vs, vs, job.len - key0 - L::N, lds[0][1], true);
        }
    } else {
        const auto next = [&] {
            // this tile is there, and the one before has been read by all
            __builtin_amdgcn_s_waitcnt(0);
            asm volatile("s_barrier" ::: "memory");
            if (key0 + L::N < block_hi) load(key0 + L::N, at ^ 1);
        };
        for (; key0 + L::N <= block_lo; key0 += L::N, at ^= 1) {
            next();
            raw_scores<TY, HD, KG>(w, s, lds[at][0] + part * L::part, lane);
            weigh<TY, HD, KG, NB>(w, s, key0, false);
            add_values<TY, HD, KG, false>(w, s, lds[at][1] + part * L::part, lane);
        }
        // the tiles that some of the block's rows see in part or not at all
        for (; key0 < block_hi; key0 += L::N, at ^= 1) {
            next();
            const int first = key0 + part * L::NW;   // the wave's part of the tile
            if (first >= hi) continue;
            raw_scores<TY, HD, KG>(w, s, lds[at][0] + part * L::part, lane_here());
            weigh<TY, HD, KG, NB>(w, s, first, true);
            add_masked(lds[at][1] + part * L::part, first);
        }
    }
    if constexpr (KG > 1) join<TY, HD, KG>(w, wave, lds_);
    else w.l += __shfl_xor(w.l, 32);
    const float inv = 1.0f / w.l;
    // (found anew where registers are short)
    const int l_ = HD > 128 ? lane_here() : lane, mine = row0 + (l_ & 31);
    if (mine >= job.nrows) return;
    const int of = HD > 128 ? mine / G : tok, h = HD > 128 ? head * G + mine - of * G : hq;
    const long long y = ((job.s + (long long)of) * a.q_heads + h) * HD + 4 * (l_ >> 5);
#pragma unroll
    for (int d = 0; d < HD / 32; ++d) {
        if (d % KG != part) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f4 x;
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = w.o[d][4 * i + r] * inv;
            const long long e = y + 32 * d + 8 * i;
            if constexpr (TY == FT_F32) *(f4*)((float*)a.y + e) = x;
            else if constexpr (TY == FT_F16) *(h4*)((_Float16*)a.y + e) = h4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
            else *(b4*)((__bf16*)a.y + e) = b4{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]};
        }
    }
}

template <int TY, int HD, int KG>
hipError_t start(const PromptAttention& a, hipStream_t s) {
    const int G = a.q_heads / a.kv_heads, blocks = (int)((long long)a.tokens * G / kBlockRows<KG>) + a.seqs;
    prompt_kernel<TY, HD, KG><<<(unsigned)blocks * a.kv_heads, PW * 64, 0, s>>>(a, G, blocks);
    return hipGetLastError();
}
// Groups by how many blocks of 128 rows there would be. With two or four, blocks are
// shorter and more, at more loads a row and a join: where the chip is not full, or
// full for so short that its last blocks count. Up to these (fp16, us, one group and
// two: heads of 64, 12 of 4096 tokens, 396 blocks 58.7, 45.7; 32 over 8 of 2048, 520
// 34.8, 35.6. Heads of 128, 453 blocks 65, 53; 516 34, 38. Heads of 256, one block
// a CU, 83 20.1, 16.3; 263 76, 68; 317 45, 58; 396 141, 170; fp32 117 153, 97; 258 1048,
// 701; 395 100, 131; 504 576, 723. fp32, bound by its products: heads of 64, 664 64.5,
// 53.3; heads of 128, 520 387, 340; 664 90, 116; heads of 96 as of 128: fp16 383 33.7, 32.9,
// 396 77.8, 68.7; 491 26.2, 29.9; fp32 480 712, 596; 520 300, 274; 658 402, 446. Four groups
// and two: heads of 64, 129 16.9, 21.0; 204 22.5, 22.7; heads of 128, 63 15.7, 18.6; 83 14.2, 10.8;
// of 96, 63 21.3, 24.1; 77 16.3, 17.5; 133 23.4, 20.4.)
template <int TY, int HD> constexpr int kTwoGroups = HD > 128 ? 272 : TY != FT_F32 ? 448 : HD == 64 ? 1024 : 512;
template <int TY, int HD> constexpr int kFourGroups = HD == 64 ? 128 : TY != FT_F32 && HD <= 128 ? 64 : 0;
template <int TY, int HD>
hipError_t by_blocks(const PromptAttention& a, hipStream_t s) {
    const long long blocks = (long long)a.tokens * a.q_heads / kBlockRows<1> + (long long)a.seqs * a.kv_heads;
    if constexpr (kFourGroups<TY, HD> > 0)
        if (blocks <= kFourGroups<TY, HD>) return start<TY, HD, 4>(a, s);
    if (blocks <= kTwoGroups<TY, HD>) return start<TY, HD, 2>(a, s);
    return start<TY, HD, 1>(a, s);
}
template <int TY>
hipError_t by_head(const PromptAttention& a, hipStream_t s) {
    switch (a.hd) {
    case 64: return by_blocks<TY, 64>(a, s);
    case 96: return by_blocks<TY, 96>(a, s);
    case 128: return by_blocks<TY, 128>(a, s);
    case 256: return by_blocks<TY, 256>(a, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_prompt_attention(const PromptAttention& a, hipStream_t s) {
    if (a.tokens == 0 || a.seqs == 0) return hipSuccess;
    return a.type == FT_F32 ? by_head<FT_F32>(a, s) : a.type == FT_F16 ? by_head<FT_F16>(a, s) : by_head<FT_BF16>(a, s);
}

}  // namespace nnrh
