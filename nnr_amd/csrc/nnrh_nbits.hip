// nnrh_nbits.hip -- y = a W^T + bias with 4-bit weights in blocks along K:
//   W[n][k] = (q[n][k] - zp[n][k / block]) * scale[n][k / block].
//
// q - zp is a whole number of at most 15 and so exact in 16 bits: the MFMA
// multiplies activations by q - zp, sums a block's (or 32 k's) products in
// fp32, and the block's scale enters in fp32 when they join the running sum.
// No weight is rounded. (So that sums before the scale fit fp32, activations are to
// be below 2^117: 128 of them times 15.) fp16 activations run on fp16 MFMAs, bf16 ones on bf16
// MFMAs; an fp32 activation is the exact sum of three bf16 pieces, one MFMA
// each.
//
// Up to 64 rows a block is a few columns with all of K split over its waves:
// every weight is read once, and there are blocks for all CUs. One row x 4096
// x 8192 columns, bf16: 18 MB in 6.5 us (a copy's rate: 3.5), bound by how long
// the first loads take; 64 x 8192 x 8192, fp16: 37 MB and 8.6 GFLOP in 19 us (7.1
// and 7.5), bound by loads: each of 256 blocks reads the 64 rows whole, 1 MB, beside
// 0.14 MB of weights (vector units 30 % busy, matrix units 18). Beyond, blocks of
// up to 128 rows share activations through LDS, and a wave's weights serve all of
// them: 512 x 4096 x 4096, bf16: 17 GFLOP in 33 to 38 us over machines (14.1), bound
// by how little two waves a SIMD can put beside each other between the barriers of
// two chunks: neither vector units (45 % busy) nor matrix units (20) are full.
#include "nnrh_decode.h"

namespace nnrh {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef u4 __attribute__((aligned(2))) u4_any;

__device__ __forceinline__ float f16_f32(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
__device__ __forceinline__ float bf16_f32(uint32_t v) { return __builtin_bit_cast(float, v << 16); }
template <int TY>
__device__ __forceinline__ float load_f32(const void* p, long long i) {
    if constexpr (TY == FT_F32) return ((const float*)p)[i];
    const uint16_t v = ((const uint16_t*)p)[i];
    return TY == FT_F16 ? f16_f32(v) : bf16_f32(v);
}
template <int TY>
__device__ __forceinline__ void store_f32(void* p, long long i, float v) {
    if constexpr (TY == FT_F32) ((float*)p)[i] = v;
    else if constexpr (TY == FT_F16) ((_Float16*)p)[i] = (_Float16)v;
    else ((__bf16*)p)[i] = (__bf16)v;
}

// bf16 pieces an activation is multiplied in
template <int TY> constexpr int kPieces = TY == FT_F32 ? 3 : 1;

// Activations of one MFMA operand: 8 consecutive K of one row
template <int TY> struct AFrag { u4 p[kPieces<TY>]; };

// the upper halves of two words: their values cut to bf16
__device__ __forceinline__ uint32_t top_halves(uint32_t lo, uint32_t hi) {
    return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
}
// x[0..7] as three bf16 each: the upper 8 bits of the significand, the next 8,
// the last 8. Cutting leaves a remainder that fp32 holds exactly. An infinity
// is its first piece alone.
__device__ __forceinline__ AFrag<FT_F32> split3(const float* x) {
    AFrag<FT_F32> f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float v[2] = {x[2 * i], x[2 * i + 1]};
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            const uint32_t u0 = __builtin_bit_cast(uint32_t, v[0]), u1 = __builtin_bit_cast(uint32_t, v[1]);
            f.p[q][i] = top_halves(u0, u1);
            if (q < 2) {
                const float t0 = __builtin_bit_cast(float, u0 & 0xffff0000u);
                const float t1 = __builtin_bit_cast(float, u1 & 0xffff0000u);
                v[0] = fabsf(v[0]) == __builtin_inff() ? 0.0f : v[0] - t0;
                v[1] = fabsf(v[1]) == __builtin_inff() ? 0.0f : v[1] - t1;
            }
        }
    }
    return f;
}

// How activations are read, 16 bytes at a time: whole pieces of K at aligned
// addresses, with the last one cut short, or at any address with the last chunk
// element by element
enum AMode : int { A_WHOLE = 0, A_EDGE = 1, A_ANY = 2 };

// Activations of MT row tiles, 64 K at a time (a chunk, two MFMA steps). An MFMA
// wants neighbouring lanes to hold neighbouring rows, and loads that are
// addressed so cost the L1 an access a lane: 64 rows x 8192 x 8192 columns took
// 34 us with them, all of it accesses. So lanes load rows 16 bytes after 16
// bytes, and operands come out of the wave's own stretch of LDS, in which the
// 16-byte cells of a row are turned by its number (eight rows a read then lie
// in different banks).
template <int TY, int MT> struct Activations {
    static constexpr int ES = TY == FT_F32 ? 4 : 2;
    static constexpr int CELLS = 64 * ES / 16;              // cells of a row
    static constexpr int NL = MT * 16 * CELLS / 64;         // cells a lane
    static constexpr int BYTES = MT * 16 * 64 * ES;         // of a wave's stretch
    u4 v[NL];
    __device__ __forceinline__ static int row_of(int i) { return (i * 64 + (int)(threadIdx.x & 63)) / CELLS; }
    __device__ __forceinline__ static int cell_of() { return (threadIdx.x & 63) % CELLS; }
    // base: row m0 (uniform over the block); rows: that many from there on exist
    // (the last one is repeated). K k0 .. k0 + 63 (uniform); elements from K on
    // are 0. Offsets from uniform addresses fit 32 bits.
    template <int AM>
    __device__ __forceinline__ void load(const char* base, int rows, int k0, int K) {
        constexpr int N = 16 / ES;
        const int c = cell_of() * N;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const uint32_t row = (uint32_t)min(row_of(i), rows - 1) * (uint32_t)(K * ES);
            if constexpr (AM == A_WHOLE) {
                v[i] = *(const u4*)(base + (long long)k0 * ES + (row + (uint32_t)(c * ES)));
            } else if constexpr (AM == A_EDGE) {   // no branch: loads stay in flight past it
                const bool in = k0 + c < K;
                const u4 x = *(const u4*)(base + (row + (uint32_t)(in ? (k0 + c) * ES : 0)));
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i][j] = in ? x[j] : 0u;
            } else if (k0 + 64 <= K) {   // (16 bytes from any address: a load like others)
                v[i] = *(const u4_any*)(base + (long long)k0 * ES + (row + (uint32_t)(c * ES)));
            } else {
                u4 x = {0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const bool in = k0 + c + j < K;
                    const uint32_t at = row + (uint32_t)(in ? (k0 + c + j) * ES : 0);
                    if constexpr (TY == FT_F32) x[j] = in ? *(const uint32_t*)(base + at) : 0u;
                    else x[j >> 1] |= (in ? (uint32_t)*(const uint16_t*)(base + at) : 0u) << (16 * (j & 1));
                }
                v[i] = x;
            }
        }
    }
    __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int r = row_of(i);
            *(u4*)(lds + (r * CELLS + (cell_of() ^ (r & (CELLS - 1)))) * 16) = v[i];
        }
    }
    // operand of step s (0, 1) and row tile t, as it lies
    struct Raw { u4 v[TY == FT_F32 ? 2 : 1]; };
    __device__ __forceinline__ static Raw read(const char* lds, int s, int t) {
        const int r = 16 * t + (int)(threadIdx.x & 15), g = (threadIdx.x & 63) >> 4;
        const auto cell = [&](int c) { return *(const u4*)(lds + (r * CELLS + (c ^ (r & (CELLS - 1)))) * 16); };
        Raw x;
        if constexpr (TY == FT_F32) {
            x.v[0] = cell(8 * s + 2 * g);
            x.v[1] = cell(8 * s + 2 * g + 1);
        } else {
            x.v[0] = cell(4 * s + g);
        }
        return x;
    }
    __device__ __forceinline__ static AFrag<TY> operand(const Raw& r) {
        if constexpr (TY == FT_F32) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __builtin_bit_cast(float, (uint32_t)r.v[j >> 2][j & 3]);
            return split3(x);
        } else {
            AFrag<TY> f;
            f.p[0] = r.v[0];
            return f;
        }
    }
};

// q - zp of a word's 8 nibbles as an MFMA operand
__device__ __forceinline__ h8 weights_f16(uint32_t w, h2 off) {
    // 0x6400 | q is 1024 + q; off = 1024 + zp. (In a vector register: mask, or
    // and word are then one instruction.)
    uint32_t magic;
    asm("v_mov_b32 %0, 0x64006400" : "=v"(magic));
    h8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const h2 v = __builtin_bit_cast(h2, ((w >> (4 * i)) & 0x000f000fu) | magic) - off;
        r[2 * i] = v[0];
        r[2 * i + 1] = v[1];
    }
    return r;
}
// A byte 0 .. 15 read as e4m3 is q * 2^-9, below 8 as a subnormal: one
// instruction turns two of them into floats, and a multiply-add gives q - zp.
__device__ __forceinline__ b8 weights_bf16(uint32_t w, float zp) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;   // elements 0 4 1 5 and 2 6 3 7
    const f2 v04 = __builtin_amdgcn_cvt_pk_f32_fp8(lo, false), v15 = __builtin_amdgcn_cvt_pk_f32_fp8(lo, true);
    const f2 v26 = __builtin_amdgcn_cvt_pk_f32_fp8(hi, false), v37 = __builtin_amdgcn_cvt_pk_f32_fp8(hi, true);
    float v[8] = {v04[0], v15[0], v26[0], v37[0], v04[1], v15[1], v26[1], v37[1]};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __builtin_fmaf(v[i], 512.0f, -zp);
    u4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r[i] = top_halves(__builtin_bit_cast(uint32_t, v[2 * i]), __builtin_bit_cast(uint32_t, v[2 * i + 1]));
    return __builtin_bit_cast(b8, r);
}

constexpr int NB_WAVES = 8;

// scales of a piece and column, as they lie
template <int TY, int NSPP> struct Scales {
    static constexpr int W = TY == FT_F32 ? NSPP : (NSPP + 1) / 2;   // words
    uint32_t w[W];
    __device__ __forceinline__ void load(const char* p, uint32_t col) {   // p: the piece's
        if constexpr (TY != FT_F32 && NSPP == 1) {
            w[0] = *(const uint16_t*)(p + col * 2);
        } else {
            typedef uint32_t vec __attribute__((ext_vector_type(W)));
            const vec v = *(const vec*)(p + col * (uint32_t)sizeof(vec));
            if constexpr (W == 1) w[0] = __builtin_bit_cast(uint32_t, v);
            else
#pragma unroll
                for (int i = 0; i < W; ++i) w[i] = v[i];
        }
    }
    __device__ __forceinline__ float get(int s) const {
        if constexpr (TY == FT_F32) return __builtin_bit_cast(float, w[s]);
        const uint32_t v = w[s / 2] >> (16 * (s & 1)) & 0xffffu;
        return TY == FT_F16 ? f16_f32((uint16_t)v) : bf16_f32(v);
    }
};

// The weights of one piece of K, loaded well before they are used
template <int TY, int NSPP, int NT> struct Stage {
    u4 w[NT];
    Scales<TY, NSPP> sc[NT];
    uint32_t zp[NT];
};

// One block: MT x 16 rows, NT x 16 columns, all of K. Its waves take pieces of
// K in turn, weights straight from memory into registers, asked for D pieces
// ahead, activations through LDS, asked for a chunk ahead. The waves' sums meet
// in LDS. DIR (a row or two): operands straight from memory like the weights;
// lanes that repeat a row cost no accesses of their own (1 x 4096 x 8192 bf16
// 6.6 us, through LDS 7.7; 16 rows 10.7 and 8.1).
template <int TY, int NSPP, int AM, int MT, int NT, int D, bool DIR>
__global__ __launch_bounds__(NB_WAVES * 64) void nbits_kernel(NbitsArgs p) {
    typedef Activations<TY, MT> Act;
    constexpr int sums = NB_WAVES * MT * NT * 1024, acts = NB_WAVES * Act::BYTES;
    __shared__ __attribute__((aligned(16))) char lds[sums > acts ? sums : acts];
    f4(*red)[MT * NT][64] = (f4(*)[MT * NT][64])lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15;
    const int tile0 = blockIdx.x * NT;
    const int m0 = blockIdx.y * (16 * MT);
    char* const mine = lds + wave * Act::BYTES;
    const char* const base = (const char*)p.a + (long long)m0 * p.K * Act::ES;
    const int rows = p.M - m0;
    f4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u) acc[t][u] = f4{0, 0, 0, 0};

    const int last = p.P - 1;
    Stage<TY, NSPP, NT> st[D];
    typename Act::Raw dir[DIR ? D : 1][4];
    Act act;
    auto load_w = [&](int d, int piece) {
        Stage<TY, NSPP, NT>& x = st[d];
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            const long long pc = (long long)(tile0 + u) * p.P + piece;
            x.w[u] = *(const u4*)((const char*)p.w + pc * 1024 + (uint32_t)(lane * 16));
            x.sc[u].load((const char*)p.scales + pc * (16 * NSPP * Act::ES), (uint32_t)col);
            x.zp[u] = *(const uint16_t*)((const char*)p.zp + (pc & p.zp_mask) * 32 + (uint32_t)(col * 2));
        }
        if constexpr (DIR)
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int i = 0; i < (TY == FT_F32 ? 2 : 1); ++i) {
                    const int k = piece * NB_PK + 32 * s + 8 * (lane >> 4) + 4 * i;   // (i: fp32 only)
                    const uint32_t row = (uint32_t)min(col, rows - 1) * (uint32_t)(p.K * Act::ES);
                    if constexpr (AM == A_WHOLE) {
                        dir[d][s].v[i] = *(const u4*)(base + (row + (uint32_t)(k * Act::ES)));
                    } else {
                        const bool in = k < p.K;
                        const u4 v = *(const u4*)(base + (row + (uint32_t)(in ? k * Act::ES : 0)));
#pragma unroll
                        for (int j = 0; j < 4; ++j) dir[d][s].v[i][j] = in ? v[j] : 0u;
                    }
                }
    };
    // Operands of the chunk at hand are in registers when its turn comes; the next
    // one's go through LDS meanwhile, and the one after is on its way.
    typename Act::Raw f[2][2][MT];
    auto pass = [&](int to, int k) {   // act -> f[to]; act <- the chunk at k
        act.store(mine);
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_sched_barrier(0);   // loads stay where they are asked for
        act.template load<AM>(base, rows, k, p.K);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int t = 0; t < MT; ++t) f[to][s][t] = Act::read(mine, s, t);
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    auto multiply = [&](int d, int next) {
        const Stage<TY, NSPP, NT>& x = st[d];
        constexpr int SPS = 4 / NSPP;   // MFMA steps a scale
        f4 part[MT][NT];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (!DIR) pass(h ^ 1, next * NB_PK + 64 * h);
#pragma unroll
            for (int s = 2 * h; s < 2 * h + 2; ++s) {
                AFrag<TY> fa[MT];
#pragma unroll
                for (int t = 0; t < MT; ++t) fa[t] = Act::operand(DIR ? dir[DIR ? d : 0][s] : f[h][s & 1][t]);
#pragma unroll
                for (int u = 0; u < NT; ++u) {
                    const uint32_t z = (x.zp[u] >> (4 * s)) & 15;
                    if constexpr (TY == FT_F16) {
                        const uint32_t o = (0x6400u + z) * 0x10001u;   // 1024 + zp, twice
                        const h8 b = weights_f16(x.w[u][s], __builtin_bit_cast(h2, o));
#pragma unroll
                        for (int t = 0; t < MT; ++t)
                            part[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                __builtin_bit_cast(h8, fa[t].p[0]), b, s % SPS ? part[t][u] : f4{0, 0, 0, 0}, 0, 0, 0);
                    } else {
                        const b8 b = weights_bf16(x.w[u][s], (float)z);
#pragma unroll
                        for (int t = 0; t < MT; ++t) {
                            if (s % SPS == 0) part[t][u] = f4{0, 0, 0, 0};
#pragma unroll
                            for (int q = 0; q < kPieces<TY>; ++q)
                                part[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, fa[t].p[q]), b,
                                                                                     part[t][u], 0, 0, 0);
                        }
                    }
                    if (s % SPS == SPS - 1) {
                        const float sc = x.sc[u].get(s / SPS);
#pragma unroll
                        for (int t = 0; t < MT; ++t)
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[t][u][i] = __builtin_fmaf(part[t][u][i], sc, acc[t][u][i]);
                    }
                }
            }
        }
    };
    if constexpr (!DIR) act.template load<AM>(base, rows, min(wave, last) * NB_PK, p.K);
#pragma unroll
    for (int d = 0; d < D; ++d) load_w(d, min(wave + d * NB_WAVES, last));
    if constexpr (!DIR) pass(0, min(wave, last) * NB_PK + 64);
    int piece = wave;
    for (; piece + D * NB_WAVES < p.P; piece += D * NB_WAVES)
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int at = piece + d * NB_WAVES;
            __builtin_amdgcn_sched_barrier(0);
            multiply(d, min(at + NB_WAVES, last));
            __builtin_amdgcn_sched_barrier(0);
            load_w(d, min(at + D * NB_WAVES, last));
        }
#pragma unroll
    for (int d = 0; d < D; ++d) {
        const int at = piece + d * NB_WAVES;
        if (at < p.P) multiply(d, min(at + NB_WAVES, last));
    }
    __syncthreads();   // every wave is done with its stretch
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u) red[wave][t * NT + u][lane] = acc[t][u];
    __syncthreads();
    // output (row, column) sits in lane 16 (row / 4) + column, element row % 4
    const int nr = min(rows, 16 * MT);
    for (int o = threadIdx.x; o < nr * (16 * NT); o += NB_WAVES * 64) {
        const int r = o / (16 * NT), c = o % (16 * NT);
        const int n = tile0 * 16 + c;
        if (n >= p.N) continue;
        const int t = (r >> 4) * NT + (c >> 4), l = (c & 15) + 16 * ((r & 15) >> 2);
        float v = 0.0f;
#pragma unroll
        for (int q = 0; q < NB_WAVES; ++q) v += ((const float*)&red[q][t][l])[r & 3];
        if (p.bias) v += load_f32<TY>(p.bias, n);
        store_f32<TY>(p.y, (long long)(m0 + r) * p.N + n, v);
    }
}

// Many rows. One block: MT x 16 rows, WN x NT x 16 columns; its waves are WN
// columns groups times 8 / WN groups that take pieces of K in turn. Waves of one
// K group share its activations: each loads a part of a chunk (64 K) and stores
// it into LDS as 16-bit operands (fp32 as its three bf16 pieces), beside the
// chunk that is being multiplied; one barrier a chunk.
template <int TY, int NSPP, int AM, int MT, int NT, int WN>
__global__ __launch_bounds__(NB_WAVES * 64) void nbits_tile_kernel(NbitsArgs p) {
    constexpr int KG = NB_WAVES / WN, NP = kPieces<TY>, ES = TY == FT_F32 ? 4 : 2, D = 2;
    constexpr int PLANE = MT * 16 * 128;                    // bytes of 64 K of the rows, 16 bits each
    constexpr int BUF = NP * PLANE;
    constexpr int CELLS = 8, NL = MT * 16 * CELLS / (64 * WN);   // cells of 8 elements: a row's, a lane's
    constexpr int V = TY == FT_F32 ? 2 : 1;                 // 16-byte loads a cell
    constexpr int acts = 2 * KG * BUF, sums = NB_WAVES * MT * NT * 1024;
    __shared__ __attribute__((aligned(16))) char lds[acts > sums ? acts : sums];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4, wn = wave % WN, kg = wave / WN;
    const int tile0 = (blockIdx.x * WN + wn) * NT;
    const int m0 = blockIdx.y * (16 * MT), rows = p.M - m0;
    const char* const base = (const char*)p.a + (long long)m0 * p.K * ES;
    const int last = p.P - 1, rounds = (p.P + KG - 1) / KG;
    char* const mine = lds + kg * BUF;                      // buffer b: mine + b KG BUF

    u4 act[NL][V];
    auto load_a = [&](int k0) {   // the wave's cells of the chunk at k0
        const int k = k0 + (lane & 7) * 8;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const uint32_t row = (uint32_t)min(((i * WN + wn) * 64 + lane) / CELLS, rows - 1) * (uint32_t)(p.K * ES);
#pragma unroll
            for (int h = 0; h < V; ++h) {
                const int kk = k + 4 * h;   // (h: fp32 only)
                if constexpr (AM == A_WHOLE) {
                    act[i][h] = *(const u4*)(base + (row + (uint32_t)(kk * ES)));
                } else if constexpr (AM == A_ANY) {
                    if (k0 + 64 <= p.K) {
                        act[i][h] = *(const u4_any*)(base + (row + (uint32_t)(kk * ES)));
                    } else {
                        u4 x = {0, 0, 0, 0};
#pragma unroll
                        for (int j = 0; j < 16 / ES; ++j) {
                            const bool in = kk + j < p.K;
                            const uint32_t at = row + (uint32_t)(in ? (kk + j) * ES : 0);
                            if constexpr (TY == FT_F32) x[j] = in ? *(const uint32_t*)(base + at) : 0u;
                            else x[j >> 1] |= (in ? (uint32_t)*(const uint16_t*)(base + at) : 0u) << (16 * (j & 1));
                        }
                        act[i][h] = x;
                    }
                } else {
                    const bool in = kk < p.K;
                    const u4 x = *(const u4*)(base + (row + (uint32_t)(in ? kk * ES : 0)));
#pragma unroll
                    for (int j = 0; j < 4; ++j) act[i][h][j] = in ? x[j] : 0u;
                }
            }
        }
    };
    auto store_a = [&](int b) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int r = ((i * WN + wn) * 64 + lane) / CELLS;
            char* to = mine + b * (KG * BUF) + (r * CELLS + ((lane & 7) ^ (r & 7))) * 16;
            if constexpr (TY == FT_F32) {
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = __builtin_bit_cast(float, (uint32_t)act[i][j >> 2][j & 3]);
                const AFrag<TY> f = split3(x);
#pragma unroll
                for (int q = 0; q < NP; ++q) *(u4*)(to + q * PLANE) = f.p[q];
            } else {
                *(u4*)to = act[i][0];
            }
        }
    };
    Stage<TY, NSPP, NT> st[D];
    auto load_w = [&](int d, int piece) {
        Stage<TY, NSPP, NT>& x = st[d];
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            const long long pc = (long long)(tile0 + u) * p.P + piece;
            x.w[u] = *(const u4*)((const char*)p.w + pc * 1024 + (uint32_t)(lane * 16));
            x.sc[u].load((const char*)p.scales + pc * (16 * NSPP * ES), (uint32_t)col);
            x.zp[u] = *(const uint16_t*)((const char*)p.zp + (pc & p.zp_mask) * 32 + (uint32_t)(col * 2));
        }
    };
    f4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u) acc[t][u] = f4{0, 0, 0, 0};
    constexpr int SPS = 4 / NSPP;   // MFMA steps a scale
    f4 part[MT][NT];
    auto half = [&](int d, int h) {   // buffer h
        const Stage<TY, NSPP, NT>& x = st[d];
        const char* from = mine + h * (KG * BUF);
#pragma unroll
        for (int s = 2 * h; s < 2 * h + 2; ++s) {
            u4 f[MT][NP];
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int q = 0; q < NP; ++q) {
                    const int r = 16 * t + col;
                    f[t][q] = *(const u4*)(from + q * PLANE + (r * CELLS + ((4 * (s & 1) + g) ^ (r & 7))) * 16);
                }
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                const uint32_t z = (x.zp[u] >> (4 * s)) & 15;
                h8 bh;
                b8 bb;
                if constexpr (TY == FT_F16) bh = weights_f16(x.w[u][s], __builtin_bit_cast(h2, (0x6400u + z) * 0x10001u));
                else bb = weights_bf16(x.w[u][s], (float)z);
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    f4 c = s % SPS ? part[t][u] : f4{0, 0, 0, 0};
#pragma unroll
                    for (int q = 0; q < NP; ++q) {
                        if constexpr (TY == FT_F16)
                            c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, f[t][q]), bh, c, 0, 0, 0);
                        else
                            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, f[t][q]), bb, c, 0, 0, 0);
                    }
                    part[t][u] = c;
                }
                if (s % SPS == SPS - 1) {
                    const float sc = x.sc[u].get(s / SPS);
#pragma unroll
                    for (int t = 0; t < MT; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[t][u][i] = __builtin_fmaf(part[t][u][i], sc, acc[t][u][i]);
                }
            }
        }
    };
    const auto piece_of = [&](int r) { return min(kg + r * KG, last); };
    load_a(piece_of(0) * NB_PK);
#pragma unroll
    for (int d = 0; d < D; ++d) load_w(d, piece_of(d));
    store_a(0);
    load_a(piece_of(0) * NB_PK + 64);
    __syncthreads();
    auto round = [&](int d, int r) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            store_a(h ^ 1);
            __builtin_amdgcn_sched_barrier(0);
            load_a(piece_of(r + 1) * NB_PK + 64 * h);
            __builtin_amdgcn_sched_barrier(0);
            if (kg + r * KG < p.P) half(d, h);
            __syncthreads();
        }
        load_w(d, piece_of(r + D));
    };
    for (int r = 0; r < rounds; r += D)
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (r + d < rounds) round(d, r + d);

    f4(*red)[MT * NT][64] = (f4(*)[MT * NT][64])lds;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u) red[wave][t * NT + u][lane] = acc[t][u];
    __syncthreads();
    constexpr int COLS = WN * NT * 16;
    const int nr = min(rows, 16 * MT);
    for (int o = threadIdx.x; o < nr * COLS; o += NB_WAVES * 64) {
        const int r = o / COLS, c = o % COLS, w = c / (NT * 16);
        const int n = blockIdx.x * COLS + c;
        if (n >= p.N) continue;
        const int t = (r >> 4) * NT + (c % (NT * 16) >> 4), l = (c & 15) + 16 * ((r & 15) >> 2);
        float v = 0.0f;
#pragma unroll
        for (int q = 0; q < KG; ++q) v += ((const float*)&red[q * WN + w][t][l])[r & 3];
        if (p.bias) v += load_f32<TY>(p.bias, n);
        store_f32<TY>(p.y, (long long)(m0 + r) * p.N + n, v);
    }
}

// One thread a lane's 16 bytes of a piece; lanes 0..15 also its scales and zero points
__global__ __launch_bounds__(256) void nbits_pack_kernel(const uint8_t* raw, const void* raw_scales,
                                                         const uint8_t* raw_zp, int N, int K, int block, int nb,
                                                         int nspp, int es, int P, long long lanes, uint32_t* w,
                                                         void* scales, uint16_t* zp) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= lanes) return;
    const int lane = (int)(i & 63);
    const long long pc = i >> 6, tile = pc / P;
    const int piece = (int)(pc - tile * P);
    const long long n = tile * 16 + (lane & 15);
    uint32_t zps = 0;
    for (int s = 0; s < 4; ++s) {
        const int k0 = piece * NB_PK + 32 * s;   // one block: its size is a multiple of 32
        const int b = k0 / block;
        uint32_t z = 8;
        if (raw_zp && n < N && k0 < K) z = (raw_zp[n * ((nb + 1) / 2) + (b >> 1)] >> (4 * (b & 1))) & 15;
        zps |= z << (4 * s);
        // eight neighbouring nibbles (behind K a block's filling, which meets zeros)
        const int k = k0 + 8 * (lane >> 4);
        uint32_t q = z * 0x11111111u;
        if (n < N && k < nb * block) q = *(const uint32_t*)(raw + ((n * nb * block + k) >> 1));
        uint32_t word = 0;
        for (int j = 0; j < 8; ++j) word |= (q >> (4 * j) & 15) << (4 * ((j >> 1) + 4 * (j & 1)));
        w[i * 4 + s] = word;
    }
    if (lane >= 16) return;
    if (raw_zp || pc == 0) zp[pc * 16 + lane] = (uint16_t)zps;   // without zero points one piece's serve all
    for (int s = 0; s < nspp; ++s) {
        const int k0 = piece * NB_PK + s * (NB_PK / nspp);
        const bool in = n < N && k0 < K;
        const long long from = n * nb + k0 / block, to = (pc * 16 + lane) * nspp + s;
        if (es == 4) ((uint32_t*)scales)[to] = in ? ((const uint32_t*)raw_scales)[from] : 0u;
        else ((uint16_t*)scales)[to] = in ? ((const uint16_t*)raw_scales)[from] : (uint16_t)0;
    }
}

template <int TY, int NSPP, int AM, int MT, int NT, int D, bool DIR = false>
hipError_t go(const NbitsArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)(nbits_cols(a.N) / 16 / NT), (unsigned)((a.M + 16 * MT - 1) / (16 * MT)));
    nbits_kernel<TY, NSPP, AM, MT, NT, D, DIR><<<grid, NB_WAVES * 64, 0, s>>>(a);
    return hipGetLastError();
}
template <int TY, int NSPP, int AM, int MT, int NT, int WN>
hipError_t go_tile(const NbitsArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)((nbits_cols(a.N) / 16 + NT * WN - 1) / (NT * WN)), (unsigned)((a.M + 16 * MT - 1) / (16 * MT)));
    nbits_tile_kernel<TY, NSPP, AM, MT, NT, WN><<<grid, NB_WAVES * 64, 0, s>>>(a);
    return hipGetLastError();
}
template <int TY, int NSPP, int AM>
hipError_t by_size(const NbitsArgs& a, hipStream_t s) {
    constexpr bool wide = TY == FT_F32;   // activations take twice the registers
    const int cols = nbits_cols(a.N);
    const auto blocks = [&](int m, int n) { return (long long)((a.M + m - 1) / m) * (cols / n); };
    if (a.M > 64) {
        // Blocks of shared rows where they fill the chip (bf16, K 4096, blocks of
        // 32, one machine: 512 x 4096 38 us, K split over waves 52; 256 x 4096 33 and
        // 25); those of 128 columns where that is so twice over (4096 x 4096 213 us,
        // 64 columns of 128 rows 251). Rows of any address too (512 x 4095 x 4096
        // bf16 54 us, K split over waves 86; fp32 73 and 156).
        if (blocks(64, 128) >= (wide ? 192 : 512)) return go_tile<TY, NSPP, AM, 4, 2, 4>(a, s);
        if constexpr (!wide)
            if (blocks(128, 64) >= 192)   // (column tiles side by side spill with few scales: 41 us, 35)
                return go_tile<TY, NSPP, AM, 8, NSPP == 4 ? 2 : 1, NSPP == 4 ? 2 : 4>(a, s);
    }
    if constexpr (AM == A_ANY) {
        return a.M <= 16 ? go<TY, NSPP, AM, 1, 1, 2>(a, s) : go<TY, NSPP, AM, 2, 2, 1>(a, s);
    } else {
        if (a.M <= 2)
            return cols >= 16384 ? go<TY, NSPP, AM, 1, 2, wide ? 2 : 3, true>(a, s) : go<TY, NSPP, AM, 1, 1, wide ? 3 : 4, true>(a, s);
        if (a.M <= 16) return cols >= 16384 ? go<TY, NSPP, AM, 1, 2, 3>(a, s) : go<TY, NSPP, AM, 1, 1, 4>(a, s);
        if constexpr (!wide)
            if (a.M > 32) return go<TY, NSPP, AM, 4, 2, 2>(a, s);
        return go<TY, NSPP, AM, 2, 2, 2>(a, s);
    }
}
template <int TY, int NSPP>
hipError_t by_loads(const NbitsArgs& a, hipStream_t s) {
    const int es = float_type_size(a.type);
    if ((long long)a.K * es % 16 || ((uintptr_t)a.a & 15)) return by_size<TY, NSPP, A_ANY>(a, s);
    return a.K % NB_PK ? by_size<TY, NSPP, A_EDGE>(a, s) : by_size<TY, NSPP, A_WHOLE>(a, s);
}
template <int TY>
hipError_t by_scales(const NbitsArgs& a, hipStream_t s) {
    return a.nspp == 4 ? by_loads<TY, 4>(a, s) : a.nspp == 2 ? by_loads<TY, 2>(a, s) : by_loads<TY, 1>(a, s);
}

}  // namespace

hipError_t launch_nbits(const NbitsArgs& a, hipStream_t s) {
    if (a.M == 0) return hipSuccess;
    return a.type == FT_F32 ? by_scales<FT_F32>(a, s)
         : a.type == FT_F16 ? by_scales<FT_F16>(a, s) : by_scales<FT_BF16>(a, s);
}

hipError_t launch_nbits_pack(const uint8_t* raw, const void* raw_scales, const uint8_t* raw_zp, int N, int K,
                             int block, int type, uint32_t* w, void* scales, uint16_t* zp, hipStream_t s) {
    const int P = nbits_pieces(K), nb = (K + block - 1) / block;
    const long long lanes = (long long)(nbits_cols(N) / 16) * P * 64;
    nbits_pack_kernel<<<(unsigned)((lanes + 255) / 256), 256, 0, s>>>(
        raw, raw_scales, raw_zp, N, K, block, nb, nbits_nspp(block), float_type_size(type), P, lanes, w, scales, zp);
    return hipGetLastError();
}

}  // namespace nnrh
