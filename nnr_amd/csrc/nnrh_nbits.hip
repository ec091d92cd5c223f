// nnrh_nbits.hip -- y = a W^T + bias with 4-bit weights in blocks along K:
//   W[n][k] = (q[n][k] - zp[n][k / block]) * scale[n][k / block].
//
// q - zp is a whole number of at most 15 and so exact in 16 bits: the MFMA
// multiplies activations by q - zp, sums a block's (or 32 k's) products in
// fp32, and the block's scale enters in fp32 when they join the running sum.
// No weight is rounded. fp16 activations run on fp16 MFMAs, bf16 ones on bf16
// MFMAs; an fp32 activation is the exact sum of three bf16 pieces, one MFMA
// each.
#include "nnrh_decode.h"

namespace nnrh {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

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

// How a block reads activations: 16 bytes at a time where addresses allow it
// (whole pieces of K, or with the last one cut short), else element by element
enum AMode : int { A_WHOLE = 0, A_EDGE = 1, A_ANY = 2 };

// k .. k + 7 of a row, as they lie; elements from K on are 0
template <int TY> struct ARaw {
    u4 v[TY == FT_F32 ? 2 : 1];
    template <int AM>
    __device__ __forceinline__ void load(const void* row, int k, int K) {
        constexpr int N = TY == FT_F32 ? 4 : 8;   // elements of 16 bytes
        constexpr int ES = TY == FT_F32 ? 4 : 2;
#pragma unroll
        for (int i = 0; i < (TY == FT_F32 ? 2 : 1); ++i, k += N) {
            if constexpr (AM == A_WHOLE) {
                v[i] = *(const u4*)((const char*)row + (long long)k * ES);
            } else if constexpr (AM == A_EDGE) {   // no branch: loads stay in flight past it
                const bool in = k < K;
                const u4 x = *(const u4*)((const char*)row + (long long)(in ? k : 0) * ES);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i][j] = in ? x[j] : 0u;
            } else {
                v[i] = u4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (k + j < K) {
                        if constexpr (TY == FT_F32) v[i][j] = ((const uint32_t*)row)[k + j];
                        else v[i][j >> 1] |= (uint32_t)((const uint16_t*)row)[k + j] << (16 * (j & 1));
                    }
            }
        }
    }
    __device__ __forceinline__ AFrag<TY> frag() const {
        if constexpr (TY == FT_F32) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __builtin_bit_cast(float, (uint32_t)v[j >> 2][j & 3]);
            return split3(x);
        } else {
            AFrag<TY> f;
            f.p[0] = v[0];
            return f;
        }
    }
};

// q - zp of a word's 8 nibbles as an MFMA operand
__device__ __forceinline__ h8 weights_f16(uint32_t w, h2 off) {
    // 0x6400 | q is 1024 + q; off = 1024 + zp
    h8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const h2 v = __builtin_bit_cast(h2, ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u) - off;
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
    __device__ __forceinline__ void load(const void* p, long long at) {   // at: piece x 16 + column
        if constexpr (TY != FT_F32 && NSPP == 1) {
            w[0] = ((const uint16_t*)p)[at];
        } else {
            typedef uint32_t vec __attribute__((ext_vector_type(W)));
            const vec v = ((const vec*)p)[at];
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
// K in turn, straight from memory into registers, in rounds of D pieces each:
// a round's weights are loaded before the one before is multiplied, a piece's
// activations as those of the piece before are used up. The waves' sums meet
// in LDS.
template <int TY, int NSPP, int AM, int MT, int NT, int D>
__global__ __launch_bounds__(NB_WAVES * 64) void nbits_kernel(NbitsArgs p) {
    __shared__ f4 red[NB_WAVES][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int tile0 = blockIdx.x * NT;
    const int m0 = blockIdx.y * (16 * MT);
    constexpr int ES = TY == FT_F32 ? 4 : 2;
    const char* row[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int m = m0 + 16 * t + col;
        row[t] = (const char*)p.a + (long long)(m < p.M ? m : p.M - 1) * p.K * ES;
    }
    f4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u) acc[t][u] = f4{0, 0, 0, 0};

    const int last = p.P - 1;
    ARaw<TY> a[4][MT];
    auto load_w = [&](Stage<TY, NSPP, NT>* x, int piece) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int at = min(piece + d * NB_WAVES, last);
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                const long long pc = (long long)(tile0 + u) * p.P + at;
                x[d].w[u] = *(const u4*)(p.w + pc * 256 + lane * 4);
                x[d].sc[u].load(p.scales, pc * 16 + col);
                x[d].zp[u] = p.zp[(pc & p.zp_mask) * 16 + col];
            }
        }
    };
    auto load_a = [&](int s, int piece) {
#pragma unroll
        for (int t = 0; t < MT; ++t) a[s][t].template load<AM>(row[t], piece * NB_PK + 32 * s + 8 * g, p.K);
    };
    auto multiply = [&](const Stage<TY, NSPP, NT>& x, int next) {
        f4 part[MT][NT];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            AFrag<TY> f[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) f[t] = a[s][t].frag();
            load_a(s, next);
            constexpr int SPS = 4 / NSPP;   // MFMA steps a scale
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                const uint32_t z = (x.zp[u] >> (4 * s)) & 15;
                if constexpr (TY == FT_F16) {
                    const uint32_t o = (0x6400u + z) * 0x10001u;   // 1024 + zp, twice
                    const h8 b = weights_f16(x.w[u][s], __builtin_bit_cast(h2, o));
#pragma unroll
                    for (int t = 0; t < MT; ++t)
                        part[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            __builtin_bit_cast(h8, f[t].p[0]), b, s % SPS ? part[t][u] : f4{0, 0, 0, 0}, 0, 0, 0);
                } else {
                    const b8 b = weights_bf16(x.w[u][s], (float)z);
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        if (s % SPS == 0) part[t][u] = f4{0, 0, 0, 0};
#pragma unroll
                        for (int q = 0; q < kPieces<TY>; ++q)
                            part[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                __builtin_bit_cast(b8, f[t].p[q]), b, part[t][u], 0, 0, 0);
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
            if (NSPP == 4 && MT == 4) __builtin_amdgcn_sched_barrier(0);   // one step's block sums at a time, or registers spill
        }
    };
    Stage<TY, NSPP, NT> cur[D];
    load_w(cur, wave);
#pragma unroll
    for (int s = 0; s < 4; ++s) load_a(s, min(wave, last));
    int piece = wave;
    for (; piece + D * NB_WAVES < p.P; piece += D * NB_WAVES) {
        Stage<TY, NSPP, NT> nxt[D];
        load_w(nxt, piece + D * NB_WAVES);
#pragma unroll
        for (int d = 0; d < D; ++d) multiply(cur[d], min(piece + (d + 1) * NB_WAVES, last));
#pragma unroll
        for (int d = 0; d < D; ++d) cur[d] = nxt[d];
    }
#pragma unroll
    for (int d = 0; d < D; ++d)
        if (piece + d * NB_WAVES < p.P) multiply(cur[d], min(piece + (d + 1) * NB_WAVES, last));
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u) red[wave][t * NT + u][lane] = acc[t][u];
    __syncthreads();
    // output (row, column) sits in lane 16 (row / 4) + column, element row % 4
    const int rows = p.M - m0 < 16 * MT ? p.M - m0 : 16 * MT;
    for (int o = threadIdx.x; o < rows * (16 * NT); o += NB_WAVES * 64) {
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
        uint32_t word = 0;
        for (int j = 0; j < 8; ++j) {
            const int k = k0 + 8 * (lane >> 4) + j;
            uint32_t q = z;
            if (n < N && k < K) q = (raw[(n * nb * block + k) >> 1] >> (4 * (k & 1))) & 15;
            word |= q << (4 * ((j >> 1) + 4 * (j & 1)));
        }
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

template <int TY, int NSPP, int AM, int MT, int NT, int D>
hipError_t go(const NbitsArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)(nbits_cols(a.N) / 16 / NT), (unsigned)((a.M + 16 * MT - 1) / (16 * MT)));
    nbits_kernel<TY, NSPP, AM, MT, NT, D><<<grid, NB_WAVES * 64, 0, s>>>(a);
    return hipGetLastError();
}
template <int TY, int NSPP, int AM>
hipError_t by_size(const NbitsArgs& a, hipStream_t s) {
    if constexpr (AM == A_ANY) {
        return a.M <= 16 ? go<TY, NSPP, AM, 1, 1, 2>(a, s) : go<TY, NSPP, AM, 2, 2, 1>(a, s);
    } else {
        const int tiles = nbits_cols(a.N) / 16;
        if (a.M <= 16) return tiles >= 1024 ? go<TY, NSPP, AM, 1, 2, 2>(a, s) : go<TY, NSPP, AM, 1, 1, 4>(a, s);
        if constexpr (TY != FT_F32)   // (fp32 activations take twice the registers)
            if (a.M > 32) return go<TY, NSPP, AM, 4, 2, 1>(a, s);
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
