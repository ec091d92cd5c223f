// nnrh_kvcache.hip -- writing tokens into the quantized key/value cache and
// reading them back. A group x of a token's elements (a head's at 8 bits, 32
// at 4 bits) is held as
//   scale = bf16(max |x| / L), code = clamp(rint(x / scale), -L, L), L = 127 or 7.
// The scale is rounded to bf16 before the codes are formed, so rounding it
// costs no accuracy beyond a step 2^-9 wider; both quotients are correctly
// rounded fp32 divisions, which decide every border between two codes (or two
// scales) as the exact quotient would: a border times the divisor has 16 bits,
// and an fp32 dividend beside it is at least 2^-24 of itself away.
// Elements that are not finite do not enter the maximum; a NaN is held as 0
// and an infinity as +-L. A scale below the normal floats is 0, and so are its
// codes.
#include "nnrh_decode.h"

namespace nnrh {
namespace {

typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kLdsRow = 40;   // bytes of an element's 32 tokens, padded

template <int TY>
__device__ __forceinline__ void load8(const void* p, long long i, float* v) {
    if constexpr (TY == FT_F32) {
        const f4 a = *(const f4*)((const float*)p + i), b = *(const f4*)((const float*)p + i + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
    } else {
        const u4 a = *(const u4*)((const uint16_t*)p + i);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t h = (a[j >> 1] >> (16 * (j & 1))) & 0xffffu;
            v[j] = TY == FT_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h) : __builtin_bit_cast(float, h << 16);
        }
    }
}
template <int TY>
__device__ __forceinline__ void store8(void* p, long long i, const float* v) {
    if constexpr (TY == FT_F32) {
        *(f4*)((float*)p + i) = f4{v[0], v[1], v[2], v[3]};
        *(f4*)((float*)p + i + 4) = f4{v[4], v[5], v[6], v[7]};
    } else {
        u4 a;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t lo, hi;
            if constexpr (TY == FT_F16) {
                lo = __builtin_bit_cast(uint16_t, (_Float16)v[2 * j]);
                hi = __builtin_bit_cast(uint16_t, (_Float16)v[2 * j + 1]);
            } else {
                lo = __builtin_bit_cast(uint16_t, (__bf16)v[2 * j]);
                hi = __builtin_bit_cast(uint16_t, (__bf16)v[2 * j + 1]);
            }
            a[j] = lo | (hi << 16);
        }
        *(u4*)((uint16_t*)p + i) = a;
    }
}

// Which tokens a wave handles: tile `x` of the positions of sequence b's newest
// seq tokens, position lens[b] - seq + token. False: no memory behind the tile.
struct TileAt {
    long long pos;      // of the tile's first token
    long long p0;       // of token 0
    long long end;      // positions from here on hold nothing
    uint8_t* part;      // the head's part of the page; NULL: none
    int in_page;        // tile within the page
};
__device__ __forceinline__ TileAt tile_at(const KvCache& c, const KvTokens& t, int b, int head, int x) {
    TileAt r;
    const long long len = t.lens[b], cap = (long long)t.max_pages * c.page_size;
    r.p0 = len - t.seq;
    r.pos = ((r.p0 >> 5) + x) * 32;
    r.end = len < cap ? len : cap;
    r.part = nullptr;
    r.in_page = 0;
    if (r.pos >= 0 && r.pos < r.end) {
        const int pi = (int)r.pos >> (31 - __builtin_clz((unsigned)c.page_size));
        const int id = t.table[(long long)b * t.max_pages + pi];
        if (id >= 0 && id < c.num_pages) {
            r.part = c.data + ((long long)id * c.heads + head) * kv_head_bytes(c.page_size, c.hd, c.bits);
            r.in_page = ((int)r.pos & (c.page_size - 1)) / 32;
        }
    }
    return r;
}
// tokens of a tile that hold something and are among the call's seq
__device__ __forceinline__ bool token_in(const TileAt& w, int seq, int t) {
    const long long p = w.pos + t;
    return w.part && p >= 0 && p >= w.p0 && p < w.end && p < w.p0 + seq;
}

__device__ __forceinline__ float finite_abs(float v) {
    const float a = fabsf(v);
    return a < __builtin_inff() ? a : 0.0f;
}
__device__ __forceinline__ float across_groups_max(float m) {   // lanes of one token
    m = fmaxf(m, __shfl_xor(m, 16));
    return fmaxf(m, __shfl_xor(m, 32));
}
__device__ __forceinline__ float scale_of(float top, float limit) {
    const float s = (float)(__bf16)(top / limit);
    return s >= 1.17549435e-38f ? s : 0.0f;
}
__device__ __forceinline__ int code_of(float v, float s, float limit) {
    if (s == 0.0f || !(v == v)) return 0;
    return (int)fminf(fmaxf(rintf(v / s), -limit), limit);
}
// Codes + zero of 8 elements, a byte each: the quotient by way of the scale's
// reciprocal, which is off by 2e-5 at most (127 x 2^-23 x 1.5), decides all that
// lie further than that from a border; the rest, and what is not finite, take
// the division. (A finite element's code needs no clamp: top / scale is below
// L + 1/2, as scale is top / L within 2^-9.)
template <int BITS>
__device__ __forceinline__ u2 codes_of(const float* v, float s, float inv) {
    constexpr float limit = BITS == 8 ? 127.0f : 7.0f, zero = BITS == 8 ? 128.0f : 8.0f;
    float c[8];
    bool near = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float t = v[j] * inv;
        c[j] = rintf(t);
        near |= !(fabsf(t - c[j]) < 0.4999f);
    }
    if (__any(near)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = (float)code_of(v[j], s, limit);
    }
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        lo = __builtin_amdgcn_cvt_pk_u8_f32(c[j] + zero, j, lo);
        hi = __builtin_amdgcn_cvt_pk_u8_f32(c[4 + j] + zero, j, hi);
    }
    return u2{lo, hi};
}
// eight codes, a byte each, as a word of nibbles (j even: nibble j / 2, j odd: 4 + j / 2; turned)
__device__ __forceinline__ uint32_t pack_nibbles(u2 q) {
    // bytes 0 4 1 5 below bytes 2 6 3 7
    const uint32_t x = __builtin_amdgcn_perm(q[1], q[0], 0x05010400u), y = __builtin_amdgcn_perm(q[1], q[0], 0x07030602u);
    return kv_turn(x | y << 4);
}
template <int BITS>
__device__ __forceinline__ int scale_slot(int values, int t) { return BITS == 4 && !values ? kv_pair(t) : kv_slot(t); }

// One block a (tile of 32 positions, head, sequence, keys or values), one wave
// 32 elements of it: a block of the layout. Lanes read 8 neighbouring elements of
// a token, form scales (at 8 bits with the other waves' maxima) and codes, and
// store keys as they are; values pass through LDS, where an element's tokens come
// together. A tile whose tokens are not all written is merged with what it holds:
// nothing else of the launch has this tile. (A wave for all of a head's elements
// ran 2000 instructions once, fetched for it: 3 x 1900 tokens of 8 x 128 bf16
// elements at 4 bits 18.6 us; so, 14.8, and 10.1 to read them, 30 MB each way or
// 5.8 us at a copy's rate.)
template <int TY, int BITS, int HD>
__global__ __launch_bounds__(HD * 2) void kv_write_kernel(KvCache c, KvTokens t) {
    constexpr int NC = HD / 32;
    constexpr float limit = BITS == 8 ? 127.0f : 7.0f;
    constexpr int BB = BITS == 8 ? 1024 : 512;   // bytes of a block
    typedef uint32_t vec __attribute__((ext_vector_type(BITS == 8 ? 4 : 2)));   // a lane's bytes of it
    __shared__ __attribute__((aligned(16))) uint8_t lds[HD * kLdsRow];
    __shared__ float tops[NC][32];
    const int lane = threadIdx.x & 63, k = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    const int values = blockIdx.y & 1, head = blockIdx.y >> 1, b = blockIdx.z;
    const TileAt w = tile_at(c, t, b, head, blockIdx.x);
    if (!w.part) return;
    const void* src = values ? t.v : t.k;
    const long long cb = kv_codes_bytes(c.page_size, HD, BITS);
    uint8_t* block = w.part + (values ? cb : 0) + ((long long)w.in_page * NC + k) * BB;
    bool in[2];   // this lane's tokens
    float x[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int tok = (lane & 15) + 16 * h;
        in[h] = token_in(w, t.seq, tok);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[h][j] = 0.0f;
        if (in[h])
            load8<TY>(src, (long long)b * t.bstride + (w.pos + tok - w.p0) * t.tstride + (long long)head * HD + 32 * k + 8 * g,
                      x[h]);
    }
    // values: what this lane's bytes hold beside the new tokens (slots 8 g .. 8 g + 7)
    uint32_t keep = 0;   // bit j: slot 8 g + j is not written
    vec old;
    if (values) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (!token_in(w, t.seq, 4 * g + (j & 3) + 16 * (j >> 2))) keep |= 1u << j;
        if (keep != 0 && keep != 0xff) old = *(const vec*)(block + lane * sizeof(vec));
    }
    float m[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        m[h] = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m[h] = fmaxf(m[h], finite_abs(x[h][j]));
        m[h] = across_groups_max(m[h]);
        if (BITS == 8 && g == 0) tops[k][(lane & 15) + 16 * h] = m[h];
    }
    if constexpr (BITS == 8) {
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < NC; ++i) m[h] = fmaxf(m[h], tops[i][(lane & 15) + 16 * h]);
    }
    __bf16* scales = (__bf16*)(w.part + 2 * cb) + (values ? (long long)c.page_size * kv_groups(HD, BITS) : 0);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int tok = (lane & 15) + 16 * h;
        const float sc = scale_of(m[h], limit), inv = sc > 0.0f ? 1.0f / sc : 0.0f;
        if (in[h] && g == 0 && (BITS == 4 || k == 0))
            scales[(long long)(BITS == 8 ? 0 : k) * c.page_size + w.in_page * 32 + scale_slot<BITS>(values, tok)] = (__bf16)sc;
        const u2 q = codes_of<BITS>(x[h], sc, inv);
        if (values) {
            uint8_t* to = lds + (32 * k + 8 * g) * kLdsRow + kv_slot(tok);
#pragma unroll
            for (int j = 0; j < 8; ++j) to[j * kLdsRow] = (uint8_t)(q[j >> 2] >> (8 * (j & 3)));
        } else if (in[h]) {
            if constexpr (BITS == 8) *(u2*)(block + lane * 16 + h * 8) = q;
            else *(uint32_t*)(block + lane * 8 + h * 4) = pack_nibbles(q);
        }
    }
    if (!values) return;
    __syncthreads();
    if (keep == 0xff) return;
    u2 e[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) e[h] = *(const u2*)(lds + (32 * k + (lane & 15) + 16 * h) * kLdsRow + 8 * g);
    vec out, mask;
    if constexpr (BITS == 8) {
        out = vec{e[0][0], e[0][1], e[1][0], e[1][1]};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            mask[i] = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (keep >> (4 * (i & 1) + j) & 1) mask[i] |= 0xffu << (8 * j);
        }
    } else {
        uint32_t mm = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (keep >> j & 1) mm |= 15u << (4 * ((j >> 1) + 4 * (j & 1)));
        out = vec{pack_nibbles(e[0]), pack_nibbles(e[1])};
        mask = vec{kv_turn(mm), kv_turn(mm)};
    }
    if (keep) out = (out & ~mask) | (old & mask);
    *(vec*)(block + lane * sizeof(vec)) = out;
}

// The same block the other way; a position that holds no token reads as zeros.
template <int TY, int BITS, int HD>
__global__ __launch_bounds__(HD * 2) void kv_read_kernel(KvCache c, KvTokens t) {
    constexpr int NC = HD / 32;
    constexpr int zero = BITS == 8 ? 128 : 8;
    constexpr int BB = BITS == 8 ? 1024 : 512;
    __shared__ __attribute__((aligned(16))) uint8_t lds[HD * kLdsRow];
    const int lane = threadIdx.x & 63, k = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    const int values = blockIdx.y & 1, head = blockIdx.y >> 1, b = blockIdx.z;
    const TileAt w = tile_at(c, t, b, head, blockIdx.x);
    const long long cb = kv_codes_bytes(c.page_size, HD, BITS);
    u2 e[2] = {{0, 0}, {0, 0}};   // codes of a half's 8 elements or tokens, a byte each
    float sc[2] = {0.0f, 0.0f};
    bool in[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) in[h] = token_in(w, t.seq, (lane & 15) + 16 * h);
    if (w.part) {
        const uint8_t* block = w.part + (values ? cb : 0) + ((long long)w.in_page * NC + k) * BB;
        const __bf16* scales = (const __bf16*)(w.part + 2 * cb) + (values ? (long long)c.page_size * kv_groups(HD, BITS) : 0);
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (in[h])
                sc[h] = (float)scales[(long long)(BITS == 8 ? 0 : k) * c.page_size + w.in_page * 32 +
                                      scale_slot<BITS>(values, (lane & 15) + 16 * h)];
        if constexpr (BITS == 8) {
            const u4 v = *(const u4*)(block + lane * 16);
            e[0] = u2{v[0], v[1]};
            e[1] = u2{v[2], v[3]};
        } else {
            const u2 v = *(const u2*)(block + lane * 8);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // bytes 0 4 1 5 and 2 6 3 7
                const uint32_t n = kv_unturn(v[h]), x = n & 0x0f0f0f0fu, y = n >> 4 & 0x0f0f0f0fu;
                e[h] = u2{__builtin_amdgcn_perm(y, x, 0x06040200u), __builtin_amdgcn_perm(y, x, 0x07050301u)};
            }
        }
    }
    if (values) {
#pragma unroll
        for (int h = 0; h < 2; ++h) *(u2*)(lds + (32 * k + (lane & 15) + 16 * h) * kLdsRow + 8 * g) = e[h];
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            e[h] = u2{0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j)
                e[h][j >> 2] |= (uint32_t)lds[(32 * k + 8 * g + j) * kLdsRow + kv_slot((lane & 15) + 16 * h)] << (8 * (j & 3));
        }
    }
    void* dst = values ? t.v : t.k;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const long long s = w.pos + (lane & 15) + 16 * h - w.p0;
        if (s < 0 || s >= t.seq) continue;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            x[j] = in[h] ? (float)((int)((e[h][j >> 2] >> (8 * (j & 3))) & 0xff) - zero) * sc[h] : 0.0f;
        store8<TY>(dst, (long long)b * t.bstride + s * t.tstride + (long long)head * HD + 32 * k + 8 * g, x);
    }
}

template <int TY, int BITS, int HD>
hipError_t go(bool write, const KvCache& c, const KvTokens& t, hipStream_t s) {
    // seq positions from anywhere in a tile on
    const dim3 grid((unsigned)(((long long)t.seq + 62) / 32), (unsigned)(2 * c.heads), (unsigned)t.batch);
    if (write) kv_write_kernel<TY, BITS, HD><<<grid, HD * 2, 0, s>>>(c, t);
    else kv_read_kernel<TY, BITS, HD><<<grid, HD * 2, 0, s>>>(c, t);
    return hipGetLastError();
}
template <int TY, int BITS>
hipError_t by_hd(bool write, const KvCache& c, const KvTokens& t, hipStream_t s) {
    switch (c.hd) {
    case 64: return go<TY, BITS, 64>(write, c, t, s);
    case 96: return go<TY, BITS, 96>(write, c, t, s);
    case 128: return go<TY, BITS, 128>(write, c, t, s);
    case 256: return go<TY, BITS, 256>(write, c, t, s);
    }
    return hipErrorInvalidValue;
}
hipError_t by_type(bool write, const KvCache& c, const KvTokens& t, hipStream_t s) {
    if (t.batch == 0 || t.seq == 0) return hipSuccess;
    if (c.bits == 8)
        return t.type == FT_F32 ? by_hd<FT_F32, 8>(write, c, t, s)
             : t.type == FT_F16 ? by_hd<FT_F16, 8>(write, c, t, s) : by_hd<FT_BF16, 8>(write, c, t, s);
    return t.type == FT_F32 ? by_hd<FT_F32, 4>(write, c, t, s)
         : t.type == FT_F16 ? by_hd<FT_F16, 4>(write, c, t, s) : by_hd<FT_BF16, 4>(write, c, t, s);
}

}  // namespace

hipError_t launch_kv_write(const KvCache& c, const KvTokens& t, hipStream_t s) { return by_type(true, c, t, s); }
hipError_t launch_kv_read(const KvCache& c, const KvTokens& t, hipStream_t s) { return by_type(false, c, t, s); }

}  // namespace nnrh
