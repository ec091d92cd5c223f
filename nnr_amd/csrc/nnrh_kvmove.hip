// nnrh_kvmove.hip -- pages copied and tokens moved within quantized key/value
// caches, several layers' at once: what a fork, a compaction and the acceptance of
// drafted tokens need. Codes and scales go as they are, so nothing is rounded a
// second time. Bound by memory and, for a few tokens, by the launch.
#include "nnrh_decode.h"

#include <algorithm>

namespace nnrh {
namespace {

typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// ---- whole pages ----------------------------------------------------------------
constexpr int CU = 4;   // 16-byte loads in flight a thread

// One block a part of a page: 256 threads x CU x 16 bytes.
__global__ __launch_bounds__(256) void kv_copy_pages_kernel(KvLayers l, const int32_t* src, const int32_t* dst, int pages,
                                                            long long bytes) {
    const int from = src[blockIdx.y], to = dst[blockIdx.y];
    if (from < 0 || from >= pages || to < 0 || to >= pages || from == to) return;
    const uint8_t* x = l.data[blockIdx.z] + from * bytes;
    uint8_t* y = l.data[blockIdx.z] + to * bytes;
    const long long at = ((long long)blockIdx.x * CU * 256 + threadIdx.x) * 16;
    u4 v[CU];
#pragma unroll
    for (int i = 0; i < CU; ++i)
        if (at + i * 4096 < bytes) v[i] = *(const u4*)(x + at + i * 4096);
#pragma unroll
    for (int i = 0; i < CU; ++i)
        if (at + i * 4096 < bytes) *(u4*)(y + at + i * 4096) = v[i];
}

// ---- tokens ---------------------------------------------------------------------
// Where a token is: the head's part of its page and its place there
struct TokenAt {
    long long part;   // bytes from the cache's start; < 0: nowhere
    int tok;          // within the page
};
__device__ __forceinline__ TokenAt token_at(const KvCache& c, const KvMoves& m, int b, int head, int pos) {
    TokenAt r = {-1, 0};
    if (pos < 0 || pos >= (long long)m.max_pages * c.page_size) return r;
    const int id = m.table[(long long)b * m.max_pages + (pos >> (31 - __builtin_clz((unsigned)c.page_size)))];
    if (id < 0 || id >= c.num_pages) return r;
    r.part = ((long long)id * c.heads + head) * kv_head_bytes(c.page_size, c.hd, c.bits);
    r.tok = pos & (c.page_size - 1);
    return r;
}

// One block a sequence, head, keys or values, layer. All of its tokens are read
// before any is written, so that a call may permute them. Keys move in words of
// 8 elements; of values, where neighbours in memory are a tile's tokens, a token's
// byte is stored by itself, and its nibble turned into the new one by an
// exclusive-or with what is there: the word's other nibbles stay as they are whoever
// else changes them, and whatever the order.
template <int BITS>
__global__ __launch_bounds__(256) void kv_move_tokens_kernel(KvCache c, KvLayers l, KvMoves m) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr int BB = BITS == 8 ? 1024 : 512, KW = BITS == 8 ? 2 : 1;   // KW: words of 8 key codes
    const int head = blockIdx.y >> 1, values = blockIdx.y & 1, b = blockIdx.x;
    const int NC = c.hd / 32, groups = BITS == 8 ? 1 : NC;
    uint8_t* data = l.data[blockIdx.z];
    TokenAt* from = (TokenAt*)lds;
    TokenAt* to = from + m.n;
    uint16_t* scales = (uint16_t*)(to + m.n);                   // [n][groups]
    uint32_t* codes = (uint32_t*)(scales + (m.n * groups + 1) / 2 * 2);   // keys: [n][hd / 8][KW]; values: a byte each
    if ((int)threadIdx.x < m.n) {
        const long long i = (long long)b * m.n + threadIdx.x;
        TokenAt x = token_at(c, m, b, head, m.src[i]), y = token_at(c, m, b, head, m.dst[i]);
        if (y.part < 0) x.part = -1;
        from[threadIdx.x] = x;
        to[threadIdx.x] = y;
    }
    __syncthreads();
    const long long cb = kv_codes_bytes(c.page_size, c.hd, BITS);
    const long long codes0 = values ? cb : 0, scales0 = 2 * cb + (values ? 2LL * c.page_size * groups : 0);
    const auto scale_place = [&](const TokenAt& t, int g) {
        const int in = t.tok & 31;
        return (uint16_t*)(data + t.part + scales0) + (long long)g * c.page_size + (t.tok & ~31) +
               (BITS == 4 && !values ? kv_pair(in) : kv_slot(in));
    };
    // eight key elements of a token
    const auto key_place = [&](const TokenAt& t, int oct) {
        const int in = t.tok & 31;
        return (uint32_t*)(data + t.part + ((long long)(t.tok >> 5) * NC + (oct >> 2)) * BB) +
               ((in & 15) + 16 * (oct & 3)) * 2 * KW + (in >> 4) * KW;
    };
    // the word that holds a token's value e, and which of its bytes or nibbles that is
    const auto value_place = [&](const TokenAt& t, int e, int* which) {
        const int slot = kv_slot(t.tok & 31), j = slot & 7;
        uint32_t* w = (uint32_t*)(data + t.part + codes0 + ((long long)(t.tok >> 5) * NC + (e >> 5)) * BB) +
                      ((e & 15) + 16 * (slot >> 3)) * 2 * KW + (e >> 4 & 1) * KW;
        *which = BITS == 8 ? j & 3 : (j >> 1) + 4 * (j & 1);
        return BITS == 8 ? w + (j >> 2) : w;
    };
    for (int i = threadIdx.x; i < m.n * groups; i += 256) {
        const TokenAt t = from[i / groups];
        if (t.part >= 0) scales[i] = *scale_place(t, i % groups);
    }
    if (!values) {
        const int octs = c.hd / 8;
        for (int i = threadIdx.x; i < m.n * octs; i += 256) {
            const TokenAt t = from[i / octs];
            if (t.part < 0) continue;
            const uint32_t* p = key_place(t, i % octs);
#pragma unroll
            for (int k = 0; k < KW; ++k) codes[i * KW + k] = p[k];
        }
    } else {
        for (int i = threadIdx.x; i < m.n * c.hd; i += 256) {
            const TokenAt t = from[i / c.hd];
            if (t.part < 0) continue;
            int which;
            const uint32_t w = *value_place(t, i % c.hd, &which);
            ((uint8_t*)codes)[i] = (uint8_t)(BITS == 8 ? w >> (8 * which) : kv_unturn(w) >> (4 * which) & 15u);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < m.n * groups; i += 256)
        if (from[i / groups].part >= 0) *scale_place(to[i / groups], i % groups) = scales[i];
    if (!values) {
        const int octs = c.hd / 8;
        for (int i = threadIdx.x; i < m.n * octs; i += 256) {
            if (from[i / octs].part < 0) continue;
            uint32_t* p = key_place(to[i / octs], i % octs);
#pragma unroll
            for (int k = 0; k < KW; ++k) p[k] = codes[i * KW + k];
        }
    } else {
        for (int i = threadIdx.x; i < m.n * c.hd; i += 256) {
            if (from[i / c.hd].part < 0) continue;
            int which;
            uint32_t* p = value_place(to[i / c.hd], i % c.hd, &which);
            const uint8_t code = ((const uint8_t*)codes)[i];
            if constexpr (BITS == 8) {
                ((uint8_t*)p)[which] = code;
            } else {
                // (what another thread does to the word meanwhile leaves this nibble)
                const uint32_t old = kv_unturn(__hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) >> (4 * which) & 15u;
                const uint32_t flip = kv_turn((old ^ code) << (4 * which));
                if (flip) __hip_atomic_fetch_xor(p, flip, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
    }
}

size_t move_lds(const KvCache& c, int n) {
    const int groups = kv_groups(c.hd, c.bits);
    return (size_t)n * 2 * sizeof(TokenAt) + (n * groups + 1) / 2 * 4 + (size_t)n * c.hd;
}

}  // namespace

hipError_t launch_kv_copy_pages(const KvCache& c, const KvLayers& l, int layers, const int32_t* src, const int32_t* dst,
                                int n, hipStream_t s) {
    const long long bytes = c.heads * kv_head_bytes(c.page_size, c.hd, c.bits), part = CU * 256 * 16;
    const unsigned parts = (unsigned)((bytes + part - 1) / part);
    // a grid's second dimension is 65535 long, and a launch has fewer than 2^32 threads
    const long long most = std::max(1LL, std::min(65535LL, (1LL << 23) / ((long long)parts * layers)));
    for (long long i = 0; i < n; i += most) {
        const dim3 grid(parts, (unsigned)std::min((long long)n - i, most), (unsigned)layers);
        kv_copy_pages_kernel<<<grid, 256, 0, s>>>(l, src + i, dst + i, c.num_pages, bytes);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_kv_move_tokens(const KvCache& c, const KvLayers& l, int layers, const KvMoves& m, hipStream_t s) {
    const dim3 grid((unsigned)m.batch, (unsigned)(2 * c.heads), (unsigned)layers);
    const size_t lds = move_lds(c, m.n);
    if (c.bits == 8) kv_move_tokens_kernel<8><<<grid, 256, lds, s>>>(c, l, m);
    else kv_move_tokens_kernel<4><<<grid, 256, lds, s>>>(c, l, m);
    return hipGetLastError();
}

}  // namespace nnrh
