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

// One block a sequence, head, keys or values, layer; its waves take its tokens in
// turn, four at a time in flight. All of them are read before any is written, so
// that a call may permute them. Keys move in words of 8 elements; of values, where
// neighbours in memory are a tile's tokens, a token's byte is stored by itself, and
// its nibble turned into the new one by an exclusive-or with what is there: the
// word's other nibbles stay as they are whoever else changes them, and whatever the
// order.
constexpr int MU = 4;
template <int BITS>
__global__ __launch_bounds__(256) void kv_move_tokens_kernel(KvCache c, KvLayers l, KvMoves m) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr int BB = BITS == 8 ? 1024 : 512, KW = BITS == 8 ? 2 : 1;   // KW: words of 8 key codes
    typedef uint32_t key_t __attribute__((ext_vector_type(KW)));
    const int head = blockIdx.y >> 1, values = blockIdx.y & 1, b = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int NC = c.hd / 32, groups = BITS == 8 ? 1 : NC;
    uint8_t* data = l.data[blockIdx.z];
    TokenAt* from = (TokenAt*)lds;
    TokenAt* to = from + m.n;
    uint16_t* scales = (uint16_t*)(to + m.n);                             // [n][groups]
    uint8_t* codes = (uint8_t*)(scales + (m.n * groups + 3) / 4 * 4);     // keys: [n][hd / 8][KW] words; values: a byte each
    for (int i = threadIdx.x; i < m.n; i += blockDim.x) {
        const long long at = (long long)b * m.n + i;
        TokenAt x = token_at(c, m, b, head, m.src[at]), y = token_at(c, m, b, head, m.dst[at]);
        if (y.part < 0) x.part = -1;
        from[i] = x;
        to[i] = y;
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
        return (key_t*)(data + t.part + ((long long)(t.tok >> 5) * NC + (oct >> 2)) * BB) + ((in & 15) + 16 * (oct & 3)) * 2 + (in >> 4);
    };
    // the word that holds a token's value e, and which of its bytes or nibbles that is
    const auto value_place = [&](const TokenAt& t, int e, int* which) {
        const int slot = kv_slot(t.tok & 31), j = slot & 7;
        uint32_t* w = (uint32_t*)(data + t.part + codes0 + ((long long)(t.tok >> 5) * NC + (e >> 5)) * BB) +
                      ((e & 15) + 16 * (slot >> 3)) * 2 * KW + (e >> 4 & 1) * KW;
        *which = BITS == 8 ? j & 3 : (j >> 1) + 4 * (j & 1);
        return BITS == 8 ? w + (j >> 2) : w;
    };
    // fn(token, place of the lane's element) over the wave's tokens and the elements `width` of a token, `load` first
    // for MU of them
    const auto each = [&](int width, auto load, auto store) {
        for (int e = lane; e < width; e += 64)
            for (int t0 = wave; t0 < m.n; t0 += MU * waves) {
                decltype(load(0, 0)) x[MU];
                bool some[MU];
#pragma unroll
                for (int u = 0; u < MU; ++u) {
                    const int t = t0 + u * waves;
                    some[u] = t < m.n && from[t].part >= 0;
                    if (some[u]) x[u] = load(t, e);
                }
#pragma unroll
                for (int u = 0; u < MU; ++u)
                    if (some[u]) store(t0 + u * waves, e, x[u]);
            }
    };
    each(groups, [&](int t, int g) { return *scale_place(from[t], g); }, [&](int t, int g, uint16_t x) { scales[t * groups + g] = x; });
    if (!values)
        each(c.hd / 8, [&](int t, int o) { return *key_place(from[t], o); },
             [&](int t, int o, key_t x) { ((key_t*)codes)[t * (c.hd / 8) + o] = x; });
    else
        each(c.hd,
             [&](int t, int e) {
                 int which;
                 const uint32_t w = *value_place(from[t], e, &which);
                 return BITS == 8 ? w >> (8 * which) & 255u : kv_unturn(w) >> (4 * which) & 15u;
             },
             [&](int t, int e, uint32_t x) { codes[t * c.hd + e] = (uint8_t)x; });
    __syncthreads();
    each(groups, [&](int t, int g) { return scales[t * groups + g]; }, [&](int t, int g, uint16_t x) { *scale_place(to[t], g) = x; });
    if (!values)
        each(c.hd / 8, [&](int t, int o) { return ((const key_t*)codes)[t * (c.hd / 8) + o]; },
             [&](int t, int o, key_t x) { *key_place(to[t], o) = x; });
    else
        each(c.hd,
             [&](int t, int e) {
                 int which;
                 const uint32_t* p = value_place(to[t], e, &which);
                 const uint32_t code = codes[t * c.hd + e];
                 if constexpr (BITS == 8) return code;
                 // (what another thread does to the word meanwhile leaves this nibble)
                 const uint32_t old = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                 return kv_turn((kv_unturn(old) >> (4 * which) & 15u ^ code) << (4 * which));
             },
             [&](int t, int e, uint32_t x) {
                 int which;
                 uint32_t* p = value_place(to[t], e, &which);
                 if constexpr (BITS == 8) ((uint8_t*)p)[which] = (uint8_t)x;
                 else if (x) __hip_atomic_fetch_xor(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
             });
}

size_t move_lds(const KvCache& c, int n) {
    const int groups = kv_groups(c.hd, c.bits);
    return (size_t)n * 2 * sizeof(TokenAt) + (n * groups + 3) / 4 * 8 + (size_t)n * c.hd;
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
    const int threads = 64 * std::min(4, (m.n + 7) / 8);
    if (c.bits == 8) kv_move_tokens_kernel<8><<<grid, threads, lds, s>>>(c, l, m);
    else kv_move_tokens_kernel<4><<<grid, threads, lds, s>>>(c, l, m);
    return hipGetLastError();
}

}  // namespace nnrh
