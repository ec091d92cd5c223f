// nnrh_kvmove.hip -- pages copied and tokens moved within quantized key/value
// caches, several layers' at once: what a fork, a compaction and the acceptance of
// drafted tokens need. Codes and scales go as they are, so nothing is rounded a
// second time. Bound by memory and, for a few tokens, by the launch.
#include "nnrh_decode.h"

#include <algorithm>
#include <type_traits>

namespace nnrh {
namespace {

typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// ---- whole pages ----------------------------------------------------------------
constexpr int CU = 4;   // 16-byte loads in flight a thread

// One block a part of a page: 256 threads x CU x 16 bytes. (700 pages of 8 caches, 413
// MB in 82 us, 5.0 TB/s, a large copy's rate; 6 of 2 caches 3.4 us.)
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

// One block a sequence, head, keys or values, layer; its waves take tokens in turn.
// All are read before any is written, so that a call may permute them. Keys move in
// words of 8 elements. Of values, a word (two, 8 bits) holds 8 tokens of an element:
// tokens that go to the same word are a chain, whose first loads it, puts all of
// them in and stores it, so that no two lanes change one word. Bound by latency: the
// positions, the table, the tokens, the words that they go to, each a trip to memory
// (4 tokens of 2 caches x 8 heads of 128, 8 bits, 4.7 us; 7 of 64 sequences, 8
// caches, 4 bits, 24: its 8192 blocks have one wave each, which makes the trips to tokens and
// words twice. A key is 4 bytes of each of 16 lines: 117 MB asked of L2, 35 of memory, a copy's 7 us).
constexpr int MU = 4;   // tokens in flight a wave

// a token's place, which is the same for all lanes, in scalar registers: a lane adds
// its own part of the address
struct Place {
    long long part;
    int tile, slot, in;   // tile of the page; of its tokens: the word of 8 (0 .. 3), the token
};
__device__ __forceinline__ Place place_of(const TokenAt& t) {
    const long long part = t.part;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)part), hi = __builtin_amdgcn_readfirstlane((int)(part >> 32));
    const int tok = __builtin_amdgcn_readfirstlane(t.tok);
    return Place{(long long)((uint64_t)hi << 32 | lo), tok >> 5, tok >> 2 & 3, tok & 31};
}

template <int BITS, int HD>
__global__ __launch_bounds__(256) void kv_move_tokens_kernel(KvCache c, KvLayers l, KvMoves m) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr int BB = BITS == 8 ? 1024 : 512, KW = BITS == 8 ? 2 : 1;   // KW: words of 8 codes
    constexpr int NC = HD / 32, groups = BITS == 8 ? 1 : NC, NE = (HD + 63) / 64, octs = HD / 8;
    typedef uint32_t word_t __attribute__((ext_vector_type(KW)));
    const int head = blockIdx.y >> 1, values = blockIdx.y & 1, b = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    uint8_t* data = l.data[blockIdx.z];
    TokenAt* from = (TokenAt*)lds;
    TokenAt* to = from + m.n;
    int* chain = (int*)(to + m.n);                                        // the next token of a word, + 1 << 16 for a first one
    uint16_t* scales = (uint16_t*)(chain + (m.n + 1) / 2 * 2);            // [n][groups]
    uint8_t* codes = (uint8_t*)(scales + (m.n * groups + 3) / 4 * 4);     // keys: [n][octs] words; values: a byte each
    for (int i = threadIdx.x; i < m.n; i += blockDim.x) {
        const long long at = (long long)b * m.n + i;
        TokenAt x = token_at(c, m, b, head, m.src[at]), y = token_at(c, m, b, head, m.dst[at]);
        if (x.part < 0) y.part = -1;
        if (y.part < 0) x.part = -1;
        from[i] = x;
        to[i] = y;
    }
    __syncthreads();
    if (values) {
        // 8 tokens share a word: 4 g .. of a tile and those 16 further
        const auto same = [&](const TokenAt& x, const TokenAt& y) {
            return x.part == y.part && (x.tok >> 5) == (y.tok >> 5) && (x.tok >> 2 & 3) == (y.tok >> 2 & 3);
        };
        for (int i = threadIdx.x; i < m.n; i += blockDim.x) {
            const TokenAt t = to[i];
            int next = i + 1, before = i - 1;
            while (next < m.n && !same(to[next], t)) ++next;
            while (before >= 0 && !same(to[before], t)) --before;
            chain[i] = next | (before < 0) << 16;
        }
    }
    const long long cb = kv_codes_bytes(c.page_size, HD, BITS);
    const long long codes0 = values ? cb : 0, scales0 = 2 * cb + (values ? 2LL * c.page_size * groups : 0);
    const auto scale_place = [&](const Place& t) {   // of group `lane`
        return (uint16_t*)(data + t.part + scales0) + (t.tile * 32 + (BITS == 4 && !values ? kv_pair(t.in) : kv_slot(t.in))) +
               lane * c.page_size;
    };
    // a key's elements 8 lane ..
    const auto key_place = [&](const Place& t) {
        return (word_t*)(data + t.part + t.tile * (NC * BB)) + ((t.in & 15) * 2 + (t.in >> 4)) + ((lane >> 2) * (BB / (KW * 4)) + 32 * (lane & 3));
    };
    // the word with a token's value e = lane + 64 k; which of its codes that is
    const auto value_place = [&](const Place& t, int k) {
        return (word_t*)(data + t.part + codes0 + t.tile * (NC * BB)) + 32 * t.slot +
               (((lane >> 5) + 2 * k) * (BB / (KW * 4)) + (lane & 15) * 2 + (lane >> 4 & 1));
    };
    const auto code_at = [](const Place& t) { return kv_slot(t.in) & 7; };
    const bool scale_lane = lane < groups, key_lane = lane < octs;
    const auto value_lane = [&](int k) { return HD % 64 == 0 || lane + 64 * k < HD; };
    for (int t0 = wave; t0 < m.n; t0 += MU * waves) {
        word_t x[MU][NE];
        uint16_t sc[MU];
        Place at[MU];
#pragma unroll
        for (int u = 0; u < MU; ++u) {
            at[u].part = -1;
            if (t0 + u * waves < m.n) at[u] = place_of(from[t0 + u * waves]);
            if (at[u].part < 0) continue;
            if (scale_lane) sc[u] = *scale_place(at[u]);
            if (values) {
#pragma unroll
                for (int k = 0; k < NE; ++k)
                    if (value_lane(k)) x[u][k] = *value_place(at[u], k);
            } else if (key_lane) {
                x[u][0] = *key_place(at[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < MU; ++u) {
            if (at[u].part < 0) continue;
            const int t = t0 + u * waves, j = code_at(at[u]);
            if (scale_lane) scales[t * groups + lane] = sc[u];
            if (values) {
#pragma unroll
                for (int k = 0; k < NE; ++k)
                    if (value_lane(k))
                        codes[t * HD + lane + 64 * k] = (uint8_t)(BITS == 8 ? x[u][k][KW - 1 & j >> 2] >> (8 * (j & 3))
                                                                            : kv_unturn(x[u][k][0]) >> (4 * ((j >> 1) + 4 * (j & 1))) & 15u);
            } else if (key_lane) {
                ((word_t*)codes)[t * octs + lane] = x[u][0];
            }
        }
    }
    __syncthreads();
    for (int t0 = wave; t0 < m.n; t0 += MU * waves) {
        word_t x[MU][NE];
        Place at[MU];
        int next[MU];
#pragma unroll
        for (int u = 0; u < MU; ++u) {
            const int t = t0 + u * waves;
            at[u].part = -1;
            if (t < m.n) at[u] = place_of(to[t]);
            if (at[u].part < 0) continue;
            if (scale_lane) *scale_place(at[u]) = scales[t * groups + lane];
            if (!values) {
                if (key_lane) *key_place(at[u]) = ((const word_t*)codes)[t * octs + lane];
                continue;
            }
            next[u] = __builtin_amdgcn_readfirstlane(chain[t]);
            if (!(next[u] >> 16)) at[u].part = -1;   // (another token's)
            else {
#pragma unroll
                for (int k = 0; k < NE; ++k)
                    if (value_lane(k)) x[u][k] = *value_place(at[u], k);
            }
        }
        if (!values) continue;
#pragma unroll
        for (int u = 0; u < MU; ++u) {
            if (at[u].part < 0) continue;
            for (int i = t0 + u * waves, n = next[u] & 0xffff; ; n = __builtin_amdgcn_readfirstlane(chain[i]) & 0xffff) {
                const int in = __builtin_amdgcn_readfirstlane(to[i].tok) & 31, j = kv_slot(in) & 7;
#pragma unroll
                for (int k = 0; k < NE; ++k) {
                    const uint32_t code = codes[min(i * HD + lane + 64 * k, m.n * HD - 1)];   // (of a lane past the head: any)
                    word_t& w = x[u][k];
                    if constexpr (BITS == 8) {
                        const uint32_t mask = 255u << (8 * (j & 3)), bits = code << (8 * (j & 3));
                        if (j >> 2) w[KW - 1] = (w[KW - 1] & ~mask) | bits;
                        else w[0] = (w[0] & ~mask) | bits;
                    } else {
                        const int sh = 4 * ((j >> 1) + 4 * (j & 1));
                        w[0] = (w[0] & ~kv_turn(15u << sh)) | kv_turn(code << sh);
                    }
                }
                i = n;
                if (i >= m.n) break;
            }
#pragma unroll
            for (int k = 0; k < NE; ++k)
                if (value_lane(k)) *value_place(at[u], k) = x[u][k];
        }
    }
}

size_t move_lds(const KvCache& c, int n) {
    const int groups = kv_groups(c.hd, c.bits);
    return (size_t)n * (2 * sizeof(TokenAt) + 4) + 8 + (n * groups + 3) / 4 * 8 + (size_t)n * c.hd;
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
    // waves: the chip's 8192, or as many as there are tokens
    const long long blocks = (long long)grid.x * grid.y * grid.z;
    const int threads = 64 * (int)std::max(1LL, std::min({4LL, (long long)m.n, 8192 / blocks}));
    const auto go = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        if (c.bits == 8) kv_move_tokens_kernel<8, HD><<<grid, threads, lds, s>>>(c, l, m);
        else kv_move_tokens_kernel<4, HD><<<grid, threads, lds, s>>>(c, l, m);
        return hipGetLastError();
    };
    switch (c.hd) {
    case 64: return go(std::integral_constant<int, 64>{});
    case 96: return go(std::integral_constant<int, 96>{});
    case 128: return go(std::integral_constant<int, 128>{});
    case 256: return go(std::integral_constant<int, 256>{});
    }
    return hipErrorInvalidValue;
}

}  // namespace nnrh
