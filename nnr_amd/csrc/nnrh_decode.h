// nnrh_decode.h -- operators of a decoder's serving step: products with 4-bit
// weights (nnrh_nbits.hip), the quantized key/value cache (nnrh_kvcache.hip) and
// the attention that reads it (nnrh_kvattn.hip). Shared with the C-ABI layer.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace nnrh {

// element types of activations
enum FloatType : int { FT_F32 = 0, FT_F16 = 1, FT_BF16 = 2 };
inline int float_type_size(int t) { return t == FT_F32 ? 4 : 2; }

// ---- 4-bit weights -----------------------------------------------------------
// Weights in memory: a piece is 16 columns x 128 K, one contiguous kilobyte,
// 16 bytes a lane: lane l holds column l & 15; its word s the K values
// 32 s + 8 (l >> 4) + j, j even in nibble j / 2, j odd in nibble 4 + j / 2
// (the operand order of a 16x16x32 MFMA whose neighbouring elements come out
// of one masked shift). Pieces of a column tile follow each other along K.
constexpr int NB_PK = 128;                 // K of a piece
struct NbitsArgs {
    const void* a;
    const uint32_t* w;                     // [Np / 16][P] pieces
    const void* scales;                    // [Np / 16][P][16][nspp], activations' type
    const uint16_t* zp;                    // [Np / 16][P][16], nibble s for word s; without
    long long zp_mask;                     // zero points one piece's 8s for all: 0, else -1
    const void* bias;                      // [N] or NULL, activations' type
    void* y;
    int M, N, K, P;
    int nspp;                              // scales a piece and column: 4, 2 or 1
    int type;                              // FloatType
};
inline int nbits_pieces(int K) { return (K + NB_PK - 1) / NB_PK; }
inline int nbits_cols(int N) { return (N + 127) / 128 * 128; }   // columns held: whole blocks of them
inline int nbits_nspp(int block) { return block >= NB_PK ? 1 : NB_PK / block; }
hipError_t launch_nbits(const NbitsArgs& a, hipStream_t s);
// raw: [N][nb][block / 2] codes, low nibble first; raw_scales [N][nb] of `type`;
// raw_zp [N][(nb + 1) / 2] or NULL
hipError_t launch_nbits_pack(const uint8_t* raw, const void* raw_scales, const uint8_t* raw_zp, int N, int K,
                             int block, int type, uint32_t* w, void* scales, uint16_t* zp, hipStream_t s);

// ---- quantized key/value cache ----------------------------------------------
// A page holds page_size tokens of every head; a head's part of it is
//   key codes | value codes | key scales | value scales
// Codes lie in blocks of 32 tokens x 32 elements, block (tile, c) of tile =
// token / 32 and c = element / 32 at tile * (head_dim / 32) + c, 16 bytes (8
// bits) or 8 bytes (4 bits) a lane of a 16x16x32 MFMA operand:
//   keys    lane (t & 15) + 16 (e >> 3): elements 8 (e >> 3) + j of token t, then of t + 16
//   values  lane (e & 15) + 16 g:        tokens kv_slot^-1(8 g + j) of element e, then of e + 16
// so attention loads operands of either product with no shuffle. 8-bit codes
// are stored as code + 128. Of 4-bit ones eight make a word, code + 8 each:
// j even in nibble j / 2, j odd in nibble 4 + j / 2, and the word turned left
// by two bits (a shift and a mask then leave a pair in its fp16 places).
// Scales are bf16, [group][page_size], a tile's 32 in the order of kv_slot; the
// keys' at 4 bits, which belong to an operand's rows, in the order of kv_pair.
struct KvCache {
    uint8_t* data;
    int num_pages, page_size, heads, hd, bits;
};
__host__ __device__ inline int kv_groups(int hd, int bits) { return bits == 8 ? 1 : hd / 32; }
__host__ __device__ inline long long kv_codes_bytes(int page, int hd, int bits) { return (long long)page * hd * bits / 8; }
// bytes of one head's part of a page
__host__ __device__ inline long long kv_head_bytes(int page, int hd, int bits) {
    return 2 * (kv_codes_bytes(page, hd, bits) + 2LL * page * kv_groups(hd, bits));
}
// place of token t of a tile among its scales and along a value operand's K:
// the order in which the two 16-token tiles of a score product leave a lane
// its four rows each
__host__ __device__ inline int kv_slot(int t) { return 8 * ((t >> 2) & 3) + 4 * (t >> 4) + (t & 3); }
__host__ __device__ inline uint32_t kv_turn(uint32_t w) { return w << 2 | w >> 30; }
__host__ __device__ inline uint32_t kv_unturn(uint32_t w) { return w >> 2 | w << 30; }
// tokens t and t + 16 side by side
__host__ __device__ inline int kv_pair(int t) { return 2 * (t & 15) + (t >> 4); }

struct KvTokens {           // write: const sources; read: destinations
    void* k;
    void* v;
    int type;               // FloatType
    long long bstride, tstride;   // elements
    int batch, seq;
    const int32_t* table;
    int max_pages;
    const int32_t* lens;
};
hipError_t launch_kv_write(const KvCache& c, const KvTokens& t, hipStream_t s);
hipError_t launch_kv_read(const KvCache& c, const KvTokens& t, hipStream_t s);

struct KvAttention {
    const void* q;
    void* y;
    int type;
    long long q_bstride, q_tstride;
    int batch, seq, q_heads;
    float scale;
    const int32_t* table;
    int max_pages;
    const int32_t* lens;
    const int32_t* prefix_table;
    int prefix_len;
};
// bytes of partial results; 0: one block sees all keys of its rows
size_t kv_attention_workspace(const KvCache& c, const KvAttention& a);
hipError_t launch_kv_attention(const KvCache& c, const KvAttention& a, void* workspace, hipStream_t s);

}  // namespace nnrh
