// The 4-bit KV cache: what its bytes mean, and the checks every entry point makes of its arguments.
//
// A pool holds pages of page_size tokens (a multiple of 16); a page holds, for each KV head, page_size / 16 tiles.
// A tile is 16 tokens of one head, K and V together, contiguous, so that one bulk copy brings all an attention step
// reads of them:
//     K codes  16 x d / 2 bytes       V codes  16 x d / 2 bytes       K words [16][d / group]       V words [16][d / group]
// A word is a group's pair (minimum m: low half, scale s: high half, bf16 each); a code c stands for c s + m.
//
// The order of the codes is the one in which tensor-core fragments are read without a shuffle (kv4_attention.cu):
//   K  a token's row of d / 2 bytes is four runs, run c holding channels 32 i + 8 c .. + 7 as the 32-bit word i, the
//      lowest channel in the lowest nibble: the four lanes that share a key in an A fragment read one run each.
//   V  blocks of eight tokens; in a block, run g (of eight) holds for each token a piece of d / 16 bytes, whose
//      half word u has channels 32 u + 4 g .. + 3: lane (g, c) reads the pieces of tokens 2 c and 2 c + 1 in one load.
#pragma once

#include "spk_common.cuh"

namespace spk::kv4 {

constexpr int kTile = 16;
constexpr int kMaxSeqs = 4096;  // sequences of a call

__host__ __device__ constexpr int tile_bytes(int d, int group) { return kTile * d + 2 * kTile * (d / group) * 4; }
__host__ __device__ constexpr int v_codes_at(int d) { return kTile * d / 2; }
__host__ __device__ constexpr int k_words_at(int d) { return kTile * d; }
__host__ __device__ constexpr int v_words_at(int d, int group) { return kTile * d + kTile * (d / group) * 4; }

// Byte of the 32-bit word that holds channels ch .. ch + 7 (ch % 8 == 0) of token t's keys.
__host__ __device__ constexpr int k_word_at(int d, int t, int ch) { return t * (d / 2) + (ch % 32 / 8) * (d / 8) + (ch / 32) * 4; }
// Byte, counted from the V codes, of the piece of token t in run g.
__host__ __device__ constexpr int v_piece_at(int d, int t, int g) { return (t / 8) * 4 * d + g * (d / 2) + (t % 8) * (d / 16); }

inline bool shape_ok(int d, int group) {
    return (d == 64 || d == 128) && (group == 32 || group == 64 || group == 128) && group <= d;
}

// What the sequences of a call are: lens[b] tokens in the cache, the last of them this call's own; the call's rows of
// sequence b are offsets[b] .. offsets[b + 1] - 1, or row b where offsets is null.
struct Batch {
    const int32_t* table;    // [seqs][width] page of each page_size tokens
    const int32_t* lens;     // [seqs]
    const int32_t* offsets;  // [seqs + 1] or null
    int seqs, rows, width;   // rows: of the call's tensors
};

struct Pool {
    unsigned char* data;
    int pages, page_size, heads, tile_bytes;
};

#ifdef __CUDACC__
__device__ __forceinline__ void bad_index(int* status) { status[kIndexWord] = SPK_BAD_INDEX; }
// First row and number of rows of sequence b, inside the call's tensors whatever the offsets say.
__device__ __forceinline__ void rows_of(const Batch& s, int b, int& first, int& count) {
    if (s.offsets == nullptr) {
        first = b, count = 1;
        return;
    }
    first = min(max(s.offsets[b], 0), s.rows);
    count = max(0, min(s.offsets[b + 1], s.rows) - first);
}
// Tokens of sequence b that are in the cache; none, which makes its rows padding, where its row of the table has no room for them.
__device__ __forceinline__ int length_of(const Batch& s, int page_size, int b, int* status) {
    const int len = s.lens[b];
    if (len >= 0 && len <= static_cast<long long>(s.width) * page_size) return len;
    bad_index(status);
    return 0;
}
__device__ __forceinline__ float word_min(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float word_scale(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
#endif

// Host checks shared by the entry points; nonzero is the status to return.
inline int check(const char* what, const void* pool, int pages, int page_size, int kv_heads, int d, int group) {
    if (pool == nullptr || !aligned16(pool)) return fail(SPK_INVALID, "%s: the pool must be a 16-byte aligned device pointer", what);
    if (!shape_ok(d, group))
        return fail(SPK_INVALID, "%s: head_dim must be 64 or 128 and group 32, 64 or 128 and at most head_dim, got head_dim=%d group=%d", what, d, group);
    if (page_size < kTile || page_size > 1024 || page_size % kTile != 0)
        return fail(SPK_INVALID, "%s: page_size must be a multiple of 16 between 16 and 1024, got %d", what, page_size);
    if (pages < 1 || kv_heads < 1 || kv_heads > 1024) return fail(SPK_INVALID, "%s: needs at least one page and 1 to 1024 KV heads, got pages=%d kv_heads=%d", what, pages, kv_heads);
    return SPK_OK;
}
inline int check_batch(const char* what, const Batch& s, int page_size) {
    if (s.seqs < 0 || s.rows < 0 || s.width < 0 || s.seqs > kMaxSeqs) return fail(SPK_INVALID, "%s: needs 0 to %d sequences and no negative sizes, got sequences=%d rows=%d table width=%d", what, kMaxSeqs, s.seqs, s.rows, s.width);
    if (static_cast<long long>(s.width) * page_size > 1 << 30) return fail(SPK_INVALID, "%s: a row of the page table may hold 2^30 tokens, got %d pages of %d", what, s.width, page_size);
    if (s.rows > 0 && s.seqs > 0 && (s.lens == nullptr || (s.table == nullptr && s.width > 0))) return fail(SPK_INVALID, "%s: null page table or lengths", what);
    if (s.offsets == nullptr && s.rows != s.seqs) return fail(SPK_INVALID, "%s: without q_offsets every sequence has one row, got %d rows and %d sequences", what, s.rows, s.seqs);
    return SPK_OK;
}

}  // namespace spk::kv4
