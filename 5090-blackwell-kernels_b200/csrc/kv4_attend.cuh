// What the two attention kernels over the 4-bit cache share: the arguments of a call, and which of its sequences goes to which.
#pragma once

#include "kv4_layout.cuh"

namespace spk::kv4 {

struct AttendParams {
    const __nv_bfloat16* q;
    long long stride;
    Pool pool;
    Batch batch;
    int q_heads, window, zero_rest;
    int prompts;  // whether sequences with many rows are another launch's (kv4_prompt.cu)
    float scale;
    __nv_bfloat16* out;
    int4* pieces;     // of kv4_attention.cu, in the workspace
    float* partials;
    int* status;
};

// A sequence is a prompt from kPromptRows rows a KV head up (rows: new tokens x query heads of a KV head), and prompts are
// taken in blocks of kBlockRows rows a CTA. With fewer than kPromptBlocks blocks in the call they would leave most SMs idle,
// while the other kernel cuts the keys as well. One sequence's chunk on 8192 keys, 32 heads over 8, d = 128: 24 blocks 195 us here and
// 164 there, 32 blocks 196 and 213, 64 blocks 197 and 414; on 2048 keys 24 blocks 62 and 69, 32 blocks 62 and 79; two sequences of
// 256 rows with 8 heads of their own, 16 blocks, 107 and 72. By rows, 32 sequences on 4096: 128 rows 184 and 413, 64 rows 181 and
// 223, 32 rows 180 and 122; 64 sequences on 512: 128 rows 77 and 201, 64 rows 71 and 104, 32 rows 70 and 62. (A tile of
// 128 rows that is half full costs as much as a full one; between 48 and 128 rows large batches would be faster here.)
constexpr int kPromptRows = 128, kBlockRows = 256, kPromptBlocks = 32;

__host__ __device__ inline long long prompt_blocks(long long rows) { return rows >= kPromptRows ? (rows + kBlockRows - 1) / kBlockRows : 0; }

#ifdef __CUDACC__
// A row's queries go into the products in fp16, times a power of two that puts the largest of them, of biased exponent e, at 2^13 to
// 2^14; lower, down to 1, where it is below 2^-50: keys that give such queries their scores are large, and the sums stay inside
// fp32. And its inverse, by which the scores are put right.
__device__ __forceinline__ float query_scale(int e) { return __uint_as_float(static_cast<uint32_t>(254 - max(e, 1) + min(max(e - 64, 0), 13)) << 23); }
__device__ __forceinline__ float query_unscale(float by) { return __uint_as_float((254u << 23) - __float_as_uint(by)); }
constexpr float kLeast = 1.4e-45f;  // above 0
#endif

// kv4_prompt.cu: the call's prompts; nothing if they are too few.
int attend_prompts(const AttendParams& p, int head_dim, int group, DeviceState* dev, cudaStream_t stream);

}  // namespace spk::kv4
