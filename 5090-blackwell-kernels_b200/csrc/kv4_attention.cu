// Attention over the 4-bit paged KV cache (its bytes: kv4_layout.cuh): for a row (token at position p, query head)
//     out = sum_j softmax_j(scale q . k_j) v_j   over the positions j <= p, with a window only p - window < j,
// k_j and v_j being c s + m. One pass over the keys with the running maximum and sum of the softmax, in fp32.
#include "kv4_layout.cuh"

namespace spk {
namespace {

using kv4::Batch;
using kv4::Pool;

struct AttendParams {
    const __nv_bfloat16* q;
    long long stride;
    Pool pool;
    Batch batch;
    int q_heads, window, zero_rest;
    float scale;
    __nv_bfloat16* out;
    int* status;
};

// The simplest right form: a warp per row and head, a lane per key for the scores, four channels a lane for the output.
template <int D, int G>
__global__ void __launch_bounds__(256) kv4_attend_rows_kernel(const AttendParams p) {
    __shared__ float qs[8][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_release();
    pdl_wait();
    const long long id = static_cast<long long>(blockIdx.x) * 8 + warp;
    const int h = static_cast<int>(id % p.q_heads), t = static_cast<int>(id / p.q_heads);
    if (t >= p.batch.rows) return;
    int b = t;
    if (p.batch.offsets != nullptr) {
        int passed = 0;
        for (int i = lane; i < p.batch.seqs; i += 32) passed += p.batch.offsets[i + 1] <= t;
        b = static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(passed)));
    }
    int pos = -1;
    if (b < p.batch.seqs) {
        int first, count;
        kv4::rows_of(p.batch, b, first, count);
        if (t >= first && t < first + count) pos = kv4::length_of(p.batch, p.pool.page_size, b, p.status) - count + (t - first);
    } else if (!p.zero_rest) {
        return;
    }
    const __nv_bfloat16* q = p.q + t * p.stride + static_cast<long long>(h) * D;
    for (int i = lane; i < D; i += 32) qs[warp][i] = __bfloat162float(q[i]) * p.scale * 1.4426950408889634f;
    __syncwarp();
    const int tiles = p.pool.page_size / kv4::kTile, kv = h / (p.q_heads / p.pool.heads);
    auto tile_of = [&](int j) -> const unsigned char* {
        const int page = p.batch.table[static_cast<size_t>(b) * p.batch.width + j / p.pool.page_size];
        if (page < 0 || page >= p.pool.pages) {
            atomicCAS(p.status, 0, SPK_BAD_INDEX);
            return nullptr;
        }
        return p.pool.data + ((static_cast<size_t>(page) * p.pool.heads + kv) * tiles + j % p.pool.page_size / kv4::kTile) * p.pool.tile_bytes;
    };
    float top = -INFINITY, sum = 0.0f, acc[4] = {};
    const int ch = 4 * lane;
    for (int j0 = p.window > 0 ? max(0, pos - p.window + 1) : 0; j0 <= pos; j0 += 32) {
        const int j = j0 + lane;
        const unsigned char* tile = j <= pos ? tile_of(j) : nullptr;
        float s = -INFINITY;
        if (tile != nullptr) {
            s = 0.0f;
            const int in = j % kv4::kTile;
            for (int c = 0; c < D; c += 8) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + kv4::k_word_at(D, in, c));
                const uint32_t word = *reinterpret_cast<const uint32_t*>(tile + kv4::k_words_at(D) + (in * (D / G) + c / G) * 4);
#pragma unroll
                for (int i = 0; i < 8; ++i) s = fmaf(fmaf(static_cast<float>(w >> (4 * i) & 15u), kv4::word_scale(word), kv4::word_min(word)), qs[warp][c + i], s);
            }
        }
        float most = s;
        for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        most = fmaxf(most, top);
        const float base = most == -INFINITY ? 0.0f : most, keep = exp2f(top - base);
        const float e = tile != nullptr ? exp2f(s - base) : 0.0f;
        top = most;
        sum = sum * keep + e;
        for (int i = 0; i < 4; ++i) acc[i] *= keep;
        const unsigned seen = __ballot_sync(0xffffffffu, tile != nullptr);
        for (int o = 0; o < 32; ++o) {
            if (!(seen >> o & 1u)) continue;
            const float w = __shfl_sync(0xffffffffu, e, o);
            const unsigned char* from = reinterpret_cast<const unsigned char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(tile), o));
            if (ch >= D) continue;
            const int in = (j0 + o) % kv4::kTile;
            const uint32_t codes = *reinterpret_cast<const uint16_t*>(from + kv4::v_codes_at(D) + kv4::v_piece_at(D, in, ch % 32 / 4) + ch / 32 * 2);
            const uint32_t word = *reinterpret_cast<const uint32_t*>(from + kv4::v_words_at(D, G) + (in * (D / G) + ch / G) * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = fmaf(w, fmaf(static_cast<float>(codes >> (4 * i) & 15u), kv4::word_scale(word), kv4::word_min(word)), acc[i]);
        }
    }
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (ch < D)
        for (int i = 0; i < 4; ++i)
            p.out[(static_cast<size_t>(t) * p.q_heads + h) * D + ch + i] = __float2bfloat16_rn(top == -INFINITY ? 0.0f : acc[i] / sum);
}

template <int D, int G>
int attend(const AttendParams& p, cudaStream_t stream) {
    const int64_t warps = int64_t{p.batch.rows} * p.q_heads;
    SPK_CUDA(launch_chained(kv4_attend_rows_kernel<D, G>, dim3(static_cast<unsigned>(cdiv64(warps, 8))), dim3(256), 0, stream, p));
    return SPK_OK;
}

}  // namespace
}  // namespace spk

extern "C" long long spk_kv4_attention_workspace(int rows, int seqs, int q_heads, int kv_heads, int head_dim) { return 16; }

extern "C" int spk_kv4_attention(const void* q, long long q_stride, const void* pool, int pages, int page_size, int q_heads, int kv_heads,
                                 int head_dim, int group, const int32_t* page_table, int table_width, const int32_t* lens,
                                 const int32_t* q_offsets, int seqs, int rows, float scale, int window, void* out, int zero_rest,
                                 void* workspace, long long workspace_bytes, void* stream_) {
    using namespace spk;
    if (int rc = kv4::check("kv4_attention", pool, pages, page_size, kv_heads, head_dim, group)) return rc;
    AttendParams p{};
    p.batch = {page_table, lens, q_offsets, seqs, rows, table_width};
    if (int rc = kv4::check_batch("kv4_attention", p.batch)) return rc;
    SPK_REQUIRE(q_heads >= 1 && q_heads <= 16384 && q_heads % kv_heads == 0, "kv4_attention: q_heads must be a multiple of kv_heads, at most 16384, got %d and %d", q_heads, kv_heads);
    SPK_REQUIRE(window >= 0, "kv4_attention: window must be 0 (none) or positive, got %d", window);
    SPK_REQUIRE(scale == scale && scale >= -3e38f && scale <= 3e38f, "kv4_attention: scale must be finite");
    if (rows == 0) return SPK_OK;
    SPK_REQUIRE(q && out && aligned16(q) && aligned16(out), "kv4_attention: q and out must be 16-byte aligned device pointers");
    SPK_REQUIRE(q_stride >= static_cast<long long>(q_heads) * head_dim && q_stride % 8 == 0, "kv4_attention: rows of q must be at least q_heads head_dim apart and a multiple of 8, got %lld", q_stride);
    SPK_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= spk_kv4_attention_workspace(rows, seqs, q_heads, kv_heads, head_dim),
                "kv4_attention: the workspace must be 16-byte aligned and hold spk_kv4_attention_workspace() bytes, got %lld", workspace_bytes);
    DeviceState* dev = nullptr;
    if (int rc = device_state(&dev)) return rc;
    p.q = static_cast<const __nv_bfloat16*>(q), p.stride = q_stride;
    p.pool = {static_cast<unsigned char*>(const_cast<void*>(pool)), pages, page_size, kv_heads, kv4::tile_bytes(head_dim, group)};
    p.q_heads = q_heads, p.window = window, p.zero_rest = zero_rest, p.scale = scale;
    p.out = static_cast<__nv_bfloat16*>(out), p.status = dev->status;
    auto stream = static_cast<cudaStream_t>(stream_);
    if (head_dim == 64) return group == 32 ? attend<64, 32>(p, stream) : attend<64, 64>(p, stream);
    return group == 32 ? attend<128, 32>(p, stream) : group == 64 ? attend<128, 64>(p, stream) : attend<128, 128>(p, stream);
}
