// Writing and reading the 4-bit paged KV cache (its bytes: kv4_layout.cuh).
//
// kv4_append  takes the output of the qkv projection, rotates q and k by their positions, writes q, and puts k and v into
//             the cache as 4-bit codes, in one launch. The definition, in fp32 except where said:
//               y1 = x1 cos - x2 sin, y2 = x2 cos + x1 sin   (x1, x2 the halves of the first rot channels; products and
//                                                            sums rounded one by one; q rounded once more, to bf16)
//               per group: m = bf16(min y), s = bf16((max y - m) * fp32(1 / 15)), 0 where that is below 2^-126,
//                          c = clamp(rint((y - m) / s), 0, 15), 0 where s is 0
//             A group that holds an infinity or a NaN, or whose range is past fp32, reads back as NaN (s = 0, m = NaN).
//             The division is a true one: bf16 inputs often lie exactly on the border between two codes.
// kv4_read    the values c s + m of named tokens, rounded once to bf16.
//
// Both are bound by memory: a token of Hq = 32, Hkv = 8, d = 128 is 12 KiB of qkv in, 8 KiB of q and 1.1 KiB of cache out.
#include <cfloat>

#include "kv4_layout.cuh"

namespace spk {
namespace {

using kv4::Batch;
using kv4::Pool;

struct AppendParams {
    const __nv_bfloat16* qkv;
    long long stride;  // elements between rows of qkv
    Pool pool;
    Batch batch;
    const float* cos_sin;  // [positions][rot]: cosines, then sines
    int positions, rot, q_heads, zero_rest;
    __nv_bfloat16* q_out;
    int* status;
};

struct Four {
    float v[4];
};

__device__ __forceinline__ Four load4(const __nv_bfloat16* p) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    return {{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u)}};
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const Four& x) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x.v[0], x.v[1]), b = __floats2bfloat162_rn(x.v[2], x.v[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// A head vector belongs to D / 4 neighbouring lanes, lane l of them holding channels 4 l .. 4 l + 3: the rotation's
// partner channels and a group's extremes are then shuffles inside the warp.
template <int D>
__device__ __forceinline__ void rotate(Four& x, int l, const float* cs, int rot) {
    const int quads = rot >> 3;  // lanes of one half
    const bool first = l < quads, in = l < 2 * quads;
    const int partner = first ? l + quads : in ? l - quads : l;
    Four other;
#pragma unroll
    for (int i = 0; i < 4; ++i) other.v[i] = __shfl_sync(0xffffffffu, x.v[i], partner, D / 4);
    if (!in) return;
    const int at = 4 * (first ? l : l - quads);
    const float4 c = *reinterpret_cast<const float4*>(cs + at), s = *reinterpret_cast<const float4*>(cs + rot / 2 + at);
    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = __fmul_rn(x.v[i], cc[i]), b = __fmul_rn(other.v[i], ss[i]);
        x.v[i] = first ? __fsub_rn(a, b) : __fadd_rn(a, b);
    }
}

// The four codes of this lane (nibble i: channel 4 l + i) and its group's word.
template <int G>
__device__ __forceinline__ uint32_t quantize4(const Four& x, uint32_t& word) {
    float lo = fminf(fminf(x.v[0], x.v[1]), fminf(x.v[2], x.v[3])), hi = fmaxf(fmaxf(x.v[0], x.v[1]), fmaxf(x.v[2], x.v[3]));
    int finite = 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) finite &= fabsf(x.v[i]) <= FLT_MAX;
#pragma unroll
    for (int o = 1; o < G / 4; o *= 2) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        finite &= __shfl_xor_sync(0xffffffffu, finite, o);
    }
    const __nv_bfloat16 mb = __float2bfloat16_rn(lo);
    const float m = __bfloat162float(mb);
    const __nv_bfloat16 sb = __float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, m), 1.0f / 15.0f));
    float s = __bfloat162float(sb);
    if (!finite || !(s <= FLT_MAX) || !(fabsf(m) <= FLT_MAX)) {
        word = 0x7fc0u;
        return 0;
    }
    if (s < FLT_MIN) s = 0.0f;  // a group of one value, or one whose minimum was rounded up past its maximum
    word = __float_as_uint(s) | __bfloat16_as_ushort(mb);
    uint32_t codes = 0;
    if (s > 0.0f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) codes |= static_cast<uint32_t>(min(max(__float2int_rn(__fdiv_rn(__fsub_rn(x.v[i], m), s)), 0), 15)) << (4 * i);
    }
    return codes;
}

// Block: eight tokens, one per warp, and the heads of slice blockIdx.y. Neighbouring tokens of a sequence share V blocks,
// so their pieces leave the SM close together.
template <int D, int G>
__global__ void __launch_bounds__(256) kv4_append_kernel(const AppendParams p) {
    constexpr int kLanes = D / 4, kPer = 32 / kLanes;  // lanes of a head vector, head vectors of a warp
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % kLanes;
    pdl_release();
    pdl_wait();
    const int t = blockIdx.x * 8 + warp;
    if (t >= p.batch.rows) return;

    // the token's sequence, position and place in the pool
    int b = t;
    if (p.batch.offsets != nullptr) {
        int passed = 0;
        for (int i = lane; i < p.batch.seqs; i += 32) passed += p.batch.offsets[i + 1] <= t;
        b = static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(passed)));
    }
    int pos = -1;
    bool known = b < p.batch.seqs;
    if (known) {
        int first, count;
        kv4::rows_of(p.batch, b, first, count);
        known = t >= first && t < first + count;
        pos = kv4::length_of(p.batch, p.pool.page_size, b, p.status) - count + (t - first);
    }
    if (!known && !p.zero_rest) return;
    if (known && pos >= p.positions) {
        if (lane == 0) atomicCAS(p.status, 0, SPK_BAD_INDEX);
        pos = -1;
    }
    const bool placed = known && pos >= 0;
    unsigned char* tile = nullptr;  // of KV head 0
    const int tiles = p.pool.page_size / kv4::kTile;
    if (placed) {
        const int page = p.batch.table[static_cast<size_t>(b) * p.batch.width + pos / p.pool.page_size];
        if (page < 0 || page >= p.pool.pages) {
            if (lane == 0) atomicCAS(p.status, 0, SPK_BAD_INDEX);
        } else {
            tile = p.pool.data + (static_cast<size_t>(page) * p.pool.heads * tiles + pos % p.pool.page_size / kv4::kTile) * p.pool.tile_bytes;
        }
    }
    const int in_tile = placed ? pos % kv4::kTile : 0;
    const float* cs = p.cos_sin + static_cast<size_t>(placed ? pos : 0) * p.rot;
    const int total = p.q_heads + 2 * p.pool.heads;
    const __nv_bfloat16* row = p.qkv + static_cast<size_t>(t) * p.stride;

    for (int h0 = blockIdx.y * kPer; h0 < total; h0 += gridDim.y * kPer) {
        const int h = h0 + lane / kLanes;
        const bool here = h < total;
        Four x = {};
        if (placed && here) x = load4(row + static_cast<size_t>(h) * D + 4 * l);
        // the shuffles below are the whole warp's: a warp of two head vectors may hold one of each kind
        if (p.rot > 0 && placed) {
            Four y = x;
            rotate<D>(y, l, cs, p.rot);
            if (h < p.q_heads + p.pool.heads) x = y;
        }
        uint32_t word = 0, codes = 0;
        if (h0 + kPer > p.q_heads) codes = quantize4<G>(x, word);
        const int kv = (h - p.q_heads) % p.pool.heads;
        const bool is_k = h < p.q_heads + p.pool.heads;
        // K: two lanes make a 32-bit word; V: the lanes of one run put their half words together
        const uint32_t upper = __shfl_down_sync(0xffffffffu, codes, 1);
        uint32_t piece[D / 64];
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
            piece[i] = __shfl_sync(0xffffffffu, codes, (l & 7) + 16 * i, kLanes) | __shfl_sync(0xffffffffu, codes, (l & 7) + 16 * i + 8, kLanes) << 16;
        if (!here) continue;
        if (h < p.q_heads) {
            store4(p.q_out + (static_cast<size_t>(t) * p.q_heads + h) * D + 4 * l, x);
            continue;
        }
        if (tile == nullptr) continue;
        unsigned char* at = tile + static_cast<size_t>(kv) * tiles * p.pool.tile_bytes;
        if (is_k) {
            if ((l & 1) == 0) *reinterpret_cast<uint32_t*>(at + kv4::k_word_at(D, in_tile, 4 * l)) = codes | upper << 16;
        } else if (l < 8) {
            unsigned char* to = at + kv4::v_codes_at(D) + kv4::v_piece_at(D, in_tile, l);
            if constexpr (D == 128) *reinterpret_cast<uint2*>(to) = make_uint2(piece[0], piece[D / 64 - 1]);
            else *reinterpret_cast<uint32_t*>(to) = piece[0];
        }
        if (l % (G / 4) == 0)
            *reinterpret_cast<uint32_t*>(at + (is_k ? kv4::k_words_at(D) : kv4::v_words_at(D, G)) + (in_tile * (D / G) + 4 * l / G) * 4) = word;
    }
}

struct ReadParams {
    Pool pool;
    const long long* slots;
    int n;
    __nv_bfloat16 *k, *v;
    int* status;
};

// A warp reads one token of one head, K and V: lane l the 4 channels 4 l .. (D = 128) or the halves of the warp one tensor each.
template <int D, int G>
__global__ void __launch_bounds__(256) kv4_read_kernel(const ReadParams p) {
    pdl_release();
    pdl_wait();
    constexpr int kQuads = D / 4;
    const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;  // (slot, head, K or V, quad)
    const int quad = static_cast<int>(i % kQuads);
    const bool is_v = (i / kQuads) & 1;
    const long long vec = i / (2 * kQuads);
    const int head = static_cast<int>(vec % p.pool.heads);
    const long long n = vec / p.pool.heads;
    if (n >= p.n) return;
    const long long slot = p.slots[n];
    Four x = {};
    if (slot >= 0 && slot < static_cast<long long>(p.pool.pages) * p.pool.page_size) {
        const int tiles = p.pool.page_size / kv4::kTile, in_page = static_cast<int>(slot % p.pool.page_size), t = in_page % kv4::kTile;
        const unsigned char* tile = p.pool.data + ((static_cast<size_t>(slot / p.pool.page_size) * p.pool.heads + head) * tiles + in_page / kv4::kTile) * p.pool.tile_bytes;
        const int ch = 4 * quad;
        const unsigned char* at = is_v ? tile + kv4::v_codes_at(D) + kv4::v_piece_at(D, t, ch % 32 / 4) + ch / 32 * 2 : tile + kv4::k_word_at(D, t, ch & ~7) + ch % 8 / 2;
        const uint32_t codes = *reinterpret_cast<const uint16_t*>(at);
        const uint32_t word = *reinterpret_cast<const uint32_t*>(tile + (is_v ? kv4::v_words_at(D, G) : kv4::k_words_at(D)) + (t * (D / G) + ch / G) * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) x.v[j] = fmaf(static_cast<float>(codes >> (4 * j) & 15u), kv4::word_scale(word), kv4::word_min(word));
    } else if (slot >= 0) {
        atomicCAS(p.status, 0, SPK_BAD_INDEX);
    }
    store4((is_v ? p.v : p.k) + (n * p.pool.heads + head) * D + 4 * quad, x);
}

template <template <int, int> class F, typename... A>
int for_shape(int d, int group, A&&... a) {
    if (d == 64) return group == 32 ? F<64, 32>::run(a...) : F<64, 64>::run(a...);
    return group == 32 ? F<128, 32>::run(a...) : group == 64 ? F<128, 64>::run(a...) : F<128, 128>::run(a...);
}

template <int D, int G>
struct Append {
    static int run(const AppendParams& p, int sms, cudaStream_t stream) {
        const int blocks = cdiv(p.batch.rows, 8), vectors = cdiv(p.q_heads + 2 * p.pool.heads, 128 / D);
        // few tokens: a slice of heads per block until the SMs hold eight blocks each
        const int slices = max(1, min(vectors, 8 * sms / blocks));
        SPK_CUDA(launch_chained(kv4_append_kernel<D, G>, dim3(blocks, slices), dim3(256), 0, stream, p));
        return SPK_OK;
    }
    static int max(int a, int b) { return a > b ? a : b; }
    static int min(int a, int b) { return a < b ? a : b; }
};
template <int D, int G>
struct Read {
    static int run(const ReadParams& p, cudaStream_t stream) {
        const int64_t threads = int64_t{p.n} * p.pool.heads * 2 * (D / 4);
        SPK_CUDA(launch_chained(kv4_read_kernel<D, G>, dim3(static_cast<unsigned>(cdiv64(threads, 256))), dim3(256), 0, stream, p));
        return SPK_OK;
    }
};

}  // namespace
}  // namespace spk

extern "C" int spk_kv4_tile_bytes(int head_dim, int group) { return spk::kv4::shape_ok(head_dim, group) ? spk::kv4::tile_bytes(head_dim, group) : 0; }

extern "C" int spk_kv4_append(const void* qkv, long long qkv_stride, void* pool, int pages, int page_size, int q_heads, int kv_heads, int head_dim,
                              int group, const int32_t* page_table, int table_width, const int32_t* lens, const int32_t* q_offsets, int seqs,
                              int rows, const float* cos_sin, int positions, int rot_dim, void* q_out, int zero_rest, void* stream) {
    using namespace spk;
    if (int rc = kv4::check("kv4_append", pool, pages, page_size, kv_heads, head_dim, group)) return rc;
    AppendParams p{};
    p.batch = {page_table, lens, q_offsets, seqs, rows, table_width};
    if (int rc = kv4::check_batch("kv4_append", p.batch)) return rc;
    SPK_REQUIRE(q_heads >= 0 && q_heads <= 16384, "kv4_append: q_heads must be in [0, 16384], got %d", q_heads);
    SPK_REQUIRE(rot_dim >= 0 && rot_dim <= head_dim && rot_dim % 8 == 0, "kv4_append: the rotated channels must be a multiple of 8, at most head_dim, got %d", rot_dim);
    if (rows == 0) return SPK_OK;
    SPK_REQUIRE(qkv && (q_out || q_heads == 0) && (cos_sin || rot_dim == 0), "kv4_append: null pointer");
    SPK_REQUIRE(rot_dim == 0 || positions >= 1, "kv4_append: the table of the rotation is empty");
    SPK_REQUIRE(aligned16(qkv) && aligned16(q_out) && aligned16(cos_sin), "kv4_append: qkv, q_out and cos_sin must be 16-byte aligned");
    SPK_REQUIRE(qkv_stride >= static_cast<long long>(q_heads + 2 * kv_heads) * head_dim && qkv_stride % 8 == 0,
                "kv4_append: rows of qkv must be at least (q_heads + 2 kv_heads) head_dim apart and a multiple of 8, got %lld", qkv_stride);
    DeviceState* dev = nullptr;
    if (int rc = device_state(&dev)) return rc;
    p.qkv = static_cast<const __nv_bfloat16*>(qkv), p.stride = qkv_stride;
    p.pool = {static_cast<unsigned char*>(pool), pages, page_size, kv_heads, kv4::tile_bytes(head_dim, group)};
    p.cos_sin = cos_sin, p.positions = rot_dim > 0 ? positions : INT32_MAX, p.rot = rot_dim, p.q_heads = q_heads, p.zero_rest = zero_rest;
    p.q_out = static_cast<__nv_bfloat16*>(q_out), p.status = dev->status;
    return for_shape<Append>(head_dim, group, p, dev->sm_count, static_cast<cudaStream_t>(stream));
}

extern "C" int spk_kv4_read(const void* pool, int pages, int page_size, int kv_heads, int head_dim, int group, const int64_t* slots, int n, void* k,
                            void* v, void* stream) {
    using namespace spk;
    if (int rc = kv4::check("kv4_read", pool, pages, page_size, kv_heads, head_dim, group)) return rc;
    SPK_REQUIRE(n >= 0 && static_cast<long long>(n) * kv_heads <= (1ll << 31), "kv4_read: slots x KV heads must be in [0, 2^31], got %d x %d", n, kv_heads);
    if (n == 0) return SPK_OK;
    SPK_REQUIRE(slots && k && v && aligned16(k) && aligned16(v), "kv4_read: null pointer, or k or v not 16-byte aligned");
    DeviceState* dev = nullptr;
    if (int rc = device_state(&dev)) return rc;
    ReadParams p{};
    p.pool = {static_cast<unsigned char*>(const_cast<void*>(pool)), pages, page_size, kv_heads, kv4::tile_bytes(head_dim, group)};
    p.slots = reinterpret_cast<const long long*>(slots), p.n = n;
    p.k = static_cast<__nv_bfloat16*>(k), p.v = static_cast<__nv_bfloat16*>(v), p.status = dev->status;
    return for_shape<Read>(head_dim, group, p, static_cast<cudaStream_t>(stream));
}
