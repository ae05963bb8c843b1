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
// Both are bound by memory first: a token of Hq = 32, Hkv = 8, d = 128 is 12 KiB of qkv in, 8 KiB of q and 1.1 KiB of cache out.
// 8192 such tokens: the append 42 us (4.3 TB/s, 0.66 of the measured copy; 29 M warp instructions at 2.7 a cycle and SM are
// what is above it), reading them back 11 us. 16 tokens: 4.7 us for the two in a graph.
#include <algorithm>
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

__device__ __forceinline__ Four unpack4(uint2 w) {
    return {{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u)}};
}
__device__ __forceinline__ uint2 load4(const __nv_bfloat16* p) { return __ldg(reinterpret_cast<const uint2*>(p)); }
__device__ __forceinline__ void store4(__nv_bfloat16* p, const Four& x) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x.v[0], x.v[1]), b = __floats2bfloat162_rn(x.v[2], x.v[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// A head vector belongs to L = D / 8 neighbouring lanes; lane l holds channels 4 l .. + 3 and, half a vector on, D / 2 + 4 l .. + 3.
// With all channels rotated these are each other's partners; with half of them or fewer the partner is another lane's first
// four channels, which come by shuffles; with a number between the two the partner's channels are loaded again.
enum class Rot { kAll, kHalf, kMost };
struct Pair {
    Four a, b;
};

// What a lane needs of the rotation of its token, the same for every head.
struct Turn {
    float4 ca, sa, cb, sb;  // of the channels in a and b
    int pa, pb;             // channel of the partners of a and b, -1: not rotated
    bool fa, fb;            // whether a and b lie in the first half of the rotated channels
};

template <int D>
__device__ __forceinline__ void turn_of(Turn& t, int l, const float* cs, int rot) {
    const int half = rot / 2;
    auto one = [&](int ch, float4& c, float4& s, int& partner, bool& first) {
        first = ch < half;
        partner = ch < rot ? (first ? ch + half : ch - half) : -1;
        c = make_float4(1.0f, 1.0f, 1.0f, 1.0f), s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (partner >= 0) {
            const float* at = cs + (first ? ch : ch - half);
            c = __ldg(reinterpret_cast<const float4*>(at)), s = __ldg(reinterpret_cast<const float4*>(at + half));
        }
    };
    one(4 * l, t.ca, t.sa, t.pa, t.fa);
    if (rot == D) {
        t.cb = t.ca, t.sb = t.sa, t.pb = 4 * l, t.fb = false;
    } else {
        one(D / 2 + 4 * l, t.cb, t.sb, t.pb, t.fb);
    }
}

// x1 cos - x2 sin or x2 cos + x1 sin, every product and sum rounded by itself.
__device__ __forceinline__ Four turned(const Four& x, const Four& partner, const float4& c, const float4& s, bool first) {
    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
    Four y;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float p = __fmul_rn(x.v[i], cc[i]), q = __fmul_rn(partner.v[i], ss[i]);
        y.v[i] = first ? __fsub_rn(p, q) : __fadd_rn(p, q);
    }
    return y;
}

// With R = kHalf all lanes of the warp call it.
template <int D, Rot R>
__device__ __forceinline__ Pair rotated(uint2 ra, uint2 rb, const __nv_bfloat16* vec, const Turn& t) {
    Pair x{unpack4(ra), unpack4(rb)};
    if constexpr (R == Rot::kAll) {
        return {turned(x.a, x.b, t.ca, t.sa, true), turned(x.b, x.a, t.ca, t.sa, false)};
    } else if constexpr (R == Rot::kHalf) {
        constexpr int L = D / 8;
        const int from = max(t.pa, 0) / 4;
        const uint2 partner = make_uint2(__shfl_sync(0xffffffffu, ra.x, from, L), __shfl_sync(0xffffffffu, ra.y, from, L));
        if (t.pa >= 0) x.a = turned(x.a, unpack4(partner), t.ca, t.sa, t.fa);
        return x;
    } else {
        if (t.pa >= 0) x.a = turned(x.a, unpack4(load4(vec + t.pa)), t.ca, t.sa, t.fa);
        if (t.pb >= 0) x.b = turned(x.b, unpack4(load4(vec + t.pb)), t.cb, t.sb, t.fb);
        return x;
    }
}

// Minimum and maximum that hand a NaN on.
__device__ __forceinline__ float min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float low4(const Four& x) { return min_nan(min_nan(x.v[0], x.v[1]), min_nan(x.v[2], x.v[3])); }
__device__ __forceinline__ float high4(const Four& x) { return max_nan(max_nan(x.v[0], x.v[1]), max_nan(x.v[2], x.v[3])); }

struct Scale {
    float m, s, inv;  // minimum, scale, 1 / scale
    uint32_t word;
};
// A group's scale from its extremes over `Lanes` neighbouring lanes.
template <int Lanes>
__device__ __forceinline__ Scale scale_of(float lo, float hi) {
#pragma unroll
    for (int o = 1; o < Lanes; o *= 2) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    Scale r;
    const __nv_bfloat16 mb = __float2bfloat16_rn(lo);
    r.m = __bfloat162float(mb);
    r.s = __bfloat162float(__float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, r.m), 1.0f / 15.0f)));
    if (r.s < FLT_MIN) r.s = 0.0f;  // a group of one value, or one whose minimum was rounded up past its maximum
    r.word = __float_as_uint(r.s) | __bfloat16_as_ushort(mb);
    // an infinity or a NaN in the group, or a range past fp32
    if (!(r.s <= FLT_MAX) || !(fabsf(r.m) <= FLT_MAX)) r.s = 0.0f, r.m = 0.0f, r.word = 0x7fc0u;
    r.inv = r.s > 0.0f ? __fdividef(1.0f, r.s) : 0.0f;
    return r;
}

// rint((x - m) / s) clamped to a code, four of them in the low 16 bits. The quotient has to be the correctly rounded one: bf16
// values often lie exactly on the border between two codes. It is had by Markstein's method (IBM Journal of Research and
// Development 34, 1990), an estimate from the reciprocal put right by its exact remainder: q + (d - q s) (1 / s) from a first
// q = d (1 / s) is that: d - q s is exact, what the last product leaves is 2^-45 of the quotient, and a quotient of 24 bits by
// s's 8 is never closer than 2^-33 to where the rounding turns. (Below 2^-100 the remainder falls out of fp32's range; there
// the division is made.) The rounding to an integer is an addition of 1.5 x 2^23, which leaves it in the low bits.
__device__ __forceinline__ uint32_t codes4(const Four& x, const Scale& g) {
    constexpr float kRound = 12582912.0f;
    int k[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float d = __fsub_rn(x.v[i], g.m), q = d * g.inv;
        k[i] = __float_as_int(fmaf(fmaf(-q, g.s, d), g.inv, q) + kRound);
    }
    if (g.s < 0x1p-100f && g.s > 0.0f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = __float_as_int(__fdiv_rn(__fsub_rn(x.v[i], g.m), g.s) + kRound);
    }
    constexpr int kZero = 0x4b400000;  // the bits of kRound: code 0
#pragma unroll
    for (int i = 0; i < 4; ++i) k[i] = min(max(k[i], kZero), kZero + 15);
    return static_cast<uint32_t>(k[0]) + 16u * k[1] + 256u * k[2] + 4096u * k[3];
}

// Block: eight tokens, one per warp, and the head vectors of slice blockIdx.y, kPer of them at a time. Neighbouring tokens
// of a sequence share V blocks, so their pieces leave the SM close together. Four blocks on an SM: with the registers that a half
// rotated head likes (71) there are three, and 5015 tokens of 20 + 2 x 20 heads of 64 take 2.9 us more of 25; with loads in
// place of the shuffles 1.1 more. (Where all channels rotate 64 registers do anyway; five blocks spill and gain nothing.)
template <int D, int G, Rot R>
__global__ void __launch_bounds__(256, 4) kv4_append_kernel(const AppendParams p) {
    constexpr int L = D / 8, kPer = 32 / L, kAhead = 4;  // lanes of a head vector, head vectors of a warp, loads in flight
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % L, sub = lane / L;
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
        if (lane == 0) kv4::bad_index(p.status);
        pos = -1;
    }
    const bool placed = known && pos >= 0;
    // this slice's head vectors: k's and v's, the longer work, then q's; a warp's step never holds q beside k or v
    const int q_steps = (p.q_heads + kPer - 1) / kPer, kv_steps = (2 * p.pool.heads + kPer - 1) / kPer;
    const int from = static_cast<int>(static_cast<long long>(q_steps + kv_steps) * blockIdx.y / gridDim.y);
    const int to = static_cast<int>(static_cast<long long>(q_steps + kv_steps) * (blockIdx.y + 1) / gridDim.y);
    const int q_from = max(from - kv_steps, 0), q_to = to - kv_steps, kv_to = min(to, kv_steps);
    if (!placed) {
        for (int i = q_from; i < q_to; ++i)
            if (i * kPer + sub < p.q_heads) {
                __nv_bfloat16* q = p.q_out + (static_cast<size_t>(t) * p.q_heads + i * kPer + sub) * D + 4 * l;
                store4(q, Four{}), store4(q + D / 2, Four{});
            }
        return;
    }
    unsigned char* tile = nullptr;  // of KV head 0
    const int tiles = p.pool.page_size / kv4::kTile, in_tile = pos % kv4::kTile;
    if (from < kv_to) {
        const int page = p.batch.table[static_cast<size_t>(b) * p.batch.width + pos / p.pool.page_size];
        if (page < 0 || page >= p.pool.pages) {
            if (lane == 0) kv4::bad_index(p.status);
        } else {
            tile = p.pool.data + (static_cast<size_t>(page) * p.pool.heads * tiles + pos % p.pool.page_size / kv4::kTile) * p.pool.tile_bytes;
        }
    }
    Turn turn;
    turn_of<D>(turn, l, p.cos_sin + static_cast<size_t>(pos) * p.rot, p.rot);
    const __nv_bfloat16* row = p.qkv + static_cast<size_t>(t) * p.stride;

    const __nv_bfloat16* kv_row = row + static_cast<size_t>(p.q_heads) * D;
    for (int i0 = from; i0 < kv_to && tile != nullptr; i0 += 2) {
        uint2 ra[2] = {}, rb[2] = {};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int h = (i0 + j) * kPer + sub;
            if (i0 + j < kv_to && h < 2 * p.pool.heads) ra[j] = load4(kv_row + h * D + 4 * l), rb[j] = load4(kv_row + h * D + D / 2 + 4 * l);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (i0 + j >= kv_to) break;  // the whole warp
            const int h = (i0 + j) * kPer + sub;
            const bool is_k = h < p.pool.heads;
            Pair x{unpack4(ra[j]), unpack4(rb[j])};
            if (R == Rot::kHalf || is_k) {
                const Pair y = rotated<D, R>(ra[j], rb[j], kv_row + h * D, turn);
                if (is_k) x = y;
            }
            uint32_t ca, cb, wa, wb;
            if constexpr (G == D) {
                const Scale g = scale_of<L>(min_nan(low4(x.a), low4(x.b)), max_nan(high4(x.a), high4(x.b)));
                ca = codes4(x.a, g), cb = codes4(x.b, g), wa = wb = g.word;
            } else {
                const Scale ga = scale_of<G / 4>(low4(x.a), high4(x.a)), gb = scale_of<G / 4>(low4(x.b), high4(x.b));
                ca = codes4(x.a, ga), cb = codes4(x.b, gb), wa = ga.word, wb = gb.word;
            }
            // K: two lanes make a 32-bit word of a and one of b; V: the lanes of one run put their half words together
            const uint32_t both = __byte_perm(ca, cb, 0x5410);
            const uint32_t next = __shfl_xor_sync(0xffffffffu, both, 1), across = __shfl_xor_sync(0xffffffffu, both, 8);
            if (h >= 2 * p.pool.heads) continue;
            unsigned char* at = tile + static_cast<size_t>(is_k ? h : h - p.pool.heads) * tiles * p.pool.tile_bytes;
            if (is_k) {
                if ((l & 1) == 0) {
                    *reinterpret_cast<uint32_t*>(at + kv4::k_word_at(D, in_tile, 4 * l)) = __byte_perm(both, next, 0x5410);
                    *reinterpret_cast<uint32_t*>(at + kv4::k_word_at(D, in_tile, D / 2 + 4 * l)) = __byte_perm(both, next, 0x7632);
                }
            } else if (l < 8) {
                unsigned char* piece = at + kv4::v_codes_at(D) + kv4::v_piece_at(D, in_tile, l);
                if constexpr (D == 128) *reinterpret_cast<uint2*>(piece) = make_uint2(__byte_perm(both, across, 0x5410), __byte_perm(both, across, 0x7632));
                else *reinterpret_cast<uint32_t*>(piece) = both;
            }
            uint32_t* words = reinterpret_cast<uint32_t*>(at + (is_k ? kv4::k_words_at(D) : kv4::v_words_at(D, G))) + in_tile * (D / G);
            if constexpr (G == D) {
                if (l == 0) words[0] = wa;
            } else {
                if (l % (G / 4) == 0) words[4 * l / G] = wa, words[(D / 2 + 4 * l) / G] = wb;
            }
        }
    }
    for (int i0 = q_from; i0 < q_to; i0 += kAhead) {
        uint2 ra[kAhead] = {}, rb[kAhead] = {};
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int h = (i0 + j) * kPer + sub;
            if (i0 + j < q_to && h < p.q_heads) ra[j] = load4(row + h * D + 4 * l), rb[j] = load4(row + h * D + D / 2 + 4 * l);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int h = (i0 + j) * kPer + sub;
            if (i0 + j >= q_to || (R != Rot::kHalf && h >= p.q_heads)) continue;
            const Pair y = rotated<D, R>(ra[j], rb[j], row + h * D, turn);
            if (h >= p.q_heads) continue;
            __nv_bfloat16* q = p.q_out + (static_cast<size_t>(t) * p.q_heads + h) * D + 4 * l;
            store4(q, y.a), store4(q + D / 2, y.b);
        }
    }
}

struct ReadParams {
    Pool pool;
    const long long* slots;
    int n;
    __nv_bfloat16 *k, *v;
    int* status;
};

// A warp reads a token: D / 8 lanes a head's keys and values, eight channels each, the heads of slice blockIdx.y. What hides
// the loads is other warps: with two or four heads' loads in flight, and the registers for them, 8192 tokens take 1.7 and 2.0 us more.
template <int D, int G>
__global__ void __launch_bounds__(256) kv4_read_kernel(const ReadParams p) {
    constexpr int L = D / 8, kPer = 32 / L;
    pdl_release();
    pdl_wait();
    const int lane = threadIdx.x & 31, ch = 8 * (lane % L), sub = lane / L, n = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (n >= p.n) return;
    const long long slot = p.slots[n];
    const bool there = slot >= 0 && slot < static_cast<long long>(p.pool.pages) * p.pool.page_size;
    if (slot >= 0 && !there) kv4::bad_index(p.status);
    const long long page = there ? slot / p.pool.page_size : 0;
    const int tiles = p.pool.page_size / kv4::kTile, in_page = there ? static_cast<int>(slot - page * p.pool.page_size) : 0, t = in_page % kv4::kTile;
    const unsigned char* tile = p.pool.data + (static_cast<size_t>(page) * p.pool.heads * tiles + in_page / kv4::kTile) * p.pool.tile_bytes;
    const int k_at = kv4::k_word_at(D, t, ch), v_at = kv4::v_codes_at(D) + kv4::v_piece_at(D, t, ch % 32 / 4) + ch / 32 * 2;
    const int word = (t * (D / G) + ch / G) * 4;
    auto write = [&](__nv_bfloat16* to, uint32_t codes, uint32_t w) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = fmaf(__uint_as_float((codes >> (4 * j) & 15u) | 0x4b000000u) - 8388608.0f, kv4::word_scale(w), kv4::word_min(w));
        uint32_t out[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
            out[j] = *reinterpret_cast<const uint32_t*>(&v);
        }
        *reinterpret_cast<uint4*>(to) = make_uint4(out[0], out[1], out[2], out[3]);
    };
#pragma unroll 1
    for (int head = blockIdx.y * kPer + sub; head < p.pool.heads; head += gridDim.y * kPer) {
        uint32_t kc = 0, vc = 0, kw = 0, vw = 0;
        if (there) {
            const unsigned char* at = tile + static_cast<size_t>(head) * tiles * p.pool.tile_bytes;
            kc = *reinterpret_cast<const uint32_t*>(at + k_at);
            vc = *reinterpret_cast<const uint16_t*>(at + v_at) | static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(at + v_at + D / 2)) << 16;
            kw = *reinterpret_cast<const uint32_t*>(at + kv4::k_words_at(D) + word), vw = *reinterpret_cast<const uint32_t*>(at + kv4::v_words_at(D, G) + word);
        }
        const size_t to = (static_cast<size_t>(n) * p.pool.heads + head) * D + ch;
        write(p.k + to, kc, kw), write(p.v + to, vc, vw);
    }
}

template <template <int, int> class F, typename... A>
int for_shape(int d, int group, A&&... a) {
    if (d == 64) return group == 32 ? F<64, 32>::run(a...) : F<64, 64>::run(a...);
    return group == 32 ? F<128, 32>::run(a...) : group == 64 ? F<128, 64>::run(a...) : F<128, 128>::run(a...);
}

template <int D, int G>
struct Append {
    static int run(const AppendParams& p, int sms, cudaStream_t stream) {
        constexpr int kPer = 256 / D;
        const int blocks = cdiv(p.batch.rows, 8), steps = cdiv(p.q_heads, kPer) + cdiv(2 * p.pool.heads, kPer);
        // the heads are sliced over blocks until there are several rounds of them (four live on an SM), or one step each
        const int slices = std::max(1, std::min(steps, 16 * sms / blocks));
        auto kernel = p.rot == D ? kv4_append_kernel<D, G, Rot::kAll> : p.rot <= D / 2 ? kv4_append_kernel<D, G, Rot::kHalf> : kv4_append_kernel<D, G, Rot::kMost>;
        SPK_CUDA(launch_chained(kernel, dim3(blocks, slices), dim3(256), 0, stream, p));
        return SPK_OK;
    }
};
template <int D, int G>
struct Read {
    static int run(const ReadParams& p, int sms, cudaStream_t stream) {
        const int blocks = cdiv(p.n, 8), steps = cdiv(p.pool.heads, 256 / D);
        const int slices = std::max(1, std::min(steps, 16 * sms / blocks));
        SPK_CUDA(launch_chained(kv4_read_kernel<D, G>, dim3(blocks, slices), dim3(256), 0, stream, p));
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
    if (int rc = kv4::check_batch("kv4_append", p.batch, page_size)) return rc;
    SPK_REQUIRE(q_heads >= 0 && q_heads <= 16384, "kv4_append: q_heads must be in [0, 16384], got %d", q_heads);
    SPK_REQUIRE(rot_dim >= 0 && rot_dim <= head_dim && rot_dim % 8 == 0, "kv4_append: the rotated channels must be a multiple of 8, at most head_dim, got %d", rot_dim);
    if (rows == 0) return SPK_OK;
    SPK_REQUIRE(qkv && (q_out || q_heads == 0) && (cos_sin || rot_dim == 0), "kv4_append: null pointer");
    SPK_REQUIRE(q_heads == 0 || qkv != q_out, "kv4_append: q_out must not be qkv's memory");
    SPK_REQUIRE(rot_dim == 0 || positions >= 1, "kv4_append: the table of the rotation is empty");
    SPK_REQUIRE(aligned16(qkv) && aligned16(q_out) && aligned16(cos_sin), "kv4_append: qkv, q_out and cos_sin must be 16-byte aligned");
    SPK_REQUIRE(qkv_stride >= static_cast<long long>(q_heads + 2 * kv_heads) * head_dim && qkv_stride % 8 == 0,
                "kv4_append: rows of qkv must be at least (q_heads + 2 kv_heads) head_dim apart and a multiple of 8, got %lld", qkv_stride);
    SPK_REQUIRE(!overlap(q_out, 2ll * rows * q_heads * head_dim, qkv, rows, qkv_stride, static_cast<long long>(q_heads + 2 * kv_heads) * head_dim),
                "kv4_append: q_out must not be in qkv's memory");
    DeviceState* dev = nullptr;
    if (int rc = device_state(&dev)) return rc;
    p.qkv = static_cast<const __nv_bfloat16*>(qkv), p.stride = qkv_stride;
    p.pool = {static_cast<unsigned char*>(pool), pages, page_size, kv_heads, kv4::tile_bytes(head_dim, group)};
    p.cos_sin = cos_sin, p.positions = rot_dim > 0 ? positions : INT32_MAX, p.rot = rot_dim, p.q_heads = q_heads, p.zero_rest = zero_rest != 0 && q_offsets != nullptr;
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
    return for_shape<Read>(head_dim, group, p, dev->sm_count, static_cast<cudaStream_t>(stream));
}
