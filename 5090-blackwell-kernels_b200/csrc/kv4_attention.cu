// Attention over the 4-bit paged KV cache (its bytes: kv4_layout.cuh): for a row (token at position p, query head)
//     out = sum_j softmax_j(scale q . k_j) v_j   over the positions j <= p, with a window only p - window < j,
// k_j and v_j being c s + m, the codes and words of the cache.
//
// One pass over the keys with the running maximum and sum of the softmax, everything between the loads and the output in
// registers. The rows that read one KV head (its query heads times the call's tokens of the sequence) are taken 8 NQ at a
// time as the n side of warp-level MMAs whose 16-row side is the cache:
//     S^T [16 tokens x rows] = K codes [16 x d] . Q^T,        O^T [channels x rows] += V codes^T [channels x 16 tokens] . P^T
// The codes go into the MMA as small integers in fp16, built by one LOP3 per pair (a nibble or-ed into the mantissa of
// 1024 reads 1024 + c, one nibble higher into that of 64 reads 64 + c); the words are applied outside it:
//     K  q . k = sum over groups of s (sum (c + o) q' - sum o q') + m sum q'   with the o-sums of q as the accumulator's start;
//        q' = q 2^(13 - e) (e the exponent of the row's largest |q|; kv4_attend.cuh) fits fp16 exactly, but for channels below
//        2^-30 of the largest; the products are exact in fp32, and four to eight MMAs a group leave the offset no room to cost precision
//     V  sum p v = sum (p s)(c - 8) + sum p (8 s + m): here the offsets are taken out before the MMA (a sum over the whole
//        sequence of values with a large common offset would drift), and the second sum is fp32. p s is rounded to fp16
//        (2^-11 of it, unbiased; bf16 would lose another half step of the output) times a power of two of its row's and
//        group's own, which puts the largest p s so far at 2^3 to 2^4: rounded in full down to 2^-17 of that, gone below
//        2^-28, so that a group loses at most keys x 2^-28 of its largest p s, however loud other groups, or tokens without
//        weight, may be. (One power for a warp, after its largest s, was 2 % faster and lost the groups 2^20 below it.)
// P^T comes out of S^T's accumulator layout by movmatrix (one 8 x 8 transpose per register).
//
// Work is cut into equal contiguous ranges of (sequence, block of rows, KV head, 16-token tile) units over the resident
// warps, whatever the lengths are; every warp finds its range itself from the lengths on the device and walks it alone,
// through a ring of its own filled by bulk copies. What a warp holds of a piece that is cut across warps is added up in
// the CTA at its end, what crosses CTAs goes through the workspace to a second, chained launch; always in the order of the
// units: the same bits every run. (Adding by whichever CTA is last, on counters, was slower: 43.2 -> 45.6 us at 64 x 4k.)
//
// Bound: instructions, then memory. A tile of 16 tokens and a head costs about 280 warp instructions (88 to build the codes'
// fragments, 32 to centre V's, 16 MMAs, the rest words, softmax and ring), at 2.3 a cycle and SM 122 cycles for 2176 to 2560
// bytes, which HBM delivers in 94 to 110. 32 heads over 8, d = 128, in a graph: 8 sequences of 65536 125.4 us = 4.55 TB/s (0.70 of the
// measured copy; the same copies without the arithmetic take 100 us); 64 sequences of up to 4096 41.7 us = 3.19 TB/s; one of
// 200 10.2 us, of which the second launch is 2.5. Prompts: kv4_prompt.cu.
#include <algorithm>

#include "kv4_attend.cuh"
#include "ptx_sm100.cuh"

namespace spk {
namespace {

using kv4::AttendParams;

constexpr int kSteps = 2;     // 16-token tiles of a ring stage
constexpr int kMinUnits = 8;  // a CTA gets at least this many units
// Units that stand in front of a piece's tiles for what its beginning costs (q, the lengths, the end's sums). Without them
// a batch with short sequences waits for the warps that got many (64 x 4k, ragged: 60.1 us with 0, 56.6 / 47.7 / 43.5 / 42.0 / 43.3
// with 1 / 3 / 6 / 10 / 16). With 0 / 5 / 10 / 20: 16 x 4097 29.5 / 26.4 / 27.7 / 28.0, 64 x 1000 31.5 / 29.4 / 28.7 / 31.7, 256 x 300 40
// with all, 8 x 65536 125 with all, 32 x 8000 with a window of 1024 24.1 / 22.2 / 22.3 / 23.7.
constexpr int kLead = 10;
constexpr int kMaxWarps = 7;  // consuming warps of a CTA, of any form

constexpr int kMaxGrid = 2 * 160, kMinGrid = 64;  // two CTAs on every SM of the part, with room; fewer than any sm_100 part has

// H = 2 is the form for at most four rows a KV head (NQ = 1): a row has two of the eight columns, each for half of the
// groups, so that the scales of one group are all a column ever meets.
//
// W consuming warps and one that fills their rings, C such blocks on an SM: seven and two, at 128 registers a thread; seven and one
// where 16 rows' accumulators take more. Five and two, with nothing spilled, is as fast at 64 x 4k and 6 % slower at 8 x 64k;
// nine and two spills in the loop and takes twice as long. 24 rows a block spills too (76 us against 45 for 16 x 5 rows on
// 6001), and 8 rows a block instead of 16 reads the cache more often (57 us). Two of the forms spill as they are, with groups of
// 32: d = 64 with 16 rows (542 bytes stored, 704 loaded) and d = 128 with 8 (458, 572). With one block on an SM they are
// faster: 64 sequences of 4096 with 16 query heads a KV head 88 us for 115, with 8 heads of 128 98 for 115.
template <int D, int G, int NQ, int H, int W, int C>
struct SplitCfg {
    static constexpr int kRows = 8 * NQ / H, kGroups = D / G / H, kWords = D / 32;
    static constexpr int kThreads = 32 * (W + 1);
    static constexpr int kTileBytes = kv4::tile_bytes(D, G), kStageBytes = kSteps * kTileBytes;
    // a task per warp; barriers and valid flags of six stages
    static constexpr int kTask = (NQ * kWords * 512 + (NQ * kGroups * 2 + NQ * 3) * 32 + 64 + 127) / 128 * 128;
    static constexpr int kSmall = W * kTask + W * 6 * 20 + 64;
    static constexpr int kFit = ((227 * 1024 - 1024 * C) / C - 2048 - kSmall) / (W * kStageBytes);
    static constexpr int kStages = kFit < 6 ? kFit : 6;
    static constexpr int kRing = W * kStages * kStageBytes, kSmem = kRing + kSmall;
    static constexpr int kPart = kRows * (D + 2);  // floats: values, then maximum and sum of every row
};

// A sequence and its place in the order of units.
struct Seq {
    int b, first, count, len;  // its rows of q, its tokens
    int lo, hi;                // tiles of 16 tokens that any of its rows sees
    bool other;                // a prompt, and the prompts are another launch's
    long long begin, units;    // units before it, its own: row blocks x KV heads x (lead + tiles)
};

__device__ __forceinline__ void load_seq(const AttendParams& p, int rows, bool prompts, Seq& s) {
    kv4::rows_of(p.batch, s.b, s.first, s.count);
    s.len = kv4::length_of(p.batch, p.pool.page_size, s.b, p.status);
    s.hi = s.count > 0 ? (s.len + kv4::kTile - 1) / kv4::kTile : 0;
    s.lo = p.window > 0 && s.count > 0 ? max(0, s.len - s.count - p.window + 1) / kv4::kTile : 0;
    const int group = p.q_heads / p.pool.heads;
    s.other = prompts && kv4::prompt_blocks(static_cast<long long>(s.count) * group) > 0;
    s.units = s.other ? 0 : static_cast<long long>((s.count * group + rows - 1) / rows) * p.pool.heads * (s.hi > s.lo ? s.hi - s.lo + kLead : 0);
}

// What a range holds of one (sequence, block of rows, KV head).
struct Piece {
    int block, head;
    int units;           // how far the range goes in it
    int tile0, tiles;    // tiles from the sequence's start; none where the range ends in the lead
    bool begins, ends;   // whether the range holds the piece's first and last tile
};

// The piece at unit u; s is the sequence that holds an earlier unit, and becomes the one that holds u.
__device__ __forceinline__ Piece piece_at(const AttendParams& p, int rows, bool prompts, long long u, long long end, Seq& s) {
    while (s.begin + s.units <= u) {
        s.begin += s.units;
        ++s.b;
        load_seq(p, rows, prompts, s);
    }
    const int n = s.hi - s.lo + kLead;
    const long long local = u - s.begin;
    const int which = local >> 32 ? static_cast<int>(local / n) : static_cast<int>(static_cast<uint32_t>(local) / n);  // a 64-bit division is long
    const int skip = static_cast<int>(local - static_cast<long long>(which) * n);
    Piece x;
    x.block = which / p.pool.heads, x.head = which - x.block * p.pool.heads;
    x.units = static_cast<int>(min(static_cast<long long>(n - skip), end - u));
    const int from = max(0, skip - kLead), to = max(0, skip + x.units - kLead);
    x.tile0 = s.lo + from, x.tiles = to - from;
    x.begins = from == 0, x.ends = skip + x.units == n;
    return x;
}

// A token's words, one per group, in one load.
template <int N>
__device__ __forceinline__ void load_words(const uint32_t* at, uint32_t (&w)[N]) {
    if constexpr (N == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(at);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(at);
        w[0] = v.x, w[1] = v.y;
    } else {
        w[0] = *at;
    }
}

// A piece as the warp that works on it needs it, in shared memory.
template <int D, int G, int NQ, int H>
struct Task {
    static constexpr int kGroups = D / G / H, kWords = D / 32;  // groups a column meets
    // the rows' q as B fragments (column g: row g, or row g % 4 in the channels of half g / 4), one 16-byte piece a lane:
    // word i's step A (even channels) b0, b1, step B (odd ones) b0, b1
    uint4 q[NQ][kWords][32];
    // by column: the offsets' start value and the sum of q' per group, the score's factor, the tokens its row sees
    float start[NQ][kGroups][8], q_sum[NQ][kGroups][8], mult[NQ][8];
    int lo[NQ][8], hi[NQ][8];
    int all_lo, all_hi, any_lo, any_hi;  // tokens that every row sees, that any row sees
    int tile0, tiles, block, head, first, count;
};

// What a warp leaves of a piece it holds in part.
struct Member {
    int block, head, first, count, seq, begins, ends;
    const float* at;  // values [rows][D], maxima and sums [rows][2]
    long long end;    // the unit behind the piece
};

// What a warp carries through the tiles of a piece.
template <int D, int G, int NQ, int H>
struct State {
    static constexpr int kGroups = D / G / H;  // groups a column meets
    // of the task, for this lane's accumulator columns 2 c and 2 c + 1
    float start[NQ][kGroups][2], q_sum[NQ][kGroups][2], mult[NQ][2];
    // the running softmax: maxima (in powers of two), sums, values (channels 32 u + 4 g + {0, 2} in o[2 u], {1, 3} in o[2 u + 1]), sum p (8 s + m)
    float top[NQ][2], sum[NQ][2], o[NQ][D / 16][4], z[NQ][kGroups][2];
    // by column and group, the power of two that p s is multiplied by before fp16 and that o carries; and, of what this lane
    // reads, the largest |s| with which no p up to 2^kSlack makes p s too large for fp16
    float lift[NQ][kGroups][2], safe[kGroups];
};

// The running maximum lags behind by up to kSlack; the largest p s of a column and group, seen from there, is lifted to 2^(kLift - 1)
// to 2^kLift, and p s may reach 2^15.
constexpr float kSlack = 6.0f;
constexpr int kLift = 4;
__device__ __forceinline__ float lift_of(float largest) {  // 2^126 for none
    const int e = static_cast<int>((__float_as_uint(largest) + 0x7fffffu) >> 23);
    return __uint_as_float(static_cast<uint32_t>(min(254 + kLift - e, 253)) << 23);
}
__device__ __forceinline__ float inverse_of(float power) { return __uint_as_float((254u << 23) - __float_as_uint(power)); }

// kSteps tiles of 16 tokens. Masked: some token is out of some row's sight, or a tile is missing (ok: the tiles that are there).
template <int D, int G, int NQ, int H, bool Masked>
__device__ __forceinline__ void attend_step(State<D, G, NQ, H>& st, const Task<D, G, NQ, H>& task, const unsigned char* tiles, int lane, int ok, int base) {
    constexpr int NG = D / G / H, NW = D / 32, kTileBytes = kv4::tile_bytes(D, G);
    const int g = lane >> 2, c = lane & 3;
    const int my_words = H == 2 ? (c >> 1) * NG * 4 : 0;  // where the words of this lane's columns begin in a token's
    float sc[NQ][kSteps][4], most[NG];
    uint32_t vw[kSteps][2][NG];
#pragma unroll
    for (int k = 0; k < NG; ++k) most[k] = 0.0f;
#pragma unroll
    for (int t = 0; t < kSteps; ++t) {
        const unsigned char* tile = tiles + t * kTileBytes;
        uint32_t kw[2][NG], code[2][NW];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            load_words(reinterpret_cast<const uint32_t*>(tile + kv4::k_words_at(D) + (g + 8 * x) * (D / G) * 4 + my_words), kw[x]);
            load_words(reinterpret_cast<const uint32_t*>(tile + kv4::v_words_at(D, G) + (g + 8 * x) * (D / G) * 4 + my_words), vw[t][x]);
            load_words(reinterpret_cast<const uint32_t*>(tile + (g + 8 * x) * (D / 2) + c * (D / 8)), code[x]);
            if (Masked) {  // what lies outside every row's sight may be anything, NaN among it
                const int j = base + t * kv4::kTile + g + 8 * x;
                const bool seen = (ok >> t & 1) && j >= task.any_lo && j < task.any_hi;
#pragma unroll
                for (int k = 0; k < NG; ++k) kw[x][k] = seen ? kw[x][k] : 0, vw[t][x][k] = seen ? vw[t][x][k] : 0;
            }
#pragma unroll
            for (int k = 0; k < NG; ++k) most[k] = fmaxf(most[k], fabsf(__uint_as_float(vw[t][x][k])));  // m in the low bits does not matter
        }
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            float acc[NQ][4];
            bool fresh = true;
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                if (32 * i / G % NG != k) continue;
                const uint32_t a0 = code[0][i], a1 = code[1][i], b0 = a0 >> 8, b1 = a1 >> 8;
                const uint32_t fa[4] = {ptx::lop3_and_or(a0, 0x000f000fu, 0x64006400u), ptx::lop3_and_or(a1, 0x000f000fu, 0x64006400u),
                                        ptx::lop3_and_or(b0, 0x000f000fu, 0x64006400u), ptx::lop3_and_or(b1, 0x000f000fu, 0x64006400u)};
                const uint32_t fb[4] = {ptx::lop3_and_or(a0, 0x00f000f0u, 0x54005400u), ptx::lop3_and_or(a1, 0x00f000f0u, 0x54005400u),
                                        ptx::lop3_and_or(b0, 0x00f000f0u, 0x54005400u), ptx::lop3_and_or(b1, 0x00f000f0u, 0x54005400u)};
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    const uint4 q = task.q[n][i][lane];
                    if (fresh) ptx::mma_f16_16816(acc[n], fa, q.x, q.y, st.start[n][k][0], st.start[n][k][1]);
                    else ptx::mma_f16_16816(acc[n], fa, q.x, q.y);
                    ptx::mma_f16_16816(acc[n], fb, q.z, q.w);
                }
                fresh = false;
            }
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const float s = kv4::word_scale(kw[x >> 1][k]), m = kv4::word_min(kw[x >> 1][k]), qs = st.q_sum[n][k][x & 1];
                    sc[n][t][x] = fmaf(s, acc[n][x], k == 0 ? m * qs : fmaf(m, qs, sc[n][t][x]));
                }
        }
        if (H == 2) {
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) sc[n][t][x] += __shfl_xor_sync(0xffffffffu, sc[n][t][x], 2);
        }
        // the scores as the softmax has them, rounded once: the largest minus the maximum is then 0 however large both are
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) sc[n][t][x] = __fmul_rn(sc[n][t][x], st.mult[n][x & 1]);
        if (Masked) {
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int j = base + t * kv4::kTile + g + 8 * (x >> 1);
                    const bool seen = (ok >> t & 1) && j >= task.lo[n][2 * c + (x & 1)] && j < task.hi[n][2 * c + (x & 1)];
                    sc[n][t][x] = seen ? sc[n][t][x] : -INFINITY;
                }
        }
    }
    // ---- running maximum and lifts: moved only when some score is 2^kSlack over the maximum or some s too large for the
    // lifts, so most steps need no shuffle
    float high[NQ][2];
    bool over = false;
#pragma unroll
    for (int k = 0; k < NG; ++k) over |= most[k] > st.safe[k];
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            float m = fmaxf(sc[n][0][x], sc[n][0][x + 2]);
#pragma unroll
            for (int t = 1; t < kSteps; ++t) m = fmaxf(m, fmaxf(sc[n][t][x], sc[n][t][x + 2]));
            high[n][x] = m;
            over |= high[n][x] > st.top[n][x] + kSlack;
        }
    if (__any_sync(0xffffffffu, over)) {
        float widest[NG];
#pragma unroll
        for (int k = 0; k < NG; ++k) widest[k] = INFINITY;
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float m = high[n][x];
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                m = fmaxf(m, st.top[n][x]);
                const float keep = st.top[n][x] == -INFINITY ? 0.0f : ptx::exp2_fast(st.top[n][x] - m);
                st.sum[n][x] *= keep;
                st.top[n][x] = m;
                const float shift = m == -INFINITY ? 0.0f : m;
                float p[kSteps][2];
#pragma unroll
                for (int t = 0; t < kSteps; ++t)
#pragma unroll
                    for (int y = 0; y < 2; ++y) p[t][y] = ptx::exp2_fast(sc[n][t][x + 2 * y] - shift);
#pragma unroll
                for (int k = 0; k < NG; ++k) {
                    st.z[n][k][x] *= keep;
                    // the largest p s: of the tokens before, of these (0 x infinity is passed over)
                    float largest = keep * 0x1p4f * inverse_of(st.lift[n][k][x]);
#pragma unroll
                    for (int t = 0; t < kSteps; ++t)
#pragma unroll
                        for (int y = 0; y < 2; ++y) largest = fmaxf(largest, p[t][y] * fabsf(kv4::word_scale(vw[t][y][k])));
                    largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 4));
                    largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 8));
                    largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 16));
                    const float lift = lift_of(largest), both = keep == 0.0f ? 0.0f : keep * (lift * inverse_of(st.lift[n][k][x]));
                    st.lift[n][k][x] = lift;
                    if (m != -INFINITY) widest[k] = fminf(widest[k], inverse_of(lift));
#pragma unroll
                    for (int i = 0; i < NW; ++i) {
                        if (32 * i / G % NG != k) continue;
#pragma unroll
                        for (int y = 0; y < 4; ++y) st.o[n][2 * i + (y >> 1)][x + 2 * (y & 1)] *= both;
                    }
                }
            }
#pragma unroll
        for (int k = 0; k < NG; ++k) st.safe[k] = 512.0f * widest[k];
    }
    // ---- weights and values
#pragma unroll
    for (int t = 0; t < kSteps; ++t) {
        const unsigned char* tile = tiles + t * kTileBytes;
        uint32_t pf[NQ][NG][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            float pr[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float m = Masked && st.top[n][x & 1] == -INFINITY ? 0.0f : st.top[n][x & 1];
                pr[x] = ptx::exp2_fast(sc[n][t][x] - m);
                st.sum[n][x & 1] += pr[x];
            }
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                float ps[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const uint32_t w = vw[t][x >> 1][k];
                    float sv = kv4::word_scale(w), mid = fmaf(8.0f, sv, kv4::word_min(w));
                    if (Masked && sc[n][t][x] == -INFINITY) sv = mid = 0.0f;  // a row that does not see the token: it may be a NaN
                    ps[x] = pr[x] * (sv * st.lift[n][k][x & 1]);
                    st.z[n][k][x & 1] = fmaf(pr[x], mid, st.z[n][k][x & 1]);
                }
                pf[n][k][0] = ptx::transpose_8x8(ptx::f16x2_pack(ps[0], ps[1]));
                pf[n][k][1] = ptx::transpose_8x8(ptx::f16x2_pack(ps[2], ps[3]));
            }
        }
        uint32_t w[2][NW];  // [half of the tile]: words of tokens 2 c, then of 2 c + 1
#pragma unroll
        for (int x = 0; x < 2; ++x) load_words(reinterpret_cast<const uint32_t*>(tile + kv4::v_codes_at(D) + x * 4 * D + g * (D / 2) + c * (D / 8)), w[x]);
#pragma unroll
        for (int unit = 0; unit < NW; ++unit) {  // channels 32 unit .. + 31
            const uint32_t pick = unit & 1 ? 0x7632u : 0x5410u;
            const uint32_t a = __byte_perm(w[0][unit / 2], w[0][unit / 2 + NW / 2], pick), b = __byte_perm(w[1][unit / 2], w[1][unit / 2 + NW / 2], pick);
            const uint32_t a8 = a >> 8, b8 = b >> 8;
            auto low = [](uint32_t v) { return ptx::f16x2_sub(ptx::lop3_and_or(v, 0x000f000fu, 0x64006400u), 0x64086408u); };   // 1024 + c - 1032
            auto high = [](uint32_t v) { return ptx::f16x2_sub(ptx::lop3_and_or(v, 0x00f000f0u, 0x54005400u), 0x54805480u); };  // 64 + c - 72
            const uint32_t fa[4] = {low(a), low(a8), low(b), low(b8)}, fb[4] = {high(a), high(a8), high(b), high(b8)};
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                ptx::mma_f16_16816(st.o[n][2 * unit], fa, pf[n][32 * unit / G % NG][0], pf[n][32 * unit / G % NG][1]);
                ptx::mma_f16_16816(st.o[n][2 * unit + 1], fb, pf[n][32 * unit / G % NG][0], pf[n][32 * unit / G % NG][1]);
            }
        }
    }
}

// Writes a task: the rows of the piece, scaled to fp16 and laid out as fragments, and what the columns need. One warp.
template <int D, int G, int NQ, int H>
__device__ __forceinline__ void write_task(const AttendParams& p, const Seq& seq, const Piece& s, Task<D, G, NQ, H>& task, int lane) {
    constexpr int NG = D / G / H, NW = D / 32, R = 8 * NQ / H;
    const int g = lane >> 2, c = lane & 3, group = p.q_heads / p.pool.heads;
    int all_lo = 0, all_hi = INT32_MAX, any_lo = INT32_MAX, any_hi = 0;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int row = s.block * R + 8 * n + (H == 2 ? g & 3 : g);  // this lane's column
        const bool there = row < seq.count * group;
        const int token = row / group;
        uint32_t raw[NW][4] = {}, most = 0;
        if (there) {
            const __nv_bfloat16* q = p.q + static_cast<long long>(seq.first + token) * p.stride + static_cast<long long>(s.head * group + row - token * group) * D + 8 * c;
#pragma unroll
            for (int i = 0; i < NW; ++i) load_words(reinterpret_cast<const uint32_t*>(q + 32 * i), raw[i]);
        }
#pragma unroll
        for (int i = 0; i < NW; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) most = __vmaxu2(most, raw[i][j] & 0x7fff7fffu);
        most = max(most >> 16, most & 0xffffu);
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int e = static_cast<int>(most >> 7);  // biased exponent of the row's largest |q|
        const bool finite = e < 255;
        const float to_fp16 = kv4::query_scale(e);
        float down = finite ? to_fp16 : 0.0f;
        const float up = finite ? kv4::query_unscale(to_fp16) : __uint_as_float(0x7fc00000u);
        if (p.scale < 0.0f) down = -down;
        uint4 q[NW];
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const bool mine = H == 1 || g / 4 == 32 * i / G / NG;
            float h[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t w = finite && mine ? raw[i][j] : 0;
                h[2 * j] = __uint_as_float(w << 16) * down, h[2 * j + 1] = __uint_as_float(w & 0xffff0000u) * down;
            }
            q[i] = make_uint4(ptx::f16x2_pack(h[0], h[4]), ptx::f16x2_pack(h[2], h[6]), ptx::f16x2_pack(h[1], h[5]), ptx::f16x2_pack(h[3], h[7]));
            task.q[n][i][lane] = q[i];
        }
        const int pos = seq.len - seq.count + token;
        const int hi = there ? max(0, pos + 1) : 0, lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
        if (c == 0) {
            // never 0: masked scores are -inf times it
            task.mult[n][g] = fmaxf(fabsf(p.scale) * (1.4426950408889634f * up), kv4::kLeast) + (up - up);
            task.lo[n][g] = lo, task.hi[n][g] = hi;
        }
        // the sums over a group of what the codes' offsets multiply: 1024 the even channels, 64 the odd ones
        const uint32_t ones[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            float even[4] = {}, odd[4] = {};
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                if (32 * i / G % NG != k) continue;
                ptx::mma_f16_16816(even, ones, q[i].x, q[i].y);
                ptx::mma_f16_16816(odd, ones, q[i].z, q[i].w);
            }
            if (g == 0) {
#pragma unroll
                for (int x = 0; x < 2; ++x) task.start[n][k][2 * c + x] = -fmaf(1024.0f, even[x], 64.0f * odd[x]), task.q_sum[n][k][2 * c + x] = even[x] + odd[x];
            }
        }
        if (there) all_lo = max(all_lo, lo), all_hi = min(all_hi, hi), any_lo = min(any_lo, lo), any_hi = max(any_hi, hi);
    }
    all_lo = __reduce_max_sync(0xffffffffu, all_lo), all_hi = __reduce_min_sync(0xffffffffu, all_hi);
    any_lo = __reduce_min_sync(0xffffffffu, any_lo), any_hi = __reduce_max_sync(0xffffffffu, any_hi);
    if (lane == 0) {
        task.all_lo = all_lo, task.all_hi = all_hi, task.any_lo = any_lo, task.any_hi = any_hi;
        task.tile0 = s.tile0, task.tiles = s.tiles, task.block = s.block, task.head = s.head;
        task.first = seq.first, task.count = seq.count;
    }
}

template <int D, int G, int NQ, int H, int W, int C>
__global__ void __launch_bounds__(32 * (W + 1), C)
kv4_attend_split_kernel(const AttendParams p) {
    using Cfg = SplitCfg<D, G, NQ, H, W, C>;
    using Task_ = Task<D, G, NQ, H>;
    constexpr int R = Cfg::kRows, NG = Cfg::kGroups, NW = Cfg::kWords, S = Cfg::kStages, kThreads = Cfg::kThreads;
    static_assert(W <= kMaxWarps, "the workspace's size");
    static_assert(S >= 2, "the ring needs two stages");
    static_assert(sizeof(Task_) <= Cfg::kTask && Cfg::kRing % 16 == 0, "the tasks' place in shared memory");
    static_assert(Cfg::kPart * 4 <= S * Cfg::kStageBytes && kThreads * 8 <= Cfg::kRing, "what the ring's memory is used for before and after");
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ Member members[2 * W];  // in the order of the units: what warp w began before its last piece, its last piece
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kRing + W * Cfg::kTask);
    int* valid_all = reinterpret_cast<int*>(bars + 2 * W * S);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    // a ring per consuming warp; the last warp's lane w fills that of warp w
    const int mine = warp < W ? warp : min(lane, W - 1);
    unsigned char* ring = smem + mine * S * Cfg::kStageBytes;
    uint64_t *full = bars + mine * 2 * S, *empty = full + S;
    int* valid = valid_all + mine * S;
    if (warp == W && lane < W) {
        for (int s = 0; s < 2 * S; ++s) ptx::mbar_init(&full[s], 1);
        ptx::fence_mbar_init();
        members[2 * lane].at = members[2 * lane + 1].at = nullptr;
    }
    pdl_release();
    pdl_wait();

    const int group = p.q_heads / p.pool.heads, tiles_per_page = p.pool.page_size / kv4::kTile;
    // rows of a sequence with nothing in sight, and rows that belong to no sequence
    auto zero_rows = [&](int from, int to) {
        const long long pieces = static_cast<long long>(max(0, to - from)) * p.q_heads * (D / 8);
        uint4* at = reinterpret_cast<uint4*>(p.out + static_cast<size_t>(from) * p.q_heads * D);
        for (long long i = threadIdx.x; i < pieces; i += kThreads) at[i] = make_uint4(0, 0, 0, 0);
    };
    // units before every chunk of sequences, one chunk a thread
    const int chunk = (p.batch.seqs + kThreads - 1) / kThreads;
    long long* chunk_start = reinterpret_cast<long long*>(smem);  // in the ring's memory, before it is used
    long long total;
    bool prompts = false;
    if (p.prompts) {  // as the other launch counts them
        __shared__ int blocks;
        if (threadIdx.x == 0) blocks = 0;
        __syncthreads();
        long long n = 0;
        for (int b = threadIdx.x; b < p.batch.seqs; b += kThreads) {
            int first, count;
            kv4::rows_of(p.batch, b, first, count);
            n += kv4::prompt_blocks(static_cast<long long>(count) * group) * p.pool.heads;
        }
        if (n > 0) atomicAdd(&blocks, static_cast<int>(min(n, 1ll << 20)));
        __syncthreads();
        prompts = blocks >= kv4::kPromptBlocks;
    }
    {
        __shared__ long long warp_sum[W + 1];
        __shared__ int empties, empty_seqs[kv4::kMaxSeqs / kMinGrid];  // of the ones that fall to this CTA
        if (threadIdx.x == 0) empties = 0;
        __syncthreads();
        long long units = 0;
        for (int i = 0; i < chunk; ++i) {
            Seq s;
            s.b = threadIdx.x * chunk + i;
            if (s.b >= p.batch.seqs) break;
            load_seq(p, R, prompts, s);
            units += s.units;
            if (s.units == 0 && !s.other && s.count > 0 && s.b % gridDim.x == blockIdx.x) empty_seqs[atomicAdd(&empties, 1)] = s.b;
        }
        long long run = units;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const long long up = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += up;
        }
        if (lane == 31) warp_sum[warp] = run;
        __syncthreads();
        long long before = 0;
        total = 0;
        for (int w = 0; w <= W; ++w) {
            if (w < warp) before += warp_sum[w];
            total += warp_sum[w];
        }
        chunk_start[threadIdx.x] = before + run - units;
        __syncthreads();
        for (int i = 0; i < empties; ++i) {
            int first, count;
            kv4::rows_of(p.batch, empty_seqs[i], first, count);
            zero_rows(first, first + count);
        }
    }
    if (p.zero_rest && blockIdx.x == gridDim.x - 1) {
        const int head = p.batch.seqs > 0 ? min(max(p.batch.offsets[0], 0), p.batch.rows) : 0;
        const int tail = p.batch.seqs > 0 ? min(max(p.batch.offsets[p.batch.seqs], 0), p.batch.rows) : 0;
        zero_rows(0, head);
        zero_rows(tail, p.batch.rows);
    }
    // the CTAs that work, and this warp's range (a filling lane: that of its warp)
    const long long active = max(1ll, min(static_cast<long long>(gridDim.x), (total + kMinUnits - 1) / kMinUnits));
    if (blockIdx.x >= active || total == 0) {
        if (threadIdx.x == 0) p.pieces[blockIdx.x] = make_int4(0, 0, 0, 0);
        return;
    }
    const long long cta_start = blockIdx.x * total / active, cta_end = (blockIdx.x + 1) * total / active;
    const long long start = cta_start + mine * (cta_end - cta_start) / W, end = cta_start + (mine + 1) * (cta_end - cta_start) / W;
    Seq seq;
    if (start < end) {
        int at = 0;
        for (int hi = kThreads - 1; at < hi;) {
            const int mid = (at + hi + 1) >> 1;
            if (chunk_start[mid] <= start) at = mid; else hi = mid - 1;
        }
        seq.b = min(at * chunk, p.batch.seqs - 1);
        seq.begin = chunk_start[at];
        load_seq(p, R, prompts, seq);
    }
    ptx::fence_proxy_async();
    __syncthreads();  // chunk_start has been read: its place is the copies' now

    float* const parts = p.partials + static_cast<size_t>(blockIdx.x) * (2 + W) * Cfg::kPart;
    if (warp == W) {
        // ---- the filling warp: each lane walks its consuming warp's range, page numbers a step early ------------------
        long long u = start;
        int left = 0, at = 0, in_page = 0, page = 0, next_page = 0, slot = 0;  // tiles left of the piece; the step's place in the table
        const int32_t* row = nullptr;
        const unsigned char* base = nullptr;
        const long long page_bytes = static_cast<long long>(p.pool.heads) * tiles_per_page * Cfg::kTileBytes;
        unsigned phase = 1;  // the first round of a ring is free
        int filled = 0;
        auto settle = [&]() {  // to this lane's next step; false at the end of the range
            while (left <= 0) {
                if (u >= end) return false;
                const Piece s = piece_at(p, R, prompts, u, end, seq);
                u += s.units;
                left = s.tiles;
                at = s.tile0 / tiles_per_page, in_page = s.tile0 - at * tiles_per_page;
                row = p.batch.table + static_cast<size_t>(seq.b) * p.batch.width;
                base = p.pool.data + static_cast<size_t>(s.head) * tiles_per_page * Cfg::kTileBytes;
            }
            page = __ldg(row + at);
            next_page = left > 1 && in_page + 1 == tiles_per_page ? __ldg(row + at + 1) : page;
            return true;
        };
        static_assert(kSteps == 2, "a step spans at most two pages");
        bool filling = lane < W && settle();
        long long since = clock64();
        while (__any_sync(0xffffffffu, filling)) {
            bool went = false;
            if (filling && ptx::mbar_test_wait(&empty[slot], phase)) {
                went = true;
                const int n = min(left, kSteps);
                int ok = (page >= 0 && page < p.pool.pages ? 1 : 0) | (next_page >= 0 && next_page < p.pool.pages ? 2 : 0);
                if (ok != 3) kv4::bad_index(p.status);
                ok &= (1 << n) - 1;
                valid[slot] = ok;
                unsigned char* to = ring + slot * Cfg::kStageBytes;
                const unsigned char* from = base + page * page_bytes + in_page * Cfg::kTileBytes;
                if (ok == 3 && in_page + 1 < tiles_per_page) {  // both tiles in one page: one copy
                    ptx::mbar_arrive_expect_tx(&full[slot], 2 * Cfg::kTileBytes);
                    ptx::bulk_g2s(to, from, 2 * Cfg::kTileBytes, &full[slot]);
                } else {
                    ptx::mbar_arrive_expect_tx(&full[slot], ((ok & 1) + (ok >> 1)) * Cfg::kTileBytes);
                    if (ok & 1) ptx::bulk_g2s(to, from, Cfg::kTileBytes, &full[slot]);
                    if (ok & 2) ptx::bulk_g2s(to + Cfg::kTileBytes, base + next_page * page_bytes, Cfg::kTileBytes, &full[slot]);
                }
                left -= kSteps;
                in_page += kSteps;
                while (in_page >= tiles_per_page) in_page -= tiles_per_page, ++at;
                if (++slot == S) slot = 0, phase ^= 1u;
                ++filled;
                filling = settle();
            }
            if (__any_sync(0xffffffffu, went)) {
                since = clock64();
            } else {
                if (__any_sync(0xffffffffu, clock64() - since > 2 * ptx::kWaitCycles)) {  // the consumers gave up
                    if (lane == 0) atomicCAS(p.status, 0, SPK_TIMEOUT);
                    break;
                }
                __nanosleep(20);
            }
        }
        // no copy is on its way when the block ends, even if its consumer gave up on it: the last one into each slot has landed
        for (int k = max(0, filled - S); k < filled; ++k) ptx::mbar_wait(&full[k % S], (k / S) & 1, p.status);
    } else {
        // ---- a consuming warp -----------------------------------------------------------------------------------------
        Task_& task = *reinterpret_cast<Task_*>(smem + Cfg::kRing + warp * Cfg::kTask);
        int slot = 0;
        unsigned phase = 0;
        bool alive = true;
        State<D, G, NQ, H> st;
        for (long long u = start; u < end;) {
            const Piece s = piece_at(p, R, prompts, u, end, seq);
            u += s.units;
            if (s.tiles == 0) continue;
            write_task<D, G, NQ, H>(p, seq, s, task, lane);
            __syncwarp();
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    st.mult[n][x] = task.mult[n][2 * c + x];
                    st.top[n][x] = -INFINITY, st.sum[n][x] = 0.0f;
#pragma unroll
                    for (int k = 0; k < NG; ++k) {
                        st.start[n][k][x] = task.start[n][k][2 * c + x], st.q_sum[n][k][x] = task.q_sum[n][k][2 * c + x];
                        st.z[n][k][x] = 0.0f, st.lift[n][k][x] = lift_of(0.0f);
                    }
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) st.o[n][i][x] = st.o[n][i][x + 2] = 0.0f;
                }
#pragma unroll
            for (int k = 0; k < NG; ++k) st.safe[k] = INFINITY;  // the first score that any row sees is over its maximum
            int base = s.tile0 * kv4::kTile;
            for (int left = s.tiles; left > 0; left -= kSteps, base += kSteps * kv4::kTile) {
                if (alive) alive = __all_sync(0xffffffffu, ptx::mbar_wait(&full[slot], phase, p.status));
                const int ok = valid[slot];  // of the tiles that the step has
                const unsigned char* tiles = ring + slot * Cfg::kStageBytes;
                if (ok != (1 << kSteps) - 1 || base < task.all_lo || base + kSteps * kv4::kTile > task.all_hi)
                    attend_step<D, G, NQ, H, true>(st, task, tiles, lane, left < kSteps ? ok & 1 : ok, base);
                else
                    attend_step<D, G, NQ, H, false>(st, task, tiles, lane, ok, base);
                __syncwarp();
                if (lane == 0 && alive) ptx::mbar_arrive(&empty[slot]);  // a copy that was given up on may still write to the slot
                if (++slot == S) slot = 0, phase ^= 1u;
            }

            // ---- what the warp has of the piece: to the output if that is all of it, else kept for the CTA's end
            const bool whole = s.begins && s.ends, last = u >= end;
            float* part = last ? reinterpret_cast<float*>(ring) : parts + (2 + warp) * Cfg::kPart;
            const int first = task.first, count = task.count, block = s.block, head = s.head;
            if (last) __syncwarp();  // every lane is past the ring
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) {
                        st.sum[n][x] += __shfl_xor_sync(0xffffffffu, st.sum[n][x], d);
#pragma unroll
                        for (int k = 0; k < NG; ++k) st.z[n][k][x] += __shfl_xor_sync(0xffffffffu, st.z[n][k][x], d);
                    }
                    const bool second = H == 2 && c >= 2;  // H = 2: a lane's columns hold one half of the channels
                    const int row = 8 * n + (H == 2 ? (2 * c + x) & 3 : 2 * c + x), r = block * R + row;
                    const float l = st.sum[n][x], k = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
                    __nv_bfloat16* to = p.out + (static_cast<size_t>(first + r / group) * p.q_heads + head * group + r % group) * D + 4 * g;
#pragma unroll
                    for (int i = 0; i < NW / H; ++i) {
                        const int ch = 32 * (second ? i + NW / 2 : i);
                        float f[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float a = st.o[n][2 * i + (j & 1)][x + (j & 2)], b = st.o[n][(2 * i + (j & 1) + (H - 1) * NW) % (D / 16)][x + (j & 2)];
                            f[j] = fmaf((second ? b : a) * k, inverse_of(st.lift[n][32 * i / G % NG][x]), st.z[n][32 * i / G % NG][x] * k);
                        }
                        if (!whole) {
                            *reinterpret_cast<float4*>(part + row * D + ch + 4 * g) = make_float4(f[0], f[1], f[2], f[3]);
                        } else if (r < count * group) {
                            const __nv_bfloat162 v = __floats2bfloat162_rn(f[0], f[1]), w = __floats2bfloat162_rn(f[2], f[3]);
                            *reinterpret_cast<uint2*>(to + ch) = make_uint2(*reinterpret_cast<const uint32_t*>(&v), *reinterpret_cast<const uint32_t*>(&w));
                        }
                    }
                    if (!whole && lane < 4 / H) part[R * D + 2 * row] = st.top[n][x], part[R * D + 2 * row + 1] = st.sum[n][x];
                }
            if (!whole && lane == 0) {
                Member& m = members[2 * warp + (last ? 1 : 0)];
                m.block = block, m.head = head, m.first = first, m.count = count, m.seq = seq.b, m.begins = s.begins, m.ends = s.ends;
                m.at = part, m.end = u + (seq.hi - s.tile0 - s.tiles);
            }
            __syncwarp();  // the task's place is free
        }
    }

    // ---- the CTA's members, chained: one begins a piece, the next ones go on with it ----------------------------------------
    __syncthreads();
    int4 entry = make_int4(0, 0, 0, 0);
    for (int i = 0; i < 2 * W;) {
        if (members[i].at == nullptr) {
            ++i;
            continue;
        }
        const Member& m = members[i];
        int stop = i + 1, n = 1;
        bool ends = m.ends;
        for (; !ends && stop < 2 * W; ++stop)
            if (members[stop].at != nullptr) ends = members[stop].ends, ++n;
        const bool whole = m.begins && ends;
        float* part = parts + (m.begins ? 1 : 0) * Cfg::kPart;
        for (int e = threadIdx.x; e < R * (D / 4); e += kThreads) {
            const int row = e / (D / 4), ch = e % (D / 4) * 4;
            float top = -INFINITY, l = 0.0f;
            for (int k = i; k < stop; ++k)
                if (members[k].at != nullptr) top = fmaxf(top, members[k].at[R * D + 2 * row]);
            float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int k = i; k < stop; ++k) {
                const float* from = members[k].at;
                if (from == nullptr) continue;
                const float t = from[R * D + 2 * row], w = t == -INFINITY ? 0.0f : ptx::exp2_fast(t - top);
                const float4 v = *reinterpret_cast<const float4*>(from + row * D + ch);
                a.x = fmaf(v.x, w, a.x), a.y = fmaf(v.y, w, a.y), a.z = fmaf(v.z, w, a.z), a.w = fmaf(v.w, w, a.w);
                l = fmaf(from[R * D + 2 * row + 1], w, l);
            }
            if (whole) {
                const int r = m.block * R + row;
                if (r >= m.count * group) break;
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                const __nv_bfloat162 x = __floats2bfloat162_rn(a.x * inv, a.y * inv), y = __floats2bfloat162_rn(a.z * inv, a.w * inv);
                *reinterpret_cast<uint2*>(p.out + (static_cast<size_t>(m.first + r / group) * p.q_heads + m.head * group + r % group) * D + ch) =
                    make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
            } else {
                *reinterpret_cast<float4*>(part + row * D + ch) = a;
                if (ch == 0) part[R * D + 2 * row] = top, part[R * D + 2 * row + 1] = l;
            }
        }
        // a piece that begins here and goes on: its parts are in this CTA and the ones after it
        if (m.begins && !ends) entry = make_int4(static_cast<int>((m.end * active - 1) / total) - static_cast<int>(blockIdx.x) + 1, m.seq, m.block, m.head);
        i = stop;
    }
    if (threadIdx.x == 0) p.pieces[blockIdx.x] = entry;
}

// Adds the parts of the pieces that were cut across CTAs: block (i, j) rows 4 j .. + 3 of the piece that began in CTA i of the launch
// before. A long sequence alone has a part in every fifth CTA: groups of threads take every so-manieth part, four loads at a time.
constexpr int kAddThreads = 512;

template <int D, int R, int W>
__global__ void __launch_bounds__(kAddThreads) kv4_attend_add_kernel(const AttendParams p) {
    pdl_release();
    pdl_wait();
    const int4 piece = p.pieces[blockIdx.x];
    if (piece.x == 0) return;
    constexpr int kPart = R * (D + 2), kPer = (2 + W) * kPart;  // a CTA's parts in the workspace
    constexpr int kGroups = kAddThreads / D;                    // a group: a thread for each four channels of the four rows
    __shared__ float4 sums[kGroups][D];
    __shared__ float2 tops[kGroups][D];
    const int head_group = p.q_heads / p.pool.heads;
    int first, count;
    kv4::rows_of(p.batch, piece.y, first, count);
    const float* mine = p.partials + static_cast<size_t>(blockIdx.x) * kPer;
    auto part = [&](int i) { return i == 0 ? mine + kPart : mine + static_cast<size_t>(i) * kPer; };
    const int item = threadIdx.x % D, group = threadIdx.x / D;
    const int row = 4 * blockIdx.y + item / (D / 4), ch = item % (D / 4) * 4, r = piece.z * R + row;
    float m = -INFINITY, l = 0.0f;
    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k0 = group; k0 < piece.x; k0 += 4 * kGroups) {
        float2 ms[4];
        float4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            ms[k] = make_float2(-INFINITY, 0.0f), v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (k0 + k * kGroups < piece.x) {
                const float* from = part(k0 + k * kGroups);
                ms[k] = *reinterpret_cast<const float2*>(from + R * D + 2 * row), v[k] = *reinterpret_cast<const float4*>(from + row * D + ch);
            }
        }
        const float now = fmaxf(fmaxf(fmaxf(ms[0].x, ms[1].x), fmaxf(ms[2].x, ms[3].x)), m);
        const float keep = m == -INFINITY ? 0.0f : ptx::exp2_fast(m - now);
        a.x *= keep, a.y *= keep, a.z *= keep, a.w *= keep, l *= keep, m = now;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float w = ms[k].x == -INFINITY ? 0.0f : ptx::exp2_fast(ms[k].x - now);
            a.x = fmaf(v[k].x, w, a.x), a.y = fmaf(v[k].y, w, a.y), a.z = fmaf(v[k].z, w, a.z), a.w = fmaf(v[k].w, w, a.w);
            l = fmaf(ms[k].y, w, l);
        }
    }
    sums[group][item] = a, tops[group][item] = make_float2(m, l);
    __syncthreads();
    if (group != 0 || r >= count * head_group) return;
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < kGroups; ++k) top = fmaxf(top, tops[k][item].x);
    a = make_float4(0.0f, 0.0f, 0.0f, 0.0f), l = 0.0f;
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
        const float2 ms = tops[k][item];
        const float4 v = sums[k][item];
        const float w = ms.x == -INFINITY ? 0.0f : ptx::exp2_fast(ms.x - top);
        a.x = fmaf(v.x, w, a.x), a.y = fmaf(v.y, w, a.y), a.z = fmaf(v.z, w, a.z), a.w = fmaf(v.w, w, a.w);
        l = fmaf(ms.y, w, l);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const __nv_bfloat162 x = __floats2bfloat162_rn(a.x * inv, a.y * inv), y = __floats2bfloat162_rn(a.z * inv, a.w * inv);
    *reinterpret_cast<uint2*>(p.out + (static_cast<size_t>(first + r / head_group) * p.q_heads + piece.w * head_group + r % head_group) * D + ch) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}

// Rows of a block. Up to four rows a KV head and sequence, and two groups or more: the form in which a row has two columns.
// Up to eight: one column each. More: sixteen at a time.
int rows_per_block(int rows, int seqs, int q_per_kv, int groups) {
    const int64_t r = static_cast<int64_t>(rows) * q_per_kv;
    return r <= int64_t{4} * seqs && groups > 1 ? 4 : r <= int64_t{8} * seqs ? 8 : 16;
}

template <int D, int G, int NQ, int H, int W, int C>
int attend(const AttendParams& p, DeviceState* dev, cudaStream_t stream) {
    using Cfg = SplitCfg<D, G, NQ, H, W, C>;
    auto kernel = kv4_attend_split_kernel<D, G, NQ, H, W, C>;
    static bool configured[kMaxDevices] = {};
    if (!configured[dev->device]) {
        SPK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem));
        configured[dev->device] = true;
    }
    const int grid = dev->sm_count * C < kMaxGrid ? dev->sm_count * C : kMaxGrid;
    if (grid < kMinGrid) return fail(SPK_UNSUPPORTED, "kv4_attention: needs at least %d SMs, the device has %d", kMinGrid, dev->sm_count);
    SPK_CUDA(launch_chained(kernel, dim3(grid), dim3(Cfg::kThreads), Cfg::kSmem, stream, p));
    SPK_CUDA(launch_chained(kv4_attend_add_kernel<D, Cfg::kRows, W>, dim3(grid, Cfg::kRows / 4), dim3(kAddThreads), 0, stream, p));
    return SPK_OK;
}
template <int D, int G>
int attend_rows(const AttendParams& p, int per_block, DeviceState* dev, cudaStream_t stream) {
    if constexpr (D / G > 1) {
        if (per_block == 4) return attend<D, G, 1, 2, 7, 2>(p, dev, stream);
    }
    if (per_block == 8) return attend<D, G, 1, 1, 7, 2>(p, dev, stream);
    if constexpr (D == 64) return attend<D, G, 2, 1, 7, 2>(p, dev, stream);
    else return attend<D, G, 2, 1, 7, 1>(p, dev, stream);
}

}  // namespace
}  // namespace spk

extern "C" long long spk_kv4_attention_workspace(int rows, int seqs, int q_heads, int kv_heads, int head_dim) {
    using namespace spk;
    if (rows < 0 || seqs < 0 || kv_heads < 1 || q_heads < kv_heads || head_dim < 1) return 0;
    return kMaxGrid * (16ll + (2ll + kMaxWarps) * rows_per_block(rows, seqs, q_heads / kv_heads, 1) * (head_dim + 2) * 4);
}

extern "C" int spk_kv4_attention(const void* q, long long q_stride, const void* pool, int pages, int page_size, int q_heads, int kv_heads,
                                 int head_dim, int group, const int32_t* page_table, int table_width, const int32_t* lens,
                                 const int32_t* q_offsets, int seqs, int rows, float scale, int window, void* out, int zero_rest,
                                 void* workspace, long long workspace_bytes, void* stream_) {
    using namespace spk;
    if (int rc = kv4::check("kv4_attention", pool, pages, page_size, kv_heads, head_dim, group)) return rc;
    AttendParams p{};
    p.batch = {page_table, lens, q_offsets, seqs, rows, table_width};
    if (int rc = kv4::check_batch("kv4_attention", p.batch, page_size)) return rc;
    SPK_REQUIRE(q_heads >= 1 && q_heads <= 16384 && q_heads % kv_heads == 0, "kv4_attention: q_heads must be a multiple of kv_heads, at most 16384, got %d and %d", q_heads, kv_heads);
    SPK_REQUIRE(window >= 0, "kv4_attention: window must be 0 (none) or positive, got %d", window);
    SPK_REQUIRE(scale == scale && scale >= -3e38f && scale <= 3e38f, "kv4_attention: scale must be finite");
    if (rows == 0) return SPK_OK;
    SPK_REQUIRE(q && out && q != out && aligned16(q) && aligned16(out), "kv4_attention: q and out must be two 16-byte aligned device pointers");
    SPK_REQUIRE(q_stride >= static_cast<long long>(q_heads) * head_dim && q_stride % 8 == 0, "kv4_attention: rows of q must be at least q_heads head_dim apart and a multiple of 8, got %lld", q_stride);
    SPK_REQUIRE(static_cast<long long>(rows) * (q_heads / kv_heads) <= INT32_MAX / 2, "kv4_attention: rows x query heads per KV head must stay below 2^30");
    SPK_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= spk_kv4_attention_workspace(rows, seqs, q_heads, kv_heads, head_dim),
                "kv4_attention: the workspace must be 16-byte aligned and hold spk_kv4_attention_workspace() bytes, got %lld", workspace_bytes);
    SPK_REQUIRE(!overlap(out, 2ll * rows * q_heads * head_dim, q, rows, q_stride, static_cast<long long>(q_heads) * head_dim), "kv4_attention: out must not be in q's memory");
    DeviceState* dev = nullptr;
    if (int rc = device_state(&dev)) return rc;
    p.q = static_cast<const __nv_bfloat16*>(q), p.stride = q_stride;
    p.pool = {static_cast<unsigned char*>(const_cast<void*>(pool)), pages, page_size, kv_heads, kv4::tile_bytes(head_dim, group)};
    p.q_heads = q_heads, p.window = window < 1 << 30 ? window : 0, p.zero_rest = zero_rest != 0 && q_offsets != nullptr, p.scale = scale;
    p.out = static_cast<__nv_bfloat16*>(out), p.status = dev->status;
    p.pieces = static_cast<int4*>(workspace);
    p.partials = reinterpret_cast<float*>(p.pieces + kMaxGrid);
    auto stream = static_cast<cudaStream_t>(stream_);
    // the most blocks of prompts there can be decides whether they are looked for at all
    const int64_t all_rows = int64_t{rows} * (q_heads / kv_heads);
    p.prompts = q_offsets != nullptr && all_rows >= kv4::kPromptRows &&
                (all_rows / kv4::kBlockRows + std::min<int64_t>(seqs, all_rows / kv4::kPromptRows)) * kv_heads >= kv4::kPromptBlocks;
    if (p.prompts) {
        if (int rc = kv4::attend_prompts(p, head_dim, group, dev, stream)) return rc;
    }
    const int per_block = rows_per_block(rows, seqs, q_heads / kv_heads, head_dim / group);
    if (head_dim == 64) return group == 32 ? attend_rows<64, 32>(p, per_block, dev, stream) : attend_rows<64, 64>(p, per_block, dev, stream);
    return group == 32 ? attend_rows<128, 32>(p, per_block, dev, stream) : group == 64 ? attend_rows<128, 64>(p, per_block, dev, stream) : attend_rows<128, 128>(p, per_block, dev, stream);
}
