// Attention of many rows over the 4-bit paged KV cache (prompts; the mathematics and the argument checks: kv4_attention.cu).
//
// A CTA takes 256 rows (new tokens x query heads of one KV head of a sequence) in two tiles of 128, one row a TMEM lane, and
// walks the keys 64 at a time:
//     S [row][key] = Q' K'^T        P = 2^(S c + b)        O [row][channel] += P V'
// with tcgen05.mma on fp16 operands, P (in S's place) from TMEM, the others from shared memory. Eight warps turn codes and
// words into K' and V', every value (c s + m) 2^-e rounded once to fp16 (2^-11 of it), e the exponent of 16 tokens' largest
// |m| + 15 s, so that nothing overflows or vanishes whatever the scale. S is put right by 2^e of the keys; for the values 2^e
// joins the softmax's exponent: with M the running maximum of score + e,
//     P = 2^(score + e - M + 4),      sum += P 2^-e,      out = O / sum,
// fp32 but for P's rounding to fp16. Values quieter than the loudest so far take the loudest's e, or one 16 above their own if that
// is less: V' has the room, and P would run out of it. So a value is held to 2^-11 of itself and 2^-32 of the largest so far, in
// whatever group, and a weight to 2^-11 and, while tokens are within 2^16 of each other, 2^-29 of the largest weight (one bit
// less for each past that). The tensor core's sums are fp32. Eight warps hold the softmax, a row a thread. M is the maximum
// of a row's first keys and moves only when weights come near fp16's end, so O (in TMEM) is rarely touched between the MMAs
// and the maximum rarely looked for (S is then read again: its 64 scores need not stay in registers until the weights are
// known to fit).
// K' rows are keys, 128 bytes = 64 channels wide (the order of the channels inside eights is the codes' own; Q' is
// stored in the same order); V' rows are keys too, and the MMA reads them MN-major; the order of its columns is the codes',
// put right when O is written.
//
// Bound: the roles' latencies, not the tensor cores (37 % active). 2 x 2048 new tokens on 6144 old ones, 32 heads over 8, d = 128:
// 680 us = 707 TFLOP/s (0.43 of the measured cuBLAS rate); a step of 64 keys takes some 2800 cycles where its MMAs take 1084
// and its exponentials 1024. By device clocks (taken at 654 us, before V's warps looked for the loudest values) a row warp has
// about 2300 cycles of work a step (1200 for the weights, the rest waits that are already over, TMEM loads and stores,
// exponents), a code warp 1900 every other step, an MMA warp 1600 (some hundred cycles for each MMA that it issues). 256 rows
// a block share the conversion of the codes; 128 keys a step would halve the fixed costs but leave TMEM no room for the
// scores to run ahead.
#include <algorithm>

#include "kv4_attend.cuh"
#include "umma_sm100.cuh"

namespace spk {
namespace {

using kv4::AttendParams;

// Five warpgroups: two of row warps, one that makes K', one that makes V', one whose first two warps issue the MMAs. The
// registers are dealt out again by warpgroup: 2 x 144 + 2 x 72 + 48 = 5 x 96.
constexpr int kKeys = 64, kRowWarps = 8, kKWarp = 8, kVWarp = 12, kMmaWarp = 16, kThreadsP = 640;
constexpr int kRowRegs = 144, kCodeRegs = 72, kMmaRegs = 48;
constexpr int kInfos = 8;       // steps whose exponents are kept: the code warps are at most four ahead of a row warp
// A weight at the maximum is 2^4, so that fp16 holds weights down to 2^-29 of it (2 x 2048 rows on 8192: 658 us with 2^0, 668 with 2^4,
// 678 with 2^6, 686 with 2^8: the higher, the more often the maximum moves).
constexpr int kLevel = 4;
constexpr float kMost = 60000.0f;  // what 16 weights may add up to before the maximum moves: then none overflows fp16
constexpr int kFit = 14;        // |K'|, |V'| < 2^14
constexpr int kSpare = 16;      // V' of tokens quieter than the loudest so far stays that many bits lower, at most

// What the code warps say of 16 keys: of the keys 2^(e - 14), and which are not finite; of the values e and 2^-e (negative if any
// is not finite), and then which, by group.
struct alignas(16) TileInfo {
    float k_unit;
    uint32_t bad_k;
    float v_exp, v_unit;
    uint32_t bad_v[4];
};

template <int N>
__device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <int D, int G>
struct PromptCfg {
    static constexpr int kTile = kv4::tile_bytes(D, G), kRaw = 4;
    static constexpr int kRows = 128 * D * 2;       // Q' of a tile of rows
    static constexpr int kOperand = kKeys * D * 2;  // K' or V' of a step
    static constexpr int kWords = 16 * (D / G);             // words of 16 keys, K's or V's
    static constexpr int kStep = kKeys / kv4::kTile * kTile;  // the cache's bytes of a step
    static constexpr int kSmem = 1024 + 2 * kRows + 4 * kOperand + kRaw * kStep + 16 * kWords * 8 + 16;
    // TMEM columns: S of both tiles, two buffers each (P in a buffer's first half), then O
    static constexpr int kS = 0, kO = 256, kCols = 512;
    static_assert(kO + 2 * D <= kCols, "TMEM");
};

struct PromptBars {
    // by stage; by tile of rows and buffer (a step's parity); by tile; by step; by slot
    uint64_t q_ready, k_full[2], v_full[2], s_full[2][2], p_full[2][2], before_last[2], o_full[2], drained[2], info[kInfos], raw_full[4], raw_empty[4];
};

// Eight codes (nibble n of w), four fp16 pairs (n, n + 4) of (c s + m).
__device__ __forceinline__ uint4 values8(uint32_t w, uint32_t s, uint32_t m) {
    const uint32_t w8 = w >> 8;
    return make_uint4(ptx::f16x2_fma(ptx::f16x2_sub(ptx::lop3_and_or(w, 0x000f000fu, 0x64006400u), 0x64006400u), s, m),
                      ptx::f16x2_fma(ptx::f16x2_sub(ptx::lop3_and_or(w, 0x00f000f0u, 0x54005400u), 0x54005400u), s, m),
                      ptx::f16x2_fma(ptx::f16x2_sub(ptx::lop3_and_or(w8, 0x000f000fu, 0x64006400u), 0x64006400u), s, m),
                      ptx::f16x2_fma(ptx::f16x2_sub(ptx::lop3_and_or(w8, 0x00f000f0u, 0x54005400u), 0x54005400u), s, m));
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(min(max(e, -126), 127) + 127) << 23); }

// Exponent above every |m| + 15 s of a warp's words (0 words for what is not there), at least -100.
__device__ __forceinline__ int exponent_of(uint32_t largest) {
    largest = __reduce_max_sync(0xffffffffu, largest);
    return max(static_cast<int>(largest >> 23) - 126, -100);
}

template <int D, int G>
__global__ void __launch_bounds__(kThreadsP, 1) kv4_attend_prompt_kernel(const AttendParams p) {
    using Cfg = PromptCfg<D, G>;
    constexpr int NG = D / G, NC = D / 8;  // groups and chunks of eight channels of a head vector
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
    unsigned char *q_smem = smem, *k_smem = q_smem + 2 * Cfg::kRows, *v_smem = k_smem + 2 * Cfg::kOperand, *raw_smem = v_smem + 2 * Cfg::kOperand;
    __shared__ PromptBars bars;
    __shared__ TileInfo infos[kInfos][4];
    __shared__ int loudest[kInfos];  // the exponent above the values of a step and of all before it
    __shared__ uint32_t raw_there[Cfg::kRaw];  // which tiles of a slot were copied
    __shared__ uint32_t tmem_slot;
    __shared__ int s_seq, s_block;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = p.q_heads / p.pool.heads, tiles_per_page = p.pool.page_size / kv4::kTile;
    pdl_wait();

    // ---- this CTA's sequence and block of rows: the last blocks, which see the most keys, first ---------------------------
    const int head = blockIdx.x % p.pool.heads, order = blockIdx.x / p.pool.heads;
    const int chunk = (p.batch.seqs + kThreadsP - 1) / kThreadsP;
    auto blocks_of = [&](int b) {
        int first, count;
        kv4::rows_of(p.batch, b, first, count);
        return static_cast<int>(kv4::prompt_blocks(static_cast<long long>(count) * group));
    };
    int n = 0;
    for (int i = 0; i < chunk; ++i)
        if (static_cast<int>(threadIdx.x) * chunk + i < p.batch.seqs) n += blocks_of(threadIdx.x * chunk + i);
    // the blocks before this thread's chunk, and all of them: each warp sums the warps before it
    __shared__ int warp_blocks[kThreadsP / 32];
    int run = n;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int up = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += up;
    }
    if (lane == 31) warp_blocks[warp] = run;
    if (threadIdx.x == 0) s_seq = s_block = 0;  // stays so only if offsets that overlap add up past 32 bits
    __syncthreads();
    int before = run - n, total = 0;
    for (int w = 0; w < kThreadsP / 32; ++w) {
        if (w < warp) before += warp_blocks[w];
        total += warp_blocks[w];
    }
    if (order >= total || static_cast<long long>(total) * p.pool.heads < kv4::kPromptBlocks) return;
    const int want = total - 1 - order;
    if (want >= before && want < before + n) {
        int at = want - before, b = threadIdx.x * chunk;
        while (at >= blocks_of(b)) at -= blocks_of(b++);
        s_seq = b, s_block = at;
    }
    if (threadIdx.x == 0) {
        ptx::mbar_init(&bars.q_ready, kRowWarps);
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&bars.k_full[i], 2), ptx::mbar_init(&bars.v_full[i], 2);
            for (int k = 0; k < 2; ++k) ptx::mbar_init(&bars.s_full[i][k], 1), ptx::mbar_init(&bars.p_full[i][k], 4);
            ptx::mbar_init(&bars.before_last[i], 1), ptx::mbar_init(&bars.o_full[i], 1), ptx::mbar_init(&bars.drained[i], 1);
        }
        for (int i = 0; i < kInfos; ++i) ptx::mbar_init(&bars.info[i], 4);
        for (int i = 0; i < Cfg::kRaw; ++i) ptx::mbar_init(&bars.raw_full[i], 1), ptx::mbar_init(&bars.raw_empty[i], 4);
        ptx::fence_mbar_init();
    }
    if (warp == kMmaWarp) umma::tmem_alloc(&tmem_slot, Cfg::kCols);
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = tmem_slot;
    pdl_release();  // only now: a kernel that starts beside this one may want TMEM too

    const int b = s_seq, block = s_block;
    int first, count;
    kv4::rows_of(p.batch, b, first, count);
    const int len = kv4::length_of(p.batch, p.pool.page_size, b, p.status), rows = count * group;
    // tokens that any row of the block sees: [any_lo, any_hi)
    const int last_row = min(rows, (block + 1) * kv4::kBlockRows) - 1;
    const int first_pos = len - count + block * kv4::kBlockRows / group, any_hi = max(0, len - count + last_row / group + 1);
    const int any_lo = p.window > 0 ? max(0, first_pos - p.window + 1) : 0;
    const int key0 = any_lo / kKeys * kKeys, steps = any_hi > key0 ? (any_hi - key0 + kKeys - 1) / kKeys : 0;
    const int tiles = last_row - block * kv4::kBlockRows >= 128 ? 2 : 1;  // tiles of 128 rows
    constexpr uint32_t kAll = 0xffffffffu;

    if (warp < kRowWarps) {
        registers_up<kRowRegs>();
        // ---- a row a thread ------------------------------------------------------------------------------------------------
        const int tile = warp >> 2;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const int row = block * kv4::kBlockRows + tile * 128 + (warp & 3) * 32 + lane;
        const bool there = row < rows;
        const int token = there ? row / group : 0;
        const __nv_bfloat16* q = p.q + static_cast<long long>(first + token) * p.stride + static_cast<long long>(head * group + (there ? row - token * group : 0)) * D;
        __nv_bfloat16* out = p.out + (static_cast<size_t>(first + token) * p.q_heads + head * group + (there ? row - token * group : 0)) * D;
        const int pos = len - count + token;
        const int hi = there ? max(0, pos + 1) : 0, lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
        uint32_t most = 0;
#pragma unroll 4
        for (int i = 0; i < NC; ++i) {
            const uint4 w = there ? __ldg(reinterpret_cast<const uint4*>(q) + i) : uint4{};
            most = __vmaxu2(__vmaxu2(most, w.x & 0x7fff7fffu), __vmaxu2(w.y & 0x7fff7fffu, __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu)));
        }
        const int e = static_cast<int>(max(most >> 16, most & 0xffffu) >> 7);  // biased exponent of the row's largest |q|
        const bool finite = e < 255;
        float down = kv4::query_scale(e);
        const float up = finite ? kv4::query_unscale(down) : __uint_as_float(0x7fc00000u);
        if (p.scale < 0.0f) down = -down;
        const float mult = fmaxf(fabsf(p.scale) * (1.4426950408889634f * up), kv4::kLeast) + (up - up);  // never 0: masked scores are -inf times it
        const bool work = tile < tiles && steps > 0;
        if (work) {
            const int r = (warp & 3) * 32 + lane;
            unsigned char* to = q_smem + tile * Cfg::kRows + r * 128;
#pragma unroll 4
            for (int i = 0; i < NC; ++i) {
                const uint4 w = there && finite ? __ldg(reinterpret_cast<const uint4*>(q) + i) : uint4{};
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
                float h[8];
#pragma unroll
                for (int k = 0; k < 4; ++k) h[2 * k] = __uint_as_float(u[k] << 16) * down, h[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u) * down;
                *reinterpret_cast<uint4*>(to + (i >> 3) * (128 * 128) + (((i & 7) ^ (r & 7)) << 4)) =
                    make_uint4(ptx::f16x2_pack(h[0], h[4]), ptx::f16x2_pack(h[1], h[5]), ptx::f16x2_pack(h[2], h[6]), ptx::f16x2_pack(h[3], h[7]));
            }
        }
        ptx::fence_proxy_async();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&bars.q_ready);

        const int all_hi = __reduce_min_sync(kAll, there ? hi : INT32_MAX), all_lo = __reduce_max_sync(kAll, there ? lo : 0);
        float top = hi > lo ? -INFINITY : 0.0f, sum = 0.0f;
        uint32_t poison = 0;  // groups of channels in which this row sees a value that is no number
        bool alive = true;
        const uint32_t o_at = tmem + lanes + Cfg::kO + tile * D;
        for (int j = 0; work && j < steps; ++j) {
            const int base = key0 + j * kKeys;
            const uint32_t s_at = tmem + lanes + Cfg::kS + tile * 128 + (j & 1) * 64;
            if (alive) alive = __all_sync(kAll, ptx::mbar_wait(&bars.s_full[tile][j & 1], (j >> 1) & 1, p.status));
            umma::fence_after_sync();
            if (alive) alive = __all_sync(kAll, ptx::mbar_wait(&bars.info[j % kInfos], (j / kInfos) & 1, p.status));
            const TileInfo* info = infos[j % kInfos];
            float unit[4], v_exp[4], v_unit[4];
            uint32_t bad = 0;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const float4 of = *reinterpret_cast<const float4*>(&info[t]);
                unit[t] = fmaxf(of.x * mult, kv4::kLeast), v_exp[t] = of.z, v_unit[t] = fabsf(of.w);
                bad |= __float_as_uint(of.y) | __float_as_uint(of.w) >> 31;
            }
            if (bad) {
                for (int t = 0; t < 4; ++t)
                    for (int i = 0; i < kv4::kTile; ++i) {
                        const int key = base + kv4::kTile * t + i;
                        if (key < lo || key >= hi) continue;
                        if (info[t].bad_k >> i & 1) poison = (1u << NG) - 1;
                        for (int k = 0; k < NG && info[t].v_unit < 0.0f; ++k) poison |= (info[t].bad_v[k] >> i & 1) << k;
                    }
            }
            // The weights under the present maximum. A row's first keys need it found, and so do scores so much larger than before that 16
            // weights add up to more than kMost: then S is read again (P does not yet stand in its place)
            uint32_t pr[32];
            float part[4], keep = 1.0f, now = 0.0f;
            bool look = __any_sync(kAll, top == -INFINITY);
#pragma unroll 1
            for (int tries = 0; tries < 2; ++tries) {
                float x[64];
                {
                    uint32_t a0[32], a1[32];
                    umma::tmem_ld_32x32(s_at, a0);
                    umma::tmem_ld_32x32(s_at + 32, a1);
                    umma::tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(a0[i]), x[i + 32] = __uint_as_float(a1[i]);
                }
                if (base < all_lo || base + kKeys > all_hi) {
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        if (base + i < lo || base + i >= hi) x[i] = -INFINITY;
                }
                if (look) {
                    float most_here = -INFINITY;
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        float m = x[16 * t];
#pragma unroll
                        for (int i = 1; i < 16; ++i) m = fmaxf(m, x[16 * t + i]);
                        most_here = fmaxf(most_here, fmaf(m, unit[t], v_exp[t]));
                    }
                    most_here -= kLevel;
                    keep = top == -INFINITY ? 0.0f : exp2f(top - fmaxf(top, most_here));
                    top = fmaxf(top, most_here);
                }
                // score + e is rounded as the maximum's was before the maximum leaves it: their difference is then 0 however large they are
                // (in one rounding what the maximum's lost would be a weight: 2^64 at a score of 10^9; 677 us for 682)
                const float shift = top == -INFINITY ? 0.0f : top;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const float2 by = make_float2(unit[t], unit[t]), add = make_float2(v_exp[t], v_exp[t]), less = make_float2(-shift, -shift);
                    float2 all = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        float2 e = ptx::add2(ptx::fma2(make_float2(x[16 * t + i], x[16 * t + i + 1]), by, add), less);
                        e.x = ptx::exp2_fast(e.x), e.y = ptx::exp2_fast(e.y);
                        all = ptx::add2(all, e);
                        pr[8 * t + i / 2] = ptx::f16x2_pack(e.x, e.y);
                    }
                    part[t] = all.x + all.y;
                }
                if (look || !__any_sync(kAll, fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])) > kMost)) break;
                look = true;
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) now = fmaf(part[t], v_unit[t], now);
            umma::tmem_st_32x32(s_at, pr);
            if (look) {
                if (j > 0) {
                    // O is the MMAs' until those of step j - 1 are done: S of step j + 1 comes after them
                    uint64_t* done = j + 1 < steps ? &bars.s_full[tile][(j + 1) & 1] : &bars.before_last[tile];
                    if (alive) alive = __all_sync(kAll, ptx::mbar_wait(done, j + 1 < steps ? ((j + 1) >> 1) & 1 : 0, p.status));
                    umma::fence_after_sync();
#pragma unroll 1
                    for (int at = 0; at < D; at += 32) {
                        uint32_t r[32];
                        umma::tmem_ld_32x32(o_at + at, r);
                        umma::tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * keep);
                        umma::tmem_st_32x32(o_at + at, r);
                    }
                }
                sum *= keep;
            }
            sum += now;
            umma::tmem_st_wait();
            umma::fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&bars.p_full[tile][j & 1]);
        }
        if (work && alive) __all_sync(kAll, ptx::mbar_wait(&bars.o_full[tile], 0, p.status));
        umma::fence_after_sync();
        if (!finite && hi > lo) poison = ~0u;
        const float inv = sum == 0.0f ? 0.0f : power_of_two(-kFit) / sum;
        if (tile < tiles) {
#pragma unroll
            for (int at = 0; at < D / 32; ++at) {
                uint32_t r[32] = {};
                if (work) {
                    umma::tmem_ld_32x32(o_at + 32 * at, r);
                    umma::tmem_ld_wait();
                }
                // column (D = 128): 16 g + 8 (u / 2) + 2 n + u % 2; (D = 64): 8 g + 2 n + u; channel 32 u + 4 g + n
#pragma unroll
                for (int u = 0; u < D / 32; ++u)
#pragma unroll
                    for (int half = 0; half < (D == 64 ? 2 : 1); ++half) {
                        uint32_t o[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            float f[2];
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                const int ch = 8 * half + 2 * k + y, g = ch / 4, nn = ch % 4;  // g within this run of 32 columns
                                const int col = D == 128 ? 16 * g + 8 * (u / 2) + 2 * nn + u % 2 : 8 * g + 2 * nn + u;
                                f[y] = poison >> (32 * u / G) & 1 ? __uint_as_float(0x7fc00000u) : __uint_as_float(r[col]) * inv;
                            }
                            const __nv_bfloat162 v = __floats2bfloat162_rn(f[0], f[1]);
                            o[k] = *reinterpret_cast<const uint32_t*>(&v);
                        }
                        if (there) *reinterpret_cast<uint4*>(out + 32 * u + (D == 128 ? 8 : 16) * at + 8 * half) = make_uint4(o[0], o[1], o[2], o[3]);
                    }
            }
        }
    } else if (warp < kMmaWarp) {
        registers_down<kCodeRegs>();
        // ---- 32 keys of every other step a warp: K's or V's codes and words to K' or V'. Two tiles at once and a step's time
        // for each: a warp alone spends most of its time on latencies -----------------------------------------------------------
        const bool is_v = warp >= kVWarp;
        const int w = warp & 1;  // keys 32 w .. + 31 of the steps of parity warp / 2 % 2
        uint2* scales = reinterpret_cast<uint2*>(raw_smem + Cfg::kRaw * Cfg::kStep) + (warp - kKWarp) * 2 * Cfg::kWords;  // (s, s), (m, m) of every word
        const int codes_at = is_v ? kv4::v_codes_at(D) : 0, words_at = is_v ? kv4::v_words_at(D, G) : kv4::k_words_at(D);
        bool alive = true;
        for (int j = warp >> 1 & 1; j < steps; j += 2) {
            const int stage = j & 1, slot = j % Cfg::kRaw, base0 = key0 + j * kKeys + 2 * w * kv4::kTile;
            if (alive) alive = __all_sync(kAll, ptx::mbar_wait(&bars.raw_full[slot], (j / Cfg::kRaw) & 1, p.status));
            const uint32_t here = raw_there[slot] >> 2 * w;
            const unsigned char* tiles_at = raw_smem + slot * Cfg::kStep + 2 * w * Cfg::kTile;
            // ---- the words, one or a few a lane: their size, and what is not finite; 0 for a key that no row sees
            constexpr int kPerLane = (Cfg::kWords + 31) / 32;
            int loud = 0;
            if (is_v) {  // the exponent above all values so far, two keys a lane; the step's two warps find the same
                const uint2* at = reinterpret_cast<const uint2*>(raw_smem + slot * Cfg::kStep + (lane >> 3) * Cfg::kTile + words_at + (lane & 7) * 8 * NG);
                const int key = key0 + j * kKeys + 2 * lane;
                uint32_t most = 0;
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    const uint2 two = at[i];
                    const uint32_t x = two.x & 0x7fff7fffu, y = two.y & 0x7fff7fffu;
                    const int kx = key + 2 * i / NG, ky = key + (2 * i + 1) / NG;
                    if (kx >= any_lo && kx < any_hi && !__vcmpgeu2(x, 0x7f807f80u)) most = __vmaxu2(most, x);
                    if (ky >= any_lo && ky < any_hi && !__vcmpgeu2(y, 0x7f807f80u)) most = __vmaxu2(most, y);
                }
                if (!(raw_there[slot] >> (lane >> 3) & 1)) most = 0;
                loud = exponent_of(__float_as_uint(fminf(fmaf(15.0f, kv4::word_scale(most), kv4::word_min(most)), 3.4e38f)));
                if (j > 0) {
                    if (alive) alive = __all_sync(kAll, ptx::mbar_wait(&bars.info[(j - 1) % kInfos], ((j - 1) / kInfos) & 1, p.status));
                    loud = max(loud, loudest[(j - 1) % kInfos]);
                }
                if (w == 0 && lane == 0) loudest[j % kInfos] = loud;
            }
#pragma unroll 1
            for (int u = 0; u < 2; ++u) {  // not unrolled, as below: the roles share the instruction caches (684 -> 654 us)
                float s[kPerLane], m[kPerLane];
                uint32_t size = 0, odd = 0;
#pragma unroll
                for (int i = 0; i < kPerLane; ++i) {
                    const int at = (lane + 32 * i) % Cfg::kWords, key = base0 + u * kv4::kTile + at / NG;  // one group: the upper lanes repeat the lower
                    uint32_t x = *reinterpret_cast<const uint32_t*>(tiles_at + u * Cfg::kTile + words_at + at * 4);
                    if (!(here >> u & 1) || key < any_lo || key >= any_hi) x = 0;
                    if ((x & 0x7f800000u) == 0x7f800000u || (x & 0x7f80u) == 0x7f80u) x = 0, odd |= 1u << i;
                    s[i] = kv4::word_scale(x), m[i] = kv4::word_min(x);
                    size = max(size, __float_as_uint(fminf(fmaf(15.0f, fabsf(s[i]), fabsf(m[i])), 3.4e38f)));
                }
                int e = exponent_of(size);
                if (is_v) e = min(loud, e + kSpare);
                const float fit = power_of_two(kFit - e);
#pragma unroll
                for (int i = 0; i < kPerLane; ++i)
                    scales[u * Cfg::kWords + (lane + 32 * i) % Cfg::kWords] = make_uint2(ptx::f16x2_pack(s[i] * fit, s[i] * fit), ptx::f16x2_pack(m[i] * fit, m[i] * fit));
                TileInfo& info = infos[j % kInfos][2 * w + u];  // its place is free: the row warps are far past step j - 8
                uint32_t bad[NG] = {};
                if (__any_sync(kAll, odd != 0)) {
#pragma unroll
                    for (int i = 0; i < kPerLane; ++i) {
                        const int at = (lane + 32 * i) % Cfg::kWords;
#pragma unroll
                        for (int k = 0; k < NG; ++k)
                            if ((odd >> i & 1) && at % NG == k) bad[k] |= 1u << (at / NG);
                    }
#pragma unroll
                    for (int k = 0; k < NG; ++k) bad[k] = __reduce_or_sync(kAll, bad[k]);
                }
                if (lane == 0) {
                    uint32_t all = 0;
#pragma unroll
                    for (int k = 0; k < NG; ++k) all |= bad[k];
                    if (is_v) {
                        const float unit = power_of_two(-e / 2) * power_of_two(-e - -e / 2);  // e up to 128: below the normal numbers, still exact
                        info.v_exp = static_cast<float>(e), info.v_unit = all ? -unit : unit;
#pragma unroll
                        for (int k = 0; k < NG; ++k) info.bad_v[k] = bad[k];
                    } else {
                        info.k_unit = power_of_two(e - kFit), info.bad_k = all;
                    }
                }
            }
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&bars.info[j % kInfos]);
            // ---- K's place is free once S of step j - 2 is there; V's once S of the step itself is, whose MMAs follow those on the
            // values of step j - 2
            const int after = is_v ? j : j - 2;
            for (int i = 0; i < tiles && after >= 0; ++i)
                if (alive) alive = __all_sync(kAll, ptx::mbar_wait(&bars.s_full[i][after & 1], (after >> 1) & 1, p.status));
            if (!is_v) {
                const int t = lane >> 1, h = lane & 1;  // a lane has half of a key's row
#pragma unroll 1
                for (int u = 0; u < 2; ++u) {
                    const unsigned char* tile = tiles_at + u * Cfg::kTile;
                    uint2 sm[NG];
#pragma unroll
                    for (int k = 0; k < NG; ++k) sm[k] = scales[u * Cfg::kWords + t * NG + k];
                    unsigned char* to = k_smem + stage * Cfg::kOperand + ((2 * w + u) * kv4::kTile + t) * 128;
#pragma unroll
                    for (int r = 0; r < 2; ++r) {  // runs 2 h and 2 h + 1
                        const unsigned char* at = tile + t * (D / 2) + (2 * h + r) * (D / 8);
                        uint32_t code[D / 32];
                        if constexpr (D == 128) {
                            const uint4 v = *reinterpret_cast<const uint4*>(at);
                            code[0] = v.x, code[1] = v.y, code[D / 32 - 2] = v.z, code[D / 32 - 1] = v.w;
                        } else {
                            const uint2 v = *reinterpret_cast<const uint2*>(at);
                            code[0] = v.x, code[1] = v.y;
                        }
#pragma unroll
                        for (int i = 0; i < D / 32; ++i)  // channels 8 chunk .. + 7, chunk = 4 i + 2 h + r
                            *reinterpret_cast<uint4*>(to + (i / 2) * (kKeys * 128) + ((((4 * i + 2 * h + r) & 7) ^ (t & 7)) << 4)) = values8(code[i], sm[32 * i / G].x, sm[32 * i / G].y);
                    }
                }
            } else {
                const int blk = lane >> 4, g = lane >> 1 & 7, th = lane & 1;  // run g of four keys of a block of eight
#pragma unroll 1
                for (int u = 0; u < 2; ++u) {
                    unsigned char* to = v_smem + stage * Cfg::kOperand + ((2 * w + u) * kv4::kTile + 8 * blk + 4 * th) * 128;
                    const unsigned char* at = tiles_at + u * Cfg::kTile + codes_at + kv4::v_piece_at(D, 8 * blk + 4 * th, g);
                    uint32_t code[4][D / 64];
                    if constexpr (D == 128) {
                        const uint4 a = *reinterpret_cast<const uint4*>(at), c = *reinterpret_cast<const uint4*>(at + 16);
                        code[0][0] = a.x, code[0][D / 64 - 1] = a.y, code[1][0] = a.z, code[1][D / 64 - 1] = a.w;
                        code[2][0] = c.x, code[2][D / 64 - 1] = c.y, code[3][0] = c.z, code[3][D / 64 - 1] = c.w;
                    } else {
                        const uint4 a = *reinterpret_cast<const uint4*>(at);
                        code[0][0] = a.x, code[1][0] = a.y, code[2][0] = a.z, code[3][0] = a.w;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint2 sm[NG];
#pragma unroll
                        for (int k = 0; k < NG; ++k) sm[k] = scales[u * Cfg::kWords + (8 * blk + 4 * th + i) * NG + k];
#pragma unroll
                        for (int jw = 0; jw < D / 64; ++jw) {  // units 2 jw (low halves) and 2 jw + 1 (high)
                            const int ka = 64 * jw / G, kb = (64 * jw + 32) / G, chunk = D / 64 * g + jw;
                            const uint32_t s2 = ka == kb ? sm[ka].x : __byte_perm(sm[ka].x, sm[kb].x, 0x5410), m2 = ka == kb ? sm[ka].y : __byte_perm(sm[ka].y, sm[kb].y, 0x5410);
                            *reinterpret_cast<uint4*>(to + (chunk >> 3) * (kKeys * 128) + i * 128 + (((chunk & 7) ^ (4 * th + i)) << 4)) = values8(code[i][jw], s2, m2);
                        }
                    }
                }
            }
            ptx::fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                ptx::mbar_arrive(is_v ? &bars.v_full[stage] : &bars.k_full[stage]);
                if (alive) ptx::mbar_arrive(&bars.raw_empty[slot]);  // a copy that was given up on may still write to the slot
            }
        }
    } else {
        registers_down<kMmaRegs>();
        const int i = warp - kMmaWarp;
        if (i == 2) {
            // ---- the copies, a step at a time; page numbers (a lane a tile) a step early ------------------------------------
            const int32_t* table = p.batch.table + static_cast<size_t>(b) * p.batch.width;
            const unsigned char* pool = p.pool.data + static_cast<size_t>(head) * tiles_per_page * Cfg::kTile;
            const long long page_bytes = static_cast<long long>(p.pool.heads) * tiles_per_page * Cfg::kTile;
            int key = key0 + (lane & 3) * kv4::kTile, at = key / kv4::kTile / tiles_per_page, in_page = key / kv4::kTile % tiles_per_page, page = -1;
            if (key < any_hi) page = __ldg(table + at);
            int j = 0;
            for (; j < steps; ++j) {
                const int slot = j % Cfg::kRaw;
                if (j >= Cfg::kRaw && !__all_sync(kAll, ptx::mbar_wait(&bars.raw_empty[slot], (j / Cfg::kRaw - 1) & 1, p.status))) break;
                const bool good = key < any_hi && page >= 0 && page < p.pool.pages;
                if (key < any_hi && !good && lane < 4) kv4::bad_index(p.status);
                const uint32_t there = __ballot_sync(kAll, good) & 15u;
                const int first_page = __shfl_sync(kAll, page, 0);
                const bool one = __ballot_sync(kAll, good && page == first_page) == kAll && __shfl_sync(kAll, in_page, 0) + 3 < tiles_per_page;
                if (lane == 0) {
                    raw_there[slot] = there;
                    ptx::mbar_arrive_expect_tx(&bars.raw_full[slot], __popc(there) * Cfg::kTile);
                }
                __syncwarp();
                unsigned char* to = raw_smem + slot * Cfg::kStep;
                const unsigned char* from = pool + page * page_bytes + in_page * Cfg::kTile;
                if (one) {  // all of the step in one page
                    if (lane == 0) ptx::bulk_g2s(to, from, Cfg::kStep, &bars.raw_full[slot]);
                } else if (lane < 4 && good) {
                    ptx::bulk_g2s(to + lane * Cfg::kTile, from, Cfg::kTile, &bars.raw_full[slot]);
                }
                key += kKeys, in_page += kKeys / kv4::kTile;
                while (in_page >= tiles_per_page) in_page -= tiles_per_page, ++at;
                if (key < any_hi) page = __ldg(table + at);
            }
            // no copy is on its way when the block ends, whoever gave up on what: the last one into each slot has landed
            for (int k = max(0, j - Cfg::kRaw); k < j; ++k) ptx::mbar_wait(&bars.raw_full[k % Cfg::kRaw], (k / Cfg::kRaw) & 1, p.status);
        } else if (i < tiles && steps > 0) {
            // ---- the MMAs of a tile of rows, a warp for each (a warp's waits and commits alone take longer than a step's MMAs). The
            // scores run two steps ahead of the values, into the buffer whose P the values have just taken: the MMAs of a
            // thread run in their order, so one commit a step tells of both
            constexpr uint32_t s_desc = umma::instr_desc(128, kKeys, 0, 0), o_desc = umma::instr_desc_b_mn(128, D, 0, 0);
            const uint64_t q0 = umma::smem_desc_k128(q_smem + i * Cfg::kRows), k0 = umma::smem_desc_k128(k_smem), v0 = umma::smem_desc_mn128(v_smem, kKeys * 128);
            const uint32_t s0 = tmem + Cfg::kS + i * 128, o0 = tmem + Cfg::kO + i * D;
            auto scores = [&](int buffer) {  // by the elected lane
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    umma::mma_f16(s0 + buffer * 64, umma::desc_advance(q0, (k / 4) * (128 * 128) + (k % 4) * 32),
                                  umma::desc_advance(k0, buffer * Cfg::kOperand + (k / 4) * (kKeys * 128) + (k % 4) * 32), s_desc, k > 0);
                umma::mma_commit(&bars.s_full[i][buffer]);
            };
            bool ok = __all_sync(kAll, ptx::mbar_wait(&bars.q_ready, 0, p.status));
            for (int j = 0; ok && j < min(steps, 2); ++j) {
                ok = __all_sync(kAll, ptx::mbar_wait(&bars.k_full[j], 0, p.status));
                umma::fence_after_sync();
                if (ok && umma::elect_one()) scores(j);
                __syncwarp();
            }
            for (int j = 0; ok && j < steps; ++j) {
                const int stage = j & 1, round = (j >> 1) & 1;
                ok = __all_sync(kAll, ptx::mbar_wait(&bars.v_full[stage], round, p.status));
                if (ok && j + 2 < steps) ok = __all_sync(kAll, ptx::mbar_wait(&bars.k_full[stage], round ^ 1, p.status));
                if (ok) ok = __all_sync(kAll, ptx::mbar_wait(&bars.p_full[i][stage], round, p.status));
                umma::fence_after_sync();
                if (ok && umma::elect_one()) {
#pragma unroll
                    for (int k = 0; k < kKeys / 16; ++k)
                        umma::mma_f16_tmem_a(o0, s0 + stage * 64 + 8 * k, umma::desc_advance(v0, stage * Cfg::kOperand + k * 2048), o_desc, j > 0 || k > 0);
                    if (j + 2 < steps) scores(stage);
                    else umma::mma_commit(j + 1 < steps ? &bars.before_last[i] : &bars.o_full[i]);
                }
                __syncwarp();
            }
            // nor an MMA, which may be on its way still if this warp or a row warp gave up
            if (umma::elect_one()) umma::mma_commit(&bars.drained[i]);
            __syncwarp();
            ptx::mbar_wait(&bars.drained[i], 0, p.status);
        }
    }
    umma::fence_before_sync();
    __syncthreads();
    if (warp == kMmaWarp) umma::tmem_dealloc(tmem, Cfg::kCols);
}

template <int D, int G>
int launch_prompts(const AttendParams& p, DeviceState* dev, cudaStream_t stream) {
    using Cfg = PromptCfg<D, G>;
    auto kernel = kv4_attend_prompt_kernel<D, G>;
    static bool configured[kMaxDevices] = {};
    if (!configured[dev->device]) {
        SPK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem));
        configured[dev->device] = true;
    }
    const int64_t rows = int64_t{p.batch.rows} * (p.q_heads / p.pool.heads);
    const int64_t blocks = rows / kv4::kBlockRows + std::min<int64_t>(p.batch.seqs, rows / kv4::kPromptRows);
    SPK_REQUIRE(blocks * p.pool.heads < (int64_t{1} << 31), "kv4_attention: too many rows for one call");
    SPK_CUDA(launch_chained(kernel, dim3(static_cast<unsigned>(blocks * p.pool.heads)), dim3(kThreadsP), Cfg::kSmem, stream, p));
    return SPK_OK;
}

}  // namespace

int kv4::attend_prompts(const AttendParams& p, int d, int group, DeviceState* dev, cudaStream_t stream) {
    if (d == 64) return group == 32 ? launch_prompts<64, 32>(p, dev, stream) : launch_prompts<64, 64>(p, dev, stream);
    return group == 32 ? launch_prompts<128, 32>(p, dev, stream) : group == 64 ? launch_prompts<128, 64>(p, dev, stream) : launch_prompts<128, 128>(p, dev, stream);
}

}  // namespace spk
