// The step between two blocks of a decoder layer, one launch:
//     z = y, or rmsnorm(y) * post_gain        (the norm after a block)
//     r = bf16(residual_scale * x + gate * z) (the residual stream)
//     h = bf16(rmsnorm(r) * gain)             (the norm before the next block, of the residual as it is stored)
// rmsnorm(v) = v / sqrt(mean(v^2) + eps). All sums in fp32; the unfused order (python/spark_kernels/engine.py:441-456 of
// the reference) writes and re-reads the residual between the two kernels. Bound by memory: x and y in, r and h out, 8
// bytes an element.
#include <initializer_list>

#include "spk_common.cuh"

namespace spk {
namespace {

struct NormParams {
    const __nv_bfloat16 *x, *y, *gain, *post_gain, *gate;
    long long x_stride, y_stride, gate_stride;
    float residual_scale, eps;
    __nv_bfloat16 *r, *h;
    int rows, hidden;
};

struct Eight {
    float v[8];
};
__device__ __forceinline__ uint4 load8(const __nv_bfloat16* p) { return *reinterpret_cast<const uint4*>(p); }  // not __ldg: r or h may take its place
__device__ __forceinline__ Eight unpack8(const uint4& w) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    Eight e;
#pragma unroll
    for (int i = 0; i < 4; ++i) e.v[2 * i] = __uint_as_float(u[i] << 16), e.v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    return e;
}
__device__ __forceinline__ uint4 pack8(const Eight& e) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(e.v[2 * i], e.v[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ float square_sum(const Eight& e, float s) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(e.v[i], e.v[i], s);
    return s;
}

// Sum over the block, the same bits in every thread: warps by shuffles, then every thread adds the warps' sums in order.
// `slots` holds one float per warp and is not reused within a row.
__device__ __forceinline__ float block_sum(float v, float* slots) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int warps = blockDim.x >> 5;
    if (warps == 1) return v;
    if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
    for (int w = 0; w < warps; ++w) s += slots[w];
    return s;
}

// A block per row; a thread holds kVec pieces of eight channels from the loads to the last store, as bf16 until they are
// used. All that the first half reads is requested at once, the second norm's gain before its sum.
template <int kVec, int kMost>
__global__ void __launch_bounds__(kMost) add_rmsnorm_kernel(const NormParams p) {
    __shared__ float slots[2][32];
    pdl_release();
    pdl_wait();
    const size_t row = blockIdx.x;
    const int pieces = p.hidden >> 3;
    const __nv_bfloat16* xr = p.x + row * p.x_stride;
    uint4 x[kVec];
    auto at = [&](int i) { return static_cast<int>(threadIdx.x + i * blockDim.x); };
#pragma unroll
    for (int i = 0; i < kVec; ++i) x[i] = at(i) < pieces ? load8(xr + 8 * at(i)) : uint4{};
    if (p.y != nullptr) {
        uint4 y[kVec], post[kVec], gate[kVec];
        const __nv_bfloat16 *yr = p.y + row * p.y_stride, *gr = p.gate + row * p.gate_stride;
#pragma unroll
        for (int i = 0; i < kVec; ++i) y[i] = at(i) < pieces ? load8(yr + 8 * at(i)) : uint4{};
        if (p.gate != nullptr) {
#pragma unroll
            for (int i = 0; i < kVec; ++i) gate[i] = at(i) < pieces ? load8(gr + 8 * at(i)) : uint4{};
        }
        float inv = 1.0f;
        if (p.post_gain != nullptr) {
#pragma unroll
            for (int i = 0; i < kVec; ++i) post[i] = at(i) < pieces ? load8(p.post_gain + 8 * at(i)) : uint4{};
            float sq = 0.0f;
#pragma unroll
            for (int i = 0; i < kVec; ++i) sq = square_sum(unpack8(y[i]), sq);
            inv = rsqrtf(block_sum(sq, slots[0]) / p.hidden + p.eps);
        }
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            if (at(i) >= pieces) continue;
            Eight z = unpack8(y[i]), r = unpack8(x[i]);
            if (p.post_gain != nullptr) {
                const Eight g = unpack8(post[i]);
#pragma unroll
                for (int j = 0; j < 8; ++j) z.v[j] *= inv * g.v[j];
            }
            if (p.gate != nullptr) {
                const Eight g = unpack8(gate[i]);
#pragma unroll
                for (int j = 0; j < 8; ++j) z.v[j] *= g.v[j];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) r.v[j] = fmaf(p.residual_scale, r.v[j], z.v[j]);
            x[i] = pack8(r);
            *reinterpret_cast<uint4*>(p.r + row * p.hidden + 8 * at(i)) = x[i];
        }
    }
    if (p.gain == nullptr) return;
    uint4 gain[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) gain[i] = at(i) < pieces ? load8(p.gain + 8 * at(i)) : uint4{};
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < kVec; ++i) sq = square_sum(unpack8(x[i]), sq);
    const float inv = rsqrtf(block_sum(sq, slots[1]) / p.hidden + p.eps);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        if (at(i) >= pieces) continue;
        Eight h = unpack8(x[i]);
        const Eight g = unpack8(gain[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) h.v[j] *= inv * g.v[j];
        *reinterpret_cast<uint4*>(p.h + row * p.hidden + 8 * at(i)) = pack8(h);
    }
}

template <int kVec, int kMost>
int launch(const NormParams& p, cudaStream_t stream) {
    const int threads = cdiv(cdiv(p.hidden >> 3, kVec), 32) * 32;
    SPK_CUDA(launch_chained(add_rmsnorm_kernel<kVec, kMost>, dim3(p.rows), dim3(threads), 0, stream, p));
    return SPK_OK;
}

}  // namespace
}  // namespace spk

extern "C" int spk_add_rmsnorm(const void* x, long long x_stride, const void* y, long long y_stride, const void* gain, const void* post_gain,
                               const void* gate, long long gate_stride, float residual_scale, float eps, void* r, void* h, int rows, int hidden,
                               void* stream_) {
    using namespace spk;
    SPK_REQUIRE(rows >= 0 && hidden >= 8 && hidden % 8 == 0 && hidden <= 65536, "add_rmsnorm: hidden must be a multiple of 8 up to 65536, got rows=%d hidden=%d", rows, hidden);
    SPK_REQUIRE(eps >= 0.0f && residual_scale == residual_scale, "add_rmsnorm: eps must not be negative, residual_scale not NaN");
    if (rows == 0) return SPK_OK;
    SPK_REQUIRE(x && (y || (!post_gain && !gate && residual_scale == 1.0f)), "add_rmsnorm: post_gain, gate and residual_scale need y");
    SPK_REQUIRE((y == nullptr || r) && (gain == nullptr) == (h == nullptr) && (y || gain), "add_rmsnorm: r goes with y, h with gain, and one of them is needed");
    SPK_REQUIRE(aligned16(x) && aligned16(y) && aligned16(gain) && aligned16(post_gain) && aligned16(gate) && aligned16(r) && aligned16(h),
                "add_rmsnorm: pointers must be 16-byte aligned");
    SPK_REQUIRE(x_stride % 8 == 0 && y_stride % 8 == 0 && gate_stride % 8 == 0 && x_stride >= 0 && y_stride >= 0 && gate_stride >= 0,
                "add_rmsnorm: row strides must be multiples of 8");
    SPK_REQUIRE(r == nullptr || r != x || x_stride == hidden || rows == 1, "add_rmsnorm: r may be x where its rows are contiguous, got a stride of %lld", x_stride);
    // a block reads its row of x, y and the gate before it writes it, so an output may take the place of one of them row by row
    const struct {
        const char* name;
        const void* at;
        long long stride;
        bool vector;
    } inputs[] = {{"x", x, x_stride, false}, {"y", y, y_stride, false}, {"the gate", gate, gate_stride, false}, {"the gain", gain, 0, true}, {"post_gain", post_gain, 0, true}};
    const long long bytes = 2ll * rows * hidden;
    for (const auto& in : inputs) {
        if (in.at == nullptr) continue;
        for (const void* out : {y == nullptr ? nullptr : r, h}) {  // r is not written without y
            if (out == nullptr || !overlap(out, bytes, in.at, in.vector ? 1 : rows, in.stride, hidden)) continue;
            SPK_REQUIRE(out == in.at && !in.vector && (in.stride == hidden || rows == 1), "add_rmsnorm: %s must not lie in the memory of %s, except in its place where its rows are contiguous",
                        out == r ? "r" : "h", in.name);
        }
    }
    SPK_REQUIRE(r == nullptr || h == nullptr || y == nullptr || !overlap(r, bytes, h, rows, hidden, hidden), "add_rmsnorm: r and h must not share memory");
    DeviceState* dev = nullptr;
    if (int rc = device_state(&dev)) return rc;
    NormParams p{};
    auto in = [](const void* a) { return static_cast<const __nv_bfloat16*>(a); };
    p.x = in(x), p.y = in(y), p.gain = in(gain), p.post_gain = in(post_gain), p.gate = in(gate);
    p.x_stride = x_stride, p.y_stride = y_stride, p.gate_stride = gate_stride, p.residual_scale = residual_scale, p.eps = eps;
    p.r = static_cast<__nv_bfloat16*>(r), p.h = static_cast<__nv_bfloat16*>(h), p.rows = rows, p.hidden = hidden;
    auto stream = static_cast<cudaStream_t>(stream_);
    const int pieces = hidden >> 3;
    // Few rows: as many threads as a block holds, for the shortest chain from load to store (1 x 4096: 2.1 us in a graph).
    // Many: four pieces a thread, so that an SM has several rows' loads in flight: 16384 x 4096 with both norms and a gate per
    // row 99 us (6.78 TB/s, 1.04 of the measured copy) against 107.5 / 101.9 / 117.8 with three, two and one piece. Sum and norm
    // alone, the blocks for few and for many: 1000 rows of 4096 5.7 and 4.9 us, 400 rows 3.6 and 3.7, 296 rows 2.7 and 2.8; of 8192 12.8
    // and 8.1, 6.4 and 4.1, 4.5 and 4.0; of 16384 28.3 and 23.4, 9.4 and 7.9, 6.8 and 5.4; of 1024 the same.
    // From 32776 channels up a thread holds eight pieces and a block 1024 threads, whose registers do not hold them (1352 bytes
    // stored, 1444 loaded); no block holds more threads.
    if (rows > 2 * dev->sm_count) {
        if (pieces <= 128) return launch<1, 128>(p, stream);
        if (pieces <= 256) return launch<2, 128>(p, stream);
        if (pieces <= 1024) return launch<4, 256>(p, stream);
        if (pieces <= 4096) return launch<8, 512>(p, stream);
    }
    return pieces <= 1024 ? launch<1, 1024>(p, stream) : pieces <= 2048 ? launch<2, 1024>(p, stream) : pieces <= 4096 ? launch<4, 1024>(p, stream) : launch<8, 1024>(p, stream);
}
