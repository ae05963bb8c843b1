// The step between two blocks of a decoder layer, one launch:
//     z = y, or rmsnorm(y) * post_gain        (the norm after a block)
//     r = bf16(residual_scale * x + gate * z) (the residual stream)
//     h = bf16(rmsnorm(r) * gain)             (the norm before the next block, of the residual as it is stored)
// rmsnorm(v) = v / sqrt(mean(v^2) + eps). All sums in fp32; the unfused order (python/spark_kernels/engine.py:441-456 of
// the reference) writes and re-reads the residual between the two kernels. Bound by memory: x and y in, r and h out, 8
// bytes an element.
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
__device__ __forceinline__ Eight load8(const __nv_bfloat16* p) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    Eight e;
#pragma unroll
    for (int i = 0; i < 4; ++i) e.v[2 * i] = __uint_as_float(u[i] << 16), e.v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    return e;
}
// Rounds to bf16, stores (if p is set) and leaves the rounded values in e.
__device__ __forceinline__ void store8(__nv_bfloat16* p, Eight& e) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(e.v[2 * i], e.v[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&b);
        e.v[2 * i] = __uint_as_float(u[i] << 16), e.v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
    if (p != nullptr) *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}

// Sum over the block, the same bits in every thread: warps by shuffles, then every thread adds the warps' sums in order.
// `slots` holds one float per warp and is not reused within a row.
__device__ __forceinline__ float block_sum(float v, float* slots) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
    for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) s += slots[w];
    return s;
}

// A block per row; a thread holds kVec pieces of eight channels in registers from the loads to the last store.
template <int kVec>
__global__ void __launch_bounds__(1024) add_rmsnorm_kernel(const NormParams p) {
    __shared__ float slots[2][32];
    pdl_release();
    pdl_wait();
    const size_t row = blockIdx.x;
    const int pieces = p.hidden >> 3;
    Eight x[kVec];
    const __nv_bfloat16* xr = p.x + row * p.x_stride;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        const int at = threadIdx.x + i * blockDim.x;
        x[i] = at < pieces ? load8(xr + 8 * at) : Eight{};
    }
    if (p.y != nullptr) {
        Eight y[kVec];
        const __nv_bfloat16* yr = p.y + row * p.y_stride;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const int at = threadIdx.x + i * blockDim.x;
            y[i] = at < pieces ? load8(yr + 8 * at) : Eight{};
        }
        float inv = 1.0f;
        if (p.post_gain != nullptr) {
            float sq = 0.0f;
#pragma unroll
            for (int i = 0; i < kVec; ++i)
                for (int j = 0; j < 8; ++j) sq = fmaf(y[i].v[j], y[i].v[j], sq);
            inv = rsqrtf(block_sum(sq, slots[0]) / p.hidden + p.eps);
        }
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const int at = threadIdx.x + i * blockDim.x;
            if (at >= pieces) continue;
            if (p.post_gain != nullptr) {
                const Eight g = load8(p.post_gain + 8 * at);
                for (int j = 0; j < 8; ++j) y[i].v[j] *= inv * g.v[j];
            }
            if (p.gate != nullptr) {
                const Eight g = load8(p.gate + row * p.gate_stride + 8 * at);
                for (int j = 0; j < 8; ++j) y[i].v[j] *= g.v[j];
            }
            for (int j = 0; j < 8; ++j) x[i].v[j] = fmaf(p.residual_scale, x[i].v[j], y[i].v[j]);
            store8(p.r + row * p.hidden + 8 * at, x[i]);
        }
    }
    if (p.gain == nullptr) return;
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < kVec; ++i)
        for (int j = 0; j < 8; ++j) sq = fmaf(x[i].v[j], x[i].v[j], sq);
    const float inv = rsqrtf(block_sum(sq, slots[1]) / p.hidden + p.eps);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        const int at = threadIdx.x + i * blockDim.x;
        if (at >= pieces) continue;
        const Eight g = load8(p.gain + 8 * at);
        for (int j = 0; j < 8; ++j) x[i].v[j] *= inv * g.v[j];
        store8(p.h + row * p.hidden + 8 * at, x[i]);
    }
}

template <int kVec>
int launch(const NormParams& p, cudaStream_t stream) {
    const int threads = cdiv(cdiv(p.hidden >> 3, kVec), 32) * 32;
    SPK_CUDA(launch_chained(add_rmsnorm_kernel<kVec>, dim3(p.rows), dim3(threads), 0, stream, p));
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
    DeviceState* dev = nullptr;
    if (int rc = device_state(&dev)) return rc;
    NormParams p{};
    auto in = [](const void* a) { return static_cast<const __nv_bfloat16*>(a); };
    p.x = in(x), p.y = in(y), p.gain = in(gain), p.post_gain = in(post_gain), p.gate = in(gate);
    p.x_stride = x_stride, p.y_stride = y_stride, p.gate_stride = gate_stride, p.residual_scale = residual_scale, p.eps = eps;
    p.r = static_cast<__nv_bfloat16*>(r), p.h = static_cast<__nv_bfloat16*>(h), p.rows = rows, p.hidden = hidden;
    auto stream = static_cast<cudaStream_t>(stream_);
    const int pieces = hidden >> 3;
    return pieces <= 1024 ? launch<1>(p, stream) : pieces <= 2048 ? launch<2>(p, stream) : pieces <= 4096 ? launch<4>(p, stream) : launch<8>(p, stream);
}
