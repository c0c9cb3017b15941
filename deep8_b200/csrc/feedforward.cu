// extern "C" layer, part four (include/d8k.h): the gated feed-forward block - the gated projection pair with its gradients,
// counter-based dropout and the root-mean-square norm.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <exception>
#include <string>

#include "../../include/d8k.h"
#include "elementwise.cuh"
#include "feedforward.cuh"
#include "gemm_host.h"

struct d8k_ctx : public d8k::Ctx {};

namespace d8k {
namespace {

#define D8K_CUDA(call)                                                                                          \
    do {                                                                                                        \
        cudaError_t e__ = (call);                                                                               \
        if (e__ != cudaSuccess) return fail(D8K_ERR_CUDA, std::string(#call) + ": " + cudaGetErrorString(e__)); \
    } while (0)

// ------------------------------------------------------------------------------------------------ gated projections
// dpre from pre and dz, four consecutive elements (one counter of the generator) per step: 5 accesses per element, bound by HBM.
// pre and dpre may be the same memory (an element is read and written by one thread), so nothing here is declared __restrict__.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) gated_grad_pre_kernel(const T* pre, const T* dz, T* dpre, size_t n, int act, DropSpec drop, int dropping) {
    constexpr bool FAST = sizeof(T) == 2;
    constexpr int V = 16 / sizeof(T);     // elements of a 16-byte access
    constexpr int E = VEC ? V : 4;        // elements per step
    const unsigned long long offset = dropping ? drop_offset(drop) : 0;
    const size_t steps = (n + E - 1) / E;
    for (size_t s = blockIdx.x * static_cast<size_t>(blockDim.x) + threadIdx.x; s < steps; s += gridDim.x * static_cast<size_t>(blockDim.x)) {
        const size_t i0 = s * E;
        alignas(16) T g[E], u[E], d[E];
        if (VEC) {
            *reinterpret_cast<uint4*>(g) = *reinterpret_cast<const uint4*>(pre + i0);
            *reinterpret_cast<uint4*>(u) = *reinterpret_cast<const uint4*>(pre + n + i0);
            *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(dz + i0);
        } else {
#pragma unroll
            for (int k = 0; k < E; ++k) {
                const bool in = i0 + k < n;
                g[k] = in ? pre[i0 + k] : narrow<T>(0.0f);
                u[k] = in ? pre[n + i0 + k] : narrow<T>(0.0f);
                d[k] = in ? dz[i0 + k] : narrow<T>(0.0f);
            }
        }
#pragma unroll
        for (int q = 0; q < E / 4; ++q) {
            uint4 words = make_uint4(0u, 0u, 0u, 0u);
            if (dropping) words = philox4x32((i0 >> 2) + q, offset, drop.seed);
            const uint32_t word[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float value, slope;
                activation<FAST, true>(act, widen(g[4 * q + k]), value, slope);
                const float dd = dropping ? widen(d[4 * q + k]) * drop.scale : widen(d[4 * q + k]);
                float dg = dd * widen(u[4 * q + k]) * slope, du = dd * value;
                if (dropping && !drop_keeps(drop, word[k])) dg = du = 0.0f;
                g[4 * q + k] = narrow<T>(dg);
                u[4 * q + k] = narrow<T>(du);
            }
        }
        if (VEC) {
            *reinterpret_cast<uint4*>(dpre + i0) = *reinterpret_cast<const uint4*>(g);
            *reinterpret_cast<uint4*>(dpre + n + i0) = *reinterpret_cast<const uint4*>(u);
        } else {
#pragma unroll
            for (int k = 0; k < E; ++k)
                if (i0 + k < n) {
                    dpre[i0 + k] = g[k];
                    dpre[n + i0 + k] = u[k];
                }
        }
    }
}

// ------------------------------------------------------------------------------------------------ dropout
// y = (residual +) dropout(x): `residual` is the accumulated gradient itself in the backward pass.  Four consecutive elements share one
// counter of the generator.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dropout_kernel(const T* x, const T* residual, T* y, size_t n, DropSpec drop) {
    constexpr int V = 16 / sizeof(T);
    constexpr int E = VEC ? V : 4;
    const unsigned long long offset = drop_offset(drop);
    const size_t steps = (n + E - 1) / E;
    for (size_t s = blockIdx.x * static_cast<size_t>(blockDim.x) + threadIdx.x; s < steps; s += gridDim.x * static_cast<size_t>(blockDim.x)) {
        const size_t i0 = s * E;
        alignas(16) T a[E], b[E];
        if (VEC) {
            *reinterpret_cast<uint4*>(a) = *reinterpret_cast<const uint4*>(x + i0);
            if (residual) *reinterpret_cast<uint4*>(b) = *reinterpret_cast<const uint4*>(residual + i0);
        } else {
#pragma unroll
            for (int k = 0; k < E; ++k) {
                a[k] = i0 + k < n ? x[i0 + k] : narrow<T>(0.0f);
                if (residual) b[k] = i0 + k < n ? residual[i0 + k] : narrow<T>(0.0f);
            }
        }
#pragma unroll
        for (int q = 0; q < E / 4; ++q) {
            const uint4 words = philox4x32((i0 >> 2) + q, offset, drop.seed);
            const uint32_t word[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float v = drop_keeps(drop, word[k]) ? widen(a[4 * q + k]) * drop.scale : 0.0f;
                if (residual) v += widen(b[4 * q + k]);
                a[4 * q + k] = narrow<T>(v);
            }
        }
        if (VEC) {
            *reinterpret_cast<uint4*>(y + i0) = *reinterpret_cast<const uint4*>(a);
        } else {
#pragma unroll
            for (int k = 0; k < E; ++k)
                if (i0 + k < n) y[i0 + k] = a[k];
        }
    }
}

// ------------------------------------------------------------------------------------------------ root-mean-square norm
// Sum over the CTA's 256 threads, the same value in every thread; `part` is 8 floats of shared memory.
__device__ __forceinline__ float cta_sum(float v, float* part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();  // the last row's sum has been read
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += part[k];
    return t;
}

// One CTA per row, the row read twice (the second time from cache).  y may be x: nothing is declared __restrict__.
template <typename T>
__global__ void __launch_bounds__(256) rms_norm_forward_kernel(const T* x, const T* weight, T* y, float* rstd, size_t rows, int cols, float eps) {
    __shared__ float part[8];
    for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* row = x + r * cols;
        float sum = 0.0f;
        for (int c = threadIdx.x; c < cols; c += 256) {
            const float v = widen(row[c]);
            sum = fmaf(v, v, sum);
        }
        sum = cta_sum(sum, part);
        const float inv = 1.0f / sqrtf(sum / cols + eps);
        if (rstd && threadIdx.x == 0) rstd[r] = inv;
        for (int c = threadIdx.x; c < cols; c += 256) y[r * cols + c] = narrow<T>(widen(row[c]) * inv * widen(weight[c]));
    }
}

template <typename T>
__global__ void __launch_bounds__(256) rms_norm_grad_x_kernel(const T* __restrict__ x, const T* __restrict__ weight, const float* __restrict__ rstd,
                                                              T* __restrict__ dx, const T* __restrict__ dy, size_t rows, int cols, int accumulate) {
    __shared__ float part[8];
    for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const size_t at = r * cols;
        const float inv = rstd[r];
        float sum = 0.0f;
        for (int c = threadIdx.x; c < cols; c += 256) sum = fmaf(widen(dy[at + c]) * widen(weight[c]), widen(x[at + c]) * inv, sum);
        const float mean = cta_sum(sum, part) / cols;
        for (int c = threadIdx.x; c < cols; c += 256) {
            float v = inv * (widen(dy[at + c]) * widen(weight[c]) - widen(x[at + c]) * inv * mean);
            if (accumulate) v += widen(dx[at + c]);
            dx[at + c] = narrow<T>(v);
        }
    }
}

// Column sums of dy * x * rstd in two fixed-order steps: a thread per column and slice of rows, then the slices in order.
template <typename T>
__global__ void __launch_bounds__(256) rms_norm_grad_w_kernel(const T* __restrict__ x, const float* __restrict__ rstd, const T* __restrict__ dy,
                                                              float* __restrict__ partial, size_t rows, int cols, size_t rows_per_slice) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    const size_t r0 = blockIdx.y * rows_per_slice;
    const size_t r1 = r0 + rows_per_slice < rows ? r0 + rows_per_slice : rows;
    float sum = 0.0f;
    for (size_t r = r0; r < r1; ++r) sum = fmaf(widen(dy[r * cols + c]), widen(x[r * cols + c]) * rstd[r], sum);
    partial[static_cast<size_t>(blockIdx.y) * cols + c] = sum;
}
template <typename T>
__global__ void __launch_bounds__(256) rms_norm_grad_w_final_kernel(T* __restrict__ dweight, const float* __restrict__ partial, int slices, int cols,
                                                                    int accumulate) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    float sum = 0.0f;
    for (int s = 0; s < slices; ++s) sum += partial[static_cast<size_t>(s) * cols + c];
    dweight[c] = narrow<T>(accumulate ? widen(dweight[c]) + sum : sum);
}

// ------------------------------------------------------------------------------------------------ host side
// The context's device is current while an entry point runs; whatever was current before is again afterwards.
class DeviceGuard {
public:
    explicit DeviceGuard(int device) {
        if (cudaGetDevice(&before_) != cudaSuccess || before_ == device) return;
        error_ = cudaSetDevice(device);
        changed_ = error_ == cudaSuccess;
    }
    ~DeviceGuard() {
        if (changed_) cudaSetDevice(before_);
    }
    cudaError_t error() const { return error_; }

private:
    int before_ = 0;
    bool changed_ = false;
    cudaError_t error_ = cudaSuccess;
};

// Runs an entry point's body with the checks every one shares; no exception leaves through the C interface.
template <class Body>
int entry(d8k_ctx* ctx, int dtype, Body body) noexcept {
    try {
        if (!ctx) return fail(D8K_ERR_ARGUMENT, "null context");
        if (dtype != D8K_F16 && dtype != D8K_F32) return fail(D8K_ERR_ARGUMENT, "type is not support: dtype must be D8K_F16 or D8K_F32");
        DeviceGuard guard(ctx->device);
        if (guard.error() != cudaSuccess) return fail(D8K_ERR_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(guard.error()));
        return body();
    } catch (const std::exception& e) {
        try {
            return fail(D8K_ERR_CUDA, e.what());
        } catch (...) {
            return D8K_ERR_CUDA;
        }
    } catch (...) {
        return D8K_ERR_CUDA;
    }
}

bool aligned16(std::initializer_list<const void*> ptrs) {
    uintptr_t bits = 0;
    for (const void* p : ptrs) bits |= reinterpret_cast<uintptr_t>(p);
    return (bits & 15) == 0;
}
bool overlap(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && x < y + nb && y < x + na;
}
size_t esize(int dtype) { return dtype == D8K_F32 ? 4 : 2; }

int grid_for(const d8k_ctx* ctx, size_t steps) {
    size_t blocks = (steps + 255) / 256;
    const size_t cap = static_cast<size_t>(ctx->num_sms) * 8;
    if (blocks > cap) blocks = cap;
    return blocks < 1 ? 1 : static_cast<int>(blocks);
}

// The launch's form of a dropout argument; *on stays 0 when there is nothing to drop (none given, or p == 0).
int make_drop(const d8k_dropout* drop, DropSpec* spec, int* on) {
    *spec = DropSpec{0, 0, nullptr, 0, 1, 1.0f};
    *on = 0;
    if (!drop) return 0;
    if (!(drop->p >= 0.0 && drop->p <= 1.0)) return fail(D8K_ERR_ARGUMENT, "dropout: p must be between 0 and 1");
    if (reinterpret_cast<uintptr_t>(drop->device_offset) & 7) return fail(D8K_ERR_ARGUMENT, "dropout: device_offset must be 8-byte aligned");
    const double threshold = std::nearbyint(drop->p * 4294967296.0);
    spec->seed = drop->seed;
    spec->offset = drop->offset;
    spec->counter = drop->device_offset;
    spec->some = threshold < 4294967296.0;
    spec->threshold = spec->some ? static_cast<uint32_t>(threshold) : 0xffffffffu;
    spec->scale = spec->some ? static_cast<float>(1.0 / (1.0 - drop->p)) : 0.0f;
    *on = drop->p > 0.0;
    return 0;
}

int check_gated(int activation, int xb, int xr, int xc, int yc) {
    if (activation < 0 || activation >= kActCount) return fail(D8K_ERR_ARGUMENT, "gated: no such activation");
    if (xb < 0 || xr < 0 || xc < 1 || yc < 1) return fail(D8K_ERR_ARGUMENT, "the shape is error");
    if (1LL * xb * xr >= (1LL << 31)) return fail(D8K_ERR_ARGUMENT, "the shape is too large");
    return 0;
}

int check_norm(size_t rows, int cols) {
    if (cols < 1) return fail(D8K_ERR_ARGUMENT, "the shape is error");
    if (cols > (1 << 30) || rows > (static_cast<size_t>(1) << 40)) return fail(D8K_ERR_ARGUMENT, "the shape is too large");
    return 0;
}

HostOperand matrix(const void* ptr, bool mn, long long ld, int batch = 1, long long stride = 0) {
    HostOperand o;
    o.ptr = ptr;
    o.mn = mn;
    o.ld = ld;
    o.batch_count = batch;
    o.batch_stride = stride;
    return o;
}

int gated_grad_pre(d8k_ctx* ctx, int dtype, int activation, const void* pre, const void* dz, void* dpre, size_t n, const d8k_dropout* drop) {
    if (activation < 0 || activation >= kActCount) return fail(D8K_ERR_ARGUMENT, "gated: no such activation");
    DropSpec spec;
    int dropping = 0;
    if (int rc = make_drop(drop, &spec, &dropping)) return rc;
    if (n == 0) return 0;
    if (!pre || !dz || !dpre) return fail(D8K_ERR_ARGUMENT, "gated: null pointer");
    const size_t bytes = n * esize(dtype);
    if ((dpre != pre && overlap(dpre, 2 * bytes, pre, 2 * bytes)) || overlap(dpre, 2 * bytes, dz, bytes))
        return fail(D8K_ERR_ARGUMENT, "gated: dpre overlaps an input");
    const int per = static_cast<int>(16 / esize(dtype));
    const bool vec = aligned16({pre, dz, dpre}) && n % per == 0;
    const int grid = grid_for(ctx, (n + per - 1) / (vec ? per : 4));
    auto run = [&](auto zero) {
        using T = decltype(zero);
        auto kernel = vec ? gated_grad_pre_kernel<T, true> : gated_grad_pre_kernel<T, false>;
        kernel<<<grid, 256, 0, ctx->stream>>>(static_cast<const T*>(pre), static_cast<const T*>(dz), static_cast<T*>(dpre), n, activation, spec, dropping);
    };
    if (dtype == D8K_F32) run(0.0f);
    else run(__half());
    D8K_CUDA(cudaGetLastError());
    count_launch();
    return 0;
}

int gated_grad_x(d8k_ctx* ctx, int dtype, void* dx, int xb, int xr, int xc, const void* w, int yc, const void* dpre, int accumulate) {
    if (int rc = check_gated(0, xb, xr, xc, yc)) return rc;
    const int rows = xb * xr;
    if (rows == 0) return 0;
    if (!dx || !w || !dpre) return fail(D8K_ERR_ARGUMENT, "gated: null pointer");
    const size_t es = esize(dtype), x_bytes = es * rows * xc;
    if (overlap(dx, x_bytes, w, 2 * es * xc * yc) || overlap(dx, x_bytes, dpre, 2 * es * rows * yc)) return fail(D8K_ERR_ARGUMENT, "gated: dx overlaps an input");
    GemmProblem g;  // the two products join one contraction: a batch of two that is summed
    g.dtype = dtype;
    g.M = rows; g.N = xc; g.K = yc;
    g.a = matrix(dpre, false, yc, 2, 1LL * rows * yc);
    g.b = matrix(w, false, yc, 2, 1LL * xc * yc);
    g.kbatch = 2;
    g.C = dx;
    g.ldc = xc;
    g.beta = accumulate ? 1 : 0;
    return run_gemm(ctx, g);
}

int gated_grad_w(d8k_ctx* ctx, int dtype, const void* x, int xb, int xr, int xc, void* dw, int yc, const void* dpre, int accumulate) {
    if (int rc = check_gated(0, xb, xr, xc, yc)) return rc;
    const int rows = xb * xr;
    const size_t es = esize(dtype), w_bytes = 2 * es * xc * yc;
    if (!dw || (rows > 0 && (!x || !dpre))) return fail(D8K_ERR_ARGUMENT, "gated: null pointer");
    if (rows == 0) {  // no row contributes
        if (!accumulate) D8K_CUDA(cudaMemsetAsync(dw, 0, w_bytes, ctx->stream));
        return 0;
    }
    if (overlap(dw, w_bytes, x, es * rows * xc) || overlap(dw, w_bytes, dpre, 2 * es * rows * yc)) return fail(D8K_ERR_ARGUMENT, "gated: dw overlaps an input");
    GemmProblem g;
    g.dtype = dtype;
    g.M = xc; g.N = yc; g.K = rows;
    g.a = matrix(x, true, xc);
    g.b = matrix(dpre, true, yc, 2, 1LL * rows * yc);
    g.batch = 2;
    g.C = dw;
    g.ldc = yc;
    g.c_batch_stride = 1LL * xc * yc;
    g.beta = accumulate ? 1 : 0;
    return run_gemm(ctx, g);
}

int dropout(d8k_ctx* ctx, int dtype, const void* x, const void* residual, void* y, size_t n, const d8k_dropout* drop) {
    if (!drop) return fail(D8K_ERR_ARGUMENT, "dropout: null pointer");
    DropSpec spec;
    int dropping = 0;
    if (int rc = make_drop(drop, &spec, &dropping)) return rc;
    if (n == 0) return 0;
    if (!x || !y) return fail(D8K_ERR_ARGUMENT, "dropout: null pointer");
    const size_t bytes = n * esize(dtype);
    if ((y != x && overlap(y, bytes, x, bytes)) || (y != residual && overlap(y, bytes, residual, bytes)))
        return fail(D8K_ERR_ARGUMENT, "dropout: the output overlaps an input");
    const int per = static_cast<int>(16 / esize(dtype));
    const bool vec = aligned16({x, residual, y}) && n % per == 0;
    const int grid = grid_for(ctx, (n + per - 1) / (vec ? per : 4));
    auto run = [&](auto zero) {
        using T = decltype(zero);
        auto kernel = vec ? dropout_kernel<T, true> : dropout_kernel<T, false>;
        kernel<<<grid, 256, 0, ctx->stream>>>(static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<T*>(y), n, spec);
    };
    if (dtype == D8K_F32) run(0.0f);
    else run(__half());
    D8K_CUDA(cudaGetLastError());
    count_launch();
    return 0;
}

template <typename T>
int rms_norm_backward(d8k_ctx* ctx, const T* x, const T* weight, const float* rstd, T* dx, T* dweight, const T* dy, size_t rows, int cols, int accumulate) {
    if (dweight) {
        const int strips = (cols + 255) / 256;
        size_t slices = (static_cast<size_t>(ctx->num_sms) * 8 + strips - 1) / strips;
        const size_t most = ctx->scratch_bytes / (static_cast<size_t>(cols) * sizeof(float));
        if (most < 1) return fail(D8K_ERR_ARGUMENT, "the context's scratch memory is smaller than one row of floats");
        if (slices > most) slices = most;
        if (slices > (rows + 7) / 8) slices = (rows + 7) / 8;
        const size_t per = (rows + slices - 1) / slices;
        slices = (rows + per - 1) / per;
        rms_norm_grad_w_kernel<T><<<dim3(strips, static_cast<unsigned>(slices)), 256, 0, ctx->stream>>>(x, rstd, dy, ctx->scratch, rows, cols, per);
        D8K_CUDA(cudaGetLastError());
        rms_norm_grad_w_final_kernel<T><<<strips, 256, 0, ctx->stream>>>(dweight, ctx->scratch, static_cast<int>(slices), cols, accumulate);
        D8K_CUDA(cudaGetLastError());
        count_launch();
        count_launch();
    }
    if (dx) {
        const size_t cap = static_cast<size_t>(ctx->num_sms) * 8;
        rms_norm_grad_x_kernel<T><<<static_cast<unsigned>(rows < cap ? rows : cap), 256, 0, ctx->stream>>>(x, weight, rstd, dx, dy, rows, cols, accumulate);
        D8K_CUDA(cudaGetLastError());
        count_launch();
    }
    return 0;
}

}  // namespace
}  // namespace d8k

using namespace d8k;

extern "C" {

int d8k_gated_forward(d8k_ctx* ctx, int dtype, int activation, const void* x, int xb, int xr, int xc, const void* w, int yc, void* pre, void* h,
                      const d8k_dropout* drop) {
    return entry(ctx, dtype, [&]() -> int {
        if (int rc = check_gated(activation, xb, xr, xc, yc)) return rc;
        DropSpec spec;
        int dropping = 0;
        if (int rc = make_drop(drop, &spec, &dropping)) return rc;
        const int rows = xb * xr;
        if (rows == 0) return 0;
        if (!x || !w || !h) return fail(D8K_ERR_ARGUMENT, "gated: null pointer");
        const size_t es = esize(dtype), xs = es * rows * xc, ws = 2 * es * xc * yc, hs = es * rows * yc;
        if (overlap(h, hs, x, xs) || overlap(h, hs, w, ws) || overlap(pre, 2 * hs, x, xs) || overlap(pre, 2 * hs, w, ws) || overlap(pre, 2 * hs, h, hs))
            return fail(D8K_ERR_ARGUMENT, "gated: an output overlaps an input or the other output");
        GatedProblem g;
        g.dtype = dtype;
        g.M = rows; g.N = yc; g.K = xc;
        g.a = x;
        g.b = w;
        g.C = h;
        g.tail = GatedTail{activation, dropping, pre, 1LL * rows * yc, spec};
        return run_gated(ctx, g);
    });
}

int d8k_gated_grad_pre(d8k_ctx* ctx, int dtype, int activation, const void* pre, const void* dz, void* dpre, size_t n, const d8k_dropout* drop) {
    return entry(ctx, dtype, [&]() -> int { return gated_grad_pre(ctx, dtype, activation, pre, dz, dpre, n, drop); });
}

int d8k_gated_grad_x_into(d8k_ctx* ctx, int dtype, void* dx, int xb, int xr, int xc, const void* w, int yc, const void* dpre, int accumulate) {
    return entry(ctx, dtype, [&]() -> int { return gated_grad_x(ctx, dtype, dx, xb, xr, xc, w, yc, dpre, accumulate); });
}

int d8k_gated_grad_w_into(d8k_ctx* ctx, int dtype, const void* x, int xb, int xr, int xc, void* dw, int yc, const void* dpre, int accumulate) {
    return entry(ctx, dtype, [&]() -> int { return gated_grad_w(ctx, dtype, x, xb, xr, xc, dw, yc, dpre, accumulate); });
}

int d8k_gated_backward(d8k_ctx* ctx, int dtype, int activation, const void* x, int xb, int xr, int xc, const void* w, int yc, const void* pre,
                       const void* dz, void* dpre, void* dx, void* dw, int accumulate, const d8k_dropout* drop) {
    return entry(ctx, dtype, [&]() -> int {
        if (int rc = check_gated(activation, xb, xr, xc, yc)) return rc;
        const size_t es = esize(dtype), rows = static_cast<size_t>(xb) * xr;
        if (rows > 0) {  // everything is checked before the first launch
            if ((dx && !w) || (dw && !x)) return fail(D8K_ERR_ARGUMENT, "gated: null pointer");
            const size_t xs = es * rows * xc, ws = 2 * es * xc * yc, hs = es * rows * yc;
            if (overlap(dpre, 2 * hs, x, xs) || overlap(dpre, 2 * hs, w, ws) || overlap(dx, xs, x, xs) || overlap(dx, xs, w, ws) || overlap(dx, xs, pre, 2 * hs) ||
                overlap(dx, xs, dz, hs) || overlap(dx, xs, dpre, 2 * hs) || overlap(dw, ws, x, xs) || overlap(dw, ws, w, ws) || overlap(dw, ws, pre, 2 * hs) ||
                overlap(dw, ws, dz, hs) || overlap(dw, ws, dpre, 2 * hs) || overlap(dx, xs, dw, ws))
                return fail(D8K_ERR_ARGUMENT, "gated: an output overlaps an input or another output");
        }
        if (int rc = gated_grad_pre(ctx, dtype, activation, pre, dz, dpre, rows * yc, drop)) return rc;
        if (dx)
            if (int rc = gated_grad_x(ctx, dtype, dx, xb, xr, xc, w, yc, dpre, accumulate)) return rc;
        if (dw)
            if (int rc = gated_grad_w(ctx, dtype, x, xb, xr, xc, dw, yc, dpre, accumulate)) return rc;
        return 0;
    });
}

int d8k_dropout_forward(d8k_ctx* ctx, int dtype, const void* x, const void* residual, void* y, size_t n, const d8k_dropout* drop) {
    return entry(ctx, dtype, [&]() -> int { return dropout(ctx, dtype, x, residual, y, n, drop); });
}

int d8k_dropout_backward(d8k_ctx* ctx, int dtype, void* dx, const void* dy, size_t n, int accumulate, const d8k_dropout* drop) {
    return entry(ctx, dtype, [&]() -> int {
        if (accumulate && n > 0 && overlap(dx, n * esize(dtype), dy, n * esize(dtype))) return fail(D8K_ERR_ARGUMENT, "dropout: dx overlaps dy");
        return dropout(ctx, dtype, dy, accumulate ? dx : nullptr, dx, n, drop);
    });
}

int d8k_rms_norm_forward(d8k_ctx* ctx, int dtype, const void* x, const void* weight, float eps, void* y, float* rstd, size_t rows, int cols) {
    return entry(ctx, dtype, [&]() -> int {
        if (int rc = check_norm(rows, cols)) return rc;
        if (!(eps >= 0.0f) || std::isinf(eps)) return fail(D8K_ERR_ARGUMENT, "rms_norm: eps must be finite and not negative");
        if (rows == 0) return 0;
        if (!x || !weight || !y) return fail(D8K_ERR_ARGUMENT, "rms_norm: null pointer");
        const size_t bytes = rows * cols * esize(dtype), wbytes = cols * esize(dtype), rbytes = rows * sizeof(float);
        if ((y != x && overlap(y, bytes, x, bytes)) || overlap(y, bytes, weight, wbytes) || overlap(rstd, rbytes, x, bytes) || overlap(rstd, rbytes, y, bytes) ||
            overlap(rstd, rbytes, weight, wbytes))
            return fail(D8K_ERR_ARGUMENT, "rms_norm: an output overlaps an input");
        const size_t cap = static_cast<size_t>(ctx->num_sms) * 8;
        const unsigned grid = static_cast<unsigned>(rows < cap ? rows : cap);
        auto run = [&](auto zero) {
            using T = decltype(zero);
            rms_norm_forward_kernel<T><<<grid, 256, 0, ctx->stream>>>(static_cast<const T*>(x), static_cast<const T*>(weight), static_cast<T*>(y), rstd,
                                                                      rows, cols, eps);
        };
        if (dtype == D8K_F32) run(0.0f);
        else run(__half());
        D8K_CUDA(cudaGetLastError());
        count_launch();
        return 0;
    });
}

int d8k_rms_norm_backward(d8k_ctx* ctx, int dtype, const void* x, const void* weight, const float* rstd, void* dx, void* dweight, const void* dy,
                          size_t rows, int cols, int accumulate) {
    return entry(ctx, dtype, [&]() -> int {
        if (int rc = check_norm(rows, cols)) return rc;
        const size_t bytes = rows * cols * esize(dtype), wbytes = cols * esize(dtype), rbytes = rows * sizeof(float);
        if (rows == 0) {  // no row contributes
            if (dweight && !accumulate) D8K_CUDA(cudaMemsetAsync(dweight, 0, wbytes, ctx->stream));
            return 0;
        }
        if (!x || !weight || !rstd || !dy) return fail(D8K_ERR_ARGUMENT, "rms_norm: null pointer");
        if (overlap(dx, bytes, x, bytes) || overlap(dx, bytes, dy, bytes) || overlap(dx, bytes, weight, wbytes) || overlap(dx, bytes, rstd, rbytes) ||
            overlap(dweight, wbytes, x, bytes) || overlap(dweight, wbytes, dy, bytes) || overlap(dweight, wbytes, weight, wbytes) ||
            overlap(dweight, wbytes, rstd, rbytes) || overlap(dweight, wbytes, dx, bytes))
            return fail(D8K_ERR_ARGUMENT, "rms_norm: an output overlaps an input or the other output");
        if (dtype == D8K_F32)
            return rms_norm_backward<float>(ctx, static_cast<const float*>(x), static_cast<const float*>(weight), rstd, static_cast<float*>(dx),
                                            static_cast<float*>(dweight), static_cast<const float*>(dy), rows, cols, accumulate);
        return rms_norm_backward<__half>(ctx, static_cast<const __half*>(x), static_cast<const __half*>(weight), rstd, static_cast<__half*>(dx),
                                         static_cast<__half*>(dweight), static_cast<const __half*>(dy), rows, cols, accumulate);
    });
}

}  // extern "C"
