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
// A pack of W consecutive elements as one memory access: 16 bytes, or a single element where rows or bases are not aligned to that.
template <typename T, int W>
struct alignas(W * sizeof(T)) Pack {
    T v[W];
};
template <typename T, int W>
__device__ __forceinline__ Pack<T, W> load_pack(const T* p) {
    return *reinterpret_cast<const Pack<T, W>*>(p);
}
template <typename T, int W>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, W>& v) {
    *reinterpret_cast<Pack<T, W>*>(p) = v;
}

// dpre from pre and dz: five accesses per element, bound by HBM (8192 x 16384 fp16: 234 us, 5.7 TB/s).  pre and dpre may be the same
// memory (an element is read and written by one thread), so nothing here is declared __restrict__.
template <int ACT, typename T, int E>
__device__ __forceinline__ void gated_grad_elements(Pack<T, E>& g, Pack<T, E>& u, const Pack<T, E>& d, size_t i0, unsigned long long offset, const DropSpec& drop,
                                                    int dropping) {
    constexpr bool FAST = sizeof(T) == 2;
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
        uint4 words = make_uint4(0u, 0u, 0u, 0u);
        if (dropping) words = philox4x32((i0 >> 2) + q, offset, drop.seed);
        const uint32_t word[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float value, slope;
            activation<ACT, FAST, true>(widen(g.v[4 * q + k]), value, slope);
            const float dd = dropping ? widen(d.v[4 * q + k]) * drop.scale : widen(d.v[4 * q + k]);
            float dg = dd * widen(u.v[4 * q + k]) * slope, du = dd * value;
            if (dropping && !drop_keeps(drop, word[k])) dg = du = 0.0f;  // whatever the projections held
            g.v[4 * q + k] = narrow<T>(dg);
            u.v[4 * q + k] = narrow<T>(du);
        }
    }
}
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) gated_grad_pre_kernel(const T* pre, const T* dz, T* dpre, size_t n, int act, DropSpec drop, int dropping) {
    constexpr int E = VEC ? 16 / sizeof(T) : 4;
    const unsigned long long offset = dropping ? drop_offset(drop) : 0;
    const size_t steps = (n + E - 1) / E, stride = gridDim.x * static_cast<size_t>(blockDim.x);
    with_activation(act, [&](auto which) {
        for (size_t s = blockIdx.x * static_cast<size_t>(blockDim.x) + threadIdx.x; s < steps; s += stride) {
            const size_t i0 = s * E;
            Pack<T, E> g, u, d;
            if (VEC) {
                g = load_pack<T, E>(pre + i0);
                u = load_pack<T, E>(pre + n + i0);
                d = load_pack<T, E>(dz + i0);
            } else {
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    const bool in = i0 + k < n;
                    g.v[k] = in ? pre[i0 + k] : narrow<T>(0.0f);
                    u.v[k] = in ? pre[n + i0 + k] : narrow<T>(0.0f);
                    d.v[k] = in ? dz[i0 + k] : narrow<T>(0.0f);
                }
            }
            gated_grad_elements<decltype(which)::value>(g, u, d, i0, offset, drop, dropping);
            if (VEC) {
                store_pack(dpre + i0, g);
                store_pack(dpre + n + i0, u);
            } else {
#pragma unroll
                for (int k = 0; k < E; ++k)
                    if (i0 + k < n) {
                        dpre[i0 + k] = g.v[k];
                        dpre[n + i0 + k] = u.v[k];
                    }
            }
        }
    });
}

// ------------------------------------------------------------------------------------------------ dropout
// One pack of y = (residual +) dropout(x), i0 the index of its first element (a multiple of four)
template <typename T, int E>
__device__ __forceinline__ void drop_pack(Pack<T, E>& a, const Pack<T, E>& b, bool add, size_t i0, unsigned long long offset, const DropSpec& drop) {
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
        const uint4 words = philox4x32((i0 >> 2) + q, offset, drop.seed);
        const uint32_t word[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float v = drop_keeps(drop, word[k]) ? widen(a.v[4 * q + k]) * drop.scale : 0.0f;
            if (add) v += widen(b.v[4 * q + k]);
            a.v[4 * q + k] = narrow<T>(v);
        }
    }
}
// y = (residual +) dropout(x): `residual` is the accumulated gradient itself in the backward pass.  VEC: bases on 16-byte boundaries; the
// last, partial pack goes element by element either way.  y may be x or residual, so nothing is declared __restrict__.
template <typename T, bool VEC, bool ADD>
__global__ void __launch_bounds__(256) dropout_kernel(const T* x, const T* residual, T* y, size_t n, DropSpec drop) {
    constexpr int E = VEC ? 16 / sizeof(T) : 4;
    const unsigned long long offset = drop_offset(drop);
    const size_t whole = n / E, stride = gridDim.x * static_cast<size_t>(blockDim.x);
    size_t s = blockIdx.x * static_cast<size_t>(blockDim.x) + threadIdx.x;
    if (VEC) {
        constexpr int U = 2;  // packs in flight per thread
        for (; s + (U - 1) * stride < whole; s += U * stride) {
            Pack<T, E> a[U], b[U] = {};
#pragma unroll
            for (int k = 0; k < U; ++k) {
                a[k] = load_pack<T, E>(x + (s + k * stride) * E);
                if (ADD) b[k] = load_pack<T, E>(residual + (s + k * stride) * E);
            }
#pragma unroll
            for (int k = 0; k < U; ++k) {
                drop_pack(a[k], b[k], ADD, (s + k * stride) * E, offset, drop);
                store_pack(y + (s + k * stride) * E, a[k]);
            }
        }
        for (; s < whole; s += stride) {
            Pack<T, E> a = load_pack<T, E>(x + s * E), b = {};
            if (ADD) b = load_pack<T, E>(residual + s * E);
            drop_pack(a, b, ADD, s * E, offset, drop);
            store_pack(y + s * E, a);
        }
    }
    for (; s * E < n; s += stride) {
        Pack<T, E> a = {}, b = {};
#pragma unroll
        for (int k = 0; k < E; ++k)
            if (s * E + k < n) {
                a.v[k] = x[s * E + k];
                if (ADD) b.v[k] = residual[s * E + k];
            }
        drop_pack(a, b, ADD, s * E, offset, drop);
#pragma unroll
        for (int k = 0; k < E; ++k)
            if (s * E + k < n) y[s * E + k] = a.v[k];
    }
}

// ------------------------------------------------------------------------------------------------ root-mean-square norm
// Rows are short enough for registers almost always: `tpr` threads (a power of two from 32 on) hold a row as N packs each, so x (and dy)
// cross from memory once.  A CTA has blockDim.x / tpr rows in work at a time.
//
// Sum over the tpr threads of a row, the same value in each of them.  part: 16 floats of shared memory that the previous row's sum does
// not use (two buffers in turn, one barrier per row).
__device__ __forceinline__ float row_sum(float v, int tpr, float* part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (tpr == 32) return v;
    const int warp = threadIdx.x >> 5, per = tpr >> 5;
    if ((threadIdx.x & 31) == 0) part[warp] = v;
    __syncthreads();
    const int first = warp & ~(per - 1);
    float t = 0.0f;
    for (int k = 0; k < per; ++k) t += part[first + k];
    return t;
}

template <typename T, int W, int N>
__global__ void __launch_bounds__(512) rms_norm_forward_kernel(const T* x, const T* weight, T* y, float* rstd, size_t rows, int cols, float eps, int tpr) {
    __shared__ float part[2][16];
    const int at = threadIdx.x & (tpr - 1), sub = threadIdx.x / tpr, group = blockDim.x / tpr;
    const int packs = cols / W;
    int buf = 0;
    for (size_t r0 = blockIdx.x * static_cast<size_t>(group); r0 < rows; r0 += gridDim.x * static_cast<size_t>(group), buf ^= 1) {
        const size_t r = r0 + sub;
        const bool live = r < rows;
        const T* row = x + r * cols;
        Pack<T, W> v[N];
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int i = at + k * tpr;
            v[k] = Pack<T, W>{};
            if (live && i < packs) v[k] = load_pack<T, W>(row + static_cast<size_t>(i) * W);
        }
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int j = 0; j < W; ++j) sum = fmaf(widen(v[k].v[j]), widen(v[k].v[j]), sum);
        sum = row_sum(sum, tpr, part[buf]);
        const float inv = 1.0f / sqrtf(sum / cols + eps);
        if (live && rstd && at == 0) rstd[r] = inv;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int i = at + k * tpr;
            if (live && i < packs) {
                const Pack<T, W> w = load_pack<T, W>(weight + static_cast<size_t>(i) * W);
#pragma unroll
                for (int j = 0; j < W; ++j) v[k].v[j] = narrow<T>(widen(v[k].v[j]) * inv * widen(w.v[j]));
                store_pack(y + r * cols + static_cast<size_t>(i) * W, v[k]);
            }
        }
    }
}

// dx (+)= and this CTA's part of dweight (partial[blockIdx.x][cols]) in one pass over x and dy: the columns a thread holds are the same for
// every row, so their sums stay in its registers.  The next row's loads are issued before this row's sum is formed.
template <typename T, int W, int N>
__global__ void __launch_bounds__(512) rms_norm_backward_kernel(const T* __restrict__ x, const T* __restrict__ weight, const float* __restrict__ rstd,
                                                                T* dx, float* __restrict__ partial, const T* __restrict__ dy, size_t rows, int cols,
                                                                int accumulate, int tpr) {
    extern __shared__ float columns[];  // (group - 1) x cols, only for several rows at a time
    __shared__ float part[2][16];
    const int at = threadIdx.x & (tpr - 1), sub = threadIdx.x / tpr, group = blockDim.x / tpr;
    const int packs = cols / W;
    const size_t step = gridDim.x * static_cast<size_t>(group);
    float dw[N][W];
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int j = 0; j < W; ++j) dw[k][j] = 0.0f;
    Pack<T, W> xs[N], gs[N];
    float inv = 0.0f;
    auto fetch = [&](size_t r) {
        const bool live = r < rows;
        inv = live ? rstd[r] : 0.0f;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int i = at + k * tpr;
            xs[k] = gs[k] = Pack<T, W>{};
            if (live && i < packs) {
                xs[k] = load_pack<T, W>(x + r * cols + static_cast<size_t>(i) * W);
                gs[k] = load_pack<T, W>(dy + r * cols + static_cast<size_t>(i) * W);
            }
        }
    };
    fetch(blockIdx.x * static_cast<size_t>(group) + sub);
    int buf = 0;
    for (size_t r0 = blockIdx.x * static_cast<size_t>(group); r0 < rows; r0 += step, buf ^= 1) {
        const size_t r = r0 + sub;
        const float scale = inv;
        float n[N][W], u[N][W], sum = 0.0f;  // x * rstd, dy * weight
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int i = at + k * tpr;
            Pack<T, W> w = {};
            if (i < packs) w = load_pack<T, W>(weight + static_cast<size_t>(i) * W);
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const float g = widen(gs[k].v[j]);
                n[k][j] = widen(xs[k].v[j]) * scale;
                u[k][j] = g * widen(w.v[j]);
                dw[k][j] = fmaf(g, n[k][j], dw[k][j]);
                sum = fmaf(u[k][j], n[k][j], sum);
            }
        }
        if (r0 + step < rows) fetch(r + step);
        if (!dx) continue;
        const float mean = row_sum(sum, tpr, part[buf]) / cols;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int i = at + k * tpr;
            if (r < rows && i < packs) {
                T* dst = dx + r * cols + static_cast<size_t>(i) * W;
                Pack<T, W> out = {};
                if (accumulate) out = load_pack<T, W>(dst);
#pragma unroll
                for (int j = 0; j < W; ++j) out.v[j] = narrow<T>(fmaf(scale, u[k][j] - n[k][j] * mean, accumulate ? widen(out.v[j]) : 0.0f));
                store_pack(dst, out);
            }
        }
    }
    if (!partial) return;
    // the CTA's rows meet in shared memory, in order
    if (sub > 0) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int i = at + k * tpr;
            if (i < packs)
#pragma unroll
                for (int j = 0; j < W; ++j) columns[static_cast<size_t>(sub - 1) * cols + i * W + j] = dw[k][j];
        }
    }
    if (group > 1) __syncthreads();
    if (sub == 0) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int i = at + k * tpr;
            if (i < packs) {
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    float t = dw[k][j];
                    for (int g = 1; g < group; ++g) t += columns[static_cast<size_t>(g - 1) * cols + i * W + j];
                    partial[static_cast<size_t>(blockIdx.x) * cols + i * W + j] = t;
                }
            }
        }
    }
}

// dweight (+)= the slices of `partial` in order: 32 columns per CTA, 32 warps that take slices w, w + 32, ... and meet in shared memory in
// warp order - a single thread per column spent one memory latency after another (39 us for 444 slices).
template <typename T>
__global__ void __launch_bounds__(1024) rms_norm_grad_w_final_kernel(T* __restrict__ dweight, const float* __restrict__ partial, int slices, int cols,
                                                                     int accumulate) {
    __shared__ float part[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float sum = 0.0f;
    if (c < cols) {
#pragma unroll 8
        for (int s = warp; s < slices; s += 32) sum += partial[static_cast<size_t>(s) * cols + c];
    }
    part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < cols) {
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < 32; ++k) t += part[k][lane];
        dweight[c] = narrow<T>(accumulate ? widen(dweight[c]) + t : t);
    }
}

// Rows too long for registers (above 16384 fp16 or 8192 fp32 columns in 16-byte packs, 8192 otherwise): one CTA per row, the row read twice,
// the second time from cache.
template <typename T>
__global__ void __launch_bounds__(512) rms_norm_forward_long_kernel(const T* x, const T* weight, T* y, float* rstd, size_t rows, int cols, float eps) {
    __shared__ float part[2][16];
    int buf = 0;
    for (size_t r = blockIdx.x; r < rows; r += gridDim.x, buf ^= 1) {
        const T* row = x + r * cols;
        float sum = 0.0f;
        for (int c = threadIdx.x; c < cols; c += 512) {
            const float v = widen(row[c]);
            sum = fmaf(v, v, sum);
        }
        sum = row_sum(sum, 512, part[buf]);
        const float inv = 1.0f / sqrtf(sum / cols + eps);
        if (rstd && threadIdx.x == 0) rstd[r] = inv;
        for (int c = threadIdx.x; c < cols; c += 512) y[r * cols + c] = narrow<T>(widen(row[c]) * inv * widen(weight[c]));
    }
}
template <typename T>
__global__ void __launch_bounds__(512) rms_norm_grad_x_long_kernel(const T* __restrict__ x, const T* __restrict__ weight, const float* __restrict__ rstd,
                                                                   T* __restrict__ dx, const T* __restrict__ dy, size_t rows, int cols, int accumulate) {
    __shared__ float part[2][16];
    int buf = 0;
    for (size_t r = blockIdx.x; r < rows; r += gridDim.x, buf ^= 1) {
        const size_t at = r * cols;
        const float inv = rstd[r];
        float sum = 0.0f;
        for (int c = threadIdx.x; c < cols; c += 512) sum = fmaf(widen(dy[at + c]) * widen(weight[c]), widen(x[at + c]) * inv, sum);
        const float mean = row_sum(sum, 512, part[buf]) / cols;
        for (int c = threadIdx.x; c < cols; c += 512) {
            float v = inv * (widen(dy[at + c]) * widen(weight[c]) - widen(x[at + c]) * inv * mean);
            if (accumulate) v += widen(dx[at + c]);
            dx[at + c] = narrow<T>(v);
        }
    }
}
template <typename T>
__global__ void __launch_bounds__(256) rms_norm_grad_w_long_kernel(const T* __restrict__ x, const float* __restrict__ rstd, const T* __restrict__ dy,
                                                                   float* __restrict__ partial, size_t rows, int cols, size_t rows_per_slice) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    const size_t r0 = blockIdx.y * rows_per_slice;
    const size_t r1 = r0 + rows_per_slice < rows ? r0 + rows_per_slice : rows;
    float sum = 0.0f;
    for (size_t r = r0; r < r1; ++r) sum = fmaf(widen(dy[r * cols + c]), widen(x[r * cols + c]) * rstd[r], sum);
    partial[static_cast<size_t>(blockIdx.y) * cols + c] = sum;
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
    const bool vec = aligned16({x, residual, y});
    const int grid = grid_for(ctx, (n + per - 1) / (vec ? per : 4));
    auto run = [&](auto zero) {
        using T = decltype(zero);
        auto kernel = residual ? (vec ? dropout_kernel<T, true, true> : dropout_kernel<T, false, true>)
                               : (vec ? dropout_kernel<T, true, false> : dropout_kernel<T, false, false>);
        kernel<<<grid, 256, 0, ctx->stream>>>(static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<T*>(y), n, spec);
    };
    if (dtype == D8K_F32) run(0.0f);
    else run(__half());
    D8K_CUDA(cudaGetLastError());
    count_launch();
    return 0;
}

// How a row of `packs` packs is spread over threads.  The register kernels hold 1, 2 or 4 packs per thread (1, 4 or 16 single elements);
// `start` is the count to begin with when there are rows enough to fill the GPU, one pack per thread and more threads per row
// otherwise, because then latency counts.  packs_per_thread == 0: too long for registers.
struct RowPlan {
    int tpr, packs_per_thread, threads, group;
};
RowPlan plan_rows(const d8k_ctx* ctx, size_t rows, int packs, bool vec, int start) {
    for (int n = rows < static_cast<size_t>(ctx->num_sms) * 4 ? 1 : start; n <= (vec ? 4 : 16); n *= vec ? 2 : 4) {
        int tpr = 32;
        while (tpr < 512 && static_cast<long long>(tpr) * n < packs) tpr *= 2;
        if (static_cast<long long>(tpr) * n < packs) continue;
        const int threads = tpr > 256 ? tpr : 256;
        return RowPlan{tpr, n, threads, threads / tpr};
    }
    return RowPlan{0, 0, 0, 0};
}

template <typename T>
int rms_norm_forward(d8k_ctx* ctx, const T* x, const T* weight, float eps, T* y, float* rstd, size_t rows, int cols) {
    constexpr int W = 16 / sizeof(T);
    const bool vec = aligned16({x, weight, y}) && cols % W == 0;
    const RowPlan p = plan_rows(ctx, rows, vec ? cols / W : cols, vec, 4);
    if (p.packs_per_thread == 0) {
        const size_t cap = static_cast<size_t>(ctx->num_sms) * 4;
        rms_norm_forward_long_kernel<T><<<static_cast<unsigned>(rows < cap ? rows : cap), 512, 0, ctx->stream>>>(x, weight, y, rstd, rows, cols, eps);
    } else {
        const size_t groups = (rows + p.group - 1) / p.group, cap = static_cast<size_t>(ctx->num_sms) * (2048 / p.threads);
        auto kernel = vec ? (p.packs_per_thread == 1 ? rms_norm_forward_kernel<T, W, 1> : p.packs_per_thread == 2 ? rms_norm_forward_kernel<T, W, 2>
                                                                                                            : rms_norm_forward_kernel<T, W, 4>)
                          : (p.packs_per_thread == 1 ? rms_norm_forward_kernel<T, 1, 1> : p.packs_per_thread == 4 ? rms_norm_forward_kernel<T, 1, 4>
                                                                                                            : rms_norm_forward_kernel<T, 1, 16>);
        kernel<<<static_cast<unsigned>(groups < cap ? groups : cap), p.threads, 0, ctx->stream>>>(x, weight, y, rstd, rows, cols, eps, p.tpr);
    }
    D8K_CUDA(cudaGetLastError());
    count_launch();
    return 0;
}

template <typename T>
int rms_norm_backward(d8k_ctx* ctx, const T* x, const T* weight, const float* rstd, T* dx, T* dweight, const T* dy, size_t rows, int cols, int accumulate) {
    constexpr int W = 16 / sizeof(T);
    const bool vec = aligned16({x, weight, dx, dy}) && cols % W == 0;
    const RowPlan p = plan_rows(ctx, rows, vec ? cols / W : cols, vec, vec ? 2 : 4);
    const size_t most = ctx->scratch_bytes / (static_cast<size_t>(cols) * sizeof(float));  // slices of column sums the scratch memory holds
    if (dweight && most < 1) return fail(D8K_ERR_ARGUMENT, "the context's scratch memory is smaller than one row of floats");
    if (!dx && !dweight) return 0;
    size_t slices = 0;
    if (p.packs_per_thread > 0) {
        const size_t groups = (rows + p.group - 1) / p.group;
        auto kernel = vec ? (p.packs_per_thread == 1 ? rms_norm_backward_kernel<T, W, 1> : p.packs_per_thread == 2 ? rms_norm_backward_kernel<T, W, 2>
                                                                                                             : rms_norm_backward_kernel<T, W, 4>)
                          : (p.packs_per_thread == 1 ? rms_norm_backward_kernel<T, 1, 1> : p.packs_per_thread == 4 ? rms_norm_backward_kernel<T, 1, 4>
                                                                                                             : rms_norm_backward_kernel<T, 1, 16>);
        const size_t dyn = dweight ? static_cast<size_t>(p.group - 1) * cols * sizeof(float) : 0;
        int per_sm = 0;
        D8K_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, p.threads, dyn));
        slices = static_cast<size_t>(ctx->num_sms) * (per_sm < 1 ? 1 : per_sm);
        if (slices > groups) slices = groups;
        if (dweight && slices > most) slices = most;
        kernel<<<static_cast<unsigned>(slices), p.threads, dyn, ctx->stream>>>(x, weight, rstd, dx, dweight ? ctx->scratch : nullptr, dy, rows, cols, accumulate,
                                                                              p.tpr);
        D8K_CUDA(cudaGetLastError());
        count_launch();
    } else {
        if (dweight) {
            const int strips = (cols + 255) / 256;
            slices = (static_cast<size_t>(ctx->num_sms) * 8 + strips - 1) / strips;
            if (slices > most) slices = most;
            if (slices > (rows + 7) / 8) slices = (rows + 7) / 8;
            const size_t per = (rows + slices - 1) / slices;
            slices = (rows + per - 1) / per;
            rms_norm_grad_w_long_kernel<T><<<dim3(strips, static_cast<unsigned>(slices)), 256, 0, ctx->stream>>>(x, rstd, dy, ctx->scratch, rows, cols, per);
            D8K_CUDA(cudaGetLastError());
            count_launch();
        }
        if (dx) {
            const size_t cap = static_cast<size_t>(ctx->num_sms) * 4;
            rms_norm_grad_x_long_kernel<T><<<static_cast<unsigned>(rows < cap ? rows : cap), 512, 0, ctx->stream>>>(x, weight, rstd, dx, dy, rows, cols, accumulate);
            D8K_CUDA(cudaGetLastError());
            count_launch();
        }
    }
    if (dweight) {
        rms_norm_grad_w_final_kernel<T><<<(cols + 31) / 32, 1024, 0, ctx->stream>>>(dweight, ctx->scratch, static_cast<int>(slices), cols, accumulate);
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
        if (dtype == D8K_F32)
            return rms_norm_forward<float>(ctx, static_cast<const float*>(x), static_cast<const float*>(weight), eps, static_cast<float*>(y), rstd, rows, cols);
        return rms_norm_forward<__half>(ctx, static_cast<const __half*>(x), static_cast<const __half*>(weight), eps, static_cast<__half*>(y), rstd, rows, cols);
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
