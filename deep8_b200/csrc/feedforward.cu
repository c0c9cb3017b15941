// extern "C" layer, part four (include/d8k.h): the gated feed-forward block - the gated projection pair with its gradients,
// counter-based dropout and the root-mean-square norm.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <exception>
#include <mutex>
#include <string>
#include <vector>

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
struct alignas(W * sizeof(T) < 16 ? W * sizeof(T) : 16) Pack {
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

// True in every thread of the CTA that is the last of `total` to arrive at `word` (Ctx::arrivals); all that the CTAs wrote before is then
// visible to it.  One atomic each, and the word is back at zero after the last: these kernels wait for nothing, so none of them can leave a
// word half-way.  (The contractions' compare-and-swap tickets, drawn by 16 CTAs at once, cost as much as a small product.)
__device__ __forceinline__ bool last_arrival(unsigned* word, unsigned total) {
    __shared__ int last;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicInc(word, total - 1) == total - 1;
    __syncthreads();
    __threadfence();
    return last;
}

__device__ __forceinline__ uint4 load_stream(const void* p) {  // read once: not kept in L1
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// The gated product for R rows of x at most (a token, or a few, while a model answers): bound by reading both weight matrices once, so
// no tensor cores.  A CTA takes a strip of 16 packs of columns (of 16 bytes) and a slice of the contraction; its 16 groups of 16 threads
// take every 16th k, each thread a pack of both projections, R products each in fp32.  The groups' sums meet in shared memory, the slices'
// in scratch memory: the CTA that finishes a strip last adds them in slice order and forms h.  fp32, 4096 -> 2 x 16384: 82 us for one row
// (6.5 TB/s), 88 for two to four, 146 for eight, whose multiply-adds no longer fit behind the loads; the tensor cores take 228 us.
template <int R>
__global__ void __launch_bounds__(256, R > 2 ? 2 : 4) gated_rows_kernel(const float* __restrict__ x, const float* __restrict__ w, float* __restrict__ h, int rows,
                                                                        int cols, int width, int k_per_slice, float* __restrict__ partial, unsigned* arrivals, GatedTail tail) {
    constexpr int V = 4, STRIP = 16 * V;
    constexpr int CHUNK = R > 4 ? 256 : 512;  // k staged at a time
    __shared__ alignas(16) float xs[CHUNK][R];
    __shared__ float sums[8][2 * R * V][16];
    const int lane = threadIdx.x & 15, kl = threadIdx.x >> 4;
    const int c = blockIdx.x * STRIP + lane * V;
    const int k_begin = blockIdx.y * k_per_slice, k_end = min(cols, k_begin + k_per_slice);
    const size_t second = static_cast<size_t>(cols) * width;
    float g[R][V] = {}, u[R][V] = {};
    for (int k0 = k_begin; k0 < k_end; k0 += CHUNK) {
        const int count = min(CHUNK, k_end - k0);
        __syncthreads();
        for (int i = threadIdx.x; i < R * CHUNK; i += 256) {
            const int r = i / CHUNK, k = i % CHUNK;
            xs[k][r] = r < rows && k < count ? x[static_cast<size_t>(r) * cols + k0 + k] : 0.0f;
        }
        __syncthreads();
        if (c < width) {
            const float* wp = w + static_cast<size_t>(k0) * width + c;
            constexpr int U = R > 4 ? 2 : 4;  // k per step: 2 U loads in flight
            for (int k0u = kl; k0u < count; k0u += 16 * U) {
                uint4 gv[U], uv[U];
#pragma unroll
                for (int q = 0; q < U; ++q) {
                    const int k = k0u + 16 * q;
                    gv[q] = uv[q] = make_uint4(0u, 0u, 0u, 0u);
                    if (k < count) {
                        gv[q] = load_stream(wp + static_cast<size_t>(k) * width);
                        uv[q] = load_stream(wp + second + static_cast<size_t>(k) * width);
                    }
                }
#pragma unroll
                for (int q = 0; q < U; ++q) {
                    const float* ge = reinterpret_cast<const float*>(&gv[q]);
                    const float* ue = reinterpret_cast<const float*>(&uv[q]);
                    // k is below CHUNK, a multiple of 16 U; from `count` on both factors are zeros
                    const Pack<float, R> a_row = *reinterpret_cast<const Pack<float, R>*>(xs[k0u + 16 * q]);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float a = a_row.v[r];
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            g[r][j] = fmaf(a, ge[j], g[r][j]);
                            u[r][j] = fmaf(a, ue[j], u[r][j]);
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            g[r][j] += __shfl_xor_sync(0xffffffffu, g[r][j], 16);
            u[r][j] += __shfl_xor_sync(0xffffffffu, u[r][j], 16);
            if ((threadIdx.x & 16) == 0) {
                sums[threadIdx.x >> 5][(2 * r) * V + j][lane] = g[r][j];
                sums[threadIdx.x >> 5][(2 * r + 1) * V + j][lane] = u[r][j];
            }
        }
    __syncthreads();
    const int slices = gridDim.y;
    float* mine = partial + (static_cast<size_t>(blockIdx.x) * slices + blockIdx.y) * (2 * R * STRIP);
    // output i of the strip: row i / STRIP, column i % STRIP; the gate's sum and, R * STRIP further, the up projection's
    auto summed = [&](int i, int which) {
        const int r = i / STRIP, col = i % STRIP;
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) t += sums[k][(2 * r + which) * V + col % V][col / V];
        return t;
    };
    if (slices > 1) {
        for (int i = threadIdx.x; i < R * STRIP; i += 256) {
            __stcg(mine + i, summed(i, 0));
            __stcg(mine + R * STRIP + i, summed(i, 1));
        }
        if (!last_arrival(arrivals + blockIdx.x, slices)) return;
    }
    const unsigned long long offset = tail.dropping ? drop_offset(tail.drop) : 0;
    const float* first = partial + static_cast<size_t>(blockIdx.x) * slices * (2 * R * STRIP);
    for (int i = threadIdx.x; i < R * STRIP; i += 256) {
        const int r = i / STRIP, col = blockIdx.x * STRIP + i % STRIP;
        if (r >= rows || col >= width) continue;
        float gate, up;
        if (slices > 1) {
            gate = up = 0.0f;
#pragma unroll 8
            for (int s = 0; s < slices; ++s) {
                gate += __ldcg(first + static_cast<size_t>(s) * (2 * R * STRIP) + i);
                up += __ldcg(first + static_cast<size_t>(s) * (2 * R * STRIP) + R * STRIP + i);
            }
        } else {
            gate = summed(i, 0);
            up = summed(i, 1);
        }
        const size_t at = static_cast<size_t>(r) * width + col;
        if (tail.pre) {
            static_cast<float*>(tail.pre)[at] = gate;
            static_cast<float*>(tail.pre)[tail.pre_stride + at] = up;
        }
        float out = 0.0f;
        with_activation(tail.act, [&](auto which) {
            float value, slope;
            activation<decltype(which)::value, false, false>(gate, value, slope);
            out = value * up;
        });
        if (tail.dropping) {
            const uint4 words = philox4x32(at >> 2, offset, tail.drop.seed);
            const uint32_t word = (at & 3) == 0 ? words.x : (at & 3) == 1 ? words.y : (at & 3) == 2 ? words.z : words.w;
            out = drop_keeps(tail.drop, word) ? out * tail.drop.scale : 0.0f;
        }
        h[at] = out;
    }
}

// widened elements of a pack and back; two halves per conversion where there are two
template <typename T, int W>
__device__ __forceinline__ void unpack(const Pack<T, W>& p, float (&f)[W]) {
    if constexpr (sizeof(T) == 2 && W % 2 == 0) {
#pragma unroll
        for (int k = 0; k < W; k += 2) {
            const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&p.v[k]));
            f[k] = t.x;
            f[k + 1] = t.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < W; ++k) f[k] = widen(p.v[k]);
    }
}
template <typename T, int W>
__device__ __forceinline__ Pack<T, W> pack_of(const float (&f)[W]) {
    Pack<T, W> p;
    if constexpr (sizeof(T) == 2 && W % 2 == 0) {
#pragma unroll
        for (int k = 0; k < W; k += 2) *reinterpret_cast<__half2*>(&p.v[k]) = __floats2half2_rn(f[k], f[k + 1]);
    } else {
#pragma unroll
        for (int k = 0; k < W; ++k) p.v[k] = narrow<T>(f[k]);
    }
    return p;
}

// 16 bytes from an address that is a multiple of the element size only: the two aligned pieces it touches, shifted together.  Both pieces must
// be readable.
template <int ESIZE>
__device__ __forceinline__ uint4 load_shifted(const char* p) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const uint4* q = reinterpret_cast<const uint4*>(at & ~static_cast<uintptr_t>(15));
    const uint4 a = __ldg(q);
    const unsigned shift = static_cast<unsigned>(at & 15);
    if (shift == 0) return a;
    const uint4 b = __ldg(q + 1);
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (shift & 8) {
#pragma unroll
        for (int k = 0; k < 6; ++k) w[k] = w[k + 2];
    }
    if (shift & 4) {
#pragma unroll
        for (int k = 0; k < 5; ++k) w[k] = w[k + 1];
    }
    if (ESIZE == 2 && (shift & 2)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Copies of row-major matrices with their rows padded by zeros to whole 128-byte pieces, so that TMA can read what starts anywhere: a
// 16-byte store per step from shifted 16-byte loads; a row's last piece, and what would touch memory around the matrix, element by element.
struct PadJobs {
    PadJob job[2];
};
template <typename T>
__global__ void __launch_bounds__(256) pad_kernel(PadJobs jobs, int count) {
    constexpr int W = 16 / sizeof(T);
    for (int q = 0; q < count; ++q) {
        const T* src = static_cast<const T*>(jobs.job[q].src);
        T* dst = static_cast<T*>(jobs.job[q].dst);
        const int cols = jobs.job[q].cols, packs = jobs.job[q].pitch / W;
        const size_t total = static_cast<size_t>(jobs.job[q].rows) * packs;
        const uintptr_t lowest = reinterpret_cast<uintptr_t>(src), highest = lowest + static_cast<size_t>(jobs.job[q].rows) * cols * sizeof(T);
        for (size_t i = blockIdx.x * 256ull + threadIdx.x; i < total; i += gridDim.x * 256ull) {
            const size_t r = total <= 0xffffffffu ? static_cast<unsigned>(i) / static_cast<unsigned>(packs) : i / packs;
            const int c = static_cast<int>(i - r * packs) * W;
            const T* from = src + r * cols + c;
            const uintptr_t piece = reinterpret_cast<uintptr_t>(from) & ~static_cast<uintptr_t>(15);
            Pack<T, W> v;
            if (c + W <= cols && piece >= lowest && piece + 32 <= highest) {
                *reinterpret_cast<uint4*>(&v) = load_shifted<sizeof(T)>(reinterpret_cast<const char*>(from));
            } else {
#pragma unroll
                for (int k = 0; k < W; ++k) v.v[k] = c + k < cols ? from[k] : narrow<T>(0.0f);
            }
            store_pack(dst + i * W, v);
        }
    }
}

// dpre from pre and dz: five accesses per element, bound by HBM (8192 x 16384 fp16: 211 us, 6.4 TB/s; 250 behind a hot product).  pre and dpre may be the same
// memory (an element is read and written by one thread), so nothing here is declared __restrict__.
// dpre is rounded to the tensors' type: the two products behind it take their operands in that type on the tensor cores, and an fp16 pair for
// each value would double their 3.3 ms.  fp16 gradients are 3.0e-4 off in norm for it, 2.1e-4 without; values of dpre below 2^-14 lose bits and
// below 2^-25 vanish, as everywhere between fp16 operators, which is what scaling the loss is for.
template <int ACT, typename T, int E>
__device__ __forceinline__ void gated_grad_elements(Pack<T, E>& g, Pack<T, E>& u, const Pack<T, E>& d, size_t i0, unsigned long long offset, const DropSpec& drop,
                                                    int dropping) {
    constexpr bool FAST = sizeof(T) == 2;
    float gate[E], up[E], dd[E];
    unpack(g, gate);
    unpack(u, up);
    unpack(d, dd);
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
        uint4 words = make_uint4(0u, 0u, 0u, 0u);
        if (dropping) words = philox4x32((i0 >> 2) + q, offset, drop.seed);
        const uint32_t word[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
        for (int k = 4 * q; k < 4 * q + 4; ++k) {
            float value, slope;
            activation<ACT, FAST, true>(gate[k], value, slope);
            if (dropping) dd[k] *= drop.scale;
            gate[k] = dd[k] * up[k] * slope;
            up[k] = dd[k] * value;
            if (dropping && !drop_keeps(drop, word[k - 4 * q])) gate[k] = up[k] = 0.0f;  // whatever the projections held
        }
    }
    g = pack_of<T, E>(gate);
    u = pack_of<T, E>(up);
}
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) gated_grad_pre_kernel(const T* pre, const T* dz, T* dpre, size_t n, int act, DropSpec drop, int dropping,
                                                             unsigned width, unsigned pitch) {
    constexpr int E = VEC ? 16 / sizeof(T) : 4;
    const unsigned long long offset = dropping ? drop_offset(drop) : 0;
    const size_t steps = (n + E - 1) / E, stride = gridDim.x * static_cast<size_t>(blockDim.x), second = n / width * pitch;
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
                // rows of dpre may be padded: where this step's first element goes
                const size_t r = n <= 0xffffffffu ? static_cast<unsigned>(i0) / width : i0 / width;
                unsigned col = static_cast<unsigned>(i0 - r * width);
                size_t at = r * pitch + col;
#pragma unroll
                for (int k = 0; k < E; ++k)
                    if (i0 + k < n) {
                        dpre[at] = g.v[k];
                        dpre[second + at] = u.v[k];
                        ++at;
                        if (++col == width) {  // on to the next row, `pitch` further than the last one began
                            col = 0;
                            at += pitch - width;
                        }
                    }
            }
        }
    });
}

// ------------------------------------------------------------------------------------------------ dropout
// One pack of y = (residual +) dropout(x); group: low word of the first four elements' counter
template <typename T, int E>
__device__ __forceinline__ Pack<T, E> drop_pack(const Pack<T, E>& a, const Pack<T, E>& b, bool add, uint32_t group, uint32_t group_hi,
                                                unsigned long long offset, const DropSpec& drop) {
    float v[E], r[E];
    unpack(a, v);
    if (add) unpack(b, r);
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
        const uint4 words = philox4x32(group + q, group_hi, offset, drop.seed);
        const uint32_t word[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
        for (int k = 4 * q; k < 4 * q + 4; ++k) {
            v[k] = drop_keeps(drop, word[k - 4 * q]) ? v[k] * drop.scale : 0.0f;
            if (add) v[k] += r[k];
        }
    }
    return pack_of<T, E>(v);
}
// y = (residual +) dropout(x): `residual` is the accumulated gradient itself in the backward pass.  VEC: bases on 16-byte boundaries; the
// last, partial pack goes element by element either way.  A launch covers at most 2^34 elements, whose counters share their high
// word.  y may be x or residual, so nothing is declared __restrict__.
// Bound by HBM in fp32 (8192 x 4096: 45.7 us, with a residual 64.7: 5.9 and 6.2 TB/s) and by the generator in fp16 (35.5 us, with a residual
// 37.5: the ten rounds alone take 27 us for these 2^25 words).  The registers are kept to what lets eight (fp32: six) CTAs hide each
// other's loads and rounds: 37.6 and 40.6 us with five.
template <typename T, bool VEC, bool ADD>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 8 : 6) dropout_kernel(const T* x, const T* residual, T* y, size_t n, uint32_t group_hi, DropSpec drop) {
    constexpr int E = VEC ? 16 / sizeof(T) : 4;
    const unsigned long long offset = drop_offset(drop);
    const size_t whole = n / E, stride = gridDim.x * static_cast<size_t>(blockDim.x);
    size_t s = blockIdx.x * static_cast<size_t>(blockDim.x) + threadIdx.x;
    if (VEC) {
        for (; s < whole; s += stride) {
            Pack<T, E> a = load_pack<T, E>(x + s * E), b = {};
            if (ADD) b = load_pack<T, E>(residual + s * E);
            store_pack(y + s * E, drop_pack(a, b, ADD, static_cast<uint32_t>(s * (E / 4)), group_hi, offset, drop));
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
        a = drop_pack(a, b, ADD, static_cast<uint32_t>(s * (E / 4)), group_hi, offset, drop);
#pragma unroll
        for (int k = 0; k < E; ++k)
            if (s * E + k < n) y[s * E + k] = a.v[k];
    }
}

// ------------------------------------------------------------------------------------------------ root-mean-square norm
// Rows are short enough for registers almost always: `tpr` threads (a power of two from 32 on) hold a row as N packs each, so x (and dy)
// cross from memory once.  A CTA has blockDim.x / tpr rows in work at a time.  Bound by HBM: forward 8192 x 4096 fp16 26.6 us (5.0 TB/s; a copy of
// the size 25), fp32 47 us (5.7 TB/s); one row of 4096 2.5 us.
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
        for (int k = 0; k < N; ++k) {
            float f[W];
            unpack(v[k], f);
#pragma unroll
            for (int j = 0; j < W; ++j) sum = fmaf(f[j], f[j], sum);
        }
        sum = row_sum(sum, tpr, part[buf]);
        const float inv = 1.0f / sqrtf(sum / cols + eps);
        if (live && rstd && at == 0) rstd[r] = inv;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int i = at + k * tpr;
            if (live && i < packs) {
                float f[W], w[W];
                unpack(v[k], f);
                unpack(load_pack<T, W>(weight + static_cast<size_t>(i) * W), w);
#pragma unroll
                for (int j = 0; j < W; ++j) f[j] *= inv * w[j];
                store_pack(y + r * cols + static_cast<size_t>(i) * W, pack_of<T, W>(f));
            }
        }
    }
}

// dx (+)= and this CTA's part of dweight (partial[blockIdx.x][cols]) in one pass over x and dy: the columns a thread holds are the same for
// every row, so their sums stay in its registers.  The next row's loads are issued before this row's sum is formed.
// 8192 x 4096: fp16 40.7 us and 6.5 for the slices' sum (4.3 TB/s together), bound by latency for want of warps: at 114 registers one CTA of 16
// fits an SM, half of the issue slots and half of the memory's bandwidth go unused (23 instructions per element); fp32 63 + 3 us (6.1 TB/s).
// Two packs per thread: 53 us with one, 65 with four.  Without the early loads fp32 took 82; a ring of rows in shared memory filled by cp.async
// was no faster.
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
    float next_inv = 0.0f;
    auto fetch = [&](size_t r) {
        const bool live = r < rows;
        next_inv = live ? rstd[r] : 0.0f;
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
        const float inv = next_inv;
        float n[N][W], u[N][W], sum = 0.0f;  // x * rstd, dy * weight
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int i = at + k * tpr;
            float w[W];
            Pack<T, W> wp = {};
            if (i < packs) wp = load_pack<T, W>(weight + static_cast<size_t>(i) * W);
            unpack(wp, w);
            unpack(xs[k], n[k]);
            unpack(gs[k], u[k]);
#pragma unroll
            for (int j = 0; j < W; ++j) {
                n[k][j] *= inv;
                dw[k][j] = fmaf(u[k][j], n[k][j], dw[k][j]);
                u[k][j] *= w[j];
                sum = fmaf(u[k][j], n[k][j], sum);
            }
        }
        if (r0 + step < rows) fetch(r + step);
        if (!dx) continue;
        const float mean = row_sum(sum, tpr, part[buf]) / cols;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int i = at + k * tpr;
            if (r >= rows || i >= packs) continue;
            T* dst = dx + r * cols + static_cast<size_t>(i) * W;
            float out[W] = {};
            if (accumulate) unpack(load_pack<T, W>(dst), out);
#pragma unroll
            for (int j = 0; j < W; ++j) out[j] = fmaf(inv, fmaf(-n[k][j], mean, u[k][j]), out[j]);
            store_pack(dst, pack_of<T, W>(out));
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
// the second time from cache, element by element (1000 x 40000 fp16 forward 79 us, 2.0 TB/s: right for any length, not fast).
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

// CTAs of `kernel` that one SM holds at once.  Asked once per kernel, block size and shared memory and kept: the driver's answer costs as
// much as a launch.
template <class Kernel>
int resident_ctas(Kernel* kernel, int threads, size_t dyn = 0) {
    struct Entry {
        const void* kernel;
        int threads;
        size_t dyn;
        int ctas;
    };
    static std::mutex mutex;
    static std::vector<Entry> known;
    std::lock_guard<std::mutex> lock(mutex);
    for (const Entry& e : known)
        if (e.kernel == reinterpret_cast<const void*>(kernel) && e.threads == threads && e.dyn == dyn) return e.ctas;
    int ctas = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, kernel, threads, dyn) != cudaSuccess || ctas < 1) ctas = 1;
    if (known.size() < 256) known.push_back(Entry{reinterpret_cast<const void*>(kernel), threads, dyn, ctas});
    return ctas;
}

// A grid for `steps` steps of one thread each, all of whose CTAs are in work at once: with a fixed eight per SM a kernel of which five fit
// ran a second, emptier round (dropout 49 us for 37).
template <class Kernel>
unsigned grid_for(const d8k_ctx* ctx, Kernel* kernel, size_t steps, int most_per_sm = 8) {
    const size_t blocks = (steps + 255) / 256;
    if (blocks <= static_cast<size_t>(ctx->num_sms)) return static_cast<unsigned>(blocks < 1 ? 1 : blocks);
    const int resident = resident_ctas(kernel, 256);
    const size_t cap = static_cast<size_t>(ctx->num_sms) * (resident < most_per_sm ? resident : most_per_sm);
    return static_cast<unsigned>(blocks > cap ? cap : blocks);
}

// The launch's form of a dropout argument; *on stays 0 when there is nothing to drop (none given, or p == 0).
int make_drop(const d8k_dropout* drop, DropSpec* spec, int* on = nullptr) {
    *spec = DropSpec{0, 0, nullptr, 0, 1, 1.0f};
    if (on) *on = 0;
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
    if (on) *on = drop->p > 0.0;
    return 0;
}

int check_gated(int activation, int xb, int xr, int xc, int yc) {
    if (activation < 0 || activation >= kActCount) return fail(D8K_ERR_ARGUMENT, "gated: no such activation");
    if (xb < 0 || xr < 0 || xc < 1 || yc < 1) return fail(D8K_ERR_ARGUMENT, "the shape is error");
    if (1LL * xb * xr > (1LL << 30) || xc > (1 << 30) || yc > (1 << 30)) return fail(D8K_ERR_ARGUMENT, "the shape is too large");
    return 0;
}

// The fp32 product for up to eight rows (nine would be two passes, 292 us where the tensor cores take 228), true when it is this kernel's: whole
// 16-byte packs of columns at 16-byte boundaries, and strips few enough for the arrival words.  (fp16 has gemm_gated_few.cu, which
// reads as fast for any of these row counts.)  As many slices as are in work at once, of at least 64 k.
bool gated_rows(d8k_ctx* ctx, const float* x, const float* w, float* h, int rows, int cols, int width, const GatedTail& tail) {
    constexpr int V = 4;
    const int strips = (width + 16 * V - 1) / (16 * V);
    if (rows > 8 || width % V != 0 || !aligned16({w}) || strips > kMaxCounters) return false;
    const int r = rows <= 2 ? rows : rows <= 4 ? 4 : 8;
    auto kernel = r == 1 ? gated_rows_kernel<1> : r == 2 ? gated_rows_kernel<2> : r == 4 ? gated_rows_kernel<4> : gated_rows_kernel<8>;
    long long slices = static_cast<long long>(ctx->num_sms) * resident_ctas(kernel, 256) / strips;
    if (slices > cols / 64) slices = cols / 64;
    const long long most = static_cast<long long>(ctx->scratch_bytes / (static_cast<size_t>(strips) * 2 * r * 16 * V * sizeof(float)));
    if (slices > most) slices = most;
    if (slices > 255) slices = 255;
    if (slices < 1) slices = 1;
    int per = static_cast<int>((cols + slices - 1) / slices);
    per = (per + 15) / 16 * 16;
    slices = (cols + per - 1) / per;
    kernel<<<dim3(strips, static_cast<unsigned>(slices)), 256, 0, ctx->stream>>>(x, w, h, rows, cols, width, per, ctx->scratch, ctx->arrivals, tail);
    return true;
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

// dpre's rows (of `width` elements, n in all) are written `pitch` apart
int gated_grad_pre(d8k_ctx* ctx, int dtype, int activation, const void* pre, const void* dz, void* dpre, size_t n, size_t width, size_t pitch,
                   const d8k_dropout* drop) {
    if (activation < 0 || activation >= kActCount) return fail(D8K_ERR_ARGUMENT, "gated: no such activation");
    DropSpec spec;
    int dropping = 0;
    if (int rc = make_drop(drop, &spec, &dropping)) return rc;
    if (n == 0) return 0;
    if (!pre || !dz || !dpre) return fail(D8K_ERR_ARGUMENT, "gated: null pointer");
    const size_t bytes = n * esize(dtype), out_bytes = n / width * pitch * esize(dtype);
    if (((dpre != pre || pitch != width) && overlap(dpre, 2 * out_bytes, pre, 2 * bytes)) || overlap(dpre, 2 * out_bytes, dz, bytes))
        return fail(D8K_ERR_ARGUMENT, "gated: dpre overlaps an input");
    const int per = static_cast<int>(16 / esize(dtype));
    const bool vec = aligned16({pre, dz, dpre}) && n % per == 0 && pitch == width;
    auto run = [&](auto zero) {
        using T = decltype(zero);
        auto kernel = vec ? gated_grad_pre_kernel<T, true> : gated_grad_pre_kernel<T, false>;
        // fp16: four CTAs per SM, though five fit (8192 x 16384: 211 us with four, 223 with five, 229 with three; 4096 x 8192: 59.4 either way)
        const int most = vec && sizeof(T) == 2 ? 4 : 8;
        kernel<<<grid_for(ctx, kernel, (n + per - 1) / (vec ? per : 4), most), 256, 0, ctx->stream>>>(
            static_cast<const T*>(pre), static_cast<const T*>(dz), static_cast<T*>(dpre), n, activation, spec, dropping, static_cast<unsigned>(width),
            static_cast<unsigned>(pitch));
    };
    if (dtype == D8K_F32) run(0.0f);
    else run(__half());
    D8K_CUDA(cudaGetLastError());
    count_launch();
    return 0;
}

// The operands of the two gradient products: x [rows, xc], w and dpre [2, ...].  Where their rows do not start on 16-byte boundaries (or are no
// whole 128-byte pieces, see below) the products read copies with padded rows (in the context's padding memory) that TMA can describe; the loader warps would fetch such rows
// element by element (333 x 250 x 1001 fp32: 203 us for both gradients).
struct GatedOperands {
    HostOperand x, w, dpre;
};
// dpre_to_come: dpre is not there yet (gated_backward writes it): its place is chosen, nothing copied.  x or w without a pointer is left out.
int gated_operands(d8k_ctx* ctx, int dtype, GatedOperands* o, const void* x, const void* w, const void* dpre, int rows, int xc, int yc, bool dpre_to_come) {
    o->x = matrix(x, true, xc);
    o->w = matrix(w, false, yc, 2, 1LL * xc * yc);
    o->dpre = matrix(dpre, false, yc, 2, 1LL * rows * yc);
    const int piece = static_cast<int>(128 / esize(dtype));
    struct Part {
        HostOperand* o;
        long long rows;
        int cols;
    } parts[3] = {{&o->x, rows, xc}, {&o->w, 2LL * xc, yc}, {&o->dpre, 2LL * rows, yc}};
    const bool dpre_whole = yc % piece == 0 || dpre_to_come || !rows_aligned(dpre, yc, dtype);
    size_t bytes = 0, at[3] = {};
    bool wanted[3] = {};
    for (int k = 0; k < 3; ++k) {
        // Rows of whole 128-byte pieces as well where that lets a faster kernel read them: x (a small copy) for the paired kernel or, in fp32, any TMA
        // kernel; dpre for the same when it costs no copy, in fp32 always; w where the paired kernel saves more than the copy costs.  The paired
        // kernel is fp16's, and out of the question for x and w while dpre's rows are neither whole pieces nor copied.
        const bool whole = parts[k].cols % piece == 0;
        const bool useful = !whole && (k == 0   ? dtype == D8K_F32 || dpre_whole
                                       : k == 1 ? dtype == D8K_F16 && dpre_whole && gated_grad_x_wants_padded_w(ctx, rows, xc, yc)
                                                : dpre_to_come || dtype == D8K_F32);
        wanted[k] = parts[k].o->ptr && (useful || !rows_aligned(parts[k].o->ptr, parts[k].cols, dtype));
        at[k] = bytes;
        if (wanted[k]) bytes += (static_cast<size_t>(parts[k].rows) * ((parts[k].cols + piece - 1) / piece * piece) * esize(dtype) + 255) & ~static_cast<size_t>(255);
    }
    char* base = bytes ? static_cast<char*>(pad_memory(ctx, bytes)) : nullptr;
    if (!base) return 0;
    PadJob jobs[3];
    int count = 0;
    for (int k = 0; k < 3; ++k) {
        if (!wanted[k]) continue;
        HostOperand& h = *parts[k].o;
        const int pitch = (parts[k].cols + piece - 1) / piece * piece;
        if (k != 2 || !dpre_to_come) {
            jobs[count].src = h.ptr;
            jobs[count].dst = base + at[k];
            jobs[count].rows = parts[k].rows;
            jobs[count].cols = parts[k].cols;
            jobs[count++].pitch = pitch;
        }
        h.ptr = base + at[k];
        h.ld = pitch;
        h.padded = true;
        if (h.batch_count == 2) h.batch_stride = parts[k].rows / 2 * pitch;
    }
    for (int k = 0; k < count; k += 2) D8K_CUDA(launch_pad(ctx, dtype, jobs + k, count - k < 2 ? count - k : 2));
    return 0;
}

int gated_grad_x(d8k_ctx* ctx, int dtype, void* dx, int rows, int xc, int yc, const GatedOperands& o, int accumulate) {
    GemmProblem g;  // the two products join one contraction: a batch of two that is summed
    g.dtype = dtype;
    g.M = rows; g.N = xc; g.K = yc;
    g.a = o.dpre;
    g.b = o.w;
    g.kbatch = 2;
    g.C = dx;
    g.ldc = xc;
    g.beta = accumulate ? 1 : 0;
    g.precise = true;
    return run_gated_grad(ctx, g);
}

int gated_grad_w(d8k_ctx* ctx, int dtype, void* dw, int rows, int xc, int yc, const GatedOperands& o, int accumulate) {
    GemmProblem g;
    g.dtype = dtype;
    g.M = xc; g.N = yc; g.K = rows;
    g.a = o.x;
    g.b = o.dpre;
    g.b.mn = true;
    g.batch = 2;
    g.C = dw;
    g.ldc = yc;
    g.c_batch_stride = 1LL * xc * yc;
    g.beta = accumulate ? 1 : 0;
    g.precise = true;
    return run_gated_grad(ctx, g);
}

int dropout(d8k_ctx* ctx, int dtype, const void* x, const void* residual, void* y, size_t n, const d8k_dropout* drop) {
    if (!drop) return fail(D8K_ERR_ARGUMENT, "dropout: null pointer");
    DropSpec spec;
    if (int rc = make_drop(drop, &spec)) return rc;
    if (n == 0) return 0;
    if (!x || !y) return fail(D8K_ERR_ARGUMENT, "dropout: null pointer");
    const size_t bytes = n * esize(dtype);
    if ((y != x && overlap(y, bytes, x, bytes)) || (y != residual && overlap(y, bytes, residual, bytes)))
        return fail(D8K_ERR_ARGUMENT, "dropout: the output overlaps an input");
    const int per = static_cast<int>(16 / esize(dtype));
    const bool vec = aligned16({x, residual, y});
    auto run = [&](auto zero) {
        using T = decltype(zero);
        auto kernel = residual ? (vec ? dropout_kernel<T, true, true> : dropout_kernel<T, false, true>)
                               : (vec ? dropout_kernel<T, true, false> : dropout_kernel<T, false, false>);
        constexpr size_t kMost = static_cast<size_t>(1) << 34;  // elements whose counters share their high word
        for (size_t first = 0; first < n; first += kMost) {
            const size_t count = n - first < kMost ? n - first : kMost;
            kernel<<<grid_for(ctx, kernel, (count + per - 1) / (vec ? per : 4)), 256, 0, ctx->stream>>>(
                static_cast<const T*>(x) + first, residual ? static_cast<const T*>(residual) + first : nullptr, static_cast<T*>(y) + first, count,
                static_cast<uint32_t>(first >> 34), spec);
            count_launch();
        }
    };
    if (dtype == D8K_F32) run(0.0f);
    else run(__half());
    D8K_CUDA(cudaGetLastError());
    return 0;
}

// How a row of `packs` packs is spread over threads.  The register kernels hold 1, 2 or 4 packs per thread (1, 4 or 16 single elements);
// `start` is the count to begin with when there are rows enough to fill the GPU, one pack per thread and more threads per row
// otherwise, because then latency counts.  packs_per_thread == 0: too long for registers.
struct RowPlan {
    int tpr, packs_per_thread, threads, group;
};
RowPlan plan_rows(const d8k_ctx* ctx, size_t rows, int packs, bool vec, int start, int least_threads) {
    for (int n = rows < static_cast<size_t>(ctx->num_sms) * 4 ? 1 : start; n <= (vec ? 4 : 16); n *= vec ? 2 : 4) {
        int tpr = 32;
        while (tpr < 512 && static_cast<long long>(tpr) * n < packs) tpr *= 2;
        if (static_cast<long long>(tpr) * n < packs) continue;
        const int threads = tpr > least_threads ? tpr : least_threads;
        return RowPlan{tpr, n, threads, threads / tpr};
    }
    return RowPlan{0, 0, 0, 0};
}

template <typename T>
int rms_norm_forward(d8k_ctx* ctx, const T* x, const T* weight, float eps, T* y, float* rstd, size_t rows, int cols) {
    constexpr int W = 16 / sizeof(T);
    const bool vec = aligned16({x, weight, y}) && cols % W == 0;
    const RowPlan p = plan_rows(ctx, rows, vec ? cols / W : cols, vec, 4, 256);
    if (p.packs_per_thread == 0) {
        const size_t cap = static_cast<size_t>(ctx->num_sms) * 4;
        rms_norm_forward_long_kernel<T><<<static_cast<unsigned>(rows < cap ? rows : cap), 512, 0, ctx->stream>>>(x, weight, y, rstd, rows, cols, eps);
    } else {
        const size_t groups = (rows + p.group - 1) / p.group;
        auto kernel = vec ? (p.packs_per_thread == 1 ? rms_norm_forward_kernel<T, W, 1> : p.packs_per_thread == 2 ? rms_norm_forward_kernel<T, W, 2>
                                                                                                            : rms_norm_forward_kernel<T, W, 4>)
                          : (p.packs_per_thread == 1 ? rms_norm_forward_kernel<T, 1, 1> : p.packs_per_thread == 4 ? rms_norm_forward_kernel<T, 1, 4>
                                                                                                            : rms_norm_forward_kernel<T, 1, 16>);
        const size_t sms = ctx->num_sms, cap = groups <= sms ? sms : sms * resident_ctas(kernel, p.threads);
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
    const RowPlan p = plan_rows(ctx, rows, vec ? cols / W : cols, vec, vec ? 2 : 4, 512);
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
        slices = static_cast<size_t>(ctx->num_sms) * resident_ctas(kernel, p.threads, dyn);
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

bool rows_aligned(const void* ptr, long long ld, int dtype) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && ld * esize(dtype) % 16 == 0; }

void* pad_memory(Ctx* ctx, size_t bytes) {
    if (bytes <= ctx->pad_bytes) return ctx->pads.back();
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(ctx->stream, &capturing) != cudaSuccess) {
        cudaGetLastError();
        return nullptr;
    }
    if (capturing != cudaStreamCaptureStatusNone) return nullptr;
    // another stream may be under capture, by this thread or another: an allocation would end it in the global mode
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    struct Restore {
        cudaStreamCaptureMode* mode;
        ~Restore() { cudaThreadExchangeStreamCaptureMode(mode); }
    } restore{&mode};
    size_t want = ctx->pad_bytes * 2 > bytes ? ctx->pad_bytes * 2 : bytes;  // the sum of all stays below twice the last
    if (want < (static_cast<size_t>(16) << 20)) want = static_cast<size_t>(16) << 20;
    ctx->pads.reserve(ctx->pads.size() + 1);
    void* p = nullptr;
    if (cudaMalloc(&p, want) != cudaSuccess) {
        cudaGetLastError();
        return nullptr;
    }
    ctx->pads.push_back(p);
    ctx->pad_bytes = want;
    return p;
}

cudaError_t launch_pad(Ctx* ctx, int dtype, const PadJob* jobs, int count) {
    PadJobs j;
    size_t steps = 0;
    for (int k = 0; k < count; ++k) {
        j.job[k] = jobs[k];
        steps += static_cast<size_t>(jobs[k].rows) * jobs[k].pitch * esize(dtype) / 16;
    }
    auto run = [&](auto kernel) { kernel<<<grid_for(static_cast<d8k_ctx*>(ctx), kernel, steps), 256, 0, ctx->stream>>>(j, count); };
    if (dtype == D8K_F32) run(pad_kernel<float>);
    else run(pad_kernel<__half>);
    count_launch();
    return cudaGetLastError();
}

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
        const GatedTail tail{activation, dropping, pre, 1LL * rows * yc, spec};
        if (dtype == D8K_F32 && gated_rows(ctx, static_cast<const float*>(x), static_cast<const float*>(w), static_cast<float*>(h), rows, xc, yc, tail)) {
            D8K_CUDA(cudaGetLastError());
            count_launch();
            set_last_kernel("f32 gated rows");
            return 0;
        }
        GatedProblem g;
        g.dtype = dtype;
        g.M = rows; g.N = yc; g.K = xc;
        g.a = x;
        g.b = w;
        g.C = h;
        g.tail = tail;
        return run_gated(ctx, g);
    });
}

int d8k_gated_grad_pre(d8k_ctx* ctx, int dtype, int activation, const void* pre, const void* dz, void* dpre, size_t n, const d8k_dropout* drop) {
    return entry(ctx, dtype, [&]() -> int { return gated_grad_pre(ctx, dtype, activation, pre, dz, dpre, n, 1, 1, drop); });
}

int d8k_gated_grad_x_into(d8k_ctx* ctx, int dtype, void* dx, int xb, int xr, int xc, const void* w, int yc, const void* dpre, int accumulate) {
    return entry(ctx, dtype, [&]() -> int {
        if (int rc = check_gated(0, xb, xr, xc, yc)) return rc;
        const int rows = xb * xr;
        if (rows == 0) return 0;
        if (!dx || !w || !dpre) return fail(D8K_ERR_ARGUMENT, "gated: null pointer");
        const size_t es = esize(dtype), x_bytes = es * rows * xc;
        if (overlap(dx, x_bytes, w, 2 * es * xc * yc) || overlap(dx, x_bytes, dpre, 2 * es * rows * yc))
            return fail(D8K_ERR_ARGUMENT, "gated: dx overlaps an input");
        GatedOperands o;
        if (int rc = gated_operands(ctx, dtype, &o, nullptr, w, dpre, rows, xc, yc, false)) return rc;
        return gated_grad_x(ctx, dtype, dx, rows, xc, yc, o, accumulate);
    });
}

int d8k_gated_grad_w_into(d8k_ctx* ctx, int dtype, const void* x, int xb, int xr, int xc, void* dw, int yc, const void* dpre, int accumulate) {
    return entry(ctx, dtype, [&]() -> int {
        if (int rc = check_gated(0, xb, xr, xc, yc)) return rc;
        const int rows = xb * xr;
        const size_t es = esize(dtype), w_bytes = 2 * es * xc * yc;
        if (!dw || (rows > 0 && (!x || !dpre))) return fail(D8K_ERR_ARGUMENT, "gated: null pointer");
        if (rows == 0) {  // no row contributes
            if (!accumulate) D8K_CUDA(cudaMemsetAsync(dw, 0, w_bytes, ctx->stream));
            return 0;
        }
        if (overlap(dw, w_bytes, x, es * rows * xc) || overlap(dw, w_bytes, dpre, 2 * es * rows * yc)) return fail(D8K_ERR_ARGUMENT, "gated: dw overlaps an input");
        GatedOperands o;
        if (int rc = gated_operands(ctx, dtype, &o, x, nullptr, dpre, rows, xc, yc, false)) return rc;
        return gated_grad_w(ctx, dtype, dw, rows, xc, yc, o, accumulate);
    });
}

int d8k_gated_backward(d8k_ctx* ctx, int dtype, int activation, const void* x, int xb, int xr, int xc, const void* w, int yc, const void* pre,
                       const void* dz, void* dpre, void* dx, void* dw, int accumulate, const d8k_dropout* drop) {
    return entry(ctx, dtype, [&]() -> int {
        if (int rc = check_gated(activation, xb, xr, xc, yc)) return rc;
        const int rows = xb * xr;
        const size_t es = esize(dtype), xs = es * rows * xc, ws = 2 * es * xc * yc, hs = es * rows * yc;
        DropSpec spec;
        int dropping = 0;
        if (int rc = make_drop(drop, &spec, &dropping)) return rc;
        if (rows == 0) {  // no row contributes
            if (dw && !accumulate) D8K_CUDA(cudaMemsetAsync(dw, 0, ws, ctx->stream));
            return 0;
        }
        // everything is checked before the first launch
        if (!pre || !dz || !dpre || (dx && !w) || (dw && !x)) return fail(D8K_ERR_ARGUMENT, "gated: null pointer");
        if ((dpre != pre && overlap(dpre, 2 * hs, pre, 2 * hs)) || overlap(dpre, 2 * hs, dz, hs) || overlap(dpre, 2 * hs, x, xs) || overlap(dpre, 2 * hs, w, ws) ||
            overlap(dx, xs, x, xs) || overlap(dx, xs, w, ws) || overlap(dx, xs, pre, 2 * hs) || overlap(dx, xs, dz, hs) || overlap(dx, xs, dpre, 2 * hs) ||
            overlap(dw, ws, x, xs) || overlap(dw, ws, w, ws) || overlap(dw, ws, pre, 2 * hs) || overlap(dw, ws, dz, hs) || overlap(dw, ws, dpre, 2 * hs) ||
            overlap(dx, xs, dw, ws))
            return fail(D8K_ERR_ARGUMENT, "gated: an output overlaps an input or another output");
        GatedOperands o;
        if (int rc = gated_operands(ctx, dtype, &o, dw ? x : nullptr, dx ? w : nullptr, dpre, rows, xc, yc, true)) return rc;
        void* where = const_cast<void*>(o.dpre.ptr);
        if (o.dpre.padded && o.dpre.ld > yc)  // the zeros behind each row
            D8K_CUDA(cudaMemset2DAsync(static_cast<char*>(where) + es * yc, es * o.dpre.ld, 0, es * (o.dpre.ld - yc), 2 * static_cast<size_t>(rows), ctx->stream));
        if (int rc = gated_grad_pre(ctx, dtype, activation, pre, dz, where, static_cast<size_t>(rows) * yc, yc, static_cast<size_t>(o.dpre.ld), drop)) return rc;
        if (dx)
            if (int rc = gated_grad_x(ctx, dtype, dx, rows, xc, yc, o, accumulate)) return rc;
        if (dw)
            if (int rc = gated_grad_w(ctx, dtype, dw, rows, xc, yc, o, accumulate)) return rc;
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
