// Instantiations of the paired-CTA fp16 kernel for the gated feed-forward block: the gated product (256 x 128 outputs per pair), its gradients'
// products with eight storing warps, and split contractions of both whose slices split_sum_kernel adds.
#include "gemm2_kernel.cuh"
#include "gemm_host.h"

namespace d8k {

GemmLaunchFn lookup_f16_gated_pair() { return launch_pair_cfg<Gemm2Cfg<false, true, 3, 2, true>>; }

GemmLaunchFn lookup_f16_gated_pair_split() { return launch_pair_cfg<Gemm2Cfg<false, true, 3, 2, true, true>>; }

// the gradient of x multiplies two K-major operands, the gradient of w two MN-major ones
GemmLaunchFn lookup_f16_pair_split(bool mn) {
    if (mn) return launch_pair_cfg<Gemm2Cfg<true, true, 3, 2, false, true>>;
    return launch_pair_cfg<Gemm2Cfg<false, false, 3, 2, false, true>>;
}
GemmLaunchFn lookup_f16_pair_store(bool mn) {
    if (mn) return launch_pair_cfg<Gemm2Cfg<true, true, 3, 2, false, false, true>>;
    return launch_pair_cfg<Gemm2Cfg<false, false, 3, 2, false, false, true>>;
}

// ------------------------------------------------------------------------------------------------ the sum of a split product's slices
// One launch over the whole output instead of a tile's last CTA: the slices of a 256 x 256 tile are 256 KB each, which one SM would read at
// 0.1 TB/s.  Four columns per thread, the slices in order (same bits every run), eight 16-byte loads in flight.
// SplitSum::ws is [slice][tile][256][256], tile = (batch * tiles_m + m) * tiles_n + n.
__device__ __forceinline__ float4 sum_slices(const float* src, int splits, size_t stride) {
    float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int s = 0; s < splits; ++s) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(src + s * stride));
        t.x += v.x; t.y += v.y; t.z += v.z; t.w += v.w;
    }
    return t;
}

template <bool GATED>
__global__ void __launch_bounds__(256) split_sum_kernel(const SplitSum q) {
    constexpr int TILE_N = GATED ? 128 : 256;
    const unsigned quads = (q.N + 3) / 4;
    const size_t total = static_cast<size_t>(q.batch) * q.M * quads;
    const size_t stride = static_cast<size_t>(q.batch) * q.tiles_m * q.tiles_n * 65536;
    const unsigned long long offset = GATED && q.gated.dropping ? drop_offset(q.gated.drop) : 0;
    for (size_t i = blockIdx.x * 256ull + threadIdx.x; i < total; i += gridDim.x * 256ull) {
        const size_t line = total <= 0xffffffffu ? static_cast<unsigned>(i) / quads : i / quads;
        const int c = static_cast<int>(i - line * quads) * 4, b = q.batch == 1 ? 0 : static_cast<int>(line / q.M), r = static_cast<int>(line - static_cast<size_t>(b) * q.M);
        const size_t tile = (static_cast<size_t>(b) * q.tiles_m + r / 256) * q.tiles_n + c / TILE_N;
        const float* src = q.ws + (tile * 256 + r % 256) * 256 + c % TILE_N;
        const float4 first = sum_slices(src, q.splits, stride);
        float v[4] = {first.x, first.y, first.z, first.w};
        __half* out = static_cast<__half*>(q.C) + b * q.c_batch_stride + static_cast<long long>(r) * q.ldc + c;
        const int count = min(4, q.N - c);
        if constexpr (GATED) {
            const GatedTail& t = q.gated;
            const float4 second = sum_slices(src + 128, q.splits, stride);
            const float up[4] = {second.x, second.y, second.z, second.w};
            if (t.pre) {
                __half* pre = static_cast<__half*>(t.pre) + static_cast<long long>(r) * q.ldc + c;
                for (int k = 0; k < count; ++k) {
                    pre[k] = __float2half_rn(v[k]);
                    pre[t.pre_stride + k] = __float2half_rn(up[k]);
                }
            }
            with_activation(t.act, [&](auto act) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float value, slope;
                    activation<decltype(act)::value, true, false>(v[k], value, slope);
                    v[k] = value * up[k];
                }
            });
            if (t.dropping) {
                const unsigned long long at = static_cast<unsigned long long>(r) * q.ldc + c;
                const uint4 w0 = philox4x32(at >> 2, offset, t.drop.seed);
                const uint4 w1 = (at & 3) ? philox4x32((at >> 2) + 1, offset, t.drop.seed) : w0;
                const uint32_t words[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
                const int skip = static_cast<int>(at & 3);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t word = skip == 0 ? words[k] : skip == 1 ? words[k + 1] : skip == 2 ? words[k + 2] : words[k + 3];
                    v[k] = drop_keeps(t.drop, word) ? v[k] * t.drop.scale : 0.0f;
                }
            }
        }
        if (count == 4 && (reinterpret_cast<uintptr_t>(out) & 7) == 0) {
            uint2 w;
            __half2* h = reinterpret_cast<__half2*>(&w);
            if (q.beta) {
                w = *reinterpret_cast<const uint2*>(out);
                const float2 a = __half22float2(h[0]), d = __half22float2(h[1]);
                v[0] += a.x; v[1] += a.y; v[2] += d.x; v[3] += d.y;
            }
            h[0] = __floats2half2_rn(v[0], v[1]);
            h[1] = __floats2half2_rn(v[2], v[3]);
            *reinterpret_cast<uint2*>(out) = w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < count) out[k] = __float2half_rn(q.beta ? v[k] + __half2float(out[k]) : v[k]);
        }
    }
}

cudaError_t launch_split_sum(const Ctx* ctx, const SplitSum& q, bool gated) {
    const size_t total = static_cast<size_t>(q.batch) * q.M * ((q.N + 3) / 4), blocks = (total + 255) / 256, cap = static_cast<size_t>(ctx->num_sms) * 8;
    const unsigned grid = static_cast<unsigned>(blocks < cap ? blocks : cap);
    if (gated) split_sum_kernel<true><<<grid, 256, 0, ctx->stream>>>(q);
    else split_sum_kernel<false><<<grid, 256, 0, ctx->stream>>>(q);
    return cudaGetLastError();
}

}  // namespace d8k
