// The gated product for a few rows (fp16, up to 128 tokens while a model answers): act(x w[0]) * (x w[1]), bound by reading the weights.
//
// The operands change places: 128 columns of a projection are the M side of the MMA (w is MN-major there), the tokens its N side, so that
// an accumulator is 128 x (16 .. 128) instead of 128 rows of which most would be padding, a partial sum of a split contraction is
// rows x 128 values, and a stage of shared memory is almost all weights.
// Measured (4096 -> 2 x 16384, whose weights alone are 41 us of HBM time): 44 us for 1 to 16 rows (6.1 TB/s), 47 for 48, 48 for 128; the ordinary
// gated kernels 57 to 77 us for 8 to 64 rows.  2048 -> 2 x 5504 (6.9 us of HBM time): 14 us for up to 8 rows, 16.5 for 48, 20 for 128; there the
// launch, the first loads and the joining of two slices take as long as the weights.
//
// Roles, barriers and bounded waits are those of d8k_gemm_kernel with one thread per role.  A work item is a strip of 128 columns and a
// slice of the contraction.  Unsplit, persistent CTAs walk over the strips, the epilogue of one (two accumulator buffers) beside the main
// loop of the next.  Split, the CTAs of a cluster take the slices of one strip and add them through each other's shared memory, each CTA
// its share of the tokens; with partial sums in scratch memory and one CTA to add them, that tail took longer than the product.
#include "gemm2_kernel.cuh"
#include "gemm_host.h"

namespace d8k {

template <int NT_>
struct FewCfg {
    static constexpr int NT = NT_;                    // tokens of a tile
    // Two k-blocks of 64 per stage where three such stages fit: a CTA reads 94 GB/s in boxes of 32 KB, 73 in boxes of 16 KB.  With more tokens
    // two stages would fit, and five of one k-block read faster.
    static constexpr int SUB = NT <= 32 ? 2 : 1;
    static constexpr int BK = 64 * SUB;
    static constexpr int W_BYTES = BK * 128 * 2;      // BK k x 128 columns of one projection, two chunks of 64 columns
    static constexpr int X_BYTES = SUB * NT * 128;    // k-major tiles of 64 k
    static constexpr int STAGE_BYTES = 2 * W_BYTES + X_BYTES;
    static constexpr int STAGES = NT <= 32 ? 3 : NT == 64 ? 5 : 4;
    static constexpr int ACC_COLS = 2 * NT;           // gate, up
    static constexpr int TMEM_COLS = 2 * ACC_COLS;
    // warps 0-3 and 6-9 are two groups of epilogue warps that take 16 tokens in turn
    static constexpr int PRODUCER_WARP = 4, MMA_WARP = 5, EPI_THREADS = 256, THREADS = 320;
    static constexpr int BAR_BYTES = 256;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + BAR_BYTES + 1024;
    static_assert(SMEM_BYTES <= 227 * 1024 && SMEM_BYTES > 114 * 1024, "one CTA per SM");
    static_assert(STAGES * STAGE_BYTES >= 2 * NT * 128 * 4, "a split CTA's sums take the ring's place");
    static_assert(8 * (2 * STAGES + 4) + 8 <= BAR_BYTES, "barrier block");
};

__device__ __forceinline__ void st_shared_f32(uint32_t addr, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }
__device__ __forceinline__ float ld_cluster_f32(uint32_t cluster_addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
    return v;
}

// One column of T tokens t0, t0 + step, ...: h, and the projections when kept.  Overwrites gate.
template <int T>
__device__ __forceinline__ void finish_tokens(const GatedFewParams& p, int t0, int step, int rows, int col, float* gate, const float* up) {
    const GatedTail& t = p.gated;
    if (t.pre) {
#pragma unroll
        for (int i = 0; i < T; ++i)
            if (t0 + i * step < rows) {
                __half* dst = static_cast<__half*>(t.pre) + static_cast<size_t>(t0 + i * step) * p.width + col;
                dst[0] = __float2half_rn(gate[i]);
                dst[t.pre_stride] = __float2half_rn(up[i]);
            }
    }
    with_activation(t.act, [&](auto act) {
#pragma unroll
        for (int i = 0; i < T; ++i) {
            float value, slope;
            activation<decltype(act)::value, true, false>(gate[i], value, slope);
            gate[i] = value * up[i];
        }
    });
    if (t.dropping) {
        const unsigned long long offset = drop_offset(t.drop);
#pragma unroll
        for (int i = 0; i < T; ++i) {
            const size_t at = static_cast<size_t>(t0 + i * step) * p.width + col;
            const uint4 words = philox4x32(at >> 2, offset, t.drop.seed);
            const uint32_t word = (at & 3) == 0 ? words.x : (at & 3) == 1 ? words.y : (at & 3) == 2 ? words.z : words.w;
            gate[i] = drop_keeps(t.drop, word) ? gate[i] * t.drop.scale : 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < T; ++i)
        if (t0 + i * step < rows) static_cast<__half*>(p.h)[static_cast<size_t>(t0 + i * step) * p.width + col] = __float2half_rn(gate[i]);
}

// tmX: x as {64 k, rows, k-block of 64, 1}, box {64, NT, SUB, 1}, or without x_chunked as {K, rows, 1}, box {64, NT, 1};  tmW: w as {64 columns, K,
// chunk of 64 columns, projection}, box {64, BK, 2, 1}, or without w_chunked as {columns, K, projection}, box {64, BK, 1}
template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, 1)
d8k_gated_few_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const GatedFewParams p) {
    constexpr int STAGES = Cfg::STAGES, NT = Cfg::NT;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bar_base = smem_base + STAGES * Cfg::STAGE_BYTES;
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
    auto tfull_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + a); };
    auto tempty_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + 2 + a); };
    const uint32_t tmem_slot = bar_base + 8u * (2 * STAGES + 4);
    __shared__ volatile int s_abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(full_bar(s), 1);
            ptx::mbar_init(empty_bar(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            ptx::mbar_init(tfull_bar(a), 1);
            ptx::mbar_init(tempty_bar(a), Cfg::EPI_THREADS);
        }
        ptx::fence_mbar_init();
    }
    if (warp == Cfg::MMA_WARP) {
        ptx::tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
        ptx::tmem_relinquish();
    }
    if (warp == Cfg::PRODUCER_WARP && lane == 0) {
        ptx::tma_prefetch_desc(&tmX);
        ptx::tma_prefetch_desc(&tmW);
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    uint32_t tmem_base;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot) : "memory");
    auto stage_w = [&](int s) { return smem_base + s * Cfg::STAGE_BYTES; };
    auto stage_x = [&](int s) { return smem_base + s * Cfg::STAGE_BYTES + 2 * Cfg::W_BYTES; };

    if (warp == Cfg::PRODUCER_WARP) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int w = blockIdx.x; ok && w < p.total_work; w += gridDim.x) {
            const int strip = w / p.splits, split = w - strip * p.splits;
            const int kb_end = min(p.num_kb, (split + 1) * p.kb_per_split);
            for (int kb = split * p.kb_per_split; kb < kb_end; ++kb) {
                ok = wait_bar(empty_bar(stage), phase ^ 1, &s_abort, p.status, (kRoleProducer << 8) | 1);
                if (!ok) break;
                if (lane == 0) {
                    const uint32_t bar = full_bar(stage);
                    ptx::mbar_arrive_expect_tx(bar, Cfg::STAGE_BYTES);
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        const uint32_t dst = stage_w(stage) + m * Cfg::W_BYTES;
                        if (p.w_chunked) {
                            ptx::tma_load_4d(dst, &tmW, bar, 0, kb * Cfg::BK, strip * 2, m);
                        } else {
                            ptx::tma_load_3d(dst, &tmW, bar, strip * 128, kb * Cfg::BK, m);
                            ptx::tma_load_3d(dst + Cfg::W_BYTES / 2, &tmW, bar, strip * 128 + 64, kb * Cfg::BK, m);
                        }
                    }
                    if (p.x_chunked) {
                        ptx::tma_load_4d(stage_x(stage), &tmX, bar, 0, 0, kb * Cfg::SUB, 0);
                    } else {
#pragma unroll
                        for (int j = 0; j < Cfg::SUB; ++j) ptx::tma_load_3d(stage_x(stage) + j * NT * 128, &tmX, bar, kb * Cfg::BK + 64 * j, 0, 0);
                    }
                }
                __syncwarp();
                if (++stage == STAGES) { stage = 0; phase ^= 1; }
            }
        }
    } else if (warp == Cfg::MMA_WARP) {
        constexpr uint32_t idesc = ptx::make_idesc(0u, true, false, 128, NT);
        int stage = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        for (int w = blockIdx.x; ok && w < p.total_work; w += gridDim.x) {
            const int strip = w / p.splits, split = w - strip * p.splits;
            const int kb_begin = split * p.kb_per_split, kb_end = min(p.num_kb, kb_begin + p.kb_per_split);
            ok = wait_bar(tempty_bar(acc), acc_phase ^ 1, &s_abort, p.status, (kRoleMma << 8) | 2);
            if (!ok) break;
            ptx::tc_fence_after_sync();
            const uint32_t d = tmem_base + acc * Cfg::ACC_COLS;
            for (int kb = kb_begin; kb < kb_end; ++kb) {
                ok = wait_bar(full_bar(stage), phase, &s_abort, p.status, (kRoleMma << 8) | 1);
                if (!ok) break;
                ptx::tc_fence_after_sync();
                if (lane == 0) {
                    const uint64_t dw = ptx::smem_desc(stage_w(stage), Cfg::BK * 128, 1024, ptx::kLayoutSw128);
                    const uint64_t dx = ptx::smem_desc(stage_x(stage), 16, 1024, ptx::kLayoutSw128);
#pragma unroll
                    for (int s = 0; s < Cfg::BK / 16; ++s) {
                        const uint32_t accumulate = (kb > kb_begin || s > 0) ? 1u : 0u;
                        const uint64_t db = dx + (((s >> 2) * (NT * 128) + (s & 3) * 32) >> 4);
                        ptx::mma_f16(d, dw + ((s * 16 * 128) >> 4), db, idesc, accumulate);
                        ptx::mma_f16(d + NT, dw + ((Cfg::W_BYTES + s * 16 * 128) >> 4), db, idesc, accumulate);
                    }
                    ptx::tc_commit(empty_bar(stage));
                    if (kb + 1 == kb_end) ptx::tc_commit(tfull_bar(acc));
                }
                __syncwarp();
                if (++stage == STAGES) { stage = 0; phase ^= 1; }
            }
            if (++acc == 2) { acc = 0; acc_phase ^= 1; }
        }
    } else {
        // epilogue: this thread's column of both projections
        const int group = warp >= 4, quarter = warp & 3;  // the accumulator lanes this warp may read: 32 quarter + lane
        const int col_in_strip = quarter * 32 + lane;
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        for (int w = blockIdx.x; ok && w < p.total_work; w += gridDim.x) {
            ok = wait_bar(tfull_bar(acc), acc_phase, &s_abort, p.status, (kRoleEpilogue << 8) | 3);
            if (!ok) break;
            ptx::tc_fence_after_sync();
            const int col = w / p.splits * 128 + col_in_strip;
            const uint32_t taddr = tmem_base + acc * Cfg::ACC_COLS + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
            for (int t0 = 16 * group; t0 < NT && t0 < p.rows; t0 += 32) {
                uint32_t g[16], u[16];
                __syncwarp();
                ptx::tmem_ld_32x16(taddr + t0, g);
                ptx::tmem_ld_32x16(taddr + NT + t0, u);
                ptx::tmem_ld_wait();
                float gate[16], up[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    gate[i] = __uint_as_float(g[i]);
                    up[i] = __uint_as_float(u[i]);
                }
                if (p.splits == 1) {
                    if (col < p.width) finish_tokens<16>(p, t0, 1, p.rows, col, gate, up);
                } else {  // every load and MMA of this CTA is over: the ring holds its sums, [projection][token][128]
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (t0 + i < p.rows) {
                            st_shared_f32(smem_base + 4u * ((t0 + i) * 128 + col_in_strip), gate[i]);
                            st_shared_f32(smem_base + 4u * ((p.rows + t0 + i) * 128 + col_in_strip), up[i]);
                        }
                }
            }
            ptx::tc_fence_before_sync();
            ptx::mbar_arrive(tempty_bar(acc));
            if (++acc == 2) { acc = 0; acc_phase ^= 1; }
        }
    }

    if (p.splits > 1) {
        // The cluster's CTAs hold one strip's slices.  CTA r finishes the tokens r, r + splits, ...: it adds the slices' sums in slice
        // order from the CTAs' shared memories.  Both barriers are reached by every thread on every path.
        __syncthreads();
        ptx::cluster_arrive();
        ptx::cluster_wait();
        const int col_in_strip = (warp & 3) * 32 + lane, col = blockIdx.x / p.splits * 128 + col_in_strip;
        if (warp != Cfg::PRODUCER_WARP && warp != Cfg::MMA_WARP && !s_abort && col < p.width) {
            const int rank = blockIdx.x % p.splits, group = warp >= 4;
#pragma unroll 1
            for (int t0 = rank + 8 * group * p.splits; t0 < p.rows; t0 += 16 * p.splits) {
                float gate[8] = {}, up[8] = {};
#pragma unroll 1
                for (int s = 0; s < p.splits; ++s) {
                    const uint32_t base = ptx::map_to_rank(smem_base, s) + 4u * col_in_strip;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int token = t0 + i * p.splits;
                        if (token < p.rows) {
                            gate[i] += ld_cluster_f32(base + 512u * token);
                            up[i] += ld_cluster_f32(base + 512u * (p.rows + token));
                        }
                    }
                }
                finish_tokens<8>(p, t0, p.splits, p.rows, col, gate, up);
            }
        }
        __syncwarp();
        ptx::cluster_arrive();  // no CTA's shared memory goes while another may read it
        ptx::cluster_wait();
    }

    if (s_abort) {
        // copies and MMAs still in flight land before shared and tensor memory are released
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (warp == Cfg::MMA_WARP) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
    }
}

template <class Cfg>
static cudaError_t launch_few(int grid, cudaStream_t stream, const CUtensorMap& tx, const CUtensorMap& tw, const GatedFewParams& p) {
    static bool configured[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(d8k_gated_few_kernel<Cfg>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(Cfg::THREADS);
    config.dynamicSmemBytes = Cfg::SMEM_BYTES;
    config.stream = stream;
    cudaLaunchAttribute cluster = {};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = p.splits;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    config.attrs = &cluster;
    config.numAttrs = p.splits > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&config, d8k_gated_few_kernel<Cfg>, tx, tw, p);
}

cudaError_t launch_gated_few(int tokens, int grid, cudaStream_t stream, const CUtensorMap& tx, const CUtensorMap& tw, const GatedFewParams& p) {
    switch (tokens) {
        case 16: return launch_few<FewCfg<16>>(grid, stream, tx, tw, p);
        case 32: return launch_few<FewCfg<32>>(grid, stream, tx, tw, p);
        case 64: return launch_few<FewCfg<64>>(grid, stream, tx, tw, p);
        default: return launch_few<FewCfg<128>>(grid, stream, tx, tw, p);
    }
}

}  // namespace d8k
