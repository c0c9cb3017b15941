// Host-side description of one contraction and the context that launches it.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cstddef>
#include <string>
#include <vector>

#include "gemm_kernel.cuh"

namespace d8k {

struct Ctx {
    int device = 0;
    int num_sms = 148;
    cudaStream_t stream = nullptr;
    float* scratch = nullptr;  // split-K partial tiles
    size_t scratch_bytes = 0;
    int* counters = nullptr;   // kMaxCounters tile ticket words (GemmParams::counters)
    unsigned epoch_counter = 0;  // this context's split launches so far, modulo 2^24 (GemmParams::epoch)
    unsigned* arrivals = nullptr;  // kMaxCounters words, zero between launches: kernels whose last CTA finishes the work count their CTAs here
    int* status = nullptr;     // device status word
    // Memory for copies of operands with padded rows, grown as calls need it (pad_memory).  What a captured graph may point at is never freed
    // before the context.
    std::vector<void*> pads;
    size_t pad_bytes = 0;  // of the last one
    GroupEntry* group_buf = nullptr;  // device memory for kMaxGroups entries of a grouped launch (null: launches are never grouped)
};
constexpr int kMaxCounters = 4096;
constexpr int kMaxGroups = 16;

// One operand as the host sees it.  mn == false: K-major (the contraction index is contiguous); mn == true: MN-major.
struct HostOperand {
    const void* ptr = nullptr;
    bool mn = false;
    bool is_virtual = false;   // virtual im2col matrix (cr) over the image at ptr
    long long ld = 0;          // pitch in elements of the stored matrix
    int rmod = 0;              // > 0: stored row g lives at (g % rmod) * ld + (g / rmod) * ld2
    long long ld2 = 0;
    long long batch_stride = 0;
    int batch_count = 1;
    bool padded = false;       // a stored matrix whose rows go on as zeros to the next multiple of 128 bytes (launch_pad)
    ConvRule cr = {};
    // halo != 0 (set by run_gemm, fp32 only): the virtual matrix is fetched as per-tile patches of halo_rows x halo_wp pixels
    int halo = 0, halo_wp = 0, halo_rows = 0;
    // A filter [oc, FH, FW, ic] restricted to the taps (f0y + ty*j, f0x + tx*i), j < nfy, i < nfx - one residue class of a
    // strided convolution.  With rmod == 0 the operand is K-major rows of filters, columns (j, i, c); with rmod > 0 it is
    // the filter read by tap, W'[((j, i), co)][ci].  TMA only.
    struct TapSubset {
        int on = 0, f0y = 0, f0x = 0, ty = 1, tx = 1, nfy = 0, nfx = 0, FH = 0, FW = 0, ic = 0, oc = 0;
    } sub;
};

struct GemmProblem {
    int dtype = 0;
    int M = 0, N = 0, K = 0;
    HostOperand a, b;
    void* C = nullptr;
    long long ldc = 0, c_batch_stride = 0;
    int batch = 1;    // independent outputs
    int kbatch = 1;   // batches summed into one output
    int beta = 0;
    int epi = 0, beta2 = 0;  // fused element-wise tail (GemmParams::epi)
    float epi_a = 0.f, epi_b = 0.f;
    void* E1 = nullptr;
    void* E2 = nullptr;
    bool precise = false;    // fp32 with short accumulation chains (GemmCfg::PRECISE); both operands K-major or both MN-major
    int force_splits = 0;    // > 0: this many splits (bounded by the k-block count and the scratch) instead of the plan's own choice
    int ticket_base = 0;     // first of the context's tickets this launch uses (grouped launches give every contraction its own range)
    bool ws_strict = false;  // split within ws / ws_bytes, never in the context's own scratch (run_gemm_group carves that up itself)
    void* ws = nullptr;  // optional caller scratch for split-K
    size_t ws_bytes = 0;
    // scatter_rows > 0: C is not used; output rows [k * scatter_rows, (k + 1) * scatter_rows) go to scatter_base[k], a
    // matrix of scatter_rows rows with pitch ldc (GemmParams::scatter_rows)
    int scatter_rows = 0, scatter_count = 0;
    void* scatter_base[kMaxScatter] = {};
    OutMap out = {};  // strided placement of rows / columns in the output tensor (GemmParams::out); FastDivs filled by run_gemm
};

// A row-major matrix stack to copy with its rows padded by zeros to whole 128-byte pieces
struct PadJob {
    const void* src = nullptr;
    void* dst = nullptr;
    long long rows = 0;  // of all matrices of the stack
    int cols = 0, pitch = 0;
};
// `bytes` of the context's padding memory, 256-byte aligned; null when it is smaller and the stream is being captured, or no more is to be had
void* pad_memory(Ctx* ctx, size_t bytes);
// up to two copies in one launch (feedforward.cu)
cudaError_t launch_pad(Ctx* ctx, int dtype, const PadJob* jobs, int count);
// whether the paired kernel saves the fp16 gradient of x more than a copy of w with padded rows costs
bool gated_grad_x_wants_padded_w(const Ctx* ctx, int rows, int xc, int yc);
// whether TMA can describe a stored matrix stack of rows of `ld` elements at ptr
bool rows_aligned(const void* ptr, long long ld, int dtype);

// act(A B[0]) * (A B[1]) for row-major A [M, K] and B [2, K, N] (GemmCfg::GATED); C [M, N]
struct GatedProblem {
    int dtype = 0;
    int M = 0, N = 0, K = 0;
    const void* a = nullptr;
    const void* b = nullptr;
    void* C = nullptr;
    GatedTail tail = {};
};

// Sum of a split paired product's slices, with the gated tail or an (accumulating) store (gemm_inst_gated_pair.cu)
struct SplitSum {
    const float* ws;
    int splits, batch, tiles_m, tiles_n, M, N;
    void* C;
    long long ldc, c_batch_stride;
    int beta;
    GatedTail gated;
};
cudaError_t launch_split_sum(const Ctx* ctx, const SplitSum& q, bool gated);

// the kernel for a few rows (gemm_gated_few.cu)
struct GatedFewParams {
    int rows, width;
    int num_kb, splits, kb_per_split;  // in stages of 64 k, or 128 for up to 32 tokens
    int total_work;                    // strips of 128 columns x splits; split launches have one CTA per item, a cluster per strip
    int x_chunked, w_chunked;
    int* status;
    void* h;
    GatedTail gated;
};
// tokens: 16, 32, 64 or 128, at least the rows
cudaError_t launch_gated_few(int tokens, int grid, cudaStream_t stream, const CUtensorMap& tx, const CUtensorMap& tw, const GatedFewParams& p);

// error reporting shared by the API layer
void set_error(const std::string& msg);
int fail(int code, const std::string& msg);
void count_launch();
void set_last_kernel(const std::string& text);

typedef cudaError_t (*GemmLaunchFn)(int grid, cudaStream_t stream, const CUtensorMap& ta, const CUtensorMap& tb, const GemmParams& p);

// Everything run_gemm works out for one contraction short of launching it
struct PreparedGemm {
    GemmParams p;
    CUtensorMap ta, tb;
    GemmLaunchFn fn = nullptr;
    int grid = 0, tiles = 0, splits = 1, total_kb = 0;
    bool pair = false, dual = false, halo = false, twin = false, f32 = false, a_mn = false, b_mn = false;
    int bn = 0;
    std::string text;  // what d8k_last_kernel reports
};

// capture != nullptr: prepare only (no clearing of tickets, no launch) and hand the result back
int run_gemm(Ctx* ctx, const GemmProblem& g, PreparedGemm* capture = nullptr);
// The gated pair of products as one launch; every extent at least 1, every pointer checked by the caller
int run_gated(Ctx* ctx, const GatedProblem& g);
// The gated block's gradient products: run_gemm, or for fp16 the paired kernel in the form that is the fastest for the problem
int run_gated_grad(Ctx* ctx, const GemmProblem& g);
// The contractions of one operator (the residue classes of a strided convolution): ONE launch whose work items are all of
// theirs when the context has a group buffer and every part runs the same one-CTA-per-SM kernel, otherwise one launch each.
int run_gemm_group(Ctx* ctx, std::vector<GemmProblem>& parts);
// scratch bytes run_gemm would use for this problem with its default split choice (0 when it runs unsplit)
size_t gemm_scratch_need(const Ctx* ctx, const GemmProblem& g);
// true when run_gemm would fetch both operands with the TMA producer (no loader warps)
bool gemm_goes_through_tma(const Ctx* ctx, const GemmProblem& g);

// one table per translation unit of instantiations; index [a_mn][b_mn][bn slot]
GemmLaunchFn lookup_f16_tma(bool a_mn, bool b_mn, int bn);
GemmLaunchFn lookup_f16_twin(bool a_mn, bool b_mn, int bn);  // lookup_f16_tma's tiles with twin issuing threads
GemmLaunchFn lookup_f16_grouped(bool a_mn, bool b_mn, int bn);  // the same for grouped launches
GemmLaunchFn lookup_f16_gather(bool a_mn, bool b_mn, int bn);
GemmLaunchFn lookup_f32_gather(bool a_mn, bool b_mn, int bn);
GemmLaunchFn lookup_f32_tma(bool a_mn, bool b_mn, int bn, bool a_in_tmem);
GemmLaunchFn lookup_f32_dual(bool a_mn, bool b_mn, int mode);  // two CTAs per SM (GemmCfg::DUAL, mode 1 or 2); launch 2 x SMs CTAs
GemmLaunchFn lookup_f32_halo(bool b_mn);  // K-major virtual A through patches, 64 columns
// the gated kernels (GemmCfg::GATED), A K-major and B MN-major; the fp32 mode is lookup_f32_dual's
GemmLaunchFn lookup_f16_gated(int bn);
GemmLaunchFn lookup_f32_gated(int mode);
GemmLaunchFn lookup_gated_gather(bool f32);  // loader warps: 128 columns fp16, 64 fp32
GemmLaunchFn lookup_f16_gated_pair();
// the same and the plain paired kernel on slices of the contraction (Gemm2Cfg::SPLIT), and the latter with eight storing warps (STORE8); both
// operands K-major, or both MN-major
GemmLaunchFn lookup_f16_gated_pair_split();
GemmLaunchFn lookup_f16_pair_split(bool mn);
GemmLaunchFn lookup_f16_pair_store(bool mn);
GemmLaunchFn lookup_f32_precise(bool mn, int mode);  // mode 1, 2 or 4 as in lookup_f32_dual, 0 the loader warps
// paired-CTA kernel: the first argument of the launch function is the number of CTA pairs
GemmLaunchFn lookup_f16_pair(bool a_mn, bool b_mn);

template <class Cfg>
cudaError_t launch_cfg(int grid, cudaStream_t stream, const CUtensorMap& ta, const CUtensorMap& tb, const GemmParams& p) {
    static bool configured[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(d8k_gemm_kernel<Cfg>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    d8k_gemm_kernel<Cfg><<<grid, Cfg::THREADS, Cfg::SMEM_BYTES, stream>>>(ta, tb, p);
    return cudaGetLastError();
}

}  // namespace d8k
