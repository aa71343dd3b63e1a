// Branches of a decode state: what the kernels of branches.cu, branch_attend.cu and branch_attend_tc.cu share.
#pragma once
#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"

namespace mbema {

static constexpr int BR_HD = 64;
static constexpr int BR_MAX_NEW = 32;              // staged tokens a branch: one per lane of a warp
static constexpr float BR_OP_SCALE = 1.0f / 64.0f;  // operand copies hold state / 64 in fp16: up to 4.19 million, saturated
static constexpr float BR_SCORE_LOG2 = 0.125f * 1.4426950408889634f;   // 1 / sqrt(64), in powers of two

static constexpr int BR_BLOCK = 16;                // branches that read a prefix together on the tensor cores
// Cost of a unit (16 slots) of a list, in the running sum that mbema_branches_extend leaves: own slots, a prefix read by one branch,
// a prefix read by sixteen.
static constexpr int BR_COST_OWN = 2, BR_COST_ONE = 2, BR_COST_BLOCK = 3;

// fp32 arithmetic: how the slot lists are cut into chunks.  A chunk of a sequence's prefix for all its branches, or one of a
// branch's own slots, leaves one partial (m, l, o[64]) for each of its rows, heads and steps, which k_branch_merge joins.
struct BranchPlan {
    int chp, cho;      // slots a chunk: prefix, own
    int SP, SO;        // chunks that the lists' capacities allow
    int steps, JP;     // steps a job of a prefix, blocks of steps
};

// Tensor cores: workers, and the lists in the running sum: prefixes (as blocks of branches read them), then the branches' own.
struct BranchShape {
    int rows, blocks;      // branches that read a prefix together; such blocks a sequence
    int warps, JW, IG;     // of a CTA: warps, steps a worker, workers
    int zb, ctas;          // blocks of steps; CTAs a head and block of steps
};

struct BranchArgs {
    mbema_branches br;
    const void* q;
    const void* Ek;
    const void* Ev;
    const float* W;
    void* O;
    float2* ml;              // maximum (of base-2 scores) and sum of every partial
    float* po;               // [.., 64] its o
    int q_dt, e_dt;
    int n, H;
    float v_total;
    int silu, listed_only;
    // fp32 arithmetic: partials [rows, H, SP + SO]
    BranchPlan plan;
    // tensor cores: a list's piece in worker w is number list + w, as lists and workers come in the same order; partials of the prefixes
    // [piece, BR_BLOCK or 1, n, H], of the own lists [own_piece0 + piece, n, H]
    int64_t n_pre, own_piece0, max_workers;
    int rows, blocks, cost_pre, ring_bytes, w_offset;
};

// The workers that a running sum of `total` occupies, each with two units or more, and where their stretches begin.
__device__ __forceinline__ int branch_workers(int total, int most) { return max(1, min(most, total / (2 * BR_COST_BLOCK))); }
__device__ __forceinline__ int branch_cut(int total, int workers, int w) { return (int)((long long)total * w / workers); }
// the worker whose stretch holds cost c < total
__device__ __forceinline__ int branch_worker_of(int total, int workers, int c) {
    return (int)((((long long)c + 1) * workers - 1) / total);
}

// Operands of a list: fp16 fragments of the gate product, 16 slots after 16 slots.  Slot k, channel c = 32 i + 8 t + 4 u + 2 p + e is half e
// of word (row / 8) + 2 p (row = k % 16) of lane 4 (row % 8) + t in fragment 2 i + u of its sixteen (512 bytes each).
__host__ __device__ inline size_t br_operand_bytes(int64_t slots, int64_t N) { return (size_t)((slots + 15) / 16) * N * 32; }

__host__ __device__ inline size_t br_index(const mbema_branches& br, int64_t r, int i) { return (size_t)r * br.max_new + i; }

// cudaFuncAttributeMaxDynamicSharedMemorySize raised to what every later call needs, once a device (the call costs the host as much
// as a launch)
template <typename Kernel>
inline cudaError_t allow_smem(Kernel kernel, size_t most, std::atomic<unsigned long long>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (e != cudaSuccess || (done.load(std::memory_order_relaxed) & bit)) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// A kernel whose CTAs may start while the kernel before it still runs (it waits for it with br_wait_for_kernel_before).
template <typename... Params, typename... Args>
inline cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, int threads, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}
__device__ __forceinline__ void br_wait_for_kernel_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void br_let_next_kernel_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

bool branch_tc_supported(int64_t N);
BranchShape branch_shape(int64_t B, int64_t S, int64_t N, int64_t n, int64_t H);
int launch_branch_attend_fp32(const BranchArgs& a, cudaStream_t st);
int launch_branch_attend_tc(BranchArgs& a, const BranchShape& p, cudaStream_t st);
int launch_branch_merge(const BranchArgs& a, bool pieces, cudaStream_t st);

}  // namespace mbema
