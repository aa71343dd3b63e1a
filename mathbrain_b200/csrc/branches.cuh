// Branches of a decode state: what the kernels of branches.cu, branch_attend.cu, branch_attend_tc.cu and branch_rows_tc.cu share.
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

// fp32 arithmetic: how the slot lists are cut into chunks.  A chunk of a sequence's prefix for all its branches, or one of a
// branch's own slots, leaves one partial (m, l, o[64]) for each of its rows, heads and steps, which k_branch_merge joins.
struct BranchPlan {
    int chp, cho;      // slots a chunk: prefix, own
    int SP, SO;        // chunks that the lists' capacities allow
    int steps, JP;     // steps a job of a prefix, blocks of steps
};

// Several branches: units of 16 slots.  Cost of one in the running sum that mbema_branches_extend leaves: of a branch's own slots, of a
// prefix for sixteen branches; a worker's least.
static constexpr int BR_COST_OWN = 2, BR_COST_BLOCK = 3, BR_LEAST_COST = 2 * BR_COST_BLOCK;
struct BranchShape {
    int blocks;            // of sixteen branches, a sequence
    int JW, IG;            // of a CTA: steps a worker, workers
    int zb, ctas;          // blocks of steps; CTAs a head and block of steps
};

// One branch: tiles of 128 slots.
static constexpr int BR_TILE = 128;
struct BranchRows {
    int JW, IG;            // steps a worker, workers a CTA
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
    // Tensor cores: a list's piece in worker w is number list + w, as lists and workers come in the same order.
    // Several branches: n_pre lists (sequence, block of sixteen), then the branches' own; partials [piece, BR_BLOCK, n, H] and
    // [own_piece0 + piece, n, H].  One branch: prefix and own list of every sequence in turn (a stretch then holds long and short ones as
    // the others do: a list's start and end cost as much as half a tile); partials [piece, 4 warps, n, H].
    int lists, n_pre, blocks, max_workers, ring_bytes, w_offset;
    int64_t own_piece0;
    __device__ __forceinline__ bool row_is_prefix(int list) const { return !(list & 1); }
    __device__ __forceinline__ int row_branch(int list) const { return list >> 1; }
    __device__ __forceinline__ const int* row_slots(int list) const {
        return list & 1 ? br.own_slot + (size_t)(list >> 1) * br.cap : br.active + (size_t)(list >> 1) * br.Kcap;
    }
    __device__ __forceinline__ const char* row_operands(int list) const;
};

// The workers that a running sum of `total` units (tiles) occupies, and where their stretches begin.
__device__ __forceinline__ int branch_workers(int total, int most, int least) { return max(1, min(most, total / least)); }
// total * w / workers in 32 bits (workers below 2^15)
__device__ __forceinline__ int branch_cut(int total, int workers, int w) {
    const int q = total / workers, r = total - q * workers;
    return q * w + r * w / workers;
}
// the worker whose stretch holds unit c < total
__device__ __forceinline__ int branch_worker_of(int total, int workers, int c) {
    if ((unsigned)total <= 0xffffffffu / (unsigned)workers) return (int)(((unsigned)(c + 1) * (unsigned)workers - 1u) / (unsigned)total);
    return (int)((((long long)c + 1) * workers - 1) / total);
}
// Where a stretch begins: the list that holds unit c, with its (running sum, length) and the next one's, by 32 samples of the running
// sum at a time.  The first samples depend on nothing but the number of lists: they are read with the total that c comes from.
struct ListSearch {
    int2 base, mine;                              // entries lo and min(lo + (lane + 1) step, hi)
    __device__ __forceinline__ void begin(const int2* work, int lists, int lane) {
        base = work[0];
        mine = work[min((lane + 1) * ((lists + 31) / 32), lists)];
    }
    __device__ __forceinline__ int find(const int2* work, int lists, int c, int lane, int2& at, int2& next) const {
        int2 first = base, s = mine;
        int lo = 0, hi = lists, step = (lists + 31) / 32;
        for (;;) {
            const unsigned below = __ballot_sync(0xffffffffu, lo + (lane + 1) * step < hi && s.x <= c);
            const int k = __popc(below);
            lo += k * step;
            if (step == 1) {
                const int before = max(k - 1, 0);
                const int2 p = make_int2(__shfl_sync(0xffffffffu, s.x, before), __shfl_sync(0xffffffffu, s.y, before));
                at = k ? p : first;
                next = make_int2(__shfl_sync(0xffffffffu, s.x, k), __shfl_sync(0xffffffffu, s.y, k));
                return lo;
            }
            hi = min(hi, lo + step);
            step = (hi - lo + 31) / 32;
            first = work[lo];
            s = work[min(lo + (lane + 1) * step, hi)];
        }
    }
};

// Operands of a list, state / 64 in fp16, tile after tile of 128 slots (the last one's other slots zero); N * 256 bytes each.
// One branch: what tcgen05 reads from shared memory, N / 64 blocks of 128 rows of 64 channels, 128 bytes a row, the 16-byte
// pieces of row k in order piece ^ (k % 8).
// Several branches: fragments of mma.sync, 16 slots after 16 slots.  Slot k, channel c = 32 i + 8 t + 4 u + 2 p + e is half e
// of word (row / 8) + 2 p (row = k % 16) of lane 4 (row % 8) + t in fragment 2 i + u of its sixteen (512 bytes each).
__host__ __device__ inline size_t br_operand_bytes(int64_t slots, int64_t N) { return (size_t)((slots + BR_TILE - 1) / BR_TILE) * N * (2 * BR_TILE); }
__device__ __forceinline__ const char* BranchArgs::row_operands(int list) const {
    return list & 1 ? reinterpret_cast<const char*>(br.own_op) + (size_t)(list >> 1) * br_operand_bytes(br.cap, br.N)
                    : reinterpret_cast<const char*>(br.pre_op) + (size_t)(list >> 1) * br_operand_bytes(br.Kcap, br.N);
}

// log2(rho) as a factor of a step count: rho = 0 (a half-life too short for fp32) keeps 0 * log2(rho) = 0
__device__ __forceinline__ float br_log2(float rho) { return fmaxf(log2f(rho), -1e30f); }

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

// A kernel whose CTAs may start while the kernel before it still runs; it waits for that one's end with br_wait_for_kernel_before.  All
// kernels here wait before their first access and only then let the next one start (but for the merge, which begins with ld_gpu); so a
// kernel's end means the end of all before it.  A launch costs about 2 us less.
template <typename... Params, typename... Args>
inline cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
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

// Loads of a kernel that has not waited yet, of what the kernels before the one directly before it wrote.  It starts only after every CTA of
// that one has waited, so those have ended and their writes are in L2; but it is the own wait that makes them visible to ordinary loads,
// which might be served from a line that L1 holds from before.  Loads at the scope of the GPU are not.  (volatile: an asm without it may
// run ahead of the condition that guards its address.)
__device__ __forceinline__ int ld_gpu(const int* p) {
    int x;
    asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(x) : "l"(p));
    return x;
}
__device__ __forceinline__ float ld_gpu(const float* p) {
    float x;
    asm volatile("ld.relaxed.gpu.global.f32 %0, [%1];" : "=f"(x) : "l"(p));
    return x;
}
__device__ __forceinline__ float2 ld_gpu(const float2* p) {
    float2 x;
    asm volatile("ld.relaxed.gpu.global.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "l"(p));
    return x;
}
__device__ __forceinline__ float2 ld_gpu_pair(const void* p, int dt, size_t i) {       // elements i, i + 1 (i even) of fp32 or bf16
    if (dt == MBEMA_F32) return ld_gpu(reinterpret_cast<const float2*>(reinterpret_cast<const float*>(p) + i));
    const uint32_t x = (uint32_t)ld_gpu(reinterpret_cast<const int*>(reinterpret_cast<const __nv_bfloat16*>(p) + i));
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}

// Two fp32 values as one operand: one instruction for two FMA, at the same rate (it is issue slots that run short).
__device__ __forceinline__ uint64_t pair2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair2(float& a, float& b, uint64_t r) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

int check_branches(const mbema_branches* br);         // sizes, pointers and alignment: what every entry point refuses
bool branch_tc_supported(int64_t N);
BranchShape branch_shape(int64_t S, int64_t n, int64_t H);
BranchRows branch_rows(int64_t n, int64_t H);
int launch_branch_rows(const BranchArgs& a, const BranchRows& p, cudaStream_t st);
int launch_branch_attend_fp32(const BranchArgs& a, cudaStream_t st);
int launch_branch_attend_tc(BranchArgs& a, const BranchShape& p, cudaStream_t st);
int launch_branch_merge(const BranchArgs& a, bool pieces, cudaStream_t st);

}  // namespace mbema
