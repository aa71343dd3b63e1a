// Branches of a decode state: what the kernels of branches.cu, branch_attend.cu and branch_attend_tc.cu share.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace mbema {

static constexpr int BR_HD = 64;
static constexpr int BR_MAX_NEW = 32;              // staged tokens a branch: one per lane of a warp
static constexpr float BR_OP_SCALE = 1.0f / 64.0f;  // operand copies hold state / 64 in fp16: up to 4.19 million, saturated
static constexpr float BR_SCORE_LOG2 = 0.125f * 1.4426950408889634f;   // 1 / sqrt(64), in powers of two

// How the slot lists are cut into jobs.  A job is one chunk of a sequence's prefix for all its branches, or one chunk of a
// branch's own slots; it leaves one partial (m, l, o[64]) for each of its rows, heads and steps, which k_branch_merge joins.
struct BranchPlan {
    int chp, cho;      // slots a chunk: prefix, own
    int SP, SO;        // chunks that the lists' capacities allow
};

struct BranchArgs {
    mbema_branches br;
    const void* q;
    const void* Ek;
    const void* Ev;
    const float* W;
    void* O;
    float2* ml;              // [rows, H, SP + SO]: maximum (of base-2 scores), sum
    float* po;               // [rows, H, SP + SO, 64]
    int q_dt, e_dt;
    int n, H;
    float v_total;
    int silu, listed_only;
    BranchPlan plan;
};

__host__ __device__ inline size_t br_index(const mbema_branches& br, int64_t r, int i) { return (size_t)r * br.max_new + i; }

// Row j of branch r cannot see slot k of the prefix: the branch has touched it, or does so with a staged token before j.
__device__ __forceinline__ bool br_hides_prefix(const mbema_branches& br, int64_t r, int j, int k) {
    const int words = (int)((br.Kcap + 31) / 32);
    if ((br.touched[(size_t)r * words + (k >> 5)] >> (k & 31)) & 1u) return true;
    for (int i = 0; i < j; ++i)
        if (br.st_pos[br_index(br, r, i)] == k) return true;
    return false;
}
__device__ __forceinline__ bool br_hides_own(const mbema_branches& br, int64_t r, int j, int u) {
    for (int i = 0; i < j; ++i)
        if (br.st_own[br_index(br, r, i)] == u) return true;
    return false;
}

bool branch_tc_supported(int64_t N);
BranchPlan branch_plan_tc(int64_t B, int64_t S, int64_t n, int64_t H, int64_t Kcap, int64_t cap);
int launch_branch_attend_tc(const BranchArgs& a, cudaStream_t st);
int launch_branch_attend_fp32(const BranchArgs& a, cudaStream_t st);
int launch_branch_merge(const BranchArgs& a, cudaStream_t st);

}  // namespace mbema
