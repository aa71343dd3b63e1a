// Verification of drafted tokens against the target's probabilities (mbema_verify_drafts).
//
// Draft j, drawn from q_j, stands with probability min(1, p_j(x) / q_j(x)): u q < p.  Behind the drafts that stand one token is
// drawn by inversion, from max(p - q, 0) where a draft was rejected, else from p; the whole then has the target's distribution.
// Products of two fp32 values, differences and sums are taken in double, so that the token does not depend on how the sum over
// the vocabulary is split (a border between tokens lies within the rounding of an fp32 sum of 50 000 terms once in a hundred draws).
// Bound by the bytes of one row of p (and of q) per sequence, behind a chain of three dependent loads that finds the row.  A
// cluster of eight CTAs takes a sequence, so that one sequence alone is not bound by what one SM can load: a warp sums its
// stretch of the vocabulary, the stretches' sums are exchanged through distributed shared memory, and the warp whose stretch
// holds the threshold walks it again.
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace mbema {

static constexpr int VD_CTAS = 8;         // a cluster: the portable size
static constexpr int VD_THREADS = 512;
static constexpr int VD_WARPS = VD_THREADS / 32;
static constexpr int VD_LANE = VD_CTAS * VD_WARPS / 32;   // stretches a lane holds

struct VerifyArgs {
    const void* p; const void* q;
    int64_t p_row, p_pos, q_row, q_pos;
    const long long* drafted; const float* u;
    long long* n_accepted; long long* tokens;
    int G, V;
};

// weight of token i: one that is negative or not finite is none
template <int DT>
__device__ __forceinline__ double vd_weight(const void* p, const void* q, size_t po, size_t qo, int i, int onehot, bool minus_q) {
    double w = (double)ld_as_f32<DT>(p, po + i);
    if (minus_q) w -= q ? (double)ld_as_f32<DT>(q, qo + i) : (i == onehot ? 1.0 : 0.0);
    return w > 0.0 && w <= 3.4028234663852886e38 ? w : 0.0;
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <int DT>
__global__ void __cluster_dims__(VD_CTAS, 1, 1) __launch_bounds__(VD_THREADS) k_verify(VerifyArgs a) {
    __shared__ double s_sum[VD_CTAS * VD_WARPS];         // sums of all stretches of the row, in vocabulary order
    __shared__ int s_acc[2];
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank();
    const int64_t r = blockIdx.x / VD_CTAS;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.G, V = a.V;
    if (warp == 0) {                                     // every CTA of the cluster finds the row by itself
        int stop = G, rejected = 0;
        for (int j0 = 0; j0 < G && stop == G; j0 += 32) {
            const int j = j0 + lane;
            const long long x = j < G ? a.drafted[r * G + j] : 0;
            bool end = j < G && (x < 0 || x >= V), stands = true;
            if (j < G && !end) {
                const double pv = (double)ld_as_f32<DT>(a.p, (size_t)(r * a.p_row + j * a.p_pos + x));
                const double qv = a.q ? (double)ld_as_f32<DT>(a.q, (size_t)(r * a.q_row + j * a.q_pos + x)) : 1.0;
                stands = (double)a.u[r * (G + 1) + j] * qv < pv;
            }
            const unsigned bad = __ballot_sync(0xffffffffu, j < G && (end || !stands));
            const unsigned ends = __ballot_sync(0xffffffffu, end);
            if (bad) {
                stop = j0 + __ffs(bad) - 1;
                rejected = !((ends >> (__ffs(bad) - 1)) & 1u);
            }
        }
        if (lane == 0) { s_acc[0] = stop; s_acc[1] = rejected; }
    }
    __syncthreads();
    const int acc = s_acc[0];
    const bool rejected = s_acc[1] != 0;
    const size_t po = (size_t)(r * a.p_row + acc * a.p_pos);
    const size_t qo = rejected ? (size_t)(r * a.q_row + acc * a.q_pos) : 0;
    const int onehot = rejected ? (int)a.drafted[r * G + acc] : -1;
    const int stretch = (V + VD_CTAS * VD_WARPS - 1) / (VD_CTAS * VD_WARPS);
    const int w_id = rank * VD_WARPS + warp;
    const int lo = min(w_id * stretch, V), hi = min(lo + stretch, V);
    bool minus_q = rejected;
    double total = 0.0;
    for (int pass = 0; pass < 2; ++pass) {
        double sum = 0.0;
#pragma unroll 8
        for (int i = lo + lane; i < hi; i += 32) sum += vd_weight<DT>(a.p, a.q, po, qo, i, onehot, minus_q);
        sum = warp_sum_d(sum);
        if (lane < VD_CTAS) cluster.map_shared_rank(s_sum, lane)[w_id] = sum;
        cluster.sync();
        total = 0.0;                                     // a lane holds four stretches; the same sums in every thread
#pragma unroll
        for (int i = 0; i < VD_LANE; ++i) total += s_sum[lane * VD_LANE + i];
        total = warp_sum_d(total);
        if (total > 0.0 || !minus_q) break;              // the same in every CTA of the cluster
        minus_q = false;                                 // p <= q everywhere: draw from p
        cluster.sync();                                  // every CTA has read the sums
    }
    // the first stretch whose running sum passes the threshold; without one (a number of 1 or more) the last that holds a token
    const double thr = (double)a.u[r * (G + 1) + G] * total;
    double before = 0.0;
    int mine;
    {
        double own[VD_LANE], lane_sum = 0.0;
#pragma unroll
        for (int i = 0; i < VD_LANE; ++i) lane_sum += own[i] = s_sum[lane * VD_LANE + i];
        double run = lane_sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += y;
        }
        run -= lane_sum;
        int hit = -1, some = -1;
        double hit_before = 0.0, some_before = 0.0;
#pragma unroll
        for (int i = 0; i < VD_LANE; ++i) {
            if (own[i] > 0.0) {
                if (hit < 0 && run + own[i] > thr) { hit = lane * VD_LANE + i; hit_before = run; }
                some = lane * VD_LANE + i;
                some_before = run;
            }
            run += own[i];
        }
        const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), somes = __ballot_sync(0xffffffffu, some >= 0);
        const int from = hits ? __ffs(hits) - 1 : 31 - __clz(somes | 1u);
        mine = __shfl_sync(0xffffffffu, hits ? hit : some, from);
        before = __shfl_sync(0xffffffffu, hits ? hit_before : some_before, from);
    }
    if (rank == 0) {
        for (int j = tid; j <= G; j += VD_THREADS)
            if (j != acc) a.tokens[r * (G + 1) + j] = j < acc ? a.drafted[r * G + j] : -1;
        if (tid == 0) {
            a.n_accepted[r] = acc;
            if (mine < 0) a.tokens[r * (G + 1) + acc] = -1;
        }
    }
    if (w_id != mine) return;
    int found = -1, tail = -1;
    for (int i0 = lo; i0 < hi && found < 0; i0 += 32) {
        const int i = i0 + lane;
        const double w = i < hi ? vd_weight<DT>(a.p, a.q, po, qo, i, onehot, minus_q) : 0.0;
        double x = w;                                    // inclusive sum over the lanes
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        const unsigned pass = __ballot_sync(0xffffffffu, w > 0.0 && before + x > thr);
        const unsigned some = __ballot_sync(0xffffffffu, w > 0.0);
        if (some) tail = i0 + 31 - __clz(some);
        if (pass) found = i0 + __ffs(pass) - 1;
        before += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) a.tokens[r * (G + 1) + acc] = found >= 0 ? found : tail;
}

}  // namespace mbema

using namespace mbema;

extern "C" int mbema_verify_drafts(const void* p, int64_t p_row, int64_t p_pos, const void* q, int64_t q_row, int64_t q_pos, int dtype,
                                   const int64_t* drafted, const float* uniforms, int64_t* n_accepted, int64_t* tokens, int64_t R,
                                   int64_t G, int64_t V, void* stream) {
    if (R < 0 || G < 0 || V < 1) return MBEMA_ERR_SHAPE;
    if (V > 0x3fffffff || G > 4096 || R > 0x7fffffff / VD_CTAS) return MBEMA_ERR_UNSUPPORTED;
    if (dtype != MBEMA_F32 && dtype != MBEMA_BF16) return MBEMA_ERR_DTYPE;
    if (R == 0) return MBEMA_OK;
    if (!p || (G > 0 && !drafted) || !uniforms || !n_accepted || !tokens) return MBEMA_ERR_NULL;
    VerifyArgs a{p, q, p_row, p_pos, q_row, q_pos, (const long long*)drafted, uniforms, (long long*)n_accepted, (long long*)tokens, (int)G, (int)V};
    const unsigned grid = (unsigned)(R * VD_CTAS);
    if (dtype == MBEMA_F32) k_verify<MBEMA_F32><<<grid, VD_THREADS, 0, (cudaStream_t)stream>>>(a);
    else k_verify<MBEMA_BF16><<<grid, VD_THREADS, 0, (cudaStream_t)stream>>>(a);
    return check_launch();
}
