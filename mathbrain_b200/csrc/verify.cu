// Verification of drafted tokens against the target's probabilities (mbema_verify_drafts).
//
// Draft j, drawn from q_j, stands with probability min(1, p_j(x) / q_j(x)): u q < p.  Behind the drafts that stand one token is
// drawn by inversion, from max(p - q, 0) where a draft was rejected, else from p; the whole then has the target's distribution.
// Products of two fp32 values, differences and sums are taken in (or with the exactness of) double, so that the token does not depend on
// how the sum over the vocabulary is split: a lane's sum of a few dozen weights is a pair of fp32 (2^-47), again in double where it leaves
// fp32's range, all others are double (a border between tokens lies within the rounding of an fp32 sum of 50 000 terms once in a
// hundred draws).
// Bound by the bytes of one row of p (and of q) per sequence, behind a chain of three dependent loads that finds the row.  A
// cluster of CTAs takes a sequence, so that one sequence alone is not bound by what one SM can load: a warp sums its
// stretch of the vocabulary, the stretches' sums are exchanged through distributed shared memory, and the CTA whose
// stretch holds the threshold deals it to its warps once more, so that a warp walks a 288th to a 1152nd of the vocabulary (175 to 44 of
// 50 257 tokens), 32 at a time.
#include <cooperative_groups.h>

#include <type_traits>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace mbema {

static constexpr int VD_THREADS = 384;
static constexpr int VD_WARPS = VD_THREADS / 32;
static constexpr int VD_BATCH = 8;         // loads of p and of q that a lane has in flight

struct VerifyArgs {
    const void* p; const void* q;
    int64_t p_row, p_pos, q_row, q_pos;
    const long long* drafted; const float* u;
    long long* n_accepted; long long* tokens;
    int G, V;
};

// weight of a token: one that is negative or not finite is none
__device__ __forceinline__ double vd_weight(double w) { return w > 0.0 && w <= 3.4028234663852886e38 ? w : 0.0; }

// s + e += weight of (p - q), as a lane's sum of a few dozen of them: the difference and every sum with its rounding error kept (Knuth's
// two-sum; relative error about 2^-47).  In double, the conversions and the compares of a whole row took longer than its bytes.
__device__ __forceinline__ void add_weight(float& s, float& e, float w) {
    const float d = w > 0.f && w <= 3.402823466e38f ? w : 0.f;
    const float t = __fadd_rn(s, d), c = __fsub_rn(t, s);
    e = __fadd_rn(e, __fadd_rn(__fsub_rn(s, __fsub_rn(t, c)), __fsub_rn(d, c)));
    s = t;
}
__device__ __forceinline__ void add_weight(float& s, float& e, float p, float q) {
    float d = __fsub_rn(p, q);
    const float b = __fsub_rn(d, p);
    float r = __fsub_rn(__fsub_rn(p, __fsub_rn(d, b)), __fadd_rn(q, b));
    const bool ok = d > 0.f && d <= 3.402823466e38f;
    d = ok ? d : 0.f;
    r = ok ? r : 0.f;
    const float t = __fadd_rn(s, d), c = __fsub_rn(t, s);
    e = __fadd_rn(e, __fadd_rn(__fadd_rn(__fsub_rn(s, __fsub_rn(t, c)), __fsub_rn(d, c)), r));
    s = t;
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Of 32 EACH sums, in shared memory: the first at which the running sum (from `before` on) passes the threshold; without one (a number
// of 1 or more, or the rounding of another order of summing) the last that is not empty; -1 if all are.  `before`: the running sum there.
template <int EACH>
__device__ __forceinline__ int pick(const double* sums, double thr, double& before) {
    const int lane = threadIdx.x & 31;
    double own[EACH], lane_sum = 0.0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) lane_sum += own[i] = sums[lane * EACH + i];
    double run = lane_sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += y;
    }
    run += before - lane_sum;
    int hit = -1, some = -1;
    double hit_before = 0.0, some_before = 0.0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        if (own[i] > 0.0) {
            if (hit < 0 && run + own[i] > thr) { hit = lane * EACH + i; hit_before = run; }
            some = lane * EACH + i;
            some_before = run;
        }
        run += own[i];
    }
    const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), somes = __ballot_sync(0xffffffffu, some >= 0);
    const int from = hits ? __ffs(hits) - 1 : 31 - __clz(somes | 1u);
    before = __shfl_sync(0xffffffffu, hits ? hit_before : some_before, from);
    return __shfl_sync(0xffffffffu, hits ? hit : some, from);
}

// CTAS: of a cluster, 2 to 8.  Four CTAs an SM, which the choice of the cluster below counts on: 42 registers a thread (with 44, 109 sequences of
// 7 drafts and 32 000 tokens take two waves, 14 us for 11).
template <int DT, int VD_CTAS>
__global__ void __launch_bounds__(VD_THREADS, 4) k_verify(VerifyArgs a) {
    constexpr int VD_LANE = (VD_CTAS * VD_WARPS + 31) / 32;      // stretches a lane holds
    __shared__ double s_sum[VD_LANE * 32];         // sums of all stretches of the row, in vocabulary order, then zeros
    __shared__ double s_sub[32];
    __shared__ int s_acc[2];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    cg::cluster_group cluster = cg::this_cluster();
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");       // (waited for before the first write to another CTA: it has started)
    const int rank = (int)cluster.block_rank();
    const int64_t r = blockIdx.x / VD_CTAS;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (VD_CTAS * VD_WARPS + tid < VD_LANE * 32) s_sum[VD_CTAS * VD_WARPS + tid] = 0.0;
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
    // what is taken off p: q, or 1 at the draft, or (not rejected; p <= q everywhere) nothing
    bool from_q = rejected && a.q, minus = rejected;
    int spike = rejected && !a.q ? onehot : -1;
    auto weight = [&](int i) {
        const double taken = from_q ? (double)ld_as_f32<DT>(a.q, qo + i) : (i == spike ? 1.0 : 0.0);
        return vd_weight((double)ld_as_f32<DT>(a.p, po + i) - taken);
    };
    double total = 0.0;
    for (int pass = 0; pass < 2; ++pass) {
        float s = 0.f, e = 0.f;
        auto batch = [&](int i0, auto whole) {            // a batch of loads is in flight, the last one (not whole) too
            float x[VD_BATCH], y[VD_BATCH];
            auto in = [&](int k) { return decltype(whole)::value || i0 + 32 * k < hi; };
#pragma unroll
            for (int k = 0; k < VD_BATCH; ++k) x[k] = in(k) ? ld_as_f32<DT>(a.p, po + i0 + 32 * k) : 0.f;
            if (from_q) {
#pragma unroll
                for (int k = 0; k < VD_BATCH; ++k) y[k] = in(k) ? ld_as_f32<DT>(a.q, qo + i0 + 32 * k) : 0.f;
#pragma unroll
                for (int k = 0; k < VD_BATCH; ++k) add_weight(s, e, x[k], y[k]);
            } else {
#pragma unroll
                for (int k = 0; k < VD_BATCH; ++k) add_weight(s, e, i0 + 32 * k == spike ? x[k] - 1.0f : x[k]);
            }
        };
        int i0 = lo + lane;
        for (; i0 + 32 * (VD_BATCH - 1) < hi; i0 += 32 * VD_BATCH) batch(i0, std::true_type());
        if (i0 < hi) batch(i0, std::false_type());
        double sum = warp_sum_d((double)s + (double)e);
        if (!(sum <= 1.7976931348623157e308)) {          // a lane's sum has left fp32's range (the weights themselves are finite): in double
            sum = 0.0;
            for (int i = lo + lane; i < hi; i += 32) sum += weight(i);
            sum = warp_sum_d(sum);
        }
        if (pass == 0) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
        if (lane < VD_CTAS) cluster.map_shared_rank(s_sum, lane)[w_id] = sum;
        cluster.sync();
        total = 0.0;                                     // (VD_LANE stretches a lane; the same sums in every thread)
#pragma unroll
        for (int i = 0; i < VD_LANE; ++i) total += s_sum[lane * VD_LANE + i];
        total = warp_sum_d(total);
        if (total > 0.0 || !minus) break;                // the same in every CTA of the cluster
        minus = from_q = false;                          // p <= q everywhere: draw from p
        spike = -1;
        cluster.sync();                                  // every CTA has read the sums
    }
    const double thr = (double)a.u[r * (G + 1) + G] * total;
    double before = 0.0;
    const int mine = pick<VD_LANE>(s_sum, thr, before);
    if (rank == 0) {
        for (int j = tid; j <= G; j += VD_THREADS)
            if (j != acc) a.tokens[r * (G + 1) + j] = j < acc ? a.drafted[r * G + j] : -1;
        if (tid == 0) {
            a.n_accepted[r] = acc;
            if (mine < 0) a.tokens[r * (G + 1) + acc] = -1;
        }
    }
    if (mine < 0 || mine / VD_WARPS != rank) return;
    // the CTA whose warp summed that stretch deals it to all its warps again; the one whose share passes the threshold walks it
    const int first = min(mine * stretch, V), behind = min(first + stretch, V);
    const int share = (stretch + VD_WARPS - 1) / VD_WARPS;
    const int from = min(first + warp * share, behind), to = min(from + share, behind);
    {
        double sum = 0.0;
        for (int i = from + lane; i < to; i += 32) sum += weight(i);
        sum = warp_sum_d(sum);
        if (lane == 0) s_sub[warp] = sum;
    }
    if (tid < 32 && tid >= VD_WARPS) s_sub[tid] = 0.0;
    __syncthreads();
    if (pick<1>(s_sub, thr, before) != warp) return;
    int found = -1, tail = -1;
    for (int i0 = from; i0 < to && found < 0; i0 += 32) {
        const int i = i0 + lane;
        const double w = i < to ? weight(i) : 0.0;
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

template <int DT, int CTAS>
static int launch(const VerifyArgs& a, int64_t R, void* stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(R * CTAS));
    cfg.blockDim = dim3(VD_THREADS);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];                         // (the launch overlaps the end of the kernel before)
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CTAS;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    MBEMA_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_verify<DT, CTAS>, a));
    return check_launch();
}

}  // namespace mbema

using namespace mbema;

extern "C" int mbema_verify_drafts(const void* p, int64_t p_row, int64_t p_pos, const void* q, int64_t q_row, int64_t q_pos, int dtype,
                                   const int64_t* drafted, const float* uniforms, int64_t* n_accepted, int64_t* tokens, int64_t R,
                                   int64_t G, int64_t V, void* stream) {
    if (R < 0 || G < 0 || V < 1) return MBEMA_ERR_SHAPE;
    if (V > 0x3fffffff || G > 4096 || R > 0x7fffffff / 8) return MBEMA_ERR_UNSUPPORTED;
    if (dtype != MBEMA_F32 && dtype != MBEMA_BF16) return MBEMA_ERR_DTYPE;
    if (R == 0) return MBEMA_OK;
    if (!p || (G > 0 && !drafted) || !uniforms || !n_accepted || !tokens) return MBEMA_ERR_NULL;
    VerifyArgs a{p, q, p_row, p_pos, q_row, q_pos, (const long long*)drafted, uniforms, (long long*)n_accepted, (long long*)tokens, (int)G, (int)V};
    // the largest cluster with which all rows' CTAs are three an SM (four fit), V = 50257, a row and its q rejected now and then: one sequence
    // 8 5.8 us, 4 6.6, 2 9.1; 64: 8 10.5, 4 9.6, 2 12.4; 128: 8 20.3, 4 16.2, 2 16.4; 256: 8 36, 4 27.5, 2 26.4
    int64_t ctas = 8;
    while (ctas > 2 && R * ctas > 3 * 148) ctas >>= 1;
    if (dtype == MBEMA_F32) return ctas == 8 ? launch<MBEMA_F32, 8>(a, R, stream) : ctas == 4 ? launch<MBEMA_F32, 4>(a, R, stream) : launch<MBEMA_F32, 2>(a, R, stream);
    return ctas == 8 ? launch<MBEMA_BF16, 8>(a, R, stream) : ctas == 4 ? launch<MBEMA_BF16, 4>(a, R, stream) : launch<MBEMA_BF16, 2>(a, R, stream);
}
