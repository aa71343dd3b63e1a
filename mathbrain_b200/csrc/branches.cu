// Branches of a decode state: bookkeeping of kept and staged tokens (the attention over them: branch_attend.cu).
//
// A branch touches few of its sequence's slots, so it holds only those: their value right after the last update and the step
// of it, as the resident state does.  A staged token's state is
//     C_i = kept value * rho^(t_i - t_kept) + sum over staged i' < i with the same token of rho^(t_i - t_i'),
// linear in its occurrences, so all staged tokens are independent of one another; powers and sums in double, rounded once (a
// token repeated at every step amplifies a bias of rho by 1/(1 - rho)).
// Bound by latency: chains of a few dependent loads for B S n rows of 4 N bytes (3 us).  The operand copies beside it move 6 N bytes a
// listed slot: 84 MB for 64 x 3400 slots of 64 channels, 17 us (13 at the memory's measured rate).
#include <algorithm>

#include "branches.cuh"

namespace mbema {

static constexpr int BS_THREADS = 128, OPERAND_THREADS = 256;

// pos[b, active[b, k]] = k over a buffer of -1; empty branches
__global__ void k_branch_init(mbema_branches br, int t_host, const int* t_dev) {
    const int b = blockIdx.y;
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < min(br.n_active[b], (int)br.Kcap)) {
        const int v = br.active[(size_t)b * br.Kcap + i];
        if (v >= 0 && v < br.V) br.pos[(size_t)b * br.V + v] = i;
    }
    const int words = (int)((br.Kcap + 31) / 32);
    const size_t all = (size_t)br.S * words;
    for (size_t w = i; w < all; w += (size_t)gridDim.x * blockDim.x) br.touched[(size_t)b * all + w] = 0u;
    for (int s = i; s < br.S; s += gridDim.x * blockDim.x) {
        br.len[b * br.S + s] = 0;
        br.own_n[b * br.S + s] = 0;
        br.own_new[b * br.S + s] = 0;
    }
    if (b == 0 && i == 0) {
        br.t0[0] = t_dev ? *t_dev : t_host;
        br.overflow[0] = 0;
    }
}

// One CTA of T threads per branch r: keeps staged tokens of the call before, then stages the new ones.
template <int T>
__device__ __forceinline__ void stage_branch(const mbema_branches& br, int64_t r, const long long* __restrict__ tok, int n,
                                             const long long* __restrict__ counts, int pending, float* __restrict__ C_q) {
    __shared__ int s_tok[BR_MAX_NEW], s_own[BR_MAX_NEW], s_dst[BR_MAX_NEW];
    __shared__ unsigned s_same[BR_MAX_NEW];
    __shared__ int s_n, s_len;
    const int b = (int)(r / br.S);
    const int tid = threadIdx.x, lane = tid & 31;
    const int N = (int)br.N, cap = (int)br.cap;
    const int t0 = br.t0[0];
    const int words = (int)((br.Kcap + 31) / 32);
    if (tid < 32) {
        int own_n = br.own_n[r], len = br.len[r];
        if (pending > 0) {
            int c = pending;
            if (counts) c = (int)min(max(counts[b], 0ll), (long long)pending);
            const bool in = lane < c;
            const size_t at = br_index(br, r, in ? lane : 0);
            const int v = in ? br.st_tok[at] : -1;
            const int own = in ? br.st_own[at] : -1, pos = in ? br.st_pos[at] : -1;
            const unsigned kept = c >= 32 ? 0xffffffffu : (1u << c) - 1u;
            const unsigned same = in ? br.st_same[at] & kept : 0u;
            const bool some = in && v >= 0;
            const int root = some ? __ffs(same) - 1 : 0;
            const bool first = some && root == lane;
            const bool last = some && (same >> lane) == 1u;              // no kept staged token behind this one repeats it
            const unsigned fresh = __ballot_sync(0xffffffffu, first && own < 0);
            const unsigned news = __ballot_sync(0xffffffffu, first && br.st_new[at] != 0);
            const int dst = own >= 0 ? own : own_n + __popc(fresh & ((1u << root) - 1u));
            s_dst[lane] = last && dst < cap ? dst : -1;
            if (first && own < 0) {
                if (dst < cap) br.own_slot[(size_t)r * cap + dst] = v;
                else atomicOr(br.overflow, 1);
            }
            if (last && dst < cap) br.own_t[(size_t)r * cap + dst] = t0 + len + lane;
            if (first && pos >= 0) atomicOr(&br.touched[(size_t)r * words + (pos >> 5)], 1u << (pos & 31));
            own_n = min(own_n + __popc(fresh), cap);
            len += c;
            if (lane == 0) {
                br.own_n[r] = own_n;
                br.own_new[r] += __popc(news);
                br.len[r] = len;
            }
        } else {
            s_dst[lane] = -1;
        }
        if (lane == 0) { s_n = own_n; s_len = len; }
    }
    __syncthreads();
    for (int i = 0; i < pending; ++i) {
        const int dst = s_dst[i];
        if (dst < 0) continue;
        for (int c = tid; c < N; c += T)
            br.own_state[((size_t)r * cap + dst) * N + c] = br.st_state[br_index(br, r, i) * N + c] + 1.0f;
    }
    if (n <= 0) return;
    __syncthreads();              // the kept values are in place (this CTA alone reads them below)
    int pos = -1;
    if (tid < 32) {
        const long long v = lane < n ? tok[r * n + lane] : -1;
        const bool some = lane < n && v >= 0 && v < br.V;
        if (lane < n && !some && v != -1) atomicOr(br.overflow, 2);
        const unsigned same = __match_any_sync(0xffffffffu, some ? (int)v : -2 - lane);
        s_tok[lane] = some ? (int)v : -1;
        s_same[lane] = same;
        s_own[lane] = -1;
        if (some) pos = br.pos[(size_t)b * br.V + v];
    }
    __syncthreads();
    const int own_n = s_n, base_t = t0 + s_len;
    for (int u = tid; u < own_n; u += T) {
        const int slot = br.own_slot[(size_t)r * cap + u];
        for (int i = 0; i < n; ++i)
            if (s_tok[i] == slot) s_own[i] = u;
    }
    __syncthreads();
    if (tid < n) {
        const bool first = s_tok[lane] >= 0 && __ffs(s_same[lane]) - 1 == lane;
        const int own = s_own[lane];
        const size_t at = br_index(br, r, lane);
        br.st_tok[at] = s_tok[lane];
        br.st_own[at] = own;
        br.st_same[at] = s_same[lane];
        br.st_pos[at] = first && own < 0 ? pos : -1;
        br.st_new[at] = first && own < 0 && pos < 0;
    }
    for (int e = tid; e < n * N; e += T) {
        const int i = e / N, c = e - i * N;
        const int v = s_tok[i], own = s_own[i];
        double x = 0.0;
        if (v >= 0) {
            const double l2 = fmax(log2((double)br.rhos[c]), -1e30);
            const int last = own >= 0 ? br.own_t[(size_t)r * cap + own] : br.last_t[(size_t)b * br.V + v];
            if (own >= 0 || last >= 0) {
                const float base = own >= 0 ? br.own_state[((size_t)r * cap + own) * N + c] : br.state[((size_t)b * br.V + v) * N + c];
                x = (double)base * exp2((double)(base_t + i - last) * l2);
            }
            for (unsigned m = s_same[i] & ((1u << i) - 1u); m; m &= m - 1u) x += exp2((double)(i - (__ffs(m) - 1)) * l2);
        }
        br.st_state[br_index(br, r, i) * N + c] = (float)x;
        C_q[((size_t)r * n + i) * N + c] = (float)x;
    }
}
__global__ void __launch_bounds__(BS_THREADS) k_branch_stage(mbema_branches br, const long long* __restrict__ tok, int n,
                                                             const long long* __restrict__ counts, int pending, float* __restrict__ C_q) {
    br_wait_for_kernel_before();
    br_let_next_kernel_start();
    stage_branch<BS_THREADS>(br, blockIdx.x, tok, n, counts, pending, C_q);
}

// Operand copies of all listed slots at the first staged step, state * rho^(t0 + len - last) / 64 in fp16 (11 significant bits; a
// state is at most 1 / (1 - rho)): what the tensor cores read for every layer, step and head, in the layouts that branches.cuh gives.
// CTA 0 leaves the running sum of the lists' units that the attention deals its work by; of the others `shares` take a list: of the
// sequences' prefixes, then of their branches 0, of their branches 1 and so on.
template <typename Count>
__device__ void running_sum(int2* out, int lists, Count count_of) {
    __shared__ int s_warp[OPERAND_THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31;
    int base = 0;
    for (int x0 = 0; x0 < lists; x0 += 256) {
        const int x = x0 + tid;
        int c = 0;
        const int count = x < lists ? count_of(x, c) : 0;
        int sum = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += y;
        }
        if (lane == 31) s_warp[tid >> 5] = sum;
        __syncthreads();
        int all = 0;
        for (int w = 0; w < 8; ++w) {
            if (w < (tid >> 5)) sum += s_warp[w];
            all += s_warp[w];
        }
        if (x < lists) out[x] = make_int2(base + sum - c, count);
        base += all;
        __syncthreads();
    }
    if (tid == 0) out[lists] = make_int2(base, 0);
}

// the largest fp16 at most; NaN stays (fminf would return the other operand: a state that is lost would count as one of 4.19 million)
__device__ __forceinline__ float half_range(float x) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(65504.f));
    return r;
}
__device__ __forceinline__ void decayed(float (&f)[8], const float* src, float dt, const float (&l2r)[8]) {
    const float4 x = *reinterpret_cast<const float4*>(src), y = *reinterpret_cast<const float4*>(src + 4);
    const float in[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = half_range(in[e] * exp2f(dt * l2r[e]) * BR_OP_SCALE);
}
__device__ __forceinline__ uint32_t half_pair(float lo, float hi) {
    const __half2 o = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&o);
}

__device__ __forceinline__ void make_operands(const mbema_branches& br, int64_t cta, int shares) {
    if (cta == 0) {
        int2* work = reinterpret_cast<int2*>(br.work);
        const int blocks = (int)((br.S + BR_BLOCK - 1) / BR_BLOCK), n_pre = (int)br.B * blocks;
        auto prefix = [&](int b) { return min(br.n_active[b], (int)br.Kcap); };
        if (br.S == 1)
            running_sum(work, (int)(2 * br.B), [&](int x, int& cost) {
                const int count = x & 1 ? br.own_n[x >> 1] : prefix(x >> 1);
                cost = (count + BR_TILE - 1) / BR_TILE;
                return count;
            });
        else
            running_sum(work, n_pre + (int)(br.B * br.S), [&](int x, int& cost) {
                const int count = x < n_pre ? prefix(x / blocks) : br.own_n[x - n_pre];
                cost = (count + 15) / 16 * (x < n_pre ? BR_COST_BLOCK : BR_COST_OWN);
                return count;
            });
        return;
    }
    const int64_t list = (cta - 1) / shares;
    const int share = (int)(cta - 1 - list * shares), z = (int)(list / br.B), b = (int)(list - z * br.B);
    const int N = (int)br.N;
    const int64_t r = (int64_t)b * br.S + (z ? z - 1 : 0);
    const int count = z ? br.own_n[r] : min(br.n_active[b], (int)br.Kcap);
    const int now = br.t0[0] + br.len[r];
    const int lane = threadIdx.x & 31, warp = share * 8 + (threadIdx.x >> 5), warps = shares * 8;
    char* out = z ? reinterpret_cast<char*>(br.own_op) + (size_t)r * br_operand_bytes(br.cap, N)
                  : reinterpret_cast<char*>(br.pre_op) + (size_t)b * br_operand_bytes(br.Kcap, N);
    auto source = [&](int slot, float& dt) {
        if (z) {
            dt = (float)(now - br.own_t[(size_t)r * br.cap + slot]);
            return (const float*)br.own_state + ((size_t)r * br.cap + slot) * N;
        }
        const int v = br.active[(size_t)b * br.Kcap + slot];
        dt = (float)(now - br.last_t[(size_t)b * br.V + v]);
        return (const float*)br.state + ((size_t)b * br.V + v) * N;
    };
    float l2r[8];
    if (br.S == 1) {                                    // rows of 64 channels: eight lanes a row, four rows a warp
        const int atoms = N / 64, atom = warp % atoms, c = 64 * atom + 8 * (lane & 7);
        const int past = (count + BR_TILE - 1) / BR_TILE * BR_TILE;
        int k = warp / atoms * 4 + (lane >> 3);
        if (k - (lane >> 3) >= past) return;
#pragma unroll
        for (int e = 0; e < 8; ++e) l2r[e] = br_log2(br.rhos[c + e]);
        for (; k - (lane >> 3) < past; k += warps / atoms * 4) {
            float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, dt;
            if (k < count) {
                const float* src = source(k, dt);
                decayed(f, src + c, dt, l2r);
            }
            const int row = k % BR_TILE;
            *reinterpret_cast<uint4*>(out + ((size_t)(k / BR_TILE) * atoms + atom) * 16384 + row * 128 + (((lane & 7) ^ (row & 7)) << 4)) =
                make_uint4(half_pair(f[0], f[1]), half_pair(f[2], f[3]), half_pair(f[4], f[5]), half_pair(f[6], f[7]));
        }
        return;
    }
    // fragments: a warp makes a pair of them, for sixteen slots
    const int half = N / 32, i = warp % half, c = 32 * i + 8 * (lane & 3);
    int k = warp / half * 16 + (lane >> 2);
    if (k - (lane >> 2) >= count) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) l2r[e] = br_log2(br.rhos[c + e]);
    for (; k - (lane >> 2) < count; k += warps / half * 16) {
        uint32_t w[2][4];                               // slots k, k + 8
#pragma unroll
        for (int hi = 0; hi < 2; ++hi) {
            float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, dt;
            if (k + 8 * hi < count) {
                const float* src = source(k + 8 * hi, dt);
                decayed(f, src + c, dt, l2r);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) w[hi][e] = half_pair(f[2 * e], f[2 * e + 1]);
        }
        char* dst = out + (size_t)(k >> 4) * N * 32 + (2 * i) * 512 + lane * 16;
        *reinterpret_cast<uint4*>(dst) = make_uint4(w[0][0], w[1][0], w[0][1], w[1][1]);
        *reinterpret_cast<uint4*>(dst + 512) = make_uint4(w[0][2], w[1][2], w[0][3], w[1][3]);
    }
}

// BESIDE: without tokens to keep, staging leaves lists and lengths alone and writes nothing that is read here; one kernel then does both,
// its first CTAs a branch each.  Otherwise the staging kernel comes before.
template <bool BESIDE>
__global__ void __launch_bounds__(OPERAND_THREADS) k_branch_operands(mbema_branches br, int shares, const long long* __restrict__ tok, int n, float* __restrict__ C_q) {
    br_wait_for_kernel_before();
    const int64_t first = BESIDE ? br.B * br.S : 0;
    if (blockIdx.x < first) stage_branch<OPERAND_THREADS>(br, blockIdx.x, tok, n, nullptr, 0, C_q);
    else make_operands(br, blockIdx.x - first, shares);
}

// One branch of every sequence moves into the prefix; step numbers move with it.  All sequences or none: every CTA looks all of them over
// (nothing that is looked at is written here).
__global__ void k_branch_adopt(mbema_branches br, const long long* __restrict__ branch, long long t_next) {
    const int b = blockIdx.x, tid = threadIdx.x;
    const int N = (int)br.N, cap = (int)br.cap, Kcap = (int)br.Kcap;
    const long long t0 = br.t0[0];
    int bad = 0;
    for (int i = tid; i < br.B; i += blockDim.x) {
        const long long s = branch[i];
        if (s < 0 || s >= br.S) bad |= 8;
        else if (t_next < t0 + br.len[(int64_t)i * br.S + s]) bad |= 4;
    }
    const int no_branch = __syncthreads_or(bad & 8), too_early = __syncthreads_or(bad & 4);
    if (no_branch || too_early) {
        if (b == 0 && tid == 0) atomicOr(br.overflow, (no_branch ? 8 : 0) | (too_early ? 4 : 0));
        return;
    }
    const int64_t r = (int64_t)b * br.S + branch[b];
    const long long shift = t_next - (t0 + br.len[r]);
    const int own_n = br.own_n[r];
    for (size_t e = tid; e < (size_t)own_n * N; e += blockDim.x) {
        const int u = (int)(e / N), c = (int)(e - (size_t)u * N);
        br.state[((size_t)b * br.V + br.own_slot[(size_t)r * cap + u]) * N + c] = br.own_state[((size_t)r * cap + u) * N + c];
    }
    for (int u = tid; u < own_n; u += blockDim.x)
        br.last_t[(size_t)b * br.V + br.own_slot[(size_t)r * cap + u]] = br.own_t[(size_t)r * cap + u];
    __shared__ int s_na;
    if (tid < 32) {                                  // slots that the prefix did not list, in the order the branch met them
        int na = min(br.n_active[b], Kcap);
        for (int u0 = 0; u0 < own_n; u0 += 32) {
            const int u = u0 + tid;
            const int v = u < own_n ? br.own_slot[(size_t)r * cap + u] : -1;
            const bool add = v >= 0 && br.pos[(size_t)b * br.V + v] < 0;
            const unsigned m = __ballot_sync(0xffffffffu, add);
            const int at = na + __popc(m & ((1u << tid) - 1u));
            if (add && at < Kcap) br.active[(size_t)b * Kcap + at] = v;
            na += __popc(m);
            if (na > Kcap) { na = Kcap; if (tid == 0) atomicOr(br.overflow, 1); }
        }
        if (tid == 0) { br.n_active[b] = na; s_na = na; }
    }
    __syncthreads();
    for (int k = tid; k < s_na; k += blockDim.x) br.last_t[(size_t)b * br.V + br.active[(size_t)b * Kcap + k]] += (int)shift;
}

int check_branches(const mbema_branches* br) {
    if (!br) return MBEMA_ERR_NULL;
    if (br->B < 0 || br->S < 1 || br->V < 1 || br->N < 1 || br->Kcap < 1 || br->cap < 1 || br->max_new < 1) return MBEMA_ERR_SHAPE;
    if (br->N > 128 || br->max_new > BR_MAX_NEW || br->B > 65535 || br->B * br->S > 0x7fffffff / 2 || br->V > 0x7fffffff ||
        br->Kcap > 0x7ffffff || br->cap > 0x7ffffff)
        return MBEMA_ERR_UNSUPPORTED;
    if (br->B == 0) return MBEMA_OK;
    const void* need[] = {br->rhos, br->state, br->last_t, br->active, br->n_active, br->pos, br->t0, br->len, br->own_n, br->own_new,
                          br->own_slot, br->own_t, br->own_state, br->touched, br->st_tok, br->st_own, br->st_pos, br->st_same,
                          br->st_new, br->st_state, br->overflow};
    for (const void* p : need)
        if (!p) return MBEMA_ERR_NULL;
    if (br->pre_op || br->own_op || br->work || br->status) {              // all four or none
        if (!branch_tc_supported(br->N) || br->S >= 65535 || br->B >= 65535) return MBEMA_ERR_UNSUPPORTED;
        if (!br->pre_op || !br->own_op || !br->work || !br->status) return MBEMA_ERR_NULL;
        if (((uintptr_t)br->pre_op | (uintptr_t)br->own_op | (uintptr_t)br->state | (uintptr_t)br->own_state) & 15 || (uintptr_t)br->work & 7) return MBEMA_ERR_ALIGN;
        const int64_t blocks = (br->S + BR_BLOCK - 1) / BR_BLOCK;                   // the running sums stay below 2^30
        if (br->B * blocks * (br->Kcap / 16 + 1) * BR_COST_BLOCK + br->B * br->S * (br->cap / 16 + 1) * BR_COST_OWN >= 1ll << 30) return MBEMA_ERR_UNSUPPORTED;
    }
    return MBEMA_OK;
}

}  // namespace mbema

using namespace mbema;

extern "C" int mbema_branches_init(const mbema_branches* br, int64_t t_now, const int32_t* t_now_dev, void* stream) {
    int rc = check_branches(br);
    if (rc != MBEMA_OK) return rc;
    if (!t_now_dev && (t_now < 0 || t_now > 0x7fffffff)) return MBEMA_ERR_SHAPE;
    if (br->B == 0) return MBEMA_OK;
    MBEMA_CUDA_TRY(cudaMemsetAsync(br->pos, 0xff, (size_t)br->B * br->V * sizeof(int32_t), (cudaStream_t)stream));
    dim3 grid((unsigned)((br->Kcap + 255) / 256), (unsigned)br->B);
    k_branch_init<<<grid, 256, 0, (cudaStream_t)stream>>>(*br, (int)t_now, t_now_dev);
    return check_launch();
}

extern "C" int mbema_branches_extend(const mbema_branches* br, const int64_t* tok, int64_t n, int64_t n_pending, float* C_q, void* stream) {
    int rc = check_branches(br);
    if (rc != MBEMA_OK) return rc;
    if (n < 1 || n > br->max_new || n_pending < 0 || n_pending > br->max_new) return MBEMA_ERR_SHAPE;
    if (br->B == 0) return MBEMA_OK;
    if (!tok || !C_q) return MBEMA_ERR_NULL;
    cudaStream_t st = (cudaStream_t)stream;
    const long long* tk = (const long long*)tok;
    const int64_t branches = br->B * br->S;
    const bool beside = br->pre_op && n_pending == 0;
    if (!beside) {
        MBEMA_CUDA_TRY(launch_early(k_branch_stage, dim3((unsigned)branches), BS_THREADS, 0, st, *br, tk, (int)n, nullptr, (int)n_pending, C_q));
        rc = check_launch();
        if (rc != MBEMA_OK || !br->pre_op) return rc;
    }
    // shares of a list: eight CTAs an SM over all lists, one for every 32 or 16 slots where that is enough
    const int64_t lists = branches + br->B, items = 32 / (br->N / 64), longest = (std::max(br->Kcap, br->cap) + items - 1) / items;
    const int64_t shares = std::min(longest, std::max<int64_t>(1, 8 * 148 / lists + 1)), ctas = lists * shares + 1;
    if (beside) MBEMA_CUDA_TRY(launch_early(k_branch_operands<true>, dim3((unsigned)(branches + ctas)), OPERAND_THREADS, 0, st, *br, (int)shares, tk, (int)n, C_q));
    else MBEMA_CUDA_TRY(launch_early(k_branch_operands<false>, dim3((unsigned)ctas), OPERAND_THREADS, 0, st, *br, (int)shares, tk, (int)n, C_q));
    return check_launch();
}

extern "C" int mbema_branches_keep(const mbema_branches* br, const int64_t* counts, int64_t n_pending, void* stream) {
    int rc = check_branches(br);
    if (rc != MBEMA_OK) return rc;
    if (n_pending < 0 || n_pending > br->max_new) return MBEMA_ERR_SHAPE;
    if (br->B == 0 || n_pending == 0) return MBEMA_OK;
    if (!counts) return MBEMA_ERR_NULL;
    MBEMA_CUDA_TRY(launch_early(k_branch_stage, dim3((unsigned)(br->B * br->S)), BS_THREADS, 0, (cudaStream_t)stream, *br, nullptr, 0, (const long long*)counts, (int)n_pending, nullptr));
    return check_launch();
}

extern "C" int mbema_branches_adopt(const mbema_branches* br, const int64_t* branch, int64_t t_next, void* stream) {
    int rc = check_branches(br);
    if (rc != MBEMA_OK || br->B == 0) return rc;
    if (!branch) return MBEMA_ERR_NULL;
    if (t_next < 0 || t_next > 0x7fffffff) return MBEMA_ERR_SHAPE;
    k_branch_adopt<<<(unsigned)br->B, 256, 0, (cudaStream_t)stream>>>(*br, (const long long*)branch, (long long)t_next);
    return check_launch();
}
