// Attention of the rows of a decode state's branches (mbema_branches_attend): fp32 arithmetic on the CUDA cores, and the merge.
//
// A slot of the prefix that a branch has not touched has the same state in every branch at the same step, so its gate
// SiLU(M W_pe), K = E_k * gate and V = E_v * gate are formed once a (sequence, step) and read by all S branches; the slots that a
// branch has touched are its own, and a row sees its prefix through a mask without them:
//     softmax over {prefix slots not touched} + {own slots} + {tokens staged before the row} + {V_total - listed, score 0, value 0}.
// A CTA takes one job (a chunk of slots, up to 32 rows) for one head: K and V tiles of 64 slots in shared memory, the branches' scores
// against them, online softmax, one partial (m, l, o) per row.  k_branch_merge joins the partials, adds the few staged
// tokens (each a dot product of N channels, in fp32) and the zero-score slots.
#include <algorithm>

#include "branches.cuh"

namespace mbema {

static constexpr int BA_THREADS = 256;
static constexpr int BA_TILE = 64;       // slots a tile
static constexpr int BA_ROWS = 32;       // branches a CTA
static constexpr int BA_LD = 68;         // floats a row of 64 in shared memory: 16-byte pieces of eight rows lie in different banks
static constexpr int BM_WARPS = 4;
static constexpr int BM_STAGED = 2 * BM_WARPS;      // staged tokens at a time: two a warp
static constexpr int BM_ROWS = 8;                   // steps a CTA, at most
static constexpr int BM_BATCH = 8;                  // partials in flight

static size_t ba_smem(int N) {
    return ((size_t)N * BR_HD + (size_t)N * BA_LD + 2 * BA_TILE * BA_LD + (size_t)BA_ROWS * (2 * BR_HD + BA_LD) + 2 * ((N + 3) & ~3) + 3 * BA_ROWS +
            2 * BA_TILE) * 4;
}

// grid: x = prefix jobs (B, blocks of 32 branches, chunks; then blocks of steps), then own jobs (B * S, chunks; all steps); y = head.
// A job's rows are (step, branch) pairs, 32 at most: the tile's states and E rows, loaded once, serve as many steps as that allows.
// The gate product is tiled 4 slots x 4 channels to a thread (three wavefronts of shared memory for 16 FMAs a warp; one slot and 16
// channels take nine); from step to step the states are multiplied by rho in place, which costs a tenth of a power in front of every row of W.
// 2 sequences x 5 branches x 3 rows, 701 slots: 30 us, bound by latency (eight meetings of the CTA a tile and step); 8 x 2 x 4, 2000 slots: 260,
// 64 % of the issue slots and of shared memory's wavefronts.
__global__ void __launch_bounds__(BA_THREADS, 2) k_branch_attend(BranchArgs a) {
    extern __shared__ __align__(16) float smem[];
    br_wait_for_kernel_before();
    br_let_next_kernel_start();
    const mbema_branches& br = a.br;
    const int N = (int)br.N;
    const int n = a.n, H = a.H, h = blockIdx.y;
    const int SP = a.plan.SP, SO = a.plan.SO;
    const int blocks = (int)((br.S + BA_ROWS - 1) / BA_ROWS);
    const int64_t n_pre = (int64_t)br.B * blocks * SP * a.plan.JP;
    const bool own = blockIdx.x >= n_pre;
    int b, s0, branches, chunk, k_lo, k_hi, j0, steps;
    if (!own) {
        chunk = (int)(blockIdx.x % SP);
        int y = (int)(blockIdx.x / SP);
        j0 = (y % a.plan.JP) * a.plan.steps;
        steps = min(a.plan.steps, n - j0);
        y /= a.plan.JP;
        b = y / blocks;
        s0 = (y % blocks) * BA_ROWS;
        branches = min(BA_ROWS, (int)br.S - s0);
        k_lo = chunk * a.plan.chp;
        k_hi = min(k_lo + a.plan.chp, min(br.n_active[b], (int)br.Kcap));
    } else {
        const int64_t x = blockIdx.x - n_pre;
        chunk = (int)(x % SO);
        const int64_t r = x / SO;
        b = (int)(r / br.S);
        s0 = (int)(r % br.S);
        branches = 1;
        j0 = 0;
        steps = n;
        k_lo = chunk * a.plan.cho;
        k_hi = min(k_lo + a.plan.cho, br.own_n[r]);
    }
    if (k_lo >= k_hi) return;
    const int64_t r0 = (int64_t)b * br.S + s0;
    const int rows = branches * steps;                    // row = step * branches + branch
    float* W_sh = smem;                                   // [N][64]
    float* A_sh = W_sh + N * BR_HD;                       // [N][68]: states at step j0, transposed; groups of four slots change places by the channel (state_row's stores)
    float* K_sh = A_sh + N * BA_LD;                       // [64][68]
    float* V_sh = K_sh + BA_TILE * BA_LD;
    float* q_sh = V_sh + BA_TILE * BA_LD;                 // [32][64], scaled to base-2 scores
    float* o_sh = q_sh + BA_ROWS * BR_HD;                 // [32][64]
    float* P_sh = o_sh + BA_ROWS * BR_HD;                 // [32][68]
    float* l2r_sh = P_sh + BA_ROWS * BA_LD;
    float* rho_sh = l2r_sh + ((N + 3) & ~3);
    float* m_sh = rho_sh + ((N + 3) & ~3);
    float* l_sh = m_sh + BA_ROWS;
    float* al_sh = l_sh + BA_ROWS;
    int* v_sh = reinterpret_cast<int*>(al_sh + BA_ROWS);  // the tile's slots, and their ages
    float* dt_sh = reinterpret_cast<float*>(v_sh + BA_TILE);
    __shared__ unsigned hid_sh[2 * BA_ROWS];              // bits of the tile's slots that a branch has touched
    __shared__ int pos_sh[BA_ROWS * BR_MAX_NEW];          // the list places that its staged tokens hide from the rows behind them
    const int tid = threadIdx.x;
    const int D = H * BR_HD;
    const int tau = br.t0[0] + br.len[r0] + j0;
    const bool whole = N % 4 == 0 && !(((uintptr_t)br.state | (uintptr_t)br.own_state) & 15);      // (a state may be a view at any offset)
    for (int i = tid; i < branches * (j0 + steps); i += BA_THREADS) {
        const int branch = i / (j0 + steps), place = i - branch * (j0 + steps);
        pos_sh[branch * BR_MAX_NEW + place] = (own ? br.st_own : br.st_pos)[br_index(br, r0 + branch, place)];
    }
    auto slots_of = [&](int k0) {                         // (the first 64 threads)
        const int k = k0 + tid;
        int v = 0;
        float dt = 0.f;
        if (k < k_hi) {
            v = own ? br.own_slot[(size_t)r0 * br.cap + k] : br.active[(size_t)b * br.Kcap + k];
            dt = (float)(tau - (own ? br.own_t[(size_t)r0 * br.cap + k] : br.last_t[(size_t)b * br.V + v]));
        }
        v_sh[tid] = v;
        dt_sh[tid] = dt;
    };
    auto state_row = [&](int k0, int k) {
        return own ? br.own_state + ((size_t)r0 * br.cap + k0 + k) * N : br.state + ((size_t)b * br.V + v_sh[k]) * N;
    };
    if (tid < BA_TILE) slots_of(k_lo);
    for (int i = tid; i < N * (BR_HD / 4); i += BA_THREADS)
        *reinterpret_cast<float4*>(W_sh + i * 4) = *reinterpret_cast<const float4*>(a.W + (size_t)(i >> 4) * D + h * BR_HD + (i & 15) * 4);
    for (int i = tid; i < N; i += BA_THREADS) {
        rho_sh[i] = br.rhos[i];
        l2r_sh[i] = br_log2(rho_sh[i]);
    }
    for (int i = tid; i < rows * BR_HD; i += BA_THREADS) {
        const int row = i >> 6, st = row / branches;
        q_sh[i] = ld_dyn_f32(a.q, a.q_dt, ((((size_t)(r0 + row - st * branches)) * n + j0 + st) * H + h) * BR_HD + (i & 63)) * BR_SCORE_LOG2;
        o_sh[i] = 0.f;
    }
    for (int i = tid; i < BA_ROWS; i += BA_THREADS) { m_sh[i] = -INFINITY; l_sh[i] = 0.f; }
    const int tx = tid & 15, ty = tid >> 4;               // gate: channels 4 tx.., slots 4 ty..
    const int slot = tid & 63, group = tid >> 6;          // states and scores: a slot, every fourth branch; output: a column, every fourth branch
    for (int k0 = k_lo; k0 < k_hi; k0 += BA_TILE) {
        const int tile = min(BA_TILE, k_hi - k0);
        __syncthreads();                                  // the slots are there
        if (tid < 2 * branches) {
            const int words = (int)((br.Kcap + 31) / 32), word = (k0 >> 5) + (tid & 1);
            hid_sh[tid] = !own && word < words ? br.touched[(size_t)(r0 + (tid >> 1)) * words + word] : 0u;
        }
        if (whole) {                                      // whole rows, 16 bytes a thread
            for (int i = tid; i < BA_TILE * (N / 4); i += BA_THREADS) {
                const int k = i / (N / 4), c = (i - k * (N / 4)) * 4;
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                if (k < tile) {
                    const float dt = dt_sh[k];
                    x = *reinterpret_cast<const float4*>(state_row(k0, k) + c);
                    x.x *= exp2f(dt * l2r_sh[c]); x.y *= exp2f(dt * l2r_sh[c + 1]);
                    x.z *= exp2f(dt * l2r_sh[c + 2]); x.w *= exp2f(dt * l2r_sh[c + 3]);
                }
                float* dst = A_sh + c * BA_LD + (k ^ (((c >> 2) & 7) << 2));
                dst[0] = x.x; dst[BA_LD] = x.y; dst[2 * BA_LD] = x.z; dst[3 * BA_LD] = x.w;
            }
        } else {
            for (int i = tid; i < BA_TILE * N; i += BA_THREADS) {
                const int k = i / N, c = i - k * N;
                A_sh[c * BA_LD + (k ^ (((c >> 2) & 7) << 2))] = k < tile ? state_row(k0, k)[c] * exp2f(dt_sh[k] * l2r_sh[c]) : 0.f;
            }
        }
        float4 ek[4], ev[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ek[i] = ev[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (4 * ty + i < tile) {
                const size_t off = (size_t)v_sh[4 * ty + i] * D + h * BR_HD + 4 * tx;
                ek[i] = ld4_dyn_f32(a.Ek, a.e_dt, off);
                ev[i] = ld4_dyn_f32(a.Ev, a.e_dt, off);
            }
        }
        for (int st = 0; st < steps; ++st) {
            const int j = j0 + st, base = st * branches;
            __syncthreads();                              // the states are there, the step before has read K, V and P
            float acc[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
#pragma unroll 8
            for (int c = 0; c < N; ++c) {
                const float4 x = *reinterpret_cast<const float4*>(A_sh + c * BA_LD + 4 * (ty ^ ((c >> 2) & 7)));
                const float4 w = *reinterpret_cast<const float4*>(W_sh + c * BR_HD + 4 * tx);
                const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    acc[i][0] = fmaf(xs[i], w.x, acc[i][0]);
                    acc[i][1] = fmaf(xs[i], w.y, acc[i][1]);
                    acc[i][2] = fmaf(xs[i], w.z, acc[i][2]);
                    acc[i][3] = fmaf(xs[i], w.w, acc[i][3]);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float g[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) g[c] = a.silu ? __fdividef(acc[i][c], 1.0f + expf(-acc[i][c])) : acc[i][c];
                const int at = (4 * ty + i) * BA_LD + 4 * tx;
                *reinterpret_cast<float4*>(K_sh + at) = make_float4(ek[i].x * g[0], ek[i].y * g[1], ek[i].z * g[2], ek[i].w * g[3]);
                *reinterpret_cast<float4*>(V_sh + at) = make_float4(ev[i].x * g[0], ev[i].y * g[1], ev[i].z * g[2], ev[i].w * g[3]);
            }
            __syncthreads();
            if (st + 1 < steps) {                         // the next step's states: every one has been read (at most 31 roundings of 2^-24)
                for (int i = tid; i < N * (BA_TILE / 4); i += BA_THREADS) {
                    float4* x = reinterpret_cast<float4*>(A_sh + (i >> 4) * BA_LD + 4 * (i & 15));
                    const float rho = rho_sh[i >> 4];
                    float4 y = *x;
                    y.x *= rho; y.y *= rho; y.z *= rho; y.w *= rho;
                    *x = y;
                }
            }
            if (st + 1 == steps && tid < BA_TILE && k0 + BA_TILE < k_hi) slots_of(k0 + BA_TILE);
            for (int br0 = group; br0 < branches; br0 += 16) {        // branches br0, br0 + 4, + 8, + 12 against one slot's K
                const float4* kp = reinterpret_cast<const float4*>(K_sh + slot * BA_LD);
                float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
                for (int i = 0; i < 16; ++i) {
                    const float4 x = kp[i];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (br0 + 4 * e < branches) {
                            const float4 y = *reinterpret_cast<const float4*>(q_sh + (base + br0 + 4 * e) * BR_HD + 4 * i);
                            s[e] = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, s[e]))));
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int branch = br0 + 4 * e;
                    if (branch < branches) {
                        bool hide = slot >= tile || ((hid_sh[2 * branch + (slot >> 5)] >> (slot & 31)) & 1u);
                        for (int i = 0; i < j; ++i) hide |= pos_sh[branch * BR_MAX_NEW + i] == k0 + slot;
                        P_sh[(base + branch) * BA_LD + slot] = hide ? -INFINITY : s[e];
                    }
                }
            }
            __syncthreads();
            for (int row = base + (tid >> 5); row < base + branches; row += BA_THREADS / 32) {
                const int lane = tid & 31;
                float* p = P_sh + row * BA_LD;
                const float x = p[lane], y = p[lane + 32];
                float mx = fmaxf(x, y);
#pragma unroll
                for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                const float m_old = m_sh[row];
                const float m_new = fmaxf(m_old, mx);
                const float ref = m_new == -INFINITY ? 0.f : m_new;      // nothing visible so far: weights are zero all the same
                const float ex = exp2f(x - ref), ey = exp2f(y - ref);
                p[lane] = ex;
                p[lane + 32] = ey;
                const float sum = warp_sum(ex + ey);
                if (lane == 0) {
                    const float alpha = exp2f(m_old - ref);
                    m_sh[row] = m_new;
                    l_sh[row] = l_sh[row] * alpha + sum;
                    al_sh[row] = alpha;
                }
            }
            __syncthreads();
            if (branches == 1) {                          // the groups share the slots, 16 each; joined in the row's old scores' place
                float x = 0.f;
#pragma unroll
                for (int c = 0; c < 16; ++c) x = fmaf(P_sh[base * BA_LD + 16 * group + c], V_sh[(16 * group + c) * BA_LD + slot], x);
                K_sh[tid] = x;                            // (the scores have been read off K)
                __syncthreads();
                if (group == 0)
                    o_sh[base * BR_HD + slot] = o_sh[base * BR_HD + slot] * al_sh[base] + ((K_sh[slot] + K_sh[64 + slot]) + (K_sh[128 + slot] + K_sh[192 + slot]));
            } else {
                for (int br0 = group; br0 < branches; br0 += 16) {
                    float o[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int row = base + br0 + 4 * e;
                        o[e] = br0 + 4 * e < branches ? o_sh[row * BR_HD + slot] * al_sh[row] : 0.f;
                    }
#pragma unroll 4
                    for (int c = 0; c < BA_TILE; c += 4) {                // (slots past the list: weight 0, value 0)
                        float v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = V_sh[(c + e) * BA_LD + slot];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (br0 + 4 * e < branches) {
                                const float4 p = *reinterpret_cast<const float4*>(P_sh + (base + br0 + 4 * e) * BA_LD + c);
                                o[e] = fmaf(p.x, v[0], fmaf(p.y, v[1], fmaf(p.z, v[2], fmaf(p.w, v[3], o[e]))));
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (br0 + 4 * e < branches) o_sh[(base + br0 + 4 * e) * BR_HD + slot] = o[e];
                }
            }
            // (the next step's K, V and P follow the meeting at its start)
        }
    }
    __syncthreads();
    const int part = own ? SP + chunk : chunk;
    for (int i = tid; i < rows * BR_HD; i += BA_THREADS) {
        const int row = i >> 6, st = row / branches;
        const size_t at = ((((size_t)(r0 + row - st * branches)) * n + j0 + st) * H + h) * (SP + SO) + part;
        a.po[at * BR_HD + (i & 63)] = o_sh[i];
        if ((i & 63) == 0) a.ml[at] = make_float2(m_sh[row], l_sh[row]);
    }
}

// A CTA takes up to RJ steps of a (branch, head): for the staged tokens its four warps share the state channels (W, 4 N * 64 bytes, is read
// once a CTA from L2, then from L1), a lane holds two output columns.  One step: the warps share its partials.  More: a step's
// partials are one warp's.
// Bound by latency: three dependent loads of staged tokens, two of partials.
// PIECES: partials of a tensor-core kernel (a list's pieces, one a worker), else of the fp32 kernel (its chunks).
template <bool PIECES>
__global__ void __launch_bounds__(BM_WARPS * 32) k_branch_merge(BranchArgs a, int RJ) {
    __shared__ __align__(16) float s_c[128][BM_STAGED];         // states of the staged tokens at this row
    __shared__ float2 s_x[BM_WARPS][BM_STAGED][32];             // partial pre-activations
    __shared__ float2 s_ml[BM_ROWS][BM_WARPS];                  // a warp's maximum and sum, and
    __shared__ float2 s_o[BM_ROWS][BM_WARPS][32];               // its o
    const mbema_branches& br = a.br;
    const int N = (int)br.N, n = a.n, H = a.H, D = H * BR_HD;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = (int)(blockIdx.x % H), JB = (n + RJ - 1) / RJ;
    const int64_t rest_id = blockIdx.x / H, r = rest_id / JB;
    const int j_first = (int)(rest_id - r * JB) * RJ, rows = min(RJ, n - j_first);
    const int b = (int)(r / br.S), s = (int)(r - (int64_t)b * br.S);
    const float2* Wc = reinterpret_cast<const float2*>(a.W + h * BR_HD + 2 * lane);
    // The staged tokens do not wait for the kernel before, and no ordinary load reads global memory up to the wait.  (With the wait here: 8 drafted
    // rows of one sequence 2 us more of 17, 64 sequences of 6 rows 18 of 335, 2 x 5 branches of 3 rows in fp32 arithmetic 3 of 33.)
    for (int jj = 0; jj < rows; ++jj) {
        const int j = j_first + jj;
        float M = -INFINITY, L = 0.f;
        float2 o = make_float2(0.f, 0.f);
        for (int i0 = 0; i0 < j; i0 += BM_STAGED) {
            const int cnt = min(BM_STAGED, j - i0);
            // loads that depend on no other first: a warp's two tokens, eight rows of W, a thread's first states; then the tokens' E rows
            auto W_rows = [&](float2 (&w)[8], int c0) {
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int c = c0 + u * BM_WARPS;
                    w[u] = c < N ? ld_gpu(Wc + (size_t)c * (D / 2)) : make_float2(0.f, 0.f);
                }
            };
            float2 w[8];
            int token[2];
            unsigned same[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const size_t at = br_index(br, r, min(i0 + warp + e * BM_WARPS, j - 1));
                token[e] = ld_gpu(br.st_tok + at);
                same[e] = (unsigned)ld_gpu(reinterpret_cast<const int*>(br.st_same) + at);
            }
            W_rows(w, warp);
            float x[4], rho[4];
            auto load_states = [&](int e0) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int e = min(e0 + u * BM_WARPS * 32, cnt * N - 1), i = e / N, c = e - i * N;
                    x[u] = ld_gpu(br.st_state + br_index(br, r, i0 + i) * N + c);
                    rho[u] = ld_gpu(br.rhos + c);
                }
            };
            load_states(threadIdx.x);
            float2 ek[2], ev[2], q = make_float2(0.f, 0.f);
            bool see[2];
            const size_t qoff = (((size_t)r * n + j) * H + h) * BR_HD + 2 * lane;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int place = i0 + warp + e * BM_WARPS;
                // none, or repeated before this row (j <= 31)
                see[e] = place < j && token[e] >= 0 && ((same[e] & ((1u << j) - 1u)) >> place) == 1u;
                ek[e] = ev[e] = make_float2(0.f, 0.f);
                if (see[e]) {
                    const size_t off = (size_t)token[e] * D + h * BR_HD + 2 * lane;
                    ek[e] = ld_gpu_pair(a.Ek, a.e_dt, off);
                    ev[e] = ld_gpu_pair(a.Ev, a.e_dt, off);
                    q = ld_gpu_pair(a.q, a.q_dt, qoff);
                }
            }
            __syncthreads();
            for (int e0 = threadIdx.x; e0 < cnt * N; e0 += 4 * BM_WARPS * 32) {
                if (e0 >= 4 * BM_WARPS * 32) load_states(e0);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int e = e0 + u * BM_WARPS * 32, i = e / N, c = e - i * N;
                    if (e < cnt * N) s_c[c][i] = (x[u] + 1.0f) * exp2f((float)(j - i0 - i) * br_log2(rho[u]));
                }
            }
            __syncthreads();
            float x0[BM_STAGED], x1[BM_STAGED];
#pragma unroll
            for (int i = 0; i < BM_STAGED; ++i) x0[i] = x1[i] = 0.f;
            for (int c0 = warp; c0 < N; c0 += BM_WARPS * 8) {     // eight rows of W in flight
                if (c0 != warp) W_rows(w, c0);
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int c = min(c0 + u * BM_WARPS, N - 1);
                    const float4 m0 = *reinterpret_cast<const float4*>(&s_c[c][0]), m1 = *reinterpret_cast<const float4*>(&s_c[c][4]);
                    const float m[8] = {m0.x, m0.y, m0.z, m0.w, m1.x, m1.y, m1.z, m1.w};
#pragma unroll
                    for (int i = 0; i < BM_STAGED; ++i) {         // (places past the last token hold whatever: their sums are not read)
                        x0[i] = fmaf(m[i], w[u].x, x0[i]);
                        x1[i] = fmaf(m[i], w[u].y, x1[i]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < BM_STAGED; ++i)
                if (i < cnt) s_x[warp][i][lane] = make_float2(x0[i], x1[i]);
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int i = warp + e * BM_WARPS;
                if (see[e]) {
                    float y0 = 0.f, y1 = 0.f;
#pragma unroll
                    for (int u = 0; u < BM_WARPS; ++u) { const float2 y = s_x[u][i][lane]; y0 += y.x; y1 += y.y; }
                    const float g0 = a.silu ? y0 / (1.0f + expf(-y0)) : y0, g1 = a.silu ? y1 / (1.0f + expf(-y1)) : y1;
                    const float score = warp_sum(q.x * (ek[e].x * g0) + q.y * (ek[e].y * g1)) * BR_SCORE_LOG2;
                    if (score == -INFINITY) continue;             // beyond fp32: no weight
                    const float m_new = fmaxf(M, score);
                    const float keep = exp2f(M - m_new), p = exp2f(score - m_new);
                    L = fmaf(L, keep, p);
                    o.x = fmaf(ev[e].x * g0, p, o.x * keep);
                    o.y = fmaf(ev[e].y * g1, p, o.y * keep);
                    M = m_new;
                }
            }
        }
        if (lane == 0) s_ml[jj][warp] = make_float2(M, L);
        s_o[jj][warp][lane] = o;
    }
    const int na = min(ld_gpu(br.n_active + b), (int)br.Kcap);
    const int own_new = ld_gpu(br.own_new + r);
    // partials of step j_first: np of the prefix from p0 on, then nq of the own slots from q0 on, p_step and q_step apart; of the next step
    // j_step further
    int np, nq;
    size_t p0, q0, p_step, q_step, j_step;
    if constexpr (PIECES) {
        auto unit_at = [&](int list) { return ld_gpu(br.work + 2 * (size_t)list); };          // the running sum of the lists' units
        struct Units { int lo, hi; };
        const size_t each = (size_t)n * H, at = (size_t)j_first * H + h;
        const bool one = br.S == 1;
        const int pre = one ? 2 * b : b * a.blocks + s / BR_BLOCK, own = one ? 2 * b + 1 : a.n_pre + (int)r;
        const int total = unit_at(a.lists);
        const Units in_pre = {unit_at(pre), unit_at(pre + 1)}, in_own = {unit_at(own), unit_at(own + 1)};
        const int workers = branch_workers(total, a.max_workers, one ? 1 : BR_LEAST_COST);
        auto pieces = [&](Units u, int unit, int& first) {
            first = 0;
            if (u.hi == u.lo) return 0;
            first = branch_worker_of(total, workers, u.lo);
            return branch_worker_of(total, workers, u.hi - unit) - first + 1;
        };
        int wp, wq;
        np = pieces(in_pre, one ? 1 : BR_COST_BLOCK, wp);
        nq = pieces(in_own, one ? 1 : BR_COST_OWN, wq);
        q_step = each;
        j_step = H;
        if (one) {
            np *= 4;
            nq *= 4;
            p_step = each;
            p0 = (size_t)(pre + wp) * 4 * each + at;
            q0 = (size_t)(own + wq) * 4 * each + at;
        } else {
            p_step = BR_BLOCK * each;
            p0 = ((size_t)(pre + wp) * BR_BLOCK + s % BR_BLOCK) * each + at;
            q0 = (size_t)(a.own_piece0 + r + wq) * each + at;
        }
    } else {
        const int SP = a.plan.SP, SO = a.plan.SO;
        np = (na + a.plan.chp - 1) / a.plan.chp;
        nq = (ld_gpu(br.own_n + r) + a.plan.cho - 1) / a.plan.cho;
        p_step = q_step = 1;
        j_step = (size_t)H * (SP + SO);
        p0 = (((size_t)r * n + j_first) * H + h) * (SP + SO);
        q0 = p0 + SP;
    }
    br_wait_for_kernel_before();
    // joins the warp's share of a step's partials (every share-th) to (M, L, o)
    auto join = [&](int jj, int first, int share, float& M, float& L, float2& o) {
        const size_t off = (size_t)jj * j_step;
        for (int p = first; p < np + nq; p += BM_BATCH * share) {
            float2 ml[BM_BATCH], x[BM_BATCH];
#pragma unroll
            for (int u = 0; u < BM_BATCH; ++u) {
                const int i = p + u * share;
                ml[u] = x[u] = make_float2(0.f, 0.f);
                if (i < np + nq) {
                    const size_t at = off + (i < np ? p0 + i * p_step : q0 + (i - np) * q_step);
                    ml[u] = a.ml[at];
                    x[u] = *reinterpret_cast<const float2*>(a.po + at * BR_HD + 2 * lane);
                }
            }
            float m_new = M;
#pragma unroll
            for (int u = 0; u < BM_BATCH; ++u) m_new = ml[u].y == 0.f ? m_new : fmaxf(m_new, ml[u].x);      // (0: every slot of it is hidden)
            const float keep = L == 0.f ? 0.f : exp2f(M - m_new);
            L *= keep;
            o.x *= keep;
            o.y *= keep;
#pragma unroll
            for (int u = 0; u < BM_BATCH; ++u) {
                if (ml[u].y == 0.f) continue;
                const float w = exp2f(ml[u].x - m_new);
                L = fmaf(ml[u].y, w, L);
                o.x = fmaf(x[u].x, w, o.x);
                o.y = fmaf(x[u].y, w, o.y);
            }
            M = m_new;
        }
    };
    if (rows == 1) {
        __syncwarp();
        float2 ml = s_ml[0][warp], o = s_o[0][warp][lane];
        join(0, warp, BM_WARPS, ml.x, ml.y, o);
        __syncwarp();
        if (lane == 0) s_ml[0][warp] = ml;
        s_o[0][warp][lane] = o;
    }
    __syncthreads();
    for (int jj = warp; jj < rows; jj += BM_WARPS) {
        const int j = j_first + jj;
        float rest = 0.f;                                       // slots that the row does not list: score 0, value 0
        if (!a.listed_only) {
            const int add = lane < j ? br.st_new[br_index(br, r, lane)] : 0;
            rest = fmaxf(a.v_total - (float)(na + own_new + __reduce_add_sync(0xffffffffu, add)), 0.f);
        }
        float M = rest > 0.f ? 0.f : -INFINITY, L = rest;
        float2 o = make_float2(0.f, 0.f);
#pragma unroll
        for (int u = 0; u < BM_WARPS; ++u) {
            const float2 ml = s_ml[jj][u];
            if (ml.y != 0.f) M = fmaxf(M, ml.x);
        }
        L = rest > 0.f ? rest * exp2f(-M) : 0.f;
#pragma unroll
        for (int u = 0; u < BM_WARPS; ++u) {
            const float2 ml = s_ml[jj][u], x = s_o[jj][u][lane];
            if (ml.y == 0.f) continue;
            const float e = exp2f(ml.x - M);
            L = fmaf(ml.y, e, L);
            o.x = fmaf(x.x, e, o.x);
            o.y = fmaf(x.y, e, o.y);
        }
        if (rows > 1) join(jj, 0, 1, M, L, o);
        const float inv = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);      // no slot at all: zero; a NaN stays one
        const size_t at = (((size_t)r * n + j) * H + h) * BR_HD + 2 * lane;
        if (a.q_dt == MBEMA_F32) {
            *reinterpret_cast<float2*>(reinterpret_cast<float*>(a.O) + at) = make_float2(o.x * inv, o.y * inv);
        } else {
            *reinterpret_cast<__nv_bfloat162*>(reinterpret_cast<__nv_bfloat16*>(a.O) + at) = __floats2bfloat162_rn(o.x * inv, o.y * inv);
        }
    }
}

// Steps a job: as many as leave it 32 rows.  Chunks: enough jobs for about four CTAs an SM, none shorter than a tile of 64 slots nor
// longer than sixteen.
static BranchPlan branch_plan(int64_t B, int64_t S, int64_t n, int64_t H, int64_t Kcap, int64_t cap) {
    BranchPlan p;
    p.steps = (int)std::max<int64_t>(1, std::min<int64_t>(n, BA_ROWS / std::min<int64_t>(S, BA_ROWS)));
    p.JP = (int)((n + p.steps - 1) / p.steps);
    auto tiles = [&](int64_t lists, int64_t slots) {
        const int64_t all = lists * H * ((slots + BA_TILE - 1) / BA_TILE);
        return std::min<int64_t>(16, std::max<int64_t>(1, all / (4 * 148)));
    };
    p.chp = (int)(BA_TILE * tiles(B * ((S + BA_ROWS - 1) / BA_ROWS) * p.JP, Kcap));
    p.cho = (int)(BA_TILE * tiles(B * S, cap));
    p.SP = (int)((Kcap + p.chp - 1) / p.chp);
    p.SO = (int)((cap + p.cho - 1) / p.cho);
    return p;
}

int launch_branch_attend_fp32(const BranchArgs& a, cudaStream_t st) {
    const mbema_branches& br = a.br;
    const int64_t jobs = br.B * ((br.S + BA_ROWS - 1) / BA_ROWS) * a.plan.SP * a.plan.JP + br.B * br.S * a.plan.SO;
    if (jobs > 0x7fffffff) return MBEMA_ERR_UNSUPPORTED;
    const size_t smem = ba_smem((int)br.N);
    static std::atomic<unsigned long long> done{0};
    MBEMA_CUDA_TRY(allow_smem(k_branch_attend, ba_smem(128), done));
    MBEMA_CUDA_TRY(launch_early(k_branch_attend, dim3((unsigned)jobs, (unsigned)a.H), BA_THREADS, smem, st, a));
    return check_launch();
}

int launch_branch_merge(const BranchArgs& a, bool pieces, cudaStream_t st) {
    // eight steps a CTA where three CTAs an SM are left: W then crosses L2 less often (64 sequences of 6 drafted rows with their attention: 335 us,
    // with a step a CTA 14 more); a step a CTA otherwise, as its loads then do not wait for one another (8 drafted rows of one sequence: 17 us,
    // with eight 15 more)
    const int64_t heads = a.br.B * a.br.S * a.H;
    const int RJ = heads * ((a.n + BM_ROWS - 1) / BM_ROWS) >= 3 * 148 ? std::min(a.n, BM_ROWS) : 1;
    const int64_t ctas = heads * ((a.n + RJ - 1) / RJ);
    if (ctas > 0x7fffffff) return MBEMA_ERR_UNSUPPORTED;
    MBEMA_CUDA_TRY(launch_early(pieces ? k_branch_merge<true> : k_branch_merge<false>, dim3((unsigned)ctas), BM_WARPS * 32, 0, st, a, RJ));
    return check_launch();
}

}  // namespace mbema

using namespace mbema;

static bool plan_sizes_ok(int64_t B, int64_t S, int64_t n, int64_t H, int64_t Kcap, int64_t cap) {
    return B >= 0 && S >= 1 && n >= 1 && n <= BR_MAX_NEW && H >= 1 && Kcap >= 1 && cap >= 1;
}

// number of partials of a call, and how it is dealt
static int64_t partials(int64_t B, int64_t S, int64_t n, int64_t H, int64_t Kcap, int64_t cap, int mode, BranchArgs* a) {
    if (mode != MBEMA_MODE_TC_BF16) {
        const BranchPlan p = branch_plan(B, S, n, H, Kcap, cap);
        if (a) a->plan = p;
        return B * S * n * H * (p.SP + p.SO);
    }
    if (S == 1) {
        const BranchRows p = branch_rows(n, H);
        if (a) {
            a->lists = (int)(2 * B);
            a->max_workers = p.ctas * p.IG;
        }
        return (2 * B + p.ctas * p.IG) * 4 * n * H;
    }
    const BranchShape p = branch_shape(S, n, H);
    const int64_t n_pre = B * p.blocks, workers = (int64_t)p.ctas * p.IG, own0 = (n_pre + workers) * BR_BLOCK;
    if (a) {
        a->lists = (int)(n_pre + B * S);
        a->n_pre = (int)n_pre;
        a->blocks = p.blocks;
        a->max_workers = (int)workers;
        a->own_piece0 = own0;
    }
    return (own0 + B * S + workers) * n * H;
}

extern "C" size_t mbema_branches_attend_workspace_bytes(int64_t B, int64_t S, int64_t n, int64_t H, int64_t Kcap, int64_t cap, int mode) {
    if (!plan_sizes_ok(B, S, n, H, Kcap, cap)) return 0;
    return align_up((size_t)partials(B, S, n, H, Kcap, cap, mode, nullptr) * (2 + BR_HD) * 4, 256) + 256;
}

extern "C" int mbema_branches_attend(const mbema_branches* br, const void* q, int q_dtype, const void* E_k, const void* E_v, int e_dtype,
                                     const float* W_pe, void* O, int64_t n, int64_t H, int64_t hd, int64_t V_total, int flags, int mode,
                                     void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_branches(br);
    if (rc != MBEMA_OK) return rc;
    if (!plan_sizes_ok(br->B, br->S, n, H, br->Kcap, br->cap) || n > br->max_new) return MBEMA_ERR_SHAPE;
    if (hd != BR_HD || H > 65535 || (mode != MBEMA_MODE_FP32 && mode != MBEMA_MODE_TC_BF16)) return MBEMA_ERR_UNSUPPORTED;
    if (mode == MBEMA_MODE_TC_BF16 && (!branch_tc_supported(br->N) || q_dtype != MBEMA_BF16 || e_dtype != MBEMA_BF16)) return MBEMA_ERR_UNSUPPORTED;
    if (br->B == 0) return MBEMA_OK;
    if (!q || !E_k || !E_v || !W_pe || !O || !workspace) return MBEMA_ERR_NULL;
    if ((q_dtype != MBEMA_F32 && q_dtype != MBEMA_BF16) || (e_dtype != MBEMA_F32 && e_dtype != MBEMA_BF16)) return MBEMA_ERR_DTYPE;
    if (((uintptr_t)q | (uintptr_t)E_k | (uintptr_t)E_v | (uintptr_t)W_pe | (uintptr_t)O | (uintptr_t)workspace) & 15) return MBEMA_ERR_ALIGN;
    if (workspace_bytes < mbema_branches_attend_workspace_bytes(br->B, br->S, n, H, br->Kcap, br->cap, mode)) return MBEMA_ERR_WORKSPACE;
    if (mode == MBEMA_MODE_TC_BF16 && (!br->pre_op || !br->own_op || !br->work || !br->status)) return MBEMA_ERR_NULL;
    BranchArgs a{};
    a.br = *br;
    a.q = q; a.Ek = E_k; a.Ev = E_v; a.W = W_pe; a.O = O;
    a.q_dt = q_dtype; a.e_dt = e_dtype; a.n = (int)n; a.H = (int)H;
    a.v_total = (float)V_total;
    a.silu = (flags & MBEMA_FLAG_SILU) ? 1 : 0;
    a.listed_only = (flags & MBEMA_FLAG_LISTED_ONLY) ? 1 : 0;
    const int64_t parts = partials(br->B, br->S, n, H, br->Kcap, br->cap, mode, &a);
    a.po = reinterpret_cast<float*>(workspace);
    a.ml = reinterpret_cast<float2*>(a.po + (size_t)parts * BR_HD);
    cudaStream_t st = (cudaStream_t)stream;
    const bool tc = mode == MBEMA_MODE_TC_BF16;
    rc = !tc ? launch_branch_attend_fp32(a, st)
         : br->S == 1 ? launch_branch_rows(a, branch_rows(n, H), st) : launch_branch_attend_tc(a, branch_shape(br->S, n, H), st);
    return rc != MBEMA_OK ? rc : launch_branch_merge(a, tc, st);
}
