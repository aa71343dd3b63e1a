// Attention of a single branch a sequence on tcgen05 (mbema_branches_attend, MBEMA_MODE_TC_BF16): drafted rows, or one row as in a
// decode step, over the prefix and the branch's own slots.
//
// A tile is 128 slots of a list; its operands lie in memory as the gate product wants them in shared memory (mbema_branches_extend),
// so one bulk copy fetches them, and rho^j of staged step j is in that step's W:  gate(j) = SiLU(A (rho^j W)),  M = 128 slots, N = 64
// channels of one head, accumulators in TMEM.  A thread owns a slot and all 64 channels: its score is a sum in the thread, it keeps its
// own running maximum, sum and o[64] over the tiles of a list, and only where the list (or the worker's stretch) ends do the 32 lanes of
// a warp join.  The gate goes back to TMEM between the two passes (q.K; P.V), since 64 of its values beside o[64] do not fit the registers.
//
// Roles: three epilogue groups of four warps; two warps gather the E_k and E_v rows (cp.async, mbarrier arrivals), one lane copies
// the operands, one issues the products.  With one step the groups are workers with stretches of their own, a tile each in turn; with
// two or three steps they take the same tile, a step each.
// 64 sequences, 3400 + 90 slots, 6 rows, 8 heads, 64 channels: 323 us (0.56e9 tanh of 16 a clock and SM would be 122).  Of a tile's 3700 cycles
// the three epilogue warps of a scheduler have MUFU work for 1540 and instructions for about 2100; the rest are waits that three warps, which
// is what o[64] leaves registers for, do not hide.  The two passes written out (372 us without), the mask before the waits, two FMA to an
// instruction (10 us).  V rounded to bf16 with P . V in mixed-precision FMA needs fewer instructions, but they and the conversions run at half
// to three quarters of the fp32 rate: an eighth slower.  The next tile's first channels loaded before this one is left: 4 % slower.
#include <algorithm>
#include <type_traits>

#include "branches.cuh"
#include "sm100_ptx.cuh"

namespace mbema {
namespace brows {

using namespace ptx;

static constexpr int TILE = BR_TILE, GROUPS = 3, EPI_WARPS = 4 * GROUPS, THREADS = (EPI_WARPS + 4) * 32;
static constexpr int WARP_K = EPI_WARPS, WARP_V = EPI_WARPS + 1, WARP_MMA = EPI_WARPS + 2, WARP_A = EPI_WARPS + 3;
// setmaxnreg: 12 * 32 * 152 (epilogue) + 4 * 32 * 56 (the other warps) = 12 * 32 * 144 + 4 * 32 * 80 = the launch allocation 512 * 128.  The
// second with three workers: each copying warp then follows three stretches, and with 56 registers keeps them in memory (64 sequences of
// one row 177 us for 121); the first otherwise (of six rows 364 us for 373).
static constexpr float W_SCALE = 64.0f;           // undoes BR_OP_SCALE

template <int ATOMS>                               // of 64 state channels
struct Smem {
    static constexpr int A_STAGES = ATOMS == 1 ? 4 : 2, E_STAGES = ATOMS == 1 ? 4 : 3, OP_BYTES = ATOMS * 16384;
    static constexpr int EK = A_STAGES * OP_BYTES, EV = EK + 16384, E_STAGE = 32768;
    static constexpr int B = EK + E_STAGES * E_STAGE, B_STEP = ATOMS * 8192, Q = B + GROUPS * B_STEP, BARS = Q + EPI_WARPS * 128, BYTES = BARS + 320 + 1024;
};

struct Bars {
    uint64_t a_full[4];            // operands have landed                                     (1 arrival and their bytes)
    uint64_t a_empty[4];           // every product that reads them has completed              (1 commit)
    uint64_t e_full[4];            // E rows have landed                                       (64: the lanes of both gathering warps)
    uint64_t e_empty[4];           // every epilogue warp of the tile has read them            (4 a step)
    uint64_t acc_full[GROUPS][2];  // gate product of a group's tile done                      (1 commit)
    uint64_t acc_empty[GROUPS][2]; // the group's warps have read its accumulators a second time (4)
    uint64_t w_full;               // W of every step is laid out                              (12: the epilogue warps)
    uint64_t drain;                // every product has completed (teardown)                   (1 commit)
    uint32_t tmem_base;
    int abort_flag;
    int tiles[GROUPS];             // of the CTA's workers
};
static_assert(sizeof(Bars) <= 320, "barrier block");

struct Cursor {                    // a worker's place in the lists
    int list, left, k, count, end; // left tiles of this list from slot k on; end: of the stretch, in tiles
    int2 n1, n2;                   // (running sum, length) of the next two lists, read ahead of their use
    __device__ __forceinline__ void start(const ListSearch& search, const int2* work, int lists, int total, int workers, int me, int lane) {
        const int c0 = branch_cut(total, workers, me);
        end = branch_cut(total, workers, me + 1);
        int2 at;
        list = search.find(work, lists, c0, lane, at, n1);
        n2 = work[min(list + 2, lists)];
        count = at.y;
        k = (c0 - at.x) * TILE;
        left = min(n1.x, end) - c0;
    }
    __device__ __forceinline__ bool next(const int2* work, int lists) {       // false: the stretch ends
        k += TILE;
        if (--left > 0) return true;
        for (;;) {
            const int2 at = n1;
            if (at.x >= end) return false;
            ++list;
            n1 = n2;
            n2 = work[min(list + 2, lists)];
            if (n1.x > at.x) { left = min(n1.x, end) - at.x; k = 0; count = at.y; return true; }
        }
    }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {        // once this thread's copies so far have landed
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
template <int OFFSET>
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4 + %5];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr), "n"(OFFSET));
    return v;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

template <int ATOMS, int IG, bool SILU>
__global__ void __launch_bounds__(THREADS, 1) k_branch_rows(BranchArgs a, int JW) {
    using L = Smem<ATOMS>;
    extern __shared__ unsigned char smem_raw[];
    br_wait_for_kernel_before();
    br_let_next_kernel_start();
    unsigned char* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    Bars* bars = reinterpret_cast<Bars*>(sm + L::BARS);
    volatile int* abort_flag = &bars->abort_flag;
    const mbema_branches& br = a.br;
    constexpr int N = 64 * ATOMS;
    const int h = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int D = a.H * BR_HD;
    const int steps = min(JW, a.n - (int)blockIdx.z * JW), j0 = blockIdx.z * JW;
    const int lists = a.lists;
    const int2* work = reinterpret_cast<const int2*>(br.work);
    ListSearch search;
    search.begin(work, lists, tid & 31);
    const int total = work[lists].x;
    const int workers = max(1, min((int)gridDim.x * IG, total));
    const int me0 = blockIdx.x * IG;
    if (total == 0 || me0 >= workers) return;                     // nothing to do (the same for all threads)
    if (tid == 0) {
        for (int i = 0; i < L::A_STAGES; ++i) {
            mbar_init(&bars->a_full[i], 1);
            mbar_init(&bars->a_empty[i], 1);
        }
        for (int i = 0; i < L::E_STAGES; ++i) {
            mbar_init(&bars->e_full[i], 64);
            mbar_init(&bars->e_empty[i], 4 * steps);
        }
        for (int g = 0; g < GROUPS; ++g)
            for (int i = 0; i < 2; ++i) {
                mbar_init(&bars->acc_full[g][i], 1);
                mbar_init(&bars->acc_empty[g][i], 4);
            }
        mbar_init(&bars->w_full, EPI_WARPS);
        mbar_init(&bars->drain, 1);
        bars->abort_flag = *reinterpret_cast<volatile int*>(br.status);
        for (int g = 0; g < IG; ++g)
            bars->tiles[g] = me0 + g < workers ? branch_cut(total, workers, me0 + g + 1) - branch_cut(total, workers, me0 + g) : 0;
        fence_barrier_init();
    }
    if (warp == WARP_MMA) {
        tmem_alloc(&bars->tmem_base, 512);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = bars->tmem_base;
    // tiles of this CTA's workers; the CTA's tiles are numbered round by round
    int rounds = 0;
#pragma unroll
    for (int g = 0; g < IG; ++g) rounds = max(rounds, bars->tiles[g]);
    const volatile int* count_of = bars->tiles;

    if (warp >= EPI_WARPS) {
        if constexpr (IG == 1) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;"); else asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        if (warp <= WARP_V) {
            // ------------------------------------------------------------ gathering warps: E_k or E_v rows, 8 lanes a row
            const char* table = reinterpret_cast<const char*>(warp == WARP_K ? a.Ek : a.Ev) + h * (BR_HD * 2) + (lane & 7) * 16;
            const uint32_t D2 = (uint32_t)D * 2;
            const int sub = lane >> 3;
            const uint32_t base = smem_u32(sm) + (warp == WARP_K ? L::EK : L::EV);
            const uint32_t even = base + sub * 128 + (((lane & 7) ^ sub) << 4), odd = base + (sub + 4) * 128 + (((lane & 7) ^ (sub + 4)) << 4);
            Cursor cur[IG] = {};
            int ids[IG][4];                                       // of each worker's next tile
            auto fetch_ids = [&](int g) {
                const int* slots = a.row_slots(cur[g].list);
#pragma unroll
                for (int i = 0; i < 4; ++i) ids[g][i] = slots[min(cur[g].k + 32 * i + lane, cur[g].count - 1)];
            };
#pragma unroll
            for (int g = 0; g < IG; ++g)
                if (count_of[g] > 0) { cur[g].start(search, work, lists, total, workers, me0 + g, lane); fetch_ids(g); }
            int st = 0, use = 0;
            bool go = true;
#pragma unroll 1
            for (int r = 0; r < rounds && go; ++r) {
#pragma unroll
                for (int g = 0; g < IG; ++g) {
                    if (!go || r >= count_of[g]) continue;
                    if (use > 0) go = __all_sync(0xffffffffu, mbar_wait(&bars->e_empty[st], (uint32_t)((use - 1) & 1), abort_flag, 1));
                    if (!go) continue;
                    uint32_t at = st * L::E_STAGE;
                    int id[4] = {ids[g][0], ids[g][1], ids[g][2], ids[g][3]};
#pragma unroll 1
                    for (int part = 0; part < 4; ++part) {        // 32 rows at a time: rows 4 x + sub
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            const uint32_t v = (uint32_t)__shfl_sync(0xffffffffu, id[0], x * 4 + sub);
                            cp_async16(at + ((x & 1) ? odd : even) + (x >> 1) * 1024, table + (uint64_t)v * D2);
                        }
                        at += 4096;
                        id[0] = id[1]; id[1] = id[2]; id[2] = id[3];
                    }
                    cp_async_arrive(&bars->e_full[st]);
                    if (++st == L::E_STAGES) { st = 0; ++use; }
                    if (cur[g].next(work, lists)) fetch_ids(g);
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        } else if (warp == WARP_A) {
            // ------------------------------------------------------------ operand copies
            Cursor cur[IG] = {};
#pragma unroll 1
            for (int g = 0; g < IG; ++g)
                if (count_of[g] > 0) cur[g].start(search, work, lists, total, workers, me0 + g, lane);
            if (lane == 0) {
                int st = 0, use = 0;
                bool go = true;
#pragma unroll 1
                for (int i = 0; go; ++i) {
                    const int r = i / IG, g = i - r * IG;
                    if (r >= rounds) break;
                    if (r >= count_of[g]) continue;
                    if (use > 0) go = mbar_wait(&bars->a_empty[st], (uint32_t)((use - 1) & 1), abort_flag, 2);
                    if (!go) break;
                    mbar_expect_tx(&bars->a_full[st], L::OP_BYTES);
                    bulk_load(sm + st * L::OP_BYTES, a.row_operands(cur[g].list) + (size_t)(cur[g].k / TILE) * L::OP_BYTES, L::OP_BYTES, &bars->a_full[st]);
                    cur[g].next(work, lists);
                    if (++st == L::A_STAGES) { st = 0; ++use; }
                }
                // given up: copies that may still be on their way (a wait that gives up returns soon after)
                for (int i = 0; !go && i < L::A_STAGES; ++i) {
                    const int uses = use + (i < st);               // times stage i was filled
                    if (uses > 0) mbar_wait(&bars->a_full[i], (uint32_t)((uses - 1) & 1), abort_flag, 6);
                }
            }
        } else if (warp == WARP_MMA && lane == 0) {
            // ------------------------------------------------------------ all products
            const uint32_t idesc = umma_idesc_16(TILE, BR_HD, 0, 0, 0, 0);
            int st = 0, use = 0;
            bool go = mbar_wait(&bars->w_full, 0, abort_flag, 5);
#pragma unroll 1
            for (int i = 0; go; ++i) {
                const int r = i / IG, g = i - r * IG;
                if (r >= rounds) break;
                if (r >= count_of[g]) continue;
                go = mbar_wait(&bars->a_full[st], (uint32_t)(use & 1), abort_flag, 3);
                const uint64_t da = umma_desc_k_sw128(smem_u32(sm + st * L::OP_BYTES));
#pragma unroll 1
                for (int s = 0; s < steps && go; ++s) {
                    const int w = IG == 1 ? s : g;
                    if (r >= 2) go = mbar_wait(&bars->acc_empty[w][r & 1], (uint32_t)(((r >> 1) - 1) & 1), abort_flag, 4);
                    if (!go) break;
                    tc_fence_after_sync();
                    const uint64_t db = umma_desc_k_sw128(smem_u32(sm + L::B + s * L::B_STEP));
#pragma unroll
                    for (int k16 = 0; k16 < 4 * ATOMS; ++k16)
                        umma_bf16_ss(tmem + (uint32_t)((w * 2 + (r & 1)) * BR_HD), da + (uint64_t)(((k16 >> 2) * 16384 + (k16 & 3) * 32) >> 4),
                                     db + (uint64_t)(((k16 >> 2) * 8192 + (k16 & 3) * 32) >> 4), idesc, k16 != 0 ? 1u : 0u);
                    umma_commit(&bars->acc_full[w][r & 1]);
                }
                if (!go) break;
                umma_commit(&bars->a_empty[st]);
                if (++st == L::A_STAGES) { st = 0; ++use; }
            }
            umma_commit(&bars->drain);
            mbar_wait(&bars->drain, 0, abort_flag, 7);
        }
    } else {
        // ---------------------------------------------------------------- epilogue: a thread a slot
        if constexpr (IG == 1) asm volatile("setmaxnreg.inc.sync.aligned.u32 152;"); else asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
        {   // W of every step, fp16, K-major rows of 64 state channels, 128-byte swizzle: a thread packs 8 channels of one output column
            const float scale = SILU ? 0.5f * W_SCALE : W_SCALE;      // SiLU(x) = h + h tanh(h), h = x / 2
            for (int i = tid; i < N * 8; i += EPI_WARPS * 32) {
                const int d = i & 63, c = (i >> 6) * 8;
                float w[8], l2r[8];
    #pragma unroll
                for (int e = 0; e < 8; ++e) {
                    w[e] = a.W[(size_t)(c + e) * D + h * BR_HD + d] * scale;
                    l2r[e] = br_log2(br.rhos[c + e]);
                }
                unsigned char* dst = sm + L::B + (c >> 6) * 8192 + d * 128 + ((((c & 63) >> 3) ^ (d & 7)) << 4);
                for (int s = 0; s < steps; ++s) {
                    float x[8];
    #pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = w[e] * exp2f((float)(j0 + s) * l2r[e]);
                    *reinterpret_cast<uint4*>(dst + s * L::B_STEP) = make_uint4(pack_h2(x[0], x[1]), pack_h2(x[2], x[3]), pack_h2(x[4], x[5]), pack_h2(x[6], x[7]));
                }
            }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->w_full);
        const int group = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
        const int jj = IG == 1 ? group : 0, j = j0 + jj;
        const int g = IG == 1 ? 0 : group;
        const int mine = count_of[g];
        if (jj < steps && mine > 0) {
            const int me = me0 + g;
            Cursor cur;
            cur.start(search, work, lists, total, workers, me, lane);
            const uint32_t taddr = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(group * 2 * BR_HD);
            uint32_t* q_sh = reinterpret_cast<uint32_t*>(sm + L::Q) + warp * 32;      // bf16; a copy a warp: the warps of a group never meet
            const uint32_t q_at = smem_u32(q_sh);
            const uint32_t e_row = smem_u32(sm) + L::EK + row * 128 + ((uint32_t)(row & 7) << 4);       // piece c of the row: ^ c * 16
            auto q_of = [&](int list) {
                return reinterpret_cast<const uint32_t*>(a.q)[((((size_t)a.row_branch(list) * a.n + j) * a.H + h) * BR_HD) / 2 + lane];
            };
            int q_list = cur.list;                                // the list whose q has been fetched
            uint32_t q_next = q_of(q_list);
            float m = -INFINITY, m8 = -INFINITY, l = 0.f, o[64];
            int staged = -1;
            const uint32_t* bits = nullptr;
            bool fresh = true, go = true;
            // this tile's number among the CTA's, as a stage and its use: tiles of one round lie one behind another
            int st = 0, use = 0;
            auto forward = [&](int by) {
                st += by;
                while (st >= L::E_STAGES) { st -= L::E_STAGES; ++use; }
            };
            int others[IG];                                       // tiles of the CTA's workers
#pragma unroll
            for (int x = 0; x < IG; ++x) others[x] = count_of[x];
#pragma unroll
            for (int x = 0; x < IG; ++x) forward(x < g && others[x] > 0 ? 1 : 0);
#pragma unroll 1
            for (int r = 0; r < mine && go; ++r) {
                if (fresh) {                                      // a new list: its row's q
                    const int64_t branch = a.row_branch(cur.list);
                    const bool prefix = a.row_is_prefix(cur.list);
                    const uint32_t x = q_list == cur.list ? q_next : q_of(cur.list);
                    __syncwarp();
                    q_sh[lane] = x;
                    __syncwarp();
                    q_list = min(cur.list + 1, lists - 1);
                    q_next = q_of(q_list);
                    staged = lane < j ? (prefix ? br.st_pos : br.st_own)[br_index(br, branch, lane)] : -1;
                    bits = prefix ? br.touched + (size_t)branch * ((br.Kcap + 31) / 32) : nullptr;
                    m = m8 = -INFINITY;
                    l = 0.f;
#pragma unroll
                    for (int i = 0; i < 64; ++i) o[i] = 0.f;
                    fresh = false;
                }
                const int k_w = cur.k + quarter * 32;             // this warp's 32 slots
                unsigned hide = bits && k_w < br.Kcap ? bits[k_w >> 5] : 0u;      // slots that the row does not see
                if (j > 0) {
                    const unsigned d = (unsigned)(staged - k_w);
                    hide |= __reduce_or_sync(0xffffffffu, d < 32u ? 1u << d : 0u);
                }
                if (cur.count - k_w < 32) hide |= 0xffffffffu << max(cur.count - k_w, 0);
                const uint32_t e_at = e_row + st * L::E_STAGE, t_at = taddr + (uint32_t)((r & 1) * BR_HD);
                go = __all_sync(0xffffffffu, mbar_wait(&bars->acc_full[group][r & 1], (uint32_t)((r >> 1) & 1), abort_flag, 8));
                if (go) go = __all_sync(0xffffffffu, mbar_wait(&bars->e_full[st], (uint32_t)(use & 1), abort_flag, 9));
                if (!go) break;
                tc_fence_after_sync();
                // 16 channels at a time, the next ones on their way.  The gate of the first 32 goes back to TMEM, the other 32 stay.
                float s0 = 0.f, s1 = 0.f, v0[16], v1[16];
                auto score = [&](float (&g16)[16], int c) {
                    const uint4 e0 = lds128<0>(e_at ^ (c << 5)), e1 = lds128<0>(e_at ^ ((c << 5) | 16));
                    const uint32_t e[8] = {e0.x, e0.y, e0.z, e0.w, e1.x, e1.y, e1.z, e1.w};
                    if (SILU) {
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            const uint64_t x2 = pair2(g16[i], g16[i + 1]);
                            unpair2(g16[i], g16[i + 1], fma2(x2, pair2(tanh_approx(g16[i]), tanh_approx(g16[i + 1])), x2));
                        }
                        if (c < 2) tmem_st_32x32b_x16(t_at + (uint32_t)(c * 16), g16);
                    }
                    const uint4 qa = lds128<0>(q_at + c * 32), qb = lds128<16>(q_at + c * 32);
                    const uint32_t q[8] = {qa.x, qa.y, qa.z, qa.w, qb.x, qb.y, qb.z, qb.w};
#pragma unroll
                    for (int i = 0; i < 8; ++i) {                 // (the product of two bf16 is exact in fp32, and needs no unpacking)
                        float x = 0.f, y = 0.f;
                        fma_f32_bf16x2(x, y, e[i], q[i]);
                        unpair2(s0, s1, fma2(pair2(x, y), pair2(g16[2 * i], g16[2 * i + 1]), pair2(s0, s1)));
                    }
                };
                tmem_ld16_nb(t_at, v0);
#pragma unroll
                for (int c = 0; c < 4; c += 2) {
                    tmem_wait_ld16(v0);
                    tmem_ld16_nb(t_at + (uint32_t)((c + 1) * 16), v1);
                    score(v0, c);
                    tmem_wait_ld16(v1);
                    if (c < 2) tmem_ld16_nb(t_at + 32, v0);
                    score(v1, c + 1);
                }
                const bool hidden = (hide >> lane) & 1u;
                const float x = (s0 + s1) * BR_SCORE_LOG2;
                const bool grow = !hidden && x > m8;        // o is scaled again only where the maximum moves by more than 2^8
                if (__any_sync(0xffffffffu, grow)) {
                    const float alpha = grow ? ex2_approx(m - x) : 1.0f;
                    if (grow) { m = x; m8 = x + 8.0f; }
                    l *= alpha;
#pragma unroll
                    for (int i = 0; i < 64; ++i) o[i] *= alpha;
                }
                const float p = hidden || x == -INFINITY ? 0.f : ex2_approx(x - m);      // (below fp32: no weight, before any maximum too)
                l += p;
                const uint64_t p2 = pair2(p, p);
                auto values = [&](float (&g16)[16], auto chunk) {
                    constexpr int c = decltype(chunk)::value;
                    const uint4 e0 = lds128<16384>(e_at ^ (c << 5)), e1 = lds128<16384>(e_at ^ ((c << 5) | 16));
                    const uint32_t e[8] = {e0.x, e0.y, e0.z, e0.w, e1.x, e1.y, e1.z, e1.w};
#pragma unroll
                    for (int i = 0; i < 8; ++i) {                 // (a hidden slot's value that is not finite: the row lists the same slot as its own)
                        const uint64_t w2 = mul2(p2, pair2(g16[2 * i], g16[2 * i + 1]));
                        unpair2(o[c * 16 + 2 * i], o[c * 16 + 2 * i + 1], fma2(w2, pair2(bf16_lo(e[i]), bf16_hi(e[i])), pair2(o[c * 16 + 2 * i], o[c * 16 + 2 * i + 1])));
                    }
                };
                values(v0, std::integral_constant<int, 2>());
                if (SILU) tmem_wait_st();
                tmem_ld16_nb(t_at, v0);
                values(v1, std::integral_constant<int, 3>());
                tmem_wait_ld16(v0);
                tmem_ld16_nb(t_at + 16, v1);
                values(v0, std::integral_constant<int, 0>());
                tmem_wait_ld16(v1);
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars->acc_empty[group][r & 1]);
                values(v1, std::integral_constant<int, 1>());
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars->e_empty[st]);
                int by = 0;                                       // to this worker's tile of the next round
#pragma unroll
                for (int x = 0; x < IG; ++x) by += (x < g ? r + 1 : r) < others[x];
                forward(by);
                const int list = cur.list;
                const bool more = cur.next(work, lists);
                if (!more || cur.list != list) {                  // the list or the stretch ends: join the lanes, two channels each
                    float M = m;
#pragma unroll
                    for (int d = 16; d; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
                    const float w = m == -INFINITY ? (l == 0.f ? 0.f : l) : ex2_approx(m - M);      // (l NaN without a maximum: keep it)
                    l = warp_sum(l == 0.f ? 0.f : l * w);
#pragma unroll
                    for (int i = 0; i < 64; ++i) o[i] *= w;
#pragma unroll
                    for (int d = 16, c = 32; d; d >>= 1, c >>= 1) {
                        const bool up = lane & d;
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            if (i < c) {
                                const float send = up ? o[i] : o[i + c], keep = up ? o[i + c] : o[i];
                                o[i] = keep + __shfl_xor_sync(0xffffffffu, send, d);
                            }
                        }
                    }
                    const size_t at = ((((size_t)(list + me)) * 4 + quarter) * a.n + j) * a.H + h;
                    *reinterpret_cast<float2*>(a.po + at * BR_HD + 2 * lane) = make_float2(o[0], o[1]);
                    if (lane == 0) a.ml[at] = make_float2(M, l);
                    fresh = true;
                }
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (warp == WARP_MMA) tmem_dealloc(tmem, 512);
    if (tid == 0 && *abort_flag) atomicOr(br.status, *abort_flag);
}

template <int ATOMS, int IG, bool SILU>
static int launch(const BranchArgs& a, const BranchRows& p, cudaStream_t st) {
    static std::atomic<unsigned long long> done{0};
    MBEMA_CUDA_TRY(allow_smem(k_branch_rows<ATOMS, IG, SILU>, Smem<ATOMS>::BYTES, done));
    MBEMA_CUDA_TRY(launch_early(k_branch_rows<ATOMS, IG, SILU>, dim3((unsigned)p.ctas, (unsigned)a.H, (unsigned)p.zb), THREADS, Smem<ATOMS>::BYTES, st, a, p.JW));
    return check_launch();
}

template <int ATOMS>
static int launch_silu(const BranchArgs& a, const BranchRows& p, cudaStream_t st) {
    if (p.IG == 1) return a.silu ? launch<ATOMS, 1, true>(a, p, st) : launch<ATOMS, 1, false>(a, p, st);
    return a.silu ? launch<ATOMS, 3, true>(a, p, st) : launch<ATOMS, 3, false>(a, p, st);
}

}  // namespace brows

// One step: three workers a CTA.  More: up to three steps a worker, whichever leaves the fewest groups idle.
BranchRows branch_rows(int64_t n, int64_t H) {
    BranchRows p;
    p.JW = n == 1 ? 1 : n == 2 || n == 4 ? 2 : 3;
    p.IG = p.JW == 1 ? 3 : 1;
    p.zb = (int)((n + p.JW - 1) / p.JW);
    p.ctas = (int)std::max<int64_t>(1, 148 / (H * p.zb));
    return p;
}

int launch_branch_rows(const BranchArgs& a, const BranchRows& p, cudaStream_t st) {
    return a.br.N == 64 ? brows::launch_silu<1>(a, p, st) : brows::launch_silu<2>(a, p, st);
}

}  // namespace mbema
