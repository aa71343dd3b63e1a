// Attention of the rows of a decode state's branches on the tensor cores (mbema_branches_attend, MBEMA_MODE_TC_BF16).
//
// The states that the rows of one call see differ from the ones at the call's first step by rho^j alone, so the operand copies
// (fp16, made once by mbema_branches_extend for all layers and steps) are the A operands of every step and rho^j goes into W:
//     gate(j) = SiLU(A . (rho^j * W)),   16 slots x 64 channels of a head to a warp (mma.sync m16n8k16, fp32 accumulators).
// A warp keeps its step's W in registers and its accumulators in the layout that the next operand needs: a thread holds the same
// 16 channels of slots g and g + 8 in the gate, in the 16-byte pieces that it loads of the E rows, and in q and O.  So nothing goes
// through shared memory, a warp is a worker of its own with its own jobs, and the E rows that one warp fetches are in L1 for the
// warps of the other steps, which take the same job.
#include <algorithm>

#include "branches.cuh"

namespace mbema {

static constexpr int BT_WARPS = 8;
static constexpr int BT_THREADS = BT_WARPS * 32;
static constexpr int BT_LDW = 70;                 // floats a row of the staged W slice, which starts up to 6 floats in (w_row)
static constexpr float BT_W_SCALE = 64.0f;        // undoes BR_OP_SCALE

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_bf2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float bf_lo(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float bf_hi(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }
__device__ __forceinline__ float tanh_fast(float x) {
    float r;
    asm("tanh.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {      // lane (g, t): element pair (g, 2t..) -> pair (2t.., g)
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// Channel maps.  Lane = 4 g + t.  Gate column (tile nt, thread t, e) is channel 32 (nt / 4) + 8 t + 2 (nt % 4) + e of the head, and
// contraction place (step ks, thread t, pair p, e) is state channel 32 (ks / 2) + 8 t + 4 (ks % 2) + 2 p + e: 16 bytes of a row each.
// Rows 8, 16 and 24 behind one another start two banks apart: a fragment's lanes read four of them, 8 channels apart.
__device__ __forceinline__ int w_row(int c) { return c * BT_LDW + 2 * ((c >> 3) & 3); }

template <int KS>
__device__ __forceinline__ void w_fragment(uint32_t (&w)[2], const float* W_sh, const float* pw, int ks, int nt, int g, int t) {
    const int c = 32 * (ks >> 1) + 8 * t + 4 * (ks & 1);
    const int d = 32 * (nt >> 2) + 8 * (g >> 1) + 2 * (nt & 3) + (g & 1);
    const float* p = W_sh + w_row(c) + d;              // c .. c + 3 lie in one group of eight
    w[0] = pack_h2(p[0] * pw[0], p[BT_LDW] * pw[1]);
    w[1] = pack_h2(p[2 * BT_LDW] * pw[2], p[3 * BT_LDW] * pw[3]);
}

// The gate product's W: in registers for 64 channels (64 of them a thread), in shared memory for 128.
template <int KS>
struct WSource {
    uint32_t w[KS == 4 ? 4 : 1][8][2];
    const uint2* sh;
    __device__ __forceinline__ void build(const float* W_sh, const float* l2r, uint2* dst, int j, float scale, int lane) {
        const int g = lane >> 2, t = lane & 3;
        sh = dst + lane;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int c = 32 * (ks >> 1) + 8 * t + 4 * (ks & 1);
            float pw[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) pw[i] = exp2f((float)j * l2r[c + i]) * scale;
#pragma unroll
            for (int nt = 0; nt < 8; ++nt) {
                if constexpr (KS == 4) {
                    w_fragment<KS>(w[ks][nt], W_sh, pw, ks, nt, g, t);
                } else {
                    uint32_t x[2];
                    w_fragment<KS>(x, W_sh, pw, ks, nt, g, t);
                    dst[(ks * 8 + nt) * 32 + lane] = make_uint2(x[0], x[1]);
                }
            }
        }
    }
    __device__ __forceinline__ void gate(float (&acc)[8][4], const uint32_t (&A)[KS][4]) const {
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int nt = 0; nt < 8; ++nt) {
                if constexpr (KS == 4) {
                    mma_f16(acc[nt], A[ks], w[ks][nt][0], w[ks][nt][1]);
                } else {
                    const uint2 x = sh[(ks * 8 + nt) * 32];
                    mma_f16(acc[nt], A[ks], x.x, x.y);
                }
            }
    }
};

// rows g and g + 8 of 16 operand rows, from this thread's first channel on
template <int KS>
__device__ __forceinline__ void load_A(uint32_t (&A)[KS][4], const __half* r0, const __half* r1) {
#pragma unroll
    for (int i = 0; i < KS / 2; ++i) {
        const uint4 x = *reinterpret_cast<const uint4*>(r0 + 32 * i);
        const uint4 y = *reinterpret_cast<const uint4*>(r1 + 32 * i);
        A[2 * i][0] = x.x; A[2 * i][2] = x.y; A[2 * i + 1][0] = x.z; A[2 * i + 1][2] = x.w;
        A[2 * i][1] = y.x; A[2 * i][3] = y.y; A[2 * i + 1][1] = y.z; A[2 * i + 1][3] = y.w;
    }
}

__device__ __forceinline__ void load_E(uint32_t (&E)[8], const char* row) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint4 x = *reinterpret_cast<const uint4*>(row + 64 * i);
        E[4 * i] = x.x; E[4 * i + 1] = x.y; E[4 * i + 2] = x.z; E[4 * i + 3] = x.w;
    }
}

// products of the halves, exact in fp32 (mixed-precision FMA: no unpacking)
__device__ __forceinline__ void mul_bf16x2(float& x, float& y, uint32_t a, uint32_t b) {
    asm("{\n\t.reg .b16 al, ah, bl, bh;\n\t"
        "mov.b32 {al, ah}, %2;\n\t"
        "mov.b32 {bl, bh}, %3;\n\t"
        "fma.rn.f32.bf16 %0, al, bl, 0f00000000;\n\t"
        "fma.rn.f32.bf16 %1, ah, bh, 0f00000000;\n\t}"
        : "=f"(x), "=f"(y) : "r"(a), "r"(b));
}

__device__ __forceinline__ void apply_gate(float (&acc)[8][4], int silu) {
    if (silu) {              // W carries 1/2: SiLU(x) = h + h tanh(h), h = x / 2
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[nt][e] = fmaf(acc[nt][e], tanh_fast(acc[nt][e]), acc[nt][e]);
    }
}

struct Job {
    const int* slots;         // slot ids of the list
    const __half* op;         // operand rows of the list
    int64_t r0;               // first branch
    int rows;                 // branches
    int lo, hi;               // slots of this job
    int part;                 // place of its partials
    bool own;
};

// chunk-major: lists shorter than their capacity leave empty jobs at the end, not between others
__device__ __forceinline__ bool find_job(Job& job, const BranchArgs& a, int64_t x, int rows_a_job) {
    const mbema_branches& br = a.br;
    const int blocks = (int)((br.S + rows_a_job - 1) / rows_a_job);
    const int64_t pre = br.B * blocks, n_pre = pre * a.plan.SP;
    job.own = x >= n_pre;
    if (!job.own) {
        const int chunk = (int)(x / pre);
        const int bb = (int)(x - chunk * pre);
        const int b = bb / blocks, s0 = (bb - b * blocks) * rows_a_job;
        job.slots = br.active + (size_t)b * br.Kcap;
        job.op = reinterpret_cast<const __half*>(br.pre_op) + (size_t)b * br.Kcap * br.N;
        job.r0 = (int64_t)b * br.S + s0;
        job.rows = min(rows_a_job, (int)br.S - s0);
        job.lo = chunk * a.plan.chp;
        job.hi = min(job.lo + a.plan.chp, min(br.n_active[b], (int)br.Kcap));
        job.part = chunk;
    } else {
        const int64_t y = x - n_pre, all = br.B * br.S;
        const int chunk = (int)(y / all);
        const int64_t r = y - chunk * all;
        job.slots = br.own_slot + (size_t)r * br.cap;
        job.op = reinterpret_cast<const __half*>(br.own_op) + (size_t)r * br.cap * br.N;
        job.r0 = r;
        job.rows = 1;
        job.lo = chunk * a.plan.cho;
        job.hi = min(job.lo + a.plan.cho, br.own_n[r]);
        job.part = a.plan.SP + chunk;
    }
    return job.lo < job.hi;
}

// bit i: slot k0 + i (i < 16) is hidden from row (r, j); staged: lane i holds the list place that staged token i < j hides, or -1
__device__ __forceinline__ unsigned hidden16(const BranchArgs& a, const Job& job, int64_t r, int k0, int staged, bool any_staged) {
    unsigned m = 0u;
    if (!job.own) {
        const int words = (int)((a.br.Kcap + 31) / 32);
        m = (a.br.touched[(size_t)r * words + (k0 >> 5)] >> (k0 & 31)) & 0xffffu;
    }
    if (any_staged) {
        const unsigned d = (unsigned)(staged - k0);
        m |= __reduce_or_sync(0xffffffffu, d < 16u ? 1u << d : 0u);
    }
    return m;
}

// One partial of a warp: the eight quads' (m, l, o[16]) joined.  A lane is left with o of channels 32 (x / 4) + 8 t + 2 (x % 4) + {0, 1},
// x = g with its bits reversed in place: see quad_columns.
__device__ __forceinline__ void join_quads(float& m, float& l, float (&o)[16], float2& out) {
    float M = m;
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
    const float w = M == -INFINITY ? 0.f : exp2f(m - M);
    l *= w;
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] *= w;
    const bool b0 = lane & 4, b1 = lane & 8, b2 = lane & 16;
    float x[8], y[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {          // keep the half that bit 0 of g names
        const float send = b0 ? o[i] : o[8 + i], keep = b0 ? o[8 + i] : o[i];
        x[i] = keep + __shfl_xor_sync(0xffffffffu, send, 4);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float send = b1 ? x[i] : x[4 + i], keep = b1 ? x[4 + i] : x[i];
        y[i] = keep + __shfl_xor_sync(0xffffffffu, send, 8);
    }
    const float s0 = b2 ? y[0] : y[2], s1 = b2 ? y[1] : y[3], k0 = b2 ? y[2] : y[0], k1 = b2 ? y[3] : y[1];
    out.x = k0 + __shfl_xor_sync(0xffffffffu, s0, 16);
    out.y = k1 + __shfl_xor_sync(0xffffffffu, s1, 16);
    m = M;
}
// first of the two head channels that join_quads leaves in this lane
__device__ __forceinline__ int quad_columns(int lane) {
    const int t = lane & 3, i = ((lane >> 2) & 1) * 8 + ((lane >> 3) & 1) * 4 + ((lane >> 4) & 1) * 2;    // index into o[16]
    return 32 * (i >> 3) + 8 * t + (i & 7);
}

// ---------------------------------------------------------------------------------------------------------------------------
// One or two branches at a time: q.K and P.V on the CUDA cores, in fp32, straight from the gate's accumulators.
// ---------------------------------------------------------------------------------------------------------------------------
template <int KS>
__device__ __forceinline__ void fma_job(const BranchArgs& a, const Job& job, const WSource<KS>& W, int j, int h, float& m, float& l,
                                        float (&o)[16]) {
    const mbema_branches& br = a.br;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t D2 = (uint32_t)a.H * BR_HD * 2;
    const char* Ek = reinterpret_cast<const char*>(a.Ek) + h * (BR_HD * 2) + 16 * t;
    const char* Ev = reinterpret_cast<const char*>(a.Ev) + h * (BR_HD * 2) + 16 * t;
    uint32_t q[8];
    load_E(q, reinterpret_cast<const char*>(a.q) + (((size_t)job.r0 * a.n + j) * a.H + h) * (BR_HD * 2) + 16 * t);
    int staged = -1;
    if (lane < j) staged = (job.own ? br.st_own : br.st_pos)[br_index(br, job.r0, lane)];
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = 0.f;
    const int last = job.hi - 1;
    const __half* op = job.op + 8 * t;
    // every load is for the unit behind: the operand rows follow the gate product that reads the registers, E_k the scores, E_v P.V
    uint32_t A[KS][4], ek0[8], ek1[8], ev0[8], ev1[8];
    int u0 = min(job.lo + g, last), u1 = min(job.lo + g + 8, last);
    int v0 = job.slots[u0], v1 = job.slots[u1];
    load_A<KS>(A, op + (size_t)u0 * br.N, op + (size_t)u1 * br.N);
    load_E(ek0, Ek + (uint64_t)v0 * D2);
    load_E(ek1, Ek + (uint64_t)v1 * D2);
    load_E(ev0, Ev + (uint64_t)v0 * D2);
    load_E(ev1, Ev + (uint64_t)v1 * D2);
    u0 = min(job.lo + 16 + g, last);
    u1 = min(job.lo + 24 + g, last);
    v0 = job.slots[u0];
    v1 = job.slots[u1];
    for (int k0 = job.lo; k0 < job.hi; k0 += 16) {
        float acc[8][4];
        W.gate(acc, A);
        load_A<KS>(A, op + (size_t)u0 * br.N, op + (size_t)u1 * br.N);
        apply_gate(acc, a.silu);
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) {
            float x = 0.f, y = 0.f;
            mul_bf16x2(x, y, ek0[nt], q[nt]);
            s0 = fmaf(x, acc[nt][0], fmaf(y, acc[nt][1], s0));
            mul_bf16x2(x, y, ek1[nt], q[nt]);
            s1 = fmaf(x, acc[nt][2], fmaf(y, acc[nt][3], s1));
        }
        load_E(ek0, Ek + (uint64_t)v0 * D2);
        load_E(ek1, Ek + (uint64_t)v1 * D2);
        unsigned hide = hidden16(a, job, job.r0, k0, staged, j > 0);
        if (job.hi - k0 < 16) hide |= 0xffffffffu << (job.hi - k0);
        s0 += __shfl_xor_sync(0xffffffffu, s0, 1);
        s1 += __shfl_xor_sync(0xffffffffu, s1, 1);
        s0 += __shfl_xor_sync(0xffffffffu, s0, 2);
        s1 += __shfl_xor_sync(0xffffffffu, s1, 2);
        const float x0 = (hide >> g) & 1u ? -INFINITY : s0 * BR_SCORE_LOG2, x1 = (hide >> (g + 8)) & 1u ? -INFINITY : s1 * BR_SCORE_LOG2;
        const float m_new = fmaxf(m, fmaxf(x0, x1));
        const float ref = m_new == -INFINITY ? 0.f : m_new;
        const float p0 = exp2f(x0 - ref), p1 = exp2f(x1 - ref);
        if (__any_sync(0xffffffffu, m_new > m)) {
            const float alpha = exp2f(m - ref);
            l *= alpha;
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] *= alpha;
        }
        m = m_new;
        l += p0 + p1;
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) {      // (a value that is not finite stays in a row that hides it: the same slot is listed as the branch's own)
            o[2 * nt] = fmaf(p0 * acc[nt][0], bf_lo(ev0[nt]), fmaf(p1 * acc[nt][2], bf_lo(ev1[nt]), o[2 * nt]));
            o[2 * nt + 1] = fmaf(p0 * acc[nt][1], bf_hi(ev0[nt]), fmaf(p1 * acc[nt][3], bf_hi(ev1[nt]), o[2 * nt + 1]));
        }
        load_E(ev0, Ev + (uint64_t)v0 * D2);
        load_E(ev1, Ev + (uint64_t)v1 * D2);
        u0 = min(u0 + 16, last);
        u1 = min(u1 + 16, last);
        v0 = job.slots[u0];
        v1 = job.slots[u1];
    }
}

// ---------------------------------------------------------------------------------------------------------------------------
// Sixteen branches at a time: q.K and P.V as products too.  K goes in as two bf16 terms (its rounding would come back
// through the exponent as an error of the score's size), V and P as one.  V's 8 x 8 blocks are transposed in registers.
// ---------------------------------------------------------------------------------------------------------------------------
static constexpr int BT_ROWS = 16;

template <int KS>
__device__ __forceinline__ void mma_job(const BranchArgs& a, const Job& job, const WSource<KS>& W, int j, int h, float (&m)[2],
                                        float (&l)[2], float (&o)[8][4]) {
    const mbema_branches& br = a.br;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t D2 = (uint32_t)a.H * BR_HD * 2;
    const char* Ek = reinterpret_cast<const char*>(a.Ek) + h * (BR_HD * 2) + 16 * t;
    const char* Ev = reinterpret_cast<const char*>(a.Ev) + h * (BR_HD * 2) + 16 * t;
    const int64_t row0 = job.r0 + min(g, job.rows - 1), row1 = job.r0 + min(g + 8, job.rows - 1);
    uint32_t q0[8], q1[8];
    load_E(q0, reinterpret_cast<const char*>(a.q) + (((size_t)row0 * a.n + j) * a.H + h) * (BR_HD * 2) + 16 * t);
    load_E(q1, reinterpret_cast<const char*>(a.q) + (((size_t)row1 * a.n + j) * a.H + h) * (BR_HD * 2) + 16 * t);
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) o[nt][0] = o[nt][1] = o[nt][2] = o[nt][3] = 0.f;
    const int words = (int)((br.Kcap + 31) / 32);
    const uint32_t* hid0 = br.touched + (size_t)row0 * words;
    const uint32_t* hid1 = br.touched + (size_t)row1 * words;
    const int last = job.hi - 1;
    const __half* op = job.op + 8 * t;
    uint32_t A[KS][4], ek0[8], ek1[8], ev0[8], ev1[8];                // loads run a unit ahead, as in fma_job
    int u0 = min(job.lo + g, last), u1 = min(job.lo + g + 8, last);
    int v0 = job.slots[u0], v1 = job.slots[u1];
    load_A<KS>(A, op + (size_t)u0 * br.N, op + (size_t)u1 * br.N);
    load_E(ek0, Ek + (uint64_t)v0 * D2);
    load_E(ek1, Ek + (uint64_t)v1 * D2);
    load_E(ev0, Ev + (uint64_t)v0 * D2);
    load_E(ev1, Ev + (uint64_t)v1 * D2);
    u0 = min(job.lo + 16 + g, last);
    u1 = min(job.lo + 24 + g, last);
    v0 = job.slots[u0];
    v1 = job.slots[u1];
    for (int k0 = job.lo; k0 < job.hi; k0 += 16) {
        float acc[8][4];
        W.gate(acc, A);
        load_A<KS>(A, op + (size_t)u0 * br.N, op + (size_t)u1 * br.N);
        unsigned hide0 = (hid0[k0 >> 5] >> (k0 & 31)) & 0xffffu, hide1 = (hid1[k0 >> 5] >> (k0 & 31)) & 0xffffu;
        apply_gate(acc, a.silu);
        float sc[2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[0][i] = sc[1][i] = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint32_t Q[4] = {q0[2 * c], q1[2 * c], q0[2 * c + 1], q1[2 * c + 1]};
            uint32_t hi[2][2], lo[2][2];                        // [slots 0-7, 8-15][channel pair]
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int nt = 2 * c + p;
                const float x0 = bf_lo(ek0[nt]) * acc[nt][0], x1 = bf_hi(ek0[nt]) * acc[nt][1];
                const float y0 = bf_lo(ek1[nt]) * acc[nt][2], y1 = bf_hi(ek1[nt]) * acc[nt][3];
                hi[0][p] = pack_bf2(x0, x1);
                hi[1][p] = pack_bf2(y0, y1);
                lo[0][p] = pack_bf2(x0 - bf_lo(hi[0][p]), x1 - bf_hi(hi[0][p]));
                lo[1][p] = pack_bf2(y0 - bf_lo(hi[1][p]), y1 - bf_hi(hi[1][p]));
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                mma_bf16(sc[x], Q, hi[x][0], hi[x][1]);
                mma_bf16(sc[x], Q, lo[x][0], lo[x][1]);
            }
        }
        load_E(ek0, Ek + (uint64_t)v0 * D2);
        load_E(ek1, Ek + (uint64_t)v1 * D2);
        if (j > 0) {
            unsigned x = 0u, y = 0u;
            for (int i = t; i < j; i += 4) {
                const unsigned d0 = (unsigned)(br.st_pos[br_index(br, row0, i)] - k0), d1 = (unsigned)(br.st_pos[br_index(br, row1, i)] - k0);
                if (d0 < 16u) x |= 1u << d0;
                if (d1 < 16u) y |= 1u << d1;
            }
            x |= __shfl_xor_sync(0xffffffffu, x, 1);
            y |= __shfl_xor_sync(0xffffffffu, y, 1);
            hide0 |= x | __shfl_xor_sync(0xffffffffu, x, 2);
            hide1 |= y | __shfl_xor_sync(0xffffffffu, y, 2);
        }
        if (job.hi - k0 < 16) {
            const unsigned past = 0xffffffffu << (job.hi - k0);
            hide0 |= past;
            hide1 |= past;
        }
        uint32_t P[4];
        bool moved = false;
        float alpha[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {                           // rows g, g + 8
            const unsigned hide = (r ? hide1 : hide0) >> (2 * t);
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = (hide >> ((i >> 1) * 8 + (i & 1))) & 1u ? -INFINITY : sc[i >> 1][2 * r + (i & 1)] * BR_SCORE_LOG2;
            float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float m_new = fmaxf(m[r], mx);
            const float ref = m_new == -INFINITY ? 0.f : m_new;
            moved |= m_new > m[r];
            alpha[r] = exp2f(m[r] - ref);
            m[r] = m_new;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = exp2f(x[i] - ref);
            l[r] = l[r] * alpha[r] + ((x[0] + x[1]) + (x[2] + x[3]));
            P[r] = pack_bf2(x[0], x[1]);
            P[2 + r] = pack_bf2(x[2], x[3]);
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int nt = 0; nt < 8; ++nt) {
                o[nt][0] *= alpha[0];
                o[nt][1] *= alpha[0];
                o[nt][2] *= alpha[1];
                o[nt][3] *= alpha[1];
            }
        }
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) {
            const uint32_t b0 = transpose8x8(pack_bf2(bf_lo(ev0[nt]) * acc[nt][0], bf_hi(ev0[nt]) * acc[nt][1]));
            const uint32_t b1 = transpose8x8(pack_bf2(bf_lo(ev1[nt]) * acc[nt][2], bf_hi(ev1[nt]) * acc[nt][3]));
            mma_bf16(o[nt], P, b0, b1);
        }
        load_E(ev0, Ev + (uint64_t)v0 * D2);
        load_E(ev1, Ev + (uint64_t)v1 * D2);
        u0 = min(u0 + 16, last);
        u1 = min(u1 + 16, last);
        v0 = job.slots[u0];
        v1 = job.slots[u1];
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
}

// grid: x = CTAs that share the jobs, y = head, z = block of JW steps.  Warp w takes step z JW + w % JW; the IG warps of a step
// take jobs of their own.  ROWS: branches that a job of a prefix takes (1: fma_job, 16: mma_job).
template <int KS, int ROWS>
__global__ void __launch_bounds__(BT_THREADS, 1) k_branch_tc(BranchArgs a, int JW, int IG) {
    extern __shared__ __align__(16) float smem[];
    __shared__ float s_l2r[16 * KS];
    const mbema_branches& br = a.br;
    constexpr int N = 16 * KS;
    const int h = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int D = a.H * BR_HD;
    float* W_sh = smem;                                                     // [N] rows at w_row
    uint2* Wf = reinterpret_cast<uint2*>(smem + (N * BT_LDW + 8));          // KS = 8: [JW][KS * 8 * 32]
    for (int i = tid; i < N * 16; i += BT_THREADS) {
        const float4 x = *reinterpret_cast<const float4*>(a.W + (size_t)(i >> 4) * D + h * BR_HD + (i & 15) * 4);
        float2* dst = reinterpret_cast<float2*>(W_sh + w_row(i >> 4) + (i & 15) * 4);
        dst[0] = make_float2(x.x, x.y);
        dst[1] = make_float2(x.z, x.w);
    }
    for (int i = tid; i < N; i += BT_THREADS) s_l2r[i] = log2f(br.rhos[i]);
    __syncthreads();
    const int jj = warp % JW, ig = warp / JW;
    const int j = blockIdx.z * JW + jj;
    if (ig >= IG || j >= a.n) return;
    WSource<KS> W;                 // KS = 8: the IG warps of a step write the same fragments, each reads what it has written
    W.build(W_sh, s_l2r, Wf + (size_t)jj * KS * 8 * 32, j, a.silu ? 0.5f * BT_W_SCALE : BT_W_SCALE, lane);
    const int blocks = (int)((br.S + ROWS - 1) / ROWS);
    const int64_t jobs = br.B * blocks * a.plan.SP + br.B * br.S * a.plan.SO;
    const int parts = a.plan.SP + a.plan.SO;
    for (int64_t x = (int64_t)blockIdx.x * IG + ig; x < jobs; x += (int64_t)gridDim.x * IG) {
        Job job;
        if (!find_job(job, a, x, ROWS)) continue;
        if (ROWS == 1 || job.own) {
            float m, l, o[16];
            fma_job<KS>(a, job, W, j, h, m, l, o);
            float2 out;
            join_quads(m, l, o, out);
            const size_t at = (((size_t)job.r0 * a.n + j) * a.H + h) * parts + job.part;
            *reinterpret_cast<float2*>(a.po + at * BR_HD + quad_columns(lane)) = out;
            if (lane == 0) a.ml[at] = make_float2(m, l);
        } else if constexpr (ROWS > 1) {
            float m[2], l[2], o[8][4];
            mma_job<KS>(a, job, W, j, h, m, l, o);
            const int g = lane >> 2, t = lane & 3;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = g + 8 * r;
                if (row < job.rows) {
                    const size_t at = (((size_t)(job.r0 + row) * a.n + j) * a.H + h) * parts + job.part;
                    float* dst = a.po + at * BR_HD + 8 * t;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<float4*>(dst + 32 * (i >> 1) + 4 * (i & 1)) =
                            make_float4(o[2 * i][2 * r], o[2 * i][2 * r + 1], o[2 * i + 1][2 * r], o[2 * i + 1][2 * r + 1]);
                    if (t == 0) a.ml[at] = make_float2(m[r], l[r]);
                }
            }
        }
    }
}

bool branch_tc_supported(int64_t N) { return N == 64 || N == 128; }

static void steps_and_shares(int n, int& JW, int& IG) {
    JW = std::min(n, BT_WARPS);
    IG = BT_WARPS / JW;
}

// One CTA an SM (the registers allow no more), dealt to the heads and blocks of steps.
static int64_t ctas_a_head(int64_t H, int64_t zb) { return std::max<int64_t>(1, 148 / (H * zb)); }

// Chunks: about four jobs a worker if all lists were full, of 2 to 32 units of 16 slots (a job costs about one unit more than its
// units: q, the joining of the quads, the partial).
BranchPlan branch_plan_tc(int64_t B, int64_t S, int64_t n, int64_t H, int64_t Kcap, int64_t cap) {
    int JW, IG;
    steps_and_shares((int)n, JW, IG);
    const int64_t zb = (n + JW - 1) / JW, workers = ctas_a_head(H, zb) * IG;
    const int64_t lists = S == 1 ? B : B * ((S + BT_ROWS - 1) / BT_ROWS);
    const int64_t units = lists * ((Kcap + 15) / 16) + B * S * ((cap + 15) / 16);
    const int64_t chunk = 16 * std::min<int64_t>(32, std::max<int64_t>(2, units / (4 * workers)));
    BranchPlan p;
    p.chp = p.cho = (int)chunk;
    p.SP = (int)((Kcap + chunk - 1) / chunk);
    p.SO = (int)((cap + chunk - 1) / chunk);
    return p;
}

template <int KS, int ROWS>
static int launch_tc(const BranchArgs& a, cudaStream_t st) {
    int JW, IG;
    steps_and_shares(a.n, JW, IG);
    const mbema_branches& br = a.br;
    const int zb = (a.n + JW - 1) / JW;
    const int64_t jobs = br.B * ((br.S + ROWS - 1) / ROWS) * a.plan.SP + br.B * br.S * a.plan.SO;
    const int64_t x = std::min((jobs + IG - 1) / IG, ctas_a_head(a.H, zb));
    const size_t smem = ((size_t)16 * KS * BT_LDW + 8) * 4 + (KS == 8 ? (size_t)JW * KS * 8 * 32 * sizeof(uint2) : 0);
    MBEMA_CUDA_TRY(cudaFuncSetAttribute(k_branch_tc<KS, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    k_branch_tc<KS, ROWS><<<dim3((unsigned)x, (unsigned)a.H, (unsigned)zb), BT_THREADS, smem, st>>>(a, JW, IG);
    return check_launch();
}

int launch_branch_attend_tc(const BranchArgs& a, cudaStream_t st) {
    const bool one = a.br.S == 1;
    if (a.H > 65535) return MBEMA_ERR_UNSUPPORTED;
    if (a.br.N == 64) return one ? launch_tc<4, 1>(a, st) : launch_tc<4, BT_ROWS>(a, st);
    return one ? launch_tc<8, 1>(a, st) : launch_tc<8, BT_ROWS>(a, st);
}

}  // namespace mbema
