// Attention of branches that share prefixes, on the tensor cores (mbema_branches_attend, MBEMA_MODE_TC_BF16, more than one branch a
// sequence; a single branch: branch_rows_tc.cu).
//
// The states that the rows of one call see differ from the ones at the call's first step by rho^j alone, so the operand copies
// (fp16, made once by mbema_branches_extend for all layers and steps) are the A operands of every step and rho^j goes into W:
//     gate(j) = SiLU(A . (rho^j * W)),   16 slots x 64 channels of a head to a warp (mma.sync m16n8k16, fp32 accumulators).
// A warp keeps its step's W in registers and its accumulators in the layout that the next operand needs: a thread holds the same
// 16 channels of slots g and g + 8 in the gate, in the 16-byte pieces that it reads of the E rows, and in q and O.
// A prefix is walked for sixteen branches at a time (q.K and P.V as products too), a branch's own slots for its row alone.
//
// Work is dealt in units of 16 slots: mbema_branches_extend leaves the running sum of all lists' units, every worker (one warp, or
// the warps of several steps together) takes an equal stretch of it and walks it without a stop; a list is cut where a stretch
// ends, and each piece leaves a partial (m, l, o[64]) a row.  The operand and E rows of a unit come by cp.async into a ring of
// shared memory, some units ahead across the ends of lists: they are gathered rows that mostly come from DRAM, and with them loaded
// a unit ahead into registers half of all cycles were spent waiting.
// Own slots go through tcgen05 in branch_rows_tc.cu's tiles of 128 slots too, but not faster: with its two gathering warps and a list's start
// and end (own lists are short) 4 x 16 branches of 400 own slots took half as long again, 64 branches of 180 a quarter.
// 64 branches of 180 own slots behind a prefix of 3400, 8 heads, 64 channels: 24 us with 11 units a warp, of which 5 us until the first
// unit is there, 3 for the ends of lists and 13 for the units' arithmetic (690 instructions each, 37 % of the issue slots: two warps a
// scheduler, as W and the accumulators leave registers for).
#include <algorithm>

#include "branches.cuh"

namespace mbema {

static constexpr int WARPS = 8;                   // of 255 registers: W (64), accumulators (32), sixteen rows' o (32) and q (16), E rows
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
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }
template <int OFFSET>
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4 + %5];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr), "n"(OFFSET));
    return v;
}
__device__ __forceinline__ void mma_f16_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
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

// The gate product's W, as fragments in shared memory: [KS][4 pairs of column tiles][32 lanes] of 16 bytes.
template <int KS>
__device__ __forceinline__ void build_W(uint32_t dst, const float* W_sh, const float* l2r, int j, float scale, int lane, int part, int parts) {
    const int g = lane >> 2, t = lane & 3;
    for (int i = part; i < KS * 4; i += parts) {
        const int ks = i >> 2, c = 32 * (ks >> 1) + 8 * t + 4 * (ks & 1);
        float pw[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) pw[e] = exp2f((float)j * l2r[c + e]) * scale;
        uint32_t x[2], y[2];
        w_fragment<KS>(x, W_sh, pw, ks, 2 * (i & 3), g, t);
        w_fragment<KS>(y, W_sh, pw, ks, 2 * (i & 3) + 1, g, t);
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst + i * 512 + lane * 16), "r"(x[0]), "r"(x[1]), "r"(y[0]), "r"(y[1]) : "memory");
    }
}
// A warp's copy of them in registers (64 a thread for 64 channels; 128 channels have no room for it): in shared memory, with twelve warps,
// 64 samples of a long prompt took 31 us for 25.
template <int KS, int I = 0>
__device__ __forceinline__ void read_W(uint4 (&w)[KS * 4], uint32_t at) {
    if constexpr (I < KS * 4) {
        w[I] = lds128<512 * I>(at);
        read_W<KS, I + 1>(w, at);
    }
}
template <int KS>
__device__ __forceinline__ void gate(float (&acc)[8][4], const uint32_t (&A)[KS][4], const uint4 (&w)[KS * 4]) {
#pragma unroll
    for (int i = 0; i < KS * 4; ++i) {
        const int ks = i / 4, nt = 2 * (i % 4);
        if (ks == 0) {
            mma_f16_first(acc[nt], A[ks], w[i].x, w[i].y);
            mma_f16_first(acc[nt + 1], A[ks], w[i].z, w[i].w);
        } else {
            mma_f16(acc[nt], A[ks], w[i].x, w[i].y);
            mma_f16(acc[nt + 1], A[ks], w[i].z, w[i].w);
        }
    }
}
template <int KS, int I = 0>
__device__ __forceinline__ void gate(float (&acc)[8][4], const uint32_t (&A)[KS][4], uint32_t w) {
    if constexpr (I < KS * 4) {
        constexpr int ks = I / 4, nt = 2 * (I % 4);
        const uint4 b = lds128<512 * I>(w);
        if (ks == 0) {
            mma_f16_first(acc[nt], A[ks], b.x, b.y);
            mma_f16_first(acc[nt + 1], A[ks], b.z, b.w);
        } else {
            mma_f16(acc[nt], A[ks], b.x, b.y);
            mma_f16(acc[nt + 1], A[ks], b.z, b.w);
        }
        gate<KS, I + 1>(acc, A, w);
    }
}

// A unit in the ring: 16 rows of E_k, of E_v (128 bytes each; in odd rows the 16-byte pieces 0-3 and 4-7 change places, so that the
// eight lanes that are served together, two rows and four pieces each, touch all banks), then the operands as the lanes' fragments.
template <int KS>
struct UnitLayout {
    static constexpr int EV = 2048, OP = 4096, OP_BYTES = 512 * KS;
    static constexpr int BYTES = OP + OP_BYTES;
};

// rows g (at_lo, at_hi: this lane's pieces of channels 0-31 and 32-63) and g + 8, OFFSET bytes into the unit
template <int OFFSET>
__device__ __forceinline__ void load_E(uint32_t (&E0)[8], uint32_t (&E1)[8], uint32_t at_lo, uint32_t at_hi) {
    const uint4 x = lds128<OFFSET>(at_lo), y = lds128<OFFSET>(at_hi), z = lds128<OFFSET + 1024>(at_lo), w = lds128<OFFSET + 1024>(at_hi);
    E0[0] = x.x; E0[1] = x.y; E0[2] = x.z; E0[3] = x.w;
    E0[4] = y.x; E0[5] = y.y; E0[6] = y.z; E0[7] = y.w;
    E1[0] = z.x; E1[1] = z.y; E1[2] = z.z; E1[3] = z.w;
    E1[4] = w.x; E1[5] = w.y; E1[6] = w.z; E1[7] = w.w;
}
template <int KS, int I = 0>
__device__ __forceinline__ void load_A(uint32_t (&A)[KS][4], uint32_t at) {
    if constexpr (I < KS) {
        const uint4 x = lds128<UnitLayout<KS>::OP + 512 * I>(at);
        A[I][0] = x.x; A[I][1] = x.y; A[I][2] = x.z; A[I][3] = x.w;
        load_A<KS, I + 1>(A, at);
    }
}
__device__ __forceinline__ void load_q(uint32_t (&E)[8], const char* row) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint4 x = *reinterpret_cast<const uint4*>(row + 64 * i);
        E[4 * i] = x.x; E[4 * i + 1] = x.y; E[4 * i + 2] = x.z; E[4 * i + 3] = x.w;
    }
}

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
            for (int e = 0; e < 4; e += 2) {
                const uint64_t x = pair2(acc[nt][e], acc[nt][e + 1]);
                unpair2(acc[nt][e], acc[nt][e + 1], fma2(x, pair2(tanh_fast(acc[nt][e]), tanh_fast(acc[nt][e + 1])), x));
            }
    }
}

// A list of slots: the prefix of a sequence as 16 of its branches read it, or a branch's own slots.
struct List {
    const int* slots;
    const char* op;           // operands, 16 slots after 16 slots
    int count;
};

__device__ __forceinline__ List get_list(const BranchArgs& a, int x, int count) {
    const mbema_branches& br = a.br;
    List t;
    t.count = count;
    if (x < a.n_pre) {
        const int b = x / a.blocks;
        t.slots = br.active + (size_t)b * br.Kcap;
        t.op = reinterpret_cast<const char*>(br.pre_op) + (size_t)b * br_operand_bytes(br.Kcap, br.N);
    } else {
        const int r = x - a.n_pre;
        t.slots = br.own_slot + (size_t)r * br.cap;
        t.op = reinterpret_cast<const char*>(br.own_op) + (size_t)r * br_operand_bytes(br.cap, br.N);
    }
    return t;
}

// bit i: own slot k0 + i (i < 16) is hidden; staged: lane i holds the list place that staged token i < j hides, or -1
__device__ __forceinline__ unsigned hidden16(int k0, int staged, bool any_staged, int count) {
    unsigned m = 0u;
    if (any_staged) {
        const unsigned d = (unsigned)(staged - k0);
        m = __reduce_or_sync(0xffffffffu, d < 16u ? 1u << d : 0u);
    }
    if (count - k0 < 16) m |= 0xffffffffu << (count - k0);
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
// One row: q.K and P.V on the CUDA cores, in fp32, straight from the gate's accumulators.  A quad of lanes has its own running
// maximum and sums, joined at the end of the piece.
// ---------------------------------------------------------------------------------------------------------------------------
struct OneRow {
    float m, l, o[16];
    uint32_t q[8];
    int staged;
    __device__ __forceinline__ void start(const BranchArgs& a, int64_t r, int j, int h, int lane) {
        load_q(q, reinterpret_cast<const char*>(a.q) + (((size_t)r * a.n + j) * a.H + h) * (BR_HD * 2) + 16 * (lane & 3));
        staged = -1;
        if (lane < j) staged = a.br.st_own[br_index(a.br, r, lane)];
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = 0.f;
    }
    __device__ __forceinline__ void unit(float (&acc)[8][4], uint32_t at_lo, uint32_t at_hi, unsigned hide, int g) {
        uint32_t e0[8], e1[8];
        load_E<0>(e0, e1, at_lo, at_hi);
        float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) {
            float x, y;                                          // (the product of two bf16 is exact in fp32, and needs no unpacking)
            mul_bf16x2(x, y, e0[nt], q[nt]);
            unpair2(s0, s1, fma2(pair2(x, y), pair2(acc[nt][0], acc[nt][1]), pair2(s0, s1)));
            mul_bf16x2(x, y, e1[nt], q[nt]);
            unpair2(s2, s3, fma2(pair2(x, y), pair2(acc[nt][2], acc[nt][3]), pair2(s2, s3)));
        }
        load_E<2048>(e0, e1, at_lo, at_hi);
        s0 += s1;
        s2 += s3;
        s0 += __shfl_xor_sync(0xffffffffu, s0, 1);
        s2 += __shfl_xor_sync(0xffffffffu, s2, 1);
        s0 += __shfl_xor_sync(0xffffffffu, s0, 2);
        s2 += __shfl_xor_sync(0xffffffffu, s2, 2);
        const float x0 = (hide >> g) & 1u ? -INFINITY : s0 * BR_SCORE_LOG2, x1 = (hide >> (g + 8)) & 1u ? -INFINITY : s2 * BR_SCORE_LOG2;
        const float m_new = fmaxf(m, fmaxf(x0, x1));
        const float ref = m_new == -INFINITY ? 0.f : m_new;
        const float p0 = ex2(x0 - ref), p1 = ex2(x1 - ref);
        if (__any_sync(0xffffffffu, m_new > m)) {
            const float alpha = ex2(m - ref);
            l *= alpha;
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] *= alpha;
        }
        m = m_new;
        l += p0 + p1;
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) {      // (a value that is not finite stays in a row that hides it: the same slot is listed as the branch's own)
            const uint64_t w0 = mul2(pair2(p0, p0), pair2(acc[nt][0], acc[nt][1])), w1 = mul2(pair2(p1, p1), pair2(acc[nt][2], acc[nt][3]));
            const uint64_t x = fma2(w1, pair2(bf_lo(e1[nt]), bf_hi(e1[nt])), pair2(o[2 * nt], o[2 * nt + 1]));
            unpair2(o[2 * nt], o[2 * nt + 1], fma2(w0, pair2(bf_lo(e0[nt]), bf_hi(e0[nt])), x));
        }
    }
    __device__ __forceinline__ void leave(const BranchArgs& a, int64_t piece, int j, int h, int lane) {
        float2 out;
        join_quads(m, l, o, out);
        const size_t at = ((size_t)piece * a.n + j) * a.H + h;
        *reinterpret_cast<float2*>(a.po + at * BR_HD + quad_columns(lane)) = out;
        if (lane == 0) a.ml[at] = make_float2(m, l);
    }
};

// ---------------------------------------------------------------------------------------------------------------------------
// Sixteen branches at a time: q.K and P.V as products too.  K goes in as two bf16 terms (its rounding would come back
// through the exponent as an error of the score's size), V and P as one.  V's 8 x 8 blocks are transposed in registers.
// ---------------------------------------------------------------------------------------------------------------------------
struct SixteenRows {
    float m[2], l[2], o[8][4];
    uint32_t q0[8], q1[8];
    const uint32_t* hid0;
    const uint32_t* hid1;
    int64_t row0, row1;
    __device__ __forceinline__ void start(const BranchArgs& a, int64_t r0, int rows, int j, int h, int lane) {
        const int g = lane >> 2, t = lane & 3;
        row0 = r0 + min(g, rows - 1);
        row1 = r0 + min(g + 8, rows - 1);
        load_q(q0, reinterpret_cast<const char*>(a.q) + (((size_t)row0 * a.n + j) * a.H + h) * (BR_HD * 2) + 16 * t);
        load_q(q1, reinterpret_cast<const char*>(a.q) + (((size_t)row1 * a.n + j) * a.H + h) * (BR_HD * 2) + 16 * t);
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) o[nt][0] = o[nt][1] = o[nt][2] = o[nt][3] = 0.f;
        const int words = (int)((a.br.Kcap + 31) / 32);
        hid0 = a.br.touched + (size_t)row0 * words;
        hid1 = a.br.touched + (size_t)row1 * words;
    }
    __device__ __forceinline__ void unit(const BranchArgs& a, float (&acc)[8][4], uint32_t at_lo, uint32_t at_hi, int k0, int count,
                                         unsigned touched0, unsigned touched1, int j, int t) {
        uint32_t e0[8], e1[8];
        load_E<0>(e0, e1, at_lo, at_hi);
        float sc[2][4], sl[2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[0][i] = sc[1][i] = sl[0][i] = sl[1][i] = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint32_t Q[4] = {q0[2 * c], q1[2 * c], q0[2 * c + 1], q1[2 * c + 1]};
            uint32_t hi[2][2], lo[2][2];                        // [slots 0-7, 8-15][channel pair]
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int nt = 2 * c + p;
                float x0, x1, y0, y1;
                unpair2(x0, x1, mul2(pair2(bf_lo(e0[nt]), bf_hi(e0[nt])), pair2(acc[nt][0], acc[nt][1])));
                unpair2(y0, y1, mul2(pair2(bf_lo(e1[nt]), bf_hi(e1[nt])), pair2(acc[nt][2], acc[nt][3])));
                hi[0][p] = pack_bf2(x0, x1);
                hi[1][p] = pack_bf2(y0, y1);
                lo[0][p] = pack_bf2(x0 - bf_lo(hi[0][p]), x1 - bf_hi(hi[0][p]));
                lo[1][p] = pack_bf2(y0 - bf_lo(hi[1][p]), y1 - bf_hi(hi[1][p]));
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                mma_bf16(sc[x], Q, hi[x][0], hi[x][1]);
                mma_bf16(sl[x], Q, lo[x][0], lo[x][1]);
            }
        }
        load_E<2048>(e0, e1, at_lo, at_hi);
#pragma unroll
        for (int i = 0; i < 4; ++i) {                           // (a product beyond fp32 stays infinite: its second term may have the other sign)
            sc[0][i] = fabsf(sc[0][i]) == INFINITY ? sc[0][i] : sc[0][i] + sl[0][i];
            sc[1][i] = fabsf(sc[1][i]) == INFINITY ? sc[1][i] : sc[1][i] + sl[1][i];
        }
        unsigned hide0 = (touched0 >> (k0 & 31)) & 0xffffu, hide1 = (touched1 >> (k0 & 31)) & 0xffffu;
        if (j > 0) {
            unsigned x = 0u, y = 0u;
            for (int i = t; i < j; i += 4) {
                const unsigned d0 = (unsigned)(a.br.st_pos[br_index(a.br, row0, i)] - k0), d1 = (unsigned)(a.br.st_pos[br_index(a.br, row1, i)] - k0);
                if (d0 < 16u) x |= 1u << d0;
                if (d1 < 16u) y |= 1u << d1;
            }
            x |= __shfl_xor_sync(0xffffffffu, x, 1);
            y |= __shfl_xor_sync(0xffffffffu, y, 1);
            hide0 |= x | __shfl_xor_sync(0xffffffffu, x, 2);
            hide1 |= y | __shfl_xor_sync(0xffffffffu, y, 2);
        }
        if (count - k0 < 16) {
            const unsigned past = 0xffffffffu << (count - k0);
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
            alpha[r] = ex2(m[r] - ref);
            m[r] = m_new;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = ex2(x[i] - ref);
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
            float x0, x1, y0, y1;
            unpair2(x0, x1, mul2(pair2(bf_lo(e0[nt]), bf_hi(e0[nt])), pair2(acc[nt][0], acc[nt][1])));
            unpair2(y0, y1, mul2(pair2(bf_lo(e1[nt]), bf_hi(e1[nt])), pair2(acc[nt][2], acc[nt][3])));
            const uint32_t b0 = transpose8x8(pack_bf2(x0, x1)), b1 = transpose8x8(pack_bf2(y0, y1));
            mma_bf16(o[nt], P, b0, b1);
        }
    }
    __device__ __forceinline__ void leave(const BranchArgs& a, int64_t piece, int rows, int j, int h, int lane) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            const int row = g + 8 * r;
            if (row < rows) {
                const size_t at = (((size_t)piece * BR_BLOCK + row) * a.n + j) * a.H + h;
                float* dst = a.po + at * BR_HD + 8 * t;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<float4*>(dst + 32 * (i >> 1) + 4 * (i & 1)) =
                        make_float4(o[2 * i][2 * r], o[2 * i][2 * r + 1], o[2 * i + 1][2 * r], o[2 * i + 1][2 * r + 1]);
                if (t == 0) a.ml[at] = make_float2(m[r], l[r]);
            }
        }
    }
};

// grid: x = CTAs that share the work, y = head, z = block of JW steps.  The CTA's warps are IG workers of JW warps each; warp w takes
// step z JW + w % JW of worker w / JW.
template <int KS, int STAGES>
__global__ void __launch_bounds__(WARPS * 32, 1) k_branch_tc(BranchArgs a, int JW, int IG) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float s_l2r[16 * KS];
    using Unit = UnitLayout<KS>;
    const mbema_branches& br = a.br;
    constexpr int N = 16 * KS;
    const int h = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int D = a.H * BR_HD;
    br_wait_for_kernel_before();
    br_let_next_kernel_start();
    const int lists = a.n_pre + (int)(br.B * br.S), n_pre = a.n_pre;
    const int2* work = reinterpret_cast<const int2*>(br.work);
    ListSearch search;
    search.begin(work, lists, lane);
    const int total = work[lists].x;
    // behind the ring the steps' fragments of W, then (or in the ring, where there is no room) the staged slice of W
    const uint32_t w_all = (uint32_t)__cvta_generic_to_shared(smem) + a.ring_bytes;
    float* W_sh = reinterpret_cast<float*>(smem + a.w_offset);
    for (int i = tid; i < N * 16; i += WARPS * 32) {
        const float4 x = *reinterpret_cast<const float4*>(a.W + (size_t)(i >> 4) * D + h * BR_HD + (i & 15) * 4);
        float2* dst = reinterpret_cast<float2*>(W_sh + w_row(i >> 4) + (i & 15) * 4);
        dst[0] = make_float2(x.x, x.y);
        dst[1] = make_float2(x.z, x.w);
    }
    for (int i = tid; i < N; i += WARPS * 32) s_l2r[i] = br_log2(br.rhos[i]);
    const int workers = branch_workers(total, (int)gridDim.x * IG, BR_LEAST_COST);
    const int jj = warp % JW, ig = warp / JW;
    const int j = blockIdx.z * JW + jj;
    const int steps = min(JW, a.n - (int)blockIdx.z * JW);       // of this CTA
    const int me = (int)blockIdx.x * IG + ig;
    const bool works = ig < IG && jj < steps && me < workers && total > 0;
    if ((int)blockIdx.x * IG >= workers || total == 0) return;   // the whole CTA has nothing to do
    const int c_end = works ? branch_cut(total, workers, me + 1) : 0;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + (works ? ig : 0) * STAGES * Unit::BYTES;
    const uint32_t ring_end = ring + STAGES * Unit::BYTES;

    // producer: `left` units of list px from slot pk on; the ids of its next unit are a unit ahead
    int px = 0, pk = 0, left = 0;
    List pl = {nullptr, nullptr, 0};
    auto units_to = [&](int from, int to, int cost) { return (min(to, c_end) - from + cost - 1) / cost; };
    auto cost_of = [&](int list) { return list < n_pre ? BR_COST_BLOCK : BR_COST_OWN; };
    auto next_list = [&](int& list, int& count) {                // the next list with units in this stretch: their number, or 0
        for (;;) {
            const int2 at = work[++list];
            if (at.x >= c_end) return 0;
            const int hi = work[list + 1].x;
            count = at.y;
            if (hi > at.x) return units_to(at.x, hi, cost_of(list));
        }
    };
    if (works) {
        const int c0 = branch_cut(total, workers, me);
        int2 lo, hi;
        px = search.find(work, lists, c0, lane, lo, hi);
        const int cost = cost_of(px), skip = (c0 - lo.x + cost - 1) / cost;     // units of the list before this stretch
        int count = lo.y;
        pk = skip * 16;
        left = max(units_to(lo.x + skip * cost, hi.x, cost), 0);
        if (left == 0) { pk = 0; left = next_list(px, count); }
        pl = get_list(a, px, count);
    }
    int x = px;                                                  // consumer: c_left units of list x from slot k0 on
    int k0 = pk, c_left = left, count = pl.count;
    // copies of a lane: 16-byte pieces of rows 4 i + sub of E_k and E_v, and of the fragments
    const int sub = lane >> 3;
    const char* Ek = reinterpret_cast<const char*>(a.Ek) + h * (BR_HD * 2) + (lane & 7) * 16;
    const char* Ev = reinterpret_cast<const char*>(a.Ev) + h * (BR_HD * 2) + (lane & 7) * 16;
    const uint32_t D2 = (uint32_t)D * 2;
    const uint32_t dst_E = sub * 128 + (((lane & 7) ^ ((sub & 1) << 2)) << 4), dst_A = Unit::OP + lane * 16;
    int ids = 0, turn = 0;                                       // the worker's warps copy a unit each in turn
    if (works && jj == 0) ids = pl.slots[min(pk + (lane & 15), pl.count - 1)];
    uint32_t fill = ring;                                        // stage that the producer fills next
    auto produce = [&]() {
        if (left > 0) {
            const char* op = pl.op + (size_t)(pk >> 4) * Unit::OP_BYTES + lane * 16;
            const int now = ids;
            const bool mine = turn == jj;
            turn = turn + 1 == steps ? 0 : turn + 1;
            pk += 16;
            if (--left == 0) {
                int next = 0;
                left = next_list(px, next);
                if (left > 0) { pl = get_list(a, px, next); pk = 0; }
            }
            if (turn == jj && left > 0) ids = pl.slots[min(pk + (lane & 15), pl.count - 1)];
            if (mine) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t v = (uint32_t)__shfl_sync(0xffffffffu, now, i * 4 + sub);
                    cp_async16(fill + dst_E + i * 512, Ek + (uint64_t)v * D2);
                    cp_async16(fill + dst_E + Unit::EV + i * 512, Ev + (uint64_t)v * D2);
                }
#pragma unroll
                for (int i = 0; i < KS; ++i) cp_async16(fill + dst_A + i * 512, op + i * 512);
            }
        }
        cp_commit();
        fill += Unit::BYTES;
        if (fill == ring_end) fill = ring;
    };
    const bool in_ring = a.w_offset == 0;
    auto fill_ring = [&]() {
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) produce();
    };
    if (works && !in_ring) fill_ring();
    __syncthreads();
    for (int i = 0; i < steps; ++i)
        build_W<KS>(w_all + i * KS * 2048, W_sh, s_l2r, blockIdx.z * JW + i, a.silu ? 0.5f * BT_W_SCALE : BT_W_SCALE, lane, warp, WARPS);
    __syncthreads();
    if (!works) return;
    if (in_ring) fill_ring();
    const uint32_t w_at = w_all + jj * KS * 2048 + lane * 16;
    constexpr bool W_REGS = KS == 4;
    uint4 w[KS * 4];
    if constexpr (W_REGS) read_W<KS>(w, w_at);
    OneRow one;
    SixteenRows many;
    bool fresh = true, own = false;
    int rows = 1;
    uint32_t at = ring;
    const uint32_t lane_lo = g * 128 + ((t ^ ((g & 1) << 2)) << 4), lane_hi = lane_lo ^ 64u;
    for (;;) {
        if (fresh) {
            own = x >= n_pre;
            if (own) {
                one.start(a, x - n_pre, j, h, lane);
            } else {
                const int b = x / a.blocks, s0 = (x - b * a.blocks) * BR_BLOCK;
                rows = min(BR_BLOCK, (int)br.S - s0);
                many.start(a, (int64_t)b * br.S + s0, rows, j, h, lane);
            }
            fresh = false;
        }
        unsigned touched0 = 0u, touched1 = 0u;
        if (!own) { touched0 = many.hid0[k0 >> 5]; touched1 = many.hid1[k0 >> 5]; }
        cp_wait<STAGES - 2>();
        if (steps == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(ig + 1), "r"(steps * 32) : "memory");
        produce();
        float acc[8][4];
        {
            uint32_t A[KS][4];
            load_A<KS>(A, at + lane * 16);
            if constexpr (W_REGS) gate<KS>(acc, A, w);
            else gate<KS>(acc, A, w_at);
        }
        apply_gate(acc, a.silu);
        if (own) one.unit(acc, at + lane_lo, at + lane_hi, hidden16(k0, one.staged, j > 0, count), g);
        else many.unit(a, acc, at + lane_lo, at + lane_hi, k0, count, touched0, touched1, j, t);
        at += Unit::BYTES;
        if (at == ring_end) at = ring;
        k0 += 16;
        if (--c_left == 0) {                                     // end of the list or of the stretch
            if (own) one.leave(a, a.own_piece0 + (x - n_pre) + me, j, h, lane);
            else many.leave(a, (int64_t)x + me, rows, j, h, lane);
            c_left = next_list(x, count);
            if (c_left == 0) break;
            k0 = 0;
            fresh = true;
        }
    }
    cp_wait<0>();
}

bool branch_tc_supported(int64_t N) { return N == 64 || N == 128; }

// How the warps of a CTA are dealt: JW steps to a worker (they share its E and operand rows), IG workers, whichever keeps the most
// warps busy over all blocks of steps; a worker of fewer steps fetches its rows more often.
static void steps_and_workers(int n, int warps, int& JW, int& IG) {
    double best = -1.0;
    for (int jw = 1; jw <= std::min(n, 8); ++jw) {
        const int zb = (n + jw - 1) / jw;
        const double busy = (double)(warps / jw) * n / zb / (1.0 + 0.25 / jw);
        if (busy >= best) { best = busy; JW = jw; }
    }
    IG = warps / JW;
}

BranchShape branch_shape(int64_t S, int64_t n, int64_t H) {
    BranchShape p;
    p.blocks = (int)((S + BR_BLOCK - 1) / BR_BLOCK);
    steps_and_workers((int)n, WARPS, p.JW, p.IG);
    p.zb = (int)((n + p.JW - 1) / p.JW);
    p.ctas = (int)std::max<int64_t>(1, 148 / (H * p.zb));       // one CTA an SM, dealt to the heads and blocks of steps
    return p;
}

template <int KS, int STAGES>
static int launch_tc(BranchArgs& a, const BranchShape& p, cudaStream_t st) {
    const size_t w_sh = align_up(((size_t)16 * KS * BT_LDW + 8) * 4, 128), w_all = (size_t)p.JW * KS * 2048;
    const size_t ring = (size_t)p.IG * STAGES * UnitLayout<KS>::BYTES, most = 232448 - 1024;
    const bool in_ring = ring + w_all + w_sh > most;
    a.ring_bytes = (int)(in_ring ? std::max(ring, w_sh) : ring);
    a.w_offset = in_ring ? 0 : a.ring_bytes + (int)w_all;
    const size_t smem = a.ring_bytes + w_all + (in_ring ? 0 : w_sh);
    static std::atomic<unsigned long long> done{0};
    MBEMA_CUDA_TRY(allow_smem(k_branch_tc<KS, STAGES>, most, done));
    MBEMA_CUDA_TRY(launch_early(k_branch_tc<KS, STAGES>, dim3((unsigned)p.ctas, (unsigned)a.H, (unsigned)p.zb), WARPS * 32, smem, st, a, p.JW, p.IG));
    return check_launch();
}

int launch_branch_attend_tc(BranchArgs& a, const BranchShape& p, cudaStream_t st) {
    return a.br.N == 64 ? launch_tc<4, 4>(a, p, st) : launch_tc<8, 3>(a, p, st);
}

}  // namespace mbema
