// gemm_kernels.hip - matrix products on the 16-bit matrix instructions, with
// the epilogues of a linear layer, of its gradients and of the Newton-Schulz
// step (thvm_hip_linear, thvm_hip_linear_grad, thvm_hip_muon_step).
//
// Operands. Every product is C[r][c] = sum_k A[r][k] B[c][k] of two packed
// operands. Packing lays an operand out as the matrix instruction
// (v_mfma_f32_32x32x16_f16) takes it: blocks of 32 rows by 16 k, 1 KB each,
// lane l's 16 bytes being k = 8 (l / 32) .. + 7 of row l % 32. A block goes
// from memory to LDS as it is (one 16-byte load a lane that writes LDS
// directly) and from LDS to registers without bank conflicts, and both
// orientations of a matrix are written by the same pass over it. Rows and k
// are padded with zeros to whole tiles, so the main loop has no bounds.
//
// 32-bit operands are two f16 planes: x 2^e = hi + lo, hi the nearest f16 and
// lo the nearest f16 of what is left, with e such that the largest value of
// the row (the products' sums never mix rows) lies in [2^14, 2^15). hi + lo
// is x 2^e to 2^-24 of itself, or to 2^-25 where x is under 2^-15 of its
// row's largest. Of the four products three are summed, hi hi + hi lo +
// lo hi; lo lo is at most 2^-24 of the product. All sums are 32 bits. So a
// 32-bit product costs three 16-bit ones, where three bf16 planes cost six.
// A row that holds an infinity or NaN is marked, and its outputs are
// computed again by plain 32-bit sums over the planes (exact_dot).
// 16-bit operands are one plane as they are.
#include <hip/hip_runtime.h>
#include "thvm_abi.h"
#include "block_args.h"
#include "block_mem.h"

typedef f16 h8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));   // a 32x32 block's sums
typedef float f4 __attribute__((ext_vector_type(4)));

// ---- activations (thvm_hip.h) ----

__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

// gelu's tanh form is z * sigmoid(2 sqrt(2/pi) (z + 0.044715 z^3))
#define GELU_U 1.5957691216057308f
#define GELU_C 0.044715f

// The normal distribution's integral up to z, by the rational approximation of
// erfc in Abramowitz and Stegun, 7.1.26: within 7.5e-8, a third of the
// instructions of erff. Taken on the side of the small tail, so that a tail is
// a small number and not what is left of 1.
__device__ __forceinline__ float normal_cdf(float z) {
    const float x = fabsf(z) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(1.0f + 0.3275911f * x);
    const float p = t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
    const float tail = 0.5f * p * __expf(-x * x);
    return z < 0.0f ? tail : 1.0f - tail;
}

__device__ __forceinline__ float act_of(u32 act, float z) {
    switch (act) {
    case ACT_RELU: return z > 0.0f ? z : 0.0f;
    case ACT_GELU: return z * normal_cdf(z);
    case ACT_GELU_TANH: return z * sigmoid(GELU_U * (z + GELU_C * z * z * z));
    case ACT_SILU: return z * sigmoid(z);
    default: return z;
    }
}

// Far from 0 the second term is 0; z is held near so that it is no product
// of 0 and infinity there.
__device__ __forceinline__ float act_slope(u32 act, float z) {
    const float near = fminf(fmaxf(z, -128.0f), 128.0f);
    switch (act) {
    case ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
    case ACT_GELU: return normal_cdf(z) + near * (0.3989422804014327f * __expf(-0.5f * near * near));
    case ACT_GELU_TANH: {
        const float s = sigmoid(GELU_U * (z + GELU_C * z * z * z));
        return s + near * (s * (1.0f - s)) * (GELU_U * (1.0f + 3.0f * GELU_C * near * near));
    }
    case ACT_SILU: {
        const float s = sigmoid(z);
        return s + near * (s * (1.0f - s));
    }
    default: return 1.0f;
    }
}

// The same of 8 values: one choice for all of them.
#define ACT_CASES(f, ...)                                                                                          \
    switch (act) {                                                                                                 \
    case ACT_RELU: ACT_EACH(f(ACT_RELU, z[j]), __VA_ARGS__) break;                                                 \
    case ACT_GELU: ACT_EACH(f(ACT_GELU, z[j]), __VA_ARGS__) break;                                                 \
    case ACT_GELU_TANH: ACT_EACH(f(ACT_GELU_TANH, z[j]), __VA_ARGS__) break;                                       \
    case ACT_SILU: ACT_EACH(f(ACT_SILU, z[j]), __VA_ARGS__) break;                                                 \
    default: break;                                                                                                \
    }
#define ACT_EACH(e, op) _Pragma("unroll") for (u32 j = 0; j < 8; j++) v[j] op e;
__device__ __forceinline__ void act8(u32 act, float *v) {
    const float *z = v;
    ACT_CASES(act_of, =)
}
__device__ __forceinline__ void slope8(u32 act, const float *z, float *v) { ACT_CASES(act_slope, *=) }

template <typename T> __device__ __forceinline__ void load8(const glob<T> *row, u32 e, u32 n, float *out) { load_n<T, 8>(row, e, n, out); }
template <typename T> __device__ __forceinline__ void store8(glob<T> *row, u32 e, u32 n, const float *in) { store_n<T, 8>(row, e, n, in); }

// ---- packed operands ----

// f16 elements of block (row block, k block) of plane pl
template <u32 PL>
__device__ __forceinline__ u64 block_at(u64 rb, u64 kb, u64 KB, u32 pl) { return ((rb * KB + kb) * PL + pl) * 512u; }

__device__ __forceinline__ void split(float v, f16 &hi, f16 &lo) {
    hi = (f16)v;
    const float h = (float)hi;
    lo = fabsf(h) < __builtin_inff() ? (f16)(v - h) : (f16)0.0f;
}

// A row's exponent word: e, and whether the row holds an infinity or NaN.
#define EXP_MARK 0x40000000
__device__ __forceinline__ int exp_of(int w) { return (w << 2) >> 2; }
__device__ __forceinline__ bool exp_marked(int w) { return ((w >> 30) & 1) != ((w >> 31) & 1); }

// The sum of a row's products with the planes as they are, in 32 bits.
template <u32 PL>
__device__ __forceinline__ float exact_dot(const glob<f16> *A, const glob<f16> *B, u32 KB, u32 r, u32 c) {
    float s = 0.0f;
    for (u32 kb = 0; kb < KB; kb++)
        for (u32 t = 0; t < 16; t++) {
            const u32 at = (t >> 3) * 256u + (t & 7u);
            const u64 ia = block_at<PL>(r >> 5, kb, KB, 0) + at + (r & 31u) * 8u;
            const u64 ib = block_at<PL>(c >> 5, kb, KB, 0) + at + (c & 31u) * 8u;
            float a = (float)A[ia], b = (float)B[ib];
            if (PL == 2) a += (float)A[ia + 512], b += (float)B[ib + 512];
            s = fmaf(a, b, s);
        }
    return s;
}

// ---- the product ----

typedef __attribute__((address_space(1))) const void *gptr;
typedef __attribute__((address_space(3))) void *lptr;

// Every load to LDS but the last `loads` of this wave and every read of LDS
// but the last `reads` are done, and every wave is here.
template <u32 loads, u32 reads> __device__ __forceinline__ void wait_stage() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(%1)\n\ts_barrier" ::"n"(loads), "n"(reads) : "memory");
}

// A tile of TM x TN by WM x WN waves. A unit is one k step of the matrix
// instruction over all planes; a stage is US units, the chunks of each row
// block that lie together in memory. LDS holds NS stages. Small tiles have
// longer stages: a barrier then stands between enough multiplications.
template <u32 TM_, u32 TN_, u32 WM_, u32 WN_, u32 PL_, u32 US_, u32 NS_>
struct Tile {
    static constexpr u32 TM = TM_, TN = TN_, WM = WM_, WN = WN_, PL = PL_, US = US_, NS = NS_;
    static constexpr u32 WAVES = WM * WN, THREADS = WAVES * 64, RBA = TM / 32, RBB = TN / 32, RB = RBA + RBB;
    static constexpr u32 MI = TM / WM / 32, NI = TN / WN / 32;
    static constexpr u32 CK = US * PL;                      // chunks of a row block in a stage
    static constexpr u32 STAGE = RB * CK * 512;             // f16 elements
    static constexpr u32 PITCH = NI * 32 + 4;               // the epilogue's staging rows
    static constexpr u32 EPI = WAVES * 32 * PITCH * 2;      // f16 elements
    static constexpr u32 LDS = NS * STAGE > EPI ? NS * STAGE : EPI;
    static constexpr u32 Q = RB / WAVES, CH = Q * CK;       // row blocks and chunks a wave brings in a stage
    static constexpr u32 READS = (MI + NI) * CK;            // fragments a wave reads of a stage
    static constexpr u32 TURN = US == 1 ? 2 : 1;            // stages a turn of the main loop
    static_assert(READS < 16 && RB % WAVES == 0 && (NS & (NS - 1)) == 0 && CK <= 4 && (US == 1 || US % 2 == 0),
                  "a wave brings whole row blocks; units alternate between two sets of registers");
    static_assert((NS - 1) * CK * 1024 <= PACK_SLACK, "loads past the end");
};

// The sums of a tile over stages s0 .. s1 - 1. A unit's fragments are read
// from LDS while the unit before is multiplied; where that begins a stage,
// the wait for the stage and the barrier come ahead of the reads, so that
// they too pass behind multiplications. A stage is brought NS - 1 ahead, into
// the buffer whose last reader has passed that barrier.
template <typename TL>
__device__ __forceinline__ void mainloop(f16 *lds, const glob<f16> *A, const glob<f16> *B, u32 KBA, u32 KBB, u32 rb0, u32 cb0, u32 s0, u32 s1,
                                         f16v (&acc)[TL::MI][TL::NI]) {
    constexpr u32 PL = TL::PL, NS = TL::NS, Q = TL::Q;
    const u32 lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const u32 wm = wave / TL::WN, wn = wave % TL::WN;
#pragma unroll
    for (u32 i = 0; i < TL::MI; i++)
#pragma unroll
        for (u32 j = 0; j < TL::NI; j++)
#pragma unroll
            for (u32 v = 0; v < 16; v++) acc[i][j][v] = 0.0f;
    if (s0 >= s1) return;
    const glob<f16> *src[Q];
#pragma unroll
    for (u32 q = 0; q < Q; q++) {
        const u32 b = wave * Q + q;
        const glob<f16> *base = b < TL::RBA ? A + block_at<PL>(rb0 + b, 0, KBA, 0) : B + block_at<PL>(cb0 + b - TL::RBA, 0, KBB, 0);
        src[q] = base + (u64)s0 * (TL::CK * 512u) + lane * 8u;
    }
    // Past the last stage what follows in memory is brought, for no one to
    // read, so that the count of loads in flight stays the same (a packed
    // operand ends PACK_SLACK short of its allocation).
    auto bring = [&](u32 buf) {
#pragma unroll
        for (u32 q = 0; q < Q; q++) {
            const u32 dst = (u32)(uintptr_t)(lptr)lds + (buf * TL::STAGE + (wave * Q + q) * (TL::CK * 512u)) * 2u;
#define BRING(c) if (c < TL::CK) __builtin_amdgcn_global_load_lds((gptr)src[q], (lptr)(uintptr_t)dst, 16, c * 1024, 0);
            BRING(0) BRING(1) BRING(2) BRING(3)
#undef BRING
            src[q] += TL::CK * 512u;
        }
    };
    h8 a[2][TL::MI][PL], b[2][TL::NI][PL];
    auto fetch = [&](u32 buf, u32 k, h8 (&fa)[TL::MI][PL], h8 (&fb)[TL::NI][PL]) {
        const f16 *st = lds + buf * TL::STAGE + lane * 8u;
#pragma unroll
        for (u32 p = 0; p < PL; p++) {
#pragma unroll
            for (u32 j = 0; j < TL::NI; j++) fb[j][p] = *(const h8 *)(st + ((TL::RBA + wn * TL::NI + j) * TL::CK + k * PL + p) * 512u);
#pragma unroll
            for (u32 i = 0; i < TL::MI; i++) fa[i][p] = *(const h8 *)(st + ((wm * TL::MI + i) * TL::CK + k * PL + p) * 512u);
        }
    };
    auto multiply = [&](const h8 (&fa)[TL::MI][PL], const h8 (&fb)[TL::NI][PL]) {
#pragma unroll
        for (u32 t = 0; t < 2 * PL - 1; t++)       // hi hi, then hi lo and lo hi
#pragma unroll
            for (u32 i = 0; i < TL::MI; i++)
#pragma unroll
                for (u32 j = 0; j < TL::NI; j++)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[i][t >> 1], fb[j][t & 1], acc[i][j], 0, 0, 0);
    };
    // One of the next unit's fragments is read after each of the first
    // multiplications: left alone, the compiler puts the reads last.
    auto unit = [&](u32 buf, u32 k, const h8 (&fa)[TL::MI][PL], const h8 (&fb)[TL::NI][PL], h8 (&na)[TL::MI][PL],
                    h8 (&nb)[TL::NI][PL]) {
        __builtin_amdgcn_sched_barrier(0);
        fetch(buf, k, na, nb);
        multiply(fa, fb);
#pragma unroll
        for (u32 i = 0; i < (TL::MI + TL::NI) * PL; i++) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (u32 i = 0; i + 1 < NS; i++) bring(i);
    wait_stage<(NS - 2) * TL::CH, 0>();
    fetch(0, 0, a[0], b[0]);
    for (u32 s = s0, buf = 0; s < s1; s += TL::TURN) {
#pragma unroll
        for (u32 u = 0; u < TL::US * TL::TURN; u++) {
            const bool fresh = (u + 1) % TL::US == 0;       // the next unit begins a stage
            if (fresh) {
                wait_stage<(NS - 3) * TL::CH, TL::READS>();
                bring((buf + NS - 1) & (NS - 1));
                buf = (buf + 1) & (NS - 1);
            }
            unit(buf, fresh ? 0 : u + 1, a[u & 1], b[u & 1], a[(u + 1) & 1], b[(u + 1) & 1]);
        }
    }
}

// Tiles in runs of neighbours per XCD (workgroup b runs on XCD b % 8), four
// tile rows at a time, so that an XCD's L2 serves a block of them.
__device__ __forceinline__ void tile_of(u32 b, u32 tm, u32 tn, u32 &i, u32 &j) {
    const u32 n = tm * tn, q = n / 8, rem = n % 8, x = b % 8;
    u32 t = x * q + (x < rem ? x : rem) + b / 8;
    const u32 g = t / (4 * tn), first = g * 4, rows = tm - first < 4 ? tm - first : 4;
    t -= g * 4 * tn;
    i = first + t % rows;
    j = t / rows;
}

// the tiles on and above the diagonal, column by column
__device__ __forceinline__ void tile_upper(u32 t, u32 &i, u32 &j) {
    j = (u32)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
    while (j * (j + 1) / 2 > t) j--;
    while ((j + 1) * (j + 2) / 2 <= t) j++;
    i = t - j * (j + 1) / 2;
}

// One wave's sums of a 32-row block into LDS, for its lanes to take rows of.
template <typename TL>
__device__ __forceinline__ void stage_rows(float *st, const f16v (&acc)[TL::NI]) {
    const u32 lane = threadIdx.x & 63u;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (u32 j = 0; j < TL::NI; j++)
#pragma unroll
        for (u32 v = 0; v < 16; v++) st[((v >> 2) * 8 + (lane >> 5) * 4 + (v & 3)) * TL::PITCH + j * 32 + (lane & 31u)] = acc[j][v];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// What an output becomes: z = sum (+ bias), y = act(z) (+ residual).
template <typename T>
__device__ __forceinline__ void finish8(const GemmArgs &a, u32 r, u32 c, float *v) {
    float t[8];
    if (a.bias) {
        load8<T>((const glob<T> *)a.bias, c, a.N, t);
#pragma unroll
        for (u32 j = 0; j < 8; j++) v[j] += t[j];
    }
    if (a.z) store8<T>((glob<T> *)a.z + (u64)r * a.N, c, a.N, v);
    act8(a.act, v);
    if (a.res) {
        load8<T>((const glob<T> *)a.res + (u64)r * a.N, c, a.N, t);
#pragma unroll
        for (u32 j = 0; j < 8; j++) v[j] += t[j];
    }
    store8<T>((glob<T> *)a.out + (u64)r * a.N, c, a.N, v);
}

// One output whose row or column is marked, its sum computed again.
template <u32 PL, typename T>
__device__ __forceinline__ void finish_marked(const GemmArgs &a, u32 r, u32 c) {
    const int e = exp_of(((const glob<int> *)a.ea)[r]) + exp_of(((const glob<int> *)a.eb)[c]);
    float v = ldexpf(exact_dot<PL>((const glob<f16> *)a.A, (const glob<f16> *)a.B, a.KB, r, c), -e);
    const u64 at = (u64)r * a.N + c;
    if (a.bias) v += (float)((const glob<T> *)a.bias)[c];
    if (a.z) ((glob<T> *)a.z)[at] = (T)v;
    v = act_of(a.act, v);
    if (a.res) v += (float)((const glob<T> *)a.res)[at];
    ((glob<T> *)a.out)[at] = (T)v;
}

// The exponents of 8 columns (padded to whole tiles), and whether one is marked.
__device__ __forceinline__ bool column_exps(const GemmArgs &a, u32 c, int *ec) {
    bool odd = false;
#pragma unroll
    for (u32 j = 0; j < 8; j++) {
        const int w = ((const glob<int> *)a.eb)[c + j];
        odd |= exp_marked(w);
        ec[j] = exp_of(w);
    }
    return odd;
}

// A tile of one product, or of one of its K splits (blockIdx.y): the partial
// sums then go to a.part[split][M][N] and gemm_join ends the work.
template <typename TL, typename T>
__device__ __forceinline__ void gemm_tile(const GemmArgs &a, f16 *lds) {
    const u32 wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    u32 ti, tj;
    tile_of(blockIdx.x, a.tm, a.tn, ti, tj);
    const u32 S = a.KB / TL::US, per = (S / TL::TURN + a.splits - 1) / a.splits * TL::TURN, s0 = blockIdx.y * per;
    const u32 s1 = s0 + per < S ? s0 + per : S;
    f16v acc[TL::MI][TL::NI];
    mainloop<TL>(lds, (const glob<f16> *)a.A, (const glob<f16> *)a.B, a.KB, a.KB, ti * TL::RBA, tj * TL::RBB, s0, s1, acc);
    wait_stage<0, 0>();
    // A lane keeps 8 columns and takes every RPP-th row of them. The residual
    // of a 32-row block is asked for before the block ahead of it is finished.
    constexpr u32 LPR = TL::NI * 4, RPP = 64 / LPR, PASSES = 32 / RPP;
    const u32 lane = threadIdx.x & 63u, dc = (lane % LPR) * 8, c = tj * TL::TN + (wave % TL::WN) * TL::NI * 32 + dc;
    const u32 r0 = ti * TL::TM + (wave / TL::WN) * TL::MI * 32 + lane / LPR;
    float *st = (float *)lds + wave * 32 * TL::PITCH;
    const float *row = st + (lane / LPR) * TL::PITCH + dc;
    if (a.splits > 1) {
#pragma unroll
        for (u32 i = 0; i < TL::MI; i++) {
            stage_rows<TL>(st, acc[i]);
#pragma unroll
            for (u32 p = 0; p < PASSES; p++) {
                const u32 r = r0 + i * 32 + p * RPP;
                float v[8];
                *(f4 *)v = *(const f4 *)(row + p * RPP * TL::PITCH);
                *(f4 *)(v + 4) = *(const f4 *)(row + p * RPP * TL::PITCH + 4);
                if (r < a.M && c < a.N) store8<float>((glob<float> *)a.part + ((u64)blockIdx.y * a.M + r) * a.N, c, a.N, v);
            }
        }
        return;
    }
    const bool whole = c + 8 <= a.N;
    float bias[8];
    int ec[8];
    bool odd = false, left = false;      // a column that is marked; outputs left for later
    if (a.bias) load8<T>((const glob<T> *)a.bias, c, a.N, bias);
    if (TL::PL == 2) odd = column_exps(a, c, ec);
    any_vec<T, 8> res[2][PASSES];
    auto ask = [&](u32 i, any_vec<T, 8> (&x)[PASSES]) {
#pragma unroll
        for (u32 p = 0; p < PASSES; p++) {
            const u32 r = r0 + i * 32 + p * RPP;
            if (a.res && whole && r < a.M) x[p] = *(const glob<any_vec<T, 8>> *)((const glob<T> *)a.res + (u64)r * a.N + c);
        }
    };
    ask(0, res[0]);
#pragma unroll
    for (u32 i = 0; i < TL::MI; i++) {
        if (i + 1 < TL::MI) ask(i + 1, res[(i + 1) & 1]);
        stage_rows<TL>(st, acc[i]);
#pragma unroll
        for (u32 p = 0; p < PASSES; p++) {
            const u32 r = r0 + i * 32 + p * RPP;
            if (r >= a.M || c >= a.N) continue;
            float v[8];
            *(f4 *)v = *(const f4 *)(row + p * RPP * TL::PITCH);
            *(f4 *)(v + 4) = *(const f4 *)(row + p * RPP * TL::PITCH + 4);
            if (TL::PL == 2) {
                const int er = ((const glob<int> *)a.ea)[r];
                if (odd || exp_marked(er)) {
                    left = true;
                    continue;
                }
#pragma unroll
                for (u32 j = 0; j < 8; j++) v[j] = ldexpf(v[j], -(er + ec[j]));
            }
            if (a.bias)
#pragma unroll
                for (u32 j = 0; j < 8; j++) v[j] += bias[j];
            const u64 at = (u64)r * a.N;
            if (a.z) store8<T>((glob<T> *)a.z + at, c, a.N, v);
            act8(a.act, v);
            if (a.res) {
                if (whole)
#pragma unroll
                    for (u32 j = 0; j < 8; j++) v[j] += (float)res[i & 1][p][j];
                else
#pragma unroll
                    for (u32 j = 0; j < 8; j++)
                        if (c + j < a.N) v[j] += (float)((const glob<T> *)a.res)[at + c + j];
            }
            store8<T>((glob<T> *)a.out + at, c, a.N, v);
        }
    }
    if (TL::PL == 2 && left)
        for (u32 q = 0; q < TL::MI * PASSES; q++) {
            const u32 r = r0 + q * RPP;
            if (r < a.M && (odd || exp_marked(((const glob<int> *)a.ea)[r])))
                for (u32 j = 0; j < 8 && c + j < a.N; j++) finish_marked<TL::PL, T>(a, r, c + j);
        }
}

// The sums of K splits, in split order, and what an output becomes.
template <u32 PL, typename T>
__device__ __forceinline__ void gemm_join(const GemmArgs &a) {
    const u32 per = (a.N + 7) / 8;
    const u64 t = (u64)blockIdx.x * 256u + threadIdx.x;
    if (t >= (u64)per * a.M) return;
    const u32 r = (u32)(t / per), c = (u32)(t % per) * 8;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0}, p[8];
    for (u32 s = 0; s < a.splits; s++) {
        load8<float>((const glob<float> *)a.part + ((u64)s * a.M + r) * a.N, c, a.N, p);
#pragma unroll
        for (u32 j = 0; j < 8; j++) v[j] += p[j];
    }
    if (PL == 2) {
        int ec[8];
        const int er = ((const glob<int> *)a.ea)[r];
        if (column_exps(a, c, ec) || exp_marked(er)) {
            for (u32 j = 0; j < 8 && c + j < a.N; j++) finish_marked<PL, T>(a, r, c + j);
            return;
        }
#pragma unroll
        for (u32 j = 0; j < 8; j++) v[j] = ldexpf(v[j], -(er + ec[j]));
    }
    finish8<T>(a, r, c, v);
}

// ---- the Newton-Schulz step's products ----

// 8 values, at the scale of their operand, into a packed operand: row r, k =
// k0 .. k0 + 7 (k0 a multiple of 8).
template <u32 PL>
__device__ __forceinline__ void put_packed(glob<f16> *out, u32 KB, u32 r, u32 k0, const float *v) {
    h8 hi, lo;
#pragma unroll
    for (u32 j = 0; j < 8; j++) {
        f16 h, l;
        split(v[j], h, l);
        hi[j] = h;
        lo[j] = l;
    }
    glob<f16> *at = out + block_at<PL>(r >> 5, k0 >> 4, KB, 0) + ((k0 >> 3) & 1u) * 256u + (r & 31u) * 8u;
    *(glob<h8> *)at = hi;
    if (PL == 2) *(glob<h8> *)(at + 512) = lo;
}

template <u32 PL>
__device__ __forceinline__ void get_packed(const glob<f16> *in, u32 KB, u32 r, u32 k0, float *v) {
    const glob<f16> *at = in + block_at<PL>(r >> 5, k0 >> 4, KB, 0) + ((k0 >> 3) & 1u) * 256u + (r & 31u) * 8u;
    const h8 hi = *(const glob<h8> *)at;
    h8 lo = {};
    if (PL == 2) lo = *(const glob<h8> *)(at + 512);
#pragma unroll
    for (u32 j = 0; j < 8; j++) v[j] = PL == 2 ? (float)hi[j] + (float)lo[j] : (float)hi[j];
}

// A tile of new = alpha * old + beta * (A B^T), written packed in its own
// orientation (out) and the other (out_t), all three at scales that alpha
// and beta hold. A symmetric product's tiles on and above the diagonal are
// computed and written to both sides. The last product of a step goes to the
// parameter instead: p = keep * p - step * new, along its rows.
template <typename TL, typename T>
__device__ __forceinline__ void ns_tile(const NsArgs &a, f16 *lds) {
    constexpr u32 PL = TL::PL;
    const u32 lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const u64 z = blockIdx.z;
    u32 ti, tj;
    if (a.sym) tile_upper(blockIdx.x, ti, tj);
    else tile_of(blockIdx.x, a.tm, a.tn, ti, tj);
    f16v acc[TL::MI][TL::NI];
    mainloop<TL>(lds, (const glob<f16> *)(a.A + z * a.stride), (const glob<f16> *)(a.B + z * a.stride), a.KB, a.KB, ti * TL::RBA, tj * TL::RBB,
                 0, a.KU / TL::US, acc);
    wait_stage<0, 0>();
    float *st = (float *)lds + wave * 32 * TL::PITCH;
    const glob<f16> *old = (const glob<f16> *)(a.old + z * a.stride);
    glob<f16> *out = (glob<f16> *)(a.out + z * a.stride), *out_t = (glob<f16> *)(a.out_t + z * a.stride);
    const bool mirror = a.out_t && !(a.sym && ti == tj);
#pragma unroll
    for (u32 i = 0; i < TL::MI; i++) {
        const u32 r0 = ti * TL::TM + ((wave / TL::WN) * TL::MI + i) * 32, c0 = tj * TL::TN + (wave % TL::WN) * TL::NI * 32;
        stage_rows<TL>(st, acc[i]);
        // own orientation: lane takes row lane % 32, 8 columns at a time
#pragma unroll
        for (u32 j = 0; j < TL::NI * 2; j++) {
            const u32 r = lane & 31u, c = j * 16 + (lane >> 5) * 8;
            float v[8], o[8];
            *(f4 *)v = *(const f4 *)(st + r * TL::PITCH + c);
            *(f4 *)(v + 4) = *(const f4 *)(st + r * TL::PITCH + c + 4);
            if (a.old) {
                get_packed<PL>(old, a.KBO, r0 + r, c0 + c, o);
#pragma unroll
                for (u32 t = 0; t < 8; t++) v[t] = a.alpha * o[t] + a.beta * v[t];
            } else {
#pragma unroll
                for (u32 t = 0; t < 8; t++) v[t] *= a.beta;
            }
            if (a.out) put_packed<PL>(out, a.KBO, r0 + r, c0 + c, v);
            if (mirror || a.last) {
                *(f4 *)(st + r * TL::PITCH + c) = *(const f4 *)v;
                *(f4 *)(st + r * TL::PITCH + c + 4) = *(const f4 *)(v + 4);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (mirror) {
            // the other: lane takes a column, 8 rows at a time
#pragma unroll
            for (u32 j = 0; j < TL::NI; j++)
#pragma unroll
                for (u32 h = 0; h < 2; h++) {
                    const u32 c = j * 32 + (lane & 31u), r = h * 16 + (lane >> 5) * 8;
                    float v[8];
#pragma unroll
                    for (u32 t = 0; t < 8; t++) v[t] = st[(r + t) * TL::PITCH + c];
                    put_packed<PL>(out_t, a.KBT, c0 + c, r0 + r, v);
                }
        }
        if (a.last) {
            // X is [n][w]; the parameter is X's shape, or its transpose (a.tall)
            glob<T> *p = (glob<T> *)a.param[z];
            float v[8], o[8];
            if (!a.tall) {
                constexpr u32 LPR = TL::NI * 4, RPP = 64 / LPR;
#pragma unroll
                for (u32 q = 0; q < 32 / RPP; q++) {
                    const u32 r = q * RPP + lane / LPR, c = (lane % LPR) * 8;
                    if (r0 + r >= a.n || c0 + c >= a.w) continue;
                    *(f4 *)v = *(const f4 *)(st + r * TL::PITCH + c);
                    *(f4 *)(v + 4) = *(const f4 *)(st + r * TL::PITCH + c + 4);
                    glob<T> *row = p + (u64)(r0 + r) * a.w;
                    load8<T>(row, c0 + c, a.w, o);
#pragma unroll
                    for (u32 t = 0; t < 8; t++) o[t] = a.keep * o[t] - a.step * v[t];
                    store8<T>(row, c0 + c, a.w, o);
                }
            } else {
#pragma unroll
                for (u32 q = 0; q < TL::NI * 2; q++) {
                    const u32 c = q * 16 + lane / 4, r = (lane & 3u) * 8;
                    if (r0 + r >= a.n || c0 + c >= a.w) continue;
#pragma unroll
                    for (u32 t = 0; t < 8; t++) v[t] = st[(r + t) * TL::PITCH + c];
                    glob<T> *row = p + (u64)(c0 + c) * a.n;
                    load8<T>(row, r0 + r, a.n, o);
#pragma unroll
                    for (u32 t = 0; t < 8; t++) o[t] = a.keep * o[t] - a.step * v[t];
                    store8<T>(row, r0 + r, a.n, o);
                }
            }
        }
    }
}

// m = beta m + g and the partial sums of u^2, u what is orthogonalised: g +
// beta m (nesterov) or m. Squares and sums in 64 bits, so that no gradient's
// size can overflow them. Workgroups of 256 lanes in steps of the grid.
template <typename T>
__device__ __forceinline__ void muon_momentum(const MuonArgs &a) {
    __shared__ double lds[4];
    const u32 z = blockIdx.y;
    const glob<T> *g = (const glob<T> *)a.grad[z];
    glob<float> *m = (glob<float> *)a.m[z];
    double s = 0.0;
    for (u64 i = ((u64)blockIdx.x * 256u + threadIdx.x) * 4u; i < a.numel; i += (u64)gridDim.x * 1024u) {
        float gv[4], mv[4];
        if (i + 4 <= a.numel) {
            const any_vec<T, 4> pg = *(const glob<any_vec<T, 4>> *)(g + i);
            const f4 pm = *(const glob<f4> *)(m + i);
#pragma unroll
            for (u32 j = 0; j < 4; j++) gv[j] = (float)pg[j], mv[j] = pm[j];
        } else {
#pragma unroll
            for (u32 j = 0; j < 4; j++) gv[j] = i + j < a.numel ? (float)g[i + j] : 0.0f, mv[j] = i + j < a.numel ? m[i + j] : 0.0f;
        }
        f4 out;
#pragma unroll
        for (u32 j = 0; j < 4; j++) {
            out[j] = a.beta * mv[j] + gv[j];
            const double u = a.nesterov ? gv[j] + a.beta * out[j] : out[j];
            s += u * u;
        }
        if (i + 4 <= a.numel) *(glob<f4> *)(m + i) = out;
        else
#pragma unroll
            for (u32 j = 0; j < 4; j++)
                if (i + j < a.numel) m[i + j] = out[j];
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63u) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) ((glob<double> *)a.sums)[z * a.blocks + blockIdx.x] = lds[0] + lds[1] + lds[2] + lds[3];
}

// ---- packing ----

__device__ __forceinline__ u32 size_word(float v) {
    const u32 b = __float_as_uint(v) & 0x7FFFFFFFu;
    return b < 0x7F800000u ? b : 0x80000000u;
}
__device__ __forceinline__ u32 size_join(u32 a, u32 b) {
    const u32 x = a & 0x7FFFFFFFu, y = b & 0x7FFFFFFFu;
    return (x > y ? x : y) | ((a | b) & 0x80000000u);
}
// the exponent word of a row whose largest finite value and mark are w
__device__ __forceinline__ int exp_word(u32 w) {
    const float v = __uint_as_float(w & 0x7FFFFFFFu);
    const int e = v > 0.0f ? 14 - ilogbf(v) : 0;
    return w & 0x80000000u ? e ^ EXP_MARK : e;
}

// What is packed at (r, c .. c + 7): the matrix itself, or dy * act'(z).
template <typename T>
__device__ __forceinline__ void source8(const PackArgs &a, u32 r, u32 c, float *v) {
    load8<T>((const glob<T> *)a.src + (u64)r * a.C, c, a.C, v);
    if (a.z) {
        float z[8];
        load8<T>((const glob<T> *)a.z + (u64)r * a.C, c, a.C, z);
        slope8(a.act, z, v);
    }
}

// The largest values of a matrix's rows and columns (as size words, a part a
// column tile of 512 and a row tile of a.rt) and the columns' sums.
// 8 waves, each every 8th row of the tile, a lane 8 columns.
template <typename T>
__device__ __forceinline__ void pack_sizes(const PackArgs &a) {
    __shared__ u32 lw[8][512];
    __shared__ float ls[8][512];
    const u32 lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const u32 c = blockIdx.x * 512u + lane * 8u;
    const u64 r0 = (u64)blockIdx.y * a.rt, r1 = r0 + a.rt < a.R ? r0 + a.rt : a.R;
    u32 cw[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    float cs[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (u64 r = r0 + wave; r < r1; r += 8) {
        float v[8];
        if (c < a.C) source8<T>(a, (u32)r, c, v);
        else
#pragma unroll
            for (u32 j = 0; j < 8; j++) v[j] = 0.0f;
        u32 rw = 0;
#pragma unroll
        for (u32 j = 0; j < 8; j++) {
            const u32 w = size_word(v[j]);
            rw = size_join(rw, w);
            cw[j] = size_join(cw[j], w);
            cs[j] += v[j];
        }
        if (a.row_part) {
#pragma unroll
            for (int d = 32; d; d >>= 1) rw = size_join(rw, __shfl_xor(rw, d));
            if (lane == 0) ((glob<u32> *)a.row_part)[(u64)blockIdx.x * a.R + r] = rw;
        }
    }
    if (!a.col_part && !a.sum_part) return;
#pragma unroll
    for (u32 j = 0; j < 8; j++) lw[wave][lane * 8 + j] = cw[j], ls[wave][lane * 8 + j] = cs[j];
    __syncthreads();
    const u32 t = threadIdx.x, ct = blockIdx.x * 512u + t;
    if (ct >= a.C) return;
    u32 w = lw[0][t];
    float s = ls[0][t];
#pragma unroll
    for (u32 k = 1; k < 8; k++) w = size_join(w, lw[k][t]), s += ls[k][t];
    if (a.col_part) ((glob<u32> *)a.col_part)[(u64)blockIdx.y * a.C + ct] = w;
    if (a.sum_part) ((glob<float> *)a.sum_part)[(u64)blockIdx.y * a.C + ct] = s;
}

// A 64 x 64 tile of a matrix [R][C] into one or both packed orientations:
// pn (rows r, k = c) and pt (rows c, k = r). 32-bit values are scaled by the
// exponents of their packed row; `unit` (the optimiser) by one factor.
// MUON: the source is u (muon_momentum) over its norm.
template <u32 PL, typename T, bool MUON>
__device__ __forceinline__ void pack_tile(const PackArgs &a, const MuonArgs *mu) {
    __shared__ float tile[64][65];
    __shared__ int er[64], ec[64];
    __shared__ float unit_lds;
    const u32 t = threadIdx.x, r0 = (blockIdx.x / a.ctiles) * 64u, c0 = (blockIdx.x % a.ctiles) * 64u, zi = blockIdx.y;
    if (PL == 2 && !MUON) {
        // the parts of this tile's rows and columns, four lanes to each
        const u32 i = t >> 2, q = t & 3u;
        u32 wr = 0, wc = 0;
        if (a.pn && r0 + i < a.R)
            for (u32 p = q; p < a.row_parts; p += 4) wr = size_join(wr, ((const glob<u32> *)a.row_part)[(u64)p * a.R + r0 + i]);
        if (a.pt && c0 + i < a.C)
            for (u32 p = q; p < a.col_parts; p += 4) wc = size_join(wc, ((const glob<u32> *)a.col_part)[(u64)p * a.C + c0 + i]);
        wr = size_join(wr, __shfl_xor(wr, 1));
        wc = size_join(wc, __shfl_xor(wc, 1));
        wr = size_join(wr, __shfl_xor(wr, 2));
        wc = size_join(wc, __shfl_xor(wc, 2));
        if (q == 0) {
            er[i] = exp_word(wr);
            ec[i] = exp_word(wc);
            if (a.pn && c0 == 0 && r0 + i < a.Rn) ((glob<int> *)a.en)[r0 + i] = er[i];
            if (a.pt && r0 == 0 && c0 + i < a.Ct) ((glob<int> *)a.et)[c0 + i] = ec[i];
        }
    }
    if (MUON) {
        if (t < 64) {
            double s = 0.0;
            for (u32 i = t; i < mu->blocks; i += 64) s += ((const glob<double> *)mu->sums)[zi * mu->blocks + i];
#pragma unroll
            for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
            if (t == 0) unit_lds = (float)(16384.0 / (sqrt(s) + 1e-7));
        }
    }
    __syncthreads();
    glob<f16> *pn = (glob<f16> *)(a.pn + zi * a.stride), *pt = (glob<f16> *)(a.pt + zi * a.stride);
#pragma unroll
    for (u32 h = 0; h < 2; h++) {
        const u32 i = h * 32 + (t >> 3), j = (t & 7u) * 8, r = r0 + i, c = c0 + j;
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (r < a.R && c < a.C) {
            if (MUON) {
                float m[8];
                load8<float>((const glob<float> *)mu->m[zi] + (u64)r * a.C, c, a.C, m);
                if (mu->nesterov) {
                    load8<T>((const glob<T> *)mu->grad[zi] + (u64)r * a.C, c, a.C, v);
#pragma unroll
                    for (u32 k = 0; k < 8; k++) v[k] += mu->beta * m[k];
                } else {
#pragma unroll
                    for (u32 k = 0; k < 8; k++) v[k] = m[k];
                }
#pragma unroll
                for (u32 k = 0; k < 8; k++) v[k] *= unit_lds;
            } else source8<T>(a, r, c, v);
        }
        if (a.pt || a.sum_part)
#pragma unroll
            for (u32 k = 0; k < 8; k++) tile[i][j + k] = v[k];
        if (a.pn && r < a.Rn && c < a.KBn * 16u) {
            if (PL == 2 && !MUON)
#pragma unroll
                for (u32 k = 0; k < 8; k++) v[k] = ldexpf(v[k], exp_of(er[i]));
            put_packed<PL>(pn, a.KBn, r, c, v);
        }
    }
    __syncthreads();
    if (a.pt)
#pragma unroll
        for (u32 h = 0; h < 2; h++) {
            const u32 j = t & 63u, i = h * 32 + (t >> 6) * 8, r = r0 + i, c = c0 + j;
            if (c >= a.Ct || r >= a.KBt * 16u) continue;
            float v[8];
#pragma unroll
            for (u32 k = 0; k < 8; k++) {
                v[k] = tile[i + k][j];
                if (PL == 2 && !MUON) v[k] = ldexpf(v[k], exp_of(ec[j]));
            }
            put_packed<PL>(pt, a.KBt, c, r, v);
        }
    if (PL == 1 && a.sum_part && t < 64 && c0 + t < a.C && r0 < a.R) {
        float s = 0.0f;
        for (u32 i = 0; i < 64; i++) s += tile[i][t];
        ((glob<float> *)a.sum_part)[(u64)(r0 / 64u) * a.C + c0 + t] = s;
    }
}

// out[c] = the sum of `parts` rows of [parts][C], 16 waves every 16th part.
template <typename T>
__device__ __forceinline__ void sum_parts(const glob<float> *part, glob<T> *out, u32 C, u32 parts) {
    __shared__ float lds[16][64];
    const u32 lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, c = blockIdx.x * 64u + lane;
    float s = 0.0f;
    if (c < C)
        for (u32 p = wave; p < parts; p += 16) s += part[(u64)p * C + c];
    lds[wave][lane] = s;
    __syncthreads();
    if (wave || c >= C) return;
#pragma unroll
    for (u32 w = 1; w < 16; w++) s += lds[w][lane];
    out[c] = (T)s;
}

// ---- few rows ----

// y = x W, MR rows a workgroup (blockIdx.z): W is read once, as it lies ([K][N] row-major),
// 16 bytes a lane, 16 lanes along a row and the workgroup's 8 waves 32 rows
// at a time, and multiplied in 32 bits. Bound by W's bytes, so K is split
// over workgroups (blockIdx.y) until the card is full; the splits' sums meet
// in gemm_join.
template <typename T, u32 MR>
__device__ __forceinline__ void few_rows(const GemmArgs &a) {
    constexpr u32 N = 16 / sizeof(T), U = 4, KSTEP = 32, COLS = 16 * N;
    __shared__ float xs[U * KSTEP][MR];
    __shared__ float comb[8][16][N * (MR > 4 ? 4 : MR) + 1];
    const u32 lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const u32 kr = wave * 4 + (lane >> 4), c = blockIdx.x * COLS + (lane & 15u) * N;
    const u32 per = a.kper, k0 = blockIdx.y * per, k1 = k0 + per < a.K ? k0 + per : a.K;
    const u32 m0 = blockIdx.z * MR;
    const glob<T> *W = (const glob<T> *)a.B, *X = (const glob<T> *)a.A + (u64)m0 * a.K;
    float acc[MR][N];
#pragma unroll
    for (u32 r = 0; r < MR; r++)
#pragma unroll
        for (u32 j = 0; j < N; j++) acc[r][j] = 0.0f;
    for (u32 kb = k0; kb < k1; kb += U * KSTEP) {
        any_vec<T, N> w[U];
#pragma unroll
        for (u32 u = 0; u < U; u++) {
            const u32 k = kb + u * KSTEP + kr;
            if (k < k1 && c + N <= a.N) w[u] = *(const glob<any_vec<T, N>> *)(W + (u64)k * a.N + c);
            else
#pragma unroll
                for (u32 j = 0; j < N; j++) w[u][j] = k < k1 && c + j < a.N ? W[(u64)k * a.N + c + j] : (T)0.0f;
        }
        __syncthreads();
        for (u32 i = threadIdx.x; i < U * KSTEP * MR; i += 512) {
            const u32 r = i / (U * KSTEP), k = i % (U * KSTEP);
            xs[k][r] = m0 + r < a.M && kb + k < k1 ? (float)X[(u64)r * a.K + kb + k] : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (u32 u = 0; u < U; u++)
            if (kb + u * KSTEP + kr < k1)     // past the end nothing is multiplied: W there is not a value
#pragma unroll
                for (u32 r = 0; r < MR; r++) {
                    const float x = xs[u * KSTEP + kr][r];
#pragma unroll
                    for (u32 j = 0; j < N; j++) acc[r][j] = fmaf(x, (float)w[u][j], acc[r][j]);
                }
    }
    // the 4 lane groups of a wave, then the 8 waves in order, 4 rows at a time
    constexpr u32 RB = MR > 4 ? 4 : MR;
#pragma unroll
    for (u32 rb = 0; rb < MR; rb += RB) {
#pragma unroll
        for (u32 r = 0; r < RB; r++)
#pragma unroll
            for (u32 j = 0; j < N; j++) {
                float s = acc[rb + r][j];
                s += __shfl_xor(s, 16);
                s += __shfl_xor(s, 32);
                if (lane < 16) comb[wave][lane][r * N + j] = s;
            }
        __syncthreads();
        for (u32 i = threadIdx.x; i < RB * COLS / 8; i += 512) {
            const u32 r = i / (COLS / 8), cc = (i % (COLS / 8)) * 8, col = blockIdx.x * COLS + cc;
            if (m0 + rb + r < a.M && col < a.N) {
                float v[8];
#pragma unroll
                for (u32 j = 0; j < 8; j++) {
                    float s = 0.0f;
#pragma unroll
                    for (u32 w = 0; w < 8; w++) s += comb[w][(cc + j) / N][r * N + (cc + j) % N];
                    v[j] = s;
                }
                if (a.splits > 1) store8<float>((glob<float> *)a.part + ((u64)blockIdx.y * a.M + m0 + rb + r) * a.N, col, a.N, v);
                else finish8<T>(a, m0 + rb + r, col, v);
            }
        }
        __syncthreads();
    }
}

// ---- the kernels ----

#define GEMM(size, TILE, name, T)                                                                                  \
    typedef TILE Tile##size##_##name;                                                                              \
    extern "C" __global__ __launch_bounds__(Tile##size##_##name::THREADS) void thvm_gemm_##size##_##name(GemmArgs a) { \
        __shared__ __attribute__((aligned(1024))) f16 lds[Tile##size##_##name::LDS];                               \
        gemm_tile<Tile##size##_##name, T>(a, lds);                                                                  \
    }                                                                                                              \
    extern "C" __global__ __launch_bounds__(Tile##size##_##name::THREADS) void thvm_ns_##size##_##name(NsArgs a) {  \
        __shared__ __attribute__((aligned(1024))) f16 lds[Tile##size##_##name::LDS];                               \
        ns_tile<Tile##size##_##name, T>(a, lds);                                                                    \
    }
#define TILE(...) Tile<__VA_ARGS__>
GEMM(256, TILE(256, 256, 2, 4, 1, 2, 4), f16, f16)
GEMM(128, TILE(128, 128, 2, 2, 1, 2, 4), f16, f16)
GEMM(64, TILE(64, 64, 2, 2, 1, 4, 4), f16, f16)
GEMM(256, TILE(256, 256, 2, 4, 2, 1, 4), f32, float)
GEMM(128, TILE(128, 128, 2, 2, 2, 1, 4), f32, float)
GEMM(64, TILE(64, 64, 2, 2, 2, 2, 4), f32, float)

#define PER_TYPE(PL, name, T)                                                                                      \
    extern "C" __global__ __launch_bounds__(256) void thvm_gemm_join_##name(GemmArgs a) { gemm_join<PL, T>(a); }    \
    extern "C" __global__ __launch_bounds__(256) void thvm_few_join_##name(GemmArgs a) { gemm_join<1, T>(a); }      \
    extern "C" __global__ __launch_bounds__(512) void thvm_pack_sizes_##name(PackArgs a) { pack_sizes<T>(a); }      \
    extern "C" __global__ __launch_bounds__(256) void thvm_pack_##name(PackArgs a) { pack_tile<PL, T, false>(a, nullptr); } \
    extern "C" __global__ __launch_bounds__(256) void thvm_muon_pack_##name(PackArgs a, MuonArgs m) {               \
        pack_tile<PL, T, true>(a, &m);                                                                              \
    }                                                                                                              \
    extern "C" __global__ __launch_bounds__(256) void thvm_muon_momentum_##name(MuonArgs m) { muon_momentum<T>(m); } \
    extern "C" __global__ __launch_bounds__(1024) void thvm_sum_parts_##name(u64 part, u64 out, u32 C, u32 parts) { \
        sum_parts<T>((const glob<float> *)part, (glob<T> *)out, C, parts);                                                      \
    }                                                                                                              \
    extern "C" __global__ __launch_bounds__(512) void thvm_few1_##name(GemmArgs a) { few_rows<T, 1>(a); }           \
    extern "C" __global__ __launch_bounds__(512) void thvm_few4_##name(GemmArgs a) { few_rows<T, 4>(a); }           \
    extern "C" __global__ __launch_bounds__(512) void thvm_few16_##name(GemmArgs a) { few_rows<T, 16>(a); }
PER_TYPE(1, f16, f16)
PER_TYPE(2, f32, float)
