// gemm_kernels.hip - matrix products on the matrix instructions, with the
// epilogues of a linear layer, of its gradients and of the Newton-Schulz
// step (thvm_hip_linear, thvm_hip_linear_grad, thvm_hip_muon_step).
//
// Three kinds, of which block.c takes the one that its estimate puts first:
// tiles on the 16-bit instruction over packed operands or 16-bit matrices as
// they lie, the bulk of this file; 64 x 64 tiles on the 32-bit instruction over
// 32-bit matrices as they lie (direct_tile), of up to a few hundred rows; and
// few rows (few_rows), which read W once.
//
// Packed operands. A product is C[r][c] = sum_k A[r][k] B[c][k]. Packing lays an operand out as the matrix instruction
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
// is x 2^e to 2^-23 of itself, or to 2^-24 where x 2^e is under 2^-2. Of the
// four products three are summed, hi hi + hi lo + lo hi; lo lo is at most 2^-22
// of the product. All sums are 32 bits. So a 32-bit product costs three 16-bit
// ones, where three bf16 planes cost six, and a sum is within (2 K + 8) 2^-24
// of its products' magnitudes (a 32-bit one: K 2^-24), with two exceptions:
//   a sum that is not finite, as each is that an infinity or NaN goes into;
//   a sum of products that are all small beside their row's and column's
//   largest, of rows with values that lost bits (doubtful).
// Those are computed again from the operands as the caller has them, in 32-bit
// sums of 32-bit products (block_again): of 4096^3 with a NaN in every row 2.0
// ms, in one row 0.72, in none 0.42.
// 16-bit operands are one plane as they are, and so is a gradient's dz = dy
// act'(z), rounded to 16 bits as a network in 16 bits holds it: of 2048^3 its
// products' error against 64 bits is 2.9e-4, that of dz in 32 bits 2.1e-4, most
// of it the outputs' own rounding, and a second plane for dz would double the
// products' instructions (now 47 of the call's 60 us). Where a dz is past 16 bits, the sums that it goes into are
// computed again, too; packing tells the products of a call that there is one.
//
// Large tiles: of 4096^3 in 16 bits as they lie 138 us, 995 TFLOP/s (a library
// product 1155 on the same card; packed ones alone 129 us), the matrix units
// busy 54 % of the cycles with one read of LDS a product; in 32 bits 324 us,
// 1272 TFLOP/s of 16-bit products, busy 73 %. Either way the card holds its clock
// near 1.7 GHz. Small ones are bound by the latency of one stage after another.
#include <hip/hip_runtime.h>
#include "thvm_abi.h"
#include "block_args.h"
#include "block_mem.h"

typedef f16 h8 __attribute__((ext_vector_type(8)));
typedef f16 h4 __attribute__((ext_vector_type(4)));
typedef int i4v __attribute__((ext_vector_type(4)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));   // a 32x32 block's sums
typedef float f4 __attribute__((ext_vector_type(4)));

// ---- activations (thvm_hip.h) ----

__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

// gelu's tanh form is z * sigmoid(2 sqrt(2/pi) (z + 0.044715 z^3))
#define GELU_U 1.5957691216057308f
#define GELU_C 0.044715f

// The normal distribution's integral up to z: the small tail, or what it leaves
// of 1. The tail is exp(-z^2 / 2) t P(t), t = 1 / (1 + 0.35 |z|), P of the least
// largest relative error, fitted to exp(z^2 / 2) erfc: 3.2e-8 up to 15. So a tail
// is as exact as a value near 1, but for the rounding of the exponential's
// argument: within (8 + 2 z^2) 2^-24 of itself. A third of erfcf's instructions; a
// polynomial of its own near 0 would make 6 units there 2, and 64 rows through
// 4096 x 4096 in f16 14.4 us instead of 13.7 (cold code, mostly).
__device__ __forceinline__ float normal_cdf(float z) {
    const float u = z * z, t = __builtin_amdgcn_rcpf(1.0f + 0.35f * fabsf(z));
    const float p = t * (0.13962125778f + t * (0.13986432552f + t * (0.11981558055f + t * (0.10557445139f + t * (-0.023262951523f +
                         t * (0.15939156711f + t * (-0.25590065122f + t * (0.14406019449f + t * -0.029163796455f))))))));
    const float tail = p * __builtin_amdgcn_exp2f(-0.72134752044f * u);
    return z < 0.0f ? tail : 1.0f - tail;
}

__device__ __forceinline__ float act_of(u32 act, float z) {
    switch (act) {
    case ACT_RELU: return z <= 0.0f ? 0.0f : z;      // NaN stays
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
    case ACT_RELU: return z > 0.0f ? 1.0f : z <= 0.0f ? 0.0f : z;
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

// The same of N values: one choice for all of them.
#define ACT_CASES(f, ...)                                                                                          \
    switch (act) {                                                                                                 \
    case ACT_RELU: ACT_EACH(f(ACT_RELU, z[j]), __VA_ARGS__) break;                                                 \
    case ACT_GELU: ACT_EACH(f(ACT_GELU, z[j]), __VA_ARGS__) break;                                                 \
    case ACT_GELU_TANH: ACT_EACH(f(ACT_GELU_TANH, z[j]), __VA_ARGS__) break;                                       \
    case ACT_SILU: ACT_EACH(f(ACT_SILU, z[j]), __VA_ARGS__) break;                                                 \
    default: break;                                                                                                \
    }
#define ACT_EACH(e, op) _Pragma("unroll") for (u32 j = 0; j < N; j++) v[j] op e;
template <u32 N> __device__ __forceinline__ void act_n(u32 act, float *v) {
    const float *z = v;
    ACT_CASES(act_of, =)
}
template <u32 N> __device__ __forceinline__ void slope_n(u32 act, const float *z, float *v) { ACT_CASES(act_slope, *=) }

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

// Of packed 32-bit operands each row has its exponent (ROW_EMPTY where all
// values are 0), and the number of its faint values: under 2^-2 as they are
// packed, and not 0, so that lo may have lost bits, 2^-24 at most. Partners are
// under 2^15, so faint values move a sum by (their number in both rows) 2^-9
// at most: by less than K 2^-25 of the sum of the products' magnitudes, if that
// is over the number times 2^16 / K.
#define ROW_EMPTY 0x4000
typedef int Row __attribute__((ext_vector_type(2)));      // exponent, faint values
__device__ __forceinline__ float faint_unit(u32 K) { return 65536.0f * __builtin_amdgcn_rcpf((float)K); }
__device__ __forceinline__ bool doubtful(Row r, Row c, float unit, float v) {
    return r.x != ROW_EMPTY && c.x != ROW_EMPTY && fabsf(v) < (float)((u32)r.y + (u32)c.y) * unit;
}

// ---- the product ----

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
    // fragments a wave reads of a stage, as far as the counter of reads goes
    static constexpr u32 READS = (MI + NI) * CK < 15 ? (MI + NI) * CK : 15;
    static constexpr u32 TURN = US == 1 ? 2 : 1;            // stages a turn of the main loop
    static_assert(RB % WAVES == 0 && (NS & (NS - 1)) == 0 && CK <= 4 && (US == 1 || US % 2 == 0),
                  "a wave brings whole row blocks; units alternate between two sets of registers");
    static_assert((NS - 1) * CK * 1024 <= PACK_SLACK, "loads past the end");
};

template <u32 v> struct Const { static constexpr u32 value = v; };

// How an operand lies in memory: packed; or, in 16 bits, row-major with k
// along its rows (ROWS: element (r, k) at r ld + k) or across them (COLS: at
// k ld + r), rows of a multiple of 8 elements. Those that are not packed go to
// LDS in chunks of the same 1 KB:
//   ROWS  two chunks hold 32 rows by 32 k, 64 bytes a row, the row's four 16
//         bytes turned by the row (octet o at place o ^ (row / 4) % 4), so that
//         the 16 rows that are read together lie in different banks;
//   COLS  a chunk holds 16 k by 32 rows, 64 bytes a k, and is turned on the
//         way to registers (ds_read_b64_tr_b16: of 16 lanes that read 4 k by 16
//         rows, lane i gets the 4 k of row i).
// Past the end of K, and past the last row, they read as 0 or as another row,
// whose sums no one takes.
enum { PACKED = 0, ROWS, COLS };

// What a wave brings to LDS: where its chunks of a stage are (bytes from a
// base that moves by `step` a stage), and the k, in the stage, that each of its
// lanes begins at. Reads past `end` give 0.
struct Operand {
    u64 base;         // of the first stage, the tile's first row
    u64 end;          // of the memory
    u32 ld, rows;     // ROWS, COLS; rows from the tile's first on
    u32 K;            // k from the first stage on
};

// The sums of a tile over n stages. A unit's fragments are read
// from LDS while the unit before is multiplied; where that begins a stage,
// the wait for the stage and the barrier come ahead of the reads, so that
// they too pass behind multiplications. A stage is brought NS - 1 ahead, into
// the buffer whose last reader has passed that barrier.
template <typename TL, u32 MA, u32 MB>
__device__ __forceinline__ void mainloop(f16 *lds, const Operand &A, const Operand &B, u64 stride_a, u64 stride_b, u32 n,
                                         f16v (&acc)[TL::MI][TL::NI]) {
    constexpr u32 PL = TL::PL, NS = TL::NS, Q = TL::Q, CK = TL::CK;
    static_assert(PL == 1 || (MA == PACKED && MB == PACKED), "planes are packed");
    const u32 lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const u32 wm = wave / TL::WN, wn = wave % TL::WN;
#pragma unroll
    for (u32 i = 0; i < TL::MI; i++)
#pragma unroll
        for (u32 j = 0; j < TL::NI; j++)
#pragma unroll
            for (u32 v = 0; v < 16; v++) acc[i][j][v] = 0.0f;
    if (!n) return;
    // a wave's row blocks are all of A or all of B
    static_assert(TL::RBA % Q == 0, "");
    const bool of_a = wave * Q < TL::RBA;
    const u32 mode = of_a ? MA : MB, ld = of_a ? A.ld : B.ld, rows = of_a ? A.rows : B.rows;
    const u32 rb0 = of_a ? wave * Q : wave * Q - TL::RBA;
    const u64 stride = of_a ? stride_a : stride_b;        // PACKED: bytes of a row block
    const u64 end = of_a ? A.end : B.end;
    const u64 step = mode == PACKED ? CK * 1024u : mode == ROWS ? CK * 32u : (u64)CK * 32u * ld;
    // this wave's first row (or the last there is), and offsets from there
    const u32 row0 = mode == PACKED || rb0 * 32 < rows ? rb0 * 32 : rows - 1;
    u64 base = (of_a ? A.base : B.base) + (mode == PACKED ? rb0 * stride : mode == ROWS ? (u64)row0 * ld * 2u : 0u);
    u32 off[Q][CK], first[CK], left = of_a ? A.K : B.K;
#pragma unroll
    for (u32 c = 0; c < CK; c++) {
        first[c] = mode == PACKED ? 0 : mode == ROWS ? (c >> 1) * 32 + ((lane & 3u) ^ (lane >> 4)) * 8 : c * 16 + (lane >> 2);
#pragma unroll
        for (u32 q = 0; q < Q; q++) {
            if (mode == PACKED) off[q][c] = (u32)(q * stride) + c * 1024u + lane * 16u;
            else if (mode == ROWS) {
                const u32 r = (rb0 + q) * 32 + (c & 1u) * 16 + (lane >> 2);
                off[q][c] = (((r < rows ? r : rows - 1) - row0) * ld + first[c]) * 2u;
            } else {
                const u32 r = (rb0 + q) * 32 + (lane & 3u) * 8;
                off[q][c] = (first[c] * ld + (r < rows ? r : rows - 8)) * 2u;
            }
        }
    }
    // Past the last stage too, for no one to read, so that the count of loads
    // in flight stays the same.
    auto bring = [&](u32 buf, u32 m) {       // the m-th chunk
        const u32 q = m / CK, c = m % CK;
        const u32 dst = (u32)(uintptr_t)(lptr)lds + (buf * TL::STAGE + ((wave * Q + q) * CK + c) * 512u) * 2u;
        const u32 room = end <= base ? 0u : end - base > 0xFFFFFFE0u ? 0xFFFFFFE0u : (u32)(end - base);
        const u32 at = first[c] < left ? off[q][c] : 0xFFFFFFF0u;      // past any room
        // Written out, so that the compiler does not know of it: it would wait
        // for every load to LDS ahead of each turning read. It has no result
        // in a register, and wait_stage and the barriers order it.
        const i4v where = {(int)(u32)base, (int)(u32)(base >> 32), (int)room, 0x00020000};
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"     // m0 is written on purpose
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(dst), "v"(at), "s"(where) : "memory", "m0");
#pragma clang diagnostic pop
        if (m == TL::CH - 1) {
            base += step;
            left = left > CK / PL * 16u ? left - CK / PL * 16u : 0u;
        }
    };
    h8 a[2][TL::MI][PL], b[2][TL::NI][PL];
    // the n-th fragment of unit k of a stage
    constexpr u32 FRAGS = (TL::MI + TL::NI) * PL;
    const u32 turned = (lane & 31u) * 32u + ((lane >> 5) ^ ((lane >> 2) & 3u)) * 8u;                             // ROWS, in elements
    const u32 across = ((lane >> 5) * 8 + ((lane & 15u) >> 2)) * 32u + ((lane >> 4) & 1u) * 16 + (lane & 3u) * 4;  // COLS
    auto fragment = [&](auto how, const f16 *block, u32 chunk) -> h8 {
        constexpr u32 mode = decltype(how)::value;
        if constexpr (mode == PACKED) return *(const h8 *)(block + chunk * 512u + lane * 8u);
        else if constexpr (mode == ROWS) return *(const h8 *)(block + (chunk >> 1) * 1024u + (chunk & 1u ? turned ^ 16u : turned));
        else {
            typedef __attribute__((address_space(3))) s4v *p;
            const u32 at = (u32)(uintptr_t)(lptr)block + (chunk * 512u + across) * 2u;
            const h4 lo = __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((p)(uintptr_t)at));
            const h4 hi = __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((p)(uintptr_t)(at + 256u)));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    };
    auto fetch = [&](u32 buf, u32 k, u32 n, h8 (&fa)[TL::MI][PL], h8 (&fb)[TL::NI][PL]) {
        const f16 *st = lds + buf * TL::STAGE;
        const u32 p = n / (TL::MI + TL::NI), x = n % (TL::MI + TL::NI);
        if (x < TL::NI) fb[x][p] = fragment(Const<MB>{}, st + (TL::RBA + wn * TL::NI + x) * (CK * 512u), k * PL + p);
        else fa[x - TL::NI][p] = fragment(Const<MA>{}, st + (wm * TL::MI + x - TL::NI) * (CK * 512u), k * PL + p);
    };
    // The products of a unit (hi hi, then hi lo and lo hi), between them the
    // reads of the next unit's fragments and, where a stage has begun, the
    // loads of a stage to come. Left alone, the compiler puts the reads last;
    // loads issued in one go hold the wave up until the address unit has
    // taken them all, and the matrix unit waits.
    // The reads come early, for the last one's latency to pass as well.
    constexpr u32 MFMAS = TL::MI * TL::NI * (2 * PL - 1), RP = FRAGS * 2 > MFMAS ? 2 : 1;
    auto unit = [&](auto fresh, u32 buf, u32 into, u32 u, const h8 (&fa)[TL::MI][PL], const h8 (&fb)[TL::NI][PL], h8 (&na)[TL::MI][PL],
                    h8 (&nb)[TL::NI][PL]) {
        constexpr u32 LOADS = decltype(fresh)::value ? TL::CH : 0;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (u32 m = 0; m < MFMAS; m++) {
            const u32 t = m / (TL::MI * TL::NI), i = m / TL::NI % TL::MI, j = m % TL::NI;
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[i][t >> 1], fb[j][t & 1], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
#pragma unroll
            for (u32 f = m * RP; f < (m + 1) * RP && f < FRAGS; f++) {
                fetch(buf, u, f, na, nb);
                if ((f % (TL::MI + TL::NI) < TL::NI ? MB : MA) == COLS) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                else __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
#pragma unroll
            for (u32 f = m * LOADS / MFMAS; f < (m + 1) * LOADS / MFMAS; f++) {
                bring(into, f);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (u32 i = 0; i + 1 < NS; i++)
#pragma unroll
        for (u32 f = 0; f < TL::CH; f++) bring(i, f);
    wait_stage<(NS - 2) * TL::CH, 0>();
#pragma unroll
    for (u32 f = 0; f < FRAGS; f++) fetch(0, 0, f, a[0], b[0]);
    for (u32 s = 0, buf = 0; s < n; s += TL::TURN) {
#pragma unroll
        for (u32 u = 0; u < TL::US * TL::TURN; u++) {
            if ((u + 1) % TL::US == 0) {       // the next unit begins a stage
                wait_stage<(NS - 3) * TL::CH, TL::READS>();
                const u32 into = (buf + NS - 1) & (NS - 1);
                buf = (buf + 1) & (NS - 1);
                unit(Const<1>{}, buf, into, 0, a[u & 1], b[u & 1], a[(u + 1) & 1], b[(u + 1) & 1]);
            } else unit(Const<0>{}, buf, 0, u + 1, a[u & 1], b[u & 1], a[(u + 1) & 1], b[(u + 1) & 1]);
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

// ---- outputs computed again ----

// Values k .. k + 15 of row r of an operand as the caller has it, zeros from
// `end` on. Loads have no conditions, which would part them: past the end they
// read the last value.
template <typename T>
__device__ __forceinline__ void origin16(const Origin &o, u32 r, u32 k, u32 end, float (&v)[16]) {
    const glob<T> *p = (const glob<T> *)o.p + (u64)r * o.row, *z = (const glob<T> *)o.z + (u64)r * o.row;
    const bool whole = k + 16 <= end;
    float at[16];
    auto each = [&](const glob<T> *from, float (&to)[16]) {
        if (o.step == 1 && whole) {
#pragma unroll
            for (u32 j = 0; j < 16; j += 4) {
                const any_vec<T, 4> q = *(const glob<any_vec<T, 4>> *)(from + k + j);
#pragma unroll
                for (u32 i = 0; i < 4; i++) to[j + i] = (float)q[i];
            }
        } else
#pragma unroll
            for (u32 j = 0; j < 16; j++) to[j] = (float)from[(u64)(k + j < end ? k + j : end - 1) * o.step];
    };
    each(p, v);
    if (o.z) {
        each(z, at);
        slope_n<16>(o.act, at, v);
    }
    if (!whole)
#pragma unroll
        for (u32 j = 0; j < 16; j++) v[j] = k + j < end ? v[j] : 0.0f;
}

// A 32 x 32 block of the product from the operands as the caller has them, on
// the 32-bit matrix instruction, by one wave: what 32-bit sums of 32-bit
// products make of infinities and NaN. Of 32 k lane half h holds k = 16 h .. +
// 15; they are asked for while the 32 before are multiplied.
template <typename T>
__device__ __forceinline__ f16v block_again(const GemmArgs &a, u32 rb, u32 cb) {
    const u32 lane = threadIdx.x & 63u, h = (lane >> 5) * 16, r = rb + (lane & 31u), c = cb + (lane & 31u);
    const u32 ra = r < a.M ? r : a.M - 1, rc = c < a.N ? c : a.N - 1;
    f16v acc = 0.0f;
    float x[16] = {}, w[16] = {}, x1[16], w1[16];
    if (!a.K) return acc;
#pragma unroll 1
    for (u32 k = 0; k < a.K + 32; k += 32) {
        origin16<T>(a.oa, ra, k + h, a.K, x1);
        origin16<T>(a.ob, rc, k + h, a.K, w1);
#pragma unroll
        for (u32 j = 0; j < 16; j++) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], w[j], acc, 0, 0, 0);
#pragma unroll
        for (u32 j = 0; j < 16; j++) x[j] = x1[j], w[j] = w1[j];
    }
    return acc;
}

// A wave's staged strip of 32 rows: small sums of faint values stand where the
// products' magnitudes (up to as many as it takes to say so) add up to enough,
// or where no product is other than 0; the others become NaN, to be computed
// again. A value's magnitude is that of hi, and lo's where hi is 0, which are
// not both 0 (count_faint).
template <typename TL>
__device__ __forceinline__ void weigh_doubtful(const GemmArgs &a, float *st, u32 rb, u32 cb) {
    const u32 lane = threadIdx.x & 63u, h = (lane >> 5) * 4;
    const float unit = faint_unit(a.K);
    typedef unsigned short us8 __attribute__((ext_vector_type(8)));
    auto magnitude = [](const glob<f16> *p) {
        const us8 hi = *(const glob<us8> *)p & (unsigned short)0x7FFF, lo = *(const glob<us8> *)(p + 512) & (unsigned short)0x7FFF;
        return __builtin_bit_cast(h8, __builtin_elementwise_max(hi, lo));
    };
#pragma unroll 1
    for (u32 j = 0; j < TL::NI; j++, cb += 32) {
        const glob<Row> *row = (const glob<Row> *)a.ea + rb + h;
        const Row col = ((const glob<Row> *)a.eb)[cb + (lane & 31u)];
        float *at = st + h * TL::PITCH + j * 32 + (lane & 31u);
        u32 open = 0, most = 0;
#pragma unroll
        for (u32 t = 0; t < 16; t++) {
            const u32 r = (t >> 2) * 8 + (t & 3u);
            const Row w = row[r];
            open |= doubtful(w, col, unit, at[r * TL::PITCH]) ? 1u << t : 0u;
            most = max(most, (u32)w.y + (u32)col.y);
        }
        const float enough = (float)most * unit;
        const glob<f16> *A = (const glob<f16> *)a.A + block_at<TL::PL>(rb >> 5, 0, a.KB, 0) + lane * 8u;
        const glob<f16> *B = (const glob<f16> *)a.B + block_at<TL::PL>(cb >> 5, 0, a.KB, 0) + lane * 8u;
        f16v sum = 0.0f;
#pragma unroll 1
        for (u32 kb = 0; kb < a.KB && __ballot(open != 0); kb += 2) {
            h8 x[2], w[2];
#pragma unroll
            for (u32 q = 0; q < 2; q++) x[q] = magnitude(A + q * (TL::PL * 512u)), w[q] = magnitude(B + q * (TL::PL * 512u));
#pragma unroll
            for (u32 q = 0; q < 2; q++) sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[q], w[q], sum, 0, 0, 0);
            A += TL::PL * 1024u, B += TL::PL * 1024u;
#pragma unroll
            for (u32 t = 0; t < 16; t++) open &= sum[t] >= enough ? ~(1u << t) : ~0u;
        }
#pragma unroll
        for (u32 t = 0; t < 16; t++)
            if (((open >> t) & 1u) && sum[t] > 0.0f) at[((t >> 2) * 8 + (t & 3u)) * TL::PITCH] = __builtin_nanf("");
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Whether 8 sums are finite (or not, if they add up to over 2^128).
__device__ __forceinline__ bool all_finite(const float *v) {
    return fabsf(((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]))) < __builtin_inff();
}

// What an output becomes: z = sum (+ bias), y = act(z) (+ residual).
template <typename T>
__device__ __forceinline__ void finish1(const GemmArgs &a, u32 r, u32 c, float v) {
    const u64 at = (u64)r * a.N + c;
    if (a.bias) v += (float)((const glob<T> *)a.bias)[c];
    if (a.z) ((glob<T> *)a.z)[at] = (T)v;
    v = act_of(a.act, v);
    if (a.res) v += (float)((const glob<T> *)a.res)[at];
    ((glob<T> *)a.out)[at] = (T)v;
}

// The operand of a tile that begins at row r0, from stage s0 on.
template <typename TL, u32 M>
__device__ __forceinline__ Operand operand(u64 p, u32 ld, u32 rows, u32 r0, u32 KB, u32 K, u32 s0) {
    Operand o;
    const u64 k0 = (u64)s0 * (TL::US * 16u);
    o.ld = ld;
    if (M == PACKED) {
        o.base = p + block_at<TL::PL>(r0 >> 5, 0, KB, 0) * 2u + (u64)s0 * (TL::CK * 1024u);
        o.end = ~0ull;        // past it: PACK_SLACK
        o.rows = 0;
        o.K = ~0u;
    } else {
        o.base = p + (M == ROWS ? (u64)r0 * ld + k0 : k0 * ld + r0) * 2u;
        o.end = p + (M == ROWS ? (u64)rows : (u64)K) * ld * 2u;
        o.rows = rows - r0;
        o.K = K > k0 ? K - (u32)k0 : 0u;
    }
    return o;
}

// ---- sums that several workgroups have parts of ----
//
// Each writes its part through to memory (sc1: the scope of the whole card,
// whose L2 caches do not see each other's lines), waits until it is there,
// and counts itself; the last to come adds all parts, its own at its place,
// in their order, so the bits do not depend on which one that is. It leaves
// the count at 0 for the next launch. No workgroup waits for another.
#define SC1 16
typedef u32 u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void put_part(u64 base, u32 at, f4 v) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, v), __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, 0x7FFFFFFF, 0x00020000),
                                           at, 0, SC1);
}
__device__ __forceinline__ f4 get_part(u64 base, u32 at) {
    return __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(
        __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, 0x7FFFFFFF, 0x00020000), at, 0, SC1));
}

// Whether this workgroup is the last of n to come.
__device__ __forceinline__ bool last_of(u64 count, u32 n) {
    __shared__ u32 before;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        u32 *c = (u32 *)count;
        before = __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (before == n - 1) __hip_atomic_store(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return before == n - 1;
}

// A tile's sums over all K splits: part s of tile t lies at (t splits + s)
// times the tile's size, as the lanes hold it.
template <typename TL>
__device__ __forceinline__ bool join_splits(u64 part, u64 count, u32 tile, u32 split, u32 splits, f16v (&acc)[TL::MI][TL::NI]) {
    constexpr u32 BYTES = TL::TM * TL::TN * 4;
    const u64 base = part + (u64)tile * splits * BYTES;
    const u32 lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const u32 at = wave * (TL::MI * TL::NI * 4096u) + lane * 16u;
#pragma unroll
    for (u32 i = 0; i < TL::MI; i++)
#pragma unroll
        for (u32 j = 0; j < TL::NI; j++)
#pragma unroll
            for (u32 q = 0; q < 4; q++)
                put_part(base + (u64)split * BYTES, at + (i * TL::NI + j) * 4096u + q * 1024u,
                         f4{acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2], acc[i][j][q * 4 + 3]});
    if (!last_of(count + tile * 4ull, splits)) return false;
#pragma unroll
    for (u32 i = 0; i < TL::MI; i++) {
        f16v sum[TL::NI];
#pragma unroll
        for (u32 j = 0; j < TL::NI; j++) sum[j] = 0.0f;
#pragma unroll 2
        for (u32 s = 0; s < splits; s++) {
            f4 p[TL::NI][4];
#pragma unroll
            for (u32 j = 0; j < TL::NI; j++)
#pragma unroll
                for (u32 q = 0; q < 4; q++) p[j][q] = get_part(base + (u64)s * BYTES, at + (i * TL::NI + j) * 4096u + q * 1024u);
#pragma unroll
            for (u32 j = 0; j < TL::NI; j++)
#pragma unroll
                for (u32 v = 0; v < 16; v++) sum[j][v] += p[j][v >> 2][v & 3];
        }
#pragma unroll
        for (u32 j = 0; j < TL::NI; j++) acc[i][j] = sum[j];
    }
    return true;
}

// A tile of one product, or of one of its K splits (blockIdx.y).
template <typename TL, typename T, u32 MA, u32 MB>
__device__ __forceinline__ void gemm_tile(const GemmArgs &a, f16 *lds) {
    const u32 wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    u32 ti, tj;
    tile_of(blockIdx.x, a.tm, a.tn, ti, tj);
    const u32 S = a.KB / TL::US, per = (S / TL::TURN + a.splits - 1) / a.splits * TL::TURN, s0 = blockIdx.y * per;
    const u32 s1 = s0 + per < S ? s0 + per : S;
    // a gradient whose 16-bit dz are infinities where dy act'(z) is not (asked for early)
    constexpr bool PACKED16 = TL::PL == 1 && MA == PACKED;
    const u32 past = PACKED16 && a.past16 ? *(const glob<u32> *)a.past16 : 0u;
    f16v acc[TL::MI][TL::NI];
    const Operand A = operand<TL, MA>(a.A, a.lda, a.M, ti * TL::TM, a.KB, a.K, s0);
    const Operand B = operand<TL, MB>(a.B, a.ldb, a.N, tj * TL::TN, a.KB, a.K, s0);
    mainloop<TL, MA, MB>(lds, A, B, (u64)a.KB * TL::PL * 1024u, (u64)a.KB * TL::PL * 1024u, s0 < s1 ? s1 - s0 : 0, acc);
    wait_stage<0, 0>();
    if (a.splits > 1 && !join_splits<TL>(a.part, a.count, blockIdx.x, blockIdx.y, a.splits, acc)) return;
    // A lane keeps 8 columns and takes every RPP-th row of them. The residual
    // of a 32-row block is asked for before the block ahead of it is finished.
    constexpr u32 LPR = TL::NI * 4, RPP = 64 / LPR, PASSES = 32 / RPP;
    const u32 lane = threadIdx.x & 63u, dc = (lane % LPR) * 8, c = tj * TL::TN + (wave % TL::WN) * TL::NI * 32 + dc;
    const u32 r0 = ti * TL::TM + (wave / TL::WN) * TL::MI * 32 + lane / LPR;
    float *st = (float *)lds + wave * 32 * TL::PITCH;
    const float *row = st + (lane / LPR) * TL::PITCH + dc;
    const bool whole = c + 8 <= a.N;
    float bias[8];
    int ec[8];
    u32 nc = 0;            // the columns' most faint values
    const float unit = faint_unit(a.K);
    u32 later[TL::MI];      // outputs of row block i that are not finished yet: bit 8 p + j
    if (a.bias) load8<T>((const glob<T> *)a.bias, c, a.N, bias);
    if (TL::PL == 2)
#pragma unroll
        for (u32 j = 0; j < 8; j++) {
            const Row w = ((const glob<Row> *)a.eb)[c + j];
            ec[j] = w.x;
            nc = max(nc, (u32)w.y);
        }
    // (with both, the largest 32-bit tile would not fit the registers)
    constexpr bool AHEAD = TL::PL == 1 || TL::MI < 4;
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
        if (AHEAD && i + 1 < TL::MI) ask(i + 1, res[(i + 1) & 1]);
        if (!AHEAD && i) ask(i, res[i & 1]);
        Row rows[PASSES];
        if (TL::PL == 2 && AHEAD)
#pragma unroll
            for (u32 p = 0; p < PASSES; p++) rows[p] = ((const glob<Row> *)a.ea)[r0 + i * 32 + p * RPP];      // there are whole tiles of them
        stage_rows<TL>(st, acc[i]);
        later[i] = 0;
        // groups of 8 columns with sums that are computed again (not finite ones
        // by now): known for all rows ahead of the rest, which has no branches for it
        u32 odd = 0;
        float all[PASSES][8];
        auto read = [&]() {
#pragma unroll
            for (u32 p = 0; p < PASSES; p++) {
                *(f4 *)all[p] = *(const f4 *)(row + p * RPP * TL::PITCH);
                *(f4 *)(all[p] + 4) = *(const f4 *)(row + p * RPP * TL::PITCH + 4);
            }
        };
        auto look = [&]() {
            odd = 0;
#pragma unroll
            for (u32 p = 0; p < PASSES; p++) odd |= !all_finite(all[p]) ? 1u << p : 0u;
        };
        read();
        if (TL::PL == 2) {
            bool small = false, doubt = false;
#pragma unroll
            for (u32 p = 0; p < PASSES; p++) {
                if (!AHEAD) rows[p] = ((const glob<Row> *)a.ea)[r0 + i * 32 + p * RPP];
                float least = fabsf(all[p][0]);
#pragma unroll
                for (u32 j = 1; j < 8; j++) least = fminf(least, fabsf(all[p][j]));
                small |= least < (float)((u32)rows[p].y + nc) * unit;
            }
            look();
            if (__builtin_expect(__ballot(small) != 0, 0)) {
#pragma unroll
                for (u32 j = 0; j < 8; j++) {
                    const Row w = ((const glob<Row> *)a.eb)[c + j];
#pragma unroll
                    for (u32 p = 0; p < PASSES; p++) doubt |= doubtful(rows[p], w, unit, all[p][j]);
                }
                if (__ballot(doubt)) {
                    weigh_doubtful<TL>(a, st, ti * TL::TM + ((wave / TL::WN) * TL::MI + i) * 32, tj * TL::TN + (wave % TL::WN) * TL::NI * 32);
                    read();
                    look();
                }
            }
        } else if (PACKED16 && __builtin_expect(past && past == a.call, 0)) look();
#pragma unroll
        for (u32 p = 0; p < PASSES; p++) {
            const u32 r = r0 + i * 32 + p * RPP;
            if (r >= a.M || c >= a.N || ((odd >> p) & 1u)) continue;
            float (&v)[8] = all[p];
            if (TL::PL == 2)
#pragma unroll
                for (u32 j = 0; j < 8; j++) v[j] = ldexpf(v[j], -(rows[p].x + ec[j]));
            if (a.bias)
#pragma unroll
                for (u32 j = 0; j < 8; j++) v[j] += bias[j];
            const u64 at = (u64)r * a.N;
            if (a.z) store8<T>((glob<T> *)a.z + at, c, a.N, v);
            act_n<8>(a.act, v);
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
        if ((TL::PL == 2 || PACKED16) && __builtin_expect(__ballot(odd != 0) != 0, 0))
            // one by one, those that stand
#pragma unroll 1
            for (u32 b = 0; b < PASSES * 8; b++) {
                const u32 r = r0 + i * 32 + b / 8 * RPP;
                if (!((odd >> b / 8) & 1u) || r >= a.M || c + b % 8 >= a.N) continue;
                const float x = row[b / 8 * RPP * TL::PITCH + b % 8];
                if (fabsf(x) < __builtin_inff())
                    finish1<T>(a, r, c + b % 8, TL::PL == 1 ? x : ldexpf(x, -(((const glob<Row> *)a.ea)[r].x + ((const glob<Row> *)a.eb)[c + b % 8].x)));
                else later[i] |= 1u << b;
            }
    }
    u32 any = 0;
#pragma unroll
    for (u32 i = 0; i < TL::MI; i++) any |= later[i];
    if ((TL::PL == 2 || PACKED16) && __builtin_expect(__ballot(any != 0) != 0, 0))
#pragma unroll 1
        for (u32 i = 0; i < TL::MI; i++) {
            u32 mine = later[0];
#pragma unroll
            for (u32 q = 1; q < TL::MI; q++) mine = q == i ? later[q] : mine;
            if (!__ballot(mine != 0)) continue;
            const u32 rb = ti * TL::TM + ((wave / TL::WN) * TL::MI + i) * 32, cb = tj * TL::TN + (wave % TL::WN) * TL::NI * 32;
#pragma unroll 1
            for (u32 j = 0; j < TL::NI; j++) {
                if (!__ballot(mine != 0 && dc / 32 == j)) continue;
                const f16v again = block_again<T>(a, rb, cb + j * 32);
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (u32 v = 0; v < 16; v++) st[((v >> 2) * 8 + (lane >> 5) * 4 + (v & 3)) * TL::PITCH + j * 32 + (lane & 31u)] = again[v];
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
            for (u32 b = 0; b < PASSES * 8; b++)
                if ((mine >> b) & 1u) finish1<T>(a, r0 + i * 32 + b / 8 * RPP, c + b % 8, row[b / 8 * RPP * TL::PITCH + b % 8]);
            __builtin_amdgcn_wave_barrier();
        }
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
// parameter instead: p = keep * p - step * new, along its rows. Of 4096 x 4096 in
// f32 188 us a symmetric product (192 x 192 tiles, 253 of them on 256 compute
// units; the whole product takes 328), of 128 x 128 4.8 us, a launch and the
// latencies of loads, four stages and the store.
template <typename TL, typename T>
__device__ __forceinline__ void ns_tile(const NsArgs &a, f16 *lds) {
    constexpr u32 PL = TL::PL;
    const u32 lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const u64 z = blockIdx.z;
    u32 ti, tj;
    if (a.sym) tile_upper(blockIdx.x, ti, tj);
    else tile_of(blockIdx.x, a.tm, a.tn, ti, tj);
    f16v acc[TL::MI][TL::NI];
    const u32 S = a.KU / TL::US, per = (S / TL::TURN + a.splits - 1) / a.splits * TL::TURN, s0 = blockIdx.y * per;
    const u32 s1 = s0 + per < S ? s0 + per : S;
    const Operand A = operand<TL, PACKED>(a.A + z * a.stride, 0, 0, ti * TL::TM, a.KB, 0, s0);
    const Operand B = operand<TL, PACKED>(a.B + z * a.stride, 0, 0, tj * TL::TN, a.KB, 0, s0);
    mainloop<TL, PACKED, PACKED>(lds, A, B, (u64)a.KB * PL * 1024u, (u64)a.KB * PL * 1024u, s0 < s1 ? s1 - s0 : 0, acc);
    wait_stage<0, 0>();
    if (a.splits > 1 && !join_splits<TL>(a.part, a.count, blockIdx.z * gridDim.x + blockIdx.x, blockIdx.y, a.splits, acc)) return;
    float *st = (float *)lds + wave * 32 * TL::PITCH;
    const glob<f16> *old = (const glob<f16> *)(a.old + z * a.stride);
    glob<f16> *out = (glob<f16> *)(a.out + z * a.stride), *out_t = (glob<f16> *)(a.out_t + z * a.stride);
    const bool mirror = a.out_t && !(a.sym && ti == tj);
#pragma unroll
    for (u32 i = 0; i < TL::MI; i++) {
        const u32 r0 = ti * TL::TM + ((wave / TL::WN) * TL::MI + i) * 32;
        const u32 c0 = tj * TL::TN + (wave % TL::WN) * TL::NI * 32;
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

// the exponent of a row whose largest magnitude's bits are w: of a row with an
// infinity or NaN, whose products are not finite whatever it is, 0
__device__ __forceinline__ int exp_of(u32 w) { return w && w < 0x7F800000u ? 14 - ilogbf(__uint_as_float(w)) : 0; }

// The matrix of a set that a workgroup works on.
__device__ __forceinline__ u32 pack_of(const PackSet &s, u32 block) {
    return (s.n > 1 && block >= s.first[1]) + (s.n > 2 && block >= s.first[2]);
}

// What is packed at (r, c .. c + N - 1): the matrix itself, or dy * act'(z).
template <typename T, u32 N>
__device__ __forceinline__ void source(const PackArgs &a, u32 r, u32 c, float *v) {
    load_n<T, N>((const glob<T> *)a.src + (u64)r * a.C, c, a.C, v);
    if (a.z) {
        float z[N];
        load_n<T, N>((const glob<T> *)a.z + (u64)r * a.C, c, a.C, z);
        slope_n<N>(a.act, z, v);
    }
}

// The largest values of a matrix's rows and columns (as the bits of their
// magnitudes, which compare as they do, with infinities and NaN the largest of
// all; a part a column tile of 512 and a row tile of a.rt) and the columns'
// sums. 8 waves, each every 8th row of the tile, a lane 8 columns; two rows are
// asked for at a time. Bound by memory: three matrices of 4096 x 4096, one with
// its act', 63 us, 4.2 TB/s.
template <typename T>
__device__ __forceinline__ void pack_sizes_of(const PackArgs &a, u32 bx, u32 by, u32 (*lw)[512], float (*ls)[512]) {
    const u32 lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const u32 c = bx * 512u + lane * 8u;
    const u64 r0 = (u64)by * a.rt, r1 = r0 + a.rt < a.R ? r0 + a.rt : a.R;
    u32 cw[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    float cs[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (u64 r = r0 + wave; r < r1; r += 16) {
        float v[2][8];
#pragma unroll
        for (u32 q = 0; q < 2; q++)
            if (r + q * 8 < r1 && c < a.C) source<T, 8>(a, (u32)r + q * 8, c, v[q]);
            else
#pragma unroll
                for (u32 j = 0; j < 8; j++) v[q][j] = 0.0f;
#pragma unroll
        for (u32 q = 0; q < 2; q++) {
            u32 rw = 0;
#pragma unroll
            for (u32 j = 0; j < 8; j++) {
                const u32 w = __float_as_uint(v[q][j]) & 0x7FFFFFFFu;
                rw = max(rw, w);
                cw[j] = max(cw[j], w);
                cs[j] += v[q][j];
            }
            if (a.row_part && r + q * 8 < r1) {
#pragma unroll
                for (int d = 32; d; d >>= 1) rw = max(rw, (u32)__shfl_xor(rw, d));
                if (lane == 0) ((glob<u32> *)a.row_part)[(u64)bx * a.R + r + q * 8] = rw;
            }
        }
    }
#pragma unroll
    for (u32 j = 0; j < 8; j++) lw[wave][lane * 8 + j] = cw[j], ls[wave][lane * 8 + j] = cs[j];
}

template <typename T>
__device__ __forceinline__ void pack_sizes(const PackArgs &a, u32 block) {
    __shared__ u32 lw[8][512];
    __shared__ float ls[8][512];
    const u32 threads = max(a.row_parts * a.col_parts, 1u) * 512u;
    for (u32 i = block * 512u + threadIdx.x; i < a.Rn; i += threads) ((glob<u32> *)a.en)[2u * i + 1u] = 0;
    for (u32 i = block * 512u + threadIdx.x; i < a.Ct; i += threads) ((glob<u32> *)a.et)[2u * i + 1u] = 0;
    if (!a.R || !a.C) return;
    const u32 bx = block % a.row_parts, by = block / a.row_parts;
    pack_sizes_of<T>(a, bx, by, lw, ls);
    __syncthreads();
    const u32 t = threadIdx.x, ct = bx * 512u + t;
    if (ct >= a.C || (!a.col_part && !a.sum_part)) return;
    u32 w = lw[0][t];
    float s = ls[0][t];
#pragma unroll
    for (u32 k = 1; k < 8; k++) w = max(w, lw[k][t]), s += ls[k][t];
    if (a.col_part) ((glob<u32> *)a.col_part)[(u64)by * a.C + ct] = w;
    if (a.sum_part) ((glob<float> *)a.sum_part)[(u64)by * a.C + ct] = s;
}

// The faint ones of 8 values of row r, for its count (pack_sizes has cleared
// it). Those that the planes would not hold
// at all become the least that they hold. Shifted left, magnitudes lose their
// sign and compare as before, and 0 less 1 is the largest of all.
__device__ __forceinline__ void count_faint(u64 words, u32 r, float *v) {
    constexpr u32 faint = (0x3E800000u << 1) - 1u;      // 2^-2
    u32 least = ~0u;
#pragma unroll
    for (u32 j = 0; j < 8; j++) least = min(least, (__float_as_uint(v[j]) << 1) - 1u);
    if (least >= faint) return;
    u32 n = 0;
#pragma unroll
    for (u32 j = 0; j < 8; j++)
        if ((__float_as_uint(v[j]) << 1) - 1u < faint) {
            n++;
            v[j] = copysignf(fmaxf(fabsf(v[j]), 5.9604645e-8f), v[j]);      // 2^-24
        }
    __hip_atomic_fetch_add((u32 *)words + 2u * r + 1u, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A 64 x 64 tile of a matrix [R][C] into one or both packed orientations:
// pn (rows r, k = c) and pt (rows c, k = r). 32-bit values are scaled by the
// exponents of their packed row; `unit` (the optimiser) by one factor.
// MUON: the source is u (muon_momentum) over its norm. Bound by memory: the same
// three matrices, one of them into both orientations, 104 us, 5.2 TB/s.
template <u32 PL, typename T, bool MUON>
__device__ __forceinline__ void pack_tile(const PackArgs &a, const MuonArgs *mu, u32 block) {
    __shared__ float tile[64][65];
    __shared__ int er[64], ec[64];
    __shared__ float unit_lds;
    const u32 t = threadIdx.x, r0 = (block / a.ctiles) * 64u, c0 = (block % a.ctiles) * 64u, zi = MUON ? blockIdx.y : 0u;
    if (PL == 2 && !MUON) {
        // the parts of this tile's rows and columns, four lanes to each
        const u32 i = t >> 2, q = t & 3u;
        u32 wr = 0, wc = 0;
        if (a.pn && r0 + i < a.R)
            for (u32 p = q; p < a.row_parts; p += 4) wr = max(wr, (u32)((const glob<u32> *)a.row_part)[(u64)p * a.R + r0 + i]);
        if (a.pt && c0 + i < a.C)
            for (u32 p = q; p < a.col_parts; p += 4) wc = max(wc, (u32)((const glob<u32> *)a.col_part)[(u64)p * a.C + c0 + i]);
        wr = max(wr, (u32)__shfl_xor(wr, 1));
        wc = max(wc, (u32)__shfl_xor(wc, 1));
        wr = max(wr, (u32)__shfl_xor(wr, 2));
        wc = max(wc, (u32)__shfl_xor(wc, 2));
        if (q == 0) {
            er[i] = exp_of(wr);
            ec[i] = exp_of(wc);
            if (a.pn && c0 == 0 && r0 + i < a.Rn) ((glob<int> *)a.en)[2u * (r0 + i)] = wr ? er[i] : ROW_EMPTY;
            if (a.pt && r0 == 0 && c0 + i < a.Ct) ((glob<int> *)a.et)[2u * (c0 + i)] = wc ? ec[i] : ROW_EMPTY;
        }
    }
    if (PL == 2 && !MUON && a.sum_out && r0 == 0 && t < 64 && c0 + t < a.C) {
        // the column sums, from the parts of pack_sizes
        float s = 0.0f;
        for (u32 p = 0; p < a.col_parts; p++) s += ((const glob<float> *)a.sum_part)[(u64)p * a.C + c0 + t];
        ((glob<T> *)a.sum_out)[c0 + t] = (T)s;
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
            } else source<T, 8>(a, r, c, v);
        }
        if (PL == 1 && !MUON && a.z) {
            float most = 0.0f;
#pragma unroll
            for (u32 k = 0; k < 8; k++) most = fmaxf(most, fabsf(v[k]));
            if (most >= 65520.0f) *(glob<u32> *)a.past16 = a.call;
        }
        if (a.pt || a.sum_part)
#pragma unroll
            for (u32 k = 0; k < 8; k++) tile[i][j + k] = v[k];
        if (a.pn && r < a.Rn && c < a.KBn * 16u) {
            if (PL == 2 && !MUON)
#pragma unroll
                for (u32 k = 0; k < 8; k++) v[k] = ldexpf(v[k], er[i]);
            if (PL == 2 && !MUON) count_faint(a.en, r, v);
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
                if (PL == 2 && !MUON) v[k] = ldexpf(v[k], ec[j]);
            }
            if (PL == 2 && !MUON) count_faint(a.et, c, v);
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

// y = x W, MR rows a workgroup (blockIdx.z). W is read once a block of rows, as
// it lies ([K][N] row-major), BYTES a lane, 16 lanes along a row. Bound by W's
// bytes where W is large: 16 bytes a lane, and K split over workgroups
// (blockIdx.y) until the card is full (1 x 4096 x 4096 f16: 11.3 us, 3 TB/s with
// the launch and the join). Bound by latency where it is small: 4 bytes a lane,
// which makes four times the workgroups without a split to join (1 x 1024 x
// 1024 f32 3.8 us against 5.6, 64 x 784 x 128 5.2).
//
// Products are 32-bit ones. One row: on the vector unit, the workgroup's 8 waves
// 32 rows of W at a time, U of a lane's loads on their way while U are
// multiplied, the split's part of x in LDS from the start. 16 rows: on the
// 32-bit matrix instruction (v_mfma_f32_16x16x4_f32: lane l holds k = l / 16 of
// row, or column, l % 16), one for each of a lane's columns and k. A wave takes
// 16 k of a unit of 128, lane group q its k = 4 q .. + 3, so that x too comes
// from memory in vectors of 4 k and neither LDS nor a barrier stands ahead of
// the sums; D units are on their way.
template <typename T, u32 MR, u32 BYTES>
__device__ __forceinline__ void few_rows(const GemmArgs &a) {
    constexpr u32 N = BYTES / sizeof(T), WAVES = 8, COLS = 16 * N, OUT = MR * COLS;
    constexpr u32 PITCH = FEW_CHUNK + 4;
    constexpr u32 XS = MR == 16 ? 0 : MR * PITCH;
    __shared__ float lds[XS > WAVES * OUT ? XS : WAVES * OUT];
    const u32 lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const u32 c = blockIdx.x * COLS + (lane & 15u) * N;
    const u32 per = a.kper, k0 = blockIdx.y * per, k1 = k0 + per < a.K ? k0 + per : a.K;
    const u32 m0 = blockIdx.z * MR, rows = a.M - m0 < MR ? a.M - m0 : MR;
    const glob<T> *W = (const glob<T> *)a.B, *X = (const glob<T> *)a.A + (u64)m0 * a.K;
    constexpr u32 R = MR < 16 ? MR : 4;      // rows of sums a lane holds
    float acc[N][R];
#pragma unroll
    for (u32 j = 0; j < N; j++)
#pragma unroll
        for (u32 r = 0; r < R; r++) acc[j][r] = 0.0f;
    // Loads have no conditions, which would part them: a lane past the last
    // columns reads the last there are, one past the last k
    // reads that, and takes 0.
    const u32 cc = c + N <= a.N ? c : a.N < N ? 0u : a.N - N;
    auto row = [&](u32 k) { return *(const glob<any_vec<T, N>> *)(W + (u64)(k < k1 ? k : k1 - 1) * a.N + cc); };
    if constexpr (MR == 16) {
        // units of 128 k; what is left of them is asked for first, and added last
        constexpr u32 D = BYTES == 4 ? 8 : 4;
        const u32 units = (k1 - k0) / 128, kr = wave * 16 + (lane >> 4) * 4, kt = k0 + units * 128 + kr;
        const glob<T> *xr = X + (u64)((lane & 15u) < rows ? lane & 15u : rows - 1) * a.K;
        any_vec<T, 4> x[D], xt;
        any_vec<T, N> w[D][4], wt[4];
        auto ask = [&](u32 u, any_vec<T, 4> &xv, any_vec<T, N> (&v)[4]) {
            const u32 k = k0 + u * 128 + kr;
            xv = *(const glob<any_vec<T, 4>> *)(xr + k);
#pragma unroll
            for (u32 i = 0; i < 4; i++) v[i] = *(const glob<any_vec<T, N>> *)(W + (u64)(k + i) * a.N + cc);
        };
        auto multiply = [&](any_vec<T, 4> xv, const any_vec<T, N> (&v)[4]) {
#pragma unroll
            for (u32 i = 0; i < 4; i++)
#pragma unroll
                for (u32 j = 0; j < N; j++) {
                    f4 t = {acc[j][0], acc[j][1], acc[j][2], acc[j][3]};
                    t = __builtin_amdgcn_mfma_f32_16x16x4f32((float)xv[i], (float)v[i][j], t, 0, 0, 0);
                    acc[j][0] = t[0], acc[j][1] = t[1], acc[j][2] = t[2], acc[j][3] = t[3];
                }
        };
        const bool rest = (k1 - k0) % 128 != 0;
        if (rest) {
#pragma unroll
            for (u32 i = 0; i < 4; i++) xt[i] = xr[kt + i < k1 ? kt + i : k1 - 1], wt[i] = row(kt + i);
        }
        if (units) {
#pragma unroll
            for (u32 d = 0; d < D; d++) ask(d < units ? d : units - 1, x[d], w[d]);
            for (u32 u = 0; u < units; u += D)
#pragma unroll
                for (u32 d = 0; d < D; d++) {
                    if (u + d < units) multiply(x[d], w[d]);
                    if (u + D < units) ask(u + D + d < units ? u + D + d : units - 1, x[d], w[d]);
                }
        }
        if (rest) {
#pragma unroll
            for (u32 i = 0; i < 4; i++) {
                xt[i] = kt + i < k1 ? xt[i] : (T)0.0f;
#pragma unroll
                for (u32 j = 0; j < N; j++) wt[i][j] = kt + i < k1 ? wt[i][j] : (T)0.0f;
            }
            multiply(xt, wt);
        }
    } else if (k0 < k1) {
        constexpr u32 U = BYTES == 4 ? 8 : 4, KSTEP = WAVES * 4;
        const u32 kr = wave * 4 + (lane >> 4);
        any_vec<T, N> w[2][U];
        auto ask = [&](u32 kb, any_vec<T, N> (&v)[U]) {
#pragma unroll
            for (u32 u = 0; u < U; u++) v[u] = row(kb + u * KSTEP + kr);
        };
        auto multiply = [&](u32 kb, const any_vec<T, N> (&v)[U]) {
#pragma unroll
            for (u32 u = 0; u < U; u++) {
                const u32 k = kb + u * KSTEP + kr;
                const float *x = lds + k - k0;
                any_vec<T, N> t = v[u];
#pragma unroll
                for (u32 j = 0; j < N; j++) t[j] = k < k1 ? t[j] : (T)0.0f;
#pragma unroll
                for (u32 r = 0; r < MR; r++)
#pragma unroll
                    for (u32 j = 0; j < N; j++) acc[j][r] = fmaf(x[r * PITCH], (float)t[j], acc[j][r]);
            }
        };
        ask(k0, w[0]);
#pragma unroll
        for (u32 r = 0; r < MR; r++)
            for (u32 k = threadIdx.x; k < per; k += 512) lds[r * PITCH + k] = r < rows && k0 + k < k1 ? (float)X[(u64)r * a.K + k0 + k] : 0.0f;
        __syncthreads();
        // per is a multiple of U * KSTEP
        for (u32 kb = k0; kb < k0 + per; kb += 2 * U * KSTEP) {
            ask(kb + U * KSTEP, w[1]);
            multiply(kb, w[0]);
            if (kb + U * KSTEP >= k0 + per) break;
            ask(kb + 2 * U * KSTEP, w[0]);
            multiply(kb + U * KSTEP, w[1]);
        }
        __syncthreads();
    }
    // the waves' sums, in order
#pragma unroll
    for (u32 r = 0; r < R; r++)
#pragma unroll
        for (u32 j = 0; j < N; j++) {
            const u32 at = cc + j - blockIdx.x * COLS;      // a lane's own columns only
            if constexpr (MR == 16) {
                if (cc + j >= c) lds[wave * OUT + ((lane >> 4) * 4 + r) * COLS + at] = acc[j][r];
            } else {
                float s = acc[j][r];
                s += __shfl_xor(s, 16);
                s += __shfl_xor(s, 32);
                if (lane < 16 && cc + j >= c) lds[wave * OUT + r * COLS + at] = s;
            }
        }
    __syncthreads();
    // a lane's outputs; what they are joined and finished with is asked for at once
    constexpr u32 PER = (OUT + 511) / 512;
    const u64 tile = (u64)blockIdx.z * gridDim.x + blockIdx.x, part = a.part + tile * a.splits * (OUT * 4u);
    float sum[PER], bias[PER], res[PER];
#pragma unroll
    for (u32 i = 0; i < PER; i++) {
        const u32 o = threadIdx.x + i * 512;
        sum[i] = lds[o % OUT];
#pragma unroll
        for (u32 q = 1; q < WAVES; q++) sum[i] += lds[q * OUT + o % OUT];
        if (a.splits > 1 && o < rows * COLS)
            __hip_atomic_store((float *)(part + ((u64)blockIdx.y * OUT + o) * 4u), sum[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (a.splits > 1 && !last_of(a.count + tile * 4u, a.splits)) return;
#pragma unroll
    for (u32 i = 0; i < PER; i++) {
        const u32 o = threadIdx.x + i * 512, r = m0 + o / COLS, col = blockIdx.x * COLS + o % COLS;
        if (o >= rows * COLS || col >= a.N) continue;
        if (a.bias) bias[i] = (float)((const glob<T> *)a.bias)[col];
        if (a.res) res[i] = (float)((const glob<T> *)a.res)[(u64)r * a.N + col];
    }
    if (a.splits > 1) {
#pragma unroll
        for (u32 i = 0; i < PER; i++) sum[i] = 0.0f;
#pragma unroll 16
        for (u32 p = 0; p < a.splits; p++)
#pragma unroll
            for (u32 i = 0; i < PER; i++)      // without a condition, which would part the loads
                sum[i] += __hip_atomic_load((const float *)(part + ((u64)p * OUT + (threadIdx.x + i * 512) % OUT) * 4u), __ATOMIC_RELAXED,
                                            __HIP_MEMORY_SCOPE_AGENT);
    }
#pragma unroll
    for (u32 i = 0; i < PER; i++) {
        const u32 o = threadIdx.x + i * 512, r = m0 + o / COLS, col = blockIdx.x * COLS + o % COLS;
        if (o >= rows * COLS || col >= a.N) continue;
        const u64 at = (u64)r * a.N + col;
        float v = a.bias ? sum[i] + bias[i] : sum[i];
        if (a.z) ((glob<T> *)a.z)[at] = (T)v;
        v = act_of(a.act, v);
        if (a.res) v += res[i];
        ((glob<T> *)a.out)[at] = (T)v;
    }
}

// ---- 32-bit products of matrices as they lie ----

// A 64 x 64 tile on the 32-bit matrix instruction (v_mfma_f32_32x32x2_f32, 64
// multiplications a cycle and compute unit where the planes' three products
// reach some 340), for sizes at which packing would take longer than that
// costs. The 4 waves of a workgroup take 16 k of 64 each and add their sums at
// the end, so nothing passes through LDS on the way in and no wave waits for
// another. Of those 16 k lane half h holds k = 8 h .. + 7: of x 8 of two rows,
// in 16-byte loads, of W two neighbouring columns at each of the 8 k. D such
// units are on their way. 128 x 4096 x 4096: 44 us, 98 TFLOP/s of the 150 that
// the instruction gives.
struct Direct {
    static constexpr u32 PITCH = 68, LDS = 4 * 64 * PITCH, D = 2;
};

// 8 k of two rows of x from k on, or of two columns of W. Past the last row or
// column a lane reads the last ones.
__device__ __forceinline__ void direct_x(const glob<float> *const (&row)[2], u32 k, float (&v)[2][8]) {
#pragma unroll
    for (u32 i = 0; i < 2; i++)
#pragma unroll
        for (u32 q = 0; q < 2; q++) {
            const any_vec<float, 4> x = *(const glob<any_vec<float, 4>> *)(row[i] + k + q * 4);
#pragma unroll
            for (u32 j = 0; j < 4; j++) v[i][q * 4 + j] = x[j];
        }
}
__device__ __forceinline__ void direct_w(const glob<float> *col, u64 ld, u32 k, float (&v)[2][8]) {
#pragma unroll
    for (u32 j = 0; j < 8; j++) {
        const any_vec<float, 2> x = *(const glob<any_vec<float, 2>> *)(col + (k + j) * ld);
        v[0][j] = x[0], v[1][j] = x[1];
    }
}

__device__ __forceinline__ void direct_tile(const GemmArgs &a, float *lds) {
    constexpr u32 D = Direct::D, PITCH = Direct::PITCH;
    const u32 lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    u32 ti, tj;
    tile_of(blockIdx.x, a.tm, a.tn, ti, tj);
    const u32 k0 = blockIdx.y * a.kper, k1 = k0 + a.kper < a.K ? k0 + a.kper : a.K;
    const u32 units = k0 < k1 ? (k1 - k0) / 64 : 0, kr = wave * 16 + (lane >> 5) * 8, kt = k0 + units * 64 + kr;
    const bool rest = k0 < k1 && (k1 - k0) % 64 != 0;
    const glob<float> *row[2];
#pragma unroll
    for (u32 i = 0; i < 2; i++) {
        const u32 r = ti * 64 + i * 32 + (lane & 31u);
        row[i] = (const glob<float> *)a.A + (u64)(r < a.M ? r : a.M - 1) * a.K;
    }
    const u32 own = tj * 64 + (lane & 31u) * 2, at = own + 2 <= a.N ? own : a.N - 2;
    const glob<float> *col = (const glob<float> *)a.B + at;
    f16v acc[2][2];
#pragma unroll
    for (u32 i = 0; i < 2; i++)
#pragma unroll
        for (u32 j = 0; j < 2; j++) acc[i][j] = 0.0f;
    float x[D][2][8], w[D][2][8], xt[2][8], wt[2][8];
    auto multiply = [&](const float (&xv)[2][8], const float (&wv)[2][8]) {
#pragma unroll
        for (u32 k = 0; k < 8; k++)
#pragma unroll
            for (u32 i = 0; i < 2; i++)
#pragma unroll
                for (u32 j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(xv[i][k], wv[j][k], acc[i][j], 0, 0, 0);
    };
    // what is left of the units is asked for first, and added last
    if (rest)
#pragma unroll
        for (u32 j = 0; j < 8; j++) {
            const u32 k = kt + j < k1 ? kt + j : k1 - 1;
            const any_vec<float, 2> v = *(const glob<any_vec<float, 2>> *)(col + (u64)k * a.N);
            xt[0][j] = row[0][k], xt[1][j] = row[1][k], wt[0][j] = v[0], wt[1][j] = v[1];
        }
    if (units) {
#pragma unroll
        for (u32 d = 0; d < D; d++) {
            const u32 k = k0 + (d < units ? d : units - 1) * 64 + kr;
            direct_x(row, k, x[d]), direct_w(col, a.N, k, w[d]);
        }
        for (u32 u = 0; u < units; u += D)
#pragma unroll
            for (u32 d = 0; d < D; d++) {
                if (u + d < units) multiply(x[d], w[d]);
                const u32 k = k0 + (u + D + d < units ? u + D + d : units - 1) * 64 + kr;
                direct_x(row, k, x[d]), direct_w(col, a.N, k, w[d]);
            }
    }
    if (rest) {
#pragma unroll
        for (u32 j = 0; j < 8; j++)
            if (kt + j >= k1) xt[0][j] = xt[1][j] = wt[0][j] = wt[1][j] = 0.0f;
        multiply(xt, wt);
    }
    // the waves' sums, in order: a lane has rows v / 4 * 8 + h * 4 + v % 4 of its columns
    float *st = lds + wave * (64 * PITCH);
#pragma unroll
    for (u32 i = 0; i < 2; i++)
#pragma unroll
        for (u32 v = 0; v < 16; v++)
#pragma unroll
            for (u32 j = 0; j < 2; j++)
                if (at + j >= own) st[(i * 32 + (v >> 2) * 8 + (lane >> 5) * 4 + (v & 3)) * PITCH + at + j - tj * 64] = acc[i][j][v];
    __syncthreads();
    const u32 dc = (threadIdx.x & 15u) * 4, dr = threadIdx.x >> 4, c = tj * 64 + dc, r0 = ti * 64 + dr;
    f4 sum[4];
#pragma unroll
    for (u32 q = 0; q < 4; q++) {
        const float *row = lds + (dr + q * 16) * PITCH + dc;
        sum[q] = *(const f4 *)row;
#pragma unroll
        for (u32 k = 1; k < 4; k++) sum[q] += *(const f4 *)(row + k * 64 * PITCH);
    }
    if (a.splits > 1) {
        const u64 base = a.part + (u64)blockIdx.x * a.splits * 16384u;
#pragma unroll
        for (u32 q = 0; q < 4; q++) put_part(base + blockIdx.y * 16384u, threadIdx.x * 16u + q * 4096u, sum[q]);
        if (!last_of(a.count + blockIdx.x * 4ull, a.splits)) return;
#pragma unroll
        for (u32 q = 0; q < 4; q++) sum[q] = f4{0, 0, 0, 0};
#pragma unroll 4
        for (u32 s = 0; s < a.splits; s++)
#pragma unroll
            for (u32 q = 0; q < 4; q++) sum[q] += get_part(base + s * 16384u, threadIdx.x * 16u + q * 4096u);
    }
    if (c >= a.N) return;
    float bias[4] = {0, 0, 0, 0}, res[4][4];
    if (a.bias) load_n<float, 4>((const glob<float> *)a.bias, c, a.N, bias);
    if (a.res)
#pragma unroll
        for (u32 q = 0; q < 4; q++)
            if (r0 + q * 16 < a.M) load_n<float, 4>((const glob<float> *)a.res + (u64)(r0 + q * 16) * a.N, c, a.N, res[q]);
#pragma unroll
    for (u32 q = 0; q < 4; q++) {
        const u32 r = r0 + q * 16;
        if (r >= a.M) break;
        float v[4];
#pragma unroll
        for (u32 j = 0; j < 4; j++) v[j] = sum[q][j] + bias[j];
        if (a.z) store_n<float, 4>((glob<float> *)a.z + (u64)r * a.N, c, a.N, v);
        act_n<4>(a.act, v);
        if (a.res)
#pragma unroll
            for (u32 j = 0; j < 4; j++) v[j] += res[q][j];
        store_n<float, 4>((glob<float> *)a.out + (u64)r * a.N, c, a.N, v);
    }
}

// ---- the kernels ----

#define GEMM(size, TILE, name, T, ...)                                                                             \
    typedef TILE Tile##size##_##name;                                                                              \
    GEMM_OF(size, name, T, , PACKED, PACKED)                                                                        \
    __VA_ARGS__
#define GEMM_OF(size, name, T, how, MA, MB)                                                                         \
    extern "C" __global__ __launch_bounds__(Tile##size##_##name::THREADS) void thvm_gemm##how##_##size##_##name(GemmArgs a) { \
        __shared__ __attribute__((aligned(1024))) f16 lds[Tile##size##_##name::LDS];                               \
        gemm_tile<Tile##size##_##name, T, MA, MB>(a, lds);                                                          \
    }
// x W with both as they lie
#define AS_THEY_LIE(size) GEMM_OF(size, f16, f16, _rc, ROWS, COLS)
#define NS(size, name, T)                                                                                          \
    extern "C" __global__ __launch_bounds__(Tile##size##_##name::THREADS) void thvm_ns_##size##_##name(NsArgs a) {  \
        __shared__ __attribute__((aligned(1024))) f16 lds[Tile##size##_##name::LDS];                               \
        ns_tile<Tile##size##_##name, T>(a, lds);                                                                    \
    }
#define TILE(...) Tile<__VA_ARGS__>
GEMM(256x256, TILE(256, 256, 2, 4, 1, 2, 4), f16, f16, AS_THEY_LIE(256x256))
GEMM(128x128, TILE(128, 128, 2, 2, 1, 4, 4), f16, f16, AS_THEY_LIE(128x128))
GEMM(64x64, TILE(64, 64, 2, 2, 1, 4, 4), f16, f16, AS_THEY_LIE(64x64))
GEMM(256x256, TILE(256, 256, 2, 4, 2, 1, 4), f32, float)
GEMM(128x128, TILE(128, 128, 2, 2, 2, 2, 4), f32, float)
GEMM(64x64, TILE(64, 64, 2, 2, 2, 2, 4), f32, float)
#undef GEMM
#define NS_TILE(size, TILE, name, T) typedef TILE Tile##size##_##name; NS(size, name, T)
NS_TILE(192x192, TILE(192, 192, 2, 2, 1, 2, 4), f16, f16)
NS_TILE(192x192, TILE(192, 192, 2, 2, 2, 1, 4), f32, float)
NS(256x256, f16, f16)
NS(128x128, f16, f16)
NS(64x64, f16, f16)
NS(256x256, f32, float)
NS(128x128, f32, float)
NS(64x64, f32, float)

#define PER_TYPE(PL, name, T)                                                                                      \
    extern "C" __global__ __launch_bounds__(256) void thvm_pack_##name(PackSet s) {                                 \
        const u32 i = pack_of(s, blockIdx.x);                                                                       \
        pack_tile<PL, T, false>(s.p[i], nullptr, blockIdx.x - s.first[i]);                                          \
    }                                                                                                              \
    extern "C" __global__ __launch_bounds__(256) void thvm_muon_pack_##name(PackArgs a, MuonArgs m) {               \
        pack_tile<PL, T, true>(a, &m, blockIdx.x);                                                                              \
    }                                                                                                              \
    extern "C" __global__ __launch_bounds__(256) void thvm_muon_momentum_##name(MuonArgs m) { muon_momentum<T>(m); } \
    extern "C" __global__ __launch_bounds__(512) void thvm_few1_##name(GemmArgs a) { few_rows<T, 1, 16>(a); }       \
    extern "C" __global__ __launch_bounds__(512) void thvm_few16_##name(GemmArgs a) { few_rows<T, 16, 16>(a); }     \
    extern "C" __global__ __launch_bounds__(512) void thvm_few1n_##name(GemmArgs a) { few_rows<T, 1, 4>(a); }       \
    extern "C" __global__ __launch_bounds__(512) void thvm_few16n_##name(GemmArgs a) { few_rows<T, 16, 4>(a); }
PER_TYPE(1, f16, f16)
PER_TYPE(2, f32, float)
// of 16-bit operands; 32-bit ones' parts are few, and added where they are packed
extern "C" __global__ __launch_bounds__(1024) void thvm_sum_parts_f16(u64 part, u64 out, u32 C, u32 parts) {
    sum_parts<f16>((const glob<float> *)part, (glob<f16> *)out, C, parts);
}
// of 32-bit operands: 16-bit ones are packed as they are
extern "C" __global__ __launch_bounds__(512, 4) void thvm_pack_sizes_f32(PackSet s) {
    const u32 i = pack_of(s, blockIdx.x);
    pack_sizes<float>(s.p[i], blockIdx.x - s.first[i]);
}
extern "C" __global__ __launch_bounds__(256) void thvm_direct_f32(GemmArgs a) {
    __shared__ __attribute__((aligned(16))) float lds[Direct::LDS];
    direct_tile(a, lds);
}
