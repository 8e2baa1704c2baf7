/*
 * block_args.h - kernel arguments of the residual block's operators (layer
 * norm, linear, their gradients, the orthogonalised step), passed by value;
 * shared by norm_kernels.hip, gemm_kernels.hip and block.c. Pointers are
 * device addresses; 0 is an absent operand.
 */
#ifndef BLOCK_ARGS_H
#define BLOCK_ARGS_H

#include "thvm_abi.h"

typedef struct {
    u64 x, gamma, beta, y, mean, rstd;
    u32 rows, cols;
    f32 eps;
    u32 pad;
} LnArgs;

typedef struct {
    u64 dy, x, mean, rstd, gamma, add, dx, dgamma, dbeta;
    u64 part;                  /* [parts][2][cols] f32: partial sums of dgamma, dbeta */
    u32 rows, cols, parts, pad;
} LnGradArgs;

/* activations: THVM_HIP_ACT_* */
enum { ACT_NONE = 0, ACT_RELU, ACT_GELU, ACT_GELU_TANH, ACT_SILU, ACT_COUNT };

/* bytes past a packed operand that a product's last loads may touch */
#define PACK_SLACK 32768

/* An operand as the caller has it: value k of row r is p[r * row + k * step]
 * (in elements; one of the two steps is 1), times act'(z) there if z is given */
typedef struct {
    u64 p, z;
    u32 row, step, act, pad;
} Origin;

/* C[M][N] = sum over k of A[r][k] B[c][k], packed operands (gemm_kernels.hip) */
typedef struct {
    u64 A, B;                  /* packed; KB blocks of 16 k */
    u64 ea, eb;                /* of each row of A and of B its exponent and number of faint values (32-bit operands) */
    Origin oa, ob;             /* what the packed operands were */
    u64 past16;                /* holds `call` if a 16-bit dz is past its type's range */
    u64 out, z, bias, res;     /* row-major [M][N]; bias [N] */
    u64 part, count;           /* the K splits' sums, and how many of a tile's are there (0 between launches) */
    u32 M, N, KB, tm, tn, splits, act;
    u32 K, lda, ldb;           /* operands as they lie */
    u32 kper;                  /* few rows: A is x [M][K], B is W [K][N], kper k a split */
    u32 call;
} GemmArgs;

/* few rows: the longest K split of a workgroup, whose part of x it holds in LDS */
#define FEW_CHUNK 1024

/* packing of a matrix [R][C] (or of dy * act'(z)) */
typedef struct {
    u64 src, z;                /* z 0: the matrix itself */
    u64 pn, pt;                /* packed with rows r (Rn of them, KBn blocks of k = c); with rows c */
    u64 en, et;                /* of each of their rows its exponent and number of faint values */
    u64 row_part, col_part;    /* the largest magnitudes' bits [row_parts][R], [col_parts][C] */
    u64 sum_part;              /* column sums [..][C] f32 */
    u64 stride;                /* bytes between the matrices of a batch in pn and pt */
    u32 R, C, act, rt;         /* rt: rows of a column part */
    u32 Rn, KBn, Ct, KBt, row_parts, col_parts;
    u64 sum_out;               /* [C]: the column sums (32-bit operands) */
    u64 past16;                /* as in GemmArgs */
    u32 ctiles, call;          /* tiles of 64 columns */
} PackArgs;

/* up to three matrices of one launch: p[i] from workgroup first[i] on */
typedef struct {
    u32 n, first[3];
    PackArgs p[3];
} PackSet;

/* the optimiser's matrices of one launch */
#define MUON_MAX 16
typedef struct {
    u64 grad[MUON_MAX], m[MUON_MAX];
    u64 sums;                  /* [count][blocks] f64: partial sums of squares */
    u64 numel;
    u32 blocks, nesterov;
    f32 beta;
    u32 pad;
} MuonArgs;

/* new = alpha old + beta A B^T over packed operands, see ns_tile */
typedef struct {
    u64 A, B, old, out, out_t; /* matrix z's operands lie z * stride bytes further */
    u64 stride, part, count;   /* part, count: as in GemmArgs, matrix by matrix */
    u64 param[MUON_MAX];
    u32 KB, KU;                /* blocks of k: in memory, and multiplied */
    u32 KBO, KBT;              /* of old and out, and of out_t */
    u32 tm, tn, sym, splits;
    u32 n, w, tall, last;
    f32 alpha, beta, keep, step;
} NsArgs;

#endif
