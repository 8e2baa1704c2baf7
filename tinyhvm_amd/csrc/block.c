/*
 * block.c - the operators of a residual feed-forward block and of its
 * training: layer norm, a linear layer with bias, activation and residual,
 * their gradients, and an orthogonalised optimiser step. Entry points of
 * thvm_hip.h with no counterpart in the engine; kernels in norm_kernels.hip
 * and gemm_kernels.hip. They take buffer ids like the Backend slots, put
 * their work on the backend's stream, and never wait on the host.
 */
#include <math.h>
#include <string.h>

#include "hipb.h"
#include "thvm_hip.h"
#include "block_args.h"

extern const unsigned char thvm_norm_kernels_co[], thvm_gemm_kernels_co[];

#define MODULES 2
#define COUNTS 4096u /* outputs of one launch whose sums several workgroups have parts of */
#define KERNELS 256 /* more than the modules have */
static struct {
    hipModule_t mod[MODULES];
    struct { char name[48]; hipFunction_t fn; } fn[KERNELS];
    u64 counts, counts_cap;     /* [COUNTS] u32: 0 between launches; and one more, see past16 */
    u32 call;                   /* of a gradient */
} B;
static Scratch block_ws;

void block_shutdown(void) {
    scratch_release(&block_ws);
    for (int i = 0; i < MODULES; i++)
        if (B.mod[i]) HIPB_CHECK(hipModuleUnload(B.mod[i]));
    pool_block_put((void *)(uintptr_t)B.counts, B.counts_cap);
    memset(&B, 0, sizeof B);
}

int block_init(void) {
    const unsigned char *co[MODULES] = {thvm_norm_kernels_co, thvm_gemm_kernels_co};
    memset(&B, 0, sizeof B);
    for (int i = 0; i < MODULES; i++) {
        hipError_t e = hipModuleLoadData(&B.mod[i], co[i]);
        if (e != hipSuccess) {
            fprintf(stderr, "tinyhvm-hip: loading an operator module failed: %s\n", hipGetErrorString(e));
            B.mod[i] = NULL;
            return -1;
        }
    }
    u32 n = COUNTS + 1, zero = 0;
    void *counts = pool_block_get(4ull * n, &B.counts_cap);
    hipFunction_t fill = rtc_static_fn("thvm_fill_u32");
    if (!counts || !fill) return -1;
    B.counts = (u64)(uintptr_t)counts;
    void *args[] = {&counts, &n, &zero};
    return hipb_launch(fill, (n + 255) / 256, 1, 1, 256, args) ? 0 : -1;
}

/* A kernel by name, looked up in the modules once. */
static hipFunction_t kernel(const char *name) {
    u32 h = 2166136261u;
    for (const char *c = name; *c; c++) h = (h ^ (u8)*c) * 16777619u;
    for (u32 p = h % KERNELS, n = 0; n < KERNELS; p = (p + 1) % KERNELS, n++) {
        if (B.fn[p].name[0] && strcmp(B.fn[p].name, name) != 0) continue;
        if (B.fn[p].name[0]) return B.fn[p].fn;
        hipFunction_t f = NULL;
        for (int i = 0; i < MODULES && !f; i++)
            if (hipModuleGetFunction(&f, B.mod[i], name) != hipSuccess) {
                (void)hipGetLastError(); /* it may be in the next module: no error of this thread's */
                f = NULL;
            }
        if (!f) {
            fprintf(stderr, "tinyhvm-hip: kernel %s not found\n", name);
            return NULL;
        }
        snprintf(B.fn[p].name, sizeof B.fn[p].name, "%s", name);
        B.fn[p].fn = f;
        return f;
    }
    return NULL;
}

/* ---- arguments ---- */

/* Two row blocks of a packed operand of this many k are reached by 32-bit
 * offsets from one address; and rows, or columns, that the launches can count. */
#define MAX_SUM (1u << 24)
#define MAX_SIDE (1u << 28)

static int refuse(const char *op, const char *why) {
    fprintf(stderr, "tinyhvm-hip: %s: %s\n", op, why);
    return THVM_HIP_EINVAL;
}

typedef struct { u32 id; u64 bytes; int out; } Operand;

/* Every named buffer exists and holds its tensor, and no output is also
 * another operand. `same` lists pairs (output, input) that may be one buffer. */
static int operands_ok(const char *op, const Operand *o, u32 n, const u32 (*same)[2], u32 n_same) {
    for (u32 i = 0; i < n; i++) {
        if (!o[i].id) continue;
        if (!pool_get(o[i].id)) { refuse(op, "an unknown buffer"); return 0; }
        if (pool_bytes(o[i].id) < o[i].bytes) { refuse(op, "a buffer shorter than its tensor"); return 0; }
        for (u32 j = 0; j < n; j++) {
            if (j == i || o[j].id != o[i].id || !o[i].out) continue;
            int ok = 0;
            for (u32 s = 0; s < n_same; s++) ok |= same[s][0] == i && same[s][1] == j;
            for (u32 s = 0; s < n_same; s++) ok |= same[s][0] == j && same[s][1] == i;
            if (!ok) { refuse(op, "an output is also another operand"); return 0; }
        }
    }
    return 1;
}

/* The operands' pending copies and host writes go ahead of the work. */
static void operands_ready(const Operand *o, u32 n) {
    for (u32 i = 0; i < n; i++)
        if (o[i].id) hipb_operand(o[i].id);
}

static void operands_written(const Operand *o, u32 n) {
    for (u32 i = 0; i < n; i++)
        if (o[i].id && o[i].out) pool_mark_device_write(o[i].id);
}

static u64 addr(u32 id) { return id ? (u64)(uintptr_t)pool_ptr(id) : 0; }

static int dtype_ok(u32 dtype) { return dtype == DTYPE_F32 || dtype == DTYPE_F16; }
static u64 esize(u32 dtype) { return dtype == DTYPE_F16 ? 2 : 4; }
static const char *tname(u32 dtype) { return dtype == DTYPE_F16 ? "f16" : "f32"; }

static u64 div_up(u64 a, u64 b) { return (a + b - 1) / b; }
static u64 round_up(u64 a, u64 b) { return div_up(a, b) * b; }

/* Work on the stream, in order; the first failure ends it. */
static int launch(const char *name, u64 gx, u32 gy, u32 gz, u32 bx, void **params) {
    if (!gx || !gy || !gz) return THVM_HIP_OK;
    if (gx * bx >= (1ull << 32) || gy > 65535 || gz > 65535) {
        fprintf(stderr, "tinyhvm-hip: %s: the grid exceeds the launch limit\n", name);
        return THVM_HIP_EINVAL;
    }
    hipFunction_t fn = kernel(name);
    if (!fn || !hipb_launch(fn, (u32)gx, gy, gz, bx, params)) return THVM_HIP_EDEVICE;
    return THVM_HIP_OK;
}
static int launch1(const char *name, u64 gx, u32 gy, u32 gz, u32 bx, void *args) {
    void *params[] = {args};
    return launch(name, gx, gy, gz, bx, params);
}

/* A workspace's parts, one after another. */
typedef struct { u64 bytes; u64 base; } Carve;
static u64 carve(Carve *c, u64 bytes) {
    u64 at = c->base + c->bytes;
    c->bytes += round_up(bytes, 1024);
    return at;
}
static int carve_reserve(Carve *c) {
    void *p = scratch_reserve(&block_ws, c->bytes ? c->bytes : 1024);
    if (!p) return 0;
    c->base = (u64)(uintptr_t)p;
    c->bytes = 0;
    return 1;
}

/* ---- layer norm ---- */

/* Lanes a row (64 a wave of its own, else a workgroup) and vectors a lane. A
 * wave of its own has no barrier and sums by shuffles alone; more lanes have
 * fewer loads one after another, and fill the card where rows are few. us with
 * 64, 256 and 1024 lanes, f32: 8192 x 512 8.1, 10.9, 36.6; 8192 x 1000 11.4, 13.4,
 * 36.8; 1024 x 512 3.1, 3.2, 6.3; 1024 x 1000 4.1, 3.5, 6.5; 4 x 512 2.7, 2.4, 2.7;
 * and with 256 and 1024: 1024 x 4096 8.7, 9.7; 256 x 4096 4.1, 3.9; 4 x 4096 3.6,
 * 3.2; 8192 x 4096 49, 59. */
static int ln_shape(u32 rows, u32 cols, u32 dtype, u32 *g, u32 *nv) {
    const u64 vecs = div_up(cols, 16 / esize(dtype));
    if (vecs <= 64 || (vecs <= 128 && rows >= 1024) || (vecs <= 256 && rows >= 4096)) *g = 64;
    else *g = vecs <= 256 || (vecs <= 1024 && rows >= 512) ? 256 : 1024;
    for (*nv = 1; *nv * *g < vecs; *nv *= 2) {}
    return *nv <= 4;
}

int thvm_hip_layer_norm(u32 y, u32 mean, u32 rstd, u32 x, u32 gamma, u32 beta, u32 rows, u32 cols, f32 eps, u32 dtype) {
    if (!hipb.initialized) return THVM_HIP_EINVAL;
    const char *op = "layer_norm";
    if (!dtype_ok(dtype)) return refuse(op, "the type is neither f32 nor f16");
    if (!y || !x) return refuse(op, "no input or no output");
    if (cols > MAX_SUM) return refuse(op, "rows of more than 2^24 values");
    const u64 n = (u64)rows * cols * esize(dtype), v = cols * esize(dtype), st = rows * 4ull;
    const Operand o[] = {{y, n, 1}, {mean, st, 1}, {rstd, st, 1}, {x, n, 0}, {gamma, v, 0}, {beta, v, 0}};
    const u32 same[][2] = {{0, 3}};
    if (!operands_ok(op, o, 6, same, 1)) return THVM_HIP_EINVAL;
    if (!rows || (!cols && !mean && !rstd)) return THVM_HIP_OK;
    operands_ready(o, 6);
    u32 g, nv;
    char name[48];
    const int fits = ln_shape(rows, cols, dtype, &g, &nv);
    if (fits) snprintf(name, sizeof name, "thvm_ln_%s_%u_%u", tname(dtype), g, nv);
    else snprintf(name, sizeof name, "thvm_ln_%s_long", tname(dtype)), g = 1024;
    int rc = THVM_HIP_OK;
    /* a launch holds fewer than 2^32 lanes */
    for (u64 r0 = 0, step = (1u << 31) / g; r0 < rows && !rc; r0 += step) {
        const u32 nr = (u32)(rows - r0 < step ? rows - r0 : step);
        const u64 off = r0 * v;
        LnArgs a = {addr(x) + off, addr(gamma), addr(beta), addr(y) + off, mean ? addr(mean) + r0 * 4 : 0,
                    rstd ? addr(rstd) + r0 * 4 : 0, nr, cols, eps, 0};
        rc = launch1(name, g < 256 ? div_up(nr, 256 / g) : nr, 1, 1, g < 256 ? 256 : g, &a);
    }
    operands_written(o, 6);
    return rc;
}

int thvm_hip_layer_norm_grad(u32 dx, u32 dgamma, u32 dbeta, u32 dy, u32 x, u32 mean, u32 rstd, u32 gamma, u32 add,
                             u32 rows, u32 cols, u32 dtype) {
    if (!hipb.initialized) return THVM_HIP_EINVAL;
    const char *op = "layer_norm_grad";
    if (!dtype_ok(dtype)) return refuse(op, "the type is neither f32 nor f16");
    if (!dy || !x || !mean || !rstd) return refuse(op, "no gradient, input or statistics");
    if (!dx && !dgamma && !dbeta) return refuse(op, "no output");
    if (cols > MAX_SUM) return refuse(op, "rows of more than 2^24 values");
    const u64 n = (u64)rows * cols * esize(dtype), v = cols * esize(dtype), st = rows * 4ull;
    const Operand o[] = {{dx, n, 1}, {dgamma, v, 1}, {dbeta, v, 1}, {dy, n, 0}, {x, n, 0},
                         {mean, st, 0}, {rstd, st, 0}, {gamma, v, 0}, {add, n, 0}};
    const u32 same[][2] = {{0, 3}, {0, 4}, {0, 8}};
    if (!operands_ok(op, o, 9, same, 3)) return THVM_HIP_EINVAL;
    if (!cols) return THVM_HIP_OK;
    const u64 vecs = div_up(cols, 16 / esize(dtype));
    const int wgrad = dgamma || dbeta, half = dtype == DTYPE_F16;
    /* The kernels' shapes (norm_kernels.hip): lanes a row, vectors a lane, and
     * workgroups, two a compute unit: of 8192x4096 in f16 52 us, against 58 with
     * one and 61 with three, whose partial sums are longer. */
    const u32 full = 2 * hipb.n_cu;
    u32 g = 0, nv = 0;
    if (vecs <= (half ? 128 : 256)) for (g = 64, nv = 1; nv * g < vecs;) nv *= 2;
    else if (vecs <= (half ? 256 : 512)) for (g = 256, nv = half ? 1 : 2; nv * g < vecs;) nv *= 2;
    else if (vecs <= (half ? 2048 : 4096)) for (g = 512, nv = half ? 1 : 2; nv * g < vecs;) nv *= 2;
    u32 parts;
    if (g) {
        const u32 per = g < 256 ? 256 / g : 1;
        parts = (u32)(div_up(rows, per) < full ? div_up(rows, per) : full);
    } else parts = (u32)(div_up(rows, 64) < 256 ? div_up(rows, 64) : 256);
    Carve c = {0, 0};
    carve(&c, wgrad ? 8ull * parts * cols : 0);
    if (!carve_reserve(&c)) return THVM_HIP_ENOMEM;
    operands_ready(o, 9);
    LnGradArgs a = {addr(dy), addr(x), addr(mean), addr(rstd), addr(gamma), addr(add), addr(dx), addr(dgamma), addr(dbeta),
                    wgrad ? carve(&c, 0) : 0, rows, cols, parts, 0};
    char name[48];
    int rc = THVM_HIP_OK;
    if (g) {
        snprintf(name, sizeof name, "thvm_lnb_%s_%u_%u", tname(dtype), g, nv);
        rc = launch1(name, parts, 1, 1, g < 256 ? 256 : g, &a);
    } else {
        if (wgrad) {
            snprintf(name, sizeof name, "thvm_lnb_%s_part", tname(dtype));
            rc = launch1(name, div_up(cols, 256), parts, 1, 256, &a);
        }
        snprintf(name, sizeof name, "thvm_lnb_%s_long", tname(dtype));
        for (u64 r0 = 0, step = 1u << 21; dx && r0 < rows && !rc; r0 += step) {
            const u64 off = r0 * v;
            LnGradArgs b = a;
            b.rows = (u32)(rows - r0 < step ? rows - r0 : step);
            b.dy += off; b.x += off; b.dx += off;
            if (b.add) b.add += off;
            b.mean += r0 * 4; b.rstd += r0 * 4;
            rc = launch1(name, b.rows, 1, 1, 1024, &b);
        }
    }
    if (wgrad && !rc) {
        snprintf(name, sizeof name, "thvm_lnb_%s_cols", tname(dtype));
        rc = launch1(name, div_up(2ull * cols, 32), 1, 1, 1024, &a);
    }
    operands_written(o, 9);
    return rc;
}

/* ---- products ---- */

/* A packed operand of `rows` rows by `k`, padded to whole tiles. */
typedef struct { u32 Rp, KB; u64 p, e; } Packed;

static u64 packed_bytes(const Packed *k, u32 dtype) { return (u64)k->Rp * k->KB * 32 * (dtype == DTYPE_F16 ? 1 : 2); }

static Packed packed_of(u32 rows, u32 k, u32 tile) {
    Packed p = {(u32)round_up(rows, tile), (u32)(round_up(k, 64) / 16), 0, 0};
    return p;
}

/* 16-bit matrices whose rows are whole 16-byte pieces are multiplied as they
 * lie. The products take 6 % longer (4096^3: 137 us against 129), packing took
 * 21 us; 2048^3 25 us against 30 in all, 512 x 4096 x 512 12 against 20. A
 * gradient packs dz in any case, and W and x with it: of 2048^3 for next to
 * nothing (12 us against 11), so that packed operands win (56 us against 60 with
 * W and x as they lie). Only that size was measured both ways; of few rows W is
 * most of what is packed (64 x 4096 x 4096: 13 of 49 us). A tile reaches up to 64
 * rows from one address by 32-bit offsets, which a longer row would pass. */
static int lies_well(u32 cols, u32 dtype) { return dtype == DTYPE_F16 && cols % 8 == 0 && cols && cols <= MAX_SUM; }

static void packed_carve(Packed *p, Carve *c, u32 dtype) {
    p->p = carve(c, packed_bytes(p, dtype) + PACK_SLACK);
    p->e = carve(c, dtype == DTYPE_F32 ? p->Rp * 8ull : 0);
}

/* A product's tile and K splits: C [M][N] over K. */
typedef struct { u32 T, tm, tn, splits, lanes; f32 time; const char *name; u32 tiles; } Plan;

/* Tiles, largest first: the larger, the fewer bytes per product, and the fewer
 * workgroups. What each takes, in us, as measured on products of 512 to 4096
 * rows and columns over K of 512 to 8192: `unit` per 16 of K (f16, f32; with
 * every compute unit at work), `fixed` for the launch, the first loads and the
 * epilogue, `join + per_join * splits` and the parts' bytes at `rate` for joining
 * K splits (optimiser steps in f32: 784 x 128, whose first product has 3 tiles,
 * 93 us with 4 splits, 97 with 2, 102 with none; 768 x 768, 78 tiles, 172 with 2,
 * 163 with none). */
static const struct {
    u32 T, lanes, slots;      /* slots: workgroups a compute unit holds, which then share its time */
    const char *name;
    f32 unit[2], fixed[2], join, per_join, rate;
} TILES[] = {
    {256, 512, 1, "256x256", {0.41f, 1.15f}, {10, 18}, 15, 1, 3e6f},
    {192, 256, 1, "192x192", {0.27f, 0.75f}, {8, 12}, 10, 1, 3e6f},     /* of a symmetric product only */
    {128, 256, 1, "128x128", {0.13f, 0.335f}, {6, 9}, 5, 1, 3e6f},
    {64, 256, 2, "64x64", {0.055f, 0.11f}, {5, 6}, 1, 0.25f, 1.3e6f},
};
#define TILE_SYM 1

/* The tile and splits that the estimate puts first, for `count` products of
 * one shape; sym: C is symmetric, and only its tiles on and above the diagonal
 * are computed. */
static Plan plan_of(u32 M, u32 N, u32 K, u32 dtype, u32 count, int sym) {
    const u32 cu = hipb.n_cu ? hipb.n_cu : 256, f = dtype == DTYPE_F32;
    const f32 units = (f32)(round_up(K, 64) / 16);
    Plan best;
    memset(&best, 0, sizeof best);
    for (u32 i = 0; i < sizeof TILES / sizeof TILES[0]; i++) {
        if (i == TILE_SYM && (!sym || K > MAX_SUM / 2)) continue;      /* it reaches three row blocks at once */
        const u32 tm = (u32)div_up(M, TILES[i].T), tn = (u32)div_up(N, TILES[i].T);
        const u64 tiles = sym ? (u64)tm * (tm + 1) / 2 : (u64)tm * tn;
        for (u32 s = 1; s <= 16; s *= 2) {
            if (s > 1 && (tiles * count > COUNTS || units / s < 12)) break;
            const u64 wgs = tiles * count * s, rounds = div_up(wgs, (u64)cu * TILES[i].slots);
            /* two workgroups of a compute unit take 1.9 times one's time */
            const f32 share = TILES[i].slots == 2 && wgs > cu ? 1.9f * (f32)rounds : (f32)rounds;
            const f32 t = TILES[i].fixed[f] + share * units / s * TILES[i].unit[f] +
                          (s > 1 ? TILES[i].join + TILES[i].per_join * s + (f32)wgs * TILES[i].T * TILES[i].T * 4 / TILES[i].rate : 0);
            if (best.T && t >= best.time) continue;
            best = (Plan){TILES[i].T, tm, tn, s, TILES[i].lanes, t, TILES[i].name, (u32)tiles};
        }
    }
    return best;
}

static u64 plan_part_bytes(const Plan *p) { return p->splits > 1 ? 4ull * p->tiles * p->splits * p->T * p->T : 0; }

/* The product of two operands with its epilogue (a: out, z, bias, res, act).
 * `lie`: A is [M][K] and B [K][N] as they lie, else both are packed (a.oa and
 * a.ob: from what). */
static int product(const Plan *pl, int lie, const Packed *pa, const Packed *pb, u32 M, u32 N, u32 K, u32 dtype, u64 part,
                   GemmArgs a) {
    char name[48];
    a.A = pa->p; a.B = pb->p; a.ea = pa->e; a.eb = pb->e;
    a.M = M; a.N = N; a.K = K; a.KB = (u32)(round_up(K, 64) / 16);
    a.tm = pl->tm; a.tn = pl->tn; a.splits = pl->splits;
    a.part = part; a.count = B.counts;
    snprintf(name, sizeof name, "thvm_gemm%s_%s_%s", lie ? "_rc" : "", pl->name, tname(dtype));
    return launch1(name, pl->tiles, pl->splits, 1, pl->lanes, &a);
}

/* A matrix [R][C] to pack (times act'(z) where z is given): `rows` with its
 * rows as rows, `cols` with its columns, either or both, and its column sums.
 * The parts of its sizes and sums lie in the workspace. */
typedef struct {
    u64 src, z;
    u32 act, R, C;
    const Packed *rows, *cols;
    u64 sums, row_part, col_part, sum_part;
    u32 rt, row_parts, col_parts;
} Source;

/* Whether a 16-bit dz of a call is past its type's range: packing writes the
 * call's number here, so that there is nothing to clear between calls (a
 * graph's launches share theirs: one that had such a dz has the next look, too). */
static u64 past16(void) { return B.counts + 4ull * COUNTS; }

#define SIZE_COLS 512u
#define SIZE_PARTS 64u
static void source_carve(Source *s, Carve *c, u32 dtype) {
    s->rt = dtype == DTYPE_F16 ? 64 : (u32)(div_up(div_up(s->R, SIZE_PARTS), 32) * 32);
    if (!s->rt) s->rt = 32;
    s->row_parts = (u32)div_up(s->C, SIZE_COLS);
    s->col_parts = (u32)div_up(s->R, s->rt);
    if (dtype == DTYPE_F32) {
        s->row_part = carve(c, s->rows ? 4ull * s->row_parts * s->R : 0);
        s->col_part = carve(c, s->cols ? 4ull * s->col_parts * s->C : 0);
    }
    s->sum_part = carve(c, s->sums ? 4ull * s->col_parts * s->C : 0);
}

/* Up to three matrices: their sizes in one launch (f32), their packing in another. */
static int pack(const Source *src, u32 n, u32 dtype) {
    char name[48];
    PackSet s, z;
    memset(&s, 0, sizeof s);
    memset(&z, 0, sizeof z);
    u64 tiles = 0, sized = 0;
    u64 sums = 0;
    for (u32 i = 0; i < n; i++) {
        const Source *m = &src[i];
        PackArgs a;
        memset(&a, 0, sizeof a);
        a.src = m->src; a.z = m->act ? m->z : 0; a.act = m->act; a.R = m->R; a.C = m->C;
        a.rt = m->rt; a.row_parts = m->row_parts; a.col_parts = m->col_parts;
        a.row_part = m->rows ? m->row_part : 0;
        a.col_part = m->cols ? m->col_part : 0;
        a.sum_part = m->sums ? m->sum_part : 0;
        u32 rmax = m->rows || m->cols || dtype == DTYPE_F16 ? (u32)round_up(m->R ? m->R : 1, 64) : 64, cmax = (u32)round_up(m->C ? m->C : 1, 64);
        if (m->rows) {
            a.pn = m->rows->p; a.en = m->rows->e; a.Rn = m->rows->Rp; a.KBn = m->rows->KB;
            if (a.Rn > rmax) rmax = a.Rn;
        }
        if (m->cols) {
            a.pt = m->cols->p; a.et = m->cols->e; a.Ct = m->cols->Rp; a.KBt = m->cols->KB;
            if (a.Ct > cmax) cmax = a.Ct;
        }
        a.sum_out = m->sums;
        a.past16 = past16(); a.call = B.call;
        if (m->sums) sums = i + 1;
        a.ctiles = cmax / 64;
        s.first[i] = (u32)tiles;
        z.first[i] = (u32)sized;
        s.p[i] = z.p[i] = a;
        tiles += (u64)(rmax / 64) * a.ctiles;
        /* of a matrix of nothing a workgroup clears the rows' numbers */
        sized += m->row_parts && m->col_parts ? (u64)m->row_parts * m->col_parts : 1;
    }
    s.n = z.n = n;
    int rc = THVM_HIP_OK;
    if (dtype == DTYPE_F32) {
        snprintf(name, sizeof name, "thvm_pack_sizes_%s", tname(dtype));
        rc = launch1(name, sized, 1, 1, 512, &z);
    }
    if (!rc) {
        snprintf(name, sizeof name, "thvm_pack_%s", tname(dtype));
        rc = launch1(name, tiles, 1, 1, 256, &s);
    }
    if (!rc && sums && dtype == DTYPE_F16) {
        const Source *m = &src[sums - 1];
        void *params[] = {(void *)&m->sum_part, (void *)&m->sums, (void *)&m->C, (void *)&m->col_parts};
        snprintf(name, sizeof name, "thvm_sum_parts_%s", tname(dtype));
        rc = launch(name, div_up(m->C, 64), 1, 1, 1024, params);
    }
    return rc;
}

/* Few rows: W is read as it lies, by blocks of 1 or 16 rows (few_rows in
 * gemm_kernels.hip); two rows take the block of 16, which is at most 6 % slower
 * for 4 than a block of 4 was (256 x 256) and up to 25 % faster (1024 x 2048). */
static u32 few_block(u32 m) { return m <= 1 ? 1 : 16; }

/* Strips of 64 bytes of a row of W with K whole, or of 256 bytes with K split
 * over workgroups: joining splits takes 2 to 4 us, but few narrow strips do not
 * read a large W as fast as the card can. f32, one row: 1024 x 2048 4.95 us
 * narrow, 5.7 wide; 1024 x 3000 7.6 and 6.9. 64 rows: 1024 x 1024 (256 workgroups)
 * 5.5 and 7.9; 512 x 4096 (1024 of them) 14 and 5.8. */
#define FEW_NARROW (8u << 20) /* bytes of W */
static int few_narrow(u32 m, u32 k, u32 n, u32 dtype) {
    if (n < 16 / esize(dtype)) return 1;      /* no wide vector */
    return k <= FEW_CHUNK && (u64)k * n * esize(dtype) <= FEW_NARROW &&
           div_up(n, 64 / esize(dtype)) * div_up(m, few_block(m)) <= 256;
}
/* Whether the kernels take the shape, and the outputs have counters or need none. */
static int few_fits(u32 m, u32 k, u32 n, u32 dtype) {
    if (k && n < 4 / esize(dtype)) return 0;      /* a lane takes 4 bytes of a row at least */
    return div_up(n, 256 / esize(dtype)) * div_up(m, few_block(m)) <= COUNTS || k <= FEW_CHUNK;
}

/* Its time in us, roughly: W's bytes once a block of rows, or 3.8 a workgroup
 * that a compute unit takes. */
static f32 few_time(u32 m, u32 k, u32 n, u32 dtype) {
    const u64 blocks = div_up(m, few_block(m));
    const f32 bytes = (f32)(3.5 + (double)k * n * esize(dtype) * blocks / 7.3e6);
    const f32 wgs = (f32)(3.8 / 256 * div_up(n, (few_narrow(m, k, n, dtype) ? 64 : 256) / esize(dtype)) * blocks);
    return bytes > wgs ? bytes : wgs;
}

static int few(u32 m, u32 k, u32 n, u32 dtype, GemmArgs a) {
    const u32 mr = few_block(m);
    /* wide strips: a workgroup a compute unit (two, of one row of 16-bit values) */
    const int narrow = few_narrow(m, k, n, dtype);
    const u32 cols = (narrow ? 64 : 256) / (u32)esize(dtype), full = mr == 1 && dtype == DTYPE_F16 ? 512 : 256;
    const u64 strips = div_up(n, cols), blocks = div_up(m, mr);
    u64 splits = narrow || !few_fits(m, FEW_CHUNK + 1, n, dtype) ? 1 : full / (strips * blocks);
    if (splits < 1) splits = 1;
    u64 per = round_up(div_up(k ? k : 1, splits), 256);
    if (per > FEW_CHUNK) per = FEW_CHUNK;
    a.kper = (u32)per;
    a.splits = (u32)div_up(k ? k : 1, per);
    a.N = n; a.K = k;
    Carve c = {0, 0};
    carve(&c, a.splits > 1 ? 4ull * a.splits * strips * cols * blocks * mr : 0);
    if (!carve_reserve(&c)) return THVM_HIP_ENOMEM;
    a.part = carve(&c, 0);
    a.count = B.counts;
    char name[48];
    snprintf(name, sizeof name, "thvm_few%u%s_%s", mr, narrow ? "n" : "", tname(dtype));
    /* a launch counts 65535 blocks of rows */
    int rc = THVM_HIP_OK;
    const u64 es = esize(dtype), step = 65535ull * mr;
    for (u64 r0 = 0; r0 < m && !rc; r0 += step) {
        GemmArgs p = a;
        p.M = (u32)(m - r0 < step ? m - r0 : step);
        p.A += r0 * k * es;
        p.out += r0 * n * es;
        if (p.z) p.z += r0 * n * es;
        if (p.res) p.res += r0 * n * es;
        rc = launch1(name, strips, a.splits, (u32)div_up(p.M, mr), 512, &p);
    }
    return rc;
}

/* 32-bit matrices as they lie, in tiles of 64 (direct_tile in gemm_kernels.hip):
 * K splits, and the time in us: 1.04 per 64 of K with a workgroup on a compute
 * unit, 40 % more with several. Of 64 x 4096 x 4096 27 us (few rows: 50; packed:
 * 63), 128 x 4096 x 4096 44 (91; 68), 256 x 4096 x 4096 75 (174; 81), but of
 * 64 x 1024 x 4096 15 (9.7; 29) and of 512 x 4096 x 4096 193 (340; 106). */
static u32 direct_splits(u32 M, u32 N, u32 K, f32 *time) {
    const u64 tiles = div_up(M, 64) * div_up(N, 64);
    const f32 units = (f32)div_up(K, 64);
    u32 best = 1;
    for (u32 s = 1; s <= 16; s *= 2) {
        if (s > 1 && (tiles > COUNTS || units / s < 4)) break;
        const u64 rounds = div_up(tiles * s, hipb.n_cu ? hipb.n_cu : 256);
        const f32 t = 3 + (f32)rounds * (5 + units / s * 1.04f) * (rounds > 1 ? 1.4f : 1) + (s > 1 ? 2.5f : 0);
        if (s > 1 && t >= *time) continue;
        *time = t;
        best = s;
    }
    return best;
}

static int direct(u32 M, u32 N, u32 K, u32 splits, u64 part, GemmArgs a) {
    a.M = M; a.N = N; a.K = K;
    a.tm = (u32)div_up(M, 64); a.tn = (u32)div_up(N, 64);
    a.kper = (u32)round_up(div_up(K, splits), 64);
    a.splits = (u32)div_up(K, a.kper);
    a.part = part; a.count = B.counts;
    return launch1("thvm_direct_f32", (u64)a.tm * a.tn, a.splits, 1, 256, &a);
}

int thvm_hip_linear(u32 y, u32 z, u32 x, u32 w, u32 bias, u32 res, u32 act, u32 m, u32 k, u32 n, u32 dtype) {
    if (!hipb.initialized) return THVM_HIP_EINVAL;
    const char *op = "linear";
    if (!dtype_ok(dtype)) return refuse(op, "the type is neither f32 nor f16");
    if (act >= ACT_COUNT) return refuse(op, "an unknown activation");
    if (!y || !x || !w) return refuse(op, "no input, weights or output");
    if (k > MAX_SUM) return refuse(op, "sums of more than 2^24 products");
    if (m > MAX_SIDE || n > MAX_SIDE) return refuse(op, "more than 2^28 rows or columns");
    const u64 es = esize(dtype), mn = (u64)m * n * es;
    const Operand o[] = {{y, mn, 1}, {z, mn, 1}, {x, (u64)m * k * es, 0}, {w, (u64)k * n * es, 0}, {bias, n * es, 0}, {res, mn, 0}};
    const u32 same[][2] = {{0, 5}};
    if (!operands_ok(op, o, 6, same, 1)) return THVM_HIP_EINVAL;
    if (!m || !n) return THVM_HIP_OK;
    GemmArgs a;
    memset(&a, 0, sizeof a);
    a.out = addr(y); a.z = addr(z); a.bias = addr(bias); a.res = addr(res); a.act = act;
    int rc;
    const Plan pl = plan_of(m, n, k, dtype, 1, 0);
    /* packing takes a launch and the operands' bytes twice over (f32: two launches, three times) */
    const f32 packed = pl.time + (dtype == DTYPE_F16 ? 6 : 12) + (f32)((double)k * (m + (double)n) * 10 / 4.8e6);
    const int as_is = lies_well(k, dtype) && lies_well(n, dtype);
    f32 straight;
    const u32 splits = direct_splits(m, n, k, &straight);
    /* as they lie, 16-bit matrices take 4.4 to 13 us for up to 64 rows; narrow strips
     * are faster than that (64 x 1024 x 1024: 6.5 us, 8.2), wide ones are not, but
     * for one row (4096 x 4096: 11.3, 12; 64 rows 38, 13) */
    const f32 rows_time = few_time(m, k, n, dtype);
    const int fast = m <= 1 || (as_is ? few_narrow(m, k, n, dtype) : rows_time < packed && (dtype != DTYPE_F32 || rows_time < straight));
    if (!k || (few_fits(m, k, n, dtype) && fast)) {
        operands_ready(o, 6);
        a.A = addr(x); a.B = addr(w);
        rc = few(m, k, n, dtype, a);
    } else if (dtype == DTYPE_F32 && n > 1 && straight < packed) {
        Carve c = {0, 0};
        carve(&c, splits > 1 ? 16384ull * splits * div_up(m, 64) * div_up(n, 64) : 0);
        if (!carve_reserve(&c)) return THVM_HIP_ENOMEM;
        operands_ready(o, 6);
        a.A = addr(x); a.B = addr(w);
        rc = direct(m, n, k, splits, carve(&c, 0), a);
    } else {
        Packed px = packed_of(m, k, pl.T), pw = packed_of(n, k, pl.T);
        Source src[2] = {{addr(x), 0, 0, m, k, &px, NULL, 0}, {addr(w), 0, 0, k, n, NULL, &pw, 0}};
        u64 part = 0;
        Carve c = {0, 0};
        for (int pass = 0; pass < 2; pass++) {
            if (!as_is) {
                packed_carve(&px, &c, dtype);
                packed_carve(&pw, &c, dtype);
                for (int i = 0; i < 2; i++) source_carve(&src[i], &c, dtype);
            }
            part = carve(&c, plan_part_bytes(&pl));
            if (!pass && !carve_reserve(&c)) return THVM_HIP_ENOMEM;
        }
        operands_ready(o, 6);
        if (as_is) {
            px.p = addr(x); pw.p = addr(w);
            a.lda = k; a.ldb = n;
            rc = product(&pl, 1, &px, &pw, m, n, k, dtype, part, a);
        } else {
            a.oa = (Origin){addr(x), 0, k, 1, 0, 0};
            a.ob = (Origin){addr(w), 0, 1, n, 0, 0};
            rc = pack(src, 2, dtype);
            if (!rc) rc = product(&pl, 0, &px, &pw, m, n, k, dtype, part, a);
        }
    }
    operands_written(o, 6);
    return rc;
}

int thvm_hip_linear_grad(u32 dx, u32 dw, u32 db, u32 dy, u32 z, u32 x, u32 w, u32 act, u32 m, u32 k, u32 n, u32 dtype) {
    if (!hipb.initialized) return THVM_HIP_EINVAL;
    const char *op = "linear_grad";
    if (!dtype_ok(dtype)) return refuse(op, "the type is neither f32 nor f16");
    if (act >= ACT_COUNT) return refuse(op, "an unknown activation");
    if (!dy || (act && !z) || (dx && !w) || (dw && !x)) return refuse(op, "no gradient, input or weights, or no values before the activation");
    if (!dx && !dw && !db) return refuse(op, "no output");
    if ((dx && n > MAX_SUM) || (dw && m > MAX_SUM)) return refuse(op, "sums of more than 2^24 products");
    if (m > MAX_SIDE || k > MAX_SIDE || n > MAX_SIDE) return refuse(op, "more than 2^28 rows or columns");
    const u64 es = esize(dtype), mn = (u64)m * n * es;
    const Operand o[] = {{dx, (u64)m * k * es, 1}, {dw, (u64)k * n * es, 1}, {db, n * es, 1}, {dy, mn, 0},
                         {act ? z : 0, mn, 0}, {dw ? x : 0, (u64)m * k * es, 0}, {dx ? w : 0, (u64)k * n * es, 0}};
    if (!operands_ok(op, o, 7, NULL, 0)) return THVM_HIP_EINVAL;
    /* an empty sum is 0: gradients over no rows or no outputs */
    if (!k) dx = dw = 0;
    if (!m) dx = 0;
    if (!n) dw = db = 0;
    if (!dx && !dw && !db) return THVM_HIP_OK;
    const Plan px_ = plan_of(m, k, n, dtype, 1, 0), pw_ = plan_of(k, n, m, dtype, 1, 0);
    Packed zr = packed_of(m, n, px_.T), wr = packed_of(k, n, px_.T);       /* dx = dz W^T */
    Packed xc = packed_of(k, m, pw_.T), zc = packed_of(n, m, pw_.T);       /* dW = x^T dz */
    Source src[3] = {{addr(dy), addr(z), act, m, n, dx ? &zr : NULL, dw ? &zc : NULL, addr(db)}};
    u32 ns = 1;
    if (dx) src[ns++] = (Source){addr(w), 0, 0, k, n, &wr, NULL, 0};
    if (dw) src[ns++] = (Source){addr(x), 0, 0, m, k, NULL, &xc, 0};
    u64 part = 0;
    Carve c = {0, 0};
    for (int pass = 0; pass < 2; pass++) {
        if (dx) packed_carve(&zr, &c, dtype), packed_carve(&wr, &c, dtype);
        if (dw) packed_carve(&xc, &c, dtype), packed_carve(&zc, &c, dtype);
        for (u32 i = 0; i < ns; i++) source_carve(&src[i], &c, dtype);
        u64 q = dx ? plan_part_bytes(&px_) : 0, q2 = dw ? plan_part_bytes(&pw_) : 0;
        part = carve(&c, q > q2 ? q : q2);
        if (!pass && !carve_reserve(&c)) return THVM_HIP_ENOMEM;
    }
    operands_ready(o, 7);
    GemmArgs a;
    memset(&a, 0, sizeof a);
    if (!++B.call) B.call = 1;
    a.past16 = act ? past16() : 0; a.call = B.call;
    int rc = pack(src, ns, dtype);
    if (dx && !rc) {
        a.out = addr(dx);
        a.oa = (Origin){addr(dy), act ? addr(z) : 0, n, 1, act, 0};
        a.ob = (Origin){addr(w), 0, n, 1, 0, 0};
        rc = product(&px_, 0, &zr, &wr, m, k, n, dtype, part, a);
    }
    if (dw && !rc) {
        a.out = addr(dw);
        a.oa = (Origin){addr(x), 0, 1, k, 0, 0};
        a.ob = (Origin){addr(dy), act ? addr(z) : 0, 1, n, act, 0};
        rc = product(&pw_, 0, &xc, &zc, k, n, m, dtype, part, a);
    }
    operands_written(o, 7);
    return rc;
}

/* ---- the orthogonalised step ---- */

/* x -> a x + b x^3 + c x^5 on the singular values: the coefficients that K.
 * Jordan et al. published for this update ("Muon", 2024), chosen for a steep
 * start at 0 that keeps [0, 1.2] within itself; five steps bring what is over
 * 1.5e-3 to 0.67 .. 1.21 */
#define NS_A 3.4445
#define NS_B (-4.7750)
#define NS_C 2.0315
/* X and A = X X^T are packed times 2^14, B = b A + c A^2 times 2^13: |X| and
 * |A| stay under 1.5 and |B| under 2.9, so all of them stay under 2^16 */

/* What a step on matrices of one shape works with: the padded sides of X [n][w],
 * the plans of X X^T, A A and B X, and bytes of X, of A and of a matrix's all. */
typedef struct {
    u32 tall, n, w, np, wp;
    Plan gram, square, apply;
    u64 xb, ab, stride, part;
} MuonPlan;

static MuonPlan muon_plan(u32 rows, u32 cols, u32 dtype, u32 count) {
    MuonPlan p;
    memset(&p, 0, sizeof p);
    p.tall = rows > cols;
    p.n = p.tall ? cols : rows;
    p.w = p.tall ? rows : cols;
    p.gram = plan_of(p.n, p.n, p.w, dtype, count, 1);
    p.square = plan_of(p.n, p.n, p.n, dtype, count, 1);
    p.apply = plan_of(p.n, p.w, p.n, dtype, count, 0);
    /* every product finds whole tiles; what no tile writes stays the packing's zeros */
    const u32 t[3] = {p.gram.T, p.square.T, p.apply.T};
    for (int i = 0; i < 3; i++) {
        const u32 np = (u32)round_up(p.n, t[i]);
        if (np > p.np) p.np = np;
    }
    p.wp = (u32)round_up(p.w, p.apply.T);
    const u64 planes = dtype == DTYPE_F16 ? 1 : 2;
    p.xb = round_up(2 * planes * p.np * p.wp, 1024);
    p.ab = round_up(2 * planes * p.np * p.np, 1024);
    p.stride = 3 * p.xb + 2 * p.ab;      /* X, X^T twice, A, B */
    const u64 parts[3] = {plan_part_bytes(&p.gram), plan_part_bytes(&p.square), plan_part_bytes(&p.apply)};
    for (int i = 0; i < 3; i++)
        if (parts[i] > p.part) p.part = parts[i];
    return p;
}

static int ns_product(const Plan *pl, NsArgs *g, u32 count, u32 dtype) {
    char name[48];
    g->tm = pl->tm; g->tn = pl->tn; g->splits = pl->splits;
    snprintf(name, sizeof name, "thvm_ns_%s_%s", pl->name, tname(dtype));
    return launch1(name, pl->tiles, pl->splits, count, pl->lanes, g);
}

static int muon_chunk(const MuonPlan *q, const u32 *param, const u32 *grad, const u32 *m, u32 count, u32 rows, u32 cols, f32 keep,
                      f32 step, f32 beta, int nesterov, u32 steps, u32 dtype) {
    char name[48];
    const u32 tall = q->tall, n = q->n, w = q->w, np = q->np, wp = q->wp;
    const u64 xb = q->xb, ab = q->ab, stride = q->stride;
    MuonArgs mu;
    memset(&mu, 0, sizeof mu);
    mu.numel = (u64)rows * cols;
    mu.blocks = (u32)(div_up(mu.numel, 1024) < 1024 ? div_up(mu.numel, 1024) : 1024);
    mu.nesterov = nesterov != 0;
    mu.beta = beta;
    NsArgs a;
    memset(&a, 0, sizeof a);
    u64 ops = 0;
    Carve c = {0, 0};
    for (int pass = 0; pass < 2; pass++) {
        ops = carve(&c, stride * count + PACK_SLACK);
        mu.sums = carve(&c, 8ull * mu.blocks * count);
        a.part = carve(&c, q->part * count);
        if (!pass && !carve_reserve(&c)) return THVM_HIP_ENOMEM;
    }
    for (u32 i = 0; i < count; i++) {
        a.param[i] = addr(param[i]);
        mu.grad[i] = addr(grad[i]);
        mu.m[i] = addr(m[i]);
    }
    snprintf(name, sizeof name, "thvm_muon_momentum_%s", tname(dtype));
    int rc = launch1(name, mu.blocks, count, 1, 256, &mu);
    if (rc) return rc;
    PackArgs p;
    memset(&p, 0, sizeof p);
    const u64 X = ops, A = ops + 3 * xb, Bm = A + ab;
    u64 xt = ops + xb, xt2 = ops + 2 * xb;
    p.R = rows; p.C = cols; p.stride = stride;
    p.pn = tall ? xt : X; p.Rn = tall ? wp : np; p.KBn = (tall ? np : wp) / 16;
    p.pt = tall ? X : xt; p.Ct = tall ? np : wp; p.KBt = (tall ? wp : np) / 16;
    p.ctiles = p.Ct / 64;
    void *pp[] = {&p, &mu};
    snprintf(name, sizeof name, "thvm_muon_pack_%s", tname(dtype));
    rc = launch(name, (u64)(p.Rn / 64) * p.ctiles, count, 1, 256, pp);
    a.stride = stride; a.n = n; a.w = w; a.tall = tall; a.keep = keep; a.step = step; a.count = B.counts;
    for (u32 s = 0; s < steps && !rc; s++) {
        NsArgs g = a;      /* A = X X^T */
        g.A = g.B = X; g.out = g.out_t = A;
        g.KB = wp / 16; g.KU = (u32)(round_up(w, 64) / 16); g.KBO = g.KBT = np / 16;
        g.sym = 1; g.beta = 1.0f / 16384;
        rc = ns_product(&q->gram, &g, count, dtype);
        g.A = g.B = g.old = A; g.out = g.out_t = Bm;      /* B = b A + c A A */
        g.KB = np / 16; g.KU = (u32)(round_up(n, 64) / 16);
        g.alpha = (f32)(NS_B / 2); g.beta = (f32)(NS_C / 32768);
        if (!rc) rc = ns_product(&q->square, &g, count, dtype);
        g.A = Bm; g.B = xt; g.old = X;                    /* X = a X + B X */
        g.KBO = wp / 16; g.sym = 0;
        g.last = s + 1 == steps;
        g.out = g.last ? 0 : X; g.out_t = g.last ? 0 : xt2;
        g.alpha = (f32)(g.last ? NS_A / 16384 : NS_A); g.beta = g.last ? 1.0f / (1 << 27) : 1.0f / 8192;
        if (!rc) rc = ns_product(&q->apply, &g, count, dtype);
        const u64 t = xt; xt = xt2; xt2 = t;
    }
    return rc;
}

int thvm_hip_muon_step(const u32 *param, const u32 *grad, const u32 *m, u32 count, u32 rows, u32 cols, f32 lr, f32 scale,
                       f32 weight_decay, f32 beta, u32 nesterov, u32 steps, u32 dtype) {
    if (!hipb.initialized) return THVM_HIP_EINVAL;
    const char *op = "muon_step";
    if (!dtype_ok(dtype)) return refuse(op, "the type is neither f32 nor f16");
    if (!steps || steps > 64) return refuse(op, "1 to 64 Newton-Schulz steps are possible");
    if (count && (!param || !grad || !m)) return refuse(op, "no parameters, gradients or momenta");
    if (rows > MAX_SUM || cols > MAX_SUM) return refuse(op, "sums of more than 2^24 products");
    const u64 numel = (u64)rows * cols, es = esize(dtype);
    for (u32 i = 0; i < count; i++) {
        if (!param[i] || !grad[i] || !m[i]) return refuse(op, "no parameter, gradient or momentum");
        const Operand o[] = {{param[i], numel * es, 1}, {m[i], numel * 4, 1}, {grad[i], numel * es, 0}};
        if (!operands_ok(op, o, 3, NULL, 0)) return THVM_HIP_EINVAL;
        for (u32 j = 0; j < i; j++)
            if (param[j] == param[i] || m[j] == m[i] || param[j] == m[i] || m[j] == param[i] || param[j] == grad[i] ||
                grad[j] == param[i] || m[j] == grad[i] || grad[j] == m[i])
                return refuse(op, "an output is also another operand");
    }
    if (!numel || !count) return THVM_HIP_OK;
    /* as many matrices at once as a launch names, in 4 GiB of workspace */
    u64 at_once = count < MUON_MAX ? count : MUON_MAX;
    MuonPlan q = muon_plan(rows, cols, dtype, (u32)at_once);
    while (at_once > 1 && at_once * (q.stride + q.part) > (4ull << 30)) q = muon_plan(rows, cols, dtype, (u32)--at_once);
    const f32 keep = (f32)(1.0 - (double)lr * weight_decay), step = (f32)((double)lr * scale);
    int rc = THVM_HIP_OK;
    for (u32 i = 0; i < count && !rc; i += (u32)at_once) {
        const u32 nc = count - i < at_once ? count - i : (u32)at_once;
        if (nc != at_once) q = muon_plan(rows, cols, dtype, nc);
        for (u32 j = i; j < i + nc; j++) hipb_operand(param[j]), hipb_operand(grad[j]), hipb_operand(m[j]);
        rc = muon_chunk(&q, param + i, grad + i, m + i, nc, rows, cols, keep, step, beta, nesterov != 0, steps, dtype);
        for (u32 j = i; j < i + nc; j++) pool_mark_device_write(param[j]), pool_mark_device_write(m[j]);
    }
    return rc;
}
