// norm_kernels.hip - layer normalisation over the rows of a matrix, forward
// and backward (thvm_hip_layer_norm, thvm_hip_layer_norm_grad):
//   mean = sum(x) / c, rstd = 1 / sqrt(sum((x - mean)^2) / c + eps),
//   y = (x - mean) * rstd * gamma + beta;
//   with xh = (x - mean) * rstd and g = dy * gamma:
//   dx = rstd * (g - mean(g) - xh * mean(g * xh)) + add,
//   dgamma = sum over rows of dy * xh, dbeta = sum over rows of dy.
// Bound by memory: a row is read once and stays in registers between the
// sums and the outputs, as vectors of 16 bytes a lane (lane i of a row's
// group takes vectors i, i + G, ...). All sums are in 32 bits; the variance
// is that of the centred values, so a large mean costs no bits. 16-bit
// values are rounded once, on the way out.
//
// Measured: forward 8192 x 4096 f32 49 to 51 us in a row of calls, 268 MB at 5.4
// TB/s (a large copy takes 54 us for as many), 42 us on inputs that lie in the
// last-level cache in part; 8 x 4096 f16 3.7 us, a launch and two memory
// latencies. Backward 8192 x 4096 f16 with what is added, 270 MB, 51 us and 4.8
// us for the column sums; 4097 x 1000 f32 14.5 and 3.9 us.
#include <hip/hip_runtime.h>
#include "thvm_abi.h"
#include "block_args.h"
#include "block_mem.h"

template <typename T> struct Vec { static constexpr u32 N = 16 / sizeof(T); };

template <typename T> __device__ __forceinline__ void load_vec(const glob<T> *row, u32 e, u32 cols, float *out) {
    load_n<T, Vec<T>::N>(row, e, cols, out);
}
template <typename T> __device__ __forceinline__ void store_vec(glob<T> *row, u32 e, u32 cols, const float *in) {
    store_n<T, Vec<T>::N>(row, e, cols, in);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// The sum over a row's group of G lanes, on every lane of it, always in the
// same order. `slot` alternates between calls, so one barrier is enough.
template <u32 G, u32 K>
__device__ __forceinline__ void group_sum(float (&v)[K], float (*lds)[16], u32 slot) {
#pragma unroll
    for (u32 k = 0; k < K; k++) v[k] = wave_sum(v[k]);
    if (G == 64) return;
    constexpr u32 W = G / 64;
    const u32 wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63u) == 0)
#pragma unroll
        for (u32 k = 0; k < K; k++) lds[slot * K + k][wave] = v[k];
    __syncthreads();
#pragma unroll
    for (u32 k = 0; k < K; k++) {
        float s = 0.0f;
#pragma unroll
        for (u32 w = 0; w < W; w++) s += lds[slot * K + k][w];
        v[k] = s;
    }
}

// ---- forward ----

template <typename T, u32 G, u32 NV>
__device__ __forceinline__ void ln_fwd(const LnArgs &a) {
    constexpr u32 N = Vec<T>::N, PER = G < 256 ? 256 / G : 1;
    __shared__ float lds[4][16];
    const u32 lane = threadIdx.x % G;
    const u32 r = blockIdx.x * PER + threadIdx.x / G;
    if (PER > 1 && r >= a.rows) return;      // whole waves of their own, no barrier below
    const glob<T> *x = (const glob<T> *)a.x + (u64)r * a.cols;
    float v[NV][N];
    float s[1] = {0.0f};
#pragma unroll
    for (u32 i = 0; i < NV; i++) load_vec<T>(x, (lane + i * G) * N, a.cols, v[i]);
#pragma unroll
    for (u32 i = 0; i < NV; i++)
#pragma unroll
        for (u32 j = 0; j < N; j++) s[0] += v[i][j];
    group_sum<G, 1>(s, lds, 0);
    const float n = (float)a.cols, mean = s[0] / n;   // divided: exact for a constant row
    s[0] = 0.0f;
#pragma unroll
    for (u32 i = 0; i < NV; i++)
#pragma unroll
        for (u32 j = 0; j < N; j++) {
            v[i][j] -= mean;
            if ((lane + i * G) * N + j < a.cols) s[0] += v[i][j] * v[i][j];
        }
    group_sum<G, 1>(s, lds, 1);
    const float rstd = 1.0f / sqrtf(s[0] / n + a.eps);
    glob<T> *y = (glob<T> *)a.y + (u64)r * a.cols;
#pragma unroll
    for (u32 i = 0; i < NV; i++) {
        const u32 e = (lane + i * G) * N;
        if (e >= a.cols) continue;
        float g[N], b[N], o[N];
        if (a.gamma) load_vec<T>((const glob<T> *)a.gamma, e, a.cols, g);
        if (a.beta) load_vec<T>((const glob<T> *)a.beta, e, a.cols, b);
#pragma unroll
        for (u32 j = 0; j < N; j++) {
            o[j] = v[i][j] * rstd;
            if (a.gamma) o[j] *= g[j];
            if (a.beta) o[j] += b[j];
        }
        store_vec<T>(y, e, a.cols, o);
    }
    if (lane == 0) {
        if (a.mean) ((glob<float> *)a.mean)[r] = mean;
        if (a.rstd) ((glob<float> *)a.rstd)[r] = rstd;
    }
}

// A row that the registers of a workgroup do not hold is read three times.
template <typename T>
__device__ __forceinline__ void ln_fwd_long(const LnArgs &a) {
    constexpr u32 N = Vec<T>::N, G = 1024;
    __shared__ float lds[4][16];
    const u32 r = blockIdx.x;
    const glob<T> *x = (const glob<T> *)a.x + (u64)r * a.cols;
    float s[1] = {0.0f}, v[N];
    for (u64 e = (u64)threadIdx.x * N; e < a.cols; e += G * N) {
        load_vec<T>(x, (u32)e, a.cols, v);
#pragma unroll
        for (u32 j = 0; j < N; j++) s[0] += v[j];
    }
    group_sum<G, 1>(s, lds, 0);
    const float n = (float)a.cols, mean = s[0] / n;   // divided: exact for a constant row
    s[0] = 0.0f;
    for (u64 e = (u64)threadIdx.x * N; e < a.cols; e += G * N) {
        load_vec<T>(x, (u32)e, a.cols, v);
#pragma unroll
        for (u32 j = 0; j < N; j++)
            if (e + j < a.cols) s[0] += (v[j] - mean) * (v[j] - mean);
    }
    group_sum<G, 1>(s, lds, 1);
    const float rstd = 1.0f / sqrtf(s[0] / n + a.eps);
    glob<T> *y = (glob<T> *)a.y + (u64)r * a.cols;
    for (u64 e = (u64)threadIdx.x * N; e < a.cols; e += G * N) {
        float g[N], b[N];
        load_vec<T>(x, (u32)e, a.cols, v);
        if (a.gamma) load_vec<T>((const glob<T> *)a.gamma, (u32)e, a.cols, g);
        if (a.beta) load_vec<T>((const glob<T> *)a.beta, (u32)e, a.cols, b);
#pragma unroll
        for (u32 j = 0; j < N; j++) {
            v[j] = (v[j] - mean) * rstd;
            if (a.gamma) v[j] *= g[j];
            if (a.beta) v[j] += b[j];
        }
        store_vec<T>(y, (u32)e, a.cols, v);
    }
    if (threadIdx.x == 0) {
        if (a.mean) ((glob<float> *)a.mean)[r] = mean;
        if (a.rstd) ((glob<float> *)a.rstd)[r] = rstd;
    }
}

// ---- backward ----

// A workgroup takes rows blockIdx.x * PER + group, + gridDim.x * PER, ...; a
// lane owns the same columns of each, so the column sums of dy * xh and dy
// stay in its registers until the workgroup's rows are done. They are then
// added over the workgroup's groups and written as one row of the partial
// sums, which ln_cols adds in row order: no atomics, the same bits each time.
// The next row is asked for, as it lies in memory, before the current row's
// sums are waited for (where the registers hold it), and so is what is added
// to the current row.
template <typename T, u32 G, u32 NV>
__device__ __forceinline__ void ln_bwd(const LnGradArgs &a) {
    constexpr u32 N = Vec<T>::N, PER = G < 256 ? 256 / G : 1;
    constexpr bool AHEAD = NV * N <= 16;
    __shared__ float lds[4][16];
    __shared__ float comb[PER > 1 ? (PER - 1) * 64 * N : 1];
    const u32 lane = threadIdx.x % G, group = threadIdx.x / G;
    const u64 step = (u64)gridDim.x * PER;
    const float inv = 1.0f / (float)a.cols;
    float dg[NV][N], db[NV][N], gm[NV][N];
#pragma unroll
    for (u32 i = 0; i < NV; i++) {
#pragma unroll
        for (u32 j = 0; j < N; j++) dg[i][j] = db[i][j] = 0.0f, gm[i][j] = 1.0f;
        if (a.gamma) load_vec<T>((const glob<T> *)a.gamma, (lane + i * G) * N, a.cols, gm[i]);
    }
    any_vec<T, N> yr[NV], xr[NV], ar[NV];
    float mean1 = 0.0f, rstd1 = 0.0f;
    auto ask = [&](u64 r) {
        mean1 = ((const glob<float> *)a.mean)[r];
        rstd1 = ((const glob<float> *)a.rstd)[r];
#pragma unroll
        for (u32 i = 0; i < NV; i++) {
            yr[i] = load_raw<T, N>((const glob<T> *)a.dy + r * a.cols, (lane + i * G) * N, a.cols);
            xr[i] = load_raw<T, N>((const glob<T> *)a.x + r * a.cols, (lane + i * G) * N, a.cols);
        }
    };
    u64 r = (u64)blockIdx.x * PER + group;
    if (AHEAD && r < a.rows) ask(r);
    for (u32 slot = 0; r < a.rows; r += step, slot ^= 1u) {
        float y[NV][N], xh[NV][N];
        if (!AHEAD) ask(r);
        const float mean = mean1, rstd = rstd1;
        if (a.add && a.dx)
#pragma unroll
            for (u32 i = 0; i < NV; i++) ar[i] = load_raw<T, N>((const glob<T> *)a.add + r * a.cols, (lane + i * G) * N, a.cols);
#pragma unroll
        for (u32 i = 0; i < NV; i++)
#pragma unroll
            for (u32 j = 0; j < N; j++) y[i][j] = (float)yr[i][j], xh[i][j] = ((float)xr[i][j] - mean) * rstd;
        if (AHEAD && r + step < a.rows) ask(r + step);
        // past the row's end dy is 0: nothing there reaches a sum
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (u32 i = 0; i < NV; i++)
#pragma unroll
            for (u32 j = 0; j < N; j++) {
                if ((lane + i * G) * N + j >= a.cols) xh[i][j] = 0.0f;
                dg[i][j] += y[i][j] * xh[i][j];
                db[i][j] += y[i][j];
                y[i][j] *= gm[i][j];
                s[0] += y[i][j];
                s[1] += y[i][j] * xh[i][j];
            }
        if (!a.dx) continue;
        group_sum<G, 2>(s, lds, slot);
        const float c0 = s[0] * inv, c1 = s[1] * inv;
#pragma unroll
        for (u32 i = 0; i < NV; i++) {
            const u32 e = (lane + i * G) * N;
            if (e >= a.cols) continue;
            float o[N];
#pragma unroll
            for (u32 j = 0; j < N; j++) {
                o[j] = rstd * (y[i][j] - c0 - xh[i][j] * c1);
                if (a.add) o[j] += (float)ar[i][j];
            }
            store_vec<T>((glob<T> *)a.dx + r * a.cols, e, a.cols, o);
        }
    }
    if (!a.part) return;
    glob<float> *pg = (glob<float> *)a.part + (u64)blockIdx.x * 2u * a.cols, *pb = pg + a.cols;
#pragma unroll
    for (u32 i = 0; i < NV; i++) {
        const u32 e = (lane + i * G) * N;
        if (PER > 1) {
#pragma unroll
            for (u32 which = 0; which < 2; which++) {
                float *v = which ? db[i] : dg[i];
                __syncthreads();
                if (group)
#pragma unroll
                    for (u32 j = 0; j < N; j++) comb[((group - 1) * N + j) * 64 + lane] = v[j];
                __syncthreads();
                if (!group)
#pragma unroll
                    for (u32 p = 0; p < PER - 1; p++)
#pragma unroll
                        for (u32 j = 0; j < N; j++) v[j] += comb[(p * N + j) * 64 + lane];
            }
        }
        if (group || e >= a.cols) continue;
#pragma unroll
        for (u32 j = 0; j < N; j++)
            if (e + j < a.cols) pg[e + j] = dg[i][j], pb[e + j] = db[i][j];
    }
}

// The long rows' dx: three reads of x and dy.
template <typename T>
__device__ __forceinline__ void ln_bwd_long(const LnGradArgs &a) {
    constexpr u32 N = Vec<T>::N, G = 1024;
    __shared__ float lds[4][16];
    const u64 r = blockIdx.x;
    const glob<T> *x = (const glob<T> *)a.x + r * a.cols, *dy = (const glob<T> *)a.dy + r * a.cols;
    const float mean = ((const glob<float> *)a.mean)[r], rstd = ((const glob<float> *)a.rstd)[r], inv = 1.0f / (float)a.cols;
    float s[2] = {0.0f, 0.0f}, v[N], y[N], g[N];
    for (u64 e = (u64)threadIdx.x * N; e < a.cols; e += G * N) {
        load_vec<T>(x, (u32)e, a.cols, v);
        load_vec<T>(dy, (u32)e, a.cols, y);
        if (a.gamma) load_vec<T>((const glob<T> *)a.gamma, (u32)e, a.cols, g);
#pragma unroll
        for (u32 j = 0; j < N; j++) {
            if (e + j >= a.cols) continue;
            const float t = a.gamma ? y[j] * g[j] : y[j];
            s[0] += t;
            s[1] += t * ((v[j] - mean) * rstd);
        }
    }
    group_sum<G, 2>(s, lds, 0);
    const float c0 = s[0] * inv, c1 = s[1] * inv;
    for (u64 e = (u64)threadIdx.x * N; e < a.cols; e += G * N) {
        float ad[N];
        load_vec<T>(x, (u32)e, a.cols, v);
        load_vec<T>(dy, (u32)e, a.cols, y);
        if (a.gamma) load_vec<T>((const glob<T> *)a.gamma, (u32)e, a.cols, g);
        if (a.add) load_vec<T>((const glob<T> *)a.add + r * a.cols, (u32)e, a.cols, ad);
#pragma unroll
        for (u32 j = 0; j < N; j++) {
            const float t = a.gamma ? y[j] * g[j] : y[j];
            v[j] = rstd * (t - c0 - (v[j] - mean) * rstd * c1);
            if (a.add) v[j] += ad[j];
        }
        store_vec<T>((glob<T> *)a.dx + r * a.cols, (u32)e, a.cols, v);
    }
}

// The long rows' partial column sums: 256 columns a workgroup, a run of rows
// each (blockIdx.y of a.parts).
template <typename T>
__device__ __forceinline__ void ln_part_long(const LnGradArgs &a) {
    const u32 c = blockIdx.x * 256u + threadIdx.x;
    if (c >= a.cols) return;
    const u64 per = ((u64)a.rows + a.parts - 1) / a.parts, r0 = per * blockIdx.y;
    const u64 r1 = r0 + per < a.rows ? r0 + per : a.rows;
    float dg = 0.0f, db = 0.0f;
    for (u64 r = r0; r < r1; r++) {
        const float y = (float)((const glob<T> *)a.dy)[r * a.cols + c];
        dg += y * (((float)((const glob<T> *)a.x)[r * a.cols + c] - ((const glob<float> *)a.mean)[r]) * ((const glob<float> *)a.rstd)[r]);
        db += y;
    }
    glob<float> *p = (glob<float> *)a.part + (u64)blockIdx.y * 2u * a.cols;
    p[c] = dg;
    p[a.cols + c] = db;
}

// dgamma and dbeta from `parts` rows of partial sums [2][cols]: a workgroup
// takes 32 of the 2 * cols columns, 32 groups of its lanes every 32nd part,
// and adds the groups' sums in order.
template <typename T>
__device__ __forceinline__ void ln_cols(const LnGradArgs &a) {
    __shared__ float lds[32][33];
    const u32 lane = threadIdx.x & 31u, group = threadIdx.x >> 5;
    const u64 c = (u64)blockIdx.x * 32u + lane, n2 = 2ull * a.cols;
    float s = 0.0f;
    if (c < n2)
#pragma unroll 8
        for (u32 p = group; p < a.parts; p += 32) s += ((const glob<float> *)a.part)[p * n2 + c];
    lds[group][lane] = s;
    __syncthreads();
    if (group || c >= n2) return;
#pragma unroll
    for (u32 w = 1; w < 32; w++) s += lds[w][lane];
    glob<T> *out = c < a.cols ? (glob<T> *)a.dgamma : (glob<T> *)a.dbeta;
    if (out) out[c < a.cols ? c : c - a.cols] = (T)s;
}

#define LN_KERNELS(T, G, NV)                                                                                       \
    extern "C" __global__ __launch_bounds__(G < 256 ? 256 : G) void thvm_ln_##T##_##G##_##NV(LnArgs a) {           \
        ln_fwd<T, G, NV>(a);                                                                                        \
    }
#define LNB_KERNELS(T, G, NV)                                                                                      \
    extern "C" __global__ __launch_bounds__(G < 256 ? 256 : G) void thvm_lnb_##T##_##G##_##NV(LnGradArgs a) {      \
        ln_bwd<T, G, NV>(a);                                                                                        \
    }
#define LN_ALL(T)                                                                                                  \
    LN_KERNELS(T, 64, 1) LN_KERNELS(T, 64, 2) LN_KERNELS(T, 64, 4)                                                 \
    LN_KERNELS(T, 256, 1) LN_KERNELS(T, 256, 2) LN_KERNELS(T, 256, 4)                                              \
    LN_KERNELS(T, 1024, 1) LN_KERNELS(T, 1024, 2) LN_KERNELS(T, 1024, 4)                                          \
    extern "C" __global__ __launch_bounds__(1024) void thvm_ln_##T##_long(LnArgs a) { ln_fwd_long<T>(a); }         \
    extern "C" __global__ __launch_bounds__(1024) void thvm_lnb_##T##_long(LnGradArgs a) { ln_bwd_long<T>(a); }    \
    extern "C" __global__ __launch_bounds__(256) void thvm_lnb_##T##_part(LnGradArgs a) { ln_part_long<T>(a); }    \
    extern "C" __global__ __launch_bounds__(1024) void thvm_lnb_##T##_cols(LnGradArgs a) { ln_cols<T>(a); }
LN_ALL(f32)
LN_ALL(f16)
LNB_KERNELS(f32, 64, 1) LNB_KERNELS(f32, 64, 2) LNB_KERNELS(f32, 64, 4)
LNB_KERNELS(f32, 256, 2) LNB_KERNELS(f32, 512, 2) LNB_KERNELS(f32, 512, 4) LNB_KERNELS(f32, 512, 8)
LNB_KERNELS(f16, 64, 1) LNB_KERNELS(f16, 64, 2)
LNB_KERNELS(f16, 256, 1) LNB_KERNELS(f16, 512, 1) LNB_KERNELS(f16, 512, 2) LNB_KERNELS(f16, 512, 4)
