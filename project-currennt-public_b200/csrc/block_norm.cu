// Norms before and after a residual block, fused with the block's gate and residual scale, and their gradients.
//
//   n = w2 * norm(f) + b2        the block's output f normalised (after the block)
//   y = x + a * gate * n         gated, scaled and added to the residual stream
//   h = w1 * norm(y) + b1        normalised for the next block (before it)
//
// norm(v) = (v - mean) / sqrt(var + eps) (layer norm) or v / sqrt(mean(v^2) + eps) (RMS norm).  y is rounded to the tensors' type before the
// second norm, so that a backward pass that reads y differentiates what the forward pass computed.  The gate has gate_rows rows; frame r
// takes row r % gate_rows: one row for all frames, one for each of the parallel sequences of a time-major fraction, or one per frame.
//
// Backward, with u1 = (y - m1) r1, u2 = (f - m2) r2 and d the gradients coming in:
//   dt = dy + r1 (w1 dh - [mean(w1 dh)] - u1 mean(w1 dh u1)),   dx = dt,   dn = a gate dt,   dgate = a dt n
//   df = r2 (w2 dn - [mean(w2 dn)] - u2 mean(w2 dn u2)),   dw1 = sum dh u1, db1 = sum dh, dw2 = sum dn u2, db2 = sum dn   (over frames)
//
// Bound by memory: a row stays in registers between its loads and its stores, so every tensor is read once and written once.  A warp
// takes a row where 4 vectors a lane hold it, a block otherwise.  The backward kernel has a fixed number of workers; a worker keeps
// the same columns for all its rows, so the sums over frames stay in registers until the end, go to the workspace once, and are
// added there in a fixed order by a second launch: no atomics, the same bits every time.
#include <math.h>

#include "typed.cuh"

namespace b2 {
namespace {

constexpr int MAX_DIM = 8192;

struct NormArgs {
    const char *pat;
    const float *w1, *b1, *w2, *b2;
    const void *gate;
    float4 *stats;                    // per row: mean and 1/deviation of f, of y
    long long rows, gate_rows, ld_gate;
    int dim, layer_norm;
    float eps, a, inv_dim;
};

// sums over the threads of a row: a warp, or all warps of the block (buffers alternate, so one barrier a sum is enough)
template <int N> __device__ __forceinline__ void row_sums(float (&x)[N], int warps, float (*red)[N], int &phase) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = warp_sum(x[i]);
    if (warps == 1) return;
    float(*buf)[N] = red + (phase & 1) * 32;
    ++phase;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) buf[threadIdx.x >> 5][i] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float y = (int)(threadIdx.x & 31) < warps ? buf[threadIdx.x & 31][i] : 0.0f;
        x[i] = warp_sum(y);
    }
}

// columns of a thread: vector i starts at column (i * tpr + lane) * W
template <typename T, int W, int NV> struct Cols {
    static __device__ __forceinline__ void load(float (&v)[NV][W], const T *row, int tpr, int lane, int dim, float other) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * tpr + lane) * W;
            if (c < dim) load_vec<T, W>(v[i], row + c);
            else
#pragma unroll
                for (int j = 0; j < W; ++j) v[i][j] = other;
        }
    }
    static __device__ __forceinline__ void store(T *row, const float (&v)[NV][W], int tpr, int lane, int dim) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * tpr + lane) * W;
            if (c < dim) store_vec<T, W>(row + c, v[i]);
        }
    }
};

// v becomes its normalised self; columns beyond dim are zero before and stay so
template <int W, int NV>
__device__ __forceinline__ void normalise(float (&v)[NV][W], const NormArgs &a, int tpr, int lane, int warps, float (*red)[1], int &phase, float &mean, float &rstd) {
    float s[1] = {0.0f};
    mean = 0.0f;
    if (a.layer_norm) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) s[0] += v[i][j];
        row_sums<1>(s, warps, red, phase);
        mean = s[0] * a.inv_dim;
        s[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if ((i * tpr + lane) * W < a.dim)
#pragma unroll
                for (int j = 0; j < W; ++j) v[i][j] -= mean;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) s[0] = fmaf(v[i][j], v[i][j], s[0]);
    row_sums<1>(s, warps, red, phase);
    rstd = 1.0f / sqrtf(fmaf(s[0], a.inv_dim, a.eps));
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) v[i][j] *= rstd;
}

template <int W, int NV> __device__ __forceinline__ void affine(float (&v)[NV][W], const float *w, const float *b, int tpr, int lane, int dim) {
    float q[NV][W];
    if (w) {
        Cols<float, W, NV>::load(q, w, tpr, lane, dim, 0.0f);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) v[i][j] *= q[i][j];
    }
    if (b) {
        Cols<float, W, NV>::load(q, b, tpr, lane, dim, 0.0f);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) v[i][j] += q[i][j];
    }
}

// tpr threads a row: 32 (the block holds 8 rows) or the whole block
template <typename T, int W, int NV>
__global__ void __launch_bounds__(NV == 8 ? 1024 : 512) block_norm_forward_kernel(const NormArgs a, const T *x, long long ld_x, const T *f, long long ld_f, T *y,
                                                                                  long long ld_y, T *h, long long ld_h, int tpr) {
    __shared__ float red[64][1];
    const int warps = tpr >> 5, lane = warps == 1 ? (threadIdx.x & 31) : threadIdx.x;
    const long long r = warps == 1 ? (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    if (r >= a.rows) return;
    int phase = 0;
    typedef Cols<T, W, NV> C;
    float v[NV][W], n[NV][W];
    float4 st = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (a.pat && a.pat[r] == PAT_NONE) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) v[i][j] = 0.0f;
        if (y) C::store(y + r * ld_y, v, tpr, lane, a.dim);
        if (h) C::store(h + r * ld_h, v, tpr, lane, a.dim);
        if (a.stats && lane == 0) a.stats[r] = st;
        return;
    }
    C::load(v, x + r * ld_x, tpr, lane, a.dim, 0.0f);
    if (f) {
        float g[NV][W];
        C::load(n, f + r * ld_f, tpr, lane, a.dim, 0.0f);
        if (a.gate) C::load(g, (const T *)a.gate + (r % a.gate_rows) * a.ld_gate, tpr, lane, a.dim, 0.0f);
        normalise<W, NV>(n, a, tpr, lane, warps, red, phase, st.x, st.y);
        affine<W, NV>(n, a.w2, a.b2, tpr, lane, a.dim);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const float s = a.gate ? a.a * g[i][j] : a.a;
                v[i][j] = to_float(from_float<T>(fmaf(s, n[i][j], v[i][j])));
            }
    }
    if (y) C::store(y + r * ld_y, v, tpr, lane, a.dim);
    if (h) {
        normalise<W, NV>(v, a, tpr, lane, warps, red, phase, st.z, st.w);
        affine<W, NV>(v, a.w1, a.b1, tpr, lane, a.dim);
        C::store(h + r * ld_h, v, tpr, lane, a.dim);
    }
    if (a.stats && lane == 0) a.stats[r] = st;
}

struct BackArgs {
    long long ld_dx, ld_df, ld_dy, ld_dh, ld_y, ld_f, ld_dgate;
    void *dgate;
    float *partial;                   // [blocks][4][dim_pad]: dw1, db1, dw2, db2 of every block
    float *partial_gate;              // [workers][dim_pad], where several workers share a row of the gate
    int dim_pad, per_group, groups_at_once;
};

// A worker is a warp (tpr = 32) or a block.  per_group workers share a row of the gate (all workers, if there is one row or none), and
// groups_at_once rows of the gate are worked on side by side.
// BIAS: means are subtracted or the norms have a bias (without both, sums are saved).
template <typename T, int W, int NV, int MAXT, bool BIAS>
__global__ void __launch_bounds__(MAXT) block_norm_backward_kernel(const NormArgs a, const BackArgs k, T *dx, T *df, const T *dy, const T *dh, const T *y, const T *f, int tpr) {
    constexpr int S = BIAS ? 2 : 1;
    __shared__ float red[64][S];
    extern __shared__ __align__(16) float join[];   // [warps][32 * W * NV], tpr = 32 only
    typedef Cols<T, W, NV> C;
    const int warps = tpr >> 5, lane = warps == 1 ? (threadIdx.x & 31) : threadIdx.x;
    const long long worker = warps == 1 ? (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    const long long G = a.gate_rows > 0 ? a.gate_rows : 1, R = a.rows / G;
    int phase = 0;
    float w1[NV][W], w2[NV][W], b2[NV][W];
    float s_w1[NV][W], s_b1[NV][W], s_w2[NV][W], s_b2[NV][W], s_g[NV][W];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) {
            w1[i][j] = w2[i][j] = 1.0f;
            b2[i][j] = s_w1[i][j] = s_b1[i][j] = s_w2[i][j] = s_b2[i][j] = s_g[i][j] = 0.0f;
        }
    if (a.w1) Cols<float, W, NV>::load(w1, a.w1, tpr, lane, a.dim, 0.0f);
    if (a.w2) Cols<float, W, NV>::load(w2, a.w2, tpr, lane, a.dim, 0.0f);
    if (BIAS && a.b2) Cols<float, W, NV>::load(b2, a.b2, tpr, lane, a.dim, 0.0f);
    const long long group0 = worker / k.per_group;
    const int member = (int)(worker - group0 * k.per_group);
    if (group0 < k.groups_at_once)
        for (long long g = group0; g < G; g += k.groups_at_once) {
            for (long long m = member; m < R; m += k.per_group) {
                const long long r = m * G + g;
                if (a.pat && a.pat[r] == PAT_NONE) {
                    float z[NV][W];
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int j = 0; j < W; ++j) z[i][j] = 0.0f;
                    if (dx) C::store(dx + r * k.ld_dx, z, tpr, lane, a.dim);
                    if (df) C::store(df + r * k.ld_df, z, tpr, lane, a.dim);
                    continue;
                }
                float t[NV][W], u[NV][W], d[NV][W], gt[NV][W];
                const float4 st = a.stats[r];
                if (dy) C::load(t, dy + r * k.ld_dy, tpr, lane, a.dim, 0.0f);
                else
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int j = 0; j < W; ++j) t[i][j] = 0.0f;
                if (dh) {
                    C::load(d, dh + r * k.ld_dh, tpr, lane, a.dim, 0.0f);
                    C::load(u, y + r * k.ld_y, tpr, lane, a.dim, st.z);
                }
                float fv[NV][W];
                if (f) {
                    C::load(fv, f + r * k.ld_f, tpr, lane, a.dim, st.x);
                    if (a.gate) C::load(gt, (const T *)a.gate + g * a.ld_gate, tpr, lane, a.dim, 0.0f);
                }
                if (dh) {
                    float s[S] = {};
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int j = 0; j < W; ++j) {
                            u[i][j] = (u[i][j] - st.z) * st.w;
                            s_w1[i][j] = fmaf(d[i][j], u[i][j], s_w1[i][j]);
                            if (BIAS) s_b1[i][j] += d[i][j];
                            d[i][j] *= w1[i][j];
                            s[0] = fmaf(d[i][j], u[i][j], s[0]);
                            if (BIAS) s[S - 1] += d[i][j];
                        }
                    row_sums<S>(s, warps, red, phase);
                    const float p = s[0] * a.inv_dim, q = BIAS && a.layer_norm ? s[S - 1] * a.inv_dim : 0.0f;
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int j = 0; j < W; ++j) t[i][j] = fmaf(st.w, fmaf(-u[i][j], p, d[i][j] - q), t[i][j]);
                }
                if (dx) C::store(dx + r * k.ld_dx, t, tpr, lane, a.dim);
                if (f) {
                    float s[S] = {};
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int j = 0; j < W; ++j) {
                            u[i][j] = (fv[i][j] - st.x) * st.y;
                            const float at = a.a * t[i][j];
                            s_g[i][j] = fmaf(at, fmaf(u[i][j], w2[i][j], b2[i][j]), s_g[i][j]);
                            const float dn = (i * tpr + lane) * W < a.dim ? (a.gate ? at * gt[i][j] : at) : 0.0f;
                            s_w2[i][j] = fmaf(dn, u[i][j], s_w2[i][j]);
                            if (BIAS) s_b2[i][j] += dn;
                            d[i][j] = dn * w2[i][j];
                            s[0] = fmaf(d[i][j], u[i][j], s[0]);
                            if (BIAS) s[S - 1] += d[i][j];
                        }
                    if (df) {
                        row_sums<S>(s, warps, red, phase);
                        const float p = s[0] * a.inv_dim, q = BIAS && a.layer_norm ? s[S - 1] * a.inv_dim : 0.0f;
#pragma unroll
                        for (int i = 0; i < NV; ++i)
#pragma unroll
                            for (int j = 0; j < W; ++j) d[i][j] = st.y * fmaf(-u[i][j], p, d[i][j] - q);
                        C::store(df + r * k.ld_df, d, tpr, lane, a.dim);
                    }
                }
            }
            if (k.dgate) {
                if (k.per_group == 1) C::store((T *)k.dgate + g * k.ld_dgate, s_g, tpr, lane, a.dim);
                else Cols<float, W, NV>::store(k.partial_gate + worker * k.dim_pad, s_g, tpr, lane, a.dim);
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < W; ++j) s_g[i][j] = 0.0f;
            }
        }
    if (!k.partial) return;
    float *out = k.partial + (size_t)blockIdx.x * 4 * k.dim_pad;
    if (warps > 1) {
        Cols<float, W, NV>::store(out, s_w1, tpr, lane, a.dim);
        Cols<float, W, NV>::store(out + k.dim_pad, s_b1, tpr, lane, a.dim);
        Cols<float, W, NV>::store(out + 2 * k.dim_pad, s_w2, tpr, lane, a.dim);
        Cols<float, W, NV>::store(out + 3 * k.dim_pad, s_b2, tpr, lane, a.dim);
    } else {
        const int w = threadIdx.x >> 5, nw = blockDim.x >> 5, width = 32 * W * NV;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            Cols<float, W, NV>::store(join + w * width, q == 0 ? s_w1 : q == 1 ? s_b1 : q == 2 ? s_w2 : s_b2, tpr, lane, width);
            __syncthreads();
            for (int c = threadIdx.x; c < a.dim; c += blockDim.x) {
                float s = 0.0f;
                for (int i = 0; i < nw; ++i) s += join[i * width + c];
                out[q * k.dim_pad + c] = s;
            }
            __syncthreads();
        }
    }
}

// Sums of the workspace over blocks (blockIdx.y < 4: one weight gradient each) or over the workers of a row of the gate.
// 32 columns x 32 phases a block; the phases are added in order.
struct ReduceArgs {
    const float *partial, *partial_gate;
    float *out[4];
    void *dgate;
    long long ld_dgate;
    int dim, dim_pad, blocks, per_group;
};
template <typename T> __global__ void __launch_bounds__(1024) block_norm_reduce_kernel(const ReduceArgs a) {
    __shared__ float part[32][33];
    grid_wait();
    const int c = blockIdx.x * 32 + threadIdx.x, y = threadIdx.y, q = blockIdx.y;
    const bool gate = q >= 4;
    if (!gate && !a.out[q]) return;
    const float *p = gate ? a.partial_gate + (size_t)(q - 4) * a.per_group * a.dim_pad : a.partial + (size_t)q * a.dim_pad;
    const size_t step = gate ? a.dim_pad : (size_t)4 * a.dim_pad;
    const int n = gate ? a.per_group : a.blocks;
    float s = 0.0f;
    if (c < a.dim)
#pragma unroll 4
        for (int i = y; i < n; i += 32) s += p[(size_t)i * step + c];
    part[y][threadIdx.x] = s;
    __syncthreads();
    if (y == 0 && c < a.dim) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += part[i][threadIdx.x];
        if (gate) ((T *)a.dgate)[(long long)(q - 4) * a.ld_dgate + c] = from_float<T>(t);
        else a.out[q][c] = t;
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------
// widest vectors (16 bytes) only where every row of every tensor starts and ends on them
struct Width {
    int w;
    int elem;
    void rows(const void *p, long long ld) { if (p && (ld % w || !aligned_to(p, 16))) w = 1; }
    void floats(const float *p) { if (!aligned_to(p, 16)) w = 1; }
};
Width width_of(const b2_block_norm *d) {
    Width x = {16 / type_size(d->type), type_size(d->type)};
    if (d->dim % x.w) x.w = 1;
    x.rows(d->gate, d->ld_gate);
    x.floats(d->w_pre); x.floats(d->b_pre); x.floats(d->w_post); x.floats(d->b_post);
    return x;
}

int check(const char *who, const b2_block_norm *d) {
    if (!d) { set_error("%s: null pointer", who); return B2_ERR_BAD_ARG; }
    const int e = type_size(d->type);
    if (!e) { set_error("%s: unknown element type %d", who, d->type); return B2_ERR_BAD_ARG; }
    if (d->rows < 0 || d->rows > 0x7fffffffll || d->dim < 1 || d->dim > MAX_DIM) {
        set_error("%s: %lld rows of %d (at most 2^31 - 1 and %d)", who, d->rows, d->dim, MAX_DIM);
        return B2_ERR_BAD_SHAPE;
    }
    if (!(d->eps >= 0.0f) || d->eps > 3.4e38f || d->residual_scale != d->residual_scale) {
        set_error("%s: epsilon %g, residual scale %g", who, (double)d->eps, (double)d->residual_scale);
        return B2_ERR_BAD_ARG;
    }
    if (d->gate) {
        if (d->gate_rows < 1 || (d->rows && d->rows % d->gate_rows)) {
            set_error("%s: a gate of %lld rows for %lld frames (the frames must be a multiple)", who, d->gate_rows, d->rows);
            return B2_ERR_BAD_SHAPE;
        }
        if (d->ld_gate < d->dim) { set_error("%s: leading dimension of the gate too small (%lld for %d columns)", who, d->ld_gate, d->dim); return B2_ERR_BAD_ARG; }
        if (!aligned_to(d->gate, e)) { set_error("%s: the gate is not aligned to its elements", who); return B2_ERR_BAD_ARG; }
    }
    if (!aligned_to(d->w_pre, 4) || !aligned_to(d->b_pre, 4) || !aligned_to(d->w_post, 4) || !aligned_to(d->b_post, 4) || !aligned_to(d->stats, 16)) {
        set_error("%s: weights have to be aligned to 4 bytes, the statistics to 16", who);
        return B2_ERR_BAD_ARG;
    }
    return B2_OK;
}
int check_rows(const char *who, const char *name, const b2_block_norm *d, const void *p, long long ld) {
    if (!p) return B2_OK;
    if (ld < d->dim) { set_error("%s: leading dimension of %s too small (%lld for %d columns)", who, name, ld, d->dim); return B2_ERR_BAD_ARG; }
    if (!aligned_to(p, type_size(d->type))) { set_error("%s: %s is not aligned to its elements", who, name); return B2_ERR_BAD_ARG; }
    return B2_OK;
}
NormArgs args_of(const b2_block_norm *d) {
    return {d->pat_types, d->w_pre, d->b_pre, d->w_post, d->b_post, d->gate, (float4 *)d->stats, d->rows, d->gate ? d->gate_rows : 1, d->ld_gate, d->dim,
            d->layer_norm ? 1 : 0, d->eps, d->residual_scale, 1.0f / (float)d->dim};
}

template <typename T, int W>
int forward(const b2_block_norm *d, const T *x, long long ld_x, const T *f, long long ld_f, T *y, long long ld_y, T *h, long long ld_h, cudaStream_t st) {
    const NormArgs a = args_of(d);
    const int vecs = (d->dim + W - 1) / W;
    const auto go = [&](auto kernel, int tpr) -> int {
        const unsigned blocks = tpr == 32 ? (unsigned)((d->rows + 7) / 8) : (unsigned)d->rows;
        kernel<<<blocks, tpr == 32 ? 256 : tpr, 0, st>>>(a, x, ld_x, f, ld_f, y, ld_y, h, ld_h, tpr);
        count_launch();
        B2_CUDA(cudaGetLastError());
        return B2_OK;
    };
    if (vecs <= 32) return go(block_norm_forward_kernel<T, W, 1>, 32);
    if (vecs <= 64) return go(block_norm_forward_kernel<T, W, 2>, 32);
    if (vecs <= 128) return go(block_norm_forward_kernel<T, W, 4>, 32);
    if (vecs <= 2048) return go(block_norm_forward_kernel<T, W, 4>, (int)pow2_at_least((unsigned)(vecs + 3) / 4));
    return go(block_norm_forward_kernel<T, W, 8>, (int)pow2_at_least((unsigned)(vecs + 7) / 8));
}

// Workers of the backward pass.  tpr: threads a row; blocks: as many as 1024 threads per multiprocessor give
struct BackPlan { int tpr, threads, blocks, workers, per_group, groups_at_once; };
int back_tpr(int vecs) {
    const int t = (int)pow2_at_least((unsigned)vecs);
    return t < 32 ? 32 : t > 1024 ? 1024 : t;
}
BackPlan back_plan(long long rows, int vecs, long long gate_rows) {
    BackPlan p;
    p.tpr = back_tpr(vecs);
    p.threads = p.tpr == 32 ? 256 : p.tpr;
    const int each = p.threads / p.tpr;
    long long blocks = (long long)sm_count() * 1024 / (p.threads < 256 ? 256 : p.threads);
    if (blocks * each > rows) blocks = (rows + each - 1) / each;
    p.blocks = (int)blocks;
    p.workers = p.blocks * each;
    const long long G = gate_rows > 0 ? gate_rows : 1;
    p.per_group = (int)(p.workers / G);
    if (p.per_group < 1) p.per_group = 1;
    if (p.per_group > rows / G) p.per_group = (int)(rows / G);
    p.groups_at_once = p.workers / p.per_group;
    return p;
}

template <typename T, int W>
int backward(const b2_block_norm *d, T *dx, long long ld_dx, T *df, long long ld_df, T *dgate, long long ld_dgate, float *const (&dw)[4], const T *dy, long long ld_dy,
             const T *dh, long long ld_dh, const T *y, long long ld_y, const T *f, long long ld_f, float *ws, cudaStream_t st) {
    const NormArgs a = args_of(d);
    const int vecs = (d->dim + W - 1) / W;
    const BackPlan p = back_plan(d->rows, vecs, d->gate ? d->gate_rows : 0);
    BackArgs k = {ld_dx, ld_df, ld_dy, ld_dh, ld_y, ld_f, ld_dgate, dgate, nullptr, nullptr, (d->dim + 15) / 16 * 16, p.per_group, p.groups_at_once};
    const bool sums = dw[0] || dw[1] || dw[2] || dw[3], gate_sums = dgate && p.per_group > 1;
    if (sums) k.partial = ws;
    k.partial_gate = ws + (size_t)p.blocks * 4 * k.dim_pad;
    const auto go = [&](auto kernel, int smem) -> int {
        kernel<<<p.blocks, p.threads, smem, st>>>(a, k, dx, df, dy, dh, y, f, p.tpr);
        count_launch();
        B2_CUDA(cudaGetLastError());
        return B2_OK;
    };
    const int smem = p.tpr == 32 ? 8 * 32 * W * 4 : 0;
    const bool bias = d->layer_norm || dw[1] || dw[3] || d->b_post;
    const auto pick = [&](auto b) {
        constexpr bool B = decltype(b)::value;
        if (vecs <= 256) return go(block_norm_backward_kernel<T, W, 1, 256, B>, smem);
        if (vecs <= 512) return go(block_norm_backward_kernel<T, W, 1, 512, B>, 0);
        if (vecs <= 1024) return go(block_norm_backward_kernel<T, W, 1, 1024, B>, 0);
        if (vecs <= 2048) return go(block_norm_backward_kernel<T, W, 2, 1024, B>, 0);
        return go(block_norm_backward_kernel<T, 1, 8, 1024, B>, 0);
    };
    B2_TRY(bias ? pick(std::true_type()) : pick(std::false_type()));
    if (!sums && !gate_sums) return B2_OK;
    const ReduceArgs r = {k.partial, k.partial_gate, {dw[0], dw[1], dw[2], dw[3]}, gate_sums ? dgate : nullptr, ld_dgate, d->dim, k.dim_pad, p.blocks, p.per_group};
    const unsigned groups = gate_sums ? (unsigned)(d->gate ? d->gate_rows : 1) : 0;
    return launch_chained(block_norm_reduce_kernel<T>, dim3((d->dim + 31) / 32, 4 + groups), dim3(32, 32), 0, st, r);
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

int b2_block_norm_forward(const b2_block_norm *d, const void *x, long long ld_x, const void *f, long long ld_f, void *y, long long ld_y, void *h, long long ld_h,
                          b2_stream stream) {
    const char *who = "b2_block_norm_forward";
    B2_TRY(check(who, d));
    B2_TRY(check_rows(who, "x", d, x, ld_x));
    B2_TRY(check_rows(who, "f", d, f, ld_f));
    B2_TRY(check_rows(who, "y", d, y, ld_y));
    B2_TRY(check_rows(who, "h", d, h, ld_h));
    if (!d->rows) return B2_OK;
    if (!x || (!y && !h) || (f && !y)) { set_error("%s: null pointer (x, and y where there is f, are needed; y or h is written)", who); return B2_ERR_BAD_ARG; }
    if (h == x || (f && (h == f || y == f)) || (h && h == y)) { set_error("%s: only y may take the place of x", who); return B2_ERR_BAD_ARG; }
    if (y == x && ld_y != ld_x) { set_error("%s: y takes the place of x with another leading dimension", who); return B2_ERR_BAD_ARG; }
    Width w = width_of(d);
    w.rows(x, ld_x); w.rows(f, ld_f); w.rows(y, ld_y); w.rows(h, ld_h);
    return with_type(d->type, [&](auto *t) {
        typedef B2_ELEM(t) T;
        constexpr int W = 16 / sizeof(T);
        if (w.w == W) return forward<T, W>(d, (const T *)x, ld_x, (const T *)f, ld_f, (T *)y, ld_y, (T *)h, ld_h, (cudaStream_t)stream);
        return forward<T, 1>(d, (const T *)x, ld_x, (const T *)f, ld_f, (T *)y, ld_y, (T *)h, ld_h, (cudaStream_t)stream);
    });
}

size_t b2_block_norm_backward_workspace(long long rows, int dim, long long gate_rows) {
    if (rows < 1 || rows > 0x7fffffffll || dim < 1 || dim > MAX_DIM || gate_rows < 0) return 0;
    // enough for any type and alignment, that is for every width of the vectors
    size_t most = 0;
    for (int w = 1; w <= 8; w *= 2) {
        const BackPlan p = back_plan(rows, (dim + w - 1) / w, gate_rows);
        const size_t n = (size_t)p.blocks * 4 + p.workers;
        if (n > most) most = n;
    }
    return most * ((dim + 15) / 16 * 16) * sizeof(float);
}

int b2_block_norm_backward(const b2_block_norm *d, void *dx, long long ld_dx, void *df, long long ld_df, void *dgate, long long ld_dgate, float *dw_pre, float *db_pre,
                           float *dw_post, float *db_post, const void *dy, long long ld_dy, const void *dh, long long ld_dh, const void *y, long long ld_y, const void *f,
                           long long ld_f, void *workspace, size_t workspace_bytes, b2_stream stream) {
    const char *who = "b2_block_norm_backward";
    B2_TRY(check(who, d));
    B2_TRY(check_rows(who, "dx", d, dx, ld_dx));
    B2_TRY(check_rows(who, "df", d, df, ld_df));
    B2_TRY(check_rows(who, "dgate", d, dgate, ld_dgate));
    B2_TRY(check_rows(who, "dy", d, dy, ld_dy));
    B2_TRY(check_rows(who, "dh", d, dh, ld_dh));
    B2_TRY(check_rows(who, "y", d, y, ld_y));
    B2_TRY(check_rows(who, "f", d, f, ld_f));
    if (!aligned_to(dw_pre, 4) || !aligned_to(db_pre, 4) || !aligned_to(dw_post, 4) || !aligned_to(db_post, 4)) {
        set_error("%s: weight gradients have to be aligned to 4 bytes", who);
        return B2_ERR_BAD_ARG;
    }
    if (dgate && !d->gate) { set_error("%s: a gradient for a gate that is not there", who); return B2_ERR_BAD_ARG; }
    if ((df || dgate || dw_post || db_post) && !f) { set_error("%s: gradients of the norm after the block need f", who); return B2_ERR_BAD_ARG; }
    if ((dw_pre || db_pre) && !dh) { set_error("%s: gradients of the norm before the block need dh", who); return B2_ERR_BAD_ARG; }
    if (!d->rows) {
        // sums over no frames
        float *w[4] = {dw_pre, db_pre, dw_post, db_post};
        for (float *p : w)
            if (p) B2_CUDA(cudaMemsetAsync(p, 0, (size_t)d->dim * sizeof(float), (cudaStream_t)stream));
        if (dgate) B2_CUDA(cudaMemset2DAsync(dgate, (size_t)ld_dgate * type_size(d->type), 0, (size_t)d->dim * type_size(d->type), (size_t)d->gate_rows, (cudaStream_t)stream));
        return B2_OK;
    }
    if (!d->stats || (!dy && !dh) || (dh && !y)) { set_error("%s: null pointer (the statistics, dy or dh, and y where there is dh, are needed)", who); return B2_ERR_BAD_ARG; }
    if (!workspace || !aligned_to(workspace, 16)) { set_error("%s: the workspace is missing or not aligned to 16 bytes", who); return B2_ERR_BAD_ARG; }
    const size_t need = b2_block_norm_backward_workspace(d->rows, d->dim, d->gate ? d->gate_rows : 0);
    if (workspace_bytes < need) { set_error("%s: %zu bytes of workspace, %zu are needed", who, workspace_bytes, need); return B2_ERR_BAD_SHAPE; }
    const void *in[4] = {dy, dh, y, f};
    const long long ld_in[4] = {ld_dy, ld_dh, ld_y, ld_f};
    for (int i = 0; i < 4; ++i)
        if ((in[i] && in[i] == dx && ld_in[i] != ld_dx) || (in[i] && in[i] == df && ld_in[i] != ld_df)) {
            set_error("%s: a gradient takes the place of an input with another leading dimension", who);
            return B2_ERR_BAD_ARG;
        }
    if (dx && dx == df) { set_error("%s: dx and df are the same", who); return B2_ERR_BAD_ARG; }
    Width w = width_of(d);
    w.rows(dx, ld_dx); w.rows(df, ld_df); w.rows(dgate, ld_dgate); w.rows(dy, ld_dy); w.rows(dh, ld_dh); w.rows(y, ld_y); w.rows(f, ld_f);
    float *const dw[4] = {dw_pre, db_pre, dw_post, db_post};
    return with_type(d->type, [&](auto *t) {
        typedef B2_ELEM(t) T;
        constexpr int W = 16 / sizeof(T);
        const auto go = [&](auto width) {
            return backward<T, decltype(width)::value>(d, (T *)dx, ld_dx, (T *)df, ld_df, (T *)dgate, ld_dgate, dw, (const T *)dy, ld_dy, (const T *)dh, ld_dh, (const T *)y,
                                                       ld_y, (const T *)f, ld_f, (float *)workspace, (cudaStream_t)stream);
        };
        return w.w == W ? go(std::integral_constant<int, W>()) : go(std::integral_constant<int, 1>());
    });
}

}  // extern "C"
