// What the two passes of the norms around a residual block (block_norm.cu, block_norm_back.cu) share: a thread's columns, sums over a row's threads,
// rows under way into shared memory, and the checks of arguments.
#pragma once
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

// Sums over the threads of a row: a warp, or all warps of the block (buffers alternate, so one barrier a sum is enough).  red holds 2 * N * 32
// floats; those of warps that are not there are zero.
template <int N> __device__ __forceinline__ void row_sums(float (&x)[N], int warps, float4 (*red)[8], int &phase) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = warp_sum(x[i]);
    if (warps == 1) return;
    float4(*buf)[8] = red + (phase & 1) * N;
    ++phase;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) reinterpret_cast<float *>(buf[i])[threadIdx.x >> 5] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float4 s = buf[i][0];
        for (int k = 1; k < (warps + 3) >> 2; ++k) {
            const float4 y = buf[i][k];
            s.x += y.x; s.y += y.y; s.z += y.z; s.w += y.w;
        }
        x[i] = (s.x + s.y) + (s.z + s.w);
    }
}
__device__ __forceinline__ void clear_sums(float4 *red, int n) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) red[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    __syncthreads();
}

// columns of a thread: vector i starts at column (i * tpr + lane) * W
template <typename T, int W, int NV, bool FULL = false> struct Cols {
    static __device__ __forceinline__ void load(float (&v)[NV][W], const T *row, int tpr, int lane, int dim, float other) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * tpr + lane) * W;
            if (FULL || c < dim) load_vec<T, W>(v[i], row + c);
            else
#pragma unroll
                for (int j = 0; j < W; ++j) v[i][j] = other;
        }
    }
    static __device__ __forceinline__ void store(T *row, const float (&v)[NV][W], int tpr, int lane, int dim) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * tpr + lane) * W;
            if (FULL || c < dim) store_vec<T, W>(row + c, v[i]);
        }
    }
};

// v becomes its normalised self; columns beyond dim are zero before and stay so
template <int W, int NV>
__device__ __forceinline__ void normalise(float (&v)[NV][W], const NormArgs &a, int tpr, int lane, int warps, float4 (*red)[8], int &phase, float &mean, float &rstd) {
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

// v * w + b; w and b (zero beyond the row) as they were loaded, 1 and 0 where there are none
template <int W, int NV> struct Affine {
    float w[NV][W], b[NV][W];
    __device__ __forceinline__ void load(const float *pw, const float *pb, int tpr, int lane, int dim) {
        if (pw) Cols<float, W, NV>::load(w, pw, tpr, lane, dim, 0.0f);
        if (pb) Cols<float, W, NV>::load(b, pb, tpr, lane, dim, 0.0f);
    }
    __device__ __forceinline__ void apply(float (&v)[NV][W], const float *pw, const float *pb) const {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) {
                if (pw) v[i][j] *= w[i][j];
                if (pb) v[i][j] += b[i][j];
            }
    }
    // one after the other: half the registers
    __device__ __forceinline__ void load_and_apply(float (&v)[NV][W], const float *pw, const float *pb, int tpr, int lane, int dim) {
        load(pw, nullptr, tpr, lane, dim);
        apply(v, pw, nullptr);
        load(nullptr, pb, tpr, lane, dim);
        apply(v, nullptr, pb);
    }
};

// Rows on their way into shared memory, `stages` of them, each with up to TENSORS tensors.  A thread copies the vectors that it will read itself,
// or (BYROW, for rows of single elements) all threads of a row copy the 16-byte pieces that hold it, and it is read element by element, so that
// loads and stores stay coalesced; a piece may begin with bytes of what lies before the row, which nobody looks at.  Stages are byte offsets.
template <typename T, int W, int NV, bool FULL, int TENSORS, bool BYROW> struct Ring {
    static constexpr int VB = W * (int)sizeof(T);         // bytes of a vector
    char *base;
    unsigned base_addr;
    int tpr, lane, dim, pitch, mine, stage_bytes, stages;
    // bytes of a stage: TENSORS rows for every row group, then 16 bytes a warp for the caller's use
    static __host__ __device__ int row_bytes(int tpr) { return tpr * NV * (int)sizeof(T) + 32; }
    static __host__ __device__ int tensor_bytes(int threads, int tpr) { return BYROW ? threads / tpr * row_bytes(tpr) : NV * threads * VB; }
    static __host__ __device__ int bytes(int threads, int tpr) { return TENSORS * tensor_bytes(threads, tpr) + threads / 32 * 16; }
    __device__ __forceinline__ Ring(char *ring, int tpr_, int lane_, int dim_, int stages_) {
        base = ring;
        base_addr = (unsigned)__cvta_generic_to_shared(ring);
        tpr = tpr_; lane = lane_; dim = dim_; stages = stages_;
        pitch = tensor_bytes(blockDim.x, tpr);
        stage_bytes = bytes(blockDim.x, tpr);
        mine = BYROW ? (tpr == 32 ? (int)(threadIdx.x >> 5) : 0) * row_bytes(tpr) : (int)threadIdx.x * VB;
    }
    __device__ __forceinline__ int column(int i) const { return (i * tpr + lane) * W; }   // of vector i
    __device__ __forceinline__ int next(int stage) const { return stage + stage_bytes < stages * stage_bytes ? stage + stage_bytes : 0; }
    __device__ __forceinline__ int spare(int stage) const { return stage + TENSORS * pitch + (int)(threadIdx.x >> 5) * 16; }
    __device__ __forceinline__ void copy(int stage, int what, const T *from) const {
        if constexpr (!BYROW) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (FULL || column(i) < dim) cp_async<VB>(base_addr + stage + mine + what * pitch + i * (int)blockDim.x * VB, from + column(i));
        } else {
            const int mis = (int)((uintptr_t)from & 15), bytes = mis + dim * (int)sizeof(T);
            const unsigned to = base_addr + stage + mine + what * pitch;
            for (int at = lane * 16; at < bytes; at += tpr * 16) cp_async(to + at, (const char *)from - mis + at, bytes - at < 16 ? bytes - at : 16);
        }
    }
    // a row as it was copied from `from`; `other` beyond its end
    __device__ __forceinline__ void take(float (&v)[NV][W], int stage, int what, const T *from, float other) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int j = 0; j < W; ++j) v[i][j] = other;
            const char *at = base + stage + mine + what * pitch;
            if constexpr (!BYROW) {
                if (FULL || column(i) < dim) load_vec<T, W>(v[i], reinterpret_cast<const T *>(at + i * (int)blockDim.x * VB));
            } else {
                if (column(i) < dim) load_vec<T, W>(v[i], reinterpret_cast<const T *>(at + (int)((uintptr_t)from & 15)) + column(i));
            }
        }
    }
    // what a thread reads and another copied is there, and nobody is still reading what is copied over next
    __device__ __forceinline__ void barrier() const {
        if (BYROW && tpr > 32) __syncthreads();
        else __syncwarp();
    }
};

// ---- host -----------------------------------------------------------------------------------------------------------------------------
// elements of an access that every row of every tensor starts and ends on: 16 bytes of them, else 2 of a 16-bit type, else 1
struct Width {
    int w, elem;
    void fit(bool wide, bool two) {
        if (w * elem == 16 && !wide) w = elem == 2 ? 2 : 1;
        if (w == 2 && elem == 2 && !two) w = 1;
    }
    void rows(const void *p, long long ld) {
        if (p) fit(ld % (16 / elem) == 0 && aligned_to(p, 16), ld % 2 == 0 && aligned_to(p, 4));
    }
    void floats(const float *p) { fit(aligned_to(p, 16), aligned_to(p, 8)); }
};
Width width_of(const b2_block_norm *d) {
    Width x = {16 / type_size(d->type), type_size(d->type)};
    x.fit(d->dim % x.w == 0, d->dim % 2 == 0);
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
        if (d->ld_gate < d->dim || d->ld_gate > 0x7fffffffll) {
            set_error("%s: leading dimension of the gate too small or beyond 2^31 (%lld for %d columns)", who, d->ld_gate, d->dim);
            return B2_ERR_BAD_ARG;
        }
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
    if (ld < d->dim || ld > 0x7fffffffll) {
        set_error("%s: leading dimension of %s too small or beyond 2^31 (%lld for %d columns)", who, name, ld, d->dim);
        return B2_ERR_BAD_ARG;
    }
    if (!aligned_to(p, type_size(d->type))) { set_error("%s: %s is not aligned to its elements", who, name); return B2_ERR_BAD_ARG; }
    return B2_OK;
}
NormArgs args_of(const b2_block_norm *d) {
    return {d->pat_types, d->w_pre, d->b_pre, d->w_post, d->b_post, d->gate, (float4 *)d->stats, d->rows, d->gate ? d->gate_rows : 1, d->ld_gate, d->dim,
            d->layer_norm ? 1 : 0, d->eps, d->residual_scale, 1.0f / (float)d->dim};
}

}  // namespace
}  // namespace b2
