// The L2 norm over a list of tensors, and the tensors scaled down to a largest norm.
//
//   n = sqrt(sum_i sum_j x_ij^2),   out_ij = x_ij * (n > max ? max / n : 1)
//
// The list travels as a kernel argument: no table in device memory, no copy, nothing kept between calls.  Every tensor is cut
// into chunks of CHUNK elements that start on 16-byte boundaries; a block takes a contiguous range of all chunks, so it looks up
// its first tensor once.  Squares are summed in fp64: the square of any finite fp32 value is a normal fp64 number, so neither large
// nor tiny gradients need a scale, and the order of the sums (thread, block, launch) is fixed.
// Bound by memory: one read for the norm, one read and one write for the scaled tensors.  The second kernel walks each range
// backwards, so that it starts with what the first one left in L2.
#include <math.h>

#include "typed.cuh"

namespace b2 {
namespace {

constexpr int THREADS = 256;
constexpr int CHUNK = 4096;
constexpr int MAX_BLOCKS = 2048;   // partial sums in the workspace

template <int CAP> struct List {
    const void *src[CAP];
    void *dst[CAP];
    unsigned long long count[CAP];
    unsigned first[CAP + 1];       // chunks before tensor i
    unsigned char src_type[CAP], dst_type[CAP];
    int n;
};

// the tensor that chunk c belongs to
template <int CAP> __device__ __forceinline__ int find_tensor(const List<CAP> &l, unsigned c) {
    int a = 0, b = l.n - 1;
    while (a < b) {
        const int m = (a + b + 1) >> 1;
        if (l.first[m] <= c) a = m; else b = m - 1;
    }
    return a;
}

__device__ __forceinline__ double block_sum(double x, double *red) {
    x = warp_sum(x);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) s += red[i];
    __syncthreads();
    return s;
}

// sum of squares of one chunk; positions are counted from the 16-byte boundary at or below the tensor's start
template <typename T> __device__ __forceinline__ double chunk_squares(const T *p, unsigned long long count, unsigned chunk) {
    constexpr int W = 16 / sizeof(T);
    const int mis = (int)(((uintptr_t)p & 15) / sizeof(T));
    const T *base = p - mis;
    const unsigned long long lo = mis, hi = mis + count, at = (unsigned long long)chunk * CHUNK;
    double s = 0.0;
    if (at >= lo && at + CHUNK <= hi) {
        constexpr int N = CHUNK / (THREADS * W);
        float v[N][W];
#pragma unroll
        for (int i = 0; i < N; ++i) load_vec<T, W>(v[i], base + at + (size_t)(i * THREADS + threadIdx.x) * W);
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) { const double x = v[i][j]; s = fma(x, x, s); }
    } else {
        const unsigned long long end = at + CHUNK < hi ? at + CHUNK : hi;
        for (unsigned long long e = (at > lo ? at : lo) + threadIdx.x; e < end; e += THREADS) {
            const double x = to_float(base[e]);
            s = fma(x, x, s);
        }
    }
    return s;
}

// partial[block] (+)= the squares of the block's chunks
template <int CAP> __global__ void __launch_bounds__(THREADS) squares_kernel(const __grid_constant__ List<CAP> l, double *__restrict__ partial, int add) {
    __shared__ double red[THREADS / 32];
    grid_wait();
    grid_release();
    const unsigned total = l.first[l.n];
    const unsigned c0 = (unsigned)((unsigned long long)total * blockIdx.x / gridDim.x), c1 = (unsigned)((unsigned long long)total * (blockIdx.x + 1) / gridDim.x);
    double s = 0.0;
    if (c0 < c1) {
        int i = find_tensor(l, c0);
        for (unsigned c = c0; c < c1; ++c) {
            while (c >= l.first[i + 1]) ++i;
            const unsigned k = c - l.first[i];
            if (l.src_type[i] == B2_F32) s += chunk_squares((const float *)l.src[i], l.count[i], k);
            else if (l.src_type[i] == B2_BF16) s += chunk_squares((const __nv_bfloat16 *)l.src[i], l.count[i], k);
            else s += chunk_squares((const __half *)l.src[i], l.count[i], k);
        }
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) partial[blockIdx.x] = add ? partial[blockIdx.x] + s : s;
}

// the norm from the partial sums; every block of a launch adds them in the same order
__device__ __forceinline__ double norm_of(const double *partial, int n, double *red) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += THREADS) s += partial[i];
    return sqrt(block_sum(s, red));
}

template <typename T, typename U>
__device__ __forceinline__ void scale_chunk(U *q, const T *p, unsigned long long count, unsigned chunk, float coef) {
    constexpr int W = 16 / sizeof(T);
    const int mis = (int)(((uintptr_t)p & 15) / sizeof(T));
    const T *base = p - mis;
    U *to = q - mis;
    const unsigned long long lo = mis, hi = mis + count, at = (unsigned long long)chunk * CHUNK;
    // the output's vectors: W elements of its own type, 16 bytes at most an access
    const bool fits = ((uintptr_t)to & (sizeof(U) * W < 16 ? sizeof(U) * W - 1 : 15)) == 0;
    if (at >= lo && at + CHUNK <= hi && fits) {
        constexpr int N = CHUNK / (THREADS * W);
        float v[N][W];
#pragma unroll
        for (int i = 0; i < N; ++i) load_vec<T, W>(v[i], base + at + (size_t)(i * THREADS + threadIdx.x) * W);
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int j = 0; j < W; ++j) v[i][j] *= coef;
            store_vec<U, W>(to + at + (size_t)(i * THREADS + threadIdx.x) * W, v[i]);
        }
    } else {
        const unsigned long long end = at + CHUNK < hi ? at + CHUNK : hi;
        for (unsigned long long e = (at > lo ? at : lo) + threadIdx.x; e < end; e += THREADS) to[e] = from_float<U>(to_float(base[e]) * coef);
    }
}
template <typename T> __device__ __forceinline__ void scale_chunk_to(void *q, int type, const T *p, unsigned long long count, unsigned chunk, float coef) {
    if (type == B2_F32) scale_chunk((float *)q, p, count, chunk, coef);
    else if (type == B2_BF16) scale_chunk((__nv_bfloat16 *)q, p, count, chunk, coef);
    else scale_chunk((__half *)q, p, count, chunk, coef);
}

template <int CAP>
__global__ void __launch_bounds__(THREADS) clip_kernel(const __grid_constant__ List<CAP> l, const double *__restrict__ partial, int n_partial, float max_norm,
                                                       float *__restrict__ norm_out) {
    __shared__ double red[THREADS / 32];
    grid_wait();
    const double norm = norm_of(partial, n_partial, red);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    // a norm that is no finite number says nothing about a scale: the values stay as they are
    const bool scale = norm > (double)max_norm && norm <= 1.7976931348623157e308;
    const float coef = scale ? (float)((double)max_norm / norm) : 1.0f;
    const unsigned total = l.first[l.n];
    const unsigned c0 = (unsigned)((unsigned long long)total * blockIdx.x / gridDim.x), c1 = (unsigned)((unsigned long long)total * (blockIdx.x + 1) / gridDim.x);
    if (c0 >= c1) return;
    int i = find_tensor(l, c1 - 1);
    for (unsigned c = c1; c-- > c0;) {
        while (c < l.first[i]) --i;
        if (!scale && l.src[i] == l.dst[i]) continue;
        const unsigned k = c - l.first[i];
        if (l.src_type[i] == B2_F32) scale_chunk_to(l.dst[i], l.dst_type[i], (const float *)l.src[i], l.count[i], k, coef);
        else if (l.src_type[i] == B2_BF16) scale_chunk_to(l.dst[i], l.dst_type[i], (const __nv_bfloat16 *)l.src[i], l.count[i], k, coef);
        else scale_chunk_to(l.dst[i], l.dst_type[i], (const __half *)l.src[i], l.count[i], k, coef);
    }
}

__global__ void __launch_bounds__(THREADS) norm_kernel(const double *__restrict__ partial, int n_partial, float *__restrict__ norm_out) {
    __shared__ double red[THREADS / 32];
    grid_wait();
    const double norm = norm_of(partial, n_partial, red);
    if (threadIdx.x == 0) *norm_out = (float)norm;
}

int check_list(const char *who, const b2_tensor *t, int n) {
    if (n < 0 || (n > 0 && !t)) { set_error("%s: a list of %d tensors without its address", who, n); return B2_ERR_BAD_ARG; }
    for (int i = 0; i < n; ++i) {
        const int sz = type_size(t[i].type);
        if (!sz) { set_error("%s: tensor %d has the unknown element type %d", who, i, t[i].type); return B2_ERR_BAD_ARG; }
        if (t[i].count && !t[i].data) { set_error("%s: tensor %d is a null pointer", who, i); return B2_ERR_BAD_ARG; }
        if (!aligned_to(t[i].data, sz)) { set_error("%s: tensor %d is not aligned to its elements", who, i); return B2_ERR_BAD_ARG; }
        if (t[i].count > ((size_t)1 << 42)) { set_error("%s: tensor %d has %zu elements", who, i, t[i].count); return B2_ERR_BAD_SHAPE; }
    }
    return B2_OK;
}

// fills l with tensors from *at on, as many as fit; false when nothing is left
template <int CAP> bool fill(List<CAP> &l, const b2_tensor *src, const b2_tensor *dst, int n, int *at) {
    int k = 0;
    unsigned long long chunks = 0;
    l.first[0] = 0;
    for (; *at < n && k < CAP; ++*at) {
        const b2_tensor &s = src[*at], &d = dst[*at];
        if (!s.count) continue;
        const size_t mis = ((uintptr_t)s.data & 15) / type_size(s.type);
        const unsigned long long c = (mis + s.count + CHUNK - 1) / CHUNK;
        if (k && chunks + c > 0xfffffffeull) break;
        chunks += c;
        l.src[k] = s.data;
        l.dst[k] = d.data;
        l.count[k] = s.count;
        l.src_type[k] = (unsigned char)s.type;
        l.dst_type[k] = (unsigned char)d.type;
        l.first[++k] = (unsigned)chunks;
    }
    l.n = k;
    return k > 0;
}

int grid_of(unsigned chunks) {
    // blocks that are resident together (8 of 256 threads per multiprocessor), one chunk each at least
    const unsigned most = (unsigned)(sm_count() * 8 < MAX_BLOCKS ? sm_count() * 8 : MAX_BLOCKS);
    return (int)(chunks < most ? chunks : most);
}

template <int CAP>
int run(const b2_tensor *src, const b2_tensor *dst, int n, bool clip, float max_norm, float *norm, double *partial, cudaStream_t st) {
    List<CAP> l;
    int blocks = 0, at = 0;
    // the first launch has the largest grid there can be when a second one follows, so that every later one only adds
    for (bool first = true; fill(l, src, dst, n, &at); first = false) {
        int grid = grid_of(l.first[l.n]);
        if (first) blocks = at < n ? grid_of(0xffffffffu) : grid;
        if (grid > blocks) grid = blocks;
        B2_TRY(launch_chained(squares_kernel<CAP>, dim3(first ? blocks : grid), dim3(THREADS), 0, st, l, partial, first ? 0 : 1));
    }
    if (!clip || !blocks) return launch_chained(norm_kernel, dim3(1), dim3(THREADS), 0, st, (const double *)partial, blocks, norm);
    at = 0;
    for (bool first = true; fill(l, src, dst, n, &at); first = false)
        B2_TRY(launch_chained(clip_kernel<CAP>, dim3(grid_of(l.first[l.n])), dim3(THREADS), 0, st, l, (const double *)partial, blocks, max_norm,
                              first ? norm : (float *)nullptr));
    return B2_OK;
}

int dispatch(const char *who, const b2_tensor *src, const b2_tensor *dst, int n, bool clip, float max_norm, float *norm, void *ws, size_t ws_bytes,
             cudaStream_t st) {
    if (!norm) { set_error("%s: null pointer for the norm", who); return B2_ERR_BAD_ARG; }
    if (!ws || !aligned_to(ws, 8)) { set_error("%s: the workspace is missing or not aligned to 8 bytes", who); return B2_ERR_BAD_ARG; }
    if (ws_bytes < b2_gradient_norm_workspace()) {
        set_error("%s: %zu bytes of workspace, %zu are needed", who, ws_bytes, b2_gradient_norm_workspace());
        return B2_ERR_BAD_SHAPE;
    }
    if (current_device() < 0) { set_error("%s: no current CUDA device", who); return B2_ERR_CUDA; }
    // short lists as a short argument: a launch copies all of it
    if (n <= 32) return run<32>(src, dst, n, clip, max_norm, norm, (double *)ws, st);
    return run<512>(src, dst, n, clip, max_norm, norm, (double *)ws, st);
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

size_t b2_gradient_norm_workspace(void) { return (size_t)MAX_BLOCKS * sizeof(double); }

int b2_gradient_norm(const b2_tensor *tensors, int n, float *norm_dev, void *workspace, size_t workspace_bytes, b2_stream stream) {
    B2_TRY(check_list("b2_gradient_norm", tensors, n));
    return dispatch("b2_gradient_norm", tensors, tensors, n, false, 0.0f, norm_dev, workspace, workspace_bytes, (cudaStream_t)stream);
}

int b2_gradient_clip(const b2_tensor *tensors, const b2_tensor *out, int n, float max_norm, float *norm_dev, void *workspace, size_t workspace_bytes,
                     b2_stream stream) {
    B2_TRY(check_list("b2_gradient_clip", tensors, n));
    if (out) {
        B2_TRY(check_list("b2_gradient_clip (outputs)", out, n));
        for (int i = 0; i < n; ++i)
            if (out[i].count != tensors[i].count) {
                set_error("b2_gradient_clip: tensor %d has %zu elements, its output %zu", i, tensors[i].count, out[i].count);
                return B2_ERR_BAD_SHAPE;
            } else if (out[i].count && out[i].data == tensors[i].data && out[i].type != tensors[i].type) {
                set_error("b2_gradient_clip: tensor %d is scaled in place to another element type", i);
                return B2_ERR_BAD_ARG;
            }
    }
    if (!(max_norm >= 0.0f)) { set_error("b2_gradient_clip: the largest norm is %g", (double)max_norm); return B2_ERR_BAD_ARG; }
    return dispatch("b2_gradient_clip", tensors, out ? out : tensors, n, true, max_norm, norm_dev, workspace, workspace_bytes, (cudaStream_t)stream);
}

}  // extern "C"
