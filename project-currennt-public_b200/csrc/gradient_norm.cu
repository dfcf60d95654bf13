// The L2 norm over a list of tensors, and the tensors scaled down to a largest norm.
//
//   n = sqrt(sum_i sum_j x_ij^2),   out_ij = x_ij * (n > max ? max / n : 1)
//
// The factor is formed from the norm as it is reported, in fp32: who reads the norm can tell what was done, and repeat it.
// The list travels as a kernel argument: no table in device memory, no copy, nothing kept between calls.  Every tensor is cut
// into chunks of CHUNK bytes that start on 16-byte boundaries; a block takes a contiguous range of all chunks, so it looks up
// its first tensor once.  Squares are summed in fp64: the square of any finite fp32 value is a normal fp64 number, so neither large
// nor tiny gradients need a scale, and the order of the sums (thread, block, launch) is fixed.
// Bound by memory: one read for the norm, one read and one write for the scaled tensors.  The second kernel walks each range
// backwards, so that it starts with what the first one left in L2.  Chunks have the same number of bytes whatever their type, and a tensor's
// ends are taken by vectors too: a block with an end taken element by element held up all others.
// Measured on a B200 (device time): 240 tensors of 260 M elements, fp32 and bf16, 385 us, three passes at 94 % of the copy bandwidth; five
// tensors of 3.7 M fp32 elements 9 us, two launches; resident blocks 3 a multiprocessor (4: 430 us, their loads spill).
#include <math.h>

#include "typed.cuh"

namespace b2 {
namespace {

constexpr int THREADS = 256;
constexpr int CHUNK = 16384;       // bytes
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

// One chunk of a tensor: bytes [at, at + CHUNK), counted from the 16-byte boundary at or below the tensor's start, `mis` bytes before it.
struct Piece {
    const char *src;
    char *dst;
    unsigned long long bytes, at;   // of the tensor; of the chunk
    int mis, src_type, dst_type;
    bool whole;                     // every byte of the chunk is the tensor's
};
template <int CAP> __device__ __forceinline__ Piece piece_of(const List<CAP> &l, int i, unsigned chunk) {
    Piece p;
    p.src_type = l.src_type[i];
    p.dst_type = l.dst_type[i];
    p.src = (const char *)l.src[i];
    p.dst = (char *)l.dst[i];
    p.bytes = l.count[i] << (p.src_type == B2_F32 ? 2 : 1);
    p.at = (unsigned long long)(chunk - l.first[i]) * CHUNK;
    p.mis = (int)((uintptr_t)p.src & 15);
    p.whole = p.at >= (unsigned)p.mis && p.at + CHUNK <= p.mis + p.bytes;
    return p;
}
constexpr int VECTORS = CHUNK / (16 * THREADS);   // of a thread, THREADS vectors apart
__device__ __forceinline__ unsigned long long place(const Piece &p, int i) { return p.at + (unsigned)(i * THREADS + threadIdx.x) * 16u; }
__device__ __forceinline__ bool inside(const Piece &p, unsigned long long at) { return p.whole || (at >= (unsigned)p.mis && at + 16 <= p.mis + p.bytes); }
// A vector that the tensor has only a part of is gathered by 2 bytes, zeros elsewhere; all of them lie at a tensor's two ends.
__device__ __forceinline__ void fetch(uint4 (&q)[VECTORS], const Piece &p) {
    const char *base = p.src - p.mis;
#pragma unroll
    for (int i = 0; i < VECTORS; ++i) {
        const unsigned long long at = place(p, i), end = p.mis + p.bytes;
        if (inside(p, at)) q[i] = *reinterpret_cast<const uint4 *>(base + at);
        else {
            unsigned w[4] = {0, 0, 0, 0};
            if (at < end && at + 16 > (unsigned)p.mis)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (at + 2 * j >= (unsigned)p.mis && at + 2 * j < end) w[j / 2] |= (unsigned)*reinterpret_cast<const unsigned short *>(base + at + 2 * j) << (16 * (j & 1));
            q[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}
template <typename T, int W> __device__ __forceinline__ void values(float (&v)[W], const uint4 &q) {
    const Vec<T, W> x = *reinterpret_cast<const Vec<T, W> *>(&q);
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = to_float(x.v[j]);
}
template <typename T> __device__ __forceinline__ double squares(const uint4 (&q)[VECTORS], double s) {
    constexpr int W = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < VECTORS; ++i) {
        float v[W];
        values<T, W>(v, q[i]);
#pragma unroll
        for (int j = 0; j < W; ++j) { const double x = v[j]; s = fma(x, x, s); }
    }
    return s;
}

// partial[block] (+)= the squares of the block's chunks; the next chunk is on its way while one is added up
template <int CAP> __global__ void __launch_bounds__(THREADS, 3) squares_kernel(const __grid_constant__ List<CAP> l, double *__restrict__ partial, int add) {
    __shared__ double red[THREADS / 32];
    grid_wait();
    grid_release();
    const unsigned total = l.first[l.n];
    const unsigned c0 = (unsigned)((unsigned long long)total * blockIdx.x / gridDim.x), c1 = (unsigned)((unsigned long long)total * (blockIdx.x + 1) / gridDim.x);
    double s = 0.0;
    if (c0 < c1) {
        int i = find_tensor(l, c0);
        Piece now = piece_of(l, i, c0), next = now;
        uint4 q[VECTORS], r[VECTORS];
        fetch(q, now);
        for (unsigned c = c0; c < c1; ++c) {
            if (c + 1 < c1) {
                while (c + 1 >= l.first[i + 1]) ++i;
                next = piece_of(l, i, c + 1);
                fetch(r, next);
            }
            if (now.src_type == B2_F32) s = squares<float>(q, s);
            else if (now.src_type == B2_BF16) s = squares<__nv_bfloat16>(q, s);
            else s = squares<__half>(q, s);
            now = next;
#pragma unroll
            for (int j = 0; j < VECTORS; ++j) q[j] = r[j];
        }
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) partial[blockIdx.x] = add ? partial[blockIdx.x] + s : s;
}

// the norm from the partial sums; every block of a launch adds them in the same order
__device__ __forceinline__ double norm_of(const double *partial, int n, double *red) {
    double s = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += THREADS) s += partial[i];
    return sqrt(block_sum(s, red));
}

// What the values are multiplied by: one factor, or two where one would be subnormal and have lost bits (the second is 1 elsewhere)
struct Factor { float a, b; };
__device__ __forceinline__ Factor factor_of(float max_norm, float norm) {
    const float c = max_norm / norm;
    if (c >= 1.17549435e-38f) return {c, 1.0f};
    const float root = (float)sqrt((double)max_norm / (double)norm);
    return {root, root};
}
// scaled vectors to where they came from
template <typename T, typename U> __device__ __forceinline__ void put(const Piece &p, const uint4 (&q)[VECTORS], const Factor &by) {
    constexpr int W = 16 / sizeof(T);
    // elements are counted from the 16-byte boundary; in the output's type its vectors may lie off theirs
    U *to = reinterpret_cast<U *>(p.dst) - p.mis / (int)sizeof(T);
    const bool fits = ((uintptr_t)to & (sizeof(U) * W < 16 ? sizeof(U) * W - 1 : 15)) == 0;
#pragma unroll
    for (int i = 0; i < VECTORS; ++i) {
        const unsigned long long at = place(p, i), end = p.mis + p.bytes;
        float v[W];
        values<T, W>(v, q[i]);
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = v[j] * by.a * by.b;
        if (fits && inside(p, at)) store_vec<U, W>(to + at / sizeof(T), v);
        else if (at < end && at + 16 > (unsigned)p.mis)
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (at + j * sizeof(T) >= (unsigned)p.mis && at + j * sizeof(T) < end) to[at / sizeof(T) + j] = from_float<U>(v[j]);
    }
}
template <typename T> __device__ __forceinline__ void put(const Piece &p, const uint4 (&q)[VECTORS], const Factor &by) {
    if (p.dst_type == B2_F32) put<T, float>(p, q, by);
    else if (p.dst_type == B2_BF16) put<T, __nv_bfloat16>(p, q, by);
    else put<T, __half>(p, q, by);
}

template <int CAP>
__global__ void __launch_bounds__(THREADS, 3) clip_kernel(const __grid_constant__ List<CAP> l, const double *partial, int n_partial, float max_norm,
                                                          float *__restrict__ norm_out) {
    __shared__ double red[THREADS / 32];
    const unsigned total = l.first[l.n];
    const unsigned c0 = (unsigned)((unsigned long long)total * blockIdx.x / gridDim.x), c1 = (unsigned)((unsigned long long)total * (blockIdx.x + 1) / gridDim.x);
    int i = 0;
    Piece now = {}, next;
    uint4 q[VECTORS], r[VECTORS];
    if (c0 < c1) {
        // The first chunk is read before the wait: this kernel starts when all blocks of the one before have passed theirs, so what they
        // read is complete.  Nothing is written before the wait: they may still be reading.
        i = find_tensor(l, c1 - 1);
        now = piece_of(l, i, c1 - 1);
        fetch(q, now);
    }
    grid_wait();
    const float norm = (float)norm_of(partial, n_partial, red);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    // a norm that is no finite number, one beyond a float among them, says nothing about a scale: the values stay as they are
    const bool scale = norm > max_norm && norm <= 3.402823466e38f;
    const Factor by = scale ? factor_of(max_norm, norm) : Factor{1.0f, 1.0f};
    next = now;
    for (unsigned c = c1; c-- > c0;) {
        if (c > c0) {
            while (c - 1 < l.first[i]) --i;
            next = piece_of(l, i, c - 1);
            if (scale || next.src != next.dst) fetch(r, next);
        }
        if (scale || now.src != now.dst) {
            if (now.src_type == B2_F32) put<float>(now, q, by);
            else if (now.src_type == B2_BF16) put<__nv_bfloat16>(now, q, by);
            else put<__half>(now, q, by);
        }
        now = next;
#pragma unroll
        for (int j = 0; j < VECTORS; ++j) q[j] = r[j];
    }
}

__global__ void __launch_bounds__(THREADS) norm_kernel(const double *partial, int n_partial, float *__restrict__ norm_out) {
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
        const unsigned long long c = (((uintptr_t)s.data & 15) + s.count * type_size(s.type) + CHUNK - 1) / CHUNK;
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
    // blocks that are resident together (3 of 256 threads per multiprocessor), one chunk each at least
    const unsigned most = (unsigned)(sm_count() * 3 < MAX_BLOCKS ? sm_count() * 3 : MAX_BLOCKS);
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
    if (!norm || !aligned_to(norm, 4)) { set_error("%s: null pointer for the norm, or not aligned to 4 bytes", who); return B2_ERR_BAD_ARG; }
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
