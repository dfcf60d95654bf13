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
// Bound by memory: a row stays in registers and shared memory between its loads and its stores, so every tensor is read once and written
// once.  What stands against it is latency: a row is a chain of two sums over its threads (four with layer norm), so the rows that follow are on
// their way into shared memory meanwhile, as many as fit (see the forward kernel); and instructions, so arithmetic is packed in the backward
// pass, the threads of a row are a constant, and full rows are compiled without tests.  The backward kernel has a fixed number of workers; a worker
// keeps the same columns for all its rows, so the sums over frames stay in registers until the end, go to the workspace once, and are added there in a
// fixed order by a second launch: no atomics, the same bits every time.
// Measured on a B200 (device time of a pass among passes over the same buffers, a third of the frames padding in the forward pass; share of the copy
// bandwidth; with buffers that change 1 to 10 % more, and cards differ by 4 %): forward, layer norm, 38400 x 512 fp32 with a gate per sequence 52 us
// (all bytes counted 92 %, of padding only zeros are written), 38400 x 512 bf16 33 us, x 1024 64 us, 8192 x 4001 without a gate 93 us (43 %; single
// elements), 64 x 1024 bf16 3.5 us.  Backward, 16384 x 2048 bf16 with a gate per frame 95 us (86 %), with layer norm and biases 137 us (60 %), 16384 x 2047
// 179 us, x 4096 250 us (one block a multiprocessor: its barriers are not hidden).
// Rows that no 16-byte access fits reach 17 to 58 %: they come into shared memory in 16-byte pieces (16-bit types), but every element is read from there and
// stored by an access of its own.
#include "block_norm.cuh"

namespace b2 {
namespace {

// Few rows: a row a warp (tpr = 32) or block, a vector a thread; nothing is loaded after anything has been waited for, so that a row costs one trip to
// memory (padding frames are loaded in vain).
template <typename T, int W>
__global__ void __launch_bounds__(512) block_norm_few_kernel(const NormArgs a, const T *x, long long ld_x, const T *f, long long ld_f, T *y, long long ld_y, T *h, long long ld_h,
                                                             int tpr) {
    __shared__ float4 red[2][8];
    const int warps = tpr >> 5, lane = warps == 1 ? (threadIdx.x & 31) : threadIdx.x;
    const long long r = warps == 1 ? (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    if (r >= a.rows) return;
    int phase = 0;
    typedef Cols<T, W, 1> C;
    float v[1][W], n[1][W], g[1][W];
    Affine<W, 1> post, pre;
    const char pat = a.pat ? a.pat[r] : 1;
    C::load(v, x + r * ld_x, tpr, lane, a.dim, 0.0f);
    if (f) {
        C::load(n, f + r * ld_f, tpr, lane, a.dim, 0.0f);
        if (a.gate) C::load(g, (const T *)a.gate + (r % a.gate_rows) * a.ld_gate, tpr, lane, a.dim, 0.0f);
        post.load(a.w2, a.b2, tpr, lane, a.dim);
    }
    if (h) pre.load(a.w1, a.b1, tpr, lane, a.dim);
    if (warps > 1) clear_sums(red[0], 16);
    float4 st = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (pat == PAT_NONE) {
#pragma unroll
        for (int j = 0; j < W; ++j) v[0][j] = 0.0f;
        if (y) C::store(y + r * ld_y, v, tpr, lane, a.dim);
        if (h) C::store(h + r * ld_h, v, tpr, lane, a.dim);
        if (a.stats && lane == 0) a.stats[r] = st;
        return;
    }
    if (f) {
        normalise<W, 1>(n, a, tpr, lane, warps, red, phase, st.x, st.y);
        post.apply(n, a.w2, a.b2);
#pragma unroll
        for (int j = 0; j < W; ++j) v[0][j] = to_float(from_float<T>(fmaf(a.gate ? a.a * g[0][j] : a.a, n[0][j], v[0][j])));
    }
    if (y) C::store(y + r * ld_y, v, tpr, lane, a.dim);
    if (h) {
        normalise<W, 1>(v, a, tpr, lane, warps, red, phase, st.z, st.w);
        pre.apply(v, a.w1, a.b1);
        C::store(h + r * ld_h, v, tpr, lane, a.dim);
    }
    if (a.stats && lane == 0) a.stats[r] = st;
}

// Many rows: workers (a warp, or a block of tpr threads) take rows one after another; the next `stages` - 1 rows are on their way while one is worked
// on, since a row is a chain of two to four sums over its threads that would leave the memory idle.  What the blocks of a multiprocessor may have of its
// shared memory gives 2 to 4 stages, but one only for fp32 rows of 129 to 4096 columns in 16-byte vectors and of 257 to 4096 single elements: there
// nothing is ahead, and the other workers' rows cover for it (38400 x 512 fp32: 92 % of the copy bandwidth).  FULL: x, f, y, h are all there and the
// threads' columns are just the row's.
__host__ __device__ constexpr int forward_threads(int per_thread) { return per_thread > 16 ? 512 : 768; }   // a multiprocessor's, by their registers
// TPR, the threads of a row (32: a warp, 8 rows a block), is a constant, which makes the offsets of a row's columns constants too: with single
// elements (W = 1) most instructions were address arithmetic (38400 x 511: 115 us, now 61 us).
template <typename T, int W, int NV, int TPR, bool FULL>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, forward_threads(NV * W) / (TPR == 32 ? 256 : TPR) > 0 ? forward_threads(NV * W) / (TPR == 32 ? 256 : TPR) : 1)
    block_norm_forward_kernel(const NormArgs a, const T *x, long long ld_x, const T *f, long long ld_f, T *y, long long ld_y, T *h, long long ld_h, int stages) {
    __shared__ float4 red[2][8];
    extern __shared__ __align__(16) char ring_memory[];
    constexpr int tpr = TPR, warps = TPR / 32;
    const int lane = warps == 1 ? (threadIdx.x & 31) : threadIdx.x;
    const unsigned worker = warps == 1 ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x, workers = warps == 1 ? gridDim.x * (blockDim.x >> 5) : gridDim.x;
    const unsigned rows = (unsigned)a.rows, G = (unsigned)a.gate_rows;
    const Ring<T, W, NV, FULL, 3, W == 1> ring(ring_memory, tpr, lane, a.dim, stages);
    typedef Cols<T, W, NV, FULL> C;
    clear_sums(red[0], 16);
    int phase = 0;
    const bool has_f = FULL || f, has_y = FULL || y, has_h = FULL || h;
    unsigned ahead = worker, on_bits = 0, on_at = 0, on_to = 0;   // which of the rows under way are no padding: bits come in at on_to, go out at on_at
    char pat_ahead = ahead < rows && a.pat ? __ldg(a.pat + ahead) : 1;
    const auto advance = [&](int stage) {
        const bool on = ahead < rows && pat_ahead != PAT_NONE;
        on_bits = (on_bits & ~(1u << on_to)) | ((unsigned)on << on_to);
        on_to = (on_to + 1) & 31;
        if (on) {
            ring.copy(stage, 0, x + ahead * ld_x);
            if (has_f) ring.copy(stage, 1, f + ahead * ld_f);
            if (has_f && a.gate) ring.copy(stage, 2, (const T *)a.gate + (ahead % G) * a.ld_gate);
        }
        cp_commit();
        ahead = rows - ahead > workers && ahead < rows ? ahead + workers : rows;
        if (a.pat && ahead < rows) pat_ahead = __ldg(a.pat + ahead);   // looked at when the next copies start
    };
    int at = 0, to = 0;
    for (int s = 0; s + 1 < stages; ++s) { advance(to); to = ring.next(to); }
    for (unsigned r = worker; r < rows; at = ring.next(at), to = ring.next(to)) {
        if (stages > 1) {
            cp_wait(stages - 2);
            ring.barrier();
            advance(to);
        } else {
            ring.barrier();
            advance(0);
            cp_wait(0);
            ring.barrier();
        }
        const bool on = on_bits >> on_at & 1;
        on_at = (on_at + 1) & 31;
        float v[NV][W];
        float4 st = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (!on) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < W; ++j) v[i][j] = 0.0f;
            if (has_y) C::store(y + r * ld_y, v, tpr, lane, a.dim);
            if (has_h) C::store(h + r * ld_h, v, tpr, lane, a.dim);
        } else {
            Affine<W, NV> w;
            if (has_f) {
                const T *gate = (const T *)a.gate + (r % G) * a.ld_gate;
                float n[NV][W];
                ring.take(n, at, 1, f + r * ld_f, 0.0f);
                normalise<W, NV>(n, a, tpr, lane, warps, red, phase, st.x, st.y);
                w.load_and_apply(n, a.w2, a.b2, tpr, lane, a.dim);
                if (a.gate) {
                    ring.take(v, at, 2, gate, 0.0f);
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int j = 0; j < W; ++j) n[i][j] *= a.a * v[i][j];
                } else
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int j = 0; j < W; ++j) n[i][j] *= a.a;
                ring.take(v, at, 0, x + r * ld_x, 0.0f);
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < W; ++j) v[i][j] = to_float(from_float<T>(v[i][j] + n[i][j]));
            } else ring.take(v, at, 0, x + r * ld_x, 0.0f);
            if (has_y) C::store(y + r * ld_y, v, tpr, lane, a.dim);
            if (has_h) {
                normalise<W, NV>(v, a, tpr, lane, warps, red, phase, st.z, st.w);
                w.load_and_apply(v, a.w1, a.b1, tpr, lane, a.dim);
                C::store(h + r * ld_h, v, tpr, lane, a.dim);
            }
        }
        if (a.stats && lane == 0) a.stats[r] = st;
        r = rows - r > workers ? r + workers : rows;
    }
    cp_wait(0);
}

template <typename T, int W>
int forward(const b2_block_norm *d, const T *x, long long ld_x, const T *f, long long ld_f, T *y, long long ld_y, T *h, long long ld_h, cudaStream_t st) {
    const NormArgs a = args_of(d);
    const int vecs = (d->dim + W - 1) / W;
    // few rows (64 x 1024 bf16: 3.5 us, with the kernel for many rows 4.3 us)
    if ((double)d->rows * vecs <= 512.0 * sm_count() && vecs <= 512) {
        const int t = (int)pow2_at_least((unsigned)vecs), tpr = t < 32 ? 32 : t;
        block_norm_few_kernel<T, W><<<tpr == 32 ? (unsigned)((d->rows + 7) / 8) : (unsigned)d->rows, tpr == 32 ? 256 : tpr, 0, st>>>(a, x, ld_x, f, ld_f, y, ld_y, h, ld_h, tpr);
        count_launch();
        B2_CUDA(cudaGetLastError());
        return B2_OK;
    }
    const auto go = [&](auto kernel, auto vectors, int tpr) -> int {
        constexpr int NV = decltype(vectors)::value;
        const int threads = tpr == 32 ? 256 : tpr, each = threads / tpr, most = 208 * 1024, per_sm = forward_threads(NV * W) / threads > 0 ? forward_threads(NV * W) / threads : 1;
        const int stage_bytes = Ring<T, W, NV, false, 3, W == 1>::bytes(threads, tpr);
        int stages = most / per_sm / stage_bytes;
        stages = stages > 4 ? 4 : stages < 1 ? 1 : stages;
        long long blocks = (long long)sm_count() * per_sm;
        if (blocks * each > d->rows) blocks = (d->rows + each - 1) / each;
        B2_TRY(set_max_dynamic_smem((const void *)kernel, most));
        kernel<<<(unsigned)blocks, threads, stages * stage_bytes, st>>>(a, x, ld_x, f, ld_f, y, ld_y, h, ld_h, stages);
        count_launch();
        B2_CUDA(cudaGetLastError());
        return B2_OK;
    };
    // 16 columns a thread, 32 in 16-byte vectors of 16-bit types up to 1024 columns: few threads a row, a warp up to 512, make the sums short
    const auto pick = [&](auto vectors, int tpr) -> int {
        constexpr int NV = decltype(vectors)::value;
        const auto sized = [&](auto threads) -> int {
            constexpr int TPR = decltype(threads)::value;
            if constexpr (W * sizeof(T) == 16)
                if (f && y && h && d->dim == NV * W * TPR) return go(block_norm_forward_kernel<T, W, NV, TPR, true>, vectors, TPR);
            return go(block_norm_forward_kernel<T, W, NV, TPR, false>, vectors, TPR);
        };
        if constexpr (NV == 16 / W) {
            if (tpr == 512) return sized(std::integral_constant<int, 512>());
            if (tpr == 256) return sized(std::integral_constant<int, 256>());
            if (tpr == 128) return sized(std::integral_constant<int, 128>());
            if (tpr == 64) return sized(std::integral_constant<int, 64>());
        }
        return sized(std::integral_constant<int, 32>());
    };
    const auto threads_for = [&](int nv) { const int t = (int)pow2_at_least((unsigned)(vecs + nv - 1) / nv); return t < 32 ? 32 : t; };
    if constexpr (W == 8)
        if (vecs > 64 && vecs <= 128) return pick(std::integral_constant<int, 4>(), 32);
    if constexpr (W * sizeof(T) == 16)
        if (vecs <= 32) return pick(std::integral_constant<int, 1>(), 32);
    constexpr int NV = 16 / W;
    if constexpr (W * sizeof(T) != 16) {
        // a lane has no more columns than the row asks for: up to 128, 4 (38400 x 101 bf16: 28.3 us, with 8 35.0, with 16 51.9);
        // up to 256, 8 (38400 x 201 bf16: 35.2 us, with 16 50.7)
        if (d->dim <= 128) return pick(std::integral_constant<int, 4 / W>(), 32);
        if (d->dim <= 256) return pick(std::integral_constant<int, 8 / W>(), 32);
    }
    return pick(std::integral_constant<int, NV>(), threads_for(NV));
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" int b2_block_norm_forward(const b2_block_norm *d, const void *x, long long ld_x, const void *f, long long ld_f, void *y, long long ld_y, void *h, long long ld_h,
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
        if constexpr (W == 8)
            if (w.w == 2) return forward<T, 2>(d, (const T *)x, ld_x, (const T *)f, ld_f, (T *)y, ld_y, (T *)h, ld_h, (cudaStream_t)stream);
        return forward<T, 1>(d, (const T *)x, ld_x, (const T *)f, ld_f, (T *)y, ld_y, (T *)h, ld_h, (cudaStream_t)stream);
    });
}
