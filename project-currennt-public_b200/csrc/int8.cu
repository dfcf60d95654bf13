// Products in 8-bit integers with a scale for each row of the activations and each channel of the weights, and the quantisation of rows.
//
//   quantise:  s_r = max_k |x_rk| / 127,  q_rk = rint(x_rk * (127 / max |x_r|))         one FMA with 1.5 * 2^23: the product is rounded once, to an integer
//   product:   out_rc = s_r * s_c * sum_k q_rk w_ck + bias_c                             exact 32-bit sums, then fma(sum, s_r * s_c, bias)
//
// The product runs on the tensor cores (tcgen05.mma kind::i8): channels are the rows of a tile (128 tensor-memory lanes), activations its columns, so that a warp
// of the epilogue, which has 32 lanes of one column, stores 32 neighbouring channels of one row of out, whatever its alignment.  The number of columns follows
// the rows of x: few rows stream the weights once through a deep ring, many rows reuse them.
// Measured on a B200 (device time; in brackets a pass over buffers that change): 50001 rows of 1024 fp32 quantised 38 us (40.9; 98 % of the copy rate); 8 bf16 rows x 50001 x 1024 11.7 us
// (14.3; the weights' floor is 8.2, 4 us are a launch, the block's set-up and its last tile); 8192 x 50001 x 1024 to bf16 379 us in a burst, 2.2 POP/s (436 at the clock
// under the power cap; twice the bf16 rate: 296), 8192 x 8192 x 4096 3.2 POP/s: short contractions are bound by the data path of the shared memory, see int8_pair_kernel.
#include <cuda.h>
#include <math.h>

#include <mutex>
#include <type_traits>

#include "ptx.cuh"
#include "typed.cuh"

namespace b2 {
namespace {

// ---- quantisation ---------------------------------------------------------------------------------------------------------------------
constexpr float TINY_ROW = 3.00926553810506e-36f;       // 2^-118: 127 over less leaves the floats

template <typename T> __device__ __forceinline__ float largest_magnitude(const uint4 &q) {
    float m = 0.0f;
    if constexpr (sizeof(T) == 4) {
        const unsigned w[4] = {q.x, q.y, q.z, q.w};
        unsigned b = 0;      // magnitudes of floats are in the order of their bits, NaN above all
#pragma unroll
        for (int i = 0; i < 4; ++i) b = max(b, w[i] & 0x7fffffffu);
        m = __uint_as_float(b);
    } else {
        const unsigned w[4] = {q.x, q.y, q.z, q.w};
        unsigned b = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) b = __vmaxu2(b, w[i] & 0x7fff7fffu);
        const unsigned short h = (unsigned short)max(b & 0xffffu, b >> 16);
        T v;
        memcpy(&v, &h, 2);
        m = to_float(v);
    }
    return m;
}
__device__ __forceinline__ float larger_magnitude(float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); }
// A row's scale and the factor of its values, from its largest magnitude
struct RowScale {
    float scale, inv;
    bool finite;
    __device__ __forceinline__ explicit RowScale(float most) {
        finite = most < __int_as_float(0x7f800000);
        const bool some = finite && most > TINY_ROW;
        inv = some ? __fdiv_rn(127.0f, most) : 0.0f;
        scale = !finite ? nanf("") : some ? __fdiv_rn(most, 127.0f) : 0.0f;
    }
    __device__ __forceinline__ unsigned char quantised(float x) const { return finite ? (unsigned char)__float_as_uint(fmaf(x, inv, 12582912.0f)) : 0; }
    template <typename T> __device__ __forceinline__ Vec<unsigned char, 16 / sizeof(T)> quantised(const uint4 &h) const {
        constexpr int W = 16 / sizeof(T);
        T e[W];
        memcpy(e, &h, 16);
        Vec<unsigned char, W> o;
#pragma unroll
        for (int j = 0; j < W; ++j) o.v[j] = quantised(to_float(e[j]));
        return o;
    }
};

// TEAM threads a row; up to U vectors of each in registers (KEPT), or the row is read twice.  WHOLE: rows of whole vectors that start on their boundaries, the integers' too.
// Else a vector's integers lie across the boundaries of what they are stored to: a lane takes the first bytes of a store from the lane before it, shifted by what
// the row's two starts differ (5000 x 8191 bf16: 43 us, with single bytes 60 us; narrow rows gain nothing, their ends cost most: 60000 x 401 41 us).
template <typename T, int TEAM, int U, bool KEPT, bool WHOLE>
__global__ void __launch_bounds__(256) int8_quantize_kernel(signed char *q, long long ld_q, float *scales, const T *x0, long long rows, int dim, long long ld_x) {
    constexpr int W = 16 / sizeof(T), TEAMS = 256 / TEAM;
    typedef std::conditional_t<W == 8, unsigned long long, unsigned> Word;         // W integers
    __shared__ float most[8];
    const int team = threadIdx.x / TEAM, at = threadIdx.x % TEAM, lane = threadIdx.x & 31;
    const long long r = (long long)blockIdx.x * TEAMS + team;
    grid_release();
    if (r >= rows) return;
    const T *x = x0 + r * ld_x;
    unsigned char *to = reinterpret_cast<unsigned char *>(q) + r * ld_q;
    // vectors hold the entries v * W - mis on; one more than there are takes the last bytes
    const int mis = WHOLE ? 0 : (int)(((uintptr_t)x & 15) / sizeof(T)), vecs = WHOLE ? dim / W : (mis + dim + W - 1) / W + 1;
    const int shift = WHOLE ? 0 : (mis - (int)((uintptr_t)to & (W - 1))) & (W - 1);      // bytes of the vector before that go to where the one behind it begins
    const auto load = [&](int v) -> uint4 {
        const int i0 = v * W - mis;
        if constexpr (WHOLE) return *reinterpret_cast<const uint4 *>(x + i0);
        else {
            if (i0 >= 0 && i0 + W <= dim) return *reinterpret_cast<const uint4 *>(x + i0);
            // the row's ends; entry by entry, in a loop: a launch fetches the code of every vector anew
            unsigned w[4] = {0, 0, 0, 0};
#pragma unroll 1
            for (int i = max(0, i0); i < min(dim, i0 + W); ++i) {
                unsigned bits = 0;
                memcpy(&bits, x + i, sizeof(T));
                const int j = i - i0, at_word = j * (int)sizeof(T) / 4, by = j * (int)sizeof(T) % 4 * 8;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (k == at_word) w[k] |= bits << by;
            }
            return make_uint4(w[0], w[1], w[2], w[3]);
        }
    };
    uint4 held[KEPT ? U : 1];
    float m = 0.0f;
    if (KEPT) {
#pragma unroll
        for (int u = 0; u < U; ++u) held[u] = at + u * TEAM < vecs ? load(at + u * TEAM) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < U; ++u) m = larger_magnitude(m, largest_magnitude<T>(held[u]));
    } else {
#pragma unroll 4
        for (int v = at; v < vecs; v += TEAM) m = larger_magnitude(m, largest_magnitude<T>(load(v)));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = larger_magnitude(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (TEAM == 256) {
        if (lane == 0) most[threadIdx.x >> 5] = m;
        __syncthreads();
        m = most[lane & 7];
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) m = larger_magnitude(m, __shfl_xor_sync(0xffffffffu, m, o));
    }
    const RowScale s(m);
    if (at == 0) scales[r] = s.scale;
    const auto word = [&](const uint4 &h) {
        const Vec<unsigned char, W> o = s.template quantised<T>(h);
        Word w;
        memcpy(&w, &o, W);
        return w;
    };
    // w: the integers of vector v, last: those of the vector before the warp's first one; whole warps come here, and a vector behind the last one stores nothing
    const auto store = [&](int v, Word w, Word last) {
        int i0 = v * W - mis;
        if constexpr (!WHOLE) {
            Word before = __shfl_up_sync(0xffffffffu, w, 1);
            if (lane == 0) before = last;
            if (shift) {
                w = (before >> (8 * shift)) | (w << (8 * (W - shift)));
                i0 += shift - W;
            }
        }
        if (v >= vecs) return;
        if (WHOLE || (i0 >= 0 && i0 + W <= dim)) *reinterpret_cast<Word *>(to + i0) = w;
        else {
#pragma unroll 1
            for (int j = max(0, -i0); j < min(W, dim - i0); ++j) to[i0 + j] = (unsigned char)(w >> (8 * j));
        }
    };
    if (KEPT && TEAM == 32) {
        Word last = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (WHOLE ? at + u * TEAM >= vecs : u * TEAM >= vecs) break;
            const Word w = word(held[u]);
            store(at + u * TEAM, w, last);
            if constexpr (!WHOLE) last = __shfl_sync(0xffffffffu, w, 31);
        }
    } else {
#pragma unroll
        for (int u = 0; KEPT && u < U; ++u) {
            const int v = at + u * TEAM;
            if (WHOLE ? v >= vecs : (v & ~31) >= vecs) break;
            store(v, word(held[u]), !WHOLE && lane == 0 && v > 0 && v <= vecs ? word(load(v - 1)) : 0);
        }
        for (int v = at; !KEPT && (WHOLE ? v < vecs : (v & ~31) < vecs); v += TEAM)
            store(v, word(v < vecs ? load(v) : make_uint4(0, 0, 0, 0)), !WHOLE && lane == 0 && v > 0 && v <= vecs ? word(load(v - 1)) : 0);
    }
}

template <typename T, bool WHOLE> int quantize_rows(signed char *q, long long ld_q, float *scales, const T *x, long long rows, int dim, long long ld_x, cudaStream_t st) {
    constexpr int W = 16 / sizeof(T);
    const int vecs = WHOLE ? dim / W : (dim + W - 1) / W + 2;      // a row may start inside a vector, and its last bytes come with one more
    const auto go = [&](auto kernel, int teams) -> int {
        const long long blocks = (rows + teams - 1) / teams;
        if (blocks > 0x7fffffffll) { set_error("b2_int8_quantize: %lld rows", rows); return B2_ERR_BAD_SHAPE; }
        kernel<<<(unsigned)blocks, 256, 0, st>>>(q, ld_q, scales, x, rows, dim, ld_x);
        count_launch();
        B2_CUDA(cudaGetLastError());
        return B2_OK;
    };
    if (vecs <= 32 * 4) return go(int8_quantize_kernel<T, 32, 4, true, WHOLE>, 8);
    if (vecs <= 32 * 8) return go(int8_quantize_kernel<T, 32, 8, true, WHOLE>, 8);
    if (vecs <= 256 * 4) return go(int8_quantize_kernel<T, 256, 4, true, WHOLE>, 1);
    if (vecs <= 256 * 8) return go(int8_quantize_kernel<T, 256, 8, true, WHOLE>, 1);
    return go(int8_quantize_kernel<T, 256, 4, false, WHOLE>, 1);
}
template <typename T> int quantize(signed char *q, long long ld_q, float *scales, const T *x, long long rows, int dim, long long ld_x, cudaStream_t st) {
    constexpr int W = 16 / sizeof(T);
    if (aligned_to(x, 16) && (rows == 1 || ld_x % W == 0) && dim % W == 0 && aligned_to(q, W) && (rows == 1 || ld_q % W == 0))
        return quantize_rows<T, true>(q, ld_q, scales, x, rows, dim, ld_x, st);
    return quantize_rows<T, false>(q, ld_q, scales, x, rows, dim, ld_x, st);
}

// ---- product --------------------------------------------------------------------------------------------------------------------------
constexpr int BM = 128, BK = 128;                 // channels of a block's tile, positions of a slab (one swizzle row of 128 bytes)
constexpr int A_BYTES = BM * BK;
constexpr int THREADS = 320;                      // warp 0 copies, 1 multiplies, 2 to 9 store
constexpr long long WAIT_CYCLES = 4000000000LL;   // about two seconds
struct ProductArgs {
    const float *x_scales, *w_scales, *bias;
    long long ld_out, rows;
    int channels, slabs;
    unsigned row_tiles, channel_tiles, splits;
    int chained;
};

// N columns (rows r0 on of out) of a thread's tensor-memory lane (channel c; real: there is one) to out.  xs: their scales in shared memory, 16-byte aligned
// more(v, j): what is added to the columns j on, of which v holds the sums
template <int N, typename O, typename F>
__device__ __forceinline__ void store_columns(uint32_t taddr, const float *xs, float ws, float bias, bool real, bool ok, O *out, long long ld, long long r0, long long rows, int c, F &&more) {
    constexpr int STEP = N < 32 ? N : 32;
    const long long left = rows - r0;
    O *p = out + r0 * ld + c;
#pragma unroll 1
    for (int j0 = 0; j0 < N; j0 += STEP) {
        if (j0 >= left) break;
        uint32_t v[STEP];
        if constexpr (STEP == 32) ptx::tmem_ld32(taddr + j0, v);
        else if constexpr (STEP == 16) ptx::tmem_ld16(taddr + j0, v);
        else ptx::tmem_ld8(taddr + j0, v);
        ptx::tmem_ld_wait();
        more(v, j0);
        const auto put = [&](bool all) {
#pragma unroll
            for (int j = 0; j < STEP; j += 4) {
                const float4 s = *reinterpret_cast<const float4 *>(xs + j0 + j);
                const float f[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // a tile that its block gave up on shows as NaN
                    const float y = ok ? fmaf((float)(int)v[j + i], f[i] * ws, bias) : nanf("");
                    if (real && (all || j0 + j + i < left)) *p = from_float<O>(y);
                    p += ld;
                }
            }
        };
        if (j0 + STEP <= left) put(true); else put(false);
    }
}
template <int N, typename O>
__device__ __forceinline__ void store_columns(uint32_t taddr, const float *xs, float ws, float bias, bool real, bool ok, O *out, long long ld, long long r0, long long rows, int c) {
    store_columns<N>(taddr, xs, ws, bias, real, ok, out, ld, r0, rows, c, [](auto &, int) {});
}
// a warp's copy of the scales of N rows from r0 on
template <int N> __device__ __forceinline__ void load_scales(float *xs, const float *x_scales, long long r0, long long rows) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < N; j += 32)
        if (j + lane < N) xs[j + lane] = r0 + j + lane < rows ? x_scales[r0 + j + lane] : 0.0f;
    __syncwarp();
}

// Up to 128 rows: a block's tile has BN columns, the weights stream through the ring.  Few channels: the blocks of a cluster (a.splits of them) share the slabs of a tile, and
// the first one adds up their sums, which the others lay down in its shared memory: whole numbers, so that the split changes nothing.
template <int BN, int STAGES_> struct Shape {
    static constexpr int STAGE_BYTES = A_BYTES + BN * BK, STAGES = STAGES_;
    static constexpr int SMEM = STAGES * STAGE_BYTES + 1024;      // slack: the swizzle wants 1024-byte alignment
    static constexpr int TMEM = 2 * BN;
};
// the most blocks that share a tile: the others' sums lie in the first one's ring
template <int BN> constexpr int most_splits() { return 4 * Shape<BN, 4>::STAGE_BYTES >= 7 * BN * BM * 4 ? 8 : 4 * Shape<BN, 4>::STAGE_BYTES >= 3 * BN * BM * 4 ? 4 : 2; }
template <int BN, int STAGES, typename O>
__global__ void __launch_bounds__(THREADS, STAGES == 4 && BN < 128 ? 2 : 1)
int8_product_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, O *out, const ProductArgs a) {
    using namespace ptx;
    typedef Shape<BN, STAGES> S;
    constexpr int HALF = BN / 2;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long bars[2 * STAGES + 5];
    __shared__ __align__(16) float scales[8][HALF];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int fail;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u, bar0 = smem_u32(bars);
    const auto full = [&](int s) { return bar0 + 8u * (uint32_t)s; };
    const auto empty = [&](int s) { return bar0 + 8u * (uint32_t)(STAGES + s); };
    const auto acc_full = [&](int b) { return bar0 + 8u * (uint32_t)(2 * STAGES + b); };
    const auto acc_empty = [&](int b) { return bar0 + 8u * (uint32_t)(2 * STAGES + 2 + b); };
    const uint32_t idle = bar0 + 8u * (uint32_t)(2 * STAGES + 4);
    // the tiles t0, t0 + step, ... (split: the one), and of each the slabs s0 on
    const unsigned tiles = a.row_tiles * a.channel_tiles, rank = a.splits > 1 ? cluster_ctarank() : 0, t0 = blockIdx.x / a.splits, step = gridDim.x / a.splits;
    const int s0 = (int)(a.slabs * rank / a.splits), slabs = (int)(a.slabs * (rank + 1) / a.splits) - s0;
    const unsigned mine = (tiles - t0 + step - 1) / step * (unsigned)slabs, first = min(mine, (unsigned)STAGES);      // slabs of this block
    const auto copy_w = [&](unsigned i) {
        const int s = (int)(i % STAGES);
        mbar_expect_tx(full(s), S::STAGE_BYTES);
        tma_load_2d(ring + (uint32_t)s * S::STAGE_BYTES, &map_w, (s0 + (int)(i % (unsigned)slabs)) * BK, (int)((t0 + i / (unsigned)slabs * step) / a.row_tiles) * BM, full(s));
    };
    const auto copy_x = [&](unsigned i) {
        const int s = (int)(i % STAGES);
        tma_load_2d(ring + (uint32_t)s * S::STAGE_BYTES + A_BYTES, &map_x, (s0 + (int)(i % (unsigned)slabs)) * BK, (int)((t0 + i / (unsigned)slabs * step) % a.row_tiles) * BN, full(s));
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(acc_full(b), 1); mbar_init(acc_empty(b), 8); }
        mbar_init(idle, 1);
        fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
        // The first slabs' weights are on the way before the block is set up, and before the activations, which the launch before this one may still be writing
        for (unsigned i = 0; i < first; ++i) copy_w(i);
    }
    if (warp == 1) tmem_alloc(smem_u32((const void *)&tmem_slot), S::TMEM);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {
            if (a.chained) { grid_wait(); fence_async_global(); }
            unsigned i = 0;
            for (; i < first; ++i) copy_x(i);
            for (; i < mine; ++i) {
                if (!mbar_wait_bounded<false>(empty((int)(i % STAGES)), ((i / STAGES) & 1u) ^ 1u, &fail, WAIT_CYCLES)) { fail = 1; ok = false; break; }
                copy_w(i);
                copy_x(i);
            }
            if (!ok)      // copies under way end before the block does
                for (unsigned j = i > (unsigned)STAGES ? i - STAGES : 0; j < i; ++j) {
                    volatile int never = 0;
                    mbar_wait_bounded<false>(full((int)(j % STAGES)), (j / STAGES) & 1u, &never, WAIT_CYCLES);
                }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = idesc_s8(BM, BN);
            unsigned i = 0, n = 0;
            for (unsigned tile = t0; tile < tiles && ok; tile += step, ++n) {
                const uint32_t d = tmem + (n & 1u) * BN;
                if (!mbar_wait_bounded<false>(acc_empty((int)(n & 1u)), ((n >> 1) & 1u) ^ 1u, &fail, WAIT_CYCLES)) { fail = 1; ok = false; break; }
                tc_fence_after();
                for (int k = 0; k < slabs; ++k, ++i) {
                    const int s = (int)(i % STAGES);
                    if (!mbar_wait_bounded<false>(full(s), (i / STAGES) & 1u, &fail, WAIT_CYCLES)) { fail = 1; ok = false; break; }
                    tc_fence_after();
                    const uint32_t at = ring + (uint32_t)s * S::STAGE_BYTES;
#pragma unroll
                    for (int kk = 0; kk < BK / 32; ++kk)
                        mma_s8(d, desc_kmajor_sw128(at + kk * 32, 1024), desc_kmajor_sw128(at + A_BYTES + kk * 32, 1024), idesc, (k | kk) ? 1u : 0u);
                    mma_commit(empty(s));
                }
                if (ok) mma_commit(acc_full((int)(n & 1u)));
            }
            if (!ok) {
                volatile int never = 0;
                mma_commit(idle);
                mbar_wait_bounded<false>(idle, 0, &never, WAIT_CYCLES);
            }
        }
    }
    // A warp reads the tensor-memory lanes 32 * (warp % 4) on; warps 2 to 5 take the first half of the columns, 6 to 9 the second
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t sums = tmem + ((uint32_t)(32 * quarter) << 16) + half * HALF;
    long long r0 = 0;
    int c = 0;
    float ws = 0.0f, bias = 0.0f;
    if (warp >= 2) {
        unsigned n = 0;
        if (a.chained) grid_wait();
        for (unsigned tile = t0; tile < tiles; tile += step, ++n) {
            r0 = (long long)(tile % a.row_tiles) * BN + half * HALF;
            c = (int)(tile / a.row_tiles) * BM + 32 * quarter + lane;
            const bool real = c < a.channels;
            ws = real ? a.w_scales[c] : 0.0f;
            bias = real && a.bias ? a.bias[c] : 0.0f;
            load_scales<HALF>(scales[warp - 2], a.x_scales, r0, a.rows);
            ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded<false>(acc_full((int)(n & 1u)), (n >> 1) & 1u, &fail, WAIT_CYCLES));
            if (!ok && lane == 0) fail = 1;
            tc_fence_after();
            if (a.splits > 1) break;
            store_columns<HALF>(sums + (n & 1u) * BN, scales[warp - 2], ws, bias, real, ok, out, a.ld_out, r0, a.rows, c);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty((int)(n & 1u)));
        }
    }
    if (a.splits > 1) {
        // the products of all blocks are complete, and the first one's ring is free
        __syncwarp();
        cluster_sync_all();
        const uint32_t place = ring + (uint32_t)(half * HALF) * (4 * BM) + 4u * (uint32_t)(32 * quarter + lane);
        if (warp >= 2 && rank) {
            const uint32_t there = map_to_rank(place + (rank - 1) * (BN * BM * 4), 0);
#pragma unroll 2
            for (int j0 = 0; j0 < HALF; j0 += 8) {
                uint32_t v[8];
                tmem_ld8(sums + j0, v);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 8; ++j) st_cluster_u32(there + (uint32_t)(j0 + j) * (4 * BM), v[j]);
            }
            if (!ok && lane == 0) st_cluster_u32(map_to_rank(smem_u32((const void *)&fail), 0), 1);
        }
        cluster_sync_all();
        if (warp >= 2 && !rank) {
            const int *others = reinterpret_cast<const int *>(smem_raw + (place - smem_u32(smem_raw)));
            store_columns<HALF>(sums, scales[warp - 2], ws, bias, c < a.channels, ok && !fail, out, a.ld_out, r0, a.rows, c, [&](auto &v, int j0) {
                for (unsigned p = 0; p + 1 < a.splits; ++p)
#pragma unroll
                    for (unsigned j = 0; j < sizeof(v) / 4; ++j) v[j] += (uint32_t)others[(p * BN + j0 + j) * BM];
            });
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, S::TMEM);
}

// Up to 8 short rows of activations that are no integers yet: every block quantises them for itself, into the layout of the tensor cores' operand, while its
// first slabs of weights are on the way.  One launch, and the activations pass through no memory.
constexpr int ROWS_BN = 16, ROWS_STAGES = 8;      // columns of a tile, slabs of the ring
constexpr int rows_smem(int slabs) { return ROWS_STAGES * A_BYTES + slabs * ROWS_BN * BK + 1024; }
template <typename T, typename O>
__global__ void __launch_bounds__(THREADS, 1)
int8_rows_kernel(const __grid_constant__ CUtensorMap map_w, const T *x, long long ld_x, int dim, O *out, const ProductArgs a) {
    using namespace ptx;
    constexpr int BN = ROWS_BN, STAGES = ROWS_STAGES, W = 16 / sizeof(T), U = sizeof(T) == 4 ? 8 : 4, TMEM = 2 * BN, HALF = BN / 2;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long bars[2 * STAGES + 6];
    __shared__ __align__(16) float scales[BN];
    __shared__ float most[8];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int fail;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w = warp - 2;
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u, bar0 = smem_u32(bars), operand = ring + STAGES * A_BYTES;
    const auto full = [&](int s) { return bar0 + 8u * (uint32_t)s; };
    const auto empty = [&](int s) { return bar0 + 8u * (uint32_t)(STAGES + s); };
    const auto acc_full = [&](int b) { return bar0 + 8u * (uint32_t)(2 * STAGES + b); };
    const auto acc_empty = [&](int b) { return bar0 + 8u * (uint32_t)(2 * STAGES + 2 + b); };
    const uint32_t idle = bar0 + 8u * (uint32_t)(2 * STAGES + 4), x_full = bar0 + 8u * (uint32_t)(2 * STAGES + 5);
    const unsigned tiles = a.channel_tiles, t0 = blockIdx.x, step = gridDim.x;
    const int slabs = a.slabs;
    const unsigned mine = (tiles - t0 + step - 1) / step * (unsigned)slabs, first = min(mine, (unsigned)STAGES);      // slabs of this block
    const auto copy = [&](unsigned i) {
        const int s = (int)(i % STAGES);
        mbar_expect_tx(full(s), A_BYTES);
        tma_load_2d(ring + (uint32_t)s * A_BYTES, &map_w, (int)(i % (unsigned)slabs) * BK, (int)(t0 + i / (unsigned)slabs * step) * BM, full(s));
    };
    // Warp w has row w % together of x, the vectors of part w / together of `parts`: with few rows several warps share one
    const int together = a.rows > 4 ? 8 : a.rows > 2 ? 4 : (int)a.rows, parts = 8 / together, part = w / together, r = w % together;
    const bool there = warp >= 2 && r < a.rows;
    const T *row = x + (there ? r : 0) * ld_x;
    // in vectors where the row allows it, else entry by entry: a launch runs through its code once, and what it has to fetch of it counts
    const bool vectors = there && (((uintptr_t)row & 15) == 0) && dim % W == 0;
    uint4 held[U];
    float m = 0.0f;
    if (vectors) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = ((part + u * parts) * 32 + lane) * W;
            held[u] = i < dim ? *reinterpret_cast<const uint4 *>(row + i) : make_uint4(0, 0, 0, 0);
        }
    } else if (there)
        for (int i = part * 32 + lane; i < dim; i += 32 * parts) m = larger_magnitude(m, fabsf(to_float(row[i])));
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(acc_full(b), 1); mbar_init(acc_empty(b), 8); }
        mbar_init(idle, 1);
        mbar_init(x_full, 8);
        fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
        // the first slabs are on the way before the block is set up
        for (unsigned i = 0; i < first; ++i) copy(i);
    }
    if (warp == 1) tmem_alloc(smem_u32((const void *)&tmem_slot), TMEM);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {
            unsigned i = first;
            for (; i < mine; ++i) {
                if (!mbar_wait_bounded<false>(empty((int)(i % STAGES)), ((i / STAGES) & 1u) ^ 1u, &fail, WAIT_CYCLES)) { fail = 1; ok = false; break; }
                copy(i);
            }
            if (!ok)      // copies under way end before the block does
                for (unsigned j = i > (unsigned)STAGES ? i - STAGES : 0; j < i; ++j) {
                    volatile int never = 0;
                    mbar_wait_bounded<false>(full((int)(j % STAGES)), (j / STAGES) & 1u, &never, WAIT_CYCLES);
                }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = idesc_s8(BM, BN);
            unsigned i = 0, n = 0;
            ok = mbar_wait_bounded<false>(x_full, 0, &fail, WAIT_CYCLES);
            if (!ok) fail = 1;
            for (unsigned tile = t0; tile < tiles && ok; tile += step, ++n) {
                const uint32_t d = tmem + (n & 1u) * BN;
                if (!mbar_wait_bounded<false>(acc_empty((int)(n & 1u)), ((n >> 1) & 1u) ^ 1u, &fail, WAIT_CYCLES)) { fail = 1; ok = false; break; }
                tc_fence_after();
                for (int k = 0; k < slabs; ++k, ++i) {
                    const int s = (int)(i % STAGES);
                    if (!mbar_wait_bounded<false>(full(s), (i / STAGES) & 1u, &fail, WAIT_CYCLES)) { fail = 1; ok = false; break; }
                    tc_fence_after();
                    const uint32_t at = ring + (uint32_t)s * A_BYTES, b = operand + (uint32_t)k * (BN * BK);
#pragma unroll
                    for (int kk = 0; kk < BK / 32; ++kk) mma_s8(d, desc_kmajor_sw128(at + kk * 32, 1024), desc_kmajor_sw128(b + kk * 32, 1024), idesc, (k | kk) ? 1u : 0u);
                    mma_commit(empty(s));
                }
                if (ok) mma_commit(acc_full((int)(n & 1u)));
            }
            if (!ok) {
                volatile int never = 0;
                mma_commit(idle);
                mbar_wait_bounded<false>(idle, 0, &never, WAIT_CYCLES);
            }
        }
    } else {
        // Columns without a row, and positions behind the last one, meet zeros of the weights or are not stored
        unsigned char *const to = smem_raw + (operand - smem_u32(smem_raw));
        if (vectors)
#pragma unroll
            for (int u = 0; u < U; ++u) m = larger_magnitude(m, largest_magnitude<T>(held[u]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = larger_magnitude(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (parts > 1) {
            if (lane == 0) most[w] = m;
            bar_named(1, 256);
            for (int p = 0; p < parts; ++p) m = larger_magnitude(m, most[r + p * together]);
        }
        if (there) {
            const RowScale q(m);
            if (lane == 0 && part == 0) scales[r] = q.scale;
            // slab, row of 128 bytes, 16-byte chunk with its index xor the row's
            const auto place = [&](int k) { return (k / BK) * (BN * BK) + r * BK + ((((k % BK) >> 4) ^ (r & 7)) << 4) + (k & 15); };
            if (vectors) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int i = ((part + u * parts) * 32 + lane) * W;
                    if (i < dim) *reinterpret_cast<Vec<unsigned char, W> *>(to + place(i)) = q.template quantised<T>(held[u]);
                }
            } else
                for (int i = part * 32 + lane; i < dim; i += 32 * parts) to[place(i)] = q.quantised(to_float(row[i]));
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(x_full);
        bar_named(1, 256);                   // the scales
    }
    // A warp reads the tensor-memory lanes 32 * (warp % 4) on; warps 2 to 5 have the first half of the columns, 6 to 9 the second
    const int quarter = warp & 3, half = w >> 2;
    const uint32_t sums = tmem + ((uint32_t)(32 * quarter) << 16) + half * HALF;
    if (warp >= 2) {
        unsigned n = 0;
        for (unsigned tile = t0; tile < tiles; tile += step, ++n) {
            const int c = (int)tile * BM + 32 * quarter + lane;
            const bool real = c < a.channels;
            const float ws = real ? a.w_scales[c] : 0.0f, bias = real && a.bias ? a.bias[c] : 0.0f;
            ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded<false>(acc_full((int)(n & 1u)), (n >> 1) & 1u, &fail, WAIT_CYCLES));
            if (!ok && lane == 0) fail = 1;
            tc_fence_after();
            store_columns<HALF>(sums + (n & 1u) * BN, scales + half * HALF, ws, bias, real, ok, out, a.ld_out, half * HALF, a.rows, c);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty((int)(n & 1u)));
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, TMEM);
}

// Many rows: a pair of blocks (cta_group::2) has a tile of 256 channels, 128 in each block, and 256 rows, of which each block holds 128 in its shared memory.  A
// slab so costs a block 32 KB of copies and 32 KB of operand reads for 512 cycles of multiplication; by itself, with the same tile, it would be 48 and 48.
// The data path of the shared memory is what bounds short contractions: with 8 slabs a tile takes 4096 cycles of multiplication, 2048 of operand reads, as many of
// copies, 1024 of accumulators read and 2200 of stores.  So up to 9 slabs of weights stay in shared memory over all tiles of their channels (RESIDENT), and only the
// activations pass through the ring.
constexpr int PAIR_BN = 256, PAIR_B = PAIR_BN / 2 * BK, PAIR_TMEM = 512, MOST_RESIDENT = 9;
template <bool RESIDENT> struct PairShape {
    static constexpr int STAGE = RESIDENT ? PAIR_B : A_BYTES + PAIR_B, STAGES = RESIDENT ? 4 : 6;
    static constexpr int SMEM = STAGES * STAGE + (RESIDENT ? MOST_RESIDENT * A_BYTES : 0) + 1024;
};
// The tiles of a pair.  Neighbouring pairs work on neighbouring channels of the same rows at the same time: where rows of `out` are not aligned, a sector between two
// tiles is written by both, and should be in the L2 still when the second one comes (8192 x 50001 x 1024: 498 us with a run of tiles for each pair).
// RESIDENT: all rows of a channel tile, round by round; the channel tiles of the last round are dealt out in runs of rows.  Else: rows first, in turn.
template <bool RESIDENT> struct PairTiles {
    unsigned pair, pairs, rows, whole, rest0, count;       // whole: tiles of the full rounds
    __device__ __forceinline__ PairTiles(const ProductArgs &a) : pair(blockIdx.x >> 1), pairs(gridDim.x >> 1), rows(a.row_tiles) {
        if (RESIDENT) {
            const unsigned rounds = a.channel_tiles / pairs;
            const unsigned long long rest = (unsigned long long)(a.channel_tiles - rounds * pairs) * rows;
            whole = rounds * rows;
            rest0 = (unsigned)(rest * pair / pairs);
            count = whole + (unsigned)(rest * (pair + 1) / pairs) - rest0;
        } else {
            whole = rest0 = 0;
            count = (rows * a.channel_tiles - pair + pairs - 1) / pairs;
        }
    }
    // row and channel tile of the n-th one; whether its weights are others than those of the one before
    __device__ __forceinline__ bool at(unsigned n, unsigned &r, unsigned &c) const {
        unsigned t, c0;
        if (!RESIDENT) { t = pair + n * pairs; c0 = 0; }
        else if (n < whole) { t = n % rows; c0 = pair + n / rows * pairs; }
        else { t = rest0 + n - whole; c0 = whole / rows * pairs; }
        r = t % rows;
        c = c0 + t / rows;
        return !RESIDENT || n == 0 || n == whole || r == 0;
    }
};
template <bool RESIDENT, typename O>
__global__ void __launch_bounds__(THREADS, 1)
int8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, O *out, const ProductArgs a) {
    using namespace ptx;
    typedef PairShape<RESIDENT> S;
    constexpr int BN = PAIR_BN, STAGES = S::STAGES, STAGE = S::STAGE;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long bars[2 * STAGES + 5];
    __shared__ __align__(16) float scales[8][BN / 2];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int fail;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u, bar0 = smem_u32(bars), held = ring + STAGES * STAGE;      // held: the weights that stay
    // full and acc_empty: the even block's count; empty, acc_full: each block has its own
    const auto full = [&](int s) { return bar0 + 8u * (uint32_t)s; };
    const auto empty = [&](int s) { return bar0 + 8u * (uint32_t)(STAGES + s); };
    const auto acc_full = [&](int b) { return bar0 + 8u * (uint32_t)(2 * STAGES + b); };
    const auto acc_empty = [&](int b) { return bar0 + 8u * (uint32_t)(2 * STAGES + 2 + b); };
    const uint32_t idle = bar0 + 8u * (uint32_t)(2 * STAGES + 4);
    const PairTiles<RESIDENT> tiles(a);
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(acc_full(b), 1); mbar_init(acc_empty(b), 16); }
        mbar_init(idle, 1);
        fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == 1) tmem_alloc_pair(smem_u32((const void *)&tmem_slot), PAIR_TMEM);
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            unsigned i = 0;
            bool ok = true;
            if (a.chained) { grid_wait(); fence_async_global(); }
            for (unsigned n = 0; n < tiles.count && ok; ++n) {
                unsigned r, c;
                const bool fresh = tiles.at(n, r, c);
                const int r0 = (int)r * BN + (int)rank * (BN / 2), c0 = (int)c * (2 * BM) + (int)rank * BM;
                for (int k = 0; k < a.slabs; ++k, ++i) {
                    const int s = (int)(i % STAGES);
                    if (!mbar_wait_bounded<false>(empty(s), ((i / STAGES) & 1u) ^ 1u, &fail, WAIT_CYCLES)) { fail = 1; ok = false; break; }
                    // The weights that were in slab k have to be read, `slabs` uses of the ring ago.  With as many slabs as slots or more, that use came before the one which freed this
                    // slot; else it is waited for.
                    if (RESIDENT && fresh && n > 0 && a.slabs < STAGES) {
                        const unsigned j = i - (unsigned)a.slabs;
                        if (!mbar_wait_bounded<false>(empty((int)(j % STAGES)), (j / STAGES) & 1u, &fail, WAIT_CYCLES)) { fail = 1; ok = false; break; }
                    }
                    const uint32_t at = ring + (uint32_t)s * STAGE, bar = map_to_rank(full(s), 0);
                    if (rank == 0) mbar_expect_tx(full(s), 2 * (PAIR_B + (fresh ? A_BYTES : 0)));
                    if (fresh) tma_load_2d_pair(RESIDENT ? held + (uint32_t)k * A_BYTES : at + PAIR_B, &map_w, k * BK, c0, bar);
                    tma_load_2d_pair(at, &map_x, k * BK, r0, bar);
                }
            }
            if (!ok && rank == 0)      // copies under way end before the blocks do
                for (unsigned j = i > (unsigned)STAGES ? i - STAGES : 0; j < i; ++j) {
                    volatile int never = 0;
                    mbar_wait_bounded<false>(full((int)(j % STAGES)), (j / STAGES) & 1u, &never, WAIT_CYCLES);
                }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            const uint32_t idesc = idesc_s8(2 * BM, BN);
            unsigned i = 0;
            bool ok = true;
            for (unsigned n = 0; n < tiles.count && ok; ++n) {
                const uint32_t d = tmem + (n & 1u) * BN;
                if (!mbar_wait_bounded<true>(acc_empty((int)(n & 1u)), ((n >> 1) & 1u) ^ 1u, &fail, WAIT_CYCLES)) { fail = 1; ok = false; break; }
                tc_fence_after();
                for (int k = 0; k < a.slabs; ++k, ++i) {
                    const int s = (int)(i % STAGES);
                    if (!mbar_wait_bounded<true>(full(s), (i / STAGES) & 1u, &fail, WAIT_CYCLES)) { fail = 1; ok = false; break; }
                    tc_fence_after();
                    const uint32_t x = ring + (uint32_t)s * STAGE, w = RESIDENT ? held + (uint32_t)k * A_BYTES : x + PAIR_B;
#pragma unroll
                    for (int kk = 0; kk < BK / 32; ++kk) mma_s8_pair(d, desc_kmajor_sw128(w + kk * 32, 1024), desc_kmajor_sw128(x + kk * 32, 1024), idesc, (k | kk) ? 1u : 0u);
                    mma_commit_pair(empty(s));
                }
                if (ok) mma_commit_pair(acc_full((int)(n & 1u)));
            }
            if (!ok) {
                volatile int never = 0;
                mma_commit_pair(idle);
                mbar_wait_bounded<false>(idle, 0, &never, WAIT_CYCLES);
            }
        }
    } else {
        constexpr int HALF = BN / 2;
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        bool ok = true;
        if (a.chained) grid_wait();
        for (unsigned n = 0; n < tiles.count; ++n) {
            unsigned row_tile, channel_tile;
            tiles.at(n, row_tile, channel_tile);
            const long long r0 = (long long)row_tile * BN + half * HALF;
            const int c = (int)channel_tile * (2 * BM) + (int)rank * BM + 32 * quarter + lane;
            const bool real = c < a.channels;
            const float ws = real ? a.w_scales[c] : 0.0f, bias = real && a.bias ? a.bias[c] : 0.0f;
            load_scales<HALF>(scales[warp - 2], a.x_scales, r0, a.rows);
            ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded<false>(acc_full((int)(n & 1u)), (n >> 1) & 1u, &fail, WAIT_CYCLES));
            if (!ok && lane == 0) fail = 1;
            tc_fence_after();
            store_columns<HALF>(tmem + ((uint32_t)(32 * quarter) << 16) + (n & 1u) * BN + half * HALF, scales[warp - 2], ws, bias, real, ok, out, a.ld_out, r0, a.rows, c);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_relaxed(map_to_rank(acc_empty((int)(n & 1u)), 0));
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();          // neither block leaves while the other's arrivals and copies may still reach it
    if (warp == 1) tmem_dealloc_pair(tmem, PAIR_TMEM);
}

// pairs of blocks that run side by side, by device
int pair_count(const void *kernel, int bytes, int *out) {
    static std::mutex mu;
    static int known[MAX_DEVICES];      // of all element types: a block has its SM to itself
    const int dev = current_device();
    if (dev < 0) { set_error("no current CUDA device (or an ordinal beyond %d)", MAX_DEVICES - 1); return B2_ERR_CUDA; }
    std::lock_guard<std::mutex> lk(mu);
    int &n = known[dev];
    if (!n) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2 * (unsigned)(sm_count() / 2 > 0 ? sm_count() / 2 : 1));
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = bytes;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = 2;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        int clusters = 0;
        B2_CUDA(cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg));
        if (clusters < 1) { set_error("b2_int8_product: no pair of blocks fits on the device"); return B2_ERR_CUDA; }
        n = clusters;
    }
    *out = n;
    return B2_OK;
}

template <int BN, int STAGES, typename O> int launch_product(const CUtensorMap &mw, const CUtensorMap &mx, O *out, const ProductArgs &a, unsigned blocks, cudaStream_t st) {
    const auto kernel = int8_product_kernel<BN, STAGES, O>;
    constexpr int BYTES = Shape<BN, STAGES>::SMEM;
    B2_TRY(set_max_dynamic_smem((const void *)kernel, BYTES));
    return launch_chained(int8_product_kernel<BN, STAGES, O>, Clusters{a.splits, a.chained}, dim3(blocks), dim3(THREADS), BYTES, st, mw, mx, out, a);
}
template <bool RESIDENT, typename O> int launch_pairs(const CUtensorMap &mw, const CUtensorMap &mx, O *out, ProductArgs a, cudaStream_t st) {
    const auto kernel = int8_pair_kernel<RESIDENT, O>;
    constexpr int BYTES = PairShape<RESIDENT>::SMEM;
    B2_TRY(set_max_dynamic_smem((const void *)kernel, BYTES));
    int pairs;
    B2_TRY(pair_count((const void *)kernel, BYTES, &pairs));
    const long long tiles = (long long)a.row_tiles * a.channel_tiles;
    const unsigned blocks = 2 * (unsigned)(tiles < pairs ? tiles : pairs);
    return launch_chained(int8_pair_kernel<RESIDENT, O>, Clusters{2, a.chained}, dim3(blocks), dim3(THREADS), BYTES, st, mw, mx, out, a);
}

size_t pitch_of(int dim) { return ((size_t)dim + 15) & ~(size_t)15; }
bool sizes_fit(long long rows, int channels, int dim) { return rows >= 0 && rows <= 0x7fffff00ll && channels >= 1 && channels <= 0x7fffff00 && dim >= 1 && dim <= 131071; }

template <typename O> int product(O *out, const signed char *x, long long ld_x, const signed char *w, long long ld_w, int dim, ProductArgs a, cudaStream_t st) {
    const auto go = [&](auto columns) -> int {
        constexpr int BN = decltype(columns)::value;
        constexpr bool PAIR = BN == PAIR_BN;
        CUtensorMap mw, mx;
        B2_TRY(make_byte_map(&mw, w, dim, a.channels, ld_w, BM));
        B2_TRY(make_byte_map(&mx, x, dim, a.rows, ld_x, PAIR ? BN / 2 : BN));
        a.row_tiles = (unsigned)((a.rows + BN - 1) / BN);
        a.channel_tiles = (unsigned)((a.channels + (PAIR ? 2 : 1) * BM - 1) / ((PAIR ? 2 : 1) * BM));
        if ((double)a.row_tiles * a.channel_tiles > 4e9) { set_error("b2_int8_product: %lld rows of %d channels", a.rows, a.channels); return B2_ERR_BAD_SHAPE; }
        if constexpr (PAIR) return a.slabs <= MOST_RESIDENT ? launch_pairs<true, O>(mw, mx, out, a, st) : launch_pairs<false, O>(mw, mx, out, a, st);
        else {
            // Where the tiles leave blocks idle, clusters share a tile, each block with 2 slabs at least: two blocks an SM then, with half the ring (8 x 4096 x 4096: 17.3 us
            // without)
            constexpr int RING = BN >= 128 ? 6 : 8, RESIDENT = BN < 128 ? 2 : 1;
            const long long tiles = (long long)a.row_tiles * a.channel_tiles;
            a.splits = 1;
            while ((int)a.splits < most_splits<BN>() && tiles * a.splits * 2 <= RESIDENT * sm_count() && a.slabs / (int)(a.splits * 2) >= 2) a.splits *= 2;
            if (a.splits > 1) return launch_product<BN, 4, O>(mw, mx, out, a, (unsigned)tiles * a.splits, st);
            return launch_product<BN, RING, O>(mw, mx, out, a, (unsigned)(tiles < sm_count() ? tiles : sm_count()), st);
        }
    };
    if (a.rows <= 16) return go(std::integral_constant<int, 16>());
    if (a.rows <= 32) return go(std::integral_constant<int, 32>());
    if (a.rows <= 64) return go(std::integral_constant<int, 64>());
    if (a.rows <= 128) return go(std::integral_constant<int, 128>());
    return go(std::integral_constant<int, PAIR_BN>());
}
// Whether the call runs as one launch that quantises in every block: up to 8 rows that fit into the registers of 8 warps, and more tiles than a split would fill
// (8 x 50001 x 1024: 10.6 us; x 1040, in two launches: 12.8 us)
bool few_rows(long long rows, int channels, int dim) {
    const int parts = rows > 4 ? 1 : rows > 2 ? 2 : rows > 1 ? 4 : 8;
    return rows <= 8 && dim <= 1024 * parts && (dim + BK - 1) / BK * (ROWS_BN * BK) <= 80 * 1024 && ((channels + BM - 1ll) / BM * 2 > sm_count() || dim <= 2 * BK);
}
template <typename T, typename O> int product_of_few(O *out, const T *x, long long ld_x, const signed char *w, long long ld_w, int dim, ProductArgs a, cudaStream_t st) {
    CUtensorMap mw;
    B2_TRY(make_byte_map(&mw, w, dim, a.channels, ld_w, BM));
    a.row_tiles = 1;
    a.channel_tiles = (unsigned)(((long long)a.channels + BM - 1) / BM);
    const auto kernel = int8_rows_kernel<T, O>;
    B2_TRY(set_max_dynamic_smem((const void *)kernel, rows_smem(80 * 1024 / (ROWS_BN * BK))));
    kernel<<<(long long)a.channel_tiles < sm_count() ? a.channel_tiles : (unsigned)sm_count(), THREADS, rows_smem(a.slabs), st>>>(mw, x, ld_x, dim, out, a);
    count_launch();
    B2_CUDA(cudaGetLastError());
    return B2_OK;
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

int b2_int8_quantize(signed char *q, long long ld_q, float *scales, const void *x, int type, long long rows, int dim, long long ld_x, b2_stream stream) {
    const int e = type_size(type);
    if (!e) { set_error("b2_int8_quantize: unknown element type %d", type); return B2_ERR_BAD_ARG; }
    if (rows < 0 || dim < 1 || dim > (1 << 27)) { set_error("b2_int8_quantize: %lld rows of %d (at most 2^27)", rows, dim); return B2_ERR_BAD_SHAPE; }
    if (ld_q < dim || ld_x < dim || ld_q > MAX_LD || ld_x > MAX_LD) {
        set_error("b2_int8_quantize: leading dimension too small or beyond 2^40 (integers %lld, input %lld for %d columns)", ld_q, ld_x, dim);
        return B2_ERR_BAD_ARG;
    }
    if (!rows) return B2_OK;
    if (!q || !scales || !x) { set_error("b2_int8_quantize: null pointer"); return B2_ERR_BAD_ARG; }
    if (!aligned_to(x, e) || !aligned_to(scales, 4)) { set_error("b2_int8_quantize: the input or the scales are not aligned to their elements"); return B2_ERR_BAD_ARG; }
    return with_type(type, [&](auto *t) { return quantize(q, ld_q, scales, (const B2_ELEM(t) *)x, rows, dim, ld_x, (cudaStream_t)stream); });
}

size_t b2_int8_product_workspace(long long rows, int channels, int dim) {
    if (!sizes_fit(rows, channels, dim)) return 0;
    return (size_t)rows * pitch_of(dim) + (size_t)rows * sizeof(float);
}

int b2_int8_product(void *out, int out_type, long long ld_out, const void *x, int x_type, long long ld_x, const float *x_scales, const signed char *w, long long ld_w,
                    const float *w_scales, const float *bias, long long rows, int channels, int dim, void *workspace, size_t workspace_bytes, b2_stream stream) {
    const int eo = type_size(out_type), ex = x_type == B2_I8 ? 1 : type_size(x_type);
    if (!eo || !ex) { set_error("b2_int8_product: unknown element type %d or %d", out_type, x_type); return B2_ERR_BAD_ARG; }
    if (!sizes_fit(rows, channels, dim)) { set_error("b2_int8_product: %lld rows, %d channels, %d positions (at most 131071)", rows, channels, dim); return B2_ERR_BAD_SHAPE; }
    if (ld_out < channels || ld_x < dim || ld_w < dim || ld_out > MAX_LD || ld_x > (1ll << 39) || ld_w > (1ll << 39)) {      // a tensor map's rows lie up to 2^40 bytes apart
        set_error("b2_int8_product: leading dimension too small or too large (out %lld for %d columns, x %lld and w %lld for %d)", ld_out, channels, ld_x, ld_w, dim);
        return B2_ERR_BAD_ARG;
    }
    if (!rows) return B2_OK;
    if (!out || !x || !w || !w_scales || (x_type == B2_I8 && !x_scales)) { set_error("b2_int8_product: null pointer"); return B2_ERR_BAD_ARG; }
    if (x_type != B2_I8 && x_scales) { set_error("b2_int8_product: scales of rows that are quantised in the call"); return B2_ERR_BAD_ARG; }
    if (!aligned_to(out, eo) || !aligned_to(x, ex) || !aligned_to(x_scales, 4) || !aligned_to(w_scales, 4) || !aligned_to(bias, 4)) {
        set_error("b2_int8_product: a tensor is not aligned to its elements");
        return B2_ERR_BAD_ARG;
    }
    // the distance from a only row to the next
    if (channels == 1) ld_w = (long long)pitch_of(dim);
    if (rows == 1 && x_type == B2_I8) ld_x = (long long)pitch_of(dim);
    if (!aligned_to(w, 16) || ld_w % 16 || (x_type == B2_I8 && (!aligned_to(x, 16) || ld_x % 16))) {
        set_error("b2_int8_product: rows of 8-bit integers that do not start at multiples of 16 bytes");
        return B2_ERR_BAD_ARG;
    }
    ProductArgs a = {};
    a.splits = 1;
    a.x_scales = x_scales; a.w_scales = w_scales; a.bias = bias;
    a.ld_out = ld_out; a.rows = rows; a.channels = channels; a.slabs = (dim + BK - 1) / BK;
    const signed char *xq = (const signed char *)x;
    const cudaStream_t st = (cudaStream_t)stream;
    if (x_type != B2_I8) {
        const size_t need = b2_int8_product_workspace(rows, channels, dim);
        if (!workspace || !aligned_to(workspace, 16)) { set_error("b2_int8_product: the workspace is missing or not aligned to 16 bytes"); return B2_ERR_BAD_ARG; }
        if (workspace_bytes < need) { set_error("b2_int8_product: a workspace of %zu bytes, %zu are needed", workspace_bytes, need); return B2_ERR_BAD_SHAPE; }
        if (few_rows(rows, channels, dim))
            return with_type(x_type, [&](auto *t) {
                const B2_ELEM(t) *in = (const B2_ELEM(t) *)x;
                return with_type(out_type, [&](auto *o) { return product_of_few((B2_ELEM(o) *)out, in, ld_x, w, ld_w, dim, a, st); });
            });
        signed char *q = (signed char *)workspace;
        float *scales = (float *)(q + (size_t)rows * pitch_of(dim));
        B2_TRY(with_type(x_type, [&](auto *t) { return quantize(q, (long long)pitch_of(dim), scales, (const B2_ELEM(t) *)x, rows, dim, ld_x, st); }));
        xq = q;
        ld_x = (long long)pitch_of(dim);
        a.x_scales = scales;
        a.chained = 1;
    }
    return with_type(out_type, [&](auto *t) { return product((B2_ELEM(t) *)out, xq, ld_x, w, ld_w, dim, a, st); });
}

}  // extern "C"
