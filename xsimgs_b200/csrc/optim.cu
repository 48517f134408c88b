// The end of a training step, over many tensors at once, for sm_100a: the
// global gradient norm, clipping by it, and the AdamW update that takes the
// clipped gradient.
//
//   N   = (sum over tensors t and elements i of |g_ti|^p)^(1/p),  p = 2, 1, inf
//   c   = min(1, max_norm / (N + 1e-6)),  g <- c g
//   g'  = c g,  m <- b1 m + (1 - b1) g',  v <- b2 v + (1 - b2) g'^2
//   w   <- w - lr wd w - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// All three are bound by HBM: 4 bytes a float for the norm, 8 more (and the
// first 4 again, where the L2 has lost them) for the scaling, 28 for the
// update.  The tensors travel as a table in the kernel's parameters, so that
// a call copies nothing to the device and can be captured in a graph.  Each
// tensor is cut into tiles.  Blocks (of small tensors, warps) take the tiles
// of all tensors in turn where they are summed, so that the order of every sum
// depends on the tensors' sizes and offsets alone: the same bits on every run.
// Where a second pass writes them, blocks fetch them from a counter; it is
// launched while the first one ends and starts at the tiles that the first one
// read last.
//
// Measured on B200, 6449 GB/s being a copy's rate: norm of 640 M floats
// 351 us (7290 GB/s), of 160 M bf16 51 us (6220); clipping 118 M floats 213 us
// (its three passes of 472 MB: 6650, of which the L2 serves some); the
// clipped update of 118 M floats 567 us (3304 MB and the norm's 472: 6660), of
// 150 M bf16 over masters 693 us (4.5 GB: 6490), of 35 % of 1 M rows of 59
// floats 159 us.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <limits>
#include <type_traits>
#include <vector>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace xsg {
namespace {

constexpr int kOptThreads = 256;
// Blocks of a launch at most: as many as run at once.  More of them keep more
// loads under way, down to the registers that four vectors a thread need (59 M
// floats with each leaf's norm: 3 43.8 us, 4 42.7, 5 41.0, 6 41.6; clipping
// 90 M bf16: 4 80.6, 5 82.5).
constexpr int kNormResident = 5;
constexpr int kScaleResident = 4;
constexpr int kOptBlocks = 148 * kNormResident;
constexpr float kClipEps = 1e-6f;
constexpr int kNormInf = 0;

// ------------------------------------------------------------- elements --
__host__ __device__ constexpr int elem_size(int dtype) { return dtype == XSG_F32 ? 4 : 2; }

__device__ __forceinline__ float load_as(const void* p, int dtype, int64_t i) {
    if (dtype == XSG_F32) return static_cast<const float*>(p)[i];
    if (dtype == XSG_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store_as(void* p, int dtype, int64_t i, float x) {
    if (dtype == XSG_F32) static_cast<float*>(p)[i] = x;
    else if (dtype == XSG_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
    else static_cast<__half*>(p)[i] = __float2half_rn(x);
}

// ---------------------------------------------------------------- tables --
// A tensor is numbered from the line boundary (128 bytes) at or below its
// first element: its elements are the numbers [lead, end) from `base`,
// whatever its offset.  The elements before the next boundary and those after
// the last whole vector go one by one, all others as aligned vectors of which
// a warp's 32 fill whole lines (from 16-byte boundaries, a warp's load spans
// five lines for four, and two warps write parts of one).  Tile k holds
// the numbers [k * tile, (k + 1) * tile); tensor t of a table owns the tiles
// [first[t], first[t + 1]) of the launch.
constexpr int kLine = 128;

struct SpanEntry {
    void* base;
    int64_t end;
    uint8_t lead, dtype;
};

template <int N>
struct SpanTable {
    SpanEntry entry[N];
    int32_t first[N + 1];
    int32_t count;
    int32_t tile_bytes;
    int32_t counters;  // of the launches of a second pass, which this one zeroes (as a
                       // parameter of its own the number costs the host 0.3 us a launch)
};

// The part of tensor t in the tiles [tile, stop): numbers [lo, hi).
struct Part {
    int64_t lo, hi;
};
template <typename Table>
__device__ __forceinline__ Part part_of(const Table& tab, int t, int32_t tile, int32_t stop) {
    const SpanEntry& e = tab.entry[t];
    const int64_t per = tab.tile_bytes >> (e.dtype == XSG_F32 ? 2 : 1);
    return {max(int64_t(e.lead), (tile - tab.first[t]) * per), min(e.end, (stop - tab.first[t]) * per)};
}

// The contiguous run of tiles of block b out of `blocks`, and the block whose
// run holds a tile.
__device__ __forceinline__ int32_t run_start(int32_t tiles, int32_t blocks, int32_t b) {
    return int32_t(int64_t(tiles) * b / blocks);
}
__device__ __forceinline__ int32_t run_of(int32_t tiles, int32_t blocks, int32_t tile) {
    return int32_t(((int64_t(tile) + 1) * blocks - 1) / tiles);
}

// The tensor that owns a tile: the last t with first[t] <= tile (tensors
// without elements own none and are passed over).
template <typename Table>
__device__ __forceinline__ int owner_of(const Table& tab, int32_t tile) {
    int lo = 0, hi = tab.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tab.first[mid] <= tile) lo = mid;
        else hi = mid;
    }
    return lo;
}

// ------------------------------------------------------------ reductions --
// Sums are held in 64 bits: a 32-bit square overflows from 1.8e19 on and is
// lost below 1e-23, and a 32-bit sum over 1e8 entries keeps few digits.  The
// maximum keeps a NaN.
template <int P>
__device__ __forceinline__ double join(double a, double b) {
    if constexpr (P == kNormInf) return (b > a || b != b) ? b : a;
    return a + b;
}

template <int P>
__device__ __forceinline__ double term(float x) {
    if constexpr (P == 2) return double(x) * double(x);
    return fabs(double(x));
}

__device__ __forceinline__ float2 halves(uint32_t u, int dtype) {
    if (dtype == XSG_BF16) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
}

// Adds 16 elements, in `x` as 32 bits.  Their sum is first taken in 32 bits
// (with every element in 64 bits the norm of 160 M bf16 takes 58 us, not 51,
// and of 200 k floats 8.0, not 6.4), and goes on as it is unless squares may
// have left the range in which 32 bits lose nothing: above 2^120, below 2^-96,
// or not finite.  Zeros, which most entries of a sparse gradient are, end
// there.
template <int P, int D>
__device__ __forceinline__ void add16(double& acc, const float (&x)[16]) {
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i & 3] = P == 2 ? fmaf(x[i], x[i], s[i & 3]) : s[i & 3] + fabsf(x[i]);
    const float sum = (s[0] + s[1]) + (s[2] + s[3]);
    const bool safe = D == XSG_F16 || (P == 2 ? sum >= 0x1p-96f && sum <= 0x1p120f : sum <= 0x1p120f);
    if (safe) {
        acc += double(sum);
        return;
    }
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) any |= __float_as_uint(x[i]);
    if ((any << 1) == 0) return;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc += term<P>(x[i]);
}

// Sum (or maximum) over the numbers [lo, hi) of a tensor, by a team of T
// threads (a block or a warp) of which this is number `me`.  kEarly: the data
// need not stay in the L2.
template <int P, int D, int T, bool kEarly>
__device__ __forceinline__ double reduce_part(const void* base, Part part, int me) {
    constexpr int V = 16 / elem_size(D);  // elements of a vector
    constexpr int kUnroll = 4;
    constexpr int L = kLine / elem_size(D);
    const int64_t first = (part.lo + L - 1) / L * (L / V), last = part.hi / V;  // whole vectors
    const uint4* vec = static_cast<const uint4*>(base) + first;
    const int n = int(max(last - first, int64_t(0)));  // a block's part is below 2^31 vectors
    double acc = 0.0;
    [[maybe_unused]] uint32_t top = 0;  // of |x|'s bits: NaN > inf > numbers
    const auto take = [&](const uint4 (&q)[kUnroll]) {
        if constexpr (P == kNormInf) {
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                const uint32_t w[4] = {q[k].x, q[k].y, q[k].z, q[k].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (D == XSG_F32) top = max(top, w[i] & 0x7fffffffu);
                    else top = __vmaxu2(top, w[i] & 0x7fff7fffu);
                }
            }
        } else if constexpr (D == XSG_F32) {
            float x[16];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                x[4 * k] = __uint_as_float(q[k].x), x[4 * k + 1] = __uint_as_float(q[k].y);
                x[4 * k + 2] = __uint_as_float(q[k].z), x[4 * k + 3] = __uint_as_float(q[k].w);
            }
            add16<P, D>(acc, x);
        } else {
#pragma unroll
            for (int k = 0; k < kUnroll; k += 2) {
                float x[16];
                const uint32_t w[8] = {q[k].x, q[k].y, q[k].z, q[k].w, q[k + 1].x, q[k + 1].y, q[k + 1].z, q[k + 1].w};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 f = halves(w[i], D);
                    x[2 * i] = f.x, x[2 * i + 1] = f.y;
                }
                add16<P, D>(acc, x);
            }
        }
    };
    int i = me;
    for (; i + (kUnroll - 1) * T < n; i += kUnroll * T) {
        uint4 q[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) q[k] = kEarly ? __ldcs(vec + i + k * T) : vec[i + k * T];
        take(q);
    }
    if (i < n) {
        uint4 q[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
            q[k] = i + k * T < n ? vec[i + k * T] : make_uint4(0, 0, 0, 0);
        take(q);
    }
    if constexpr (P == kNormInf) {
        const uint32_t one = D == XSG_F32 ? top : max(top & 0xffffu, top >> 16);
        acc = double(D == XSG_F32 ? __uint_as_float(one) : halves(one, D).x);
    }
    // the elements before the first and after the last of these vectors, each fewer than a line's
    const int64_t head = min(first * V, part.hi), tail = max(last * V, head);
    if (head == part.lo && tail == part.hi) return acc;
    for (int j = me; j < 2 * L; j += T) {
        const int64_t odd = j < L ? part.lo + j : tail + j - L;
        if (odd < (j < L ? head : part.hi)) acc = join<P>(acc, term<P>(load_as(base, D, odd)));
    }
    return acc;
}

template <int P, int T, bool kEarly = false, typename Table>
__device__ __forceinline__ double reduce_part(const Table& tab, int t, Part part, int me) {
    const int dtype = tab.entry[t].dtype;
    if (dtype == XSG_F32) return reduce_part<P, XSG_F32, T, kEarly>(tab.entry[t].base, part, me);
    if (dtype == XSG_BF16) return reduce_part<P, XSG_BF16, T, kEarly>(tab.entry[t].base, part, me);
    return reduce_part<P, XSG_F16, T, kEarly>(tab.entry[t].base, part, me);
}

// Over the block, in a fixed order; every thread gets the result.  `smem`
// holds 33 doubles.
template <int P>
__device__ double block_reduce(double v, double* smem) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o; o >>= 1) v = join<P>(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if (lane == 0) smem[warp] = v;
    __syncthreads();
    v = lane < warps ? smem[lane] : 0.0;
#pragma unroll
    for (int o = 16; o; o >>= 1) v = join<P>(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

template <int P>
__device__ __forceinline__ float root(double s) {
    return float(P == 2 ? sqrt(s) : s);
}

__device__ __forceinline__ float clip_coefficient(float norm, float max_norm) {
    const float c = max_norm / (norm + kClipEps);
    return c >= 1.f ? 1.f : c;  // a NaN stays
}

// Partial sums of a launch: sums[b] of all tiles of block b, which takes them
// in turn.  What comes before the last 80 MB is read as data that need not
// stay in the L2 (clipping 118 M floats: 236 us without, 227.5 with 64 to 120
// MB; the second pass finds as much in the L2 as before, 76 MB, so what gains
// is the write-back of the lines that the pass before has left there).
constexpr int64_t kKeptBytes = int64_t(80) << 20;

template <int P, int N>
__global__ void __launch_bounds__(kOptThreads, kNormResident)
    norm_partial_kernel(const __grid_constant__ SpanTable<N> tab, double* __restrict__ sums,
                        unsigned* __restrict__ fetched) {
    __shared__ double smem[33];
    pdl_trigger();
    if (fetched && blockIdx.x == 0)  // the tile counters of the second pass
        for (int i = threadIdx.x; i < tab.counters; i += blockDim.x) fetched[i] = 0;
    const int32_t tiles = tab.first[tab.count];
    double acc = 0.0;
    int t = -1;
    for (int32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        if (t < 0) t = owner_of(tab, tile);
        while (tile >= tab.first[t + 1]) ++t;
        const Part part = part_of(tab, t, tile, tile + 1);
        if (int64_t(tiles - tile) * tab.tile_bytes > kKeptBytes)
            acc = join<P>(acc, reduce_part<P, kOptThreads, true>(tab, t, part, threadIdx.x));
        else
            acc = join<P>(acc, reduce_part<P, kOptThreads>(tab, t, part, threadIdx.x));
    }
    acc = block_reduce<P>(acc, smem);
    if (threadIdx.x == 0) sums[blockIdx.x] = acc;
}

// The same where each tensor's norm is asked for.  A block takes a contiguous
// run of tiles, and slots[b + t] is its part of tensor t: b + t grows along
// the runs, so that no two parts share a slot, and blocks + tensors of them
// are enough.
template <int P, int N>
__global__ void __launch_bounds__(kOptThreads, kNormResident)
    norm_partial_each_kernel(const __grid_constant__ SpanTable<N> tab, double* __restrict__ sums,
                             double* __restrict__ slots) {
    __shared__ double smem[33];
    pdl_trigger();
    const int32_t tiles = tab.first[tab.count], end = run_start(tiles, gridDim.x, blockIdx.x + 1);
    int32_t tile = run_start(tiles, gridDim.x, blockIdx.x);
    // no second pass follows (largest entry of 160 M bf16: 54.8 us, 56.4 without)
    const bool early = int64_t(tiles) * tab.tile_bytes > kKeptBytes;
    double whole = 0.0;
    for (int t = owner_of(tab, tile); tile < end; ++t) {
        const int32_t stop = min(end, tab.first[t + 1]);
        if (stop <= tile) continue;
        // tile by tile, so that the same entries meet in 32 bits as in the kernel above
        double acc = 0.0;
        if (early) {
            for (; tile < stop; ++tile)
                acc = join<P>(acc, reduce_part<P, kOptThreads, true>(tab, t, part_of(tab, t, tile, tile + 1),
                                                                     threadIdx.x));
        } else {
            for (; tile < stop; ++tile)
                acc = join<P>(acc, reduce_part<P, kOptThreads>(tab, t, part_of(tab, t, tile, tile + 1), threadIdx.x));
        }
        acc = block_reduce<P>(acc, smem);
        if (threadIdx.x == 0) slots[blockIdx.x + t] = acc;
        whole = join<P>(whole, acc);
    }
    if (threadIdx.x == 0) sums[blockIdx.x] = whole;
}

// All partial sums of a call, by every block for itself.  (The first pass may
// still run when a kernel that reads them starts: plain loads, after pdl_wait.)
template <int P>
__device__ __forceinline__ float total_norm(const double* sums, int n, double* smem) {
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) v = join<P>(v, __ldcg(sums + i));
    return root<P>(block_reduce<P>(v, smem));
}

// Block 0: the norm of all tensors (if `norm`).  The others: a tensor each.
template <int P, int N>
__global__ void __launch_bounds__(kOptThreads)
    norm_finish_kernel(const __grid_constant__ SpanTable<N> tab, int blocks, const double* sums,
                       int n_sums, const double* slots, float* __restrict__ norm,
                       float* __restrict__ norms) {
    __shared__ double smem[33];
    pdl_wait();
    if (blockIdx.x == 0) {
        if (!norm) return;
        const float v = total_norm<P>(sums, n_sums, smem);
        if (threadIdx.x == 0) *norm = v;
        return;
    }
    const int t = blockIdx.x - 1;
    const int32_t tiles = tab.first[tab.count], begin = tab.first[t], end = tab.first[t + 1];
    float v = 0.f;
    if (end > begin) {
        const int b0 = run_of(tiles, blocks, begin), b1 = run_of(tiles, blocks, end - 1);
        v = total_norm<P>(slots + b0 + t, b1 - b0 + 1, smem);
    }
    if (threadIdx.x == 0) norms[t] = v;
}

// g <- c g over the numbers [lo, hi) of a tensor, by a team of T threads, from
// the end to the start.  The product is taken in 32 bits and rounded once to g's type.
template <int D>
__device__ __forceinline__ uint32_t scaled(uint32_t w, float c) {
    if constexpr (D == XSG_F32) return __float_as_uint(__uint_as_float(w) * c);
    const float2 f = halves(w, D);
    uint32_t r;
    if constexpr (D == XSG_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f.x * c, f.y * c);
        memcpy(&r, &h, 4);
    } else {
        const __half2 h = __floats2half2_rn(f.x * c, f.y * c);
        memcpy(&r, &h, 4);
    }
    return r;
}

template <int D, int T>
__device__ __forceinline__ void scale_part(void* base, Part part, float c, int me) {
    constexpr int V = 16 / elem_size(D);
    constexpr int kUnroll = 4, kStep = kUnroll * T;
    constexpr int L = kLine / elem_size(D);
    const int64_t first = (part.lo + L - 1) / L * (L / V), last = part.hi / V;
    uint4* vec = static_cast<uint4*>(base) + first;
    const int n = int(max(last - first, int64_t(0)));  // a block's part is below 2^31 vectors
    int i = n / kStep * kStep + me;
    for (int j = i; j < n; j += T) {
        const uint4 q = vec[j];
        vec[j] = make_uint4(scaled<D>(q.x, c), scaled<D>(q.y, c), scaled<D>(q.z, c), scaled<D>(q.w, c));
    }
    for (i -= kStep; i >= 0; i -= kStep) {
        uint4 q[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) q[k] = vec[i + k * T];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
            vec[i + k * T] =
                make_uint4(scaled<D>(q[k].x, c), scaled<D>(q[k].y, c), scaled<D>(q[k].z, c), scaled<D>(q[k].w, c));
    }
    const int64_t head = min(first * V, part.hi), tail = max(last * V, head);
    if (head == part.lo && tail == part.hi) return;
    for (int j = me; j < 2 * L; j += T) {
        const int64_t odd = j < L ? part.lo + j : tail + j - L;
        if (odd < (j < L ? head : part.hi)) store_as(base, D, odd, load_as(base, D, odd) * c);
    }
}

template <int T, typename Table>
__device__ __forceinline__ void scale_part(const Table& tab, int t, Part part, float c, int me) {
    const int dtype = tab.entry[t].dtype;
    if (dtype == XSG_F32) scale_part<XSG_F32, T>(tab.entry[t].base, part, c, me);
    else if (dtype == XSG_BF16) scale_part<XSG_BF16, T>(tab.entry[t].base, part, c, me);
    else scale_part<XSG_F16, T>(tab.entry[t].base, part, c, me);
}

// The second pass of clipping.  c = 1 leaves the data alone.  The tiles are
// taken from the last to the first, so that what the first pass read last, and
// the L2 still holds, comes first.  A block fetches the next tile while it
// works on one: the reads and writes then go through the memory in order,
// with the blocks out of step, which HBM likes better than blocks that take
// every 592nd tile (clipping 118 M floats: 214 us against 227, 90 M bf16 78.9
// against 80.9) or a block for each tile (216.5, and 4 us more where nothing
// has to be scaled).  Which block has which tile changes no result.
template <int P, int N>
__global__ void __launch_bounds__(kOptThreads, kScaleResident)
    clip_scale_kernel(const __grid_constant__ SpanTable<N> tab, const double* sums, int n_sums,
                      float max_norm, float* __restrict__ norm, unsigned* fetched) {
    __shared__ double smem[33];
    __shared__ int32_t next[2];
    pdl_wait();
    const float total = total_norm<P>(sums, n_sums, smem);
    if (blockIdx.x == 0 && threadIdx.x == 0 && norm) *norm = total;
    const float c = clip_coefficient(total, max_norm);
    if (c == 1.f) return;
    const int32_t tiles = tab.first[tab.count];
    if (threadIdx.x == 0) next[0] = int32_t(atomicAdd(fetched, 1u));
    __syncthreads();
    int t = -1;
    for (int turn = 0; next[turn] < tiles; turn ^= 1) {
        const int32_t tile = tiles - 1 - next[turn];
        if (threadIdx.x == 0) next[turn ^ 1] = int32_t(atomicAdd(fetched, 1u));
        if (t < 0) t = owner_of(tab, tile);
        while (tile < tab.first[t]) --t;
        scale_part<kOptThreads>(tab, t, part_of(tab, t, tile, tile + 1), c, threadIdx.x);
        __syncthreads();
    }
}

// --------------------------------------------------------- small tensors --
// What a few SMs read in one round of loads goes in one launch: a cluster of
// blocks whose warps each take small tiles, so that all loads are under way
// at once; the blocks' sums meet over the cluster's shared memory.  Bound by
// the launch and the latency of its few dependent steps.
constexpr int kSmallThreads = 1024;
constexpr int kSmallBlocks = 8;
constexpr int kSmallSpans = 32;
constexpr int kSmallTile = 4096;  // bytes: eight vectors a lane

// A block's sums, where the others of the cluster read them.
struct ClusterSums {
    double whole;
    double each[kSmallSpans];
    double warp[33];
};

// This warp among the cluster's.
struct Worker {
    int id, count, lane;
};
__device__ __forceinline__ Worker worker_of(const cg::cluster_group& cluster) {
    const int warps = int(blockDim.x >> 5);
    return {int(cluster.block_rank()) * warps + int(threadIdx.x >> 5), int(cluster.num_blocks()) * warps,
            int(threadIdx.x & 31)};
}

// body(t, tile) for the tiles of a worker, in turn.
template <typename Table, typename F>
__device__ __forceinline__ void for_tiles(const Table& tab, int32_t first, int32_t step, F&& body) {
    const int32_t tiles = tab.first[tab.count];
    int t = -1;
    for (int32_t tile = first; tile < tiles; tile += step) {
        if (t < 0) t = owner_of(tab, tile);
        while (tile >= tab.first[t + 1]) ++t;
        body(t, tile);
    }
}

// Over the cluster, in the order of the ranks; every thread gets it.
template <int P>
__device__ __forceinline__ double cluster_join(cg::cluster_group& cluster, double* mine) {
    double v = 0.0;
    for (unsigned r = 0; r < cluster.num_blocks(); ++r) v = join<P>(v, *cluster.map_shared_rank(mine, r));
    return v;
}

// The norm of all tensors, for every thread of the cluster.
template <int P>
__device__ __forceinline__ float cluster_norm(const SpanTable<kSmallSpans>& tab, cg::cluster_group& cluster,
                                              ClusterSums& sums) {
    const Worker w = worker_of(cluster);
    double acc = 0.0;
    for_tiles(tab, w.id, w.count, [&](int t, int32_t tile) {
        acc = join<P>(acc, reduce_part<P, 32>(tab, t, part_of(tab, t, tile, tile + 1), w.lane));
    });
    acc = block_reduce<P>(acc, sums.warp);
    if (cluster.num_blocks() == 1) return root<P>(acc);
    if (threadIdx.x == 0) sums.whole = acc;
    cluster.sync();
    const float total = root<P>(cluster_join<P>(cluster, &sums.whole));
    cluster.sync();  // the others' sums stay until all have read them
    return total;
}

template <int P>
__global__ void __launch_bounds__(kSmallThreads)
    norm_small_kernel(const __grid_constant__ SpanTable<kSmallSpans> tab, float* __restrict__ norm) {
    __shared__ ClusterSums sums;
    cg::cluster_group cluster = cg::this_cluster();
    const float total = cluster_norm<P>(tab, cluster, sums);
    if (cluster.block_rank() == 0 && threadIdx.x == 0) *norm = total;
}

// With each tensor's norm: a warp adds its tile's sum to its own row.
template <int P>
__global__ void __launch_bounds__(kSmallThreads)
    norm_small_each_kernel(const __grid_constant__ SpanTable<kSmallSpans> tab, float* __restrict__ norm,
                           float* __restrict__ norms) {
    __shared__ ClusterSums sums;
    __shared__ double rows[kSmallThreads / 32][kSmallSpans];
    cg::cluster_group cluster = cg::this_cluster();
    const Worker w = worker_of(cluster);
    double* row = rows[threadIdx.x >> 5];
    row[w.lane] = 0.0;
    __syncwarp();
    for_tiles(tab, w.id, w.count, [&](int t, int32_t tile) {
        double v = reduce_part<P, 32>(tab, t, part_of(tab, t, tile, tile + 1), w.lane);
#pragma unroll
        for (int o = 16; o; o >>= 1) v = join<P>(v, __shfl_xor_sync(0xffffffffu, v, o));
        if (w.lane == 0) row[t] = join<P>(row[t], v);
    });
    __syncthreads();
    if (threadIdx.x < 32) {
        double each = 0.0;
        for (int r = 0; r < int(blockDim.x >> 5); ++r) each = join<P>(each, rows[r][threadIdx.x]);
        sums.each[threadIdx.x] = each;
    }
    cluster.sync();
    if (cluster.block_rank() == 0 && threadIdx.x < 32) {
        double v = cluster_join<P>(cluster, &sums.each[threadIdx.x]);
        if (int(threadIdx.x) < tab.count) norms[threadIdx.x] = root<P>(v);
#pragma unroll
        for (int o = 16; o; o >>= 1) v = join<P>(v, __shfl_xor_sync(0xffffffffu, v, o));
        if (threadIdx.x == 0) *norm = root<P>(v);
    }
    cluster.sync();
}

template <int P>
__global__ void __launch_bounds__(kSmallThreads)
    clip_small_kernel(const __grid_constant__ SpanTable<kSmallSpans> tab, float max_norm, float* __restrict__ norm) {
    __shared__ ClusterSums sums;
    cg::cluster_group cluster = cg::this_cluster();
    const float total = cluster_norm<P>(tab, cluster, sums);
    if (cluster.block_rank() == 0 && threadIdx.x == 0) *norm = total;
    const float c = clip_coefficient(total, max_norm);
    if (c == 1.f) return;
    // the tiles that this warp has read, and no other
    const Worker w = worker_of(cluster);
    for_tiles(tab, w.id, w.count, [&](int t, int32_t tile) {
        scale_part<32>(tab, t, part_of(tab, t, tile, tile + 1), c, w.lane);
    });
}

// ----------------------------------------------------------------- AdamW --
// Bound by HBM: 16 bytes a lane from each of four arrays are under way in five
// blocks an SM.  Moments and arithmetic are in 32 bits; w is rounded once to a
// 16-bit parameter's type.
constexpr int kAdamLine = 64;     // elements: whole lines for every type
// Blocks an SM: more have too few registers, fewer too few loads under way
// (150 M bf16 over masters: 4 728 us, 5 699, 6 737; 118 M floats, clipped: 3
// 610 us, 4 574, 5 571, 6 608; 1 M masked rows: 4 171 us, 5 158, 6 161).
constexpr int kAdamResident = 5;
// Elements of a tile at most: without row masks (150 M bf16 over masters: 4096
// 699 us, 8192 710), and with them, where each of a block's eight warps goes
// through a stretch of 1024 (1 M masked rows: 4096 201 us, 8192 158, 16384 171).
constexpr int32_t kAdamTile = 4096, kRowsTile = 8192;
constexpr int kAdamGroups = 32;

struct AdamHyper {
    float beta1, rest1, beta2, rest2, lr, lr_decay, eps;  // rest = 1 - beta, lr_decay = lr * weight decay
    float log_beta1, log_beta2;
};

// Elements are numbered from `lead` on, as above, in vectors of four; the
// pointers are those of number 0, which is a multiple of 64 elements for the
// parameter.  All arrays of a tensor have to be as far past a multiple of
// four elements for that (`vec`); where they are not, lead is 0 and elements
// go one by one.
struct AdamEntry {
    void* param;
    const void* grad;
    float* exp_avg;
    float* exp_avg_sq;
    float* master;
    const uint8_t* rows;
    int64_t end;
    int32_t row_size;
    uint32_t row_magic;  // 2^31 / row_size, rounded up
    uint8_t lead, vec, group, param_dtype, grad_dtype;
};

template <int N>
struct AdamTable {
    AdamEntry entry[N];
    int32_t first[N + 1];
    int32_t count;
    int32_t tile;  // elements
    AdamHyper hyper[kAdamGroups];
};

struct AdamCall {
    unsigned long long* step;  // [0] updates taken, [1] blocks that are done, modulo the launch's
    unsigned* fetched;         // tiles fetched (behind a norm, which zeroes it)
    const double* sums;        // the gradients' partial sums, or null
    int32_t n_sums;
    int32_t advance;      // the call's last launch counts the update
    int32_t clip;
    int32_t skip_nonfinite;
    float max_norm;
    float* norm;
};

struct AdamScale {
    float c, beta1, rest1, beta2, rest2, lr_decay, eps, step_size, root_scale;
};

__device__ __forceinline__ void adam_element(const AdamScale& h, float g, float& m, float& v, float& w) {
    g *= h.c;
    m = fmaf(h.beta1, m, h.rest1 * g);
    v = fmaf(h.beta2, v, h.rest2 * g * g);
    w = fmaf(-h.lr_decay, w, w);
    const float den = fmaf(sqrtf(v), h.root_scale, h.eps);
    // A moment whose gradients have long been zero stays among the subnormal
    // numbers, on which a division takes a slow path (59 M of them: 326 us
    // against 272); a product does not.  The reciprocal is exact to half an
    // ulp and finite from 2^-126 on; the limit leaves that a wide margin, and
    // only an eps below 1e-30 lets a denominator under it.
    const float q = den >= 0x1p-100f ? m * __frcp_rn(den) : m / den;
    w -= h.step_size * q;
}

__device__ __forceinline__ void load4(float (&x)[4], const void* p, int dtype, int64_t i) {
    if (dtype == XSG_F32) {
        const float4 q = static_cast<const float4*>(p)[i];
        x[0] = q.x, x[1] = q.y, x[2] = q.z, x[3] = q.w;
    } else {
        const uint2 q = static_cast<const uint2*>(p)[i];
        const float2 a = halves(q.x, dtype), b = halves(q.y, dtype);
        x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
    }
}

__device__ __forceinline__ void store4(void* p, int dtype, int64_t i, const float (&x)[4]) {
    if (dtype == XSG_F32) {
        static_cast<float4*>(p)[i] = make_float4(x[0], x[1], x[2], x[3]);
    } else if (dtype == XSG_BF16) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
        uint2 q;
        memcpy(&q.x, &a, 4);
        memcpy(&q.y, &b, 4);
        static_cast<uint2*>(p)[i] = q;
    } else {
        const __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
        uint2 q;
        memcpy(&q.x, &a, 4);
        memcpy(&q.y, &b, 4);
        static_cast<uint2*>(p)[i] = q;
    }
}

// The update over the numbers [lo, hi) of a tensor, by a team of T threads.  kF32: all
// arrays are in 32 bits and there is no master, so no branch on the types
// stands between the loads.
template <bool kF32>
struct AdamAt {
    const AdamEntry& e;
    const AdamScale& h;

    __device__ __forceinline__ int param_dtype() const { return kF32 ? XSG_F32 : e.param_dtype; }
    __device__ __forceinline__ int grad_dtype() const { return kF32 ? XSG_F32 : e.grad_dtype; }
    __device__ __forceinline__ float* master() const { return kF32 ? nullptr : e.master; }

    // Element i.
    __device__ __forceinline__ void one(int64_t i) const {
        float m = e.exp_avg[i], v = e.exp_avg_sq[i];
        float w = master() ? master()[i] : load_as(e.param, param_dtype(), i);
        adam_element(h, load_as(e.grad, grad_dtype(), i), m, v, w);
        e.exp_avg[i] = m;
        e.exp_avg_sq[i] = v;
        if (master()) master()[i] = w;
        store_as(e.param, param_dtype(), i, w);
    }
    struct Four {
        float w[4], g[4], m[4], v[4];
    };
    // Vector i; `keep` has a bit for each of its elements that is updated.
    __device__ __forceinline__ void load(Four& x, int64_t i) const {
        load4(x.g, e.grad, grad_dtype(), i);
        load4(x.m, e.exp_avg, XSG_F32, i);
        load4(x.v, e.exp_avg_sq, XSG_F32, i);
        if (master()) load4(x.w, master(), XSG_F32, i);
        else load4(x.w, e.param, param_dtype(), i);
    }
    __device__ __forceinline__ void update(Four& x, int64_t i, uint32_t keep) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float m = x.m[j], v = x.v[j], w = x.w[j];
            adam_element(h, x.g[j], m, v, w);
            if (keep >> j & 1) x.m[j] = m, x.v[j] = v, x.w[j] = w;
        }
        store4(e.exp_avg, XSG_F32, i, x.m);
        store4(e.exp_avg_sq, XSG_F32, i, x.v);
        if (master()) store4(master(), XSG_F32, i, x.w);
        if (keep == 15u || (!master() && param_dtype() == XSG_F32)) {
            store4(e.param, param_dtype(), i, x.w);
        } else {
            // a row that is passed over keeps its parameter's bits, whatever its master says
            for (int j = 0; j < 4; ++j)
                if (keep >> j & 1) store_as(e.param, param_dtype(), 4 * i + j, x.w[j]);
        }
    }
};

// Rows of a part's elements: of its first by a 64-bit division, of the others
// from their distance x to that row's start.  x is below the row's size plus
// a tile's 8192 + 64 elements: below twice the size of rows of 16384 and more,
// and exact by the multiplication for shorter ones (x * size < 2^31).
struct RowsAt {
    const uint8_t* rows;
    uint32_t size, rem, magic;

    __device__ __forceinline__ RowsAt(const AdamEntry& e, int64_t element)
        : size(uint32_t(e.row_size)), magic(e.row_magic) {
        const int64_t row = element / e.row_size;
        rows = e.rows + row;
        rem = uint32_t(element - row * e.row_size);
    }
    __device__ __forceinline__ uint32_t row(uint32_t x) const {
        return size >= 16384u ? uint32_t(x >= size) : uint32_t((uint64_t(x) * magic) >> 31);
    }
    // Whether the element at a distance from the first is updated.
    __device__ __forceinline__ bool keeps(uint32_t distance) const { return rows[row(rem + distance)] != 0; }
    // The same for four elements from there on, as bits.
    __device__ __forceinline__ uint32_t keeps4(uint32_t distance) const {
        const uint32_t x = rem + distance, r = row(x);
        if (size >= 3u) {  // two rows at most
            const uint32_t left = (r + 1u) * size - x;  // of row r
            const uint32_t a = rows[r] ? 15u : 0u;
            if (left >= 4u) return a;
            const uint32_t mask = (1u << left) - 1u;
            return (a & mask) | (rows[r + 1u] ? 15u & ~mask : 0u);
        }
        uint32_t k = 0;
#pragma unroll
        for (uint32_t j = 0; j < 4u; ++j) k |= rows[size == 1u ? x + j : (x + j) >> 1] ? 1u << j : 0u;
        return k;
    }
};

template <bool kF32, bool kRows, int T>
__device__ __forceinline__ void adam_part(const AdamEntry& e, Part part, const AdamScale& h, int me) {
    const AdamAt<kF32> at{e, h};
    if (kRows && e.rows) {
        const RowsAt rows(e, part.lo - e.lead);
        if (!e.vec) {
            for (int64_t i = part.lo + me; i < part.hi; i += T)
                if (rows.keeps(uint32_t(i - part.lo))) at.one(i);
            return;
        }
        constexpr int L = kAdamLine;
        const int64_t first = (part.lo + L - 1) / L * (L / 4), last = part.hi / 4;
        const int n = int(max(last - first, int64_t(0)));
        const uint32_t skip = uint32_t(4 * first - part.lo);
        constexpr int kRowsWarps = T == 32 ? kSmallThreads / 32 : T / 32;
        // Each warp lists the vectors of a stretch that have something to
        // update, and then goes through the list with all lanes at work.
        constexpr int kStretch = 8 * 32;
        __shared__ uint16_t lists[kRowsWarps][kStretch];
        uint16_t* list = lists[threadIdx.x >> 5];
        const int lane = int(threadIdx.x & 31);
        for (int base = me / 32 * kStretch; base < n; base += T / 32 * kStretch) {
            int count = 0;
#pragma unroll
            for (int k = 0; k < kStretch; k += 32) {
                const int j = base + k + lane;
                const uint32_t keep = j < n ? rows.keeps4(skip + 4u * uint32_t(j)) : 0u;
                const uint32_t some = __ballot_sync(0xffffffffu, keep != 0u);
                if (keep) list[count + __popc(some & ((1u << lane) - 1u))] = uint16_t((k + lane) << 4 | keep);
                count += __popc(some);
            }
            __syncwarp();
            for (int q = lane; q < count; q += 32) {
                const uint32_t entry = list[q];
                const int64_t i = first + base + (entry >> 4);
                typename AdamAt<kF32>::Four x;
                at.load(x, i);
                at.update(x, i, entry & 15u);
            }
            __syncwarp();
        }
        const int64_t head = min(first * 4, part.hi), tail = max(last * 4, head);
        if (head == part.lo && tail == part.hi) return;
        for (int j = me; j < 2 * L; j += T) {
            const int64_t odd = j < L ? part.lo + j : tail + j - L;
            if (odd < (j < L ? head : part.hi) && rows.keeps(uint32_t(odd - part.lo))) at.one(odd);
        }
        return;
    }
    if (!e.vec) {
        for (int64_t i = part.lo + me; i < part.hi; i += T) at.one(i);
        return;
    }
    constexpr int L = kAdamLine;
    const int64_t first = (part.lo + L - 1) / L * (L / 4), last = part.hi / 4;
    const int n = int(max(last - first, int64_t(0)));
    for (int j = me; j < n; j += T) {
        typename AdamAt<kF32>::Four x;
        at.load(x, first + j);
        at.update(x, first + j, 15u);
    }
    const int64_t head = min(first * 4, part.hi), tail = max(last * 4, head);
    if (head == part.lo && tail == part.hi) return;
    for (int j = me; j < 2 * L; j += T) {
        const int64_t odd = j < L ? part.lo + j : tail + j - L;
        if (odd < (j < L ? head : part.hi)) at.one(odd);
    }
}

// The options of a tensor's group at this step.
__device__ __forceinline__ void set_group(AdamScale& h, const AdamHyper& y, float steps) {
    h.beta1 = y.beta1, h.rest1 = y.rest1, h.beta2 = y.beta2, h.rest2 = y.rest2;
    h.lr_decay = y.lr_decay, h.eps = y.eps;
    // 1 - b^t without the cancellation of 1 - pow(b, t)
    h.step_size = y.lr / -expm1f(steps * y.log_beta1);
    h.root_scale = rsqrtf(-expm1f(steps * y.log_beta2));
}

// One tile of tensor t, by a team of T threads.
template <bool kF32, bool kRows, int T, typename Table>
__device__ __forceinline__ void adam_tile(const Table& tab, int t, int32_t tile, const AdamScale& h, int me) {
    const AdamEntry& e = tab.entry[t];
    const int64_t at = int64_t(tile - tab.first[t]) * tab.tile;
    adam_part<kF32, kRows, T>(e, {max(int64_t(e.lead), at), min(e.end, at + tab.tile)}, h, me);
}

// Behind a norm, blocks fetch tiles as in clipping, from the last to the first.
// Every block fetches one past the last; the last of them to do so counts the
// update, when all blocks that have had a tile have long read step[0].  The
// counter is in the call's scratch, where the norm's pass zeroes it.  A call
// without a norm has no scratch and nothing in the L2 to meet: a block for each
// tile (118 M floats: 495 us, 494 with a counter; 1.4 M floats:
// 8.2 us, 11.2), under row masks, which cost more to set out on, 740 blocks that
// take tiles in turn (1 M rows, 35 % seen: 158.7 us, 157.8 with a counter; 200 k
// rows: 41.5, 42.0).  There the last block to be done counts the update, by
// step[1] modulo the number of blocks: if that word is not zero, blocks count
// too early, but each tile is still updated once.
template <int N, bool kF32, bool kRows>
__global__ void __launch_bounds__(kOptThreads, kAdamResident)
    adamw_kernel(const __grid_constant__ AdamTable<N> tab, const __grid_constant__ AdamCall call) {
    __shared__ double smem[33];
    __shared__ uint32_t next[2];
    AdamScale h;
    h.c = 1.f;
    if (call.sums) {
        pdl_wait();
        const float total = total_norm<2>(call.sums, call.n_sums, smem);
        if (blockIdx.x == 0 && threadIdx.x == 0 && call.norm) *call.norm = total;
        if (call.skip_nonfinite && !isfinite(total)) return;  // every block alike: nothing changes
        if (call.clip) h.c = clip_coefficient(total, call.max_norm);
    }
    const float steps = float(call.step[0] + 1);
    const uint32_t tiles = uint32_t(tab.first[tab.count]);
    const auto fetch = [&](uint32_t before) {
        return call.fetched ? atomicAdd(call.fetched, 1u) : before + gridDim.x;
    };
    if (threadIdx.x == 0) next[0] = call.fetched ? fetch(0) : blockIdx.x;
    __syncthreads();
    int t = -1, turn = 0;
    for (; next[turn] < tiles; turn ^= 1) {
        const int32_t tile = int32_t(tiles - 1u - next[turn]);
        if (threadIdx.x == 0) next[turn ^ 1] = fetch(next[turn]);
        if (t < 0 || tile < tab.first[t]) {
            if (t < 0) t = owner_of(tab, tile);
            while (tile < tab.first[t]) --t;
            set_group(h, tab.hyper[tab.entry[t].group], steps);
        }
        adam_tile<kF32, kRows, kOptThreads>(tab, t, tile, h, threadIdx.x);
        __syncthreads();
    }
    if (threadIdx.x == 0 && call.advance) {
        const bool last = call.fetched ? next[turn] == tiles + gridDim.x - 1u
                                       : atomicInc(reinterpret_cast<unsigned*>(call.step + 1), gridDim.x - 1u) ==
                                             gridDim.x - 1u;
        if (last) atomicAdd(call.step, 1ull);
    }
}

// Norm and update of small tensors in one launch (see norm_small_kernel).
template <bool kF32>
__global__ void __launch_bounds__(kSmallThreads)
    adamw_small_kernel(const __grid_constant__ SpanTable<kSmallSpans> grads,
                       const __grid_constant__ AdamTable<kSmallSpans> tab, const __grid_constant__ AdamCall call) {
    __shared__ ClusterSums sums;
    cg::cluster_group cluster = cg::this_cluster();
    const float steps = float(call.step[0] + 1);
    const float total = cluster_norm<2>(grads, cluster, sums);
    const bool first = cluster.block_rank() == 0 && threadIdx.x == 0;
    if (first && call.norm) *call.norm = total;
    if (call.skip_nonfinite && !isfinite(total)) return;
    AdamScale h;
    h.c = call.clip ? clip_coefficient(total, call.max_norm) : 1.f;
    const Worker w = worker_of(cluster);
    int group_of = -1;
    for_tiles(tab, w.id, w.count, [&](int t, int32_t tile) {
        if (t != group_of) set_group(h, tab.hyper[tab.entry[t].group], steps);
        group_of = t;
        adam_tile<kF32, true, 32>(tab, t, tile, h, w.lane);
    });
    if (first) atomicAdd(call.step, 1ull);  // all have read it before the norm's barriers
}

// ------------------------------------------------------------------ host --
constexpr int kSpans = 1024;
constexpr int kAdamSpans = 380;
static_assert(sizeof(SpanTable<kSpans>) <= 32000 && sizeof(AdamTable<kAdamSpans>) + sizeof(AdamCall) <= 32000,
              "kernel parameters hold 32764 bytes");
// One launch of a cluster up to these sizes, two of the whole GPU above, which
// cost the host one launch more and have all SMs' loads and stores.  Norm:
// 4.3 us against 6.8 at 14 k floats, 6.2 against 7.3 at 140 k, 6.4 (two) at
// 280 k.  Clipping: 5.1 against 6.4 at 1 k floats, 6.2 against 6.8 at 14 k,
// 8.2 against 6.6 at 28 k.  Clipped update: 6.7 us against 8.5 at 420 floats,
// 8.5 and 8.5 at 2 k, 10.2 against 8.5 at 4 k.
constexpr int64_t kSmallNormBytes = 1 << 20;
constexpr int64_t kSmallClipBytes = 1 << 16;
constexpr int64_t kSmallAdamElems = 1 << 11;
constexpr int32_t kSmallAdamTile = 256;  // elements, a warp's: two vectors a lane

bool small_norm(int64_t n_spans, int64_t bytes) { return n_spans <= kSmallSpans && bytes <= kSmallNormBytes; }
bool small_clip(int64_t n_spans, int64_t bytes) { return n_spans <= kSmallSpans && bytes <= kSmallClipBytes; }
bool small_adamw(int64_t n_spans, int64_t elems) { return n_spans <= kSmallSpans && elems <= kSmallAdamElems; }

// The smallest tile that leaves each block one, up to `most`.
int32_t tile_for(int64_t size, int32_t least, int32_t most, int64_t blocks) {
    while (least < most && size > least * blocks) least *= 2;
    return least;
}

template <typename T>
struct Same {
    using type = T;
};

// A launch by reference: the tables are copied once, by the driver.
template <typename... P>
void launch_table(void (*kernel)(P...), unsigned grid, unsigned block, unsigned cluster, bool pdl, cudaStream_t st,
                  const typename Same<P>::type&... args) {
    count_launch();
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    if (cluster > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim = {cluster, 1, 1};
        ++cfg.numAttrs;
    }
    if (pdl) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        ++cfg.numAttrs;
    }
    void* pointers[] = {const_cast<void*>(static_cast<const void*>(&args))...};
    (void)cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(kernel), pointers);  // errors surface in check_launch
}

bool known_dtype(int d) { return d == XSG_F32 || d == XSG_BF16 || d == XSG_F16; }

constexpr int64_t kMaxElems = int64_t(1) << 40;  // keeps tile numbers inside 31 bits

int check_spans(const xsg_span* spans, int64_t n, const char* what) {
    XSG_REQUIRE(n > 0 && spans, std::string(what) + ": at least one tensor is needed");
    int64_t total = 0;
    for (int64_t i = 0; i < n; ++i) {
        XSG_REQUIRE(known_dtype(spans[i].dtype), std::string(what) + ": unknown element type");
        XSG_REQUIRE(spans[i].n >= 0 && spans[i].n < kMaxElems - total, std::string(what) + ": bad element count");
        total += spans[i].n;
        XSG_REQUIRE(spans[i].n == 0 || spans[i].data, std::string(what) + ": null pointer");
        XSG_REQUIRE(reinterpret_cast<uintptr_t>(spans[i].data) % elem_size(spans[i].dtype) == 0,
                    std::string(what) + ": misaligned pointer");
    }
    return XSG_OK;
}

// The words of a call that are no tensors: norms, the counter (64 bits), and
// the scratch, which begins with sums in 64 bits.
bool aligned(const void* p, size_t size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

int check_words(const float* norm, const float* norms, const int64_t* step, const Arena& arena, const char* what) {
    XSG_REQUIRE(aligned(norm, sizeof(float)) && aligned(norms, sizeof(float)), std::string(what) + ": misaligned norm");
    XSG_REQUIRE(aligned(step, sizeof(int64_t)), std::string(what) + ": misaligned step counter");
    XSG_REQUIRE(aligned(arena.base, sizeof(double)), std::string(what) + ": misaligned workspace");
    return XSG_OK;
}

// The tensors of one launch.
template <int N>
struct SpanLaunch {
    SpanTable<N> tab;
    int blocks = 0;
    int64_t first_span = 0, sums_at = 0, slots_at = 0, bytes = 0;

    void add(const void* data, int64_t n, int dtype) {
        SpanEntry& e = tab.entry[tab.count++];
        const auto at = reinterpret_cast<uintptr_t>(data);
        e.base = reinterpret_cast<void*>(at - at % kLine);
        e.lead = uint8_t(at % kLine / elem_size(dtype));
        e.end = e.lead + n;
        e.dtype = uint8_t(dtype);
        bytes += n * elem_size(dtype);
    }
    // The tiles, when all tensors are in.
    int32_t cut(int32_t tile_bytes) {
        tab.tile_bytes = tile_bytes;
        int64_t tiles = 0;
        for (int t = 0; t < tab.count; ++t) {
            const SpanEntry& e = tab.entry[t];
            const int64_t per = tile_bytes / elem_size(e.dtype);
            tab.first[t] = int32_t(tiles);
            tiles += e.end > e.lead ? (e.end + per - 1) / per : 0;
        }
        tab.first[tab.count] = int32_t(tiles);
        return int32_t(tiles);
    }
    void close(int64_t& sums, int64_t& slots) {
        // clipping 90 M bf16 in 201 tensors: 73 us with tiles of 32 KB, 77 of 16; 118 M floats: 213, 217
        blocks = std::max(1, std::min(cut(tile_for(bytes, 4096, 32768, kOptBlocks)), kOptBlocks));
        sums_at = sums;
        sums += blocks;
        slots_at = slots;
        slots += blocks + tab.count;
    }
    SpanLaunch() { tab.count = tab.counters = 0; }
};

size_t sums_count(int64_t n_spans) { return size_t((n_spans + kSpans - 1) / kSpans) * kOptBlocks; }
size_t slots_count(int64_t n_spans) { return sums_count(n_spans) + size_t(n_spans); }

// Tile counters, one for each launch of a second pass: an update's takes
// kAdamGroups tensors at least unless it is the last, clipping's more.
static_assert(kAdamGroups <= kSmallSpans && kAdamGroups <= kSpans && kAdamGroups <= kAdamSpans, "counters_count");
int64_t counters_count(int64_t n_spans) { return n_spans / kAdamGroups + 1; }

// All launches over `n` tensors, tensor i from get(i): one of a small table
// where that holds them, else as many of the large table as it takes.
template <int N>
struct SpanPlan {
    std::vector<SpanLaunch<N>> launches;
    int64_t sums = 0, slots = 0;

    template <typename Get>
    SpanPlan(int64_t n, Get&& get) : launches((n + N - 1) / N) {
        for (int64_t i = 0; i < n; ++i) {
            SpanLaunch<N>& L = launches[i / N];
            if (L.tab.count == 0) L.first_span = i;
            get(i, L);
        }
        for (auto& L : launches) L.close(sums, slots);
        launches[0].tab.counters = int32_t(counters_count(n));
    }

    int64_t bytes() const { return launches[0].bytes; }

    template <int P>
    void partials(double* sums_at, double* slots_at, unsigned* fetched, cudaStream_t st) const {
        for (size_t l = 0; l < launches.size(); ++l) {
            const auto& L = launches[l];
            if (slots_at)
                launch_table(norm_partial_each_kernel<P, N>, L.blocks, kOptThreads, 1, false, st, L.tab,
                             sums_at + L.sums_at, slots_at + L.slots_at);
            else
                launch_table(norm_partial_kernel<P, N>, L.blocks, kOptThreads, 1, false, st, L.tab,
                             sums_at + L.sums_at, fetched);
        }
    }
};

// The cluster's form of a launch: its table cut into warps' tiles, and as many
// threads as there are tiles, up to kSmallBlocks blocks.
struct SmallLaunch {
    SpanTable<kSmallSpans> tab;
    unsigned cluster = 1, threads = 32;

    explicit SmallLaunch(const SpanPlan<kSmallSpans>& plan) {
        SpanLaunch<kSmallSpans> L = plan.launches[0];
        const int32_t tiles = L.cut(kSmallTile);
        while (threads < kSmallThreads && int32_t(threads) < 32 * tiles) threads *= 2;
        while (cluster < kSmallBlocks && int32_t(cluster) * (kSmallThreads / 32) < tiles) cluster *= 2;
        tab = L.tab;
    }
};

template <int P, int N>
void launch_norm_finish(const SpanLaunch<N>& L, const double* sums, int n_sums, const double* slots, float* norm,
                        float* norms, bool pdl, cudaStream_t st) {
    launch_table(norm_finish_kernel<P, N>, 1 + (slots ? L.tab.count : 0), kOptThreads, 1, pdl, st, L.tab, L.blocks,
                 sums, n_sums, slots, norm, norms);
}

template <int P, int N>
int norm_all(const SpanPlan<N>& plan, float* norm, float* norms, Arena arena, int64_t n, cudaStream_t st) {
    if constexpr (N == kSmallSpans) {
        if (small_norm(n, plan.bytes())) {
            const SmallLaunch s(plan);
            if (norms) launch_table(norm_small_each_kernel<P>, s.cluster, s.threads, s.cluster, false, st, s.tab, norm, norms);
            else launch_table(norm_small_kernel<P>, s.cluster, s.threads, s.cluster, false, st, s.tab, norm);
            return XSG_OK;
        }
    }
    double* sums = arena.take<double>(sums_count(n));
    double* slots = norms ? arena.take<double>(slots_count(n)) : nullptr;
    plan.template partials<P>(sums, slots, nullptr, st);
    for (size_t l = 0; l < plan.launches.size(); ++l) {
        const SpanLaunch<N>& L = plan.launches[l];
        const bool last = l + 1 == plan.launches.size();
        if (!slots && !last) continue;
        // the first of these follows the last first pass directly
        launch_norm_finish<P>(L, sums, int(plan.sums), slots ? slots + L.slots_at : nullptr, last ? norm : nullptr,
                              norms ? norms + L.first_span : nullptr, !slots || l == 0, st);
    }
    return XSG_OK;
}

template <int P, int N>
int clip_all(const SpanPlan<N>& plan, float max_norm, float* norm, Arena arena, int64_t n, cudaStream_t st) {
    if constexpr (N == kSmallSpans) {
        if (small_clip(n, plan.bytes())) {
            const SmallLaunch s(plan);
            launch_table(clip_small_kernel<P>, s.cluster, s.threads, s.cluster, false, st, s.tab, max_norm, norm);
            return XSG_OK;
        }
    }
    double* sums = arena.take<double>(sums_count(n));
    unsigned* fetched = arena.take<unsigned>(counters_count(n));
    plan.template partials<P>(sums, nullptr, fetched, st);
    for (size_t l = plan.launches.size(); l-- > 0;)
        launch_table(clip_scale_kernel<P, N>, std::min(plan.launches[l].blocks, 148 * kScaleResident), kOptThreads, 1, l + 1 == plan.launches.size(),
                     st, plan.launches[l].tab, sums, int(plan.sums), max_norm, l == 0 ? norm : nullptr, fetched + l);
    return XSG_OK;
}

// body(P) for a norm type.
template <typename F>
int with_norm_type(int norm_type, const char* what, F&& body) {
    switch (norm_type) {
        case XSG_NORM_2: return body(std::integral_constant<int, 2>{});
        case XSG_NORM_1: return body(std::integral_constant<int, 1>{});
        case XSG_NORM_INF: return body(std::integral_constant<int, kNormInf>{});
        default: return set_error(XSG_ERR_INVALID_ARGUMENT, std::string(what) + ": unknown norm type");
    }
}

// body(plan) with the table that the number of tensors asks for.
template <typename Get, typename F>
int with_plan(int64_t n, Get&& get, F&& body) {
    if (n <= kSmallSpans) return body(SpanPlan<kSmallSpans>(n, get));
    return body(SpanPlan<kSpans>(n, get));
}

int grad_norm(const xsg_span* spans, int64_t n, int norm_type, float* norm, float* norms, Arena arena,
              cudaStream_t st) {
    if (int rc = check_spans(spans, n, "grad_norm")) return rc;
    XSG_REQUIRE(norm, "grad_norm: null output");
    if (int rc = check_words(norm, norms, nullptr, arena, "grad_norm")) return rc;
    if (arena.cap < xsg_grad_norm_workspace_bytes(spans, n))
        return set_error(XSG_ERR_WORKSPACE, "grad_norm: workspace too small");
    const auto get = [&](int64_t i, auto& L) { L.add(spans[i].data, spans[i].n, spans[i].dtype); };
    ScopedTimer tm("grad_norm", st);
    const int rc = with_plan(n, get, [&](const auto& plan) {
        return with_norm_type(norm_type, "grad_norm",
                              [&](auto p) { return norm_all<decltype(p)::value>(plan, norm, norms, arena, n, st); });
    });
    return rc ? rc : check_launch("grad_norm");
}

int clip_grads(const xsg_span* spans, int64_t n, int norm_type, float max_norm, float* norm, Arena arena,
               cudaStream_t st) {
    if (int rc = check_spans(spans, n, "clip_grads")) return rc;
    XSG_REQUIRE(norm, "clip_grads: null output");
    if (int rc = check_words(norm, nullptr, nullptr, arena, "clip_grads")) return rc;
    XSG_REQUIRE(max_norm >= 0.f && std::isfinite(max_norm), "clip_grads: max_norm must be finite and not negative");
    if (arena.cap < xsg_clip_grads_workspace_bytes(spans, n))
        return set_error(XSG_ERR_WORKSPACE, "clip_grads: workspace too small");
    const auto get = [&](int64_t i, auto& L) { L.add(spans[i].data, spans[i].n, spans[i].dtype); };
    ScopedTimer tm("clip_grads", st);
    const int rc = with_plan(n, get, [&](const auto& plan) {
        return with_norm_type(norm_type, "clip_grads",
                              [&](auto p) { return clip_all<decltype(p)::value>(plan, max_norm, norm, arena, n, st); });
    });
    return rc ? rc : check_launch("clip_grads");
}

// ---- AdamW
int check_adamw(const xsg_adamw_span* spans, int64_t n) {
    XSG_REQUIRE(n > 0 && spans, "adamw_update: at least one tensor is needed");
    int64_t total = 0;
    for (int64_t i = 0; i < n; ++i) {
        const xsg_adamw_span& s = spans[i];
        XSG_REQUIRE(known_dtype(s.param_dtype) && known_dtype(s.grad_dtype), "adamw_update: unknown element type");
        XSG_REQUIRE(s.n >= 0 && s.n < kMaxElems - total, "adamw_update: bad element count");
        total += s.n;
        XSG_REQUIRE(s.n == 0 || (s.param && s.grad && s.exp_avg && s.exp_avg_sq), "adamw_update: null pointer");
        XSG_REQUIRE(!s.row_mask || (s.row_size > 0 && s.row_size < (int64_t(1) << 30)),
                    "adamw_update: a row mask needs a row size below 2^30");
        // the mask has n / row_size entries: elements past the last whole row have none
        XSG_REQUIRE(!s.row_mask || s.n % s.row_size == 0,
                    "adamw_update: the element count under a row mask must be a multiple of the row size");
        const auto off = [](const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % size != 0; };
        XSG_REQUIRE(!off(s.param, elem_size(s.param_dtype)) && !off(s.grad, elem_size(s.grad_dtype)) &&
                        !off(s.exp_avg, 4) && !off(s.exp_avg_sq, 4) && !off(s.master, 4),
                    "adamw_update: misaligned pointer");
        XSG_REQUIRE(s.beta1 >= 0 && s.beta1 < 1 && s.beta2 >= 0 && s.beta2 < 1, "adamw_update: betas must be in [0, 1)");
        XSG_REQUIRE(s.eps >= 0 && std::isfinite(s.lr) && std::isfinite(s.weight_decay),
                    "adamw_update: bad learning rate, eps or weight decay");
        // finite in 64 bits is not enough: inf * 0 would make NaN of entries without gradient
        XSG_REQUIRE(std::isfinite(float(s.lr)) && std::isfinite(float(s.lr * s.weight_decay)),
                    "adamw_update: learning rate, or its product with the weight decay, beyond 32 bits");
    }
    return XSG_OK;
}

// How far the parameter is past a multiple of 64 elements, or -1 if another
// array of the update is not as far past a multiple of four.
int common_lead(const xsg_adamw_span& s) {
    const auto past = [](const void* p, int size, int of) { return int(reinterpret_cast<uintptr_t>(p) / size % of); };
    const int lead = past(s.param, elem_size(s.param_dtype), kAdamLine);
    const bool all = past(s.grad, elem_size(s.grad_dtype), 4) == lead % 4 && past(s.exp_avg, 4, 4) == lead % 4 &&
                     past(s.exp_avg_sq, 4, 4) == lead % 4 && (!s.master || past(s.master, 4, 4) == lead % 4);
    return all ? lead : -1;
}

AdamHyper hyper_of(const xsg_adamw_span& s) {
    AdamHyper h{};
    h.beta1 = float(s.beta1);
    h.rest1 = float(1.0 - s.beta1);
    h.beta2 = float(s.beta2);
    h.rest2 = float(1.0 - s.beta2);
    h.lr = float(s.lr);
    h.lr_decay = float(s.lr * s.weight_decay);
    // an eps above 0 stays above 0, so that an entry that never had a gradient gives 0 / eps = 0, not NaN
    h.eps = s.eps > 0 ? std::max(float(s.eps), std::numeric_limits<float>::denorm_min()) : 0.f;
    h.log_beta1 = float(std::log(s.beta1));
    h.log_beta2 = float(std::log(s.beta2));
    return h;
}

// Fills a table with tensors from `i` on, as many as it holds (tensors and
// different groups of options); returns the first that is not in.
template <int N>
int64_t fill_adam(AdamTable<N>& tab, const xsg_adamw_span* spans, int64_t i, int64_t n, int32_t tile, bool& f32, bool& rows) {
    int groups = 0, t = 0, g = 0;
    int64_t tiles = 0;
    tab.tile = tile;
    f32 = true, rows = false;
    for (; t < N && i < n; ++t, ++i) {
        const xsg_adamw_span& s = spans[i];
        const auto same = [&](const xsg_adamw_span& o) {
            return s.lr == o.lr && s.beta1 == o.beta1 && s.beta2 == o.beta2 && s.eps == o.eps &&
                   s.weight_decay == o.weight_decay;
        };
        if (t == 0 || !same(spans[i - 1])) {  // the options of the one before are its own, mostly
            const AdamHyper h = hyper_of(s);
            for (g = 0; g < groups && std::memcmp(&tab.hyper[g], &h, sizeof(h)) != 0;) ++g;
            if (g == kAdamGroups) break;
            if (g == groups) tab.hyper[groups++] = h;
        }
        AdamEntry& e = tab.entry[t];
        const int lead = common_lead(s);
        const auto back = [&](const void* p, int size) {
            return const_cast<char*>(static_cast<const char*>(p)) - std::max(lead, 0) * size;
        };
        e.vec = lead >= 0;
        e.lead = uint8_t(std::max(lead, 0));
        e.group = uint8_t(g);
        e.param = back(s.param, elem_size(s.param_dtype));
        e.grad = back(s.grad, elem_size(s.grad_dtype));
        e.exp_avg = reinterpret_cast<float*>(back(s.exp_avg, 4));
        e.exp_avg_sq = reinterpret_cast<float*>(back(s.exp_avg_sq, 4));
        e.master = s.master ? reinterpret_cast<float*>(back(s.master, 4)) : nullptr;
        e.rows = s.row_mask;
        e.end = e.lead + s.n;
        e.row_size = int32_t(std::max<int64_t>(s.row_size, 1));
        e.row_magic = uint32_t(((int64_t(1) << 31) + e.row_size - 1) / e.row_size);
        e.param_dtype = uint8_t(s.param_dtype);
        e.grad_dtype = uint8_t(s.grad_dtype);
        f32 = f32 && s.param_dtype == XSG_F32 && s.grad_dtype == XSG_F32 && !s.master;
        rows = rows || (s.row_mask && s.n);
        tab.first[t] = int32_t(tiles);
        tiles += s.n ? (e.lead + s.n + tile - 1) / tile : 0;
    }
    tab.first[t] = int32_t(tiles);
    tab.count = t;
    return i;
}

template <int N>
void adamw_all(const xsg_adamw_span* spans, int64_t n, int64_t elems, AdamCall call, float* norm, cudaStream_t st) {
    AdamTable<N> tab;
    bool masked = false;
    for (int64_t i = 0; i < n; ++i) masked = masked || spans[i].row_mask;
    const int32_t tile = tile_for(elems, 1024, masked ? kRowsTile : kAdamTile, 148 * kAdamResident);
    bool pdl = call.sums != nullptr;  // the first launch follows the norm's directly
    for (int64_t i = 0; i < n;) {
        bool f32, rows;
        i = fill_adam(tab, spans, i, n, tile, f32, rows);
        call.advance = i >= n;
        call.norm = i >= n ? norm : nullptr;
        const int32_t tiles = tab.first[tab.count];
        const int32_t blocks = std::max(1, call.fetched || rows ? std::min(tiles, 148 * kAdamResident) : tiles);
        launch_table(f32 ? (rows ? adamw_kernel<N, true, true> : adamw_kernel<N, true, false>)
                         : (rows ? adamw_kernel<N, false, true> : adamw_kernel<N, false, false>),
                     blocks, kOptThreads, 1, pdl, st, tab, call);
        pdl = false;
        if (call.fetched) ++call.fetched;
    }
}

int adamw_update(const xsg_adamw_span* spans, int64_t n, int64_t* step, float max_norm, bool skip_nonfinite,
                 float* norm, Arena arena, cudaStream_t st) {
    if (int rc = check_adamw(spans, n)) return rc;
    XSG_REQUIRE(step, "adamw_update: null step counter");
    if (int rc = check_words(norm, nullptr, step, arena, "adamw_update")) return rc;
    XSG_REQUIRE(max_norm < 0.f || std::isfinite(max_norm), "adamw_update: max_norm must be finite");
    ScopedTimer tm("adamw_update", st);
    AdamCall call{};
    call.step = reinterpret_cast<unsigned long long*>(step);
    call.clip = max_norm >= 0.f;
    call.skip_nonfinite = skip_nonfinite;
    call.max_norm = max_norm;
    int64_t elems = 0;
    for (int64_t i = 0; i < n; ++i) elems += spans[i].n;
    int rc = XSG_OK;
    bool done = false;
    if (call.clip || skip_nonfinite || norm) {
        if (arena.cap < xsg_adamw_workspace_bytes(spans, n))
            return set_error(XSG_ERR_WORKSPACE, "adamw_update: workspace too small");
        const auto get = [&](int64_t i, auto& L) { L.add(spans[i].grad, spans[i].n, spans[i].grad_dtype); };
        rc = with_plan(n, get, [&](const auto& plan) {
            if constexpr (std::is_same_v<std::decay_t<decltype(plan)>, SpanPlan<kSmallSpans>>) {
                if (small_adamw(n, elems)) {
                    const SmallLaunch s(plan);
                    AdamTable<kSmallSpans> tab;
                    bool f32, rows;
                    fill_adam(tab, spans, 0, n, kSmallAdamTile, f32, rows);
                    call.norm = norm;
                    launch_table(f32 ? adamw_small_kernel<true> : adamw_small_kernel<false>, s.cluster, s.threads,
                                 s.cluster, false, st, s.tab, tab, call);
                    done = true;
                    return int(XSG_OK);
                }
            }
            double* sums = arena.take<double>(sums_count(n));
            call.fetched = arena.take<unsigned>(counters_count(n));
            plan.template partials<2>(sums, nullptr, call.fetched, st);
            call.sums = sums;
            call.n_sums = int(plan.sums);
            return int(XSG_OK);
        });
    }
    if (rc) return rc;
    if (!done) {
        if (n <= kSmallSpans) adamw_all<kSmallSpans>(spans, n, elems, call, norm, st);
        else adamw_all<kAdamSpans>(spans, n, elems, call, norm, st);
    }
    return check_launch("adamw_update");
}

// No C++ exception leaves a C entry.
template <typename F>
int guarded(const char* what, F&& body) {
    try {
        return body();
    } catch (const std::exception& e) {
        return set_error(XSG_ERR_INVALID_ARGUMENT, std::string(what) + ": " + e.what());
    }
}

Arena arena_of(void* workspace, size_t bytes) { return Arena(workspace, workspace ? bytes : 0); }

}  // namespace
}  // namespace xsg

using namespace xsg;

extern "C" size_t xsg_grad_norm_workspace_size(int64_t n_spans) {
    if (n_spans <= 0) return 0;
    return Arena::round(sums_count(n_spans) * sizeof(double)) + Arena::round(slots_count(n_spans) * sizeof(double));
}

// Bytes of at most kSmallSpans tensors (no more are asked for).
static int64_t small_bytes(const xsg_span* spans, int64_t n) {
    int64_t bytes = 0;
    for (int64_t i = 0; i < n && n <= kSmallSpans; ++i) bytes += spans[i].n * elem_size(spans[i].dtype);
    return bytes;
}

extern "C" size_t xsg_grad_norm_workspace_bytes(const xsg_span* spans_host, int64_t n_spans) {
    if (n_spans <= 0 || !spans_host) return 0;
    return small_norm(n_spans, small_bytes(spans_host, n_spans)) ? 0 : xsg_grad_norm_workspace_size(n_spans);
}

extern "C" size_t xsg_clip_grads_workspace_bytes(const xsg_span* spans_host, int64_t n_spans) {
    if (n_spans <= 0 || !spans_host) return 0;
    return small_clip(n_spans, small_bytes(spans_host, n_spans)) ? 0 : xsg_grad_norm_workspace_size(n_spans);
}

extern "C" size_t xsg_adamw_workspace_bytes(const xsg_adamw_span* spans_host, int64_t n_spans) {
    if (n_spans <= 0 || !spans_host) return 0;
    int64_t elems = 0;
    for (int64_t i = 0; i < n_spans && n_spans <= kSmallSpans; ++i) elems += spans_host[i].n;
    return small_adamw(n_spans, elems) ? 0 : xsg_grad_norm_workspace_size(n_spans);
}

extern "C" int xsg_grad_norm(const xsg_span* spans_host, int64_t n_spans, int norm_type, float* norm, float* norms,
                             void* workspace, size_t workspace_bytes, xsg_stream_t stream) {
    return guarded("grad_norm", [&] {
        return grad_norm(spans_host, n_spans, norm_type, norm, norms, arena_of(workspace, workspace_bytes),
                         as_cuda(stream));
    });
}

extern "C" int xsg_clip_grads(const xsg_span* spans_host, int64_t n_spans, int norm_type, float max_norm, float* norm,
                              void* workspace, size_t workspace_bytes, xsg_stream_t stream) {
    return guarded("clip_grads", [&] {
        return clip_grads(spans_host, n_spans, norm_type, max_norm, norm, arena_of(workspace, workspace_bytes),
                          as_cuda(stream));
    });
}

extern "C" int xsg_adamw_update(const xsg_adamw_span* spans_host, int64_t n_spans, int64_t* step, float max_norm,
                                int skip_nonfinite, float* norm, void* workspace, size_t workspace_bytes,
                                xsg_stream_t stream) {
    return guarded("adamw_update", [&] {
        return adamw_update(spans_host, n_spans, step, max_norm, skip_nonfinite != 0, norm,
                            arena_of(workspace, workspace_bytes), as_cuda(stream));
    });
}
