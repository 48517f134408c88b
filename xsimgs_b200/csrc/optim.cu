// The end of a training step, over many tensors at once, for sm_100a: the
// global gradient norm, clipping by it, and the AdamW update that takes the
// clipped gradient.
//
//   N   = (sum over tensors t and elements i of |g_ti|^p)^(1/p),  p = 2, 1, inf
//   c   = min(1, max_norm / (N + 1e-6)),  g <- c g
//   g'  = c g,  m <- b1 m + (1 - b1) g',  v <- b2 v + (1 - b2) g'^2
//   w   <- w - lr wd w - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// All three are HBM-bound.  The tensors travel as a table in the kernel's
// parameters, so that a call copies nothing to the device and can be captured
// in a graph.  Each tensor is cut into tiles; every block takes one
// contiguous run of the tiles of all tensors, so that tensors of any size
// share the work evenly and the order of every sum depends on the tensors'
// sizes alone: no atomics, the same bits on every run.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <vector>

#include "common.cuh"

namespace xsg {
namespace {

constexpr int kOptThreads = 256;
constexpr int kOptBlocks = 148 * 4;      // blocks a launch at most
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
// A tensor is numbered from the 16-byte boundary at or below its first
// element: its elements are the numbers [lead, end) from `base`, whatever its
// offset, and every 16 bytes in between are one aligned vector.  Tile k holds
// the numbers [k * tile, (k + 1) * tile); tensor t of a table owns the tiles
// [first[t], first[t + 1]) of the launch.
constexpr int kTileBytes = 16384;

template <int N>
struct SpanTable {
    void* base[N];
    int64_t end[N];
    int32_t first[N + 1];
    uint8_t lead[N];
    uint8_t dtype[N];
    int32_t count;
};

// The part of tensor t in the tiles [tile, stop): numbers [lo, hi).
struct Part {
    int64_t lo, hi;
};
template <typename Table>
__device__ __forceinline__ Part part_of(const Table& tab, int t, int32_t tile, int32_t stop) {
    const int64_t per = kTileBytes / elem_size(tab.dtype[t]);
    return {max(int64_t(tab.lead[t]), (tile - tab.first[t]) * per), min(tab.end[t], (stop - tab.first[t]) * per)};
}

// The run of tiles of block b out of `blocks`, and back.
__host__ __device__ __forceinline__ int32_t run_start(int32_t tiles, int32_t blocks, int32_t b) {
    return int32_t(int64_t(tiles) * b / blocks);
}
__host__ __device__ __forceinline__ int32_t block_of(int32_t tiles, int32_t blocks, int32_t tile) {
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
// (the conversions to 64 bits run at a quarter of the rate that a full-speed
// read of 16-bit data needs), and goes on as it is unless squares may have
// left the range in which 32 bits lose nothing: above 2^120, below 2^-96, or
// not finite.  Zeros, which most entries of a sparse gradient are, end there.
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

// Sum (or maximum) over the numbers [lo, hi) of a tensor, by the block.
template <int P, int D>
__device__ __forceinline__ double reduce_part(const void* base, Part part) {
    constexpr int V = 16 / elem_size(D);  // elements of a vector
    constexpr int kUnroll = 4;
    const auto* vec = static_cast<const uint4*>(base);
    const int64_t first = (part.lo + V - 1) / V, last = part.hi / V;  // whole vectors
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
    int64_t i = first + threadIdx.x;
    for (; i + (kUnroll - 1) * kOptThreads < last; i += kUnroll * kOptThreads) {
        uint4 q[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) q[k] = __ldg(vec + i + k * kOptThreads);
        take(q);
    }
    if (i < last) {
        uint4 q[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
            q[k] = i + k * kOptThreads < last ? __ldg(vec + i + k * kOptThreads) : make_uint4(0, 0, 0, 0);
        take(q);
    }
    if constexpr (P == kNormInf) {
        const uint32_t one = D == XSG_F32 ? top : max(top & 0xffffu, top >> 16);
        acc = double(D == XSG_F32 ? __uint_as_float(one) : halves(one, D).x);
    }
    // the elements before the first and after the last whole vector
    const int64_t head = min(first * V, part.hi), tail = max(last * V, head);
    const int64_t odd = threadIdx.x < V ? part.lo + threadIdx.x : tail + threadIdx.x - V;
    if (threadIdx.x < 2 * V && odd < (threadIdx.x < V ? head : part.hi))
        acc = join<P>(acc, term<P>(load_as(base, D, odd)));
    return acc;
}

template <int P>
__device__ __forceinline__ double reduce_part(const void* base, int dtype, Part part) {
    if (dtype == XSG_F32) return reduce_part<P, XSG_F32>(base, part);
    if (dtype == XSG_BF16) return reduce_part<P, XSG_BF16>(base, part);
    return reduce_part<P, XSG_F16>(base, part);
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

// Partial sums of a launch: sums[b] for the whole run of block b and, where
// each tensor's norm is asked for, slots[b + t] for its part of tensor t
// (b + t grows along the runs, so that no two parts share a slot).
template <int P, int N>
__global__ void __launch_bounds__(kOptThreads)
    norm_partial_kernel(const __grid_constant__ SpanTable<N> tab, double* __restrict__ sums,
                        double* __restrict__ slots) {
    __shared__ double smem[33];
    const int32_t tiles = tab.first[tab.count];
    int32_t tile = run_start(tiles, gridDim.x, blockIdx.x);
    const int32_t end = run_start(tiles, gridDim.x, blockIdx.x + 1);
    double whole = 0.0;
    for (int t = owner_of(tab, tile); tile < end; ++t) {
        const int32_t stop = min(end, tab.first[t + 1]);
        if (stop <= tile) continue;
        double acc = reduce_part<P>(tab.base[t], tab.dtype[t], part_of(tab, t, tile, stop));
        if (slots) {
            acc = block_reduce<P>(acc, smem);
            if (threadIdx.x == 0) slots[blockIdx.x + t] = acc;
            whole = join<P>(whole, acc);
        } else {
            whole = join<P>(whole, acc);
        }
        tile = stop;
    }
    if (!slots) whole = block_reduce<P>(whole, smem);
    if (threadIdx.x == 0) sums[blockIdx.x] = whole;
}

// All partial sums of a call, by every block for itself.
template <int P>
__device__ __forceinline__ float total_norm(const double* sums, int n, double* smem) {
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) v = join<P>(v, sums[i]);
    return root<P>(block_reduce<P>(v, smem));
}

// Block 0: the norm of all tensors (if `norm`).  The others: a warp for each
// tensor of the table.
template <int P, int N>
__global__ void __launch_bounds__(kOptThreads)
    norm_finish_kernel(const __grid_constant__ SpanTable<N> tab, int blocks, const double* __restrict__ sums,
                       int n_sums, const double* __restrict__ slots, float* __restrict__ norm,
                       float* __restrict__ norms) {
    __shared__ double smem[33];
    if (blockIdx.x == 0) {
        if (!norm) return;
        const float v = total_norm<P>(sums, n_sums, smem);
        if (threadIdx.x == 0) *norm = v;
        return;
    }
    const int t = (blockIdx.x - 1) * (kOptThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (t >= tab.count) return;
    double v = 0.0;
    const int32_t tiles = tab.first[tab.count];
    if (tab.first[t + 1] > tab.first[t]) {
        const int b0 = block_of(tiles, blocks, tab.first[t]), b1 = block_of(tiles, blocks, tab.first[t + 1] - 1);
        for (int b = b0 + lane; b <= b1; b += 32) v = join<P>(v, slots[b + t]);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) v = join<P>(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (lane == 0) norms[t] = root<P>(v);
}

// g <- c g.  The product is taken in 32 bits and rounded once to g's type;
// c = 1 leaves the data alone.
template <int P, int N>
__global__ void __launch_bounds__(kOptThreads)
    clip_scale_kernel(const __grid_constant__ SpanTable<N> tab, const double* __restrict__ sums, int n_sums,
                      float max_norm, float* __restrict__ norm) {
    __shared__ double smem[33];
    const float total = total_norm<P>(sums, n_sums, smem);
    if (blockIdx.x == 0 && threadIdx.x == 0 && norm) *norm = total;
    const float c = clip_coefficient(total, max_norm);
    if (c == 1.f) return;
    const int32_t tiles = tab.first[tab.count];
    int32_t tile = run_start(tiles, gridDim.x, blockIdx.x);
    const int32_t end = run_start(tiles, gridDim.x, blockIdx.x + 1);
    for (int t = owner_of(tab, tile); tile < end; ++t) {
        const int32_t stop = min(end, tab.first[t + 1]);
        if (stop <= tile) continue;
        const int dtype = tab.dtype[t];
        const Part part = part_of(tab, t, tile, stop);
        for (int64_t i = part.lo + threadIdx.x; i < part.hi; i += kOptThreads)
            store_as(tab.base[t], dtype, i, load_as(tab.base[t], dtype, i) * c);
        tile = stop;
    }
}

// ----------------------------------------------------------------- AdamW --
constexpr int kAdamTile = 2048;  // elements
constexpr int kAdamGroups = 32;

struct AdamHyper {
    float beta1, rest1, beta2, rest2, lr, lr_decay, eps;  // rest = 1 - beta, lr_decay = lr * weight decay
    float log_beta1, log_beta2;
};

template <int N>
struct AdamTable {
    void* param[N];
    const void* grad[N];
    float* exp_avg[N];
    float* exp_avg_sq[N];
    float* master[N];
    const uint8_t* rows[N];
    int64_t n[N];
    int64_t row_size[N];
    int32_t first[N + 1];
    uint8_t param_dtype[N];
    uint8_t grad_dtype[N];
    uint8_t group[N];
    AdamHyper hyper[kAdamGroups];
    int32_t count;
};

struct AdamCall {
    long long* step;      // [0] updates taken, [1] blocks that are done (zero between launches)
    const double* sums;   // the gradients' partial sums, or null
    int32_t n_sums;
    int32_t advance;      // the call's last launch counts the update
    int32_t clip;
    int32_t skip_nonfinite;
    float max_norm;
    float* norm;
};

template <int N>
__global__ void __launch_bounds__(kOptThreads)
    adamw_kernel(const __grid_constant__ AdamTable<N> tab, const __grid_constant__ AdamCall call) {
    __shared__ double smem[33];
    float c = 1.f;
    if (call.sums) {
        const float total = total_norm<2>(call.sums, call.n_sums, smem);
        if (blockIdx.x == 0 && threadIdx.x == 0 && call.norm) *call.norm = total;
        if (call.skip_nonfinite && !isfinite(total)) return;  // every block alike: nothing changes
        if (call.clip) c = clip_coefficient(total, call.max_norm);
    }
    const float steps = float(call.step[0] + 1);
    const int32_t tiles = tab.first[tab.count];
    int32_t tile = run_start(tiles, gridDim.x, blockIdx.x);
    const int32_t end = run_start(tiles, gridDim.x, blockIdx.x + 1);
    for (int t = owner_of(tab, tile); tile < end; ++t) {
        const int32_t stop = min(end, tab.first[t + 1]);
        if (stop <= tile) continue;
        const AdamHyper h = tab.hyper[tab.group[t]];
        // 1 - b^t without the cancellation of 1 - pow(b, t)
        const float step_size = h.lr / -expm1f(steps * h.log_beta1);
        const float scale2 = rsqrtf(-expm1f(steps * h.log_beta2));
        const int64_t lo = int64_t(tile - tab.first[t]) * kAdamTile;
        const int64_t hi = min(tab.n[t], int64_t(stop - tab.first[t]) * kAdamTile);
        for (int64_t i = lo + threadIdx.x; i < hi; i += kOptThreads) {
            if (tab.rows[t] && !tab.rows[t][i / tab.row_size[t]]) continue;
            const float g = load_as(tab.grad[t], tab.grad_dtype[t], i) * c;
            const float m = fmaf(h.beta1, tab.exp_avg[t][i], h.rest1 * g);
            const float v = fmaf(h.beta2, tab.exp_avg_sq[t][i], h.rest2 * g * g);
            float w = tab.master[t] ? tab.master[t][i] : load_as(tab.param[t], tab.param_dtype[t], i);
            w = fmaf(-h.lr_decay, w, w);
            w -= step_size * m / fmaf(sqrtf(v), scale2, h.eps);
            tab.exp_avg[t][i] = m;
            tab.exp_avg_sq[t][i] = v;
            if (tab.master[t]) tab.master[t][i] = w;
            store_as(tab.param[t], tab.param_dtype[t], i, w);
        }
        tile = stop;
    }
    if (call.advance) {
        // the last block to come counts the update: all have read step[0] by then
        __syncthreads();
        if (threadIdx.x == 0) {
            auto* word = reinterpret_cast<unsigned long long*>(call.step);
            if (atomicAdd(word + 1, 1ull) == gridDim.x - 1) {
                word[0] += 1;
                word[1] = 0;
            }
        }
    }
}

// ------------------------------------------------------------------ host --
constexpr int kSpans = 1024;
constexpr int kAdamSpans = 320;
static_assert(sizeof(SpanTable<kSpans>) <= 32000 && sizeof(AdamTable<kAdamSpans>) <= 32000,
              "kernel parameters hold 32764 bytes");

struct SpanLaunch {
    SpanTable<kSpans> tab;
    int blocks = 0;
    int64_t first_span = 0, sums_at = 0, slots_at = 0;
};

bool known_dtype(int d) { return d == XSG_F32 || d == XSG_BF16 || d == XSG_F16; }

int64_t span_launches(int64_t n_spans) { return (n_spans + kSpans - 1) / kSpans; }

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

// Cuts the spans into launches of at most kSpans tensors.
std::vector<SpanLaunch> plan_spans(const xsg_span* spans, int64_t n) {
    std::vector<SpanLaunch> out(span_launches(n));
    int64_t sums = 0, slots = 0;
    for (size_t l = 0; l < out.size(); ++l) {
        SpanLaunch& L = out[l];
        L.first_span = int64_t(l) * kSpans;
        L.tab.count = int32_t(std::min<int64_t>(kSpans, n - L.first_span));
        int64_t tiles = 0;
        for (int t = 0; t < L.tab.count; ++t) {
            const xsg_span& s = spans[L.first_span + t];
            const int64_t per = kTileBytes / elem_size(s.dtype);
            const auto at = reinterpret_cast<uintptr_t>(s.data);
            const int64_t lead = int64_t(at % 16) / elem_size(s.dtype);
            L.tab.base[t] = reinterpret_cast<void*>(at - at % 16);
            L.tab.lead[t] = uint8_t(lead);
            L.tab.end[t] = lead + s.n;
            L.tab.dtype[t] = uint8_t(s.dtype);
            L.tab.first[t] = int32_t(tiles);
            tiles += s.n ? (lead + s.n + per - 1) / per : 0;
        }
        L.tab.first[L.tab.count] = int32_t(tiles);
        L.blocks = int(std::max<int64_t>(1, std::min<int64_t>(tiles, kOptBlocks)));
        L.sums_at = sums;
        L.slots_at = slots;
        sums += L.blocks;
        slots += L.blocks + L.tab.count;
    }
    return out;
}

size_t sums_bytes(int64_t n_spans) { return Arena::round(span_launches(n_spans) * kOptBlocks * sizeof(double)); }
size_t slots_bytes(int64_t n_spans) {
    return Arena::round((span_launches(n_spans) * kOptBlocks + n_spans) * sizeof(double));
}

template <int P>
void launch_partials(const std::vector<SpanLaunch>& plan, double* sums, double* slots, cudaStream_t st) {
    for (const SpanLaunch& L : plan)
        launch(norm_partial_kernel<P, kSpans>, L.blocks, kOptThreads, 0, st, L.tab, sums + L.sums_at,
               slots ? slots + L.slots_at : nullptr);
}

int total_sums(const std::vector<SpanLaunch>& plan) { return int(plan.back().sums_at) + plan.back().blocks; }

template <int P>
void norm_all(const std::vector<SpanLaunch>& plan, double* sums, double* slots, float* norm, float* norms,
              cudaStream_t st) {
    launch_partials<P>(plan, sums, slots, st);
    for (size_t l = 0; l < plan.size(); ++l) {
        const SpanLaunch& L = plan[l];
        const bool last = l + 1 == plan.size();
        if (!slots && !last) continue;
        const unsigned grid = 1 + (slots ? blocks_for(L.tab.count, kOptThreads / 32) : 0);
        launch(norm_finish_kernel<P, kSpans>, grid, kOptThreads, 0, st, L.tab, L.blocks,
               static_cast<const double*>(sums), total_sums(plan),
               static_cast<const double*>(slots ? slots + L.slots_at : nullptr), last ? norm : nullptr,
               norms ? norms + L.first_span : nullptr);
    }
}

template <int P>
void clip_all(const std::vector<SpanLaunch>& plan, double* sums, float max_norm, float* norm, cudaStream_t st) {
    launch_partials<P>(plan, sums, nullptr, st);
    for (size_t l = plan.size(); l-- > 0;)
        launch(clip_scale_kernel<P, kSpans>, plan[l].blocks, kOptThreads, 0, st, plan[l].tab,
               static_cast<const double*>(sums), total_sums(plan), max_norm, l == 0 ? norm : nullptr);
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

}  // namespace
}  // namespace xsg

using namespace xsg;

extern "C" size_t xsg_grad_norm_workspace_size(int64_t n_spans) {
    if (n_spans <= 0) return 0;
    return sums_bytes(n_spans) + slots_bytes(n_spans);
}

static int grad_norm(const xsg_span* spans_host, int64_t n_spans, int norm_type, float* norm, float* norms,
                             void* workspace, size_t workspace_bytes, xsg_stream_t stream) {
    if (int rc = check_spans(spans_host, n_spans, "grad_norm")) return rc;
    XSG_REQUIRE(norm, "grad_norm: null output");
    Arena arena(workspace, workspace ? workspace_bytes : 0);
    double* sums = arena.take<double>(span_launches(n_spans) * kOptBlocks);
    double* slots = norms ? arena.take<double>(span_launches(n_spans) * kOptBlocks + n_spans) : nullptr;
    if (!sums || (norms && !slots)) return set_error(XSG_ERR_WORKSPACE, "grad_norm: workspace too small");
    const auto plan = plan_spans(spans_host, n_spans);
    switch (norm_type) {
        case XSG_NORM_2: norm_all<2>(plan, sums, slots, norm, norms, as_cuda(stream)); break;
        case XSG_NORM_1: norm_all<1>(plan, sums, slots, norm, norms, as_cuda(stream)); break;
        case XSG_NORM_INF: norm_all<kNormInf>(plan, sums, slots, norm, norms, as_cuda(stream)); break;
        default: return set_error(XSG_ERR_INVALID_ARGUMENT, "grad_norm: unknown norm type");
    }
    return check_launch("grad_norm");
}

static int clip_grads(const xsg_span* spans_host, int64_t n_spans, int norm_type, float max_norm, float* norm,
                              void* workspace, size_t workspace_bytes, xsg_stream_t stream) {
    if (int rc = check_spans(spans_host, n_spans, "clip_grads")) return rc;
    XSG_REQUIRE(norm, "clip_grads: null output");
    XSG_REQUIRE(max_norm >= 0.f && std::isfinite(max_norm), "clip_grads: max_norm must be finite and not negative");
    Arena arena(workspace, workspace ? workspace_bytes : 0);
    double* sums = arena.take<double>(span_launches(n_spans) * kOptBlocks);
    if (!sums) return set_error(XSG_ERR_WORKSPACE, "clip_grads: workspace too small");
    const auto plan = plan_spans(spans_host, n_spans);
    switch (norm_type) {
        case XSG_NORM_2: clip_all<2>(plan, sums, max_norm, norm, as_cuda(stream)); break;
        case XSG_NORM_1: clip_all<1>(plan, sums, max_norm, norm, as_cuda(stream)); break;
        case XSG_NORM_INF: clip_all<kNormInf>(plan, sums, max_norm, norm, as_cuda(stream)); break;
        default: return set_error(XSG_ERR_INVALID_ARGUMENT, "clip_grads: unknown norm type");
    }
    return check_launch("clip_grads");
}

static int adamw_update(const xsg_adamw_span* spans_host, int64_t n_spans, int64_t* step, float max_norm,
                                int skip_nonfinite, float* norm, void* workspace, size_t workspace_bytes,
                                xsg_stream_t stream) {
    XSG_REQUIRE(n_spans > 0 && spans_host, "adamw_update: at least one tensor is needed");
    XSG_REQUIRE(step, "adamw_update: null step counter");
    XSG_REQUIRE(max_norm < 0.f || std::isfinite(max_norm), "adamw_update: max_norm must be finite");
    const bool clip = max_norm >= 0.f, normed = clip || skip_nonfinite || norm;
    std::vector<xsg_span> grads(normed ? n_spans : 0);
    int64_t total = 0;
    for (int64_t i = 0; i < n_spans; ++i) {
        const xsg_adamw_span& s = spans_host[i];
        XSG_REQUIRE(known_dtype(s.param_dtype) && known_dtype(s.grad_dtype), "adamw_update: unknown element type");
        XSG_REQUIRE(s.n >= 0 && s.n < kMaxElems - total, "adamw_update: bad element count");
        total += s.n;
        XSG_REQUIRE(s.n == 0 || (s.param && s.grad && s.exp_avg && s.exp_avg_sq), "adamw_update: null pointer");
        XSG_REQUIRE(!s.row_mask || s.row_size > 0, "adamw_update: a row mask needs a row size");
        const auto off = [](const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % size != 0; };
        XSG_REQUIRE(!off(s.param, elem_size(s.param_dtype)) && !off(s.grad, elem_size(s.grad_dtype)) &&
                        !off(s.exp_avg, 4) && !off(s.exp_avg_sq, 4) && !off(s.master, 4),
                    "adamw_update: misaligned pointer");
        XSG_REQUIRE(s.beta1 >= 0 && s.beta1 < 1 && s.beta2 >= 0 && s.beta2 < 1, "adamw_update: betas must be in [0, 1)");
        XSG_REQUIRE(s.eps >= 0 && std::isfinite(s.lr) && std::isfinite(s.weight_decay),
                    "adamw_update: bad learning rate, eps or weight decay");
        if (normed) grads[i] = {const_cast<void*>(s.grad), s.n, s.grad_dtype};
    }
    AdamCall call{};
    call.step = reinterpret_cast<long long*>(step);
    call.clip = clip;
    call.skip_nonfinite = skip_nonfinite != 0;
    call.max_norm = max_norm;
    if (normed) {
        Arena arena(workspace, workspace ? workspace_bytes : 0);
        double* sums = arena.take<double>(span_launches(n_spans) * kOptBlocks);
        if (!sums) return set_error(XSG_ERR_WORKSPACE, "adamw_update: workspace too small");
        const auto plan = plan_spans(grads.data(), n_spans);
        launch_partials<2>(plan, sums, nullptr, as_cuda(stream));
        call.sums = sums;
        call.n_sums = total_sums(plan);
    }
    AdamTable<kAdamSpans> tab;
    for (int64_t i = 0; i < n_spans;) {
        int64_t tiles = 0;
        int groups = 0, t = 0;
        for (; t < kAdamSpans && i < n_spans; ++t, ++i) {
            const xsg_adamw_span& s = spans_host[i];
            AdamHyper h{};
            h.beta1 = float(s.beta1);
            h.rest1 = float(1.0 - s.beta1);
            h.beta2 = float(s.beta2);
            h.rest2 = float(1.0 - s.beta2);
            h.lr = float(s.lr);
            h.lr_decay = float(s.lr * s.weight_decay);
            h.eps = float(s.eps);
            h.log_beta1 = float(std::log(s.beta1));
            h.log_beta2 = float(std::log(s.beta2));
            int g = 0;
            while (g < groups && std::memcmp(&tab.hyper[g], &h, sizeof(h)) != 0) ++g;
            if (g == kAdamGroups) break;
            if (g == groups) tab.hyper[groups++] = h;
            tab.group[t] = uint8_t(g);
            tab.param[t] = s.param;
            tab.grad[t] = s.grad;
            tab.exp_avg[t] = s.exp_avg;
            tab.exp_avg_sq[t] = s.exp_avg_sq;
            tab.master[t] = s.master;
            tab.rows[t] = s.row_mask;
            tab.n[t] = s.n;
            tab.row_size[t] = s.row_size;
            tab.param_dtype[t] = uint8_t(s.param_dtype);
            tab.grad_dtype[t] = uint8_t(s.grad_dtype);
            tab.first[t] = int32_t(tiles);
            tiles += (s.n + kAdamTile - 1) / kAdamTile;
        }
        tab.first[t] = int32_t(tiles);
        tab.count = t;
        const bool last = i >= n_spans;
        call.advance = last;
        call.norm = last ? norm : nullptr;
        const unsigned blocks = unsigned(std::max<int64_t>(1, std::min<int64_t>(tiles, kOptBlocks)));
        launch(adamw_kernel<kAdamSpans>, blocks, kOptThreads, 0, as_cuda(stream), tab, call);
    }
    return check_launch("adamw_update");
}

extern "C" int xsg_grad_norm(const xsg_span* spans_host, int64_t n_spans, int norm_type, float* norm, float* norms,
                             void* workspace, size_t workspace_bytes, xsg_stream_t stream) {
    return guarded("grad_norm", [&] {
        return grad_norm(spans_host, n_spans, norm_type, norm, norms, workspace, workspace_bytes, stream);
    });
}

extern "C" int xsg_clip_grads(const xsg_span* spans_host, int64_t n_spans, int norm_type, float max_norm, float* norm,
                              void* workspace, size_t workspace_bytes, xsg_stream_t stream) {
    return guarded("clip_grads", [&] {
        return clip_grads(spans_host, n_spans, norm_type, max_norm, norm, workspace, workspace_bytes, stream);
    });
}

extern "C" int xsg_adamw_update(const xsg_adamw_span* spans_host, int64_t n_spans, int64_t* step, float max_norm,
                                int skip_nonfinite, float* norm, void* workspace, size_t workspace_bytes,
                                xsg_stream_t stream) {
    return guarded("adamw_update", [&] {
        return adamw_update(spans_host, n_spans, step, max_norm, skip_nonfinite, norm, workspace, workspace_bytes,
                            stream);
    });
}
