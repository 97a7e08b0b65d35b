// Balance loss of a router over E experts and T tokens, of which Tv count:
//
//   p[t, e] = softmax(logits[t, :])[e]      n[e] = pairs (t, k) with idx[t, k] == e
//   loss = coef * E * sum_e f[e] P[e],      f[e] = n[e] / (top Tv),  P[e] = sum_t p[t, e] / Tv
//   d loss / d logits[t, e] = p[t, e] (w[e] - sum_j p[t, j] w[j]),   w[e] = coef E / Tv * (f[e] - mean f)
//
// (f has no gradient; a constant taken off f leaves the gradient as it is, since the p of a row add up to one,
// and without it the difference would cancel to a few digits where the experts are evenly used.)
//
// Two passes over the logits, since the gradient of every token needs the sums over all of them.  Bound by
// memory or by launches.  A group of W lanes holds a row in registers, W the power of two that covers it,
// up to a warp, so that short rows share a warp.  The sums are formed without floating-point atomics: lanes over
// their rows, warps of a CTA in order, CTAs of a cluster in order through distributed shared memory, clusters in
// order by the second kernel: the same bits in every run.  Problems that one cluster of eight CTAs can do in a few
// microseconds take one launch, the cluster's barrier between the passes.
#include "balance.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "launch_count.h"

namespace cg = cooperative_groups;

namespace mgk {
namespace balance {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kCluster = 8;

__device__ __forceinline__ float at(const float* p) { return *p; }
__device__ __forceinline__ float at(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

template <int VEC>
__device__ __forceinline__ void load_vec(const float* p, float (&f)[VEC]) {
    if (VEC == 4) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        f[0] = v.x; f[1 % VEC] = v.y; f[2 % VEC] = v.z; f[3 % VEC] = v.w;
    } else {
        f[0] = *p;
    }
}
template <int VEC>
__device__ __forceinline__ void load_vec(const __nv_bfloat16* p, float (&f)[VEC]) {
    if (VEC == 4) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        f[0] = __uint_as_float(v.x << 16); f[1 % VEC] = __uint_as_float(v.x & 0xffff0000u);
        f[2 % VEC] = __uint_as_float(v.y << 16); f[3 % VEC] = __uint_as_float(v.y & 0xffff0000u);
    } else {
        f[0] = __bfloat162float(*p);
    }
}
template <int VEC>
__device__ __forceinline__ void store_vec(float* p, const float (&f)[VEC]) {
    if (VEC == 4)
        *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1 % VEC], f[2 % VEC], f[3 % VEC]);
    else
        *p = f[0];
}
template <int VEC>
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&f)[VEC]) {
    if (VEC == 4) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1 % VEC]), b = __floats2bfloat162_rn(f[2 % VEC], f[3 % VEC]);
        *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
        *p = __float2bfloat16_rn(f[0]);
    }
}

// One row over W lanes: x becomes the probabilities of its columns (zero beyond the last one).  A row
// that holds nothing but -infinity has no probabilities.
template <int VEC, int NC>
__device__ __forceinline__ void softmax_row(float (&x)[NC][VEC], int W) {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            top = fmaxf(top, x[i][v]);
    for (int o = W >> 1; o > 0; o >>= 1)
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top == -INFINITY)
        top = 0.f;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            x[i][v] = __expf(x[i][v] - top);
            sum += x[i][v];
        }
    for (int o = W >> 1; o > 0; o >>= 1)
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float inv = sum == 0.f ? 0.f : __fdividef(1.f, sum);
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            x[i][v] *= inv;
}

template <class T, int VEC, int NC>
__device__ __forceinline__ void load_row(const T* row, int W, int sub, int experts, float (&x)[NC][VEC]) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int c = (i * W + sub) * VEC;
        if (c < experts) {
            load_vec<VEC>(row + c, x[i]);
        } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                x[i][v] = -INFINITY;
        }
    }
}

// Shared memory of a CTA: float sums [kWarps][E] whose first row becomes the CTA's, int counts [E], int valid,
// then float w [E] and room for the totals.
struct Smem {
    float* sums;
    int* counts;
    int* valid;
    float* w;
    float* red;
};
__device__ __forceinline__ Smem carve(char* base, int experts) {
    Smem s;
    s.sums = reinterpret_cast<float*>(base);
    s.counts = reinterpret_cast<int*>(s.sums + kWarps * experts);
    s.valid = s.counts + experts;
    s.w = reinterpret_cast<float*>(s.valid + 4);
    s.red = s.w + experts;
    return s;
}
size_t smem_bytes(int experts) { return sizeof(float) * (kWarps * experts + experts + 4 + experts + 2 * kWarps + 4); }

// The rows of CTA `cta` of `ctas`: sums over them into s.sums[0..E), s.counts and s.valid.
template <class T, int VEC, int NC>
__device__ __forceinline__ void cta_stats(const Router& r, int W, int cta, int ctas, const Smem& s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int e = threadIdx.x; e < r.experts; e += kThreads)
        s.counts[e] = 0;
    if (threadIdx.x == 0)
        *s.valid = 0;
    __syncthreads();
    const int sub = lane & (W - 1), per_warp = 32 / W;
    const T* logits = static_cast<const T*>(r.logits);
    float acc[NC][VEC] = {};
    int valid = 0;
    const int64_t step = static_cast<int64_t>(ctas) * kWarps * per_warp;
    // (all lanes of a warp go round alike: the shuffles are warp-wide)
    for (int64_t base = (static_cast<int64_t>(cta) * kWarps + warp) * per_warp; base < r.tokens; base += step) {
        const int64_t t = base + lane / W;
        const bool live = t < r.tokens && (r.mask == nullptr || r.mask[t] != 0);
        float x[NC][VEC];
        if (live) {
            load_row<T, VEC, NC>(logits + t * r.ld, W, sub, r.experts, x);
            for (int k = sub; k < r.top; k += W) {
                const int64_t e = r.idx64 ? static_cast<const int64_t*>(r.idx)[t * r.top + k]
                                          : static_cast<const int*>(r.idx)[t * r.top + k];
                if (e >= 0 && e < r.experts)
                    atomicAdd(&s.counts[e], 1);
            }
            valid += sub == 0 ? 1 : 0;
        } else {
#pragma unroll
            for (int i = 0; i < NC; ++i)
#pragma unroll
                for (int v = 0; v < VEC; ++v)
                    x[i][v] = -INFINITY;
        }
        softmax_row<VEC, NC>(x, W);
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                acc[i][v] += x[i][v];
    }
    // groups of a warp that hold the same columns, then the warps of the CTA
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            for (int o = W; o < 32; o <<= 1)
                acc[i][v] += __shfl_xor_sync(0xffffffffu, acc[i][v], o);
            const int c = (i * W + sub) * VEC + v;
            if (lane < W && c < r.experts)
                s.sums[warp * r.experts + c] = acc[i][v];
        }
    if (valid)
        atomicAdd(s.valid, valid);
    __syncthreads();
    for (int e = threadIdx.x; e < r.experts; e += kThreads) {
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k)
            sum += s.sums[k * r.experts + e];
        s.sums[e] = sum;
    }
    __syncthreads();
}

// From the totals of one expert a thread: w in shared memory, and the loss and the counts by the CTA
// that is to write them.  `total(e, sum, count)` gives the totals of expert e.
template <class F>
__device__ __forceinline__ void weights(const Router& r, const Result& out, const Smem& s, int valid, bool write, F total) {
    // (the number of pairs counted is needed for the mean share: first the counts)
    int pairs = 0;
    double dot = 0.0;
    for (int e = threadIdx.x; e < r.experts; e += kThreads) {
        double sum;
        int count;
        total(e, sum, count);
        pairs += count;
        dot += sum * count;
        s.w[e] = __int_as_float(count);
        if (write)
            out.counts[e] = count;
    }
    for (int o = 16; o > 0; o >>= 1) {
        pairs += __shfl_xor_sync(0xffffffffu, pairs, o);
        dot += __shfl_xor_sync(0xffffffffu, dot, o);
    }
    __shared__ int pairs_of[kWarps];
    __shared__ double dot_of[kWarps];
    if ((threadIdx.x & 31) == 0) {
        pairs_of[threadIdx.x >> 5] = pairs;
        dot_of[threadIdx.x >> 5] = dot;
    }
    __syncthreads();
    int64_t all = 0;
    double loss = 0.0;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
        all += pairs_of[k];
        loss += dot_of[k];
    }
    const double tv = valid > 0 ? valid : 1, factor = static_cast<double>(out.coef) * r.experts / (tv * tv * r.top);
    if (write && threadIdx.x == 0)
        *out.loss = static_cast<float>(loss * factor);
    // w = factor * (n - all / E) with the difference formed in whole numbers
    const double scale = factor / r.experts;
    for (int e = threadIdx.x; e < r.experts; e += kThreads) {
        const int64_t n = __float_as_int(s.w[e]);
        s.w[e] = static_cast<float>(scale * static_cast<double>(n * r.experts - all));
    }
    __syncthreads();
}

// dlogits of the rows of CTA `cta` of `ctas`
template <class T, class D, int VEC, int NC>
__device__ __forceinline__ void cta_grads(const Router& r, const Result& out, int W, int cta, int ctas, const Smem& s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = lane & (W - 1), per_warp = 32 / W;
    const T* logits = static_cast<const T*>(r.logits);
    float w[NC][VEC];
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const int c = (i * W + sub) * VEC + v;
            w[i][v] = c < r.experts ? s.w[c] : 0.f;
        }
    const int64_t step = static_cast<int64_t>(ctas) * kWarps * per_warp;
    for (int64_t base = (static_cast<int64_t>(cta) * kWarps + warp) * per_warp; base < r.tokens; base += step) {
        const int64_t t = base + lane / W;
        const bool here = t < r.tokens, live = here && (r.mask == nullptr || r.mask[t] != 0);
        float x[NC][VEC];
        if (live) {
            load_row<T, VEC, NC>(logits + t * r.ld, W, sub, r.experts, x);
        } else {
#pragma unroll
            for (int i = 0; i < NC; ++i)
#pragma unroll
                for (int v = 0; v < VEC; ++v)
                    x[i][v] = -INFINITY;
        }
        softmax_row<VEC, NC>(x, W);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                dot += x[i][v] * w[i][v];
        for (int o = W >> 1; o > 0; o >>= 1)
            dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (!here || (out.accumulate && !live))
            continue;
        D* row = static_cast<D*>(out.dlogits) + t * out.ldd;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = (i * W + sub) * VEC;
            if (c >= r.experts)
                continue;
            float d[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                d[v] = x[i][v] * (w[i][v] - dot);
            if (out.accumulate) {
                float o[VEC];
                load_vec<VEC>(row + c, o);
#pragma unroll
                for (int v = 0; v < VEC; ++v)
                    d[v] += o[v];
            }
            store_vec<VEC>(row + c, d);
        }
    }
}

template <class T, int VEC, int NC>
__global__ void __launch_bounds__(kThreads) __cluster_dims__(kCluster) stats_kernel(const Router r, int W, char* partial) {
    extern __shared__ __align__(16) char raw[];
    const Smem s = carve(raw, r.experts);
    cg::cluster_group cluster = cg::this_cluster();
    cta_stats<T, VEC, NC>(r, W, blockIdx.x, gridDim.x, s);
    cluster.sync();
    float* sums = reinterpret_cast<float*>(partial) + static_cast<size_t>(blockIdx.x / kCluster) * partial_words(r.experts);
    int* counts = reinterpret_cast<int*>(sums + r.experts);
    for (int e = cluster.block_rank() * kThreads + threadIdx.x; e < r.experts; e += kCluster * kThreads) {
        float sum = 0.f;
        int count = 0;
        for (int c = 0; c < kCluster; ++c) {
            sum += *cluster.map_shared_rank(s.sums + e, c);
            count += *cluster.map_shared_rank(s.counts + e, c);
        }
        sums[e] = sum;
        counts[e] = count;
    }
    if (cluster.block_rank() == 0 && threadIdx.x == 0) {
        int valid = 0;
        for (int c = 0; c < kCluster; ++c)
            valid += *cluster.map_shared_rank(s.valid, c);
        counts[r.experts] = valid;
    }
    cluster.sync();  // no CTA leaves while its shared memory may be read
}

template <class T, class D, int VEC, int NC>
__global__ void __launch_bounds__(kThreads) grad_kernel(const Router r, int W, const char* partial, int n_partials, const Result out) {
    extern __shared__ __align__(16) char raw[];
    const Smem s = carve(raw, r.experts);
    const float* sums = reinterpret_cast<const float*>(partial);
    const int words = partial_words(r.experts);
    int valid = 0;
    for (int k = 0; k < n_partials; ++k)
        valid += reinterpret_cast<const int*>(sums)[static_cast<size_t>(k) * words + 2 * r.experts];
    weights(r, out, s, valid, blockIdx.x == 0, [&](int e, double& sum, int& count) {
        sum = 0.0;
        count = 0;
        for (int k = 0; k < n_partials; ++k) {
            const float* one = sums + static_cast<size_t>(k) * words;
            sum += one[e];
            count += reinterpret_cast<const int*>(one)[r.experts + e];
        }
    });
    if (out.dlogits != nullptr)
        cta_grads<T, D, VEC, NC>(r, out, W, blockIdx.x, gridDim.x, s);
}

template <class T, class D, int VEC, int NC>
__global__ void __launch_bounds__(kThreads) __cluster_dims__(kCluster) small_kernel(const Router r, int W, const Result out) {
    extern __shared__ __align__(16) char raw[];
    const Smem s = carve(raw, r.experts);
    cg::cluster_group cluster = cg::this_cluster();
    cta_stats<T, VEC, NC>(r, W, blockIdx.x, gridDim.x, s);
    cluster.sync();
    int valid = 0;
    for (int c = 0; c < kCluster; ++c)
        valid += *cluster.map_shared_rank(s.valid, c);
    weights(r, out, s, valid, blockIdx.x == 0, [&](int e, double& sum, int& count) {
        sum = 0.0;
        count = 0;
        for (int c = 0; c < kCluster; ++c) {
            sum += *cluster.map_shared_rank(s.sums + e, c);
            count += *cluster.map_shared_rank(s.counts + e, c);
        }
    });
    cluster.sync();
    if (out.dlogits != nullptr)
        cta_grads<T, D, VEC, NC>(r, out, W, blockIdx.x, gridDim.x, s);
}

// How a row is laid over lanes: vectors of four where the rows' addresses allow it
struct Shape {
    int vec, W, nc;
};
Shape shape(const Router& r, const Result* out) {
    const uintptr_t size = r.bf16 ? 2 : 4;
    bool four = r.experts % 4 == 0 && r.ld % 4 == 0 && reinterpret_cast<uintptr_t>(r.logits) % (4 * size) == 0;
    if (out != nullptr && out->dlogits != nullptr) {
        const uintptr_t d = out->d_bf16 ? 2 : 4;
        four = four && out->ldd % 4 == 0 && reinterpret_cast<uintptr_t>(out->dlogits) % (4 * d) == 0;
    }
    Shape s;
    s.vec = four ? 4 : 1;
    const int units = (r.experts + s.vec - 1) / s.vec;
    s.W = 1;
    while (s.W < 32 && s.W < units)
        s.W *= 2;
    s.nc = 1;
    while (s.nc * 32 < units)
        s.nc *= 2;
    return s;
}

bool bad(const Router& r) {
    // (pairs are counted in 32 bits)
    return r.tokens < 0 || static_cast<int64_t>(r.tokens) * r.top > 0x7fffffffll || r.experts < 1 || r.experts > kMaxExperts || r.top < 1 || r.top > kMaxTop || r.ld < r.experts ||
           (r.tokens > 0 && (r.logits == nullptr || r.idx == nullptr)) ||
           reinterpret_cast<uintptr_t>(r.logits) % (r.bf16 ? 2 : 4) != 0 || reinterpret_cast<uintptr_t>(r.idx) % (r.idx64 ? 8 : 4) != 0;
}
bool bad(const Router& r, const Result& o) {
    return o.loss == nullptr || o.counts == nullptr ||
           (o.dlogits != nullptr && (o.ldd < r.experts || (o.d_bf16 && !r.bf16) ||
                                     reinterpret_cast<uintptr_t>(o.dlogits) % (o.d_bf16 ? 2 : 4) != 0));
}

// Calls go(kernel tag) with the types and the layout as template arguments
template <class T, class F>
cudaError_t pick_row(const Shape& s, F go) {
    if (s.vec == 4) {
        switch (s.nc) {
            case 1: return go(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
            case 2: return go(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});
            case 4: return go(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
            default: return go(std::integral_constant<int, 4>{}, std::integral_constant<int, 8>{});
        }
    }
    switch (s.nc) {
        case 1: return go(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
        case 2: return go(std::integral_constant<int, 1>{}, std::integral_constant<int, 2>{});
        case 4: return go(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
        case 8: return go(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
        case 16: return go(std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{});
        default: return go(std::integral_constant<int, 1>{}, std::integral_constant<int, 32>{});
    }
}

// CTAs for `tokens` rows: at most two rounds of four resident CTAs per SM
int row_ctas(const Router& r, const Shape& s, int most) {
    const int64_t per_cta = static_cast<int64_t>(kWarps) * (32 / s.W);
    const int64_t need = (r.tokens + per_cta - 1) / per_cta;
    return static_cast<int>(need < 1 ? 1 : need > most ? most : need);
}

}  // namespace

int partials(int tokens, int experts) {
    // as many clusters as there is work for: at least 32 KB of float32 logits a CTA
    const int64_t elements = static_cast<int64_t>(tokens) * experts;
    const int64_t want = elements / (8192 * kCluster);
    return static_cast<int>(want < 1 ? 1 : want > kMaxPartials ? kMaxPartials : want);
}

cudaError_t launch_stats(const Router& r, void* partial, cudaStream_t stream) {
    if (bad(r) || partial == nullptr || reinterpret_cast<uintptr_t>(partial) % 16 != 0)
        return cudaErrorInvalidValue;
    const Shape s = shape(r, nullptr);
    const int grid = partials(r.tokens, r.experts) * kCluster;
    auto typed = [&](auto t) {
        using T = decltype(t);
        return pick_row<T>(s, [&](auto vec, auto nc) {
            stats_kernel<T, decltype(vec)::value, decltype(nc)::value>
                    <<<grid, kThreads, smem_bytes(r.experts), stream>>>(r, s.W, static_cast<char*>(partial));
            count_launch();
            return cudaGetLastError();
        });
    };
    return r.bf16 ? typed(__nv_bfloat16{}) : typed(float{});
}

cudaError_t launch_grad(const Router& r, const void* partial, int n_partials, const Result& out, cudaStream_t stream) {
    if (bad(r) || bad(r, out) || partial == nullptr || reinterpret_cast<uintptr_t>(partial) % 16 != 0 || n_partials < 1 ||
        n_partials > kMaxPartials)
        return cudaErrorInvalidValue;
    const Shape s = shape(r, &out);
    const int grid = row_ctas(r, s, 148 * 8);
    auto typed = [&](auto t, auto d) {
        using T = decltype(t);
        using D = decltype(d);
        return pick_row<T>(s, [&](auto vec, auto nc) {
            grad_kernel<T, D, decltype(vec)::value, decltype(nc)::value><<<grid, kThreads, smem_bytes(r.experts), stream>>>(
                    r, s.W, static_cast<const char*>(partial), n_partials, out);
            count_launch();
            return cudaGetLastError();
        });
    };
    if (!r.bf16)
        return typed(float{}, float{});
    return out.d_bf16 ? typed(__nv_bfloat16{}, __nv_bfloat16{}) : typed(__nv_bfloat16{}, float{});
}

cudaError_t launch_small(const Router& r, const Result& out, cudaStream_t stream) {
    if (bad(r) || bad(r, out))
        return cudaErrorInvalidValue;
    if (static_cast<int64_t>(r.tokens) * r.experts > 65536)
        return cudaErrorNotSupported;
    const Shape s = shape(r, &out);
    auto typed = [&](auto t, auto d) {
        using T = decltype(t);
        using D = decltype(d);
        return pick_row<T>(s, [&](auto vec, auto nc) {
            small_kernel<T, D, decltype(vec)::value, decltype(nc)::value>
                    <<<kCluster, kThreads, smem_bytes(r.experts), stream>>>(r, s.W, out);
            count_launch();
            return cudaGetLastError();
        });
    };
    if (!r.bf16)
        return typed(float{}, float{});
    return out.d_bf16 ? typed(__nv_bfloat16{}, __nv_bfloat16{}) : typed(__nv_bfloat16{}, float{});
}

}  // namespace balance
}  // namespace mgk
