// Balance loss of a router over E experts and T tokens, of which Tv count:
//
//   p[t, e] = softmax(logits[t, :])[e]      n[e] = pairs (t, k) with idx[t, k] == e
//   loss = coef * E * sum_e f[e] P[e],      f[e] = n[e] / (top Tv),  P[e] = sum_t p[t, e] / Tv
//   d loss / d logits[t, e] = p[t, e] (w[e] - sum_j p[t, j] w[j]),   w[e] = coef E / Tv * (f[e] - mean f)
//
// (f has no gradient; a constant taken off f leaves the gradient as it is, since the p of a row add up to one,
// and without it the difference would cancel to a few digits where the experts are evenly used.)
//
// Two passes over the logits, since the gradient of every token needs the sums over all of them; the first leaves
// every row's maximum and reciprocal sum behind (8 bytes a row), so that the second has one sum over a row to
// form.  Bound by memory or by launches.  A group of W lanes holds a row in registers, W the power of two that covers
// it, up to a warp, so that short rows share a warp; a warp has several rows in flight.  The sums are
// formed without floating-point atomics: lanes over their rows, warps of a CTA in order, CTAs of a cluster in order
// through distributed shared memory, clusters in order by the second kernel: the same bits in every run.  The
// second kernel's clusters share the work of adding the partial sums up.  Problems that one cluster of eight CTAs
// can do in a few microseconds take one launch, the cluster's barrier between the passes.
#include "balance.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "f32x2.cuh"
#include "launch_count.h"

namespace cg = cooperative_groups;

namespace mgk {
namespace balance {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kCluster = 8;

template <int VEC>
__device__ __forceinline__ void load_vec(const float* p, float (&f)[VEC]) {
    static_assert(VEC == 4 || VEC == 1, "16 bytes or one element");
    if constexpr (VEC == 4) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    } else {
        f[0] = *p;
    }
}
template <int VEC>
__device__ __forceinline__ void load_vec(const __nv_bfloat16* p, float (&f)[VEC]) {
    static_assert(VEC == 8 || VEC == 4 || VEC == 1, "16 or 8 bytes or one element");
    if constexpr (VEC == 1) {
        f[0] = __bfloat162float(*p);
    } else {
        uint32_t w[VEC / 2];
        if constexpr (VEC == 8)
            *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
        else
            *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}
// (float32 gradients beside bf16 logits are stored eight elements at a time too)
template <int VEC>
__device__ __forceinline__ void load_old(const float* p, float (&f)[VEC]) {
    if constexpr (VEC == 8) {
        float lo[4], hi[4];
        load_vec<4>(p, lo);
        load_vec<4>(p + 4, hi);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = lo[i];
            f[4 + i] = hi[i];
        }
    } else {
        load_vec<VEC>(p, f);
    }
}
template <int VEC>
__device__ __forceinline__ void load_old(const __nv_bfloat16* p, float (&f)[VEC]) {
    load_vec<VEC>(p, f);
}
template <int VEC>
__device__ __forceinline__ void store_vec(float* p, const float (&f)[VEC]) {
    if constexpr (VEC == 1) {
        *p = f[0];
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 4)
            *reinterpret_cast<float4*>(p + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
    }
}
template <int VEC>
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&f)[VEC]) {
    if constexpr (VEC == 1) {
        *p = __float2bfloat16_rn(f[0]);
    } else {
        uint32_t w[VEC / 2];
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        if constexpr (VEC == 8)
            *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(w);
        else
            *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(w);
    }
}

// Rows that a group of lanes has in flight: 16 registers of logits where a row takes fewer
template <int VEC, int NC>
__host__ __device__ constexpr int rows_in_flight() {
    return VEC * NC >= 16 ? 1 : VEC * NC >= 8 ? 2 : 4;
}

constexpr float LOG2E = 1.4426950408889634f;

// x <- x f + g;  sum of x y;  y <- y + x f: in pairs where there are pairs
template <int NC, int VEC>
__device__ __forceinline__ void scale_add(float (&x)[NC][VEC], float f, float g) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        if constexpr (VEC == 1) {
            x[i][0] = fmaf(x[i][0], f, g);
        } else {
#pragma unroll
            for (int v = 0; v < VEC; v += 2) {
                const f32x2::Pair p = f32x2::fma({x[i][v], x[i][v + 1]}, f32x2::both(f), f32x2::both(g));
                x[i][v] = p.x;
                x[i][v + 1] = p.y;
            }
        }
    }
}
template <int NC, int VEC>
__device__ __forceinline__ float dot_of(const float (&x)[NC][VEC], const float (&y)[NC][VEC]) {
    if constexpr (VEC == 1) {
        float d = 0.f;
#pragma unroll
        for (int i = 0; i < NC; ++i)
            d = fmaf(x[i][0], y[i][0], d);
        return d;
    } else {
        f32x2::Pair d = f32x2::both(0.f);
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int v = 0; v < VEC; v += 2)
                d = f32x2::fma({x[i][v], x[i][v + 1]}, {y[i][v], y[i][v + 1]}, d);
        return d.x + d.y;
    }
}
template <int NC, int VEC>
__device__ __forceinline__ float sum_of(const float (&x)[NC][VEC]) {
    if constexpr (VEC == 1) {
        float d = 0.f;
#pragma unroll
        for (int i = 0; i < NC; ++i)
            d += x[i][0];
        return d;
    } else {
        f32x2::Pair d = f32x2::both(0.f);
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int v = 0; v < VEC; v += 2)
                d = f32x2::add(d, {x[i][v], x[i][v + 1]});
        return d.x + d.y;
    }
}
template <int NC, int VEC>
__device__ __forceinline__ void add_scaled(float (&y)[NC][VEC], const float (&x)[NC][VEC], float f) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        if constexpr (VEC == 1) {
            y[i][0] = fmaf(x[i][0], f, y[i][0]);
        } else {
#pragma unroll
            for (int v = 0; v < VEC; v += 2) {
                const f32x2::Pair p = f32x2::fma({x[i][v], x[i][v + 1]}, f32x2::both(f), {y[i][v], y[i][v + 1]});
                y[i][v] = p.x;
                y[i][v + 1] = p.y;
            }
        }
    }
}

// x <- exp(x - top), with what is below the normal numbers as zero.  One fused step in front of 2^x; its rounding of
// top log2e is the same in every term of a row and drops out where they are divided by their sum, as long as 2 to the
// power of that error is an ordinary number: at |top| < 2^20 the error is below 2^-3.  (From 1.5e9 on it would pass 128.)
// Beyond, the difference comes first: it is exact for what is near top, and for the rest too large to count.
template <int NC, int VEC>
__device__ __forceinline__ void exponentials(float (&x)[NC][VEC], float top) {
    if (fabsf(top) < 0x1p20f) {
        scale_add<NC, VEC>(x, LOG2E, -top * LOG2E);
    } else {
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                x[i][v] = (x[i][v] - top) * LOG2E;
    }
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(x[i][v]) : "f"(x[i][v]));
}

// Sums (or maxima) of U values over groups of W lanes, the U chains side by side
template <int U>
__device__ __forceinline__ void group_sum(float (&v)[U], int W) {
    for (int o = W >> 1; o > 0; o >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u)
            v[u] += __shfl_xor_sync(0xffffffffu, v[u], o);
}
template <int U>
__device__ __forceinline__ void group_max(float (&v)[U], int W) {
    if (W == 32) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            asm volatile("redux.sync.max.f32 %0, %0, 0xffffffff;" : "+f"(v[u]));
        return;
    }
    for (int o = W >> 1; o > 0; o >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u)
            v[u] = fmaxf(v[u], __shfl_xor_sync(0xffffffffu, v[u], o));
}

// A lane's part of a row as words: one element, or 8 or 16 bytes; what is not there is -infinity
template <class T, int VEC>
constexpr int words_of() { return VEC == 1 ? 1 : static_cast<int>(VEC * sizeof(T) / 4); }
template <class T, int VEC, int NC>
__device__ __forceinline__ void load_row(const T* row, bool live, int W, int sub, int experts,
                                         uint32_t (&w)[NC][words_of<T, VEC>()]) {
    constexpr int N = words_of<T, VEC>();
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int c = (i * W + sub) * VEC;
        if (live && c < experts) {
            if constexpr (VEC == 1) {
                w[i][0] = sizeof(T) == 4 ? *reinterpret_cast<const uint32_t*>(row + c)
                                         : static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(row + c)) << 16;
            } else if constexpr (N == 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(row + c);
                w[i][0] = v.x; w[i][1] = v.y; w[i][2] = v.z; w[i][3] = v.w;
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(row + c);
                w[i][0] = v.x; w[i][1] = v.y;
            }
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k)
                w[i][k] = sizeof(T) == 4 || VEC == 1 ? 0xff800000u : 0xff80ff80u;
        }
    }
}
template <class T, int VEC>
__device__ __forceinline__ float element(const uint32_t (&w)[words_of<T, VEC>()], int v) {
    if (sizeof(T) == 4 || VEC == 1)
        return __uint_as_float(w[v]);
    return __uint_as_float((v & 1) ? w[v / 2] & 0xffff0000u : w[v / 2] << 16);
}

// The rows of a lane: U at a time, 32 / W apart, `left` of them from row `at` on (negative behind the end)
template <class T, int VEC, int NC>
struct Walk {
    static constexpr int U = rows_in_flight<VEC, NC>();
    const T* p;
    const uint8_t* mask;
    int64_t row_step, u_step;
    int at, left, left_of_warp, step, per_warp;

    __device__ __forceinline__ Walk(const Router& r, int W, int cta, int ctas) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        per_warp = 32 / W;
        step = ctas * kWarps * per_warp * U;
        const int first = (cta * kWarps + warp) * per_warp * U;
        at = first + lane / W;
        left = r.tokens - at;
        left_of_warp = r.tokens - first;
        row_step = step * r.ld;
        u_step = per_warp * r.ld;
        p = static_cast<const T*>(r.logits) + at * r.ld;
        mask = r.mask != nullptr ? r.mask + at : nullptr;
    }
    // which of the rows count
    __device__ __forceinline__ void fetch(uint8_t (&live)[U]) const {
#pragma unroll
        for (int u = 0; u < U; ++u)
            live[u] = u * per_warp >= left ? 0 : mask == nullptr ? 1 : mask[u * per_warp];
    }
    __device__ __forceinline__ const T* row(int u) const { return p + u * u_step; }
    __device__ __forceinline__ void next() {
        p += row_step;
        if (mask != nullptr)
            mask += step;
        // (unsigned: the sum may pass the last int once behind the end, where it is not used)
        at = static_cast<int>(static_cast<uint32_t>(at) + step);
        left -= step;
        left_of_warp -= step;
    }
};

// Shared memory of a CTA: float sums [kWarps][E] whose first row becomes the CTA's (where the first pass runs) or
// double totals [E] (where it does not), int counts [E], float w [E], int valid.
struct Smem {
    double* total;
    float* sums;
    int* counts;
    int* valid;
    float* w;
};
__device__ __forceinline__ Smem carve(char* base, int experts, bool sums) {
    Smem s;
    s.total = reinterpret_cast<double*>(base);
    s.sums = reinterpret_cast<float*>(base);
    s.counts = reinterpret_cast<int*>(base) + (sums ? kWarps : 2) * experts;
    s.w = reinterpret_cast<float*>(s.counts + experts);
    s.valid = s.counts + 2 * experts;
    return s;
}
size_t smem_bytes(int experts, bool sums) { return sizeof(float) * (((sums ? kWarps : 2) + 2) * experts + 1); }

// The rows of CTA `cta` of `ctas`: sums over them into s.sums[0..E), s.counts and s.valid, and every row's
// maximum and reciprocal sum into `rows` (zeros for a row that holds nothing but -infinity: it has no probabilities).
template <class T, int VEC, int NC>
__device__ __forceinline__ void cta_stats(const Router& r, int W, int cta, int ctas, const Smem& s, float2* rows) {
    constexpr int U = rows_in_flight<VEC, NC>();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane & (W - 1), per_warp = 32 / W;
    for (int e = threadIdx.x; e < r.experts; e += kThreads)
        s.counts[e] = 0;
    if (threadIdx.x == 0)
        *s.valid = 0;
    __syncthreads();
    // pairs, apart from the rows: contiguous whatever the number per token
    {
        const uint32_t pairs = static_cast<uint32_t>(r.tokens) * r.top, by = static_cast<uint32_t>(ctas) * kThreads;
        constexpr int AT_ONCE = 8;
        for (uint64_t base = static_cast<uint64_t>(cta) * kThreads + threadIdx.x; base < pairs; base += static_cast<uint64_t>(by) * AT_ONCE) {
            int64_t e[AT_ONCE];
            uint8_t counts[AT_ONCE];
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                const uint64_t i = base + static_cast<uint64_t>(k) * by;
                e[k] = -1;
                counts[k] = 1;
                if (i < pairs) {  // (the two loads do not wait for one another)
                    e[k] = r.idx64 ? static_cast<const int64_t*>(r.idx)[i] : static_cast<const int*>(r.idx)[i];
                    if (r.mask != nullptr)
                        counts[k] = r.mask[static_cast<uint32_t>(i) / static_cast<uint32_t>(r.top)];
                }
            }
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k)
                if (counts[k] != 0 && e[k] >= 0 && e[k] < r.experts)
                    atomicAdd(&s.counts[e[k]], 1);
        }
    }
    float acc[NC][VEC] = {};
    int valid = 0;
    Walk<T, VEC, NC> walk(r, W, cta, ctas);
    uint32_t raw[U][NC][words_of<T, VEC>()];
    // rows that are on their way while others are worked on, and the masks of the rows after them: whether a row is read
    // hangs on its mask
    uint8_t live[U];
    int next_at = 0, next_left = 0, next_of_warp = 0;
    auto load = [&]() {
        next_at = walk.at;
        next_left = walk.left;
        next_of_warp = walk.left_of_warp;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            load_row<T, VEC, NC>(walk.row(u), live[u] != 0, W, sub, r.experts, raw[u]);
            valid += live[u] != 0 && sub == 0 ? 1 : 0;
        }
        walk.next();
        walk.fetch(live);
    };
    walk.fetch(live);
    load();
    // (all lanes of a warp go round alike: the shuffles are warp-wide)
    while (next_of_warp > 0) {
        const int at = next_at, left = next_left;
        float x[U][NC][VEC], top[U], sum[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < NC; ++i)
#pragma unroll
                for (int v = 0; v < VEC; ++v)
                    x[u][i][v] = element<T, VEC>(raw[u][i], v);
        load();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            top[u] = -INFINITY;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                if constexpr (VEC == 1) {
                    top[u] = fmaxf(top[u], x[u][i][0]);
                } else {
#pragma unroll
                    for (int v = 0; v < VEC; v += 2)
                        asm("max.f32 %0, %0, %1, %2;" : "+f"(top[u]) : "f"(x[u][i][v]), "f"(x[u][i][v + 1]));
                }
            }
        }
        group_max<U>(top, W);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            top[u] = top[u] == -INFINITY ? 0.f : top[u];
            exponentials<NC, VEC>(x[u], top[u]);
            sum[u] = sum_of<NC, VEC>(x[u]);
        }
        group_sum<U>(sum, W);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float inv = sum[u] == 0.f ? 0.f : __fdividef(1.f, sum[u]);
            if (sub == 0 && u * per_warp < left)
                rows[at + u * per_warp] = make_float2(top[u], inv);
            add_scaled<NC, VEC>(acc, x[u], inv);
        }
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
__device__ __forceinline__ void cta_grads(const Router& r, const Result& out, int W, int cta, int ctas, const Smem& s,
                                          const float2* rows) {
    constexpr int U = rows_in_flight<VEC, NC>();
    const int sub = threadIdx.x & (W - 1), per_warp = 32 / W;
    float w[NC][VEC];
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const int c = (i * W + sub) * VEC + v;
            w[i][v] = c < r.experts ? s.w[c] : 0.f;
        }
    Walk<T, VEC, NC> walk(r, W, cta, ctas);
    uint32_t raw[U][NC][words_of<T, VEC>()];
    float2 row[U];
    bool here[U];
    uint8_t mask[U];
    int next_at = 0, next_left = 0, next_of_warp = 0;
    auto load = [&]() {
        next_at = walk.at;
        next_left = walk.left;
        next_of_warp = walk.left_of_warp;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            here[u] = mask[u] != 0;
            row[u] = u * per_warp < walk.left ? rows[walk.at + u * per_warp] : make_float2(0.f, 0.f);
            load_row<T, VEC, NC>(walk.row(u), here[u], W, sub, r.experts, raw[u]);
        }
        walk.next();
        walk.fetch(mask);
    };
    walk.fetch(mask);
    load();
    while (next_of_warp > 0) {
        const int at = next_at, left = next_left;
        float x[U][NC][VEC], inv[U], dot[U];
        bool live[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            live[u] = here[u];
            inv[u] = row[u].y;
#pragma unroll
            for (int i = 0; i < NC; ++i)
#pragma unroll
                for (int v = 0; v < VEC; ++v)
                    x[u][i][v] = element<T, VEC>(raw[u][i], v);
            exponentials<NC, VEC>(x[u], row[u].x);
            dot[u] = dot_of<NC, VEC>(x[u], w);
        }
        load();
        group_sum<U>(dot, W);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u * per_warp >= left || (out.accumulate && !live[u]))
                continue;
            D* to = static_cast<D*>(out.dlogits) + static_cast<int64_t>(at + u * per_warp) * out.ldd;
            dot[u] *= inv[u];
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                const int c = (i * W + sub) * VEC;
                if (c >= r.experts)
                    continue;
                // p (w - dot) with p = x inv: x (w inv - dot inv)
                float d[VEC];
                if constexpr (VEC == 1) {
                    d[0] = x[u][i][0] * fmaf(w[i][0], inv[u], -dot[u] * inv[u]);
                } else {
#pragma unroll
                    for (int v = 0; v < VEC; v += 2) {
                        const f32x2::Pair q = f32x2::mul({x[u][i][v], x[u][i][v + 1]},
                                                         f32x2::fma({w[i][v], w[i][v + 1]}, f32x2::both(inv[u]), f32x2::both(-dot[u] * inv[u])));
                        d[v] = q.x;
                        d[v + 1] = q.y;
                    }
                }
                if (out.accumulate) {
                    float o[VEC];
                    load_old<VEC>(to + c, o);
#pragma unroll
                    for (int v = 0; v < VEC; ++v)
                        d[v] += o[v];
                }
                store_vec<VEC>(to + c, d);
            }
        }
    }
}

// (three CTAs on an SM, or two, where the registers of a row allow it)
template <class T, int VEC, int NC>
__global__ void __launch_bounds__(kThreads, VEC * NC <= 16 ? 3 : VEC * NC <= 32 ? 2 : 1) __cluster_dims__(kCluster)
        stats_kernel(const Router r, int W, char* partial, float2* rows) {
    extern __shared__ __align__(16) char raw[];
    const Smem s = carve(raw, r.experts, true);
    cg::cluster_group cluster = cg::this_cluster();
    // the second kernel may be set up meanwhile; it waits for this one's end before it reads anything
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    cta_stats<T, VEC, NC>(r, W, blockIdx.x, gridDim.x, s, rows);
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
__global__ void __launch_bounds__(kThreads, VEC * NC <= 16 ? 3 : VEC * NC <= 32 ? 2 : 1) __cluster_dims__(kCluster)
        grad_kernel(const Router r, int W, const char* partial, int n_partials, const float2* rows, const Result out) {
    extern __shared__ __align__(16) char raw[];
    const Smem s = carve(raw, r.experts, false);
    cg::cluster_group cluster = cg::this_cluster();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const float* sums = reinterpret_cast<const float*>(partial);
    const int words = partial_words(r.experts);
    // this CTA's eighth of the experts, G lanes each on the partial sums
    const int per = (r.experts + kCluster - 1) / kCluster;
    int G = 32;
    while (G * per > kThreads)
        G >>= 1;
    {
        const int mine = threadIdx.x / G, e = cluster.block_rank() * per + mine;
        double sum = 0.0;
        int count = 0;
        if (mine < per && e < r.experts)
            for (int k = threadIdx.x % G; k < n_partials; k += G) {
                const float* one = sums + static_cast<size_t>(k) * words;
                sum += one[e];
                count += reinterpret_cast<const int*>(one)[r.experts + e];
            }
        for (int o = G >> 1; o > 0; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            count += __shfl_xor_sync(0xffffffffu, count, o);
        }
        if (mine < per && e < r.experts && threadIdx.x % G == 0) {
            s.total[e] = sum;
            s.counts[e] = count;
        }
    }
    int valid = 0;
    for (int k = threadIdx.x & 31; k < n_partials; k += 32)
        valid += reinterpret_cast<const int*>(sums)[static_cast<size_t>(k) * words + 2 * r.experts];
    valid = __reduce_add_sync(0xffffffffu, valid);
    cluster.sync();
    weights(r, out, s, valid, blockIdx.x == 0, [&](int e, double& sum, int& count) {
        sum = *cluster.map_shared_rank(s.total + e, e / per);
        count = *cluster.map_shared_rank(s.counts + e, e / per);
    });
    cluster.sync();
    if (out.dlogits != nullptr)
        cta_grads<T, D, VEC, NC>(r, out, W, blockIdx.x, gridDim.x, s, rows);
}

template <class T, class D, int VEC, int NC>
__global__ void __launch_bounds__(kThreads) __cluster_dims__(kCluster)
        small_kernel(const Router r, int W, float2* rows, const Result out) {
    extern __shared__ __align__(16) char raw[];
    const Smem s = carve(raw, r.experts, true);
    cg::cluster_group cluster = cg::this_cluster();
    cta_stats<T, VEC, NC>(r, W, blockIdx.x, gridDim.x, s, rows);  // (a CTA reads the rows that it wrote itself)
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
        cta_grads<T, D, VEC, NC>(r, out, W, blockIdx.x, gridDim.x, s, rows);
}

// How a row is laid over lanes: 16-byte vectors where the rows' addresses allow it, then 8 bytes of bf16
struct Shape {
    int vec, W, nc;
};
bool vectors(const Router& r, const Result* out, int vec) {
    bool ok = r.experts % vec == 0 && r.ld % vec == 0 && reinterpret_cast<uintptr_t>(r.logits) % (vec * (r.bf16 ? 2 : 4)) == 0;
    if (out != nullptr && out->dlogits != nullptr)
        ok = ok && out->ldd % vec == 0 && reinterpret_cast<uintptr_t>(out->dlogits) % (out->d_bf16 ? vec * 2 : 16) == 0;
    return ok;
}
Shape shape(const Router& r, const Result* out) {
    Shape s;
    s.vec = r.bf16 && vectors(r, out, 8) ? 8 : vectors(r, out, 4) ? 4 : 1;
    const int units = (r.experts + s.vec - 1) / s.vec;
    // Two vectors a lane before more lanes: a warp then has more rows, and what is done once a row, the sums over lanes
    // above all, is done for all of them at once.  (More take the registers of other warps: 200003 x 256 bf16 logits
    // 105 us with one vector, 136 with four.)
    s.W = 1;
    while (s.W < 32 && s.W * 2 < units)
        s.W *= 2;
    s.nc = 1;
    while (s.nc * s.W < units)
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

// Calls go(vector, columns) with the layout as template arguments
template <class T, class F>
cudaError_t pick_row(const Shape& s, F go) {
#define MGK_ROW(V, N) \
    if (s.vec == V && s.nc == N) \
    return go(std::integral_constant<int, V>{}, std::integral_constant<int, N>{})
    if constexpr (sizeof(T) == 2) {
        MGK_ROW(8, 1);
        MGK_ROW(8, 2);
        MGK_ROW(8, 4);
    }
    MGK_ROW(4, 1);
    MGK_ROW(4, 2);
    MGK_ROW(4, 4);
    MGK_ROW(4, 8);
    MGK_ROW(1, 1);
    MGK_ROW(1, 2);
    MGK_ROW(1, 4);
    MGK_ROW(1, 8);
    MGK_ROW(1, 16);
    MGK_ROW(1, 32);
#undef MGK_ROW
    return cudaErrorInvalidValue;
}

float2* rows_of(void* workspace, const Router& r) {
    return reinterpret_cast<float2*>(static_cast<char*>(workspace) +
                                     static_cast<size_t>(kMaxPartials) * partial_words(r.experts) * 4);
}

}  // namespace

size_t workspace_bytes(int tokens, int experts) {
    if (tokens < 0 || experts < 1)
        return 0;
    return static_cast<size_t>(kMaxPartials) * partial_words(experts) * 4 + static_cast<size_t>(tokens) * sizeof(float2);
}

int partials(int tokens, int experts) {
    // as many clusters as there is work for: at least 16 KB of float32 logits a CTA, three CTAs an SM at most
    const int64_t elements = static_cast<int64_t>(tokens) * experts;
    const int64_t want = elements / (4096 * kCluster);
    return static_cast<int>(want < 1 ? 1 : want > kMaxPartials ? kMaxPartials : want);
}

cudaError_t launch_stats(const Router& r, void* workspace, cudaStream_t stream) {
    if (bad(r) || workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
        return cudaErrorInvalidValue;
    const Shape s = shape(r, nullptr);
    const int grid = partials(r.tokens, r.experts) * kCluster;
    auto typed = [&](auto t) {
        using T = decltype(t);
        return pick_row<T>(s, [&](auto vec, auto nc) {
            stats_kernel<T, decltype(vec)::value, decltype(nc)::value><<<grid, kThreads, smem_bytes(r.experts, true), stream>>>(
                    r, s.W, static_cast<char*>(workspace), rows_of(workspace, r));
            count_launch();
            return cudaGetLastError();
        });
    };
    return r.bf16 ? typed(__nv_bfloat16{}) : typed(float{});
}

cudaError_t launch_grad(const Router& r, const void* partial, int n_partials, const void* workspace, const Result& out,
                        bool follows_stats, cudaStream_t stream) {
    if (bad(r) || bad(r, out) || partial == nullptr || reinterpret_cast<uintptr_t>(partial) % 16 != 0 || n_partials < 1 ||
        n_partials > kMaxPartials || workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
        return cudaErrorInvalidValue;
    const Shape s = shape(r, &out);
    auto typed = [&](auto t, auto d) {
        using T = decltype(t);
        using D = decltype(d);
        return pick_row<T>(s, [&](auto vec, auto nc) {
            constexpr int V = decltype(vec)::value, N = decltype(nc)::value;
            const int64_t per_cta = static_cast<int64_t>(kWarps) * (32 / s.W) * rows_in_flight<V, N>();
            int64_t clusters = (r.tokens + per_cta * kCluster - 1) / (per_cta * kCluster);
            clusters = clusters < 1 ? 1 : clusters > kMaxPartials ? kMaxPartials : clusters;
            cudaLaunchAttribute attr{};
            attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr.val.programmaticStreamSerializationAllowed = 1;
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = static_cast<unsigned>(clusters * kCluster);
            cfg.blockDim = kThreads;
            cfg.dynamicSmemBytes = smem_bytes(r.experts, false);
            cfg.stream = stream;
            cfg.attrs = &attr;
            cfg.numAttrs = follows_stats ? 1 : 0;
            const cudaError_t e = cudaLaunchKernelEx(&cfg, grad_kernel<T, D, V, N>, r, s.W, static_cast<const char*>(partial),
                                                     n_partials, static_cast<const float2*>(rows_of(const_cast<void*>(workspace), r)), out);
            count_launch();
            return e;
        });
    };
    if (!r.bf16)
        return typed(float{}, float{});
    return out.d_bf16 ? typed(__nv_bfloat16{}, __nv_bfloat16{}) : typed(__nv_bfloat16{}, float{});
}

bool is_small(int tokens, int experts) { return static_cast<int64_t>(tokens) * experts <= 65536; }

cudaError_t launch_small(const Router& r, void* workspace, const Result& out, cudaStream_t stream) {
    if (bad(r) || bad(r, out) || !is_small(r.tokens, r.experts) || workspace == nullptr ||
        reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
        return cudaErrorInvalidValue;
    const Shape s = shape(r, &out);
    auto typed = [&](auto t, auto d) {
        using T = decltype(t);
        using D = decltype(d);
        return pick_row<T>(s, [&](auto vec, auto nc) {
            small_kernel<T, D, decltype(vec)::value, decltype(nc)::value>
                    <<<kCluster, kThreads, smem_bytes(r.experts, true), stream>>>(r, s.W, rows_of(workspace, r), out);
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
