// AdamW over a list of tensors:
//
//   m <- b1 m + (1 - b1) g        v <- b2 v + (1 - b2) g^2        (g times grad_scale)
//   p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
//
// 8-bit moments: blocks of 256 elements of one tensor hold m and r = sqrt(v) as e4m3 numbers times a
// float32 scale, the block's largest magnitude over 448.  The root and not v itself: e4m3 spans 2^18, which is
// 2^36 of v, and its half step of 2^-4 then is one of the denominator too.  A root that is not zero is never
// rounded to zero, so no update is divided by eps alone.  The arithmetic of the step is float32; only what is
// kept between steps is rounded.  A NaN or an infinity in a block's gradients makes the block's scale NaN or
// infinite and with it the block.
//
// m and v are formed with every operation rounded on its own, in the order of the formulas (no contraction into fused
// multiply-adds): they are those of a list of elementary float32 operations bit for bit, so that an
// 8-bit m next to the border of two numbers falls to the same side everywhere.  The root that 8-bit moments keep is up to
// one float32 step off the rounded one, and which of two ways it is found goes by all eight numbers of a lane: the same
// blocks give the same bits however a list is split, the same number among others may not.  The update itself uses the
// hardware's approximate reciprocal, a few float32 steps off.
//
// Bound by HBM, with the issue slots close behind: 10 bytes an element with 8-bit moments and bf16 tensors leave
// about 55 instructions for it; products and sums are issued in pairs.  A warp takes blocks of 256 elements, two
// runs of four a lane so that every access of the warp is contiguous whatever the types, and loads the next block
// before it works on one (without: 550 us for 176 M elements at four CTAs an SM, 430 with).  A scale is found with one
// warp-wide integer maximum (float magnitudes order as integers, NaN above all) and nothing is read twice.
// Tensors' addresses travel as kernel parameters: no copy to the device before the launch, and a captured
// graph replays them.
#include "adamw.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <memory>
#include <new>
#include <type_traits>

#include "f32x2.cuh"
#include "launch_count.h"

namespace mgk {
namespace adamw {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr float kTop = 448.f;        // largest e4m3 number
constexpr float kLeast = 0x1p-100f;  // a block whose largest magnitude is below is kept as zeros

struct Entry {
    void* p;
    const void* g;
    void* copy;
    uint64_t n;
    uint64_t block;
};
// CAP tensors a launch; the larger one stays below the 32764 bytes of parameters that a kernel may have
template <int CAP>
struct Table {
    Entry e[CAP];
    uint32_t first_cta[CAP];
    int count;
    int per_warp;  // neighbouring blocks that a warp takes, 32 at most
};

struct Args {
    void *m, *v;
    float *m_scale, *v_scale;
    float b1, c1, b2, c2, eps, keep, rate, root, grad_scale;
    const float *lr_dev, *grad_scale_dev, *step_dev;
    double lr, beta1, beta2, weight_decay, step;
};

// A lane's eight elements are [4 lane, 4 lane + 4) and [128 + 4 lane, ...) of its warp's block.  They are loaded as
// words, float32 one and bf16 two to a word.
template <class T>
constexpr int words_of() { return static_cast<int>(2 * sizeof(T)); }

__device__ __forceinline__ uint32_t bits_of(float x) { return __float_as_uint(x); }
__device__ __forceinline__ uint32_t bits_of(__nv_bfloat16 x) { return __bfloat16_as_ushort(x); }

// As vectors where the block's address and length allow it, else one by one; `live` counts the elements from the
// lane's first on
template <class T>
__device__ __forceinline__ void load_words(const T* s, bool whole, int live, uint32_t (&w)[words_of<T>()]) {
    if (whole) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (sizeof(T) == 4) {
                const uint4 a = __ldcs(reinterpret_cast<const uint4*>(s + 128 * h));
                w[4 * h] = a.x; w[4 * h + 1] = a.y; w[4 * h + 2] = a.z; w[4 * h + 3] = a.w;
            } else {
                const uint2 a = __ldcs(reinterpret_cast<const uint2*>(s + 128 * h));
                w[2 * h] = a.x; w[2 * h + 1] = a.y;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < words_of<T>(); ++i)
            w[i] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int at = (i >> 2) * 128 + (i & 3);
            if (at < live)
                w[i * words_of<T>() / 8] |= bits_of(s[at]) << (sizeof(T) == 4 ? 0 : 16 * (i & 1));
        }
    }
}
template <class T>
__device__ __forceinline__ void unpack(const uint32_t (&w)[words_of<T>()], float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (sizeof(T) == 4)
            f[i] = __uint_as_float(w[i]);
        else
            f[i] = __uint_as_float((i & 1) ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
}
__device__ __forceinline__ void put(float* d, float x) { *d = x; }
__device__ __forceinline__ void put(__nv_bfloat16* d, float x) { *d = __float2bfloat16_rn(x); }
__device__ __forceinline__ void store4(float* d, const float* f) {
    *reinterpret_cast<float4*>(d) = make_float4(f[0], f[1], f[2], f[3]);
}
__device__ __forceinline__ void store4(__nv_bfloat16* d, const float* f) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
    *reinterpret_cast<uint2*>(d) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
template <class T>
__device__ __forceinline__ void store_some(T* d, bool whole, int live, const float (&f)[8]) {
    if (whole) {
        store4(d, f);
        store4(d + 128, f + 4);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int at = (i >> 2) * 128 + (i & 3);
            if (at < live)
                put(d + at, f[i]);
        }
    }
}
template <class T>
__device__ __forceinline__ bool vector_ok(const T* p) {
    return (reinterpret_cast<uintptr_t>(p) & (4 * sizeof(T) - 1)) == 0;
}

using f32x2::both;
using f32x2::fma;
using f32x2::mul;
using f32x2::Pair;
__device__ __forceinline__ Pair add_apart(Pair a, Pair b) { return {__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y)}; }

// four e4m3 numbers times a scale
__device__ __forceinline__ void decode4(uint32_t code, float scale, float* f) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(code >> (16 * i)), __NV_E4M3);
        const float2 x = __half22float2(__half2(h));
        const Pair y = mul({x.x, x.y}, both(scale));
        f[2 * i] = y.x;
        f[2 * i + 1] = y.y;
    }
}
__device__ __forceinline__ float min3(float a, float b, float c) {
    float d;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Square roots of eight numbers by one step of Newton's method for s^2 = x, that is s + (x - s^2) / (2 s), from
// s = x y with the hardware's approximate y = 1 / sqrt(x): a relative error e of s becomes e^2 / 2, so what is left is the
// last rounding, at most one float32 step.  Zeros, numbers near the denormal ones and infinities take CUDA's
// function.
__device__ __forceinline__ void roots8(const float (&v)[8], float (&r)[8]) {
    const float lo = fminf(min3(v[0], v[1], v[2]), fminf(min3(v[3], v[4], v[5]), fminf(v[6], v[7])));
    const float hi = fmaxf(max3(v[0], v[1], v[2]), fmaxf(max3(v[3], v[4], v[5]), fmaxf(v[6], v[7])));
    if (lo >= 0x1p-100f && hi <= 0x1p100f) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            Pair y;
            asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(v[i]));
            asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(v[i + 1]));
            const Pair x{v[i], v[i + 1]}, s = mul(x, y);
            const Pair q = fma(fma({-s.x, -s.y}, s, x), mul(y, both(0.5f)), s);
            r[i] = q.x;
            r[i + 1] = q.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            r[i] = __fsqrt_rn(v[i]);
    }
}
// e4m3 numbers of a block over its scale, which is returned
template <bool KEEP>
__device__ __forceinline__ float encode8(const float (&f)[8], uint32_t (&code)[2]) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i += 2)
        t = f32x2::max3_nan(t, fabsf(f[i]), fabsf(f[i + 1]));
    const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(t)));
    const float inv = top < kLeast ? 0.f : __fmul_rn(__frcp_rn(top), kTop);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float* x = f + 4 * i;
        const Pair y = mul({x[0], x[1]}, both(inv)), z = mul({x[2], x[3]}, both(inv));
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y.x, y.y), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(z.x, z.y), __NV_SATFINITE, __NV_E4M3);
        code[i] = lo | (hi << 16);
        // seldom: a number that came out as zero
        if (KEEP && ((code[i] - 0x01010101u) & ~code[i] & 0x80808080u) != 0) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (((code[i] >> (8 * k)) & 0xffu) == 0 && x[k] > 0.f)
                    code[i] |= 1u << (8 * k);
        }
    }
    return top < kLeast ? 0.f : __fmul_rn(top, 1.f / kTop);
}

// What a lane reads of a block
template <class P, class G, int BITS>
struct Raw {
    static constexpr int MW = BITS == 8 ? 2 : 8;
    uint32_t p[words_of<P>()], g[words_of<G>()], m[MW], v[MW];
};

template <class P, class G, int BITS, int CAP>
__global__ void __launch_bounds__(kThreads, BITS == 8 ? 4 : 3) adamw_kernel(const __grid_constant__ Table<CAP> t, const Args a) {
    __shared__ float from_device[3];
    float keep = a.keep, rate = a.rate, root = a.root, grad_scale = a.grad_scale;
    if (a.lr_dev != nullptr || a.step_dev != nullptr || a.grad_scale_dev != nullptr) {
        if (threadIdx.x == 0) {
            const double lr = a.lr_dev != nullptr ? static_cast<double>(*a.lr_dev) : a.lr;
            const double step = a.step_dev != nullptr ? static_cast<double>(*a.step_dev) : a.step;
            from_device[0] = static_cast<float>(1.0 - lr * a.weight_decay);
            from_device[1] = static_cast<float>(lr / (1.0 - pow(a.beta1, step)));
            from_device[2] = static_cast<float>(1.0 / sqrt(1.0 - pow(a.beta2, step)));
        }
        __syncthreads();
        keep = from_device[0];
        rate = from_device[1];
        root = from_device[2];
        if (a.grad_scale_dev != nullptr)
            grad_scale = *a.grad_scale_dev;
    }
    // the last tensor that begins at or before this CTA
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first_cta[mid] <= blockIdx.x)
            lo = mid;
        else
            hi = mid;
    }
    const Entry& e = t.e[lo];
    const int lane = threadIdx.x & 31;
    // from the CTA's first element on everything fits 32 bits
    const uint64_t cta_block = static_cast<uint64_t>(blockIdx.x - t.first_cta[lo]) * (kWarps * t.per_warp);
    const uint64_t cta_at = cta_block * kBlock, sb0 = e.block + cta_block;
    const int n = static_cast<int>(min(e.n - cta_at, static_cast<uint64_t>(kBlock * kWarps * t.per_warp)));
    P* const p0 = static_cast<P*>(e.p) + cta_at;
    const G* const g0 = static_cast<const G*>(e.g) + cta_at;
    __nv_bfloat16* const c0 = e.copy != nullptr ? static_cast<__nv_bfloat16*>(e.copy) + cta_at : nullptr;
    using M = typename std::conditional<BITS == 8, uint8_t, float>::type;
    M* const m0 = static_cast<M*>(a.m) + sb0 * kBlock;
    M* const v0 = static_cast<M*>(a.v) + sb0 * kBlock;
    const bool p_ok = vector_ok(p0), g_ok = vector_ok(g0), c_ok = vector_ok(c0);
    const Pair gs = both(grad_scale), b1 = both(a.b1), c1 = both(a.c1), b2 = both(a.b2), c2 = both(a.c2);

    auto load = [&](int block, Raw<P, G, BITS>& r) {
        const int at = block * kBlock + lane * 4, live = n - at;
        const bool full = block * kBlock + kBlock <= n;  // (the same in all lanes)
        load_words(p0 + at, full && p_ok, live, r.p);
        load_words(g0 + at, full && g_ok, live, r.g);
        if constexpr (BITS == 8) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                r.m[h] = __ldcs(reinterpret_cast<const uint32_t*>(m0 + at + 128 * h));
                r.v[h] = __ldcs(reinterpret_cast<const uint32_t*>(v0 + at + 128 * h));
            }
        } else {
            load_words(m0 + at, true, 0, r.m);
            load_words(v0 + at, true, 0, r.v);
        }
    };

    Raw<P, G, BITS> raw;
    const int first = (threadIdx.x >> 5) * t.per_warp, past = min(first + t.per_warp, (n + kBlock - 1) / kBlock);
    float scales[2] = {0.f, 0.f}, new_scales[2] = {0.f, 0.f};  // of block first + lane
    if (BITS == 8 && first + lane < past) {
        scales[0] = a.m_scale[sb0 + first + lane];
        scales[1] = a.v_scale[sb0 + first + lane];
    }
    if (first < past)
        load(first, raw);
#pragma unroll 1
    for (int block = first; block < past; ++block) {
        float p[8], g[8], m[8], v[8];
        unpack<P>(raw.p, p);
        unpack<G>(raw.g, g);
        if constexpr (BITS == 8) {
            const float sm = __shfl_sync(0xffffffffu, scales[0], block - first);
            const float sv = __shfl_sync(0xffffffffu, scales[1], block - first);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                decode4(raw.m[h], sm, m + 4 * h);
                decode4(raw.v[h], sv, v + 4 * h);
            }
        } else {
            unpack<float>(raw.m, m);
            unpack<float>(raw.v, v);
        }
        if (block + 1 < past)
            load(block + 1, raw);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            Pair mm{m[i], m[i + 1]}, vv{v[i], v[i + 1]};
            if (BITS == 8)
                vv = mul(vv, vv);
            const Pair x = mul({g[i], g[i + 1]}, gs);
            mm = add_apart(mul(mm, b1), mul(x, c1));
            vv = add_apart(mul(vv, b2), mul(mul(x, x), c2));
            m[i] = mm.x;
            m[i + 1] = mm.y;
            v[i] = vv.x;
            v[i + 1] = vv.y;
        }
        float r[8];
        roots8(v, r);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const Pair d = fma({r[i], r[i + 1]}, both(root), both(a.eps));
            const Pair u = mul({m[i], m[i + 1]}, {rcp_approx(d.x), rcp_approx(d.y)});
            const Pair q = fma(u, both(-rate), mul({p[i], p[i + 1]}, both(keep)));
            p[i] = q.x;
            p[i + 1] = q.y;
        }
        const int at = block * kBlock + lane * 4, live = n - at;
        const bool full = block * kBlock + kBlock <= n;
        store_some(p0 + at, full && p_ok, live, p);
        if (c0 != nullptr)
            store_some(c0 + at, full && c_ok, live, p);
        if constexpr (BITS == 8) {
            uint32_t code[2];
            const float sm = encode8<false>(m, code);
            uint32_t* to = reinterpret_cast<uint32_t*>(m0 + at);
            to[0] = code[0];
            to[32] = code[1];
            const float sv = encode8<true>(r, code);
            to = reinterpret_cast<uint32_t*>(v0 + at);
            to[0] = code[0];
            to[32] = code[1];
            if (lane == block - first) {
                new_scales[0] = sm;
                new_scales[1] = sv;
            }
        } else {
            store_some(m0 + at, true, 0, m);
            store_some(v0 + at, true, 0, v);
        }
    }
    if (BITS == 8 && first + lane < past) {
        a.m_scale[sb0 + first + lane] = new_scales[0];
        a.v_scale[sb0 + first + lane] = new_scales[1];
    }
}

template <class P, class G, int BITS, int CAP>
cudaError_t launch_table(const Tensor* tensors, int count, const Args& a, cudaStream_t stream) {
    Table<CAP> t;
    uint64_t blocks = 0;
    for (int k = 0; k < count; ++k)
        blocks += (tensors[k].n + kBlock - 1) / kBlock;
    // Several blocks a warp once that still fills the chip (what a warp does once, finding its tensor above all, costs
    // as many instructions as a block), eight of 8-bit moments, whose scales then are one whole sector to read and
    // to write: written one by one they held everything else up (176 M elements: 430 us, 297 so; at 4 a warp 310).
    // With 32 bits eight are 3 % slower than four.
    const uint64_t resident = 148ull * 4 * kWarps;
    t.per_warp = BITS == 8 && blocks >= resident * 8 * 4 ? 8 : blocks >= resident * 4 * 3 ? 4 : 1;
    const uint64_t chunk = static_cast<uint64_t>(kBlock) * kWarps * t.per_warp;
    int i = 0;
    while (i < count) {
        uint64_t ctas = 0;
        t.count = 0;
        for (; i < count && t.count < CAP; ++i) {
            const uint64_t need = (tensors[i].n + chunk - 1) / chunk;
            if (need == 0)
                continue;
            if (need > 0x7fffffffull)
                return cudaErrorInvalidValue;
            if (ctas + need > 0x7fffffffull)
                break;
            t.e[t.count] = {tensors[i].p, tensors[i].g, tensors[i].copy, tensors[i].n, tensors[i].block};
            t.first_cta[t.count++] = static_cast<uint32_t>(ctas);
            ctas += need;
        }
        if (t.count == 0)
            continue;
        adamw_kernel<P, G, BITS, CAP><<<static_cast<unsigned>(ctas), kThreads, 0, stream>>>(t, a);
        count_launch();
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess)
            return e;
    }
    return cudaSuccess;
}

template <class P, class G>
cudaError_t launch_typed(const Tensor* tensors, int count, int bits, const Args& a, cudaStream_t stream) {
    // a short list travels as 2.8 KB of parameters, a long one as 31 KB a launch
    if (count <= 64)
        return bits == 8 ? launch_table<P, G, 8, 64>(tensors, count, a, stream)
                         : launch_table<P, G, 32, 64>(tensors, count, a, stream);
    return bits == 8 ? launch_table<P, G, 8, 720>(tensors, count, a, stream)
                     : launch_table<P, G, 32, 720>(tensors, count, a, stream);
}

// Whether ranges of `size` bytes an element overlap that `place` gives for the tensors: these would be written by
// several CTAs at once.  Views of one buffer in their order take one look each, others are sorted.
template <class F>
cudaError_t refuse_overlap(const Tensor* tensors, int count, uint64_t size, F place) {
    struct Range {
        uint64_t begin, end;
    };
    auto range = [&](const Tensor& t) {
        const uint64_t at = t.n != 0 ? reinterpret_cast<uintptr_t>(place(t)) : 0;
        return Range{at, at != 0 ? at + t.n * size : 0};
    };
    uint64_t end = 0;
    int i = 0;
    for (; i < count; ++i) {
        const Range r = range(tensors[i]);
        if (r.begin == 0)
            continue;
        if (r.begin < end)
            break;
        end = r.end;
    }
    if (i == count)
        return cudaSuccess;
    const std::unique_ptr<Range[]> all(new (std::nothrow) Range[count]);
    if (all == nullptr)
        return cudaErrorMemoryAllocation;
    for (int k = 0; k < count; ++k)
        all[k] = range(tensors[k]);
    std::sort(all.get(), all.get() + count, [](const Range& a, const Range& b) { return a.begin < b.begin; });
    for (int k = 1; k < count; ++k)
        if (all[k].begin < all[k - 1].end)
            return cudaErrorInvalidValue;
    return cudaSuccess;
}

}  // namespace

cudaError_t launch(const Tensor* tensors, int count, const Step& s, cudaStream_t stream) {
    static_assert(sizeof(Table<720>) + sizeof(Args) <= 32764, "kernel parameters");
    if (count < 0 || (count > 0 && tensors == nullptr) || (s.bits != 8 && s.bits != 32))
        return cudaErrorInvalidValue;
    const uintptr_t moments = reinterpret_cast<uintptr_t>(s.m) | reinterpret_cast<uintptr_t>(s.v);
    const uintptr_t scales = reinterpret_cast<uintptr_t>(s.m_scale) | reinterpret_cast<uintptr_t>(s.v_scale);
    bool work = false;
    for (int i = 0; i < count; ++i) {
        const Tensor& t = tensors[i];
        if (t.n == 0)
            continue;
        work = true;
        const uintptr_t pm = s.p_bf16 ? 1 : 3, gm = s.g_bf16 ? 1 : 3;
        if (t.p == nullptr || t.g == nullptr || (reinterpret_cast<uintptr_t>(t.p) & pm) ||
            (reinterpret_cast<uintptr_t>(t.g) & gm) || (reinterpret_cast<uintptr_t>(t.copy) & 1))
            return cudaErrorInvalidValue;
    }
    if (!work)
        return cudaSuccess;
    if (s.m == nullptr || s.v == nullptr || (moments & 15) ||
        (s.bits == 8 && (s.m_scale == nullptr || s.v_scale == nullptr || (scales & 3))))
        return cudaErrorInvalidValue;
    cudaError_t e = refuse_overlap(tensors, count, s.p_bf16 ? 2 : 4, [](const Tensor& t) { return t.p; });
    if (e == cudaSuccess)
        e = refuse_overlap(tensors, count, 2, [](const Tensor& t) { return t.copy; });
    if (e != cudaSuccess)
        return e;
    Args a{};
    a.m = s.m;
    a.v = s.v;
    a.m_scale = s.m_scale;
    a.v_scale = s.v_scale;
    a.b1 = static_cast<float>(s.beta1);
    a.c1 = static_cast<float>(1.0 - s.beta1);
    a.b2 = static_cast<float>(s.beta2);
    a.c2 = static_cast<float>(1.0 - s.beta2);
    a.eps = static_cast<float>(s.eps);
    a.keep = static_cast<float>(1.0 - s.lr * s.weight_decay);
    a.rate = static_cast<float>(s.lr / (1.0 - std::pow(s.beta1, s.step)));
    a.root = static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(s.beta2, s.step)));
    a.grad_scale = static_cast<float>(s.grad_scale);
    a.lr_dev = s.lr_dev;
    a.grad_scale_dev = s.grad_scale_dev;
    a.step_dev = s.step_dev;
    a.lr = s.lr;
    a.beta1 = s.beta1;
    a.beta2 = s.beta2;
    a.weight_decay = s.weight_decay;
    a.step = s.step;
    if (s.p_bf16)
        return s.g_bf16 ? launch_typed<__nv_bfloat16, __nv_bfloat16>(tensors, count, s.bits, a, stream)
                        : launch_typed<__nv_bfloat16, float>(tensors, count, s.bits, a, stream);
    return s.g_bf16 ? launch_typed<float, __nv_bfloat16>(tensors, count, s.bits, a, stream)
                    : launch_typed<float, float>(tensors, count, s.bits, a, stream);
}

}  // namespace adamw
}  // namespace mgk
