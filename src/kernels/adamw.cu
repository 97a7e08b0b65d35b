// AdamW over a list of tensors:
//
//   m <- b1 m + (1 - b1) g        v <- b2 v + (1 - b2) g^2        (g times grad_scale)
//   p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
//
// Every operation is rounded on its own (no contraction into fused multiply-adds), so that the update is
// the one that a list of elementary float32 operations gives, bit for bit, on any split of the work: an 8-bit
// moment next to the border of two numbers falls to the same side.
//
// 8-bit moments: blocks of 256 elements of one tensor hold m and r = sqrt(v) as e4m3 numbers times a
// float32 scale, the block's largest magnitude over 448.  The root and not v itself: e4m3 spans 2^18, which is
// 2^36 of v, and its half step of 2^-4 then is one of the denominator too.  A root that is not zero is never
// rounded to zero, so no update is divided by eps alone.  The arithmetic of the step is float32; only what is
// kept between steps is rounded.  A NaN or an infinity in a block's gradients makes the block's scale NaN or
// infinite and with it the block.
//
// Bound by HBM.  A warp takes one block of 256 elements, eight a lane, so a scale is found with one
// warp-wide integer maximum (float magnitudes order as integers, NaN above all) and nothing is read twice.
// Tensors' addresses travel as kernel parameters: no copy to the device before the launch, and a captured
// graph replays them.
#include "adamw.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cmath>
#include <type_traits>

#include "launch_count.h"

namespace mgk {
namespace adamw {

namespace {

constexpr int kThreads = 256;
constexpr int kBlocksPerCta = kThreads / 32;
constexpr float kTop = 448.f;          // largest e4m3 number
constexpr float kLeast = 0x1p-100f;    // a block whose largest magnitude is below is kept as zeros

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
};

struct Args {
    void *m, *v;
    float *m_scale, *v_scale;
    float b1, c1, b2, c2, eps, keep, rate, root, grad_scale;
    const float *lr_dev, *grad_scale_dev, *step_dev;
    double lr, beta1, beta2, weight_decay, step;
};

__device__ __forceinline__ void load8(const float* s, float (&f)[8]) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(s)), b = __ldcs(reinterpret_cast<const float4*>(s) + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* s, float (&f)[8]) {
    const uint4 a = __ldcs(reinterpret_cast<const uint4*>(s));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void store8(float* d, const float (&f)[8]) {
    reinterpret_cast<float4*>(d)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(d)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* d, const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* d, float x) { *d = x; }
__device__ __forceinline__ void put(__nv_bfloat16* d, float x) { *d = __float2bfloat16_rn(x); }

// Eight values of a lane, the whole vector where it may be read as one, else one by one up to `live`
template <class T>
__device__ __forceinline__ void load_some(const T* s, bool whole, int live, float (&f)[8]) {
    if (whole) {
        load8(s, f);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            f[i] = i < live ? to_float(s[i]) : 0.f;
    }
}
template <class T>
__device__ __forceinline__ void store_some(T* d, bool whole, int live, const float (&f)[8]) {
    if (whole) {
        store8(d, f);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < live)
                put(d + i, f[i]);
    }
}
template <class T>
__device__ __forceinline__ bool vector_ok(const T* p) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

__device__ __forceinline__ void decode8(uint2 code, float scale, float (&f)[8]) {
    const uint32_t w[2] = {code.x, code.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i >> 1] >> (16 * (i & 1))),
                                                         __NV_E4M3);
        const float2 x = __half22float2(__half2(h));
        f[2 * i] = __fmul_rn(x.x, scale);
        f[2 * i + 1] = __fmul_rn(x.y, scale);
    }
}
__device__ __forceinline__ uint32_t warp_top(const float (&f)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
    return __reduce_max_sync(0xffffffffu, top);
}
// e4m3 numbers of f over the block's scale, which is returned too
template <bool KEEP>
__device__ __forceinline__ uint2 encode8(const float (&f)[8], float& scale) {
    const float top = __uint_as_float(warp_top(f));
    const float inv = top < kLeast ? 0.f : __fmul_rn(__frcp_rn(top), kTop);
    scale = top < kLeast ? 0.f : __fmul_rn(top, 1.f / kTop);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = __fmul_rn(f[2 * i], inv), b = __fmul_rn(f[2 * i + 1], inv);
        w[i] = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
        if (KEEP) {
            w[i] |= (w[i] & 0xffu) == 0 && f[2 * i] > 0.f ? 1u : 0u;
            w[i] |= (w[i] & 0xff00u) == 0 && f[2 * i + 1] > 0.f ? 0x100u : 0u;
        }
    }
    return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

template <class P, class G, int BITS, int CAP>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ Table<CAP> t, const Args a) {
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
    const uint64_t block = static_cast<uint64_t>(blockIdx.x - t.first_cta[lo]) * kBlocksPerCta + (threadIdx.x >> 5);
    if (block * kBlock >= e.n)
        return;
    const int lane = threadIdx.x & 31;
    const uint64_t at = block * kBlock + lane * 8;
    const int live = at >= e.n ? 0 : static_cast<int>(min(static_cast<uint64_t>(8), e.n - at));
    const bool full = live == 8;
    P* pp = static_cast<P*>(e.p) + at;
    const G* gp = static_cast<const G*>(e.g) + at;
    const uint64_t sb = e.block + block;           // block in the moment buffers
    const uint64_t sat = sb * kBlock + lane * 8;

    float p[8], g[8], m[8], v[8];
    load_some(pp, full && vector_ok(pp), live, p);
    load_some(gp, full && vector_ok(gp), live, g);
    if (BITS == 8) {
        decode8(__ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.m) + sat)), a.m_scale[sb], m);
        decode8(__ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.v) + sat)), a.v_scale[sb], v);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = __fmul_rn(v[i], v[i]);
    } else {
        load8(static_cast<const float*>(a.m) + sat, m);
        load8(static_cast<const float*>(a.v) + sat, v);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = __fmul_rn(g[i], grad_scale);
        m[i] = __fadd_rn(__fmul_rn(m[i], a.b1), __fmul_rn(x, a.c1));
        v[i] = __fadd_rn(__fmul_rn(v[i], a.b2), __fmul_rn(__fmul_rn(x, x), a.c2));
        const float r = __fsqrt_rn(v[i]);
        const float u = __fdiv_rn(m[i], __fadd_rn(__fmul_rn(r, root), a.eps));
        p[i] = __fsub_rn(__fmul_rn(p[i], keep), __fmul_rn(u, rate));
        if (BITS == 8)
            v[i] = r;
    }
    store_some(pp, full && vector_ok(pp), live, p);
    if (e.copy != nullptr) {
        __nv_bfloat16* cp = static_cast<__nv_bfloat16*>(e.copy) + at;
        store_some(cp, full && vector_ok(cp), live, p);
    }
    if (BITS == 8) {
        float sm, sr;
        const uint2 cm = encode8<false>(m, sm), cr = encode8<true>(v, sr);
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.m) + sat) = cm;
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.v) + sat) = cr;
        if (lane == 0) {
            a.m_scale[sb] = sm;
            a.v_scale[sb] = sr;
        }
    } else {
        store8(static_cast<float*>(a.m) + sat, m);
        store8(static_cast<float*>(a.v) + sat, v);
    }
}

template <class P, class G, int BITS, int CAP>
cudaError_t launch_table(const Tensor* tensors, int count, const Args& a, cudaStream_t stream) {
    Table<CAP> t;
    int i = 0;
    while (i < count) {
        uint64_t ctas = 0;
        t.count = 0;
        for (; i < count && t.count < CAP; ++i) {
            const uint64_t need = (tensors[i].n + kBlock * kBlocksPerCta - 1) / (kBlock * kBlocksPerCta);
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
