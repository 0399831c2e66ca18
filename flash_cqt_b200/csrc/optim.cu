// AdamW over many tensors in one launch, moments in 32 or in 8 bits, and the
// global gradient norm that scales the gradients.
//
// For every element, in 32 bits, with t the tensor's own count of steps:
//   g' = g c                       c = min(1, max_norm / (norm + 1e-6)), or 1
//   m  = b1 m + (1 - b1) g'
//   v  = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// Each product and sum is rounded by itself (no fused multiply-add), so the
// result does not depend on how a variant of the kernel is compiled.
//
// Moments in 8 bits: blocks of 256 elements (one warp, 8 elements a lane)
// share a power-of-two scale per moment, one byte each.  m is held in e4m3, v
// in e5m2 (its values span the square of the gradients' range); the scale is
// the least that brings the block's largest finite value to the format's
// largest or below.  The rounding is stochastic, with 16 bits of a hash of
// (seed, t, tensor, element) each: at b2 = 0.999 a step moves v by 0.1 %,
// and an 8-bit float rounded to nearest (steps of 12 to 25 %) would never
// move.  Under the smallest normal value m becomes 0, and v, unless it is 0,
// the smallest normal value: a denominator must not vanish.
//
// The table of tensors rides in the kernel parameters (up to 32 KB): no copy
// before the launch, and a captured graph holds it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "internal.h"

namespace fcqt {

namespace {

constexpr int kThreads = 256;
constexpr int kLane = 8;                        // consecutive elements a thread
constexpr int kChunk = kThreads * kLane;        // elements a CTA takes at a time
static_assert(kChunk % kOptBlock == 0 && 32 * kLane == kOptBlock, "a warp is one block");

template <int N>
struct OptTable {
    OptTensor t[N];
    int count;
    unsigned chunks;
};

// shifts and odd multipliers (the fractional bits of the square roots of 2
// and 3); every bit of the input reaches every bit of the output
__host__ __device__ __forceinline__ unsigned mix32(unsigned x) {
    x ^= x >> 16;
    x *= 0x6A09E667u;
    x ^= x >> 15;
    x *= 0xBB67AE85u;
    return x ^ (x >> 16);
}

// ---- 8 consecutive values as 32-bit floats.  `vec`: all 8 are there, at an
// address that is a multiple of 32 (2) or 16 (1) bytes; else (0) the first n of
// them one by one
__device__ __forceinline__ void load8(const float* p, int vec, int n, float (&x)[8]) {
    if (vec == 2) {
        load_v8(p, x);
    } else if (vec) {
        const float4 a = reinterpret_cast<const float4*>(p)[0];
        const float4 b = reinterpret_cast<const float4*>(p)[1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = i < n ? p[i] : 0.f;
    }
}
__device__ __forceinline__ void store8(float* p, int vec, int n, const float (&x)[8]) {
    if (vec == 2) {
        store_v8(p, x);
    } else if (vec) {
        reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = x[i];
    }
}
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
// 16-bit parameters are rounded once, to nearest even, from the 32-bit result
__device__ __forceinline__ void from_float(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_float(float x, __half& y) { y = __float2half_rn(x); }
template <class T>
__device__ __forceinline__ float2 pair_to_float(unsigned w) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) {
        return __half22float2(*reinterpret_cast<const __half2*>(&w));
    } else {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
}
template <class T>
__device__ __forceinline__ unsigned pair_from_float(float a, float b) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const unsigned*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const unsigned*>(&h);
    }
}
template <class T>
__device__ __forceinline__ void load8(const T* p, int vec, int n, float (&x)[8]) {
    if (vec) {
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = pair_to_float<T>(u[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = i < n ? to_float(p[i]) : 0.f;
    }
}
template <class T>
__device__ __forceinline__ void store8(T* p, int vec, int n, const float (&x)[8]) {
    if (vec) {
        *reinterpret_cast<uint4*>(p) =
            make_uint4(pair_from_float<T>(x[0], x[1]), pair_from_float<T>(x[2], x[3]),
                       pair_from_float<T>(x[4], x[5]), pair_from_float<T>(x[6], x[7]));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) from_float(x[i], p[i]);
    }
}
// 8 codes, the first in the low byte of x
__device__ __forceinline__ uint2 load_codes(const uint8_t* p, int vec, int n) {
    if (vec) return *reinterpret_cast<const uint2*>(p);
    uint2 c = make_uint2(0, 0);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) (i < 4 ? c.x : c.y) |= (unsigned)p[i] << (8 * (i & 3));
    return c;
}
__device__ __forceinline__ void store_codes(uint8_t* p, int vec, int n, uint2 c) {
    if (vec) {
        *reinterpret_cast<uint2*>(p) = c;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = (uint8_t)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
    }
}
__device__ __forceinline__ float sqrt_approx(float x) {
    float y;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// the low bytes of 8 words
__device__ __forceinline__ uint2 pack8(const unsigned (&c)[8]) {
    return make_uint2(
        __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410),
        __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410));
}
// the values of 8 codes times s
template <__nv_fp8_interpretation_t F>
__device__ __forceinline__ void decode8(uint2 c, float s, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned w = i < 2 ? c.x : c.y;
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
            (__nv_fp8x2_storage_t)((i & 1) ? w >> 16 : w & 0xffffu), F);
        const float2 f = __half22float2(__half2(h));
        x[2 * i] = __fmul_rn(f.x, s);
        x[2 * i + 1] = __fmul_rn(f.y, s);
    }
}
// 2^(byte - 127); a byte of 0 is the subnormal 2^-127
__device__ __forceinline__ float scale_of(uint8_t byte) {
    return __uint_as_float(byte ? (unsigned)byte << 23 : 0x400000u);
}

// what one step needs of one tensor's count: lr / (1 - b1^t), 1 / sqrt(1 -
// b2^t), in 64 bits up to the last rounding
struct StepScalars {
    float decay, rate, root, clip;
};

// New 8-bit moments of one lane's 8 elements, the first n of them real.  The
// scales follow from the largest values of the warp's 256.
//
// RARE: some moment of the block is not finite, or a scale is the largest
// there is.  Values that are not finite then do not count for the scale and
// get the formats' own codes; and a value next to 2^128 does not round up to
// it (code 119 is 240 in e4m3 and 1.75 * 2^14 in e5m2).
template <bool RARE>
__device__ __forceinline__ void encode_moments(const float (&m)[8], const float (&v)[8], int n,
                                               unsigned mtop, unsigned vtop, unsigned index,
                                               unsigned key, uint2& mc, uint2& vc, int& mk,
                                               int& vk) {
    if constexpr (RARE) {
        mtop = vtop = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned mb = __float_as_uint(m[i]) & 0x7fffffffu;
            const unsigned vb = __float_as_uint(v[i]) & 0x7fffffffu;
            if (i < n && mb < 0x7f800000u) mtop = max(mtop, mb);
            if (i < n && vb < 0x7f800000u) vtop = max(vtop, vb);
        }
        mtop = __reduce_max_sync(0xffffffffu, mtop);
        vtop = __reduce_max_sync(0xffffffffu, vtop);
    }
    // 448 = 1.75 * 2^8 and 57344 = 1.75 * 2^15: the exponent of the largest
    // value, one more where its fraction is above 1.75
    mk = max(1, (int)((mtop + 0x1fffffu) >> 23) - 8);
    vk = max(1, (int)((vtop + 0x1fffffu) >> 23) - 15);
    const float mi = __uint_as_float((unsigned)(254 - mk) << 23);
    const float vi = __uint_as_float((unsigned)(254 - vk) << 23);
    unsigned a[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // the noise goes in below the last bit that is kept; the exponent's
        // bias changes with the same addition
        const unsigned h = mix32((index + i) ^ key);
        const unsigned mb = __float_as_uint(__fmul_rn(m[i], mi));
        const unsigned vb = __float_as_uint(__fmul_rn(v[i], vi));
        int c = (int)((mb & 0x7fffffffu) + ((h << 4) & 0xffff0u) + (8u - (120u << 23))) >> 20;
        int d = (int)(vb + ((h >> 11) & 0x1fffe0u) + (16u - (112u << 23))) >> 21;
        d = max(d, 4);
        if constexpr (RARE) {
            c = min(c, mk == 247 ? 119 : 126);
            d = min(d, vk == 240 ? 119 : 123);
        }
        a[i] = (unsigned)(c < 8 ? 0 : c) | ((mb >> 24) & 0x80u);
        b[i] = v[i] > 0.f ? (unsigned)d : 0u;
        if constexpr (RARE) {
            const unsigned vr = __float_as_uint(v[i]) & 0x7fffffffu;
            if ((__float_as_uint(m[i]) & 0x7fffffffu) >= 0x7f800000u) a[i] = 0x7fu;
            if (vr >= 0x7f800000u) b[i] = vr == 0x7f800000u ? 0x7cu : 0x7fu;
        }
    }
    mc = pack8(a);
    vc = pack8(b);
}

template <class T, int BITS>
__device__ __forceinline__ void update8(const OptTensor& t, long long base, const OptArgs& a,
                                        const StepScalars& s, unsigned key) {
    const long long left = t.n - base;
    const int n = left >= 8 ? 8 : (left > 0 ? (int)left : 0);
    const int full = n == 8 ? t.vec : 0;
    float g[8], p[8], m[8], v[8];
    load8(static_cast<const T*>(t.g) + base, full, n, g);
    if (t.master) load8(t.master + base, full, n, p);
    else load8(static_cast<const T*>(t.p) + base, full, n, p);
    const long long block = base / kOptBlock;
    if constexpr (BITS == 8) {
        const uint2 mc = load_codes(static_cast<const uint8_t*>(t.m) + base, full, n);
        const uint2 vc = load_codes(static_cast<const uint8_t*>(t.v) + base, full, n);
        // a lane behind the tensor's end may be behind the scales' end too.
        // The scales are powers of two: b (code s) = code (b s)
        const float ms = scale_of(n > 0 ? t.ms[block] : 1), vs = scale_of(n > 0 ? t.vs[block] : 1);
        decode8<__NV_E4M3>(mc, __fmul_rn(ms, a.b1), m);
        decode8<__NV_E5M2>(vc, __fmul_rn(vs, a.b2), v);
    } else {
        load8(static_cast<const float*>(t.m) + base, full, n, m);
        load8(static_cast<const float*>(t.v) + base, full, n, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            m[i] = __fmul_rn(m[i], a.b1);
            v[i] = __fmul_rn(v[i], a.b2);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float gi = __fmul_rn(g[i], s.clip);
        m[i] = __fadd_rn(m[i], __fmul_rn(gi, a.omb1));
        v[i] = __fadd_rn(v[i], __fmul_rn(__fmul_rn(gi, gi), a.omb2));
        // root and quotient to 2^-22: their last bits are far below the
        // update's own, and correctly rounded ones take half of the instructions
        const float d = __fadd_rn(__fmul_rn(sqrt_approx(v[i]), s.root), a.eps);
        p[i] = __fsub_rn(__fmul_rn(p[i], s.decay), __fmul_rn(__fdividef(m[i], d), s.rate));
    }
    if (t.master) store8(t.master + base, full, n, p);
    store8(static_cast<T*>(t.p) + base, full, n, p);
    if constexpr (BITS == 8) {
        // elements behind the end are zeros: they change no maximum
        unsigned mtop = 0, vtop = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            mtop = max(mtop, __float_as_uint(m[i]) & 0x7fffffffu);
            vtop = max(vtop, __float_as_uint(v[i]) & 0x7fffffffu);
        }
        mtop = __reduce_max_sync(0xffffffffu, mtop);
        vtop = __reduce_max_sync(0xffffffffu, vtop);
        uint2 mc, vc;
        int mk, vk;
        // above 1.75 * 2^127 the scales are the largest (or there is none)
        if (max(mtop, vtop) > 0x7f600000u)
            encode_moments<true>(m, v, n, mtop, vtop, (unsigned)base, key, mc, vc, mk, vk);
        else
            encode_moments<false>(m, v, n, mtop, vtop, (unsigned)base, key, mc, vc, mk, vk);
        store_codes(static_cast<uint8_t*>(t.m) + base, full, n, mc);
        store_codes(static_cast<uint8_t*>(t.v) + base, full, n, vc);
        if ((threadIdx.x & 31) == 0 && n > 0) {
            t.ms[block] = (uint8_t)mk;
            t.vs[block] = (uint8_t)vk;
        }
    } else {
        store8(static_cast<float*>(t.m) + base, full, n, m);
        store8(static_cast<float*>(t.v) + base, full, n, v);
    }
}

// the tensor that chunk c lies in: the last one whose first chunk is <= c
template <int N>
__device__ __forceinline__ int find_tensor(const OptTable<N>& tab, unsigned c) {
    int lo = 0, hi = tab.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tab.t[mid].chunk0 <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

struct ChunkPlan {
    int tensor;
    float rate, root;
    unsigned key;
};

template <int N, int BITS>
__global__ void __launch_bounds__(kThreads)
adamw_kernel(const __grid_constant__ OptTable<N> tab, const __grid_constant__ OptArgs a) {
    __shared__ ChunkPlan plan[kThreads];
    const double lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
    StepScalars s{};
    s.decay = (float)(1.0 - lr * a.wd);
    s.clip = 1.f;
    if (a.norm) {
        const double c = a.max_norm / (*a.norm + 1e-6);
        s.clip = c > 1.0 ? 1.f : (float)c;   // NaN stays NaN
    }
    // the CTA's chunks are one grid apart (neighbouring CTAs share DRAM pages).
    // What each of them needs of its tensor -- which one it is, powers of the
    // betas in 64 bits -- is worked out by one thread a chunk, a CTA's width of
    // chunks at a time
    for (unsigned c0 = blockIdx.x; c0 < tab.chunks; c0 += kThreads * gridDim.x) {
        __syncthreads();
        const unsigned long long mine = c0 + (unsigned long long)threadIdx.x * gridDim.x;
        if (mine < tab.chunks) {
            ChunkPlan q;
            q.tensor = find_tensor(tab, (unsigned)mine);
            const OptTensor& t = tab.t[q.tensor];
            const long long step = *t.step + 1;
            q.rate = (float)(lr / (1.0 - exp2((double)step * a.lb1)));
            q.root = (float)(1.0 / sqrt(1.0 - exp2((double)step * a.lb2)));
            q.key = BITS == 8 ? mix32(mix32(a.seed_key + (unsigned)step) + (unsigned)t.ordinal) : 0;
            plan[threadIdx.x] = q;
        }
        __syncthreads();
        unsigned c = c0;
        for (int k = 0; k < kThreads && c < tab.chunks; ++k, c += gridDim.x) {
            const ChunkPlan q = plan[k];
            const OptTensor& t = tab.t[q.tensor];
            const long long base = (long long)(c - t.chunk0) * kChunk + threadIdx.x * kLane;
            s.rate = q.rate;
            s.root = q.root;
            const unsigned key = BITS == 8 ? mix32(q.key + (unsigned)(base >> 32)) : 0;
            if (t.dtype == kOptF32) update8<float, BITS>(t, base, a, s, key);
            else if (t.dtype == kOptBf16) update8<__nv_bfloat16, BITS>(t, base, a, s, key);
            else update8<__half, BITS>(t, base, a, s, key);
        }
    }
    // every CTA has read the counts it needs: the last one to come here
    // advances them
    __shared__ unsigned order;
    __syncthreads();
    if (threadIdx.x == 0) order = atomicAdd(a.ticket, 1u);
    __syncthreads();
    if (order != gridDim.x - 1) return;
    for (int i = threadIdx.x; i < tab.count; i += kThreads) *tab.t[i].step += 1;
    if (threadIdx.x == 0) *a.ticket = 0;
}

// ---- sqrt(sum of squares over all gradients), summed in 64 bits in a fixed
// order: threads, warps, CTAs, launches
template <class T>
__device__ __forceinline__ void squares8(const T* p, long long base, long long size, int vec,
                                         double (&sum)[4]) {
    const long long left = size - base;
    const int n = left >= 8 ? 8 : (left > 0 ? (int)left : 0);
    float x[8];
    load8(p + base, n == 8 ? vec : 0, n, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i & 3] = fma((double)x[i], (double)x[i], sum[i & 3]);
}

__device__ __forceinline__ double cta_sum(double x) {
    __shared__ double part[kThreads / 32];
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x / 32] = x;
    __syncthreads();
    x = 0;
    for (int i = 0; i < kThreads / 32; ++i) x += part[i];
    return x;
}

template <int N>
__global__ void __launch_bounds__(kThreads)
norm_kernel(const __grid_constant__ OptTable<N> tab, double* partial, int first, int last,
            unsigned* ticket, double* norm, float* norm32) {
    __shared__ int tensor[kThreads];   // of the CTA's next chunks, as above
    double part[4] = {0, 0, 0, 0};
    for (unsigned c0 = blockIdx.x; c0 < tab.chunks; c0 += kThreads * gridDim.x) {
        __syncthreads();
        const unsigned long long mine = c0 + (unsigned long long)threadIdx.x * gridDim.x;
        if (mine < tab.chunks) tensor[threadIdx.x] = find_tensor(tab, (unsigned)mine);
        __syncthreads();
        unsigned c = c0;
#pragma unroll 2
        for (int k = 0; k < kThreads && c < tab.chunks; ++k, c += gridDim.x) {
            const OptTensor& t = tab.t[tensor[k]];
            const long long base = (long long)(c - t.chunk0) * kChunk + threadIdx.x * kLane;
            if (t.dtype == kOptF32) squares8(static_cast<const float*>(t.g), base, t.n, t.vec, part);
            else if (t.dtype == kOptBf16)
                squares8(static_cast<const __nv_bfloat16*>(t.g), base, t.n, t.vec, part);
            else squares8(static_cast<const __half*>(t.g), base, t.n, t.vec, part);
        }
    }
    double sum = (part[0] + part[1]) + (part[2] + part[3]);
    sum = cta_sum(sum);
    __shared__ unsigned order;
    if (threadIdx.x == 0) {
        partial[first + blockIdx.x] = sum;
        __threadfence();
        order = atomicAdd(ticket, 1u);
    }
    __syncthreads();
    if (order != gridDim.x - 1) return;
    __threadfence();
    if (threadIdx.x == 0) *ticket = 0;
    if (!last) return;
    sum = 0;
    const int n = first + gridDim.x;
    for (int i = threadIdx.x; i < n; i += kThreads) sum += __ldcg(partial + i);
    sum = cta_sum(sum);
    if (threadIdx.x == 0) {
        *norm = sqrt(sum);
        *norm32 = (float)sqrt(sum);
    }
}

// CTAs of one launch: all chunks at once up to what the SMs hold, then a loop
unsigned opt_grid(unsigned chunks, unsigned most) {
    return chunks < 1 ? 1 : (chunks < most ? chunks : most);
}

template <int N>
void fill(OptTable<N>* tab, const OptTensor* t, int count) {
    tab->count = count;
    unsigned c = 0;
    for (int i = 0; i < count; ++i) {
        tab->t[i] = t[i];
        tab->t[i].chunk0 = c;
        c += (unsigned)((t[i].n + kChunk - 1) / kChunk);
    }
    tab->chunks = c;
}

template <int N>
cudaError_t adamw_part(const OptTensor* t, int count, int bits, const OptArgs& a, cudaStream_t s) {
    OptTable<N> tab;
    fill(&tab, t, count);
    const unsigned grid = opt_grid(tab.chunks, kOptCtas);
    if (bits == 8) adamw_kernel<N, 8><<<grid, kThreads, 0, s>>>(tab, a);
    else adamw_kernel<N, 32><<<grid, kThreads, 0, s>>>(tab, a);
    return cudaGetLastError();
}

template <int N>
cudaError_t norm_part(const OptTensor* t, int count, double* partial, int* first, bool last,
                      unsigned* ticket, double* norm, float* norm32, cudaStream_t s) {
    OptTable<N> tab;
    fill(&tab, t, count);
    const unsigned grid = opt_grid(tab.chunks, kNormCtas);
    norm_kernel<N><<<grid, kThreads, 0, s>>>(tab, partial, *first, last ? 1 : 0, ticket, norm,
                                             norm32);
    *first += (int)grid;
    return cudaGetLastError();
}

// kernel parameters are copied with every launch: a short list takes a small
// table
constexpr int kSmall = 12, kMiddle = 100;

}  // namespace

cudaError_t launch_adamw(const OptTensor* t, int count, int bits, OptArgs a, cudaStream_t s) {
    a.seed_key = mix32(a.seed_key);
    if (count <= kSmall) return adamw_part<kSmall>(t, count, bits, a, s);
    if (count <= kMiddle) return adamw_part<kMiddle>(t, count, bits, a, s);
    return adamw_part<kOptTensors>(t, count, bits, a, s);
}

cudaError_t launch_grad_norm(const OptTensor* t, int count, double* partial, int* first, bool last,
                             unsigned* ticket, double* norm, float* norm32, cudaStream_t s) {
    if (count <= kSmall)
        return norm_part<kSmall>(t, count, partial, first, last, ticket, norm, norm32, s);
    if (count <= kMiddle)
        return norm_part<kMiddle>(t, count, partial, first, last, ticket, norm, norm32, s);
    return norm_part<kOptTensors>(t, count, partial, first, last, ticket, norm, norm32, s);
}

long long opt_chunks(long long n) { return (n + kChunk - 1) / kChunk; }

}  // namespace fcqt
