// AdamW over many tensors in one launch, moments in 32 or in 8 bits, and the
// global gradient norm that scales the gradients.
//
// For every element, in 32 bits, with t the tensor's own count of steps:
//   g' = g c                       c = min(1, max_norm / (norm + 1e-6)), or 1
//   m  = b1 m + (1 - b1) g'
//   v  = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// Each product and sum of m and v is rounded by itself (no fused multiply-add),
// so their bits do not depend on how a variant of the kernel is compiled.
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
//
// Every byte is touched once, so DRAM bounds the step: 144 M bf16 elements with
// a master copy 660 us (6.1 TB/s), 67 M floats with 8-bit moments 180 to 193 us
// (6.0 to 5.6 TB/s, from one GPU to another).  16-bit parameters with 8-bit moments
// move 10 bytes for 57 instructions an element, which would take as long as the
// bytes if they were issued without a pause, and stay at 4.3 TB/s (96 M elements,
// 221 us).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "internal.h"

namespace fcqt {

namespace {

constexpr int kLane = 8;                        // consecutive elements a thread
static_assert(32 * kLane == kOptBlock, "a warp is one block");
// CTA sizes.  Measured with 8-bit moments, 67 M float and 96 M bf16 elements: 181
// and 225 us with 7 CTAs of 128 threads an SM (72 registers), 190 and 233 with 3
// of 256, 192 and 233 with 4 of 192, 210 and 224 with 4 of 224, 221 and 315 with
// 4 of 256 (64 registers, spilled).  A table of more than 100 tensors takes 42 KB of
// shared memory and leaves room for 5 of the 7: 25 M bf16 elements with clipping
// 80 us as 100 tensors, 125 as 101.  32-bit moments move more bytes an element
// and want fewer threads: 144 M bf16 elements with a master copy 660 us with 16
// warps an SM, 675 with 24, 750 with 32.
template <int BITS>
constexpr int kStepThreads = BITS == 8 ? 128 : 256;
template <int BITS>
constexpr int kStepCtas = BITS == 8 ? 7 : 2;    // of an SM
constexpr int kNormThreads = 256;

template <int N>
struct OptTable {
    OptTensor t[N];
    int count;
    unsigned chunks;
};

// shifts and odd multipliers (the fractional bits of the square roots of 2
// and 3); every bit of the input reaches every bit of the output
__host__ __device__ __forceinline__ unsigned mix_first(unsigned x) { return x ^ (x >> 16); }
__host__ __device__ __forceinline__ unsigned mix_middle(unsigned x) {
    x *= 0x6A09E667u;
    x ^= x >> 15;
    return x * 0xBB67AE85u;
}
__host__ __device__ __forceinline__ unsigned mix32(unsigned x) {
    x = mix_middle(mix_first(x));
    return x ^ (x >> 16);
}

// Two 32-bit floats in one instruction (sm_100).  A product and a sum that takes
// it may come out as one fused operation, so what has to have the bits of two
// roundings is added with __fadd_rn.
struct F2 {
    unsigned long long w;
};
__device__ __forceinline__ F2 two(float a, float b) {
    F2 x;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x.w) : "f"(a), "f"(b));
    return x;
}
__device__ __forceinline__ F2 two(float a) { return two(a, a); }
__device__ __forceinline__ void split(F2 x, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.w));
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
    F2 x;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(x.w) : "l"(a.w), "l"(b.w));
    return x;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
    F2 x;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(x.w) : "l"(a.w), "l"(b.w));
    return x;
}

// the largest of three, NaN if one of them is
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

// ---- 8 consecutive values.  `vec`: all 8 are there, at an address that is a
// multiple of 32 (2) or 16 (1) bytes; else (0) the first n of them one by one,
// zeros behind.  They stay as loaded (Raw8) until they are needed: a load waits
// for nothing.
template <class T>
struct Raw8 {
    uint4 w;
};
template <>
struct Raw8<float> {
    float f[8];
};
__device__ __forceinline__ void load8(const float* p, int vec, int n, Raw8<float>& x) {
    if (vec == 2) {
        load_v8(p, x.f);
    } else if (vec) {
        const float4 a = reinterpret_cast<const float4*>(p)[0];
        const float4 b = reinterpret_cast<const float4*>(p)[1];
        x.f[0] = a.x; x.f[1] = a.y; x.f[2] = a.z; x.f[3] = a.w;
        x.f[4] = b.x; x.f[5] = b.y; x.f[6] = b.z; x.f[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x.f[i] = i < n ? p[i] : 0.f;
    }
}
template <class T>
__device__ __forceinline__ void load8(const T* p, int vec, int n, Raw8<T>& x) {
    if (vec) {
        x.w = *reinterpret_cast<const uint4*>(p);
    } else {
        const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
        unsigned w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) w[i / 2] |= (unsigned)h[i] << (16 * (i & 1));
        x.w = make_uint4(w[0], w[1], w[2], w[3]);
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
// 16-bit parameters are rounded once, to nearest even, from the 32-bit result
__device__ __forceinline__ void from_float(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_float(float x, __half& y) { y = __float2half_rn(x); }
template <class T>
__device__ __forceinline__ float2 pair_to_float(unsigned w) {
    if constexpr (std::is_same<T, __half>::value) {
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
__device__ __forceinline__ void unpack(const Raw8<float>& r, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = r.f[i];
}
template <class T>
__device__ __forceinline__ void unpack(const Raw8<T>& r, float (&x)[8]) {
    const unsigned u[4] = {r.w.x, r.w.y, r.w.z, r.w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = pair_to_float<T>(u[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
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
// square root and reciprocal to one unit in the last place
__device__ __forceinline__ float root_of(float x) {
    float y;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float one_over(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 8 values to codes, the first in the low byte
template <__nv_fp8_interpretation_t F>
__device__ __forceinline__ uint2 to_fp8(const float (&x)[8]) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * i], x[2 * i + 1]), __NV_SATFINITE, F);
    return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}
__device__ __forceinline__ void put_byte(uint2& c, int i, unsigned byte) {
    unsigned& w = i < 4 ? c.x : c.y;
    w = (w & ~(0xffu << (8 * (i & 3)))) | byte << (8 * (i & 3));
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
        split(two(f.x, f.y) * two(s), x[2 * i], x[2 * i + 1]);
    }
}
// 2^(byte - 127); a byte of 0 is the subnormal 2^-127
__device__ __forceinline__ float scale_of(uint8_t byte) {
    return __uint_as_float(byte ? (unsigned)byte << 23 : 0x400000u);
}

// 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t) and the gradients' factor
struct StepScalars {
    float decay, rate, root, clip;
};

// New 8-bit moments of one lane's 8 elements, the first n of them real, from
// the largest magnitudes of the warp's 256 (NaN where one of them is).
//
// A value over its scale gets its noise added below the last bit that is kept,
// as integers, and the bits below that cut off: the conversion to 8 bits then
// rounds nothing.
//
// RARE: some moment of the block is not finite, or a scale is the largest
// there is.  Values that are not finite then do not count for the scale and
// get the formats' own codes; and a value next to 2^128 does not round up to
// it (it stays at 240 in e4m3 and at 1.75 * 2^14 in e5m2).
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
    // mix32 of (index + i) ^ key for i < 8, index a multiple of 8: its first
    // step is the same for all of them
    const unsigned first = mix_first(index ^ key);
    float a[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        split(two(m[i], m[i + 1]) * two(mi), a[i], a[i + 1]);
        split(two(v[i], v[i + 1]) * two(vi), b[i], b[i + 1]);
#pragma unroll
        for (int j = i; j < i + 2; ++j) {
            const unsigned h = mix_middle(first ^ j);
            // the low and the high half of mix32's result (its last step folds
            // the high half into the low one), and half a step below
            const unsigned hm = (((h << 4) ^ (h >> 12)) & 0xffff0u) + 8u;
            const unsigned hv = ((h >> 11) & 0x1fffe0u) + 16u;
            a[j] = __uint_as_float((__float_as_uint(a[j]) + hm) & 0xfff00000u);
            b[j] = __uint_as_float((__float_as_uint(b[j]) + hv) & 0xffe00000u);
            if constexpr (RARE) {
                const float mmost = mk == 247 ? 240.f : 448.f, vmost = vk == 240 ? 28672.f : 57344.f;
                a[j] = fminf(fmaxf(a[j], -mmost), mmost);
                b[j] = fminf(b[j], vmost);
            }
        }
        // below the smallest normal value: 0 for m, that value for v.  |a| is at
        // most 1.875 * 2^-7 or at least 2^-6, its square 0.88 * 2^-12 or 2^-12:
        // a factor of 0 or 1, worked out beside the integer adders, which this
        // kernel has least of
        const F2 ai = two(a[i], a[i + 1]);
        float qa, qb, la, lb;
        split(ai * ai, qa, qb);
        qa = __saturatef(fmaf(qa, 0x1p40f, -0.94f * 0x1p28f));
        qb = __saturatef(fmaf(qb, 0x1p40f, -0.94f * 0x1p28f));
        split(ai * two(qa, qb), a[i], a[i + 1]);
        split(two(v[i], v[i + 1]) * two(0x1p100f) * two(0x1p100f), la, lb);
        b[i] = fmaxf(b[i], fminf(la, 0x1p-14f));
        b[i + 1] = fmaxf(b[i + 1], fminf(lb, 0x1p-14f));
    }
    mc = to_fp8<__NV_E4M3>(a);
    vc = to_fp8<__NV_E5M2>(b);
    if constexpr (RARE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned vr = __float_as_uint(v[i]) & 0x7fffffffu;
            if ((__float_as_uint(m[i]) & 0x7fffffffu) >= 0x7f800000u) put_byte(mc, i, 0x7fu);
            if (vr >= 0x7f800000u) put_byte(vc, i, vr == 0x7f800000u ? 0x7cu : 0x7fu);
        }
    }
}

// one thread's elements of one chunk, as loaded.  MASTER: the parameter's value
// is its 32-bit copy
template <class T, int BITS, bool MASTER>
struct Chunk {
    using P = typename std::conditional<MASTER, float, T>::type;
    long long base;
    Raw8<T> g;
    Raw8<P> p;
    Raw8<float> m, v;   // BITS 32
    uint2 mc, vc;       // BITS 8

    __device__ __forceinline__ void load(const OptTensor& t, long long at, int n, int vec) {
        base = at;
        load8(static_cast<const T*>(t.g) + base, vec, n, g);
        load8((MASTER ? reinterpret_cast<const P*>(t.master) : static_cast<const P*>(t.p)) + base,
              vec, n, p);
        if constexpr (BITS == 8) {
            mc = load_codes(static_cast<const uint8_t*>(t.m) + base, vec, n);
            vc = load_codes(static_cast<const uint8_t*>(t.v) + base, vec, n);
        } else {
            load8(static_cast<const float*>(t.m) + base, vec, n, m);
            load8(static_cast<const float*>(t.v) + base, vec, n, v);
        }
    }
};

// EXACT: the denominator and the quotient as the formula says, each rounded
// once (see launch_adamw)
template <class T, int BITS, bool MASTER, bool EXACT>
__device__ __forceinline__ void update8(const OptTensor& t, const Chunk<T, BITS, MASTER>& c,
                                        const OptArgs& a, const StepScalars& s, unsigned key,
                                        int n, int vec, uint8_t* ms, uint8_t* vs) {
    float g[8], p[8], m[8], v[8];
    unpack(c.g, g);
    unpack(c.p, p);
    if constexpr (BITS == 8) {
        // the scales are powers of two: b (code s) = code (b s)
        decode8<__NV_E4M3>(c.mc, __fmul_rn(scale_of(*ms), a.b1), m);
        decode8<__NV_E5M2>(c.vc, __fmul_rn(scale_of(*vs), a.b2), v);
    } else {
        unpack(c.m, m);
        unpack(c.v, v);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            split(two(m[i], m[i + 1]) * two(a.b1), m[i], m[i + 1]);
            split(two(v[i], v[i + 1]) * two(a.b2), v[i], v[i + 1]);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const F2 gi = two(g[i], g[i + 1]) * two(s.clip);
        // the sums one by one: a sum of packed products would be fused with
        // them, and the moments' bits are those of separate roundings
        float qa, qb, ra, rb;
        split(gi * two(a.omb1), qa, qb);
        m[i] = __fadd_rn(m[i], qa);
        m[i + 1] = __fadd_rn(m[i + 1], qb);
        split(gi * gi * two(a.omb2), ra, rb);
        v[i] = __fadd_rn(v[i], ra);
        v[i + 1] = __fadd_rn(v[i + 1], rb);
        if constexpr (EXACT) {
#pragma unroll
            for (int j = i; j < i + 2; ++j) {
                const float d = __fadd_rn(__fmul_rn(__fsqrt_rn(v[j]), s.root), a.eps);
                p[j] = __fadd_rn(__fmul_rn(p[j], s.decay), __fmul_rn(-s.rate, __fdiv_rn(m[j], d)));
            }
            continue;
        }
        // root and reciprocal to 2^-23: their last bits are far below the
        // parameter's own, and correctly rounded ones took a third of all
        // instructions.  2^-126 under the root keeps what is subnormal
        // from being read as 0; it moves the root by 2^-63 at most.
        float da, db;
        split(two(v[i], v[i + 1]) + two(0x1p-126f), ra, rb);
        split(two(root_of(ra), root_of(rb)) * two(s.root) + two(a.eps), da, db);
        const F2 step = two(m[i], m[i + 1]) * two(one_over(da), one_over(db)) * two(-s.rate);
        split(two(p[i], p[i + 1]) * two(s.decay) + step, p[i], p[i + 1]);
    }
    uint2 mc, vc;
    int mk, vk;
    if constexpr (BITS == 8) {
        // elements behind the end are zeros: they change no maximum
        float mmax = 0.f, vmax = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            mmax = max_nan(mmax, fabsf(m[i]), fabsf(m[i + 1]));
            vmax = max_nan(vmax, v[i], v[i + 1]);
        }
        const unsigned mtop = __reduce_max_sync(0xffffffffu, __float_as_uint(mmax));
        const unsigned vtop = __reduce_max_sync(0xffffffffu, __float_as_uint(vmax));
        // above 1.75 * 2^127 the scales are the largest (or there is none)
        if (max(mtop, vtop) > 0x7f600000u)
            encode_moments<true>(m, v, n, mtop, vtop, (unsigned)c.base, key, mc, vc, mk, vk);
        else
            encode_moments<false>(m, v, n, mtop, vtop, (unsigned)c.base, key, mc, vc, mk, vk);
    }
    if constexpr (MASTER) store8(t.master + c.base, vec, n, p);
    store8(static_cast<T*>(t.p) + c.base, vec, n, p);
    if constexpr (BITS == 8) {
        store_codes(static_cast<uint8_t*>(t.m) + c.base, vec, n, mc);
        store_codes(static_cast<uint8_t*>(t.v) + c.base, vec, n, vc);
        if ((threadIdx.x & 31) == 0) {
            *ms = (uint8_t)mk;
            *vs = (uint8_t)vk;
        }
    } else {
        store8(static_cast<float*>(t.m) + c.base, vec, n, m);
        store8(static_cast<float*>(t.v) + c.base, vec, n, v);
    }
}

// a chunk that the tensor ends in, or whose arrays are not aligned
template <class T, int BITS, bool MASTER, bool EXACT>
__device__ __forceinline__ void update_part(const OptTensor& t, long long base, const OptArgs& a,
                                            const StepScalars& s, unsigned key, uint8_t* ms,
                                            uint8_t* vs) {
    const long long left = t.n - base;
    const int n = left >= 8 ? 8 : (left > 0 ? (int)left : 0);
    const int vec = n == 8 ? t.vec : 0;
    Chunk<T, BITS, MASTER> c;
    c.load(t, base, n, vec);
    update8<T, BITS, MASTER, EXACT>(t, c, a, s, key, n, vec, ms, vs);
}

constexpr int kWhole = 1 << 30;   // every thread has 8 aligned elements

// the chunks of a tensor before this one have all their elements, aligned
__device__ __forceinline__ unsigned whole_end(const OptTensor& t, int chunk) {
    return t.chunk0 + (t.vec == 2 ? (unsigned)(t.n / chunk) : 0);
}

// The table rides in the kernel's parameters and is copied to shared memory with
// ordinary loads, all of them at once: read as constants, 80 tensors' entries
// miss the constant cache one after the other (10 us before the first chunk).
template <int N>
__device__ __forceinline__ void copy_table(const OptTable<N>& tab, OptTensor* to) {
    static_assert(sizeof(OptTensor) % 8 == 0, "copied in words of 64 bits");
    const unsigned long long* from = reinterpret_cast<const unsigned long long*>(tab.t);
    unsigned long long* words = reinterpret_cast<unsigned long long*>(to);
    for (int i = threadIdx.x; i < tab.count * (int)(sizeof(OptTensor) / 8); i += blockDim.x) {
        unsigned long long w;
        asm volatile("ld.u64 %0, [%1];" : "=l"(w) : "l"(from + i));
        words[i] = w;
    }
}

// the tensor that chunk c lies in: the last one whose first chunk is <= c
__device__ __forceinline__ int find_tensor(const OptTensor* table, int count, unsigned c) {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (table[mid].chunk0 <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

struct TensorPlan {
    float rate, root;
    unsigned key;
    unsigned chunk0;
};

template <int N, class T, int BITS, bool MASTER, bool EXACT>
__global__ void __launch_bounds__(kStepThreads<BITS>, kStepCtas<BITS>)
adamw_kernel(const __grid_constant__ OptTable<N> tab, const __grid_constant__ OptArgs a) {
    constexpr int kThreads = kStepThreads<BITS>, kChunk = kThreads * kLane;
    __shared__ __align__(8) OptTensor table[N];
    __shared__ TensorPlan tensor[N];
    __shared__ int chunk[kThreads];      // tensor of each of the CTA's next chunks, and kWhole
    __shared__ uint8_t scale[2][BITS == 8 ? kThreads * (kThreads / 32) : 1];
    __shared__ long long steps[N];
    __shared__ StepScalars same;
    __shared__ unsigned order;
    // The CTA's chunks are one grid apart (neighbouring CTAs share DRAM pages).
    // The next one is on its way while one is computed, and the first one while
    // what follows works out the scalars.
    Chunk<T, BITS, MASTER> here;
    const long long lane = threadIdx.x * kLane;
    copy_table(tab, table);
    __syncthreads();
    const int first = find_tensor(table, tab.count, blockIdx.x);
    if (blockIdx.x < whole_end(table[first], kChunk))
        here.load(table[first], (long long)(blockIdx.x - table[first].chunk0) * kChunk + lane, 8, 2);
    if (threadIdx.x == kThreads - 1) {
        if (a.norm) pdl_wait();   // what else this kernel reads, the norm's does not write
        same.decay = (float)(1.0 - (a.lr_dev ? (double)*a.lr_dev : a.lr) * a.wd);
        const double c = a.norm ? a.max_norm / (*a.norm + 1e-6) : 1.0;
        same.clip = c > 1.0 ? 1.f : (float)c;   // NaN stays NaN
    }
    // 1 - b^t = -expm1(t ln b), which 32 bits hold to 2^-22 for every t
    const float lr = a.lr_dev ? *a.lr_dev : (float)a.lr;
    for (int i = threadIdx.x; i < tab.count; i += kThreads) {
        const OptTensor& t = table[i];
        const long long step = *t.step + 1;
        TensorPlan q;
        q.rate = lr / -expm1f((float)step * a.ln1);
        q.root = rsqrtf(-expm1f((float)step * a.ln2));
        q.key = BITS == 8 ? mix32(mix32(a.seed_key + (unsigned)step) + (unsigned)t.ordinal) : 0;
        q.chunk0 = t.chunk0;
        tensor[i] = q;
        steps[i] = step;
    }
    // tensors are looked up by one thread a chunk, a CTA's width at a time (the
    // last one of a width is the first of the next).  The scale bytes of a width
    // are read and written together: a byte at a time from every warp, 32 of
    // them to a sector of the L2 cache, cost a quarter of the kernel's time.
    constexpr unsigned kWidth = kThreads - 1;
    constexpr int kWarps = kThreads / 32;
    for (unsigned c0 = blockIdx.x; c0 < tab.chunks; c0 += kWidth * gridDim.x) {
        __syncthreads();
        const unsigned long long mine = c0 + (unsigned long long)threadIdx.x * gridDim.x;
        if (mine < tab.chunks) {
            const int i = find_tensor(table, tab.count, (unsigned)mine);
            chunk[threadIdx.x] = i | ((unsigned)mine < whole_end(table[i], kChunk) ? kWhole : 0);
        }
        __syncthreads();
        const unsigned left = (tab.chunks - c0 - 1) / gridDim.x + 1;
        const unsigned width = left < kWidth ? left : kWidth;
        // calls f(place in shared memory, tensor, block) for every block
        const auto each_block = [&](auto f) {
            for (unsigned i = threadIdx.x; i < width * kWarps; i += kThreads) {
                const unsigned k = i / kWarps, w = i - k * kWarps;
                const OptTensor& t = table[chunk[k] & ~kWhole];
                const long long block = (long long)(c0 + k * gridDim.x - t.chunk0) * kWarps + w;
                if (block * kOptBlock < t.n) f(i, t, block);
            }
        };
        if constexpr (BITS == 8) {
            each_block([&](unsigned i, const OptTensor& t, long long block) {
                scale[0][i] = t.ms[block];
                scale[1][i] = t.vs[block];
            });
            __syncthreads();
        }
        StepScalars s = same;
        unsigned c = c0;
        for (unsigned k = 0; k < width; ++k, c += gridDim.x) {
            const int i = chunk[k];
            const OptTensor& t = table[i & ~kWhole];
            const TensorPlan q = tensor[i & ~kWhole];
            s.rate = q.rate;
            s.root = q.root;
            const bool more = c + gridDim.x < tab.chunks;
            const int j = more ? chunk[k + 1] : 0;
            Chunk<T, BITS, MASTER> next;
            if (j & kWhole) {
                const OptTensor& u = table[j & ~kWhole];
                next.load(u, (long long)(c + gridDim.x - u.chunk0) * kChunk + lane, 8, 2);
            }
            const long long base = (long long)(c - q.chunk0) * kChunk + lane;
            const unsigned key = BITS == 8 ? mix32(q.key + (unsigned)(base >> 32)) : 0;
            uint8_t* ms = &scale[0][BITS == 8 ? k * kWarps + threadIdx.x / 32 : 0];
            uint8_t* vs = &scale[1][BITS == 8 ? k * kWarps + threadIdx.x / 32 : 0];
            if (i & kWhole) update8<T, BITS, MASTER, EXACT>(t, here, a, s, key, 8, 2, ms, vs);
            else update_part<T, BITS, MASTER, EXACT>(t, base, a, s, key, ms, vs);
            here = next;
        }
        if constexpr (BITS == 8) {
            __syncthreads();
            each_block([&](unsigned i, const OptTensor& t, long long block) {
                t.ms[block] = scale[0][i];
                t.vs[block] = scale[1][i];
            });
        }
    }
    // every CTA has read the counts: the last one to come here advances them
    __syncthreads();
    if (threadIdx.x == 0) order = atomicAdd(a.ticket, 1u);
    __syncthreads();
    if (order != gridDim.x - 1) return;
    for (int i = threadIdx.x; i < tab.count; i += kThreads) *table[i].step = steps[i];
    if (threadIdx.x == 0) *a.ticket = 0;
}

// ---- sqrt(sum of squares over all gradients), summed in 64 bits in a fixed
// order: threads, warps, CTAs, launches.  Bound by what its start and its end cost
// and by loads on their way: 210 MB take 46 us (4.6 TB/s), 50 MB 16, nothing 4.

// elements of a chunk: 32 bytes a thread, so that 16-bit gradients have as many
// bytes on their way as 32-bit ones
__host__ __device__ constexpr int norm_chunk(int dtype) {
    return kNormThreads * (dtype == kOptF32 ? 8 : 16);
}

__device__ __forceinline__ void add_square(float x, double& sum) {
    sum = fma((double)x, (double)x, sum);
}

// a thread's elements of chunk `chunk` of a tensor, some of them or none
template <class T>
__device__ __forceinline__ void squares(const OptTensor& t, long long chunk, bool whole,
                                        double (&sum)[4]) {
    constexpr int kEach = 32 / sizeof(T);
    const long long base = (chunk * kNormThreads + threadIdx.x) * kEach;
    const T* g = static_cast<const T*>(t.g) + base;
    if (whole) {
        float w[8];
        load_v8(reinterpret_cast<const float*>(g), w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (sizeof(T) == 4) {
                add_square(w[i], sum[i & 3]);
            } else {
                const float2 f = pair_to_float<T>(__float_as_uint(w[i]));
                add_square(f.x, sum[i & 1]);
                add_square(f.y, sum[2 + (i & 1)]);
            }
        }
    } else {
        for (int k = 0; k < kEach; k += 8) {
            const long long left = t.n - base - k;
            const int n = left >= 8 ? 8 : (left > 0 ? (int)left : 0);
            Raw8<T> r;
            float x[8];
            load8(g + k, n == 8 ? t.vec : 0, n, r);
            unpack(r, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) add_square(x[i], sum[i & 3]);
        }
    }
}

__device__ __forceinline__ double cta_sum(double x) {
    __shared__ double part[kNormThreads / 32];
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x / 32] = x;
    __syncthreads();
    x = 0;
    for (int i = 0; i < kNormThreads / 32; ++i) x += part[i];
    return x;
}

template <int N>
__global__ void __launch_bounds__(kNormThreads, kNormCtas / 148)
norm_kernel(const __grid_constant__ OptTable<N> tab, double* partial, int first, int last,
            unsigned* ticket, double* norm, float* norm32) {
    __shared__ __align__(8) OptTensor table[N];
    __shared__ int tensor[kNormThreads];   // of each of the CTA's next chunks, and kWhole
    pdl_launch_dependents();
    copy_table(tab, table);
    double part[4] = {0, 0, 0, 0};
    for (unsigned c0 = blockIdx.x; c0 < tab.chunks; c0 += kNormThreads * gridDim.x) {
        __syncthreads();
        const unsigned long long mine = c0 + (unsigned long long)threadIdx.x * gridDim.x;
        if (mine < tab.chunks) {
            const int i = find_tensor(table, tab.count, (unsigned)mine);
            tensor[threadIdx.x] = i | ((unsigned)mine < whole_end(table[i], norm_chunk(table[i].dtype)) ? kWhole : 0);
        }
        __syncthreads();
        unsigned c = c0;
        for (int k = 0; k < kNormThreads && c < tab.chunks; ++k, c += gridDim.x) {
            const int i = tensor[k];
            const OptTensor& t = table[i & ~kWhole];
            const long long at = (long long)(c - t.chunk0);
            if (t.dtype == kOptF32) squares<float>(t, at, i & kWhole, part);
            else if (t.dtype == kOptBf16) squares<__nv_bfloat16>(t, at, i & kWhole, part);
            else squares<__half>(t, at, i & kWhole, part);
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
    for (int i = threadIdx.x; i < n; i += kNormThreads) sum += __ldcg(partial + i);
    sum = cta_sum(sum);
    if (threadIdx.x == 0) {
        *norm = sqrt(sum);
        *norm32 = (float)sqrt(sum);
    }
}

// CTAs of one launch: one a chunk, up to what the SMs hold at a time
unsigned opt_grid(unsigned chunks, unsigned most) {
    return chunks < 1 ? 1 : (chunks < most ? chunks : most);
}

template <int N>
void fill(OptTable<N>* tab, const OptTensor* t, int count, int chunk_of) {
    tab->count = count;
    unsigned c = 0;
    for (int i = 0; i < count; ++i) {
        const int chunk = chunk_of ? chunk_of : norm_chunk(t[i].dtype);   // 0: the norm's
        tab->t[i] = t[i];
        tab->t[i].chunk0 = c;
        c += (unsigned)((t[i].n + chunk - 1) / chunk);
    }
    tab->chunks = c;
}

// CTAs of a kernel that the GPU holds at a time (asked once)
template <class K>
unsigned resident_ctas(K kernel, int threads) {
    int device = 0, sms = 148, per_sm = 1;
    if (cudaGetDevice(&device) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, 0) != cudaSuccess ||
        per_sm < 1) {
        cudaGetLastError();
        return 148;
    }
    return (unsigned)(sms * per_sm);
}

template <int N, class T, int BITS, bool MASTER, bool EXACT>
cudaError_t adamw_launch(const OptTensor* t, int count, const OptArgs& a, cudaStream_t s) {
    constexpr int kThreads = kStepThreads<BITS>;
    OptTable<N> tab;
    fill(&tab, t, count, kThreads * kLane);
    const auto kernel = adamw_kernel<N, T, BITS, MASTER, EXACT>;
    static const unsigned most = resident_ctas(kernel, kThreads);
    // right behind the norm, the kernel may start on what the norm leaves free
    return launch_pdl(a.behind_norm, kernel, dim3(opt_grid(tab.chunks, most)), dim3(kThreads), 0, s,
                      tab, a);
}

template <int N, bool EXACT, class T, bool MASTER>
cudaError_t adamw_part(const OptTensor* t, int count, int bits, const OptArgs& a, cudaStream_t s) {
    return bits == 8 ? adamw_launch<N, T, 8, MASTER, EXACT>(t, count, a, s)
                     : adamw_launch<N, T, 32, MASTER, EXACT>(t, count, a, s);
}

template <int N, bool EXACT>
cudaError_t adamw_typed(const OptTensor* t, int count, int bits, const OptArgs& a, cudaStream_t s) {
    if (t->dtype == kOptF32) return adamw_part<N, EXACT, float, false>(t, count, bits, a, s);
    if (t->dtype == kOptBf16)
        return t->master ? adamw_part<N, EXACT, __nv_bfloat16, true>(t, count, bits, a, s)
                         : adamw_part<N, EXACT, __nv_bfloat16, false>(t, count, bits, a, s);
    return t->master ? adamw_part<N, EXACT, __half, true>(t, count, bits, a, s)
                     : adamw_part<N, EXACT, __half, false>(t, count, bits, a, s);
}

template <int N>
cudaError_t norm_part(const OptTensor* t, int count, double* partial, int* first, bool last,
                      unsigned* ticket, double* norm, float* norm32, cudaStream_t s) {
    OptTable<N> tab;
    fill(&tab, t, count, 0);
    const unsigned grid = opt_grid(tab.chunks, kNormCtas);
    norm_kernel<N><<<grid, kNormThreads, 0, s>>>(tab, partial, *first, last ? 1 : 0, ticket, norm,
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
    // sqrt(v + 2^-126) is off by 2^-63 at most, so the denominator by 2^-63 /
    // sqrt(1 - b2) (its bias correction at t = 1): under 2^-28 of eps, a sixteenth
    // of a rounding, if eps is at least 2^-35 / sqrt(1 - b2) (9.2e-10 for b2 =
    // 0.999).  Above 2^100 the reciprocal would come near to underflowing.  Other
    // values of eps, which training has little use for, take the exact operations:
    // as fast with 32-bit moments (302 us for 67 M floats), 234 us instead of 179
    // with 8-bit ones, 310 instead of 221 for 96 M bf16 elements with those.
    if (!(a.eps >= 0x1p-35 / sqrt(1.0 - a.beta2) && a.eps <= 0x1p100))
        return adamw_typed<kOptTensors, true>(t, count, bits, a, s);
    if (count <= kSmall) return adamw_typed<kSmall, false>(t, count, bits, a, s);
    if (count <= kMiddle) return adamw_typed<kMiddle, false>(t, count, bits, a, s);
    return adamw_typed<kOptTensors, false>(t, count, bits, a, s);
}

cudaError_t launch_grad_norm(const OptTensor* t, int count, double* partial, int* first, bool last,
                             unsigned* ticket, double* norm, float* norm32, cudaStream_t s) {
    if (count <= kSmall)
        return norm_part<kSmall>(t, count, partial, first, last, ticket, norm, norm32, s);
    if (count <= kMiddle)
        return norm_part<kMiddle>(t, count, partial, first, last, ticket, norm, norm32, s);
    return norm_part<kOptTensors>(t, count, partial, first, last, ticket, norm, norm32, s);
}

// (of the smallest kind)
long long opt_chunks(long long n) {
    constexpr int least = kStepThreads<8> * kLane;
    return (n + least - 1) / least;
}

}  // namespace fcqt
