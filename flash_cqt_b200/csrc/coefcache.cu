// Coefficient cache: the newest slices of a set of streams, held in 8 bits.
//
// Every stream has a ring of `capacity` slices; slice number k of a stream
// lies in slot k mod capacity.  A slice is the heap of its ncoef complex
// coefficients, two codes each.  16 consecutive coefficients (32 codes; no
// band is shorter) share a scale 2^e, one byte e + 127, the least that brings
// the largest finite magnitude to the format's largest or below:
//   int8: code = round(x 2^-e) in [-127, 127], -128 for a value that is not
//         finite;    e4m3: the nearest e4m3 value of x 2^-e, its NaN likewise.
// Scaling by powers of two is exact, so a value is rounded once (to nearest
// even) when it is written, and reading it back in 32 or 16 bits (bf16)
// rounds nothing.
//
// Both kernels move bytes and do little else.  A thread takes 4 coefficients
// (32 bytes of complex64, 8 bytes of codes); 4 lanes share a scale.  Work is
// cut into units of one tile of one slice; a stream's length is read on the
// device, so a captured graph follows it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "internal.h"

namespace fcqt {

namespace {

constexpr int kThreads = 256;
constexpr int kQuads = 2;                            // quads of a thread in one unit
constexpr int kTile = kThreads * kQuads;             // quads (4 coefficients) of a unit

struct Place {          // where a quad lies in the groups' tensors
    int group;
    long long at;       // offset in complex values
};

__device__ __forceinline__ Place place(const CacheGroups& gr, int j, long long row, long long slice) {
    int g = 0;
#pragma unroll
    for (int step = kMaxGroups / 2; step; step >>= 1)
        if (g + step < gr.count && j >= gr.off[g + step]) g += step;
    const int k = j - gr.off[g];
    const int band = k >> gr.shift[g], t = k & ((1 << gr.shift[g]) - 1);
    return {g, row * gr.row[g] + slice * gr.slice[g] + band * gr.band[g] + t};
}

__device__ __forceinline__ unsigned slot_of(long long number, int capacity) {
    const unsigned long long n = (unsigned long long)number;
    return n >> 32 ? (unsigned)(n % (unsigned)capacity) : (unsigned)n % (unsigned)capacity;
}

template <bool INT8>
__device__ __forceinline__ uint2 encode(const float (&x)[8], int& e) {
    unsigned top = 0;
    bool fine = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned b = __float_as_uint(x[i]) & 0x7fffffffu;
        if (b < 0x7f800000u) top = max(top, b);
        else fine = false;
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 127 = (1 + 63/64) 2^6 and 448 = 1.75 2^8: the exponent of the largest
    // value, one more where its fraction is above the format's
    e = INT8 ? (int)((top + 0x1ffffu) >> 23) - 6 : (int)((top + 0x1fffffu) >> 23) - 8;
    e = max(e, 1);
    const float inv = __uint_as_float((unsigned)(254 - e) << 23);
    // at the largest scale a value next to 2^128 must not round up to it
    const float most = INT8 ? (e == 249 ? 63.f : 127.f) : (e == 247 ? 240.f : 448.f);
    uint2 c;
    if constexpr (INT8) {
        unsigned b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // adding 1.5 * 2^23 rounds to the nearest integer, which the low
            // bits then hold in two's complement
            const float y = fminf(fmaxf(__fmul_rn(x[i], inv), -most), most);
            b[i] = __float_as_uint(__fadd_rn(y, 12582912.f));
            if (!fine && (__float_as_uint(x[i]) & 0x7fffffffu) >= 0x7f800000u) b[i] = 0x80u;
        }
        c.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
        c.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
    } else {
        unsigned h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float2 f = make_float2(fminf(fmaxf(__fmul_rn(x[2 * i], inv), -most), most),
                                   fminf(fmaxf(__fmul_rn(x[2 * i + 1], inv), -most), most));
            if (!fine) {   // infinities would be held as the largest value, NaN too
                const float nan = __int_as_float(0x7fffffff);
                if (!isfinite(x[2 * i])) f.x = nan;
                if (!isfinite(x[2 * i + 1])) f.y = nan;
            }
            h[i] = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
        }
        c.x = h[0] | h[1] << 16;
        c.y = h[2] | h[3] << 16;
    }
    return c;
}

template <bool INT8>
__device__ __forceinline__ void decode(uint2 c, uint8_t e, float (&x)[8]) {
    const float s = __uint_as_float(e ? (unsigned)e << 23 : 0x400000u);
    if constexpr (INT8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // the code plus 128 in the low bits of 2^23
            const unsigned w = (i < 4 ? c.x : c.y) ^ 0x80808080u;
            const float f = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | (i & 3)));
            x[i] = f == 8388608.f ? __int_as_float(0x7fffffff) : (f - 8388736.f) * s;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned w = i < 2 ? c.x : c.y;
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
                (__nv_fp8x2_storage_t)((i & 1) ? w >> 16 : w & 0xffffu), __NV_E4M3);
            const float2 f = __half22float2(__half2(h));
            x[2 * i] = f.x * s;
            x[2 * i + 1] = f.y * s;
        }
    }
}

struct Unit {
    unsigned tile, slice, row;
};
__device__ __forceinline__ Unit unit_of(unsigned u, unsigned tiles, unsigned slices) {
    const unsigned rs = u / tiles;
    return {u - rs * tiles, rs % slices, rs / slices};
}

template <bool INT8>
__global__ void __launch_bounds__(kThreads)
append_kernel(const __grid_constant__ CacheStore st, const __grid_constant__ CacheGroups gr,
              int slices, const long long* counts, unsigned units) {
    const unsigned tiles = (unsigned)(st.ncoef / 4 + kTile - 1) / kTile;
    for (unsigned u = blockIdx.x; u < units; u += gridDim.x) {
        const Unit w = unit_of(u, tiles, slices);
        long long count = counts ? counts[w.row] : slices;
        count = count < 0 ? 0 : (count > slices ? slices : count);
        // slices behind the stream's last one are left out, and so are those
        // that newer ones of this call would overwrite
        if (w.slice >= count || (long long)w.slice + st.capacity < count) continue;
        const long long length = max(st.length[w.row], 0ll);
        const long long at = (long long)w.row * st.capacity + slot_of(length + w.slice, st.capacity);
        uint2* codes = reinterpret_cast<uint2*>(st.codes + at * 2 * st.ncoef);
        uint8_t* scales = st.scales + at * (st.ncoef / 16);
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
            const int q = w.tile * kTile + i * kThreads + threadIdx.x;
            const bool in = q < st.ncoef / 4;   // ncoef is a multiple of 16: 4 lanes agree
            float x[8] = {};
            if (in) {
                const Place p = place(gr, 4 * q, w.row, w.slice);
                const float2* src = static_cast<const float2*>(gr.data[p.group]) + p.at;
                if (gr.wide) {
                    const float4 a = reinterpret_cast<const float4*>(src)[0];
                    const float4 b = reinterpret_cast<const float4*>(src)[1];
                    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
                    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float2 a = src[k];
                        x[2 * k] = a.x;
                        x[2 * k + 1] = a.y;
                    }
                }
            }
            int e;
            const uint2 c = encode<INT8>(x, e);
            if (in) {
                codes[q] = c;
                if ((threadIdx.x & 3) == 0) scales[q / 4] = (uint8_t)e;
            }
        }
    }
    // every CTA has read the lengths: the last one to come here advances them
    __shared__ unsigned order;
    __syncthreads();
    if (threadIdx.x == 0) order = atomicAdd(st.ticket, 1u);
    __syncthreads();
    if (order != gridDim.x - 1) return;
    for (int r = threadIdx.x; r < st.rows; r += kThreads) {
        long long count = counts ? counts[r] : slices;
        count = count < 0 ? 0 : (count > slices ? slices : count);
        st.length[r] = max(st.length[r], 0ll) + count;
    }
    if (threadIdx.x == 0) *st.ticket = 0;
}

__device__ __forceinline__ void store_quad(float* dst, const float (&x)[8]) {
    reinterpret_cast<float4*>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store_quad(__nv_bfloat16* dst, const float (&x)[8]) {
    alignas(16) __nv_bfloat16 h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = __float2bfloat16_rn(x[i]);
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(h);
}
__device__ __forceinline__ void store_quad(__half* dst, const float (&x)[8]) {
    alignas(16) __half h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = __float2half_rn(x[i]);
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(h);
}

template <bool INT8, class T>
__global__ void __launch_bounds__(kThreads)
window_kernel(const __grid_constant__ CacheStore st, const __grid_constant__ CacheGroups gr,
              int slices, const long long* ends, unsigned units) {
    const unsigned tiles = (unsigned)(st.ncoef / 4 + kTile - 1) / kTile;
    for (unsigned u = blockIdx.x; u < units; u += gridDim.x) {
        const Unit w = unit_of(u, tiles, slices);
        const long long length = st.length[w.row];
        const long long end = ends ? ends[w.row] : length;
        const long long number = end - slices + w.slice;
        const bool held = number >= 0 && number < length && number >= length - st.capacity;
        const long long at =
            (long long)w.row * st.capacity + (held ? slot_of(number, st.capacity) : 0);
        const uint2* codes = reinterpret_cast<const uint2*>(st.codes + at * 2 * st.ncoef);
        const uint8_t* scales = st.scales + at * (st.ncoef / 16);
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
            const int q = w.tile * kTile + i * kThreads + threadIdx.x;
            if (q >= st.ncoef / 4) continue;
            float x[8] = {};
            if (held) decode<INT8>(codes[q], scales[q / 4], x);
            const Place p = place(gr, 4 * q, w.row, w.slice);
            store_quad(static_cast<T*>(gr.data[p.group]) + 2 * p.at, x);
        }
    }
}

// CTAs: every unit at once up to eight CTAs an SM, then a loop
unsigned cache_units(const CacheStore& st, int slices) {
    const unsigned tiles = (unsigned)(st.ncoef / 4 + kTile - 1) / kTile;
    return tiles * (unsigned)slices * (unsigned)st.rows;
}
unsigned cache_grid(unsigned units) {
    constexpr unsigned most = 148 * 8;
    return units < most ? units : most;
}

}  // namespace

long long cache_unit_count(const CacheStore& st, long long slices) {
    return (long long)((st.ncoef / 4 + kTile - 1) / kTile) * slices * st.rows;
}

cudaError_t launch_cache_append(const CacheStore& st, const CacheGroups& gr, int slices,
                                const long long* counts, cudaStream_t s) {
    const unsigned units = cache_units(st, slices);
    if (units == 0) return cudaSuccess;
    if (st.int8) append_kernel<true><<<cache_grid(units), kThreads, 0, s>>>(st, gr, slices, counts, units);
    else append_kernel<false><<<cache_grid(units), kThreads, 0, s>>>(st, gr, slices, counts, units);
    return cudaGetLastError();
}

template <class T>
static cudaError_t window_as(const CacheStore& st, const CacheGroups& gr, int slices,
                             const long long* ends, cudaStream_t s) {
    const unsigned units = cache_units(st, slices);
    if (st.int8) window_kernel<true, T><<<cache_grid(units), kThreads, 0, s>>>(st, gr, slices, ends, units);
    else window_kernel<false, T><<<cache_grid(units), kThreads, 0, s>>>(st, gr, slices, ends, units);
    return cudaGetLastError();
}

cudaError_t launch_cache_window(const CacheStore& st, const CacheGroups& gr, int slices,
                                const long long* ends, int dtype, cudaStream_t s) {
    if (cache_units(st, slices) == 0) return cudaSuccess;
    if (dtype == kOptF32) return window_as<float>(st, gr, slices, ends, s);
    if (dtype == kOptBf16) return window_as<__nv_bfloat16>(st, gr, slices, ends, s);
    return window_as<__half>(st, gr, slices, ends, s);
}

}  // namespace fcqt
