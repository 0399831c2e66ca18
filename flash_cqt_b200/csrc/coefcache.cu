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
// rounds nothing (but e4m3 values under 2^-130 in bf16, whose steps are 2^-133).
//
// Both kernels move bytes and do little else, so what a byte costs in
// instructions decides.  A thread takes 8 coefficients (64 bytes of complex64,
// 16 of codes; two lanes share a scale), a CTA 4096 of one slice; a slice's
// addresses in the groups' tensors are laid out in shared memory once for the
// CTA.  Whatever is rare (values that are not finite, the largest scales, NaN
// codes) is found by one test over a thread's values and left to a second
// version of the loop body.  A stream's length is read on the device, so a
// captured graph follows it.
//
// Measured: 490 slices of 132,992 coefficients written as e4m3 in 110 us (6.0
// TB/s), windows of 16 x 64 slices read as complex64 in 185 us (6.8 TB/s, four
// fifths of it writes), as bf16 pairs from int8 68 M coefficients in 73 us (5.6
// TB/s; 24 instructions a coefficient).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "internal.h"

namespace fcqt {

namespace {

constexpr int kThreads = 256;
constexpr int kOcts = 2;                             // octs (8 coefficients) a thread
constexpr int kTile = kThreads * kOcts;              // octs of a CTA

// where the slice (row, slice) begins in every group's tensor
struct SliceBase {
    char* data[kMaxGroups];       // first coefficient of the slice
    long long band[kMaxGroups];   // bytes from band to band
};


__device__ __forceinline__ void find_slice(const CacheGroups& gr, int item, long long row,
                                           long long slice, SliceBase& sb) {
    const int g = threadIdx.x;
    if (g < kMaxGroups) {
        sb.data[g] = static_cast<char*>(gr.data[g]) +
                     (row * gr.row[g] + slice * gr.slice[g]) * item;
        sb.band[g] = gr.band[g] * item;
    }
    __syncthreads();
}

// address of heap coefficient j of the slice
__device__ __forceinline__ char* place(const CacheGroups& gr, const SliceBase& sb, int item, int j) {
    int g = 0;
#pragma unroll
    for (int step = kMaxGroups / 2; step; step >>= 1)
        if (j >= gr.off[g + step]) g += step;   // unused groups lie behind every j
    const int k = j - gr.off[g], shift = gr.shift[g];
    const int band = k >> shift, t = k - (band << shift);
    return sb.data[g] + (band * sb.band[g] + (long long)t * item);
}

__device__ __forceinline__ unsigned slot_of(long long number, int capacity) {
    const unsigned long long n = (unsigned long long)number;
    return n >> 32 ? (unsigned)(n % (unsigned)capacity) : (unsigned)n % (unsigned)capacity;
}

// the larger magnitude, NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(fabsf(b)));
    return y;
}
__device__ __forceinline__ bool finite(float x) {
    return (__float_as_uint(x) & 0x7fffffffu) < 0x7f800000u;
}

// 16 values to codes.  RARE: some value of the run is not finite, or the scale
// is the largest there is, where a value next to 2^128 must not round up to it
template <bool INT8, bool RARE>
__device__ __forceinline__ uint4 encode(const float (&x)[16], float peak, int& e) {
    if constexpr (RARE) {
        peak = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (finite(x[i])) peak = fmaxf(peak, fabsf(x[i]));
        peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
    }
    // 127 = (1 + 63/64) 2^6 and 448 = 1.75 2^8: the exponent of the largest
    // value, one more where its fraction is above the format's
    const unsigned top = __float_as_uint(peak);
    e = INT8 ? (int)((top + 0x1ffffu) >> 23) - 6 : (int)((top + 0x1fffffu) >> 23) - 8;
    e = max(e, 1);
    const float inv = __uint_as_float((unsigned)(254 - e) << 23);
    const float most = INT8 ? (e == 249 ? 63.f : 127.f) : (e == 247 ? 240.f : 448.f);
    unsigned c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            y[k] = x[4 * i + k];
            if constexpr (RARE) y[k] = fminf(fmaxf(y[k] * inv, -most), most);
        }
        if constexpr (INT8) {
            unsigned b[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                // adding 1.5 * 2^23 rounds to the nearest integer, which the low
                // bits then hold in two's complement
                b[k] = __float_as_uint(RARE ? y[k] + 12582912.f : fmaf(y[k], inv, 12582912.f));
                if constexpr (RARE)
                    if (!finite(x[4 * i + k])) b[k] = 0x80u;
            }
            c[i] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040),
                               0x5410);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (RARE) {
                    if (!finite(x[4 * i + k])) y[k] = __int_as_float(0x7fffffff);
                } else {
                    y[k] *= inv;
                }
            }
            const unsigned lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE,
                                                         __NV_E4M3);
            const unsigned hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE,
                                                         __NV_E4M3);
            c[i] = lo | hi << 16;
        }
    }
    return make_uint4(c[0], c[1], c[2], c[3]);
}

// 16 codes to values
template <bool INT8>
__device__ __forceinline__ void decode(uint4 c, uint8_t e, float (&x)[16]) {
    const float s = __uint_as_float(e ? (unsigned)e << 23 : 0x400000u);
    const unsigned w[4] = {c.x, c.y, c.z, c.w};
    if constexpr (INT8) {
        unsigned nan = 0;
        const float off = -8388736.f * s;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned u = w[i] ^ 0x80808080u;   // the codes plus 128
            nan |= (u - 0x01010101u) & ~u;           // bit 7 of a byte that is 0, the code of NaN
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                // 2^23 + byte, less 2^23 + 128, times s, rounded once (exactly)
                const float f = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 | k));
                x[4 * i + k] = fmaf(f, s, off);
            }
        }
        // that needs (2^23 + 128) s to be finite
        if ((nan & 0x80808080u) != 0 || e > 200) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int code = (int)(w[i / 4] << (24 - 8 * (i & 3))) >> 24;
                x[i] = code == -128 ? __int_as_float(0x7fffffff) : (float)code * s;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
                (__nv_fp8x2_storage_t)((i & 1) ? w[i / 2] >> 16 : w[i / 2] & 0xffffu), __NV_E4M3);
            const float2 f = __half22float2(__half2(h));
            x[2 * i] = f.x * s;
            x[2 * i + 1] = f.y * s;
        }
    }
}

// 8 coefficients from memory
__device__ __forceinline__ void load16(const char* src, int wide, float (&x)[16]) {
    float a[8], b[8];
    if (wide == 2) {
        load_v8(reinterpret_cast<const float*>(src), a);
        load_v8(reinterpret_cast<const float*>(src) + 8, b);
    } else {   // float2 at a time: 8 bytes is what any complex64 tensor has
        const float2* p = reinterpret_cast<const float2*>(src);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 u = p[i], w = p[4 + i];
            a[2 * i] = u.x; a[2 * i + 1] = u.y;
            b[2 * i] = w.x; b[2 * i + 1] = w.y;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = a[i];
        x[8 + i] = b[i];
    }
}

__device__ __forceinline__ long long clamped(const long long* counts, int row, int slices) {
    const long long n = counts ? counts[row] : slices;
    return n < 0 ? 0 : (n > slices ? slices : n);
}

template <bool INT8>
__global__ void __launch_bounds__(kThreads)
append_kernel(const __grid_constant__ CacheStore st, const __grid_constant__ CacheGroups gr,
              int slices, const long long* counts) {
    __shared__ SliceBase sb;
    __shared__ unsigned order;
    const int octs = st.ncoef / 8;
    for (int row = blockIdx.z; row < st.rows; row += gridDim.z) {
        const long long count = clamped(counts, row, slices);
        const long long length = max(st.length[row], 0ll);
        for (int slice = blockIdx.y; slice < slices; slice += gridDim.y) {
            // slices behind the stream's last one are left out, and so are
            // those that newer ones of this call would overwrite
            if (slice >= count || (long long)slice + st.capacity < count) continue;
            __syncthreads();
            find_slice(gr, 8, row, slice, sb);
            const long long at = (long long)row * st.capacity + slot_of(length + slice, st.capacity);
            uint4* codes = reinterpret_cast<uint4*>(st.codes + at * 2 * st.ncoef);
            uint8_t* scales = st.scales + at * (st.ncoef / 16);
            float x[kOcts][16];
            // ncoef is a multiple of 16, so the two lanes of a run agree on `in`
#pragma unroll
            for (int i = 0; i < kOcts; ++i) {
                const int q = blockIdx.x * kTile + i * kThreads + threadIdx.x;
                if (q < octs) {
                    load16(place(gr, sb, 8, 8 * q), gr.wide, x[i]);
                } else {
#pragma unroll
                    for (int k = 0; k < 16; ++k) x[i][k] = 0.f;
                }
            }
#pragma unroll
            for (int i = 0; i < kOcts; ++i) {
                const int q = blockIdx.x * kTile + i * kThreads + threadIdx.x;
                float peak = fabsf(x[i][0]);
#pragma unroll
                for (int k = 1; k < 16; ++k) peak = max_nan(peak, x[i][k]);
                peak = max_nan(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
                int e;
                uint4 c;
                // only values above it take the largest scales; NaN fails too
                if (__any_sync(0xffffffffu, !(peak < 0x1p127f))) c = encode<INT8, true>(x[i], peak, e);
                else c = encode<INT8, false>(x[i], peak, e);
                if (q < octs) {
                    codes[q] = c;
                    if ((threadIdx.x & 1) == 0) scales[q / 2] = (uint8_t)e;
                }
            }
        }
        // every CTA of the row has read its length: the last one to come here
        // advances it
        __syncthreads();
        if (threadIdx.x == 0) {
            order = atomicAdd(st.ticket + row, 1u);
            if (order == gridDim.x * gridDim.y - 1) {
                st.length[row] = length + count;
                st.ticket[row] = 0;
            }
        }
    }
}

// 8 coefficients to memory: 64 bytes of float, 32 of the others
__device__ __forceinline__ void store16(float* dst, int wide, const float (&x)[16]) {
    float a[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        a[i] = x[i];
        b[i] = x[8 + i];
    }
    if (wide == 2) {
        store_v8(dst, a);
        store_v8(dst + 8, b);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            reinterpret_cast<float4*>(dst)[i] =
                make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    }
}
__device__ __forceinline__ float pair(__nv_bfloat16, float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const float*>(&h);
}
__device__ __forceinline__ float pair(__half, float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const float*>(&h);
}
template <class T>
__device__ __forceinline__ void store16(T* dst, int wide, const float (&x)[16]) {
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = pair(T(), x[2 * i], x[2 * i + 1]);
    if (wide == 2) {
        store_v8(reinterpret_cast<float*>(dst), w);
    } else {
        reinterpret_cast<float4*>(dst)[0] = make_float4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(w[4], w[5], w[6], w[7]);
    }
}

template <bool INT8, class T>
__global__ void __launch_bounds__(kThreads)
window_kernel(const __grid_constant__ CacheStore st, const __grid_constant__ CacheGroups gr,
              int slices, const long long* ends) {
    __shared__ SliceBase sb;
    constexpr int item = 2 * sizeof(T);
    const int octs = st.ncoef / 8;
    for (int row = blockIdx.z; row < st.rows; row += gridDim.z) {
        const long long length = st.length[row];
        const long long end = ends ? ends[row] : length;
        for (int slice = blockIdx.y; slice < slices; slice += gridDim.y) {
            const long long number = end - slices + slice;
            const bool held = number >= 0 && number < length && number >= length - st.capacity;
            const long long at =
                (long long)row * st.capacity + (held ? slot_of(number, st.capacity) : 0);
            const uint4* codes = reinterpret_cast<const uint4*>(st.codes + at * 2 * st.ncoef);
            const uint8_t* scales = st.scales + at * (st.ncoef / 16);
            __syncthreads();
            find_slice(gr, item, row, slice, sb);
            uint4 c[kOcts];
            uint8_t e[kOcts];
#pragma unroll
            for (int i = 0; i < kOcts; ++i) {
                const int q = blockIdx.x * kTile + i * kThreads + threadIdx.x;
                const bool in = held && q < octs;
                c[i] = in ? codes[q] : make_uint4(0, 0, 0, 0);   // codes of zero
                e[i] = in ? scales[q / 2] : 1;
            }
#pragma unroll
            for (int i = 0; i < kOcts; ++i) {
                const int q = blockIdx.x * kTile + i * kThreads + threadIdx.x;
                if (q >= octs) continue;
                T* dst = reinterpret_cast<T*>(place(gr, sb, item, 8 * q));
                float y[16];
                decode<INT8>(c[i], e[i], y);
                store16(dst, gr.wide, y);
            }
        }
    }
}

constexpr unsigned kMaxYZ = 65535;

dim3 cache_grid(const CacheStore& st, int slices) {
    const unsigned tiles = (unsigned)((st.ncoef / 8 + kTile - 1) / kTile);
    return dim3(tiles, (unsigned)slices < kMaxYZ ? (unsigned)slices : kMaxYZ,
                (unsigned)st.rows < kMaxYZ ? (unsigned)st.rows : kMaxYZ);
}

}  // namespace

cudaError_t launch_cache_append(const CacheStore& st, const CacheGroups& gr, int slices,
                                const long long* counts, cudaStream_t s) {
    if (slices == 0 || st.rows == 0) return cudaSuccess;
    const dim3 grid = cache_grid(st, slices);
    if (st.int8) append_kernel<true><<<grid, kThreads, 0, s>>>(st, gr, slices, counts);
    else append_kernel<false><<<grid, kThreads, 0, s>>>(st, gr, slices, counts);
    return cudaGetLastError();
}

template <class T>
static cudaError_t window_as(const CacheStore& st, const CacheGroups& gr, int slices,
                             const long long* ends, cudaStream_t s) {
    const dim3 grid = cache_grid(st, slices);
    if (st.int8) window_kernel<true, T><<<grid, kThreads, 0, s>>>(st, gr, slices, ends);
    else window_kernel<false, T><<<grid, kThreads, 0, s>>>(st, gr, slices, ends);
    return cudaGetLastError();
}

cudaError_t launch_cache_window(const CacheStore& st, const CacheGroups& gr, int slices,
                                const long long* ends, int dtype, cudaStream_t s) {
    if (slices == 0 || st.rows == 0) return cudaSuccess;
    if (dtype == kOptF32) return window_as<float>(st, gr, slices, ends, s);
    if (dtype == kOptBf16) return window_as<__nv_bfloat16>(st, gr, slices, ends, s);
    return window_as<__half>(st, gr, slices, ends, s);
}

}  // namespace fcqt
