// numeric.h -- element types and reductions shared by the operators that take f32, bf16 and f16 tensors.
#pragma once
#include "common.h"

namespace mz {

#define MZ_GLOBAL __attribute__((address_space(1)))

// one element type: its storage, how many of them a 16-byte load brings, and the exact widening / nearest-even narrowing
template <int DT> struct Elem;
template <> struct Elem<MZ_F32> {
    using T = uint32_t;
    static constexpr int VEC = 4;
    static __device__ __forceinline__ float up(uint32_t v) { return __uint_as_float(v); }
    static __device__ __forceinline__ uint32_t down(float f) { return __float_as_uint(f); }
};
template <> struct Elem<MZ_BF16> {
    using T = uint16_t;
    static constexpr int VEC = 8;
    static __device__ __forceinline__ float up(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ uint16_t down(float f) {
        const __bf16 h = (__bf16)f;   // the hardware's conversion: to nearest even, NaN stays NaN
        uint16_t v;
        __builtin_memcpy(&v, &h, 2);
        return v;
    }
};
template <> struct Elem<MZ_F16> {
    using T = uint16_t;
    static constexpr int VEC = 8;
    static __device__ __forceinline__ float up(uint16_t v) { _Float16 h; __builtin_memcpy(&h, &v, 2); return (float)h; }
    static __device__ __forceinline__ uint16_t down(float f) { const _Float16 h = (_Float16)f; uint16_t v; __builtin_memcpy(&v, &h, 2); return v; }
};

// N elements as the 32-bit words that hold them (16-bit ones stay in pairs, half the registers of one word each)
template <int DT, int N> struct Words {
    static constexpr int SIZE = sizeof(typename Elem<DT>::T), COUNT = N * SIZE / 4;
    uint32_t w[COUNT];
    __device__ __forceinline__ float get(int j) const {
        if constexpr (DT == MZ_F32) return __uint_as_float(w[j]);
        else if constexpr (DT == MZ_BF16) return __uint_as_float(j & 1 ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16);
        else return Elem<DT>::up((uint16_t)(j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xFFFFu));
    }
    __device__ __forceinline__ void set(int j, typename Elem<DT>::T v) {
        if constexpr (DT == MZ_F32) w[j] = v;
        else w[j / 2] = j & 1 ? (w[j / 2] & 0xFFFFu) | (uint32_t)v << 16 : (w[j / 2] & 0xFFFF0000u) | v;
    }
    // elements 2 j and 2 j + 1, each rounded once
    __device__ __forceinline__ void set_pair(int j, float a, float b) {
        if constexpr (DT == MZ_F32) {
            w[2 * j] = __float_as_uint(a);
            w[2 * j + 1] = __float_as_uint(b);
        } else {
            typedef float F2 __attribute__((ext_vector_type(2)));
            typedef __bf16 B2 __attribute__((ext_vector_type(2)));
            typedef _Float16 H2 __attribute__((ext_vector_type(2)));
            const F2 f = {a, b};
            if constexpr (DT == MZ_BF16) {
                const B2 h = __builtin_convertvector(f, B2);
                __builtin_memcpy(&w[j], &h, 4);
            } else {
                const H2 h = __builtin_convertvector(f, H2);
                __builtin_memcpy(&w[j], &h, 4);
            }
        }
    }
};

// Global loads and stores of this target may start at any element, so rows and views that begin at an odd one take the same 16-byte
// accesses as aligned ones.
template <int DT, int N> __device__ __forceinline__ Words<DT, N> load_words(const void *base, int64_t at) {
    Words<DT, N> r;
    __builtin_memcpy(r.w, (const MZ_GLOBAL typename Elem<DT>::T *)base + at, sizeof(r.w));
    return r;
}
template <int DT, int N> __device__ __forceinline__ void store_words(void *base, int64_t at, const Words<DT, N> &r) {
    __builtin_memcpy((MZ_GLOBAL typename Elem<DT>::T *)base + at, r.w, sizeof(r.w));
}
// eight truth values of a byte each, from any address
struct __attribute__((packed, aligned(1))) Flags { uint64_t v; };
__device__ __forceinline__ uint64_t load_flags(const uint8_t *base, int64_t at) { return ((const MZ_GLOBAL Flags *)((const MZ_GLOBAL uint8_t *)base + at))->v; }

template <int DT> __device__ __forceinline__ float load_one(const void *base, int64_t at) {
    return Elem<DT>::up(((const MZ_GLOBAL typename Elem<DT>::T *)base)[at]);
}
template <int DT> __device__ __forceinline__ void store_one(void *base, int64_t at, float f) {
    ((MZ_GLOBAL typename Elem<DT>::T *)base)[at] = Elem<DT>::down(f);
}

// the sum over a wave in a fixed order, the same in every lane
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

// the sum over a workgroup of W waves in a fixed order, the same in every thread; `red` holds W values and may be used again after the call
template <int W> __device__ __forceinline__ double block_sum(double v, double *red) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < W; ++w) s += red[w];
    __syncthreads();
    return s;
}

static inline int elem_bytes(int dtype) { return dtype == MZ_F32 ? 4 : 2; }
static inline bool elem_known(int dtype) { return dtype == MZ_F32 || dtype == MZ_BF16 || dtype == MZ_F16; }

}  // namespace mz
