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

// N elements of 16 or 32 bits that lie together.  Global loads and stores of this target may start at any element, so rows and
// views that begin at an odd element take the same 16-byte accesses as aligned ones.
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[N]; };

template <int DT, int N> __device__ __forceinline__ Pack<typename Elem<DT>::T, N> load_pack(const void *base, int64_t at) {
    typedef Pack<typename Elem<DT>::T, N> P;
    const MZ_GLOBAL P *p = (const MZ_GLOBAL P *)((const MZ_GLOBAL typename Elem<DT>::T *)base + at);
    P r;
    __builtin_memcpy(&r, p, sizeof(P));
    return r;
}
template <int DT, int N> __device__ __forceinline__ void store_pack(void *base, int64_t at, const Pack<typename Elem<DT>::T, N> &r) {
    typedef Pack<typename Elem<DT>::T, N> P;
    MZ_GLOBAL P *p = (MZ_GLOBAL P *)((MZ_GLOBAL typename Elem<DT>::T *)base + at);
    __builtin_memcpy(p, &r, sizeof(P));
}
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
