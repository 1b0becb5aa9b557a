// gradnorm_kernels.hip -- the 2-norm over all elements of many gradient tensors, and their scaling by min(1, max_norm / (norm + 1e-6)).
//
//   norm = sqrt(sum over tensors and elements of g^2),   dst = src * min(1, max_norm / (norm + 1e-6))
//
// Both passes are bound by memory: the norm of 400 M bf16 gradients takes 183 us (4.4 TB/s), their scaling into f32 500 us (4.8 TB/s; a large copy
// reaches 4.7).  The tensors are cut into chunks of equal bytes and a fixed number of workgroups walks over them, so a list of forty ragged tensors
// costs what one flat buffer of their size does: one launch per 256 tensors for the norm, per 128 for the scaling.  The list travels in the kernel's
// arguments (no copy to the device, so a call can be captured).  Squares and sums are held in 64 bits: no overflow above 1.8e19, no underflow below
// 1e-23, and the order of the sums is fixed by the chunks, so the norm has the same bits on every call.
#include <algorithm>
#include <new>
#include "numeric.h"

namespace {

using namespace mz;

constexpr int GRID = 1024;     // workgroups of 256 threads: four per CU

// Tensors of one launch: as many as fit the 4 KB that a launch's arguments may take.  A tensor is its pointers, its first chunk and, in 16 bits, the
// size of its last chunk less one (at most 2^14 - 1) and its type.
template <bool DST> struct GradList {
    static constexpr int LIST = DST ? 128 : 256;
    const void *src[LIST];
    const void *dst[DST ? LIST : 1];
    uint32_t start[LIST];      // first chunk of each tensor; above the last one 0xFFFFFFFF
    uint16_t last[LIST];       // (size of the last chunk - 1) | dtype << 14
    uint8_t dst_dt[DST ? LIST : 1];
    uint32_t chunks;
};
static_assert(sizeof(GradList<false>) + 64 <= 4096 && sizeof(GradList<true>) + 64 <= 4096, "the list has to fit a launch's arguments");

// chunk c of the list: its tensor (the last one that starts at or before it), its first element, and how many there are
template <int U, bool DST> struct Chunk {
    int i, dt;
    int64_t at;
    int left;
    __device__ __forceinline__ Chunk(const GradList<DST> &L, uint32_t c) {
        const int lane = threadIdx.x & 63;
        int k = 0;
#pragma unroll
        for (int j = 0; j < GradList<DST>::LIST; j += 64) k += (int)__popcll(__ballot(L.start[j + lane] <= c));
        i = __builtin_amdgcn_readfirstlane(k - 1);
        const uint32_t end = i + 1 < GradList<DST>::LIST ? min(L.start[i + 1], L.chunks) : L.chunks;
        const uint32_t last = L.last[i];
        dt = (int)(last >> 14);
        const int full = U * 256 * (dt == MZ_F32 ? 4 : 8);
        at = (int64_t)(c - L.start[i]) * full;
        left = c + 1 == end ? (int)(last & 0x3FFF) + 1 : full;
    }
};

// U vectors of 16 bytes per lane; a tensor's last chunk keeps whole vectors too, so that all of its loads are in flight together, and one element a
// lane behind them
template <int DT, int U> __device__ __forceinline__ double square_sum(const void *src, int64_t at, int left) {
    constexpr int VEC = Elem<DT>::VEC;
    double acc = 0.0;
    Words<DT, VEC> p[U];
    if (left == U * 256 * VEC) {
#pragma unroll
        for (int k = 0; k < U; ++k) p[k] = load_words<DT, VEC>(src, at + (k * 256 + (int)threadIdx.x) * VEC);
    } else {
        const int whole = left / VEC, rest = left % VEC;
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int v = k * 256 + threadIdx.x;
            p[k] = {};
            if (v < whole) p[k] = load_words<DT, VEC>(src, at + (int64_t)v * VEC);
        }
        acc = (int)threadIdx.x < rest ? (double)load_one<DT>(src, at + (int64_t)whole * VEC + threadIdx.x) : 0.0;
        acc *= acc;
    }
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const double g = (double)p[k].get(j);
            acc = fma(g, g, acc);
        }
    return acc;
}

template <int U> __global__ void __launch_bounds__(256) k_norm_partial(GradList<false> L, double *partial) {
    __shared__ double red[4];
    double acc = 0.0;
    for (uint32_t c = blockIdx.x; c < L.chunks; c += gridDim.x) {
        const Chunk<U, false> k(L, c);
        if (k.dt == MZ_F32) acc += square_sum<MZ_F32, U>(L.src[k.i], k.at, k.left);
        else if (k.dt == MZ_BF16) acc += square_sum<MZ_BF16, U>(L.src[k.i], k.at, k.left);
        else acc += square_sum<MZ_F16, U>(L.src[k.i], k.at, k.left);
    }
    acc = block_sum<4>(acc, red);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

__global__ void __launch_bounds__(1024) k_norm_final(const double *partial, int count, float *norm) {
    __shared__ double red[16];
    double s = 0.0;
    for (int k = threadIdx.x; k < count; k += 1024) s += partial[k];
    s = block_sum<16>(s, red);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

template <int SD, int DD, int U> __device__ __forceinline__ void scale_chunk(const void *src, void *dst, int64_t at, int left, float scale) {
    constexpr int VEC = Elem<SD>::VEC;
    const int whole = left / VEC;
    const int64_t end = at + (int64_t)whole * VEC + threadIdx.x;
    if ((int)threadIdx.x < left % VEC) store_one<DD>(dst, end, load_one<SD>(src, end) * scale);
    Words<SD, VEC> p[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
        const int v = k * 256 + threadIdx.x;
        if (v < whole) p[k] = load_words<SD, VEC>(src, at + (int64_t)v * VEC);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
        const int v = k * 256 + threadIdx.x;
        if (v < whole) {
            Words<DD, VEC> q;
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) q.set_pair(j, p[k].get(2 * j) * scale, p[k].get(2 * j + 1) * scale);
            store_words<DD, VEC>(dst, at + (int64_t)v * VEC, q);
        }
    }
}

// every workgroup adds up the partial sums itself (the same order, so the same norm), which saves a launch between the passes
template <int U> __global__ void __launch_bounds__(256) k_clip(GradList<true> L, const double *partial, int count, double max_norm, float *norm, int write_norm) {
    __shared__ double red[4];
    double s = 0.0;
    for (int k = threadIdx.x; k < count; k += 256) s += partial[k];
    s = sqrt(block_sum<4>(s, red));
    if (write_norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)s;
    const double ratio = max_norm / (s + 1e-6);
    const float scale = ratio >= 1.0 ? 1.0f : (float)ratio;   // a NaN stays one
    for (uint32_t c = blockIdx.x; c < L.chunks; c += gridDim.x) {
        const Chunk<U, true> k(L, c);
        const int sd = k.dt, dd = L.dst_dt[k.i], left = k.left;
        const int64_t at = k.at;
        const void *src = L.src[k.i];
        void *dst = (void *)L.dst[k.i];
        if (scale == 1.0f && src == dst) continue;            // in place and not clipped: the values stay as they are
        if (sd == MZ_F32) scale_chunk<MZ_F32, MZ_F32, U>(src, dst, at, left, scale);
        else if (sd == MZ_BF16) {
            if (dd == MZ_F32) scale_chunk<MZ_BF16, MZ_F32, U>(src, dst, at, left, scale);
            else scale_chunk<MZ_BF16, MZ_BF16, U>(src, dst, at, left, scale);
        } else {
            if (dd == MZ_F32) scale_chunk<MZ_F16, MZ_F32, U>(src, dst, at, left, scale);
            else scale_chunk<MZ_F16, MZ_F16, U>(src, dst, at, left, scale);
        }
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------------
struct Range {
    uintptr_t lo, hi;
    int of;          // tensor
    bool written;
};

int check_list(const char *who, const mz_grad_tensor *t, int32_t count, bool clip, int64_t *bytes) {
    MZ_REQUIRE(count >= 1, "%s: needs at least one tensor", who);
    MZ_REQUIRE(t, "%s: null list", who);
    *bytes = 0;
    for (int i = 0; i < count; ++i) {
        MZ_REQUIRE(t[i].n >= 0, "%s: tensor %d has a negative size", who, i);
        MZ_REQUIRE(elem_known(t[i].src_dtype), "%s: tensor %d has an unknown dtype %d", who, i, t[i].src_dtype);
        if (t[i].n == 0) continue;
        MZ_REQUIRE(t[i].n <= (int64_t)1 << 40, "%s: tensor %d is too large", who, i);
        const int sb = elem_bytes(t[i].src_dtype);
        MZ_REQUIRE(t[i].src && (uintptr_t)t[i].src % sb == 0, "%s: tensor %d has a null or misaligned pointer", who, i);
        *bytes += t[i].n * sb;
        if (!clip) continue;
        MZ_REQUIRE(t[i].dst_dtype == t[i].src_dtype || t[i].dst_dtype == MZ_F32, "%s: tensor %d: the output has its dtype or is f32", who, i);
        MZ_REQUIRE(t[i].dst && (uintptr_t)t[i].dst % elem_bytes(t[i].dst_dtype) == 0, "%s: output %d has a null or misaligned pointer", who, i);
    }
    MZ_REQUIRE(*bytes < (int64_t)1 << 42, "%s: the tensors are too large", who);
    return MZ_OK;
}

// what one workgroup writes no other may read or write: outputs lie apart from each other, and from every gradient but their own
int check_overlap(const char *who, const mz_grad_tensor *t, int32_t count) {
    Range *r = new (std::nothrow) Range[2 * (size_t)count];
    MZ_REQUIRE(r, "%s: out of host memory", who);
    int m = 0;
    for (int i = 0; i < count; ++i) {
        if (t[i].n == 0) continue;
        const uintptr_t s = (uintptr_t)t[i].src, d = (uintptr_t)t[i].dst;
        r[m++] = {d, d + (uintptr_t)t[i].n * elem_bytes(t[i].dst_dtype), i, true};
        if (s != d || t[i].src_dtype != t[i].dst_dtype) r[m++] = {s, s + (uintptr_t)t[i].n * elem_bytes(t[i].src_dtype), i, false};
    }
    std::sort(r, r + m, [](const Range &a, const Range &b) { return a.lo < b.lo; });
    int bad = -1;
    uintptr_t any_end = 0, written_end = 0;   // how far what came before reaches
    for (int k = 0; k < m && bad < 0; ++k) {
        if (r[k].lo < (r[k].written ? any_end : written_end)) bad = r[k].of;
        any_end = std::max(any_end, r[k].hi);
        if (r[k].written) written_end = std::max(written_end, r[k].hi);
    }
    delete[] r;
    MZ_REQUIRE(bad < 0, "%s: tensor %d overlaps another one that is written, or its own output in part", who, bad);
    return MZ_OK;
}

// the next list of non-empty tensors from *i on; returns their count
template <bool DST> int next_list(const mz_grad_tensor *t, int32_t count, int *i, int chunk_bytes, GradList<DST> *L) {
    int k = 0;
    uint32_t chunks = 0;
    for (; *i < count && k < GradList<DST>::LIST; ++*i) {
        const mz_grad_tensor &x = t[*i];
        if (x.n == 0) continue;
        const int64_t full = chunk_bytes / elem_bytes(x.src_dtype), parts = (x.n + full - 1) / full;
        L->src[k] = x.src;
        if (DST) {
            L->dst[k] = x.dst;
            L->dst_dt[k] = (uint8_t)x.dst_dtype;
        }
        L->start[k] = chunks;
        L->last[k] = (uint16_t)((x.n - (parts - 1) * full - 1) | x.src_dtype << 14);
        chunks += (uint32_t)parts;
        ++k;
    }
    L->chunks = chunks;
    for (int j = k; j < GradList<DST>::LIST; ++j) {
        L->start[j] = 0xFFFFFFFFu;
        L->last[j] = 0;
        L->src[j] = nullptr;
        if (DST) {
            L->dst[j] = nullptr;
            L->dst_dt[j] = 0;
        }
    }
    return k;
}

// Chunks of 32 KB keep eight 16-byte loads of every lane in flight; lists under 4 MB are cut into 8 KB so that more CUs get some.  Measured with 32 / 8 KB:
// clipping 0.4 MB 7.2 / 6.0 us, 8 MB 9.2 / 9.6 us, 32 MB 18.4 / 21.2 us; the norm of 800 MB 143 / 155 us.
inline int unroll_for(int64_t bytes) { return bytes < ((int64_t)4 << 20) ? 2 : 8; }

int partial_sums(const mz_grad_tensor *t, int32_t count, int unroll, double *partial, int *partials, hipStream_t s) {
    *partials = 0;
    for (int i = 0; i < count;) {
        GradList<false> L;
        if (!next_list(t, count, &i, unroll * 4096, &L)) break;
        const int grid = (int)std::min<uint32_t>(L.chunks, GRID);
        if (unroll == 2) hipLaunchKernelGGL((k_norm_partial<2>), dim3(grid), dim3(256), 0, s, L, partial + *partials);
        else hipLaunchKernelGGL((k_norm_partial<8>), dim3(grid), dim3(256), 0, s, L, partial + *partials);
        MZ_LAUNCH_CHECK("k_norm_partial");
        *partials += grid;
    }
    return MZ_OK;
}

}  // namespace

extern "C" int64_t mz_grad_workspace_bytes(int32_t count) {
    if (count < 1) return -1;
    constexpr int LIST = GradList<false>::LIST;
    return (((int64_t)count + LIST - 1) / LIST) * GRID * (int64_t)sizeof(double);
}

extern "C" int mz_grad_norm(const mz_grad_tensor *tensors, int32_t count, void *workspace, int64_t workspace_bytes, float *norm, void *stream) {
    int64_t bytes;
    if (int rc = check_list("mz_grad_norm", tensors, count, false, &bytes)) return rc;
    MZ_REQUIRE(norm && workspace && ((uintptr_t)workspace & 7) == 0, "mz_grad_norm: null or misaligned workspace or result");
    MZ_REQUIRE(workspace_bytes >= mz_grad_workspace_bytes(count), "mz_grad_norm: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
               (long long)mz_grad_workspace_bytes(count));
    hipStream_t s = (hipStream_t)stream;
    int partials;
    if (int rc = partial_sums(tensors, count, unroll_for(bytes), (double *)workspace, &partials, s)) return rc;
    hipLaunchKernelGGL(k_norm_final, dim3(1), dim3(1024), 0, s, (const double *)workspace, partials, norm);
    MZ_LAUNCH_CHECK("k_norm_final");
    return MZ_OK;
}

extern "C" int mz_grad_clip(const mz_grad_tensor *tensors, int32_t count, double max_norm, void *workspace, int64_t workspace_bytes, float *norm,
                            void *stream) {
    int64_t bytes;
    if (int rc = check_list("mz_grad_clip", tensors, count, true, &bytes)) return rc;
    MZ_REQUIRE(max_norm >= 0.0, "mz_grad_clip: max_norm has to be 0 or more");
    MZ_REQUIRE(norm && workspace && ((uintptr_t)workspace & 7) == 0, "mz_grad_clip: null or misaligned workspace or result");
    MZ_REQUIRE(workspace_bytes >= mz_grad_workspace_bytes(count), "mz_grad_clip: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
               (long long)mz_grad_workspace_bytes(count));
    if (int rc = check_overlap("mz_grad_clip", tensors, count)) return rc;
    hipStream_t s = (hipStream_t)stream;
    const int unroll = unroll_for(bytes);
    int partials, first = 1;
    if (int rc = partial_sums(tensors, count, unroll, (double *)workspace, &partials, s)) return rc;
    for (int i = 0; i < count || first;) {
        GradList<true> L;
        if (!next_list(tensors, count, &i, unroll * 4096, &L) && !first) break;   // with nothing but empty tensors the norm is written all the same
        const int grid = (int)std::max<uint32_t>(1, std::min<uint32_t>(L.chunks, GRID));
        if (unroll == 2) hipLaunchKernelGGL((k_clip<2>), dim3(grid), dim3(256), 0, s, L, (const double *)workspace, partials, max_norm, norm, first);
        else hipLaunchKernelGGL((k_clip<8>), dim3(grid), dim3(256), 0, s, L, (const double *)workspace, partials, max_norm, norm, first);
        MZ_LAUNCH_CHECK("k_clip");
        first = 0;
    }
    return MZ_OK;
}
