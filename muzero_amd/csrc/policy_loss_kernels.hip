// policy_loss_kernels.hip -- the policy's cross-entropy against target distributions, and its gradient.
//
// For row i with logits x, targets t >= 0 and weight w, over the actions that `legal` leaves:
//   m = max x,  z = sum exp(x - m),  T = sum t,    loss_i = w (T log z - sum t (x - m))        [= -w sum t log softmax(x)]
//   d loss_i / d x = w (T exp(x - m) / z - t)
// A term with t = 0 counts as 0 also where x is -inf.  A row without a legal action, or of weight 0, gives 0 and a zero gradient.
//
// Bound by memory: x and t are read, the gradient is written.  So the loss and the gradient come out of ONE pass: the row stays in registers between
// its sums and its gradient (one wave per row up to 512 actions, one workgroup above), and a training step reads x and t once, not twice:
// 4096 x 32768 bf16 takes 155 us, 5.2 TB/s, where a large copy reaches 4.7.  Rows that are too long for a workgroup's registers are cut into chunks:
// one launch for the chunks' sums, one that joins them and writes the gradient (both read x and t: 5 parts of traffic for 3; in slabs of rows that
// would stay in the last-level cache between the two launches it was slower, 512 x 131072 f32: 310 us in slabs of 96 MB, 263 us without).
// Softmax statistics and row sums are f32, sums over rows 64 bits; 16-bit gradients are rounded once.  Above 512 actions the exponentials of 16-bit
// logits are the hardware's, also those in the f32 loss (exp_of).
#include <math.h>
#include <algorithm>
#include "numeric.h"

namespace {

using namespace mz;

struct LossArgs {
    const void *x, *t;
    const uint8_t *allowed;        // (n, v) bytes, or null
    const uint64_t *board;         // (n) bitboards of 64 squares, action 64 legal where none is set, or null
    const float *weight;           // (n) or null
    const float *go;               // the gradient of the loss: one value, or one per row
    float *row_loss;               // (n) or null
    void *grad;                    // or null
    int64_t x_stride, t_stride, allowed_stride, grad_stride;   // between rows, in elements
    int64_t n;
    int v, go_stride, skip_one;
    float scale;                   // of the gradient: 1 / n for a mean
};

constexpr float NEG_INF = -INFINITY;

// what one lane, wave or workgroup knows of a row: the maximum, sum exp(x - m), sum t, sum t (x - m)
struct Stat {
    float m, z, t, a;
};
__device__ __forceinline__ float shift_of(float m) { return m == NEG_INF ? 0.0f : m; }
__device__ __forceinline__ Stat join(const Stat &p, const Stat &q) {
    Stat r;
    r.m = fmaxf(p.m, q.m);
    const float s = shift_of(r.m);
    const float dp = shift_of(p.m) - s, dq = shift_of(q.m) - s;
    // an empty part has m = -inf, z = 0 and only zero terms: its shift is 0 and must not bring in exp(0 - s)
    r.z = (p.m == NEG_INF ? p.z : p.z * expf(dp)) + (q.m == NEG_INF ? q.z : q.z * expf(dq));
    r.t = p.t + q.t;
    r.a = (p.t != 0.0f ? fmaf(p.t, dp, p.a) : p.a) + (q.t != 0.0f ? fmaf(q.t, dq, q.a) : q.a);
    return r;
}
__device__ __forceinline__ Stat wave_join(Stat s) {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const Stat o = {__shfl_xor(s.m, d, 64), __shfl_xor(s.z, d, 64), __shfl_xor(s.t, d, 64), __shfl_xor(s.a, d, 64)};
        s = join(s, o);
    }
    return s;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
    return v;
}
__device__ __forceinline__ float wave_sumf(float v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

__device__ __forceinline__ float row_weight(const LossArgs &A, int64_t row) { return A.weight ? A.weight[row] : 1.0f; }
__device__ __forceinline__ float row_scale(const LossArgs &A, int64_t row, float w) {
    const float go = A.go ? A.go[A.go_stride ? row : 0] : 1.0f;
    return go * (w * A.scale);
}
// no action left: the maximum is -inf and nothing was added (a NaN would have been)
__device__ __forceinline__ bool row_empty(const Stat &s) { return s.m == NEG_INF && s.z == 0.0f; }
__device__ __forceinline__ float loss_of(const Stat &s, float w) { return (row_empty(s) || w == 0.0f) ? 0.0f : w * (s.t * logf(s.z) - s.a); }

// ---- one wave per row, up to 64 E actions ------------------------------------------------------------------------------------
template <int XD, int TD, int E> __global__ void __launch_bounds__(256) k_loss_wave(LossArgs A) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= A.n) return;
    if (A.skip_one && A.go[0] == 1.0f) return;
    const float w = row_weight(A, row);
    const bool dead = w == 0.0f;
    const int64_t xo = row * A.x_stride, to = row * A.t_stride, ao = row * A.allowed_stride;
    const uint64_t board = A.board ? A.board[row] : 0;
    float x[E], t[E];
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const int j = k * 64 + lane;
        bool ok = j < A.v && !dead;
        if (ok && A.allowed) ok = A.allowed[ao + j] != 0;
        if (ok && A.board) ok = j < 64 ? (board >> j) & 1 : board == 0;
        x[k] = NEG_INF;
        t[k] = 0.0f;
        if (ok) {
            x[k] = load_one<XD>(A.x, xo + j);
            t[k] = load_one<TD>(A.t, to + j);
        }
    }
    Stat s = {NEG_INF, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < E; ++k) s.m = fmaxf(s.m, x[k]);
    s.m = wave_max(s.m);
    const float shift = shift_of(s.m);
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const float d = x[k] - shift;
        x[k] = expf(d);
        s.z += x[k];
        s.t += t[k];
        if (t[k] != 0.0f) s.a = fmaf(t[k], d, s.a);
    }
    s.z = wave_sumf(s.z);
    s.t = wave_sumf(s.t);
    s.a = wave_sumf(s.a);
    if (A.row_loss && lane == 0) A.row_loss[row] = loss_of(s, w);
    if (!A.grad) return;
    const bool zero = dead || row_empty(s);
    const float scale = row_scale(A, row, w), tz = s.t / s.z;
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const int j = k * 64 + lane;
        if (j < A.v) store_one<XD>(A.grad, row * A.grad_stride + j, zero ? 0.0f : (x[k] * tz - t[k]) * scale);
    }
}

// e^d for d <= 0.  16-bit logits: 2^(d log2 e) on the hardware's exponential, |d| 2^-24 relative, far below a step of theirs; f32 ones: exact to the
// last places.
template <int XD> __device__ __forceinline__ float exp_of(float d) { return XD == MZ_F32 ? expf(d) : __builtin_amdgcn_exp2f(d * 1.44269504f); }

// ---- a run of VEC actions in registers ---------------------------------------------------------------------------------------
template <int XD, int TD> struct Run {
    static constexpr int VEC = Elem<XD>::VEC;
    Words<XD, VEC> x;
    Words<TD, VEC> t;
    // actions at..at+VEC-1 of a row; what lies behind its end or is not legal becomes x = -inf, t = 0
    __device__ __forceinline__ void load(const LossArgs &A, int64_t xo, int64_t to, int64_t ao, int at) {
        if (at + VEC <= A.v) {
            x = load_words<XD, VEC>(A.x, xo + at);
            t = load_words<TD, VEC>(A.t, to + at);
            if (A.allowed) {
                uint32_t ok[VEC / 4];
                __builtin_memcpy(ok, (const MZ_GLOBAL uint8_t *)A.allowed + ao + at, VEC);
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (!((ok[j / 4] >> (j & 3) * 8) & 0xFF)) clear(j);
            }
        } else {
            x = {};
            t = {};
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                clear(j);
                if (at + j < A.v && (!A.allowed || A.allowed[ao + at + j])) {
                    x.set(j, ((const MZ_GLOBAL typename Elem<XD>::T *)A.x)[xo + at + j]);
                    t.set(j, ((const MZ_GLOBAL typename Elem<TD>::T *)A.t)[to + at + j]);
                }
            }
        }
    }
    __device__ __forceinline__ void clear(int j) {
        x.set(j, (typename Elem<XD>::T)(XD == MZ_F32 ? 0xFF800000u : XD == MZ_BF16 ? 0xFF80u : 0xFC00u));
        t.set(j, 0);
    }
    __device__ __forceinline__ float xf(int j) const { return x.get(j); }
    __device__ __forceinline__ float tf(int j) const { return t.get(j); }
    __device__ __forceinline__ void add(Stat &s, float shift) const {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float d = xf(j) - shift, tv = tf(j);
            s.z += exp_of<XD>(d);
            s.t += tv;
            if (tv != 0.0f) s.a = fmaf(tv, d, s.a);
        }
    }
    __device__ __forceinline__ void store_grad(const LossArgs &A, int64_t go, int at, bool zero, float shift, float tz, float scale) const {
        Words<XD, VEC> g;
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
            float f[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) f[i] = zero ? 0.0f : fmaf(exp_of<XD>(xf(2 * j + i) - shift), tz, -tf(2 * j + i)) * scale;
            g.set_pair(j, f[0], f[1]);
        }
        if (at + VEC <= A.v) store_words<XD, VEC>(A.grad, go + at, g);
        else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (at + j < A.v) store_one<XD>(A.grad, go + at + j, g.get(j));
        }
    }
};

// ---- one workgroup per row, up to THREADS x NV x VEC actions, held in registers --------------------------------------------------
template <int XD, int TD, int THREADS, int NV> __global__ void __launch_bounds__(THREADS) k_loss_row(LossArgs A) {
    constexpr int VEC = Elem<XD>::VEC, W = THREADS / 64;
    __shared__ float red[4][W];
    if (A.skip_one && A.go[0] == 1.0f) return;
    const int64_t row = blockIdx.x;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const float w = row_weight(A, row);
    const int64_t xo = row * A.x_stride, to = row * A.t_stride, ao = row * A.allowed_stride, gro = row * A.grad_stride;
    const bool dead = w == 0.0f;
    Run<XD, TD> r[NV];
    Stat s = {NEG_INF, 0.0f, 0.0f, 0.0f};
    if (!dead) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int at = (k * THREADS + threadIdx.x) * VEC;
            if (at < A.v) r[k].load(A, xo, to, ao, at);
        }
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if ((k * THREADS + threadIdx.x) * VEC < (unsigned)A.v)
#pragma unroll
                for (int j = 0; j < VEC; ++j) s.m = fmaxf(s.m, r[k].xf(j));
        s.m = wave_max(s.m);
        if (lane == 0) red[0][wave] = s.m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < W; ++i) s.m = fmaxf(s.m, red[0][i]);
        const float shift = shift_of(s.m);
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if ((k * THREADS + threadIdx.x) * VEC < (unsigned)A.v) r[k].add(s, shift);
        s.z = wave_sumf(s.z);
        s.t = wave_sumf(s.t);
        s.a = wave_sumf(s.a);
        if (lane == 0) {
            red[1][wave] = s.z;
            red[2][wave] = s.t;
            red[3][wave] = s.a;
        }
        __syncthreads();
        s.z = s.t = s.a = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            s.z += red[1][i];
            s.t += red[2][i];
            s.a += red[3][i];
        }
    }
    if (A.row_loss && threadIdx.x == 0) A.row_loss[row] = loss_of(s, w);
    if (!A.grad) return;
    const bool zero = dead || row_empty(s);
    const float scale = row_scale(A, row, w), tz = s.t / s.z, shift = shift_of(s.m);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int at = (k * THREADS + threadIdx.x) * VEC;
        if (at < A.v) r[k].store_grad(A, gro, at, zero, shift, tz, scale);
    }
}

// ---- rows in chunks ------------------------------------------------------------------------------------------------------------
constexpr int CHUNKS = 256;    // at most: one thread of the joining workgroup reads one chunk's sums

template <int XD, int TD> __global__ void __launch_bounds__(256) k_loss_part(LossArgs A, int64_t row0, int chunk, Stat *part) {
    constexpr int VEC = Elem<XD>::VEC;
    __shared__ Stat red[4];
    if (A.skip_one && A.go[0] == 1.0f) return;
    const int64_t row = row0 + blockIdx.y;
    const int64_t xo = row * A.x_stride, to = row * A.t_stride, ao = row * A.allowed_stride;
    const int begin = blockIdx.x * chunk, end = min(begin + chunk, A.v);
    Stat s = {NEG_INF, 0.0f, 0.0f, 0.0f};
    if (row_weight(A, row) != 0.0f)
        for (int at = begin + threadIdx.x * VEC; at < end; at += 256 * VEC) {
            Run<XD, TD> r;
            r.load(A, xo, to, ao, at);
            Stat q = {NEG_INF, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < VEC; ++j) q.m = fmaxf(q.m, r.xf(j));
            r.add(q, shift_of(q.m));
            s = join(s, q);
        }
    s = wave_join(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = join(join(red[0], red[1]), join(red[2], red[3]));
}

template <int XD, int TD> __global__ void __launch_bounds__(256) k_loss_join(LossArgs A, int64_t row0, int chunk, const Stat *part) {
    constexpr int VEC = Elem<XD>::VEC;
    __shared__ Stat red[4];
    if (A.skip_one && A.go[0] == 1.0f) return;
    const int64_t row = row0 + blockIdx.y;
    Stat s = {NEG_INF, 0.0f, 0.0f, 0.0f};
    if (threadIdx.x < gridDim.x) s = part[(int64_t)blockIdx.y * gridDim.x + threadIdx.x];
    s = wave_join(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = join(join(red[0], red[1]), join(red[2], red[3]));
    const float w = row_weight(A, row);
    if (A.row_loss && blockIdx.x == 0 && threadIdx.x == 0) A.row_loss[row] = loss_of(s, w);
    if (!A.grad) return;
    const int64_t xo = row * A.x_stride, to = row * A.t_stride, ao = row * A.allowed_stride, gro = row * A.grad_stride;
    const bool zero = w == 0.0f || row_empty(s);
    const float scale = row_scale(A, row, w), tz = s.t / s.z, shift = shift_of(s.m);
    const int begin = blockIdx.x * chunk, end = min(begin + chunk, A.v);
    for (int at = begin + threadIdx.x * VEC; at < end; at += 256 * VEC) {
        Run<XD, TD> r;
        r.load(A, xo, to, ao, at);
        r.store_grad(A, gro, at, zero, shift, tz, scale);
    }
}

__global__ void __launch_bounds__(1024) k_loss_sum(const float *row_loss, int64_t n, double scale, float *loss) {
    __shared__ double red[16];
    double s = 0.0;
    for (int64_t k = threadIdx.x; k < n; k += 1024) s += (double)row_loss[k];
    s = block_sum<16>(s, red);
    if (threadIdx.x == 0) *loss = (float)(s * scale);
}

// ---- host side -------------------------------------------------------------------------------------------------------------------
constexpr int64_t MAX_V = 1 << 24, MAX_N = (1 << 22) - 1;   // a launch has fewer than 2^32 threads

constexpr int64_t SLAB = 65535;         // rows of one pair of launches: what a grid's second dimension takes
// Chunks of 8192 actions or more; with few rows of 2048 or more, for more CUs (131,072 f32 actions, in 2048 / 8192: 1 row 14.9 / 19.8 us, 8 rows
// 17.3 / 20.8 us, 64 rows 47.1 / 40.9 us)
int chunk_size(int64_t n, int64_t v) {
    return (int)std::max<int64_t>(n <= 16 ? 2048 : 8192, ((v + CHUNKS - 1) / CHUNKS + 2047) / 2048 * 2048);
}
int chunk_count(int64_t n, int64_t v) { return (int)((v + chunk_size(n, v) - 1) / chunk_size(n, v)); }

template <int XD, int TD> int launch(const LossArgs &A, Stat *part, hipStream_t s) {
    constexpr int VEC = Elem<XD>::VEC;
    const unsigned rows = (unsigned)A.n;
    const int64_t vecs = ((int64_t)A.v + VEC - 1) / VEC;
    // The smallest workgroup whose registers hold a row, so that a CU has several to overlap one's loads with another's stores: 4096 x 500 f32 by a
    // wave 14.1 us, by a workgroup 16.9; 4096 x 16384 f32 by 512 threads 193 us, by 1024 218; 64 x 16384 f32 by a workgroup 15.2 us, in chunks 20.4;
    // 256 x 32768 f32 32.9 and 41.3.
    if (A.v <= 128) hipLaunchKernelGGL((k_loss_wave<XD, TD, 2>), dim3((rows + 3) / 4), dim3(256), 0, s, A);
    else if (A.v <= 512) hipLaunchKernelGGL((k_loss_wave<XD, TD, 8>), dim3((rows + 3) / 4), dim3(256), 0, s, A);
    else if (vecs <= 256 * 2) hipLaunchKernelGGL((k_loss_row<XD, TD, 256, 2>), dim3(rows), dim3(256), 0, s, A);
    else if (vecs <= 256 * 4) hipLaunchKernelGGL((k_loss_row<XD, TD, 256, 4>), dim3(rows), dim3(256), 0, s, A);
    else if (vecs <= 512 * 4) hipLaunchKernelGGL((k_loss_row<XD, TD, 512, 4>), dim3(rows), dim3(512), 0, s, A);
    else if (vecs <= 512 * 8) hipLaunchKernelGGL((k_loss_row<XD, TD, 512, 8>), dim3(rows), dim3(512), 0, s, A);
    else if (XD == TD && vecs <= 1024 * 8) {   // f32 targets beside 16-bit logits do not fit the registers
        if constexpr (XD == TD) hipLaunchKernelGGL((k_loss_row<XD, TD, 1024, 8>), dim3(rows), dim3(1024), 0, s, A);
    }
    else {
        const int chunk = chunk_size(A.n, A.v);
        for (int64_t r = 0; r < A.n; r += SLAB) {
            const dim3 grid((unsigned)chunk_count(A.n, A.v), (unsigned)std::min(SLAB, A.n - r));
            hipLaunchKernelGGL((k_loss_part<XD, TD>), grid, dim3(256), 0, s, A, r, chunk, part);
            MZ_LAUNCH_CHECK("k_loss_part");
            hipLaunchKernelGGL((k_loss_join<XD, TD>), grid, dim3(256), 0, s, A, r, chunk, (const Stat *)part);
            MZ_LAUNCH_CHECK("k_loss_join");
        }
    }
    MZ_LAUNCH_CHECK("k_loss");
    return MZ_OK;
}

}  // namespace

extern "C" int64_t mz_policy_loss_workspace_bytes(int64_t n, int64_t v) {
    if (n < 0 || n > MAX_N || v < 1 || v > MAX_V) return -1;
    return std::max<int64_t>(n, 1) * 4 + 16 + std::min(SLAB, n) * chunk_count(n, v) * (int64_t)sizeof(Stat);
}

extern "C" int mz_policy_loss(const mz_policy_loss_args *a, void *workspace, int64_t workspace_bytes, void *stream) {
    const char *who = "mz_policy_loss";
    MZ_REQUIRE(a, "%s: null arguments", who);
    MZ_REQUIRE(a->n >= 0 && a->n <= MAX_N, "%s: n has to be 0 .. 2^22 - 1", who);
    MZ_REQUIRE(a->v >= 1 && a->v <= MAX_V, "%s: v has to be 1 .. 2^24", who);
    MZ_REQUIRE(elem_known(a->dtype), "%s: unknown dtype %d", who, a->dtype);
    MZ_REQUIRE(a->target_dtype == a->dtype || a->target_dtype == MZ_F32, "%s: targets have the logits' dtype or are f32", who);
    MZ_REQUIRE(!a->board || a->v == 65, "%s: a bitboard needs v = 65", who);
    MZ_REQUIRE(!(a->board && a->allowed), "%s: allowed or board, not both", who);
    MZ_REQUIRE(a->row_loss || a->loss || a->grad, "%s: no output", who);
    MZ_REQUIRE(!a->skip_one || (a->grad_out && a->grad_out_stride == 0), "%s: skip_one needs one grad_out", who);
    MZ_REQUIRE(!a->skip_one || (!a->loss && !a->row_loss), "%s: skip_one leaves the loss out", who);
    MZ_REQUIRE(a->grad_out_stride == 0 || a->grad_out_stride == 1, "%s: grad_out_stride is 0 or 1", who);
    if (a->n == 0) return MZ_OK;
    MZ_REQUIRE(a->logits && a->targets, "%s: null logits or targets", who);
    const int xb = elem_bytes(a->dtype), tb = elem_bytes(a->target_dtype);
    MZ_REQUIRE((uintptr_t)a->logits % xb == 0 && (uintptr_t)a->targets % tb == 0 && (uintptr_t)a->grad % xb == 0, "%s: misaligned logits, targets or grad", who);
    MZ_REQUIRE(a->logits_stride >= 0 && a->targets_stride >= 0 && a->allowed_stride >= 0, "%s: negative row strides", who);
    MZ_REQUIRE(!a->grad || a->grad_stride >= a->v, "%s: the gradient's rows overlap", who);
    MZ_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0, "%s: null or misaligned workspace", who);
    MZ_REQUIRE(workspace_bytes >= mz_policy_loss_workspace_bytes(a->n, a->v), "%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes,
               (long long)mz_policy_loss_workspace_bytes(a->n, a->v));
    float *rows = (float *)workspace;
    Stat *part = (Stat *)((char *)workspace + (std::max<int64_t>(a->n, 1) * 4 + 15) / 16 * 16);
    LossArgs A;
    A.x = a->logits;
    A.t = a->targets;
    A.allowed = a->allowed;
    A.board = a->board;
    A.weight = a->weight;
    A.go = a->grad_out;
    A.row_loss = a->row_loss ? a->row_loss : a->loss ? rows : nullptr;
    A.grad = a->grad;
    A.x_stride = a->logits_stride;
    A.t_stride = a->targets_stride;
    A.allowed_stride = a->allowed_stride;
    A.grad_stride = a->grad_stride;
    A.n = a->n;
    A.v = (int)a->v;
    A.go_stride = a->grad_out_stride;
    A.skip_one = a->skip_one;
    A.scale = (float)a->scale;
    hipStream_t s = (hipStream_t)stream;
    int rc;
    if (a->dtype == MZ_F32) rc = launch<MZ_F32, MZ_F32>(A, part, s);
    else if (a->dtype == MZ_BF16) rc = a->target_dtype == MZ_F32 ? launch<MZ_BF16, MZ_F32>(A, part, s) : launch<MZ_BF16, MZ_BF16>(A, part, s);
    else rc = a->target_dtype == MZ_F32 ? launch<MZ_F16, MZ_F32>(A, part, s) : launch<MZ_F16, MZ_F16>(A, part, s);
    if (rc) return rc;
    if (a->loss) {
        hipLaunchKernelGGL(k_loss_sum, dim3(1), dim3(1024), 0, s, (const float *)A.row_loss, a->n, a->scale, a->loss);
        MZ_LAUNCH_CHECK("k_loss_sum");
    }
    return MZ_OK;
}
