// policy_sample_kernels.hip -- one action per row of logits from ONE given uniform number, under a temperature, top-k, top-p and min-p.
//
// For row x with temperature T > 0, over the actions that `legal` leaves and whose logit is above -inf, with m = max x:
//   w_j = exp((x_j - m) / T), and the actions ordered by (x descending, index ascending).
//   top-k keeps the first k;  top-p keeps those of them before which less than p times their total mass lies;  min-p keeps w_j >= min_p;
//   the first is always kept.  With R the mass that is kept, the answer is the lowest index j with sum over kept i <= j of w_i > u R.
// T = 0 answers the first action of the order.  Every filter keeps a PREFIX of the order, so the kept set is "x above a threshold, and the first r
// actions on it": nothing is sorted.
//
// All masses are held in 64 bits, because a draw next to the border of two actions has to fall on its own side: at 131,072 actions f32 sums would put
// one draw in a thousand wrong.  Sums run in a fixed order, or over integers (units of the total's 2^61st part, so that atomics give the same total in any
// order).  The groups' masses of long rows are right to 2e-12.
//
// Up to 512 actions: one wave per row.  Up to 8192: one workgroup of 4, 8 or 16 waves per row.  Both hold the row in registers, one launch; few rows are
// bound by latency (4096 x 65 f32 without a filter 4.3 us, 256 x 4096 bf16 top-p 9 us), thousands under top-p by the search for its cut (4096 x 500 f32
// 27 us, 4096 x 4096 bf16 75 us, over ten times what reading them takes): a 64-bit exponential for every action, and above 512 of them an LDS atomic.
// Longer rows, two launches: k_sample_groups reads the logits once, across all CUs, and leaves the maximum of every 128 actions and, where the
// row's settings need the total, their mass (256 x 131072 bf16: without the masses 13 us, the memory's time; with them 30 us, the 64-bit exponentials', which
// keep the vector ALUs 70 % busy).  k_sample_row, a workgroup per row, works from those: bounds on what can be kept leave few groups, it reads only these
// again, takes the actions above the bound into registers (up to 4096 or 8192) and goes on as for a shorter row (median row 15 us, bound by the
// latency of about ten dependent steps).
#include <math.h>
#include <algorithm>
#include <type_traits>
#include "numeric.h"

namespace {

using namespace mz;

struct SampleArgs {
    const void *x;
    const uint8_t *allowed;
    const uint64_t *board;
    const double *u;
    const float *temperature_of, *top_p_of, *min_p_of;
    const int32_t *top_k_of;
    int32_t *action;
    double temperature, c, top_p, min_p;   // c = log2(e) / temperature
    int64_t x_stride, allowed_stride, n;
    int v, top_k;
};

// one row's settings; a filter that keeps everything is switched off here
struct Setting {
    double c, top_p, min_p;   // c = log2(e) / T
    bool greedy, bad;
    int k;                    // 0 = off
    bool p_on, m_on;
};
__device__ __forceinline__ Setting setting_of(const SampleArgs &A, int64_t row) {
    Setting s;
    const double T = A.temperature_of ? (double)A.temperature_of[row] : A.temperature;
    s.bad = !(T < INFINITY);
    s.top_p = fmax(A.top_p_of ? (double)A.top_p_of[row] : A.top_p, 0.0);
    const double min_p = A.min_p_of ? (double)A.min_p_of[row] : A.min_p;
    s.min_p = fmin(min_p, 1.0);
    const int k = A.top_k_of ? A.top_k_of[row] : A.top_k;
    s.k = k > 0 && k < A.v ? k : 0;
    s.greedy = !(T > 0.0) || s.k == 1;
    s.c = s.greedy ? 0.0 : A.temperature_of ? 1.4426950408889634 / T : A.c;
    s.p_on = (A.top_p_of ? (double)A.top_p_of[row] : A.top_p) < 1.0;   // a NaN is no limit
    s.m_on = min_p > 0.0;
    return s;
}

// 32-bit keys in the order of the values; -0 counts as +0
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }
// (those of a 16-bit type end in bits that are 0 above zero and 1 below)
template <int XD> constexpr int key_ends() { return XD == MZ_F32 ? 0 : XD == MZ_BF16 ? 16 : 13; }
constexpr uint32_t KEY_NONE = 0x007FFFFFu;     // -inf: an action that cannot be played
constexpr uint32_t KEY_LOWEST = 0x00800000u;   // the lowest finite value
constexpr uint32_t KEY_INF = 0xFF800000u;      // +inf, and above it NaN: no distribution

// 2^t for t <= 0: 2^round(t) times a polynomial at f = t - round(t) in [-1/2, 1/2], 1 + f q(f) with q the interpolation of (2^f - 1) / f at the
// Chebyshev nodes (2^0 is 1 exactly): of degree 9, relative error 6e-16, or where FINE is false of degree 7, 2e-12.  Adding 1.5 2^52 rounds t and
// leaves the integer in the low word.  Below 2^-1075 it is 0, as any 64-bit exponential: u = 0 takes none of those.
template <bool FINE> __device__ __forceinline__ double exp2_neg(double t) {
    t = fmax(t, -1100.0);
    const double big = 6755399441055744.0, r = t + big, f = t - (r - big);
    double q;
    if (FINE) {
        q = 7.070977866508138e-09;
        q = fma(q, f, 1.0205905413765595e-07);
        q = fma(q, f, 1.3215451633221434e-06);
        q = fma(q, f, 1.5252672924850737e-05);
        q = fma(q, f, 0.00015403530424776529);
        q = fma(q, f, 0.0013333558200794592);
        q = fma(q, f, 0.009618129107618665);
        q = fma(q, f, 0.05550410866465167);
        q = fma(q, f, 0.24022650695910075);
        q = fma(q, f, 0.6931471805599462);
    } else {
        q = 1.325080551750225e-06;
        q = fma(q, f, 1.5303700711365693e-05);
        q = fma(q, f, 0.00015403475186530786);
        q = fma(q, f, 0.0013333478473685416);
        q = fma(q, f, 0.00961812913523614);
        q = fma(q, f, 0.055504109063258665);
        q = fma(q, f, 0.24022650695888503);
        q = fma(q, f, 0.6931471805568324);
    }
    return ldexp(fma(q, f, 1.0), (int)(uint32_t)__double_as_longlong(r));
}
template <bool FINE = true> __device__ __forceinline__ double mass_of(float x, double m, double c) { return exp2_neg<FINE>(((double)x - m) * c); }

// ---- reductions and scans over a wave in registers: rows of 16 lanes by shifts, then across the rows (lanes that get nothing add 0) ----------
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS> __device__ __forceinline__ double dpp(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)((uint64_t)dpp<CTRL, ROWS>((uint32_t)(b >> 32)) << 32 | dpp<CTRL, ROWS>((uint32_t)b)));
}
template <int CTRL, int ROWS> __device__ __forceinline__ uint64_t dpp(uint64_t v) {
    return (uint64_t)dpp<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | dpp<CTRL, ROWS>((uint32_t)v);
}
template <typename T> __device__ __forceinline__ T scan(T v) {   // inclusive
    v += dpp<0x111, 0xF>(v);
    v += dpp<0x112, 0xF>(v);
    v += dpp<0x114, 0xF>(v);
    v += dpp<0x118, 0xF>(v);
    v += dpp<0x142, 0xA>(v);
    v += dpp<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) { return (uint64_t)lane_of((uint32_t)(v >> 32), lane) << 32 | lane_of((uint32_t)v, lane); }
__device__ __forceinline__ double lane_of(double v, int lane) { return __longlong_as_double((long long)lane_of((uint64_t)__double_as_longlong(v), lane)); }
template <typename T> __device__ __forceinline__ T total(T v) { return lane_of(scan(v), 63); }
// the largest over 16 lanes in their last one, and over the wave in every lane
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    v = max(v, dpp<0x111, 0xF>(v));
    v = max(v, dpp<0x112, 0xF>(v));
    v = max(v, dpp<0x114, 0xF>(v));
    return max(v, dpp<0x118, 0xF>(v));
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    v = max16(v);
    v = max(v, dpp<0x142, 0xA>(v));
    return lane_of(max(v, dpp<0x143, 0xC>(v)), 63);
}
__device__ __forceinline__ uint32_t lane_last16(uint32_t v) { return (uint32_t)__builtin_amdgcn_ds_swizzle((int)v, 0x1F0); }   // lane 15 of each 16
__device__ __forceinline__ double sum16(double v) {   // in the last of 16 lanes
    v += dpp<0x111, 0xF>(v);
    v += dpp<0x112, 0xF>(v);
    v += dpp<0x114, 0xF>(v);
    return v + dpp<0x118, 0xF>(v);
}
__device__ __forceinline__ uint64_t lanes_below(int lane) { return lane ? ~0ull >> (64 - lane) : 0ull; }

// ---- up to 64 E values in one wave's registers, the i-th of them in x[i / 64] of lane i % 64 (-inf: none) ------------------------------------
// The answer's i.  top: the largest key.  all: the mass that top-p shares out, if it is known (> 0).  Thresholds are found among the bits in which the
// keys differ, for top-k one at a time, for top-p by parting the range into WAYS (4 where the wave is alone: three sums at once take little longer
// than one; 2 where many waves share the CU: 4096 x 65 f32, top-p 0.9: 15.0 us against 20.6).
template <int XD, int E, int WAYS> __device__ __forceinline__ int wave_pick(const float *x, const Setting &s, double u, uint32_t top, double all) {
    const int lane = threadIdx.x & 63;
    uint32_t key[E];
#pragma unroll
    for (int k = 0; k < E; ++k) key[k] = key_of(x[k]);
    // the kept set: keys above tau, and the first `ties` on it
    uint32_t tau = KEY_NONE;
    int ties = 0;
    double w[E];
    if (s.greedy) {
        tau = top;
        ties = 1;
#pragma unroll
        for (int k = 0; k < E; ++k) w[k] = key[k] == top ? 1.0 : 0.0;
    } else {
        const double m = (double)value_of(top);
#pragma unroll
        for (int k = 0; k < E; ++k) w[k] = key[k] > KEY_NONE ? mass_of(x[k], m, s.c) : 0.0;
        constexpr int ENDS = key_ends<XD>();
        uint32_t least = 0xFFFFFFFFu;
        int there = 0;
#pragma unroll
        for (int k = 0; k < E; ++k) {
            if (key[k] > KEY_NONE) least = min(least, key[k]);
            there += __popcll(__ballot(key[k] > KEY_NONE));
        }
        least = ~wave_max_u32(~least);
        if (s.k && s.k < there) {   // the largest tau that at least k keys reach
            const uint32_t differ = least ^ top;
            uint32_t bit = differ ? 0x80000000u >> __clz((int)differ) : 0, t = differ ? top & ~(bit | (bit - 1)) : top;
            for (; bit >> ENDS; bit >>= 1) {
                int c = 0;
#pragma unroll
                for (int k = 0; k < E; ++k) c += __popcll(__ballot(key[k] >= (t | bit)));
                if (c >= s.k) t |= bit;
            }
            tau = 0xFFFFFFFFu;
            int above = 0;
#pragma unroll
            for (int k = 0; k < E; ++k)
                if (key[k] >= t) tau = min(tau, key[k]);
            tau = ~wave_max_u32(~tau);
#pragma unroll
            for (int k = 0; k < E; ++k) above += __popcll(__ballot(key[k] > tau));
            ties = s.k - above;
        }
        if (s.p_on) {   // the lowest tau above which less than p of the mass lies
            double sum = 0.0;
#pragma unroll
            for (int k = 0; k < E; ++k) sum += key[k] > tau ? w[k] : 0.0;
            sum = total(sum) + (tau > KEY_NONE ? ties * mass_of(value_of(tau), m, s.c) : 0.0);
            const double limit = lane_of(s.top_p * (all > 0.0 ? all : sum), 0);   // the same in every lane: the search below branches for the whole wave
            // the answer lies in [lo, hi]: the least key that can be kept, and the largest, above which nothing is (in steps of 2^ENDS, which part all keys)
            uint32_t lo = max(least, tau) >> ENDS, hi = top >> ENDS;
            while (lo < hi) {
                const uint32_t step = max(1u, (hi - lo + 1) / WAYS);
                uint32_t mid[WAYS - 1];
                double over[WAYS - 1];
#pragma unroll
                for (int i = 0; i < WAYS - 1; ++i) {
                    mid[i] = min(hi, lo + step * (i + 1) - 1);
                    const uint32_t edge = mid[i] << ENDS | ((1u << ENDS) - 1);
                    over[i] = 0.0;
#pragma unroll
                    for (int k = 0; k < E; ++k) over[i] += key[k] > edge ? w[k] : 0.0;
                }
#pragma unroll
                for (int i = 0; i < WAYS - 1; ++i) over[i] = scan(over[i]);
                uint32_t from = lo, upto = hi;
#pragma unroll
                for (int i = WAYS - 2; i >= 0; --i) {
                    const bool below = __builtin_amdgcn_readfirstlane(lane_of(over[i], 63) < limit);
                    upto = below ? mid[i] : upto;
                    from = !below && from == lo ? mid[i] + 1 : from;
                }
                lo = min(from, upto);
                hi = upto;
            }
            lo = ENDS ? (lo << ENDS) | (lo << ENDS & 0x80000000u ? 0 : (1u << ENDS) - 1) : lo;
            double above = 0.0;
            int on = 0;
#pragma unroll
            for (int k = 0; k < E; ++k) {
                above += key[k] > lo ? w[k] : 0.0;
                on += __popcll(__ballot(key[k] == lo));
            }
            above = total(above);
            const double wl = mass_of(value_of(lo), m, s.c);
            int r = 0;
            while (r < on && above + r * wl < limit) ++r;
            if (lo == top && r < 1) r = 1;
            if (lo > tau) {
                tau = lo;
                ties = r;
            } else ties = min(ties, r);
        }
    }
    // cumulated in the actions' own order
    double part[E], base = 0.0;
    int seen = 0;
    uint64_t keep[E];
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const uint64_t on = __ballot(key[k] == tau);
        bool kept = key[k] > tau || (key[k] == tau && seen + (int)__popcll(on & lanes_below(lane)) < ties);
        if (!s.greedy && s.m_on) kept = kept && (w[k] >= s.min_p || key[k] == top);
        seen += __popcll(on);
        keep[k] = __ballot(kept);
        part[k] = 0.0;
        if (keep[k]) {
            part[k] = base + scan(kept ? w[k] : 0.0);
            base = lane_of(part[k], 63);
        }
    }
    const double target = u * base;
    int pick = -1, last = -1;
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const uint64_t hit = __ballot(part[k] > target) & keep[k];
        if (pick < 0 && hit) pick = k * 64 + __ffsll((unsigned long long)hit) - 1;
        if (keep[k]) last = k * 64 + 63 - __clzll((long long)keep[k]);
    }
    return pick < 0 ? last : pick;
}

// ---- up to 512 actions: one wave per row ---------------------------------------------------------------------------------------------
template <int XD, int E> __global__ void __launch_bounds__(256) k_sample_wave(SampleArgs A) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= A.n) return;
    const Setting s = setting_of(A, row);
    const int64_t xo = row * A.x_stride, ao = row * A.allowed_stride;
    const uint64_t board = A.board ? A.board[row] : 0;
    float x[E];
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const int j = k * 64 + lane;
        bool ok = j < A.v;
        if (ok && A.allowed) ok = A.allowed[ao + j] != 0;
        if (ok && A.board) ok = j < 64 ? (board >> j) & 1 : board == 0;
        x[k] = ok ? load_one<XD>(A.x, xo + j) : -INFINITY;
        top = max(top, x[k] != x[k] ? 0xFFFFFFFFu : key_of(x[k]));
    }
    top = wave_max_u32(top);
    if (top <= KEY_NONE || top >= KEY_INF || s.bad) {
        if (lane == 0) A.action[row] = -1;
        return;
    }
    const int pick = wave_pick<XD, E, 2>(x, s, A.u[row], top, 0.0);
    if (lane == 0) A.action[row] = pick;
}

// eight actions of a row as they lie there (so that their loads can be under way while others are worked on)
template <int XD> struct Eight {
    Words<XD, 8> words;
    uint64_t ok;                                 // with a mask: a byte each, 0 = not legal
    __device__ __forceinline__ void none() {
#pragma unroll
        for (int j = 0; j < 8; ++j) words.set(j, (typename Elem<XD>::T)(XD == MZ_F32 ? 0xFF800000u : XD == MZ_BF16 ? 0xFF80u : 0xFC00u));
        ok = ~0ull;
    }
    __device__ __forceinline__ void load(const SampleArgs &A, int64_t xo, int64_t ao, int at) {
        if (at + 8 <= A.v) {
            words = load_words<XD, 8>(A.x, xo + at);
            if (A.allowed) ok = load_flags(A.allowed, ao + at);
        } else {                                 // behind the row's end: -inf
            none();
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (at + j < A.v) {
                    words.set(j, ((const MZ_GLOBAL typename Elem<XD>::T *)A.x)[xo + at + j]);
                    if (A.allowed && !A.allowed[ao + at + j]) ok &= ~(0xFFull << j * 8);
                }
        }
    }
    __device__ __forceinline__ void unpack(const SampleArgs &A, float *x) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = words.get(j);
        if (A.allowed)                           // the same for the whole launch
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = (ok >> j * 8) & 0xFF ? x[j] : -INFINITY;
    }
};

// ---- what a workgroup of W waves does together -----------------------------------------------------------------------------------------
template <int W> struct Shared {
    static constexpr int THREADS = 64 * W, BINS = 4 * THREADS, FEW = 64;
    unsigned long long hist[BINS];
    unsigned long long few_amount[FEW];
    uint32_t few_key[FEW];
    unsigned long long wave_u64[W];
    double wave_f64[W];
    uint32_t wave_u32[W];
    unsigned long long above;
    double base;
    int bin, few, pick;
};

template <int W, typename T> __device__ __forceinline__ T block_total(T v, T *of_wave) {   // of_wave may be used again after the call
    v = total(v);
    if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = v;
    __syncthreads();
    T t = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) t += of_wave[i];
    __syncthreads();
    return t;
}
template <int W> __device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t *of_wave) {
    v = wave_max_u32(v);
    if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) v = max(v, of_wave[i]);
    __syncthreads();
    return v;
}

// The bin of the histogram that takes the amounts from below `limit` to it, counted from bin 0; -1: their total stays below.  `above`: what lies
// in the bins before it, on entry and on return together with what was there.
template <int W> __device__ __forceinline__ int crossing_bin(Shared<W> &S, uint64_t limit, uint64_t *above) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t h[4], own = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) own += h[i] = S.hist[threadIdx.x * 4 + i];
    const uint64_t sum = scan(own);
    if (lane == 63) S.wave_u64[wave] = sum;
    __syncthreads();
    uint64_t before = *above + sum - own;
#pragma unroll
    for (int i = 0; i < W; ++i) before += i < wave ? S.wave_u64[i] : 0;
    if (before < limit && before + own >= limit) {   // one thread at most
        int i = 0;
        while (before + h[0] < limit) {
            before += h[0];
            h[0] = h[1];
            h[1] = h[2];
            h[2] = h[3];
            ++i;
        }
        S.bin = threadIdx.x * 4 + i;
        S.above = before;
    }
    __syncthreads();
    if (S.bin >= 0) *above = S.above;
    return S.bin;
}

// The lowest tau in [lo, hi] with (amount above tau) < limit, where `each` hands (key, value, function of the amount) of everything in the row to
// its argument; *above = that amount.  False: all of it together stays below the limit.  Amounts are integers, so the order of the atomics does
// not matter.  `guess` >= lo: where tau is looked for first; `ends` = bits of a key that its type leaves empty.
// The first histogram, from `guess` on, has bins of equal width in the value, which few logits share; the up to 64 of the bin that reaches the limit
// are ranked in registers.  More: histograms over the bits of that bin's keys, each narrowing to one bin of the one before, unless they are all equal
// (256 x 131072 bf16, flat, p = 0.9: 190 us; from all keys 259).  Tau below the guess: the same from all keys.
template <int W, class EACH>
__device__ __forceinline__ bool find_threshold(EACH each, uint32_t lo, uint32_t guess, uint32_t hi, uint64_t limit, int ends, Shared<W> &S,
                                               uint32_t *tau, uint64_t *above_out) {
    constexpr int BINS = Shared<W>::BINS, BITS = W == 4 ? 10 : W == 8 ? 11 : 12, FEW = Shared<W>::FEW;
    static_assert(1 << BITS == BINS, "a bin for each key of that many bits");
    const int lane = threadIdx.x & 63;
    auto clear = [&] {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) S.hist[threadIdx.x * 4 + i] = 0;
        if (threadIdx.x == 0) {
            S.bin = -1;
            S.few = 0;
        }
        __syncthreads();
    };
    uint64_t above = 0;
    const float xh = value_of(hi), width = xh - value_of(guess), scale = BINS / width;
    if (((hi - guess) >> ends) >= BINS && scale > 0.0f && scale < 1e30f) {
        auto bin_of = [&](float x) { return min(BINS - 1, (int)((xh - x) * scale)); };
        clear();
        each([&](uint32_t key, float x, auto amount) {
            if (key >= guess && key <= hi) atomicAdd(&S.hist[bin_of(x)], (unsigned long long)amount());
        });
        __syncthreads();
        const int bin = crossing_bin(S, limit, &above);
        if (bin < 0 && guess == lo) return false;
        uint32_t least = 0xFFFFFFFFu, most = 0;
        if (bin >= 0) each([&](uint32_t key, float x, auto amount) {
            if (key >= guess && key <= hi && bin_of(x) == bin) {
                const int i = atomicAdd(&S.few, 1);
                least = min(least, key);
                most = max(most, key);
                if (i < FEW) {
                    S.few_key[i] = key;
                    S.few_amount[i] = (unsigned long long)amount();
                }
            }
        });
        __syncthreads();
        const int few = S.few;
        if (bin >= 0 && few <= FEW) {
            const uint32_t key = lane < few ? S.few_key[lane] : 0;
            const uint64_t amount = lane < few ? (uint64_t)S.few_amount[lane] : 0;
            uint64_t over = above;
            for (int i = 0; i < few; ++i) {
                const uint32_t k = lane_of(key, i);
                const uint64_t a = lane_of(amount, i);
                if (k > key) over += a;
            }
            const uint32_t best = lane < few && over < limit ? key : 0xFFFFFFFFu;
            *tau = ~wave_max_u32(~best);
            *above_out = lane_of(over, __ffsll((unsigned long long)__ballot(best == *tau)) - 1);
            return true;
        }
        if (bin >= 0) {           // above: what lies above the bin
            lo = ~block_max<W>(~least, S.wave_u32);
            hi = block_max<W>(most, S.wave_u32);
            if (lo == hi) {
                *tau = lo;
                *above_out = above;
                return true;
            }
        }
    }
    for (;;) {
        const int shift = max(0, 32 - __clz((int)(hi - lo)) - BITS);   // (hi - lo) >> shift < BINS
        clear();
        each([&](uint32_t key, float, auto amount) {
            if (key >= lo && key <= hi) atomicAdd(&S.hist[(hi - key) >> shift], (unsigned long long)amount());
        });
        __syncthreads();
        const int bin = crossing_bin(S, limit, &above);
        if (bin < 0) return false;
        hi -= (uint32_t)bin << shift;
        if (shift <= ends) {      // one key: the one whose low bits are what its type leaves there, 0 above zero and 1 below
            const uint32_t low = (1u << ends) - 1;
            uint32_t t = hi & 0x80000000u ? hi & ~low : hi | low;
            if (t > hi) t -= low + 1;
            *tau = t;
            *above_out = above;
            return true;
        }
        lo = hi - lo < (1u << shift) ? lo : hi - (1u << shift) + 1;
    }
}

// Masses as integers, for sums that the order of atomics does not change: the total that is shared out becomes 2^61 .. 2^62, so a unit is 2^-61 of it at
// most and 2^19 masses, each rounded by half a unit, are 2^-43 of it off together.  (In units of 2^-44 of the BEST mass a long tail behind one action
// far ahead would be cut a fifth too short.)
__device__ __forceinline__ double int_scale(double total) { return ldexp(1.0, 61 - ilogb(total)); }
__device__ __forceinline__ uint64_t int_mass(double w, double scale) { return (uint64_t)fma(w, scale, 0.5); }
// how many of up to `ties` actions of mass w begin before `left` is used up
__device__ __forceinline__ uint32_t ties_within(double left, double w, uint32_t ties) { return left > 0.0 ? (uint32_t)fmin(ceil(left / w), (double)ties) : 0; }

// The answer for what the workgroup's threads hold in registers, thread by thread in the actions' order, N in each: the place of the picked one
// (thread N + j), in every thread.  best: the largest key.  low: nothing below it is kept.  all: the mass that top-p shares out, if it is known (> 0).
template <int XD, int W, int N>
__device__ __forceinline__ int pick(const float *x, const Setting &s, double u, int v, uint32_t best, uint32_t low, double all, Shared<W> &S) {
    constexpr int ENDS = key_ends<XD>();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const double m = (double)value_of(best);
    uint32_t tau = KEY_NONE, ties = 0;           // the kept set: keys above tau, and the first `ties` on it
    double w[N];
    {
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = mass_of(x[j], m, s.c);
        uint64_t above;
        if (low == KEY_LOWEST && (s.k || s.p_on)) {   // no bound yet: the least value that is there
            uint32_t least = 0xFFFFFFFFu;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint32_t key = key_of(x[j]);
                if (key > KEY_NONE) least = min(least, key);
            }
            low = ~block_max<W>(~least, S.wave_u32);
        }
        if (s.k) {
            auto each = [&](auto take) {
#pragma unroll
                for (int j = 0; j < N; ++j) take(key_of(x[j]), x[j], [] { return 1ull; });
            };
            uint32_t t;
            if (find_threshold(each, low, low, best, (uint64_t)s.k, ENDS, S, &t, &above)) {
                tau = t;
                ties = (uint32_t)(s.k - above);
            }
        }
        if (s.p_on) {
            // The cut is looked for above top-k's threshold (on it lie more actions than top-k keeps); where those above do not fill p, on it.
            double over = 0.0;
            const double wt = tau > KEY_NONE ? mass_of(value_of(tau), m, s.c) : 0.0;
            if (!(all > 0.0)) {
#pragma unroll
                for (int j = 0; j < N; ++j) over += key_of(x[j]) > tau ? w[j] : 0.0;
                over = block_total<W>(over, S.wave_f64);
                all = over + ties * wt;
            }
            const uint32_t from = tau > KEY_NONE ? tau + 1 : low;
            const double scale = int_scale(all);
            const uint64_t amount = (uint64_t)fmax(1.0, ceil(s.top_p * all * scale));
            auto each = [&](auto take) {
                double by = scale;
                asm volatile("" : "+v"(by));     // not the same value to the compiler, which would keep all integers beside the masses
#pragma unroll
                for (int j = 0; j < N; ++j) take(key_of(x[j]), x[j], [&] { return int_mass(w[j], by); });
            };
            uint32_t t;
            if (from <= best && find_threshold(each, from, from, best, amount, ENDS, S, &t, &above)) {
                ties = ties_within((double)(amount - above), mass_of(value_of(t), m, s.c) * scale, v);
                tau = t;
            } else if (tau > KEY_NONE) ties = max(tau == best ? 1u : 0u, ties_within(s.top_p * all - over, wt, ties));
        }
    }
    // cumulated in the actions' order
    uint32_t on = 0;
    if (tau > KEY_NONE)
#pragma unroll
        for (int j = 0; j < N; ++j) on += key_of(x[j]) == tau;
    const uint32_t on_upto = scan(on);
    __syncthreads();
    if (lane == 63) S.wave_u32[wave] = on_upto;
    if (threadIdx.x == 0) S.pick = 0x7FFFFFFF;
    __syncthreads();
    uint32_t rank = on_upto - on;
#pragma unroll
    for (int i = 0; i < W; ++i) rank += i < wave ? S.wave_u32[i] : 0;
    double own = 0.0;
    uint32_t keep = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint32_t key = key_of(x[j]);
        bool kept = key > tau;
        if (key == tau && on) kept = rank++ < ties;
        if (s.m_on) kept = kept && (w[j] >= s.min_p || key == best);
        if (kept) {
            keep |= 1u << j;
            own += w[j];
        }
    }
    const double sum = scan(own);
    if (lane == 63) S.wave_f64[wave] = sum;
    __syncthreads();
    double cum = sum - own, everything = 0.0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        cum += i < wave ? S.wave_f64[i] : 0.0;
        everything += S.wave_f64[i];
    }
    const double target = u * everything;
    int mine = -1, last = -1;
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (keep >> j & 1) {
            cum += w[j];
            last = j;
            if (mine < 0 && cum > target) mine = j;
        }
    if (mine >= 0) atomicMin(&S.pick, (int)threadIdx.x * N + mine);
    __syncthreads();
    int at = S.pick;
    if (at == 0x7FFFFFFF) {                      // rounding, or u >= 1: the last that is kept
        __syncthreads();
        if (threadIdx.x == 0) S.pick = -1;
        __syncthreads();
        if (last >= 0) atomicMax(&S.pick, (int)threadIdx.x * N + last);
        __syncthreads();
        at = S.pick;
    }
    return at;
}

// ---- up to 512 W actions: a workgroup of W waves per row, eight neighbouring actions in a thread -----------------------------------------
template <int XD, int W> __global__ void __launch_bounds__(64 * W) k_sample_block(SampleArgs A) {
    __shared__ Shared<W> S;
    const int64_t row = blockIdx.x;
    const Setting s = setting_of(A, row);
    float x[8];
    Eight<XD> e;
    e.load(A, row * A.x_stride, row * A.allowed_stride, threadIdx.x * 8);
    e.unpack(A, x);
    uint32_t best = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) best = max(best, x[j] != x[j] ? 0xFFFFFFFFu : key_of(x[j]));
    best = block_max<W>(best, S.wave_u32);
    if (best <= KEY_NONE || best >= KEY_INF || s.bad) {
        if (threadIdx.x == 0) A.action[row] = -1;
        return;
    }
    if (s.greedy) {
        if (threadIdx.x == 0) S.pick = 0x7FFFFFFF;
        __syncthreads();
#pragma unroll
        for (int j = 7; j >= 0; --j)
            if (key_of(x[j]) == best) atomicMin(&S.pick, (int)threadIdx.x * 8 + j);
        __syncthreads();
        if (threadIdx.x == 0) A.action[row] = S.pick;
        return;
    }
    const int at = pick<XD, W, 8>(x, s, A.u[row], A.v, best, KEY_LOWEST, 0.0, S);
    if (threadIdx.x == 0) A.action[row] = at;
}

// ---- longer rows ---------------------------------------------------------------------------------------------------------------------
constexpr int GROUP = 128;          // actions whose maximum and mass are kept together: 16 lanes of 8
constexpr int MAX_V = 1 << 19;      // 4096 groups
// rows that one workgroup holds in registers from the start
inline bool in_block(int64_t n, int64_t v) { return v <= 4096 || (v <= 8192 && n <= 512); }

// whether a row's total mass has to come from all of its actions
__device__ __forceinline__ bool needs_mass(const Setting &s) { return !s.greedy && !s.k && (s.p_on || !s.m_on); }

// a workgroup takes TILES x 2048 actions of one row, sixteen lanes a group, the next tile's loads under way
template <int XD, int TILES> __global__ void __launch_bounds__(256) k_sample_groups(SampleArgs A, int groups, double *mass, uint32_t *top) {
    const int64_t row = blockIdx.y;
    const Setting s = setting_of(A, row);
    const bool massed = needs_mass(s);
    const int64_t xo = row * A.x_stride, ao = row * A.allowed_stride;
    const int first = blockIdx.x * (TILES * 2048) + threadIdx.x * 8;
    Eight<XD> e, e2;
    e.load(A, xo, ao, first);                    // behind the row's end: nothing is read
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        const int at = first + t * 2048, g = at / GROUP;
        if (t + 1 < TILES) e2.load(A, xo, ao, at + 2048);
        float x[8], m = -INFINITY;
        e.unpack(A, x);
        bool nan = false;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            m = fmaxf(m, fmaxf(x[j], x[j + 1]));
            nan |= __builtin_isunordered(x[j], x[j + 1]);
        }
        const uint32_t key = lane_last16(max16(nan ? 0xFFFFFFFFu : key_of(m)));
        const bool writes = (threadIdx.x & 15) == 15 && g < groups;
        if (writes) top[row * groups + g] = key;
        if (massed) {
            double w = 0.0;
            if (key > KEY_NONE && key < KEY_INF) {
                const double md = (double)value_of(key);
#pragma unroll
                for (int j = 0; j < 8; ++j) w += mass_of<false>(x[j], md, s.c);   // 2e-12 of a group's mass moves no draw that 1e-12 of the row would not
            }
            w = sum16(w);
            if (writes) mass[row * groups + g] = w;
        }
        if (t + 1 < TILES) e = e2;
    }
}

// LDS of a row: its groups, then the actions that its bounds leave, SEG to each wave
template <int W, int N> struct RowShared {
    static constexpr int SEG = 64 * N;
    Shared<W> S;
    float x[W * SEG];
    int32_t index[W * SEG];
    uint16_t list[MAX_V / GROUP];
};

template <int XD, int W, int N> __global__ void __launch_bounds__(64 * W) k_sample_row(SampleArgs A, int groups, const double *mass_in, const uint32_t *top_in) {
    constexpr int THREADS = 64 * W, SEG = RowShared<W, N>::SEG, ENDS = key_ends<XD>();
    __shared__ RowShared<W, N> R;
    extern __shared__ double dyn[];
    Shared<W> &S = R.S;
    double *mass = dyn;                          // of a group: all of it, later what is kept of it
    uint32_t *top = (uint32_t *)(dyn + groups);  // its largest key, later how many actions on the threshold come before it
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Setting s = setting_of(A, row);
    const int64_t xo = row * A.x_stride, ao = row * A.allowed_stride;
    const bool massed = needs_mass(s), filtered = s.k || s.p_on || s.m_on;

    uint32_t best = 0;
    for (int g = threadIdx.x; g < groups; g += THREADS) {
        top[g] = top_in[row * groups + g];
        if (massed) mass[g] = mass_in[row * groups + g];
        best = max(best, top[g]);
    }
    if (threadIdx.x == 0) S.pick = 0x7FFFFFFF;
    best = block_max<W>(best, S.wave_u32);
    if (best <= KEY_NONE || best >= KEY_INF || s.bad) {
        if (threadIdx.x == 0) A.action[row] = -1;
        return;
    }
    const double m = (double)value_of(best), u = A.u[row];
    uint32_t tau = KEY_NONE, ties = 0;           // the kept set: keys above tau, and the first `ties` on it
    double target = -1.0;
    int found;

    if (s.greedy) {
        for (int g = threadIdx.x; g < groups; g += THREADS)
            if (top[g] == best) atomicMin(&S.pick, g);
        __syncthreads();
        found = S.pick;
        tau = best - 1;
        if (threadIdx.x == 0) S.base = 0.0;
        __syncthreads();
    } else {
        if (massed)
            for (int g = threadIdx.x; g < groups; g += THREADS) mass[g] = top[g] > KEY_NONE ? mass[g] * mass_of(value_of(top[g]), m, s.c) : 0.0;
        if (filtered) {
            // Nothing below `low` is kept, nor counts in what top-p shares out.  (With top-k, top-p shares out the mass of the k first, also of
            // those that min-p drops, so min-p gives no bound there.)
            uint32_t low = KEY_LOWEST;
            bool bounded = true;
            auto bound = [&](double x) {         // the key of a value a little below x
                const float f = (float)(x - 1e-6 * (fabs(x) + fabs(m)));
                return max(low, min(best, max(key_of(f), KEY_LOWEST + 2) - 2));
            };
            // (1e-12: w rounds up to min_p at that distance too, and at a high temperature a step of w is far in x.)
            if (s.m_on && !(s.k && s.p_on)) low = bound(m + (log2(s.min_p) - 1e-12) / s.c);
            if (s.k) {                           // each wave takes every W-th group: if q = k / W of them reach a value in every wave, k actions do
                const int q = (s.k + W - 1) / W;
                uint32_t t = 0;
                bounded = q <= groups / W;
                if (bounded) {
                    constexpr int PER = MAX_V / GROUP / THREADS;
                    uint32_t mine[PER];
#pragma unroll
                    for (int i = 0; i < PER; ++i) {
                        const int g = wave + lane * W + i * THREADS;
                        mine[i] = g < groups ? top[g] : 0;
                    }
                    // the low bits stay 0: a little lower is a bound too
                    if (groups <= THREADS) {
                        for (uint32_t bit = 0x80000000u; bit > 0x2000; bit >>= 1)
                            if ((int)__popcll(__ballot(mine[0] >= (t | bit))) >= q) t |= bit;
                    } else
                        for (uint32_t bit = 0x80000000u; bit > 0x2000; bit >>= 1) {
                            int c = 0;
#pragma unroll
                            for (int i = 0; i < PER; ++i) c += (int)__popcll(__ballot(mine[i] >= (t | bit)));
                            if (c >= q) t |= bit;
                        }
                }
                t = ~block_max<W>(~t, S.wave_u32);
                low = max(low, t);
            }
            double all = 0.0;
            if (massed) {
                for (int g = threadIdx.x; g < groups; g += THREADS) all += mass[g];
                all = block_total<W>(all, S.wave_f64);
                // Actions of a mass below b have less than (1 - p) of the total together if the groups' masses, each at most 128 b, do: then none of
                // them is kept.  True for b = (1 - p) of the mean mass; the waves try 4, 16, ... times that.
                const double rest = (1.0 - s.top_p) * all * (1.0 - 1e-9);
                double b = rest / ((double)groups * GROUP);
                uint32_t good = 0;
                if (s.p_on) {
#pragma unroll
                    for (int i = 0; i < 16 / W; ++i) {
                        const int step = wave * (16 / W) + i + 1;
                        const double most = ldexp(b, 2 * step) * GROUP;
                        double sum = 0.0;
#pragma unroll 8
                        for (int g = lane; g < groups; g += 64) sum += fmin(mass[g], most);
                        if (total(sum) < rest) good = step;
                    }
                    good = block_max<W>(good, S.wave_u32);
                    low = bound(m + (log2(b) + 2.0 * good) / s.c);
                }
            }
            // the groups that reach `need`, in order, in R.list; their number
            auto list_groups = [&](uint32_t need) {
                const int run0 = (int)((int64_t)groups * wave / W), run1 = (int)((int64_t)groups * (wave + 1) / W);
                int n = 0;
                for (int g = run0; g < run1; g += 64) n += (int)__popcll(__ballot(g + lane < run1 && top[min(g + lane, groups - 1)] >= need));
                __syncthreads();
                if (lane == 0) S.wave_u32[wave] = (uint32_t)n;
                __syncthreads();
                int to = 0, all_of_them = 0;
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const int c = (int)S.wave_u32[i];
                    to += i < wave ? c : 0;
                    all_of_them += c;
                }
                for (int g = run0; g < run1; g += 64) {
                    const bool reach = g + lane < run1 && top[min(g + lane, groups - 1)] >= need;
                    const uint64_t b = __ballot(reach);
                    if (reach) R.list[to + (int)__popcll(b & lanes_below(lane))] = (uint16_t)(g + lane);
                    to += (int)__popcll(b);
                }
                __syncthreads();
                return all_of_them;
            };
            // Every wave walks over an equal share of the listed groups, in order, sixteen lanes to a group, the loads of DEPTH times four groups under way
            // together; `take` gets a lane's group (-1: none) and its eight actions, and says whether to go on.
            auto walk = [&](int listed, auto take) {
                constexpr int DEPTH = XD == MZ_F32 ? 3 : 4;   // what fits 128 registers
                const int q1 = (int)((int64_t)listed * (wave + 1) / W);
                for (int q = (int)((int64_t)listed * wave / W); q < q1; q += 4 * DEPTH) {
                    Eight<XD> e[DEPTH];
                    int mine[DEPTH];
#pragma unroll
                    for (int d = 0; d < DEPTH; ++d) {
                        const int i = q + 4 * d + (lane >> 4);
                        mine[d] = i < q1 ? (int)R.list[i] : -1;
                        if (mine[d] >= 0) e[d].load(A, xo, ao, mine[d] * GROUP + (lane & 15) * 8);
                        else e[d].none();
                    }
#pragma unroll
                    for (int d = 0; d < DEPTH; ++d) {
                        if (q + 4 * d >= q1) return;
                        float x[8];
                        e[d].unpack(A, x);
                        if (!take(mine[d], x)) return;
                    }
                }
            };
            // where the k-th is looked for first: `low` or, without a bound, twice as far below the best as the least of the groups' maxima
            auto first_guess = [&]() -> uint32_t {
                if (bounded) return low;
                uint32_t least = 0xFFFFFFFFu;
                for (int g = threadIdx.x; g < groups; g += THREADS)
                    if (top[g] > KEY_NONE) least = min(least, top[g]);
                least = ~block_max<W>(~least, S.wave_u32);
                return bound(m - 2.0 * (m - (double)value_of(least)));
            };
            // The actions from `low` on, in their order, each wave's in a segment of its own.  Too many (or no bound yet) where top-k keeps at most half of
            // what fits: the k-th largest's place in a histogram of the values is a closer bound, and once more (k = 2000, that / the row read again
            // for each step: 256 x 131072 bf16 64 / 118 us, 64 x 10000 f32 25 / 30 us).
            int count, listed, many, most, start[W + 1];
            for (bool closer = false;;) {
                count = 0;
                listed = list_groups(low);
                if (bounded) {
                    const float least = value_of(low);
                    walk(listed, [&](int g, const float *x) {
                        uint32_t n = 0;
#pragma unroll
                        for (int j = 0; j < 8; ++j) n += x[j] >= least;
                        const uint32_t upto = scan(n);
                        int to = count + (int)(upto - n);
                        count += (int)lane_of(upto, 63);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (x[j] >= least) {
                                if (to < SEG) {
                                    R.x[wave * SEG + to] = x[j];
                                    R.index[wave * SEG + to] = g * GROUP + (lane & 15) * 8 + j;
                                }
                                ++to;
                            }
                        return count <= SEG;
                    });
                }
                __syncthreads();
                if (lane == 0) S.wave_u32[wave] = bounded ? (uint32_t)count : SEG + 1u;
                __syncthreads();
                many = most = start[0] = 0;
                const uint32_t of_wave = lane < W ? S.wave_u32[lane] : 0;
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const int c = (int)lane_of(of_wave, i);
                    most = max(most, c);
                    many += c;
                    start[i + 1] = many;
                }
                if (most <= SEG || closer || !s.k || s.k > W * SEG / 2) break;
                closer = true;
                __syncthreads();                 // wave_u32 is used again
                constexpr int BINS = Shared<W>::BINS;
                const uint32_t from = first_guess();
                const float high = value_of(best), width = high - value_of(from), scale = BINS / width;
                if (!(scale > 0.0f && scale < 1e30f)) break;
#pragma unroll
                for (int i = 0; i < 4; ++i) S.hist[threadIdx.x * 4 + i] = 0;
                if (threadIdx.x == 0) S.bin = -1;
                __syncthreads();
                walk(listed, [&](int, const float *x) {
                    const float least = value_of(from);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (x[j] >= least) atomicAdd(&S.hist[min(BINS - 1, (int)((high - x[j]) * scale))], 1ull);
                    return true;
                });
                __syncthreads();
                uint64_t above = 0;
                const int bin = crossing_bin(S, (uint64_t)s.k, &above);
                if (bin < 0) break;
                low = bound((double)high - (bin + 1.0) / BINS * (double)width);
                bounded = true;
            }
            // few: one wave goes on without the others (4 x 131072 f32, top-k 50 and top-p: 17.9 us; the workgroup together 24.0)
            if (most <= SEG && many <= 512) {
                if (wave) return;
                auto finish = [&](auto size) {
                    constexpr int E = decltype(size)::value;
                    int slot[E];
                    float x[E];
#pragma unroll
                    for (int k = 0; k < E; ++k) {
                        const int i = k * 64 + lane;
                        slot[k] = i;
#pragma unroll
                        for (int j = 1; j < W; ++j) slot[k] = i >= start[j] ? j * SEG + i - start[j] : slot[k];
                        x[k] = i < many ? R.x[slot[k]] : -INFINITY;
                    }
                    const int at = wave_pick<XD, E, 4>(x, s, u, best, massed ? all : 0.0);
#pragma unroll
                    for (int k = 0; k < E; ++k)
                        if (at >= 0 && at >> 6 == k && (at & 63) == lane) A.action[row] = R.index[slot[k]];
                };
                if (many <= 64) finish(std::integral_constant<int, 1>());
                else if (many <= 192) finish(std::integral_constant<int, 3>());
                else finish(std::integral_constant<int, 8>());
                return;
            }
            __syncthreads();                     // wave_u32 is used again
            if (most <= SEG) {
                float x[N];
#pragma unroll
                for (int j = 0; j < N; ++j) x[j] = lane * N + j < count ? R.x[wave * SEG + lane * N + j] : -INFINITY;
                const int at = pick<XD, W, N>(x, s, u, A.v, best, low, massed ? all : 0.0, S);
                if (threadIdx.x == 0) A.action[row] = at >= 0 ? R.index[at] : -1;
                return;
            }

            // Too many for the registers: the same steps with the row read again for each.
            uint64_t above;
            if (s.k) {
                uint32_t t;
                auto each = [&](auto take) {
                    walk(listed, [&](int, const float *x) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) take(key_of(x[j]), x[j], [] { return 1ull; });
                        return true;
                    });
                };
                if (find_threshold(each, low, first_guess(), best, (uint64_t)s.k, ENDS, S, &t, &above)) {
                    tau = t;
                    ties = (uint32_t)(s.k - above);
                }
            }
            if (s.p_on) {
                const uint32_t from = tau > KEY_NONE ? tau + 1 : low;   // as in `pick`
                double over = 0.0;
                const double wt = tau > KEY_NONE ? mass_of(value_of(tau), m, s.c) : 0.0;
                listed = list_groups(from);
                if (!massed) {
                    walk(listed, [&](int, const float *x) {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (key_of(x[j]) >= from) over += mass_of(x[j], m, s.c);
                        return true;
                    });
                    over = block_total<W>(over, S.wave_f64);
                }
                const double shared = massed ? all : over + ties * wt, scale = int_scale(shared);
                const uint64_t amount = (uint64_t)fmax(1.0, ceil(s.top_p * shared * scale));
                uint32_t t;
                auto each = [&](auto take) {
                    walk(listed, [&](int, const float *x) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) take(key_of(x[j]), x[j], [&] { return int_mass(mass_of(x[j], m, s.c), scale); });
                        return true;
                    });
                };
                if (from <= best && find_threshold(each, from, from, best, amount, ENDS, S, &t, &above)) {
                    ties = ties_within((double)(amount - above), mass_of(value_of(t), m, s.c) * scale, A.v);
                    tau = t;
                } else if (tau > KEY_NONE) ties = max(tau == best ? 1u : 0u, ties_within(s.top_p * shared - over, wt, ties));
                else tau = low - 1;   // rounding: everything from `low` on
            }
            // what is kept of every group, and how many actions on the threshold come before it
            uint32_t on = 0;
            listed = list_groups(max(low, tau));
            if (tau > KEY_NONE)
                walk(listed, [&](int, const float *x) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) on += key_of(x[j]) == tau;
                    return true;
                });
            on = total(on);
            __syncthreads();
            if (lane == 0) S.wave_u32[wave] = on;
            for (int g = threadIdx.x; g < groups; g += THREADS) mass[g] = 0.0;
            if (threadIdx.x == 0) S.pick = 0x7FFFFFFF;
            __syncthreads();
            uint32_t seen = 0;
#pragma unroll
            for (int i = 0; i < W; ++i) seen += i < wave ? S.wave_u32[i] : 0;
            walk(listed, [&](int g, const float *x) {
                uint32_t c = 0;
                if (tau > KEY_NONE)
#pragma unroll
                    for (int j = 0; j < 8; ++j) c += key_of(x[j]) == tau;
                const uint32_t upto = scan(c);
                uint32_t rank = seen + upto - c;
                const uint32_t rank0 = rank;
                double w = 0.0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t key = key_of(x[j]);
                    bool kept = key > tau;
                    if (key == tau && c) kept = rank++ < ties;
                    if (kept) {
                        const double wj = mass_of(x[j], m, s.c);
                        if (!s.m_on || wj >= s.min_p || key == best) w += wj;
                    }
                }
                w = sum16(w);
                const uint32_t first = (uint32_t)__shfl((int)rank0, lane & 48, 64);
                if (g >= 0 && (lane & 15) == 15) {
                    mass[g] = w;
                    top[g] = first;
                }
                seen += lane_of(upto, 63);
                return true;
            });
        }
        __syncthreads();
        // the group that the draw falls into: every thread adds up a run of groups, then the runs
        const int per = (groups + THREADS - 1) / THREADS, g0 = min(groups, (int)threadIdx.x * per), g1 = min(groups, g0 + per);
        double own = 0.0;
        for (int g = g0; g < g1; ++g) own += mass[g];
        const double sum = scan(own);
        if (lane == 63) S.wave_f64[wave] = sum;
        __syncthreads();
        double cum = sum - own, everything = 0.0;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            cum += i < wave ? S.wave_f64[i] : 0.0;
            everything += S.wave_f64[i];
        }
        target = u * everything;
        int mine = 0x7FFFFFFF, last = -1;
        double base = 0.0;
        for (int g = g0; g < g1; ++g) {
            if (mass[g] > 0.0) last = g;
            if (mine == 0x7FFFFFFF && mass[g] > 0.0 && cum + mass[g] > target) {
                mine = g;
                base = cum;
            }
            cum += mass[g];
        }
        if (mine != 0x7FFFFFFF) atomicMin(&S.pick, mine);
        if (threadIdx.x == 0) S.bin = -1;
        __syncthreads();
        found = S.pick;
        if (found == mine && mine != 0x7FFFFFFF) S.base = base;
        if (found == 0x7FFFFFFF && last >= 0) atomicMax(&S.bin, last);
        __syncthreads();
        if (found == 0x7FFFFFFF) {               // rounding, or u >= 1: the last action that is kept
            found = max(S.bin, 0);
            target = INFINITY;
        }
    }
    if (wave) return;
    // inside the group: two actions a lane, in order
    float x2[2];
    uint32_t key[2], c = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int at = found * GROUP + lane * 2 + j;
        x2[j] = at < A.v && (!A.allowed || A.allowed[ao + at]) ? load_one<XD>(A.x, xo + at) : -INFINITY;
        key[j] = key_of(x2[j]);
        c += key[j] == tau && tau > KEY_NONE;
    }
    uint32_t rank = scan(c) - c;
    if (!s.greedy && filtered) rank += top[found];
    bool kept[2];
    double w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        kept[j] = key[j] > tau;
        if (key[j] == tau && tau > KEY_NONE) kept[j] = rank++ < ties;
        w[j] = kept[j] ? (s.greedy ? 1.0 : mass_of(x2[j], m, s.c)) : 0.0;
        if (!s.greedy && s.m_on && kept[j] && !(w[j] >= s.min_p || key[j] == best)) {
            kept[j] = false;
            w[j] = 0.0;
        }
    }
    const double upto = S.base + scan(w[0] + w[1]);
    const uint64_t any = __ballot(kept[0] || kept[1]), hit = __ballot(upto > target) & any;
    const int at = hit ? __ffsll((unsigned long long)hit) - 1 : 63 - __clzll((long long)any);
    if (lane == at) {
        // of this lane's two: the first if it is kept and reaches the target, or if the second is not kept
        const bool first = kept[0] && (!kept[1] || (hit && upto - w[1] > target));
        A.action[row] = found * GROUP + lane * 2 + (first ? 0 : 1);
    }
}

template <int XD> int launch(const SampleArgs &A, void *workspace, hipStream_t s) {
    const unsigned rows = (unsigned)A.n;
    // top-p, 4096 x 500 f32: a wave a row 26.6 us, a workgroup 32.6.  4096 x 2000 f32: four waves a row 34.1 us, eight 72.6.  4096 x 4096 bf16: in one
    // launch 75 us, in two 100.  8192 f32: 256 rows 13.3 and 21.7 us, 2048 rows 97 and 76.
    if (A.v <= 128) hipLaunchKernelGGL((k_sample_wave<XD, 2>), dim3((rows + 3) / 4), dim3(256), 0, s, A);
    else if (A.v <= 512) hipLaunchKernelGGL((k_sample_wave<XD, 8>), dim3((rows + 3) / 4), dim3(256), 0, s, A);
    else if (A.v <= 2048) hipLaunchKernelGGL((k_sample_block<XD, 4>), dim3(rows), dim3(256), 0, s, A);
    else if (A.v <= 4096) hipLaunchKernelGGL((k_sample_block<XD, 8>), dim3(rows), dim3(512), 0, s, A);
    else if (in_block(A.n, A.v)) hipLaunchKernelGGL((k_sample_block<XD, 16>), dim3(rows), dim3(1024), 0, s, A);
    else {
        const int groups = (A.v + GROUP - 1) / GROUP;
        double *mass = (double *)workspace;
        uint32_t *top = (uint32_t *)(mass + A.n * groups);
        for (int64_t r = 0; r < A.n; r += 65535) {   // rows of one pair of launches
            SampleArgs B = A;
            B.n = std::min<int64_t>(65535, A.n - r);
            B.x = (const char *)A.x + r * A.x_stride * elem_bytes(XD);
            if (A.allowed) B.allowed = A.allowed + r * A.allowed_stride;
            B.u = A.u + r;
            if (A.temperature_of) B.temperature_of = A.temperature_of + r;
            if (A.top_k_of) B.top_k_of = A.top_k_of + r;
            if (A.top_p_of) B.top_p_of = A.top_p_of + r;
            if (A.min_p_of) B.min_p_of = A.min_p_of + r;
            B.action = A.action + r;
            double *row_mass = mass + r * groups;
            uint32_t *row_top = top + r * groups;
            // four tiles a workgroup share its settings; not where that leaves CUs without one (131,072 bf16, no filter, four tiles / one: 4 rows
            // 12.8 / 10.8 us, 64 rows 20.0 / 20.3 us, 1024 rows 139 / 153 us)
            const bool many = B.n * ((A.v + 8191) / 8192) >= 1024;
            if (many)
                hipLaunchKernelGGL((k_sample_groups<XD, 4>), dim3((A.v + 8191) / 8192, (unsigned)B.n), dim3(256), 0, s, B, groups, row_mass, row_top);
            else
                hipLaunchKernelGGL((k_sample_groups<XD, 1>), dim3((A.v + 2047) / 2048, (unsigned)B.n), dim3(256), 0, s, B, groups, row_mass, row_top);
            MZ_LAUNCH_CHECK("k_sample_groups");
            // up to a row per CU: sixteen waves each; more rows: eight waves each, so that a CU works on two (131,072 bf16, sixteen / eight: 256 rows top-p
            // 54 / 57 us, top-k 1000 68 / 95 us; 400 rows top-p 84 / 73 us, top-k 50 44 / 36 us)
            const size_t lds = (size_t)groups * 12;
            const double *m = row_mass;
            const uint32_t *t = row_top;
            if (A.n <= 256) hipLaunchKernelGGL((k_sample_row<XD, 16, 8>), dim3((unsigned)B.n), dim3(1024), lds, s, B, groups, m, t);
            else hipLaunchKernelGGL((k_sample_row<XD, 8, 8>), dim3((unsigned)B.n), dim3(512), lds, s, B, groups, m, t);
            MZ_LAUNCH_CHECK("k_sample_row");
        }
    }
    MZ_LAUNCH_CHECK("k_sample");
    return MZ_OK;
}

constexpr int64_t MAX_N = (1 << 22) - 1;

}  // namespace

extern "C" int64_t mz_sample_actions_workspace_bytes(int64_t n, int64_t v) {
    if (n < 0 || n > MAX_N || v < 1 || v > MAX_V) return -1;
    return in_block(n, v) ? 0 : std::max<int64_t>(n, 1) * ((v + GROUP - 1) / GROUP) * 12;
}

extern "C" int mz_sample_actions(const mz_sample_args *a, void *workspace, int64_t workspace_bytes, void *stream) {
    const char *who = "mz_sample_actions";
    MZ_REQUIRE(a, "%s: null arguments", who);
    MZ_REQUIRE(a->n >= 0 && a->n <= MAX_N, "%s: n has to be 0 .. 2^22 - 1", who);
    MZ_REQUIRE(a->v >= 1 && a->v <= MAX_V, "%s: v has to be 1 .. 2^19", who);
    MZ_REQUIRE(elem_known(a->dtype), "%s: unknown dtype %d", who, a->dtype);
    MZ_REQUIRE(!a->board || a->v == 65, "%s: a bitboard needs v = 65", who);
    MZ_REQUIRE(!(a->board && a->allowed), "%s: allowed or board, not both", who);
    MZ_REQUIRE(a->temperature_of || a->temperature == 0.0 || (a->temperature >= 1e-30 && a->temperature <= 1e30),
               "%s: the temperature has to be 0, or 1e-30 .. 1e30", who);
    MZ_REQUIRE(a->top_k_of || a->top_k >= 0, "%s: top_k has to be 0 (off) or more", who);
    MZ_REQUIRE(a->top_p_of || (a->top_p >= 0.0 && a->top_p <= 1.0), "%s: top_p has to be in [0, 1]", who);
    MZ_REQUIRE(a->min_p_of || (a->min_p >= 0.0 && a->min_p <= 1.0), "%s: min_p has to be in [0, 1]", who);
    if (a->n == 0) return MZ_OK;
    MZ_REQUIRE(a->logits && a->u && a->action, "%s: null logits, u or action", who);
    MZ_REQUIRE((uintptr_t)a->logits % elem_bytes(a->dtype) == 0, "%s: misaligned logits", who);
    MZ_REQUIRE(a->logits_stride >= 0 && a->allowed_stride >= 0, "%s: negative row strides", who);
    const int64_t need = mz_sample_actions_workspace_bytes(a->n, a->v);
    MZ_REQUIRE(need == 0 || (workspace && ((uintptr_t)workspace & 7) == 0), "%s: null or misaligned workspace", who);
    MZ_REQUIRE(workspace_bytes >= need, "%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes, (long long)need);
    SampleArgs A;
    A.x = a->logits;
    A.allowed = a->allowed;
    A.board = a->board;
    A.u = a->u;
    A.temperature_of = a->temperature_of;
    A.top_k_of = a->top_k_of;
    A.top_p_of = a->top_p_of;
    A.min_p_of = a->min_p_of;
    A.action = a->action;
    A.temperature = a->temperature;
    A.c = a->temperature > 0.0 ? 1.4426950408889634 / a->temperature : 0.0;
    A.top_p = a->top_p;
    A.min_p = a->min_p;
    A.top_k = (int)std::min<int64_t>(a->top_k, a->v);
    A.x_stride = a->logits_stride;
    A.allowed_stride = a->allowed_stride;
    A.n = a->n;
    A.v = (int)a->v;
    hipStream_t s = (hipStream_t)stream;
    if (a->dtype == MZ_F32) return launch<MZ_F32>(A, workspace, s);
    if (a->dtype == MZ_BF16) return launch<MZ_BF16>(A, workspace, s);
    return launch<MZ_F16>(A, workspace, s);
}
