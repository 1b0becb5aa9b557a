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
// one draw in a thousand wrong.  Sums run in a fixed order, or over integers (w scaled to 2^s, so that atomics give the same total in any order).
//
// Short rows (up to 512 actions): one wave per row, everything in registers, thresholds bit by bit.
// Long rows, two launches: k_sample_groups reads the logits once, across all CUs, and leaves the maximum of every 128 actions and, where the
// row's settings need the total, their mass; k_sample_row, a workgroup per row, works from those: it finds a lower bound of what can be
// kept, reads again only the groups that reach it, and finds the thresholds by histograms over the logits' bits, 1024 bins at a time.
#include <math.h>
#include <algorithm>
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
    double temperature, top_p, min_p;
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
    s.min_p = A.min_p_of ? (double)A.min_p_of[row] : A.min_p;
    const int k = A.top_k_of ? A.top_k_of[row] : A.top_k;
    s.k = k > 0 && k < A.v ? k : 0;
    s.greedy = !(T > 0.0) || s.k == 1;
    s.c = s.greedy ? 0.0 : 1.4426950408889634 / T;
    s.p_on = (A.top_p_of ? (double)A.top_p_of[row] : A.top_p) < 1.0;   // a NaN is no limit
    s.m_on = s.min_p > 0.0;
    return s;
}

// 32-bit keys in the order of the values; -0 counts as +0
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }
constexpr uint32_t KEY_NONE = 0x007FFFFFu;     // -inf: an action that cannot be played
constexpr uint32_t KEY_LOWEST = 0x00800000u;   // the lowest finite value
constexpr uint32_t KEY_INF = 0xFF800000u;      // +inf, and above it NaN: no distribution

// 2^t for t <= 0: 2^round(t) times the series of e^y at y = ln 2 (t - round(t)), |y| <= 0.3466; y^13 / 13! < 2e-16
__device__ __forceinline__ double exp2_neg(double t) {
    t = fmax(t, -1100.0);
    const double r = rint(t);
    const double y = (t - r) * 0.6931471805599453;
    double q = 1.0 / 479001600.0;
    q = fma(q, y, 1.0 / 39916800.0);
    q = fma(q, y, 1.0 / 3628800.0);
    q = fma(q, y, 1.0 / 362880.0);
    q = fma(q, y, 1.0 / 40320.0);
    q = fma(q, y, 1.0 / 5040.0);
    q = fma(q, y, 1.0 / 720.0);
    q = fma(q, y, 1.0 / 120.0);
    q = fma(q, y, 1.0 / 24.0);
    q = fma(q, y, 1.0 / 6.0);
    q = fma(q, y, 0.5);
    q = fma(q, y, 1.0);
    q = fma(q, y, 1.0);
    return ldexp(q, (int)r);
}
__device__ __forceinline__ double mass_of(float x, double m, double c) { return exp2_neg(((double)x - m) * c); }

__device__ __forceinline__ double wave_scan(double v, int lane) {   // inclusive
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    return v;
}
__device__ __forceinline__ int wave_scan_int(int v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    return v;
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d, 64));
    return v;
}
__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += (uint64_t)__shfl_xor((long long)v, d, 64);
    return v;
}
__device__ __forceinline__ uint64_t lanes_below(int lane) { return lane ? ~0ull >> (64 - lane) : 0ull; }

// ---- short rows: one wave each, action j = 64 k + lane --------------------------------------------------------------------------------
template <int XD, int E> __global__ void __launch_bounds__(256) k_sample_wave(SampleArgs A) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= A.n) return;
    const Setting s = setting_of(A, row);
    const int64_t xo = row * A.x_stride, ao = row * A.allowed_stride;
    const uint64_t board = A.board ? A.board[row] : 0;
    float x[E];
    uint32_t key[E];
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const int j = k * 64 + lane;
        bool ok = j < A.v;
        if (ok && A.allowed) ok = A.allowed[ao + j] != 0;
        if (ok && A.board) ok = j < 64 ? (board >> j) & 1 : board == 0;
        x[k] = ok ? load_one<XD>(A.x, xo + j) : -INFINITY;
        key[k] = x[k] != x[k] ? 0xFFFFFFFFu : key_of(x[k]);
        top = max(top, key[k]);
    }
    top = wave_max_u32(top);
    if (top <= KEY_NONE || top >= KEY_INF || s.bad) {
        if (lane == 0) A.action[row] = -1;
        return;
    }
    // the kept set: keys above tau, and the first `ties` on it
    uint32_t tau = KEY_NONE;
    int ties = 0;
    double w[E];
#pragma unroll
    for (int k = 0; k < E; ++k) w[k] = 0.0;
    if (s.greedy) {
        tau = top;
        ties = 1;
#pragma unroll
        for (int k = 0; k < E; ++k) w[k] = key[k] == top ? 1.0 : 0.0;
    } else {
        const double m = (double)value_of(top);
#pragma unroll
        for (int k = 0; k < E; ++k) w[k] = key[k] > KEY_NONE ? mass_of(x[k], m, s.c) : 0.0;
        if (s.k) {   // the largest tau that at least k keys reach, bit by bit from the top
            uint32_t t = 0;
            for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
                int c = 0;
#pragma unroll
                for (int k = 0; k < E; ++k) c += __popcll(__ballot(key[k] >= (t | bit)));
                if (c >= s.k) t |= bit;
            }
            if (t > KEY_NONE) {
                int above = 0;
#pragma unroll
                for (int k = 0; k < E; ++k) above += __popcll(__ballot(key[k] > t));
                tau = t;
                ties = s.k - above;
            }
        }
        if (s.p_on) {   // the lowest tau above which less than p of the mass lies
            const double w_tau = tau > KEY_NONE ? mass_of(value_of(tau), m, s.c) : 0.0;
            double total = 0.0;
#pragma unroll
            for (int k = 0; k < E; ++k) total += key[k] > tau ? w[k] : 0.0;
            total = wave_sum(total) + (tau > KEY_NONE ? ties * w_tau : 0.0);
            const double limit = s.top_p * total;
            uint32_t lo = tau > KEY_NONE ? tau : KEY_LOWEST, hi = top;   // the answer lies in [lo, hi]: nothing is above the largest key
            while (lo < hi) {
                const uint32_t mid = lo + (hi - lo) / 2;
                double above = 0.0;
#pragma unroll
                for (int k = 0; k < E; ++k) above += key[k] > mid ? w[k] : 0.0;
                if (wave_sum(above) < limit) hi = mid;
                else lo = mid + 1;
            }
            double above = 0.0;
            int on = 0;
#pragma unroll
            for (int k = 0; k < E; ++k) {
                above += key[k] > lo ? w[k] : 0.0;
                on += __popcll(__ballot(key[k] == lo));
            }
            above = wave_sum(above);
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
            part[k] = base + wave_scan(kept ? w[k] : 0.0, lane);
            base = __shfl(part[k], 63, 64);
        }
    }
    const double target = A.u[row] * base;
    int pick = -1, last = -1;
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const uint64_t hit = __ballot(part[k] > target) & keep[k];
        if (pick < 0 && hit) pick = k * 64 + __ffsll((unsigned long long)hit) - 1;
        if (keep[k]) last = k * 64 + 63 - __clzll((long long)keep[k]);
    }
    if (lane == 0) A.action[row] = pick < 0 ? last : pick;
}

// ---- long rows ------------------------------------------------------------------------------------------------------------------------
constexpr int GROUP = 128;          // actions whose maximum and mass are kept together: 16 lanes of 8
constexpr int MAX_V = 1 << 19;      // 4096 groups: 48 KB of LDS for a row
constexpr int BINS = 1024;

// eight actions of a row; what lies behind its end or is not legal is -inf
template <int XD> __device__ __forceinline__ void load_eight(const SampleArgs &A, int64_t xo, int64_t ao, int at, float *x) {
    if (at + 8 <= A.v) {
        const Words<XD, 8> p = load_words<XD, 8>(A.x, xo + at);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = p.get(j);
        if (A.allowed) {
            const uint64_t ok = load_flags(A.allowed, ao + at);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = (ok >> j * 8) & 0xFF ? x[j] : -INFINITY;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = at + j < A.v && (!A.allowed || A.allowed[ao + at + j]) ? load_one<XD>(A.x, xo + at + j) : -INFINITY;
    }
}

// whether a row's total mass has to come from all of its actions
__device__ __forceinline__ bool needs_mass(const Setting &s) { return !s.greedy && !s.k && (s.p_on || !s.m_on); }

// a workgroup takes 2048 actions of one row, sixteen lanes a group
template <int XD> __global__ void __launch_bounds__(256) k_sample_groups(SampleArgs A, int groups, double *mass, uint32_t *top) {
    const int64_t row = blockIdx.y;
    const int at = blockIdx.x * 2048 + threadIdx.x * 8, g = at / GROUP;
    if (g >= groups) return;
    const Setting s = setting_of(A, row);
    float x[8];
    load_eight<XD>(A, row * A.x_stride, row * A.allowed_stride, at, x);
    float m = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        m = fmaxf(m, x[j]);
        nan |= x[j] != x[j];
    }
    uint32_t key = nan ? 0xFFFFFFFFu : key_of(m);
#pragma unroll
    for (int d = 8; d; d >>= 1) key = max(key, (uint32_t)__shfl_xor((int)key, d, 16));
    if ((threadIdx.x & 15) == 0) top[row * groups + g] = key;
    if (!needs_mass(s)) return;
    double w = 0.0;
    if (key > KEY_NONE && key < KEY_INF) {
        const double md = (double)value_of(key);
#pragma unroll
        for (int j = 0; j < 8; ++j) w += mass_of(x[j], md, s.c);
    }
#pragma unroll
    for (int d = 8; d; d >>= 1) w += __shfl_xor(w, d, 16);
    if ((threadIdx.x & 15) == 0) mass[row * groups + g] = w;
}

constexpr int ROW_THREADS = 1024, ROW_WAVES = ROW_THREADS / 64;

struct RowShared {
    unsigned long long hist[BINS];
    unsigned long long wave_u64[ROW_WAVES];
    double wave_f64[ROW_WAVES];
    uint32_t wave_u32[ROW_WAVES];
    unsigned long long above;
    double base;
    int bin, group;
};

__device__ __forceinline__ uint64_t block_sum_u64(uint64_t v, RowShared &S) {
    v = wave_sum_u64(v);
    if ((threadIdx.x & 63) == 0) S.wave_u64[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t t = 0;
#pragma unroll
    for (int i = 0; i < ROW_WAVES; ++i) t += S.wave_u64[i];
    __syncthreads();
    return t;
}

// The lowest tau in [lo, hi] with (amount above tau) < limit, where `each` hands every (key, function of its amount) of the row to its argument; `above` = that
// amount.  Histograms over [lo, hi], the bin that reaches the limit becomes the next range, down to a single key.  Amounts are integers, so the order of
// the atomics does not matter.  False: all of them together stay below the limit.
template <class EACH> __device__ bool find_threshold(EACH each, uint32_t lo, uint32_t hi, uint64_t limit, RowShared &S, uint32_t *tau, uint64_t *above_out) {
    uint64_t above = 0;
    for (;;) {
        const uint32_t width = hi - lo;
        const int shift = max(0, 32 - __clz((int)width) - 10);    // width >> shift < 1024
        S.hist[threadIdx.x] = 0;
        if (threadIdx.x == 0) S.bin = -1;
        __syncthreads();
        each([&](uint32_t key, auto amount) {
            if (key >= lo && key <= hi) atomicAdd(&S.hist[(hi - key) >> shift], (unsigned long long)amount());
        });
        __syncthreads();
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const uint64_t own = S.hist[threadIdx.x];
        uint64_t sum = own;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint64_t o = (uint64_t)__shfl_up((long long)sum, d, 64);
            if (lane >= d) sum += o;
        }
        if (lane == 63) S.wave_u64[wave] = sum;
        __syncthreads();
        uint64_t before = above;
        for (int i = 0; i < wave; ++i) before += S.wave_u64[i];
        if (before + sum - own < limit && before + sum >= limit) {    // one thread at most
            S.bin = threadIdx.x;
            S.above = before + sum - own;
        }
        __syncthreads();
        const int bin = S.bin;
        above = S.above;
        __syncthreads();
        if (bin < 0) return false;
        hi -= (uint32_t)bin << shift;
        if (shift == 0) {
            *tau = hi;
            *above_out = above;
            return true;
        }
        lo = hi - lo < (1u << shift) ? lo : hi - (1u << shift) + 1;
    }
}

template <int XD> __global__ void __launch_bounds__(ROW_THREADS) k_sample_row(SampleArgs A, int groups, const double *mass_in, const uint32_t *top_in) {
    extern __shared__ double dyn[];
    __shared__ RowShared S;
    double *mass = dyn;                          // of a group: all of it, later what is kept of it
    uint32_t *top = (uint32_t *)(dyn + groups);  // its largest key, later how many actions on the threshold come before it
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Setting s = setting_of(A, row);
    const int64_t xo = row * A.x_stride, ao = row * A.allowed_stride;
    const bool massed = needs_mass(s);

    uint32_t best = 0;
    for (int g = threadIdx.x; g < groups; g += ROW_THREADS) {
        top[g] = top_in[row * groups + g];
        mass[g] = massed ? mass_in[row * groups + g] : 0.0;
        best = max(best, top[g]);
    }
    best = wave_max_u32(best);
    if (lane == 0) S.wave_u32[wave] = best;
    if (threadIdx.x == 0) S.group = 0x7FFFFFFF;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ROW_WAVES; ++i) best = max(best, S.wave_u32[i]);
    if (best <= KEY_NONE || best >= KEY_INF || s.bad) {
        if (threadIdx.x == 0) A.action[row] = -1;
        return;
    }
    const double m = (double)value_of(best);
    uint32_t tau = KEY_NONE, ties = 0;           // the kept set: keys above tau, and the first `ties` on it
    double target = -1.0;
    int found;

    if (s.greedy) {
        for (int g = threadIdx.x; g < groups; g += ROW_THREADS)
            if (top[g] == best) atomicMin(&S.group, g);
        __syncthreads();
        found = S.group;
        tau = best - 1;
        if (threadIdx.x == 0) S.base = 0.0;
        __syncthreads();
    } else {
        if (massed)
            for (int g = threadIdx.x; g < groups; g += ROW_THREADS) mass[g] = top[g] > KEY_NONE ? mass[g] * mass_of(value_of(top[g]), m, s.c) : 0.0;
        if (s.k || s.p_on || s.m_on) {
            // Nothing below `low` is kept, nor counts in what top-p shares out.  (With top-k, top-p shares out the mass of the k first, also of
            // those that min-p drops, so min-p gives no bound there.)
            uint32_t low = KEY_LOWEST;
            auto bound = [&](double x) {         // the key of a value a little below x
                const float f = (float)(x - 1e-6 * (fabs(x) + fabs(m)));
                return max(low, min(best, max(key_of(f), KEY_LOWEST + 2) - 2));
            };
            if (s.m_on && !(s.k && s.p_on)) low = bound(m + log2(fmin(s.min_p, 1.0)) / s.c);
            if (s.k && s.k <= groups) {          // k groups reach the k-th largest of their maxima, so k actions do
                uint32_t t;
                uint64_t a;
                auto each = [&](auto take) {
                    for (int g = threadIdx.x; g < groups; g += ROW_THREADS) take(top[g], [] { return 1ull; });
                };
                if (find_threshold(each, low, best, (uint64_t)s.k, S, &t, &a)) low = t;
            }
            double total = 0.0;
            if (massed) {
                __syncthreads();
                for (int g = threadIdx.x; g < groups; g += ROW_THREADS) total += mass[g];
                total = block_sum<ROW_WAVES>(total, S.wave_f64);
                // the actions below (1 - p) of the mean mass have less than (1 - p) of the total together
                low = bound(m + log2((1.0 - s.top_p) * total / A.v) / s.c);
            }
            // every wave owns a run of the row and walks over the groups of it that reach `low`, in order
            const int steps = (groups + 3) / 4, i0 = (int)((int64_t)steps * wave / ROW_WAVES), i1 = (int)((int64_t)steps * (wave + 1) / ROW_WAVES);
            const uint32_t need = low;
            auto walk = [&](auto take) {
                for (int i = i0; i < i1; ++i) {
                    const int g = i * 4 + (lane >> 4);
                    const bool q = g < groups && top[g] >= need;
                    if (!__ballot(q)) continue;
                    float x[8];
                    if (q) load_eight<XD>(A, xo, ao, i * 512 + lane * 8, x);
                    else
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[j] = -INFINITY;
                    take(g, q, x);
                }
            };
            // masses as integers: at most 2^50 each, their sum below 2^63
            const double to_int = ldexp(1.0, min(50, 62 - (32 - __clz(A.v))));
            auto int_mass = [&](float x) { return (uint64_t)(mass_of(x, m, s.c) * to_int + 0.5); };
            uint64_t above;
            if (s.k) {
                uint32_t t;
                auto each = [&](auto take) {
                    walk([&](int, bool, const float *x) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) take(key_of(x[j]), [] { return 1ull; });
                    });
                };
                if (find_threshold(each, low, best, (uint64_t)s.k, S, &t, &above)) {
                    tau = t;
                    ties = (uint32_t)(s.k - above);
                }
            }
            if (s.p_on) {
                const uint32_t lowest = tau > KEY_NONE ? tau : low;
                double limit;
                if (massed) limit = s.top_p * total * to_int;
                else {
                    uint64_t sum = 0;
                    walk([&](int, bool, const float *x) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint32_t key = key_of(x[j]);
                            if (key > tau && key >= lowest) sum += int_mass(x[j]);
                        }
                    });
                    sum = block_sum_u64(sum, S);
                    if (tau > KEY_NONE) sum += ties * int_mass(value_of(tau));
                    limit = s.top_p * (double)sum;
                }
                const uint64_t amount = max((uint64_t)1, (uint64_t)ceil(limit));
                uint32_t t;
                auto each = [&](auto take) {
                    walk([&](int, bool, const float *x) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) take(key_of(x[j]), [&] { return int_mass(x[j]); });
                    });
                };
                if (find_threshold(each, lowest, best, amount, S, &t, &above)) {
                    const uint64_t one = int_mass(value_of(t));
                    const uint32_t r = (uint32_t)min((amount - above + one - 1) / one, (uint64_t)A.v);
                    if (t > tau) {
                        tau = t;
                        ties = r;
                    } else ties = min(ties, r);
                }
            }
            // what is kept of every group, and how many actions on the threshold come before it
            int on = 0;
            walk([&](int, bool, const float *x) {
#pragma unroll
                for (int j = 0; j < 8; ++j) on += key_of(x[j]) == tau;
            });
            if (tau <= KEY_NONE) on = 0;
            on = (int)wave_sum_u64((uint64_t)on);
            __syncthreads();
            if (lane == 0) S.wave_u32[wave] = (uint32_t)on;
            for (int g = threadIdx.x; g < groups; g += ROW_THREADS) mass[g] = 0.0;
            __syncthreads();
            uint32_t seen = 0;
            for (int i = 0; i < wave; ++i) seen += S.wave_u32[i];
            walk([&](int g, bool q, const float *x) {
                int c = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) c += key_of(x[j]) == tau;
                if (tau <= KEY_NONE) c = 0;
                const int upto = wave_scan_int(c, lane);
                uint32_t rank = seen + (uint32_t)(upto - c);
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
#pragma unroll
                for (int d = 8; d; d >>= 1) w += __shfl_xor(w, d, 16);
                if (q && (lane & 15) == 0) {
                    mass[g] = w;
                    top[g] = rank0;
                }
                seen += (uint32_t)__shfl(upto, 63, 64);
            });
        }
        __syncthreads();
        // the group that the draw falls into: every thread adds up a run of groups, then the runs
        const int per = (groups + ROW_THREADS - 1) / ROW_THREADS, g0 = min(groups, (int)threadIdx.x * per), g1 = min(groups, g0 + per);
        double own = 0.0;
        for (int g = g0; g < g1; ++g) own += mass[g];
        const double sum = wave_scan(own, lane);
        if (lane == 63) S.wave_f64[wave] = sum;
        __syncthreads();
        double before = 0.0, all = 0.0;
#pragma unroll
        for (int i = 0; i < ROW_WAVES; ++i) {
            before += i < wave ? S.wave_f64[i] : 0.0;
            all += S.wave_f64[i];
        }
        before += sum - own;
        target = A.u[row] * all;
        double cum = before;
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
        if (mine != 0x7FFFFFFF) atomicMin(&S.group, mine);
        if (threadIdx.x == 0) S.bin = -1;
        __syncthreads();
        found = S.group;
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
    uint32_t key[2];
    int c = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int at = found * GROUP + lane * 2 + j;
        x2[j] = at < A.v && (!A.allowed || A.allowed[ao + at]) ? load_one<XD>(A.x, xo + at) : -INFINITY;
        key[j] = key_of(x2[j]);
        c += key[j] == tau && tau > KEY_NONE;
    }
    uint32_t rank = wave_scan_int(c, lane) - c;
    if (!s.greedy && (s.k || s.p_on || s.m_on)) rank += top[found];
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
    const double upto = S.base + wave_scan(w[0] + w[1], lane);
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
    if (A.v <= 128) hipLaunchKernelGGL((k_sample_wave<XD, 2>), dim3((rows + 3) / 4), dim3(256), 0, s, A);
    else if (A.v <= 512) hipLaunchKernelGGL((k_sample_wave<XD, 8>), dim3((rows + 3) / 4), dim3(256), 0, s, A);
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
            hipLaunchKernelGGL((k_sample_groups<XD>), dim3((A.v + 2047) / 2048, (unsigned)B.n), dim3(256), 0, s, B, groups, mass + r * groups, top + r * groups);
            MZ_LAUNCH_CHECK("k_sample_groups");
            hipLaunchKernelGGL((k_sample_row<XD>), dim3((unsigned)B.n), dim3(ROW_THREADS), (size_t)groups * 12, s, B, groups, (const double *)(mass + r * groups),
                               (const uint32_t *)(top + r * groups));
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
    return v <= 512 ? 0 : std::max<int64_t>(n, 1) * ((v + GROUP - 1) / GROUP) * 12;
}

extern "C" int mz_sample_actions(const mz_sample_args *a, void *workspace, int64_t workspace_bytes, void *stream) {
    const char *who = "mz_sample_actions";
    MZ_REQUIRE(a, "%s: null arguments", who);
    MZ_REQUIRE(a->n >= 0 && a->n <= MAX_N, "%s: n has to be 0 .. 2^22 - 1", who);
    MZ_REQUIRE(a->v >= 1 && a->v <= MAX_V, "%s: v has to be 1 .. 2^19", who);
    MZ_REQUIRE(elem_known(a->dtype), "%s: unknown dtype %d", who, a->dtype);
    MZ_REQUIRE(!a->board || a->v == 65, "%s: a bitboard needs v = 65", who);
    MZ_REQUIRE(!(a->board && a->allowed), "%s: allowed or board, not both", who);
    MZ_REQUIRE(a->temperature_of || a->temperature == 0.0 || (a->temperature >= 1e-30 && a->temperature <= 1e30), "%s: the temperature has to be 0, or 1e-30 .. 1e30", who);
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
