// tune.hip - losses over rows of logits that tune a trained model: the clipped policy loss with a KL term and the paired
// preference loss, and their gradients.
//
// Row r chose class a of C:   logp = (x_a - max) - ln(sum exp(x - max)),   d logp / d x_j = [j = a] - softmax_j.
// Rows of one sequence are consecutive (seq_ptr); a row counts if its mask is set and 0 <= a < C.  With the log-ratio
// to the policy that generated, rho = exp(logp - old), advantage A and gap = ref - logp:
//     term = -min(rho A, clip(rho, 1 - lo, 1 + hi) A) + kl_coef (exp(gap) - gap - 1)
//     d term / d logp = -(rho A where the clip does not bind) - kl_coef (exp(gap) - 1)
// and a sequence's loss is the mean (or sum) of its counted rows' terms.  A pair's loss reads the difference of two
// sequences' sums of logp - ref.  A row that does not count has gradient 0 whatever its logits hold: it is written, not
// multiplied.
//
// Bound by HBM for many classes: 2 bytes a bf16 logit in, 2 out.  The one-pass form reads a row once, keeps it in
// registers while its sum is taken, and writes its gradient; rows too long for that are read a second time right after
// the first, from cache.  The log-probability and its differences (to old, to ref) are fp64, a few operations a row:
// their error would enter every value of the gradient.  What follows from a difference is fp32 in forms that do not cancel.
// A row's exponentials are summed in fp64 (rows of more than 64 threads: eights of them), so that the sum is better than each:
// a log-probability is off by 1e-8.  Whether the clip binds is decided on the logarithm in fp64.  Sums over a sequence's
// rows are fp64, in a fixed order.
#include "common.h"
#include "prof.h"
#include "vec.h"
#include <math.h>

// 8-value pieces of its row a thread keeps (64 registers)
#define TN_KEEP(DT) ((DT) == EDGEHIP_F32 ? 8 : 16)
// Classes up to which a thread takes a row alone.  Rows that are read once and kept: 128 bytes (10^6 x 33 / 10^6 x 48 bf16,
// policy loss and gradient: four threads a row 111 / 109 us, one 65 / 72 us; 10^6 x 48 fp32: 142 us either way, preference
// loss and gradient 135, 144 us).  Only written (preference loss and gradient, 10^6 x 24 / 10^6 x 32 bf16: one 70 / 99 us, four
// 59 / 66 us): 16 classes.
#define TN_ALONE(DT, MODE) ((MODE) == 1 ? 16 : (DT) != EDGEHIP_F32 ? 64 : 32)

struct tn_rows {
    const void* logits; int64_t ld;     // values from one row to the next
    int64_t R; int C;
    const void* taken; int taken8;      // int64, or uint8
    const uint8_t* mask;
    const int64_t* seq_ptr; int S;
    // policy
    const float *old_logp, *adv, *ref;
    int adv_per_row;
    double kl_coef, lo, hi;             // 1 - lo, 1 + hi
    double ln_lo, ln_hi;                // their logarithms
    // per row
    float* logp;                        // log-probability (0 where the row does not count)
    double* logp64;                     // the same, for sums whose differences matter
    float* rowstat;                     // [R][2] max and 1 / sum
    double* term; float* kl; float* dterm; uint8_t* clipped;
    // per sequence
    const double* scale;                // factor of dterm in the gradient; NULL: weight[s], or each
    const float* weight; double each;
    double* part;                       // partial sums of the rows' terms (rows a thread takes alone: made with the terms)
    void* dlogits;                      // dense [R][C]
};

__device__ static inline bool tn_counts(const tn_rows& T, int64_t r, int64_t& a) {
    // (all requests at once, no branch between them)
    a = T.taken8 ? (int64_t)static_cast<const uint8_t*>(T.taken)[r] : static_cast<const int64_t*>(T.taken)[r];
    bool on = (a >= 0) & (a < T.C);
    if (T.mask) on &= T.mask[r] != 0;
    if (T.seq_ptr) on &= (r >= T.seq_ptr[0]) & (r < T.seq_ptr[T.S]);
    return on;
}
// the sequence of row r (r below seq_ptr[S])
__device__ static inline int tn_seq(const int64_t* __restrict__ ptr, int S, int64_t r) {
    int lo = 0, hi = S - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ptr[mid + 1] <= r) lo = mid + 1; else hi = mid;
    }
    return lo;
}

// the same in a wave of up to RPW consecutive rows, r counted: searched once, by the scalar unit, where they all lie in the
// sequence of the first
__device__ static inline int64_t tn_first(int64_t r) {
    return ((int64_t)__builtin_amdgcn_readfirstlane((int)(r >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)r);
}
template <int RPW>
__device__ static inline int tn_wave_seq(const int64_t* __restrict__ ptr, int S, int64_t r) {
    const int64_t first = tn_first(r);
    const int g = tn_seq(ptr, S, first);
    return RPW == 1 || first + RPW - 1 < ptr[g + 1] ? g : tn_seq(ptr, S, r);
}

__device__ static inline double tn_scale(const tn_rows& T, int seq) {
    return T.scale ? T.scale[seq] : T.weight ? (double)T.weight[seq] : T.each;
}

// exp(d) - 1 - d and its derivative exp(d) - 1, to a few ulp: near 0 the series (d^2 / 2 + ...; the term after the last is
// below 2^-25 of the first), which d added to is no cancellation; else each by itself, so that a large -d is not rounded into
// the derivative and an infinite one (a class that the reference forbids) leaves it -1
__device__ static inline float tn_kl(float d, float& slope) {
    if (fabsf(d) < 1.0f) {
        float s = 1.0f / 479001600.0f;
        s = s * d + 1.0f / 39916800.0f;
        s = s * d + 1.0f / 3628800.0f;
        s = s * d + 1.0f / 362880.0f;
        s = s * d + 1.0f / 40320.0f;
        s = s * d + 1.0f / 5040.0f;
        s = s * d + 1.0f / 720.0f;
        s = s * d + 1.0f / 120.0f;
        s = s * d + 1.0f / 24.0f;
        s = s * d + 1.0f / 6.0f;
        s = s * d + 0.5f;
        s *= d * d;
        slope = s + d;
        return s;
    }
    const float e = expf(d);
    slope = e - 1.0f;
    return d > 80.0f ? e : slope - d;                            // (an infinite gap is not NaN)
}

// e^x, x <= 700 or NaN (below -150: e^-150), in fp64 to 3.5e-8 (rms 6e-9, mean below 2e-10).  e^x = 2^n (1 + q):
// n = rint(x log2 e), r = x - n ln 2, ln 2 as 16 bits (n times them is exact) and the rest; q = e^r - 1 = r + r^2 P(r) in fp32,
// where its rounding is at most 2^-26; P has the smallest largest error over |r| <= ln 2 / 2, 5e-10.  A row of few classes has no many terms to average over and a
// preference's margin is the difference of sums over many such rows: rounded to fp32 and added up there, a row's
// log-probability was off by 3e-8 to 7e-8, all margins by that times the root of their rows and more.
__device__ static inline double tn_exp64(float x) {
    x = x < -150.0f ? -150.0f : x;                               // (-inf; NaN stays)
    const float t = __builtin_fmaf(x, 1.44269504f, 12582912.0f), n = t - 12582912.0f;     // n in t's last bits
    const float r1 = __builtin_fmaf(n, -0.693145751953125f, x), c = n * -1.42860682e-6f, r = r1 + c;
    float p = 0.00020303126f;
    p = __builtin_fmaf(p, r, 0.001393498f);
    p = __builtin_fmaf(p, r, 0.008332706f);
    p = __builtin_fmaf(p, r, 0.04166643f);
    p = __builtin_fmaf(p, r, 0.16666669f);
    p = __builtin_fmaf(p, r, 0.5f);
    // (c not by way of r: x - n 16 bits lies on r's grid, so that c would be rounded to the same side for all x of an n)
    const float q = r1 + __builtin_fmaf(r * r, p, c);
    return __builtin_ldexp(1.0 + (double)q, __float_as_int(t) - 0x4b400000);
}

// The policy terms of one counted row; returns d term / d logp.  The ratio is rounded to fp32 once, its product with the
// advantage is exact in the fp64 term (the terms of a sequence nearly cancel where its advantages sum to zero).  An advantage of 0
// times a ratio past fp32's range is 0, times an infinite one NaN.
__device__ static inline float tn_policy(const tn_rows& T, int64_t r, int seq, double logp, float old, float ref, double& term, float& kl, bool& cut) {
    const float A = T.adv[T.adv_per_row ? r : seq];
    const double gain = logp - (double)old;
    const float gain32 = (float)gain;
    const float rho = gain > 700.0 ? __builtin_inff() : gain < -700.0 ? 0.0f : (float)(tn_exp64(gain32) * (1.0 + (gain - (double)gain32)));
    cut = A > 0.0f ? gain > T.ln_hi : (A < 0.0f && gain < T.ln_lo);
    const double bound = A > 0.0f ? T.hi : T.lo, gained = A == 0.0f && gain < (double)__builtin_inff() ? 0.0 : (double)A * (double)rho;
    term = cut ? -(double)A * bound : -gained;
    float d = cut ? 0.0f : (float)-gained;
    kl = 0.0f;
    if (T.ref) {
        const float gap = (float)((double)ref - logp);
        float slope;
        kl = tn_kl(gap, slope);
        if (T.kl_coef != 0.0) {                                  // (only watched: an infinite or NaN kl stays out of loss and gradient)
            term += T.kl_coef * (double)kl;
            d -= (float)T.kl_coef * slope;
        }
    }
    return d;
}

// The sequence of this lane's row r (64 consecutive rows a wave), -1 where it lies in none.  Where the wave's first and last
// row lie in one sequence - most waves - the search is done once, by the scalar unit.
__device__ static inline int tn_lane_seq(const tn_rows& T, int64_t r) {
    const int64_t first = tn_first(r);
    if (first >= T.seq_ptr[0] && first < T.seq_ptr[T.S]) {
        const int g = tn_seq(T.seq_ptr, T.S, first);
        if (first + 63 < T.seq_ptr[g + 1] && first + 63 < T.R) return g;
    }
    return r < T.R && r >= T.seq_ptr[0] && r < T.seq_ptr[T.S] ? tn_seq(T.seq_ptr, T.S, r) : -1;
}

// Sums over the lanes of a wave that share a sequence (g from tn_lane_seq; lanes that do not count have zeros): of v (WHAT 0:
// nothing; 1: two values; 2: one), and how many lanes have `cut` and `counts`.  The last lane of a run writes them as partial (wave w, sequence g), at slot
// w + g: along the rows one of the two grows by one at each border, so the slots are distinct and waves + sequences of
// them are enough.
#define TN_WAVE 64
template <int WHAT>
__device__ static inline void tn_wave_part(double (&v)[WHAT == 1 ? 2 : 1], bool cut, bool counts, int g, int64_t w, double* __restrict__ part) {
    constexpr int NV = WHAT == 0 ? 0 : WHAT == 1 ? 2 : 1;
    const int lane = threadIdx.x & 63;
    const int before = __shfl_up(g, 1, 64), after = __shfl_down(g, 1, 64);
    const uint64_t starts = __ballot(lane == 0 || before != g);
    // lanes of this lane's run up to itself
    const uint64_t upto = ~0ull >> (63 - lane), run = upto & ~((1ull << (63 - __builtin_clzll(starts & upto))) - 1);
    const uint64_t cuts = __ballot(cut), all = __ballot(counts);
    if (starts == 1) {                                           // one run: any order of pairs
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] += __shfl_xor(v[i], o, 64);
        }
    } else {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const bool same = lane >= o && (run >> (lane >= o ? lane - o : 0) & 1);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const double u = __shfl_up(v[i], o, 64);
                if (same) v[i] += u;
            }
        }
    }
    if (g >= 0 && (lane == 63 || after != g)) {
        double* p = part + (w + g) * 4;
        p[0] = NV > 0 ? v[0] : 0.0;
        p[1] = NV > 1 ? v[WHAT == 1] : 0.0;
        p[2] = (double)__popcll(cuts & run);
        p[3] = (double)__popcll(all & run);
    }
}

// e^x in fp32 by the hardware's power of two, for the sums of rows of many classes and for every value of a gradient.  The fp32
// constant log2(e) alone is 1.3e-8 off: every term of a row would be off to the same side by that times |x|.  With the
// constant's second part the error of a term is that of rounding x log2(e), to either side, and the instruction's own (mean -3e-9).
__device__ static inline float tn_exp(float x) {
    constexpr float HI = 1.44269502162933349609f, LO = 1.92596298909109e-8f;
    return __builtin_amdgcn_exp2f(__builtin_fmaf(x, HI, x * LO));
}

// ln(s) to 1e-9, s > 0 (NaN: NaN).  s = 2^k f, f in [sqrt(1/2), sqrt(2)), z = (f - 1) / (f + 1):
// ln f = 2 z (1 + z^2 / 3 + z^4 / 5 + ...), the bracket's sum, below 0.01, in fp32
__device__ static inline double tn_ln(double s) {
    double f = __builtin_amdgcn_frexp_mant(s);
    int k = __builtin_amdgcn_frexp_exp(s);
    if (f < 0.70710678118654752440) { f += f; --k; }
    const double num = f - 1.0, den = f + 1.0, r = (double)__builtin_amdgcn_rcpf((float)den), z0 = num * r;
    const double z = __builtin_fma(r, __builtin_fma(-z0, den, num), z0);
    const float w = (float)z * (float)z;
    float p = 1.0f / 11.0f;
    p = __builtin_fmaf(p, w, 1.0f / 9.0f);
    p = __builtin_fmaf(p, w, 1.0f / 7.0f);
    p = __builtin_fmaf(p, w, 1.0f / 5.0f);
    p = __builtin_fmaf(p, w, 1.0f / 3.0f);
    return __builtin_fma((double)k, 0.69314718055994530942, __builtin_fma(2.0 * z, (double)(p * w), 2.0 * z));
}

// The TPR threads' running pairs (largest value, sum of exponentials below it) become the row's, in every one of them: the
// largest first, so that each sum is scaled once.
template <int TPR>
__device__ static inline void tn_row_merge(float& m, double& s, float* lds_m, double* lds_s) {
    if (TPR == 1) return;
    float top = m;
#pragma unroll
    for (int o = 1; o < (TPR < 64 ? TPR : 64); o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    if (TPR > 64) {
        if ((threadIdx.x & 63) == 0) lds_m[threadIdx.x >> 6] = top;
        __syncthreads();
        top = lds_m[0];
#pragma unroll
        for (int w = 1; w < TPR / 64; ++w) top = fmaxf(top, lds_m[w]);
    }
    s *= tn_exp64(m - top);                                      // (a row of -inf alone: NaN, as its log-probability)
    m = top;
#pragma unroll
    for (int o = 1; o < (TPR < 64 ? TPR : 64); o <<= 1) s += __shfl_xor(s, o, 64);
    if (TPR > 64) {
        if ((threadIdx.x & 63) == 0) lds_s[threadIdx.x >> 6] = s;
        __syncthreads();
        s = lds_s[0];
#pragma unroll
        for (int w = 1; w < TPR / 64; ++w) s += lds_s[w];
    }
}

// n of eight more values into the running pair.  NaN: the sum becomes NaN and stays it.  FEW: each
// exponential and the sum in fp64; else eight are added up in fp32, which many pieces average, and the pieces in fp64.
template <bool FEW>
__device__ static inline void tn_add8(float& m, double& s, const float (&v)[8], int n = 8) {
    float top = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
    top = fmaxf(top, m);
    if (top > m) { s *= FEW ? tn_exp64(m - top) : (double)tn_exp(m - top); m = top; }     // m = -inf: s is 0 (or NaN) before
    const float base = m == -__builtin_inff() ? 0.0f : m;                            // all -inf so far: exp(-inf) = 0
    if (FEW) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i >= n) break;
            s += tn_exp64(v[i] - base);
        }
    } else {
        float a = 0.0f, b = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            a += tn_exp(v[i] - base);
            b += tn_exp(v[i + 1] - base);
        }
        s += (double)(a + b);
    }
}

// MODE 0: row statistics (and the policy's per-row terms where T.old_logp is given)
// MODE 1: the gradient from row statistics;  MODE 2: both at once
// PIECES: of a row that one thread keeps (8 classes or less: 1)
// Waves a SIMD: kept rows take 64 registers beside some 34 others, and two fewer of those make five waves of four where a row is
// whole blocks (30000 x 4099 fp32, policy loss and gradient: four 236 us, five 217 us; four threads a row, 10^6 x 48 fp32: 142,
// 147 us).
#define TN_WAVES(TPR, MODE) ((MODE) == 2 && ((TPR) == 256 || (TPR) == 512) ? 5 : 1)
template <int DT, int TPR, int MODE, int PIECES = 4>
__global__ __launch_bounds__((TPR < 256 ? 256 : TPR), TN_WAVES(TPR, MODE)) void k_tn_rows(tn_rows T) {
    constexpr int RPB = (TPR < 256 ? 256 : TPR) / TPR;
    constexpr int RPW = TPR < 64 ? 64 / TPR : 1;
    __shared__ float lds_m[TPR < 64 ? 1 : TPR / 64];
    __shared__ double lds_s[TPR < 64 ? 1 : TPR / 64];
    const int t = threadIdx.x % TPR;
    const int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
    if (TPR > 1 && TPR <= 64 && r >= T.R) return;                // (TPR > 64: one row per block, none too many)
    const int C = T.C;
    const int64_t base = r * T.ld;
    int64_t a = -1;
    float old = 0.0f, ref = 0.0f;
    if (MODE != 1 && T.old_logp && r < T.R) {
        old = T.old_logp[r];
        if (T.ref) ref = T.ref[r];
    }
    const bool counts = r < T.R && tn_counts(T, r, a);
    constexpr int KEEP = MODE == 1 ? 1 : TPR == 1 ? PIECES : MODE == 2 ? TN_KEEP(DT) : 1;
    eh_raw8<DT> keep[KEEP];
    float m = -__builtin_inff(), inv = 0.0f;
    double s = 0.0;
    float coef = 0.0f;
    // Pieces of eight values, all whole: the last one of a row ends with it and begins inside the one before, those values are
    // left out of the sum and their gradient is written twice, to the same bits.  (8 classes or less: one piece, value by value.)
    constexpr bool WHOLE = TPR > 1 || PIECES > 1;
    const typename eh_elem<DT>::type* const row = reinterpret_cast<const typename eh_elem<DT>::type*>(T.logits) + base;
    auto start = [&](int c) { return WHOLE && c > C - 8 ? C - 8 : c; };
    auto add = [&](float (&v)[8], int c) {
        if (WHOLE && c > C - 8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < c - (C - 8) ? -__builtin_inff() : v[i];
        }
        tn_add8<(TPR <= 64)>(m, s, v);
    };
    float only[8];                                                // 8 classes or less: the row
    if (!WHOLE && r < T.R) eh_load8<DT>(row, 0, C, only, -__builtin_inff());
    const bool kept = MODE != 1 && WHOLE && C <= TPR * 8 * KEEP;
    if (MODE != 1) {
        if (counts) {
            if (kept) {
#pragma unroll
                for (int k = 0; k < KEEP; ++k) {
                    if (k * TPR * 8 >= C) break;
                    keep[k].load(row + start((k * TPR + t) * 8));
                }
#pragma unroll
                for (int k = 0; k < KEEP; ++k) {
                    if (k * TPR * 8 >= C) break;
                    const int c = (k * TPR + t) * 8;
                    float v[8];
                    keep[k].get(v);
                    if (c < C) add(v, c);
                }
            } else if (WHOLE) {
                for (int c = t * 8; c < C; c += TPR * 8) {
                    float v[8];
                    eh_load8<DT>(row, start(c), 8, v);
                    add(v, c);
                }
            } else {
                tn_add8<true>(m, s, only, C);
            }
            tn_row_merge<TPR>(m, s, lds_m, lds_s);                         // (a row counts for all of its threads or none)
        }
        double logp = 0.0;
        double term = 0.0;
        float d = 0.0f, kl = 0.0f;
        bool cut = false;
        int seq = -1;
        if (TPR == 1 && T.old_logp) seq = tn_lane_seq(T, r);
        if (counts) {
            const float xa = (float)row[a];
            logp = (double)xa - (double)m - tn_ln(s);
            const float s32 = (float)s;
            inv = 1.0f / s32;
            inv = __builtin_fmaf(-inv * inv, (float)(s - (double)s32), inv);
            if (T.old_logp) {
                if (TPR > 1) seq = tn_wave_seq<RPW>(T.seq_ptr, T.S, r);
                d = tn_policy(T, r, seq, logp, old, ref, term, kl, cut);
                if (MODE == 2) coef = (float)((double)d * tn_scale(T, seq));
            }
        }
        if (t == 0 && r < T.R) {
            if (T.logp) T.logp[r] = (float)logp;
            if (T.logp64) T.logp64[r] = logp;
            if (T.rowstat) { T.rowstat[2 * r] = m; T.rowstat[2 * r + 1] = inv; }
            if (T.dterm) T.dterm[r] = d;
            if (T.term && TPR > 1) {
                T.term[r] = term;
                T.kl[r] = kl;
                T.clipped[r] = cut;
            }
        }
        if (TPR == 1 && T.old_logp) {
            double v[2] = {term, (double)kl};
            tn_wave_part<1>(v, cut, counts, seq, r / TN_WAVE, T.part);
        }
        if (TPR == 1 && r >= T.R) return;
    } else if (counts) {
        m = T.rowstat[2 * r];
        inv = T.rowstat[2 * r + 1];
        const int seq = tn_wave_seq<RPW>(T.seq_ptr, T.S, r);
        coef = (float)(T.dterm ? (double)T.dterm[r] * tn_scale(T, seq) : tn_scale(T, seq));
    }
    if (MODE != 0 && (TPR > 1 || r < T.R)) {
        const float f = -coef * inv;
#pragma unroll
        for (int k = 0; k < KEEP; ++k) {
            if (k * TPR * 8 >= C) break;
            for (int from = (k * TPR + t) * 8; from < C; from += TPR * 8) {
                const int c = start(from);
                float v[8];
                if (!counts) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
                } else {
                    if (kept) keep[k].get(v);
                    else if (WHOLE) eh_load8<DT>(row, c, 8, v);
                    else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = only[i];
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = f * tn_exp(v[i] - m);
                    if (a >= c && a < c + 8) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) if (a == c + i) v[i] += coef;
                    }
                }
                eh_store8<DT>(T.dlogits, r * C + c, WHOLE ? 8 : C, v);
                if (kept) break;
            }
            if (!kept) break;
        }
    }
}

// ---- sums over the rows of a sequence (tn_wave_part), a lane a row ----------------------------------------------------
// WHAT 0: counted rows; 1: policy (term, kl, clipped, count); 2: preference (logp - ref, count)
template <int WHAT>
__global__ __launch_bounds__(256) void k_tn_part(tn_rows T) {
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    double v[WHAT == 1 ? 2 : 1] = {0.0};
    bool cut = false, counts = false;
    if (r < T.R) {                                                // requested before the search
        int64_t cls;
        counts = tn_counts(T, r, cls);
        if (WHAT == 1) { v[0] = T.term[r]; v[WHAT == 1] = T.kl[r]; cut = T.clipped[r]; }
        if (WHAT == 2) v[0] = T.logp64[r] - (T.ref ? (double)T.ref[r] : 0.0);
    }
    const int g = tn_lane_seq(T, r);
    if (!counts) {
        v[0] = v[WHAT == 1] = 0.0;
        cut = false;
    }
    tn_wave_part<WHAT>(v, cut, counts, g, r / TN_WAVE, T.part);
}

struct tn_final {
    const int64_t* seq_ptr; int64_t R; int S; const double* part;
    int mean; const float* weight; double each;       // weight of a sequence's (pair's) loss in the gradient: weight[s], or each
    float *loss, *kl; int32_t* clipped;
    double* scale;                                    // d (weighted loss) / d (dterm or logp) of the sequence's rows
    // preference
    int kind; double beta, smooth; float* margin;
};
// Few rows: a sequence's block of 1024 threads adds them up itself (16 rows a thread at most), a launch less, two where the
// count comes first.  More rows, which may all lie in one sequence, or more sequences than blocks that run at once go through
// tn_sum's partials.  150 x 1000 fp32, preference loss and gradient: 24 us, 21 us; 8192 x 32003 bf16, policy: 242, 238 us.
static bool tn_direct(const tn_rows& T) { return T.R <= 16384 && T.S <= 512; }
// totals of sequence g in every thread of the block, from the partials or from the rows (WHAT as in k_tn_part)
template <int WHAT, bool DIRECT>
__device__ static inline void tn_total(const tn_final& F, const tn_rows& T, int g, double (&v)[4], double (&red)[16][4]) {
    int64_t a = F.seq_ptr[g], b = F.seq_ptr[g + 1];
    if (a < 0) a = 0;
    if (b > F.R) b = F.R;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = 0.0;
    if (DIRECT) {
#pragma unroll 4
        for (int64_t r = a + threadIdx.x; r < b; r += 1024) {
            double x = 0.0, y = 0.0;
            bool cut = false;
            if (WHAT == 1) { x = T.term[r]; y = T.kl[r]; cut = T.clipped[r]; }
            if (WHAT == 2) x = T.logp64[r] - (T.ref ? (double)T.ref[r] : 0.0);
            int64_t cls;
            const bool counts = tn_counts(T, r, cls);
            if (WHAT) v[0] += counts ? x : 0.0;
            if (WHAT == 1) { v[1] += counts ? y : 0.0; v[2] += counts && cut ? 1.0 : 0.0; }
            v[3] += counts ? 1.0 : 0.0;
        }
    } else if (a < b) {
        for (int64_t c = a / TN_WAVE + threadIdx.x; c <= (b - 1) / TN_WAVE; c += 256) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += F.part[(c + g) * 4 + i];
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += __shfl_xor(v[i], o, 64);
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) red[threadIdx.x >> 6][i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (red[0][i] + red[1][i]) + (red[2][i] + red[3][i]);
    if (DIRECT) {
#pragma unroll 1
        for (int w = 4; w < 16; w += 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += (red[w][i] + red[w + 1][i]) + (red[w + 2][i] + red[w + 3][i]);
        }
    }
}
// a block a sequence.  PASS 0: the gradient's scale from the counted rows; 1: the losses
template <int PASS, bool DIRECT>
__global__ __launch_bounds__(DIRECT ? 1024 : 256) void k_tn_policy_final(tn_final F, tn_rows T) {
    __shared__ double red[16][4];
    const int g = blockIdx.x;
    double v[4];
    tn_total<PASS, DIRECT>(F, T, g, v, red);
    if (threadIdx.x) return;
    const double inv = F.mean ? 1.0 / (v[3] > 0.0 ? v[3] : 1.0) : 1.0;
    if (F.scale) F.scale[g] = (F.weight ? (double)F.weight[g] : F.each) * inv;
    if (PASS == 1) {
        F.loss[g] = (float)(v[0] * inv);
        F.kl[g] = (float)(v[1] * inv);
        F.clipped[g] = (int32_t)v[2];
    }
}
// a block a pair: chosen sequence g, rejected sequence g + pairs
template <bool DIRECT>
__global__ __launch_bounds__(DIRECT ? 1024 : 256) void k_tn_pref_final(tn_final F, tn_rows T) {
    __shared__ double red[16][4];
    const int g = blockIdx.x, P = F.S / 2;
    double c[4], r[4];
    tn_total<2, DIRECT>(F, T, g, c, red);
    tn_total<2, DIRECT>(F, T, g + P, r, red);
    if (threadIdx.x) return;
    const double ic = F.mean ? 1.0 / (c[3] > 0.0 ? c[3] : 1.0) : 1.0, ir = F.mean ? 1.0 / (r[3] > 0.0 ? r[3] : 1.0) : 1.0;
    const double margin = c[0] * ic - r[0] * ir;
    double loss, d;
    if (F.kind == EDGEHIP_PREFER_SIGMOID) {
        const double x = F.beta * margin, w = exp(-fabs(x));
        // -ln sigmoid(x), smoothed: ln(1 + e^-|x|) and (1 - smooth) |x| below 0, smooth |x| above (no smooth, no term: a margin may
        // be infinite, where a class that may not be taken was)
        loss = log1p(w) + (x < 0.0 ? (F.smooth - 1.0) * x : F.smooth > 0.0 ? F.smooth * x : 0.0);
        d = F.beta * (F.smooth - (x >= 0.0 ? w : 1.0) / (1.0 + w));               // smooth - sigmoid(-x)
    } else {
        const double off = margin - 0.5 / F.beta;
        loss = off * off;
        d = 2.0 * off;
    }
    if (F.loss) F.loss[g] = (float)loss;
    if (F.margin) F.margin[g] = (float)margin;
    if (F.scale) {
        d *= F.weight ? (double)F.weight[g] : F.each;
        F.scale[g] = d * ic;
        F.scale[g + P] = -d * ir;
    }
}

// ---- entry points -------------------------------------------------------------------------------------------------
template <int DT, int MODE>
static void tn_go(const tn_rows& T, int tpr, dim3 grid, dim3 block, hipStream_t s) {
#define TN_RUN(...) EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_tn_rows<__VA_ARGS__>), grid, block, 0, s, T))
    if (T.C <= 8) { TN_RUN(DT, 1, MODE, 1); return; }
    if constexpr (TN_ALONE(DT, MODE) > 32) {
        if (tpr == 1 && T.C > 32) { TN_RUN(DT, 1, MODE, 8); return; }
    }
    switch (tpr) {
        case 1: TN_RUN(DT, 1, MODE); break;
        case 4: TN_RUN(DT, 4, MODE); break;
        case 8: TN_RUN(DT, 8, MODE); break;
        case 16: TN_RUN(DT, 16, MODE); break;
        case 32: TN_RUN(DT, 32, MODE); break;
        case 64: TN_RUN(DT, 64, MODE); break;
        case 256: TN_RUN(DT, 256, MODE); break;
        case 512: TN_RUN(DT, 512, MODE); break;
        default: TN_RUN(DT, 1024, MODE);
    }
#undef TN_RUN
}
template <int MODE> static int tn_alone(int dtype) { return dtype == EDGEHIP_F32 ? TN_ALONE(EDGEHIP_F32, MODE) : TN_ALONE(EDGEHIP_BF16, MODE); }
template <int MODE>
static int tn_threads(int dtype, int C) {
    // Threads of a row: one for few classes (10^6 x 9 bf16, policy loss and gradient: eight threads a row 143 us, one
    // 40 us), else as few as can keep it whole: what is done once per row is done by all of them, and a CU has rows in
    // different phases (8192 x 32003 bf16: 1024 threads a row 369 us, 256 238 us).
    const int per = 8 * (dtype == EDGEHIP_F32 ? TN_KEEP(EDGEHIP_F32) : TN_KEEP(EDGEHIP_BF16));
    if (C <= tn_alone<MODE>(dtype)) return 1;
    // (only written: wider runs pay more where a row has more than 128 bytes; preference over 10^6 x 48 fp32: four threads
    // 156 us, eight 135 us; over 10^6 x 33 bf16: 77 us, 87 us)
    int tpr = MODE == 1 && C > (dtype == EDGEHIP_F32 ? 32 : 64) ? 8 : 4;
    while (tpr < 64 && C > tpr * per) tpr *= 2;
    if (C > 64 * per) tpr = 256;
    while (tpr < 1024 && C > tpr * per) tpr *= 2;
    return tpr;
}
template <int MODE>
static int64_t tn_row_blocks(int dtype, int64_t R, int C) {
    const int tpr = tn_threads<MODE>(dtype, C), rpb = (tpr < 256 ? 256 : tpr) / tpr;
    return (R + rpb - 1) / rpb;
}
// whether a launch takes all rows: up to 2^31 - 1 of few classes, fewer with several threads a row
template <int MODE>
static int tn_fits(const edgehip_logit_rows* Q) {
    const int tpr = tn_threads<MODE>(Q->dtype, Q->classes);
    return eh_grid_ok(tn_row_blocks<MODE>(Q->dtype, Q->rows, Q->classes), tpr < 256 ? 256 : tpr) ? EDGEHIP_OK : EDGEHIP_ERR_TOO_LARGE;
}
template <int MODE>
static int tn_launch(int dtype, const tn_rows& T, hipStream_t s) {
    if (T.R == 0) return EDGEHIP_OK;
    const int tpr = tn_threads<MODE>(dtype, T.C);
    const dim3 grid((unsigned)tn_row_blocks<MODE>(dtype, T.R, T.C)), block(tpr < 256 ? 256 : tpr);
    if (dtype == EDGEHIP_F32) tn_go<EDGEHIP_F32, MODE>(T, tpr, grid, block, s);
    else if (dtype == EDGEHIP_BF16) tn_go<EDGEHIP_BF16, MODE>(T, tpr, grid, block, s);
    else tn_go<EDGEHIP_F16, MODE>(T, tpr, grid, block, s);
    EH_LAUNCH_CHECK();
    return EDGEHIP_OK;
}

#define TN_TRY(x) do { const int rc_ = (x); if (rc_ != EDGEHIP_OK) return rc_; } while (0)
static int tn_check(const edgehip_logit_rows* Q, bool seqs = true) {
    EH_CHECK_ARG(Q && eh_dtype_ok(Q->dtype) && Q->rows >= 0 && Q->classes >= 1);
    EH_CHECK_ARG(seqs ? Q->seq_ptr && Q->num_seqs >= 1 : (Q->seq_ptr != nullptr) == (Q->num_seqs >= 1) && Q->num_seqs >= 0);
    EH_CHECK_ARG(Q->taken_type == EDGEHIP_TAKEN_I64 || Q->taken_type == EDGEHIP_TAKEN_U8);
    EH_CHECK_ARG(Q->rows == 0 || (Q->logits && Q->taken && Q->row_stride >= Q->classes));
    // (sequences: a block each)
    if (Q->rows > (((int64_t)1 << 31) - 1) || !eh_grid_ok(Q->num_seqs, 256) || Q->classes > (1 << 30)) return EDGEHIP_ERR_TOO_LARGE;
    return EDGEHIP_OK;
}
static tn_rows tn_fill(const edgehip_logit_rows* Q) {
    tn_rows T = {};
    T.logits = Q->logits; T.ld = Q->row_stride; T.R = Q->rows; T.C = Q->classes;
    T.taken = Q->taken; T.taken8 = Q->taken_type == EDGEHIP_TAKEN_U8; T.mask = Q->mask; T.seq_ptr = Q->seq_ptr; T.S = Q->num_seqs;
    return T;
}
// workspace: [S] fp64 scales, [chunks + S][4] fp64 partials, per row fp64 term, log-probability, fp32 kl, dterm, stat and a byte
struct tn_ws { double *scale, *part, *term, *logp; float *kl, *dterm, *stat; uint8_t* clipped; size_t bytes; };
static tn_ws tn_layout(const edgehip_logit_rows* Q, void* ws) {
    tn_ws W;
    const size_t R = (size_t)Q->rows, S = (size_t)Q->num_seqs, chunks = (R + TN_WAVE - 1) / TN_WAVE;
    char* p = reinterpret_cast<char*>(ws);
    size_t o = 0;
    auto take = [&](size_t n) { char* q = p + o; o += (n + 15) & ~(size_t)15; return q; };
    W.scale = (double*)take(S * 8);
    W.part = (double*)take((chunks + S) * 32);
    W.term = (double*)take(R * 8);
    W.kl = (float*)take(R * 4);
    W.dterm = (float*)take(R * 4);
    W.logp = (double*)take(R * 8);
    W.stat = (float*)take(R * 8);
    W.clipped = (uint8_t*)take(R);
    W.bytes = o;
    return W;
}
extern "C" size_t edgehip_tune_workspace_bytes(const edgehip_logit_rows* Q) {
    return tn_check(Q) == EDGEHIP_OK ? tn_layout(Q, nullptr).bytes : 0;
}

template <int WHAT>
static int tn_sum(const tn_rows& T, hipStream_t s) {
    if (T.R == 0) return EDGEHIP_OK;
    EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_tn_part<WHAT>), dim3((unsigned)((T.R + 255) / 256)), dim3(256), 0, s, T));
    EH_LAUNCH_CHECK();
    return EDGEHIP_OK;
}


extern "C" int edgehip_row_logp(const edgehip_logit_rows* Q, float* logp, void* stream) {
    TN_TRY(tn_check(Q, false));
    EH_CHECK_ARG(Q->rows == 0 || logp);
    TN_TRY(tn_fits<0>(Q));
    tn_rows T = tn_fill(Q);
    T.logp = logp;
    return tn_launch<0>(Q->dtype, T, eh_stream(stream));
}

static int tn_policy_args(const edgehip_logit_rows* Q, const edgehip_policy* O, tn_rows& T, tn_final& F, tn_ws& W, void* ws, size_t ws_bytes) {
    TN_TRY(tn_check(Q));
    EH_CHECK_ARG(O && (Q->rows == 0 || (O->old_logp && O->advantage)) && O->clip_lo >= 0.0 && O->clip_hi >= 0.0);
    EH_CHECK_ARG(O->kl_coef == 0.0 || O->ref_logp || Q->rows == 0);
    if (ws_bytes < edgehip_tune_workspace_bytes(Q)) return EDGEHIP_ERR_WORKSPACE;
    EH_CHECK_ARG(ws && ((uintptr_t)ws & 15) == 0);
    W = tn_layout(Q, ws);
    T = tn_fill(Q);
    T.old_logp = O->old_logp; T.adv = O->advantage; T.ref = O->ref_logp; T.adv_per_row = O->advantage_per_row;
    T.kl_coef = O->kl_coef; T.lo = 1.0 - O->clip_lo; T.hi = 1.0 + O->clip_hi;
    T.ln_lo = O->clip_lo < 1.0 ? log1p(-O->clip_lo) : -HUGE_VAL; T.ln_hi = log1p(O->clip_hi);
    T.term = W.term; T.kl = W.kl; T.clipped = W.clipped; T.part = W.part;
    T.weight = O->weight; T.each = 1.0 / (double)Q->num_seqs;
    F = tn_final{};
    F.seq_ptr = Q->seq_ptr; F.R = Q->rows; F.S = Q->num_seqs; F.part = W.part;
    F.mean = O->mean; F.weight = O->weight; F.each = 1.0 / (double)Q->num_seqs;
    return EDGEHIP_OK;
}

// rows: the sequences' totals are taken from the rows, not from partials
template <int PASS>
static int tn_policy_final(const tn_final& F, const tn_rows& T, bool rows, hipStream_t s) {
    if (rows) EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_tn_policy_final<PASS, true>), dim3(F.S), dim3(1024), 0, s, F, T));
    else EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_tn_policy_final<PASS, false>), dim3(F.S), dim3(256), 0, s, F, T));
    EH_LAUNCH_CHECK();
    return EDGEHIP_OK;
}
// the losses, after the rows' terms
template <int MODE>
static int tn_policy_sums(int dtype, const tn_final& F, const tn_rows& T, hipStream_t s) {
    const bool made = T.C <= tn_alone<MODE>(dtype);              // (the row kernel has made the partials)
    if (!made && !tn_direct(T)) TN_TRY(tn_sum<1>(T, s));
    return tn_policy_final<1>(F, T, !made && tn_direct(T), s);
}

extern "C" int edgehip_policy_loss_fwd(const edgehip_logit_rows* Q, const edgehip_policy* O, float* loss, float* kl, int32_t* clipped,
                                       float* logp, void* ws, size_t ws_bytes, void* stream) {
    tn_rows T; tn_final F; tn_ws W;
    TN_TRY(tn_policy_args(Q, O, T, F, W, ws, ws_bytes));
    EH_CHECK_ARG(loss && kl && clipped);
    TN_TRY(tn_fits<0>(Q));
    hipStream_t s = eh_stream(stream);
    T.logp = logp; T.rowstat = W.stat; T.dterm = W.dterm;
    TN_TRY(tn_launch<0>(Q->dtype, T, s));
    F.loss = loss; F.kl = kl; F.clipped = clipped;
    return tn_policy_sums<0>(Q->dtype, F, T, s);
}
extern "C" int edgehip_policy_loss_bwd(const edgehip_logit_rows* Q, const edgehip_policy* O, void* dlogits, void* ws, size_t ws_bytes,
                                       void* stream) {
    tn_rows T; tn_final F; tn_ws W;
    TN_TRY(tn_policy_args(Q, O, T, F, W, ws, ws_bytes));
    EH_CHECK_ARG(Q->rows == 0 || dlogits);
    TN_TRY(tn_fits<1>(Q));
    hipStream_t s = eh_stream(stream);
    if (F.mean) {                               // the partial sums of the forward, if it made some, are still in the workspace
        F.scale = W.scale;
        T.scale = W.scale;
        TN_TRY(tn_policy_final<0>(F, T, tn_direct(T), s));
    }
    T.rowstat = W.stat; T.dterm = W.dterm; T.dlogits = dlogits;
    return tn_launch<1>(Q->dtype, T, s);
}
extern "C" int edgehip_policy_loss_grad(const edgehip_logit_rows* Q, const edgehip_policy* O, float* loss, float* kl, int32_t* clipped,
                                        float* logp, void* dlogits, void* ws, size_t ws_bytes, void* stream) {
    tn_rows T; tn_final F; tn_ws W;
    TN_TRY(tn_policy_args(Q, O, T, F, W, ws, ws_bytes));
    EH_CHECK_ARG(loss && kl && clipped && (Q->rows == 0 || dlogits));
    TN_TRY(tn_fits<2>(Q));
    hipStream_t s = eh_stream(stream);
    if (F.mean) {                               // a mean needs the number of counted rows before the gradient
        if (!tn_direct(T)) TN_TRY(tn_sum<0>(T, s));
        F.scale = W.scale;
        TN_TRY(tn_policy_final<0>(F, T, tn_direct(T), s));
        T.scale = W.scale;
    }
    T.logp = logp; T.dlogits = dlogits;
    TN_TRY(tn_launch<2>(Q->dtype, T, s));
    F.scale = nullptr; F.loss = loss; F.kl = kl; F.clipped = clipped;
    return tn_policy_sums<2>(Q->dtype, F, T, s);
}

static int tn_pref_args(const edgehip_logit_rows* Q, const edgehip_preference* O, tn_rows& T, tn_final& F, tn_ws& W, void* ws, size_t ws_bytes) {
    TN_TRY(tn_check(Q));
    EH_CHECK_ARG(O && Q->num_seqs % 2 == 0 && (O->kind == EDGEHIP_PREFER_SIGMOID || O->kind == EDGEHIP_PREFER_SQUARE) && O->beta > 0.0);
    EH_CHECK_ARG(O->label_smoothing >= 0.0 && O->label_smoothing < 0.5 && (O->kind == EDGEHIP_PREFER_SIGMOID || O->label_smoothing == 0.0));
    if (ws_bytes < edgehip_tune_workspace_bytes(Q)) return EDGEHIP_ERR_WORKSPACE;
    EH_CHECK_ARG(ws && ((uintptr_t)ws & 15) == 0);
    W = tn_layout(Q, ws);
    T = tn_fill(Q);
    T.ref = O->ref_logp; T.part = W.part;
    F = tn_final{};
    F.seq_ptr = Q->seq_ptr; F.R = Q->rows; F.S = Q->num_seqs; F.part = W.part;
    F.mean = O->mean; F.weight = O->weight; F.each = 2.0 / (double)Q->num_seqs;
    F.kind = O->kind; F.beta = O->beta; F.smooth = O->label_smoothing;
    return EDGEHIP_OK;
}
static int tn_pref_final(const tn_final& F, const tn_rows& T, hipStream_t s) {
    if (tn_direct(T)) EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_tn_pref_final<true>), dim3(F.S / 2), dim3(1024), 0, s, F, T));
    else EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_tn_pref_final<false>), dim3(F.S / 2), dim3(256), 0, s, F, T));
    EH_LAUNCH_CHECK();
    return EDGEHIP_OK;
}
static int tn_pref_fwd(const edgehip_logit_rows* Q, tn_rows& T, tn_final& F, tn_ws& W, float* loss, float* margin, hipStream_t s) {
    EH_CHECK_ARG(loss && margin);
    TN_TRY(tn_fits<0>(Q));
    T.logp64 = W.logp; T.rowstat = W.stat;
    TN_TRY(tn_launch<0>(Q->dtype, T, s));
    if (!tn_direct(T)) TN_TRY(tn_sum<2>(T, s));
    F.loss = loss; F.margin = margin;
    TN_TRY(tn_pref_final(F, T, s));
    return EDGEHIP_OK;
}
extern "C" int edgehip_preference_loss_fwd(const edgehip_logit_rows* Q, const edgehip_preference* O, float* loss, float* margin,
                                           void* ws, size_t ws_bytes, void* stream) {
    tn_rows T; tn_final F; tn_ws W;
    TN_TRY(tn_pref_args(Q, O, T, F, W, ws, ws_bytes));
    return tn_pref_fwd(Q, T, F, W, loss, margin, eh_stream(stream));
}
extern "C" int edgehip_preference_loss_grad(const edgehip_logit_rows* Q, const edgehip_preference* O, float* loss, float* margin,
                                            void* dlogits, void* ws, size_t ws_bytes, void* stream) {
    tn_rows T; tn_final F; tn_ws W;
    TN_TRY(tn_pref_args(Q, O, T, F, W, ws, ws_bytes));
    EH_CHECK_ARG(Q->rows == 0 || dlogits);
    TN_TRY(tn_fits<1>(Q));
    F.scale = W.scale;
    TN_TRY(tn_pref_fwd(Q, T, F, W, loss, margin, eh_stream(stream)));
    T.logp64 = nullptr; T.scale = W.scale; T.dlogits = dlogits;
    return tn_launch<1>(Q->dtype, T, eh_stream(stream));
}
extern "C" int edgehip_preference_loss_bwd(const edgehip_logit_rows* Q, const edgehip_preference* O, void* dlogits, void* ws,
                                           size_t ws_bytes, void* stream) {
    tn_rows T; tn_final F; tn_ws W;
    TN_TRY(tn_pref_args(Q, O, T, F, W, ws, ws_bytes));
    EH_CHECK_ARG(Q->rows == 0 || dlogits);
    TN_TRY(tn_fits<1>(Q));
    hipStream_t s = eh_stream(stream);
    F.scale = W.scale;
    T.logp64 = W.logp;                          // (what the forward left there)
    TN_TRY(tn_pref_final(F, T, s));
    T.rowstat = W.stat; T.scale = W.scale; T.dlogits = dlogits;
    return tn_launch<1>(Q->dtype, T, s);
}
