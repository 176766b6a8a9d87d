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
// registers (64 values a thread) while its sum is taken, and writes its gradient; rows too long for that are read a
// second time right after the first, from cache.  The log-probability and everything that follows from it is fp64, once
// per row: its error would enter every value of the gradient, and gaps near 0 cancel in fp32; the exponentials are
// fp32 (1e-7 relative each), their sum of many is better than each.  Sums over a sequence's rows are fp64, in a fixed order.
#include "common.h"
#include "prof.h"
#include "vec.h"

#define TN_KEEP 8                       // 8-value pieces of its row a thread keeps
#define TN_LOG2E 1.44269504088896341f

struct tn_rows {
    const void* logits; int64_t ld;     // values from one row to the next
    int64_t R; int C;
    const int64_t* taken; const uint8_t* mask;
    const int64_t* seq_ptr; int S;
    // policy
    const float *old_logp, *adv, *ref;
    int adv_per_row;
    float kl_coef; double lo, hi;       // 1 - lo, 1 + hi
    // per row
    float* logp;                        // log-probability (0 where the row does not count)
    double* logp64;                     // the same, for sums whose differences matter
    float* rowstat;                     // [R][2] max and 1 / sum
    float* term; float* kl; float* dterm; uint8_t* clipped;
    // per sequence
    const double* scale;                // factor of dterm in the gradient
    const float* coef;                  // per row instead: factor of (onehot - softmax)
    void* dlogits;                      // dense [R][C]
};

__device__ static inline bool tn_counts(const tn_rows& T, int64_t r, int64_t& a) {
    a = T.taken[r];
    if (a < 0 || a >= T.C || (T.mask && !T.mask[r])) return false;
    return !T.seq_ptr || (r >= T.seq_ptr[0] && r < T.seq_ptr[T.S]);
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

// exp(d) - 1 - d without cancellation near 0
__device__ static inline double tn_kl(double d) {
    if (fabs(d) < 0.125) {
        double s = 1.0 / 39916800.0;                             // d^11 / 11!: next term 1e-19 of the first
        s = s * d + 1.0 / 3628800.0;
        s = s * d + 1.0 / 362880.0;
        s = s * d + 1.0 / 40320.0;
        s = s * d + 1.0 / 5040.0;
        s = s * d + 1.0 / 720.0;
        s = s * d + 1.0 / 120.0;
        s = s * d + 1.0 / 24.0;
        s = s * d + 1.0 / 6.0;
        s = s * d + 0.5;
        return s * d * d;
    }
    return d > 700.0 ? exp(d) : expm1(d) - d;                    // (an infinite gap is not NaN)
}

// the policy terms of one counted row; returns d term / d logp
__device__ static inline double tn_policy(const tn_rows& T, int64_t r, int seq, double logp, double& term, double& kl, bool& cut) {
    const double A = T.adv[T.adv_per_row ? r : seq];
    const double rho = exp(logp - (double)T.old_logp[r]);
    cut = A > 0.0 ? rho > T.hi : (A < 0.0 && rho < T.lo);
    const double bound = A > 0.0 ? T.hi : T.lo;
    term = -A * (cut ? bound : rho);
    double d = cut ? 0.0 : -A * rho;
    kl = 0.0;
    if (T.ref) {
        const double gap = (double)T.ref[r] - logp;
        kl = tn_kl(gap);
        term += (double)T.kl_coef * kl;
        d -= (double)T.kl_coef * (kl + gap);                     // exp(gap) - 1
    }
    return d;
}

// max and sum over the TPR threads of a row: the running pair of a softmax, merged
__device__ static inline void tn_merge(float& m, float& s, float m2, float s2) {
    const float top = fmaxf(m, m2);
    // equal (also both -inf): no exponent of a difference of infinities
    s = (m == top ? s : s * __builtin_amdgcn_exp2f((m - top) * TN_LOG2E)) + (m2 == top ? s2 : s2 * __builtin_amdgcn_exp2f((m2 - top) * TN_LOG2E));
    m = top;
}
template <int TPR>
__device__ static inline void tn_row_merge(float& m, float& s, float* lds) {
#pragma unroll
    for (int o = 1; o < (TPR < 64 ? TPR : 64); o <<= 1) {
        const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64);
        tn_merge(m, s, m2, s2);
    }
    if (TPR > 64) {
        constexpr int NW = TPR / 64;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) { lds[(threadIdx.x >> 6) * 2] = m; lds[(threadIdx.x >> 6) * 2 + 1] = s; }
        __syncthreads();
        m = lds[0]; s = lds[1];
#pragma unroll
        for (int w = 1; w < NW; ++w) tn_merge(m, s, lds[2 * w], lds[2 * w + 1]);
    }
}

// eight more values into the running pair.  NaN: the sum becomes NaN and stays it.
__device__ static inline void tn_add8(float& m, float& s, const float (&v)[8]) {
    float top = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
    top = fmaxf(top, m);
    if (top > m) { s *= __builtin_amdgcn_exp2f((m - top) * TN_LOG2E); m = top; }     // m = -inf: s is 0 (or NaN) before
    const float base = m == -__builtin_inff() ? 0.0f : m;                            // all -inf so far: exp(-inf) = 0
    float a = 0.0f, b = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        a += __builtin_amdgcn_exp2f((v[i] - base) * TN_LOG2E);
        b += __builtin_amdgcn_exp2f((v[i + 1] - base) * TN_LOG2E);
    }
    s += a + b;
}

// MODE 0: row statistics (and the policy's per-row terms where T.old_logp is given)
// MODE 1: the gradient from row statistics;  MODE 2: both at once
template <int DT, int TPR, int MODE>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_tn_rows(tn_rows T) {
    constexpr int RPB = (TPR < 256 ? 256 : TPR) / TPR;
    __shared__ float lds[2 * (TPR < 64 ? 1 : TPR / 64)];
    const int t = threadIdx.x % TPR;
    const int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
    if (TPR <= 64 && r >= T.R) return;                           // (TPR > 64: one row per block, none too many)
    const int C = T.C;
    const int64_t base = r * T.ld;
    int64_t a;
    const bool counts = tn_counts(T, r, a);
    eh_raw8<DT> keep[TN_KEEP];
    float m = -__builtin_inff(), s = 0.0f, inv = 0.0f;
    float coef = 0.0f;
    const int full = C - 7;                                       // pieces starting below it are whole
    const bool kept = MODE == 2 && C <= TPR * 8 * TN_KEEP;
    if (MODE != 1) {
        if (counts) {
            if (kept) {
#pragma unroll
                for (int k = 0; k < TN_KEEP; ++k) {
                    const int c = (k * TPR + t) * 8;
                    if (c < full) keep[k].load(reinterpret_cast<const typename eh_elem<DT>::type*>(T.logits) + base + c);
                }
#pragma unroll
                for (int k = 0; k < TN_KEEP; ++k) {
                    const int c = (k * TPR + t) * 8;
                    float v[8];
                    if (c < full) { keep[k].get(v); tn_add8(m, s, v); }
                    else if (c < C) { eh_load8<DT>(T.logits, base + c, C - c, v, -__builtin_inff()); tn_add8(m, s, v); }
                }
            } else {
                for (int c = t * 8; c < C; c += TPR * 8) {
                    float v[8];
                    eh_load8<DT>(T.logits, base + c, C - c, v, -__builtin_inff());
                    tn_add8(m, s, v);
                }
            }
            tn_row_merge<TPR>(m, s, lds);                         // (a row counts for all of its threads or none)
        }
        double logp = 0.0, d = 0.0, term = 0.0, kl = 0.0;
        bool cut = false;
        int seq = 0;
        if (counts) {
            const float xa = (float)reinterpret_cast<const typename eh_elem<DT>::type*>(T.logits)[base + a];
            logp = (double)xa - (double)m - log((double)s);
            inv = 1.0f / s;
            if (T.old_logp) {
                seq = tn_seq(T.seq_ptr, T.S, r);
                d = tn_policy(T, r, seq, logp, term, kl, cut);
                if (MODE == 2) coef = (float)(d * T.scale[seq]);
            }
        }
        if (t == 0) {
            if (T.logp) T.logp[r] = (float)logp;
            if (T.logp64) T.logp64[r] = logp;
            if (T.rowstat) { T.rowstat[2 * r] = m; T.rowstat[2 * r + 1] = inv; }
            if (T.term) {
                T.term[r] = (float)term;
                T.kl[r] = (float)kl;
                T.clipped[r] = cut;
                if (T.dterm) T.dterm[r] = (float)d;
            }
        }
    } else if (counts) {
        m = T.rowstat[2 * r];
        inv = T.rowstat[2 * r + 1];
        const int seq = tn_seq(T.seq_ptr, T.S, r);
        coef = T.dterm ? (float)((double)T.dterm[r] * T.scale[seq]) : (float)T.scale[seq];
    }
    if (MODE != 0) {
        const float f = -coef * inv;
#pragma unroll
        for (int k = 0; k < (MODE == 2 ? TN_KEEP : 1); ++k) {
            for (int c = (k * TPR + t) * 8; c < C; c += TPR * 8) {
                float v[8];
                if (!counts) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
                } else {
                    if (kept && c < full) keep[k].get(v);
                    else eh_load8<DT>(T.logits, base + c, C - c, v, 0.0f);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = f * __builtin_amdgcn_exp2f((v[i] - m) * TN_LOG2E);
                    if (a >= c && a < c + 8) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) if (a == c + i) v[i] += coef;
                    }
                }
                eh_store8<DT>(T.dlogits, r * C + c, C - c, v);
                if (kept) break;
            }
            if (!kept) break;
        }
    }
}

// ---- sums over the rows of a sequence ----------------------------------------------------------------------------
// A block owns TN_CHUNK consecutive rows and writes one partial per (block c, sequence g) it meets, at slot c + g: along
// the rows one of the two grows by one at each border, so the slots are distinct and blocks + S of them are enough.
// WHAT 0: counted rows; 1: policy (term, kl, clipped, count); 2: preference (logp - ref)
#define TN_CHUNK 2048
template <int WHAT>
__global__ __launch_bounds__(256) void k_tn_part(tn_rows T, double* __restrict__ part) {
    __shared__ double red[4][4];
    const int64_t r0 = (int64_t)blockIdx.x * TN_CHUNK;
    int64_t r1 = r0 + TN_CHUNK < T.R ? r0 + TN_CHUNK : T.R;
    if (r1 > T.seq_ptr[T.S]) r1 = T.seq_ptr[T.S];
    if (r0 >= r1) return;
    int g = tn_seq(T.seq_ptr, T.S, r0);
    for (int64_t a = r0; a < r1;) {
        while (g < T.S - 1 && T.seq_ptr[g + 1] <= a) ++g;
        int64_t b = T.seq_ptr[g + 1];
        if (b > r1 || g == T.S - 1) b = r1;
        double v[4] = {0.0, 0.0, 0.0, 0.0};
        for (int64_t r = a + threadIdx.x; r < b; r += 256) {
            int64_t cls;
            if (!tn_counts(T, r, cls)) continue;
            v[3] += 1.0;
            if (WHAT == 1) { v[0] += T.term[r]; v[1] += T.kl[r]; v[2] += T.clipped[r]; }
            if (WHAT == 2) v[0] += T.logp64[r] - (T.ref ? (double)T.ref[r] : 0.0);
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
        if (threadIdx.x < 4) part[((int64_t)blockIdx.x + g) * 4 + threadIdx.x] = red[0][threadIdx.x] + red[1][threadIdx.x] + red[2][threadIdx.x] + red[3][threadIdx.x];
        a = b;
    }
}

struct tn_final {
    const int64_t* seq_ptr; int64_t R; int S; const double* part;
    int mean; const float* weight; double each;       // weight of a sequence's (pair's) loss in the gradient: weight[s], or each
    float *loss, *kl; int32_t* clipped;
    double* scale;                                    // d (weighted loss) / d (dterm or logp) of the sequence's rows
    float* inv_count;
    // preference
    int kind; double beta, smooth; float* margin;
};
__device__ static inline void tn_total(const tn_final& F, int g, double (&v)[4]) {
    int64_t a = F.seq_ptr[g], b = F.seq_ptr[g + 1];
    if (a < 0) a = 0;
    if (b > F.R) b = F.R;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = 0.0;
    if (a < b) {
        for (int64_t c = a / TN_CHUNK + (threadIdx.x & 63); c <= (b - 1) / TN_CHUNK; c += 64) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += F.part[(c + g) * 4 + i];
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += __shfl_xor(v[i], o, 64);
    }
}
// one wave per sequence.  PASS 0: the gradient's scale from the counted rows; 1: the losses
template <int PASS>
__global__ __launch_bounds__(64) void k_tn_policy_final(tn_final F) {
    const int g = blockIdx.x;
    double v[4];
    tn_total(F, g, v);
    if (threadIdx.x) return;
    const double inv = F.mean ? 1.0 / (v[3] > 0.0 ? v[3] : 1.0) : 1.0;
    if (F.scale) F.scale[g] = (F.weight ? (double)F.weight[g] : F.each) * inv;
    if (PASS == 1) {
        F.loss[g] = (float)(v[0] * inv);
        F.kl[g] = (float)(v[1] * inv);
        F.clipped[g] = (int32_t)v[2];
    }
}
// one wave per pair: chosen sequence g, rejected sequence g + pairs
__global__ __launch_bounds__(64) void k_tn_pref_final(tn_final F) {
    const int g = blockIdx.x, P = F.S / 2;
    double c[4], r[4];
    tn_total(F, g, c);
    tn_total(F, g + P, r);
    if (threadIdx.x) return;
    const double ic = F.mean ? 1.0 / (c[3] > 0.0 ? c[3] : 1.0) : 1.0, ir = F.mean ? 1.0 / (r[3] > 0.0 ? r[3] : 1.0) : 1.0;
    const double margin = c[0] * ic - r[0] * ir;
    double loss, d;
    if (F.kind == EDGEHIP_PREFER_SIGMOID) {
        const double x = F.beta * margin, w = exp(-fabs(x));
        loss = log1p(w) + (x < 0.0 ? -x : 0.0) + F.smooth * x;                   // -ln sigmoid(x), smoothed
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
template <int MODE>
static int tn_launch(int dtype, const tn_rows& T, hipStream_t s) {
    if (T.R == 0) return EDGEHIP_OK;
    // threads of a row: eight values each at least, 64 at most while the row can be kept
    int tpr = 1;
    if (T.C > 8) tpr = 8;
    if (T.C > 512) tpr = 64;
    if (T.C > 4096) tpr = 256;
    if (T.C > 16384) tpr = 1024;
    const int rpb = (tpr < 256 ? 256 : tpr) / tpr;
    const dim3 grid((unsigned)((T.R + rpb - 1) / rpb)), block(tpr < 256 ? 256 : tpr);
#define TN_TPR(DT, N) case N: EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_tn_rows<DT, N, MODE>), grid, block, 0, s, T)); break;
#define TN_DT(DT) switch (tpr) { TN_TPR(DT, 1) TN_TPR(DT, 8) TN_TPR(DT, 64) TN_TPR(DT, 256) TN_TPR(DT, 1024) }
    if (dtype == EDGEHIP_F32) { TN_DT(EDGEHIP_F32) }
    else if (dtype == EDGEHIP_BF16) { TN_DT(EDGEHIP_BF16) }
    else { TN_DT(EDGEHIP_F16) }
#undef TN_DT
#undef TN_TPR
    EH_LAUNCH_CHECK();
    return EDGEHIP_OK;
}

static int tn_check(const edgehip_logit_rows* Q, bool seqs = true) {
    EH_CHECK_ARG(Q && eh_dtype_ok(Q->dtype) && Q->rows >= 0 && Q->classes >= 1);
    EH_CHECK_ARG(seqs ? Q->seq_ptr && Q->num_seqs >= 1 : (Q->seq_ptr != nullptr) == (Q->num_seqs >= 1) && Q->num_seqs >= 0);
    EH_CHECK_ARG(Q->rows == 0 || (Q->logits && Q->taken && Q->row_stride >= Q->classes));
    if (Q->rows > (((int64_t)1 << 31) - 1) || Q->num_seqs > (1 << 30)) return EDGEHIP_ERR_TOO_LARGE;
    return EDGEHIP_OK;
}
static tn_rows tn_fill(const edgehip_logit_rows* Q) {
    tn_rows T = {};
    T.logits = Q->logits; T.ld = Q->row_stride; T.R = Q->rows; T.C = Q->classes;
    T.taken = Q->taken; T.mask = Q->mask; T.seq_ptr = Q->seq_ptr; T.S = Q->num_seqs;
    return T;
}
// workspace: [S] fp64 scales, [chunks + S][4] fp64 partials, per row fp32 term, kl, dterm (or stat) and a byte
struct tn_ws { double *scale, *part, *logp; float *term, *kl, *dterm, *stat; uint8_t* clipped; size_t bytes; };
static tn_ws tn_layout(const edgehip_logit_rows* Q, void* ws) {
    tn_ws W;
    const size_t R = (size_t)Q->rows, S = (size_t)Q->num_seqs, chunks = (R + TN_CHUNK - 1) / TN_CHUNK;
    char* p = reinterpret_cast<char*>(ws);
    size_t o = 0;
    auto take = [&](size_t n) { char* q = p + o; o += (n + 15) & ~(size_t)15; return q; };
    W.scale = (double*)take(S * 8);
    W.part = (double*)take((chunks + S) * 32);
    W.term = (float*)take(R * 4);
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
static int tn_sum(const tn_rows& T, double* part, hipStream_t s) {
    if (T.R == 0) return EDGEHIP_OK;
    EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_tn_part<WHAT>), dim3((unsigned)((T.R + TN_CHUNK - 1) / TN_CHUNK)), dim3(256), 0, s, T, part));
    EH_LAUNCH_CHECK();
    return EDGEHIP_OK;
}

#define TN_TRY(x) do { const int rc_ = (x); if (rc_ != EDGEHIP_OK) return rc_; } while (0)

extern "C" int edgehip_row_logp(const edgehip_logit_rows* Q, float* logp, void* stream) {
    TN_TRY(tn_check(Q, false));
    EH_CHECK_ARG(Q->rows == 0 || logp);
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
    T.kl_coef = (float)O->kl_coef; T.lo = 1.0 - O->clip_lo; T.hi = 1.0 + O->clip_hi;
    T.term = W.term; T.kl = W.kl; T.clipped = W.clipped;
    F = tn_final{};
    F.seq_ptr = Q->seq_ptr; F.R = Q->rows; F.S = Q->num_seqs; F.part = W.part;
    F.mean = O->mean; F.weight = O->weight; F.each = 1.0 / (double)Q->num_seqs;
    return EDGEHIP_OK;
}

extern "C" int edgehip_policy_loss_fwd(const edgehip_logit_rows* Q, const edgehip_policy* O, float* loss, float* kl, int32_t* clipped,
                                       float* logp, void* ws, size_t ws_bytes, void* stream) {
    tn_rows T; tn_final F; tn_ws W;
    TN_TRY(tn_policy_args(Q, O, T, F, W, ws, ws_bytes));
    EH_CHECK_ARG(loss && kl && clipped);
    hipStream_t s = eh_stream(stream);
    T.logp = logp; T.rowstat = W.stat; T.dterm = W.dterm;
    TN_TRY(tn_launch<0>(Q->dtype, T, s));
    TN_TRY(tn_sum<1>(T, W.part, s));
    F.loss = loss; F.kl = kl; F.clipped = clipped;
    EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_tn_policy_final<1>), dim3(F.S), dim3(64), 0, s, F));
    EH_LAUNCH_CHECK();
    return EDGEHIP_OK;
}
extern "C" int edgehip_policy_loss_bwd(const edgehip_logit_rows* Q, const edgehip_policy* O, void* dlogits, void* ws, size_t ws_bytes,
                                       void* stream) {
    tn_rows T; tn_final F; tn_ws W;
    TN_TRY(tn_policy_args(Q, O, T, F, W, ws, ws_bytes));
    EH_CHECK_ARG(Q->rows == 0 || dlogits);
    hipStream_t s = eh_stream(stream);
    F.scale = W.scale;                          // the partial sums of the forward are still in the workspace
    EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_tn_policy_final<0>), dim3(F.S), dim3(64), 0, s, F));
    EH_LAUNCH_CHECK();
    T.rowstat = W.stat; T.dterm = W.dterm; T.scale = W.scale; T.dlogits = dlogits;
    return tn_launch<1>(Q->dtype, T, s);
}
extern "C" int edgehip_policy_loss_grad(const edgehip_logit_rows* Q, const edgehip_policy* O, float* loss, float* kl, int32_t* clipped,
                                        float* logp, void* dlogits, void* ws, size_t ws_bytes, void* stream) {
    tn_rows T; tn_final F; tn_ws W;
    TN_TRY(tn_policy_args(Q, O, T, F, W, ws, ws_bytes));
    EH_CHECK_ARG(loss && kl && clipped && (Q->rows == 0 || dlogits));
    hipStream_t s = eh_stream(stream);
    F.scale = W.scale;
    TN_TRY(tn_sum<0>(T, W.part, s));
    EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_tn_policy_final<0>), dim3(F.S), dim3(64), 0, s, F));
    EH_LAUNCH_CHECK();
    T.logp = logp; T.scale = W.scale; T.dlogits = dlogits;
    TN_TRY(tn_launch<2>(Q->dtype, T, s));
    TN_TRY(tn_sum<1>(T, W.part, s));
    F.scale = nullptr; F.loss = loss; F.kl = kl; F.clipped = clipped;
    EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_tn_policy_final<1>), dim3(F.S), dim3(64), 0, s, F));
    EH_LAUNCH_CHECK();
    return EDGEHIP_OK;
}

static int tn_pref_args(const edgehip_logit_rows* Q, const edgehip_preference* O, tn_rows& T, tn_final& F, tn_ws& W, void* ws, size_t ws_bytes) {
    TN_TRY(tn_check(Q));
    EH_CHECK_ARG(O && Q->num_seqs % 2 == 0 && (O->kind == EDGEHIP_PREFER_SIGMOID || O->kind == EDGEHIP_PREFER_SQUARE) && O->beta > 0.0);
    EH_CHECK_ARG(O->label_smoothing >= 0.0 && O->label_smoothing < 0.5 && (O->kind == EDGEHIP_PREFER_SIGMOID || O->label_smoothing == 0.0));
    if (ws_bytes < edgehip_tune_workspace_bytes(Q)) return EDGEHIP_ERR_WORKSPACE;
    EH_CHECK_ARG(ws && ((uintptr_t)ws & 15) == 0);
    W = tn_layout(Q, ws);
    T = tn_fill(Q);
    T.ref = O->ref_logp;
    F = tn_final{};
    F.seq_ptr = Q->seq_ptr; F.R = Q->rows; F.S = Q->num_seqs; F.part = W.part;
    F.mean = O->mean; F.weight = O->weight; F.each = 2.0 / (double)Q->num_seqs;
    F.kind = O->kind; F.beta = O->beta; F.smooth = O->label_smoothing;
    return EDGEHIP_OK;
}
extern "C" int edgehip_preference_loss_fwd(const edgehip_logit_rows* Q, const edgehip_preference* O, float* loss, float* margin,
                                           void* ws, size_t ws_bytes, void* stream) {
    tn_rows T; tn_final F; tn_ws W;
    TN_TRY(tn_pref_args(Q, O, T, F, W, ws, ws_bytes));
    EH_CHECK_ARG(loss && margin);
    hipStream_t s = eh_stream(stream);
    T.logp64 = W.logp; T.rowstat = W.stat;
    TN_TRY(tn_launch<0>(Q->dtype, T, s));
    TN_TRY(tn_sum<2>(T, W.part, s));
    F.loss = loss; F.margin = margin;
    EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL(k_tn_pref_final, dim3(F.S / 2), dim3(64), 0, s, F));
    EH_LAUNCH_CHECK();
    return EDGEHIP_OK;
}
extern "C" int edgehip_preference_loss_bwd(const edgehip_logit_rows* Q, const edgehip_preference* O, void* dlogits, void* ws,
                                           size_t ws_bytes, void* stream) {
    tn_rows T; tn_final F; tn_ws W;
    TN_TRY(tn_pref_args(Q, O, T, F, W, ws, ws_bytes));
    EH_CHECK_ARG(Q->rows == 0 || dlogits);
    hipStream_t s = eh_stream(stream);
    F.scale = W.scale;
    EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL(k_tn_pref_final, dim3(F.S / 2), dim3(64), 0, s, F));
    EH_LAUNCH_CHECK();
    T.rowstat = W.stat; T.scale = W.scale; T.dlogits = dlogits;
    return tn_launch<1>(Q->dtype, T, s);
}
