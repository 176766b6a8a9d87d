// ckpt8.hip - activations kept for the backward pass in 8 bits, and the backward passes that read them.
//
// A row of K values is cut into groups of 64 (the last may be shorter).  A group shares a step 2^e, e the smallest
// integer of [-120, 121] with max|x| <= 127 2^e, and keeps round-to-nearest-even(x 2^-e), a whole number of [-127, 127]:
// off by at most 2^(e-1) <= max|x| / 127.  (Above 127 2^121 there is no such e: 121, and the codes end at 127 - a larger
// step would stand for infinity at the top.)  A POWER OF TWO as the step makes a kept value code * 2^e exact in bf16 (7 significant
// bits; bf16 has fp32's range), so in the weight gradient
//     dW[n][k] = sum over m of dY[m][n] X8[m][k]
// X8 enters the matrix instructions as ONE bf16 operand without error, and dY as 1 (bf16), 2 (fp16) or 3 (fp32) bf16
// terms that add up to it exactly: every product is exact, sums are fp32.  An fp32 product needs 3 matrix
// instructions where the six-term split of gemm.h needs 6.  A group that holds an infinity or NaN keeps e = -128: all of
// it stands for NaN, so that a bad activation stays visible in the gradients.
#include "common.h"
#include "prof.h"
#include "vec.h"

#define CK_GROUP 64
#define CK_E_MIN (-120)
#define CK_E_MAX 121
#define CK_E_BAD (-128)

typedef float ck_f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 ck_bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int ck_u32x4 __attribute__((ext_vector_type(4)));

// step of a group, or NaN
__device__ static inline float ck_step(int e) { return e == CK_E_BAD ? __uint_as_float(0x7fc00000u) : __uint_as_float((unsigned)(127 + e) << 23); }

// e of a group whose largest |x| has the bits a:  |x| = 1.m 2^(E-127) <= 127 2^e  iff  e >= E - 133, one more where
// 1.m > 127/64, that is m > 63/64 2^23
__device__ static inline int ck_exponent(unsigned a) {
    if (a >= 0x7f800000u) return CK_E_BAD;
    const int e = (int)(a >> 23) - 133 + ((a & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    return e < CK_E_MIN ? CK_E_MIN : e > CK_E_MAX ? CK_E_MAX : e;
}

// log(1 + exp(x)) and its derivative; the larger of 0 and x is split off, so nothing overflows
__device__ static inline float ck_tanh_softplus(float x) {
    // tanh(log(1 + e^x)) = ((1 + e^x)^2 - 1) / ((1 + e^x)^2 + 1) = s / (s + 2), s = e^x (e^x + 2); for x > 0 in e^-x:
    // (1 + 2 w) / (1 + 2 w + 2 w^2)
    const float w = expf(-fabsf(x));
    const float a = x > 0.0f ? 1.0f + 2.0f * w : w * (w + 2.0f);
    const float b = x > 0.0f ? 2.0f * w * w : 2.0f;
    return a / (a + b);
}
__device__ static inline float ck_sigmoid(float x) {
    const float w = expf(-fabsf(x));
    return (x >= 0.0f ? 1.0f : w) / (1.0f + w);
}
__device__ static inline float ck_act(int kind, float x) {
    return kind == EDGEHIP_ACT_SILU ? x / (1.0f + expf(-x)) : x * ck_tanh_softplus(x);
}
__device__ static inline float ck_dact(int kind, float x) {
    const float p = ck_sigmoid(x);
    if (kind == EDGEHIP_ACT_SILU) return p * (1.0f + x * (1.0f - p));
    const float t = ck_tanh_softplus(x);
    return t + x * (1.0f - t * t) * p;
}

// Eight threads a group, eight values a thread.  HBM bound: reads x, writes the codes, 1/64 exponent a value (and y).
// K a multiple of 64: group u starts at value 64 u; else its row is u / groups-per-row.
struct ck_place { int64_t off; int n; };
__device__ static inline ck_place ck_locate(unsigned u, unsigned KG, int K, int sub) {
    if ((K & 63) == 0) return ck_place{(int64_t)u * 64 + sub * 8, 8};
    const unsigned row = u / KG, g = u - row * KG;
    const int c = (int)g * 64 + sub * 8;
    return ck_place{(int64_t)row * K + c, K - c};
}

template <int DT, bool ACT>
__global__ __launch_bounds__(256) void k_ck_pack(const void* __restrict__ x, int kind, void* __restrict__ y, int8_t* __restrict__ codes,
                                                 int8_t* __restrict__ exps, unsigned ngroups, unsigned KG, int K) {
    const unsigned u = blockIdx.x * 32u + (threadIdx.x >> 3);
    const int sub = threadIdx.x & 7;
    const bool live = u < ngroups;
    ck_place p = ck_locate(live ? u : 0, KG, K, sub);
    if (!live) p.n = 0;
    float v[8];
    eh_load8<DT>(x, p.off, p.n, v);
    unsigned a = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned b = __float_as_uint(v[i]) & 0x7fffffffu;      // as whole numbers: NaN > infinity > the rest
        a = a > b ? a : b;
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        const unsigned b = (unsigned)__shfl_xor((int)a, o, 64);
        a = a > b ? a : b;
    }
    const int e = ck_exponent(a);
    const float down = e == CK_E_BAD ? 0.0f : __uint_as_float((unsigned)(127 - e) << 23);
    unsigned w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int q = e == CK_E_BAD ? 0 : (int)fminf(fmaxf(rintf(v[i] * down), -127.0f), 127.0f);    // exact product
        w[i >> 2] |= ((unsigned)q & 0xffu) << (8 * (i & 3));
    }
    if (p.n >= 8) {
        *reinterpret_cast<eh_u32x2u*>(codes + p.off) = eh_u32x2u{w[0], w[1]};
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < p.n) codes[p.off + i] = (int8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
    if (live && sub == 0) exps[u] = (int8_t)e;
    if (ACT) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = ck_act(kind, v[i]);
        eh_store8<DT>(y, p.off, p.n, v);
    }
}

__device__ static inline void ck_load_codes(const int8_t* codes, int64_t off, int n, float step, float (&o)[8]) {
    if (n >= 8) {
        const eh_u32x2u w = *reinterpret_cast<const eh_u32x2u*>(codes + off);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3))) * step;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = i < n ? (float)codes[off + i] * step : 0.0f;
    }
}

// BWD: dx = dy act'(kept x); else out = kept x
template <int DT, bool BWD>
__global__ __launch_bounds__(256) void k_ck_read(const void* __restrict__ dy, int kind, const int8_t* __restrict__ codes,
                                                 const int8_t* __restrict__ exps, void* __restrict__ out, unsigned ngroups, unsigned KG,
                                                 int K) {
    const unsigned u = blockIdx.x * 32u + (threadIdx.x >> 3);
    if (u >= ngroups) return;
    const ck_place p = ck_locate(u, KG, K, threadIdx.x & 7);
    float v[8], d[8];
    ck_load_codes(codes, p.off, p.n, ck_step(exps[u]), v);
    if (BWD) {
        eh_load8<DT>(dy, p.off, p.n, d);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = d[i] * ck_dact(kind, v[i]);
    }
    eh_store8<DT>(out, p.off, p.n, v);
}

static int ck_size(int64_t M, int64_t K, unsigned& KG, unsigned& ngroups) {
    EH_CHECK_ARG(M >= 0 && K >= 1);
    if (K > ((int64_t)1 << 31) - 64) return EDGEHIP_ERR_TOO_LARGE;
    const int64_t kg = (K + CK_GROUP - 1) / CK_GROUP;
    if (M > 0 && kg > (((int64_t)1 << 31) - 1) / M) return EDGEHIP_ERR_TOO_LARGE;
    KG = (unsigned)kg;
    ngroups = (unsigned)(M * kg);
    return EDGEHIP_OK;
}

template <bool ACT>
static int ck_pack(int dtype, const void* x, int kind, void* y, int64_t M, int64_t K, int8_t* codes, int8_t* exps, void* stream) {
    unsigned KG, ng;
    const int rc = ck_size(M, K, KG, ng);
    if (rc != EDGEHIP_OK) return rc;
    EH_CHECK_ARG(eh_dtype_ok(dtype) && (!ACT || kind == EDGEHIP_ACT_SILU || kind == EDGEHIP_ACT_MISH));
    if (ng == 0) return EDGEHIP_OK;
    EH_CHECK_ARG(x && codes && exps && (!ACT || y));
    hipStream_t s = eh_stream(stream);
    const dim3 grid((ng + 31) / 32), block(256);
#define CK_GO(DT) EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_ck_pack<DT, ACT>), grid, block, 0, s, x, kind, y, codes, exps, ng, KG, (int)K))
    if (dtype == EDGEHIP_F32) CK_GO(EDGEHIP_F32);
    else if (dtype == EDGEHIP_BF16) CK_GO(EDGEHIP_BF16);
    else CK_GO(EDGEHIP_F16);
#undef CK_GO
    EH_LAUNCH_CHECK();
    return EDGEHIP_OK;
}
template <bool BWD>
static int ck_read(int dtype, const void* dy, int kind, int64_t M, int64_t K, const int8_t* codes, const int8_t* exps, void* out, void* stream) {
    unsigned KG, ng;
    const int rc = ck_size(M, K, KG, ng);
    if (rc != EDGEHIP_OK) return rc;
    EH_CHECK_ARG(eh_dtype_ok(dtype) && (!BWD || kind == EDGEHIP_ACT_SILU || kind == EDGEHIP_ACT_MISH));
    if (ng == 0) return EDGEHIP_OK;
    EH_CHECK_ARG(codes && exps && out && (!BWD || dy));
    hipStream_t s = eh_stream(stream);
    const dim3 grid((ng + 31) / 32), block(256);
#define CK_GO(DT) EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_ck_read<DT, BWD>), grid, block, 0, s, dy, kind, codes, exps, out, ng, KG, (int)K))
    if (dtype == EDGEHIP_F32) CK_GO(EDGEHIP_F32);
    else if (dtype == EDGEHIP_BF16) CK_GO(EDGEHIP_BF16);
    else CK_GO(EDGEHIP_F16);
#undef CK_GO
    EH_LAUNCH_CHECK();
    return EDGEHIP_OK;
}

extern "C" int edgehip_pack8(int32_t dtype, const void* x, int64_t M, int64_t K, int8_t* codes, int8_t* exps, void* stream) {
    return ck_pack<false>(dtype, x, 0, nullptr, M, K, codes, exps, stream);
}
extern "C" int edgehip_unpack8(int32_t dtype, const int8_t* codes, const int8_t* exps, int64_t M, int64_t K, void* x, void* stream) {
    return ck_read<false>(dtype, nullptr, 0, M, K, codes, exps, x, stream);
}
extern "C" int edgehip_act8_fwd(int32_t dtype, int32_t kind, const void* x, int64_t M, int64_t K, void* y, int8_t* codes, int8_t* exps,
                                void* stream) {
    return ck_pack<true>(dtype, x, kind, y, M, K, codes, exps, stream);
}
extern "C" int edgehip_act8_bwd(int32_t dtype, int32_t kind, const void* dy, const int8_t* codes, const int8_t* exps, int64_t M, int64_t K,
                                void* dx, void* stream) {
    return ck_read<true>(dtype, dy, kind, M, K, codes, exps, dx, stream);
}

// ------------------------------------------------------------------------------------------------------------------
// dW[N][K] = dY[M][N]^T X8[M][K], db[n] = sum over m of dY[m][n].
//
// The sum runs over the ROWS of both operands, the slow axis of both: a matrix instruction wants eight consecutive m of
// one column per lane.  A thread therefore stages an 8 x 8 block (eight rows, eight columns: 16-byte reads of 16-bit
// rows), turns it in registers - two rows' values of a column side by side are one v_perm - and writes eight 16-byte
// pieces [column][eight m] to LDS.  Tile image: piece (m / 8, column c) at ((m / 8) * 128 + c') * 16 bytes, c' = c with
// its low three bits xored by the next three: the eight writers of a bank phase hold columns 8 apart and land in eight
// different 16-byte slots, and a fragment (32 consecutive columns) still reads 32 consecutive pieces.
//
// A block owns a 128 x 128 tile of dW and a run of rows (blockIdx.z); four waves, 64 x 64 each.  The rows are split
// when the tiles alone do not fill the chip; partial tiles go to the workspace and are added in order by k_ck_dw_sum.
// ------------------------------------------------------------------------------------------------------------------
#define DW_T 128
#define DW_M 32
#define DW_PIECES (DW_M / 8 * DW_T)          // 16-byte pieces of one operand plane

template <int DT> struct dw_planes { static constexpr int value = DT == EDGEHIP_BF16 ? 1 : DT == EDGEHIP_F16 ? 2 : 3; };

// x = t[0] + t[1] + ... by truncation to 8 significant bits each; the upper halves of two rows' values in one dword.
// An infinity or NaN stays in the first term (its remainder would be NaN: zero instead).
template <int P>
__device__ static inline void dw_split(float x0, float x1, unsigned (&o)[P]) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const unsigned u0 = __float_as_uint(x0), u1 = __float_as_uint(x1);
        o[p] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
        if (p + 1 < P) {
            x0 = (u0 & 0x7f800000u) == 0x7f800000u ? 0.0f : x0 - __uint_as_float(u0 & 0xffff0000u);
            x1 = (u1 & 0x7f800000u) == 0x7f800000u ? 0.0f : x1 - __uint_as_float(u1 & 0xffff0000u);
        }
    }
}
// (truncation would turn a NaN whose payload lies in the low half into an infinity: such values are made quiet first)
__device__ static inline float dw_quiet(float x) { return x != x ? __uint_as_float(0x7fc00000u) : x; }

__device__ static inline int dw_piece(int mblk, int c) { return mblk * DW_T + ((c & ~7) | ((c ^ (c >> 3)) & 7)); }

template <int DT>
__global__ __launch_bounds__(256) void k_ck_dw(const void* __restrict__ dY, const int8_t* __restrict__ codes, const int8_t* __restrict__ exps,
                                               int64_t M, int N, int K, int KG, int64_t rows_per_split, float* __restrict__ out,
                                               float* __restrict__ db) {
    constexpr int P = dw_planes<DT>::value;
    __shared__ ck_u32x4 ya[P][DW_PIECES], xa[DW_PIECES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int k0 = blockIdx.x * DW_T, n0 = blockIdx.y * DW_T;
    const int64_t m0 = (int64_t)blockIdx.z * rows_per_split;
    const int64_t m1 = m0 + rows_per_split < M ? m0 + rows_per_split : M;
    // staging: threads 0..63 the 8x8 blocks of dY, 64..127 those of X (4 x 16 blocks each)
    const int c8 = (lane & 15) * 8, mb = lane >> 4;
    const bool want_db = db && blockIdx.x == 0;
    float bsum[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) bsum[i] = 0.0f;
    ck_f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    const int wn = (wave & 1) * 64, wk = (wave >> 1) * 64;
    for (int64_t m = m0; m < m1; m += DW_M) {
        __syncthreads();
        if (wave < 2) {
            float v[8][8];
            const int64_t r = m + mb * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool in = r + i < m1;
                if (wave == 0) {
                    eh_load8<DT>(dY, (r + i) * N + n0 + c8, in ? N - n0 - c8 : 0, v[i]);
                } else {
                    const int n = K - k0 - c8;
                    const float st = in && n > 0 ? ck_step(exps[(r + i) * KG + ((k0 + c8) >> 6)]) : 0.0f;
                    ck_load_codes(codes, (r + i) * K + k0 + c8, in ? n : 0, st, v[i]);
                }
            }
            if (wave == 0) {
                if (want_db) {
#pragma unroll
                    for (int c = 0; c < 8; ++c)
#pragma unroll
                        for (int i = 0; i < 8; ++i) bsum[c] += v[i][c];
                }
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    ck_u32x4 w[P];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        unsigned o[P];
                        dw_split<P>(dw_quiet(v[2 * i][c]), dw_quiet(v[2 * i + 1][c]), o);
#pragma unroll
                        for (int p = 0; p < P; ++p) w[p][i] = o[p];
                    }
#pragma unroll
                    for (int p = 0; p < P; ++p) ya[p][dw_piece(mb, c8 + c)] = w[p];
                }
            } else {
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    ck_u32x4 w;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        unsigned o[1];
                        dw_split<1>(v[2 * i][c], v[2 * i + 1][c], o);
                        w[i] = o[0];
                    }
                    xa[dw_piece(mb, c8 + c)] = w;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < DW_M / 16; ++s) {
            const int mblk = s * 2 + (lane >> 5);
            ck_bf16x8 b[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) b[j] = __builtin_bit_cast(ck_bf16x8, xa[dw_piece(mblk, wk + j * 32 + (lane & 31))]);
#pragma unroll
            for (int p = P - 1; p >= 0; --p) {                  // small terms first
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const ck_bf16x8 a = __builtin_bit_cast(ck_bf16x8, ya[p][dw_piece(mblk, wn + i * 32 + (lane & 31))]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b[j], acc[i][j], 0, 0, 0);
                }
            }
        }
    }
    float* o = out + (int64_t)blockIdx.z * N * K;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int n = n0 + wn + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5), k = k0 + wk + j * 32 + (lane & 31);
                if (n < N && k < K) o[(int64_t)n * K + k] = acc[i][j][r];
            }
    if (want_db && wave == 0) {
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            bsum[c] += __shfl_xor(bsum[c], 16, 64);
            bsum[c] += __shfl_xor(bsum[c], 32, 64);
            if (lane < 16 && n0 + c8 + c < N) db[(int64_t)blockIdx.z * N + n0 + c8 + c] = bsum[c];
        }
    }
}

// sum of the splits' partial results, in order
__global__ __launch_bounds__(256) void k_ck_dw_sum(const float* __restrict__ part, int64_t n, int splits, float* __restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float a = 0.0f;
    for (int z = 0; z < splits; ++z) a += part[z * n + i];
    out[i] = a;
}

// Splits of the rows: enough blocks for the 256 CUs, but at least 256 rows a split
static int dw_splits(int64_t M, int N, int K, int64_t& rows) {
    const int64_t tiles = (int64_t)eh_cdiv(N, DW_T) * eh_cdiv(K, DW_T);
    int64_t s = (512 + tiles - 1) / tiles;
    const int64_t most = (M + 255) / 256;
    if (s > most) s = most;
    if (s < 1) s = 1;
    rows = (M + s - 1) / s;
    rows = (rows + DW_M - 1) / DW_M * DW_M;
    if (rows < DW_M) rows = DW_M;
    return (int)((M + rows - 1) / rows > 0 ? (M + rows - 1) / rows : 1);
}

static int dw_check(int32_t dtype, int64_t M, int32_t N, int32_t K) {
    EH_CHECK_ARG(eh_dtype_ok(dtype) && M >= 0 && N >= 1 && K >= 1);
    if (N > (1 << 22) || K > (1 << 22)) return EDGEHIP_ERR_TOO_LARGE;        // grid limits and 32-bit column arithmetic
    return EDGEHIP_OK;
}

extern "C" size_t edgehip_linear8_workspace_bytes(int32_t dtype, int64_t M, int32_t N, int32_t K) {
    if (dw_check(dtype, M, N, K) != EDGEHIP_OK) return 0;
    int64_t rows;
    const int s = dw_splits(M, N, K, rows);
    return s > 1 ? (size_t)s * ((size_t)N * K + N) * sizeof(float) : 16;
}

extern "C" int edgehip_linear8_bwd_weight(int32_t dtype, const void* dY, const int8_t* codes, const int8_t* exps, int64_t M, int32_t N,
                                          int32_t K, float* dW, float* db, void* ws, size_t ws_bytes, void* stream) {
    const int rc = dw_check(dtype, M, N, K);
    if (rc != EDGEHIP_OK) return rc;
    EH_CHECK_ARG(dW && (M == 0 || (dY && codes && exps)));
    if (ws_bytes < edgehip_linear8_workspace_bytes(dtype, M, N, K)) return EDGEHIP_ERR_WORKSPACE;
    int64_t rows;
    const int splits = dw_splits(M, N, K, rows);
    EH_CHECK_ARG(splits == 1 || (ws && ((uintptr_t)ws & 3) == 0));
    hipStream_t s = eh_stream(stream);
    float* part = splits > 1 ? reinterpret_cast<float*>(ws) : dW;
    float* pdb = !db ? nullptr : splits > 1 ? part + (int64_t)splits * N * K : db;
    const dim3 grid(eh_cdiv(K, DW_T), eh_cdiv(N, DW_T), splits), block(256);
    const int KG = (K + CK_GROUP - 1) / CK_GROUP;
#define DW_GO(DT) EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_ck_dw<DT>), grid, block, 0, s, dY, codes, exps, M, N, K, KG, rows, part, pdb))
    if (dtype == EDGEHIP_F32) DW_GO(EDGEHIP_F32);
    else if (dtype == EDGEHIP_BF16) DW_GO(EDGEHIP_BF16);
    else DW_GO(EDGEHIP_F16);
#undef DW_GO
    EH_LAUNCH_CHECK();
    if (splits > 1) {
        const int64_t n = (int64_t)N * K;
        EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL(k_ck_dw_sum, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, part, n, splits, dW));
        EH_LAUNCH_CHECK();
        if (db) {
            EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL(k_ck_dw_sum, dim3((N + 255) / 256), dim3(256), 0, s, pdb, (int64_t)N, splits, db));
            EH_LAUNCH_CHECK();
        }
    }
    return EDGEHIP_OK;
}
