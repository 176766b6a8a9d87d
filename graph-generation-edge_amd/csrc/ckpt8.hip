// ckpt8.hip - activations kept for the backward pass in 8 bits, and the backward passes that read them.
//
// A row of K values is cut into groups of 64 (the last may be shorter).  A group shares a step 2^e, e the smallest
// integer of [-120, 121] with max|x| <= 127 2^e, and keeps round-to-nearest-even(x 2^-e), a whole number of [-127, 127]:
// off by at most 2^(e-1), which is at most max|x| / 127 but for a group at the smallest step, off by up to 2^-121 however
// small its values are.  (Above 127 2^121 there is no such e: 121, and the codes end at 127 - a larger step would stand for
// infinity at the top.)  A POWER OF TWO as the step makes a kept value code * 2^e exact in bf16 (7 significant bits; bf16 has
// fp32's range), so in the weight gradient
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
typedef unsigned int ck_u32u __attribute__((aligned(1)));
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

// The activations and their derivatives.  FAST, for 16-bit results: e^-|x| and 1 / (1 + .) by the hardware's instructions
// (together 1e-6 relative, their rounding is 2^-9 or 2^-12); fp32 results take the library's.
template <bool FAST> __device__ static inline float ck_exp_neg(float x) {       // e^-|x|
    return FAST ? __builtin_amdgcn_exp2f(fabsf(x) * -1.44269504088896341f) : expf(-fabsf(x));
}
template <bool FAST> __device__ static inline float ck_div(float a, float b) { return FAST ? a * __builtin_amdgcn_rcpf(b) : a / b; }
// tanh(log(1 + e^x)) = ((1 + e^x)^2 - 1) / ((1 + e^x)^2 + 1) = s / (s + 2), s = w (w + 2), w = e^x; for x > 0 in w = e^-x:
// (1 + 2 w) / (1 + 2 w + 2 w^2)
template <bool FAST> __device__ static inline float ck_tanh_softplus(float x, float w) {
    const float a = x > 0.0f ? 1.0f + 2.0f * w : w * (w + 2.0f);
    const float b = x > 0.0f ? 2.0f * w * w : 2.0f;
    return ck_div<FAST>(a, a + b);
}
template <bool FAST> __device__ static inline float ck_sigmoid(float x, float w) { return ck_div<FAST>(x >= 0.0f ? 1.0f : w, 1.0f + w); }
template <bool FAST> __device__ static inline float ck_act(int kind, float x) {
    const float w = ck_exp_neg<FAST>(x);
    return x * (kind == EDGEHIP_ACT_SILU ? ck_sigmoid<FAST>(x, w) : ck_tanh_softplus<FAST>(x, w));
}
template <bool FAST> __device__ static inline float ck_dact(int kind, float x) {
    const float w = ck_exp_neg<FAST>(x), p = ck_sigmoid<FAST>(x, w);
    if (kind == EDGEHIP_ACT_SILU) return p * (1.0f + x * (1.0f - p));
    const float t = ck_tanh_softplus<FAST>(x, w);
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

template <int DT, bool ACT, bool TINY>
__global__ __launch_bounds__(256) void k_ck_pack(const void* __restrict__ x, int kind, void* __restrict__ y, int8_t* __restrict__ codes,
                                                 int8_t* __restrict__ exps, unsigned ngroups, unsigned KG, int K, int64_t end) {
    const unsigned u = blockIdx.x * 32u + (threadIdx.x >> 3);
    const int sub = threadIdx.x & 7;
    const bool live = u < ngroups;
    ck_place p = ck_locate(live ? u : 0, KG, K, sub);
    if (!live) p.n = 0;
    const eh_at at = eh_place(p.off, p.n, end);
    eh_raw8<DT> in;
    float v[8];
    eh_get<DT, TINY>(in, x, at);
    in.get(v);
    eh_own<TINY>(v, at.n, at.back);
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
    int8_t* q = codes + p.off;
    if (p.n >= 8) {
        *reinterpret_cast<eh_u32x2u*>(q) = eh_u32x2u{w[0], w[1]};
    } else if (p.n > 0) {                                        // in pieces of four, two and one
        if (p.n & 4) *reinterpret_cast<ck_u32u*>(q) = w[0];
        const unsigned rest = p.n & 4 ? w[1] : w[0];
        q += p.n & 4;
        if (p.n & 2) { q[0] = (int8_t)rest; q[1] = (int8_t)(rest >> 8); }
        if (p.n & 1) q[p.n & 2] = (int8_t)(p.n & 2 ? rest >> 16 : rest);
    }
    if (live && sub == 0) exps[u] = (int8_t)e;
    if (ACT) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = ck_act<DT != EDGEHIP_F32>(kind, v[i]);
        eh_store8<DT>(y, p.off, p.n, v);
    }
}

// eight codes where eh_place puts them, as values; what lies behind a row's end stays what it is
template <bool TINY>
__device__ static inline void ck_load_codes(const int8_t* codes, const eh_at& at, float step, float (&o)[8]) {
    uint64_t w = 0;
    if (!TINY) {
        const eh_u32x2u v = *reinterpret_cast<const eh_u32x2u*>(codes + at.off);
        w = ((uint64_t)v[1] << 32 | v[0]) >> (8 * at.back);
    } else {
        for (int i = 0; i < at.n; ++i) w |= (uint64_t)(uint8_t)codes[at.off + at.back + i] << (8 * i);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (float)(int8_t)(w >> (8 * i)) * step;
}

// BWD: dx = dy act'(kept x); else out = kept x
template <int DT, bool BWD, bool TINY>
__global__ __launch_bounds__(256) void k_ck_read(const void* __restrict__ dy, int kind, const int8_t* __restrict__ codes,
                                                 const int8_t* __restrict__ exps, void* __restrict__ out, unsigned ngroups, unsigned KG,
                                                 int K, int64_t end) {
    const unsigned u = blockIdx.x * 32u + (threadIdx.x >> 3);
    if (u >= ngroups) return;
    const ck_place p = ck_locate(u, KG, K, threadIdx.x & 7);
    const eh_at at = eh_place(p.off, p.n, end);
    eh_raw8<DT> in;
    float v[8], d[8];
    if (BWD) eh_get<DT, TINY>(in, dy, at);
    ck_load_codes<TINY>(codes, at, ck_step(exps[u]), v);
    if (BWD) {
        in.get(d);
        eh_own<TINY>(d, at.n, at.back);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = d[i] * ck_dact<DT != EDGEHIP_F32>(kind, v[i]);
    }
    eh_store8<DT>(out, p.off, p.n, v);
}

static int ck_size(int64_t M, int64_t K, unsigned& KG, unsigned& ngroups) {
    EH_CHECK_ARG(M >= 0 && K >= 1);
    if (K > ((int64_t)1 << 31) - 64) return EDGEHIP_ERR_TOO_LARGE;
    const int64_t kg = (K + CK_GROUP - 1) / CK_GROUP;
    if (M > 0 && (kg > (((int64_t)1 << 31) - 1) / M || !eh_grid_ok((M * kg + 31) / 32, 256))) return EDGEHIP_ERR_TOO_LARGE;
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
#define CK_AS(DT, TINY) EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_ck_pack<DT, ACT, TINY>), grid, block, 0, s, x, kind, y, codes, exps, ng, KG, (int)K, M * K))
#define CK_GO(DT) do { if (M * K < 8) CK_AS(DT, true); else CK_AS(DT, false); } while (0)
    if (dtype == EDGEHIP_F32) CK_GO(EDGEHIP_F32);
    else if (dtype == EDGEHIP_BF16) CK_GO(EDGEHIP_BF16);
    else CK_GO(EDGEHIP_F16);
#undef CK_GO
#undef CK_AS
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
#define CK_AS(DT, TINY) EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_ck_read<DT, BWD, TINY>), grid, block, 0, s, dy, kind, codes, exps, out, ng, KG, (int)K, M * K))
#define CK_GO(DT) do { if (M * K < 8) CK_AS(DT, true); else CK_AS(DT, false); } while (0)
    if (dtype == EDGEHIP_F32) CK_GO(EDGEHIP_F32);
    else if (dtype == EDGEHIP_BF16) CK_GO(EDGEHIP_BF16);
    else CK_GO(EDGEHIP_F16);
#undef CK_GO
#undef CK_AS
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
// The sum runs over the ROWS of both operands, the slow axis of both, while a matrix instruction wants eight consecutive
// m of one column in a lane.  A thread therefore stages 8-row x CW-column pieces of each operand, turns them in registers - two rows' values of a column side by side are one v_perm - and writes CW 16-byte
// pieces [column][eight m] to LDS.  The piece (m / 8, column c) stands at ((m / 8) T + c') 16 bytes, c' = c with its low
// three bits xored by the next three: the eight writers of a bank phase, whose columns are 4 or 8 apart, land in eight
// different slots, and a fragment (32 consecutive columns) still reads 32 consecutive pieces: no bank conflicts.
//
// A block owns a T x T tile of dW and a run of rows; four waves, T/2 x T/2 each.  T = 256 needs half the LDS reads per flop
// of T = 128 and is taken for large products (dw_choose); its 256 accumulators leave one wave a SIMD, so everything
// else is placed between its matrix instructions: two LDS images, and while a chunk of BM rows is multiplied, the next
// one's registers (requested a chunk earlier) are turned and written and the one after is requested, in one run of
// instructions without a branch; one barrier a chunk, which waits for LDS only, so that the requests stay in flight
// across it.  Launches back to back, the sums of partials with them: 16384 x 4096 x 4096 bf16 519-529 us, 1040-1060 TFLOP/s - the
// library's bf16 product of that shape, which has no codes to turn, 520-527 us; the matrix pipe is busy 45 % of the cycles, vector
// instructions issue in 34 %.  fp16 / fp32: 570 / 399 TFLOP/s (two / three terms).  78208 x 512 x 128 fp32, T = 128 with two
// blocks a CU: 58 us, 2.9 TB/s of dY and codes; matrix pipe 23 %, vector instructions 36 % of the cycles, waves wait 36 % of
// their time for their turn to issue and 23 % for memory or a barrier.  (One launch at a time, as a tracer runs them, the first is
// 550-590 us, the second 61-63 us and 9 us.)
// Not kept: a fixed pattern of one matrix instruction and 5 or 6 others (630-670 us); pieces of four rows with wider
// reads and the exponents group by group (617 us).
//
// The rows are split where the tiles alone do not fill the chip; partial tiles go to the workspace and are added in
// order by k_ck_dw_sum.  db: the block of k-tile j adds up the chunks with number j modulo the k-tiles, so that this work
// is spread over them (up to 128 rows: the first block's alone); partials by (split, k-tile).
// ------------------------------------------------------------------------------------------------------------------
#define CK_BARRIER() asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory")

template <int DT> struct dw_planes { static constexpr int value = DT == EDGEHIP_BF16 ? 1 : DT == EDGEHIP_F16 ? 2 : 3; };
// rows a chunk: two images of (planes + 1) x T x BM x 2 bytes must fit the 160 KB of LDS, twice for two blocks a CU (T = 128)
template <int DT> struct dw_rows { static constexpr int value = DT == EDGEHIP_BF16 ? 64 : 32; };

// x = t[0] + t[1] + ... by truncation to 8 significant bits each; the upper halves of two rows' values in one dword.  An
// infinity leaves a NaN in the second term (as a NaN does, whose payload truncation could lose): with two or three terms
// whatever is not finite makes the gradients it reaches NaN.
template <int P>
__device__ static inline void dw_split(float x0, float x1, unsigned (&o)[P]) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const unsigned u0 = __float_as_uint(x0), u1 = __float_as_uint(x1);
        o[p] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
        if (p + 1 < P) {
            x0 -= __uint_as_float(u0 & 0xffff0000u);
            x1 -= __uint_as_float(u1 & 0xffff0000u);
        }
    }
}

template <int CW> struct dw_word { typedef unsigned type __attribute__((aligned(1))); };
template <> struct dw_word<2> { typedef unsigned short type __attribute__((aligned(1))); };
template <bool B> struct dw_flag { static constexpr bool value = B; };

template <int T>
__device__ static inline int dw_piece(int mblk, int c) { return mblk * T + ((c & ~7) | ((c ^ (c >> 3)) & 7)); }

// a global address whose base is in scalar registers
#define DW_GLOBAL __attribute__((address_space(1)))
typedef const DW_GLOBAL char* dw_addr;
__device__ static inline dw_addr dw_uniform(const void* p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const unsigned lo = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)v), hi = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(v >> 32));
    return reinterpret_cast<dw_addr>(((uint64_t)hi << 32) | lo);
}

// CW consecutive values of a dY row as they stand in memory: DWORDS registers
template <int DT, int CW> struct dw_y {
    static constexpr int DWORDS = CW * (DT == EDGEHIP_F32 ? 4 : 2) / 4;
    unsigned d[DWORDS];
    __device__ inline void load(dw_addr p) {
        typedef unsigned vec __attribute__((ext_vector_type(DWORDS), aligned(2)));
        const vec v = *reinterpret_cast<const DW_GLOBAL vec*>(p);
#pragma unroll
        for (int i = 0; i < DWORDS; ++i) d[i] = v[i];
    }
    __device__ inline void clear() {
#pragma unroll
        for (int i = 0; i < DWORDS; ++i) d[i] = 0u;
    }
    __device__ inline float get(int c) const {
        if (DT == EDGEHIP_F32) return __uint_as_float(d[c < DWORDS ? c : 0]);
        const unsigned w = d[c / 2 < DWORDS ? c / 2 : 0];
        if (DT == EDGEHIP_BF16) return __uint_as_float(c & 1 ? w & 0xffff0000u : w << 16);
        return (float)__builtin_bit_cast(_Float16, (unsigned short)(c & 1 ? w >> 16 : w));
    }
};

template <int DT, int T>
__global__ __launch_bounds__(256, T == 256 ? 1 : 2) void k_ck_dw(const void* __restrict__ dY, const int8_t* __restrict__ codes,
                                                                const int8_t* __restrict__ exps, int64_t M, int N, int K, int KG,
                                                                int64_t rows_per_split, int nt, int kt, int kb, float* __restrict__ out,
                                                                float* __restrict__ db) {
    constexpr int P = dw_planes<DT>::value, BM = dw_rows<DT>::value, CW = T * BM >= 8192 ? 4 : 2, W = T / 2, F = W / 32;
    constexpr int MB = 256 / (T / CW), U = BM / 8 / MB;         // m-blocks staged at once, times the U pieces of a thread
    constexpr int D = T == 256 ? 1 : 2;                          // chunks requested ahead of the one being staged
    constexpr int PIECES = BM / 8 * T, ES = DT == EDGEHIP_F32 ? 4 : 2;
    __shared__ ck_u32x4 img[2][(P + 1) * PIECES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // tiles in runs of four n-tiles; consecutive tiles to one XCD (blocks are dealt to the eight of them in turn), so that
    // its L2 holds the few panels its blocks share
    int id = blockIdx.x;
    const int total = nt * kt;
    if ((total & 7) == 0) id = (id & 7) * (total >> 3) + (id >> 3);
    const int band = id / (4 * kt), left = nt - band * 4 < 4 ? nt - band * 4 : 4, in = id - band * 4 * kt;
    const int ktile = in / left, k0 = ktile * T;
    // the last n-tile is moved back to end with dY: its first columns are then made twice, to the same bits
    int n0 = (band * 4 + in % left) * T;
    if (n0 + T > N) n0 = N > T ? N - T : 0;
    const int64_t m0 = (int64_t)blockIdx.y * rows_per_split;
    const int64_t m1 = m0 + rows_per_split < M ? m0 + rows_per_split : M;
    // Staging: CW (2 or 4) columns and, U times, eight rows of both operands a thread.  No access leaves its tensor: columns behind
    // the end of a dY narrower than the tile are those of its last CW (written again where they belong), a word of codes
    // that passes the end of its row reads into the next one (columns behind the end go nowhere), in the last chunk it is
    // read further left and shifted.  Rows behind the last one are read from it, with step 0.
    const int c0 = (tid % (T / CW)) * CW, mb = tid / (T / CW);
    const int yc = c0 + CW <= N - n0 ? c0 : N - n0 - CW;
    const int kc = k0 + c0 < K ? k0 + c0 : K - 1, kw = kc + CW <= K ? kc : K - CW, xs = (kc - kw) * 8;
    const unsigned yv = (unsigned)(((int64_t)mb * 8 * N + n0 + yc) * ES), xv = (unsigned)(mb * 8 * K + kc), ev = (unsigned)(mb * 8 * KG + (kc >> 6));
    dw_y<DT, CW> y[D * U][8];
    unsigned x[D * U][8];
    int e[D * U][8];
    typedef typename dw_word<CW>::type word;
    // piece u (of register set u / U) of the chunk at row m
    auto request = [&](int64_t m, int u, auto whole) {
        const int64_t mu = m + u % U * MB * 8;
        if constexpr (decltype(whole)::value) {
            // (bases of the scalar unit, one 32-bit offset a lane: no address arithmetic in the vector unit)
            const dw_addr yp = dw_uniform(reinterpret_cast<const char*>(dY) + mu * N * ES), xp = dw_uniform(codes + mu * K),
                          ep = dw_uniform(exps + mu * KG);
            unsigned yo = yv, xo = xv, eo = ev;
            asm("" : "+v"(yo), "+v"(xo), "+v"(eo));             // extended to 64 bits here, where the load can fold it
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                y[u][i].load(yp + (int64_t)i * N * ES + yo);
                x[u][i] = *reinterpret_cast<const DW_GLOBAL word*>(xp + (int64_t)i * K + xo);
                e[u][i] = *reinterpret_cast<const DW_GLOBAL int8_t*>(ep + (int64_t)i * KG + eo);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int64_t r = mu + mb * 8 + i, q = r < m1 ? r : m1 - 1;
                y[u][i].load(reinterpret_cast<dw_addr>(reinterpret_cast<uint64_t>(dY)) + (q * N + n0 + yc) * ES);
                if (r >= m1) y[u][i].clear();                    // (an infinity there times step 0 would be NaN)
                x[u][i] = (unsigned)*reinterpret_cast<const word*>(codes + q * K + kw) >> xs;
                e[u][i] = r < m1 ? exps[q * KG + (kc >> 6)] : -127;
            }
        }
    };
    float bsum[CW];
#pragma unroll
    for (int c = 0; c < CW; ++c) bsum[c] = 0.0f;
    auto put = [&](ck_u32x4* im, int u) {
        const int mblk = u % U * MB + mb;
#pragma unroll
        for (int c = 0; c < CW; ++c) {
            ck_u32x4 w[P];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                unsigned o[P];
                if (DT == EDGEHIP_BF16) o[0] = __builtin_amdgcn_perm(y[u][2 * i + 1].d[c / 2], y[u][2 * i].d[c / 2], c & 1 ? 0x07060302u : 0x05040100u);
                else dw_split<P>(y[u][2 * i].get(c), y[u][2 * i + 1].get(c), o);
#pragma unroll
                for (int p = 0; p < P; ++p) w[p][i] = o[p];
            }
#pragma unroll
            for (int p = 0; p < P; ++p) im[p * PIECES + dw_piece<T>(mblk, yc + c)] = w[p];
        }
        float st[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            // exponent -128 gives -infinity, and such a group's codes are 0: code * step is NaN, as it should be
            st[i] = __uint_as_float((unsigned)(127 + e[u][i]) << 23);
#pragma unroll
        for (int c = 0; c < CW; ++c) {
            ck_u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) v[h] = (float)(int8_t)(x[u][2 * i + h] >> (8 * c)) * st[2 * i + h];
                w[i] = __builtin_amdgcn_perm(__float_as_uint(v[1]), __float_as_uint(v[0]), 0x07060302u);
            }
            im[P * PIECES + dw_piece<T>(mblk, c0 + c)] = w;
        }
    };
    ck_f32x16 acc[F][F];
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    const int wn = (wave & 1) * W, wk = (wave >> 1) * W, fr = lane & 31, fh = lane >> 5;
    int turn = 0, chunk = 0;
    // the column sums of the chunk at row m, which register set `set` holds
    auto count_db = [&](int64_t m, int set) {
        if (db && chunk % kb == ktile) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const bool live = m + (u * MB + mb) * 8 + i < m1;
#pragma unroll
                    for (int c = 0; c < CW; ++c) bsum[c] += live ? y[set * U + u][i].get(c) : 0.0f;
                }
        }
        ++chunk;
    };
    if (m0 < m1) {
#pragma unroll
        for (int u = 0; u < D * U; ++u)
            if (m0 + u / U * BM < m1) request(m0 + u / U * BM, u, dw_flag<false>{});
        count_db(m0, 0);
#pragma unroll
        for (int u = 0; u < U; ++u) put(img[0], u);
        if (m0 + D * BM < m1) {
#pragma unroll
            for (int u = 0; u < U; ++u) request(m0 + D * BM, u, dw_flag<false>{});
        }
    }
    // one chunk: S x P x F x F matrix instructions; STAGE: the next chunk's registers are turned and written in between, in
    // the same run of instructions, so that the vector unit works while the matrix unit does
    constexpr int S = BM / 16;
    auto fetch_b = [&](const ck_u32x4* im, int s, ck_bf16x8 (&b)[F]) {
#pragma unroll
        for (int j = 0; j < F; ++j) b[j] = __builtin_bit_cast(ck_bf16x8, im[P * PIECES + dw_piece<T>(s * 2 + fh, wk + j * 32 + fr)]);
    };
    auto fetch_a = [&](const ck_u32x4* im, int s, int p, ck_bf16x8 (&a)[F]) {
#pragma unroll
        for (int i = 0; i < F; ++i) a[i] = __builtin_bit_cast(ck_bf16x8, im[p * PIECES + dw_piece<T>(s * 2 + fh, wn + i * 32 + fr)]);
    };
    auto multiply = [&](const ck_u32x4* im, ck_u32x4* next, int64_t after, int set, auto stage, auto whole) {
        ck_bf16x8 a[2][F], b[2][F];
        fetch_b(im, 0, b[0]);
        fetch_a(im, 0, P - 1, a[0]);
#pragma unroll
        for (int q = 0; q < S * P; ++q) {                       // small terms first
            const int s = q / P, s1 = (q + 1) / P;
            if (q + 1 < S * P) {
                if (s1 != s) fetch_b(im, s1, b[s1 & 1]);
                fetch_a(im, s1, P - 1 - (q + 1) % P, a[(q + 1) & 1]);
            }
            if constexpr (decltype(stage)::value) {
                if (q % (S * P / U) == 0) put(next, set * U + q / (S * P / U));
            }
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < F; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[q & 1][i], b[s & 1][j], acc[i][j], 0, 0, 0);
            if constexpr (decltype(stage)::value) {
                // the registers just written are free again: they are filled for the chunk D behind the one they held, most of D
                // chunks' time before they are needed
                if (q % (S * P / U) == 0 && (decltype(whole)::value || after < m1)) request(after, set * U + q / (S * P / U), whole);
            }
        }
    };
    int64_t m = m0;
    while (m + (2 * D + 1) * BM < m1) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            CK_BARRIER();
            count_db(m + BM, (d + 1) % D);
            multiply(img[turn], img[turn ^ 1], m + (D + 1) * BM, (d + 1) % D, dw_flag<true>{}, dw_flag<true>{});
            turn ^= 1;
            m += BM;
        }
    }
    while (m + BM < m1) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (m + BM >= m1) break;
            CK_BARRIER();
            count_db(m + BM, (d + 1) % D);
            multiply(img[turn], img[turn ^ 1], m + (D + 1) * BM, (d + 1) % D, dw_flag<true>{}, dw_flag<false>{});
            turn ^= 1;
            m += BM;
        }
    }
    if (m < m1) {
        CK_BARRIER();
        multiply(img[turn], nullptr, m1, 0, dw_flag<false>{}, dw_flag<false>{});
    }
    float* o = out + (int64_t)blockIdx.y * N * K;
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int n = n0 + wn + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * fh, k = k0 + wk + j * 32 + fr;
                if (n < N && k < K) o[(int64_t)n * K + k] = acc[i][j][r];
            }
    if (db && ktile < kb) {
        // the MB threads that hold one column's sums, through LDS
        __syncthreads();
        float* red = reinterpret_cast<float*>(img[0]);
#pragma unroll
        for (int c = 0; c < CW; ++c) red[mb * T + yc + c] = bsum[c];
        __syncthreads();
        if (tid < T && n0 + tid < N) {
            float s = 0.0f;
#pragma unroll
            for (int b = 0; b < MB; ++b) s += red[b * T + tid];
            db[((int64_t)blockIdx.y * kb + ktile) * N + n0 + tid] = s;
        }
    }
}

// Fewer than four columns on one side: nothing for a tile.  A thread owns one value of dW, 256 of them a block; rows as
// above.  HBM bound (the wide side is read once, by neighbouring threads).
template <int DT>
__global__ __launch_bounds__(256) void k_ck_dw_thin(const void* __restrict__ dY, const int8_t* __restrict__ codes, const int8_t* __restrict__ exps,
                                                    int64_t M, int N, int K, int KG, int64_t rows_per_split, float* __restrict__ out,
                                                    float* __restrict__ db) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)N * K) return;
    const int n = (int)(i / K), k = (int)(i % K);
    const int64_t m0 = (int64_t)blockIdx.y * rows_per_split, m1 = m0 + rows_per_split < M ? m0 + rows_per_split : M;
    float a = 0.0f, b = 0.0f;
#pragma unroll 4
    for (int64_t m = m0; m < m1; ++m) {
        const float y = (float)reinterpret_cast<const typename eh_elem<DT>::type*>(dY)[m * N + n];
        a = __builtin_fmaf(y, (float)codes[m * K + k] * ck_step(exps[m * KG + (k >> 6)]), a);
        b += y;
    }
    out[(int64_t)blockIdx.y * N * K + i] = a;
    if (db && k == 0) db[(int64_t)blockIdx.y * N + n] = b;
}

// Sums of partial results, in order: LANES columns of four x STRIPS strips of partials a block; the strips meet in LDS.
template <int STRIPS, int LANES>
__device__ static inline void dw_sum(const float* __restrict__ src, int64_t len, int np, float* __restrict__ out, int64_t block, float* lds) {
    constexpr int PAD = LANES * 4 + 16;
    const int lane = threadIdx.x % LANES, strip = threadIdx.x / LANES;
    const int64_t first = block * LANES * 4, at = first + lane * 4;
    float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const int left = at < len ? (len - at < 4 ? (int)(len - at) : 4) : 0;
    if (len >= 4) {                                              // the last four columns are read whole and moved down
        const int64_t from = at + 4 <= len ? at : len - 4;
#pragma unroll 4
        for (int z = strip; z < np; z += STRIPS) {
            const eh_f32x4u v = *reinterpret_cast<const eh_f32x4u*>(src + z * len + from);
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] += v[i];
        }
        const int by = left ? (int)(at - from) : 0;
        const float a1 = a[1], a2 = a[2], a3 = a[3];
        a[0] = by == 1 ? a1 : by == 2 ? a2 : by == 3 ? a3 : a[0];
        a[1] = by == 1 ? a2 : by == 2 ? a3 : a1;
        a[2] = by == 1 ? a3 : a2;
    } else if (left) {
        for (int z = strip; z < np; z += STRIPS)
#pragma unroll
            for (int i = 0; i < 3; ++i) a[i] += src[z * len + (i < left ? i : 0)];
    }
    if (STRIPS == 1) {
        if (left == 4) *reinterpret_cast<eh_f32x4u*>(out + at) = eh_f32x4u{a[0], a[1], a[2], a[3]};
        else for (int i = 0; i < left; ++i) out[at + i] = a[i];
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) lds[strip * PAD + lane * 4 + i] = a[i];
    __syncthreads();
    const int c = threadIdx.x;
    if (c < LANES * 4 && first + c < len) {
        float v = 0.0f;
#pragma unroll
        for (int z = 0; z < STRIPS; ++z) v += lds[z * PAD + c];
        out[first + c] = v;
    }
}
// The first `blocks` blocks add the tiles, the rest db.  One strip for few partials, or where the values fill the chip
// anyway (1024 rows of 1024 x 1024 bf16, the whole gradient: 16 strips 40 us, one 30 us).
static bool dw_one_strip(int parts, int64_t n) { return parts <= 4 || (parts <= 16 && n >= (1 << 18)); }
template <int STRIPS, int LANES>
__global__ __launch_bounds__(STRIPS * LANES) void k_ck_dw_sum(const float* __restrict__ part, int64_t n, int parts, float* __restrict__ out,
                                                              const float* __restrict__ part_b, int64_t nb, int parts_b,
                                                              float* __restrict__ out_b, int blocks) {
    constexpr int LB = STRIPS * LANES / 16;
    __shared__ float lds[16 * (LB * 4 + 16)];
    if ((int)blockIdx.x < blocks) dw_sum<STRIPS, LANES>(part, n, parts, out, blockIdx.x, lds);
    else dw_sum<16, LB>(part_b, nb, parts_b, out_b, (int64_t)blockIdx.x - blocks, lds);
}

struct dw_plan { int tile, nt, kt, splits, kb; int64_t rows; };
// The tile and the splits of the rows: the chip holds one block of the larger tile a CU, two of the smaller.  The larger one
// pays where its tiles fill the chip, or each of a few has thousands of rows (tiles x 64-row pieces: 4096); below, four times
// the blocks do (4096 rows of 1024 x 1024 bf16: larger 39 us, smaller 29 us; 1024 of 2048 x 2048: 40, 33 us; 2048 of 2048 x
// 2048 fp32: 73, 74 us; 512 of 4096 x 4096 bf16: 36, 40 us).
static dw_plan dw_choose(int64_t M, int N, int K) {
    dw_plan p;
    const int64_t most = (M + 63) / 64;
    const int64_t large = (int64_t)eh_cdiv(N, 256) * eh_cdiv(K, 256);
    p.tile = N > 128 && K > 128 && large * most >= (large >= 256 ? 1024 : 4096) ? 256 : 128;
    p.nt = eh_cdiv(N, p.tile);
    p.kt = eh_cdiv(K, p.tile);
    if (N < 4 || K < 4) {                        // k_ck_dw_thin: blocks of 256 values
        p.tile = 0;
        p.nt = eh_cdiv((int64_t)N * K, 256);
        p.kt = 1;
    }
    const int64_t tiles = (int64_t)p.nt * p.kt;
    const int64_t room = p.tile == 256 ? 256 : 512;      // blocks the chip holds at once
    int64_t s = tiles >= room ? 1 : room / tiles;
    if (s > most) s = most;
    if (s < 1) s = 1;
    // Up to 128 rows one block goes over all of them and the first k-tile makes all of db: no partials, no second launch
    // (16 rows of 64 x 1000: 15 us, 12 us a call; 128 rows of 100 x 100 fp32: 9.3 us, 10.4 us on the device, 15 us, 12 us a call).
    p.kb = p.kt;
    if (M <= 128) s = p.kb = 1;
    p.rows = ((M + s - 1) / s + 63) / 64 * 64;
    if (p.rows < 64) p.rows = 64;
    p.splits = (int)((M + p.rows - 1) / p.rows);
    if (p.splits < 1) p.splits = 1;
    return p;
}

static int dw_check(int32_t dtype, int64_t M, int32_t N, int32_t K) {
    EH_CHECK_ARG(eh_dtype_ok(dtype) && M >= 0 && N >= 1 && K >= 1);
    if (N > (1 << 22) || K > (1 << 22)) return EDGEHIP_ERR_TOO_LARGE;        // offsets within 64 rows are 32 bits
    const dw_plan p = dw_choose(M, N, K);
    return eh_grid_ok((int64_t)p.nt * p.kt, 256) ? EDGEHIP_OK : EDGEHIP_ERR_TOO_LARGE;
}

static size_t dw_floats(const dw_plan& p, int N, int K, size_t& db_at) {
    db_at = p.splits > 1 ? (size_t)p.splits * N * K : 0;
    return db_at + (p.splits * p.kb > 1 ? (size_t)p.splits * p.kb * N : 0);
}

extern "C" size_t edgehip_linear8_workspace_bytes(int32_t dtype, int64_t M, int32_t N, int32_t K) {
    if (dw_check(dtype, M, N, K) != EDGEHIP_OK) return 0;
    size_t at;
    return dw_floats(dw_choose(M, N, K), N, K, at) * sizeof(float) + 16;
}

extern "C" int edgehip_linear8_bwd_weight(int32_t dtype, const void* dY, const int8_t* codes, const int8_t* exps, int64_t M, int32_t N,
                                          int32_t K, float* dW, float* db, void* ws, size_t ws_bytes, void* stream) {
    const int rc = dw_check(dtype, M, N, K);
    if (rc != EDGEHIP_OK) return rc;
    EH_CHECK_ARG(dW && (M == 0 || (dY && codes && exps)));
    if (ws_bytes < edgehip_linear8_workspace_bytes(dtype, M, N, K)) return EDGEHIP_ERR_WORKSPACE;
    const dw_plan p = dw_choose(M, N, K);
    size_t at;
    const size_t need = dw_floats(p, N, K, at);
    EH_CHECK_ARG(need == 0 || (ws && ((uintptr_t)ws & 3) == 0));
    hipStream_t s = eh_stream(stream);
    float* base = reinterpret_cast<float*>(ws);
    const bool many_b = p.splits * p.kb > 1;
    float* part = p.splits > 1 ? base : dW;
    float* pdb = !db ? nullptr : many_b ? base + at : db;
    const dim3 grid(p.nt * p.kt, p.splits), block(256);
    const int KG = (K + CK_GROUP - 1) / CK_GROUP;
#define DW_GO(DT, T) EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_ck_dw<DT, T>), grid, block, 0, s, dY, codes, exps, M, N, K, KG, p.rows, p.nt, p.kt, p.kb, part, pdb))
#define DW_THIN(DT) EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_ck_dw_thin<DT>), grid, block, 0, s, dY, codes, exps, M, N, K, KG, p.rows, part, pdb))
#define DW_TILE(DT) do { if (p.tile == 256) DW_GO(DT, 256); else if (p.tile) DW_GO(DT, 128); else DW_THIN(DT); } while (0)
    if (dtype == EDGEHIP_F32) DW_TILE(EDGEHIP_F32);
    else if (dtype == EDGEHIP_BF16) DW_TILE(EDGEHIP_BF16);
    else DW_TILE(EDGEHIP_F16);
#undef DW_TILE
#undef DW_THIN
#undef DW_GO
    EH_LAUNCH_CHECK();
    const int64_t n = (int64_t)N * K;
    const bool few = dw_one_strip(p.splits, n);
    const int blocks = p.splits > 1 ? eh_cdiv(n, few ? 1024 : 256) : 0, more = db && many_b ? eh_cdiv(N, few ? 64 : 256) : 0;
#define DW_SUM(S, L) EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_ck_dw_sum<S, L>), dim3(blocks + more), dim3(S * L), 0, s, part, n, p.splits, dW, pdb, \
                                                               (int64_t)N, p.splits * p.kb, db, blocks))
    if (blocks + more) {
        if (few) DW_SUM(1, 256);
        else DW_SUM(16, 64);
        EH_LAUNCH_CHECK();
    }
#undef DW_SUM
    return EDGEHIP_OK;
}
