// block.hip - the step between two blocks of a deep network, forward and backward in one kernel each:
//
//     u  = N_post(z)                 z: what the block put out
//     h' = res_scale h + gate u      h: the residual stream
//     y  = N_pre(h')                 what the next block reads
//
// N(x) = (x - mean) r w + b with r = 1 / sqrt(mean((x - mean)^2) + eps); the root-mean-square kind has mean = 0.
// With xhat = (x - mean) r and t = dN w:   dx = r (t - mean(t) - xhat mean(t xhat)),   dw = sum over rows of dN xhat,
// db = sum of dN (the root-mean-square kind drops mean(t)).  Hence, with t_pre = dy w_pre:
//     D  = dh' + N_pre^T(dy),  dh = res_scale D,  dgate = D u (summed as the gate was spread),  dz = N_post^T(gate D).
//
// Bound by HBM: 14 flops a value forward, 26 backward.  Everything between the reads of h, z (dh', dy) and the writes
// of h', y (dh, dz) stays in registers: a thread owns 8 columns of a row (one 16-byte access of a 16-bit type), the
// threads of a row meet in a wave reduction (and, where it has more than 64, in LDS).  16384 x 4096 bf16: forward 104 us,
// 5.2 TB/s, backward 177 us, 4.5 TB/s (+ 7 us for the partials), against 5.1 TB/s of a large copy; 78208 x 64 fp32 with a
// gate per graph: 21 us and 32 us (3.8 TB/s), there the start and end of the launches tell.  The backward pass recomputes u, h' from
// h and z instead of reading a kept h': the same bytes, and the gradient is that of the unrounded h'.  y, too, is made
// from the unrounded h'.  All statistics and sums are fp32; each output is rounded once.
//
// Sums over rows (dw, db, dgate): a block owns a run of consecutive rows and its threads keep the sums of their columns
// in registers over all of them, so a column costs one partial per block instead of an atomic per row; a second kernel
// adds the partials in block order.  No atomics: results do not depend on the order blocks run in.  A gate per group of
// rows flushes at every group border; the pair (block c, group g) owns partial c + g: along the rows one of the two
// grows by one at each border, so no two pairs share a slot, and nblocks + groups slots are enough.
#include "common.h"
#include "prof.h"
#include "vec.h"

#define GN_MAX_DIM 8192

struct gn_args {
    const void *h, *z, *dho, *dy;
    void *ho, *y, *dh, *dz, *dgate;
    float* stats;               // [rows][4]: mean and r of z, mean and r of h'
    const float* stats_in;
    const void *w_pre, *b_pre, *w_post, *b_post;
    const void* gate;
    const int32_t* row_ptr;
    float* part;                // [5][nblk][D]: dw_pre, db_pre, dw_post, db_post, dgate (a gate that is one vector)
    float* gpart;               // [nblk + groups][D]
    int64_t rows;
    int rows_per_block, nblk, D, pre, post, wdt, gkind, gdt, groups;
    float alpha, eps, inv_d;
    int want_pre, want_post, want_gate;
};

// TPR threads a row: 8, 16, 32 or 64 (several rows a block of 256), or GN_ROW: the whole block, whole waves of it, as many
// as the row has pieces of 512 columns.
#define GN_ROW 1024
#define GN_WIDE 512                      // blocks up to this size have their own kernels: twice the registers a thread
#define GN_THREADS(TPR) ((TPR) <= 64 ? 256 : (TPR))

template <int CTRL> __device__ static inline float gn_add_dpp(float v) {
    return v + __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xF, 0xF, true));
}
// sum over the threads of a row, in every one of them.  Within 16 lanes by lane exchanges of the vector unit (pairs, quads,
// mirrored halves); the four sums of 16 by the scalar unit's reads.  The waves of a row meet in LDS, two buffers in turn (a
// wave can only write the buffer of sum k + 2 after every wave has passed the barrier of k + 1, that is after it has read
// that of k); the barrier waits for LDS only: the next row's requests stay in flight.
template <int TPR, int NV>
__device__ static inline void gn_row_sum(float (&v)[NV], float* lds, int& turn) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        v[i] = gn_add_dpp<0xB1>(v[i]);                           // quad_perm [1,0,3,2]
        v[i] = gn_add_dpp<0x4E>(v[i]);                           // quad_perm [2,3,0,1]
        v[i] = gn_add_dpp<0x141>(v[i]);                          // row_half_mirror
        if (TPR >= 16) v[i] = gn_add_dpp<0x140>(v[i]);           // row_mirror
        if (TPR == 32) v[i] += __shfl_xor(v[i], 16, 64);
        if (TPR >= 64) {
            const int b = (int)__float_as_uint(v[i]);
            const float s0 = __uint_as_float((unsigned)__builtin_amdgcn_readlane(b, 0)), s1 = __uint_as_float((unsigned)__builtin_amdgcn_readlane(b, 16));
            const float s2 = __uint_as_float((unsigned)__builtin_amdgcn_readlane(b, 32)), s3 = __uint_as_float((unsigned)__builtin_amdgcn_readlane(b, 48));
            v[i] = (s0 + s1) + (s2 + s3);
        }
    }
    if (TPR > 64) {
        const int waves = blockDim.x >> 6;
        float* b = lds + turn * 32;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) b[(threadIdx.x >> 6) * 2 + i] = v[i];
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = 0.0f;
        for (int w = 0; w < waves; ++w) {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] += b[w * 2 + i];
        }
    }
}

// first group whose end lies behind `row` (groups may be empty); `groups` where the row lies behind the last one
__device__ static inline int gn_group_of(const int32_t* __restrict__ row_ptr, int groups, int64_t row) {
    int lo = 0, hi = groups;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if ((int64_t)row_ptr[mid + 1] <= row) lo = mid + 1; else hi = mid;
    }
    return lo;
}

template <bool LAYER, int TPR>
__device__ static inline void gn_stats(const float (&x)[8], int n, float inv_d, float eps, float& mean, float& r, float* lds, int& turn) {
    float s[1];
    mean = 0.0f;
    if (LAYER) {
        s[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s[0] += x[i];
        gn_row_sum<TPR, 1>(s, lds, turn);
        mean = s[0] * inv_d;
    }
    s[0] = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float c = i < n ? x[i] - mean : 0.0f;
        s[0] += c * c;
    }
    gn_row_sum<TPR, 1>(s, lds, turn);
    r = 1.0f / sqrtf(s[0] * inv_d + eps);
}

// the gate of a row
template <int DZ, bool TINY>
__device__ static inline void gn_row_gate(const gn_args& A, const eh_at& at, float (&g)[8]) {
    if constexpr (DZ == EDGEHIP_F32) {
        eh_raw8<EDGEHIP_F32> r;
        eh_get<EDGEHIP_F32, TINY>(r, A.gate, at);
        r.get(g);
    } else {
        eh_raw8<EDGEHIP_F32> r;
        eh_raw8<DZ> q;
        float o[8];
        const bool wide = A.gdt == EDGEHIP_F32;
        if (wide) eh_get<EDGEHIP_F32, TINY>(r, A.gate, at);
        else eh_get<DZ, TINY>(q, A.gate, at);
        r.get(g);
        q.get(o);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = wide ? +g[i] : +o[i];
    }
    eh_own<TINY>(g, at.n, at.back);
}

// what a thread slot reads of its row
template <int DH, int DZ> struct gn_in {
    eh_raw8<DZ> z;
    eh_raw8<DH> h;
};

template <int DH, int DZ, bool LAYER, int TPR, bool TINY = false>
__global__ __launch_bounds__(GN_THREADS(TPR)) void k_gn_fwd(gn_args A) {
    constexpr int RPB = TPR <= 64 ? 256 / TPR : 1;
    __shared__ float lds[64];
    int turn = 0;
    const int slot = TPR <= 64 ? threadIdx.x / TPR : 0, t = TPR <= 64 ? threadIdx.x % TPR : threadIdx.x, col = t * 8, n = A.D - col;
    float wpre[8], wpost[8], bpre[8], bpost[8], g[8];
    const int np = n < 0 ? 0 : n;
    eh_load8_any(A.w_pre, A.wdt, col, A.w_pre ? np : 0, wpre, 1.0f);
    eh_load8_any(A.w_post, A.wdt, col, A.w_post ? np : 0, wpost, 1.0f);
    if (LAYER) {
        eh_load8_any(A.b_pre, A.wdt, col, A.b_pre ? np : 0, bpre, 0.0f);
        eh_load8_any(A.b_post, A.wdt, col, A.b_post ? np : 0, bpost, 0.0f);
    }
    eh_load8_any(A.gate, A.gdt, col, A.gkind == EDGEHIP_GATE_VECTOR ? np : 0, g, 1.0f);
    const int64_t end = A.rows * A.D, r0 = (int64_t)blockIdx.x * A.rows_per_block;
    const int64_t r1 = r0 + A.rows_per_block < A.rows ? r0 + A.rows_per_block : A.rows;
    int grp = A.gkind == EDGEHIP_GATE_GROUP ? gn_group_of(A.row_ptr, A.groups, r0) : 0, held = -1;
    auto request = [&](gn_in<DH, DZ>& in, int64_t row) {
        const eh_at at = eh_place(row * A.D + col, row < r1 ? n : 0, end);
        eh_get<DZ, TINY>(in.z, A.z, at);
        eh_get<DH, TINY>(in.h, A.h, at);
    };
    gn_in<DH, DZ> next;
    request(next, r0 + slot);
    for (int64_t base = r0; base < r1; base += RPB) {
        const int64_t row = base + slot;
        const bool live = row < r1;
        const eh_at at = eh_place(row * A.D + col, live ? n : 0, end);
        float z[8], h[8];
        if (A.gkind == EDGEHIP_GATE_ROW) gn_row_gate<DZ, TINY>(A, at, g);
        next.z.get(z);
        next.h.get(h);
        eh_own<TINY>(z, at.n, at.back);
        eh_own<TINY>(h, at.n, at.back);
        request(next, row + RPB);                                // a row ahead
        if (A.gkind == EDGEHIP_GATE_GROUP && live) {
            while (grp < A.groups && (int64_t)A.row_ptr[grp + 1] <= row) ++grp;
            if (grp != held) {
                held = grp;
                eh_load8_any(A.gate, A.gdt, (int64_t)grp * A.D + col, grp < A.groups ? np : 0, g, 0.0f);
            }
        }
        float mz = 0.0f, rz = 1.0f, mh = 0.0f, rh = 1.0f;
        if (A.post) {
            gn_stats<LAYER, TPR>(z, n, A.inv_d, A.eps, mz, rz, lds, turn);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                z[i] = (z[i] - mz) * rz * wpost[i];
                if (LAYER) z[i] += bpost[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = A.alpha * h[i] + g[i] * z[i];
        if (live) eh_store8<DH>(A.ho, row * A.D + col, n, h);
        if (A.pre) {
            if (n < 8) {
#pragma unroll
                for (int i = 0; i < 8; ++i) if (i >= n) h[i] = 0.0f;
            }
            gn_stats<LAYER, TPR>(h, n, A.inv_d, A.eps, mh, rh, lds, turn);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                h[i] = (h[i] - mh) * rh * wpre[i];
                if (LAYER) h[i] += bpre[i];
            }
            if (live) eh_store8<DZ>(A.y, row * A.D + col, n, h);
        }
        if (A.stats && live && t == 0) *reinterpret_cast<float4*>(A.stats + row * 4) = make_float4(mz, rz, mh, rh);
    }
}

// column sums of the block's row slots -> one partial row
template <int TPR>
__device__ static inline void gn_flush(float (&acc)[8], float* lds, float* dst, int D, int slot, int t) {
    constexpr int RPB = TPR <= 64 ? 256 / TPR : 1;
    const int col = t * 8;
    if (RPB > 1) {
        // slots in turn through LDS: [RPB][TPR * 8] floats, 8 KiB
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) lds[(slot * 8 + i) * TPR + t] = acc[i];
        __syncthreads();
        for (int c = threadIdx.x; c < TPR * 8; c += 256) {
            const int i = c / TPR, tt = c % TPR;
            float s = 0.0f;
#pragma unroll 8
            for (int k = 0; k < RPB; ++k) s += lds[(k * 8 + i) * TPR + tt];
            if (tt * 8 + i < D) dst[tt * 8 + i] = s;
        }
    } else {
        eh_store8<EDGEHIP_F32>(dst, col, D - col, acc);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
}

// The backward kernel needs the norms' weights three times a row; in registers they (and b_post) would cost 24 a thread
// and with them half of the waves a CU holds.  They stand in LDS instead, as fp32: [vector][half of a thread's
// eight][thread][4].
template <int TPR>
__device__ static inline void gn_par_put(float* par, int t, const float (&v)[8]) {
    const int T = TPR <= 64 ? TPR : blockDim.x;
    *reinterpret_cast<float4*>(par + t * 4) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(par + (T + t) * 4) = make_float4(v[4], v[5], v[6], v[7]);
}
template <int TPR>
__device__ static inline void gn_par_get(const float* par, int vec, int t, float (&v)[8]) {
    const int T = TPR <= 64 ? TPR : blockDim.x;
    const float4 a = *reinterpret_cast<const float4*>(par + (vec * 2 * T + t) * 4), b = *reinterpret_cast<const float4*>(par + ((vec * 2 + 1) * T + t) * 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

template <int DH, int DZ> struct gn_grad {
    eh_raw8<DZ> z, dy;
    eh_raw8<DH> h, d;
    float4 st;
};

// Waves a SIMD the registers are cut to: four (128 registers) with a 16-bit stream, three with fp32 (blocks of 1024 threads: four).
// At four, up to 64 threads a row, the mean-and-variance kind spills 50-53 registers, the other kind 5-7; a row of whole waves spills
// none, and with an fp32 stream takes 105-128, so that four waves fit there too.
#define GN_BWD_WAVES(DH) ((DH) == EDGEHIP_F32 ? 3 : 4)
template <int DH, int DZ, bool LAYER, int TPR, bool TINY = false>
__global__ __launch_bounds__(GN_THREADS(TPR), (TPR == GN_ROW ? 4 : GN_BWD_WAVES(DH))) void k_gn_bwd(gn_args A) {
    constexpr int RPB = TPR <= 64 ? 256 / TPR : 1;
    constexpr bool AHEAD = DH != EDGEHIP_F32 && TPR > 64 && !LAYER;   // requests a row ahead, where they fit the registers
    extern __shared__ float par[];
    __shared__ float lds[64];
    __shared__ float fl[RPB > 1 ? 256 * 8 : 1];
    int turn = 0;
    const int slot = TPR <= 64 ? threadIdx.x / TPR : 0, t = TPR <= 64 ? threadIdx.x % TPR : threadIdx.x, col = t * 8, n = A.D - col;
    // (gradients that are not given: any tensor of their shape, cleared when it is taken)
    const void* const dho = A.dho ? A.dho : A.h;
    const void* const dyp = A.dy ? A.dy : A.z;
    const bool has_dy = A.dy && A.pre;
    const int np = n < 0 ? 0 : n;
    float g[8];
    if (slot == 0) {
        const int T = TPR <= 64 ? TPR : blockDim.x;
        float v[8];
        eh_load8_any(A.w_pre, A.wdt, col, A.w_pre ? np : 0, v, 1.0f);
        gn_par_put<TPR>(par, t, v);
        eh_load8_any(A.w_post, A.wdt, col, A.w_post ? np : 0, v, 1.0f);
        gn_par_put<TPR>(par + 8 * T, t, v);
        if (LAYER) {
            eh_load8_any(A.b_post, A.wdt, col, A.b_post ? np : 0, v, 0.0f);
            gn_par_put<TPR>(par + 16 * T, t, v);
        }
    }
    __syncthreads();
    eh_load8_any(A.gate, A.gdt, col, A.gkind == EDGEHIP_GATE_VECTOR ? np : 0, g, 1.0f);
    float awpre[8], awpost[8], abpre[8], abpost[8], ag[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { awpre[i] = awpost[i] = abpre[i] = abpost[i] = ag[i] = 0.0f; }
    const int64_t end = A.rows * A.D, r0 = (int64_t)blockIdx.x * A.rows_per_block;
    const int64_t r1 = r0 + A.rows_per_block < A.rows ? r0 + A.rows_per_block : A.rows;
    int grp = A.gkind == EDGEHIP_GATE_GROUP ? gn_group_of(A.row_ptr, A.groups, r0) : 0;
    // u = zhat w_post + b_post
    auto get_u = [&](const float (&z)[8], float (&u)[8]) {
        if (!A.post) {
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = z[i];
            return;
        }
        float w[8], b[8];
        gn_par_get<TPR>(par, 1, t, w);
        if (LAYER) gn_par_get<TPR>(par, 2, t, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = LAYER ? z[i] * w[i] + b[i] : z[i] * w[i];
    };
    for (int64_t s0 = r0; s0 < r1;) {
        // rows of one group (all rows where the gate is not per group)
        int64_t s1 = r1;
        if (A.gkind == EDGEHIP_GATE_GROUP) {
            while (grp < A.groups && (int64_t)A.row_ptr[grp + 1] <= s0) ++grp;
            if (grp < A.groups && (int64_t)A.row_ptr[grp + 1] < r1) s1 = A.row_ptr[grp + 1];
            eh_load8_any(A.gate, A.gdt, (int64_t)grp * A.D + col, grp < A.groups ? np : 0, g, 0.0f);
        }
        gn_grad<DH, DZ> in;
        auto request = [&](int64_t row) {
            const eh_at at = eh_place(row * A.D + col, row < s1 ? n : 0, end);
            eh_get<DZ, TINY>(in.z, A.z, at);
            eh_get<DH, TINY>(in.h, A.h, at);
            eh_get<DH, TINY>(in.d, dho, at);
            eh_get<DZ, TINY>(in.dy, dyp, at);
            in.st = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (row < s1) in.st = *reinterpret_cast<const float4*>(A.stats_in + row * 4);
        };
        if (AHEAD) request(s0 + slot);
        for (int64_t base = s0; base < s1; base += RPB) {
            const int64_t row = base + slot;
            const bool live = row < s1;
            const int64_t off = row * A.D + col;
            const eh_at at = eh_place(off, live ? n : 0, end);
            float z[8], h[8], d[8], dy[8], w[8];
            if (!AHEAD) request(row);
            if (A.gkind == EDGEHIP_GATE_ROW) gn_row_gate<DZ, TINY>(A, at, g);
            in.z.get(z);
            in.h.get(h);
            in.d.get(d);
            in.dy.get(dy);
            eh_own<TINY>(z, at.n, at.back);
            eh_own<TINY>(h, at.n, at.back);
            eh_own<TINY>(d, A.dho ? at.n : 0, at.back);
            eh_own<TINY>(dy, has_dy ? at.n : 0, at.back);
            const float4 st = in.st;
            if (AHEAD) request(row + RPB);
            if (A.post) {
#pragma unroll
                for (int i = 0; i < 8; ++i) z[i] = (z[i] - st.x) * st.y;          // zhat
            }
            if (A.pre) {
                float u[8];
                get_u(z, u);
                gn_par_get<TPR>(par, 0, t, w);
                float c[2] = {0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    h[i] = (A.alpha * h[i] + g[i] * u[i] - st.z) * st.w;         // hhat
                    awpre[i] += dy[i] * h[i];
                    if (LAYER) abpre[i] += dy[i];
                    dy[i] *= w[i];
                    c[0] += i < n ? dy[i] * h[i] : 0.0f;
                    if (LAYER) c[1] += dy[i];
                }
                gn_row_sum<TPR, LAYER ? 2 : 1>(reinterpret_cast<float (&)[LAYER ? 2 : 1]>(c), lds, turn);
                asm volatile("" ::: "memory");                                   // the weights are read again below, not held
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] += st.w * (dy[i] - h[i] * (c[0] * A.inv_d) - (LAYER ? c[1] * A.inv_d : 0.0f));
            }
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = A.alpha * d[i];
            if (live) eh_store8<DH>(A.dh, off, n, o);
            if (A.want_gate) {
                get_u(z, o);
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = live && i < n ? d[i] * o[i] : 0.0f;
                if (A.gkind == EDGEHIP_GATE_ROW) {
                    if (live) {
                        if (DZ == EDGEHIP_F32 || A.gdt == EDGEHIP_F32) eh_store8<EDGEHIP_F32>(A.dgate, off, n, o);
                        else eh_store8<DZ>(A.dgate, off, n, o);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) ag[i] += o[i];
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = live && i < n ? d[i] * g[i] : 0.0f;      // du
            if (A.post) {
                float c[2] = {0.0f, 0.0f};
                gn_par_get<TPR>(par, 1, t, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    awpost[i] += d[i] * z[i];
                    if (LAYER) abpost[i] += d[i];
                    d[i] *= w[i];
                    c[0] += d[i] * z[i];
                    if (LAYER) c[1] += d[i];
                }
                gn_row_sum<TPR, LAYER ? 2 : 1>(reinterpret_cast<float (&)[LAYER ? 2 : 1]>(c), lds, turn);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] = st.y * (d[i] - z[i] * (c[0] * A.inv_d) - (LAYER ? c[1] * A.inv_d : 0.0f));
            }
            if (live) eh_store8<DZ>(A.dz, off, n, d);
        }
        if (A.gkind == EDGEHIP_GATE_GROUP && A.want_gate) {
            if (grp < A.groups) {
                gn_flush<TPR>(ag, fl, A.gpart + ((int64_t)blockIdx.x + grp) * A.D, A.D, slot, t);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) ag[i] = 0.0f;
            }
        }
        s0 = s1;
    }
    const int64_t plane = (int64_t)A.nblk * A.D;
    float* p = A.part + (int64_t)blockIdx.x * A.D;
    if (A.want_pre) {
        gn_flush<TPR>(awpre, fl, p, A.D, slot, t);
        if (LAYER) gn_flush<TPR>(abpre, fl, p + plane, A.D, slot, t);
    }
    if (A.want_post) {
        gn_flush<TPR>(awpost, fl, p + 2 * plane, A.D, slot, t);
        if (LAYER) gn_flush<TPR>(abpost, fl, p + 3 * plane, A.D, slot, t);
    }
    if (A.gkind == EDGEHIP_GATE_VECTOR && A.want_gate) gn_flush<TPR>(ag, fl, p + 4 * plane, A.D, slot, t);
}

// partials -> sums, in block order.  blockIdx.x: which vector, then which group of the gate; 32 columns x 32 strips
struct gn_red {
    const float *part, *gpart;
    int64_t plane;
    int nblk, D, rows_per_block, vectors;
    int64_t rows;
    void *out[5], *dgate;
    int dt[5], gdt;
    const int32_t* row_ptr;
};
__global__ __launch_bounds__(1024) void k_gn_reduce(gn_red R) {
    __shared__ float s[32][33];
    const int c = threadIdx.x & 31, strip = threadIdx.x >> 5, col = blockIdx.y * 32 + c, v = blockIdx.x, g = v - R.vectors;
    int64_t b0 = 0, b1 = R.nblk;
    const float* src;
    void* out;
    int dt;
    int64_t at = col;
    if (g >= 0) {
        int64_t a = R.row_ptr[g], b = R.row_ptr[g + 1];
        if (a < 0) a = 0;
        if (b > R.rows) b = R.rows;
        b0 = a / R.rows_per_block;
        b1 = a < b ? (b - 1) / R.rows_per_block + 1 : b0;
        src = R.gpart + (int64_t)g * R.D;                      // partial of (block, group): row block + group
        out = R.dgate; dt = R.gdt;
        at += (int64_t)g * R.D;
    } else {
        out = R.out[v]; dt = R.dt[v];
        if (!out) return;
        src = R.part + v * R.plane;
    }
    float a = 0.0f;
    if (col < R.D) {
#pragma unroll 8
        for (int64_t b = b0 + strip; b < b1; b += 32) a += src[b * R.D + col];
    }
    s[strip][c] = a;
    __syncthreads();
    if (strip == 0 && col < R.D) {
#pragma unroll
        for (int i = 1; i < 32; ++i) a += s[i][c];
        eh_store1_any(out, dt, at, a);
    }
}

// threads of a row (see GN_ROW): 8 columns each
static int gn_tpr(int D) {
    if (D > GN_WIDE * 8) return GN_ROW;
    if (D > 512) return GN_WIDE;
    int t = 8;
    while (t * 8 < D) t *= 2;
    return t;
}
static size_t gn_par_bytes(int D, bool layer) { return (size_t)(D <= 512 ? gn_tpr(D) : (D + 511) / 512 * 64) * 8 * sizeof(float) * (layer ? 3 : 2); }
static int gn_threads(int D) { return D <= 512 ? 256 : (D + 511) / 512 * 64; }
// Rows a block owns.  Backward: no more blocks than GN_BWD_WAVES waves a SIMD make, whole blocks a CU; more of them add partials
// (5 D floats a block at most) and a second, partly filled round.  (With an fp32 stream and rows of whole waves a fourth wave a
// SIMD would fit; 7 or 8 waves a block, of 12 that are counted on, are one block a CU.)  Forward, no partials: two rounds of blocks, four where a block is one row
// (16384 x 4096 bf16: 1024 blocks 110 us, 2048 96 us), but four rows a block where there are enough of them, as a block
// reads the parameters once (5003 x 1101: one row a block 38 us, four 33 us).
static int gn_rows_per_block(int64_t rows, int D, int stream_dtype, int bwd) {
    const int rpb = D <= 512 ? 256 / gn_tpr(D) : 1, waves = gn_threads(D) / 64;
    const int simd = D > GN_WIDE * 8 ? 4 : GN_BWD_WAVES(stream_dtype);
    const int64_t target = (int64_t)256 * (4 * simd / waves) * (bwd ? 1 : D <= 512 ? 2 : 4);
    int64_t per = (rows + target - 1) / target;
    if (!bwd && D > 512 && per < 4) per = rows >= 4096 ? 4 : rows >= 2048 ? 2 : per;
    per = (per + rpb - 1) / rpb * rpb;
    return (int)(per < rpb ? rpb : per);
}

static int gn_check(const edgehip_gate_norm* G) {
    EH_CHECK_ARG(G && G->rows >= 0 && G->dim >= 1);
    EH_CHECK_ARG(eh_dtype_ok(G->stream_dtype) && eh_dtype_ok(G->branch_dtype));
    if (G->stream_dtype != G->branch_dtype && G->stream_dtype != EDGEHIP_F32) return EDGEHIP_ERR_UNSUPPORTED;
    EH_CHECK_ARG(G->kind == EDGEHIP_NORM_RMS || G->kind == EDGEHIP_NORM_LAYER);
    EH_CHECK_ARG(G->kind == EDGEHIP_NORM_LAYER || (!G->b_pre && !G->b_post));
    EH_CHECK_ARG(G->param_dtype == EDGEHIP_F32 || G->param_dtype == G->branch_dtype);
    EH_CHECK_ARG(G->gate_kind >= EDGEHIP_GATE_NONE && G->gate_kind <= EDGEHIP_GATE_ROW);
    EH_CHECK_ARG((G->gate_kind == EDGEHIP_GATE_NONE) == (G->gate == nullptr));
    EH_CHECK_ARG(G->gate_kind == EDGEHIP_GATE_NONE || G->gate_dtype == EDGEHIP_F32 || G->gate_dtype == G->branch_dtype);
    EH_CHECK_ARG(G->gate_kind != EDGEHIP_GATE_GROUP || (G->row_ptr && G->groups >= 1));
    if (G->dim > GN_MAX_DIM) return EDGEHIP_ERR_UNSUPPORTED;
    if (G->rows > ((int64_t)1 << 31) - 1 || (G->gate_kind == EDGEHIP_GATE_GROUP && G->groups > 65535)) return EDGEHIP_ERR_TOO_LARGE;
    return EDGEHIP_OK;
}

static gn_args gn_fill(const edgehip_gate_norm* G) {
    gn_args A = {};
    A.w_pre = G->w_pre; A.b_pre = G->b_pre; A.w_post = G->w_post; A.b_post = G->b_post;
    A.gate = G->gate; A.row_ptr = G->row_ptr;
    A.rows = G->rows; A.D = G->dim; A.pre = G->pre != 0; A.post = G->post != 0; A.wdt = G->param_dtype;
    A.gkind = G->gate_kind; A.gdt = G->gate_dtype; A.groups = G->groups;
    A.alpha = G->res_scale; A.eps = G->eps; A.inv_d = 1.0f / (float)G->dim;
    return A;
}

template <int DH, int DZ, bool LAYER>
static int gn_launch(const gn_args& A, int nblk, bool bwd, hipStream_t s) {
    const dim3 block(gn_threads(A.D));
    if (A.rows * A.D < 8) {
        if (bwd) EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_gn_bwd<DH, DZ, LAYER, 8, true>), dim3(nblk), block, gn_par_bytes(A.D, LAYER), s, A));
        else EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_gn_fwd<DH, DZ, LAYER, 8, true>), dim3(nblk), block, 0, s, A));
        EH_LAUNCH_CHECK();
        return EDGEHIP_OK;
    }
    switch (gn_tpr(A.D)) {
#define GN_CASE(T) case T: \
        if (bwd) EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_gn_bwd<DH, DZ, LAYER, T>), dim3(nblk), block, gn_par_bytes(A.D, LAYER), s, A)); \
        else EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL((k_gn_fwd<DH, DZ, LAYER, T>), dim3(nblk), block, 0, s, A)); \
        break;
        GN_CASE(8) GN_CASE(16) GN_CASE(32) GN_CASE(64) GN_CASE(GN_WIDE) GN_CASE(GN_ROW)
#undef GN_CASE
        default: return EDGEHIP_ERR_UNSUPPORTED;
    }
    EH_LAUNCH_CHECK();
    return EDGEHIP_OK;
}
static int gn_dispatch(const edgehip_gate_norm* G, const gn_args& A, int nblk, bool bwd, hipStream_t s) {
    const int key = G->stream_dtype * 4 + G->branch_dtype;
    const bool layer = G->kind == EDGEHIP_NORM_LAYER;
    switch (key) {
#define GN_TYPES(H, Z) case (H) * 4 + (Z): return layer ? gn_launch<H, Z, true>(A, nblk, bwd, s) : gn_launch<H, Z, false>(A, nblk, bwd, s);
        GN_TYPES(EDGEHIP_F32, EDGEHIP_F32)
        GN_TYPES(EDGEHIP_BF16, EDGEHIP_BF16)
        GN_TYPES(EDGEHIP_F16, EDGEHIP_F16)
        GN_TYPES(EDGEHIP_F32, EDGEHIP_BF16)
        GN_TYPES(EDGEHIP_F32, EDGEHIP_F16)
#undef GN_TYPES
    }
    return EDGEHIP_ERR_UNSUPPORTED;
}

extern "C" int edgehip_gate_norm_fwd(const edgehip_gate_norm* G, const void* h, const void* z, void* h_out, void* y,
                                     float* stats, void* stream) {
    const int rc = gn_check(G);
    if (rc != EDGEHIP_OK) return rc;
    if (G->rows == 0) return EDGEHIP_OK;
    EH_CHECK_ARG(h && z && h_out && (!G->pre || y) && ((uintptr_t)stats & 15) == 0);
    gn_args A = gn_fill(G);
    A.h = h; A.z = z; A.ho = h_out; A.y = y; A.stats = stats;
    A.rows_per_block = gn_rows_per_block(G->rows, G->dim, G->stream_dtype, 0);
    return gn_dispatch(G, A, eh_cdiv(G->rows, A.rows_per_block), false, eh_stream(stream));
}

static int gn_blocks(const edgehip_gate_norm* G) { return eh_cdiv(G->rows, gn_rows_per_block(G->rows, G->dim, G->stream_dtype, 1)); }

extern "C" size_t edgehip_gate_norm_workspace_bytes(const edgehip_gate_norm* G) {
    if (gn_check(G) != EDGEHIP_OK) return 0;
    const size_t nblk = (size_t)gn_blocks(G);
    size_t rows = 5 * nblk;
    if (G->gate_kind == EDGEHIP_GATE_GROUP) rows += nblk + (size_t)G->groups;
    return (rows * (size_t)G->dim + 4) * sizeof(float);
}

extern "C" int edgehip_gate_norm_bwd(const edgehip_gate_norm* G, const void* dh_out, const void* dy, const void* h, const void* z,
                                     const float* stats, void* dh, void* dz, void* dgate, void* dw_pre, void* db_pre,
                                     void* dw_post, void* db_post, void* ws, size_t ws_bytes, void* stream) {
    const int rc = gn_check(G);
    if (rc != EDGEHIP_OK) return rc;
    const bool layer = G->kind == EDGEHIP_NORM_LAYER;
    EH_CHECK_ARG(layer || (!db_pre && !db_post));
    EH_CHECK_ARG((G->pre || (!dw_pre && !db_pre)) && (G->post || (!dw_post && !db_post)));
    EH_CHECK_ARG(!dgate || G->gate_kind != EDGEHIP_GATE_NONE);
    EH_CHECK_ARG(G->rows == 0 || (h && z && stats && dh && dz));
    EH_CHECK_ARG(((uintptr_t)stats & 15) == 0);
    if (ws_bytes < edgehip_gate_norm_workspace_bytes(G)) return EDGEHIP_ERR_WORKSPACE;
    EH_CHECK_ARG(ws && ((uintptr_t)ws & 15) == 0);
    hipStream_t s = eh_stream(stream);
    gn_args A = gn_fill(G);
    A.h = h; A.z = z; A.dho = dh_out; A.dy = dy; A.dh = dh; A.dz = dz; A.dgate = dgate; A.stats_in = stats;
    A.rows_per_block = gn_rows_per_block(G->rows, G->dim, G->stream_dtype, 1);
    A.nblk = gn_blocks(G);
    A.part = reinterpret_cast<float*>(ws);
    A.gpart = A.part + (size_t)5 * A.nblk * A.D;
    A.want_pre = dw_pre || db_pre;
    A.want_post = dw_post || db_post;
    A.want_gate = dgate != nullptr;
    if (A.nblk) {
        const int rl = gn_dispatch(G, A, A.nblk, true, s);
        if (rl != EDGEHIP_OK) return rl;
    }
    gn_red R = {};
    R.part = A.part; R.plane = (int64_t)A.nblk * A.D; R.nblk = A.nblk; R.D = A.D; R.rows = G->rows; R.rows_per_block = A.rows_per_block;
    void* outs[5] = {dw_pre, db_pre, dw_post, db_post, G->gate_kind == EDGEHIP_GATE_VECTOR ? dgate : nullptr};
    for (int i = 0; i < 5; ++i) { R.out[i] = outs[i]; R.dt[i] = i < 4 ? G->param_dtype : G->gate_dtype; }
    R.vectors = outs[0] || outs[1] || outs[2] || outs[3] || outs[4] ? 5 : 0;
    R.gpart = A.gpart; R.row_ptr = G->row_ptr; R.dgate = dgate; R.gdt = G->gate_dtype;
    const int sums = R.vectors + (G->gate_kind == EDGEHIP_GATE_GROUP && dgate ? G->groups : 0);
    if (sums) {
        EH_PROF(EH_K_TRAIN, s, hipLaunchKernelGGL(k_gn_reduce, dim3(sums, eh_cdiv(A.D, 32)), dim3(1024), 0, s, R));
        EH_LAUNCH_CHECK();
    }
    return EDGEHIP_OK;
}
