// vec.h - eight consecutive values of a fp32 / bf16 / fp16 row, at any alignment, as fp32 registers.
//
// gfx950 takes 16-byte global accesses at any element-aligned address, so a row of odd length or a view that starts in
// the middle of a line is read with the same vector accesses as an aligned one: the vector types below only promise the
// alignment of their element.  What a row's last vector does with the values it lacks: eh_place, or eh_load8 value by value.
#pragma once
#include "common.h"

template <int DT> struct eh_elem;
template <> struct eh_elem<EDGEHIP_F32> { typedef float type; };
template <> struct eh_elem<EDGEHIP_BF16> { typedef __bf16 type; };
template <> struct eh_elem<EDGEHIP_F16> { typedef _Float16 type; };

typedef float eh_f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned int eh_u32x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int eh_u32x2u __attribute__((ext_vector_type(2), aligned(1)));
typedef unsigned int eh_u32x2h __attribute__((ext_vector_type(2), aligned(2)));

// whether a launch takes that many threads along x (its size is a 32-bit number of threads)
static inline int eh_grid_ok(int64_t blocks, int64_t threads) { return blocks < ((int64_t)1 << 32) / threads; }
static inline int eh_dtype_ok(int dt) { return dt == EDGEHIP_F32 || dt == EDGEHIP_BF16 || dt == EDGEHIP_F16; }

// eight raw values as they stand in memory (4 or 8 registers)
template <int DT> struct eh_raw8 {
    eh_u32x4u v;
    __device__ inline void load(const void* p) { v = *reinterpret_cast<const eh_u32x4u*>(p); }
    __device__ inline void get(float (&o)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (DT == EDGEHIP_BF16) {
                o[2 * i] = __uint_as_float(v[i] << 16);
                o[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
            } else {
                o[2 * i] = (float)__builtin_bit_cast(_Float16, (unsigned short)(v[i] & 0xffffu));
                o[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (unsigned short)(v[i] >> 16));
            }
        }
    }
};
template <> struct eh_raw8<EDGEHIP_F32> {
    eh_f32x4u a, b;
    __device__ inline void load(const void* p) {
        a = *reinterpret_cast<const eh_f32x4u*>(p);
        b = *(reinterpret_cast<const eh_f32x4u*>(p) + 1);
    }
    __device__ inline void get(float (&o)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) { o[i] = a[i]; o[4 + i] = b[i]; }
    }
};

// Where a thread's eight values of a row are read, without a branch and without looking at them while the request is in
// flight: a row's last, partial vector is read whole, into the next row; at the very end of the tensor it is read `back`
// values earlier; a thread without values (n <= 0) reads whatever its clamped place holds.  eh_own puts that right: values
// are moved down by `back`, what is not the row's own becomes 0.  The tensor has at least eight values (TINY kernels
// take smaller ones, value by value).
struct eh_at { int64_t off; int n, back; };
__device__ static inline eh_at eh_place(int64_t off, int n, int64_t end) {
    const int64_t o = off + 8 <= end ? off : end - 8;
    return eh_at{o, n > 8 ? 8 : n, n > 0 ? (int)(off - o) : 0};
}
template <int DT, bool TINY>
__device__ static inline void eh_get(eh_raw8<DT>& r, const void* base, const eh_at& a) {
    typedef typename eh_elem<DT>::type T;
    const T* p = reinterpret_cast<const T*>(base);
    if (!TINY) {
        r.load(p + a.off);
    } else {                                                     // (off is below 0 by 8 - end there, back as much larger)
        T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < a.n ? p[a.off + a.back + i] : (T)0.0f;
        __builtin_memcpy(&r, v, sizeof(v));
    }
}
template <bool TINY>
__device__ static inline void eh_own(float (&v)[8], int n, int back) {
    if (n < 8) {
        if (!TINY && back) {
#pragma unroll
            for (int s = 1; s < 8; s *= 2)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float here = v[i], there = v[i + s < 8 ? i + s : 7];
                    v[i] = back & s ? there : here;
                }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? v[i] : 0.0f;
    }
}

// n of eight values (n <= 0: none); the others read as `fill`
template <int DT>
__device__ static inline void eh_load8(const void* base, int64_t off, int n, float (&o)[8], float fill = 0.0f) {
    typedef typename eh_elem<DT>::type T;
    const T* p = reinterpret_cast<const T*>(base) + off;
    if (n >= 8) {
        eh_raw8<DT> r;
        r.load(p);
        r.get(o);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = i < n ? (float)p[i] : fill;
    }
}

// one rounding to the type, to nearest even
template <int DT>
__device__ static inline unsigned eh_pack2(float a, float b) {
    typedef typename eh_elem<DT == EDGEHIP_F32 ? EDGEHIP_BF16 : DT>::type T;
    return (unsigned)__builtin_bit_cast(unsigned short, (T)a) | ((unsigned)__builtin_bit_cast(unsigned short, (T)b) << 16);
}
template <int DT>
__device__ static inline void eh_store8(void* base, int64_t off, int n, const float (&v)[8]) {
    typedef typename eh_elem<DT>::type T;
    T* p = reinterpret_cast<T*>(base) + off;
    if (n >= 8) {
        if (DT == EDGEHIP_F32) {
            *reinterpret_cast<eh_f32x4u*>(p) = eh_f32x4u{v[0], v[1], v[2], v[3]};
            *(reinterpret_cast<eh_f32x4u*>(p) + 1) = eh_f32x4u{v[4], v[5], v[6], v[7]};
        } else {
            *reinterpret_cast<eh_u32x4u*>(p) = eh_u32x4u{eh_pack2<DT>(v[0], v[1]), eh_pack2<DT>(v[2], v[3]), eh_pack2<DT>(v[4], v[5]), eh_pack2<DT>(v[6], v[7])};
        }
    } else if (n > 0) {                                          // in pieces of four, two and one
        const bool four = n & 4;
        if (DT == EDGEHIP_F32) {
            if (four) *reinterpret_cast<eh_f32x4u*>(p) = eh_f32x4u{v[0], v[1], v[2], v[3]};
        } else {
            if (four) *reinterpret_cast<eh_u32x2h*>(p) = eh_u32x2h{eh_pack2<DT>(v[0], v[1]), eh_pack2<DT>(v[2], v[3])};
        }
        const int at = n & 4, last = n & 6;
        // (values read first, then chosen: a choice of places would keep v in memory)
        const float v0 = v[0], v1 = v[1], v2 = v[2], v4 = v[4], v5 = v[5], v6 = v[6];
        const float x0 = four ? v4 : v0, x1 = four ? v5 : v1;
        float x = v0;
        x = last == 2 ? v2 : x;
        x = last == 4 ? v4 : x;
        x = last == 6 ? v6 : x;
        if (n & 2) {
            p[at] = (T)x0;
            p[at + 1] = (T)x1;
        }
        if (n & 1) p[last] = (T)x;
    }
}

// the type known at run time only (parameters: read once per block)
__device__ static inline void eh_load8_any(const void* base, int dt, int64_t off, int n, float (&o)[8], float fill) {
    if (dt == EDGEHIP_F32) eh_load8<EDGEHIP_F32>(base, off, n, o, fill);
    else if (dt == EDGEHIP_BF16) eh_load8<EDGEHIP_BF16>(base, off, n, o, fill);
    else eh_load8<EDGEHIP_F16>(base, off, n, o, fill);
}
__device__ static inline void eh_store1_any(void* base, int dt, int64_t i, float v) {
    if (dt == EDGEHIP_F32) reinterpret_cast<float*>(base)[i] = v;
    else if (dt == EDGEHIP_BF16) reinterpret_cast<__bf16*>(base)[i] = (__bf16)v;
    else reinterpret_cast<_Float16*>(base)[i] = (_Float16)v;
}
