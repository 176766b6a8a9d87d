// vec.h - eight consecutive values of a fp32 / bf16 / fp16 row, at any alignment, as fp32 registers.
//
// gfx950 takes 16-byte global accesses at any element-aligned address, so a row of odd length or a view that starts in
// the middle of a line is read with the same vector accesses as an aligned one: the vector types below only promise the
// alignment of their element.  The last, partial vector of a row goes element by element.
#pragma once
#include "common.h"

template <int DT> struct eh_elem;
template <> struct eh_elem<EDGEHIP_F32> { typedef float type; };
template <> struct eh_elem<EDGEHIP_BF16> { typedef __bf16 type; };
template <> struct eh_elem<EDGEHIP_F16> { typedef _Float16 type; };

typedef float eh_f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned int eh_u32x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int eh_u32x2u __attribute__((ext_vector_type(2), aligned(1)));

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
__device__ static inline void eh_store8(void* base, int64_t off, int n, const float (&v)[8]) {
    typedef typename eh_elem<DT>::type T;
    T* p = reinterpret_cast<T*>(base) + off;
    if (n >= 8) {
        if (DT == EDGEHIP_F32) {
            *reinterpret_cast<eh_f32x4u*>(p) = eh_f32x4u{v[0], v[1], v[2], v[3]};
            *(reinterpret_cast<eh_f32x4u*>(p) + 1) = eh_f32x4u{v[4], v[5], v[6], v[7]};
        } else {
            eh_u32x4u w;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned lo = __builtin_bit_cast(unsigned short, (typename eh_elem<DT == EDGEHIP_F32 ? EDGEHIP_BF16 : DT>::type)v[2 * i]);
                const unsigned hi = __builtin_bit_cast(unsigned short, (typename eh_elem<DT == EDGEHIP_F32 ? EDGEHIP_BF16 : DT>::type)v[2 * i + 1]);
                w[i] = lo | (hi << 16);
            }
            *reinterpret_cast<eh_u32x4u*>(p) = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = (T)v[i];
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
