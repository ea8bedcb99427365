// Element types of the kernels that take fp32, bf16 or fp16 tensors: conversion to the 32-bit working type and back (round to
// nearest even), and vectors of 16 bytes.
#pragma once
#include "common.h"

template <typename T> __device__ inline float sis3d_f32(T v) { return (float)v; }
template <typename T> __device__ inline T sis3d_from_f32(float v) { return (T)v; }

// 16 bytes of elements (VEC = 16 / sizeof(T)) or one element (VEC = 1: rows or strides that are not 16-byte aligned).  The 16 bytes are
// held as four words and taken apart by the word: as an array of 16-bit elements the compiler moves them about one by one.
template <typename T, int VEC> struct SisVec { uint32_t w[4]; };
template <typename T> struct SisVec<T, 1> { T v; };

typedef uint32_t sis3d_u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 sis3d_f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 sis3d_bf16x2 __attribute__((ext_vector_type(2)));

template <typename T, int VEC, bool ONCE = false> __device__ inline SisVec<T, VEC> sis3d_raw(const T *p)
{
    SisVec<T, VEC> r;
    if constexpr (VEC == 1) r.v = *p;
    else {
        const sis3d_u32x4 *q = reinterpret_cast<const sis3d_u32x4 *>(p);
        sis3d_u32x4 v;
        if constexpr (ONCE) v = __builtin_nontemporal_load(q);
        else v = *q;
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = v[i];
    }
    return r;
}
// A vector that is read once: marked so that it does not displace what is read again.  Streaming 256 MB reads, 16 bytes a lane, four in
// flight: 6.0 TB/s without the mark, 6.8 TB/s with it.
template <typename T, int VEC> __device__ inline SisVec<T, VEC> sis3d_load_once(const T *p) { return sis3d_raw<T, VEC, true>(p); }

template <typename T, int VEC> __device__ inline void sis3d_unpack(const SisVec<T, VEC> &r, float (&out)[VEC])
{
    if constexpr (VEC == 1) out[0] = (float)r.v;
    else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = __uint_as_float(r.w[i]);
    } else if constexpr (__is_same(T, __bf16)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            out[2 * i] = __uint_as_float(r.w[i] << 16);
            out[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const sis3d_f16x2 h = __builtin_bit_cast(sis3d_f16x2, r.w[i]);
            out[2 * i] = (float)h[0];
            out[2 * i + 1] = (float)h[1];
        }
    }
}
template <typename T, int VEC> __device__ inline void sis3d_load(const T *p, float (&out)[VEC]) { sis3d_unpack<T, VEC>(sis3d_raw<T, VEC>(p), out); }

template <typename T, int VEC, bool ONCE = false> __device__ inline void sis3d_store(T *p, const float (&in)[VEC])
{
    if constexpr (VEC == 1) *p = (T)in[0];
    else {
        sis3d_u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) v[i] = __float_as_uint(in[i]);
            else if constexpr (__is_same(T, __bf16)) v[i] = __builtin_bit_cast(uint32_t, sis3d_bf16x2{(__bf16)in[2 * i], (__bf16)in[2 * i + 1]});
            else v[i] = __builtin_bit_cast(uint32_t, sis3d_f16x2{(_Float16)in[2 * i], (_Float16)in[2 * i + 1]});
        }
        if constexpr (ONCE) __builtin_nontemporal_store(v, reinterpret_cast<sis3d_u32x4 *>(p));
        else *reinterpret_cast<sis3d_u32x4 *>(p) = v;
    }
}

static inline int sis3d_elem_bytes(int dtype) { return dtype == SIS3D_F32 ? 4 : (dtype == SIS3D_BF16 || dtype == SIS3D_F16) ? 2 : 0; }
