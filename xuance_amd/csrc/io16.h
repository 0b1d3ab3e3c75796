// Activations stored as f32 or bf16: element and vector access of the sequence-policy kernels.  Arithmetic is f32; a value is rounded
// (to nearest even) only where it is stored.
#pragma once
#include "common.h"
#include "split3.h"

namespace xrl {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));

struct bf16_t { unsigned short bits; };

__device__ __forceinline__ float io_load(const float* p) { return *p; }
__device__ __forceinline__ float io_load(const bf16_t* p) { return bf16_bits_to_float(p->bits); }
__device__ __forceinline__ void io_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void io_store(bf16_t* p, float v) { p->bits = (unsigned short)cvt_pk_bf16(v, 0.f); }

// 16 bytes of a row at any element: the hardware takes such an access at any address
typedef u32x4_t u32x4_any4_t __attribute__((aligned(4)));
typedef u32x4_t u32x4_any2_t __attribute__((aligned(2)));
typedef f32x4_t f32x4_any_t __attribute__((aligned(4)));

template <typename E> struct row16;
template <> struct row16<float> {
    static constexpr int PER = 4;
    static constexpr unsigned LOW = 0xff800000u;                // -inf in every element
    static __device__ __forceinline__ u32x4_t load(const float* p) { return *reinterpret_cast<const u32x4_any4_t*>(p); }
    static __device__ __forceinline__ void store(float* p, u32x4_t v) { *reinterpret_cast<u32x4_any4_t*>(p) = v; }
    static __device__ __forceinline__ unsigned bits(const float* p) { return __float_as_uint(*p); }
    static __device__ __forceinline__ float get(const u32x4_t& v, int j) { return __uint_as_float(v[j]); }
    static __device__ __forceinline__ void put(u32x4_t& v, int j, unsigned b) { v[j] = b; }
    static __device__ __forceinline__ u32x4_t pack(const float* f) {
        const u32x4_t v = {__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
        return v;
    }
};
template <> struct row16<bf16_t> {
    static constexpr int PER = 8;
    static constexpr unsigned LOW = 0xff80ff80u;
    static __device__ __forceinline__ u32x4_t load(const bf16_t* p) { return *reinterpret_cast<const u32x4_any2_t*>(p); }
    static __device__ __forceinline__ void store(bf16_t* p, u32x4_t v) { *reinterpret_cast<u32x4_any2_t*>(p) = v; }
    static __device__ __forceinline__ unsigned bits(const bf16_t* p) { return p->bits; }
    static __device__ __forceinline__ float get(const u32x4_t& v, int j) { return __uint_as_float(j & 1 ? v[j >> 1] & 0xffff0000u : v[j >> 1] << 16); }
    static __device__ __forceinline__ void put(u32x4_t& v, int j, unsigned b) {
        v[j >> 1] = j & 1 ? (v[j >> 1] & 0xffffu) | (b << 16) : (v[j >> 1] & 0xffff0000u) | (b & 0xffffu);
    }
    static __device__ __forceinline__ u32x4_t pack(const float* f) {
        const u32x4_t v = {cvt_pk_bf16(f[0], f[1]), cvt_pk_bf16(f[2], f[3]), cvt_pk_bf16(f[4], f[5]), cvt_pk_bf16(f[6], f[7])};
        return v;
    }
};

}  // namespace xrl
