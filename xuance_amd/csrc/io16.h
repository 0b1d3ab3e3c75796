// Activations stored as f32 or bf16: element and vector access of the sequence-policy kernels.  Arithmetic is f32; a value is rounded
// (to nearest even) only where it is stored.
#pragma once
#include "common.h"
#include "split3.h"

namespace xrl {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));

struct bf16_t { unsigned short bits; };

__device__ __forceinline__ float io_load(const float* p) { return *p; }
__device__ __forceinline__ float io_load(const bf16_t* p) { return bf16_bits_to_float(p->bits); }
__device__ __forceinline__ void io_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void io_store(bf16_t* p, float v) { p->bits = (unsigned short)cvt_pk_bf16(v, 0.f); }

}  // namespace xrl
