// dg_half.h -- element types of the layer and optimizer operators (adamw.hip, groupnorm.hip, grouped.hip): fp32, bf16 and fp16 values
// in memory, fp32 in registers; vectors of them in one load or store.
#pragma once
#include "dg_common.h"

#ifdef DG_EMU      // (host compilers have no conversion instruction for bf16: the same round-to-nearest-even in integers)
static inline uint16_t dg_f32_to_bf16(float f) {
  const uint32_t u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
#else
__device__ __forceinline__ uint16_t dg_f32_to_bf16(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
#endif

struct DgF32 {
  typedef float S;
  static constexpr int FULL = 4;      // elements of a 16-byte access
  static __device__ __forceinline__ float to(float s) { return s; }
  static __device__ __forceinline__ float from(float f) { return f; }
};
struct DgBF16 {
  typedef uint16_t S;
  static constexpr int FULL = 8;
  static __device__ __forceinline__ float to(uint16_t s) { return __uint_as_float((uint32_t)s << 16); }
  static __device__ __forceinline__ uint16_t from(float f) { return dg_f32_to_bf16(f); }
};
struct DgF16 {
  typedef uint16_t S;
  static constexpr int FULL = 8;
  static __device__ __forceinline__ float to(uint16_t s) { return (float)__builtin_bit_cast(_Float16, s); }
  static __device__ __forceinline__ uint16_t from(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
};

// VEC elements as they lie in memory
template <class D, int VEC> struct DgRaw {
  typedef typename D::S T __attribute__((ext_vector_type(VEC)));
  T v;
  __device__ __forceinline__ float get(int i) const { return D::to(v[i]); }
  __device__ __forceinline__ void set(int i, float f) { v[i] = D::from(f); }
};
template <class D> struct DgRaw<D, 1> {
  typedef typename D::S T;
  T v;
  __device__ __forceinline__ float get(int) const { return D::to(v); }
  __device__ __forceinline__ void set(int, float f) { v = D::from(f); }
};
template <class D, int VEC> __device__ __forceinline__ DgRaw<D, VEC> dg_load(const typename D::S* p) {
  DgRaw<D, VEC> r;
  r.v = *reinterpret_cast<const typename DgRaw<D, VEC>::T*>(p);
  return r;
}
template <class D, int VEC> __device__ __forceinline__ void dg_store(typename D::S* p, const DgRaw<D, VEC>& r) {
  *reinterpret_cast<typename DgRaw<D, VEC>::T*>(p) = r.v;
}
template <class D, int VEC> __device__ __forceinline__ DgRaw<D, VEC> dg_zero() {
  DgRaw<D, VEC> r;
  r.v = (typename DgRaw<D, VEC>::T)(0);
  return r;
}
// the vectors' bits become opaque: what was computed from them is computed again where it is needed again, not held in registers
template <class D, int VEC, int N> __device__ __forceinline__ void dg_hide(DgRaw<D, VEC>* r) {
#ifndef DG_EMU
  constexpr int B = VEC * sizeof(typename D::S);
  typedef uint32_t W __attribute__((ext_vector_type(B >= 8 ? B / 4 : 2)));
#pragma unroll
  for (int i = 0; i < N; ++i)
    if constexpr (B >= 8) { W w = __builtin_bit_cast(W, r[i].v); asm volatile("" : "+v"(w)); r[i].v = __builtin_bit_cast(typename DgRaw<D, VEC>::T, w); }
#endif
}
// one element of a tensor whose type is known at run time (weights and biases may differ in type from the activations)
__device__ __forceinline__ float dg_load_as(const void* p, int64_t i, int dtype) {
  if (dtype == DGCNN_F32) return static_cast<const float*>(p)[i];
  const uint16_t s = static_cast<const uint16_t*>(p)[i];
  return dtype == DGCNN_BF16 ? DgBF16::to(s) : DgF16::to(s);
}
__device__ __forceinline__ void dg_store_as(void* p, int64_t i, int dtype, float f) {
  if (dtype == DGCNN_F32) static_cast<float*>(p)[i] = f;
  else static_cast<uint16_t*>(p)[i] = dtype == DGCNN_BF16 ? DgBF16::from(f) : DgF16::from(f);
}
static inline bool dg_dtype_ok(int d) { return d == DGCNN_F32 || d == DGCNN_BF16 || d == DGCNN_F16; }
static inline int dg_dtype_size(int d) { return d == DGCNN_F32 ? 4 : 2; }
