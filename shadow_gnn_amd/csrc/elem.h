// Element types of the node-wise MLP operators (layer_norm.hip, dropout.hip, linear16.hip, label_logprobs.hip): fp32, bf16 and fp16
// in memory, fp32 in registers, and vectors of V elements that are loaded and stored whole.
#pragma once
#include "actnorm_common.h"

namespace shadow {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void ldv(const T *p, float (&x)[V]) {
  const Vec<T, V> a = *reinterpret_cast<const Vec<T, V> *>(p);
#pragma unroll
  for (int j = 0; j < V; j++) x[j] = (float)a.v[j];
}
// (conversions to 16 bits round to nearest even: v_cvt_pk_bf16_f32 / v_cvt_f16_f32)
template <typename T, int V>
__device__ __forceinline__ void stv(T *p, const float (&x)[V]) {
  Vec<T, V> a;
#pragma unroll
  for (int j = 0; j < V; j++) a.v[j] = (T)x[j];
  *reinterpret_cast<Vec<T, V> *>(p) = a;
}

// elements per 16-byte word
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

inline uint32_t elem_bytes(int dtype) { return dtype == SL_F32 ? 4u : 2u; }
inline bool elem_dtype_ok(int dtype) { return dtype == SL_F32 || dtype == SL_BF16 || dtype == SL_F16; }
// rows of whole 16-byte words: pointer, pitch and width
inline bool rows_of_words(const void *p, int64_t ld, uint32_t F, int dtype) {
  const uint32_t V = 16u / elem_bytes(dtype);
  return !p || (!(reinterpret_cast<uintptr_t>(p) & 15) && ld % V == 0 && F % V == 0);
}

// the statement with T the C++ type of DTYPE
#define SHD_DISPATCH_ELEM(DTYPE, ...)                              \
  switch (DTYPE) {                                                 \
    case SL_F32: { using T = float; __VA_ARGS__; break; }          \
    case SL_BF16: { using T = shadow::bf16_t; __VA_ARGS__; break; }\
    default: { using T = shadow::f16_t; __VA_ARGS__; break; }      \
  }

}  // namespace shadow
