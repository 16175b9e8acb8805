// Element types of the entry points that take fp32, bf16 and fp16 tensors (glx_layernorm.hip, glx_attention.hip,
// glx_orthogonal.hip): GLX_F32 / GLX_BF16 / GLX_F16 of glenet_hip.h.
#pragma once
#include "glx_common.h"

static inline size_t glx_elem_size(int dtype) { return dtype == GLX_F32 ? 4 : 2; }
static inline bool glx_elem_ok(int dtype) { return dtype == GLX_F32 || dtype == GLX_BF16 || dtype == GLX_F16; }

// VEC elements at any address that is a multiple of the ELEMENT size: one wide load / store (global memory takes unaligned
// dwordx4 accesses; a row of an odd width starts anywhere)
template <typename T, int VEC>
struct GlxVec {
  typedef T vec __attribute__((ext_vector_type(VEC)));
  struct __attribute__((packed, aligned(sizeof(T)))) loose { vec v; };
  static __device__ __forceinline__ vec load(const T* p) { return reinterpret_cast<const loose*>(p)->v; }
  static __device__ __forceinline__ void store(T* p, vec v) { reinterpret_cast<loose*>(p)->v = v; }
};
