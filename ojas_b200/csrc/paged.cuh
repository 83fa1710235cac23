// Shared by the kernels over a paged KV cache: the pages' view, the pass's index tables and the rotation of a pair.
#pragma once
#include "common.cuh"

// [P, page, Hkv, D] through strides in elements; D contiguous
template <class P>
struct PagesView {
  P* ptr;
  int64_t sp, st, sh;   // page, place in the page, head
};
template <class P>
inline PagesView<P> pages_view(const ojc_tensor* t) { return PagesView<P>{(P*)t->data, t->stride[0], t->stride[1], t->stride[2]}; }

// [N, H, D] through strides; D contiguous
template <class P>
struct RowsView {
  P* ptr;
  int64_t sn, sh;
};
template <class P>
inline RowsView<P> rows_view(const ojc_tensor* t) { return RowsView<P>{(P*)t->data, t->stride[0], t->stride[1]}; }

// A tensor that is written through its strides: no axis may lie on itself (a broadcast one, of stride 0, would take the writes of all its entries)
inline ojc_status own_places(const char* op, const char* what, const ojc_tensor* t) {
  for (int i = 0; i < t->rank; ++i)
    if (t->shape[i] > 1 && t->stride[i] == 0) return ojc_fail(OJC_ERR_SHAPE, op, std::string(what) + " is written and cannot be a broadcast view");
  return OJC_OK;
}

#ifdef __CUDACC__
// Rotation of a pair: the angle is position x frequency with the frequency in 2^-64 turns, so the product modulo 2^64 IS the angle's fraction of a
// turn, exact to position x 2^-64 however far the position; its upper half as a signed integer is the angle / pi in [-1, 1) x 2^31. What is rounded to
// BF16 (2^-8) takes the special-function unit's sine and cosine, whose absolute error on [-pi, pi] is about 2^-21; F32 results take sincospif.
template <bool F32_RESULT>
__device__ __forceinline__ void rope_turn(uint64_t turns, uint32_t position, float amplitude, float* c, float* s) {
  const uint64_t t = turns * position;
  const float half_turns = (float)(int32_t)(uint32_t)(t >> 32) * 4.656612873077393e-10f;
  if (F32_RESULT) sincospif(half_turns, s, c);
  else __sincosf(half_turns * 3.14159265358979f, s, c);
  *c = __fmul_rn(*c, amplitude);
  *s = __fmul_rn(*s, amplitude);
}
// (u, v) turned: one product rounded, then a fused multiply-add, spelled out so that every kernel gives the same bits
__device__ __forceinline__ float turned_first(float u, float v, float c, float s) { return __fmaf_rn(u, c, -__fmul_rn(v, s)); }
__device__ __forceinline__ float turned_second(float u, float v, float c, float s) { return __fmaf_rn(v, c, __fmul_rn(u, s)); }
#endif

ojc_status rope_check(const char* op, const ojc_rope* rope, int64_t head_dim);
