// kvq8.cuh -- paged KV cache in 8 bits: shared device definitions.
//
// A page holds page_tokens consecutive positions of one sequence.  For each
// page and KV head, keys and values are codes c in [-127, 127] with one fp32
// scale s: the value is c * s.  Sequences name their pages through a block
// table; entries outside [0, pages) stand for absent pages (their rows are
// dropped by the append and never attended to).
#pragma once

#include <math.h>

#include "kib_common.cuh"

namespace kib {

struct Kvq8Cache {
  int8_t *k, *v;
  float *k_scale, *v_scale;  // [pages][kv_heads]
  int pages, kv_heads, page_tokens, page_shift, head_dim;
  int64_t page_stride, head_stride, token_stride;  // elements (bytes)
};

struct Kvq8Batch {
  const int32_t *table, *lengths, *row_start;
  int sequences, table_stride, rows, max_rows;
  int max_length;  // keys at positions past it are not attended to
};

// New rows and length of one sequence.  Row i of n sits at position
// length - n + i; everything is clamped so that no bad entry reads or writes
// outside the tensors.
struct Kvq8Seq {
  int first, n, length;
};

KIB_DEV Kvq8Seq kvq8_seq(const Kvq8Batch& b, int s) {
  Kvq8Seq q;
  q.first = max(0, min(b.row_start[s], b.rows));
  q.n = max(0, min(b.row_start[s + 1], b.rows) - q.first);
  q.length = max(-(1 << 30), min(b.lengths[s], 1 << 30));
  return q;
}

KIB_DEV int kvq8_page(const Kvq8Cache& c, const Kvq8Batch& b, int s, int page_index) {
  if (page_index < 0 || page_index >= b.table_stride) return -1;
  const int p = b.table[static_cast<int64_t>(s) * b.table_stride + page_index];
  return p >= 0 && p < c.pages ? p : -1;
}

template <typename T>
KIB_DEV float to_f32(T x);
template <>
KIB_DEV float to_f32<float>(float x) { return x; }
template <>
KIB_DEV float to_f32<__half>(__half x) { return __half2float(x); }
template <typename T>
KIB_DEV T from_f32(float x);
template <>
KIB_DEV float from_f32<float>(float x) { return x; }
template <>
KIB_DEV __half from_f32<__half>(float x) { return __float2half_rn(x); }

// V consecutive elements through the widest loads their alignment allows
// (V * sizeof(T) bytes: 4, 8, 16 or 32).
template <typename T, int V>
KIB_DEV void load_vec(const T* p, float (&x)[V]) {
  constexpr int B = V * static_cast<int>(sizeof(T));
  constexpr int W = B >= 16 ? 16 : B;
  alignas(16) T raw[V];
#pragma unroll
  for (int i = 0; i < B / W; ++i) {
    if constexpr (W == 16) reinterpret_cast<uint4*>(raw)[i] = reinterpret_cast<const uint4*>(p)[i];
    else if constexpr (W == 8) reinterpret_cast<uint2*>(raw)[i] = reinterpret_cast<const uint2*>(p)[i];
    else reinterpret_cast<uint32_t*>(raw)[i] = reinterpret_cast<const uint32_t*>(p)[i];
  }
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = to_f32<T>(raw[i]);
}

template <typename T, int V>
KIB_DEV void store_vec(T* p, const float (&x)[V]) {
  constexpr int B = V * static_cast<int>(sizeof(T));
  constexpr int W = B >= 16 ? 16 : B;
  alignas(16) T raw[V];
#pragma unroll
  for (int i = 0; i < V; ++i) raw[i] = from_f32<T>(x[i]);
#pragma unroll
  for (int i = 0; i < B / W; ++i) {
    if constexpr (W == 16) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(raw)[i];
    else if constexpr (W == 8) reinterpret_cast<uint2*>(p)[i] = reinterpret_cast<const uint2*>(raw)[i];
    else reinterpret_cast<uint32_t*>(p)[i] = reinterpret_cast<const uint32_t*>(raw)[i];
  }
}

// V codes packed in V bytes (2, 4 or 8).
template <int V>
KIB_DEV void load_codes(const int8_t* p, int (&c)[V]) {
  alignas(8) int8_t raw[V];
  if constexpr (V == 8) *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(p);
  else if constexpr (V == 4) *reinterpret_cast<uint32_t*>(raw) = *reinterpret_cast<const uint32_t*>(p);
  else *reinterpret_cast<uint16_t*>(raw) = *reinterpret_cast<const uint16_t*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) c[i] = raw[i];
}

}  // namespace kib
