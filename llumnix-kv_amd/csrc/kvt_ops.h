// Internal declarations shared by the operators that fill and read the registered cache's pages
// (rotary positions, append, attention of one new token): argument checks and device helpers.
#ifndef KVT_OPS_H_
#define KVT_OPS_H_

#include <initializer_list>
#include <string>

#include "kvt_runtime.h"

struct kvt_rotary {
  uint32_t dim = 0;            // rotated elements of a row
  bool interleaved = false;
  float magnitude = 1.0f;
  double turns[128] = {};      // turns (not radians) per position, pair by pair
};

namespace kvt {

// Bytes of an element; 0 for an unknown dtype.
uint32_t dtype_bytes(uint32_t dtype);

// What kvt_kv_layout promises, checked; *extent = bytes from the tensor's start to behind its
// last row. The message starts with `who`.
int check_kv_layout(const kvt_kv_layout* l, const char* who, uint64_t* extent);
// The layer's tensor: KVT_OK and its base when the (checked) layout's extent fits into it.
int check_cache_layer(const kvt_cache* c, uint32_t layer, const kvt_kv_layout* l, uint64_t extent,
                      const char* who, uint8_t** base);

// n_tokens x n_heads rows of row_bytes bytes at token * token_stride + head * head_stride.
struct Rows {
  const void* ptr;
  uint64_t token_stride, head_stride;
};
// Alignment to the element, a span that can be formed, rows apart where they are written.
// *span = bytes from ptr to behind the last row.
int check_rows(const Rows& r, uint64_t n_tokens, uint32_t n_heads, uint64_t row_bytes,
               uint32_t elem, bool written, const char* who, const char* what, uint64_t* span);
// Refuses rows that are read (`what`) where they share bytes with rows that are written by the
// same launch, unless they are the very same rows and `in_place` allows that. Slices of one wider
// tensor that interleave without sharing a byte are told apart, token by token or (with equal strides)
// head by head.
int check_apart(const Rows& in, uint32_t in_heads, const Rows& out, uint32_t out_heads, uint64_t n_tokens,
                uint64_t row_bytes, bool in_place, const char* who, const char* what);

// check_device_span() of several buffers; the text of a refusal is only made for one.
struct Span {
  const void* ptr;
  uint64_t bytes;
  const char* what;
};
int check_spans(const char* who, std::initializer_list<Span> spans);
// Refuses a buffer that reaches into one of the others.
int check_distinct(const char* who, const Span& a, std::initializer_list<Span> others);

inline bool rows_aligned16(const Rows& r) {
  return ((reinterpret_cast<uintptr_t>(r.ptr) | r.token_stride | r.head_stride) & 15u) == 0;
}

// n / d for 32-bit n by a multiplication: m = ceil(2^64 / d), 0 standing for d = 1.
inline uint64_t division_magic(uint32_t d) { return d <= 1 ? 0 : ~0ull / d + 1; }

__device__ __forceinline__ uint32_t divided(uint32_t n, uint64_t m) {
  if (m == 0) return n;
  return static_cast<uint32_t>(((m >> 32) * n + __umulhi(static_cast<uint32_t>(m), n)) >> 32);
}

}  // namespace kvt

#endif  // KVT_OPS_H_
