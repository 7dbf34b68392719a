// Rotary positions, and the append of a step's keys and values to the paged cache.
//
// Both are one kernel over a flat list of items. An item is what a lane moves: two pieces of a
// row, N = 16 bytes' worth of elements each (or 1 where an alignment forbids vectors). Of a rotated
// part in the half layout they are the two sides of N pairs; everywhere else the i-th piece of the
// part's first half and the i-th of its second, which leaves every load and store 16 bytes a lane,
// lanes side by side. The items of a token -- its query rows, key rows, value rows -- follow one
// another, and so do the tokens, so that every lane of every workgroup has work whatever the head
// counts are.
//
// The angle position * frequency is formed in 64 bits, in turns, and reduced there to the nearest
// quarter: a product in 32 bits would be off by 2^-24 of the angle, half a radian at position
// 10^7. A pair's cosine and sine serve all heads of the token: a workgroup computes those of the
// tokens that it meets once, while its loads are on their way, and passes them on through LDS.
//
// Bound by HBM: 3 operations per element moved. Microseconds a call, and TB/s of what it reads and
// writes, where a 1 GiB copy reaches 6.6: 16384 x 64 rows of 128 f16, interleaved, 85 (6.3); a prompt of
// 16384, heads of 32 + 8 + 8 x 128 bf16, 67 (6.0); one of 10007, 16 + 2 + 2 x 256, to e4m3 pages, 33 (5.9).
// A step of few tokens is one round trip to memory after a launch: 2.6 for one token, 4.0 for 256 x 80
// rows of 128, less than a caller's host needs to issue it.
#include <hip/hip_runtime.h>

#include "kvt_ops.h"

namespace kvt {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
// One / two / four, microseconds: a prompt of 16384 66.6 / 68.6 / 72.2, one to e4m3 33.4 / 36.4 / 40.0,
// 16384 x 64 rows of f16 85.3 / 89.9 / 91.1 -- more loads in flight per lane, fewer lanes.
constexpr uint32_t kItemsPerLane = 1;
// Stores are non-temporal. Loads are so where the launch reads more than this: less is still in the
// 256 MiB memory-side cache after the projection that made it. Microseconds a call, heads of 32 + 8
// + 8 x 128 bf16, all plain / plain loads, non-temporal stores / both non-temporal: 2048 tokens
// (25 MB read) 9.6 / 9.0 / 10.2, 4096 18.8 / 15.9 / 18.4, 8192 38.0 / 33.4 / 34.1, 16384 (201 MB)
// 73.9 / 69.8 / 66.4.
constexpr uint64_t kCachedInput = 128ull << 20;
constexpr uint32_t kItemsPerWg = kThreads * kItemsPerLane;

struct RotateParams {
  const uint8_t *q, *k, *v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;
  uint8_t* q_out;
  int64_t q_out_token, q_out_head;
  uint8_t* cache;
  int64_t block_stride, kv_stride, token_stride, head_stride;
  const int64_t *positions, *slots;
  uint64_t n_tokens, n_slots;
  uint64_t items_magic, row_magic, half_magic, block_magic;
  uint32_t items, q_items, qk_items;   // per token: all, of the queries, of queries and keys
  uint32_t row_items, rot_items;       // per row; of a query or key row, the rotated ones in front
  uint32_t half, dim, ntpb;            // pairs and elements of a row
  bool once;                           // for the launcher: more is read than kCachedInput
  float k_mul, v_mul, magnitude;
};

// The frequencies travel with the launch; 64 of them (heads of 128) where they are enough, since
// a launch's arguments cost host time by their size (a rotary call: 5.3 us with room for 128, 4.2 with 64).
template <int PAIRS>
struct Turns {
  double per_position[PAIRS];
};

// Every pointer here is to global memory, also where the compiler cannot tell.
template <class V, class P>
__device__ __forceinline__ __attribute__((address_space(1))) V* global(P* p) {
  return (__attribute__((address_space(1))) V*)(p);
}

struct Bf16 {
  static __device__ __forceinline__ float wide(uint32_t bits) { return __uint_as_float(bits << 16); }
  static __device__ __forceinline__ uint32_t pair(float a, float b) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), b2));
  }
};
struct F16 {
  static __device__ __forceinline__ float wide(uint32_t bits) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
  }
  static __device__ __forceinline__ uint32_t pair(float a, float b) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), h2));
  }
};
struct F32 {};

// Two values to e4m3, as the converting pack rounds (kvt_kernels.hip): to nearest even,
// saturating, NaN kept with its sign. The instruction's overflow result depends on a mode bit, so
// the operands are clamped first and NaNs, which the clamp turns into numbers, patched after.
template <bool HIGH>
__device__ __forceinline__ uint32_t to_e4m3(float a, float b, uint32_t acc) {
  uint32_t r = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_fmed3f(a, -448.0f, 448.0f),
                                               __builtin_amdgcn_fmed3f(b, -448.0f, 448.0f), acc, HIGH);
  constexpr uint32_t sh = HIGH ? 16u : 0u;
  if (a != a) r = (r & ~(0xFFu << sh)) | (((__float_as_uint(a) >> 24) & 0x80u) | 0x7Fu) << sh;
  if (b != b) r = (r & ~(0xFF00u << sh)) | (((__float_as_uint(b) >> 24) & 0x80u) | 0x7Fu) << (sh + 8u);
  return r;
}

// N elements of type T as they lie in memory.
template <class T, int N>
struct Piece {
  static constexpr int kElem = std::is_same<T, F32>::value ? 4 : 2;
  static constexpr int kWords = N == 1 ? 1 : N * kElem / 4;
  uint32_t w[kWords];

  template <bool ONCE>
  __device__ __forceinline__ void load(const uint8_t* p) {
    if constexpr (N == 1) {
      if constexpr (kElem == 4)
        w[0] = *global<const uint32_t>(p);
      else
        w[0] = *global<const uint16_t>(p);
    } else {
      const auto at = global<const u32x4>(p);
      const u32x4 v = ONCE ? __builtin_nontemporal_load(at) : *at;
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    }
  }
  __device__ __forceinline__ void store(uint8_t* p) const {
    if constexpr (N == 1) {
      if constexpr (kElem == 4)
        *global<uint32_t>(p) = w[0];
      else
        *global<uint16_t>(p) = static_cast<uint16_t>(w[0]);
    } else {
      __builtin_nontemporal_store((u32x4{w[0], w[1], w[2], w[3]}), global<u32x4>(p));
    }
  }
  __device__ __forceinline__ void widen(float* f) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (kElem == 4)
        f[i] = __uint_as_float(w[i]);
      else
        f[i] = T::wide(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xFFFFu);
    }
  }
  __device__ __forceinline__ void round(const float* f) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (kElem == 4)
        w[i] = __float_as_uint(f[i]);
      else if constexpr (N == 1)
        w[i] = T::pair(f[0], 0.0f);
      else
        w[i] = T::pair(f[2 * i], f[2 * i + 1]);
    }
  }
};

// N values to N bytes of e4m3.
template <int N>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float* f) {
  if constexpr (N == 8) {
    u32x2 r;
    r.x = to_e4m3<true>(f[2], f[3], to_e4m3<false>(f[0], f[1], 0u));
    r.y = to_e4m3<true>(f[6], f[7], to_e4m3<false>(f[4], f[5], 0u));
    __builtin_nontemporal_store(r, global<u32x2>(p));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) *global<uint8_t>(p + i) = static_cast<uint8_t>(to_e4m3<false>(f[i], 0.0f, 0u));
  }
}

// What a lane has of one item between its load and its store.
template <class T, int N>
struct Item {
  Piece<T, N> a, b;
  uint8_t* out;           // where the row starts; nullptr: no item, or a slot that is none
  uint32_t at_a, at_b;    // elements into the row; at_b == 0: there is no second piece
  uint32_t angle;         // first pair's place in the workgroup's table
  float mul;              // of the cache's scale
  bool rotated, narrow;   // narrow: to the cache's 8-bit type
};

// T: type of queries, keys and values. E4M3: the cache holds that instead of T. N: elements of
// a piece. INTER: pairs lie next to each other. PAIRS: room for frequencies. ONCE: read with
// non-temporal loads.
template <class T, bool E4M3, int N, bool INTER, int PAIRS, bool ONCE>
__global__ __launch_bounds__(kThreads) void rotate_append_kernel(const RotateParams p, const Turns<PAIRS> turns) {
  extern __shared__ float2 cs[];
  constexpr int kElem = Piece<T, N>::kElem;
  const uint32_t first = blockIdx.x * kItemsPerWg, tokens_before = divided(first, p.items_magic);
  const uint32_t rem = first - tokens_before * p.items;
  const uint64_t token0 = tokens_before;

  Item<T, N> it[kItemsPerLane];
#pragma unroll
  for (uint32_t n = 0; n < kItemsPerLane; ++n) {
    Item<T, N>& x = it[n];
    x.out = nullptr;
    const uint32_t f = rem + threadIdx.x + n * kThreads;
    const uint32_t tl = divided(f, p.items_magic);
    const uint64_t t = token0 + tl;
    if (t >= p.n_tokens) continue;
    uint32_t i = f - tl * p.items;
    const bool to_cache = i >= p.q_items, value = i >= p.qk_items;
    i -= value ? p.qk_items : to_cache ? p.q_items : 0u;
    const uint32_t row = divided(i, p.row_magic), u = i - row * p.row_items;
    x.rotated = !value && u < p.rot_items;
    x.narrow = E4M3 && to_cache;
    if (x.rotated) {
      x.at_a = INTER && N == 1 ? 2 * u : u * N;
      x.at_b = INTER && N == 1 ? 2 * u + 1 : p.half + u * N;
      // the first pair of the item (of each piece, where a piece holds its pairs whole)
      x.angle = tl * p.half + (INTER && N > 1 ? u * N / 2 : u * N);
    } else {
      const uint32_t front = value ? 0u : 2 * p.half, rest = p.dim - front;
      const uint32_t v = value ? u : u - p.rot_items;
      x.at_a = front + v * N;
      x.at_b = x.at_a + (rest + 1) / 2;
      if (N == 1 && x.at_b >= p.dim) x.at_b = 0;   // the middle one of an odd number
    }
    const uint8_t* in;
    if (to_cache) {
      in = value ? p.v + t * p.v_token + row * p.v_head : p.k + t * p.k_token + row * p.k_head;
      x.mul = value ? p.v_mul : p.k_mul;
      const uint64_t slot = static_cast<uint64_t>(p.slots[t]);
      if (slot >= p.n_slots) continue;   // none (padding): no row
      const uint64_t block =
          p.n_slots <= 0xFFFFFFFFull ? divided(static_cast<uint32_t>(slot), p.block_magic) : slot / p.ntpb;
      x.out = p.cache + block * p.block_stride + (slot - block * p.ntpb) * p.token_stride + row * p.head_stride +
              (value ? p.kv_stride : 0);
    } else {
      in = p.q + t * p.q_token + row * p.q_head;
      x.out = p.q_out + t * p.q_out_token + row * p.q_out_head;
      x.mul = 1.0f;
    }
    x.a.template load<ONCE>(in + x.at_a * kElem);
    if (N > 1 || x.at_b != 0) x.b.template load<ONCE>(in + x.at_b * kElem);
  }

  if (p.half != 0) {
    const uint64_t left = p.n_tokens - token0;
    const uint32_t span = divided(rem + kItemsPerWg - 1, p.items_magic) + 1;
    const uint32_t tokens = left < span ? static_cast<uint32_t>(left) : span;
    for (uint32_t n = threadIdx.x; n < tokens * p.half; n += kThreads) {
      const uint32_t tl = divided(n, p.half_magic);
      double turn = static_cast<double>(p.positions[token0 + tl]) * turns.per_position[n - tl * p.half];
      turn -= rint(turn);
      const double quarter = rint(4.0 * turn);
      float s, c;
      sincospif(static_cast<float>(2.0 * (turn - 0.25 * quarter)), &s, &c);
      const int k = static_cast<int>(quarter) & 3;
      const float cc = k & 1 ? s : c, ss = k & 1 ? c : s;
      cs[n] = make_float2(p.magnitude * (k == 1 || k == 2 ? -cc : cc),
                          p.magnitude * (k >= 2 ? -ss : ss));
    }
    __syncthreads();
  }

#pragma unroll
  for (uint32_t n = 0; n < kItemsPerLane; ++n) {
    Item<T, N>& x = it[n];
    if (!x.out) continue;
    if (x.rotated || (E4M3 && x.narrow)) {
      float a[2 * N];
      x.a.widen(a);
      if (N > 1 || x.at_b != 0) x.b.widen(a + N);
      if (x.rotated) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          // pair j of the item: across its two pieces, or within one of them
          constexpr bool kWithin = INTER && N > 1;
          const int i0 = kWithin ? 2 * j : j, i1 = kWithin ? 2 * j + 1 : N + j;
          const uint32_t at = kWithin && j >= N / 2 ? x.angle + p.half / 2 + j - N / 2 : x.angle + j;
          const float2 t = cs[at];
          const float x0 = a[i0], x1 = a[i1];
          a[i0] = x0 * t.x - x1 * t.y;
          a[i1] = x0 * t.y + x1 * t.x;
        }
      }
      if (E4M3 && x.narrow) {
#pragma unroll
        for (int j = 0; j < 2 * N; ++j) a[j] *= x.mul;
        store_e4m3<N>(x.out + x.at_a, a);
        if (N > 1 || x.at_b != 0) store_e4m3<N>(x.out + x.at_b, a + N);
        continue;
      }
      x.a.round(a);
      x.b.round(a + N);
    }
    x.a.store(x.out + x.at_a * kElem);
    if (N > 1 || x.at_b != 0) x.b.store(x.out + x.at_b * kElem);
  }
}

template <class T, bool E4M3, int N, bool INTER>
void launch_turns(const RotateParams& p, const double* turns, uint32_t wgs, uint32_t lds, hipStream_t s) {
  const auto filled = [&](auto& t) -> auto& {
    for (uint32_t i = 0; i < p.half; ++i) t.per_position[i] = turns[i];
    return t;
  };
  const auto go = [&](auto room, auto once) {
    Turns<decltype(room)::value> t{};
    rotate_append_kernel<T, E4M3, N, INTER, decltype(room)::value, N != 1 && decltype(once)::value>
        <<<wgs, kThreads, lds, s>>>(p, filled(t));
  };
  const std::integral_constant<int, 64> few;
  const std::integral_constant<int, 128> many;
  if (p.half <= 64)
    p.once ? go(few, std::true_type()) : go(few, std::false_type());
  else
    p.once ? go(many, std::true_type()) : go(many, std::false_type());
}

template <class T, bool E4M3, int N>
void launch_pairs(const RotateParams& p, const double* turns, bool inter, uint32_t wgs, uint32_t lds, hipStream_t s) {
  if (inter)
    launch_turns<T, E4M3, N, true>(p, turns, wgs, lds, s);
  else
    launch_turns<T, E4M3, N, false>(p, turns, wgs, lds, s);
}

template <class T, bool E4M3>
void launch_pieces(const RotateParams& p, const double* turns, bool vec, bool inter, uint32_t wgs, uint32_t lds,
                   hipStream_t s) {
  if (vec)
    launch_pairs<T, E4M3, 16 / Piece<T, 1>::kElem>(p, turns, inter, wgs, lds, s);
  else
    launch_pairs<T, E4M3, 1>(p, turns, inter, wgs, lds, s);
}

struct RotateCall {
  const kvt_rotary* rotary;
  uint32_t dtype, head_dim, n_q_heads, n_kv_heads;
  bool e4m3;
  bool aligned;   // every pointer and stride is a multiple of 16 bytes
  hipStream_t stream;
};

struct RotateGrid {
  uint32_t wgs, lds;
  bool vec, inter;
};

// What follows from the sizes. One token's items must fit 32 bits: they do with at most 65536 heads
// of each kind. A launch has fewer than 2^32 lanes.
int size_rotate(const RotateCall& c, RotateParams& p, const char* who, RotateGrid* grid) {
  const uint32_t dim = c.rotary ? c.rotary->dim : 0, n_vec = 16 / dtype_bytes(c.dtype);
  grid->inter = c.rotary && c.rotary->interleaved;
  // vectors need an even number of whole pieces in both parts of a row
  grid->vec = c.aligned && dim % (2 * n_vec) == 0 && c.head_dim % (2 * n_vec) == 0;
  const uint32_t n = grid->vec ? n_vec : 1;
  p.half = dim / 2;
  p.dim = c.head_dim;
  p.rot_items = p.half / n;
  p.row_items = p.rot_items + (c.head_dim - dim + 1) / 2 / n;
  p.q_items = c.n_q_heads * p.row_items;
  p.qk_items = p.q_items + c.n_kv_heads * p.row_items;
  p.items = p.qk_items + c.n_kv_heads * p.row_items;
  p.items_magic = division_magic(p.items);
  p.row_magic = division_magic(p.row_items);
  p.half_magic = division_magic(p.half);
  p.block_magic = division_magic(p.ntpb);
  if (c.rotary) p.magnitude = c.rotary->magnitude;
  const unsigned __int128 all = static_cast<unsigned __int128>(p.n_tokens) * p.items;
  const unsigned __int128 wgs = (all + kItemsPerWg - 1) / kItemsPerWg;
  if (wgs > 0xFFFFFFFFu / kThreads) return fail(KVT_ERR_INVALID, std::string(who) + ": too many rows for one launch");
  p.once = all * 2 * n * dtype_bytes(c.dtype) > kCachedInput;
  grid->wgs = static_cast<uint32_t>(wgs);
  // tokens that one workgroup's items can belong to
  const uint32_t span = p.items ? (kItemsPerWg - 2) / p.items + 2 : 0;
  grid->lds = span * p.half * static_cast<uint32_t>(sizeof(float2));
  return KVT_OK;
}

int launch_rotate(const RotateCall& c, const RotateParams& p, const RotateGrid& g, const char* who) {
  const double* turns = c.rotary ? c.rotary->turns : nullptr;
  switch (c.dtype) {
    case KVT_DTYPE_BF16:
      if (c.e4m3) launch_pieces<Bf16, true>(p, turns, g.vec, g.inter, g.wgs, g.lds, c.stream);
      else launch_pieces<Bf16, false>(p, turns, g.vec, g.inter, g.wgs, g.lds, c.stream);
      break;
    case KVT_DTYPE_F16:
      if (c.e4m3) launch_pieces<F16, true>(p, turns, g.vec, g.inter, g.wgs, g.lds, c.stream);
      else launch_pieces<F16, false>(p, turns, g.vec, g.inter, g.wgs, g.lds, c.stream);
      break;
    default:
      launch_pieces<F32, false>(p, turns, g.vec, g.inter, g.wgs, g.lds, c.stream);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return hip_fail(e, who);
  return KVT_OK;
}

bool being_captured(hipStream_t s) {
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(s, &cap) != hipSuccess) (void)hipGetLastError();
  return cap != hipStreamCaptureStatusNone;
}

}  // namespace
}  // namespace kvt

using namespace kvt;

extern "C" {

int kvt_rotary_apply(const kvt_rotary* r, int device, uint32_t dtype, const void* x,
                     uint64_t x_token_stride, uint64_t x_head_stride, void* out,
                     uint64_t out_token_stride, uint64_t out_head_stride, const int64_t* positions,
                     uint64_t n_tokens, uint32_t n_heads, uint32_t head_dim, void* stream) {
  return guarded([&]() -> int {
    static const char* who = "kvt_rotary_apply";
    if (!r) return fail(KVT_ERR_INVALID, "kvt_rotary_apply: null rotation");
    if (dtype != KVT_DTYPE_BF16 && dtype != KVT_DTYPE_F16 && dtype != KVT_DTYPE_F32)
      return fail(KVT_ERR_UNSUPPORTED, "kvt_rotary_apply: rows are bf16, f16 or f32");
    if (head_dim < r->dim || head_dim > 256 || n_heads > 65536)
      return fail(KVT_ERR_INVALID, "kvt_rotary_apply: head_dim must be at least the rotated part and at most 256, "
                                   "n_heads at most 65536");
    const uint32_t elem = dtype_bytes(dtype);
    const Rows in{x, x_token_stride, x_head_stride}, to{out, out_token_stride, out_head_stride};
    uint64_t in_span = 0, out_span = 0;
    if (int rc = check_rows(in, n_tokens, n_heads, head_dim * elem, elem, false, who, "x", &in_span)) return rc;
    if (int rc = check_rows(to, n_tokens, n_heads, head_dim * elem, elem, true, who, "out", &out_span)) return rc;
    if (int rc = check_apart(in, n_heads, to, n_heads, n_tokens, head_dim * elem, true, who, "x")) return rc;
    if (in_span != 0 && (!positions || reinterpret_cast<uintptr_t>(positions) & 7u))
      return fail(KVT_ERR_INVALID, "kvt_rotary_apply: positions are null or not aligned");
    if (int rc = check_distinct(who, {out, out_span, "out"}, {{positions, 8 * n_tokens, "positions"}})) return rc;
    RotateParams p{};
    p.q = static_cast<const uint8_t*>(x);
    p.q_token = x_token_stride, p.q_head = x_head_stride;
    p.q_out = static_cast<uint8_t*>(out);
    p.q_out_token = out_token_stride, p.q_out_head = out_head_stride;
    p.positions = positions;
    p.n_tokens = n_tokens;
    p.ntpb = 1;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const RotateCall call{r, dtype, head_dim, n_heads, 0, false, rows_aligned16(in) && rows_aligned16(to), s};
    RotateGrid grid{};
    if (int rc = size_rotate(call, p, who, &grid)) return rc;
    if (int rc = check_device(device)) return rc;
    if (in_span == 0) return KVT_OK;
    DeviceGuard g;
    if (int rc = g.enter(device)) return rc;
    if (!being_captured(s))
      if (int rc = check_spans(who, {{x, in_span, "x"}, {out, out_span, "out"}, {positions, 8 * n_tokens, "positions"}}))
        return rc;
    return launch_rotate(call, p, grid, who);
  });
}

int kvt_kv_append(const kvt_cache* cache, uint32_t layer, const kvt_kv_layout* layout,
                  const kvt_rotary* rotary, uint32_t dtype, const void* k, uint64_t k_token_stride,
                  uint64_t k_head_stride, const void* v, uint64_t v_token_stride,
                  uint64_t v_head_stride, const void* q, uint64_t q_token_stride,
                  uint64_t q_head_stride, uint32_t n_q_heads, void* q_out,
                  uint64_t q_out_token_stride, uint64_t q_out_head_stride,
                  const int64_t* positions, const int64_t* slots, uint64_t n_tokens, float k_scale,
                  float v_scale, void* stream) {
  return guarded([&]() -> int {
    static const char* who = "kvt_kv_append";
    uint64_t extent = 0;
    if (int rc = check_kv_layout(layout, who, &extent)) return rc;
    if (dtype != KVT_DTYPE_BF16 && dtype != KVT_DTYPE_F16)
      return fail(KVT_ERR_UNSUPPORTED, "kvt_kv_append: keys and values are bf16 or f16");
    const bool e4m3 = layout->dtype == KVT_DTYPE_E4M3;
    if (!e4m3 && layout->dtype != dtype)
      return fail(KVT_ERR_UNSUPPORTED, "kvt_kv_append: the cache holds the keys' own type or e4m3");
    // a scale whose reciprocal overflows would turn every row into infinities
    if (!(k_scale > 0) || !(v_scale > 0) || !(1.0f / k_scale > 0) || !(1.0f / v_scale > 0) ||
        1.0f / k_scale > 3.0e38f || 1.0f / v_scale > 3.0e38f || (!e4m3 && (k_scale != 1.0f || v_scale != 1.0f)))
      return fail(KVT_ERR_INVALID, "kvt_kv_append: scales must be positive, with finite reciprocals, and 1 for a 16-bit cache");
    if (n_q_heads > 65536 || (n_q_heads != 0 && !rotary))
      return fail(KVT_ERR_INVALID, "kvt_kv_append: queries need a rotation, and at most 65536 heads");
    if (rotary && rotary->dim > layout->head_dim)
      return fail(KVT_ERR_INVALID, "kvt_kv_append: the rotated part is longer than the head");
    const uint32_t elem = dtype_bytes(dtype), heads = layout->n_kv_heads;
    const uint64_t row = static_cast<uint64_t>(layout->head_dim) * elem;
    const Rows kr{k, k_token_stride, k_head_stride}, vr{v, v_token_stride, v_head_stride};
    const Rows qr{q, q_token_stride, q_head_stride}, qo{q_out, q_out_token_stride, q_out_head_stride};
    uint64_t k_span = 0, v_span = 0, q_span = 0, qo_span = 0;
    if (int rc = check_rows(kr, n_tokens, heads, row, elem, false, who, "k", &k_span)) return rc;
    if (int rc = check_rows(vr, n_tokens, heads, row, elem, false, who, "v", &v_span)) return rc;
    if (int rc = check_rows(qr, n_tokens, n_q_heads, row, elem, false, who, "q", &q_span)) return rc;
    if (int rc = check_rows(qo, n_tokens, n_q_heads, row, elem, true, who, "q_out", &qo_span)) return rc;
    if (int rc = check_apart(qr, n_q_heads, qo, n_q_heads, n_tokens, row, true, who, "q")) return rc;
    if (int rc = check_apart(kr, heads, qo, n_q_heads, n_tokens, row, false, who, "k")) return rc;
    if (int rc = check_apart(vr, heads, qo, n_q_heads, n_tokens, row, false, who, "v")) return rc;
    if (n_tokens != 0 && (!slots || reinterpret_cast<uintptr_t>(slots) & 7u))
      return fail(KVT_ERR_INVALID, "kvt_kv_append: slots are null or not aligned");
    if (n_tokens != 0 && rotary && (!positions || reinterpret_cast<uintptr_t>(positions) & 7u))
      return fail(KVT_ERR_INVALID, "kvt_kv_append: positions are null or not aligned");
    const Span slot_array{slots, 8 * n_tokens, "slots"}, position_array{positions, rotary ? 8 * n_tokens : 0, "positions"};
    if (int rc = check_distinct(who, {q_out, qo_span, "q_out"}, {slot_array, position_array})) return rc;
    RotateParams p{};
    p.q = static_cast<const uint8_t*>(q), p.k = static_cast<const uint8_t*>(k), p.v = static_cast<const uint8_t*>(v);
    p.q_token = q_token_stride, p.q_head = q_head_stride;
    p.k_token = k_token_stride, p.k_head = k_head_stride;
    p.v_token = v_token_stride, p.v_head = v_head_stride;
    p.q_out = static_cast<uint8_t*>(q_out);
    p.q_out_token = q_out_token_stride, p.q_out_head = q_out_head_stride;
    p.block_stride = layout->block_stride, p.kv_stride = layout->kv_stride;
    p.token_stride = layout->token_stride, p.head_stride = layout->head_stride;
    p.positions = positions, p.slots = slots;
    p.n_tokens = n_tokens, p.n_slots = layout->n_blocks * layout->ntpb;
    p.ntpb = layout->ntpb;
    p.k_mul = 1.0f / k_scale, p.v_mul = 1.0f / v_scale;
    const bool aligned = rows_aligned16(kr) && rows_aligned16(vr) &&
                         (n_q_heads == 0 || (rows_aligned16(qr) && rows_aligned16(qo)));
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const RotateCall call{rotary, dtype, layout->head_dim, n_q_heads, heads, e4m3, aligned, s};
    RotateGrid grid{};
    if (int rc = size_rotate(call, p, who, &grid)) return rc;
    if (int rc = check_cache_layer(cache, layer, layout, extent, who, &p.cache)) return rc;
    if (n_tokens == 0) return KVT_OK;
    if (int rc = check_distinct(who, {p.cache, extent, "the cache's tensor"},
                                {{k, k_span, "k"}, {v, v_span, "v"}, {q, q_span, "q"}, {q_out, qo_span, "q_out"},
                                 slot_array, position_array}))
      return rc;
    DeviceGuard g;
    if (int rc = g.enter(cache->device)) return rc;
    if (!being_captured(s))
      if (int rc = check_spans(who, {{k, k_span, "k"}, {v, v_span, "v"}, {q, q_span, "q"}, {q_out, qo_span, "q_out"},
                                     slot_array, position_array}))
        return rc;
    return launch_rotate(call, p, grid, who);
  });
}

}  // extern "C"
