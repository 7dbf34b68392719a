// Attention of one new token per sequence over the paged cache.
//
// out = sum_t p_t v_t / sum_t p_t with p_t = exp(s_t - max s), s_t = scale q . k_t, in one pass
// over the keys and values with the running maximum and sum of the softmax. All query heads of a
// KV head read the same rows, so a wavefront takes up to 16 of them at once and the products are
// matrix products of 16 columns:
//   S^T [16 tokens x 16 heads] = K [tokens x dim] Q^T    (v_mfma_f32_16x16x32: A = K, B = Q^T)
//   O^T [dim x 16 heads]      += V^T [dim x tokens] P^T  (A = V^T, B = P^T), 32 tokens at a time
// The matrix instruction's contracted index may be numbered at will as long as both operands
// agree, which is used twice: (1) the result of the first product (lane: head = lane % 16, tokens
// 4 (lane / 16) ... + 3) is the second product's operand as it stands, no value changes lanes; (2)
// a lane loads whole vectors of rows of V, for the eight tokens whose weights it holds, and
// turns the 8 x n block inside its registers. The accumulators and the softmax's statistics then
// lie on lanes of the same head.
//
// Weights are split into two 16-bit values each (the weight cut off and what that left, rounded),
// so that the product with V loses nothing that counts beside the output's own rounding: rounding
// them once costs as much error as the output's rounding does, the second product costs a few
// matrix instructions in a kernel that is bound by HBM. Both values are positive (the rest at
// least the smallest positive number), so that an infinity in V times a weight is that infinity,
// as in the formula, and not the difference of two.
//
// An 8-bit cache is widened on load: every e4m3 value is a bf16 and an f16 value.
#include <hip/hip_runtime.h>

#include <cmath>
#include <thread>

#include "kvt_ops.h"

namespace kvt {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256, kWaves = 4;
constexpr uint32_t kTile = 32;                   // tokens a wavefront takes at a time
constexpr uint32_t kStep = kTile * kWaves;       // ... and a workgroup
constexpr uint32_t kMaxSplits = 256;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;

struct DecodeParams {
  const uint8_t* base;
  int64_t block_stride, kv_stride, token_stride, head_stride;
  const uint8_t* q;
  int64_t q_token, q_head;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* lens;
  uint8_t* out;
  int64_t out_token, out_head;
  float* lse;
  float* part_o;       // [seq][head][split][head_dim]: sums not yet divided
  float2* part_ml;     // [seq][head][split]: maximum (times log2 e), sum
  uint32_t* counters;  // [seq][group of heads]: workgroups that have left their part
  uint64_t block_magic, visible_max;
  uint32_t ntpb, n_blocks, n_heads, group, head_tiles, head_dim, window, chunk, splits;
  float scale_log2, cap, cap_in, v_scale;
  bool q_vec, out_vec;
};

struct Bf16 {
  typedef __bf16 x8 __attribute__((ext_vector_type(8)));
  typedef __bf16 x2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  template <bool HIGH>
  static __device__ __forceinline__ uint32_t widen(uint32_t e4m3) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(e4m3, 1.0f, HIGH));
  }
  // two values cut off to this type, and the smallest positive rest worth adding (see Weights)
  static __device__ __forceinline__ uint32_t cut(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
  }
  static constexpr float kLeast = 0x1p-126f;
};
struct F16 {
  typedef _Float16 x8 __attribute__((ext_vector_type(8)));
  typedef _Float16 x2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  template <bool HIGH>
  static __device__ __forceinline__ uint32_t widen(uint32_t e4m3) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(e4m3, 1.0f, HIGH));
  }
  static __device__ __forceinline__ uint32_t cut(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
  }
  static constexpr float kLeast = 0x1p-24f;
};

// The maximum / sum over the four lanes that hold one head's tokens (lane, +16, +32, +48).
__device__ __forceinline__ float over_tokens_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float over_tokens_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// One part's statistics of a head. sum < 0 stands for "scores were there, all of them minus
// infinity": that softmax is NaN, while a head that saw no token at all gives zeros.
struct Stat {
  float max, sum;
};
__device__ __forceinline__ float weight_of(const Stat& s, float top) {
  return s.max == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s.max - top);
}

// T: queries' type. E4M3: the cache holds that instead. D: head_dim rounded up to 64, 128, 256;
// EXACT: it is D.
template <class T, bool E4M3, int D, bool EXACT>
__global__ __launch_bounds__(kThreads) void decode_kernel(const DecodeParams p) {
  constexpr int CB = E4M3 ? 1 : 2;                         // bytes of a cached element
  constexpr int KP = D * CB / 64;                          // 16-byte pieces of a K row per lane
  constexpr int VP = D / 16 < 16 / CB ? D / 16 : 16 / CB;  // elements of a V piece
  constexpr int NP = D / 16 / VP;                          // V pieces per row and lane
  constexpr int VW = VP * CB / 4;                          // words of a V piece
  constexpr int NA = NP * VP;                              // accumulators: 16 dims each
  extern __shared__ float lds[];

  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t col = lane & 15u, kg = lane >> 4;
  const uint32_t kv_head = blockIdx.x / p.head_tiles, tile = blockIdx.x - kv_head * p.head_tiles;
  const uint32_t split = blockIdx.y, seq = blockIdx.z;
  const uint32_t head0 = kv_head * p.group + tile * 16u;
  const uint32_t n_heads = p.group - tile * 16u < 16u ? p.group - tile * 16u : 16u;
  const uint32_t dim = EXACT ? D : p.head_dim;

  // the tokens this sequence sees, and this workgroup's share of them
  const int32_t raw_len = p.lens[seq];
  const uint32_t len = raw_len <= 0 ? 0u
                       : static_cast<uint64_t>(raw_len) < p.visible_max ? static_cast<uint32_t>(raw_len)
                                                                        : static_cast<uint32_t>(p.visible_max);
  const uint32_t start = p.window != 0 && len > p.window ? len - p.window : 0u;
  const uint32_t first = start & ~(kTile - 1);
  uint32_t chunk = (len - first + p.splits - 1) / p.splits;
  chunk = (chunk + kStep - 1) / kStep * kStep;
  if (chunk < p.chunk) chunk = p.chunk;
  const uint32_t parts = len == 0 ? 1u : (len - first + chunk - 1) / chunk;
  if (split >= parts) return;
  const uint32_t begin = first + split * chunk;
  const uint32_t end = len - begin < chunk ? len : begin + chunk;

  // queries: lane = head, the same numbering of the dims as the pieces of K
  u32x4 qf[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    const uint32_t d = E4M3 ? (c / 2) * 64u + kg * 16u + (c & 1) * 8u : c * 32u + kg * 8u;
    u32x4 v = {0, 0, 0, 0};
    if (col < n_heads && (EXACT || d < dim)) {
      const uint8_t* a = p.q + seq * p.q_token + (head0 + col) * p.q_head + d * 2u;
      if (p.q_vec) {
        v = *reinterpret_cast<const u32x4*>(a);
      } else {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(a);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = h[2 * j] | static_cast<uint32_t>(h[2 * j + 1]) << 16;
      }
    }
    qf[c] = v;
  }

  const uint8_t* kbase = p.base + kv_head * p.head_stride;
  const uint8_t* vbase = kbase + p.kv_stride;
  const int32_t* table = p.tables + seq * p.table_stride;

  f32x4 acc[NA];
#pragma unroll
  for (int x = 0; x < NA; ++x) acc[x] = f32x4{0, 0, 0, 0};
  float top = -INFINITY, sum = 0.0f;
  bool any = false;

  for (uint32_t t0 = begin + wave * kTile; t0 < end; t0 += kStep) {
    // where the tile's 32 rows lie: lane's column is token col and 16 + col
    int64_t off[2];
    uint32_t seen = 0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint32_t t = t0 + s * 16u + col;
      bool valid = t >= start && t < end;
      const uint32_t page = divided(t, p.block_magic);
      const int32_t block = valid ? table[page] : -1;
      valid = static_cast<uint32_t>(block) < p.n_blocks;
      // a token that is not seen reads the cache's first row and takes no part below
      off[s] = valid ? block * p.block_stride + (t - page * p.ntpb) * p.token_stride : 0;
      seen |= static_cast<uint32_t>(__ballot(valid) & 0xFFFFu) << (16 * s);
    }
    any = any || seen != 0;

    u32x4 kr[2][KP];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int c = 0; c < KP; ++c) {
        const uint32_t at = c * 64u + kg * 16u;
        kr[s][c] = EXACT || at < dim * CB ? *reinterpret_cast<const u32x4*>(kbase + off[s] + at) : u32x4{0, 0, 0, 0};
      }
    // V: the eight tokens whose weights this lane will hold, 4 kg ... + 3 of both halves
    uint32_t vr[8][NP][VW];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t o = __shfl(off[i >> 2], kg * 4 + (i & 3));
#pragma unroll
      for (int h = 0; h < NP; ++h) {
        const uint32_t d = (h * 16u + col) * VP;
        const uint8_t* a = vbase + o + d * CB;
        const bool in = EXACT || d < dim;
        if constexpr (VW == 4) {
          const u32x4 v = in ? *reinterpret_cast<const u32x4*>(a) : u32x4{0, 0, 0, 0};
          vr[i][h][0] = v.x, vr[i][h][1] = v.y, vr[i][h][2] = v.z, vr[i][h][3] = v.w;
        } else if constexpr (VW == 2) {
          const u32x2 v = in ? *reinterpret_cast<const u32x2*>(a) : u32x2{0, 0};
          vr[i][h][0] = v.x, vr[i][h][1] = v.y;
        } else {
          vr[i][h][0] = in ? *reinterpret_cast<const uint32_t*>(a) : 0u;
        }
      }
    }

    // scores
    f32x4 sc[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      sc[s] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < KP; ++c) {
        if constexpr (E4M3) {
          const u32x4 w = kr[s][c];
          const u32x4 a = {T::template widen<false>(w.x), T::template widen<true>(w.x),
                           T::template widen<false>(w.y), T::template widen<true>(w.y)};
          const u32x4 b = {T::template widen<false>(w.z), T::template widen<true>(w.z),
                           T::template widen<false>(w.w), T::template widen<true>(w.w)};
          sc[s] = T::mma(a, qf[2 * c], sc[s]);
          sc[s] = T::mma(b, qf[2 * c + 1], sc[s]);
        } else {
          sc[s] = T::mma(kr[s][c], qf[c], sc[s]);
        }
      }
    }
    float high = -INFINITY;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v = sc[s][r] * p.scale_log2;
        if (p.cap != 0.0f) v = p.cap * tanhf(sc[s][r] * p.cap_in);
        v = (seen >> (16 * s + 4 * kg + r)) & 1u ? v : -INFINITY;
        sc[s][r] = v;
        high = fmaxf(high, v);
      }
    high = fmaxf(over_tokens_max(high), top);
    if (__any(high != top)) {
      // a head with nothing but minus infinity so far: exp2(-inf - 0) = 0 below
      const float shrink = __builtin_amdgcn_exp2f(top - (high == -INFINITY ? 0.0f : high));
      sum *= shrink;
#pragma unroll
      for (int x = 0; x < NA; ++x) acc[x] *= shrink;
      top = high;
    }
    const float ref = high == -INFINITY ? 0.0f : high;
    u32x4 ph, pl;   // weights cut off, and what that left
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const float a = __builtin_amdgcn_exp2f(sc[s][r] - ref), b = __builtin_amdgcn_exp2f(sc[s][r + 1] - ref);
        sum += a + b;
        const uint32_t hi = T::cut(a, b);
        const f32x2 kept = __builtin_convertvector(__builtin_bit_cast(typename T::x2, hi), f32x2);
        const f32x2 left = {fmaxf(a - kept.x, T::kLeast), fmaxf(b - kept.y, T::kLeast)};
        ph[s * 2 + r / 2] = hi;
        pl[s * 2 + r / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(left, typename T::x2));
      }

    if (seen != 0xFFFFFFFFu) {
      // rows that are not seen may hold anything, and zero times anything is not zero
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (!((seen >> (16 * (i >> 2) + 4 * kg + (i & 3))) & 1u))
#pragma unroll
          for (int h = 0; h < NP; ++h)
#pragma unroll
            for (int w = 0; w < VW; ++w) vr[i][h][w] = 0;
    }
#pragma unroll
    for (int h = 0; h < NP; ++h)
#pragma unroll
      for (int w = 0; w < VP / 2; ++w) {   // two dims at a time
        uint32_t x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (E4M3)
            x[i] = w & 1 ? T::template widen<true>(vr[i][h][w / 2]) : T::template widen<false>(vr[i][h][w / 2]);
          else
            x[i] = vr[i][h][w];
        }
        u32x4 even, odd;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          even[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x05040100u);
          odd[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x07060302u);
        }
        f32x4& a = acc[h * VP + 2 * w];
        f32x4& b = acc[h * VP + 2 * w + 1];
        a = T::mma(even, ph, a);
        b = T::mma(odd, ph, b);
        a = T::mma(even, pl, a);
        b = T::mma(odd, pl, b);
      }
  }

  // the four wavefronts' parts meet in LDS: [wave][head][dim], rows 4 floats apart from a
  // multiple of the banks
  constexpr uint32_t kRow = D + 4;
  float* part = lds;
  Stat* stats = reinterpret_cast<Stat*>(lds + kWaves * n_heads * kRow);   // [wave][16]
  sum = over_tokens_sum(sum);
  if (sum == 0.0f && any) sum = -1.0f;
  if (kg == 0) stats[wave * 16 + col] = Stat{top, sum};
  if (col < n_heads) {
    float* row = part + (wave * n_heads + col) * kRow;
#pragma unroll
    for (int h = 0; h < NP; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int x = 0; x < VP; x += 4) {
          const f32x4 v = {acc[h * VP + x][r], acc[h * VP + x + 1][r], acc[h * VP + x + 2][r], acc[h * VP + x + 3][r]};
          *reinterpret_cast<f32x4*>(row + (h * 16 + kg * 4 + r) * VP + x) = v;
        }
  }
  __syncthreads();

  const uint32_t quads = dim / 4, work = n_heads * quads;
  const auto finish = [&](uint32_t head, uint32_t d, f32x4 o, float m, float l, bool nothing_but_inf) {
    const float inv = l == 0.0f ? (nothing_but_inf ? NAN : 0.0f) : p.v_scale / l;
    uint8_t* a = p.out + seq * p.out_token + (head0 + head) * p.out_head + d * 2u;
    o *= inv;
    const f32x2 lo = {o.x, o.y}, hi = {o.z, o.w};
    const u32x2 w = {__builtin_bit_cast(uint32_t, __builtin_convertvector(lo, typename T::x2)),
                     __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, typename T::x2))};
    if (p.out_vec) {
      *reinterpret_cast<u32x2*>(a) = w;
    } else {
      uint16_t* h = reinterpret_cast<uint16_t*>(a);
      h[0] = w.x, h[1] = w.x >> 16, h[2] = w.y, h[3] = w.y >> 16;
    }
    if (d == 0 && p.lse)
      p.lse[static_cast<uint64_t>(seq) * p.n_heads + head0 + head] =
          l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
  };
  const uint64_t row0 = (static_cast<uint64_t>(seq) * p.n_heads + head0) * p.splits;
  for (uint32_t n = threadIdx.x; n < work; n += kThreads) {
    const uint32_t head = n / quads, d = (n - head * quads) * 4;
    float m = -INFINITY, l = 0.0f;
    bool inf = false;
    f32x4 o = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, stats[w * 16 + head].max);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const Stat s = stats[w * 16 + head];
      const float f = weight_of(s, m);
      inf = inf || s.sum < 0.0f;
      if (f != 0.0f) {
        l += f * s.sum;
        o += f * *reinterpret_cast<const f32x4*>(part + (w * n_heads + head) * kRow + d);
      }
    }
    if (parts == 1) {
      finish(head, d, o, m, l, inf);
    } else {
      const uint64_t row = row0 + head * p.splits + split;
      *reinterpret_cast<f32x4*>(p.part_o + row * dim + d) = o;
      if (d == 0) p.part_ml[row] = make_float2(m, l == 0.0f && inf ? -1.0f : l);
    }
  }
  if (parts == 1) return;

  // the last workgroup of this group of heads to get here joins the parts, in their order
  uint32_t* counter = p.counters + static_cast<uint64_t>(seq) * gridDim.x + blockIdx.x;
  __threadfence();
  __syncthreads();
  uint32_t* arrived = reinterpret_cast<uint32_t*>(lds);
  if (threadIdx.x == 0)
    *arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  const bool last = *arrived == parts - 1;
  if (!last) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) *counter = 0;   // as the next launch on this workspace wants to find it
  float2* ml = reinterpret_cast<float2*>(lds);   // [head][part]
  for (uint32_t n = threadIdx.x; n < n_heads * parts; n += kThreads) {
    const uint32_t head = n / parts, s = n - head * parts;
    ml[n] = p.part_ml[row0 + head * p.splits + s];
  }
  __syncthreads();
  for (uint32_t n = threadIdx.x; n < work; n += kThreads) {
    const uint32_t head = n / quads, d = (n - head * quads) * 4;
    const float2* mine = ml + head * parts;
    float m = -INFINITY, l = 0.0f;
    bool inf = false;
    for (uint32_t s = 0; s < parts; ++s) m = fmaxf(m, mine[s].x);
    f32x4 o = {0, 0, 0, 0};
    const float* src = p.part_o + (row0 + head * p.splits) * dim + d;
    for (uint32_t s = 0; s < parts; ++s) {
      const Stat st = {mine[s].x, mine[s].y};
      const float f = weight_of(st, m);
      inf = inf || st.sum < 0.0f;
      if (f != 0.0f) {
        l += f * st.sum;
        o += f * *reinterpret_cast<const f32x4*>(src + static_cast<uint64_t>(s) * dim);
      }
    }
    finish(head, d, o, m, l, inf);
  }
}

struct Launch {
  dim3 grid;
  uint32_t lds;
  hipStream_t stream;
};

template <class T, bool E4M3, int D>
void launch_exact(const DecodeParams& p, const Launch& l) {
  if (p.head_dim == D)
    decode_kernel<T, E4M3, D, true><<<l.grid, kThreads, l.lds, l.stream>>>(p);
  else
    decode_kernel<T, E4M3, D, false><<<l.grid, kThreads, l.lds, l.stream>>>(p);
}

template <class T, bool E4M3>
void launch_dim(const DecodeParams& p, const Launch& l) {
  if (p.head_dim <= 64)
    launch_exact<T, E4M3, 64>(p, l);
  else if (p.head_dim <= 128)
    launch_exact<T, E4M3, 128>(p, l);
  else
    launch_exact<T, E4M3, 256>(p, l);
}

// Workgroups a split launch aims at: 8 of 4 wavefronts on each of the 256 CUs. A part is at
// least kMinPart tokens and need not be longer than kMaxPart.
constexpr uint32_t kAimWgs = 2048, kMinPart = kStep, kMaxPart = 2048;
// Rows (of one head and part) that a workspace has room for, at most.
constexpr uint64_t kMaxRowsPerHead = 4096;

}  // namespace
}  // namespace kvt

using namespace kvt;

// Sums and statistics of split launches live in a workspace; two launches that may run at the
// same time must not share one. Launches on one stream never do run at the same time, and neither
// do those recorded into one capture on one stream, so a workspace belongs to a stream (eager
// launches) or to a capture and its stream, from the first launch there on.
struct kvt_decode {
  int device = 0;
  kvt_kv_layout layout{};
  uint64_t extent = 0;
  uint32_t dtype = 0, n_heads = 0, group = 0, head_tiles = 0, window = 0, max_seqs = 0;
  float scale = 0, cap = 0;
  uint64_t rows = 0, ws_bytes = 0;
  uint8_t* arena = nullptr;
  struct Owner {
    bool taken = false;
    hipStream_t stream = nullptr;
    unsigned long long capture = 0;     // 0: eager
    std::thread::id thread;             // of a per-thread default stream
  };
  std::mutex mu;
  std::vector<Owner> owners;

  uint64_t ml_at() const { return round_up(rows * layout.head_dim * 4ull, 256); }
  uint64_t counters_at() const { return round_up(ml_at() + rows * 8ull, 256); }

  int workspace(hipStream_t s, unsigned long long capture, uint8_t** out) {
    const std::thread::id me = s == hipStreamPerThread ? std::this_thread::get_id() : std::thread::id();
    std::lock_guard<std::mutex> lock(mu);
    size_t free = owners.size();
    for (size_t i = 0; i < owners.size(); ++i) {
      const Owner& o = owners[i];
      if (!o.taken) {
        if (free == owners.size()) free = i;
      } else if (o.stream == s && o.capture == capture && o.thread == me) {
        *out = arena + i * ws_bytes;
        return KVT_OK;
      }
    }
    if (free == owners.size())
      return fail(KVT_ERR_INVALID, "kvt_decode_attention: other streams and captures hold all " +
                                       std::to_string(owners.size()) +
                                       " workspaces (kvt_decode_create's n_workspaces, kvt_decode_release)");
    owners[free] = Owner{true, s, capture, me};
    *out = arena + free * ws_bytes;
    return KVT_OK;
  }
};

extern "C" {

int kvt_decode_create(int device, const kvt_kv_layout* layout, uint32_t dtype, uint32_t n_q_heads,
                      float softmax_scale, float logit_cap, uint32_t window, uint32_t max_seqs,
                      uint32_t n_workspaces, kvt_decode** out) {
  return guarded([&]() -> int {
    static const char* who = "kvt_decode_create";
    if (!out) return fail(KVT_ERR_INVALID, "kvt_decode_create: null argument");
    std::unique_ptr<kvt_decode> d(new kvt_decode());
    if (int rc = check_kv_layout(layout, who, &d->extent)) return rc;
    if (dtype != KVT_DTYPE_BF16 && dtype != KVT_DTYPE_F16)
      return fail(KVT_ERR_UNSUPPORTED, "kvt_decode_create: queries are bf16 or f16");
    if (layout->dtype != KVT_DTYPE_E4M3 && layout->dtype != dtype)
      return fail(KVT_ERR_UNSUPPORTED, "kvt_decode_create: the cache holds the queries' own type or e4m3");
    if (n_q_heads == 0 || n_q_heads % layout->n_kv_heads != 0 || n_q_heads > 65536)
      return fail(KVT_ERR_INVALID, "kvt_decode_create: the query heads must be a multiple of the KV heads, at most 65536");
    if (!std::isfinite(softmax_scale) || !std::isfinite(logit_cap) || logit_cap < 0)
      return fail(KVT_ERR_INVALID, "kvt_decode_create: bad softmax_scale or logit_cap");
    if (max_seqs == 0 || max_seqs > 65535 || n_workspaces == 0 || n_workspaces > 1024)
      return fail(KVT_ERR_INVALID, "kvt_decode_create: max_seqs must be in [1, 65535], n_workspaces in [1, 1024]");
    if (int rc = check_device(device)) return rc;
    d->device = device;
    d->layout = *layout;
    d->dtype = dtype;
    d->n_heads = n_q_heads;
    d->group = n_q_heads / layout->n_kv_heads;
    d->head_tiles = (d->group + 15) / 16;
    d->window = window;
    d->max_seqs = max_seqs;
    d->scale = softmax_scale != 0 ? softmax_scale : 1.0f / std::sqrt(static_cast<float>(layout->head_dim));
    d->cap = logit_cap;
    d->rows = std::min<uint64_t>(kMaxRowsPerHead * std::min(d->group, 16u),
                                 static_cast<uint64_t>(max_seqs) * n_q_heads * kMaxSplits);
    const uint64_t counters = static_cast<uint64_t>(max_seqs) * layout->n_kv_heads * d->head_tiles;
    d->ws_bytes = round_up(d->counters_at() + counters * 4, 256);
    d->owners.resize(n_workspaces);
    DeviceGuard g;
    if (int rc = g.enter(device)) return rc;
    KVT_HIP(hipMalloc(reinterpret_cast<void**>(&d->arena), d->ws_bytes * n_workspaces));
    // the counters start at zero and every launch leaves them so
    for (uint32_t i = 0; i < n_workspaces; ++i) {
      const hipError_t e = hipMemset(d->arena + i * d->ws_bytes + d->counters_at(), 0, counters * 4);
      if (e != hipSuccess) {
        (void)hipFree(d->arena);
        return hip_fail(e, "hipMemset(decode workspace)");
      }
    }
    const hipError_t e = hipDeviceSynchronize();
    if (e != hipSuccess) {
      (void)hipFree(d->arena);
      return hip_fail(e, "hipDeviceSynchronize");
    }
    *out = d.release();
    return KVT_OK;
  });
}

void kvt_decode_destroy(kvt_decode* d) {
  if (!d) return;
  DeviceGuard g;
  if (g.enter(d->device) == KVT_OK) {
    forget_device_spans();
    if (d->arena) (void)hipFree(d->arena);
  }
  delete d;
}

int kvt_decode_release(kvt_decode* d, void* stream) {
  if (!d) return fail(KVT_ERR_INVALID, "kvt_decode_release: null argument");
  std::lock_guard<std::mutex> lock(d->mu);
  for (kvt_decode::Owner& o : d->owners)
    if (o.taken && o.stream == static_cast<hipStream_t>(stream)) o = kvt_decode::Owner{};
  return KVT_OK;
}

int kvt_decode_attention(kvt_decode* d, const kvt_cache* cache, uint32_t layer, const void* q,
                         uint64_t q_token_stride, uint64_t q_head_stride, const int32_t* block_tables,
                         uint64_t table_stride, uint32_t table_blocks, const int32_t* seq_lens,
                         uint32_t n_seqs, uint64_t max_len, float k_scale, float v_scale, void* out,
                         uint64_t out_token_stride, uint64_t out_head_stride, float* lse, void* stream) {
  return guarded([&]() -> int {
    static const char* who = "kvt_decode_attention";
    if (!d) return fail(KVT_ERR_INVALID, "kvt_decode_attention: null argument");
    uint8_t* base = nullptr;
    if (int rc = check_cache_layer(cache, layer, &d->layout, d->extent, who, &base)) return rc;
    if (cache->device != d->device) return fail(KVT_ERR_INVALID, "kvt_decode_attention: the cache is on another device");
    if (n_seqs > d->max_seqs) return fail(KVT_ERR_INVALID, "kvt_decode_attention: more sequences than max_seqs");
    const bool e4m3 = d->layout.dtype == KVT_DTYPE_E4M3;
    if (!std::isfinite(k_scale) || !std::isfinite(v_scale) || !(k_scale > 0) || !(v_scale > 0) ||
        (!e4m3 && (k_scale != 1.0f || v_scale != 1.0f)))
      return fail(KVT_ERR_INVALID, "kvt_decode_attention: scales must be positive, and 1 for a 16-bit cache");
    const uint32_t dim = d->layout.head_dim;
    const Rows qr{q, q_token_stride, q_head_stride}, outr{out, out_token_stride, out_head_stride};
    uint64_t q_span = 0, out_span = 0;
    if (int rc = check_rows(qr, n_seqs, d->n_heads, dim * 2ull, 2, false, who, "q", &q_span)) return rc;
    if (int rc = check_rows(outr, n_seqs, d->n_heads, dim * 2ull, 2, true, who, "out", &out_span)) return rc;
    if (int rc = check_apart(qr, d->n_heads, outr, d->n_heads, n_seqs, dim * 2ull, false, who, "q")) return rc;
    if (n_seqs == 0) return KVT_OK;
    if (!seq_lens || (reinterpret_cast<uintptr_t>(seq_lens) & 3u) || (reinterpret_cast<uintptr_t>(lse) & 3u) ||
        (table_blocks != 0 && (!block_tables || (reinterpret_cast<uintptr_t>(block_tables) & 3u))))
      return fail(KVT_ERR_INVALID, "kvt_decode_attention: tables, lengths or lse are null or not aligned");
    if (table_stride > (1ull << 40)) return fail(KVT_ERR_INVALID, "kvt_decode_attention: table_stride out of range");
    DeviceGuard g;
    if (int rc = g.enter(d->device)) return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    unsigned long long capture = 0;
    if (hipStreamIsCapturing(s, &cap) != hipSuccess) (void)hipGetLastError();
    if (cap == hipStreamCaptureStatusNone) {
      if (int rc = check_device_span(q, q_span, "kvt_decode_attention: q")) return rc;
      if (int rc = check_device_span(out, out_span, "kvt_decode_attention: out")) return rc;
      if (int rc = check_device_span(seq_lens, 4ull * n_seqs, "kvt_decode_attention: seq_lens")) return rc;
      if (int rc = check_device_span(block_tables, table_blocks ? 4 * ((n_seqs - 1) * table_stride + table_blocks) : 0,
                                     "kvt_decode_attention: block_tables"))
        return rc;
      if (lse)
        if (int rc = check_device_span(lse, 4ull * n_seqs * d->n_heads, "kvt_decode_attention: lse")) return rc;
    } else if (hipStreamGetCaptureInfo(s, &cap, &capture) != hipSuccess || capture == 0) {
      (void)hipGetLastError();
      return fail(KVT_ERR_HIP, "kvt_decode_attention: the stream's capture cannot be told apart");
    }

    DecodeParams p{};
    p.base = base;
    p.block_stride = d->layout.block_stride, p.kv_stride = d->layout.kv_stride;
    p.token_stride = d->layout.token_stride, p.head_stride = d->layout.head_stride;
    p.q = static_cast<const uint8_t*>(q), p.q_token = q_token_stride, p.q_head = q_head_stride;
    p.tables = block_tables, p.table_stride = table_stride;
    p.lens = seq_lens;
    p.out = static_cast<uint8_t*>(out), p.out_token = out_token_stride, p.out_head = out_head_stride;
    p.lse = lse;
    p.block_magic = division_magic(d->layout.ntpb);
    p.visible_max = std::min<uint64_t>(static_cast<uint64_t>(table_blocks) * d->layout.ntpb, 0x7FFFFFFFull);
    p.ntpb = d->layout.ntpb, p.n_blocks = static_cast<uint32_t>(d->layout.n_blocks);
    p.n_heads = d->n_heads, p.group = d->group, p.head_tiles = d->head_tiles, p.head_dim = dim, p.window = d->window;
    const float scale = d->scale * k_scale;
    p.scale_log2 = scale * kLog2e;
    p.cap = d->cap * kLog2e, p.cap_in = d->cap != 0 ? scale / d->cap : 0;
    p.v_scale = v_scale;
    p.q_vec = rows_aligned16(qr);
    p.out_vec = ((reinterpret_cast<uintptr_t>(out) | out_token_stride | out_head_stride) & 7u) == 0;

    // how far to split: max_len is the caller's word and decides nothing but speed
    uint64_t longest = max_len == 0 || max_len > p.visible_max ? p.visible_max : max_len;
    if (d->window != 0) longest = std::min<uint64_t>(longest, d->window + kTile);
    const uint64_t groups = static_cast<uint64_t>(d->layout.n_kv_heads) * d->head_tiles;
    uint64_t chunk = longest * n_seqs * groups / kAimWgs;
    chunk = round_up(std::min<uint64_t>(std::max<uint64_t>(chunk, kMinPart), kMaxPart), kStep);
    uint64_t splits = std::max<uint64_t>(1, (longest + chunk - 1) / chunk);
    splits = std::min<uint64_t>(splits, kMaxSplits);
    splits = std::max<uint64_t>(1, std::min<uint64_t>(splits, d->rows / (static_cast<uint64_t>(n_seqs) * d->n_heads)));
    p.chunk = static_cast<uint32_t>(chunk), p.splits = static_cast<uint32_t>(splits);
    if (splits > 1) {
      uint8_t* ws = nullptr;
      if (int rc = d->workspace(s, capture, &ws)) return rc;
      p.part_o = reinterpret_cast<float*>(ws);
      p.part_ml = reinterpret_cast<float2*>(ws + d->ml_at());
      p.counters = reinterpret_cast<uint32_t*>(ws + d->counters_at());
    }
    const uint32_t heads = std::min(d->group, 16u), full = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
    const uint32_t meet = kWaves * (heads * (full + 4) * 4 + 16 * static_cast<uint32_t>(sizeof(Stat)));
    const Launch l{dim3(static_cast<uint32_t>(groups), p.splits, n_seqs),
                   std::max<uint32_t>(meet, splits > 1 ? heads * p.splits * static_cast<uint32_t>(sizeof(float2)) : 0), s};
    if (d->dtype == KVT_DTYPE_BF16) {
      if (e4m3) launch_dim<Bf16, true>(p, l);
      else launch_dim<Bf16, false>(p, l);
    } else {
      if (e4m3) launch_dim<F16, true>(p, l);
      else launch_dim<F16, false>(p, l);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return hip_fail(e, who);
    return KVT_OK;
  });
}

}  // extern "C"
