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
// matrix instructions in a kernel that is bound by HBM. Both values are at least the smallest
// positive number, so that an infinity in V times a weight is that infinity, as in the formula, and
// neither the difference of two nor zero times one. For f16 the weights are taken times 2^16, which
// makes its smallest positive number 2^-40 of the largest weight: 2^-24 of it, for each of the many
// small weights of a long sequence in which one token stands out, would add up to more than the
// output's own rounding. (The largest weights, cut off to f16's largest number of 65504, leave the rest
// of 65536 as any other.) For bf16 rows they are taken times the power of two next below 1 / length,
// so that no sum over the tokens leaves 32 bits, whatever V holds.
//
// An 8-bit cache is widened on load: every e4m3 value is a bf16 and an f16 value.
//
// Bound by HBM once a launch has some ten microseconds of rows to read. The formula has 2 operations
// per cached element and query head; the products do 2 per element of K and 4 per element of V for 16
// heads at a time, whether there are as many or not: 24 a byte of a 16-bit cache, 48 of an 8-bit one, for
// every 16 query heads that share a KV head, against the 178 a byte at which the matrix units would take
// over (more than 112 heads, or 48). What the rest of this file is about is keeping enough reads in
// flight from every CU, and leaving nothing but reads between the first row and the last:
//   shares   the units of 128 tokens of all sequences, one list, cut into as many equal shares as
//            workgroups are resident, wherever that falls: no workgroup waits for a longer one, no second
//            wave of workgroups starts (one and a half to four times as many: 131071 tokens 94 -> 100-120
//            us, 128 x 4096 of 256 160 -> 174-187). Every wavefront finds its share itself from the
//            lengths (a scan, 1 us), so lengths stay on the device and a captured launch serves any.
//   joins    a row that is split is joined by whichever workgroup is last, in the parts' order (the same
//            bits each time). Parts are written through and read past the L2s (sc1) and counted by one
//            relaxed atomic: a device-wide fence per workgroup, which writes back and drops whole L2s,
//            took 543 us where this takes 292 (64 x 1k-8k tokens, the form before K went through LDS).
//   K        by whole rows through LDS, without passing registers: reading 64-byte pieces of 16 rows
//            straight into the matrix operand took 225 us (195), 178 (160) for 256 f16. V stays in
//            registers, transposed by byte permutes; through LDS as well it gains nothing (196).
//   ahead    the next tile's rows are asked for before this one's are used up, the block ids of the one
//            behind before that. Loads are non-temporal: plain ones 230 us (219), 134 (118) for one
//            long sequence (both before K went through LDS).
// Microseconds, and TB/s of the bytes a launch cannot do without, where a 1 GiB copy reaches 6.6: 64
// sequences of 1k-8k tokens, 32 heads on 8 of 128 bf16, 182 (6.4); 128 of 4096, 16 on 2 of 256 f16, 160 (6.7);
// one of 131071, 64 on 8 of 128 bf16 HND, 93 (5.8: 4 us to the first rows, 10 for the join of 64 parts);
// 96 of 1-16384, 16 on 2 of 128 e4m3, 75 (5.2: the same, and the vector units 40 % busy with widening); one of 512, 9.0
// (one round trip after another: lengths 1, table 2, rows 1.3, the wavefronts' join 0.4, parts out 1.3, the
// count 0.4, parts in 2).
#include <hip/hip_runtime.h>

#include <cmath>
#include <thread>

#include "kvt_ops.h"

namespace kvt {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256, kWaves = 4;
constexpr uint32_t kTile = 32;                   // tokens a wavefront takes at a time
constexpr uint32_t kStep = kTile * kWaves;       // ... and a workgroup
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
  float* part_o;       // [workgroup][first, last, joined][head][head_dim]: sums not yet divided
  float2* part_ml;     // [workgroup][first, last, joined][head]: maximum (times log2 e), sum
  uint32_t* counters;  // [step][workgroup]: parts, of those that begin with its own, that have been left
  uint64_t block_magic;
  uint32_t visible_max, ntpb, n_blocks, n_seqs, n_heads, head_dim, window;
  uint32_t group, spread, head_rows, rows, teams, slot_heads;
  float scale_log2, cap, cap_in, v_scale;
  bool q_vec, out_vec, abreast;
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
  // two values cut off to this type, its smallest positive number (here of the normal ones) and
  // the bits of two of them, and what the largest weight of a sequence is in the product with V
  static __device__ __forceinline__ uint32_t cut(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
  }
  template <bool E4M3>
  static __device__ __forceinline__ float top(uint32_t len) {
    return E4M3 ? 1.0f : __uint_as_float((95u + __builtin_clz(len)) << 23);
  }
  static constexpr float kLeast = 0x1p-126f;
  static constexpr uint32_t kLeastTwice = 0x00800080u;
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
  template <bool E4M3>
  static __device__ __forceinline__ float top(uint32_t) { return 0x1p16f; }
  static constexpr float kLeast = 0x1p-24f;
  static constexpr uint32_t kLeastTwice = 0x00010001u;
};

// N pieces of 16 bytes from LDS, once all but the newest `NEWER` vector memory operations are done:
// what loads that go to LDS have written is not there before, and the compiler, which does not tell
// their targets apart, would wait for every load there is.
template <int N, int NEWER>
__device__ __forceinline__ void read_k(const uint32_t* at, int offset, u32x4* r) {
  if constexpr (N == 1) {
    if (offset == 0)
      asm volatile("s_waitcnt vmcnt(%2)\n\tds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(r[0]) : "v"(at[0]), "n"(NEWER) : "memory");
    else
      asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(r[0]) : "v"(at[0] + offset) : "memory");
  } else if constexpr (N == 2) {
    if (offset == 0)
      asm volatile("s_waitcnt vmcnt(%4)\n\tds_read_b128 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)"
                   : "=&v"(r[0]), "=&v"(r[1]) : "v"(at[0]), "v"(at[1]), "n"(NEWER) : "memory");
    else
      asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)"
                   : "=&v"(r[0]), "=&v"(r[1]) : "v"(at[0] + offset), "v"(at[1] + offset) : "memory");
  } else {
#pragma unroll
    for (int n = 0; n < N; n += 4) {
      if (offset == 0 && n == 0)
        asm volatile("s_waitcnt vmcnt(%8)\n\tds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %6\n\t"
                     "ds_read_b128 %3, %7\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
                     : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(NEWER) : "memory");
      else
        asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %6\n\t"
                     "ds_read_b128 %3, %7\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(r[n]), "=&v"(r[n + 1]), "=&v"(r[n + 2]), "=&v"(r[n + 3])
                     : "v"(at[n] + offset), "v"(at[n + 1] + offset), "v"(at[n + 2] + offset), "v"(at[n + 3] + offset) : "memory");
    }
  }
}

// The maximum / sum over the four lanes that hold one head's tokens (lane, +16, +32, +48).
// Both operands of a swap are the value: what comes back are its even and its odd rows (of 16, of
// 32 lanes), each in both places.
__device__ __forceinline__ float over_tokens_max(float v) {
  const uint32_t a = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  const uint32_t b = __float_as_uint(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
  const auto q = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float over_tokens_sum(float v) {
  const uint32_t a = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  const uint32_t b = __float_as_uint(__uint_as_float(r[0]) + __uint_as_float(r[1]));
  const auto q = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

// Cache policies of the buffer instructions: bit 1 = non-temporal (rows of the cache are read
// once), bit 4 = sc1, the scope of the device.
constexpr int kStreamed = 2, kShared = 16;
template <class V>
__device__ __forceinline__ V streamed(const uint8_t* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
}

// Parts of split sequences pass from one workgroup to another, on whatever XCD: written through
// to, and read from, where all XCDs see them (sc1: the scope of the device).
typedef __amdgpu_buffer_rsrc_t rsrc_t;
constexpr uint32_t kNowhere = 0xFFFFF000u;   // the end of every buffer
__device__ __forceinline__ rsrc_t rsrc_of(void* base) {
  return __builtin_amdgcn_make_buffer_rsrc(base, 0, kNowhere, 0x00020000);
}

__device__ __forceinline__ uint64_t uniform(uint64_t v) {
  return static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32))) << 32 |
         __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
}

// 16 bytes per lane from rows + at to LDS, the lanes' pieces one after the other from `to` on.
__device__ __forceinline__ void load_to_lds(rsrc_t rows, uint32_t at, __attribute__((address_space(3))) void* to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rows, to, 16, at, 0, 0, kStreamed);
}

// Uniform reads through the scalar cache.
typedef __attribute__((address_space(4))) const int32_t* constant_t;
__device__ __forceinline__ constant_t constant(const int32_t* p) { return (constant_t)(p); }

// Tokens that a sequence of this length may see, and the units that they take.
__device__ __forceinline__ uint32_t seen_of(const DecodeParams& p, int32_t len) {
  const uint32_t n = len < 0 ? 0u : static_cast<uint32_t>(len);
  return n < p.visible_max ? n : p.visible_max;
}
__device__ __forceinline__ uint32_t units_of(const DecodeParams& p, int32_t raw) {
  const uint32_t len = seen_of(p, raw), start = p.window != 0 && len > p.window ? len - p.window : 0u;
  return (len - (start & ~(kTile - 1)) + kStep - 1) / kStep;
}

// A row's parts are joined in two steps where they are more than kFan and, together, more than kAlone float4s: one
// workgroup reads some 25 GB/s of them. One / two steps, microseconds: 2 sequences of 65000, 64 heads on one of
// 128, 212 / 68 (their rows take 10 at the rate of a copy: it is the join that bounds such launches); one of 131071,
// 128 on 8 of 128 (64 parts of 512) 127 / 108; 4 of 9343, 32 on 2 of 192 (33 of 768) 31.1 / 30.0 (not kept for such
// heads; rows 9); but 64 parts of 256 92.4 / 93.5, 16 of 384 15.4 / 16.1. The code of it slows launches
// that do not need it (e4m3 74.2 / 75.6, 512 tokens 9.1 / 9.8), so that it is a kernel of its own, taken where
// equally long sequences would be split that far; each of the two is right for any lengths.
constexpr uint32_t kFan = 8, kAlone = 20480;
// One part's statistics of a head. sum < 0 stands for "scores were there, all of them minus
// infinity": that softmax is NaN, while a head that saw no token at all gives zeros.
struct Stat {
  float max, sum;
};
// (the maximum passes over NaN: a part of nothing but NaN has no maximum, and a NaN sum)
__device__ __forceinline__ float weight_of(const Stat& s, float top) {
  return s.max != -INFINITY ? __builtin_amdgcn_exp2f(s.max - top) : s.sum != s.sum ? s.sum : 0.0f;
}
// What sums of V are multiplied with for a weight: never zero, which would make an infinity NaN. One in a
// row that is seen then comes through wherever the sequence is split, as it does within a tile. (A NaN weight
// ends here, and makes the row NaN by its sum.)
__device__ __forceinline__ float carried(float weight) { return fmaxf(weight, 0x1p-126f); }

// The launch's arguments, loaded where this is called and not kept in registers from the start.
typedef __attribute__((address_space(4))) const DecodeParams* params_t;
__device__ __forceinline__ params_t arguments() {
  uint64_t at = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
  asm volatile("" : "+s"(at));
  return (params_t)at;
}

enum { kWhole, kNear, kFar };

// Workgroups of a launch, per CU: what is resident at once. Rows of 128 need 160 registers, and three
// workgroups a CU would fit, but read no faster than two (e4m3 76.6 us against 73.9: shorter shares,
// more parts); two of rows of 256 take 170 us where one takes 160.
constexpr uint32_t per_cu(uint32_t dim) { return dim <= 64 ? 4 : dim <= 128 ? 2 : 1; }

// T: queries' type. E4M3: the cache holds that instead. D: head_dim rounded up to 64, 128, 256;
// EXACT: it is D. PAGES: kWhole where 16 tokens that start at a multiple of 16 lie within one page;
// else, of a cache whose offsets fit 32 bits, kNear, or kFar. TWO: parts may be joined in two steps.
template <class T, bool E4M3, int D, bool EXACT, int PAGES, bool TWO>
__global__ __launch_bounds__(kThreads, per_cu(D)) void decode_kernel(const DecodeParams p) {
  constexpr int CB = E4M3 ? 1 : 2;                         // bytes of a cached element
  constexpr int KP = D * CB / 64;                          // 16-byte pieces of a K row per lane
  constexpr int VP = D / 16 < 16 / CB ? D / 16 : 16 / CB;  // elements of a V piece
  constexpr int NP = D / 16 / VP;                          // V pieces per row and lane
  constexpr int VW = VP * CB / 4;                          // words of a V piece
  constexpr int NA = NP * VP;                              // accumulators: 16 dims each
  constexpr bool WHOLE = PAGES == kWhole;
  typedef typename std::conditional<PAGES == kNear, uint32_t, int64_t>::type offset_t;
  extern __shared__ float lds[];

  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t col = lane & 15u, kg = lane >> 4;
  const uint32_t team = blockIdx.x / p.rows, member = blockIdx.x - team * p.rows;
  const uint32_t dim = EXACT ? D : p.head_dim;

  // --- the work: units of kStep tokens, sequence after sequence; team t takes units [t U / n,
  // (t + 1) U / n) of all U, and each of its workgroups one row (KV head, tiles of its query heads)
  // of them. Found by every wavefront for itself: lane i adds up the i-th share of the sequences.
  uint64_t total, before;   // units of all sequences; of those in front of `seq`
  uint64_t u = 0, u_end = 0;
  uint32_t n_teams, seq, len;
  {
    const uint32_t each = (p.n_seqs + 63u) / 64u, lanes = (p.n_seqs + each - 1) / each;
    const uint32_t s0 = lane * each, s1 = s0 + each < p.n_seqs ? s0 + each : p.n_seqs;
    uint64_t mine = 0;
    int32_t raw = 0;   // the length of the last sequence looked at
    for (uint32_t s = s0; s < s1; ++s) raw = p.lens[s], mine += units_of(p, raw);
    uint64_t upto = mine;
    for (uint32_t d = 1; d < lanes; d *= 2) {
      const uint64_t other = __shfl_up(upto, d);
      if (lane >= d) upto += other;
    }
    total = uniform(__shfl(upto, lanes - 1));
    n_teams = total < p.teams ? static_cast<uint32_t>(total) : p.teams;
    if (team < n_teams) {
      u = team * total / n_teams;
      u_end = (team + 1) * total / n_teams;
    }
    uint64_t at = upto - mine;
    uint32_t s = s0;
    const bool here = u >= at && u < upto;
    if (here && each > 1)
      for (;; ++s) {
        raw = p.lens[s];
        const uint32_t n = units_of(p, raw);
        if (u < at + n) break;
        at += n;
      }
    const uint32_t owner = __builtin_ctzll(__ballot(here) | 1ull << 63);
    seq = __builtin_amdgcn_readlane(s, owner);
    len = seen_of(p, __builtin_amdgcn_readlane(raw, owner));
    before = uniform(__shfl(at, owner));
  }
  const uint64_t u_begin = u;

  // a sequence that sees nothing belongs to no row: zeros
  for (uint32_t s = blockIdx.x; s < p.n_seqs; s += gridDim.x) {
    if (seen_of(p, p.lens[s]) != 0) continue;
    for (uint32_t n = threadIdx.x; n < p.n_heads * dim; n += kThreads) {
      const uint32_t head = n / dim;
      reinterpret_cast<uint16_t*>(p.out + s * p.out_token + head * p.out_head)[n - head * dim] = 0;
    }
    if (p.lse)
      for (uint32_t n = threadIdx.x; n < p.n_heads; n += kThreads) p.lse[static_cast<uint64_t>(s) * p.n_heads + n] = -INFINITY;
  }

  // this workgroup's heads: `spread` bundles of at most 16 that its wavefronts take side by side
  // before they share out the tokens -- tiles of one KV head's, or (abreast) those of neighbouring KV heads
  const uint32_t bundle = p.group < 16u ? p.group : 16u;
  const uint32_t tile = wave & (p.spread - 1), turn = wave / p.spread;
  const uint32_t kv_first = p.abreast ? member * p.spread : member / p.head_rows;
  const uint32_t head_row = p.abreast ? 0u : member - kv_first * p.head_rows;
  const uint32_t kv_head = kv_first + (p.abreast ? tile : 0u);
  const uint32_t head0 = kv_first * p.group + head_row * p.spread * 16u;
  const uint32_t left = p.abreast ? p.spread * p.group : p.group - head_row * p.spread * 16u;
  const uint32_t n_heads = left < p.spread * bundle ? left : p.spread * bundle;
  const uint32_t my_heads = n_heads <= tile * bundle ? 0u : n_heads - tile * bundle < bundle ? n_heads - tile * bundle : bundle;
  const uint32_t step = kStep / p.spread;

  const uint8_t* kbase = p.base + kv_head * p.head_stride;
  const uint8_t* vbase = kbase + p.kv_stride;
  const rsrc_t part_o = rsrc_of(p.part_o), part_ml = rsrc_of(p.part_ml);
  // K goes through LDS: a load instruction there takes whole rows, one lane after the other 16
  // bytes, and a row's pieces are stored in an order that lets the 16 rows of a read differ in bank
  constexpr uint32_t RB = D * CB, PR = RB / 16, RI = 64 / PR, KI = 16 / RI;   // row bytes, pieces; rows per load, loads per half
  uint8_t* const k_tile = reinterpret_cast<uint8_t*>(lds) + wave * kTile * RB;
  const auto turned = [](uint32_t row, uint32_t piece) -> uint32_t {
    return piece ^ ((row / (PR >= 16 ? 1u : 16u / (PR < 16 ? PR : 16u))) & ((PR >= 16 ? 16u : PR) - 1u));
  };
  uint32_t k_read[KP];
#pragma unroll
  for (int c = 0; c < KP; ++c)
    k_read[c] = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)(k_tile))) +
                col * RB + turned(col, c * 4u + kg) * 16u;
  uint32_t k_lane[KI];
#pragma unroll
  for (uint32_t j = 0; j < KI; ++j) {
    const uint32_t row = j * RI + lane / PR;
    k_lane[j] = (WHOLE ? row * static_cast<uint32_t>(p.token_stride) : 0u) + turned(row, lane % PR) * 16u;
    // pieces behind the head's end: behind the buffer's end too, so that nothing is read
    if (!EXACT && turned(row, lane % PR) * 16u >= dim * CB) k_lane[j] = kNowhere;
  }
  uint32_t v_piece[NP];   // (what dims behind the head's end are read as does not matter)
#pragma unroll
  for (uint32_t h = 0; h < NP; ++h) v_piece[h] = EXACT || (h * 16u + col) * VP < dim ? (h * 16u + col) * VP * CB : 0u;
  uint32_t v_lane[4];
#pragma unroll
  for (int r = 0; r < 4; ++r)
    v_lane[r] = WHOLE ? (kg * 4 + r) * static_cast<uint32_t>(p.token_stride) : 0u;

  while (u < u_end) {
    // the sequence that unit u belongs to, and how much of it is this workgroup's
    const uint32_t start = p.window != 0 && len > p.window ? len - p.window : 0u;
    const uint32_t first = start & ~(kTile - 1), units = (len - first + kStep - 1) / kStep;
    if (u >= before + units) {
      before += units;
      len = seen_of(p, constant(p.lens)[++seq]);
      continue;
    }
    const float top_weight = T::template top<E4M3>(len);
    const uint32_t unit0 = static_cast<uint32_t>(u - before);
    const uint32_t n_units = u_end - u < units - unit0 ? static_cast<uint32_t>(u_end - u) : units - unit0;
    const uint32_t begin = first + unit0 * kStep;
    const uint32_t end = len - begin < n_units * kStep ? len : begin + n_units * kStep;

    // queries: lane = head, the same numbering of the dims as the pieces of K
    u32x4 qf[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const uint32_t d = E4M3 ? (c / 2) * 64u + kg * 16u + (c & 1) * 8u : c * 32u + kg * 8u;
      u32x4 v = {0, 0, 0, 0};
      if (col < my_heads && (EXACT || d < dim)) {
        const uint8_t* a = p.q + seq * p.q_token + (head0 + tile * bundle + col) * p.q_head + d * 2u;
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

    const int32_t* table = p.tables + seq * p.table_stride;
    // Block ids of a tile's two halves: one each where a half lies within a page (WHOLE, through
    // the scalar cache, so that waiting for them is not waiting for rows), else one for the lane's
    // token of each half. Behind the end the last token's are asked for again.
    const auto fetch = [&](uint32_t t0, int32_t (&id)[2]) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint32_t t = t0 + s * 16u + (WHOLE ? 0u : col), in = t < len ? t : len - 1;
        id[s] = WHOLE ? constant(table)[divided(in, p.block_magic)] : table[divided(in, p.block_magic)];
      }
    };
    // ... and where the halves' rows lie: bytes of the half's first row (WHOLE), or of the lane's
    // token. What is not seen reads some row of the cache and takes no part below. -> seen, a bit each
    const auto place = [&](uint32_t t0, const int32_t (&id)[2], offset_t (&off)[2]) -> uint32_t {
      uint32_t seen = 0;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint32_t t = t0 + s * 16u + (WHOLE ? 0u : col);
        bool valid = static_cast<uint32_t>(id[s]) < p.n_blocks;
        if (!WHOLE) valid = valid && t >= start && t < end;
        const uint32_t in = t - divided(t, p.block_magic) * p.ntpb;
        if constexpr (PAGES == kNear)
          off[s] = valid ? id[s] * static_cast<uint32_t>(p.block_stride) + in * static_cast<uint32_t>(p.token_stride) : 0u;
        else
          off[s] = valid ? id[s] * p.block_stride + in * p.token_stride : 0;
        if (WHOLE) {
          const uint32_t upto = end > t ? (end - t < 16u ? (1u << (end - t)) - 1u : 0xFFFFu) : 0u;
          const uint32_t from = start > t ? (start - t < 16u ? (1u << (start - t)) - 1u : 0xFFFFu) : 0u;
          seen |= (valid ? upto & ~from : 0u) << (16 * s);
        } else {
          seen |= static_cast<uint32_t>(__ballot(valid) & 0xFFFFu) << (16 * s);
        }
      }
      return seen;
    };
    const auto load_k = [&](const offset_t (&off)[2]) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        // (a buffer instruction where it can be: the compiler counts it apart from the loads of V)
        const rsrc_t rows = rsrc_of(const_cast<uint8_t*>(kbase + (WHOLE ? off[s] : 0)));
#pragma unroll
        for (uint32_t j = 0; j < KI; ++j) {
          const uint32_t row = j * RI + lane / PR;
          const auto to = (__attribute__((address_space(3))) void*)(k_tile + (s * KI + j) * 1024u);
          if constexpr (PAGES == kWhole) {
            load_to_lds(rows, k_lane[j], to);
          } else if constexpr (PAGES == kNear) {
            const uint32_t at = __shfl(off[s], row) + k_lane[j];
            load_to_lds(rows, EXACT || k_lane[j] != kNowhere ? at : kNowhere, to);
          } else {
            // (by all lanes: one whose own piece lies behind the head's end still tells others where a row is)
            const int64_t at = __shfl(off[s], row);
            if (EXACT || k_lane[j] != kNowhere)
              __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(kbase + at + k_lane[j]), to,
                                               16, 0, kStreamed);
          }
        }
      }
    };
    if (!EXACT) {   // pieces behind the head's end are never written
      for (uint32_t n = lane; n < kTile * PR; n += 64) reinterpret_cast<u32x4*>(k_tile)[n] = u32x4{0, 0, 0, 0};
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    // V: the eight tokens whose weights this lane will hold, 4 kg ... + 3 of both halves
    uint32_t vr[8][NP][VW];
    const auto load_v = [&](const offset_t (&off)[2]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint8_t* row = vbase + (WHOLE ? off[i >> 2] : __shfl(off[i >> 2], kg * 4 + (i & 3)));
#pragma unroll
        for (int h = 0; h < NP; ++h) {
          const uint8_t* a = row + v_lane[i & 3] + v_piece[h];
          if constexpr (VW == 4) {
            const u32x4 v = streamed<u32x4>(a);
            vr[i][h][0] = v.x, vr[i][h][1] = v.y, vr[i][h][2] = v.z, vr[i][h][3] = v.w;
          } else if constexpr (VW == 2) {
            const u32x2 v = streamed<u32x2>(a);
            vr[i][h][0] = v.x, vr[i][h][1] = v.y;
          } else {
            vr[i][h][0] = streamed<uint32_t>(a);
          }
        }
      }
    };

    f32x4 acc[NA];
#pragma unroll
    for (int x = 0; x < NA; ++x) acc[x] = f32x4{0, 0, 0, 0};
    float top = -INFINITY, sum = 0.0f;
    bool any = false;

    // While a tile is worked on, the next one's rows are on their way (K from where this one's
    // scores are done, V from where its sums are) and the block ids of the one behind.
    uint32_t t0 = begin + turn * kTile, seen = 0;
    int32_t id[2];
    offset_t off[2];
    const auto work_on = [&](auto more) {
      constexpr bool MORE = decltype(more)::value;
      any = any || seen != 0;
      uint32_t seen_next = 0;
      if constexpr (MORE) {
        seen_next = place(t0 + step, id, off);
        fetch(t0 + 2 * step, id);
      }

      // scores
      f32x4 sc[2];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        u32x4 kr[KP];
        read_k<KP, 8 * NP>(k_read, s * 16 * RB, kr);
        sc[s] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < KP; ++c) {
          if constexpr (E4M3) {
            const u32x4 w = kr[c];
            const u32x4 a = {T::template widen<false>(w.x), T::template widen<true>(w.x),
                             T::template widen<false>(w.y), T::template widen<true>(w.y)};
            const u32x4 b = {T::template widen<false>(w.z), T::template widen<true>(w.z),
                             T::template widen<false>(w.w), T::template widen<true>(w.w)};
            sc[s] = T::mma(a, qf[2 * c], sc[s]);
            sc[s] = T::mma(b, qf[2 * c + 1], sc[s]);
          } else {
            sc[s] = T::mma(kr[c], qf[c], sc[s]);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (MORE) load_k(off);
      __builtin_amdgcn_sched_barrier(0);
      if (p.cap != 0.0f) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[s][r] = p.cap * tanhf(sc[s][r] * p.cap_in);
      } else {
        sc[0] *= p.scale_log2;
        sc[1] *= p.scale_log2;
      }
      if (seen != 0xFFFFFFFFu) {
        const uint32_t bits = seen >> (4 * kg);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (!((bits >> (16 * (i >> 2) + (i & 3))) & 1u)) {
            sc[i >> 2][i & 3] = -INFINITY;
            // rows that are not seen may hold anything, and zero times anything is not zero
#pragma unroll
            for (int h = 0; h < NP; ++h)
#pragma unroll
              for (int w = 0; w < VW; ++w) vr[i][h][w] = 0;
          }
      }
      float high = top;
#pragma unroll
      for (int i = 0; i < 8; ++i) high = fmaxf(high, sc[i >> 2][i & 3]);
      high = over_tokens_max(high);
      if (__any(high != top)) {
        // a head with nothing but minus infinity so far: exp2(-inf - 0) = 0, of a sum of zero
        const float shrink = carried(__builtin_amdgcn_exp2f(top - (high == -INFINITY ? 0.0f : high)));
        sum *= shrink;
#pragma unroll
        for (int x = 0; x < NA; ++x) acc[x] *= shrink;
        top = high;
      }
      const float ref = high == -INFINITY ? 0.0f : high;
      u32x4 ph, pl;   // weights cut off, and what that left
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int s = i >> 1, r = 2 * (i & 1);
        float a = __builtin_amdgcn_exp2f(sc[s][r] - ref), b = __builtin_amdgcn_exp2f(sc[s][r + 1] - ref);
        sum += a + b;
        a *= top_weight, b *= top_weight;
        // (positive numbers, and NaN above them, are in the order of their bits)
        const uint32_t hi = __builtin_bit_cast(
            uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, T::cut(a, b)), __builtin_bit_cast(u16x2, T::kLeastTwice)));
        const f32x2 kept = __builtin_convertvector(__builtin_bit_cast(typename T::x2, hi), f32x2);
        const f32x2 rest = {fmaxf(a - kept.x, T::kLeast), fmaxf(b - kept.y, T::kLeast)};
        ph[i] = hi;
        pl[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, typename T::x2));
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
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (MORE) load_v(off);
      __builtin_amdgcn_sched_barrier(0);
      seen = seen_next;
    };
    if (t0 < end && my_heads != 0) {
      fetch(t0, id);
      seen = place(t0, id, off);
      fetch(t0 + step, id);
      // the queries are here before rows are asked for: waiting for them later would be waiting for
      // rows too
#pragma unroll
      for (int c = 0; c < D / 32; ++c) asm volatile("" : "+v"(qf[c]));
      load_k(off);
      __builtin_amdgcn_sched_barrier(0);
      load_v(off);
      __builtin_amdgcn_sched_barrier(0);
      for (; t0 + step < end; t0 += step) work_on(std::true_type());
      work_on(std::false_type());
    }
    __syncthreads();   // no rows of K are in LDS, or on the way there, any more

    // the wavefronts' parts meet in LDS: [wave][head of its tile][dim], rows 4 floats apart from
    // a multiple of the banks
    constexpr uint32_t kRow = D + 4;
    Stat* stats = reinterpret_cast<Stat*>(lds);   // [wave][16]
    float* part = lds + kWaves * 16 * 2;
    sum = over_tokens_sum(sum);
    if (sum == 0.0f && any) sum = -1.0f;
    if (kg == 0) stats[wave * 16 + col] = Stat{top, sum};
    if (col < my_heads) {
      float* row = part + (wave * bundle + col) * kRow;
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

    // (made anew for every row: the compiler would otherwise work out all that follows from them, for
    // every way below, before the first row is read: one sequence of 512 9.4 us, 9.1)
    uint32_t tid = threadIdx.x, heads = n_heads;
    asm volatile("" : "+v"(tid), "+s"(heads));
    const uint32_t quads = dim / 4, work = heads * quads;
    const bool whole = n_units == units;
    const auto finish = [&](uint32_t head, uint32_t d, f32x4 o, float m, float l, bool nothing_but_inf) {
      const float inv = l == 0.0f ? (nothing_but_inf ? NAN : 0.0f) : p.v_scale / top_weight / l;
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
    const auto leave = [&](uint32_t at, uint32_t d, f32x4 o, float m, float l, bool nothing_but_inf) {
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), part_o, (at * dim + d) * 4u, 0, kShared);
      if (d == 0)
        __builtin_amdgcn_raw_buffer_store_b64(
            u32x2{__float_as_uint(m), __float_as_uint(l == 0.0f && nothing_but_inf ? -1.0f : l)}, part_ml, at * 8u, 0, kShared);
    };
    for (uint32_t n = tid; n < work; n += kThreads) {
      const uint32_t head = n / quads, d = (n - head * quads) * 4;
      const uint32_t t = head / bundle, h = head - t * bundle;
      float m = -INFINITY, l = 0.0f;
      bool inf = false;
      f32x4 o = {0, 0, 0, 0};
      for (uint32_t w = t; w < kWaves; w += p.spread) m = fmaxf(m, stats[w * 16 + h].max);
      for (uint32_t w = t; w < kWaves; w += p.spread) {
        const Stat s = stats[w * 16 + h];
        const float f = weight_of(s, m);
        inf = inf || s.sum < 0.0f;
        if (f != 0.0f) l += f * s.sum;
        o += carried(f) * *reinterpret_cast<const f32x4*>(part + (w * bundle + h) * kRow + d);
      }
      if (whole) {
        finish(head, d, o, m, l, inf);
      } else {
        const uint32_t at = (3u * blockIdx.x + (u != u_begin)) * p.slot_heads + head;
        leave(at, d, o, m, l, inf);
      }
    }
    // Q float4s of a head (a piece of the head apart, so that lanes side by side ask for bytes side by
    // side: one after the other 93.5 us for 131071 tokens, 92.5) by one lane, or by several (crews) that
    // share the parts; kBatch parts at a time, all asked for at once, then weighed against their maximum. Two where that saves
    // a pass (32 heads of 192, 21 parts: 35 -> 28 us for the launch), else one, whose crews have
    // less to tell one another.
    const auto join = [&](auto quads_each, uint32_t count, const auto& slot, const auto& sink) {
      constexpr uint32_t Q = decltype(quads_each)::value, kBatch = 8;
      const uint32_t per_head = dim / (4 * Q), jobs = heads * per_head;
      const uint32_t crews = jobs < kThreads ? kThreads / jobs : 1u;
      for (uint32_t n0 = 0; n0 < jobs; n0 += kThreads) {
        const uint32_t crew = jobs < kThreads ? tid / jobs : 0u;
        const uint32_t n = jobs < kThreads ? tid - crew * jobs : n0 + tid;
        const bool active = n < jobs && crew < crews;
        const uint32_t head = n / per_head, d = (n - head * per_head) * 4, apart = dim / Q;
        float m = -INFINITY, l = 0.0f;
        bool inf = false;
        f32x4 o[Q] = {};
        for (uint32_t s0 = crew; s0 < count; s0 += kBatch * crews) {
          u32x2 st[kBatch];
          u32x4 v[kBatch][Q];
#pragma unroll
          for (uint32_t k = 0; k < kBatch; ++k) {
            // a part that is none is behind the buffer's end: zeros come back
            const uint32_t s = s0 + k * crews, at = slot(s) + head;
            const bool is = active && s < count;
            st[k] = __builtin_amdgcn_raw_buffer_load_b64(part_ml, is ? at * 8u : kNowhere, 0, kShared);
#pragma unroll
            for (uint32_t x = 0; x < Q; ++x)
              v[k][x] = __builtin_amdgcn_raw_buffer_load_b128(part_o, is ? (at * dim + d + x * apart) * 4u : kNowhere, 0, kShared);
          }
          float up = m;
#pragma unroll
          for (uint32_t k = 0; k < kBatch; ++k) {
            if (s0 + k * crews >= count) st[k].x = __float_as_uint(-INFINITY);
            up = fmaxf(up, __uint_as_float(st[k].x));
          }
          const float f_old = weight_of(Stat{m, l}, up);
          if (f_old != 1.0f) {
            l *= f_old;
#pragma unroll
            for (uint32_t x = 0; x < Q; ++x) o[x] *= carried(f_old);
          }
#pragma unroll
          for (uint32_t k = 0; k < kBatch; ++k) {
            const Stat part_st = {__uint_as_float(st[k].x), __uint_as_float(st[k].y)};
            const float f = weight_of(part_st, up);
            inf = inf || part_st.sum < 0.0f;
            l += f != 0.0f ? f * part_st.sum : 0.0f;
#pragma unroll
            for (uint32_t x = 0; x < Q; ++x) o[x] += carried(f) * __builtin_bit_cast(f32x4, v[k][x]);
          }
          m = up;
        }
        if (crews > 1) {
          f32x4* os = reinterpret_cast<f32x4*>(lds);
          Stat* mls = reinterpret_cast<Stat*>(lds + kThreads * 4 * Q);
          if (active && crew != 0) {
#pragma unroll
            for (uint32_t x = 0; x < Q; ++x) os[Q * tid + x] = o[x];
            mls[tid] = Stat{m, l == 0.0f && inf ? -1.0f : l};
          }
          __syncthreads();
          if (active && crew == 0)
            for (uint32_t t = 1; t < crews; ++t) {
              const uint32_t at = t * jobs + n;
              const Stat other = mls[at];
              const float up = fmaxf(m, other.max), f_old = weight_of(Stat{m, l}, up), f = weight_of(other, up);
              inf = inf || other.sum < 0.0f;
              l = (f_old != 0.0f ? f_old * l : 0.0f) + (f != 0.0f ? f * other.sum : 0.0f);
#pragma unroll
              for (uint32_t x = 0; x < Q; ++x) o[x] = carried(f_old) * o[x] + carried(f) * os[Q * at + x];
              m = up;
            }
        }
        if (active && crew == 0)
#pragma unroll
          for (uint32_t x = 0; x < Q; ++x) sink(head, d + x * apart, o[x], m, l, inf);
      }
    };
    if (!whole) {
      // the last workgroup of this row to get here joins the parts, in their order: those of the
      // teams w0 ... w1, the first's behind whatever it did before
      const uint32_t w0 = static_cast<uint32_t>(((before + 1) * n_teams - 1) / total);
      const uint32_t w1 = static_cast<uint32_t>(((before + units) * n_teams - 1) / total);
      const uint32_t parts = w1 - w0 + 1;
      const bool behind = w0 * total / n_teams < before;
      const auto last_of = [&](uint32_t* counter, uint32_t count) -> bool {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wavefront's part is where all can see it
        __syncthreads();
        uint32_t* arrived = reinterpret_cast<uint32_t*>(lds);
        if (tid == 0)
          *arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        const bool last = *arrived == count - 1;
        __syncthreads();
        if (last && tid == 0)   // as the next launch on this workspace wants to find it
          __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return last;
      };
      if (!TWO || parts <= kFan || parts * work <= kAlone) {
        if (last_of(p.counters + w0 * p.rows + member, parts)) {
          const auto slot = [&](uint32_t s) -> uint32_t {
            return (3u * ((w0 + s) * p.rows + member) + (s == 0 && behind)) * p.slot_heads;
          };
          if (D > 64 && work >= kThreads)
            join(std::integral_constant<uint32_t, D == 64 ? 1 : 2>(), parts, slot, finish);
          else
            join(std::integral_constant<uint32_t, 1>(), parts, slot, finish);
        }
      } else if constexpr (TWO) {
        // in two steps: `fan` neighbouring parts by the last of their workgroups, what those leave by
        // the last of these
        const params_t a = arguments();
        const uint32_t rows = a->rows, slot_heads = a->slot_heads;
        uint32_t fan = kFan;
        while (fan * fan < parts) fan *= 2;
        const uint32_t from = (team - w0) / fan * fan, some = parts - from < fan ? parts - from : fan;
        const uint32_t sum_slot = (3u * ((w0 + from) * rows + member) + 2u) * slot_heads;
        bool second = false;
        for (uint32_t count = some;;) {
          if (count > 1) {
            if (!last_of(a->counters + (second ? a->teams + w0 : w0 + from) * rows + member, count)) break;
            join(std::integral_constant<uint32_t, D == 64 ? 1 : 2>(), count,
                 [&](uint32_t s) -> uint32_t {
                   const uint32_t at = second ? s * fan : from + s;
                   const uint32_t which = second && at + 1 < parts ? 2u : at == 0 && behind ? 1u : 0u;
                   return (3u * ((w0 + at) * rows + member) + which) * slot_heads;
                 },
                 [&](uint32_t head, uint32_t d, f32x4 o, float m, float l, bool nothing_but_inf) {
                   if (second)
                     finish(head, d, o, m, l, nothing_but_inf);
                   else
                     leave(sum_slot + head, d, o, m, l, nothing_but_inf);
                 });
          }
          if (second) break;
          second = true;
          count = (parts + fan - 1) / fan;
        }
      }
    }
    u += n_units;
    __syncthreads();   // LDS is the next row's
  }
}

// Where the rows of neighbouring KV heads are neighbours in memory and short, a workgroup takes two
// of them side by side, so that it reads 512 bytes in a row instead of 256 (twice the sums to join,
// hence only where every workgroup has this many units). One / two heads, microseconds, 8 KV heads of
// 128 bf16 in [.., h, d] rows: 64 sequences of 1k-8k 196.6 / 182.7, 16 of them 49.2 / 45.8, 12 38.9 /
// 39.9, 8 31.9 / 36.6; rows of 512 bytes (dim 256) 310 / 316; 2 KV heads (e4m3) 74.5 / 75.7; pages that
// keep a head's rows together 169.8 / 171.2.
constexpr uint32_t kAbreastUnits = 8;

// Whether 32 bits hold what scores are multiplied with.
bool scores_held(float scale, float cap) {
  return std::isfinite(scale * kLog2e) && (cap == 0 || (std::isfinite(cap * kLog2e) && std::isfinite(scale / cap)));
}

struct Launch {
  dim3 grid;
  uint32_t lds;
  int pages;
  bool two_steps;
  hipStream_t stream;
};

template <class T, bool E4M3, int D, bool EXACT>
void launch_pages(const DecodeParams& p, const Launch& l) {
  if (l.pages == kNear) {
    decode_kernel<T, E4M3, D, EXACT, kNear, false><<<l.grid, kThreads, l.lds, l.stream>>>(p);
  } else if (l.pages == kFar) {
    decode_kernel<T, E4M3, D, EXACT, kFar, false><<<l.grid, kThreads, l.lds, l.stream>>>(p);
  } else {
    // (two steps for the usual head sizes and pages alone: every kernel takes its seconds to compile)
    if constexpr (EXACT)
      if (l.two_steps) {
        decode_kernel<T, E4M3, D, EXACT, kWhole, true><<<l.grid, kThreads, l.lds, l.stream>>>(p);
        return;
      }
    decode_kernel<T, E4M3, D, EXACT, kWhole, false><<<l.grid, kThreads, l.lds, l.stream>>>(p);
  }
}

template <class T, bool E4M3, int D>
void launch_exact(const DecodeParams& p, const Launch& l) {
  if (p.head_dim == D)
    launch_pages<T, E4M3, D, true>(p, l);
  else
    launch_pages<T, E4M3, D, false>(p, l);
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
  uint32_t dtype = 0, n_heads = 0, group = 0, spread = 0, head_rows = 0, slot_heads = 0, rows = 0, window = 0, max_seqs = 0;
  float scale = 0, cap = 0;
  uint64_t ws_bytes = 0;
  uint8_t* arena = nullptr;
  struct Owner {
    bool taken = false;
    hipStream_t stream = nullptr;
    unsigned long long capture = 0;     // 0: eager
    std::thread::id thread;             // of a per-thread default stream
  };
  std::mutex mu;
  std::vector<Owner> owners;

  uint32_t n_wgs = 0, teams = 0;
  bool pairs = false;   // neighbouring KV heads may be taken side by side
  uint64_t ml_at() const { return round_up(n_wgs * 3ull * slot_heads * (pairs ? 2 : 1) * layout.head_dim * 4, 256); }
  uint64_t counters_at() const { return round_up(ml_at() + n_wgs * 3ull * slot_heads * (pairs ? 2 : 1) * 8, 256); }

  // hipStreamPerThread is one handle for a stream of every thread: what tells them apart.
  static std::thread::id thread_of(hipStream_t s) {
    return s == hipStreamPerThread ? std::this_thread::get_id() : std::thread::id();
  }

  int workspace(hipStream_t s, unsigned long long capture, uint8_t** out) {
    const std::thread::id me = thread_of(s);
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
    d->scale = softmax_scale != 0 ? softmax_scale : 1.0f / std::sqrt(static_cast<float>(layout->head_dim));
    d->cap = logit_cap;
    if (!scores_held(d->scale, d->cap))
      return fail(KVT_ERR_INVALID, "kvt_decode_create: 32 bits do not hold softmax_scale or logit_cap, or their ratio");
    if (max_seqs == 0 || max_seqs > 65535 || n_workspaces == 0 || n_workspaces > 1024)
      return fail(KVT_ERR_INVALID, "kvt_decode_create: max_seqs must be in [1, 65535], n_workspaces in [1, 1024]");
    if (int rc = check_device(device)) return rc;
    d->device = device;
    d->layout = *layout;
    d->dtype = dtype;
    d->n_heads = n_q_heads;
    d->group = n_q_heads / layout->n_kv_heads;
    const uint32_t tiles = (d->group + 15) / 16;
    d->spread = tiles >= 3 ? 4 : tiles;
    d->head_rows = (tiles + d->spread - 1) / d->spread;
    d->slot_heads = std::min(d->group, 16 * d->spread);
    d->window = window;
    d->max_seqs = max_seqs;
    d->rows = layout->n_kv_heads * d->head_rows;
    d->teams = std::max(1u, device_cu_count(device) * per_cu(layout->head_dim) / d->rows);
    d->n_wgs = d->teams * d->rows;
    const uint32_t row = layout->head_dim * dtype_bytes(layout->dtype);
    d->pairs = d->group <= 16 && layout->n_kv_heads >= 4 && layout->n_kv_heads % 2 == 0 && row <= 256 &&
               layout->head_stride == row;
    const uint64_t counters = 2ull * d->n_wgs;
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
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const std::thread::id me = kvt_decode::thread_of(s);
  for (kvt_decode::Owner& o : d->owners)
    if (o.taken && o.stream == s && o.thread == me) o = kvt_decode::Owner{};
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
    const float scale = d->scale * k_scale;
    if (!scores_held(scale, d->cap))
      return fail(KVT_ERR_INVALID, "kvt_decode_attention: 32 bits do not hold softmax_scale k_scale, or its ratio to logit_cap");
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
    const Span outs{out, out_span, "out"}, lses{lse, lse ? 4ull * n_seqs * d->n_heads : 0, "lse"};
    if (int rc = check_distinct(who, {base, d->extent, "the cache's tensor"}, {outs, lses})) return rc;
    if (int rc = check_distinct(who, lses, {outs, {q, q_span, "q"}})) return rc;
    if (table_stride > (1ull << 40)) return fail(KVT_ERR_INVALID, "kvt_decode_attention: table_stride out of range");
    // (workgroups that read different lengths would wait for different numbers of parts)
    const Span lens{seq_lens, 4ull * n_seqs, "seq_lens"};
    const Span tables{block_tables, table_blocks ? 4 * ((n_seqs - 1) * table_stride + table_blocks) : 0, "block_tables"};
    if (int rc = check_distinct(who, outs, {lens, tables})) return rc;
    if (int rc = check_distinct(who, lses, {lens, tables})) return rc;
    DeviceGuard g;
    if (int rc = g.enter(d->device)) return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    unsigned long long capture = 0;
    if (hipStreamIsCapturing(s, &cap) != hipSuccess) (void)hipGetLastError();
    if (cap == hipStreamCaptureStatusNone) {
      if (int rc = check_spans(who, {{q, q_span, "q"}, outs, lens, tables, lses})) return rc;
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
    p.visible_max = static_cast<uint32_t>(std::min<uint64_t>(static_cast<uint64_t>(table_blocks) * d->layout.ntpb, 0x7FFFFFFFull));
    p.ntpb = d->layout.ntpb, p.n_blocks = static_cast<uint32_t>(d->layout.n_blocks);
    p.n_heads = d->n_heads, p.group = d->group, p.spread = d->spread, p.head_rows = d->head_rows, p.slot_heads = d->slot_heads, p.head_dim = dim, p.window = d->window;
    p.scale_log2 = scale * kLog2e;
    p.cap = d->cap * kLog2e, p.cap_in = d->cap != 0 ? scale / d->cap : 0;
    p.v_scale = v_scale;
    p.q_vec = rows_aligned16(qr);
    p.out_vec = ((reinterpret_cast<uintptr_t>(out) | out_token_stride | out_head_stride) & 7u) == 0;

    p.n_seqs = n_seqs;
    p.rows = d->rows;
    uint64_t longest = max_len == 0 || max_len > p.visible_max ? p.visible_max : max_len;
    const uint64_t units = (longest + kStep - 1) / kStep * n_seqs;
    uint32_t teams = d->teams;
    if (d->pairs && units >= kAbreastUnits * d->n_wgs / (d->rows / 2)) {
      p.abreast = true;
      p.spread = 2, p.head_rows = 1, p.slot_heads = 2 * d->group;
      p.rows = d->rows / 2;
      teams = d->n_wgs / p.rows;
    }
    p.teams = static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>(teams, units)));
    const uint32_t wgs = p.teams * p.rows;
    {
      uint8_t* ws = nullptr;
      if (int rc = d->workspace(s, capture, &ws)) return rc;
      p.part_o = reinterpret_cast<float*>(ws);
      p.part_ml = reinterpret_cast<float2*>(ws + d->ml_at());
      p.counters = reinterpret_cast<uint32_t*>(ws + d->counters_at());
    }
    const uint32_t heads = std::min(d->group, 16u), full = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
    const uint32_t meet = std::max<uint32_t>(kWaves * (heads * (full + 4) * 4 + 16 * static_cast<uint32_t>(sizeof(Stat))),
                                             kWaves * kTile * full * (e4m3 ? 1 : 2));
    const int pages = d->layout.ntpb % 16 == 0 && d->layout.token_stride <= (1u << 27) ? kWhole
                      : d->extent < kNowhere                                          ? kNear
                                                                                      : kFar;
    // parts of a sequence, of equally long ones (14 of 1536 float4s: one step 28.6 us, two 30.3)
    const uint32_t split = p.teams / n_seqs;
    const bool two_steps = split > 2 * kFan && static_cast<uint64_t>(split) * p.slot_heads * dim / 4 > kAlone;
    const Launch l{dim3(wgs), std::max<uint32_t>(meet, kThreads * 40), pages, two_steps, s};
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
