// Host side of the operators on the registered cache: the layouts of the cache shapes, the
// checks of their arguments, and the frequencies of rotary positions.
#include <algorithm>
#include <cmath>

#include "kvt_ops.h"

namespace kvt {

uint32_t dtype_bytes(uint32_t dtype) {
  switch (dtype) {
    case KVT_DTYPE_BF16:
    case KVT_DTYPE_F16: return 2;
    case KVT_DTYPE_F32: return 4;
    case KVT_DTYPE_E4M3: return 1;
    default: return 0;
  }
}

namespace {

struct Dim {
  uint64_t n, stride;
};

// Whether the rows of a strided nest lie apart: taken from the smallest stride up, every
// stride must step over what the dimensions below it span. false also where the span leaves
// 62 bits. *span = bytes from the first row's start to the last row's end.
bool rows_apart(Dim* dims, size_t n_dims, uint64_t row_bytes, uint64_t* span) {
  std::sort(dims, dims + n_dims, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
  unsigned __int128 reach = row_bytes;
  for (size_t i = 0; i < n_dims; ++i) {
    if (dims[i].n <= 1) continue;
    if (dims[i].stride < reach) return false;
    reach += static_cast<unsigned __int128>(dims[i].n - 1) * dims[i].stride;
    if (reach >> 62) return false;
  }
  *span = static_cast<uint64_t>(reach);
  return true;
}

std::string text(const char* who, const std::string& what) { return std::string(who) + ": " + what; }

}  // namespace

int check_kv_layout(const kvt_kv_layout* l, const char* who, uint64_t* extent) {
  if (!l) return fail(KVT_ERR_INVALID, text(who, "null layout"));
  if (l->dtype != KVT_DTYPE_BF16 && l->dtype != KVT_DTYPE_F16 && l->dtype != KVT_DTYPE_E4M3)
    return fail(KVT_ERR_UNSUPPORTED, text(who, "the cache holds bf16, f16 or e4m3"));
  if (l->head_dim == 0 || l->head_dim % 16 != 0 || l->head_dim > 256)
    return fail(KVT_ERR_UNSUPPORTED, text(who, "head_dim must be a multiple of 16 up to 256"));
  if (l->tensor >= KVT_MAX_TENSORS || l->n_kv_heads == 0 || l->n_kv_heads > 65536)
    return fail(KVT_ERR_INVALID, text(who, "bad tensor index or number of KV heads"));
  if (l->ntpb == 0 || l->ntpb > 65536)
    return fail(KVT_ERR_INVALID, text(who, "tokens per block must be in [1, 65536]"));
  if (l->n_blocks == 0 || l->n_blocks > 0x7FFFFFFFull)
    return fail(KVT_ERR_INVALID, text(who, "the number of blocks must be in [1, 2^31)"));
  if ((l->block_stride | l->kv_stride | l->token_stride | l->head_stride) & 15u)
    return fail(KVT_ERR_INVALID, text(who, "the layout's strides must be multiples of 16 bytes"));
  Dim dims[4] = {{l->n_blocks, l->block_stride}, {2, l->kv_stride}, {l->ntpb, l->token_stride},
                 {l->n_kv_heads, l->head_stride}};
  if (!rows_apart(dims, 4, static_cast<uint64_t>(l->head_dim) * dtype_bytes(l->dtype), extent))
    return fail(KVT_ERR_INVALID, text(who, "the layout's rows overlap, or leave 62 bits"));
  return KVT_OK;
}

int check_cache_layer(const kvt_cache* c, uint32_t layer, const kvt_kv_layout* l, uint64_t extent,
                      const char* who, uint8_t** base) {
  if (!c) return fail(KVT_ERR_INVALID, text(who, "null cache"));
  if (layer >= c->n_layers || l->tensor >= c->n_tensors)
    return fail(KVT_ERR_OUT_OF_RANGE, text(who, "the cache has no such layer or tensor"));
  if (extent > c->capacity[l->tensor])
    return fail(KVT_ERR_OUT_OF_RANGE,
                text(who, "the layout spans " + std::to_string(extent) + " bytes, the cache's tensor has " +
                              std::to_string(c->capacity[l->tensor])));
  void* p = c->host_ptrs[static_cast<uint64_t>(layer) * c->n_tensors + l->tensor];
  if (reinterpret_cast<uintptr_t>(p) & 15u)
    return fail(KVT_ERR_INVALID, text(who, "the layer's tensor is not 16-byte aligned"));
  *base = static_cast<uint8_t*>(p);
  return KVT_OK;
}

int check_rows(const Rows& r, uint64_t n_tokens, uint32_t n_heads, uint64_t row_bytes,
               uint32_t elem, bool written, const char* who, const char* what, uint64_t* span) {
  *span = 0;
  if (n_tokens == 0 || n_heads == 0) return KVT_OK;
  if (!r.ptr) return fail(KVT_ERR_INVALID, text(who, std::string(what) + " is null"));
  if ((reinterpret_cast<uintptr_t>(r.ptr) | r.token_stride | r.head_stride) & (elem - 1))
    return fail(KVT_ERR_INVALID, text(who, std::string(what) + " is not aligned to its elements"));
  Dim dims[2] = {{n_tokens, r.token_stride}, {n_heads, r.head_stride}};
  if (written) {
    if (!rows_apart(dims, 2, row_bytes, span))
      return fail(KVT_ERR_INVALID, text(who, std::string("the rows of ") + what + " overlap, or leave 62 bits"));
    return KVT_OK;
  }
  unsigned __int128 reach = row_bytes;
  for (const Dim& d : dims) reach += static_cast<unsigned __int128>(d.n - 1) * d.stride;
  if (reach >> 62) return fail(KVT_ERR_INVALID, text(who, std::string(what) + " leaves 62 bits"));
  *span = static_cast<uint64_t>(reach);
  return KVT_OK;
}

int check_apart(const Rows& in, uint32_t in_heads, const Rows& out, uint32_t out_heads, uint64_t n_tokens,
                uint64_t row_bytes, bool in_place, const char* who, const char* what) {
  if (n_tokens == 0 || in_heads == 0 || out_heads == 0) return KVT_OK;
  // bytes of one token's rows, and of all (both were found to stay within 62 bits)
  const uint64_t in_token = (in_heads - 1) * in.head_stride + row_bytes;
  const uint64_t out_token = (out_heads - 1) * out.head_stride + row_bytes;
  const uint64_t a = reinterpret_cast<uintptr_t>(in.ptr), b = reinterpret_cast<uintptr_t>(out.ptr);
  if (a + (n_tokens - 1) * in.token_stride + in_token <= b || b + (n_tokens - 1) * out.token_stride + out_token <= a)
    return KVT_OK;
  // (a stride of one token or one head is no stride)
  const bool same_tokens = n_tokens == 1 || in.token_stride == out.token_stride;
  const bool same_heads = in_heads == 1 || out_heads == 1 || in.head_stride == out.head_stride;
  if (in_place && a == b && same_tokens && in_heads == out_heads && same_heads) return KVT_OK;
  const uint64_t stride = out.token_stride;
  if (in.token_stride == stride && in_token <= stride && out_token <= stride) {
    // both repeat with the same period: apart when one period's intervals are
    const uint64_t gap = a >= b ? (a - b) % stride : (stride - (b - a) % stride) % stride;   // a behind b
    if (gap >= out_token && gap + in_token <= stride) return KVT_OK;
  }
  if (same_tokens && same_heads) {
    // rows interleave head by head (or token by token within a head): those of two tokens dt apart and two
    // heads dh apart meet where |a - b + dt token_stride + dh head_stride| < row_bytes
    // (spans stay within 62 bits and addresses far below that, so that 64 bits hold every sum)
    const int64_t t_stride = n_tokens == 1 ? 0 : in.token_stride, most = n_tokens - 1, row = row_bytes;
    const int64_t h_stride = in_heads > 1 ? in.head_stride : out_heads > 1 ? out.head_stride : 0;
    const auto floored = [](int64_t n, int64_t d) { return n / d - (n % d < 0); };
    bool meet = false;
    for (int64_t dh = -(static_cast<int64_t>(out_heads) - 1); dh < in_heads && !meet; ++dh) {
      const int64_t c = static_cast<int64_t>(a - b) + dh * h_stride;
      if (t_stride == 0)
        meet = -row < c && c < row;
      else
        meet = std::max(floored(-row - c, t_stride) + 1, -most) <= std::min(floored(row - c - 1, t_stride), most);
    }
    if (!meet) return KVT_OK;
  }
  return fail(KVT_ERR_INVALID, text(who, std::string("the output shares bytes with ") + what +
                                             " without being the same rows"));
}

int check_distinct(const char* who, const Span& a, std::initializer_list<Span> others) {
  const uint64_t a0 = reinterpret_cast<uintptr_t>(a.ptr);
  for (const Span& b : others) {
    const uint64_t b0 = reinterpret_cast<uintptr_t>(b.ptr);
    if (a.bytes != 0 && b.bytes != 0 && a0 < b0 + b.bytes && b0 < a0 + a.bytes)
      return fail(KVT_ERR_INVALID, text(who, std::string(a.what) + " shares bytes with " + b.what));
  }
  return KVT_OK;
}

int check_spans(const char* who, std::initializer_list<Span> spans) {
  static const std::string none;
  for (const Span& s : spans)
    if (check_device_span(s.ptr, s.bytes, none) != KVT_OK)
      return check_device_span(s.ptr, s.bytes, std::string(who) + ": " + s.what);
  return KVT_OK;
}

}  // namespace kvt

using namespace kvt;

extern "C" {

int kvt_kv_layout_of(int cache_shape, uint32_t dtype, uint64_t n_blocks, uint32_t ntpb,
                     uint32_t n_kv_heads, uint32_t head_dim, kvt_kv_layout* out) {
  return guarded([&]() -> int {
    static const char* who = "kvt_kv_layout_of";
    if (!out) return fail(KVT_ERR_INVALID, "kvt_kv_layout_of: null argument");
    const uint64_t row = static_cast<uint64_t>(head_dim) * dtype_bytes(dtype);
    // products of 32-bit sizes: refused below where they leave what a layout may hold
    if (n_kv_heads > 65536 || ntpb > 65536 || head_dim > 256 || n_blocks > 0x7FFFFFFFull)
      return fail(KVT_ERR_INVALID, "kvt_kv_layout_of: sizes out of range");
    const uint64_t token = row * n_kv_heads, half = token * ntpb;
    kvt_kv_layout l{};
    l.dtype = dtype;
    l.n_kv_heads = n_kv_heads;
    l.head_dim = head_dim;
    l.ntpb = ntpb;
    l.n_blocks = n_blocks;
    switch (cache_shape) {
      case KVT_SHAPE_FLASH:                  // [2, nblk, bs, h, d]
        l.block_stride = half;
        if (half != 0 && n_blocks > (1ull << 62) / half)
          return fail(KVT_ERR_INVALID, "kvt_kv_layout_of: sizes out of range");
        l.kv_stride = half * n_blocks, l.token_stride = token, l.head_stride = row;
        break;
      case KVT_SHAPE_RAGGED_FLASH:           // [nblk, bs, 2, h, d]
        l.block_stride = 2 * half, l.kv_stride = token, l.token_stride = 2 * token, l.head_stride = row;
        break;
      case KVT_SHAPE_QWEN3_NEXT_FLASH:       // [nblk, 2, bs, h, d]
        l.block_stride = 2 * half, l.kv_stride = half, l.token_stride = token, l.head_stride = row;
        break;
      case KVT_SHAPE_FLASHINFER:             // [nblk, 2, h, bs, d]
      case KVT_SHAPE_QWEN3_NEXT_FLASHINFER:
        l.block_stride = 2 * half, l.kv_stride = half, l.token_stride = row, l.head_stride = row * ntpb;
        break;
      default:
        return fail(KVT_ERR_UNSUPPORTED, "kvt_kv_layout_of: no keys and values per head in this cache shape");
    }
    uint64_t extent = 0;
    if (int rc = check_kv_layout(&l, who, &extent)) return rc;
    *out = l;
    return KVT_OK;
  });
}

int kvt_rotary_frequencies(const kvt_rotary_opts* o, double* freq, double* magnitude) {
  return guarded([&]() -> int {
    if (!o || !freq || !magnitude) return fail(KVT_ERR_INVALID, "kvt_rotary_frequencies: null argument");
    if (o->rotary_dim < 2 || o->rotary_dim > 256 || o->rotary_dim % 2 != 0)
      return fail(KVT_ERR_INVALID, "kvt_rotary_frequencies: rotary_dim must be even, 2 to 256");
    if (o->scaling > KVT_ROTARY_RAMP)
      return fail(KVT_ERR_UNSUPPORTED, "kvt_rotary_frequencies: unknown scaling");
    const bool ramp = o->scaling == KVT_ROTARY_RAMP, bands = o->scaling == KVT_ROTARY_BANDS;
    const double low = o->low == 0 ? 1.0 : o->low;
    const double high = o->high == 0 ? (ramp ? 32.0 : 4.0) : o->high;
    const auto finite_above = [](double v, double than) { return std::isfinite(v) && v > than; };
    if (!finite_above(o->base, 1.0) || !std::isfinite(o->magnitude) || o->magnitude < 0 ||
        (o->scaling != KVT_ROTARY_PLAIN && !finite_above(o->factor, 0.0)) ||
        ((bands || ramp) &&
         (!finite_above(o->original_max_position, 0.0) || !finite_above(low, 0.0) || !finite_above(high, low))))
      return fail(KVT_ERR_INVALID, "kvt_rotary_frequencies: base, factor, original_max_position, low, high or "
                                   "magnitude out of range");
    const double pi = 3.14159265358979323846;
    const uint32_t pairs = o->rotary_dim / 2;
    // the pair (a real number) that makes `turns` turns over the original length
    const auto pair_of = [&](double turns) {
      return o->rotary_dim * std::log(o->original_max_position / (turns * 2 * pi)) / (2 * std::log(o->base));
    };
    double first = 0, last = 0;
    if (ramp) {
      first = std::max(std::floor(pair_of(high)), 0.0);
      last = std::min(std::ceil(pair_of(low)), static_cast<double>(o->rotary_dim) - 1);
    }
    for (uint32_t i = 0; i < pairs; ++i) {
      const double w = std::pow(o->base, -2.0 * i / o->rotary_dim);
      double keep = 0;
      if (o->scaling == KVT_ROTARY_PLAIN) keep = 1;
      if (bands) keep = (o->original_max_position * w / (2 * pi) - low) / (high - low);
      if (ramp) keep = 1 - (i - first) / std::max(last - first, 1e-3);
      keep = std::min(1.0, std::max(0.0, keep));
      freq[i] = keep == 1 ? w : w * keep + w / o->factor * (1 - keep);
    }
    *magnitude = o->magnitude != 0 ? o->magnitude : ramp && o->factor > 1 ? 0.1 * std::log(o->factor) + 1 : 1.0;
    return KVT_OK;
  });
}

int kvt_rotary_create(uint32_t rotary_dim, int interleaved, const double* freq, double magnitude,
                      kvt_rotary** out) {
  return guarded([&]() -> int {
    if (!freq || !out) return fail(KVT_ERR_INVALID, "kvt_rotary_create: null argument");
    if (rotary_dim < 2 || rotary_dim > 256 || rotary_dim % 2 != 0)
      return fail(KVT_ERR_INVALID, "kvt_rotary_create: rotary_dim must be even, 2 to 256");
    if (!std::isfinite(static_cast<float>(magnitude)))
      return fail(KVT_ERR_INVALID, "kvt_rotary_create: magnitude is not finite in 32 bits");
    for (uint32_t i = 0; i < rotary_dim / 2; ++i)
      if (!std::isfinite(freq[i])) return fail(KVT_ERR_INVALID, "kvt_rotary_create: a frequency is not finite");
    std::unique_ptr<kvt_rotary> r(new kvt_rotary());
    r->dim = rotary_dim;
    r->interleaved = interleaved != 0;
    r->magnitude = static_cast<float>(magnitude);
    for (uint32_t i = 0; i < rotary_dim / 2; ++i) r->turns[i] = freq[i] / (2 * 3.14159265358979323846);
    *out = r.release();
    return KVT_OK;
  });
}

void kvt_rotary_destroy(kvt_rotary* r) { delete r; }

}  // extern "C"
