// Rotary positions: the query and key heads of a layer turned by the angles
// of their tokens' positions, on their own or on the way into the paged
// cache (the keys rotated and stored, the values stored, one launch).
//
// Pair j of a head's first rotary_dim dims, (x1, x2) = dims (j, j +
// rotary_dim / 2) in the half layout or (2 j, 2 j + 1) in the interleaved
// one, becomes
//   (x1 cos a - x2 sin a, x2 cos a + x1 sin a),  a = position * inv_freq[j],
// in fp32 with one rounding to the element type; the other dims pass
// through.  The angles of far positions need more than fp32 (position 131071
// at one radian per position has an fp32 spacing of 2^-7), so cosine and
// sine come from a table built once in fp64, [max_position][rotary_dim / 2]
// float2; a factor of the scaling multiplies both.
#include <type_traits>

#include "nkv_common.h"

namespace nkv {
namespace {

__global__ __launch_bounds__(256) void rotary_table_kernel(const double* __restrict__ inv_freq,
                                                           double factor, int64_t entries,
                                                           int32_t half, float2* __restrict__ table) {
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; e < entries; e += stride) {
    const int64_t position = e / half;
    double sine, cosine;
    sincos(static_cast<double>(position) * inv_freq[e - position * half], &sine, &cosine);
    table[e] = make_float2(static_cast<float>(cosine * factor), static_cast<float>(sine * factor));
  }
}

// Element types: to and from fp32 (rounded to nearest even).
struct Bf16 {
  typedef uint16_t T;
  static __device__ __forceinline__ float get(T v) { return __uint_as_float(static_cast<uint32_t>(v) << 16); }
  static __device__ __forceinline__ T put(float f) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f)); }
};
struct Fp16 {
  typedef uint16_t T;
  static __device__ __forceinline__ float get(T v) { return static_cast<float>(__builtin_bit_cast(_Float16, v)); }
  // The empty asm keeps the conversion apart from the fma before it: as one
  // instruction it rounds once, and the compiler takes that in some forms of
  // the kernel and not in others.
  static __device__ __forceinline__ T put(float f) {
    asm("" : "+v"(f));
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
  }
};
struct Fp32 {
  typedef float T;
  static __device__ __forceinline__ float get(T v) { return v; }
  static __device__ __forceinline__ T put(float f) { return f; }
};

// One launch: strides in elements.  A null k_out, or key_cache, is not written.
struct RotaryArgs {
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  void* k_out;
  void* key_cache;
  void* value_cache;
  const void* positions;
  const int32_t* slots;
  const float2* table;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;
  int64_t q_out_token, q_out_head, k_out_token, k_out_head;
  int64_t position_row;  // elements between position rows (sections), 0 without
  int64_t max_position, num_slots;
  int32_t num_tokens, q_heads, kv_heads, head_dim, half, wide_positions;
  int32_t section_end0, section_end1;  // first pairs of the second and third position row
  int32_t lanes;  // threads of a head
};

constexpr int kRotaryThreads = 256;

// Streaming accesses of a vector (16 bytes) or a single element.
template <typename P>
__device__ __forceinline__ P load_once(const P* p) {
  if constexpr (sizeof(P) == 16) return __builtin_bit_cast(P, load_stream(reinterpret_cast<const u32x4*>(p)));
  return *p;
}
template <typename P>
__device__ __forceinline__ void store_once(P* p, const P& v) {
  if constexpr (sizeof(P) == 16) {
    store_stream(reinterpret_cast<u32x4*>(p), __builtin_bit_cast(u32x4, v));
  } else {
    *p = v;
  }
}

// One thread per two W-element vectors of a head, of every q, k and (stored) v
// head of a token.  Its vectors lie in the two halves of the rotated dims, of
// the dims behind them, or of a v head, so that neighbouring threads move
// neighbouring vectors: in the half layout they hold the two sides of W pairs,
// in the interleaved one W / 2 pairs each (with 2 W dims in a row per thread
// that form took 44.3 us where the half layout took 37.0, 8,192 tokens of 32 q
// and 8 kv heads).
//
// Bound by HBM: every row is read and written once, next to which the 6
// operations of a pair and the table (512 bytes per token at 128 dims, from
// the caches for all heads but one) are little.  Flat over tokens and heads
// the grid is large for a single chunk and one round for a decode step.  What
// no later kernel reads from the caches (inputs, cache rows) streams past
// them; q_out, read next by the attention, does not.  With the store, bf16:
// 8,192 tokens of 28 q and 4 kv heads, three position rows, 27.6 us, 5.5 TB/s,
// in fp32 49.9 us, 6.1 TB/s; 64 tokens 3.1 us, a launch's latency.  The half
// layout's angles as two runs of loads instead of one lost 15 %.
template <typename E, int W, bool kInterleaved, bool kStore>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryArgs a) {
  typedef typename E::T T;
  struct alignas(sizeof(T) * W) Pack {
    T e[W];
  };
  const uint32_t heads = a.q_heads + (kStore ? 2 : 1) * a.kv_heads;
  const uint32_t thread = blockIdx.x * kRotaryThreads + threadIdx.x;  // below 2^31 (the launch)
  const uint32_t head_of_all = thread / a.lanes;
  const int32_t lane = static_cast<int32_t>(thread - head_of_all * a.lanes);
  const int64_t token = head_of_all / heads;
  const int32_t h = static_cast<int32_t>(head_of_all - static_cast<uint32_t>(token) * heads);
  if (token >= a.num_tokens) return;
  const int32_t kh = h - a.q_heads, vh = kh - a.kv_heads;
  const bool is_v = kStore && vh >= 0;
  const int32_t j0 = lane * W;
  const bool rotated = j0 < a.half && !is_v;
  int32_t at1, at2;
  if (W == 1 && (kInterleaved || !rotated)) {  // single elements: two in a row
    at1 = 2 * j0;
    at2 = 2 * j0 + 1;
  } else {
    const int32_t begin = rotated || is_v ? 0 : a.half;  // in vectors' dims, of a half
    const int32_t width = rotated ? a.half : is_v ? a.head_dim / 2 : a.head_dim / 2 - a.half;
    at1 = 2 * begin + (j0 - begin);
    at2 = at1 + width;
  }
  const bool both = at2 < a.head_dim;  // (an odd dim at the end, W == 1)

  // The vectors are on their way while the angles are looked up.
  const T* const src = kh < 0  ? static_cast<const T*>(a.q) + token * a.q_token + h * a.q_head
                       : is_v ? static_cast<const T*>(a.v) + token * a.v_token + vh * a.v_head
                              : static_cast<const T*>(a.k) + token * a.k_token + kh * a.k_head;
  Pack x = load_once(reinterpret_cast<const Pack*>(src + at1)), y{};
  if (both) y = load_once(reinterpret_cast<const Pack*>(src + at2));
  int64_t position[3];
#pragma unroll
  for (int r = 0; r < 3; ++r) {
    const int64_t at = r * a.position_row + token;
    position[r] = a.wide_positions ? static_cast<const int64_t*>(a.positions)[at]
                                   : static_cast<const int32_t*>(a.positions)[at];
  }
  int64_t slot = -1;
  if (kStore && kh >= 0) slot = a.slots[token];
  const bool known = position[0] >= 0 && position[0] < a.max_position && position[1] >= 0 &&
                     position[1] < a.max_position && position[2] >= 0 && position[2] < a.max_position;
  if (rotated && known) {
    auto row_of = [&](int32_t j) { return j < a.section_end0 ? 0 : j < a.section_end1 ? 1 : 2; };
    auto entry = [&](int32_t j) {
      const int row = row_of(j);
      const int64_t p = row == 0 ? position[0] : row == 1 ? position[1] : position[2];
      return a.table + p * a.half + j;
    };
    float cosine[W], sine[W];
    if constexpr (W == 1) {
      const float2 cs = *entry(j0);
      cosine[0] = cs.x;
      sine[0] = cs.y;
    } else {
      constexpr int kSegments = kInterleaved ? 2 : 1;
      constexpr int kPairs = W / kSegments;
#pragma unroll
      for (int s = 0; s < kSegments; ++s) {  // W / 2 pairs, of the first and the second vector's (interleaved)
        const int32_t j = kInterleaved ? (j0 + s * a.half) / 2 : j0;
        float* const c = cosine + s * kPairs;
        float* const d = sine + s * kPairs;
        if (row_of(j) == row_of(j + kPairs - 1)) {  // one position: 16 bytes at a time
          const float4* const from = reinterpret_cast<const float4*>(entry(j));
#pragma unroll
          for (int w = 0; w < kPairs / 2; ++w) {
            const float4 cs = from[w];
            c[2 * w] = cs.x;
            d[2 * w] = cs.y;
            c[2 * w + 1] = cs.z;
            d[2 * w + 1] = cs.w;
          }
        } else {
#pragma unroll
          for (int w = 0; w < kPairs; ++w) {
            const float2 cs = *entry(j + w);
            c[w] = cs.x;
            d[w] = cs.y;
          }
        }
      }
    }
    float f[2 * W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      f[w] = E::get(x.e[w]);
      f[W + w] = E::get(y.e[w]);
    }
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int i1 = kInterleaved ? 2 * w : w, i2 = kInterleaved ? 2 * w + 1 : W + w;
      const float x1 = f[i1], x2 = f[i2];
      // Fused alike in every form, so that all give the same bits.
      f[i1] = __builtin_fmaf(x1, cosine[w], -(x2 * sine[w]));
      f[i2] = __builtin_fmaf(x2, cosine[w], x1 * sine[w]);
    }
#pragma unroll
    for (int w = 0; w < W; ++w) {
      x.e[w] = E::put(f[w]);
      y.e[w] = E::put(f[W + w]);
    }
  } else if (!known) {
    x = Pack{};
    y = Pack{};
  }

  if (kh < 0) {
    T* const dst = static_cast<T*>(a.q_out) + token * a.q_out_token + h * a.q_out_head;
    *reinterpret_cast<Pack*>(dst + at1) = x;
    if (both) *reinterpret_cast<Pack*>(dst + at2) = y;
    return;
  }
  if (!is_v && a.k_out != nullptr) {
    T* const dst = static_cast<T*>(a.k_out) + token * a.k_out_token + kh * a.k_out_head;
    *reinterpret_cast<Pack*>(dst + at1) = x;
    if (both) *reinterpret_cast<Pack*>(dst + at2) = y;
  }
  if (kStore && slot >= 0 && slot < a.num_slots && known) {
    T* const cache = static_cast<T*>(is_v ? a.value_cache : a.key_cache);
    T* const dst = cache + (slot * a.kv_heads + (is_v ? vh : kh)) * a.head_dim;
    store_once(reinterpret_cast<Pack*>(dst + at1), x);
    if (both) store_once(reinterpret_cast<Pack*>(dst + at2), y);
  }
}

template <typename E, int W>
void (*rotary_kernel_for(bool interleaved, bool store))(RotaryArgs) {
  if (interleaved) return store ? rotary_kernel<E, W, true, true> : rotary_kernel<E, W, true, false>;
  return store ? rotary_kernel<E, W, false, true> : rotary_kernel<E, W, false, false>;
}

// [tokens, heads, dim] elements of one tensor, addresses and strides in elements.
struct HeadsView {
  int64_t at, token, head, heads;
};
// The elements from the first to past the last of a token's heads, of all.
int64_t span_of(const HeadsView& v, int64_t dim) { return (v.heads - 1) * v.head + dim; }
int64_t extent_of(const HeadsView& v, int64_t tokens, int64_t dim) {
  return (tokens - 1) * v.token + span_of(v, dim);
}
bool same_view(const HeadsView& a, const HeadsView& b, int64_t tokens) {
  return a.at == b.at && a.heads == b.heads && (tokens == 1 || a.token == b.token) &&
         (a.heads == 1 || a.head == b.head);
}
// Whether two elements of a view are one.
bool folds(const HeadsView& v, int64_t tokens, int64_t dim) {
  if (v.heads > 1 && v.head < dim) return true;
  if (tokens > 1 && v.token < dim) return true;
  return tokens > 1 && v.heads > 1 && v.token < span_of(v, dim) && v.head < (tokens - 1) * v.token + dim;
}
// Whether two views may have an element in common.  Views whose ranges meet
// have none where they lie apart within one row or within one head's step of
// the rows they are cut from (q, k and v of a fused projection).
bool meet(const HeadsView& a, const HeadsView& b, int64_t tokens, int64_t dim) {
  if (a.at + extent_of(a, tokens, dim) <= b.at || b.at + extent_of(b, tokens, dim) <= a.at) return false;
  auto apart = [](int64_t step, int64_t delta, int64_t la, int64_t lb) {
    const int64_t d = ((delta % step) + step) % step;
    return d >= la && d + lb <= step;
  };
  if (tokens > 1 && a.token == b.token && a.token > 0 &&
      apart(a.token, b.at - a.at, span_of(a, dim), span_of(b, dim))) {
    return false;
  }
  return !(a.heads > 1 && b.heads > 1 && a.head == b.head && a.head > 0 &&
           (tokens == 1 || (a.token % a.head == 0 && b.token % a.head == 0)) &&
           apart(a.head, b.at - a.at, dim, dim));
}

}  // namespace
}  // namespace nkv

extern "C" int nkv_rotary_table(const double* inv_freq, double factor, int64_t max_position,
                                int64_t rotary_dim, float* table, void* stream) {
  using namespace nkv;
  if (rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > NKV_ROTARY_MAX_HEAD_DIM ||
      max_position <= 0 || max_position > INT32_MAX) {
    return nkv_fail(NKV_E_INVALID,
                    "nkv_rotary_table: need an even rotary_dim in [2, %d] and max_position in [1, 2^31)",
                    NKV_ROTARY_MAX_HEAD_DIM);
  }
  if (!inv_freq || !table) return nkv_fail(NKV_E_INVALID, "nkv_rotary_table: null pointer");
  if (reinterpret_cast<uint64_t>(table) % 16 != 0) {
    return nkv_fail(NKV_E_INVALID, "nkv_rotary_table: table must be 16-byte aligned");
  }
  const int64_t entries = max_position * (rotary_dim / 2);
  const int64_t blocks = (entries + 255) / 256;
  rotary_table_kernel<<<dim3(static_cast<unsigned>(blocks < 8192 ? blocks : 8192)), dim3(256), 0,
                        static_cast<hipStream_t>(stream)>>>(
      inv_freq, factor, entries, static_cast<int32_t>(rotary_dim / 2), reinterpret_cast<float2*>(table));
  return nkv_check_launch("nkv_rotary_table");
}

extern "C" int nkv_rotary(const nkv_rotary_desc* d, void* stream) {
  using namespace nkv;
  if (d == nullptr) return nkv_fail(NKV_E_INVALID, "nkv_rotary: null descriptor");
  const int eb = element_bytes(d->dtype);
  if (eb == 0) return nkv_fail(NKV_E_INVALID, "nkv_rotary: unknown dtype %d", d->dtype);
  if (d->num_tokens < 0 || d->num_q_heads < 0 || d->num_kv_heads < 0 || d->head_dim <= 0 ||
      d->head_dim > NKV_ROTARY_MAX_HEAD_DIM || d->num_q_heads > NKV_ROTARY_MAX_HEADS ||
      d->num_kv_heads > NKV_ROTARY_MAX_HEADS || d->num_tokens > INT32_MAX) {
    return nkv_fail(NKV_E_INVALID,
                    "nkv_rotary: tokens outside [0, 2^31), heads outside [0, %d] or head_dim outside [1, %d]",
                    NKV_ROTARY_MAX_HEADS, NKV_ROTARY_MAX_HEAD_DIM);
  }
  if (d->rotary_dim < 2 || d->rotary_dim % 2 != 0 || d->rotary_dim > d->head_dim) {
    return nkv_fail(NKV_E_INVALID, "nkv_rotary: rotary_dim must be even, in [2, head_dim]");
  }
  if (d->layout != NKV_ROTARY_HALF && d->layout != NKV_ROTARY_INTERLEAVED) {
    return nkv_fail(NKV_E_INVALID, "nkv_rotary: unknown layout %d", d->layout);
  }
  if (d->position_bytes != 4 && d->position_bytes != 8) {
    return nkv_fail(NKV_E_INVALID, "nkv_rotary: positions must be 4 or 8 bytes each");
  }
  if (d->max_position <= 0 || d->max_position > INT32_MAX) {
    return nkv_fail(NKV_E_INVALID, "nkv_rotary: max_position must be in [1, 2^31)");
  }
  const int64_t half = d->rotary_dim / 2;
  if (d->position_row_stride < 0 ||
      (d->position_row_stride > 0 &&
       (d->section_ends[0] < 0 || d->section_ends[1] < d->section_ends[0] || d->section_ends[1] > half))) {
    return nkv_fail(NKV_E_INVALID,
                    "nkv_rotary: sections must split the pairs in order: 0 <= end0 <= end1 <= rotary_dim / 2");
  }
  const bool store = d->key_cache != nullptr || d->value_cache != nullptr;
  if (d->num_slots < 0 || d->num_slots > INT32_MAX) {
    return nkv_fail(NKV_E_INVALID, "nkv_rotary: num_slots outside [0, 2^31)");
  }
  for (int64_t s : {d->q_token_stride, d->q_head_stride, d->k_token_stride, d->k_head_stride,
                    d->v_token_stride, d->v_head_stride, d->q_out_token_stride, d->q_out_head_stride,
                    d->k_out_token_stride, d->k_out_head_stride}) {
    if (s < 0) return nkv_fail(NKV_E_INVALID, "nkv_rotary: negative stride");
  }
  if (d->num_tokens == 0 || d->num_q_heads + d->num_kv_heads == 0) return NKV_OK;
  if (!d->positions || !d->table || (d->num_q_heads > 0 && (!d->q || !d->q_out)) ||
      (d->num_kv_heads > 0 && (!d->k || (!store && !d->k_out))) ||
      (store && (!d->key_cache || !d->value_cache || !d->v || !d->slot_mapping))) {
    return nkv_fail(NKV_E_INVALID, "nkv_rotary: null pointer");
  }
  // 16-byte vectors where every pointer, stride and part of a head allows
  // them, single elements otherwise (head views cut at odd places).
  const uint64_t vec = 16 / static_cast<uint64_t>(eb);
  uint64_t bits = 0;
  for (const void* p : {d->q, d->k, static_cast<const void*>(d->q_out), static_cast<const void*>(d->k_out),
                        store ? d->v : nullptr, static_cast<const void*>(d->key_cache),
                        static_cast<const void*>(d->value_cache)}) {
    bits |= reinterpret_cast<uint64_t>(p);
  }
  if (bits % static_cast<uint64_t>(eb) != 0 || reinterpret_cast<uint64_t>(d->table) % 16 != 0 ||
      reinterpret_cast<uint64_t>(d->positions) % static_cast<uint64_t>(d->position_bytes) != 0) {
    return nkv_fail(NKV_E_INVALID, "nkv_rotary: pointers not aligned to their elements (table: 16 bytes)");
  }
  // Outputs: their own input or memory of their own, and no element twice.
  auto view = [&](const void* p, int64_t token, int64_t head, int64_t n) {
    return HeadsView{static_cast<int64_t>(reinterpret_cast<uint64_t>(p) / static_cast<uint64_t>(eb)), token, head, n};
  };
  const HeadsView q = view(d->q, d->q_token_stride, d->q_head_stride, d->num_q_heads);
  const HeadsView k = view(d->k, d->k_token_stride, d->k_head_stride, d->num_kv_heads);
  const HeadsView v = view(store ? d->v : nullptr, d->v_token_stride, d->v_head_stride, d->num_kv_heads);
  const HeadsView qo = view(d->q_out, d->q_out_token_stride, d->q_out_head_stride, d->num_q_heads);
  const HeadsView ko = view(d->k_out, d->k_out_token_stride, d->k_out_head_stride, d->num_kv_heads);
  const bool has_q = d->num_q_heads > 0, has_k = d->num_kv_heads > 0, has_ko = has_k && d->k_out != nullptr;
  const int64_t n = d->num_tokens, dim = d->head_dim;
  if ((has_q && (folds(qo, n, dim) || (!same_view(qo, q, n) && meet(qo, q, n, dim)) ||
                 (has_k && meet(qo, k, n, dim)) || (has_k && store && meet(qo, v, n, dim)))) ||
      (has_ko && (folds(ko, n, dim) || (!same_view(ko, k, n) && meet(ko, k, n, dim)) ||
                  (store && meet(ko, v, n, dim)) || (has_q && (meet(ko, q, n, dim) || meet(ko, qo, n, dim)))))) {
    return nkv_fail(NKV_E_INVALID,
                    "nkv_rotary: an output must be its own input or overlap no tensor of the call, "
                    "and hold each element once");
  }
  uint64_t strides = 0;
  for (int64_t s : {d->q_token_stride, d->q_head_stride, d->k_token_stride, d->k_head_stride,
                    d->q_out_token_stride, d->q_out_head_stride}) {
    strides |= static_cast<uint64_t>(s);
  }
  if (store) strides |= static_cast<uint64_t>(d->v_token_stride) | static_cast<uint64_t>(d->v_head_stride);
  if (d->k_out) strides |= static_cast<uint64_t>(d->k_out_token_stride) | static_cast<uint64_t>(d->k_out_head_stride);
  const bool wide = bits % 16 == 0 && strides % vec == 0 && half % static_cast<int64_t>(vec) == 0 &&
                    d->head_dim % static_cast<int64_t>(2 * vec) == 0;
  const int64_t w = wide ? static_cast<int64_t>(vec) : 1;
  const int64_t lanes = (d->head_dim + 2 * w - 1) / (2 * w);
  const int64_t heads = d->num_q_heads + (store ? 2 : 1) * d->num_kv_heads;
  // Threads are numbered in 31 bits: more tokens than that are several launches.
  const int64_t most = INT32_MAX / (lanes * heads);
  RotaryArgs a{};
  a.q = d->q;
  a.k = d->k;
  a.v = d->v;
  a.q_out = d->q_out;
  a.k_out = d->k_out;
  a.key_cache = d->key_cache;
  a.value_cache = d->value_cache;
  a.positions = d->positions;
  a.slots = d->slot_mapping;
  a.table = reinterpret_cast<const float2*>(d->table);
  a.q_token = d->q_token_stride;
  a.q_head = d->q_head_stride;
  a.k_token = d->k_token_stride;
  a.k_head = d->k_head_stride;
  a.v_token = d->v_token_stride;
  a.v_head = d->v_head_stride;
  a.q_out_token = d->q_out_token_stride;
  a.q_out_head = d->q_out_head_stride;
  a.k_out_token = d->k_out_token_stride;
  a.k_out_head = d->k_out_head_stride;
  a.position_row = d->position_row_stride;
  a.max_position = d->max_position;
  a.num_slots = d->num_slots;
  a.q_heads = static_cast<int32_t>(d->num_q_heads);
  a.kv_heads = static_cast<int32_t>(d->num_kv_heads);
  a.head_dim = static_cast<int32_t>(d->head_dim);
  a.half = static_cast<int32_t>(half);
  a.wide_positions = d->position_bytes == 8 ? 1 : 0;
  a.section_end0 = static_cast<int32_t>(d->section_ends[0]);
  a.section_end1 = static_cast<int32_t>(d->section_ends[1]);
  a.lanes = static_cast<int32_t>(lanes);
  const bool inter = d->layout == NKV_ROTARY_INTERLEAVED;
  void (*kernel)(RotaryArgs) = nullptr;
  if (d->dtype == NKV_DTYPE_FLOAT32) {
    kernel = wide ? rotary_kernel_for<Fp32, 4>(inter, store) : rotary_kernel_for<Fp32, 1>(inter, store);
  } else if (d->dtype == NKV_DTYPE_FLOAT16) {
    kernel = wide ? rotary_kernel_for<Fp16, 8>(inter, store) : rotary_kernel_for<Fp16, 1>(inter, store);
  } else {
    kernel = wide ? rotary_kernel_for<Bf16, 8>(inter, store) : rotary_kernel_for<Bf16, 1>(inter, store);
  }
  auto advance = [](auto*& p, int64_t bytes) {
    if (p != nullptr) p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(reinterpret_cast<uintptr_t>(p) + bytes);
  };
  for (int64_t done = 0; done < d->num_tokens; done += most) {
    const int64_t tokens = d->num_tokens - done < most ? d->num_tokens - done : most;
    a.num_tokens = static_cast<int32_t>(tokens);
    const int64_t blocks = (tokens * heads * lanes + kRotaryThreads - 1) / kRotaryThreads;
    kernel<<<dim3(static_cast<unsigned>(blocks)), dim3(kRotaryThreads), 0, static_cast<hipStream_t>(stream)>>>(a);
    if (int rc = nkv_check_launch("nkv_rotary")) return rc;
    advance(a.q, most * a.q_token * eb);
    advance(a.k, most * a.k_token * eb);
    advance(a.v, most * a.v_token * eb);
    advance(a.q_out, most * a.q_out_token * eb);
    advance(a.k_out, most * a.k_out_token * eb);
    advance(a.positions, most * d->position_bytes);
    advance(a.slots, most * 4);
  }
  return NKV_OK;
}
