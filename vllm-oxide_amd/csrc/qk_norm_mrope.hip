// The attention prologue with positions on several axes, fused with the KV append: per
// token, RMSNorm of q and k per head, rotation of each frequency by the position on its
// own axis, q written for attention, k and v into their cache slots.
//
//   y = x * w / sqrt(mean(x^2) + eps),  j < D/2, r = row positions[axis(j)][t] of the table:
//   out[j]       = y[j] cos_r[j] - y[j + D/2] sin_r[j]
//   out[j + D/2] = y[j + D/2] cos_r[j] + y[j] sin_r[j]
// all in fp32 and rounded once.  The single-axis prologue (qk_norm_rope.hip) rounds
// after norm, weight and rotation as the reference does; this one has no reference to
// agree with bit for bit, and one rounding is the more exact result.
//
// Bound by HBM: 4 bytes an element (in and out), about 10 flops.  A wave works on one
// token: D / 16 lanes hold a head (lane i elements [8 i, 8 i + 8) of each half, so
// rotation partners meet in a lane and rows move 16 bytes at a time), 8 heads at D = 128
// at once, and it walks the token's heads with the next rows' loads issued before the
// present ones are worked on.  The positions, the cos / sin values of the lane's eight
// frequencies and the norm weights are then loaded once for all of the token's heads.
// 16384 tokens of 32 + 8 + 8 heads, D 128 (403 MB): 67 us into outputs that stay where they
// are (6.0 TB/s), 80 where the caches have to be written back as well (5.05 TB/s); a copy
// of this size runs at 5.4.  64 tokens take 3.8 us, a launch and three dependent loads.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "cdna4_tile.hpp"
#include "oxide_common.hpp"

namespace {

constexpr int kMropeThreads = 256;
constexpr int kMaxAxes = 4;
constexpr int64_t kMaxTokens = 1 << 25;  // a wave each: a launch holds fewer than 2^32 lanes
constexpr int E = 8;  // elements of each half per lane

__device__ __forceinline__ float lo_f32(Bf16Tag, uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f32(Bf16Tag, uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ float lo_f32(F16Tag, uint32_t w) {
  return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w)));
}
__device__ __forceinline__ float hi_f32(F16Tag, uint32_t w) {
  return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w >> 16)));
}

struct MropeParams {
  uint16_t* q_out;            // [T, Hq, D]
  uint16_t* k_out;            // [T, Hkv, D] or null
  const uint16_t* qkv;        // [T, qkv_stride], row = q | k | v
  const uint16_t* q_weight;   // [D] or null (no norm)
  const uint16_t* k_weight;   // [D] or null
  const float* cos_sin;       // [max_position, D]
  const int32_t* positions;   // [axes, T]
  uint16_t* key_cache;        // [num_slots, Hkv, D]
  uint16_t* value_cache;
  const int64_t* slot_mapping;  // [T] or null
  int64_t num_slots;
  int64_t qkv_stride;
  int64_t num_tokens;
  int max_position;
  int num_axes;
  int num_heads;
  int num_kv_heads;
  int rounds;  // of kHeads heads that a wave walks
  float eps;
  uint32_t axis[4];  // axis of frequency j: bits 2 (j % 16) of word j / 16
};

// The two 16-byte slices of a head row that a lane holds.
struct Slices {
  uint4 a, b;
};

template <int D, bool V, bool ONCE>
__device__ __forceinline__ Slices load_slices(const uint16_t* row, int sub) {
  Slices s;
  if constexpr (V && !ONCE) {
    s.a = *reinterpret_cast<const uint4*>(row + sub * E);
    s.b = *reinterpret_cast<const uint4*>(row + D / 2 + sub * E);
  } else if constexpr (V) {
    // Rows read once: non-temporal loads keep them from displacing cached lines.
    typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
    s.a = __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(row + sub * E)));
    s.b = __builtin_bit_cast(uint4,
                             __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(row + D / 2 + sub * E)));
  } else {
    uint16_t r1[E], r2[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      r1[e] = row[sub * E + e];
      r2[e] = row[D / 2 + sub * E + e];
    }
    __builtin_memcpy(&s.a, r1, sizeof(s.a));
    __builtin_memcpy(&s.b, r2, sizeof(s.b));
  }
  return s;
}

template <int D, bool V>
__device__ __forceinline__ void store_slices(uint16_t* row, int sub, Slices s) {
  if constexpr (V) {
    *reinterpret_cast<uint4*>(row + sub * E) = s.a;
    *reinterpret_cast<uint4*>(row + D / 2 + sub * E) = s.b;
  } else {
    uint16_t r1[E], r2[E];
    __builtin_memcpy(r1, &s.a, sizeof(s.a));
    __builtin_memcpy(r2, &s.b, sizeof(s.b));
#pragma unroll
    for (int e = 0; e < E; ++e) {
      row[sub * E + e] = r1[e];
      row[D / 2 + sub * E + e] = r2[e];
    }
  }
}

template <class Tag>
__device__ __forceinline__ void widen(Slices s, float* x1, float* x2) {
  const uint32_t a[4] = {s.a.x, s.a.y, s.a.z, s.a.w}, b[4] = {s.b.x, s.b.y, s.b.z, s.b.w};
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    x1[e] = lo_f32(Tag{}, a[e / 2]);
    x1[e + 1] = hi_f32(Tag{}, a[e / 2]);
    x2[e] = lo_f32(Tag{}, b[e / 2]);
    x2[e + 1] = hi_f32(Tag{}, b[e / 2]);
  }
}

template <class Tag>
__device__ __forceinline__ Slices narrow(const float* y1, const float* y2) {
  uint32_t a[4], b[4];
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    a[e / 2] = pack2(Tag{}, y1[e], y1[e + 1]);
    b[e / 2] = pack2(Tag{}, y2[e], y2[e + 1]);
  }
  return Slices{make_uint4(a[0], a[1], a[2], a[3]), make_uint4(b[0], b[1], b[2], b[3])};
}

template <class Tag, int D, bool V>
__global__ __launch_bounds__(kMropeThreads) void qk_norm_mrope_cache_kernel(MropeParams p) {
  constexpr int kLanes = D / 16;        // of a head
  constexpr int kHeads = 64 / kLanes;   // that a wave holds at once
  const int lane = threadIdx.x & 63;
  const int sub = lane % kLanes;
  // The wave's token, positions and slot are scalars.
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kMropeThreads / 64) +
                    __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= p.num_tokens) return;
  const int q_heads = p.num_heads, qk_heads = p.num_heads + p.num_kv_heads, heads = qk_heads + p.num_kv_heads;
  const uint16_t* row = p.qkv + t * p.qkv_stride;
  int h = static_cast<int>(blockIdx.y) * p.rounds * kHeads + lane / kLanes;
  const int end = min(heads, h - lane / kLanes + p.rounds * kHeads);

  // Positions first: the table's rows wait for them, and loads return in order.
  int32_t pos[kMaxAxes];
#pragma unroll
  for (int a = 0; a < kMaxAxes; ++a) pos[a] = p.positions[min(a, p.num_axes - 1) * p.num_tokens + t];
  int64_t slot = *(p.slot_mapping ? p.slot_mapping + t : reinterpret_cast<const int64_t*>(p.cos_sin));
  // Past the last head a lane reads the last head's row and writes nothing.
  Slices next = load_slices<D, V, true>(row + static_cast<int64_t>(min(h, heads - 1)) * D, sub);
  if (!p.slot_mapping || slot >= p.num_slots) slot = -1;
  uint32_t owner = p.axis[0];
#pragma unroll
  for (int w = 1; w < D / 32; ++w) owner = sub / 2 == w ? p.axis[w] : owner;
  owner >>= 16 * (sub & 1);
#pragma unroll
  for (int a = 0; a < kMaxAxes; ++a) pos[a] = min(max(pos[a], 0), p.max_position - 1);
  float c[E], s[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const uint32_t a = (owner >> (2 * e)) & 3u;
    int at = pos[0];
#pragma unroll
    for (int b = 1; b < kMaxAxes; ++b) at = a == static_cast<uint32_t>(b) ? pos[b] : at;
    const float* cs = p.cos_sin + static_cast<int64_t>(at) * D + sub * E + e;
    c[e] = cs[0];
    s[e] = cs[D / 2];
  }
  Slices wq{}, wk{};
  if (p.q_weight) wq = load_slices<D, V, false>(p.q_weight, sub);
  if (p.k_weight) wk = load_slices<D, V, false>(p.k_weight, sub);

  for (int h0 = h - lane / kLanes; h0 < end; h0 += kHeads, h += kHeads) {
    const Slices now = next;
    if (h0 + kHeads < end) next = load_slices<D, V, true>(row + static_cast<int64_t>(min(h + kHeads, heads - 1)) * D, sub);
    const bool is_q = h < q_heads;
    float x1[E], x2[E];
    widen<Tag>(now, x1, x2);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) ss += x1[e] * x1[e] + x2[e] * x2[e];
#pragma unroll
    for (int m = 1; m < kLanes; m <<= 1) ss += __shfl_xor(ss, m);
    if ((is_q ? p.q_weight : p.k_weight) != nullptr) {
      const float inv = 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
      float w1[E], w2[E];
      widen<Tag>(is_q ? wq : wk, w1, w2);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        x1[e] = x1[e] * inv * w1[e];
        x2[e] = x2[e] * inv * w2[e];
      }
    }
    float y1[E], y2[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      y1[e] = x1[e] * c[e] - x2[e] * s[e];
      y2[e] = x2[e] * c[e] + x1[e] * s[e];
    }
    const Slices turned = narrow<Tag>(y1, y2);
    if (is_q) {
      store_slices<D, V>(p.q_out + (t * p.num_heads + h) * D, sub, turned);
    } else if (h < qk_heads) {
      const int kh = h - q_heads;
      if (p.k_out) store_slices<D, V>(p.k_out + (t * p.num_kv_heads + kh) * D, sub, turned);
      if (slot >= 0) store_slices<D, V>(p.key_cache + (slot * p.num_kv_heads + kh) * D, sub, turned);
    } else if (h < heads && slot >= 0) {
      store_slices<D, V>(p.value_cache + (slot * p.num_kv_heads + (h - qk_heads)) * D, sub, now);
    }
  }
}

template <class Tag, int D>
void launch_mrope(MropeParams p, bool vec, hipStream_t s) {
  constexpr int kHeads = 64 / (D / 16);
  const int rounds = (p.num_heads + 2 * p.num_kv_heads + kHeads - 1) / kHeads;
  // A wave for a token's heads, or for a round of them where that leaves most of the chip
  // idle: 5.9 against 7.2 us at 64 tokens of 32 + 8 + 8 heads, 149 against 70 at 16k.
  const int parts = static_cast<int>(std::min<int64_t>(rounds, std::max<int64_t>(1, 2048 / p.num_tokens)));
  p.rounds = (rounds + parts - 1) / parts;
  const dim3 grid(static_cast<unsigned>((p.num_tokens + kMropeThreads / 64 - 1) / (kMropeThreads / 64)),
                  static_cast<unsigned>((rounds + p.rounds - 1) / p.rounds));
  if (vec)
    hipLaunchKernelGGL((qk_norm_mrope_cache_kernel<Tag, D, true>), grid, dim3(kMropeThreads), 0, s, p);
  else
    hipLaunchKernelGGL((qk_norm_mrope_cache_kernel<Tag, D, false>), grid, dim3(kMropeThreads), 0, s, p);
}

}  // namespace

extern "C" void qk_norm_mrope_and_cache(void* q_out, void* k_out, const void* qkv, int64_t qkv_row_stride,
                                        const void* q_norm_weight, const void* k_norm_weight, double eps,
                                        const float* cos_sin_cache, int64_t max_position, const int32_t* positions,
                                        int64_t num_axes, const int32_t* sections, int interleaved, void* key_cache,
                                        void* value_cache, int64_t num_slots, const int64_t* slot_mapping,
                                        int64_t num_tokens, int64_t num_heads, int64_t num_kv_heads,
                                        int64_t head_dim, int dtype, void* stream) {
  if (dtype != OXIDE_DTYPE_BF16 && dtype != OXIDE_DTYPE_F16) {
    oxide::set_error(OXIDE_ERR_UNSUPPORTED_DTYPE);
    return;
  }
  if (head_dim != 64 && head_dim != 128) {
    oxide::set_error(OXIDE_ERR_UNSUPPORTED_SHAPE);
    return;
  }
  if (num_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_tokens > kMaxTokens ||
      num_heads > 4096 || num_kv_heads > 4096 || max_position <= 0 || max_position > INT32_MAX || num_slots < 0 ||
      qkv_row_stride < (num_heads + 2 * num_kv_heads) * head_dim || num_axes < 1 || num_axes > kMaxAxes ||
      !sections) {
    oxide::set_error(OXIDE_ERR_INVALID_ARGUMENT);
    return;
  }
  // The axis of every frequency.
  const int half = static_cast<int>(head_dim / 2), axes = static_cast<int>(num_axes);
  int64_t sum = 0;
  bool good = true;
  for (int a = 0; a < axes; ++a) {
    good = good && sections[a] >= 0;
    sum += sections[a];
    if (interleaved && a > 0 && sections[a] > 0)
      good = good && int64_t{axes} * (sections[a] - 1) + a < half;
  }
  if (!good || sum != half) {
    oxide::set_error(OXIDE_ERR_INVALID_ARGUMENT);
    return;
  }
  MropeParams p{};
  for (int j = 0, a = 0, left = sections[0]; j < half; ++j) {
    int owner = 0;
    if (interleaved) {
      owner = j % axes > 0 && j < axes * sections[j % axes] ? j % axes : 0;
    } else {
      while (left == 0) left = sections[++a];
      --left;
      owner = a;
    }
    p.axis[j / 16] |= static_cast<uint32_t>(owner) << (2 * (j % 16));
  }
  if (num_tokens == 0) return;
  const int64_t qkv_elems = (num_tokens - 1) * qkv_row_stride + (num_heads + 2 * num_kv_heads) * head_dim;
  if (!q_out || !qkv || !cos_sin_cache || !positions || (slot_mapping && (!key_cache || !value_cache)) ||
      oxide::overlap16(q_out, num_tokens * num_heads * head_dim, qkv, qkv_elems) ||
      (k_out && oxide::overlap16(k_out, num_tokens * num_kv_heads * head_dim, qkv, qkv_elems))) {
    oxide::set_error(OXIDE_ERR_INVALID_ARGUMENT);
    return;
  }
  p.q_out = static_cast<uint16_t*>(q_out);
  p.k_out = static_cast<uint16_t*>(k_out);
  p.qkv = static_cast<const uint16_t*>(qkv);
  p.q_weight = static_cast<const uint16_t*>(q_norm_weight);
  p.k_weight = static_cast<const uint16_t*>(k_norm_weight);
  p.cos_sin = cos_sin_cache;
  p.positions = positions;
  p.key_cache = static_cast<uint16_t*>(key_cache);
  p.value_cache = static_cast<uint16_t*>(value_cache);
  p.slot_mapping = slot_mapping;
  p.num_slots = num_slots;
  p.qkv_stride = qkv_row_stride;
  p.num_tokens = num_tokens;
  p.max_position = static_cast<int>(max_position);
  p.num_axes = axes;
  p.num_heads = static_cast<int>(num_heads);
  p.num_kv_heads = static_cast<int>(num_kv_heads);
  p.eps = static_cast<float>(eps);
  // Head slices are D * 2 bytes apart (a multiple of 16): 16-byte accesses need the base
  // pointers and the qkv row stride aligned.
  const bool vec = oxide::aligned16(qkv) && oxide::aligned16(q_out) && oxide::aligned16(k_out) &&
                   oxide::aligned16(key_cache) && oxide::aligned16(value_cache) && oxide::aligned16(q_norm_weight) &&
                   oxide::aligned16(k_norm_weight) && qkv_row_stride % 8 == 0;
  hipStream_t s = oxide::as_stream(stream);
  const bool bf16 = dtype == OXIDE_DTYPE_BF16;
  if (head_dim == 128)
    bf16 ? launch_mrope<Bf16Tag, 128>(p, vec, s) : launch_mrope<F16Tag, 128>(p, vec, s);
  else
    bf16 ? launch_mrope<Bf16Tag, 64>(p, vec, s) : launch_mrope<F16Tag, 64>(p, vec, s);
  oxide::check_launch();
}
