// Linear attention with a decay for each head, for gfx950: per sequence and kv head n a
// state S [D, D] (key dimension first), fp32,
//   S_t = lambda_n S_{t-1} + k_t v_t^T,   lambda_n = exp(log_decay[n]),
//   out_t[h] = scale * q_t[h]^T S_t       for the query heads h of n.
// No reference counterpart: every layer of its models is softmax attention.
//
// linear_decode: one token.  Bound by HBM, the state read and written once (8 D^2 bytes
// a head against 4 D^2 + 2 G D^2 operations).  A workgroup holds kCols columns of one
// state in registers -- out's columns need S's columns only -- so nothing is joined
// between workgroups; the sum over the key dimension goes over the lanes that share a
// column, then over the waves through LDS.
#include <math.h>

#include <type_traits>

#include "cdna4_tile.hpp"
#include "oxide_common.hpp"

namespace {

__device__ __forceinline__ float to_f32(Bf16Tag, uint16_t h) { return __uint_as_float(static_cast<uint32_t>(h) << 16); }
__device__ __forceinline__ float to_f32(F16Tag, uint16_t h) {
  return static_cast<float>(__builtin_bit_cast(_Float16, h));
}

struct LinearParams {
  uint16_t* out;      // [T, Hq, D]
  const uint16_t* q;  // T rows of [Hq, D], q_stride apart
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_stride, k_stride, v_stride;
  const float* log_decay;        // [Hkv]
  float* state;                  // [num_slots, Hkv, D, D]
  const int32_t* slots;          // [batch]
  const uint32_t* context_lens;  // [batch] or null (prefill)
  const uint32_t* cu_q;          // [batch + 1] (prefill)
  int64_t total_q;
  int64_t num_slots;
  int batch, num_heads, num_kv_heads, group, max_q;
  float scale;
};

// lambda^n as a sum of two fp32: a rounded lambda is off by up to 2^-25, the same way
// in every step, so a state that a slowly decaying head carries over thousands of
// tokens would drift by thousands of times that.
struct Decay {
  float hi, lo;
  __device__ __forceinline__ float operator*(float x) const { return fmaf(x, hi, x * lo); }
};
__device__ __forceinline__ Decay decay_power(float log_decay, int n) {
  // Below -1e4 every power but the zeroth is 0 (also for -inf, whose zeroth is 1).
  const double e = exp(static_cast<double>(log_decay < -1e4f ? -1e4f : log_decay) * n);
  const float hi = static_cast<float>(e);
  // Grown out of fp32's range: no remainder to an infinity.
  return Decay{hi, __builtin_isinf(hi) ? 0.f : static_cast<float>(e - static_cast<double>(hi))};
}

constexpr int kDecodeThreads = 256;
constexpr int kDecodeCols = 32;  // state columns of a workgroup

// One token with the state's columns in registers: s[i] are 4 columns of key row
// i * kRows + row.  q (G heads) and k are in LDS as fp32.  Writes G x kDecodeCols
// outputs.
template <class Tag, int D>
__global__ __launch_bounds__(kDecodeThreads) void linear_decode(LinearParams p) {
  constexpr int kLanes = kDecodeCols / 4;           // lanes of a row's columns
  constexpr int kRows = kDecodeThreads / kLanes;    // rows that the workgroup holds at once
  constexpr int N = D / kRows;
  constexpr int kHeads = 8;  // query heads joined at a time
  __shared__ float s_q[kHeads][D];
  __shared__ float s_part[kHeads][kDecodeThreads / 64][kDecodeCols];
  const int slices = D / kDecodeCols;
  const int slice = blockIdx.x % slices;
  const int n = blockIdx.x / slices % p.num_kv_heads;
  const int b = blockIdx.x / slices / p.num_kv_heads;
  const int64_t slot = p.slots[b];
  if (slot < 0 || slot >= p.num_slots) return;
  const int lane = threadIdx.x % kLanes, row = threadIdx.x / kLanes;
  const int col = slice * kDecodeCols + lane * 4;
  float* state = p.state + (slot * p.num_kv_heads + n) * D * D + col;
  floatx4 s[N];
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = *reinterpret_cast<const floatx4*>(state + (i * kRows + row) * D);
  const uint16_t* k = p.k + b * p.k_stride + n * D;
  const uint16_t* v = p.v + b * p.v_stride + n * D + col;
  const Decay decay = decay_power(p.log_decay[n], 1);
  float vv[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) vv[e] = to_f32(Tag{}, v[e]);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float kk = to_f32(Tag{}, k[i * kRows + row]);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[i][e] = fmaf(kk, vv[e], decay * s[i][e]);
    *reinterpret_cast<floatx4*>(state + (i * kRows + row) * D) = s[i];
  }
  const int64_t heads0 = static_cast<int64_t>(b) * p.num_heads + n * p.group;
  const uint16_t* q = p.q + b * p.q_stride + n * p.group * D;
  for (int g0 = 0; g0 < p.group; g0 += kHeads) {
    const int heads = min(kHeads, p.group - g0);
    __syncthreads();
    for (int i = threadIdx.x; i < heads * D; i += kDecodeThreads) s_q[i / D][i % D] = to_f32(Tag{}, q[g0 * D + i]);
    __syncthreads();
    for (int g = 0; g < heads; ++g) {
      floatx4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float qq = s_q[g][i * kRows + row];
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = fmaf(qq, s[i][e], sum[e]);
      }
#pragma unroll
      for (int m = kLanes; m < 64; m <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += __shfl_xor(sum[e], m);
      if ((threadIdx.x & 63) < kLanes)
        *reinterpret_cast<floatx4*>(&s_part[g][threadIdx.x >> 6][lane * 4]) = sum;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < heads * kDecodeCols; i += kDecodeThreads) {
      const int g = i / kDecodeCols, c = i % kDecodeCols;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kDecodeThreads / 64; ++w) sum += s_part[g][w][c];
      p.out[(heads0 + g0 + g) * D + slice * kDecodeCols + c] = pack1(Tag{}, sum * p.scale);
    }
  }
}

// Prompts, token by token: a workgroup walks a sequence with 32 columns of the state in
// registers.
template <class Tag, int D>
__global__ __launch_bounds__(kDecodeThreads) void linear_prefill_recurrent(LinearParams p) {
  constexpr int kLanes = kDecodeCols / 4;
  constexpr int kRows = kDecodeThreads / kLanes;
  constexpr int N = D / kRows;
  __shared__ float s_part[kDecodeThreads / 64][kDecodeCols];
  const int slices = D / kDecodeCols;
  const int slice = blockIdx.x % slices;
  const int n = blockIdx.x / slices % p.num_kv_heads;
  const int b = blockIdx.x / slices / p.num_kv_heads;
  const int64_t slot = p.slots[b];
  if (slot < 0 || slot >= p.num_slots) return;
  const int64_t begin = p.cu_q[b];
  const int64_t end = min(min(static_cast<int64_t>(p.cu_q[b + 1]), p.total_q), begin + p.max_q);
  if (end <= begin) return;
  const int lane = threadIdx.x % kLanes, row = threadIdx.x / kLanes;
  const int col = slice * kDecodeCols + lane * 4;
  float* state = p.state + (slot * p.num_kv_heads + n) * D * D + col;
  const bool fresh = p.context_lens && p.context_lens[b] == 0;
  floatx4 s[N];
#pragma unroll
  for (int i = 0; i < N; ++i)
    s[i] = fresh ? floatx4{0.f, 0.f, 0.f, 0.f} : *reinterpret_cast<const floatx4*>(state + (i * kRows + row) * D);
  const Decay decay = decay_power(p.log_decay[n], 1);
  for (int64_t t = begin; t < end; ++t) {
    const uint16_t* k = p.k + t * p.k_stride + n * D;
    const uint16_t* v = p.v + t * p.v_stride + n * D + col;
    float vv[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) vv[e] = to_f32(Tag{}, v[e]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float kk = to_f32(Tag{}, k[i * kRows + row]);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] = fmaf(kk, vv[e], decay * s[i][e]);
    }
    for (int g = 0; g < p.group; ++g) {
      const uint16_t* q = p.q + t * p.q_stride + (n * p.group + g) * D;
      floatx4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float qq = to_f32(Tag{}, q[i * kRows + row]);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = fmaf(qq, s[i][e], sum[e]);
      }
#pragma unroll
      for (int m = kLanes; m < 64; m <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += __shfl_xor(sum[e], m);
      __syncthreads();
      if ((threadIdx.x & 63) < kLanes) *reinterpret_cast<floatx4*>(&s_part[threadIdx.x >> 6][lane * 4]) = sum;
      __syncthreads();
      if (threadIdx.x < kDecodeCols) {
        float o = 0.f;
#pragma unroll
        for (int w = 0; w < kDecodeThreads / 64; ++w) o += s_part[w][threadIdx.x];
        p.out[(t * p.num_heads + n * p.group + g) * D + slice * kDecodeCols + threadIdx.x] =
            pack1(Tag{}, o * p.scale);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) *reinterpret_cast<floatx4*>(state + (i * kRows + row) * D) = s[i];
}

// Argument checks of both entries; OXIDE_OK, or the error to record.
int check_linear(const LinearParams& p, int64_t rows, int64_t batch, int64_t num_heads, int64_t num_kv_heads,
                 int64_t head_dim, int dtype) {
  if (dtype != OXIDE_DTYPE_BF16 && dtype != OXIDE_DTYPE_F16) return OXIDE_ERR_UNSUPPORTED_DTYPE;
  if (head_dim != 64 && head_dim != 128) return OXIDE_ERR_UNSUPPORTED_SHAPE;
  if (batch < 0 || rows < 0 || batch > 65535 || rows > INT32_MAX || num_heads <= 0 || num_kv_heads <= 0 ||
      num_heads > 4096 || num_heads % num_kv_heads != 0 || p.num_slots < 0 || p.q_stride < num_heads * head_dim ||
      p.k_stride < num_kv_heads * head_dim || p.v_stride < num_kv_heads * head_dim || p.q_stride % 8 != 0 ||
      p.k_stride % 8 != 0 || p.v_stride % 8 != 0)
    return OXIDE_ERR_INVALID_ARGUMENT;
  if (batch == 0 || rows == 0) return OXIDE_OK;
  const void* ptrs[] = {p.out, p.q, p.k, p.v, p.state};
  for (const void* x : ptrs)
    if (!x || !oxide::aligned16(x)) return OXIDE_ERR_INVALID_ARGUMENT;
  if (!p.log_decay || !p.slots) return OXIDE_ERR_INVALID_ARGUMENT;
  const int64_t q_row = num_heads * head_dim, k_row = num_kv_heads * head_dim;
  if (oxide::overlap16(p.out, rows * q_row, p.q, (rows - 1) * p.q_stride + q_row) ||
      oxide::overlap16(p.out, rows * q_row, p.k, (rows - 1) * p.k_stride + k_row) ||
      oxide::overlap16(p.out, rows * q_row, p.v, (rows - 1) * p.v_stride + k_row))
    return OXIDE_ERR_INVALID_ARGUMENT;
  return OXIDE_OK;
}

// Calls f with the tag and the head dimension as types.
template <class F>
void dispatch(int dtype, int64_t head_dim, F f) {
  auto with_dim = [&](auto tag) {
    if (head_dim == 128)
      f(tag, std::integral_constant<int, 128>{});
    else
      f(tag, std::integral_constant<int, 64>{});
  };
  if (dtype == OXIDE_DTYPE_BF16)
    with_dim(Bf16Tag{});
  else
    with_dim(F16Tag{});
}

LinearParams linear_params(void* out, const void* q, const void* k, const void* v, int64_t q_row_stride,
                           int64_t k_row_stride, int64_t v_row_stride, const float* log_decay, float* state,
                           const int32_t* state_slots, int64_t num_slots, float scale) {
  LinearParams p{};
  p.out = static_cast<uint16_t*>(out);
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.q_stride = q_row_stride;
  p.k_stride = k_row_stride;
  p.v_stride = v_row_stride;
  p.log_decay = log_decay;
  p.state = state;
  p.slots = state_slots;
  p.num_slots = num_slots;
  p.scale = scale;
  return p;
}

void set_heads(LinearParams& p, int64_t batch, int64_t num_heads, int64_t num_kv_heads) {
  p.batch = static_cast<int>(batch);
  p.num_heads = static_cast<int>(num_heads);
  p.num_kv_heads = static_cast<int>(num_kv_heads);
  p.group = static_cast<int>(num_heads / num_kv_heads);
}

}  // namespace

extern "C" void linear_attention_decode(void* out, const void* q, const void* k, const void* v, int64_t q_row_stride,
                                        int64_t k_row_stride, int64_t v_row_stride, const float* log_decay,
                                        float* state, const int32_t* state_slots, int64_t num_slots, int64_t batch,
                                        int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, float scale,
                                        int dtype, void* stream) {
  LinearParams p = linear_params(out, q, k, v, q_row_stride, k_row_stride, v_row_stride, log_decay, state,
                                 state_slots, num_slots, scale);
  if (const int e = check_linear(p, batch, batch, num_heads, num_kv_heads, head_dim, dtype)) {
    oxide::set_error(e);
    return;
  }
  if (batch == 0) return;
  set_heads(p, batch, num_heads, num_kv_heads);
  dispatch(dtype, head_dim, [&](auto tag, auto d) {
    using Tag = decltype(tag);
    constexpr int D = decltype(d)::value;
    hipLaunchKernelGGL((linear_decode<Tag, D>), dim3(static_cast<unsigned>(batch * num_kv_heads * (D / kDecodeCols))),
                       dim3(kDecodeThreads), 0, oxide::as_stream(stream), p);
  });
  oxide::check_launch();
}

extern "C" size_t linear_attention_prefill_workspace_size(int64_t total_q, int64_t batch, int64_t num_heads,
                                                          int64_t num_kv_heads, int64_t head_dim,
                                                          int64_t max_seqlen_q) {
  return 0;
}

extern "C" void linear_attention_prefill(void* out, const void* q, const void* k, const void* v, int64_t q_row_stride,
                                         int64_t k_row_stride, int64_t v_row_stride, const float* log_decay,
                                         float* state, const int32_t* state_slots, const uint32_t* context_lens,
                                         const uint32_t* cu_seqlens_q, int64_t num_slots, int64_t total_q,
                                         int64_t batch, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                                         int64_t max_seqlen_q, float scale, void* workspace, size_t workspace_bytes,
                                         int dtype, void* stream) {
  LinearParams p = linear_params(out, q, k, v, q_row_stride, k_row_stride, v_row_stride, log_decay, state,
                                 state_slots, num_slots, scale);
  if (const int e = check_linear(p, total_q, batch, num_heads, num_kv_heads, head_dim, dtype)) {
    oxide::set_error(e);
    return;
  }
  if (max_seqlen_q < 0 || (batch > 0 && !cu_seqlens_q)) {
    oxide::set_error(OXIDE_ERR_INVALID_ARGUMENT);
    return;
  }
  if (batch == 0 || total_q == 0 || max_seqlen_q == 0) return;
  set_heads(p, batch, num_heads, num_kv_heads);
  p.context_lens = context_lens;
  p.cu_q = cu_seqlens_q;
  p.total_q = total_q;
  p.max_q = static_cast<int>(max_seqlen_q < total_q ? max_seqlen_q : total_q);
  dispatch(dtype, head_dim, [&](auto tag, auto d) {
    using Tag = decltype(tag);
    constexpr int D = decltype(d)::value;
    hipLaunchKernelGGL((linear_prefill_recurrent<Tag, D>),
                       dim3(static_cast<unsigned>(batch * num_kv_heads * (D / kDecodeCols))), dim3(kDecodeThreads), 0,
                       oxide::as_stream(stream), p);
  });
  oxide::check_launch();
}
