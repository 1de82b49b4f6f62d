// Linear attention with a decay for each head, for gfx950: per sequence and kv head n a
// state S [D, D] (key dimension first), fp32,
//   S_t = lambda_n S_{t-1} + k_t v_t^T,   lambda_n = exp(log_decay[n]),
//   out_t[h] = scale * q_t[h]^T S_t       for the query heads h of n.
// No reference counterpart: every layer of its models is softmax attention.
//
// linear_decode: one token.  Bound by HBM, the state read and written once (8 D^2 bytes
// a head against 4 D^2 + 2 G D^2 operations).  A workgroup holds COLS columns of one
// state in registers -- out's columns need S's columns only -- so nothing is joined
// between workgroups; the sum over the key dimension goes over the lanes that share a
// column, then over the waves through LDS.  Heads run fastest in the grid, so that with
// kv heads a multiple of the eight XCDs one of them gets all columns of a state: 64
// sequences on 32 heads at D = 128 (268 MB) 56 -> 52 us, and with the choices of
// launch_tokens 46.8 (5.78 TB/s, above the rate of a copy that writes as much as it
// reads, 5.4 at this size).  4 sequences on 16 heads (8.4 MB) take 4.3 us: a launch.
#include <math.h>

#include <algorithm>
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
  float* workspace;              // pieces' states (prefill)
  int64_t total_q;
  int64_t num_slots;
  int64_t units;  // states of each kv head in the workspace
  int batch, num_heads, num_kv_heads, group, max_q;
  int piece_tokens;
  int part_heads;  // query heads of a kv head that a workgroup takes, where they are dealt out
  bool joined;  // the workspace holds the states at the pieces' begins, not the pieces' sums
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

template <int I>
using Int = std::integral_constant<int, I>;

// Powers of lambda one after the other, each a single fp32 factor: what its rounding leaves
// out is put into the next one, so the product of any run of them is off by a few 2^-25.
struct DecaySteps {
  float off = 0.f;  // relative, of the factors so far
  __device__ __forceinline__ float next(Decay d) {
    const bool plain = d.hi > 0.f && !__builtin_isinf(d.hi);
    const float add = plain ? fmaf(d.hi, off, d.lo) : d.lo;
    const float f = d.hi + add;
    off = plain ? (add - (f - d.hi)) * __builtin_amdgcn_rcpf(d.hi) : 0.f;
    return f;
  }
};

constexpr int kDecodeThreads = 256;

// Values that are the same in every lane, in scalar registers.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ float uniform(float x) { return __int_as_float(uniform(__float_as_int(x))); }
__device__ __forceinline__ Decay uniform(Decay d) { return Decay{uniform(d.hi), uniform(d.lo)}; }

// A sequence's slot, rows (at most max_q, and none past the last there is) and whether it
// starts from zero, and a head's decay: asked for together, before any is looked at.
struct Sequence {
  int slot, begin, end;
  bool fresh;
  float log_decay;
};
__device__ __forceinline__ Sequence sequence_of(const LinearParams& p, int b, int n) {
  const int slot = p.slots[b];
  const uint32_t from = p.cu_q[b], to = p.cu_q[b + 1];
  const uint32_t context = *(p.context_lens ? p.context_lens + b : p.cu_q);
  const float log_decay = p.log_decay[n];
  const int64_t begin = min(static_cast<int64_t>(from), p.total_q);
  const int64_t end = min(min(static_cast<int64_t>(to), p.total_q), begin + p.max_q);
  return Sequence{uniform(slot), uniform(static_cast<int>(begin)), uniform(static_cast<int>(end)),
                  p.context_lens && uniform(static_cast<int>(context)) == 0, uniform(log_decay)};
}

// One token a sequence, or (MANY) a few, with the state's columns in registers: s[i] are 4
// columns of key row i * kRows + row.  ONCE: the states pass through the caches without a
// claim on them.
template <class Tag, int D, int COLS, bool ONCE, bool MANY>
__global__ __launch_bounds__(kDecodeThreads) void linear_decode(LinearParams p) {
  constexpr int kLanes = COLS / 4;                  // lanes of a row's columns
  constexpr int kRows = kDecodeThreads / kLanes;    // rows that the workgroup holds at once
  constexpr int N = D / kRows;
  constexpr int kHeads = 8;  // query heads joined at a time
  __shared__ float s_q[kHeads][D];
  __shared__ float s_part[kHeads][kDecodeThreads / 64][COLS];
  constexpr int kSlices = D / COLS;
  const int n = blockIdx.x % p.num_kv_heads;
  const int slice = blockIdx.x / p.num_kv_heads % kSlices;
  const int b = blockIdx.x / p.num_kv_heads / kSlices;
  Sequence seq{p.slots[b], b, b + 1, false, p.log_decay[n]};
  if constexpr (MANY) seq = sequence_of(p, b, n);
  if (seq.slot < 0 || seq.slot >= p.num_slots || seq.begin >= seq.end) return;
  const int lane = threadIdx.x % kLanes, row = threadIdx.x / kLanes;
  const int col = slice * COLS + lane * 4;
  float* state = p.state + (static_cast<int64_t>(seq.slot) * p.num_kv_heads + n) * D * D + col;
  floatx4 s[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const floatx4* at = reinterpret_cast<const floatx4*>(state + (i * kRows + row) * D);
    s[i] = floatx4{0.f, 0.f, 0.f, 0.f};
    if (!MANY || !seq.fresh) s[i] = ONCE ? __builtin_nontemporal_load(at) : *at;
  }
  auto store_state = [&] {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      floatx4* at = reinterpret_cast<floatx4*>(state + (i * kRows + row) * D);
      if constexpr (ONCE)
        __builtin_nontemporal_store(s[i], at);
      else
        *at = s[i];
    }
  };
  uint16_t k[N];
  uint2 v;
  auto read_token = [&](int t) {
#pragma unroll
    for (int i = 0; i < N; ++i) k[i] = p.k[t * p.k_stride + n * D + i * kRows + row];
    v = *reinterpret_cast<const uint2*>(p.v + t * p.v_stride + n * D + col);
  };
  read_token(seq.begin);
  const Decay decay = decay_power(seq.log_decay, 1);
  for (int t = seq.begin; t < seq.end; ++t) {
    const float vv[4] = {to_f32(Tag{}, static_cast<uint16_t>(v.x)), to_f32(Tag{}, static_cast<uint16_t>(v.x >> 16)),
                         to_f32(Tag{}, static_cast<uint16_t>(v.y)), to_f32(Tag{}, static_cast<uint16_t>(v.y >> 16))};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float kk = to_f32(Tag{}, k[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] = fmaf(kk, vv[e], decay * s[i][e]);
    }
    if (MANY && t + 1 < seq.end) read_token(t + 1);
    if (!MANY) store_state();
    const uint16_t* q = p.q + t * p.q_stride + n * p.group * D;
    uint16_t* out = p.out + (static_cast<int64_t>(t) * p.num_heads + n * p.group) * D + slice * COLS;
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
        // Over the lanes that hold the same columns: lanes 8 apart by a rotation of the row
        // of 16, rows of 16 by exchanging them.
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (kLanes == 8)
            sum[e] += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(sum[e]), 0x128, 0xf, 0xf, true));
          sum[e] = sum_over_lane_groups(sum[e]);
        }
        if ((threadIdx.x & 63) < kLanes)
          *reinterpret_cast<floatx4*>(&s_part[g][threadIdx.x >> 6][lane * 4]) = sum;
      }
      __syncthreads();
      for (int i = threadIdx.x; i < heads * COLS; i += kDecodeThreads) {
        const int g = i / COLS, c = i % COLS;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kDecodeThreads / 64; ++w) sum += s_part[g][w][c];
        out[static_cast<int64_t>(g0 + g) * D + c] = pack1(Tag{}, sum * p.scale);
      }
    }
  }
  if (MANY) store_state();
}

// Prompts, 64 tokens at a time on the matrix cores.  With S the state before a chunk,
// rows i, j of the chunk and n tokens in it:
//   P_ij = (q_i . k_j) lambda^(i - j) for j <= i, else 0
//   out_i = scale * (lambda^(i + 1) S^T q_i + sum_j P_ij v_j)
//   S <- lambda^n S + sum_j k_j (lambda^(n - 1 - j) v_j)^T
// A workgroup has a wave for each 32 value columns; a wave keeps its columns of S (all
// key rows) in matrix-core accumulators from chunk to chunk.  Scores are shared: each
// wave computes 16 query rows of P (two such strips at D = 64) and puts them into LDS.
// A last chunk of fewer than 64 tokens is padded with zero rows in FRONT, so weights and
// decays have their places in every chunk.
//
// Matrix-core layouts (cdna4_tile.hpp): the accumulator of K^T V has a value column in
// each lane and key rows in registers, which is the operand layout of S^T if the eight
// rows of a register run are those of an operand's k run: key columns are dealt to the
// rows of a tile with bits 2 and 3 exchanged (deal), which the transposing LDS reads do
// for nothing.  The same order for value columns hands a lane eight consecutive output
// columns.
//
// What is rounded to 16 bits, and why: P and S are operands of 16-bit matrix products,
// each rounded once (half a step of the type, as the output is); v times its weight
// would be too, but lands in the fp32 state, so it goes through the products as a sum of
// 16-bit values, three of bf16 or two of f16, with at least 22 bits.  f16 has the bits but not the
// range: P's rows, a wave's part of S and of v are scaled by powers of two to about 2^14.
//
// v is used for every earlier row of a chunk as 0 * v, which is NaN for an infinity or
// NaN: a chunk that holds one adds its products one by one instead.
//
// Few sequences on few heads leave most of the chip idle, so long ones are cut into pieces:
// a launch for the pieces' sums, one that joins many of them, one for the outputs.  That
// reads k and v twice (the second time largely from the last-level cache), and moves a
// state of 4 D^2 bytes three to five times a piece.
//
// What bounds it: the chunk's chain of phases (scores, barrier, outputs, sums, barrier) at
// the two waves that 256 registers leave a SIMD.  Of its cycles at D = 128 the matrix cores
// are busy for 28 % and the vector units for 31 %; with all rows read from the caches the
// kernels take about five sixths of the time.  1 x 8192 tokens on 32 heads (268 MB in and
// out, 55 us at the rate of a copy) 97.4 us, its kernels 35 + 13 + 53 one by one; 4 x 4096
// in f16 163 us; 100 tokens on 16 heads 9.7 us, 2 chunks.
constexpr int kChunk = 64;

template <int D>
struct Tiles {
  static constexpr int kWaves = D / 32;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kGranules = D / 8;       // 16-byte pieces of a row
  static constexpr int kLoads = kChunk * kGranules / kThreads;  // granules of a tile a thread moves
  static constexpr int kTileBytes = kChunk * kRowBytes;
  static constexpr int kStrips = 4 / kWaves;  // 16-row strips of P a wave computes
  static constexpr int kRegs = D * D / kThreads;  // state values of a lane
  // Granule g of a row lies at g ^ turn(row): 16 rows' granules of one column, and four
  // rows' of 32 columns, fall into different banks.  turn repeats every 16 rows, so an
  // address is a lane's own offset, exclusive-or the granule, plus 16-row steps.
  static __device__ __forceinline__ int turn(int row) {
    if constexpr (D == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
    return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  }
  static __device__ __forceinline__ int at(int row, int granule) {
    return row * kRowBytes + ((granule ^ turn(row)) << 4);
  }
  static constexpr int kStep = 16 * kRowBytes;
  // P's rows: 64 scores, 128 bytes.
  static __device__ __forceinline__ int score_at(int row, int granule) {
    return row * 128 + ((granule ^ ((row >> 1) & 7)) << 4);
  }
};

// Column of a 32-column tile whose values row (or lane) m holds.
__device__ __forceinline__ int deal(int m) { return (m & 0x13) | ((m & 4) << 1) | ((m & 8) >> 1); }

// Offset of a lane's transposing reads of rows 8 (lane / 32) + 4 x + 0..3, columns dealt to
// the lanes of a tile at column 0.
template <int D>
__device__ __forceinline__ int columns_at(int lane, int x) {
  const int in_group = lane & 15, q = in_group & 3;
  const int col = 16 * ((lane >> 4) & 1) + 8 * (q & 1) + 4 * (q >> 1);
  return Tiles<D>::at(8 * (lane >> 5) + 4 * x + (in_group >> 2), col >> 3) + (col & 4) * 2;
}
// Operand of tokens 16 kb + 8 (lane / 32) + 0..7, column 32 t + deal(lane % 32).
template <int D>
__device__ __forceinline__ uint4 columns_operand(const char* tile, int at0, int at1, int kb, int t) {
  const uint2 a = lds_read_tr16(tile + (at0 ^ (t << 6)) + kb * Tiles<D>::kStep);
  const uint2 b = lds_read_tr16(tile + (at1 ^ (t << 6)) + kb * Tiles<D>::kStep);
  return make_uint4(a.x, a.y, b.x, b.y);
}

// The compiler's scheduler moves nothing across: left alone it reads operands far ahead of
// their products, into more registers than there are.
__device__ __forceinline__ void fence_schedule() { __builtin_amdgcn_sched_barrier(0); }

// Asks for READS LDS reads first, then PRODUCTS matrix products with VALU others between
// each two: a product keeps the matrix cores busy for as long as eight of those take.
template <int READS, int PRODUCTS, int VALU>
__device__ __forceinline__ void interleave() {
  __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
  for (int i = 0; i < PRODUCTS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
  }
}

// Keeps a lane's offset one register: what is computed from it is not kept from chunk to
// chunk in registers of its own.
__device__ __forceinline__ int fresh_copy(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

__device__ __forceinline__ uint4 lds_read16(const char* p) { return *reinterpret_cast<const uint4*>(p); }

// acc + 0 * (each of eight packed bf16 values): NaN once one of them is an infinity or NaN.
__device__ __forceinline__ float add_zeros(uint4 v, float acc) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_in_t, w[e]), __builtin_bit_cast(bf16x2_in_t, 0u), acc,
                                          false);
  return acc;
}
// The larger of `most` and the magnitudes of eight packed f16 values, as bit patterns (which
// are ordered as the magnitudes are), low and high ones apart; 0x7c00 on: infinity, NaN.
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u16x2_t max_bits(uint4 v, u16x2_t most) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, w[e] & 0x7fff7fffu));
  return most;
}

template <class Tag>
__device__ __forceinline__ void unpack8(uint4 v, float* x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = to_f32(Tag{}, static_cast<uint16_t>(w[e]));
    x[2 * e + 1] = to_f32(Tag{}, static_cast<uint16_t>(w[e] >> 16));
  }
}
template <class Tag>
__device__ __forceinline__ uint4 pack8(const float* x) {
  return make_uint4(pack2_cvt(Tag{}, x[0], x[1]), pack2_cvt(Tag{}, x[2], x[3]), pack2_cvt(Tag{}, x[4], x[5]),
                    pack2_cvt(Tag{}, x[6], x[7]));
}

// 2^e with |x| 2^-e in [2^14, 2^15), e cut to +-40: beyond that 2^-65 of an f16 product's
// range is lost, or an f16 overflow is honest.
struct Pow2 {
  float up, down;  // 2^e, 2^-e
};
__device__ __forceinline__ Pow2 scale_for_f16(float x) {
  const int e = min(max(static_cast<int>((__float_as_uint(x) >> 23) & 255) - 127 - 14, -40), 40);
  return Pow2{__uint_as_float(static_cast<uint32_t>(127 + e) << 23), __uint_as_float(static_cast<uint32_t>(127 - e) << 23)};
}
// Largest of a wave's values, in every lane: over rows of 16 lanes by rotations within them
// (an LDS shuffle would be a round trip each), then over the four rows.
__device__ __forceinline__ float wave_max(float x) {
#define OXIDE_ROTATED_MAX(N) \
  x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + N, 0xf, 0xf, true)))
  OXIDE_ROTATED_MAX(1);
  OXIDE_ROTATED_MAX(2);
  OXIDE_ROTATED_MAX(4);
  OXIDE_ROTATED_MAX(8);
#undef OXIDE_ROTATED_MAX
  return max_over_lane_groups(x);
}

// The last sequence whose key is at most x, -1 if there is none: every wave by itself, 64
// sequences at a time.  key(b) grows with b and is computed from the row b starts at.
template <class Key>
__device__ __forceinline__ int last_sequence(const LinearParams& p, int x, Key key) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = p.batch;
  while (true) {
    const int step = (n + 63) / 64, at = lo + lane * step;
    bool ok = false;
    if (lane * step < n) ok = key(at, static_cast<int>(min(static_cast<int64_t>(p.cu_q[at]), p.total_q))) <= x;
    const int found = __popcll(__ballot(ok));
    if (found == 0) return -1;
    lo += (found - 1) * step;
    n = min(step, n - (found - 1) * step);
    if (step == 1) return uniform(lo);
  }
}

// The sequence and piece at a place of the grid.  Up to 64 sequences have their pieces one
// after the other, by a scan of their numbers, and the grid's spare places come last (places
// with nothing to do in between leave compute units idle: 39 -> 48 us for four prompts of
// 1024 on 16 heads).  More have them from floor(begin / piece_tokens) + b on: no two
// sequences' are the same and none is past total_q / piece_tokens + batch.
struct Place {
  int sequence, piece;
};
__device__ __forceinline__ Place place_of(const LinearParams& p, int at) {
  if (p.batch == 1) return Place{0, at};
  if (p.batch > 64) {
    const int b = last_sequence(p, at, [&](int i, int begin) { return begin / p.piece_tokens + i; });
    if (b < 0) return Place{-1, 0};
    const int begin = uniform(static_cast<int>(min(static_cast<int64_t>(p.cu_q[b]), p.total_q)));
    return Place{b, at - b - begin / p.piece_tokens};
  }
  const int lane = threadIdx.x & 63;
  const int64_t begin = min(static_cast<int64_t>(p.cu_q[min(lane, p.batch)]), p.total_q);
  const int64_t end = min(min(static_cast<int64_t>(p.cu_q[min(lane + 1, p.batch)]), p.total_q), begin + p.max_q);
  const int own = end > begin ? static_cast<int>((end - begin - 1) / p.piece_tokens) + 1 : 0;
  int before = own;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int add = __shfl_up(before, off);
    if (lane >= off) before += add;
  }
  before -= own;
  const int b = __popcll(__ballot(lane < p.batch && before <= at)) - 1;
  return Place{uniform(b), at - uniform(__shfl(before, max(b, 0)))};
}

// What a workgroup does with its piece of a sequence.
enum Mode {
  kWhole,  // a sequence from its slot's state to its end
  // A piece's own sum, from a zero state (the first: from the slot's, which it also copies),
  // into the workspace.
  kSums,
  // A piece's outputs, from its begin's state in the workspace.  Its own state is for them
  // alone: of bf16 it takes v as two values, 16 bits of it.
  kPieces,
  kLast,  // also the slot's new state, which no other piece reads in this launch
};

// OUTPUTS: a kernel that computes them.
template <int D, bool OUTPUTS>
struct alignas(16) ChunkTiles {
  char k[Tiles<D>::kTileBytes], v[Tiles<D>::kTileBytes];
  char q[OUTPUTS ? Tiles<D>::kTileBytes : 16], p[OUTPUTS ? kChunk * 128 : 16];
  float weight[kChunk];                            // lambda^(63 - j)
  float power[kChunk + 1], power_low[kChunk + 1];  // lambda^m, and what its rounding leaves
  float up[kChunk];                                // f16: 2^e of P's rows
  // Of even and odd chunks: bf16, whether v holds an infinity or NaN; f16, its largest
  // magnitude's bits (0x7c00 on: one of those).
  int most[2];
};

// Rows t0 .. t1 - 1 of a sequence and kv head n, its piece `piece`; outputs for `heads` query
// heads of n's, from g0 on (the first workgroup's write the state).
template <class Tag, int D, int MODE, class Lds>
__device__ __forceinline__ void walk_chunks(const LinearParams& p, const Sequence& seq, int n, int piece, int t0,
                                            int t1, int g0, int heads, Lds& lds) {
  using T = Tiles<D>;
  constexpr bool kF16 = std::is_same<Tag, F16Tag>::value;
  constexpr int kMt = D / 32;  // tiles of 32 key rows
  char *const s_k = lds.k, *const s_v = lds.v, *const s_q = lds.q, *const s_p = lds.p;
  float *const s_weight = lds.weight, *const s_power = lds.power, *const s_power_low = lds.power_low;
  float* const s_up = lds.up;
  int* const s_most = lds.most;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), half = lane >> 5;
  const float ld = seq.log_decay;
  // The workspace's states: sums of all pieces but the last, every sequence's from
  // floor(begin / piece_tokens) on; and `units` behind its first, a copy of the slot's state
  // that a cut sequence starts from.
  const int64_t first_unit = MODE == kWhole ? 0 : seq.begin / p.piece_tokens;
  const int64_t unit = first_unit + piece - (MODE == kPieces || MODE == kLast ? 1 : 0);
  if (MODE == kSums && unit >= p.units) return;
  float* const ws = p.workspace + (unit * p.num_kv_heads + n) * D * D + tid * 4;
  auto copy = [&] { return p.workspace + ((p.units + first_unit) * p.num_kv_heads + n) * D * D + tid * 4; };
  float* const state =
      p.state + (static_cast<int64_t>(seq.slot) * p.num_kv_heads + n) * D * D + 32 * wave + deal(lane & 31);
  const int chunks = (t1 - t0 + kChunk - 1) / kChunk;

  // A thread moves granule tid % kGranules of rows tid / kGranules + 16 i of a tile.
  const int tile_row = tid / T::kGranules, tile_at = T::at(tile_row, tid % T::kGranules);
  // Computed where it is needed: kept in registers, the four tensors' would spill others.
  auto lane_bytes = [&](int64_t stride) {
    const uint32_t t = fresh_copy(tid);
    return t / T::kGranules * static_cast<uint32_t>(stride * 2) + t % T::kGranules * 16;
  };
  // Rows from `first` (of the chunk) on hold tokens; in place of those before, row `first`
  // is read, and zeros are stored for k and v.
  struct Granules {
    oxide::u32x4 r[T::kLoads];
  };
  // Without a branch, of which the addresses would be 64-bit registers of their own.
  auto load_tile = [&](const uint16_t* base, int64_t stride, int64_t row0, int first, auto once) {
    const char* rows = reinterpret_cast<const char*>(base) + row0 * stride * 2;
    const uint32_t step = static_cast<uint32_t>(stride) * 32, at = lane_bytes(stride);
    const uint32_t least = fresh_copy(tid) % T::kGranules * 16 + first * static_cast<uint32_t>(stride * 2);
    Granules x;
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) {
      const oxide::u32x4* from = reinterpret_cast<const oxide::u32x4*>(rows + max(at + i * step, least));
      if constexpr (decltype(once)::value)
        x.r[i] = __builtin_nontemporal_load(from);
      else
        x.r[i] = *from;
    }
    return x;
  };
  auto store_tile = [&](char* tile, const Granules& x) {
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) *reinterpret_cast<oxide::u32x4*>(tile + tile_at + i * T::kStep) = x.r[i];
  };
  // Loaded rows are first looked at here: otherwise what the next chunk does with them is
  // begun where they are asked for, with a wait for memory.
  auto arrived = [&](Granules x) {
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) {
      asm volatile("" : "+v"(x.r[i]));
    }
    return x;
  };
  auto without_padding = [&](Granules x, int first) {
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i)
      if (16 * i + tile_row < first) x.r[i] = oxide::u32x4{0, 0, 0, 0};
    return x;
  };

  // q and out pass through the caches without a claim on them: keys and values are there
  // when the second launch reads them again.
  constexpr std::true_type kOnce{};
  constexpr std::false_type kKeep{};
  const int64_t h0 = static_cast<int64_t>(n) * p.group + g0;
  const uint16_t* const qn = p.q + h0 * D;
  const uint16_t* const kn = p.k + static_cast<int64_t>(n) * D;
  const uint16_t* const vn = p.v + static_cast<int64_t>(n) * D;
  // Chunk c is rows row0(c) + 0..63 of which the first first(c) are padding.
  auto first_of = [&](int c) { return c + 1 < chunks ? 0 : chunks * kChunk - (t1 - t0); };
  auto row0_of = [&](int c) { return static_cast<int64_t>(t0) + c * kChunk - first_of(c); };

  // In the order in which they are asked for later.
  Granules rq{};
  if constexpr (MODE != kSums) rq = load_tile(qn, p.q_stride, row0_of(0), first_of(0), kOnce);
  Granules rk = load_tile(kn, p.k_stride, row0_of(0), first_of(0), kKeep);
  Granules rv = load_tile(vn, p.v_stride, row0_of(0), first_of(0), kKeep);

  for (int m = tid; m <= kChunk; m += T::kThreads) {
    const Decay x = decay_power(ld, m);
    s_power[m] = x.hi;
    s_power_low[m] = x.lo;
    if (m < kChunk) s_weight[kChunk - 1 - m] = x.hi;
  }
  if (tid < 2) s_most[tid] = 0;

  // Lane's state values: register 8 a + i of tile mt is key row 32 mt + 16 a + 8 half + i.
  floatx16 S[kMt];
#pragma unroll
  for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
    for (int r = 0; r < 16; ++r) S[mt][r] = 0.f;
  // The workspace keeps a state as its threads hold it: four registers of all threads, the
  // next four.
  auto read_dump = [&](const float* from, auto of) {
#pragma unroll
    for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const floatx4 x = *reinterpret_cast<const floatx4*>(from + (mt * 4 + r / 4) * T::kThreads * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) S[mt][r + e] = of(S[mt][r + e], x[e]);
      }
  };
  auto write_dump = [&](float* to) {
#pragma unroll
    for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<floatx4*>(to + (mt * 4 + r / 4) * T::kThreads * 4) =
            floatx4{S[mt][r], S[mt][r + 1], S[mt][r + 2], S[mt][r + 3]};
  };
  if (piece == 0 && !seq.fresh) {
    if (MODE == kPieces) {
      read_dump(copy(), [](float, float x) { return x; });
    } else {
#pragma unroll
      for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[mt][r] = state[(32 * mt + 16 * (r / 8) + 8 * half + r % 8) * D];
      if (MODE == kSums) write_dump(copy());
    }
  }
  if ((MODE == kPieces || MODE == kLast) && piece > 0 && unit < p.units) {
    // The state at the piece's begin, or the earlier pieces' sums one after the other.
    const Decay over_piece = decay_power(ld, p.piece_tokens);
    const bool joined = p.joined;
    for (int back = joined ? 0 : piece - 1; back >= 0; --back)
      read_dump(ws - static_cast<int64_t>(back) * p.num_kv_heads * D * D,
                [&](float now, float x) { return joined ? x : over_piece * now + x; });
  }

  // Decays of the wave's scores (bf16: with the outputs' scale): query 16 strip + lane % 16,
  // keys 16 kt + 4 (lane / 16) + r.  Strips have one to four tiles of keys: of two workgroups
  // on a compute unit (neighbours in the grid 8 or 256 apart) one deals them out in reverse,
  // so that its SIMDs get even work.
  const int strip0 = T::kStrips == 1 && ((blockIdx.x >> 3 ^ blockIdx.x >> 8) & 1) ? 3 - wave : wave;
  float fade[T::kStrips][4][4];
  __syncthreads();
  if constexpr (MODE != kSums) {
#pragma unroll
    for (int x = 0; x < T::kStrips; ++x) {
      const int strip = x == 0 ? strip0 : 3 - strip0;
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          fade[x][kt][r] = s_power[max(16 * strip + (lane & 15) - (16 * kt + 4 * (lane >> 4) + r), 0)] *
                           (kF16 ? 1.f : p.scale);
    }
  }

  // Offsets of the lane's operands in the tiles.
  const int rows16 = T::at(lane & 15, lane >> 4), rows32 = T::at(lane & 31, half);
  const int cols0 = columns_at<D>(lane, 0), cols1 = columns_at<D>(lane, 1);
  const int scores16 = T::score_at(lane & 15, half) + ((lane >> 4) & 1) * 8, scores32 = T::score_at(lane & 31, half);

  const int in_last = t1 - t0 - (chunks - 1) * kChunk;
  const Decay over_chunk = uniform(Decay{s_power[kChunk], s_power_low[kChunk]});
  const Decay over_last = uniform(Decay{s_power[in_last], s_power_low[in_last]});
  const float carries[2] = {s_power[(lane & 31) + 1], s_power[(lane & 31) + 33]};  // without padding
  DecaySteps steps;
  float s_unit = 1.f;

  // The rows that are in registers, of which the first `first` are padding, into the tiles.
  auto put_rows = [&](int c, int first) {
    rk = arrived(rk);
    rv = arrived(rv);
    if (first > 0) {
      rk = without_padding(rk, first);
      rv = without_padding(rv, first);
    }
    store_tile(s_k, rk);
    store_tile(s_v, rv);
    if constexpr (kF16) {
      u16x2_t most = {0, 0};
#pragma unroll
      for (int i = 0; i < T::kLoads; ++i) most = max_bits(__builtin_bit_cast(uint4, rv.r[i]), most);
      // As fp32 whole numbers they keep their order.
      const int top = static_cast<int>(wave_max(static_cast<float>(max(most.x, most.y))));
      if (lane == 0) atomicMax(&s_most[c & 1], top);
    } else if constexpr (MODE != kSums) {
      float zero = 0.f;
#pragma unroll
      for (int i = 0; i < T::kLoads; ++i) zero = add_zeros(__builtin_bit_cast(uint4, rv.r[i]), zero);
      if (zero != zero) s_most[c & 1] = 1;
    }
  };
  put_rows(0, first_of(0));
  if constexpr (MODE != kSums) store_tile(s_q, arrived(rq));

  // All chunks but the last ask for the next one's rows and have no padding.  Rows go into
  // their tiles in the chunk that asked for them: where a wait for loads may meet paths with
  // and without them, or with and without later stores, it waits for all of these as well.
  auto chunk = [&](int c, auto more_constant) __attribute__((always_inline)) {
    constexpr bool more = decltype(more_constant)::value;
    const int first = more ? 0 : first_of(c);
    const int64_t row0 = row0_of(c);
    __syncthreads();
    const int most = uniform(s_most[c & 1]);
    if (tid == 0) s_most[(c + 1) & 1] = 0;  // last read before the barrier that ended chunk c - 1
    // A thread moves the granules of the output tile in whose place it puts the next queries.
    auto read_out = [&] {
      Granules x;
#pragma unroll
      for (int i = 0; i < T::kLoads; ++i)
        x.r[i] = *reinterpret_cast<const oxide::u32x4*>(s_q + tile_at + i * T::kStep);
      return x;
    };
    auto store_out = [&](int g, const Granules& x) {
      char* const out = reinterpret_cast<char*>(p.out + (row0 * p.num_heads + h0 + g) * D);
      const int64_t stride = static_cast<int64_t>(p.num_heads) * D;
      const uint32_t at = lane_bytes(stride), step = static_cast<uint32_t>(stride) * 32;
#pragma unroll
      for (int i = 0; i < T::kLoads; ++i)
        if (more || 16 * i + tile_row >= first)
          __builtin_nontemporal_store(x.r[i], reinterpret_cast<oxide::u32x4*>(out + (at + i * step)));
    };
    // The next chunk's rows are asked for a tile at a time, between the phases of this one: all
    // at once they fill the memory pipe and every wave waits to get its loads into it.
    const int next_first = first_of(c + 1);
    const int64_t next_row0 = row0_of(c + 1);
    // The state's decay over the chunk.  f16: what is added to it comes scaled by v's power
    // of two, so the registers hold the state over `s_unit`.
    constexpr bool update = more || MODE != kPieces;
    Pow2 v_scale{1.f, 1.f};
    // An infinity or NaN has no part in the power: other columns keep their values.  A head
    // whose states grow weighs v by up to lambda^n.
    if constexpr (kF16)
      v_scale = scale_for_f16(to_f32(Tag{}, static_cast<uint16_t>(min(most, 0x7bff))) *
                              fmaxf((more ? over_chunk : over_last).hi, 1.f));
    float fall = 1.f;
    if constexpr (update) fall = steps.next(more ? over_chunk : over_last) * (kF16 ? s_unit * v_scale.down : 1.f);
    if constexpr (MODE != kSums) {
      Pow2 s_scale{1.f, 1.f};
      if constexpr (kF16) {
        float m = 0.f;
#pragma unroll
        for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
          for (int r = 0; r < 16; ++r) m = fmaxf(m, fabsf(S[mt][r]));
        m = wave_max(m);
        if (!(m < INFINITY)) {  // nor here
          m = 0.f;
#pragma unroll
          for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
            for (int r = 0; r < 16; ++r) m = fabsf(S[mt][r]) < INFINITY ? fmaxf(m, fabsf(S[mt][r])) : m;
          m = wave_max(m);
        }
        s_scale = scale_for_f16(m);  // of the registers' values
      }

      auto head = [&](int g, auto same_constant) __attribute__((always_inline)) {
        constexpr bool same = decltype(same_constant)::value;  // the next tile of queries is this chunk's
        const float fall_now = same ? 1.f : fall;

        // Scores: K Q^T tiles, a query in each lane and four keys in its registers.
        const int r16 = fresh_copy(rows16), p16 = fresh_copy(scores16);
        auto score_strip = [&](auto strip_constant, const float (&fade_x)[4][4]) {
          constexpr int strip = decltype(strip_constant)::value;
          uint4 qb[D / 32], kb[strip + 1][D / 32];
          floatx4 score[4] = {};
#pragma unroll
          for (int kk = 0; kk < D / 32; ++kk) {
            qb[kk] = lds_read16(s_q + (r16 ^ (kk << 6)) + strip * T::kStep);
#pragma unroll
            for (int kt = 0; kt <= strip; ++kt) kb[kt][kk] = lds_read16(s_k + (r16 ^ (kk << 6)) + kt * T::kStep);
          }
#pragma unroll
          for (int kk = 0; kk < D / 32; ++kk)
#pragma unroll
            for (int kt = 0; kt <= strip; ++kt) score[kt] = mfma16x16x32(Tag{}, kb[kt][kk], qb[kk], score[kt]);
#pragma unroll
          for (int kt = 0; kt <= strip; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const bool seen = kt < strip || 4 * (lane >> 4) + r <= (lane & 15);
              score[kt][r] = seen ? score[kt][r] * fade_x[kt][r] : 0.f;
            }
          Pow2 p_scale{1.f, 1.f};
          if constexpr (kF16) {
            float m = 0.f;
#pragma unroll
            for (int kt = 0; kt <= strip; ++kt)
#pragma unroll
              for (int r = 0; r < 4; ++r) m = fmaxf(m, fabsf(score[kt][r]));
            p_scale = scale_for_f16(max_over_lane_groups(m));
            if (lane < 16) s_up[16 * strip + lane] = p_scale.up;
          }
          // Tiles of keys behind the strip are read only where they share a block of 32.
#pragma unroll
          for (int kt = 0; kt <= (strip | 1); ++kt) {
            float y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = kF16 ? score[kt][r] * p_scale.down : score[kt][r];
            *reinterpret_cast<uint2*>(s_p + (p16 ^ (kt << 5)) + strip * 16 * 128) =
                make_uint2(pack2_cvt(Tag{}, y[0], y[1]), pack2_cvt(Tag{}, y[2], y[3]));
          }
          fence_schedule();
        };
        if constexpr (T::kStrips == 1) {
          switch (strip0) {
            case 0: score_strip(Int<0>{}, fade[0]); break;
            case 1: score_strip(Int<1>{}, fade[0]); break;
            case 2: score_strip(Int<2>{}, fade[0]); break;
            default: score_strip(Int<3>{}, fade[0]);
          }
        } else if (strip0 == 0) {
          score_strip(Int<0>{}, fade[0]);
          score_strip(Int<3>{}, fade[T::kStrips - 1]);
        } else {
          score_strip(Int<1>{}, fade[0]);
          score_strip(Int<2>{}, fade[T::kStrips - 1]);
        }

        if (same || more)
          rq = load_tile(same ? qn + (g + 1) * D : qn, p.q_stride, same ? row0 : next_row0,
                         same ? first : next_first, kOnce);

        // Outputs, transposed: a query (of both halves of the chunk) in each lane, value
        // columns in its registers.  First what the state gives, while other waves' scores
        // are still to come; the next key rows' operands are read ahead.
        fence_schedule();
        const int r32 = fresh_copy(rows32), p32 = fresh_copy(scores32);
        floatx16 acc[2];
#pragma unroll
        for (int it = 0; it < 2; ++it)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[it][r] = 0.f;
        uint4 qa[2][2];
        auto read_queries = [&](int mt) {
#pragma unroll
          for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int it = 0; it < 2; ++it)
              qa[a][it] = lds_read16(s_q + (r32 ^ ((4 * mt + 2 * a) << 4)) + it * 2 * T::kStep);
        };
        uint4 s16[2];
        auto pack_state = [&](int mt) {
          // Not kept packed from head to head, in 32 more registers.
          asm volatile("" : "+v"(S[mt]));
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = kF16 ? S[mt][8 * a + i] * s_scale.down : S[mt][8 * a + i];
            s16[a] = pack8<Tag>(x);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) S[mt][r] *= fall_now;
        };
        read_queries(0);
        pack_state(0);
#pragma unroll
        for (int mt = 0; mt < kMt; ++mt) {
          uint4 now[2][2], part[2];
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            part[a] = s16[a];
#pragma unroll
            for (int it = 0; it < 2; ++it) now[a][it] = qa[a][it];
          }
          if (mt + 1 < kMt) {
            read_queries(mt + 1);
            pack_state(mt + 1);
          }
#pragma unroll
          for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int it = 0; it < 2; ++it) acc[it] = mfma32x32x16(Tag{}, part[a], now[a][it], acc[it]);
          interleave<4, 4, 7>();
          fence_schedule();
        }
        if (!same && more) rk = load_tile(kn, p.k_stride, next_row0, next_first, kKeep);
        const int v0 = fresh_copy(cols0), v1 = fresh_copy(cols1);
        uint4 v[4], ps[2][4];
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) v[kb] = columns_operand<D>(s_v, v0, v1, kb, wave);
        __syncthreads();

#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
          for (int it = kb / 2; it < 2; ++it) ps[it][kb] = lds_read16(s_p + (p32 ^ (kb << 5)) + it * 32 * 128);
        }
        Pow2 p_scale[2] = {{1.f, 1.f}, {1.f, 1.f}};
#pragma unroll
        for (int it = 0; it < 2; ++it) {
          const int query = 32 * it + (lane & 31);
          float carry = more ? carries[it] : s_power[max(query + 1 - first, 0)];
          if constexpr (kF16) {
            p_scale[it].up = s_up[query];
            p_scale[it].down = __uint_as_float(0x7f000000u - __float_as_uint(p_scale[it].up));  // 1 / 2^e
            carry *= s_scale.up * s_unit * p_scale[it].down;
            p_scale[it].up *= p.scale;
          } else {
            carry *= p.scale;
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[it][r] *= carry;
        }
        if (most >= (kF16 ? 0x7c00 : 1)) {  // one by one, and nothing left for the products
#pragma unroll
          for (int it = 0; it < 2; ++it) {
            const int query = 32 * it + (lane & 31);
            for (int j = 0; j < 32 * it + 32; ++j) {
              const float pj = to_f32(
                  Tag{}, *reinterpret_cast<const uint16_t*>(s_p + T::score_at(query, j >> 3) + (j & 7) * 2));
#pragma unroll
              for (int a = 0; a < 2; ++a) {
                float x[8];
                unpack8<Tag>(lds_read16(s_v + T::at(j, 4 * wave + 2 * a + half)), x);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  if (j <= query) acc[it][8 * a + i] = fmaf(pj, x[i], acc[it][8 * a + i]);
              }
            }
          }
#pragma unroll
          for (int kb = 0; kb < 4; ++kb) v[kb] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
#pragma unroll
          for (int it = kb / 2; it < 2; ++it) acc[it] = mfma32x32x16(Tag{}, v[kb], ps[it][kb], acc[it]);
        // Into the place of the queries, which every wave is done with: rows then leave whole,
        // 256 bytes at a time, instead of 16 bytes of 64 rows by each wave.
#pragma unroll
        for (int it = 0; it < 2; ++it)
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = kF16 ? acc[it][8 * a + i] * p_scale[it].up : acc[it][8 * a + i];
            *reinterpret_cast<uint4*>(s_q + (r32 ^ ((4 * wave + 2 * a) << 4)) + it * 2 * T::kStep) = pack8<Tag>(x);
          }
        if (same) {
          __syncthreads();
          store_out(g, read_out());
          store_tile(s_q, arrived(rq));
          __syncthreads();
        }
      };
      for (int g = 0; g + 1 < heads; ++g) head(g, std::true_type{});
      head(heads - 1, std::false_type{});
    }

    fence_schedule();
    if (more) {
      if constexpr (MODE == kSums) rk = load_tile(kn, p.k_stride, next_row0, next_first, kKeep);
      rv = load_tile(vn, p.v_stride, next_row0, next_first, kKeep);
    }
    if constexpr (update) {
      const int k0 = fresh_copy(cols0), k1 = fresh_copy(cols1);
      if constexpr (MODE == kSums) {
#pragma unroll
        for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
          for (int r = 0; r < 16; ++r) S[mt][r] *= fall;
      }
      // The products of 16 tokens, while the next 16's operands are read and weighted.
      constexpr int kTerms = kF16 || MODE == kPieces ? 2 : 3;
      uint4 term[kTerms], k[kMt];
      auto weigh = [&](uint4 v, int kb) {
        float x[8], y[8];
        unpack8<Tag>(v, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] *= s_weight[16 * kb + 8 * half + i];
          if constexpr (kF16) x[i] *= v_scale.down;
        }
#pragma unroll
        for (int t = 0; t < kTerms; ++t) {
          term[t] = pack8<Tag>(x);
          unpack8<Tag>(term[t], y);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] -= y[i];
        }
      };
      uint4 v = columns_operand<D>(s_v, k0, k1, 0, wave);
#pragma unroll
      for (int mt = 0; mt < kMt; ++mt) k[mt] = columns_operand<D>(s_k, k0, k1, 0, mt);
      weigh(v, 0);
      v = columns_operand<D>(s_v, k0, k1, 1, wave);
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
        uint4 now[kMt], part[kTerms];
#pragma unroll
        for (int mt = 0; mt < kMt; ++mt) now[mt] = k[mt];
#pragma unroll
        for (int t = 0; t < kTerms; ++t) part[t] = term[t];
        const uint4 v_next = v;
        if (kb < 2) v = columns_operand<D>(s_v, k0, k1, kb + 2, wave);
        if (kb < 3) {
#pragma unroll
          for (int mt = 0; mt < kMt; ++mt) k[mt] = columns_operand<D>(s_k, k0, k1, kb + 1, mt);
        }
#pragma unroll
        for (int t = 0; t < kTerms; ++t)
#pragma unroll
          for (int mt = 0; mt < kMt; ++mt) S[mt] = mfma32x32x16(Tag{}, now[mt], part[t], S[mt]);
        if (kb < 3) weigh(v_next, kb + 1);
        interleave<2 * kMt + 2, kTerms * kMt, 6>();
        fence_schedule();
      }
      if constexpr (kF16) s_unit = v_scale.up;
    }
    __syncthreads();
    Granules x{};
    if constexpr (MODE != kSums) x = read_out();
    if constexpr (more) put_rows(c + 1, next_first);
    if constexpr (MODE != kSums) {
      store_out(heads - 1, x);
      if constexpr (more) store_tile(s_q, arrived(rq));
    }
  };
  for (int c = 0; c + 1 < chunks; ++c) chunk(c, std::true_type{});
  chunk(chunks - 1, std::false_type{});
  if (MODE == kPieces) return;

  if constexpr (kF16) {
#pragma unroll
    for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r) S[mt][r] *= s_unit;
  }
  if (MODE == kSums) {
    write_dump(ws);
  } else if (g0 == 0) {
#pragma unroll
    for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r) state[(32 * mt + 16 * (r / 8) + 8 * half + r % 8) * D] = S[mt][r];
  }
}

template <class Tag, int D, int MODE>
__global__ __launch_bounds__(Tiles<D>::kThreads, 2) void linear_prefill_chunks(LinearParams p) {
  __shared__ ChunkTiles<D, MODE != kSums> lds;
  const int n = blockIdx.x % p.num_kv_heads;
  int piece = 0, b = blockIdx.x / p.num_kv_heads;
  if constexpr (MODE != kWhole) {
    const Place at = place_of(p, b);
    b = at.sequence;
    piece = at.piece;
    if (b < 0) return;
  }
  const Sequence seq = sequence_of(p, b, n);
  const int begin = seq.begin, end = seq.end;
  if (seq.slot < 0 || seq.slot >= p.num_slots) return;
  if (piece < 0 || begin >= end || piece > (end - begin - 1) / max(p.piece_tokens, 1)) return;
  if constexpr (MODE == kWhole) {
    walk_chunks<Tag, D, kWhole>(p, seq, n, 0, begin, end, 0, p.group, lds);
  } else {
    const int t0 = begin + piece * p.piece_tokens, t1 = t0 + min(end - t0, p.piece_tokens);
    int g0 = 0, heads = p.group;
    if constexpr (MODE == kPieces) {
      // A sequence that is not cut starts from its slot, which the workgroup that writes it
      // has to have for itself.
      if (piece > 0 || t1 < end) {
        g0 = static_cast<int>(blockIdx.y) * p.part_heads;
        heads = min(p.part_heads, p.group - g0);
      }
      if (heads <= 0 || (blockIdx.y > 0 && g0 == 0)) return;
    }
    if (t1 < end)
      walk_chunks<Tag, D, MODE>(p, seq, n, piece, t0, t1, g0, heads, lds);
    else if constexpr (MODE == kPieces)
      walk_chunks<Tag, D, kLast>(p, seq, n, piece, t0, t1, g0, heads, lds);
  }
}

// The pieces' sums become the states at the next pieces' begins, in place:
//   start(1) = sum(0), start(i + 1) = lambda^piece_tokens start(i) + sum(i).
// A thread carries four values of a state through its sequence's pieces.
template <int D>
__global__ __launch_bounds__(256) void linear_prefill_join(LinearParams p) {
  constexpr int kQuads = D * D / 4;
  const int blocks = kQuads / 256;
  // Heads run fastest in all three grids: with kv heads a multiple of the eight XCDs, a
  // head's pieces, and with them what the workspace holds of it, stay on one.
  const int n = blockIdx.x % p.num_kv_heads;
  const int quad = blockIdx.x / p.num_kv_heads % blocks * 256 + threadIdx.x;
  // The cut sequence, if there is one, whose first sum is this unit: the last that starts in
  // its piece_tokens rows.
  const int unit = blockIdx.x / p.num_kv_heads / blocks;
  const int b = last_sequence(p, unit, [&](int, int begin) { return begin / p.piece_tokens; });
  if (b < 0) return;
  const Sequence seq = sequence_of(p, b, n);
  const int slot = seq.slot, begin = seq.begin;
  if (slot < 0 || slot >= p.num_slots || begin / p.piece_tokens != unit) return;
  const int sums = seq.end > begin ? (seq.end - begin - 1) / p.piece_tokens : 0;  // all pieces but the last
  if (sums == 0) return;
  floatx4 s = {0.f, 0.f, 0.f, 0.f};
  const Decay fall = decay_power(seq.log_decay, p.piece_tokens);
  const int64_t first = begin / p.piece_tokens;
  const int count = static_cast<int>(min(static_cast<int64_t>(sums), p.units - first));
  const int64_t step = static_cast<int64_t>(p.num_kv_heads) * D * D;
  float* const ws = p.workspace + (first * p.num_kv_heads + n) * D * D + quad * 4;
  constexpr int kAhead = 4;  // sums asked for before the first is needed
  floatx4 next[kAhead];
#pragma unroll
  for (int a = 0; a < kAhead; ++a) next[a] = *reinterpret_cast<const floatx4*>(ws + min(a, count - 1) * step);
  for (int i0 = 0; i0 < count; i0 += kAhead) {
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const floatx4 add = next[a];
      next[a] = *reinterpret_cast<const floatx4*>(ws + min(i0 + a + kAhead, count - 1) * step);
      if (i0 + a < count) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = fall * s[e] + add[e];
        *reinterpret_cast<floatx4*>(ws + (i0 + a) * step) = s;
      }
    }
  }
}

// Tokens of a piece, 0 where sequences are walked whole.
struct Plan {
  int64_t piece_tokens, units;
};
Plan plan_prefill(int64_t total_q, int64_t batch, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                  int64_t max_seqlen_q) {
  const Plan whole{0, 0};
  if (total_q <= 0 || batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      (head_dim != 64 && head_dim != 128) || max_seqlen_q <= 0)
    return whole;
  // As many pieces as workgroups are resident (LDS and registers hold two on a compute unit
  // at D = 128, four at 64), but none whose rows are fewer bytes than its state costs
  // (written, joined, read: 16 D^2, against 4 D (1 + group) a token), unless compute units
  // are left without one: 512 tokens on 16 heads 28 us whole, 18.7 in pieces of 64, 1000 on
  // 32/8 in f16 35.2 -> 25.2, 2048 on 8 31.9 -> 25.2 (2048 on 32, a piece for each at 256:
  // 39.9, at 128 47).  Nor more than 32 for that of a sequence, whose join is a chain: 8192
  // on 2 heads 36.8 us in 32 pieces, 45.7 in 128.
  const int64_t cus = oxide::device_cu_count(), resident = (head_dim == 128 ? 2 : 4) * cus;
  const int64_t group = num_heads / num_kv_heads, rows = total_q * num_kv_heads;
  int64_t piece = std::max((rows + cus - 1) / cus, (std::min(max_seqlen_q, total_q) + 31) / 32);
  piece = std::max(std::min(piece, 4 * head_dim / (1 + group)), (rows + resident - 1) / resident);
  piece = (piece + kChunk - 1) / kChunk * kChunk;
  if (max_seqlen_q <= 2 * piece) return whole;
  return Plan{piece, total_q / piece};
}

constexpr int64_t kMaxStride = 1 << 25;  // elements: a chunk's rows' offsets in bytes fit 32 bits

// Argument checks of both entries; OXIDE_OK, or the error to record.
int check_linear(const LinearParams& p, int64_t rows, int64_t batch, int64_t num_heads, int64_t num_kv_heads,
                 int64_t head_dim, int dtype) {
  if (dtype != OXIDE_DTYPE_BF16 && dtype != OXIDE_DTYPE_F16) return OXIDE_ERR_UNSUPPORTED_DTYPE;
  if (head_dim != 64 && head_dim != 128) return OXIDE_ERR_UNSUPPORTED_SHAPE;
  if (batch < 0 || rows < 0 || batch > 65535 || rows > INT32_MAX || num_heads <= 0 || num_kv_heads <= 0 ||
      num_heads > 4096 || num_heads % num_kv_heads != 0 || p.num_slots < 0 || p.q_stride < num_heads * head_dim ||
      p.k_stride < num_kv_heads * head_dim || p.v_stride < num_kv_heads * head_dim || p.q_stride % 8 != 0 ||
      p.k_stride % 8 != 0 || p.v_stride % 8 != 0 || p.q_stride > kMaxStride || p.k_stride > kMaxStride ||
      p.v_stride > kMaxStride)
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

// Prompts of so few tokens are walked one by one, as single tokens are: against a chunk
// padded to 64, 4 tokens of one sequence on 16 heads 6.2 for 7.0 us, of 24 on 32/8 heads
// 11.6 for 12.5, of 64 on 32 heads 40 for 38; 8 tokens 8.9 for 6.7, 20 for 13 and 65 for 37.
constexpr int kFewTokens = 4;

// One token a sequence, or a few.
template <bool MANY>
void launch_tokens(const LinearParams& p, int64_t head_dim, int dtype, hipStream_t s) {
  const int64_t states = int64_t{p.batch} * p.num_kv_heads;
  // 64 columns a workgroup where it saves more than latency: whole rows at D = 64 (200
  // sequences on 32 heads 42.6 -> 40.0 us), half as many walks over a group's queries (64
  // sequences on 32/8 heads of 128 16.5 -> 14.7); else 32, four times as many workgroups for
  // a small batch as states (4 sequences on 16 heads 4.05 against 4.54).
  const bool wide = (head_dim == 64 || p.group > 1) && states >= oxide::device_cu_count();
  // States past half the 256 MB last-level cache are not there any more when they are next
  // needed: non-temporal (64 sequences on 32 heads, 134 MB of states, 51.7 -> 48.7 us; with 16
  // sequences, 34 MB, 12.7 -> 14.7).
  const bool once = states * head_dim * head_dim * 4 >= (int64_t{128} << 20);
  dispatch(dtype, head_dim, [&](auto tag, auto d) {
    using Tag = decltype(tag);
    constexpr int D = decltype(d)::value;
    auto launch = [&](auto kernel, int cols) {
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(states * (D / cols))), dim3(kDecodeThreads), 0,
                         s, p);
    };
    if (wide)
      once ? launch(linear_decode<Tag, D, 64, true, MANY>, 64) : launch(linear_decode<Tag, D, 64, false, MANY>, 64);
    else
      once ? launch(linear_decode<Tag, D, 32, true, MANY>, 32) : launch(linear_decode<Tag, D, 32, false, MANY>, 32);
  });
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
  launch_tokens<false>(p, head_dim, dtype, oxide::as_stream(stream));
  oxide::check_launch();
}

extern "C" size_t linear_attention_prefill_workspace_size(int64_t total_q, int64_t batch, int64_t num_heads,
                                                          int64_t num_kv_heads, int64_t head_dim,
                                                          int64_t max_seqlen_q) {
  const Plan plan = plan_prefill(total_q, batch, num_heads, num_kv_heads, head_dim, max_seqlen_q);
  return static_cast<size_t>(2 * plan.units * num_kv_heads * head_dim * head_dim) * sizeof(float);
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
  if (p.max_q <= kFewTokens) {
    launch_tokens<true>(p, head_dim, dtype, oxide::as_stream(stream));
    oxide::check_launch();
    return;
  }
  const Plan plan = plan_prefill(total_q, batch, num_heads, num_kv_heads, head_dim, max_seqlen_q);
  const size_t need = static_cast<size_t>(2 * plan.units * num_kv_heads * head_dim * head_dim) * sizeof(float);
  const bool cut = plan.piece_tokens > 0 && workspace && oxide::aligned16(workspace) && workspace_bytes >= need;
  hipStream_t s = oxide::as_stream(stream);
  dispatch(dtype, head_dim, [&](auto tag, auto d) {
    using Tag = decltype(tag);
    constexpr int D = decltype(d)::value;
    const dim3 threads(Tiles<D>::kThreads);
    const unsigned heads = static_cast<unsigned>(batch * num_kv_heads);
    if (!cut) {
      hipLaunchKernelGGL((linear_prefill_chunks<Tag, D, kWhole>), dim3(heads), threads, 0, s, p);
      return;
    }
    p.workspace = static_cast<float*>(workspace);
    p.units = plan.units;
    p.piece_tokens = static_cast<int>(plan.piece_tokens);
    const dim3 grid(static_cast<unsigned>((plan.units + batch) * num_kv_heads));
    hipLaunchKernelGGL((linear_prefill_chunks<Tag, D, kSums>), grid, threads, 0, s, p);
    // A piece adds up the sums before it by itself where they are few: over P pieces that
    // reads P (P - 1) / 2 states, where joining first moves 3 (P - 1) and is a launch more.
    p.joined = p.max_q > 8 * plan.piece_tokens;
    if (p.joined)
      hipLaunchKernelGGL((linear_prefill_join<D>),
                         dim3(static_cast<unsigned>(plan.units * num_kv_heads * (D * D / 4 / 256))), dim3(256), 0, s, p);
    // Query heads of one kv head are dealt out to workgroups, each with the state for itself,
    // where compute units would have none (at D = 64: two, which fit four): 2 x 500 tokens on
    // 28/4 heads of 64 24.1 -> 16.2 us, 2 x 1000 on 32/2 of 128 45.4 -> 32.7; dealt out to
    // every resident place, 4 x 700 on 32/8 would take 36.6 instead of 32.2.
    const int64_t places = (D == 128 ? 1 : 2) * oxide::device_cu_count();
    const int64_t idle = places / std::max<int64_t>(plan.units * num_kv_heads, 1);
    p.part_heads = static_cast<int>(p.group / std::clamp<int64_t>(idle, 1, p.group));
    const dim3 parts(grid.x, static_cast<unsigned>((p.group + p.part_heads - 1) / p.part_heads));
    hipLaunchKernelGGL((linear_prefill_chunks<Tag, D, kPieces>), parts, threads, 0, s, p);
  });
  oxide::check_launch();
}
