// Metadata of a mixed step on the device: prefix sums of the requests' lengths, blocks
// handed out of a free list into the block tables, and every token's slot and position.
//
// With C cached and Q new tokens of request b, pages of P tokens and tables of W entries:
//   held = min(W, ceil(C / P)), need = min(W, ceil((C + Q) / P)),
//   cu_q, cu_k, cu_new = prefix sums of Q, C + Q, need - held,
//   table[b][held + i] = free[cu_new[b] + i], i < need - held, if cu_new[b + 1] <= F,
//   slot of token p = C + i is table[b][p / P] * P + p % P.
// A decode step with complete tables is build_decode_metadata_device's; the reference
// fills both kinds on the host (crates/vllm-oxide/src/engine/mod.rs:160-196, 247-267).
//
// A token's block comes from the table where the request held it before the step and
// from the free list where it is new, so tokens never wait for the table's writers and
// one launch does both.  Bound by latency: a round trip for the lengths, the scan, a
// bisection, a round trip for the block id.  Every workgroup scans all requests by itself
// (up to 1024: four a lane, wave scans joined in LDS) and then serves its share of the
// tokens and of the new table entries, finding a token's request by bisection of the
// prefix sums in LDS.  64 single tokens 3.7 us, 700 requests with 63k tokens 6.3, of which
// a launch is 2-3; what is read and written would take 0.3 us.  Beyond 1024 requests a
// first launch of one workgroup writes the prefix sums and the second bisects them in
// memory (60,000 requests 93 us).
#include "oxide_common.hpp"

namespace {

constexpr int kThreads = 256;
constexpr int kFusedBatch = 1024;  // requests that every workgroup scans by itself
constexpr int kScanThreads = 1024;

// Division of 32-bit numbers by one that a launch keeps, as a multiplication and shifts
// (T. Granlund, P. L. Montgomery, "Division by invariant integers using multiplication",
// PLDI 1994, figure 4.1); the general divide is ten times the operations, and a scan's
// lane does four for each request.
struct Divisor {
  uint32_t d, m;
  int shift1, shift2;
};
Divisor divisor_of(uint32_t d) {
  int l = 0;
  while (l < 32 && (uint64_t{1} << l) < d) ++l;
  const uint64_t m = ((uint64_t{1} << 32) * ((uint64_t{1} << l) - d)) / d + 1;
  return Divisor{d, static_cast<uint32_t>(m), l < 1 ? l : 1, l > 1 ? l - 1 : 0};
}
__device__ __forceinline__ uint32_t divide(uint32_t x, Divisor by) {
  const uint32_t t = __umulhi(by.m, x);
  return (t + ((x - t) >> by.shift1)) >> by.shift2;
}
__device__ __forceinline__ uint64_t divide(uint64_t x, Divisor by) {
  return (x >> 32) == 0 ? divide(static_cast<uint32_t>(x), by) : x / by.d;
}

struct StepParams {
  const uint32_t* context_lens;
  const uint32_t* query_lens;
  const int32_t* position_offsets;  // [batch] or null
  int32_t* block_table;             // [batch, width]
  const int32_t* free_blocks;       // [num_free]
  uint32_t* cu_q;
  uint32_t* cu_k;
  uint32_t* cu_new;
  int64_t* slots;      // [num_tokens]
  int32_t* positions;  // [num_axes, num_tokens] or null
  int64_t num_tokens;
  int64_t num_free;
  uint32_t width;
  Divisor block_size;
  int batch;
  int num_axes;
};

// Blocks of the first `tokens` tokens that the table has room for.
__device__ __forceinline__ uint32_t blocks_of(const StepParams& p, uint64_t tokens) {
  const uint64_t whole = divide(tokens, p.block_size);
  const uint64_t n = whole + (whole * p.block_size.d != tokens);
  return static_cast<uint32_t>(min(n, static_cast<uint64_t>(p.width)));
}

struct Sums {
  uint32_t q, k, n;
};

// Exclusive prefix sums over the workgroup of each lane's three totals, and all lanes'.
template <int THREADS>
__device__ __forceinline__ Sums scan_totals(Sums own, Sums* s_wave, Sums& all) {
  Sums acc = own;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t q = __shfl_up(acc.q, off), k = __shfl_up(acc.k, off), n = __shfl_up(acc.n, off);
    if (lane >= off) acc.q += q, acc.k += k, acc.n += n;
  }
  if (lane == 63) s_wave[wave] = acc;
  __syncthreads();
  acc.q -= own.q, acc.k -= own.k, acc.n -= own.n;
  all = Sums{0, 0, 0};
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    const Sums s = s_wave[w];
    if (w < wave) acc.q += s.q, acc.k += s.k, acc.n += s.n;
    all.q += s.q, all.k += s.k, all.n += s.n;
  }
  return acc;
}

// THREADS * PER requests at a time, PER neighbours a lane; put(b, context, sums) is called
// with the sums before request b, and end(sums) with all requests'.
template <int THREADS, int PER, class Put, class End>
__device__ __forceinline__ void scan_requests(const StepParams& p, Sums* s_wave, Put put, End end) {
  Sums before{0, 0, 0};  // of the rounds so far
  for (int first = 0; first < p.batch; first += THREADS * PER) {
    const int b0 = first + static_cast<int>(threadIdx.x) * PER;
    uint32_t c[PER], q[PER];
    Sums each[PER], own{0, 0, 0};
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      c[i] = p.context_lens[min(b0 + i, p.batch - 1)];
      q[i] = p.query_lens[min(b0 + i, p.batch - 1)];
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint64_t total = static_cast<uint64_t>(c[i]) + q[i];
      each[i] = Sums{q[i], static_cast<uint32_t>(total), blocks_of(p, total) - blocks_of(p, c[i])};
      if (b0 + i >= p.batch) each[i] = Sums{0, 0, 0};
      own.q += each[i].q, own.k += each[i].k, own.n += each[i].n;
    }
    if (first > 0) __syncthreads();  // the wave totals of the round before are read
    Sums round;
    Sums at = scan_totals<THREADS>(own, s_wave, round);
    at.q += before.q, at.k += before.k, at.n += before.n;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (b0 + i < p.batch) put(b0 + i, c[i], at);
      at.q += each[i].q, at.k += each[i].k, at.n += each[i].n;
    }
    before.q += round.q, before.k += round.k, before.n += round.n;
  }
  if (threadIdx.x == 0) end(before);
}

// The last request whose prefix sum is at most x (sums: batch + 1 of them, sums[batch] > x).
__device__ __forceinline__ int request_of(const uint32_t* sums, int batch, uint32_t x) {
  int lo = 0, hi = batch;  // sums[lo] <= x < sums[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ void put_token(const StepParams& p, const uint32_t* cu_q, const uint32_t* cu_new,
                                          const uint32_t* context, int64_t t, uint32_t total) {
  int64_t slot = -1;
  int32_t position = 0;
  if (t < total) {
    const int b = request_of(cu_q, p.batch, static_cast<uint32_t>(t));
    const uint64_t c = context[b];
    const uint64_t pos = c + (static_cast<uint32_t>(t) - cu_q[b]);
    position = static_cast<int32_t>(static_cast<uint32_t>(pos));
    if (p.position_offsets)
      position = static_cast<int32_t>(static_cast<uint32_t>(position) + static_cast<uint32_t>(p.position_offsets[b]));
    const uint64_t block = divide(pos, p.block_size), in_block = pos - block * p.block_size.d;
    if (block < p.width) {
      const uint32_t held = blocks_of(p, c);
      const uint64_t at = cu_new[b] + (block - held);  // where in the free list a new block is
      const int32_t* id = nullptr;
      if (block < held) {
        id = p.block_table + static_cast<int64_t>(b) * p.width + static_cast<int64_t>(block);
      } else if (cu_new[b + 1] <= p.num_free && at < cu_new[b + 1]) {
        id = p.free_blocks + at;
      }
      if (id) slot = static_cast<int64_t>(*id) * p.block_size.d + static_cast<int64_t>(in_block);
    }
  }
  p.slots[t] = slot;
  if (p.positions)
    for (int a = 0; a < p.num_axes; ++a) p.positions[a * p.num_tokens + t] = position;
}

// Tokens, then new table entries, over the whole grid.
__device__ __forceinline__ void serve(const StepParams& p, const uint32_t* cu_q, const uint32_t* cu_new,
                                      const uint32_t* context) {
  const uint32_t total = cu_q[p.batch];
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t t = first; t < p.num_tokens; t += stride) put_token(p, cu_q, cu_new, context, t, total);
  const int64_t handed = min(static_cast<int64_t>(cu_new[p.batch]), p.num_free);
  for (int64_t n = first; n < handed; n += stride) {
    const int b = request_of(cu_new, p.batch, static_cast<uint32_t>(n));
    if (cu_new[b + 1] > p.num_free) continue;  // the list ends inside this request's blocks
    const uint32_t entry = blocks_of(p, context[b]) + static_cast<uint32_t>(n) - cu_new[b];
    p.block_table[static_cast<int64_t>(b) * p.width + entry] = p.free_blocks[n];
  }
}

template <int PER>
__global__ __launch_bounds__(kThreads) void step_metadata_fused(StepParams p) {
  constexpr int kMost = kThreads * PER;
  __shared__ uint32_t s_q[kMost + 1], s_new[kMost + 1], s_context[kMost];
  __shared__ Sums s_wave[kThreads / 64];
  auto put = [&](int b, const Sums& s) {
    s_q[b] = s.q;
    s_new[b] = s.n;
    if (blockIdx.x == 0) {
      p.cu_q[b] = s.q;
      p.cu_k[b] = s.k;
      p.cu_new[b] = s.n;
    }
  };
  scan_requests<kThreads, PER>(
      p, s_wave,
      [&](int b, uint32_t context, const Sums& s) {
        s_context[b] = context;
        put(b, s);
      },
      [&](const Sums& s) { put(p.batch, s); });
  __syncthreads();
  serve(p, s_q, s_new, s_context);
}

__global__ __launch_bounds__(kScanThreads) void step_metadata_scan(StepParams p) {
  __shared__ Sums s_wave[kScanThreads / 64];
  auto put = [&](int b, const Sums& s) {
    p.cu_q[b] = s.q;
    p.cu_k[b] = s.k;
    p.cu_new[b] = s.n;
  };
  scan_requests<kScanThreads, 4>(
      p, s_wave, [&](int b, uint32_t, const Sums& s) { put(b, s); }, [&](const Sums& s) { put(p.batch, s); });
}

__global__ __launch_bounds__(kThreads) void step_metadata_serve(StepParams p) {
  serve(p, p.cu_q, p.cu_new, p.context_lens);
}

}  // namespace

extern "C" void build_step_metadata_device(const uint32_t* context_lens, const uint32_t* query_lens,
                                           const int32_t* position_offsets, int32_t* block_table,
                                           int64_t max_blocks_per_seq, const int32_t* free_blocks,
                                           int64_t num_free_blocks, int64_t batch, int64_t block_size,
                                           int64_t num_tokens, int64_t num_axes, uint32_t* cu_seqlens_q,
                                           uint32_t* cu_seqlens_k, uint32_t* cu_new_blocks, int64_t* slot_mapping,
                                           int32_t* positions, void* stream) {
  if (batch < 0 || batch > 65535 || max_blocks_per_seq < 0 || batch * max_blocks_per_seq > INT32_MAX ||
      max_blocks_per_seq > INT32_MAX || num_free_blocks < 0 || block_size <= 0 || block_size > INT32_MAX ||
      num_tokens < 0 || num_tokens > INT32_MAX || (positions && (num_axes < 1 || num_axes > 4)) || !cu_seqlens_q ||
      !cu_seqlens_k || !cu_new_blocks || (num_tokens > 0 && !slot_mapping) ||
      (batch > 0 && (!context_lens || !query_lens)) || (batch * max_blocks_per_seq > 0 && !block_table) ||
      (num_free_blocks > 0 && !free_blocks)) {
    oxide::set_error(OXIDE_ERR_INVALID_ARGUMENT);
    return;
  }
  StepParams p{};
  p.context_lens = context_lens;
  p.query_lens = query_lens;
  p.position_offsets = position_offsets;
  p.block_table = block_table;
  p.free_blocks = free_blocks;
  p.cu_q = cu_seqlens_q;
  p.cu_k = cu_seqlens_k;
  p.cu_new = cu_new_blocks;
  p.slots = slot_mapping;
  p.positions = positions;
  p.num_tokens = num_tokens;
  p.num_free = num_free_blocks;
  p.width = static_cast<uint32_t>(max_blocks_per_seq);
  p.block_size = divisor_of(static_cast<uint32_t>(block_size));
  p.batch = static_cast<int>(batch);
  p.num_axes = static_cast<int>(num_axes);
  hipStream_t s = oxide::as_stream(stream);
  const int64_t items = num_tokens > batch ? num_tokens : batch;
  const int64_t wgs = (items + kThreads - 1) / kThreads, most = oxide::device_cu_count();
  const dim3 grid(static_cast<unsigned>(wgs < 1 ? 1 : wgs > most ? most : wgs));
  if (batch <= kFusedBatch) {
    hipLaunchKernelGGL(batch <= kThreads ? step_metadata_fused<1> : step_metadata_fused<kFusedBatch / kThreads>, grid,
                       dim3(kThreads), 0, s, p);
  } else {
    hipLaunchKernelGGL(step_metadata_scan, dim3(1), dim3(kScanThreads), 0, s, p);
    hipLaunchKernelGGL(step_metadata_serve, grid, dim3(kThreads), 0, s, p);
  }
  oxide::check_launch();
}
