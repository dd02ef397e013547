// Block tables, cache slots, positions and row offsets of a ragged batch from its request lengths.
//
// With counts[i] cache blocks and q[i] new tokens per sequence, F[i] = sum counts[:i], S[i] = sum q[:i]:
//   table[i, j]  = ids[F[i] + j]               (j < counts[i], else pad)
//   position[t]  = cached[i] + t - S[i]        (S[i] <= t < S[i + 1])
//   slot[t]      = ids[F[i] + position / B] * B + position % B
// Nothing is computed to speak of: a call lasts as long as one dependent chain (lengths -> sums -> block id -> store),
// plus the time to write the tables when they are large. So there is one launch and no second pass over partial sums:
// every CTA reads all lengths at once and sums them itself (a few KB out of L2, n / 256 per thread) and then takes its
// share of the output in pieces of four elements, 16 bytes a store. 8 sequences: 3.3 us, 256: 4.1 us. Lengths are read
// as at least 0, and sums saturate at 2^30 - 1, so no input
// reaches an index out of range: a token whose sequence has no block for it, and a row behind the last sequence, gets
// the pad block.
#include "common.cuh"
#include "serving_args.h"

namespace ajb {
namespace maps {

constexpr int kThreads = 256;
constexpr int kMaxSeqs = 16384;              // two sums and a length of 4 bytes per sequence in shared memory
constexpr int kCap = (1 << 30) - 1;

__device__ __forceinline__ int sat_add(int a, int b) { return min(a + b, kCap); }     // both in [0, kCap]

struct Params {
  const int *ids, *counts, *cached, *q_lens;
  int n_ids, seqs, total, width, block_size, pad;
  int *tables, *positions;
  long long* slots;
  int *q_start, *context;
};

// blocks[i] and tokens[i] = saturated sums of max(0, counts[:i]) and max(0, q_lens[:i]) for i in [0, n], lengths[i] =
// max(0, cached[i]); all threads of the CTA, `n` uniform. The three loads go out together.
__device__ void stage_lengths(const Params& p, int* blocks, int* tokens, int* lengths, int2* warp_sums) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, n = p.seqs;
  int carry_b = 0, carry_t = 0;
  for (int base = 0; base < n; base += kThreads) {
    const int i = base + t;
    int b = 0, q = 0;
    if (i < n) {
      b = p.counts[i];
      q = p.q_lens[i];
      const int c = p.cached[i];
      b = min(max(b, 0), kCap);
      q = min(max(q, 0), kCap);
      lengths[i] = max(c, 0);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up_b = __shfl_up_sync(0xffffffffu, b, o), up_q = __shfl_up_sync(0xffffffffu, q, o);
      if (lane >= o) { b = sat_add(b, up_b); q = sat_add(q, up_q); }
    }
    if (lane == 31) warp_sums[warp] = make_int2(b, q);
    __syncthreads();
    int before_b = carry_b, all_b = carry_b, before_t = carry_t, all_t = carry_t;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w == warp) { before_b = all_b; before_t = all_t; }
      const int2 sum = warp_sums[w];
      all_b = sat_add(all_b, sum.x);
      all_t = sat_add(all_t, sum.y);
    }
    // saturated sums cannot be taken back apart: the exclusive sum comes from the neighbour's inclusive one
    const int left_b = __shfl_up_sync(0xffffffffu, b, 1), left_q = __shfl_up_sync(0xffffffffu, q, 1);
    if (i < n) {
      blocks[i] = lane > 0 ? sat_add(before_b, left_b) : before_b;
      tokens[i] = lane > 0 ? sat_add(before_t, left_q) : before_t;
    }
    carry_b = all_b;
    carry_t = all_t;
    __syncthreads();
  }
  if (t == 0) { blocks[n] = carry_b; tokens[n] = carry_t; }
}

// last i in [0, n) with sums[i] <= t (n >= 1, sums[0] = 0 <= t)
__device__ __forceinline__ int find(const int* sums, int n, int t) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kThreads) batch_maps_kernel(const Params p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ int sums[];
  __shared__ int2 warp_sums[kThreads / 32];
  int* first_block = sums;
  int* first_token = sums + p.seqs + 1;
  int* cached = first_token + p.seqs + 1;
  stage_lengths(p, first_block, first_token, cached, warp_sums);
  __syncthreads();
  const int tokens = min(first_token[p.seqs], p.total);        // rows that belong to a sequence
  const long long thread = blockIdx.x * (long long)kThreads + threadIdx.x, threads = (long long)gridDim.x * kThreads;

  for (long long i = thread; i <= p.seqs; i += threads) {
    p.q_start[i] = min(first_token[i], p.total);
    if (i < p.seqs) p.context[i] = (int)min((long long)cached[i] + max(p.q_lens[i], 0), 0x7fffffffll);
  }

  // four tokens per thread: one search, then a step to the next sequence where one ends
  const int token_pieces = (p.total + 3) >> 2;
  for (long long piece = thread; piece < token_pieces; piece += threads) {
    const int t0 = (int)piece * 4;
    int pos[4];
    long long slot[4];
    int i = t0 < tokens ? find(first_token, p.seqs, t0) : p.seqs;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int t = t0 + k;
      pos[k] = 0;
      slot[k] = (long long)p.pad * p.block_size;
      if (t < tokens) {
        while (first_token[i + 1] <= t) ++i;                   // empty sequences are stepped over
        const unsigned at = (unsigned)cached[i] + (unsigned)(t - first_token[i]);        // below 2^31 + 2^30
        const unsigned b = at / (unsigned)p.block_size;
        const unsigned offset = at - b * (unsigned)p.block_size;
        const int first = first_block[i];
        const bool has = b < (unsigned)(first_block[i + 1] - first) && (unsigned)first + b < (unsigned)p.n_ids;
        const int id = has ? p.ids[first + (int)b] : p.pad;
        pos[k] = (int)min(at, 0x7fffffffu);
        slot[k] = (long long)id * p.block_size + offset;
      }
    }
    if (t0 + 4 <= p.total) {
      *reinterpret_cast<int4*>(p.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *reinterpret_cast<longlong2*>(p.slots + t0) = make_longlong2(slot[0], slot[1]);
      *reinterpret_cast<longlong2*>(p.slots + t0 + 2) = make_longlong2(slot[2], slot[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (t0 + k < p.total) {
          p.positions[t0 + k] = pos[k];
          p.slots[t0 + k] = slot[k];
        }
    }
  }

  // four table entries per thread; rows of any width, so a piece may end in the next row
  const long long cells = (long long)p.seqs * p.width;
  for (long long piece = thread; piece < (cells + 3) >> 2; piece += threads) {
    const long long c0 = piece * 4;
    int row = c0 <= 0xffffffffll ? (int)((unsigned)c0 / (unsigned)p.width) : (int)(c0 / p.width);
    int col = (int)(c0 - (long long)row * p.width);
    int v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = p.pad;
      if (row < p.seqs) {
        const long long at = (long long)first_block[row] + col;
        if (at < first_block[row + 1] && at < p.n_ids) v[k] = p.ids[at];
      }
      if (++col == p.width) { col = 0; ++row; }
    }
    if (c0 + 4 <= cells) {
      *reinterpret_cast<int4*>(p.tables + c0) = make_int4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c0 + k < cells) p.tables[c0 + k] = v[k];
    }
  }
}

}  // namespace maps
}  // namespace ajb

// ids [n_ids] block ids of all sequences, one after another; counts / cached / q_lens [seqs]; all int32 on the device.
// tables [seqs, width], positions [total], slots [total] (int64), q_start [seqs + 1], context [seqs]; tables, positions
// and slots 16-byte aligned.
extern "C" int ajb_batch_maps(const void* arguments) {
  using namespace ajb;
  const BatchMapsArgs& args = *static_cast<const BatchMapsArgs*>(arguments);
  AJB_REQUIRE(args.size == (int)sizeof(args), "batch maps: arguments of %d bytes, not %d", args.size, (int)sizeof(args));
  const auto& [size, ids, counts, cached, q_lens, n_ids, seqs, total, width, block_size, pad, tables,
               positions, slots, q_start, context, stream] = args;
  AJB_REQUIRE(seqs >= 0 && seqs <= maps::kMaxSeqs, "batch maps: %d sequences (at most %d)", seqs, maps::kMaxSeqs);
  AJB_REQUIRE(total >= 0 && total <= maps::kCap && n_ids >= 0 && n_ids <= maps::kCap && width >= 1 && block_size >= 1,
              "batch maps: %d tokens, %d block ids, %d blocks per table row, %d tokens per block are out of range", total, n_ids,
              width, block_size);
  AJB_REQUIRE(((reinterpret_cast<uintptr_t>(tables) | reinterpret_cast<uintptr_t>(positions) | reinterpret_cast<uintptr_t>(slots)) & 15) == 0,
              "batch maps: tables, positions and slots must be 16-byte aligned");
  // every CTA reads all lengths while others write: results must lie apart from them, and from one another
  const long long n = seqs;
  const MemoryRange results[5] = {{tables, 4 * n * width}, {positions, 4ll * total}, {slots, 8ll * total}, {q_start, 4 * (n + 1)}, {context, 4 * n}};
  const MemoryRange inputs[4] = {{ids, 4ll * n_ids}, {counts, 4 * n}, {cached, 4 * n}, {q_lens, 4 * n}};
  for (int i = 0; i < 5; ++i) {
    for (int j = 0; j < i; ++j) AJB_REQUIRE(!results[i].meets(results[j]), "batch maps: results %d and %d overlap", j, i);
    for (int j = 0; j < 4; ++j) AJB_REQUIRE(!results[i].meets(inputs[j]), "batch maps: result %d overlaps input %d", i, j);
  }
  maps::Params p;
  p.ids = (const int*)ids; p.counts = (const int*)counts; p.cached = (const int*)cached; p.q_lens = (const int*)q_lens;
  p.n_ids = n_ids; p.seqs = seqs; p.total = total; p.width = width; p.block_size = block_size; p.pad = pad;
  p.tables = (int*)tables; p.positions = (int*)positions; p.slots = (long long*)slots; p.q_start = (int*)q_start;
  p.context = (int*)context;
  const int smem = 3 * (seqs + 1) * (int)sizeof(int);
  // Function attributes belong to a device: raised once on each, to what the largest call takes, and never lowered, as
  // another thread may be between this and its launch. (What a launch may use without it, 48 KB, holds the static array too.)
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  AJB_CUDA_OK(cudaGetDevice(&dev));
  if (dev >= kMaxDevices || !configured[dev]) {
    AJB_CUDA_OK(cudaFuncSetAttribute(maps::batch_maps_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     3 * (maps::kMaxSeqs + 1) * (int)sizeof(int)));
    if (dev < kMaxDevices) configured[dev] = true;
  }
  const long long pieces = ((long long)total + 3) / 4 + ((long long)seqs * width + 3) / 4 + 1;
  const long long blocks = (pieces + maps::kThreads - 1) / maps::kThreads;
  return launch_early(maps::batch_maps_kernel, dim3((unsigned)(blocks < 4ll * sm_count() ? blocks : 4ll * sm_count())),
                      dim3(maps::kThreads), smem, reinterpret_cast<cudaStream_t>(stream), p);
}
