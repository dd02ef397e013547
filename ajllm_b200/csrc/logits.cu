// Logits processing ahead of the sampler: penalties for repeated tokens, token biases and grammar bit masks, from bf16 or
// fp32 logits to fp32 logits in one launch.
//
// For token v of a row, c(v) = how often it was generated, seen(v) = whether it is anywhere in the history (prompt and
// generated tokens), r / p / f = the row's repetition, presence and frequency penalty:
//   x = logit;  x = seen ? (x > 0 ? x / r : x * r) : x;  x = x - f * c - p * (c > 0);  x = x + bias;  x = masked ? -inf : x
// Every step rounds to fp32 once and nothing is contracted (and this file is compiled without fast math, so that subnormal
// numbers stay what they are): the result equals elementary fp32 operations bit for bit.
//
// Bound by memory: 6 bytes per bf16 logit (read, write) and a bit of the mask; where a mask shuts four neighbouring
// tokens their logits are not read. Only the few tokens of the history and of the bias list need arithmetic, so the rows
// are streamed through (widen, mask) and those tokens then mended one by one: history tokens are counted in a table in
// shared memory, and the thread that takes a token's count out of the table (an atomic that leaves 0) is the one that
// writes that token. Counts are whole numbers, so the order of the additions does not show. Biases follow in list order
// within one warp; lanes that hold the same token take turns.
//
// Few logits (kTwoLaunches below): one launch, a CTA streams a piece of a row with eight warps while four count the
// history tokens of that piece, then mends them. Many: a launch that only streams, and one with a CTA per row that counts
// and works out the new logits while the first still runs, waits for it on the device and stores them: every piece no
// longer looks through its row's whole history, and no streaming warp waits for one that counts (256 rows of 128256 with
// 2560 tokens of history, biases and a mask: 56 us in one launch, 46 us in two; 36 us of that is the streaming alone).
#include "common.cuh"
#include "serving_args.h"

namespace ajb {
namespace logits {

constexpr int kStreamThreads = 256;
constexpr int kHistoryThreads = 128;             // launched in addition when there is a history
constexpr int kUnroll = 4;
constexpr int kHistoryUnroll = 4;
// Logits from which two launches are faster: 128 rows of 128256 with 2048 tokens of history take 35 us in one launch and
// 27 us in two, 64 rows 20 us and 24 us.
constexpr long long kTwoLaunches = 1 << 23;
constexpr unsigned kMinusInf = 0xff800000u;

// Counts of the tokens of a piece. A cell has one bit for "in the prompt" and the rest for "times generated"; histories
// of up to 32767 tokens fit 16-bit cells, two to a word of shared memory (pieces of 16384 tokens), longer ones take whole
// words (pieces of 8192): 32 KB either way.
template <bool kNarrow>
struct Table {
  static constexpr int kMaxChunk = kNarrow ? 16384 : 8192;
  static constexpr unsigned kPrompt = kNarrow ? 0x8000u : 0x80000000u;
  static __device__ __forceinline__ int words(int chunk) { return kNarrow ? chunk >> 1 : chunk; }
  static __device__ __forceinline__ void add(unsigned* t, int i, bool prompt) {
    const int shift = kNarrow ? 16 * (i & 1) : 0;
    unsigned* word = t + (kNarrow ? i >> 1 : i);
    if (prompt) atomicOr(word, kPrompt << shift);
    else atomicAdd(word, 1u << shift);
  }
  static __device__ __forceinline__ unsigned take(unsigned* t, int i) {
    if (!kNarrow) return atomicExch(t + i, 0u);
    const int shift = 16 * (i & 1);
    return (atomicAnd(t + (i >> 1), ~(0xffffu << shift)) >> shift) & 0xffffu;
  }
};

// (Inputs are read through pointers that have passed behind_wait: the kernels start before the launch in front of them, which
// may write those inputs, has ended.)
struct Params {
  const void* in;
  long long in_pitch;
  float* out;                    // [rows, vocab]
  int rows, vocab;
  const int* history;            // [rows, history_width] token ids, null: no penalties
  long long history_pitch;
  int history_width;
  const int *prompt_lens, *history_lens;
  const float *repetition, *presence, *frequency;      // [rows], null: 1, 0, 0
  const int* bias_ids;           // [rows, biases], ids out of range are skipped
  const float* bias_values;
  int biases;
  const unsigned* mask;          // [rows, mask_pitch] words, bit v % 32 of word v / 32 set = token v allowed; null: all are
  long long mask_pitch;
  int chunk, chunks;             // tokens per piece (a multiple of 32), pieces per row
  int pieces;                    // in all (two launches)
};

template <typename T>
__device__ __forceinline__ float load1(const T* p);
template <>
__device__ __forceinline__ float load1<float>(const float* p) { return ld_settled(p); }
template <>
__device__ __forceinline__ float load1<__nv_bfloat16>(const __nv_bfloat16* p) {
  return __uint_as_float((unsigned)ld_settled(reinterpret_cast<const unsigned short*>(p)) << 16);
}
// four neighbouring logits, as loaded and as fp32 bits
template <typename T>
struct Four;
template <>
struct Four<float> {
  uint4 v;
  __device__ __forceinline__ void load(const float* p) { v = ld_settled(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ uint4 wide() const { return v; }
};
template <>
struct Four<__nv_bfloat16> {
  uint2 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = ld_settled(reinterpret_cast<const uint2*>(p)); }
  __device__ __forceinline__ uint4 wide() const { return make_uint4(v.x << 16, v.x & 0xffff0000u, v.y << 16, v.y & 0xffff0000u); }
};

__device__ __forceinline__ bool open_token(const unsigned* mask, int v) {
  return mask == nullptr || ((ld_settled(mask + (v >> 5)) >> (v & 31)) & 1u);
}

// Tokens [lo, hi) of a row, widened and masked, by `threads` threads.
template <typename T>
__device__ __forceinline__ void stream_piece(const T* in, float* out, const unsigned* mask, int lo, int hi, int thread, int threads) {
  // four-token groups start where `out` is 16-byte aligned; the input rows have to agree with that to be read in groups
  const int lead = (int)((4 - ((reinterpret_cast<uintptr_t>(out + lo) >> 2) & 3)) & 3);
  const int first = min(hi, lo + lead);
  const bool wide = (reinterpret_cast<uintptr_t>(in + lo + lead) & (4 * sizeof(T) - 1)) == 0;
  auto one = [&](int v) { out[v] = open_token(mask, v) ? load1<T>(in + v) : __uint_as_float(kMinusInf); };
  if (!wide) {
    for (int v = lo + thread; v < hi; v += threads) one(v);
    return;
  }
  for (int v = lo + thread; v < first; v += threads) one(v);
  const int groups = (hi - first) >> 2;
  for (int g0 = thread; g0 < groups; g0 += threads * kUnroll) {
    unsigned open[kUnroll];
    Four<T> x[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int g = g0 + u * threads, v = first + 4 * g;
      open[u] = g < groups ? 15u : 0u;
      if (mask != nullptr && g < groups) {
        // a group lies in one word, or in two neighbours when the row does not start on a 16-byte boundary
        const unsigned w0 = ld_settled(mask + (v >> 5)), w1 = (v & 31) > 28 ? ld_settled(mask + (v >> 5) + 1) : 0u;
        open[u] = __funnelshift_r(w0, w1, v & 31) & 15u;
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (open[u]) x[u].load(in + first + 4 * (g0 + u * threads));
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int g = g0 + u * threads;
      if (g < groups) {
        uint4 w = x[u].wide();
        if (!(open[u] & 1u)) w.x = kMinusInf;
        if (!(open[u] & 2u)) w.y = kMinusInf;
        if (!(open[u] & 4u)) w.z = kMinusInf;
        if (!(open[u] & 8u)) w.w = kMinusInf;
        *reinterpret_cast<uint4*>(out + first + 4 * g) = w;
      }
    }
  }
  for (int v = first + 4 * groups + thread; v < hi; v += threads) one(v);
}

// visit(place, token) for the history tokens in [lo, hi); `threads` threads, several loads in flight
template <typename Visit>
__device__ __forceinline__ void for_history(const int* history, int len, int lo, int hi, int thread, int threads, Visit visit) {
  for (int i0 = thread; i0 < len; i0 += threads * kHistoryUnroll) {
    int v[kHistoryUnroll];
#pragma unroll
    for (int u = 0; u < kHistoryUnroll; ++u) {
      const int i = i0 + u * threads;
      v[u] = i < len ? ld_settled(history + i) : -1;
    }
#pragma unroll
    for (int u = 0; u < kHistoryUnroll; ++u)
      if (v[u] >= lo && v[u] < hi) visit(i0 + u * threads, v[u]);
  }
}

// The row's first biases, as loaded by the first warp well before they are added.
struct FirstBiases {
  int id[2];
  float value[2];
  __device__ __forceinline__ void load(const Params& p, int row) {
    const int* ids = behind_wait(p.bias_ids);
    const float* values = behind_wait(p.bias_values);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = 32 * u + (int)threadIdx.x;
      const bool there = threadIdx.x < 32 && i < p.biases;
      id[u] = there ? ld_settled(ids + (size_t)row * p.biases + i) : -1;
      value[u] = there ? ld_settled(values + (size_t)row * p.biases + i) : 0.0f;
    }
  }
};

// The row's biases of tokens in [lo, hi), by the first warp: in list order, lanes with the same token one after another.
__device__ __forceinline__ void add_biases(const Params& p, const FirstBiases& ahead, int row, float* out, const unsigned* mask, int lo,
                                           int hi) {
  if (threadIdx.x >= 32) return;
  const int* ids = behind_wait(p.bias_ids) + (size_t)row * p.biases;
  const float* values = behind_wait(p.bias_values) + (size_t)row * p.biases;
#pragma unroll 1
  for (int base = 0; base < p.biases; base += 32) {
    const int i = base + (int)threadIdx.x;
    const bool later = base >= 64 && i < p.biases;
    const int v = base == 0 ? ahead.id[0] : base == 32 ? ahead.id[1] : later ? ld_settled(ids + i) : -1;
    const float value = base == 0 ? ahead.value[0] : base == 32 ? ahead.value[1] : later ? ld_settled(values + i) : 0.0f;
    const bool mine = v >= lo && v < hi && open_token(mask, v);
    // turn of this lane among the lanes with the same token
    const unsigned same = __match_any_sync(0xffffffffu, mine ? v : -1);
    const int turn = __popc(same & ((1u << threadIdx.x) - 1u));
    const int turns = __reduce_max_sync(0xffffffffu, mine ? __popc(same) : 0);
    for (int k = 0; k < turns; ++k) {
      if (mine && turn == k) {
        volatile float* at = out + v;
        *at = __fadd_rn(*at, value);
      }
      __syncwarp();
    }
  }
}

template <typename T, bool kNarrow>
__global__ void __launch_bounds__(kStreamThreads + kHistoryThreads) process_logits_kernel(const Params p) {
  extern __shared__ unsigned table[];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  using Tab = Table<kNarrow>;
  const int row = (int)(blockIdx.x / (unsigned)p.chunks), part = (int)(blockIdx.x % (unsigned)p.chunks);
  const int lo = part * p.chunk, hi = min(p.vocab, lo + p.chunk);
  const T* in = behind_wait(reinterpret_cast<const T*>(p.in)) + (size_t)row * p.in_pitch;
  float* out = p.out + (size_t)row * p.vocab;
  const unsigned* mask = p.mask != nullptr ? behind_wait(p.mask) + (size_t)row * p.mask_pitch : nullptr;
  const int* history = p.history != nullptr ? behind_wait(p.history) + (size_t)row * p.history_pitch : nullptr;
  const int thread = threadIdx.x;
  // what is needed behind the streaming is asked for in front of it
  const int stored = history != nullptr ? p.history_lens[row] : 0;
  float r = 1.0f, pr = 0.0f, f = 0.0f;
  if (history != nullptr) {
    if (p.repetition != nullptr) r = p.repetition[row];
    if (p.presence != nullptr) pr = p.presence[row];
    if (p.frequency != nullptr) f = p.frequency[row];
  }
  FirstBiases ahead;
  ahead.load(p, row);
  const int len = min(max(stored, 0), p.history_width);
  if (thread < kStreamThreads) {
    stream_piece<T>(in, out, mask, lo, hi, thread, kStreamThreads);
  } else if (len > 0) {
    const int t = thread - kStreamThreads;
    for (int i = t; i < (Tab::words(p.chunk) >> 2); i += kHistoryThreads) reinterpret_cast<uint4*>(table)[i] = make_uint4(0, 0, 0, 0);
    asm volatile("bar.sync 1, %0;" ::"n"(kHistoryThreads) : "memory");
    const int prompt = p.prompt_lens[row];
    for_history(history, len, lo, hi, t, kHistoryThreads, [&](int i, int v) { Tab::add(table, v - lo, i < prompt); });
  }

  // ---- tokens of the history
  if (len > 0) {
    __syncthreads();
    for_history(history, len, lo, hi, thread, kStreamThreads + kHistoryThreads, [&](int, int v) {
      const unsigned held = Tab::take(table, v - lo);
      if (held == 0u || !open_token(mask, v)) return;
      float x = load1<T>(in + v);
      x = x > 0.0f ? __fdiv_rn(x, r) : __fmul_rn(x, r);
      const unsigned count = held & ~Tab::kPrompt;
      if (count > 0u) x = __fsub_rn(__fsub_rn(x, __fmul_rn(f, (float)count)), pr);
      out[v] = x;
    });
  }

  if (p.biases > 0) {
    __syncthreads();
    add_biases(p, ahead, row, out, mask, lo, hi);
  }
}


// ---- two launches
// The first: rows streamed by as many CTAs as run at once, each with every gridDim-th piece; the mask words of a piece are
// fetched a piece ahead and lie in shared memory, so that a group's bits do not cost it a second latency.
constexpr int kStreamCtas = 4;                   // per SM: two CTAs of the second launch fit beside them
constexpr int kStreamChunk = 8192;

template <typename T, bool kMasked>
__global__ void __launch_bounds__(kStreamThreads, 6) stream_logits_kernel(const Params p) {
  constexpr int kWords = kStreamChunk / 32 + 1;          // one more than a piece has: groups look at the next word too
  constexpr int kEach = (kWords + kStreamThreads - 1) / kStreamThreads;
  __shared__ unsigned shared[2][kMasked ? kWords : 1];
  // in this order: the second launch reads the inputs without waiting for anything but its start
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int thread = threadIdx.x, step = (int)gridDim.x, all = (p.vocab + 31) / 32;
  const T* const logits = behind_wait(reinterpret_cast<const T*>(p.in));
  const unsigned* const mask = behind_wait(p.mask);
  unsigned ahead[kEach];
  auto load_words = [&](int piece) {
    const int row = piece / p.chunks, first = (piece - row * p.chunks) * (kStreamChunk / 32);
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int i = thread + u * kStreamThreads;
      ahead[u] = i < kWords && first + i < all ? ld_settled(mask + (size_t)row * p.mask_pitch + first + i) : 0u;
    }
  };
  if (kMasked && (int)blockIdx.x < p.pieces) load_words((int)blockIdx.x);
  int turn = 0;
#pragma unroll 1
  for (int piece = (int)blockIdx.x; piece < p.pieces; piece += step, turn ^= 1) {
    const int row = piece / p.chunks, part = piece - row * p.chunks;
    const int lo = part * kStreamChunk, hi = min(p.vocab, lo + kStreamChunk);
    const T* in = logits + (size_t)row * p.in_pitch;
    float* out = p.out + (size_t)row * p.vocab;
    const unsigned* words = shared[turn];
    if (kMasked) {
#pragma unroll
      for (int u = 0; u < kEach; ++u)
        if (thread + u * kStreamThreads < kWords) shared[turn][thread + u * kStreamThreads] = ahead[u];
      if (piece + step < p.pieces) load_words(piece + step);
      __syncthreads();                                   // (the buffer two pieces back was read before the last one)
    }
    // four-token groups start where `out` is 16-byte aligned; the input rows have to agree with that to be read in groups
    const int lead = (int)((4 - ((reinterpret_cast<uintptr_t>(out + lo) >> 2) & 3)) & 3);
    const int first = min(hi, lo + lead);
    const bool wide = (reinterpret_cast<uintptr_t>(in + lo + lead) & (4 * sizeof(T) - 1)) == 0;
    const int groups = wide ? (hi - first) >> 2 : 0;
#pragma unroll 1
    for (int g0 = thread; g0 < groups; g0 += kStreamThreads * kUnroll) {
      unsigned open[kUnroll];
      Four<T> x[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int g = g0 + u * kStreamThreads, at = first - lo + 4 * g;
        open[u] = g < groups ? 15u : 0u;
        if (kMasked && g < groups) open[u] = __funnelshift_r(words[at >> 5], words[(at >> 5) + 1], at & 31) & 15u;
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (open[u]) x[u].load(in + first + 4 * (g0 + u * kStreamThreads));
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int g = g0 + u * kStreamThreads;
        if (g < groups) {
          uint4 w = x[u].wide();
          if (kMasked) {
            if (!(open[u] & 1u)) w.x = kMinusInf;
            if (!(open[u] & 2u)) w.y = kMinusInf;
            if (!(open[u] & 4u)) w.z = kMinusInf;
            if (!(open[u] & 8u)) w.w = kMinusInf;
          }
          *reinterpret_cast<uint4*>(out + first + 4 * g) = w;
        }
      }
    }
    // what is in front of and behind the groups (everything, when rows cannot be read in groups)
    const int before = wide ? first - lo : 0, rest = hi - lo - 4 * groups;
#pragma unroll 1
    for (int i = thread; i < rest; i += kStreamThreads) {
      const int v = lo + (i < before ? i : i + 4 * groups);
      const bool open = !kMasked || ((words[(v - lo) >> 5] >> ((v - lo) & 31)) & 1u);
      out[v] = open ? load1<T>(in + v) : __uint_as_float(kMinusInf);
    }
  }
}

// The second: a CTA per row. The vocabulary is gone through in ranges of the table's size, and the row's history once per
// range. Up to kHeld tokens the history and the logits of its tokens lie in shared memory, and the new logits wait there
// until the streaming launch has ended; longer histories are read and counted after that.
constexpr int kMendThreads = 256;
constexpr int kBatch = 4;
constexpr int kHeld = 4096;
constexpr int kMendRange = 32768;                // tokens per range: 64 KB of 16-bit cells, or half as many of 32 bits

template <typename T, bool kNarrow>
__global__ void __launch_bounds__(kMendThreads, 6) mend_logits_kernel(const Params p) {
  extern __shared__ __align__(16) unsigned table[];
  using Tab = Table<kNarrow>;
  constexpr int kRange = kNarrow ? kMendRange : kMendRange / 2;
  const int row = blockIdx.x, thread = threadIdx.x;
  // the launches that write the inputs have ended when this one starts: every CTA of the streaming launch has waited for them
  const T* in = reinterpret_cast<const T*>(p.in) + (size_t)row * p.in_pitch;
  float* out = p.out + (size_t)row * p.vocab;
  const unsigned* mask = p.mask != nullptr ? p.mask + (size_t)row * p.mask_pitch : nullptr;
  FirstBiases ahead;
  ahead.load(p, row);
  if (p.history != nullptr) {
    const int cells = min(kRange, (p.vocab + 7) & ~7);
    int* tokens = reinterpret_cast<int*>(table + Tab::words(cells));
    float* values = reinterpret_cast<float*>(tokens + min(kHeld, p.history_width));
    const int* history = p.history + (size_t)row * p.history_pitch;
    const int len = min(max(p.history_lens[row], 0), p.history_width), prompt = p.prompt_lens[row];
    const float r = p.repetition != nullptr ? p.repetition[row] : 1.0f;
    const float pr = p.presence != nullptr ? p.presence[row] : 0.0f;
    const float f = p.frequency != nullptr ? p.frequency[row] : 0.0f;
    auto changed = [&](float x, unsigned got) {
      x = x > 0.0f ? __fdiv_rn(x, r) : __fmul_rn(x, r);
      const unsigned count = got & ~Tab::kPrompt;
      return count > 0u ? __fsub_rn(__fsub_rn(x, __fmul_rn(f, (float)count)), pr) : x;
    };
#pragma unroll 1
    for (int i = thread; i < (Tab::words(cells) >> 2); i += kMendThreads) reinterpret_cast<uint4*>(table)[i] = make_uint4(0, 0, 0, 0);
    const bool held = len <= kHeld;
    if (held) {
#pragma unroll 4
      for (int i = thread; i < len; i += kMendThreads) {
        const int v = ld_settled(history + i);
        tokens[i] = (unsigned)v < (unsigned)p.vocab ? v : -1;          // below -1 stand tokens whose count has been taken
      }
    } else {
      asm volatile("griddepcontrol.wait;" ::: "memory");
    }
    __syncthreads();
#pragma unroll 1
    for (int lo = 0; lo < p.vocab; lo += kRange) {
      const int hi = min(p.vocab, lo + kRange);
      if (held) {
#pragma unroll 4
        for (int i = thread; i < len; i += kMendThreads) {
          const int v = tokens[i];
          if (v >= lo && v < hi) Tab::add(table, v - lo, i < prompt);
        }
        __syncthreads();
        // the thread that finds a count keeps it (with the token as -2 - v); the same token elsewhere is done with
#pragma unroll 4
        for (int i = thread; i < len; i += kMendThreads) {
          const int v = tokens[i];
          if (v >= lo && v < hi) {
            const unsigned got = Tab::take(table, v - lo);
            values[i] = __uint_as_float(got);
            tokens[i] = got != 0u ? -2 - v : -1;
          }
        }
      } else {
        for_history(history, len, lo, hi, thread, kMendThreads, [&](int i, int v) { Tab::add(table, v - lo, i < prompt); });
        __syncthreads();
        for_history(history, len, lo, hi, thread, kMendThreads, [&](int, int v) {
          const unsigned got = Tab::take(table, v - lo);
          if (got != 0u && open_token(mask, v)) out[v] = changed(load1<T>(in + v), got);
        });
      }
      __syncthreads();
    }
    if (held) {
      // all counts are there: one round of reads, once per token (reading every occurrence ahead of counting cost the
      // streaming launch a quarter of its bandwidth, reading range by range a latency per range)
#pragma unroll 1
      for (int i0 = thread; i0 < len; i0 += kBatch * kMendThreads) {
        int v[kBatch];
        unsigned word[kBatch];
        float x[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int i = i0 + u * kMendThreads;
          v[u] = i < len ? -2 - tokens[i] : -1;
          if (v[u] >= 0) {
            x[u] = load1<T>(in + v[u]);
            word[u] = mask != nullptr ? ld_settled(mask + (v[u] >> 5)) : 0xffffffffu;
          }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          if (v[u] >= 0) {
            const int i = i0 + u * kMendThreads;
            if ((word[u] >> (v[u] & 31)) & 1u) values[i] = changed(x[u], __float_as_uint(values[i]));
            else tokens[i] = -1;
          }
        }
      }
      asm volatile("griddepcontrol.wait;" ::: "memory");
#pragma unroll 4
      for (int i = thread; i < len; i += kMendThreads) {
        const int v = tokens[i];
        if (v <= -2) out[-2 - v] = values[i];
      }
    }
  } else {
    asm volatile("griddepcontrol.wait;" ::: "memory");
  }
  if (p.biases > 0) {
    __syncthreads();
    add_biases(p, ahead, row, out, mask, 0, p.vocab);
  }
}

}  // namespace logits
}  // namespace ajb

// logits [rows, vocab] (dtype 0: bf16, 1: fp32) with in_pitch elements between rows; out fp32 [rows, vocab] contiguous,
// not overlapping the logits. Null pointers switch the parts off: history (with lens), repetition / presence /
// frequency, bias_ids (biases = 0), mask.
extern "C" int ajb_process_logits(const void* arguments) {
  using namespace ajb;
  const ProcessLogitsArgs& args = *static_cast<const ProcessLogitsArgs*>(arguments);
  AJB_REQUIRE(args.size == (int)sizeof(args), "process logits: arguments of %d bytes, not %d", args.size, (int)sizeof(args));
  const auto& [size, logits, dtype, in_pitch, out, rows, vocab, history, history_pitch, history_width,
               prompt_lens, history_lens, repetition, presence, frequency, bias_ids, bias_values, biases,
               mask, mask_pitch, stream] = args;
  AJB_REQUIRE(dtype == 0 || dtype == 1, "process logits: unknown type %d", dtype);
  AJB_REQUIRE(rows >= 0 && vocab >= 1 && vocab <= (1 << 30) && history_width >= 0 && biases >= 0, "process logits: sizes out of range");
  AJB_REQUIRE(history == nullptr || (prompt_lens != nullptr && history_lens != nullptr), "process logits: a history comes with its lengths");
  AJB_REQUIRE(biases == 0 || (bias_ids != nullptr && bias_values != nullptr), "process logits: biases come with ids and values");
  if (rows == 0) return 0;
  logits::Params p;
  p.in = logits; p.in_pitch = in_pitch; p.out = (float*)out; p.rows = rows; p.vocab = vocab;
  p.history = (const int*)history; p.history_pitch = history_pitch; p.history_width = history_width;
  p.prompt_lens = (const int*)prompt_lens; p.history_lens = (const int*)history_lens;
  p.repetition = (const float*)repetition; p.presence = (const float*)presence; p.frequency = (const float*)frequency;
  p.bias_ids = (const int*)bias_ids; p.bias_values = (const float*)bias_values; p.biases = biases;
  p.mask = (const unsigned*)mask; p.mask_pitch = mask_pitch;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool counts = history != nullptr && history_width > 0, narrow = history_width <= 32767;
  if (!counts) p.history = nullptr;
  const bool mends = counts || biases > 0;
  if (!mends || (long long)rows * vocab >= logits::kTwoLaunches) {
    p.chunk = logits::kStreamChunk;
    p.chunks = (vocab + p.chunk - 1) / p.chunk;
    const long long pieces = (long long)rows * p.chunks;
    AJB_REQUIRE(pieces <= 0x3fffffffll, "process logits: %d rows of %d tokens are too many", rows, vocab);
    p.pieces = (int)pieces;
    const long long most = (long long)logits::kStreamCtas * sm_count(), each = (pieces + most - 1) / most;
    const int grid = (int)((pieces + each - 1) / each);          // as many pieces for each CTA
    void (*const stream_kernels[4])(logits::Params) = {
        logits::stream_logits_kernel<__nv_bfloat16, false>, logits::stream_logits_kernel<__nv_bfloat16, true>,
        logits::stream_logits_kernel<float, false>, logits::stream_logits_kernel<float, true>};
    const int which = 2 * dtype + (mask != nullptr);
    // function attributes belong to a device: set once on each
    static bool configured[8][kMaxDevices] = {};
    int dev = 0;
    AJB_CUDA_OK(cudaGetDevice(&dev));
    if (dev >= kMaxDevices || !configured[which][dev]) {
      // with an SM's memory divided the way the second launch needs it, that one's CTAs can start beside these
      AJB_CUDA_OK(cudaFuncSetAttribute(stream_kernels[which], cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
      if (dev < kMaxDevices) configured[which][dev] = true;
    }
    if (const int rc = launch_early(stream_kernels[which], dim3(grid), dim3(logits::kStreamThreads), 0, s, p)) return rc;
    if (!mends) return 0;
    void (*const mend_kernels[4])(logits::Params) = {
        logits::mend_logits_kernel<__nv_bfloat16, false>, logits::mend_logits_kernel<__nv_bfloat16, true>,
        logits::mend_logits_kernel<float, false>, logits::mend_logits_kernel<float, true>};
    auto kernel = mend_kernels[2 * dtype + narrow];
    const int range = narrow ? logits::kMendRange : logits::kMendRange / 2, cells = vocab < range ? (vocab + 7) & ~7 : range;
    const int held = history_width < logits::kHeld ? history_width : logits::kHeld;
    const int smem = counts ? cells * (narrow ? 2 : 4) + held * 8 : 0;
    bool& done = configured[4 + 2 * dtype + narrow][dev < kMaxDevices ? dev : 0];
    if (dev >= kMaxDevices || !done) {
      AJB_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, logits::kMendRange * 2 + logits::kHeld * 8));
      AJB_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
      if (dev < kMaxDevices) done = true;
    }
    return launch_early(kernel, dim3(rows), dim3(logits::kMendThreads), smem, s, p);
  }
  // A piece of a row per CTA: large, because every piece looks at the row's whole history, but not larger than leaves three
  // for each SM (48 x 128256 with two: 16.6 us, with three: 13.9 us; 16 x 128256 with eight: 10.5 us, with three: 5.7 us).
  int chunk = narrow ? logits::Table<true>::kMaxChunk : logits::Table<false>::kMaxChunk;
  while (chunk > 1024 && (long long)rows * ((vocab + chunk - 1) / chunk) < 3ll * sm_count()) chunk >>= 1;
  p.chunk = chunk;
  p.chunks = (vocab + chunk - 1) / chunk;
  const int smem = counts ? chunk * (narrow ? 2 : 4) : 0;
  const int grid = rows * p.chunks, threads = logits::kStreamThreads + (counts ? logits::kHistoryThreads : 0);
  auto kernel = dtype == 0 ? (narrow ? logits::process_logits_kernel<__nv_bfloat16, true> : logits::process_logits_kernel<__nv_bfloat16, false>)
                           : (narrow ? logits::process_logits_kernel<float, true> : logits::process_logits_kernel<float, false>);
  return launch_early(kernel, dim3(grid), dim3(threads), smem, s, p);
}
