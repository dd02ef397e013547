// Logits processing ahead of the sampler: penalties for repeated tokens, token biases and grammar bit masks, from bf16 or
// fp32 logits to fp32 logits in one launch.
//
// For token v of a row, c(v) = how often it was generated, seen(v) = whether it is anywhere in the history (prompt and
// generated tokens), r / p / f = the row's repetition, presence and frequency penalty:
//   x = logit;  x = seen ? (x > 0 ? x / r : x * r) : x;  x = x - f * c - p * (c > 0);  x = x + bias;  x = masked ? -inf : x
// Every step rounds to fp32 once and nothing is contracted, so the result equals elementary fp32 operations bit for bit.
//
// Bound by memory: 6 bytes per bf16 logit (read, write) and a bit of the mask; where a mask shuts four neighbouring
// tokens their logits are not read. Only the few tokens of the history and of the bias list need arithmetic, so a CTA
// streams its piece of the row through (widen, mask) and then mends those tokens one by one. Four more warps count the
// history tokens of the piece in a table in shared memory while the others stream, so that neither waits for the other;
// the thread that then takes a token's count out of the table (an atomic that leaves 0) is the one that writes that
// token. Counts are whole numbers, so the order of the additions does not show. Biases follow in list order within one
// warp; lanes that hold the same token take turns.
#include "common.cuh"

namespace ajb {
namespace logits {

constexpr int kStreamThreads = 256;
constexpr int kHistoryThreads = 128;             // launched in addition when there is a history
constexpr int kUnroll = 4;
constexpr int kHistoryUnroll = 4;
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
  int chunk, chunks;             // tokens per CTA (a multiple of 32), CTAs per row
};

template <typename T>
__device__ __forceinline__ float load1(const T* p);
template <>
__device__ __forceinline__ float load1<float>(const float* p) { return __ldg(p); }
template <>
__device__ __forceinline__ float load1<__nv_bfloat16>(const __nv_bfloat16* p) {
  return __uint_as_float((unsigned)__ldg(reinterpret_cast<const unsigned short*>(p)) << 16);
}
// four neighbouring logits, as loaded and as fp32 bits
template <typename T>
struct Four;
template <>
struct Four<float> {
  uint4 v;
  __device__ __forceinline__ void load(const float* p) { v = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ uint4 wide() const { return v; }
};
template <>
struct Four<__nv_bfloat16> {
  uint2 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = __ldg(reinterpret_cast<const uint2*>(p)); }
  __device__ __forceinline__ uint4 wide() const { return make_uint4(v.x << 16, v.x & 0xffff0000u, v.y << 16, v.y & 0xffff0000u); }
};

__device__ __forceinline__ bool open_token(const unsigned* mask, int v) {
  return mask == nullptr || ((__ldg(mask + (v >> 5)) >> (v & 31)) & 1u);
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
        const unsigned w0 = __ldg(mask + (v >> 5)), w1 = (v & 31) > 28 ? __ldg(mask + (v >> 5) + 1) : 0u;
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
      v[u] = i < len ? __ldg(history + i) : -1;
    }
#pragma unroll
    for (int u = 0; u < kHistoryUnroll; ++u)
      if (v[u] >= lo && v[u] < hi) visit(i0 + u * threads, v[u]);
  }
}

template <typename T, bool kNarrow>
__global__ void __launch_bounds__(kStreamThreads + kHistoryThreads) process_logits_kernel(const Params p) {
  extern __shared__ unsigned table[];
  using Tab = Table<kNarrow>;
  const int row = (int)(blockIdx.x / (unsigned)p.chunks), part = (int)(blockIdx.x % (unsigned)p.chunks);
  const int lo = part * p.chunk, hi = min(p.vocab, lo + p.chunk);
  const T* in = reinterpret_cast<const T*>(p.in) + (size_t)row * p.in_pitch;
  float* out = p.out + (size_t)row * p.vocab;
  const unsigned* mask = p.mask != nullptr ? p.mask + (size_t)row * p.mask_pitch : nullptr;
  const int* history = p.history != nullptr ? p.history + (size_t)row * p.history_pitch : nullptr;
  const int thread = threadIdx.x;
  int len = 0;

  if (history != nullptr) len = min(max(p.history_lens[row], 0), p.history_width);
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
    const float r = p.repetition != nullptr ? p.repetition[row] : 1.0f;
    const float pr = p.presence != nullptr ? p.presence[row] : 0.0f;
    const float f = p.frequency != nullptr ? p.frequency[row] : 0.0f;
    for_history(history, len, lo, hi, thread, kStreamThreads + kHistoryThreads, [&](int, int v) {
      const unsigned held = Tab::take(table, v - lo);
      if (held == 0u || !open_token(mask, v)) return;
      float x = load1<T>(in + v);
      x = x > 0.0f ? __fdiv_rn(x, r) : __fmul_rn(x, r);
      const unsigned count = held & ~Tab::kPrompt;
      x = __fsub_rn(x, __fmul_rn(f, (float)count));
      out[v] = __fsub_rn(x, count > 0u ? pr : 0.0f);
    });
  }

  // ---- biases
  if (p.biases > 0) {
    __syncthreads();
    if (threadIdx.x < 32) {
      const int* ids = p.bias_ids + (size_t)row * p.biases;
      const float* values = p.bias_values + (size_t)row * p.biases;
      for (int base = 0; base < p.biases; base += 32) {
        const int i = base + (int)threadIdx.x;
        const int v = i < p.biases ? __ldg(ids + i) : -1;
        const bool mine = v >= lo && v < hi && open_token(mask, v);
        // turn of this lane among the lanes with the same token
        const unsigned same = __match_any_sync(0xffffffffu, mine ? v : -1);
        const int turn = __popc(same & ((1u << threadIdx.x) - 1u));
        int turns = mine ? __popc(same) : 0;
        turns = __reduce_max_sync(0xffffffffu, turns);
        for (int k = 0; k < turns; ++k) {
          if (mine && turn == k) {
            volatile float* at = out + v;
            *at = __fadd_rn(*at, __ldg(values + i));
          }
          __syncwarp();
        }
      }
    }
  }
}

}  // namespace logits
}  // namespace ajb

// logits [rows, vocab] (dtype 0: bf16, 1: fp32) with in_pitch elements between rows; out fp32 [rows, vocab] contiguous,
// not overlapping the logits. Null pointers switch the parts off: history (with lens), repetition / presence /
// frequency, bias_ids (biases = 0), mask.
extern "C" int ajb_process_logits(const void* logits, int dtype, long long in_pitch, void* out, int rows, int vocab,
                                  const void* history, long long history_pitch, int history_width, const void* prompt_lens,
                                  const void* history_lens, const void* repetition, const void* presence,
                                  const void* frequency, const void* bias_ids, const void* bias_values, int biases,
                                  const void* mask, long long mask_pitch, void* stream) {
  using namespace ajb;
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
  // a piece of a row per CTA: large, because every piece looks at the row's whole history, but not larger than leaves
  // two CTAs for each SM
  const bool counts = history != nullptr && history_width > 0, narrow = history_width <= 32767;
  int chunk = narrow ? logits::Table<true>::kMaxChunk : logits::Table<false>::kMaxChunk;
  while (chunk > 1024 && (long long)rows * ((vocab + chunk - 1) / chunk) < 2ll * sm_count()) chunk >>= 1;
  p.chunk = chunk;
  p.chunks = (vocab + chunk - 1) / chunk;
  AJB_REQUIRE((long long)rows * p.chunks <= 0x7fffffffll, "process logits: %d rows of %d tokens are too many", rows, vocab);
  if (!counts) p.history = nullptr;
  const int smem = counts ? chunk * (narrow ? 2 : 4) : 0;
  const int grid = rows * p.chunks, threads = logits::kStreamThreads + (counts ? logits::kHistoryThreads : 0);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == 0 && narrow) logits::process_logits_kernel<__nv_bfloat16, true><<<grid, threads, smem, s>>>(p);
  else if (dtype == 0) logits::process_logits_kernel<__nv_bfloat16, false><<<grid, threads, smem, s>>>(p);
  else if (narrow) logits::process_logits_kernel<float, true><<<grid, threads, smem, s>>>(p);
  else logits::process_logits_kernel<float, false><<<grid, threads, smem, s>>>(p);
  AJB_CUDA_OK(cudaGetLastError());
  return 0;
}
