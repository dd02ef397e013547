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
// first streams its piece of the row through (widen, mask), then mends those tokens one by one: it has counted the
// history tokens of its piece in a table in shared memory, and the thread that takes a token's count out of the table
// (an exchange with 0) is the one that writes that token. Counts are whole numbers, so the order of the additions does
// not show. Biases follow in list order within one warp; lanes that hold the same token take turns.
#include "common.cuh"

namespace ajb {
namespace logits {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;
constexpr unsigned kInPrompt = 0x80000000u;      // table entry: bit 31 = in the prompt, the rest = times generated

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
__device__ __forceinline__ uint4 load4(const float* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
__device__ __forceinline__ uint4 load4(const __nv_bfloat16* p) {
  const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
  return make_uint4(v.x << 16, v.x & 0xffff0000u, v.y << 16, v.y & 0xffff0000u);
}

constexpr unsigned kMinusInf = 0xff800000u;

template <typename T>
__global__ void __launch_bounds__(kThreads) process_logits_kernel(const Params p) {
  extern __shared__ unsigned table[];
  const int row = (int)(blockIdx.x / (unsigned)p.chunks), part = (int)(blockIdx.x % (unsigned)p.chunks);
  const int lo = part * p.chunk, hi = min(p.vocab, lo + p.chunk);
  const T* in = reinterpret_cast<const T*>(p.in) + (size_t)row * p.in_pitch;
  float* out = p.out + (size_t)row * p.vocab;
  const unsigned* mask = p.mask != nullptr ? p.mask + (size_t)row * p.mask_pitch : nullptr;
  const int* history = p.history != nullptr ? p.history + (size_t)row * p.history_pitch : nullptr;
  const int len = history != nullptr ? min(max(p.history_lens[row], 0), p.history_width) : 0;

  if (len > 0) {
    for (int i = threadIdx.x; i < (p.chunk >> 2); i += kThreads) reinterpret_cast<uint4*>(table)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const int prompt = p.prompt_lens[row];
    for (int i = threadIdx.x; i < len; i += kThreads) {
      const int v = __ldg(history + i);
      if (v >= lo && v < hi) {
        if (i < prompt) atomicOr(&table[v - lo], kInPrompt);
        else atomicAdd(&table[v - lo], 1u);
      }
    }
  }

  // ---- the whole piece: widen and mask
  {
    // four-token groups start where `out` is 16-byte aligned; the input rows have to agree with that to be read in groups
    const int lead = (int)((4 - ((reinterpret_cast<uintptr_t>(out + lo) >> 2) & 3)) & 3);
    const int first = min(hi, lo + lead);
    const bool wide = (reinterpret_cast<uintptr_t>(in + lo + lead) & (4 * sizeof(T) - 1)) == 0;
    auto one = [&](int v) {
      const bool open = mask == nullptr || ((__ldg(mask + (v >> 5)) >> (v & 31)) & 1u);
      out[v] = open ? load1<T>(in + v) : __uint_as_float(kMinusInf);
    };
    if (wide) {
      for (int v = lo + (int)threadIdx.x; v < first; v += kThreads) one(v);
      const int groups = (hi - first) >> 2;
      for (int g0 = threadIdx.x; g0 < groups; g0 += kThreads * kUnroll) {
        unsigned open[kUnroll];
        uint4 x[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int g = g0 + u * kThreads, v = first + 4 * g;
          open[u] = g < groups ? 15u : 0u;
          if (mask != nullptr && g < groups) {
            // a group lies in one word, or in two neighbours when the row does not start on a 16-byte boundary
            const unsigned w0 = __ldg(mask + (v >> 5)), w1 = (v & 31) > 28 ? __ldg(mask + (v >> 5) + 1) : 0u;
            open[u] = __funnelshift_r(w0, w1, v & 31) & 15u;
          }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          x[u] = make_uint4(kMinusInf, kMinusInf, kMinusInf, kMinusInf);
          if (open[u]) x[u] = load4(in + first + 4 * (g0 + u * kThreads));
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int g = g0 + u * kThreads;
          if (g < groups) {
            if (!(open[u] & 1u)) x[u].x = kMinusInf;
            if (!(open[u] & 2u)) x[u].y = kMinusInf;
            if (!(open[u] & 4u)) x[u].z = kMinusInf;
            if (!(open[u] & 8u)) x[u].w = kMinusInf;
            *reinterpret_cast<uint4*>(out + first + 4 * g) = x[u];
          }
        }
      }
      for (int v = first + 4 * groups + (int)threadIdx.x; v < hi; v += kThreads) one(v);
    } else {
      for (int v = lo + (int)threadIdx.x; v < hi; v += kThreads) one(v);
    }
  }

  // ---- tokens of the history
  if (len > 0) {
    __syncthreads();
    const float r = p.repetition != nullptr ? p.repetition[row] : 1.0f;
    const float pr = p.presence != nullptr ? p.presence[row] : 0.0f;
    const float f = p.frequency != nullptr ? p.frequency[row] : 0.0f;
    for (int i = threadIdx.x; i < len; i += kThreads) {
      const int v = __ldg(history + i);
      if (v < lo || v >= hi) continue;
      const unsigned held = atomicExch(&table[v - lo], 0u);
      if (held == 0u || (mask != nullptr && !((__ldg(mask + (v >> 5)) >> (v & 31)) & 1u))) continue;
      float x = load1<T>(in + v);
      x = x > 0.0f ? __fdiv_rn(x, r) : __fmul_rn(x, r);
      const unsigned count = held & ~kInPrompt;
      x = __fsub_rn(x, __fmul_rn(f, (float)count));
      x = __fsub_rn(x, count > 0u ? pr : 0.0f);
      out[v] = x;
    }
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
        const bool mine = v >= lo && v < hi && (mask == nullptr || ((__ldg(mask + (v >> 5)) >> (v & 31)) & 1u));
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
  int chunk = 8192;
  while (chunk > 1024 && (long long)rows * ((vocab + chunk - 1) / chunk) < 2ll * sm_count()) chunk >>= 1;
  p.chunk = chunk;
  p.chunks = (vocab + chunk - 1) / chunk;
  AJB_REQUIRE((long long)rows * p.chunks <= 0x7fffffffll, "process logits: %d rows of %d tokens are too many", rows, vocab);
  const int smem = history != nullptr ? chunk * (int)sizeof(unsigned) : 0;
  const int grid = rows * p.chunks;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == 0) logits::process_logits_kernel<__nv_bfloat16><<<grid, logits::kThreads, smem, s>>>(p);
  else logits::process_logits_kernel<float><<<grid, logits::kThreads, smem, s>>>(p);
  AJB_CUDA_OK(cudaGetLastError());
  return 0;
}
