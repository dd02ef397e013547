// Paged-KV attention for decoding and speculative verification on sm_100a.
//
// A CTA's piece of work is a (sequence, KV head), or a share of its keys: the `group * q_len` query rows that share this
// KV head (group = Hq / Hkv query heads, q_len new tokens: 1 for plain decoding, k + 1 when verifying k draft tokens) are
// worked on together, so every K/V byte of the sequence is read once for all of them, in tiles of keys that TMA fetches
// block by block (16 tokens, addressed through the block table). S = Q K^T and O += P V run on the tensor cores with
// accumulators in tensor memory, the softmax between them in registers with fp32 maxima and sums; probabilities are rounded
// to bf16 as the operand of the second product, whose other operand, the cached values, is bf16 too. Row (head h, new token
// i) may see keys 0 .. context_len - q_len + i.
//
// The caches are streamed once with little arithmetic per byte, so the bytes in flight per SM and the length of a step's
// dependent chain (wait for the tile, one product, a softmax over it, a second product) decide. There are two kernels, by
// query rows per piece, with two CTAs per SM so that one's chain hides behind the other's loads (one for 17 to 32 rows of 128):
//   up to 32 (paged_decode_kernel): keys on the 128-row side of the tensor-core tile, 128 of them per step;
//   more (paged_attention_kernel): query rows on it, 64 keys per step.
// 256 sequences of 1280 tokens, 8 KV heads of 128, 4 rows each: 191 us, 7.0 TB/s; 16 sequences of 1000: 15.7 us.
//
// Long contexts at small batch: with `splits` > 1 the tiles of a sequence are divided over that many pieces. Each leaves
// its un-normalised fp32 output rows and (reference maximum, row sum) in a workspace, and a second small kernel joins them
// with the usual log-sum-exp weights.
//
// Layouts: q [tokens, Hq, hd] bf16 (rows of a sequence are contiguous, `q_start[seq]` is its first row); caches
// [num_blocks, block_size = 16, Hkv, hd] bf16; block_tables [num_seqs, max_blocks] int32; out like q.
//
// Behind a shared prefix (csrc/prefix_attention.cu) the kernels cover the rest of every sequence: they start at key
// `first_key` and always leave un-normalised parts, and sequences with more query rows than one CTA holds are cut into
// `chunks` of q_len tokens each. paged_decode_kernel may take the prefix itself along, in pieces for rows of several
// sequences.
#include "common.cuh"
#include "paged_attention.h"

namespace ajb {
namespace paged {

constexpr int TILE = 64;           // keys per step
constexpr int QROWS = 128;         // rows of the query / probability operand tiles (the MMA's M)
constexpr int BLOCK_TOKENS = 16;   // tokens per cache block
constexpr int kThreads = 192;
constexpr int kMaxRows = 64;       // group * q_len of ajb_paged_attention
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kPagedKernelId = 5;

template <int HD>
struct Cfg {
  static constexpr int kQ = QROWS * HD * 2;          // the query rows, staged once
  static constexpr int kTile = TILE * HD * 2;        // one K or V tile
  static constexpr int kP = QROWS * TILE * 2;        // probabilities of one step (A operand of P V)
  static constexpr int kSmem = kQ + 4 * kTile /*2 x (K,V)*/ + kP + 256;
  static constexpr int kOCol = 2 * TILE;             // S0 at 0, S1 at TILE, O behind them
  static constexpr int kTmemCols = 256;              // 2 * 64 + HD <= 256: two CTAs fit the SM's 512 columns
};

struct Params {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  const int* block_tables;
  const int* context_lens;
  const int* q_start;         // null: sequence i's rows start at i * q_total
  long long q_pitch;          // elements between the rows of two tokens in q
  int max_blocks;
  int heads, kv_heads, group, q_len;
  int seqs, chunks;           // sequences; CTAs that a sequence's new tokens are cut over
  int q_total;                // new tokens per sequence; q_len of them are a CTA's, chunk after chunk
  int first_key;              // first cached token this launch looks at (a multiple of the block size)
  float scale;
  int splits;                 // CTAs per (sequence, KV head, chunk)
  int prefix_splits;          // divisions of the keys in front of first_key (0: not covered); their CTAs are ahead of the others
  int prefix_tokens;          // query tokens that one of these CTAs takes
  int prefix_pieces;          // and how many of them a KV head's query tokens are
  int early;                  // this launch may have started before the one in front of it ended: wait for that first
  int part_stride, part_base; // parts per row in the workspace and the first one of this launch; part_stride 0: no parts
  float* part_o;              // [tokens, Hq, part_stride, hd] fp32, un-normalised
  float2* part_ml;            // [tokens, Hq, part_stride] (reference maximum in log2 units, row sum); sum 0 = no keys seen
  DeviceStatus* status;
};

// Rows [first, TILE) of a V tile become zero: they belong to no key (the unused end of the last block, or a block fetched
// again to fill the tile), their probabilities are zero, and zero times whatever an old sequence left there (an
// infinity, a NaN) must not reach the sums. `t` is the caller's index among the 128 threads that share the work.
template <int HD>
__device__ __forceinline__ void zero_value_rows(uint8_t* tile, int first, int t) {
  for (int i = first * 8 + t; i < TILE * 8; i += 128) {
#pragma unroll
    for (int b = 0; b < HD / 64; ++b) reinterpret_cast<uint4*>(tile + b * (TILE * 128))[i] = make_uint4(0, 0, 0, 0);
  }
}

// 16-byte chunk `ch` of row `row` of a K-major operand tile of QROWS rows (128-byte swizzle, 64-element boxes).
__device__ __forceinline__ void store_chunk(uint8_t* tile, int row, int ch, uint4 val) {
  uint8_t* dst = tile + (ch >> 3) * (QROWS * 128) + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
  *reinterpret_cast<uint4*>(dst) = val;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 2)
paged_attention_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const Params p) {
  using C = Cfg<HD>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw;
  uint8_t* sQ = smem;
  uint8_t* sP = sQ + C::kQ;
  uint8_t* sKV = sP + C::kP;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + 4 * C::kTile);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (smem_misaligned(smem, p.status, kPagedKernelId, reinterpret_cast<uint32_t*>(bars) + 60)) return;
  // K and V tiles have their own barriers: a K tile is free again after the first product of its step, long before
  // the V tile of the same step, and the issuing warp must never find the next K tile missing when it gets there
  uint64_t* k_full = bars;         // 2
  uint64_t* k_empty = bars + 2;    // 2
  uint64_t* v_full = bars + 4;     // 2
  uint64_t* v_empty = bars + 6;    // 2
  uint64_t* s_full = bars + 8;     // 2
  uint64_t* s_free = bars + 10;    // 2
  uint64_t* p_ready = bars + 12;   // 1
  uint64_t* pv_done = bars + 13;   // 1
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 14);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int seq = blockIdx.x, kv_head = (int)blockIdx.y % p.kv_heads;
  const int group = p.heads / p.kv_heads;
  const int q0 = ((int)blockIdx.y / p.kv_heads) * p.q_len;          // first of this CTA's new tokens
  const int q_len = min(p.q_len, p.q_total - q0);
  const int rows = group * q_len;                   // real rows, packed head-major: row = h_in_group * q_len + i
  const int token0 = (p.q_start != nullptr ? p.q_start[seq] : seq * p.q_total) + q0;
  // keys are counted from first_key; the block table bounds them whatever the context length says
  const int ctx = p.context_lens[seq] - (p.q_total - q0 - q_len) - p.first_key;
  const int keys = min(max(ctx, 0), p.max_blocks * BLOCK_TOKENS - p.first_key);
  const int all_tiles = (keys + TILE - 1) / TILE;
  // this CTA's share of the sequence's tiles: [t0, t0 + n_tiles)
  const int per_split = (all_tiles + p.splits - 1) / p.splits;
  const int t0 = min(all_tiles, (int)blockIdx.z * per_split);
  const int n_tiles = min(all_tiles - t0, per_split);
  const int active_quarters = (rows + 31) / 32;
  // the tile that the last key does not fill, if it is this CTA's (always its last one)
  const int ragged_tile = (keys % TILE != 0 && n_tiles > 0 && t0 + n_tiles == all_tiles) ? n_tiles - 1 : -1;
  const int* table = p.block_tables + (size_t)seq * p.max_blocks + p.first_key / BLOCK_TOKENS;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);
    }
    mbar_init(p_ready, 4);
    mbar_init(pv_done, 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tensor_map(&map_k);
    prefetch_tensor_map(&map_v);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  // stage Q: rows beyond `rows` are zero (their scores are never used)
  if (warp >= 2) {
    const int t = threadIdx.x - 64;                 // 0..127 == tile row
    const bool real = t < rows;
    const int h = real ? t / q_len : 0, i = real ? t % q_len : 0;
    const __nv_bfloat16* src = p.q + (size_t)(token0 + i) * p.q_pitch + (size_t)(kv_head * group + h) * HD;
#pragma unroll
    for (int ch = 0; ch < HD / 8; ++ch) {
      const uint4 v = real ? reinterpret_cast<const uint4*>(src)[ch] : make_uint4(0, 0, 0, 0);
      store_chunk(sQ, t, ch, v);
    }
    fence_proxy_async_smem();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // Producer. The block ids of eight tiles (32 blocks) are fetched by the 32 lanes with one coalesced load, a group
    // ahead of their use, and handed to the issuing lane by shuffles: a dependent table lookup per block in front of
    // its copies would cost more than the copies themselves.
    constexpr int kBlocksPerTile = TILE / BLOCK_TOKENS;
    constexpr int kTilesPerGroup = 32 / kBlocksPerTile;
    const int last_block = (keys + BLOCK_TOKENS - 1) / BLOCK_TOKENS - 1;
    // blocks past the end of the sequence re-read the last valid block (masked later); keeps the byte count fixed
    auto fetch_ids = [&](int group) { return table[max(0, min(last_block, (t0 + group * kTilesPerGroup) * kBlocksPerTile + lane))]; };
    int ids_next = n_tiles > 0 ? fetch_ids(0) : 0;
    bool ok = true;
    // K tiles run one step ahead of V tiles: K(j + 1) goes out as soon as the first product of step j - 1 has read
    // its slot, V(j) when the second product of step j - 2 has
    int ids_k = ids_next, ids_prev = ids_next;      // block ids of K's group of tiles and of the group before it
    int k_group = -1;
    for (int j = 0; j <= n_tiles && ok; ++j) {
      if (j < n_tiles) {
        if (j % kTilesPerGroup == 0) {
          ids_prev = ids_k;
          ids_k = ids_next;
          k_group = j / kTilesPerGroup;
          if (j + kTilesPerGroup < n_tiles) ids_next = fetch_ids(k_group + 1);
        }
        const int s = j & 1;
        int id[kBlocksPerTile];
#pragma unroll
        for (int b = 0; b < kBlocksPerTile; ++b) id[b] = __shfl_sync(0xffffffffu, ids_k, (j % kTilesPerGroup) * kBlocksPerTile + b);
        if (lane == 0) {
          ok = mbar_wait(&k_empty[s], (((uint32_t)j >> 1) & 1) ^ 1, abort_flag, p.status, kPagedKernelId, 1);
          if (ok) {
            uint8_t* sK = sKV + s * 2 * C::kTile;
            mbar_arrive_expect_tx(&k_full[s], C::kTile);
#pragma unroll
            for (int b = 0; b < kBlocksPerTile; ++b) {
#pragma unroll
              for (int i = 0; i < HD / 64; ++i)
                tma_load_3d(sK + i * (TILE * 128) + b * (BLOCK_TOKENS * 128), &map_k, &k_full[s], kv_head * HD + 64 * i, 0, id[b]);
            }
          }
        }
      }
      if (j >= 1) {
        const int jv = j - 1;
        const int ids_v = (jv / kTilesPerGroup == k_group) ? ids_k : ids_prev;     // V is one step behind K
        const int s = jv & 1;
        int id[kBlocksPerTile];
#pragma unroll
        for (int b = 0; b < kBlocksPerTile; ++b) id[b] = __shfl_sync(0xffffffffu, ids_v, (jv % kTilesPerGroup) * kBlocksPerTile + b);
        if (lane == 0 && ok) {
          ok = mbar_wait(&v_empty[s], (((uint32_t)jv >> 1) & 1) ^ 1, abort_flag, p.status, kPagedKernelId, 2);
          if (ok) {
            uint8_t* sV = sKV + s * 2 * C::kTile + C::kTile;
            mbar_arrive_expect_tx(&v_full[s], C::kTile);
#pragma unroll
            for (int b = 0; b < kBlocksPerTile; ++b) {
#pragma unroll
              for (int i = 0; i < HD / 64; ++i)
                tma_load_3d(sV + i * (TILE * 128) + b * (BLOCK_TOKENS * 128), &map_v, &v_full[s], kv_head * HD + 64 * i, 0, id[b]);
            }
          }
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc_s = make_idesc(QROWS, TILE, 1, false, false);
    constexpr uint32_t idesc_o = make_idesc(QROWS, HD, 1, false, true);
    // descriptor low words; a k-step is a compile-time offset added to one of these (see common.cuh)
    const uint32_t q_km = desc_lo_k_major(smem_u32(sQ)), p_km = desc_lo_k_major(smem_u32(sP));
    const uint32_t k_km0 = desc_lo_k_major(smem_u32(sKV));
    const uint32_t v_mn0 = desc_lo_mn_major(smem_u32(sKV) + C::kTile, TILE * 128);
    constexpr uint32_t kStageStep = (2 * C::kTile) >> 4;
    bool ok = true;
    auto issue_s = [&](int j) -> bool {
      const int s = j & 1;
      const uint32_t use = (uint32_t)j >> 1;
      if (!mbar_wait(&k_full[s], use & 1, abort_flag, p.status, kPagedKernelId, 3)) return false;
      if (!mbar_wait(&s_free[s], (use & 1) ^ 1, abort_flag, p.status, kPagedKernelId, 4)) return false;
      tc_fence_after_sync();
      if (lane == 0) {
        const uint32_t k_km = k_km0 + (uint32_t)s * kStageStep;
        const uint32_t d = tmem_base + (uint32_t)(s * TILE);
        umma_f16_c<false>(d, desc_at(q_km, 0), desc_at(k_km, 0), idesc_s);
#pragma unroll
        for (int k = 1; k < HD / 16; ++k)
          umma_f16_c<true>(d, desc_at(q_km, k_major_step(k, QROWS * 128)), desc_at(k_km, k_major_step(k, TILE * 128)), idesc_s);
        tc_commit(&s_full[s]);
        tc_commit(&k_empty[s]);
      }
      __syncwarp();
      return true;
    };
    if (n_tiles > 0) ok = issue_s(0);
    for (int j = 0; j < n_tiles && ok; ++j) {
      if (j + 1 < n_tiles) {
        ok = issue_s(j + 1);
        if (!ok) break;
      }
      if (!mbar_wait(p_ready, (uint32_t)j & 1, abort_flag, p.status, kPagedKernelId, 5)) { ok = false; break; }
      if (!mbar_wait(&v_full[j & 1], ((uint32_t)j >> 1) & 1, abort_flag, p.status, kPagedKernelId, 10)) { ok = false; break; }
      tc_fence_after_sync();
      if (lane == 0) {
        const uint32_t v_mn = v_mn0 + (uint32_t)(j & 1) * kStageStep;
        umma_f16(tmem_base + C::kOCol, desc_at(p_km, 0), desc_at(v_mn, 0), idesc_o, j != 0);
#pragma unroll
        for (int k = 1; k < TILE / 16; ++k)
          umma_f16_c<true>(tmem_base + C::kOCol, desc_at(p_km, k_major_step(k, QROWS * 128)), desc_at(v_mn, mn_major_step(k)), idesc_o);
        tc_commit(pv_done);
        tc_commit(&v_empty[j & 1]);
      }
      __syncwarp();
    }
  } else {
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const bool active = quarter < active_quarters;     // warp-uniform
    const bool real = row < rows;
    const int h = real ? row / q_len : 0, qi = real ? row % q_len : 0;
    const int k_max = real ? min(ctx - q_len + qi, keys - 1) : -1;   // last visible key
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const float sl = p.scale * kLog2e;
    float m_run = -INFINITY, l_run = 0.0f;
    bool ok = true;
    for (int j = 0; j < n_tiles && ok; ++j) {
      const int s = j & 1;
      if (!mbar_wait(&s_full[s], ((uint32_t)j >> 1) & 1, abort_flag, p.status, kPagedKernelId, 6)) { ok = false; break; }
      tc_fence_after_sync();
      const int k0 = (t0 + j) * TILE;
      uint32_t pk[TILE / 2];
      float alpha = 1.0f;
      bool moved = false;
      if (active) {
        uint32_t sv[TILE / 32][32];
#pragma unroll
        for (int c = 0; c < TILE / 32; ++c) tmem_ld_32x32(tmem_base + lane_addr + (uint32_t)(s * TILE + c * 32), sv[c]);
        tc_wait_ld();
        float m_tile = -INFINITY;
#pragma unroll
        for (int c = 0; c < TILE / 32; ++c) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float x = __uint_as_float(sv[c][i]);
            if (k0 + c * 32 + i > k_max) x = -INFINITY;
            sv[c][i] = __float_as_uint(x);
            m_tile = fmaxf(m_tile, x);
          }
        }
        // lazy reference maximum (see flash_fwd.cu): O is rescaled only when a row would overflow 2^8
        moved = (m_tile - m_run) * sl > 8.0f;
        const float m_new = moved ? m_tile : m_run;
        const float m_safe = (m_new == -INFINITY) ? 0.0f : m_new;
        alpha = moved ? exp2f((m_run - m_safe) * sl) : 1.0f;
        const float neg = -m_safe * sl;
        float l_tile = 0.0f;
#pragma unroll
        for (int c = 0; c < TILE / 32; ++c) {
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float p0 = exp2f(fmaf(__uint_as_float(sv[c][i]), sl, neg));
            const float p1 = exp2f(fmaf(__uint_as_float(sv[c][i + 1]), sl, neg));
            l_tile += p0 + p1;
            pk[c * 16 + i / 2] = pack_bf16x2(p0, p1);
          }
        }
        l_run = l_run * alpha + l_tile;
        m_run = m_new;
      } else {
#pragma unroll
        for (int i = 0; i < TILE / 2; ++i) pk[i] = 0u;
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_free[s]);
      if (j > 0 && !mbar_wait(pv_done, (uint32_t)(j - 1) & 1, abort_flag, p.status, kPagedKernelId, 7)) { ok = false; break; }
      tc_fence_after_sync();
      // inactive quarters write their (zero) rows only once: they never change
      if (active || j == 0) {
#pragma unroll
        for (int ch = 0; ch < TILE / 8; ++ch) store_chunk(sP, row, ch, make_uint4(pk[ch * 4], pk[ch * 4 + 1], pk[ch * 4 + 2], pk[ch * 4 + 3]));
      }
      if (ragged_tile == j) {
        if (!mbar_wait(&v_full[s], ((uint32_t)j >> 1) & 1, abort_flag, p.status, kPagedKernelId, 11)) { ok = false; break; }
        zero_value_rows<HD>(sKV + s * 2 * C::kTile + C::kTile, keys - (t0 + j) * TILE, quarter * 32 + lane);
      }
      if (active && j > 0 && __any_sync(0xffffffffu, moved)) {
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t ov[32];
          tmem_ld_32x32(tmem_base + lane_addr + (uint32_t)(C::kOCol + c * 32), ov);
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
          tmem_st_32x32(tmem_base + lane_addr + (uint32_t)(C::kOCol + c * 32), ov);
        }
        tc_wait_st();
      }
      fence_proxy_async_smem();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready);
    }
    const size_t out_row = (size_t)(token0 + qi) * p.heads + kv_head * group + h;
    const size_t part_row = out_row * p.part_stride + p.part_base + blockIdx.z;
    if (p.part_stride > 0 && real && (n_tiles == 0 || !ok))
      p.part_ml[part_row] = make_float2(0.0f, 0.0f);        // nothing to merge from this part
    if (ok && n_tiles > 0 && mbar_wait(pv_done, (uint32_t)(n_tiles - 1) & 1, abort_flag, p.status, kPagedKernelId, 8)) {
      tc_fence_after_sync();
      if (active && p.part_stride > 0) {
        if (real) p.part_ml[part_row] = make_float2(m_run == -INFINITY ? 0.0f : m_run * sl, l_run);
        float* part = p.part_o + part_row * HD;
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t ov[32];
          tmem_ld_32x32(tmem_base + lane_addr + (uint32_t)(C::kOCol + c * 32), ov);
          tc_wait_ld();
          if (real) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              reinterpret_cast<uint4*>(part + c * 32)[i] = make_uint4(ov[4 * i], ov[4 * i + 1], ov[4 * i + 2], ov[4 * i + 3]);
          }
        }
      } else if (active) {
        const float inv_l = l_run > 0.0f ? 1.0f / l_run : 0.0f;
        __nv_bfloat16* dst = p.out + out_row * HD;
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t ov[32];
          tmem_ld_32x32(tmem_base + lane_addr + (uint32_t)(C::kOCol + c * 32), ov);
          tc_wait_ld();
          if (real) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint4 q;
              q.x = pack_bf16x2(__uint_as_float(ov[8 * i]) * inv_l, __uint_as_float(ov[8 * i + 1]) * inv_l);
              q.y = pack_bf16x2(__uint_as_float(ov[8 * i + 2]) * inv_l, __uint_as_float(ov[8 * i + 3]) * inv_l);
              q.z = pack_bf16x2(__uint_as_float(ov[8 * i + 4]) * inv_l, __uint_as_float(ov[8 * i + 5]) * inv_l);
              q.w = pack_bf16x2(__uint_as_float(ov[8 * i + 6]) * inv_l, __uint_as_float(ov[8 * i + 7]) * inv_l);
              reinterpret_cast<uint4*>(dst + c * 32)[i] = q;
            }
          }
        }
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
  // a launch that joins the parts waits for this one only: this one does not end before the launch in front of it has
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---------------------------------------------------------------------------------------------------------------------
// At most 32 query rows per (sequence, KV head, part): the work of plain decoding, and of verifying a few tokens.
//
// Keys and head dimension fill the 128-row side of the tensor-core tile, the few query rows the narrow one:
//   S^T [128 keys, N] = K Q^T,   O^T [hd, N] += V^T P^T    (N = 16 or 32 rows, the real ones first)
// so a step reads every K and V byte from shared memory once and nothing else of size, each softmax thread owns one key
// and all its query rows (4 of 16 columns used in the worst ordinary case, instead of 4 of 128 rows), and what a CTA
// holds besides its ring of K and V tiles is a few KB. The row maxima of a tile are a warp reduction per query row and
// one exchange between the four warps; row sums stay in registers until the end.
//
// A CTA does not end with its first piece of work: while it computes, it takes over a CTA of the launch that has not
// started yet (the hardware gives out each exactly once, so sequences of any mix of lengths balance). Its producing warp
// runs on into the next piece's keys and values as ring slots fall free, the next piece's query rows are loaded while the
// last tile of the piece before is worked on, and barriers and tensor memory are set up once: tile, slot and exchange
// numbers simply count over all pieces.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int DTILE = 128;         // keys per step

template <int HD, int N>
struct DecodeCfg {
  static constexpr int kTile = DTILE * HD * 2;                    // one K or V tile
  static constexpr int kCtas = HD == 128 && N == 32 ? 1 : 2;      // per SM
  static constexpr int kSlots = HD == 64 ? 5 : kCtas == 2 ? 3 : 6;
  static constexpr int kQ = N * HD * 2;                           // query rows of a piece
  static constexpr int kP = N * DTILE * 2;                        // probabilities of a step; two of them
  static constexpr int kExchange = 4 * 4 * 32 * 4;                // [slot][warp][query row]
  // 64-wide heads: the product with V^T runs 128 rows high all the same, its second half reads the next 8-row groups (for
  // the last one: up to 1 KB behind the ring) into accumulator rows that nobody reads
  static constexpr int kSmem = kSlots * kTile + kQ + 2 * kP + kExchange + 512;
  // an SM has 228 KB, of which each CTA takes 1 KB more than it asks for
  static_assert(kCtas * (kSmem + 1024) <= 228 * 1024, "shared memory for the CTAs of an SM");
  static constexpr int kOCol = 2 * N;                             // S^T twice, O^T behind them
  static constexpr int kTmemCols = N == 16 ? 64 : 128;
};

// What one CTA of a launch does, from the coordinates that the grid gives it and the lengths behind them. The producing
// warp works it out once per piece (the divisions in it take longer than a tile's exponentials) and hands it to the
// other warps through shared memory.
struct Work {
  int n_tiles;          // of 128 keys; -1: no more work
  int t0;               // the first of them
  int kv_head, rows;    // real query rows, packed token by token: row = new token * group + head of the group
  int token0;           // the first new token
  int ctx;              // keys that the last new token sees; the others see one less each
  int keys;             // keys that there are (the block table bounds them whatever the context length says)
  int part;             // its place among the parts of a row
  __device__ __forceinline__ Work() {}
  __device__ __forceinline__ Work(const Params& p, int y, int z, int context, int first_token) {
    int chunk = 0;
    kv_head = y;
    if (p.chunks > 1) { chunk = y / p.kv_heads; kv_head = y - chunk * p.kv_heads; }
    const int q0 = chunk * p.q_len, q_len = min(p.q_len, p.q_total - q0);
    rows = p.group * q_len;
    token0 = first_token + q0;
    // keys are counted from first_key
    ctx = context - (p.q_total - q0 - q_len) - p.first_key;
    keys = min(max(ctx, 0), p.max_blocks * BLOCK_TOKENS - p.first_key);
    const int all_tiles = (keys + DTILE - 1) / DTILE;
    t0 = 0;
    n_tiles = all_tiles;
    if (p.splits > 1) {       // this CTA's share of the sequence's tiles
      const int per_split = (all_tiles + p.splits - 1) / p.splits;
      t0 = min(all_tiles, z * per_split);
      n_tiles = min(all_tiles - t0, per_split);
    }
    part = p.part_base + z;
  }
  __device__ __forceinline__ void store(int4* to) const {
    to[0] = make_int4(n_tiles, t0, kv_head, rows);
    to[1] = make_int4(token0, ctx, keys, part);
  }
  __device__ __forceinline__ void load(const int4* from) {
    const int4 a = from[0], b = from[1];
    n_tiles = a.x; t0 = a.y; kv_head = a.z; rows = a.w;
    token0 = b.x; ctx = b.y; keys = b.z; part = b.w;
  }
};

__device__ __forceinline__ float warp_max_f32(float x) {
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(x));
  return m;
}

template <int R>
__device__ __forceinline__ void tmem_ld_rows(uint32_t taddr, uint32_t (&r)[R]) {
  if constexpr (R == 4) tmem_ld_32x4(taddr, r);
  else if constexpr (R == 8) tmem_ld_32x8(taddr, r);
  else if constexpr (R == 16) tmem_ld_32x16(taddr, r);
  else tmem_ld_32x32(taddr, r);
}
template <int R>
__device__ __forceinline__ void tmem_st_rows(uint32_t taddr, const uint32_t (&r)[R]) {
  if constexpr (R == 4) tmem_st_32x4(taddr, r);
  else if constexpr (R == 8) tmem_st_32x8(taddr, r);
  else if constexpr (R == 16) tmem_st_32x16(taddr, r);
  else tmem_st_32x32(taddr, r);
}

// R: query rows that the softmax warps work on (the real ones rounded up to 4, 8, 16 or 32; what comes of the others is not
// used). A piece of work may be a single tile, so a warp walks through most of its code once per piece: the code is kept
// short (one place for each wait, load and product, rows as a template parameter instead of branches), as instruction
// fetches cost short contexts more than arithmetic (256 sequences x 32..512 keys: 80 us before, 60 % of the fetches hit; 20
// rows x 20 keys: 8.4 us with some 35 instructions per row, 5.9 us with some 20).
template <int HD, int R>
__global__ void __launch_bounds__(kThreads, (DecodeCfg<HD, (R < 16 ? 16 : R)>::kCtas))
paged_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params p) {
  constexpr int N = R < 16 ? 16 : R;
  using C = DecodeCfg<HD, N>;
  constexpr int kSlots = C::kSlots;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* ring = smem_raw;
  uint8_t* sQ = ring + kSlots * C::kTile;
  uint8_t* sP = sQ + C::kQ;
  float* sExchange = reinterpret_cast<float*>(sP + 2 * C::kP);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sP + 2 * C::kP + C::kExchange);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (p.early) asm volatile("griddepcontrol.wait;" ::: "memory");
  if (smem_misaligned(smem_raw, p.status, kPagedKernelId, reinterpret_cast<uint32_t*>(bars) + 120)) return;
  uint64_t* full = bars;           // kSlots (<= 6)
  uint64_t* empty = bars + 6;      // kSlots
  uint64_t* s_full = bars + 12;    // 2
  uint64_t* s_free = bars + 14;    // 2
  uint64_t* p_ready = bars + 16;   // 2
  uint64_t* pv_done = bars + 18;   // 2
  uint64_t* w_full = bars + 20;    // 2: a piece of work is announced
  uint64_t* w_empty = bars + 22;   // 2: and has been read by the five other warps
  uint64_t* q_ready = bars + 24;   // the query rows of a piece are staged
  uint64_t* xbar = bars + 25;      // the four softmax warps exchange maxima / sums
  uint64_t* taken = bars + 26;     // the answer about the next piece is there
  void* answer = bars + 28;                                     // 16 bytes
  int4* announced = reinterpret_cast<int4*>(bars + 30);         // 2 pieces of two words each
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 38);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto wait = [&](uint64_t* bar, uint32_t parity, int stage) {
    return mbar_wait_compact(bar, parity, abort_flag, p.status, kPagedKernelId, stage);
  };

  if (threadIdx.x == 0) {
#pragma unroll 1
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);
      mbar_init(&p_ready[i], 4);
      mbar_init(&pv_done[i], 1);
      mbar_init(&w_full[i], 1);
      mbar_init(&w_empty[i], 5);
    }
    mbar_init(q_ready, 4);
    mbar_init(xbar, 4);
    mbar_init(taken, 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tensor_map(&map_k);
    prefetch_tensor_map(&map_v);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  if (warp >= 2) {
    // query rows that no piece fills, and their probabilities, stay zero (or an earlier piece's): their columns of the
    // accumulators are never used
#pragma unroll 1
    for (int i = threadIdx.x - 64; i < (C::kQ + 2 * C::kP) / 16; i += 128) reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  // Tiles pass through the ring in the order K0 K1 V0 K2 V1 ... K(n-1) V(n-2) V(n-1): a K tile goes out a step ahead, as
  // its product is issued a step ahead. Number of a tile among its piece's 2 n:
  auto k_number = [](int j) { return j == 0 ? 0 : 2 * j - 1; };
  auto v_number = [](int j, int n) { return j < n - 1 ? 2 * j + 2 : 2 * n - 1; };

  if (warp == 0) {
    // Producer. The block ids of four tiles (32 blocks) are fetched by the 32 lanes with one coalesced load, a group
    // ahead of their use; for a tile, eight lanes then copy a block each.
    constexpr int kBlocksPerTile = DTILE / BLOCK_TOKENS;
    constexpr int kTilesPerGroup = 32 / kBlocksPerTile;
    const int first_block = p.first_key / BLOCK_TOKENS, table_end = p.max_blocks - 1;
    // The KV heads of a sequence are neighbours in the grid: their rows of a cache block are neighbours in memory, and
    // they are read at about the same time.
    const int columns = p.kv_heads * p.chunks, prefix_ctas = p.kv_heads * p.prefix_pieces * p.prefix_splits;
    int cta = blockIdx.x, ids_next = 0;
    bool ok = true, asked = false;
    uint32_t base = 0;                                // tiles of all pieces before this one, K and V counted
    uint32_t piece = 0;
#pragma unroll 1
    for (; ok; ++piece) {
      // ---- what the piece is
      Work w;
      int seq = 0, from_block = first_block;
      if (cta >= 0 && cta < prefix_ctas) {
        // keys that all sequences share, for as many of their query rows as the launch's CTAs hold
        from_block = 0;
        const int units = p.kv_heads * p.prefix_pieces, split = cta / units, unit = cta - split * units, piece_of = unit / p.kv_heads;
        const int tiles = (p.first_key + DTILE - 1) / DTILE, each = (tiles + p.prefix_splits - 1) / p.prefix_splits;
        w.kv_head = unit - piece_of * p.kv_heads;
        w.token0 = piece_of * p.prefix_tokens;
        const int tokens = min(p.prefix_tokens, p.seqs * p.q_total - w.token0);
        w.rows = tokens * p.group;
        w.keys = p.first_key;
        w.ctx = p.first_key + tokens - 1;
        w.t0 = min(tiles, split * each);
        w.n_tiles = min(tiles - w.t0, each);
        w.part = split;
      } else if (cta >= 0) {
        cta -= prefix_ctas;
        const int rest = cta / columns;
        int z = 0;
        seq = rest;
        if (p.splits > 1) { z = rest / p.seqs; seq = rest - z * p.seqs; }
        // a single part starts at tile 0 whatever the context is: its ids need not wait for the length
        const int context = p.context_lens[seq], first_token = p.q_start != nullptr ? p.q_start[seq] : seq * p.q_total;
        if (p.splits == 1) ids_next = p.block_tables[(size_t)seq * p.max_blocks + min(table_end, first_block + lane)];
        w = Work(p, cta - rest * columns, z, context, first_token);
        cta += prefix_ctas;
      } else {
        w.n_tiles = -1;
      }
      if (lane == 0) {
        ok = wait(&w_empty[piece & 1], ((piece >> 1) & 1) ^ 1, 12);
        if (ok) {
          w.store(announced + 2 * (piece & 1));
          mbar_arrive(&w_full[piece & 1]);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      const int n_tiles = w.n_tiles;
      if (!ok || n_tiles < 0) break;
      // ids are read up to the end of the table's row; those past the sequence's last block are not used
      auto fetch_ids = [&](int j) {
        return p.block_tables[(size_t)seq * p.max_blocks + min(table_end, from_block + (w.t0 + j) * kBlocksPerTile + lane)];
      };
      if ((p.splits > 1 || cta < prefix_ctas) && n_tiles > 0) ids_next = fetch_ids(0);
      const int blocks = (w.keys + BLOCK_TOKENS - 1) / BLOCK_TOKENS - w.t0 * kBlocksPerTile;
      // ---- its tiles, and meanwhile the next piece: asked for as the last K tile goes out (the answer takes about a
      // microsecond, and a CTA with a long piece should not sit on another one)
      int ids_k = 0, ids_prev = 0;                    // block ids of the last K tile's group of four tiles, and of the one before
      const int ask_at = n_tiles > 1 ? 2 * n_tiles - 3 : 0;
#pragma unroll 1
      for (int t = 0; t < max(1, 2 * n_tiles) && ok; ++t) {
        if (t < 2 * n_tiles) {
          const bool is_k = t == 0 || ((t & 1) && t < 2 * n_tiles - 1);
          const int j = is_k ? (t + 1) >> 1 : t == 2 * n_tiles - 1 ? n_tiles - 1 : (t >> 1) - 1;
          if (is_k && j % kTilesPerGroup == 0) {
            ids_prev = ids_k;
            ids_k = ids_next;
            if (j + kTilesPerGroup < n_tiles) ids_next = fetch_ids(j + kTilesPerGroup);
          }
          // V of the last tile of a group goes out after K of the next group's first
          const int ids = !is_k && j % kTilesPerGroup == kTilesPerGroup - 1 && j + 1 < n_tiles ? ids_prev : ids_k;
          const int id = __shfl_sync(0xffffffffu, ids, (j % kTilesPerGroup) * kBlocksPerTile + lane % kBlocksPerTile);
          const uint32_t g = base + (uint32_t)t;
          const uint32_t s = g % kSlots;
          const int here = min(kBlocksPerTile, blocks - j * kBlocksPerTile);      // blocks that hold keys
          if (lane == 0) {
            ok = wait(&empty[s], ((g / kSlots) & 1) ^ 1, is_k ? 1 : 2);
            if (ok) mbar_arrive_expect_tx(&full[s], (uint32_t)here * BLOCK_TOKENS * HD * 2);
          }
          ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
          if (ok && lane < here)
            tma_load_5d(ring + s * C::kTile + lane * (BLOCK_TOKENS * HD * 2), is_k ? &map_k : &map_v, &full[s], 0, 0, w.kv_head * (HD / 64), 0, id);
        }
        if (t == ask_at && lane == 0 && ok) {
          fence_proxy_async_smem();                   // the answer before has been read
          mbar_arrive_expect_tx(taken, 16);
          launch_take_request(answer, taken);
          asked = true;
        }
      }
      if (!ok) break;
      base += 2u * (uint32_t)n_tiles;
      cta = -1;
      if (lane == 0) {
        ok = wait(taken, piece & 1, 13);
        if (ok) {
          asked = false;
          if (!launch_take_answer(answer, cta)) cta = -1;
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      cta = __shfl_sync(0xffffffffu, cta, 0);
    }
    // after a wait that ran out: the answer may still be on its way into this CTA's shared memory (bounded as well)
    if (lane == 0 && asked) {
      const unsigned long long since = global_timer_ns();
      while (!mbar_try_wait(taken, piece & 1) && global_timer_ns() - since < kWaitBudgetNs) {}
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc_s = make_idesc(DTILE, N, 1, false, false);
    constexpr uint32_t idesc_o = make_idesc(128, N, 1, true, false);
    const uint32_t q_km = desc_lo_k_major(smem_u32(sQ)), p_km0 = desc_lo_k_major(smem_u32(sP));
    const uint32_t k_km0 = desc_lo_k_major(smem_u32(ring));
    const uint32_t v_mn0 = desc_lo_mn_major(smem_u32(ring), 1024);
    constexpr uint32_t kSlotStep = C::kTile >> 4;
    bool ok = true;
    uint32_t base = 0, slots = 0, staged = 0;         // steps, ring tiles and pieces with keys before this piece
#pragma unroll 1
    for (uint32_t piece = 0; ok; ++piece) {
      if (!wait(&w_full[piece & 1], (piece >> 1) & 1, 14)) break;
      Work w;
      w.load(announced + 2 * (piece & 1));
      const int n_tiles = w.n_tiles;
      __syncwarp();
      if (lane == 0) mbar_arrive(&w_empty[piece & 1]);
      if (n_tiles < 0) break;
      if (n_tiles == 0) continue;
      if (!wait(q_ready, staged & 1, 15)) break;
      ++staged;
#pragma unroll 1
      for (int j = -1; j < n_tiles; ++j) {
        if (j + 1 < n_tiles) {
          // S^T of step j + 1, before the second product of step j
          const uint32_t g = base + (uint32_t)(j + 1), t = slots + (uint32_t)k_number(j + 1), slot = t % kSlots;
          if (!wait(&full[slot], (t / kSlots) & 1, 3) || !wait(&s_free[g & 1], ((g >> 1) & 1) ^ 1, 4)) { ok = false; break; }
          tc_fence_after_sync();
          if (elect_one()) {
            const uint32_t k_km = k_km0 + slot * kSlotStep, d = tmem_base + (g & 1) * N;
            umma_f16_c<false>(d, desc_cache<HD>(k_km, 0), desc_at(q_km, 0), idesc_s);
#pragma unroll
            for (int k = 1; k < HD / 16; ++k)
              umma_f16_c<true>(d, desc_cache<HD>(k_km, cache_column_step(k)), desc_at(q_km, k_major_step(k, N * 128)), idesc_s);
            tc_commit(&s_full[g & 1]);
            tc_commit(&empty[slot]);
          }
          __syncwarp();
        }
        if (j < 0) continue;
        const uint32_t g = base + (uint32_t)j, t = slots + (uint32_t)v_number(j, n_tiles), slot = t % kSlots;
        if (!wait(&p_ready[g & 1], (g >> 1) & 1, 5) || !wait(&full[slot], (t / kSlots) & 1, 10)) { ok = false; break; }
        // Keys of this tile, 16 to a product. The unused end of the last block becomes zero: its probabilities are zero,
        // and zero times whatever an old sequence left there (an infinity, a NaN) must not reach the sums. Blocks past
        // that one have not been fetched and are not multiplied.
        const int keys = min(DTILE, w.keys - (w.t0 + j) * DTILE);
        if (keys % BLOCK_TOKENS != 0) {
          uint8_t* tile = ring + slot * C::kTile;
          const int rows = BLOCK_TOKENS - keys % BLOCK_TOKENS;
#pragma unroll 1
          for (int i = lane; i < rows * (HD / 8); i += 32)      // (row, 64-column half, 16 bytes of 128)
            *reinterpret_cast<uint4*>(tile + cache_row_offset<HD>(keys + i / (HD / 8)) + (i % (HD / 8)) / 8 * 1024 + i % 8 * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
          __syncwarp();
        }
        tc_fence_after_sync();
        if (elect_one()) {
          const uint32_t v_mn = v_mn0 + slot * kSlotStep, p_km = p_km0 + (g & 1) * (uint32_t)(C::kP >> 4);
#pragma unroll 1
          for (int k = 0; k * 16 < keys; ++k)
            umma_f16(tmem_base + C::kOCol, desc_cache<HD>(v_mn, cache_row_step<HD>(k)), desc_at(p_km, k_major_step(k, N * 128)), idesc_o, j != 0 || k != 0);
          tc_commit(&pv_done[g & 1]);
          tc_commit(&empty[slot]);
        }
        __syncwarp();
      }
      base += (uint32_t)n_tiles;
      slots += 2u * (uint32_t)n_tiles;
    }
  } else {
    const int quarter = warp & 3;
    const int key_lane = quarter * 32 + lane;         // this thread's key of a tile, and its row of O^T
    const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const float sl = p.scale * kLog2e;
    bool ok = true;
    // The four warps exchange one value per query row (lane r: row r) through a ring of four slots: a warp writes its
    // value of exchange number x and arrives, and waits (bounded) until all four have before it reads them. It does so
    // before it writes x + 1, so the barrier never runs two phases ahead of a waiter.
    uint32_t exchange = 0;
    float* my_exchange = sExchange + quarter * 32 + lane;
    auto publish = [&](float mine) {
      my_exchange[(exchange & 3) * 128] = mine;
      __syncwarp();
      if (lane == 0) mbar_arrive(xbar);
    };
    auto collect = [&](float (&all)[4]) -> bool {
      if (!wait(xbar, exchange & 1, 9)) return false;
#pragma unroll
      for (int q = 0; q < 4; ++q) all[q] = sExchange[(exchange & 3) * 128 + q * 32 + lane];
      ++exchange;
      return true;
    };
    // Query rows of a piece, 16 bytes at a time over the 128 threads: loaded into registers as soon as the piece is known,
    // stored when the products of the piece before have read theirs. Which of them a thread moves is the same for every
    // piece.
    constexpr int kChunks = HD / 8, kHeld = (R * kChunks + 127) / 128;
    uint4 held[kHeld];
    long long held_from[kHeld];
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      const int r = (key_lane + 128 * u) / kChunks, ch = (key_lane + 128 * u) % kChunks;
      held_from[u] = (r / p.group) * p.q_pitch + (r % p.group) * HD + 8 * ch;
    }
    // lane r looks after query row r: new token r / group, head r % group of the KV head's group
    const int my_token = lane / p.group, my_head = lane - my_token * p.group;
    uint32_t base = 0;                                // steps of all pieces before this one
    Work w;
    w.n_tiles = -1;                                   // nothing before the first piece
#pragma unroll 1
    for (uint32_t piece = 0;; ++piece) {
      const int n_tiles = w.n_tiles, rows = w.rows;
      const int sees_least = w.ctx - (rows - 1) / p.group;           // keys that the first new token sees
      float m_run = -INFINITY;                        // of row `lane`
      float l[R];                                     // of every row, this thread's keys only
#pragma unroll
      for (int r = 0; r < R; ++r) l[r] = 0.0f;
#pragma unroll 1
      for (int j = 0; j < n_tiles; ++j) {
        const uint32_t g = base + (uint32_t)j;
        const int b = g & 1;
        if (!wait(&s_full[b], (g >> 1) & 1, 6)) { ok = false; break; }
        tc_fence_after_sync();
        uint32_t sv[R];
        tmem_ld_rows<R>(lane_base + (uint32_t)(b * N), sv);
        tc_wait_ld();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[b]);
        if ((w.t0 + j + 1) * DTILE > min(sees_least, w.keys)) {      // some row does not see the whole tile
          // rows are packed token by token: hidden from the tokens in front of the one at this key
          const int key = (w.t0 + j) * DTILE + key_lane;
          const int hidden = key < w.keys ? max(key - sees_least + 1, 0) * p.group : R;
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (r < hidden) sv[r] = 0xff800000u;       // -inf
        }
        float mine = -INFINITY;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float m = warp_max_f32(__uint_as_float(sv[r]));
          if (lane == r) mine = m;
        }
        publish(lane < rows ? mine : -INFINITY);
        float part[4];
        if (!collect(part)) { ok = false; break; }
        const float m_tile = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
        // lazy reference maximum (see flash_fwd.cu); every warp sees the same m_tile and decides alike
        const bool moved = (m_tile - m_run) * sl > 8.0f;
        const float m_new = moved ? m_tile : m_run;
        const float m_safe = (m_new == -INFINITY) ? 0.0f : m_new;
        const float alpha = moved ? exp2f((m_run - m_safe) * sl) : 1.0f;
        const float neg = -m_safe * sl;
        m_run = m_new;
        const bool any_moved = __any_sync(0xffffffffu, moved);
        // probability tile b was last read by the second product of step g - 2, and O^T changes scale only when every
        // product up to step g - 1 has landed
        if (g > 1 && !wait(&pv_done[b], ((g - 2) >> 1) & 1, 7)) { ok = false; break; }
        if (any_moved && j > 0) {
          if (!wait(&pv_done[b ^ 1], ((g - 1) >> 1) & 1, 7)) { ok = false; break; }
          tc_fence_after_sync();
          uint32_t ov[R];
          tmem_ld_rows<R>(lane_base + C::kOCol, ov);
          tc_wait_ld();
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float shrink = __shfl_sync(0xffffffffu, alpha, r);
            l[r] *= shrink;
            ov[r] = __float_as_uint(__uint_as_float(ov[r]) * shrink);
          }
          tmem_st_rows<R>(lane_base + C::kOCol, ov);
          tc_wait_st();
        }
        // P^T rows are query rows, 64 keys to 128 bytes; two lanes trade so that each stores two keys of one row
        uint8_t* tile_p = sP + b * C::kP + (quarter >> 1) * (N * 128);
        const int pair_key = (quarter & 1) * 32 + (lane & ~1);
#pragma unroll
        for (int r = 0; r < R; r += 2) {
          const float p0 = exp2f(fmaf(__uint_as_float(sv[r]), sl, __shfl_sync(0xffffffffu, neg, r)));
          const float p1 = exp2f(fmaf(__uint_as_float(sv[r + 1]), sl, __shfl_sync(0xffffffffu, neg, r + 1)));
          l[r] += p0;
          l[r + 1] += p1;
          const float other = __shfl_xor_sync(0xffffffffu, (lane & 1) ? p0 : p1, 1);
          const int row = r + (lane & 1);
          *reinterpret_cast<uint32_t*>(tile_p + row * 128 + (((pair_key >> 3) ^ (row & 7)) << 4) + (pair_key & 7) * 2) =
              (lane & 1) ? pack_bf16x2(other, p1) : pack_bf16x2(p0, other);
        }
        fence_proxy_async_smem();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[b]);
      }
      // ---- the next piece: its query rows on their way while this one's sums are joined
      Work next;
      ok = ok && wait(&w_full[piece & 1], (piece >> 1) & 1, 14);
      if (ok) {
        next.load(announced + 2 * (piece & 1));
        __syncwarp();
        if (lane == 0) mbar_arrive(&w_empty[piece & 1]);
        if (next.n_tiles > 0) {
          const __nv_bfloat16* q = p.q + (size_t)next.token0 * p.q_pitch + (size_t)(next.kv_head * p.group) * HD;
#pragma unroll
          for (int u = 0; u < kHeld; ++u)
            if ((key_lane + 128 * u) / kChunks < next.rows) held[u] = ld_v4(reinterpret_cast<const uint4*>(q + held_from[u]));
        }
      }
      const bool real = lane < rows && n_tiles >= 0;
      const int out_row = (w.token0 + my_token) * p.heads + w.kv_head * p.group + my_head;
      auto part_row = [&](int row) { return (size_t)row * p.part_stride + w.part; };
      if (p.part_stride > 0 && quarter == 0 && real && (n_tiles == 0 || !ok)) p.part_ml[part_row(out_row)] = make_float2(0.0f, 0.0f);
      if (!ok) break;
      if (n_tiles > 0) {
        // Lane r is to have the sum of row r over this warp's keys. Two lanes trade halves of their rows, then quarters, ...:
        // R - 1 exchanges, where summing every row over all lanes takes 5 R.
#pragma unroll
        for (int half = R / 2; half > 0; half >>= 1) {
          const bool upper = (lane & half) != 0;
#pragma unroll
          for (int r = 0; r < half; ++r) {
            const float theirs = upper ? l[r] : l[r + half], mine = upper ? l[r + half] : l[r];
            l[r] = mine + __shfl_xor_sync(0xffffffffu, theirs, half);
          }
        }
#pragma unroll
        for (int o = R; o < 32; o <<= 1) l[0] += __shfl_xor_sync(0xffffffffu, l[0], o);
        publish(l[0]);
      }
      if (next.n_tiles > 0) {
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
          const int r = (key_lane + 128 * u) / kChunks, ch = (key_lane + 128 * u) % kChunks;
          if (r < next.rows) *reinterpret_cast<uint4*>(sQ + (ch >> 3) * (N * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = held[u];
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_ready);
      }
      // ---- this piece's output
      if (n_tiles > 0) {
        float sums[4];
        base += (uint32_t)n_tiles;
        if (!collect(sums) || !wait(&pv_done[(base - 1) & 1], ((base - 1) >> 1) & 1, 8)) break;
        tc_fence_after_sync();
        const float l_all = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        const float inv_l = l_all > 0.0f ? 1.0f / l_all : 0.0f;
        if (p.part_stride > 0 && quarter == 0 && real) p.part_ml[part_row(out_row)] = make_float2(m_run == -INFINITY ? 0.0f : m_run * sl, l_all);
        if (HD == 128 || quarter < 2) {
          uint32_t ov[R];
          tmem_ld_rows<R>(lane_base + C::kOCol, ov);
          tc_wait_ld();
          // 32 neighbouring elements of row r per warp; rows and parts are counted in 32 bits (each is 256 bytes at least)
          if (p.part_stride > 0) {
            const int place = (int)part_row(out_row);
            float* dst = p.part_o + key_lane;
#pragma unroll
            for (int r = 0; r < R; ++r) {
              const int at = __shfl_sync(0xffffffffu, place, r);
              if (r < rows) dst[(long long)at * HD] = __uint_as_float(ov[r]);
            }
          } else {
            __nv_bfloat16* dst = p.out + key_lane;
#pragma unroll
            for (int r = 0; r < R; ++r) {
              const int at = __shfl_sync(0xffffffffu, out_row, r);
              const float scale = __shfl_sync(0xffffffffu, inv_l, r);
              if (r < rows) dst[(long long)at * HD] = __float2bfloat16(__uint_as_float(ov[r]) * scale);
            }
          }
        }
        tc_fence_before_sync();
      }
      if (next.n_tiles < 0) break;
      w = next;
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
  // a launch that joins the parts waits for this one only: this one does not end before the launch in front of it has
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// out[row, head, :] = sum_z w_z O_z / sum_z w_z l_z with w_z = 2^(m_z - max m): one warp per (row, head), HD / 32
// neighbouring elements per lane. A part whose sum is 0 saw no key and has no row; any other counts, however small its weight
// and also if its sum is NaN: what went wrong in front of the kernel must not come out as attention over the other parts. The
// parts are read at once, before their weights are known: what bounds the kernel is the latency of two dependent reads, not
// the bytes. It is launched while the launch in front of it still runs and waits
// for it (and so for everything that one has waited for) on the device. It does not let the next launch start among its own
// CTAs in turn: a prefix kernel then takes whole pairs of SMs instead of one of each, and the suffixes are left with fewer
// of the paths to memory that pairs share (33 x 5 rows, back to back: 33 us instead of 28).
template <int HD>
__global__ void __launch_bounds__(128) merge_splits_kernel(const float* part_o, const float2* part_ml,
                                                           __nv_bfloat16* out, const int* q_start, int q_len,
                                                           int heads, int splits, long long pairs /* sequences * q_len * heads */) {
  const int lane = threadIdx.x & 31;
  const long long w = (blockIdx.x * (long long)blockDim.x + threadIdx.x) >> 5;
  if (w >= pairs) return;
  size_t out_row = (size_t)w;
  if (q_start != nullptr) {
    const long long local_row = w / heads;
    const int seq = (int)(local_row / q_len);
    out_row = (size_t)(q_start[seq] + (int)(local_row - (long long)seq * q_len)) * heads + (size_t)(w - local_row * heads);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kPerLane = HD / 32;
  constexpr int kBatch = 4;
  float acc[kPerLane];
#pragma unroll
  for (int c = 0; c < kPerLane; ++c) acc[c] = 0.0f;
  const float* src = part_o + out_row * splits * HD + lane * kPerLane;
  // lane z: part z (and z + 32: at most 64 parts)
  const float2* ml = part_ml + out_row * splits;
  const float2 none = make_float2(0.0f, 0.0f);
  const float2 a = lane < splits ? ld_l2(ml + lane) : none, b = lane + 32 < splits ? ld_l2(ml + lane + 32) : none;
  const unsigned saw_a = __ballot_sync(0xffffffffu, a.y != 0.0f), saw_b = __ballot_sync(0xffffffffu, b.y != 0.0f);
  float weight_a = 0.0f, weight_b = 0.0f;
  bool weighed = false;
#pragma unroll 1
  for (int z0 = 0; z0 < splits; z0 += kBatch) {
    float v[kBatch][kPerLane];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (z0 + u < splits) {
        if constexpr (kPerLane == 4) *reinterpret_cast<float4*>(v[u]) = ld_l2(reinterpret_cast<const float4*>(src + (size_t)(z0 + u) * HD));
        else *reinterpret_cast<float2*>(v[u]) = ld_l2(reinterpret_cast<const float2*>(src + (size_t)(z0 + u) * HD));
      }
    }
    if (!weighed) {
      float m = fmaxf(a.y != 0.0f ? a.x : -INFINITY, b.y != 0.0f ? b.x : -INFINITY);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      weight_a = a.y != 0.0f ? exp2f(a.x - m) : 0.0f;
      weight_b = b.y != 0.0f ? exp2f(b.x - m) : 0.0f;
      float l = weight_a * a.y + weight_b * b.y;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      const float inv = l != 0.0f ? 1.0f / l : 0.0f;
      weight_a *= inv;
      weight_b *= inv;
      weighed = true;
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (z0 + u < splits) {
        const float weight = __shfl_sync(0xffffffffu, z0 + u < 32 ? weight_a : weight_b, (z0 + u) & 31);
        if (((z0 + u < 32 ? saw_a : saw_b) >> ((z0 + u) & 31)) & 1u) {
#pragma unroll
          for (int c = 0; c < kPerLane; ++c) acc[c] += weight * v[u][c];
        }
      }
    }
  }
  if constexpr (kPerLane == 4)
    *reinterpret_cast<uint2*>(out + out_row * HD + lane * 4) = make_uint2(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]));
  else
    *reinterpret_cast<uint32_t*>(out + out_row * HD + lane * 2) = pack_bf16x2(acc[0], acc[1]);
}

// `kernel` on `grid`, with all the shared memory that its CTAs per SM need
template <typename Kernel>
static int launch_on(Kernel kernel, bool (&configured)[kMaxDevices], dim3 grid, int smem, const CUtensorMap& map_k,
                     const CUtensorMap& map_v, const Params& p, bool beside_previous, cudaStream_t stream) {
  // function attributes belong to a device: set once on each
  int dev = 0;
  AJB_CUDA_OK(cudaGetDevice(&dev));
  if (dev >= kMaxDevices || !configured[dev]) {
    AJB_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    // two CTAs per SM need the whole shared-memory carve-out
    AJB_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    if (dev < kMaxDevices) configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = beside_previous ? 1 : 0;
  AJB_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, map_k, map_v, p));
  return 0;
}

template <int HD>
static int launch_kernel(const Launch& a, cudaStream_t stream) {
  Params p;
  p.q = (const __nv_bfloat16*)a.q; p.out = (__nv_bfloat16*)a.out; p.block_tables = (const int*)a.block_tables;
  p.context_lens = (const int*)a.context_lens; p.q_start = (const int*)a.q_start; p.q_pitch = a.q_pitch;
  p.max_blocks = a.max_blocks; p.heads = a.heads; p.kv_heads = a.kv_heads; p.group = a.heads / a.kv_heads; p.q_len = a.q_len;
  p.seqs = a.num_seqs; p.chunks = (a.q_total + a.q_len - 1) / a.q_len; p.q_total = a.q_total;
  p.first_key = a.first_key; p.scale = a.scale; p.status = device_status_buffer();
  p.early = a.early;
  p.splits = a.splits; p.prefix_splits = a.prefix_splits; p.part_stride = a.part_stride; p.part_base = a.part_base;
  p.part_o = (float*)a.part_o; p.part_ml = (float2*)a.part_ml;
  static bool configured[5][kMaxDevices] = {};
  p.prefix_tokens = a.prefix_tokens;
  p.prefix_pieces = a.prefix_splits > 0 ? (a.num_seqs * a.q_total + a.prefix_tokens - 1) / a.prefix_tokens : 0;
  const int rows = p.group * (a.prefix_splits > 0 ? max(a.q_len, min(a.prefix_tokens, a.num_seqs * a.q_total)) : a.q_len);
  if (rows <= 32) {
    const long long ctas = (long long)a.kv_heads * p.prefix_pieces * a.prefix_splits + (long long)a.num_seqs * a.kv_heads * p.chunks * a.splits;
    AJB_REQUIRE(ctas <= 0x7fffffffll, "paged attention: %lld CTAs are too many for one launch", ctas);
    const dim3 grid((unsigned)ctas);
    CUtensorMap map_k, map_v;
    if (a.map_k != nullptr) {
      map_k = *a.map_k;
      map_v = *a.map_v;
    } else {
      int rc = make_tensor_map_cache(&map_k, a.k_cache, a.num_blocks, a.kv_heads, HD);
      if (rc == 0) rc = make_tensor_map_cache(&map_v, a.v_cache, a.num_blocks, a.kv_heads, HD);
      if (rc) return rc;
    }
    const int smem16 = DecodeCfg<HD, 16>::kSmem, smem32 = DecodeCfg<HD, 32>::kSmem;
    if (rows <= 4) return launch_on(paged_decode_kernel<HD, 4>, configured[0], grid, smem16, map_k, map_v, p, a.beside_previous || a.early, stream);
    if (rows <= 8) return launch_on(paged_decode_kernel<HD, 8>, configured[1], grid, smem16, map_k, map_v, p, a.beside_previous || a.early, stream);
    if (rows <= 16) return launch_on(paged_decode_kernel<HD, 16>, configured[2], grid, smem16, map_k, map_v, p, a.beside_previous || a.early, stream);
    return launch_on(paged_decode_kernel<HD, 32>, configured[3], grid, smem32, map_k, map_v, p, a.beside_previous || a.early, stream);
  }
  AJB_REQUIRE(a.prefix_splits == 0, "paged attention: more than 32 query rows per CTA cannot take a shared prefix along");
  AJB_REQUIRE((long long)a.kv_heads * p.chunks <= 65535, "paged attention: %d new tokens per sequence are too many for one launch", a.q_total);
  CUtensorMap map_k, map_v;
  const uint64_t row_pitch = (uint64_t)a.kv_heads * HD * 2;
  int rc = make_tensor_map_3d(&map_k, a.k_cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.num_blocks, BLOCK_TOKENS,
                              (uint64_t)a.kv_heads * HD, row_pitch * BLOCK_TOKENS, row_pitch, BLOCK_TOKENS, 64);
  if (rc) return rc;
  rc = make_tensor_map_3d(&map_v, a.v_cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.num_blocks, BLOCK_TOKENS,
                          (uint64_t)a.kv_heads * HD, row_pitch * BLOCK_TOKENS, row_pitch, BLOCK_TOKENS, 64);
  if (rc) return rc;
  return launch_on(paged_attention_kernel<HD>, configured[4], dim3(a.num_seqs, a.kv_heads * p.chunks, a.splits), Cfg<HD>::kSmem, map_k, map_v, p,
                   a.beside_previous, stream);
}

int launch(const Launch& a, int head_dim, cudaStream_t stream) {
  if (head_dim == 128) return launch_kernel<128>(a, stream);
  if (head_dim == 64) return launch_kernel<64>(a, stream);
  set_error("paged attention: head_dim %d is not supported (64 and 128 are)", head_dim);
  return 2;
}

template <int HD>
static int launch_merge(const Launch& a, cudaStream_t stream) {
  const long long pairs = (long long)a.num_seqs * a.q_total * a.heads;
  return launch_early(merge_splits_kernel<HD>, dim3((unsigned)((pairs * 32 + 127) / 128)), dim3(128), 0, stream, (const float*)a.part_o,
                      (const float2*)a.part_ml, (__nv_bfloat16*)a.out, (const int*)a.q_start, a.q_total, a.heads, a.part_stride, pairs);
}

int merge_parts(const Launch& a, int head_dim, cudaStream_t stream) {
  return head_dim == 128 ? launch_merge<128>(a, stream) : launch_merge<64>(a, stream);
}

}  // namespace paged
}  // namespace ajb

// Every sequence of the launch contributes exactly q_len new rows; (heads / kv_heads) * q_len <= 64.
// splits > 1 divides every sequence's tiles over that many CTAs: part_o must hold rows * heads * splits * head_dim
// floats and part_ml rows * heads * splits * 2 floats, where rows = the total number of query rows of the batch.
extern "C" int ajb_paged_attention(const void* q, const void* k_cache, const void* v_cache, const void* block_tables,
                                   const void* context_lens, const void* q_start, void* out, int num_seqs,
                                   int num_blocks, int block_size, int max_blocks, int heads, int kv_heads,
                                   int head_dim, int q_len, float scale, int splits, void* part_o, void* part_ml,
                                   void* stream) {
  using namespace ajb;
  AJB_REQUIRE(splits >= 1 && splits <= 64 && (splits == 1 || (part_o != nullptr && part_ml != nullptr)),
              "paged attention: splits must be in [1, 64] and come with a workspace");
  AJB_REQUIRE(block_size == paged::BLOCK_TOKENS, "paged attention: cache block size must be %d", paged::BLOCK_TOKENS);
  AJB_REQUIRE(heads % kv_heads == 0 && (heads / kv_heads) * q_len <= paged::kMaxRows && q_len >= 1,
              "paged attention: (heads / kv_heads) * q_len = %d exceeds %d", (heads / kv_heads) * q_len, paged::kMaxRows);
  if (num_seqs <= 0) return 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  paged::Launch a;
  a.q = q; a.k_cache = k_cache; a.v_cache = v_cache; a.block_tables = block_tables; a.context_lens = context_lens;
  a.q_start = q_start; a.out = out; a.q_pitch = (long long)heads * head_dim;
  a.num_seqs = num_seqs; a.num_blocks = num_blocks; a.max_blocks = max_blocks; a.heads = heads; a.kv_heads = kv_heads;
  a.q_len = q_len; a.q_total = q_len; a.first_key = 0; a.scale = scale; a.splits = splits; a.prefix_splits = a.prefix_tokens = 0;
  a.part_stride = splits > 1 ? splits : 0; a.part_base = 0; a.part_o = part_o; a.part_ml = part_ml;
  a.map_k = a.map_v = nullptr; a.beside_previous = a.early = false;
  int rc = paged::launch(a, head_dim, s);
  if (rc == 0 && splits > 1) rc = paged::merge_parts(a, head_dim, s);
  return rc;
}
