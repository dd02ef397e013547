// Attention of a batch whose sequences begin with the same cached prefix, for decoding and verification on sm_100a.
//
// softmax over the keys of one row is a sum over key ranges: with (m, l, O) = (reference maximum, sum of 2^(s - m),
// sum of 2^(s - m) v) of each range, out = sum_z 2^(m_z - m) O_z / sum_z 2^(m_z - m) l_z. The prefix range is the same
// for every sequence, so its keys and values need to be read once per batch, not once per sequence, and its scores are
// a dense product: all query rows of a KV head (tokens * group of them, no mask, the prefix lies before every new
// token) fill 128-row tensor-core tiles. The rest of each sequence runs on the paged kernel (paged_attention.cu) from
// key `shared` on; both leave un-normalised fp32 parts, which a small kernel joins.
//
// The prefix kernel takes a share of the prefix in steps of 128 keys, with two streams of 128 query rows per CTA
// (S = Q K^T, softmax, O += P V with S, P and O in tensor memory, P written over the scores it came from): while eight
// warps turn one stream's scores into probabilities, the tensor pipe runs the other's products. A 128 x 128 step is two
// products of 512 cycles and 16384 exponentials, 1024 cycles of the SM's exponential unit, for which it takes 1600 to 1900:
// the chain of waits (scores, maxima of the other half of the keys, probabilities, products) is what bounds it, with no
// exponentials it is 2 % faster. The streams are two row tiles that share every K and V tile; when all rows fit one tile they are
// two halves of the keys instead (even and odd tiles, two parts; one part when a CTA has a single tile).
//
// A prefix CTA has an SM to itself (shared memory), the suffix launch, which does not read what this one writes, starts
// as soon as every CTA here has and takes the other SMs: the prefix is bound by its steps (one of 256 rows x 128 keys of
// 128 takes 1.7 us: on 148 SMs 1.46 PFLOP/s, 0.91 of what a library product reaches without the exponentials; with its start
// and end a launch of 128 CTAs and 60 steps each reaches 0.96 PFLOP/s), the suffix by memory, and the number of prefix CTAs
// divides the SMs so that both last about as long.
//
// Scores, maxima, sums and parts are fp32. Probabilities are rounded to bf16 (half a step: 2^-8 of each) as the operand of the
// second product, whose other operand, the cached values, is bf16: kept in fp32 they would take two such products. The sums
// are of the unrounded ones. Against 64 bits results are off by 0.0019 to 0.0023 (2-norm), 0.0017 of which is the rounding of
// the result itself.
//
// This kernel starts slowly (11 to 14 us until its first parts are stored, for barriers, 512 columns of tensor memory and
// two dependent products). With few rows, or many rows and a short prefix, the prefix runs in the paged launch itself, as
// more pieces of its work for 16 query rows each: one launch less, and products that are as narrow as the rows are few.
// ops/serving.py estimates both and takes the shorter: 24 sequences of 4 rows per KV head behind 2048 + 32 tokens take
// 11.9 us in pieces and 16.1 us with this kernel; behind 6144 + 256, 20.2 us and 19.7 us. 256 sequences behind 7680 tokens:
// 80 us, of which the suffixes alone take 54 us.
#include "common.cuh"
#include "serving_args.h"
#include "paged_attention.h"

namespace ajb {
namespace prefix {

constexpr int TILE = 128;          // keys per step
constexpr int ROWS = 128;          // query rows of a stream
constexpr int BLOCK_TOKENS = 16;   // tokens per cache block
constexpr int kThreads = 576;      // TMA warp, product warp, 16 softmax warps: per stream four tensor-memory quarters x two key halves
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kPrefixKernelId = 12;

template <int HD>
struct Cfg {
  static constexpr int kTile = TILE * HD * 2;            // Q, one K tile, one V tile: same size
  static constexpr int kStages = HD == 64 ? 5 : 2;       // K and V tiles held at a time
  static constexpr int kStagePitch = 12;                 // floats per row of a store block: 8 columns and 16 bytes of padding
  static constexpr int kStoreBlock = 32 * kStagePitch * 4;
  static constexpr int kExchange = 2 * 2 * 2 * ROWS * 4; // [stream][parity][key half][row]
  static constexpr int kSmem = kTile * (2 + 2 * kStages) + 16 * kStoreBlock + kExchange + 512;
  static constexpr int kOCol = 2 * TILE;                 // S (and P) of stream s at s * 128, O behind them
  static constexpr int kTmemCols = 512;
  // a CTA of the suffix launch (three or five tiles of 128 keys at least) on the same SM would wait for its tensor memory
  // until this one leaves: it must not fit
  static_assert(kSmem <= 227 * 1024 && kSmem + 3 * kTile > 227 * 1024, "shared memory of a prefix CTA");
};

struct Params {
  const __nv_bfloat16* q;
  const int* table;             // block ids of the prefix
  float inv_group;
  long long q_pitch;
  int rows;                     // tokens * group: query rows of one KV head
  int group, heads;
  int keys;                     // shared prefix length (a multiple of the block size)
  int pairs;                    // row tiles two by two; 0: one row tile, its streams take even and odd key tiles
  int kv_heads, splits;
  float scale;
  int part_stride;
  float* part_o;
  float2* part_ml;
  DeviceStatus* status;
};

__device__ __forceinline__ void store_chunk(uint8_t* tile, int row, int ch, uint4 val) {
  *reinterpret_cast<uint4*>(tile + (ch >> 3) * (ROWS * 128) + row * 128 + (((ch & 7) ^ (row & 7)) << 4)) = val;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
prefix_attention_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params p) {
  using C = Cfg<HD>;
  constexpr int kStages = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;                                    // two row tiles
  uint8_t* sK = sQ + 2 * C::kTile;
  uint8_t* sV = sK + kStages * C::kTile;
  uint8_t* sStore = sV + kStages * C::kTile;
  float* sExchange = reinterpret_cast<float*>(sStore + 16 * C::kStoreBlock);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sStore + 16 * C::kStoreBlock + C::kExchange);
  // in this order: the suffix launch reads the inputs without waiting for anything but its start
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (smem_misaligned(smem, p.status, kPrefixKernelId, reinterpret_cast<uint32_t*>(bars) + 120)) return;
  uint64_t* k_full = bars;               // kStages (<= 5)
  uint64_t* k_empty = bars + 5;
  uint64_t* v_full = bars + 10;
  uint64_t* v_empty = bars + 15;
  uint64_t* s_full = bars + 20;          // per stream
  uint64_t* p_ready = bars + 22;
  uint64_t* pv_done = bars + 24;
  uint64_t* pair_bar = bars + 26;        // per stream and quarter: the two warps that share 32 rows
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 34);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto wait = [&](uint64_t* bar, uint32_t parity, int stage) {
    return mbar_wait_compact(bar, parity, abort_flag, p.status, kPrefixKernelId, stage);
  };
  // row tile pairs of one (KV head, share of the keys) are neighbours: they read the same tiles out of L2
  const bool paired = p.pairs > 0;
  const int pairs = paired ? p.pairs : 1;
  const int pair = (int)blockIdx.x % pairs;
  const int kv_head = ((int)blockIdx.x / pairs) % p.kv_heads;
  const int split = (int)blockIdx.x / (pairs * p.kv_heads);
  const int all_tiles = (p.keys + TILE - 1) / TILE;
  const int per_split = (all_tiles + p.splits - 1) / p.splits;
  const int t0 = min(all_tiles, split * per_split);
  const int n_tiles = min(all_tiles - t0, per_split);
  // stream s: its rows, and how many steps it has; step i is tile i (paired) or 2 i + s
  auto row0_of = [&](int s) { return (paired ? 2 * pair + s : 0) * ROWS; };
  auto steps_of = [&](int s) { return paired ? (row0_of(s) < p.rows ? n_tiles : 0) : (n_tiles + 1 - s) / 2; };

  const int group4 = (warp - 2) >> 2;                    // of a softmax warp: four warps, one per tensor-memory quarter
  const int stream = group4 >> 1, half = group4 & 1;
  // query row r of a tile (0 .. 127) that starts at head `head0` of token `token0`
  const int row0 = row0_of(stream & 1), rows = p.rows - row0;      // rows may pass 128: then all of this tile's are real
  const int token0 = row0 / p.group, head0 = row0 - token0 * p.group;
  auto row_place = [&](int r, int& token, int& head) {
    const int t = (int)((float)(head0 + r) * p.inv_group + 0.5f * p.inv_group);       // below 256: exact
    token = token0 + t;
    head = head0 + r - t * p.group;
  };

  if (threadIdx.x == 0) {
#pragma unroll 1
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
#pragma unroll 1
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_ready[s], 8);
      mbar_init(&pv_done[s], 1);
    }
#pragma unroll 1
    for (int i = 0; i < 8; ++i) mbar_init(&pair_bar[i], 2);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tensor_map(&map_k);
    prefetch_tensor_map(&map_v);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  if (warp >= 2 && (paired || stream == 0)) {
    // query rows: HD / 8 neighbouring threads per row; rows past the last are zero
    constexpr int kChunks = HD / 8, kEach = ROWS * kChunks / 256;
    const int t = (threadIdx.x - 64) & 255;
    uint4 v[kEach];
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int r = (t + 256 * u) / kChunks, ch = (t + 256 * u) % kChunks;
      int token, h;
      row_place(r, token, h);
      v[u] = make_uint4(0, 0, 0, 0);
      if (r < rows) v[u] = ld_v4(reinterpret_cast<const uint4*>(p.q + (size_t)token * p.q_pitch + (size_t)(kv_head * p.group + h) * HD) + ch);
    }
#pragma unroll
    for (int u = 0; u < kEach; ++u) store_chunk(sQ + stream * C::kTile, (t + 256 * u) / kChunks, (t + 256 * u) % kChunks, v[u]);
    fence_proxy_async_smem();
  }
  if (warp != 0) {
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
  }

  if (warp == 0) {
    // block ids: eight per tile, four tiles by the 32 lanes of one coalesced load, a group of tiles ahead; eight lanes copy
    // a block of a tile each. K tiles run one ahead of V tiles: a K slot is free again long before the V slot of the same
    // tile. The first tiles go out before the other warps are let go.
    constexpr int kBlocksPerTile = TILE / BLOCK_TOKENS;
    constexpr int kTilesPerGroup = 32 / kBlocksPerTile;
    const int last_block = p.keys / BLOCK_TOKENS - 1;
    __syncwarp();
    auto fetch_ids = [&](int g) { return p.table[min(last_block, (t0 + g * kTilesPerGroup) * kBlocksPerTile + lane)]; };
    int ids_next = n_tiles > 0 ? fetch_ids(0) : 0, ids_k = ids_next, ids_prev = ids_next;
    bool ok = true;
#pragma unroll 1
    for (int i = 0; i < 2 * n_tiles + (n_tiles == 0); ++i) {
      // order K0 K1 V0 K2 V1 ...
      if (i == 3 || (i == 2 * n_tiles - 1 && i < 3) || n_tiles == 0) {
        tc_fence_before_sync();
        __syncthreads();
        tc_fence_after_sync();
        if (n_tiles == 0) break;
      }
      const bool is_k = i == 0 || ((i & 1) && i < 2 * n_tiles - 1);
      const int t = is_k ? (i + 1) >> 1 : i == 2 * n_tiles - 1 ? n_tiles - 1 : (i >> 1) - 1;
      if (is_k && t % kTilesPerGroup == 0) {
        ids_prev = ids_k;
        ids_k = ids_next;
        if (t + kTilesPerGroup < n_tiles) ids_next = fetch_ids(t / kTilesPerGroup + 1);
      }
      // V of the last tile of a group goes out after K of the next group's first
      const int ids = !is_k && t % kTilesPerGroup == kTilesPerGroup - 1 && t + 1 < n_tiles ? ids_prev : ids_k;
      const int id = __shfl_sync(0xffffffffu, ids, (t % kTilesPerGroup) * kBlocksPerTile + lane % kBlocksPerTile);
      const int slot = t % kStages;
      uint64_t* full = (is_k ? k_full : v_full) + slot;
      if (lane == 0) {
        ok = wait((is_k ? k_empty : v_empty) + slot, ((uint32_t)(t / kStages) & 1) ^ 1, is_k ? 1 : 2);
        if (ok) mbar_arrive_expect_tx(full, C::kTile);
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      if (!ok) break;
      if (lane < kBlocksPerTile)
        tma_load_5d((is_k ? sK : sV) + slot * C::kTile + lane * (BLOCK_TOKENS * HD * 2), is_k ? &map_k : &map_v, full, 0, 0,
                    kv_head * (HD / 64), 0, id);
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc_s = make_idesc(ROWS, TILE, 1, false, false);
    constexpr uint32_t idesc_o = make_idesc(ROWS, HD, 1, false, true);
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t q_km0 = desc_lo_k_major(smem_u32(sQ));
    const uint32_t k_km0 = desc_lo_k_major(smem_u32(sK));
    const uint32_t v_mn0 = desc_lo_mn_major(smem_u32(sV), 1024);
    constexpr uint32_t kStep = C::kTile >> 4;
    const int steps0 = steps_of(0), steps1 = steps_of(1);          // stream 0 never has fewer
    const bool both = paired && steps1 > 0;              // both streams use every tile; stream 1 comes second
    // Per round: the second product of stream 0's last step, then the first one of its next, which overwrites the scores
    // that the probabilities lay over (the tensor pipe runs in issue order), then the same of stream 1. `at` is the ring
    // slot (and phase) of the tile whose scores come next, `was` of the one whose probabilities do; with the keys divided
    // over the streams each takes every other tile. What a product needs is known before its wait ends.
    int at = 0;
    uint32_t at_phase = 0;
    int was[2] = {0, 0};
    uint32_t was_phase[2] = {0, 0};
    bool ok = true;
#pragma unroll 1
    for (int i = 0; i <= steps0 && ok; ++i) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int steps = s == 0 ? steps0 : steps1;
        const uint32_t d = tmem_base + (uint32_t)(s * TILE), o = tmem_base + (uint32_t)(C::kOCol + s * HD);
        const bool release = !both || s == 1;
        const uint32_t q_km = q_km0 + (paired ? (uint32_t)s * kStep : 0u);
        if (i < steps && !wait(&k_full[at], at_phase, 3)) { ok = false; break; }
        if (i > 0 && i <= steps) {
          const uint32_t v_mn = v_mn0 + (uint32_t)was[s] * kStep;
          if (!wait(&v_full[was[s]], was_phase[s], 5) || !wait(&p_ready[s], (uint32_t)(i - 1) & 1, 4)) { ok = false; break; }
          tc_fence_after_sync();
          if (elect_one()) {
            umma_f16_ts(o, d, desc_cache<HD>(v_mn, 0), idesc_o, i != 1);
#pragma unroll
            for (int k = 1; k < TILE / 16; ++k)            // keys 0..63 in columns [0, 32) of the scores, 64..127 in [64, 96)
              umma_f16_ts_c<true>(o, d + (uint32_t)(k < 4 ? k * 8 : 64 + (k - 4) * 8), desc_cache<HD>(v_mn, cache_row_step<HD>(k)), idesc_o);
            tc_commit(&pv_done[s]);
            if (release) tc_commit(&v_empty[was[s]]);
          }
          __syncwarp();
        }
        if (i < steps) {
          tc_fence_after_sync();
          if (elect_one()) {
            const uint32_t k_km = k_km0 + (uint32_t)at * kStep;
            umma_f16_c<false>(d, desc_at(q_km, 0), desc_cache<HD>(k_km, 0), idesc_s);
#pragma unroll
            for (int k = 1; k < HD / 16; ++k)
              umma_f16_c<true>(d, desc_at(q_km, k_major_step(k, ROWS * 128)), desc_cache<HD>(k_km, cache_column_step(k)), idesc_s);
            tc_commit(&s_full[s]);
            if (release) tc_commit(&k_empty[at]);
          }
          __syncwarp();
          was[s] = at;
          was_phase[s] = at_phase;
          if (release && ++at == kStages) { at = 0; at_phase ^= 1; }
        }
      }
    }
  } else {
    const uint32_t tmem_base = *tmem_slot;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int n = steps_of(stream);
    const bool active = quarter * 32 < rows;           // warp-uniform: quarters without query rows only keep the pace
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_col = tmem_base + lane_addr + (uint32_t)(stream * TILE + half * 64);
    const uint32_t o_col = tmem_base + lane_addr + (uint32_t)(C::kOCol + stream * HD + half * (HD / 2));
    const float sl = p.scale * kLog2e;
    float m_run = -INFINITY, l_run = 0.0f;             // l_run: this warp's half of the keys only
    bool ok = true;
    // one float per row, exchanged with the warp that holds the other half of the keys (bounded, like every wait)
    float* slots = sExchange + stream * (4 * ROWS) + row;
    auto exchange = [&](uint32_t phase, float mine, float& theirs) -> bool {
      float* slot = slots + (phase & 1) * (2 * ROWS);
      slot[half * ROWS] = mine;
      __syncwarp();
      if (lane == 0) mbar_arrive(&pair_bar[stream * 4 + quarter]);
      if (!wait(&pair_bar[stream * 4 + quarter], phase & 1, 10)) return false;
      theirs = slot[(half ^ 1) * ROWS];
      return true;
    };
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      if (!wait(&s_full[stream], (uint32_t)j & 1, 6)) { ok = false; break; }
      const int t = paired ? j : 2 * j + stream;
      const int left = p.keys - (t0 + t) * TILE;        // keys of this tile; the last tile may have fewer than 128
      if (left < TILE) {
        // the blocks that fill the tile up are copies of the last one: their probabilities are zero, and zero times an
        // infinity must not reach the sums (all that wait for the tile write the same zeros)
        const int slot = t % kStages;
        if (!wait(&v_full[slot], (uint32_t)(t / kStages) & 1, 9)) { ok = false; break; }
#pragma unroll 1
        for (int i = (half * ROWS + row); i < (TILE - left) * (HD / 8); i += 256)
          *reinterpret_cast<uint4*>(sV + slot * C::kTile + cache_row_offset<HD>(left + i / (HD / 8)) + (i % (HD / 8)) / 8 * 1024 + i % 8 * 16) =
              make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
      }
      if (active) {
        tc_fence_after_sync();
        uint32_t sv[2][32];
        tmem_ld_32x32(s_col, sv[0]);
        tmem_ld_32x32(s_col + 32u, sv[1]);
        tc_wait_ld();
        if (left < TILE) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (half * 64 + c * 32 + i >= left) sv[c][i] = 0xff800000u;      // -inf
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) m4[i & 3] = fmaxf(m4[i & 3], __uint_as_float(sv[c][i]));
        const float m_half = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        float m_other;
        if (!exchange((uint32_t)j, m_half, m_other)) { ok = false; break; }
        const float m_tile = fmaxf(m_half, m_other);
        // lazy reference maximum (see flash_fwd.cu): O is rescaled only when a row would pass 2^8
        const bool moved = (m_tile - m_run) * sl > 8.0f;
        const float m_new = moved ? m_tile : m_run;
        const float m_safe = (m_new == -INFINITY) ? 0.0f : m_new;
        const float alpha = moved ? exp2f((m_run - m_safe) * sl) : 1.0f;
        const float neg = -m_safe * sl;
        float l2[2] = {0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float p0 = exp2f(fmaf(__uint_as_float(sv[c][i]), sl, neg));
            const float p1 = exp2f(fmaf(__uint_as_float(sv[c][i + 1]), sl, neg));
            l2[0] += p0;
            l2[1] += p1;
            pk[i / 2] = pack_bf16x2(p0, p1);
          }
          tmem_st_32x16(s_col + (uint32_t)(c * 16), pk);
        }
        l_run = l_run * alpha + (l2[0] + l2[1]);
        m_run = m_new;
        if (j > 0 && __any_sync(0xffffffffu, moved)) {
          // each half of the warps rescales half of the head's columns
          if (!wait(&pv_done[stream], (uint32_t)(j - 1) & 1, 7)) { ok = false; break; }
          tc_fence_after_sync();
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t ov[16];
            tmem_ld_32x16(o_col + (uint32_t)(c * 16), ov);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
            tmem_st_32x16(o_col + (uint32_t)(c * 16), ov);
          }
        }
        tc_wait_st();
        tc_fence_before_sync();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[stream]);
    }
    // with one tile per CTA the second stream has nothing to do, and no part
    const bool lone = !paired && per_split == 1;
    const int part = paired || lone ? split : 2 * split + stream;
    auto part_row = [&](int r) {
      int token, h;
      row_place(r, token, h);
      return ((size_t)token * p.heads + kv_head * p.group + h) * p.part_stride + part;
    };
    float l_other = 0.0f;
    if (ok && active && n > 0) ok = exchange((uint32_t)n, l_run, l_other);
    const bool real = row < rows && half == 0 && !(lone && stream == 1);
    if (real && (n == 0 || !ok)) p.part_ml[part_row(row)] = make_float2(0.0f, 0.0f);       // nothing to join from this part
    if (ok && active && n > 0 && wait(&pv_done[stream], (uint32_t)(n - 1) & 1, 8)) {
      tc_fence_after_sync();
      if (real) p.part_ml[part_row(row)] = make_float2(m_run * sl, l_run + l_other);
      // rows leave as 32-byte segments through a padded block of shared memory: two lanes per row, sixteen rows at a time
      float* block = reinterpret_cast<float*>(sStore + (warp - 2) * C::kStoreBlock);
      const int sub = lane >> 1, piece = lane & 1;
      float* dst[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = quarter * 32 + 16 * i + sub;
        dst[i] = r < rows ? p.part_o + part_row(r) * HD + half * (HD / 2) + 4 * piece : nullptr;
      }
#pragma unroll 1
      for (int c = 0; c < HD / 16; ++c) {
        uint32_t ov[8];
        tmem_ld_32x8(o_col + (uint32_t)(c * 8), ov);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<uint4*>(block + lane * C::kStagePitch + 4 * i) = make_uint4(ov[4 * i], ov[4 * i + 1], ov[4 * i + 2], ov[4 * i + 3]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 v = *reinterpret_cast<const uint4*>(block + (16 * i + sub) * C::kStagePitch + 4 * piece);
          if (dst[i] != nullptr) *reinterpret_cast<uint4*>(dst[i] + c * 8) = v;
        }
        __syncwarp();
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(*tmem_slot, C::kTmemCols);
  }
}

template <int HD>
static int launch_prefix(const paged::Launch& a, int shared, int splits, cudaStream_t stream) {
  using C = Cfg<HD>;
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  AJB_CUDA_OK(cudaGetDevice(&dev));
  if (dev >= kMaxDevices || !configured[dev]) {
    AJB_CUDA_OK(cudaFuncSetAttribute(prefix_attention_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    AJB_CUDA_OK(cudaFuncSetAttribute(prefix_attention_kernel<HD>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                     cudaSharedmemCarveoutMaxShared));
    if (dev < kMaxDevices) configured[dev] = true;
  }
  Params p;
  p.q = (const __nv_bfloat16*)a.q; p.table = (const int*)a.block_tables; p.q_pitch = a.q_pitch;
  p.group = a.heads / a.kv_heads; p.inv_group = 1.0f / (float)p.group; p.heads = a.heads; p.rows = a.num_seqs * a.q_total * p.group; p.keys = shared;
  p.pairs = p.rows <= ROWS ? 0 : (p.rows + 2 * ROWS - 1) / (2 * ROWS);
  p.kv_heads = a.kv_heads; p.scale = a.scale;
  p.splits = splits;
  p.part_stride = a.part_stride; p.part_o = (float*)a.part_o; p.part_ml = (float2*)a.part_ml;
  p.status = device_status_buffer();
  const long long grid = (long long)(p.pairs == 0 ? 1 : p.pairs) * p.kv_heads * p.splits;
  AJB_REQUIRE(grid <= 0x7fffffffll, "shared prefix attention: too many query rows");
  return launch_early(prefix_attention_kernel<HD>, dim3((unsigned)grid), dim3(kThreads), C::kSmem, stream, *a.map_k, *a.map_v, p);
}

}  // namespace prefix
}  // namespace ajb

// q [num_seqs * q_len, heads, head_dim] bf16 with q_pitch elements between tokens, out the same, contiguous; the first
// `shared` tokens (a multiple of 16; 0: plain paged attention) of every sequence are the ones that the first row of
// block_tables names. With prefix_tokens > 0 it is pieces of the paged launch, prefix_splits of them for each KV head and
// prefix_tokens query tokens (32 query rows at most); otherwise the prefix kernel divides it over prefix_splits CTAs per
// (256 query rows, KV head). parts = what is left per row: suffix_splits, and prefix_splits more, or twice as many when the
// prefix kernel has at most 128 query rows per KV head and a CTA more than one tile of 128 keys. part_o holds
// num_seqs * q_len * heads * parts * head_dim floats, part_ml two per part.
extern "C" int ajb_shared_prefix_attention(const void* arguments) {
  using namespace ajb;
  const SharedPrefixArgs& args = *static_cast<const SharedPrefixArgs*>(arguments);
  AJB_REQUIRE(args.size == (int)sizeof(args), "shared prefix attention: arguments of %d bytes, not %d", args.size, (int)sizeof(args));
  const auto& [size, q, k_cache, v_cache, block_tables, context_lens, out, q_pitch, num_seqs, num_blocks,
               block_size, max_blocks, heads, kv_heads, head_dim, q_len, shared, scale, prefix_tokens,
               prefix_splits, suffix_splits, parts, part_o, part_ml, stream] = args;
  AJB_REQUIRE(block_size == prefix::BLOCK_TOKENS, "shared prefix attention: cache block size must be %d", prefix::BLOCK_TOKENS);
  AJB_REQUIRE(head_dim == 64 || head_dim == 128, "shared prefix attention: head_dim %d is not supported (64 and 128 are)", head_dim);
  AJB_REQUIRE(kv_heads >= 1 && heads % kv_heads == 0 && heads / kv_heads <= prefix::ROWS && q_len >= 1,
              "shared prefix attention: %d query heads cannot share %d KV heads", heads, kv_heads);
  AJB_REQUIRE(shared >= 0 && shared % prefix::BLOCK_TOKENS == 0 && shared / prefix::BLOCK_TOKENS <= max_blocks,
              "shared prefix attention: %d shared tokens are not whole blocks of the table", shared);
  AJB_REQUIRE((long long)num_seqs * q_len * (heads / kv_heads) <= (1ll << 30), "shared prefix attention: too many query rows");
  const int group = heads / kv_heads, tiles = (shared + prefix::TILE - 1) / prefix::TILE;
  const int rows = num_seqs * q_len * group;      // query rows per KV head
  const bool few = prefix_tokens > 0;             // the paged kernel takes the prefix along
  AJB_REQUIRE(!few || (shared > 0 && prefix_tokens * group <= 32 && q_len * group <= 32),
              "shared prefix attention: CTAs of %d and %d tokens with %d query heads each are too large", prefix_tokens, q_len, group);
  AJB_REQUIRE((prefix_splits > 0) == (shared > 0) && prefix_splits >= 0 && prefix_splits <= (tiles > 0 ? tiles : 0) &&
                  suffix_splits >= 1 && part_o != nullptr && part_ml != nullptr,
              "shared prefix attention: %d and %d divisions of %d shared tokens and of the rest do not fit, or there is no workspace",
              prefix_splits, suffix_splits, shared);
  const int prefix_parts = !few && rows <= prefix::ROWS && prefix_splits < tiles ? 2 * prefix_splits : prefix_splits;
  AJB_REQUIRE(parts == prefix_parts + suffix_splits && parts <= 64, "shared prefix attention: %d parts per row, not %d", parts,
              prefix_parts + suffix_splits);
  AJB_REQUIRE(scale >= 0.99e-30f && scale <= 1000.0f, "shared prefix attention: scale %g is not between 1e-30 and 1e3", (double)scale);
  AJB_REQUIRE(q_pitch % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0, "shared prefix attention: query rows must be 16-byte aligned");
  AJB_REQUIRE((reinterpret_cast<uintptr_t>(out) & 15) == 0, "shared prefix attention: out must be 16-byte aligned");
  if (num_seqs <= 0) return 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  paged::Launch a;
  a.q = q; a.k_cache = k_cache; a.v_cache = v_cache; a.block_tables = block_tables; a.context_lens = context_lens;
  a.q_start = nullptr; a.out = out; a.q_pitch = q_pitch; a.num_seqs = num_seqs; a.num_blocks = num_blocks;
  a.max_blocks = max_blocks; a.heads = heads; a.kv_heads = kv_heads; a.q_total = q_len;
  // up to 32 rows run on the paged kernel that puts the keys on the tensor-core rows; otherwise 128 query rows at a time
  a.q_len = group * q_len <= 32 ? q_len : min(q_len, prefix::ROWS / group);
  a.first_key = shared; a.scale = scale; a.splits = suffix_splits; a.part_stride = parts;
  a.part_base = prefix_parts; a.part_o = part_o; a.part_ml = part_ml; a.beside_previous = shared > 0 && !few;
  a.prefix_splits = few ? prefix_splits : 0;
  a.prefix_tokens = prefix_tokens;
  a.early = few;
  CUtensorMap map_k, map_v;
  int rc = make_tensor_map_cache(&map_k, a.k_cache, a.num_blocks, a.kv_heads, head_dim);
  if (rc == 0) rc = make_tensor_map_cache(&map_v, a.v_cache, a.num_blocks, a.kv_heads, head_dim);
  if (rc) return rc;
  a.map_k = &map_k;
  a.map_v = &map_v;
  if (shared > 0 && !few)
    rc = head_dim == 128 ? prefix::launch_prefix<128>(a, shared, prefix_splits, s) : prefix::launch_prefix<64>(a, shared, prefix_splits, s);
  if (rc == 0) rc = paged::launch(a, head_dim, s);
  if (rc == 0) rc = paged::merge_parts(a, head_dim, s);
  return rc;
}
