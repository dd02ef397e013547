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
// (S = Q K^T, softmax, O += P V with S, P and O in tensor memory, P written over the scores it came from): while four
// warps turn one stream's scores into probabilities, the tensor pipe runs the other's products. A 128 x 128 step is two
// products of 512 cycles and 16384 exponentials, 1024 cycles of the SM's exponential unit, so the two streams keep both
// about equally busy. The streams are two row tiles that share every K and V tile; when all rows fit one tile they are
// two halves of the keys instead (even and odd tiles, two parts).
//
// A prefix CTA has an SM to itself (shared memory), the suffix launch, which does not read what this one writes, starts
// as soon as every CTA here has and takes the other SMs: the prefix is bound by arithmetic, the suffix by memory, and
// the number of prefix CTAs divides the SMs so that both last about as long.
#include "common.cuh"
#include "paged_attention.h"

namespace ajb {
namespace prefix {

constexpr int TILE = 128;          // keys per step
constexpr int ROWS = 128;          // query rows of a stream
constexpr int BLOCK_TOKENS = 16;   // tokens per cache block
constexpr int kThreads = 384;      // TMA warp, product warp, two idle, 2 x 4 softmax warps (one per tensor-memory quarter)
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kPrefixKernelId = 12;
constexpr int kMaxParts = 32;      // parts of the prefix; as many again behind it

template <int HD>
struct Cfg {
  static constexpr int kTile = TILE * HD * 2;            // Q, one K tile, one V tile: same size
  static constexpr int kStages = HD == 64 ? 5 : 2;       // K and V tiles held at a time
  static constexpr int kStagePitch = 20;                 // floats per row of a store block: 16 columns and 16 bytes of padding
  static constexpr int kStoreBlock = 32 * kStagePitch * 4;
  static constexpr int kSmem = kTile * (2 + 2 * kStages) + 8 * kStoreBlock + 512;
  static constexpr int kOCol = 2 * TILE;                 // S (and P) of stream s at s * 128, O behind them
  static constexpr int kTmemCols = 512;
  // a CTA of the suffix launch on the same SM would wait for its tensor memory until this one leaves: it must not fit
  static_assert(kSmem + 64 * HD * 2 * 4 + ROWS * HD * 2 + ROWS * 64 * 2 > 227 * 1024, "a suffix CTA would fit beside");
};

struct Params {
  const __nv_bfloat16* q;
  const int* table;             // block ids of the prefix
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
  uint64_t* bars = reinterpret_cast<uint64_t*>(sStore + 8 * C::kStoreBlock);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (smem_misaligned(smem, p.status, kPrefixKernelId, reinterpret_cast<uint32_t*>(bars) + 120)) return;
  uint64_t* k_full = bars;               // kStages (<= 5)
  uint64_t* k_empty = bars + 5;
  uint64_t* v_full = bars + 10;
  uint64_t* v_empty = bars + 15;
  uint64_t* s_full = bars + 20;          // per stream
  uint64_t* p_ready = bars + 22;
  uint64_t* pv_done = bars + 24;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 26);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
  const int steps[2] = {steps_of(0), steps_of(1)};

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_ready[s], 4);
      mbar_init(&pv_done[s], 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tensor_map(&map_k);
    prefetch_tensor_map(&map_v);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  const int stream = warp >> 2 == 2 ? 1 : 0;             // of a softmax warp (4..7, 8..11)
  if (warp >= 4 && (paired || stream == 0)) {
    // query rows: HD / 8 neighbouring threads per row; rows past the last are zero
    constexpr int kChunks = HD / 8;
    const int row0 = row0_of(stream), rows = p.rows - row0;
#pragma unroll 4
    for (int i = threadIdx.x & 127; i < ROWS * kChunks; i += 128) {
      const int r = i / kChunks, ch = i % kChunks;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < rows) {
        const int token = (row0 + r) / p.group, h = (row0 + r) % p.group;
        v = reinterpret_cast<const uint4*>(p.q + (size_t)token * p.q_pitch + (size_t)(kv_head * p.group + h) * HD)[ch];
      }
      store_chunk(sQ + stream * C::kTile, r, ch, v);
    }
    fence_proxy_async_smem();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // block ids: eight per tile, four tiles by the 32 lanes of one coalesced load, a group of tiles ahead. K tiles run
    // one ahead of V tiles: a K slot is free again long before the V slot of the same tile.
    constexpr int kBlocksPerTile = TILE / BLOCK_TOKENS;
    constexpr int kTilesPerGroup = 32 / kBlocksPerTile;
    const int last_block = p.keys / BLOCK_TOKENS - 1;
    auto fetch_ids = [&](int g) { return p.table[min(last_block, (t0 + g * kTilesPerGroup) * kBlocksPerTile + lane)]; };
    int ids_next = n_tiles > 0 ? fetch_ids(0) : 0, ids_k = ids_next, ids_prev = ids_next, k_group = -1;
    bool ok = true;
    auto load = [&](int t, int ids, uint8_t* ring, uint64_t* full, uint64_t* empty, const CUtensorMap* map, int stage_id) {
      int id[kBlocksPerTile];
#pragma unroll
      for (int b = 0; b < kBlocksPerTile; ++b) id[b] = __shfl_sync(0xffffffffu, ids, (t % kTilesPerGroup) * kBlocksPerTile + b);
      if (lane == 0 && ok) {
        const int s = t % kStages;
        ok = mbar_wait_compact(&empty[s], ((uint32_t)(t / kStages) & 1) ^ 1, abort_flag, p.status, kPrefixKernelId, stage_id);
        if (ok) {
          mbar_arrive_expect_tx(&full[s], C::kTile);
#pragma unroll
          for (int b = 0; b < kBlocksPerTile; ++b) {
#pragma unroll
            for (int i = 0; i < HD / 64; ++i)
              tma_load_3d(ring + s * C::kTile + i * (TILE * 128) + b * (BLOCK_TOKENS * 128), map, &full[s], kv_head * HD + 64 * i, 0, id[b]);
          }
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
    };
    for (int t = 0; t <= n_tiles && ok; ++t) {
      if (t < n_tiles) {
        if (t % kTilesPerGroup == 0) {
          ids_prev = ids_k;
          ids_k = ids_next;
          k_group = t / kTilesPerGroup;
          if (t + kTilesPerGroup < n_tiles) ids_next = fetch_ids(k_group + 1);
        }
        load(t, ids_k, sK, k_full, k_empty, &map_k, 1);
      }
      if (t >= 1) load(t - 1, (t - 1) / kTilesPerGroup == k_group ? ids_k : ids_prev, sV, v_full, v_empty, &map_v, 2);
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc_s = make_idesc(ROWS, TILE, 1, false, false);
    constexpr uint32_t idesc_o = make_idesc(ROWS, HD, 1, false, true);
    const uint32_t q_km0 = desc_lo_k_major(smem_u32(sQ));
    const uint32_t k_km0 = desc_lo_k_major(smem_u32(sK));
    const uint32_t v_mn0 = desc_lo_mn_major(smem_u32(sV), TILE * 128);
    constexpr uint32_t kStep = C::kTile >> 4;
    const bool both = paired && steps[1] > 0;            // both streams use every tile; stream 1 comes second
    auto issue_s = [&](int s, int i) -> bool {
      const int t = paired ? i : 2 * i + s, slot = t % kStages;
      // S overwrites P(i - 1): the product that reads it was issued before, and the tensor pipe runs in issue order
      if (!mbar_wait_compact(&k_full[slot], (uint32_t)(t / kStages) & 1, abort_flag, p.status, kPrefixKernelId, 3)) return false;
      tc_fence_after_sync();
      if (lane == 0) {
        const uint32_t k_km = k_km0 + (uint32_t)slot * kStep, q_km = q_km0 + (paired ? (uint32_t)s * kStep : 0u);
        const uint32_t d = tmem_base + (uint32_t)(s * TILE);
        umma_f16_c<false>(d, desc_at(q_km, 0), desc_at(k_km, 0), idesc_s);
#pragma unroll
        for (int k = 1; k < HD / 16; ++k)
          umma_f16_c<true>(d, desc_at(q_km, k_major_step(k, ROWS * 128)), desc_at(k_km, k_major_step(k, TILE * 128)), idesc_s);
        tc_commit(&s_full[s]);
        if (!both || s == 1) tc_commit(&k_empty[slot]);
      }
      __syncwarp();
      return true;
    };
    bool ok = true;
    for (int s = 0; s < 2; ++s)
      if (steps[s] > 0 && ok) ok = issue_s(s, 0);
    for (int i = 0; i < steps[0] && ok; ++i) {           // stream 0 never has fewer steps than stream 1
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if (i >= steps[s] || !ok) continue;
        const int t = paired ? i : 2 * i + s, slot = t % kStages;
        if (!mbar_wait_compact(&p_ready[s], (uint32_t)i & 1, abort_flag, p.status, kPrefixKernelId, 4)) { ok = false; break; }
        if (!mbar_wait_compact(&v_full[slot], (uint32_t)(t / kStages) & 1, abort_flag, p.status, kPrefixKernelId, 5)) { ok = false; break; }
        tc_fence_after_sync();
        if (lane == 0) {
          const uint32_t v_mn = v_mn0 + (uint32_t)slot * kStep;
          const uint32_t o = tmem_base + (uint32_t)(C::kOCol + s * HD), pr = tmem_base + (uint32_t)(s * TILE);
          umma_f16_ts(o, pr, desc_at(v_mn, 0), idesc_o, i != 0);
#pragma unroll
          for (int k = 1; k < TILE / 16; ++k) umma_f16_ts_c<true>(o, pr + (uint32_t)(k * 8), desc_at(v_mn, mn_major_step(k)), idesc_o);
          tc_commit(&pv_done[s]);
          if (!both || s == 1) tc_commit(&v_empty[slot]);
        }
        __syncwarp();
        if (i + 1 < steps[s]) ok = issue_s(s, i + 1);
      }
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int row0 = row0_of(stream), rows = p.rows - row0;      // rows may pass 128: then all of this tile's are real
    const int n = steps[stream];
    const bool active = quarter * 32 < rows;           // warp-uniform: quarters without query rows only keep the pace
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_col = tmem_base + lane_addr + (uint32_t)(stream * TILE);
    const uint32_t o_col = tmem_base + lane_addr + (uint32_t)(C::kOCol + stream * HD);
    const float sl = p.scale * kLog2e;
    float m_run = -INFINITY, l_run = 0.0f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      if (!mbar_wait_compact(&s_full[stream], (uint32_t)j & 1, abort_flag, p.status, kPrefixKernelId, 6)) { ok = false; break; }
      const int t = paired ? j : 2 * j + stream;
      const int left = p.keys - (t0 + t) * TILE;        // keys of this tile; the last tile may have fewer than 128
      if (left < TILE) {
        // the blocks that fill the tile up are copies of the last one: their probabilities are zero, and zero times an
        // infinity must not reach the sums (paired streams both write the same zeros)
        const int slot = t % kStages;
        if (!mbar_wait_compact(&v_full[slot], (uint32_t)(t / kStages) & 1, abort_flag, p.status, kPrefixKernelId, 9)) { ok = false; break; }
        for (int i = left * 8 + row; i < TILE * 8; i += 128) {
#pragma unroll
          for (int b = 0; b < HD / 64; ++b)
            reinterpret_cast<uint4*>(sV + slot * C::kTile + b * (TILE * 128))[i] = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
      }
      if (active) {
        tc_fence_after_sync();
        uint32_t sv[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32(s_col + (uint32_t)(c * 32), sv[c]);
        tc_wait_ld();
        if (left < TILE) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c * 32 + i >= left) sv[c][i] = 0xff800000u;      // -inf
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) m4[i & 3] = fmaxf(m4[i & 3], __uint_as_float(sv[c][i]));
        const float m_tile = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        // lazy reference maximum (see flash_fwd.cu): O is rescaled only when a row would pass 2^8
        const bool moved = (m_tile - m_run) * sl > 8.0f;
        const float m_new = moved ? m_tile : m_run;
        const float m_safe = (m_new == -INFINITY) ? 0.0f : m_new;
        const float alpha = moved ? exp2f((m_run - m_safe) * sl) : 1.0f;
        const float neg = -m_safe * sl;
        float l2[2] = {0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
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
          if (!mbar_wait_compact(&pv_done[stream], (uint32_t)(j - 1) & 1, abort_flag, p.status, kPrefixKernelId, 7)) { ok = false; break; }
          tc_fence_after_sync();
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t ov[32];
            tmem_ld_32x32(o_col + (uint32_t)(c * 32), ov);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
            tmem_st_32x32(o_col + (uint32_t)(c * 32), ov);
          }
        }
        tc_wait_st();
        tc_fence_before_sync();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[stream]);
    }
    const int part = paired ? split : 2 * split + stream;
    auto part_row = [&](int r) {
      const int token = (row0 + r) / p.group, h = (row0 + r) % p.group;
      return ((size_t)token * p.heads + kv_head * p.group + h) * p.part_stride + part;
    };
    const bool real = row < rows;
    if (real && (n == 0 || !ok)) p.part_ml[part_row(row)] = make_float2(0.0f, 0.0f);       // nothing to join from this part
    if (ok && active && n > 0 && mbar_wait_compact(&pv_done[stream], (uint32_t)(n - 1) & 1, abort_flag, p.status, kPrefixKernelId, 8)) {
      tc_fence_after_sync();
      if (real) p.part_ml[part_row(row)] = make_float2(m_run * sl, l_run);
      // rows leave as 64-byte segments through a padded block of shared memory: four lanes per row, eight rows at a time
      float* block = reinterpret_cast<float*>(sStore + (warp - 4) * C::kStoreBlock);
      const int sub = lane >> 2, piece = lane & 3;
      float* dst[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = quarter * 32 + 8 * i + sub;
        dst[i] = r < rows ? p.part_o + part_row(r) * HD + 4 * piece : nullptr;
      }
#pragma unroll 1
      for (int c = 0; c < HD / 16; ++c) {
        uint32_t ov[16];
        tmem_ld_32x16(o_col + (uint32_t)(c * 16), ov);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<uint4*>(block + lane * C::kStagePitch + 4 * i) = make_uint4(ov[4 * i], ov[4 * i + 1], ov[4 * i + 2], ov[4 * i + 3]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 v = *reinterpret_cast<const uint4*>(block + (8 * i + sub) * C::kStagePitch + 4 * piece);
          if (dst[i] != nullptr) *reinterpret_cast<uint4*>(dst[i] + c * 16) = v;
        }
        __syncwarp();
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
}

template <int HD>
static int launch_prefix(const paged::Launch& a, int shared, int parts, cudaStream_t stream) {
  using C = Cfg<HD>;
  CUtensorMap map_k, map_v;
  const uint64_t row_pitch = (uint64_t)a.kv_heads * HD * 2;
  int rc = make_tensor_map_3d(&map_k, a.k_cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.num_blocks, BLOCK_TOKENS,
                              (uint64_t)a.kv_heads * HD, row_pitch * BLOCK_TOKENS, row_pitch, BLOCK_TOKENS, 64);
  if (rc) return rc;
  rc = make_tensor_map_3d(&map_v, a.v_cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.num_blocks, BLOCK_TOKENS,
                          (uint64_t)a.kv_heads * HD, row_pitch * BLOCK_TOKENS, row_pitch, BLOCK_TOKENS, 64);
  if (rc) return rc;
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
  p.group = a.heads / a.kv_heads; p.heads = a.heads; p.rows = a.num_seqs * a.q_total * p.group; p.keys = shared;
  p.pairs = p.rows <= ROWS ? 0 : (p.rows + 2 * ROWS - 1) / (2 * ROWS);
  p.kv_heads = a.kv_heads; p.scale = a.scale;
  p.splits = p.pairs == 0 ? parts / 2 : parts;
  p.part_stride = a.part_stride; p.part_o = (float*)a.part_o; p.part_ml = (float2*)a.part_ml;
  p.status = device_status_buffer();
  const long long grid = (long long)(p.pairs == 0 ? 1 : p.pairs) * p.kv_heads * p.splits;
  AJB_REQUIRE(grid <= 0x7fffffffll, "shared prefix attention: too many query rows");
  prefix_attention_kernel<HD><<<(int)grid, kThreads, C::kSmem, stream>>>(map_k, map_v, p);
  AJB_CUDA_OK(cudaGetLastError());
  return 0;
}

}  // namespace prefix
}  // namespace ajb

// q [num_seqs * q_len, heads, head_dim] bf16 with q_pitch elements between tokens, out the same, contiguous; the first
// `shared` tokens (a multiple of 16; 0: plain paged attention) of every sequence are the ones that the first row of
// block_tables names.
// part_o holds num_seqs * q_len * heads * (prefix_parts + suffix_parts) * head_dim floats, part_ml two per part.
extern "C" int ajb_shared_prefix_attention(const void* q, const void* k_cache, const void* v_cache, const void* block_tables,
                                           const void* context_lens, void* out, long long q_pitch, int num_seqs,
                                           int num_blocks, int block_size, int max_blocks, int heads, int kv_heads,
                                           int head_dim, int q_len, int shared, float scale, int prefix_parts,
                                           int suffix_parts, void* part_o, void* part_ml, void* stream) {
  using namespace ajb;
  AJB_REQUIRE(block_size == prefix::BLOCK_TOKENS, "shared prefix attention: cache block size must be %d", prefix::BLOCK_TOKENS);
  AJB_REQUIRE(head_dim == 64 || head_dim == 128, "shared prefix attention: head_dim %d is not supported (64 and 128 are)", head_dim);
  AJB_REQUIRE(kv_heads >= 1 && heads % kv_heads == 0 && heads / kv_heads <= prefix::ROWS && q_len >= 1,
              "shared prefix attention: %d query heads cannot share %d KV heads", heads, kv_heads);
  AJB_REQUIRE(shared >= 0 && shared % prefix::BLOCK_TOKENS == 0 && shared / prefix::BLOCK_TOKENS <= max_blocks,
              "shared prefix attention: %d shared tokens are not whole blocks of the table", shared);
  const bool one_tile = (long long)num_seqs * q_len * (heads / kv_heads) <= prefix::ROWS;
  AJB_REQUIRE(!one_tile || prefix_parts % 2 == 0, "shared prefix attention: up to %d query rows per KV head leave their parts in pairs",
              prefix::ROWS);
  AJB_REQUIRE((prefix_parts > 0) == (shared > 0) && prefix_parts >= 0 && prefix_parts <= prefix::kMaxParts && suffix_parts >= 1 && suffix_parts <= prefix::kMaxParts &&
                  part_o != nullptr && part_ml != nullptr,
              "shared prefix attention: parts must be in [1, %d] (none of a prefix of length 0) and come with a workspace", prefix::kMaxParts);
  AJB_REQUIRE(q_pitch % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0, "shared prefix attention: query rows must be 16-byte aligned");
  AJB_REQUIRE((long long)num_seqs * q_len * (heads / kv_heads) <= (1ll << 30), "shared prefix attention: too many query rows");
  if (num_seqs <= 0) return 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int group = heads / kv_heads;
  paged::Launch a;
  a.q = q; a.k_cache = k_cache; a.v_cache = v_cache; a.block_tables = block_tables; a.context_lens = context_lens;
  a.q_start = nullptr; a.out = out; a.q_pitch = q_pitch; a.num_seqs = num_seqs; a.num_blocks = num_blocks;
  a.max_blocks = max_blocks; a.heads = heads; a.kv_heads = kv_heads; a.q_total = q_len;
  // up to 32 rows the paged kernel works with four replicas of them (cheaper per step); otherwise 128 rows at a time
  a.q_len = group * q_len <= 32 ? q_len : min(q_len, prefix::ROWS / group);
  a.first_key = shared; a.scale = scale; a.splits = suffix_parts; a.part_stride = prefix_parts + suffix_parts;
  a.part_base = prefix_parts; a.part_o = part_o; a.part_ml = part_ml; a.beside_previous = shared > 0;
  int rc = 0;
  if (shared > 0)
    rc = head_dim == 128 ? prefix::launch_prefix<128>(a, shared, prefix_parts, s) : prefix::launch_prefix<64>(a, shared, prefix_parts, s);
  if (rc == 0) rc = paged::launch(a, head_dim, s);
  if (rc == 0) rc = paged::merge_parts(a, head_dim, s);
  return rc;
}
