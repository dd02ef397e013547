// Internal interface of the paged-attention kernel, for operators that combine it with parts of their own.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace ajb {
namespace paged {

struct Launch {
  const void *q, *k_cache, *v_cache, *block_tables, *context_lens;
  const void* q_start;          // null: sequence i's rows start at i * q_total
  void* out;
  long long q_pitch;            // elements between two tokens of q
  int num_seqs, num_blocks, max_blocks, heads, kv_heads;
  int q_len;                    // tokens of a sequence that one CTA takes
  int q_total;                  // new tokens per sequence
  int first_key;                // cached tokens in front of this one are left out (a multiple of the block size)
  float scale;
  int splits;                   // parts this launch leaves per row
  int prefix_splits;            // > 0: this launch also covers the keys in front of first_key, the same for all sequences (row 0
                                // of the tables), divided in that many parts per row, which come first; at most 32 query
  int prefix_tokens;            // rows per CTA: so many tokens of the batch for these keys, q_len tokens of a sequence for its own
  int part_stride, part_base;   // parts per row in the workspace, first one of this launch; stride 0: no parts, `out` is written
  void *part_o, *part_ml;
  const CUtensorMap *map_k, *map_v;   // of make_tensor_map_cache, when the caller has them already (else null)
  bool early;                   // may start before the launch in front of it has ended, and waits for that (up to 32 rows per CTA)
  bool beside_previous;         // may start while the launch in front of it still runs (which must have said so)
};

int launch(const Launch& a, int head_dim, cudaStream_t stream);
// out = the log-sum-exp weighted sum of all a.part_stride parts
int merge_parts(const Launch& a, int head_dim, cudaStream_t stream);

}  // namespace paged
}  // namespace ajb
