// Arguments of the serving entry points that take them in one structure; ops/native.py packs the same layouts.
#pragma once

struct BatchMapsArgs {
  int size;                 // of the structure: a caller with another layout is refused
  const void *ids, *counts, *cached, *q_lens;
  int n_ids, seqs, total, width, block_size, pad;
  void *tables, *positions, *slots, *q_start, *context, *stream;
};

struct SharedPrefixArgs {
  int size;
  const void *q, *k_cache, *v_cache, *block_tables, *context_lens;
  void *out;
  long long q_pitch;
  int num_seqs, num_blocks, block_size, max_blocks, heads, kv_heads, head_dim, q_len, shared;
  float scale;
  int prefix_tokens, prefix_splits, suffix_splits, parts;
  void *part_o, *part_ml, *stream;
};

struct ProcessLogitsArgs {
  int size;
  const void *logits;
  int dtype;
  long long in_pitch;
  void *out;
  int rows, vocab;
  const void *history;
  long long history_pitch;
  int history_width;
  const void *prompt_lens, *history_lens, *repetition, *presence, *frequency, *bias_ids, *bias_values;
  int biases;
  const void *mask;
  long long mask_pitch;
  void *stream;
};
