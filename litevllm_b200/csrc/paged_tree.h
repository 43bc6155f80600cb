// Parameters and launchers of the drafted-tree / 8-bit-cache attention
// kernel (paged_tree.cuh), one launcher per cache format so that the
// instantiations compile in separate files.
#pragma once

#include "lk_host.h"

namespace lk {

struct TreeParams {
  void* out;
  int64_t out_stride;           // elements between tokens of out
  const void* q;
  int64_t q_stride;
  const void* k;                // [num_blocks, bs, H_kv, D], 16-bit or bytes
  const void* v;
  const float* k_scale;         // [num_blocks, H_kv, bs] (8-bit caches)
  const float* v_scale;
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* context_lens;
  const int32_t* cu_seqlens_q;  // NULL: one query per sequence (decode)
  const int64_t* mask;          // [T, mask_stride] bit words; NULL: causal chain
  int64_t mask_stride;
  int mask_words;
  int32_t* status;
  int T;                        // rows of q and out
  int B, H_kv, G, bs, max_blocks;
  uint32_t bs_mul;              // key / bs: key >> bs_shift if 0, else umulhi(key, bs_mul) >> bs_shift
  int bs_shift;
  int64_t num_blocks;
  int max_q;                    // most query tokens of a sequence
  float scale_log2;             // scale * log2(e)
  int cluster;                  // > 1: a unit's splits are one cluster of that many CTAs
  int chunk;                    // keys per split (cluster: set by each context)
  int nsplit;                   // 1: every CTA writes out itself
  float4* part_ml;              // [T * H][nsplit]: m, l, M, unused
  float* part_o;                // [T * H][nsplit][D]
};

// NT (1, 2, 4): groups of eight query rows a CTA takes.
int tree_launch_16(const TreeParams& p, int dtype, int D, int NT, unsigned grid, cudaStream_t s);
int tree_launch_i8(const TreeParams& p, int dtype, int D, int NT, unsigned grid, cudaStream_t s);
int tree_launch_e4m3(const TreeParams& p, int dtype, int D, int NT, unsigned grid, cudaStream_t s);

}  // namespace lk
