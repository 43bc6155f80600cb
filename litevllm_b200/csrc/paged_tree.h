// Parameters and launchers of the drafted-tree / 8-bit-cache attention kernels
// (paged_tree.cuh on mma.sync, paged_tree_tc.cuh on tcgen05), one launcher per
// cache format so that the instantiations compile in separate files.
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
  uint32_t g_mul;               // row / G in the same way
  int g_shift;
  int64_t num_blocks;
  int max_q;                    // most query tokens of a sequence
  float scale_log2;             // scale * log2(e)
  int cluster;                  // > 1: a unit's splits are one cluster of that many CTAs
  int chunk;                    // keys per split (cluster: set by each context)
  int nsplit;                   // 1: every CTA writes out itself
  float4* part_ml;              // [T * H][nsplit]: m, l, M, unused
  float* part_o;                // [T * H][nsplit][D]
};

#ifdef __CUDACC__
// Query tokens of sequence b, rows row0 .. of q. A cu_seqlens_q that passes q or max_q is
// flagged and cut to what lies inside both. In 64 bits: the difference of two entries and
// the end of the rows may pass 32.
__device__ __forceinline__ int tree_tokens(const TreeParams& p, int b, int* row0) {
  *row0 = b;
  if (!p.cu_seqlens_q) return 1;
  const int64_t first = p.cu_seqlens_q[b];
  const int64_t count = p.cu_seqlens_q[b + 1] - first;
  *row0 = static_cast<int>(first);
  if (count <= p.max_q && first >= 0 && first + count <= p.T)
    return static_cast<int>(max(count, static_cast<int64_t>(0)));
  if (threadIdx.x == 0 && p.status) atomicOr(p.status, LK_STATUS_CTX_OOB);
  if (first < 0 || first >= p.T || count <= 0) return 0;
  return static_cast<int>(min(min(count, static_cast<int64_t>(p.max_q)), p.T - first));
}
// key / p.bs, key < 2^31.
__device__ __forceinline__ int tree_quotient(const TreeParams& p, int key) {
  return static_cast<int>(p.bs_mul ? __umulhi(key, p.bs_mul) >> p.bs_shift
                                   : static_cast<uint32_t>(key) >> p.bs_shift);
}
// Query token of a KV head's query row, row / G.
__device__ __forceinline__ int tree_token(const TreeParams& p, int row) {
  return static_cast<int>(p.g_mul ? __umulhi(row, p.g_mul) >> p.g_shift
                                  : static_cast<uint32_t>(row) >> p.g_shift);
}
#endif

// NT (1, 2, 4): groups of eight query rows a CTA takes; 0: the tcgen05 kernel.
int tree_launch_16(const TreeParams& p, int dtype, int D, int NT, unsigned grid, cudaStream_t s);
int tree_launch_i8(const TreeParams& p, int dtype, int D, int NT, unsigned grid, cudaStream_t s);
int tree_launch_e4m3(const TreeParams& p, int dtype, int D, int NT, unsigned grid, cudaStream_t s);

}  // namespace lk
