// Entry points of drafted-tree attention and of decode over an 8-bit cache:
// argument checks, the split plan and the kernel that joins the splits. The
// attention kernel itself is in paged_tree.cuh.
#include <algorithm>

#include "lk_common.cuh"
#include "paged_tree.h"

namespace lk {
namespace {

struct JoinParams {
  void* out;
  int64_t out_stride;
  const float4* part_ml;  // [T * H][nsplit]: m, l, M
  const float* part_o;    // [T * H][nsplit][D]
  const int32_t* cu_seqlens_q;
  const int32_t* context_lens;
  uint32_t rows;  // T * H
  int B, H, nsplit, chunk, max_keys, max_q;
};

template <typename T> LK_DEVINL T join_round(float x);
template <> LK_DEVINL __nv_bfloat16 join_round<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> LK_DEVINL __half join_round<__half>(float x) { return __float2half_rn(x); }

// out = sum_s O_s 2^(M_s - M) / sum_s l_s 2^(m_s - m) * 2^(M - m), in split
// order whatever order the splits ended in. Four warps: a query row each where rows
// are many and splits few (29K rows of up to four: 17 us from a cold cache, 21 with a
// CTA per row), else all four on one row, W = 4 (256 rows of up to eight: 7.0 and 9.5).
template <typename T, int D, int W>
__global__ void __launch_bounds__(128) tree_join_kernel(const JoinParams p) {
  pdl_wait();
  const uint32_t row = W > 1 ? blockIdx.x : blockIdx.x * 4u + (threadIdx.x >> 5);  // < 2^31 + 4
  if (row >= p.rows) return;
  const int t = row / static_cast<uint32_t>(p.H), h = row - t * static_cast<uint32_t>(p.H);
  int b = t;
  if (p.cu_seqlens_q) {
    if (t < p.cu_seqlens_q[0] || t >= p.cu_seqlens_q[p.B]) return;
    int lo = 0, hi = p.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.cu_seqlens_q[mid] <= t) lo = mid;
      else hi = mid;
    }
    b = lo;
    if (t - p.cu_seqlens_q[b] >= p.max_q) return;  // not computed
  }
  const int ctx = max(min(p.context_lens[b], p.max_keys), 0);
  const int ns = (ctx + p.chunk - 1) / p.chunk;
  if (ns <= 1) return;  // written by its only split
  const int warp = W > 1 ? threadIdx.x >> 5 : 0, lane = threadIdx.x & 31;
  const float4* ml = p.part_ml + static_cast<int64_t>(row) * p.nsplit;
  float a = -3.402823466e38f, A = a;
  for (int s = lane; s < ns; s += 32) {
    const float4 w = ml[s];
    a = fmaxf(a, w.x);
    A = fmaxf(A, w.z);
  }
  a = warp_max(a);
  A = warp_max(A);
  constexpr int V = D / 32;
  float acc[V], L = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int s = warp; s < ns; s += W) {
    const float4 w = ml[s];
    const float f = ex2_mufu(w.z - A);
    L += w.y * ex2_mufu(w.x - a);
    const float* po = p.part_o + (static_cast<int64_t>(row) * p.nsplit + s) * D + lane * V;
    __align__(16) float x[V];
    if constexpr (V == 4) *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(po);
    else *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(po);
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] += x[i] * f;
  }
  if constexpr (W > 1) {
    __shared__ float sm[W][D + 1];
#pragma unroll
    for (int i = 0; i < V; ++i) sm[warp][lane * V + i] = acc[i];
    if (lane == 0) sm[warp][D] = L;
    __syncthreads();
    if (warp != 0) return;
    L = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      L += sm[w][D];
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += sm[w][lane * V + i];
    }
  }
  const float fin = exp2f(A - a) / L;
  T* dst = static_cast<T*>(p.out) + t * p.out_stride + h * D + lane * V;
#pragma unroll
  for (int i = 0; i < V; ++i) dst[i] = join_round<T>(acc[i] * fin);
}

struct Plan {
  int NT, cluster, chunk, nsplit;  // NT 0: the tcgen05 kernel
  int64_t grid;
};

// How a call is cut into CTAs, from its sizes alone (contexts are on the device;
// `keys`, the table's width, bounds them). A unit is (sequence, KV head, group of
// query rows). Measured on B200, 8 KV heads, G = 4, D = 128, graph-replayed, in us.
//  * The tcgen05 kernel (128 rows a CTA) where a key row meets more than 16 query rows
//    (32 x 1000, 24 rows: 16-bit 27 and 33 on mma.sync, int8 32 and 35; 16 rows: 27 and
//    28, 32 and 25) and the whole call outweighs its longer set-up (1 x 4000, 128 rows:
//    16 and 28; 8 x 512, 64 rows: 16 and 14; 1 x 256, 256 rows: 12 and 9). Its TMA boxes
//    want block sizes that are multiples of 16: with others wide trees stay on mma.sync
//    (16 x 1K-8K, 192-256 rows, int8: blocks of 24 441 us, of 16 200).
//  * Else NT, the smallest of 1, 2, 4 whose 8 NT rows hold a KV head's, or a smaller
//    one while its units still leave room on the SMs: a warp with fewer accumulators
//    is faster, and re-reads come from L2 (16 rows, 8 x 1000: NT 1 13.3, NT 2 13.8;
//    16 x 4000: 59.8 and 47.5).
//  * Contexts are cut while one wave of CTAs has room for the pieces: pieces of one
//    wave share HBM evenly and end together (decode, 8 x 16K-32K, int8: 4096 keys a
//    piece 70, 1024 keys 81), and every CTA pays 3 to 4 us of latencies. A piece is at
//    least 256 keys and at most 1 MB of rows, which a CTA alone on its SM streams in
//    about 30 us (tcgen05: 2048 keys), so that one long context in a batch does not
//    outlast the others by more (48-64 nodes, 16 x 1K-8K, int8: 206 then, at 1024 keys 228, at 4096 234).
//  * Pieces of short contexts (a table of at most 2048 keys) with four or more to a
//    unit are a cluster, else the workspace and the joining kernel hold them (decode,
//    1 x 1000: cluster 7.0, joined 7.8, and 5 us less host time for the second launch
//    and the workspace; 8 x 4000: 19.0 and 17.6).
Plan plan_of(int B, int max_q, int H, int H_kv, int D, int fmt, int bs, int max_blocks) {
  auto round_up = [](int64_t x, int64_t m) { return (x + m - 1) / m * m; };
  Plan r;
  const int64_t rows = static_cast<int64_t>(max_q) * (H / H_kv);
  const int64_t heads = static_cast<int64_t>(B) * H_kv;
  const int64_t keys = std::max<int64_t>(1, static_cast<int64_t>(max_blocks) * bs);
  int64_t units = 0, slots = 0;  // resident CTAs
  if (rows > 16 && bs % 16 == 0 && heads * keys * rows > (2 << 20)) {
    r.NT = 0;
    units = heads * ((rows + 127) / 128);
    slots = 2 * num_sms();
  } else {
    for (r.NT = 1;; r.NT *= 2) {
      units = heads * ((rows + 8 * r.NT - 1) / (8 * r.NT));
      slots = static_cast<int64_t>(num_sms()) * (r.NT == 1 ? 3 : 2);
      if (r.NT == 4 || rows <= 8 * r.NT || (r.NT == 1 ? 2 : 1) * units <= slots) break;
    }
  }
  const int64_t per = std::max<int64_t>(1, slots / units);  // pieces of a unit in one wave
  r.cluster = 1;
  if (r.NT > 0 && keys <= 2048 && per >= 4)
    while (r.cluster < 8 && r.cluster * 2 <= per && keys > 128 * r.cluster) r.cluster *= 2;
  if (r.cluster > 1) {
    r.nsplit = 1;
    r.chunk = 0;
    r.grid = units * r.cluster;
    return r;
  }
  const int64_t cap = r.NT == 0 ? 2048 : (1 << 20) / (2 * D * (fmt == LK_KV_16BIT ? 2 : 1));
  int64_t chunk = round_up((keys + per - 1) / per, 64);
  chunk = std::min(std::max<int64_t>(chunk, 256), cap);
  // a wide table of a large batch: no more than 65536 CTAs, most of them empty
  const int64_t most = std::max<int64_t>(1, 65536 / units);
  chunk = std::max(chunk, round_up((keys + most - 1) / most, 64));
  r.chunk = static_cast<int>(std::min<int64_t>(chunk, 1 << 30));
  r.nsplit = static_cast<int>((keys + r.chunk - 1) / r.chunk);
  r.grid = units * r.nsplit;
  return r;
}

size_t plan_bytes(const Plan& r, int64_t T, int H, int D) {
  return r.nsplit == 1 ? 0 : static_cast<size_t>(T) * H * r.nsplit * (D + 4) * 4;
}

template <typename T, int D>
cudaError_t join(const JoinParams& j, unsigned rows, cudaStream_t s) {
  if (j.nsplit <= 8 && rows > 2048)
    return launch_after_previous(tree_join_kernel<T, D, 1>, dim3((rows + 3) / 4), dim3(128), 0, s, j);
  return launch_after_previous(tree_join_kernel<T, D, 4>, dim3(rows), dim3(128), 0, s, j);
}

// Multiplier and shift for exact quotients by d of numbers below 2^31 (0: a shift
// alone). With l = ceil(log2 d), m = floor(2^(31 + l) / d) + 1 < 2^32 exceeds
// 2^(31 + l) / d by at most 1, so x m / 2^(31 + l) passes x / d by less than 1 / d.
void divisor(int d, uint32_t* mul, int* shift) {
  int l = 0;
  while ((1LL << l) < d) ++l;
  const bool power = (1LL << l) == d;
  *mul = power ? 0u : static_cast<uint32_t>((1ull << (31 + l)) / d + 1);
  *shift = power ? l : l - 1;
}

int run(TreeParams& p, int T, int H, int D, float scale, int dtype, int fmt, void* workspace,
        size_t workspace_bytes, cudaStream_t s) {
  const Plan r = plan_of(p.B, p.max_q, H, p.H_kv, D, fmt, p.bs, p.max_blocks);
  if (r.grid > 0x7fffffffLL || static_cast<int64_t>(T) * H > 0x7fffffffLL) return LK_ERR_INVALID_ARG;
  const size_t need = plan_bytes(r, T, H, D);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need ||
                   (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0))
    return LK_ERR_WORKSPACE;
  divisor(p.bs, &p.bs_mul, &p.bs_shift);
  divisor(p.G, &p.g_mul, &p.g_shift);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.cluster = r.cluster;
  p.chunk = r.chunk;
  p.nsplit = r.nsplit;
  p.part_ml = static_cast<float4*>(workspace);
  p.part_o = r.nsplit == 1 ? nullptr
                           : reinterpret_cast<float*>(p.part_ml + static_cast<int64_t>(T) * H * r.nsplit);
  const unsigned grid = static_cast<unsigned>(r.grid);
  int rc = fmt == LK_KV_16BIT  ? tree_launch_16(p, dtype, D, r.NT, grid, s)
           : fmt == LK_KV_INT8 ? tree_launch_i8(p, dtype, D, r.NT, grid, s)
                               : tree_launch_e4m3(p, dtype, D, r.NT, grid, s);
  if (rc != LK_OK || r.nsplit == 1) return rc;
  JoinParams j;
  j.out = p.out;
  j.out_stride = p.out_stride;
  j.part_ml = p.part_ml;
  j.part_o = p.part_o;
  j.cu_seqlens_q = p.cu_seqlens_q;
  j.context_lens = p.context_lens;
  j.rows = static_cast<uint32_t>(T) * H;
  j.B = p.B;
  j.H = H;
  j.nsplit = r.nsplit;
  j.chunk = r.chunk;
  j.max_keys = p.max_blocks * p.bs;
  j.max_q = p.max_q;
  const unsigned rows = static_cast<unsigned>(T) * H;
  cudaError_t e;
  if (dtype == LK_DTYPE_BF16)
    e = D == 128 ? join<__nv_bfloat16, 128>(j, rows, s) : join<__nv_bfloat16, 64>(j, rows, s);
  else
    e = D == 128 ? join<__half, 128>(j, rows, s) : join<__half, 64>(j, rows, s);
  return e == cudaSuccess ? check_launch() : LK_ERR_CUDA;
}

bool shape_ok(int H, int H_kv, int D, int bs, int max_blocks, int64_t num_blocks, int dtype,
              int fmt, int* rc) {
  *rc = LK_OK;
  if (H <= 0 || H_kv <= 0 || H % H_kv != 0 || bs <= 0 || max_blocks <= 0 || num_blocks < 0) {
    *rc = LK_ERR_INVALID_ARG;
  } else if ((D != 64 && D != 128) || (dtype != LK_DTYPE_F16 && dtype != LK_DTYPE_BF16) ||
             (fmt != LK_KV_16BIT && fmt != LK_KV_INT8 && fmt != LK_KV_E4M3) ||
             num_blocks > 0x7fffffffLL / bs || max_blocks > 0x7fff0000 / bs) {
    *rc = LK_ERR_UNSUPPORTED;
  }
  return *rc == LK_OK;
}

bool aligned(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15u) == 0; }

}  // namespace
}  // namespace lk

extern "C" size_t lk_paged_tree_workspace_bytes(int32_t num_tokens, int32_t num_seqs,
                                                int32_t max_q_len, int32_t H, int32_t H_kv,
                                                int32_t D, int32_t block_size,
                                                int32_t max_blocks_per_seq, int32_t kv_format) {
  if (num_tokens <= 0 || num_seqs <= 0 || max_q_len <= 0 || H <= 0 || H_kv <= 0 ||
      H % H_kv != 0 || D <= 0 || block_size <= 0 || max_blocks_per_seq <= 0)
    return 0;
  return lk::plan_bytes(
      lk::plan_of(num_seqs, max_q_len, H, H_kv, D, kv_format, block_size, max_blocks_per_seq),
      num_tokens, H, D);
}

extern "C" int lk_paged_tree_attention(
    void* out, int64_t out_token_stride, const void* q, int64_t q_token_stride,
    const void* k_cache, const float* k_scale, const void* v_cache, const float* v_scale,
    int64_t num_blocks, const int32_t* block_tables, int64_t block_table_stride,
    const int32_t* cu_seqlens_q, const int32_t* context_lens, const int64_t* tree_mask,
    int64_t mask_stride, int32_t mask_words, int32_t num_tokens, int32_t num_seqs,
    int32_t max_q_len, int32_t H, int32_t H_kv, int32_t D, int32_t block_size,
    int32_t max_blocks_per_seq, float scale, int32_t dtype, int32_t kv_format, void* workspace,
    size_t workspace_bytes, int32_t* status, void* stream) {
  int rc;
  if (num_tokens < 0 || num_seqs < 0 || max_q_len < 0) return LK_ERR_INVALID_ARG;
  if (!lk::shape_ok(H, H_kv, D, block_size, max_blocks_per_seq, num_blocks, dtype, kv_format, &rc))
    return rc;
  if (num_tokens == 0 || num_seqs == 0 || max_q_len == 0) return LK_OK;
  const bool q8 = kv_format != LK_KV_16BIT;
  if (!out || !q || !k_cache || !v_cache || !block_tables || !context_lens ||
      (q8 && (!k_scale || !v_scale)) || (!cu_seqlens_q && (max_q_len != 1 || tree_mask)) ||
      (!cu_seqlens_q && num_tokens != num_seqs) ||
      (tree_mask && (mask_words <= 0 || static_cast<int64_t>(mask_words) * 64 < max_q_len)) ||
      static_cast<int64_t>(max_q_len) * (H / H_kv) > 0x7fffffffLL / 2)
    return LK_ERR_INVALID_ARG;
  if (!lk::aligned(k_cache) || !lk::aligned(v_cache)) return LK_ERR_ALIGNMENT;
  lk::TreeParams p = {};
  p.out = out;
  p.out_stride = out_token_stride;
  p.q = q;
  p.q_stride = q_token_stride;
  p.k = k_cache;
  p.v = v_cache;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.block_tables = block_tables;
  p.bt_stride = block_table_stride;
  p.context_lens = context_lens;
  p.cu_seqlens_q = cu_seqlens_q;
  p.mask = tree_mask;
  p.mask_stride = mask_stride;
  p.mask_words = mask_words;
  p.status = status;
  p.T = num_tokens;
  p.B = num_seqs;
  p.H_kv = H_kv;
  p.G = H / H_kv;
  p.bs = block_size;
  p.max_blocks = max_blocks_per_seq;
  p.num_blocks = num_blocks;
  p.max_q = max_q_len;
  return lk::run(p, num_tokens, H, D, scale, dtype, kv_format, workspace, workspace_bytes,
                 static_cast<cudaStream_t>(stream));
}

extern "C" int lk_paged_decode_q8(void* out, int64_t out_token_stride, const void* q,
                                  int64_t q_token_stride, const void* k_data,
                                  const float* k_scale, const void* v_data, const float* v_scale,
                                  int64_t num_blocks, const int32_t* block_tables,
                                  int64_t block_table_stride, const int32_t* context_lens,
                                  int32_t B, int32_t H, int32_t H_kv, int32_t D,
                                  int32_t block_size, int32_t max_blocks_per_seq, float scale,
                                  int32_t dtype, int32_t kv_format, void* workspace,
                                  size_t workspace_bytes, int32_t* status, void* stream) {
  if (kv_format == LK_KV_16BIT) return LK_ERR_UNSUPPORTED;  // lk_paged_decode reads those
  return lk_paged_tree_attention(out, out_token_stride, q, q_token_stride, k_data, k_scale,
                                 v_data, v_scale, num_blocks, block_tables, block_table_stride,
                                 nullptr, context_lens, nullptr, 0, 0, B, B, 1, H, H_kv, D,
                                 block_size, max_blocks_per_seq, scale, dtype, kv_format,
                                 workspace, workspace_bytes, status, stream);
}
