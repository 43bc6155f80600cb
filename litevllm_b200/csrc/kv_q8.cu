// The 8-bit KV cache: quantising K / V rows as they are written, and reading
// whole contexts back in 16 or 32 bits. Formats and formulas: lk_q8.cuh. A value read
// back is the fp32 product q s, rounded once more for a 16-bit output: at most half a
// step of the type and 2^-24 off, and the bits that other fp32 arithmetic then gives.
//
// Cache layout: bytes [num_blocks, block_size, H_kv, D] as the 16-bit cache
// (so block tables, slot mappings and block copies are unchanged) and fp32
// scales [num_blocks, H_kv, block_size]: the attention warp of one KV head
// then reads a block's scales as one contiguous piece.
//
// Both kernels move every byte once and do a few operations per element, so
// HBM bounds them once the call is large; small calls are launch latency. At 8 KV
// heads of 128, bf16: storing 16384 tokens takes 17.1 us (101 MB, 5.9 TB/s), 256
// tokens 2.2 us; reading 69K rows back 68 us (427 MB, 6.3 TB/s), 6.2K rows 7.8 us
// (4.9 TB/s). As blocks for prefill (caches cold, the call included): 9108 rows of four
// contexts under a table of 4096 each 16 us; 8 x 500 rows under a tight table 11, under
// one of 32768 each 35, the start of 262144 warps of which 4000 have a row to move.
#include <type_traits>

#include "lk_common.cuh"
#include "lk_host.h"
#include "lk_q8.cuh"

namespace {

constexpr int kQThreads = 256;

// Largest |x| of eight packed 16-bit values, as the bits of the type: without
// its sign a 16-bit float orders like an unsigned integer, NaN above infinity.
LK_DEVINL uint32_t abs_max2(uint32_t m, uint32_t w) { return __vmaxu2(m, w & 0x7fff7fffu); }

template <typename T> LK_DEVINL float from_bits16(uint32_t b);
template <> LK_DEVINL float from_bits16<__nv_bfloat16>(uint32_t b) { return __uint_as_float(b << 16); }
template <> LK_DEVINL float from_bits16<__half>(uint32_t b) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(b)));
}
template <typename T> constexpr uint32_t inf_bits();
template <> constexpr uint32_t inf_bits<__nv_bfloat16>() { return 0x7f80u; }
template <> constexpr uint32_t inf_bits<__half>() { return 0x7c00u; }

struct StoreQ8Params {
  const void* src[2];   // key, value
  int64_t stride[2];    // elements between tokens
  uint8_t* data[2];
  float* scale[2];
  const int64_t* slot_mapping;
  int64_t num_slots;
  int rows;             // tokens * H_kv
  int H_kv, bs;
  int32_t* status;
};

// D / 16 lanes hold one (token, head): its K and its V row, 16 values of each a
// lane (four 16-byte loads under way at once), a packed maximum, log2(D / 16)
// shuffles, two 16-byte stores. With one of the two a CTA, the loads behind the
// slot's and 64-bit quotients, 16384 tokens took 35.7 us.
template <typename T, int FMT, int D, bool VEC>
__global__ void __launch_bounds__(kQThreads) store_kv_q8_kernel(const StoreQ8Params p) {
  // A following attention kernel may start launching; it waits for this grid.
  lk::pdl_launch_dependents();
  constexpr int LPR = D / 16;
  const int lane = threadIdx.x % LPR;
  const uint32_t row = blockIdx.x * (kQThreads / LPR) + threadIdx.x / LPR;
  const bool inside = row < static_cast<uint32_t>(p.rows);
  const uint32_t t = inside ? row / static_cast<uint32_t>(p.H_kv) : 0u;
  const uint32_t h = inside ? row - t * p.H_kv : 0u;
  const int64_t slot = inside ? p.slot_mapping[t] : -1;
  // the rows are read while their slot is on its way: a skipped token's too
  uint32_t w[2][8];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const T* src = static_cast<const T*>(p.src[which]) + t * p.stride[which] + h * D + lane * 16;
    if constexpr (VEC) {
      const uint4 a = reinterpret_cast<const uint4*>(src)[0];
      const uint4 b = reinterpret_cast<const uint4*>(src)[1];
      w[which][0] = a.x; w[which][1] = a.y; w[which][2] = a.z; w[which][3] = a.w;
      w[which][4] = b.x; w[which][5] = b.y; w[which][6] = b.z; w[which][7] = b.w;
    } else {
      const uint16_t* s16 = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[which][i] = s16[2 * i] | (static_cast<uint32_t>(s16[2 * i + 1]) << 16);
    }
  }
  uint32_t top[2];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = abs_max2(m, w[which][i]);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
    top[which] = max(m & 0xffffu, m >> 16);
  }
  if (slot < 0 || slot >= p.num_slots) {
    if (inside && slot != -1 && p.status != nullptr && lane == 0)
      atomicOr(p.status, LK_STATUS_SLOT_OOB);
    return;
  }
  const uint32_t blk = static_cast<uint32_t>(slot) / static_cast<uint32_t>(p.bs);  // < 2^31
  const uint32_t off = static_cast<uint32_t>(slot) - blk * p.bs;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const bool fine = top[which] < inf_bits<T>();
    const float a = fmaxf(from_bits16<T>(top[which]), 7.888609052210118e-31f);  // 2^-100
    const float r = __fdiv_rn(lk::Q8<FMT>::kMax, a);
    uint4 q = make_uint4(0u, 0u, 0u, 0u);
    if (fine) {
      uint32_t* qw = &q.x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = w[which][2 * i], hi = w[which][2 * i + 1];
        const float x[4] = {from_bits16<T>(lo & 0xffffu), from_bits16<T>(lo >> 16),
                            from_bits16<T>(hi & 0xffffu), from_bits16<T>(hi >> 16)};
        qw[i] = lk::Q8<FMT>::pack4(x, r);
      }
    }
    *reinterpret_cast<uint4*>(p.data[which] + (slot * p.H_kv + h) * D + lane * 16) = q;
    if (lane == 0)
      p.scale[which][(static_cast<int64_t>(blk) * p.H_kv + h) * p.bs + off] =
          fine ? __fdiv_rn(a, lk::Q8<FMT>::kMax) : __int_as_float(0x7fc00000);
  }
}

struct LoadQ8Params {
  const uint8_t* data[2];
  const float* scale[2];
  void* out[2];               // [num_rows, H_kv, D]
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* context_lens;
  const int32_t* cu_rows;     // [B + 1]
  int32_t* out_tables;        // [B, max_blocks], instead of cu_rows: whole blocks
  int64_t num_blocks;
  int64_t num_rows;
  int B, H_kv, bs, max_blocks;
  int32_t* status;
};

template <typename T> LK_DEVINL void put8(T* dst, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(dst) =
      make_uint4(lk::pack2<T>(x[0], x[1]), lk::pack2<T>(x[2], x[3]), lk::pack2<T>(x[4], x[5]),
                 lk::pack2<T>(x[6], x[7]));
}
template <> LK_DEVINL void put8<float>(float* dst, const float (&x)[8]) {
  reinterpret_cast<float4*>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// One warp per output row: it finds its sequence in cu_rows, then moves the row's K
// and V together, eight values a lane and access (8-byte loads, 16-byte stores, both
// contiguous over the warp), up to eight loads under way at once. K and V one after
// the other took 82 us instead of 68 for 69K rows of 8 x 128; two rows a warp, to
// share the search, 70, four 71 (and short calls lose warps: 6.2K rows 7.8, 8.0, 10).
// BLOCKS: the output is blocks in the table's order, of which those with a token of the
// context are written (zeros behind it); a row that is not costs its warp's start.
template <typename T, int FMT, int D, bool BLOCKS>
__global__ void __launch_bounds__(kQThreads) load_kv_q8_kernel(const LoadQ8Params p) {
  const int lane = threadIdx.x & 31;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * (kQThreads / 32) + (threadIdx.x >> 5);
  if (at >= p.num_rows || (!BLOCKS && (at < p.cu_rows[0] || at >= p.cu_rows[p.B]))) return;
  const int row = static_cast<int>(at);
  int b, pos;
  if constexpr (BLOCKS) {
    const uint32_t cap = p.max_blocks * p.bs;
    b = static_cast<uint32_t>(row) / cap;
    pos = row - b * cap;
  } else {
    // b = the last sequence that starts at or before row: 32 probes a step
    int lo = 0, hi = p.B;  // cu_rows[lo] <= row < cu_rows[hi]
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32;
      const int probe = min(lo + lane * step, hi);
      const uint32_t le = __ballot_sync(0xffffffffu, p.cu_rows[probe] <= row);
      const int k = 31 - __clz(le);  // lane 0 always holds
      const int nlo = min(lo + k * step, hi - 1);
      hi = min(hi, nlo + step);
      lo = nlo;
    }
    b = lo;
    pos = row - p.cu_rows[b];
  }
  int ctx = p.context_lens[b];
  if (ctx > p.max_blocks * static_cast<int64_t>(p.bs)) {
    if (lane == 0 && p.status) atomicOr(p.status, LK_STATUS_CTX_OOB);
    ctx = p.max_blocks * p.bs;
  }
  const int page = static_cast<uint32_t>(max(pos, 0)) / static_cast<uint32_t>(p.bs);
  const int off = pos - page * p.bs;
  if constexpr (BLOCKS) {
    if (off == 0 && lane == 0) p.out_tables[row / p.bs] = row / p.bs;
    if (page * p.bs >= ctx) return;
  }
  int blk = -1;
  if (pos >= 0 && pos < ctx) {
    blk = p.block_tables[b * p.bt_stride + page];
    if (blk < 0 || blk >= p.num_blocks) {
      if (lane == 0 && p.status) atomicOr(p.status, LK_STATUS_BLOCK_OOB);
      blk = -1;
    }
  }
  const int width = p.H_kv * D;
  const int64_t o = static_cast<int64_t>(row) * width;
  if (blk < 0) {
    const float zero[8] = {};
    for (int i = lane * 8; i < width; i += 256) {
      put8<T>(static_cast<T*>(p.out[0]) + o + i, zero);
      put8<T>(static_cast<T*>(p.out[1]) + o + i, zero);
    }
    return;
  }
  const int64_t src = (static_cast<int64_t>(blk) * p.bs + off) * width;
  const int64_t sc = static_cast<int64_t>(blk) * p.H_kv * p.bs + off;
  auto put = [&](int which, int i, uint2 w, float s) {
    float a[4], c[4];
    lk::Q8<FMT>::unpack4(w.x, a);
    lk::Q8<FMT>::unpack4(w.y, c);
    const float x[8] = {a[0] * s, a[1] * s, a[2] * s, a[3] * s,
                        c[0] * s, c[1] * s, c[2] * s, c[3] * s};
    put8<T>(static_cast<T*>(p.out[which]) + o + i, x);
  };
  int i = lane * 8;
  for (; i + 3 * 256 < width; i += 4 * 256) {
    uint2 w[2][4];
    float s[2][4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        w[which][k] = *reinterpret_cast<const uint2*>(p.data[which] + src + i + k * 256);
        s[which][k] = p.scale[which][sc + (i + k * 256) / D * p.bs];
      }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int which = 0; which < 2; ++which) put(which, i + k * 256, w[which][k], s[which][k]);
  }
  for (; i < width; i += 256) {
#pragma unroll
    for (int which = 0; which < 2; ++which)
      put(which, i, *reinterpret_cast<const uint2*>(p.data[which] + src + i),
          p.scale[which][sc + i / D * p.bs]);
  }
}

bool kv_q8_shape(int32_t H_kv, int32_t D, int32_t bs, int64_t num_blocks, int32_t fmt, int* rc) {
  if (H_kv <= 0 || D <= 0 || bs <= 0 || num_blocks < 0) {
    *rc = LK_ERR_INVALID_ARG;
    return false;
  }
  if ((D != 64 && D != 128) || (fmt != LK_KV_INT8 && fmt != LK_KV_E4M3) || H_kv > 65535 ||
      num_blocks > 0x7fffffffLL / bs) {
    *rc = LK_ERR_UNSUPPORTED;
    return false;
  }
  return true;
}

bool aligned16(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15u) == 0; }

// Shared by the two entry points: cu_rows or out_tables is NULL.
int load_kv_q8(void* key_out, void* value_out, const void* k_data, const float* k_scale,
               const void* v_data, const float* v_scale, const int32_t* block_tables,
               int64_t block_table_stride, const int32_t* context_lens, const int32_t* cu_rows,
               int32_t* out_tables, int32_t num_seqs, int64_t num_rows, int32_t H_kv, int32_t D,
               int64_t num_blocks, int32_t block_size, int32_t max_blocks_per_seq, int32_t dtype,
               int32_t kv_format, int32_t* status, void* stream) {
  int rc = LK_OK;
  if (num_seqs < 0 || num_rows < 0 || max_blocks_per_seq < 0) return LK_ERR_INVALID_ARG;
  if (!kv_q8_shape(H_kv, D, block_size, num_blocks, kv_format, &rc)) return rc;
  if (dtype != LK_DTYPE_F32 && dtype != LK_DTYPE_F16 && dtype != LK_DTYPE_BF16)
    return LK_ERR_UNSUPPORTED;
  if (num_seqs == 0 || num_rows == 0) return LK_OK;
  if (!key_out || !value_out || !k_data || !k_scale || !v_data || !v_scale || !context_lens ||
      (!cu_rows && !out_tables) || (max_blocks_per_seq > 0 && !block_tables) ||
      num_rows > 0x7fffffffLL || max_blocks_per_seq > 0x7fffffff / block_size)
    return LK_ERR_INVALID_ARG;
  if (!aligned16(k_data) || !aligned16(v_data) || !aligned16(key_out) || !aligned16(value_out))
    return LK_ERR_ALIGNMENT;
  LoadQ8Params p;
  p.data[0] = static_cast<const uint8_t*>(k_data);
  p.data[1] = static_cast<const uint8_t*>(v_data);
  p.scale[0] = k_scale;
  p.scale[1] = v_scale;
  p.out[0] = key_out;
  p.out[1] = value_out;
  p.block_tables = block_tables;
  p.bt_stride = block_table_stride;
  p.context_lens = context_lens;
  p.cu_rows = cu_rows;
  p.out_tables = out_tables;
  p.num_blocks = num_blocks;
  p.num_rows = num_rows;
  p.B = num_seqs;
  p.H_kv = H_kv;
  p.bs = block_size;
  p.max_blocks = max_blocks_per_seq;
  p.status = status;
  const int per_cta = kQThreads / 32;
  const unsigned grid = static_cast<unsigned>((num_rows + per_cta - 1) / per_cta);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto by_dim = [&](auto type, auto fmt) {
    using T = decltype(type);
    constexpr int F = decltype(fmt)::value;
    if (out_tables && D == 128) load_kv_q8_kernel<T, F, 128, true><<<grid, kQThreads, 0, s>>>(p);
    else if (out_tables) load_kv_q8_kernel<T, F, 64, true><<<grid, kQThreads, 0, s>>>(p);
    else if (D == 128) load_kv_q8_kernel<T, F, 128, false><<<grid, kQThreads, 0, s>>>(p);
    else load_kv_q8_kernel<T, F, 64, false><<<grid, kQThreads, 0, s>>>(p);
  };
  auto by_fmt = [&](auto type) {
    if (kv_format == LK_KV_INT8) by_dim(type, std::integral_constant<int, LK_KV_INT8>());
    else by_dim(type, std::integral_constant<int, LK_KV_E4M3>());
  };
  if (dtype == LK_DTYPE_BF16) by_fmt(__nv_bfloat16());
  else if (dtype == LK_DTYPE_F16) by_fmt(__half());
  else by_fmt(float());
  return lk::check_launch();
}

}  // namespace

extern "C" int lk_store_kv_q8(const void* key, const void* value, void* k_data, float* k_scale,
                              void* v_data, float* v_scale, const int64_t* slot_mapping,
                              int32_t num_tokens, int32_t H_kv, int32_t D,
                              int64_t key_token_stride, int64_t value_token_stride,
                              int64_t num_blocks, int32_t block_size, int32_t dtype,
                              int32_t kv_format, int32_t* status, void* stream) {
  int rc = LK_OK;
  if (num_tokens < 0) return LK_ERR_INVALID_ARG;
  if (!kv_q8_shape(H_kv, D, block_size, num_blocks, kv_format, &rc)) return rc;
  if (dtype != LK_DTYPE_F16 && dtype != LK_DTYPE_BF16) return LK_ERR_UNSUPPORTED;
  if (num_tokens == 0) return LK_OK;
  if (!key || !value || !k_data || !k_scale || !v_data || !v_scale || !slot_mapping)
    return LK_ERR_INVALID_ARG;
  if (!aligned16(k_data) || !aligned16(v_data)) return LK_ERR_ALIGNMENT;
  if (static_cast<int64_t>(num_tokens) * H_kv > 0x7fffffffLL) return LK_ERR_INVALID_ARG;
  StoreQ8Params p;
  p.src[0] = key;
  p.src[1] = value;
  p.stride[0] = key_token_stride;
  p.stride[1] = value_token_stride;
  p.data[0] = static_cast<uint8_t*>(k_data);
  p.data[1] = static_cast<uint8_t*>(v_data);
  p.scale[0] = k_scale;
  p.scale[1] = v_scale;
  p.slot_mapping = slot_mapping;
  p.num_slots = num_blocks * block_size;
  p.rows = num_tokens * H_kv;
  p.H_kv = H_kv;
  p.bs = block_size;
  p.status = status;
  const bool vec = aligned16(key) && aligned16(value) && (key_token_stride & 7) == 0 &&
                   (value_token_stride & 7) == 0;
  const int per_cta = kQThreads / (D / 16);
  const unsigned grid = (static_cast<unsigned>(p.rows) + per_cta - 1) / per_cta;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto by_vec = [&](auto type, auto fmt, auto dim) {
    using T = decltype(type);
    constexpr int F = decltype(fmt)::value, N = decltype(dim)::value;
    if (vec) store_kv_q8_kernel<T, F, N, true><<<grid, kQThreads, 0, s>>>(p);
    else store_kv_q8_kernel<T, F, N, false><<<grid, kQThreads, 0, s>>>(p);
  };
  auto by_dim = [&](auto type, auto fmt) {
    if (D == 128) by_vec(type, fmt, std::integral_constant<int, 128>());
    else by_vec(type, fmt, std::integral_constant<int, 64>());
  };
  auto by_fmt = [&](auto type) {
    if (kv_format == LK_KV_INT8) by_dim(type, std::integral_constant<int, LK_KV_INT8>());
    else by_dim(type, std::integral_constant<int, LK_KV_E4M3>());
  };
  if (dtype == LK_DTYPE_BF16) by_fmt(__nv_bfloat16());
  else by_fmt(__half());
  return lk::check_launch();
}

extern "C" int lk_load_kv_q8(void* key_out, void* value_out, const void* k_data,
                             const float* k_scale, const void* v_data, const float* v_scale,
                             const int32_t* block_tables, int64_t block_table_stride,
                             const int32_t* context_lens, const int32_t* cu_rows,
                             int32_t num_seqs, int64_t num_rows, int32_t H_kv, int32_t D,
                             int64_t num_blocks, int32_t block_size, int32_t max_blocks_per_seq,
                             int32_t dtype, int32_t kv_format, int32_t* status, void* stream) {
  return load_kv_q8(key_out, value_out, k_data, k_scale, v_data, v_scale, block_tables,
                    block_table_stride, context_lens, cu_rows, nullptr, num_seqs, num_rows, H_kv, D,
                    num_blocks, block_size, max_blocks_per_seq, dtype, kv_format, status, stream);
}

extern "C" int lk_load_kv_q8_blocks(void* key_out, void* value_out, int32_t* out_tables,
                                    const void* k_data, const float* k_scale, const void* v_data,
                                    const float* v_scale, const int32_t* block_tables,
                                    int64_t block_table_stride, const int32_t* context_lens,
                                    int32_t num_seqs, int32_t H_kv, int32_t D, int64_t num_blocks,
                                    int32_t block_size, int32_t max_blocks_per_seq, int32_t dtype,
                                    int32_t kv_format, int32_t* status, void* stream) {
  if (num_seqs > 0 && max_blocks_per_seq > 0 && !out_tables) return LK_ERR_INVALID_ARG;
  if (num_seqs < 0 || max_blocks_per_seq < 0 || block_size <= 0) return LK_ERR_INVALID_ARG;
  const int64_t blocks = static_cast<int64_t>(num_seqs) * max_blocks_per_seq;
  if (blocks > 0x7fffffffLL / block_size) return LK_ERR_INVALID_ARG;
  return load_kv_q8(key_out, value_out, k_data, k_scale, v_data, v_scale, block_tables,
                    block_table_stride, context_lens, nullptr, out_tables, num_seqs,
                    blocks * block_size, H_kv, D, num_blocks, block_size, max_blocks_per_seq, dtype,
                    kv_format, status, stream);
}
