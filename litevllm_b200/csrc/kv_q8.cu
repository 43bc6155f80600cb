// The 8-bit KV cache: quantising K / V rows as they are written, and reading
// whole contexts back in 16 or 32 bits. Formats and formulas: lk_q8.cuh.
//
// Cache layout: bytes [num_blocks, block_size, H_kv, D] as the 16-bit cache
// (so block tables, slot mappings and block copies are unchanged) and fp32
// scales [num_blocks, H_kv, block_size]: the attention warp of one KV head
// then reads a block's scales as one contiguous piece.
//
// Both kernels move every byte once and do a few operations per element, so
// HBM bounds them once the call is large; small calls are launch latency.
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

// D / 16 lanes hold one row, 16 values each: two 16-byte loads, a packed
// maximum, log2(D / 16) shuffles, one 16-byte store. blockIdx.y: K or V.
template <typename T, int FMT, int D, bool VEC>
__global__ void __launch_bounds__(kQThreads) store_kv_q8_kernel(const StoreQ8Params p) {
  // A following attention kernel may start launching; it waits for this grid.
  lk::pdl_launch_dependents();
  constexpr int LPR = D / 16;
  const int lane = threadIdx.x % LPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kQThreads / LPR) + threadIdx.x / LPR;
  const int which = blockIdx.y;
  const bool inside = row < p.rows;
  const int t = inside ? static_cast<int>(row / p.H_kv) : 0;
  const int h = inside ? static_cast<int>(row % p.H_kv) : 0;
  const int64_t slot = inside ? p.slot_mapping[t] : -1;
  const bool store = slot >= 0 && slot < p.num_slots;
  if (inside && !store && slot != -1 && p.status != nullptr && lane == 0)
    atomicOr(p.status, LK_STATUS_SLOT_OOB);
  uint32_t w[8];
  if (store) {
    const T* src = static_cast<const T*>(p.src[which]) + t * p.stride[which] + h * D + lane * 16;
    if constexpr (VEC) {
      const uint4 a = reinterpret_cast<const uint4*>(src)[0];
      const uint4 b = reinterpret_cast<const uint4*>(src)[1];
      w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
      w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    } else {
      const uint16_t* s16 = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i] = s16[2 * i] | (static_cast<uint32_t>(s16[2 * i + 1]) << 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0u;
  }
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = abs_max2(m, w[i]);
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (!store) return;
  const uint32_t top = max(m & 0xffffu, m >> 16);
  const bool fine = top < inf_bits<T>();
  const float a = fmaxf(from_bits16<T>(top), 7.888609052210118e-31f);  // 2^-100
  const float r = __fdiv_rn(lk::Q8<FMT>::kMax, a);
  uint4 q = make_uint4(0u, 0u, 0u, 0u);
  if (fine) {
    uint32_t* qw = &q.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x[4] = {from_bits16<T>(w[2 * i] & 0xffffu), from_bits16<T>(w[2 * i] >> 16),
                          from_bits16<T>(w[2 * i + 1] & 0xffffu), from_bits16<T>(w[2 * i + 1] >> 16)};
      qw[i] = lk::Q8<FMT>::pack4(x, r);
    }
  }
  *reinterpret_cast<uint4*>(p.data[which] + (slot * p.H_kv + h) * D + lane * 16) = q;
  if (lane == 0) {
    const int64_t blk = slot / p.bs;
    p.scale[which][(blk * p.H_kv + h) * p.bs + (slot - blk * p.bs)] =
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

// One warp per output row: it finds its sequence in cu_rows, then moves the
// row's K and V, eight values a lane (8-byte loads, 16-byte stores, both
// contiguous over the warp).
template <typename T, int FMT, int D>
__global__ void __launch_bounds__(kQThreads) load_kv_q8_kernel(const LoadQ8Params p) {
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kQThreads / 32) + (threadIdx.x >> 5);
  if (row >= p.num_rows || row < p.cu_rows[0] || row >= p.cu_rows[p.B]) return;
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
  const int b = lo;
  const int pos = static_cast<int>(row - p.cu_rows[b]);
  int ctx = p.context_lens[b];
  if (ctx > p.max_blocks * static_cast<int64_t>(p.bs)) {
    if (lane == 0 && p.status) atomicOr(p.status, LK_STATUS_CTX_OOB);
    ctx = p.max_blocks * p.bs;
  }
  int blk = -1;
  if (pos < ctx) {
    blk = p.block_tables[b * p.bt_stride + pos / p.bs];
    if (blk < 0 || blk >= p.num_blocks) {
      if (lane == 0 && p.status) atomicOr(p.status, LK_STATUS_BLOCK_OOB);
      blk = -1;
    }
  }
  const int off = pos % p.bs;
  const int64_t width = static_cast<int64_t>(p.H_kv) * D;
  const int chunks = p.H_kv * (D / 8);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const uint8_t* src = p.data[which] + (static_cast<int64_t>(blk) * p.bs + off) * width;
    const float* sc = p.scale[which] + static_cast<int64_t>(blk) * p.H_kv * p.bs + off;
    T* dst = static_cast<T*>(p.out[which]) + row * width;
#pragma unroll 4
    for (int i = lane; i < chunks; i += 32) {
      float x[8];
      if (blk >= 0) {
        const uint2 w = reinterpret_cast<const uint2*>(src)[i];
        const float s = sc[(i / (D / 8)) * p.bs];
        float a[4], c[4];
        lk::Q8<FMT>::unpack4(w.x, a);
        lk::Q8<FMT>::unpack4(w.y, c);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] = a[j] * s;
          x[4 + j] = c[j] * s;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = 0.f;
      }
      put8<T>(dst + i * 8, x);
    }
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
  const dim3 grid((p.rows + per_cta - 1) / per_cta, 2);
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
  int rc = LK_OK;
  if (num_seqs < 0 || num_rows < 0 || max_blocks_per_seq < 0) return LK_ERR_INVALID_ARG;
  if (!kv_q8_shape(H_kv, D, block_size, num_blocks, kv_format, &rc)) return rc;
  if (dtype != LK_DTYPE_F32 && dtype != LK_DTYPE_F16 && dtype != LK_DTYPE_BF16)
    return LK_ERR_UNSUPPORTED;
  if (num_seqs == 0 || num_rows == 0) return LK_OK;
  if (!key_out || !value_out || !k_data || !k_scale || !v_data || !v_scale || !context_lens ||
      !cu_rows || (max_blocks_per_seq > 0 && !block_tables) || num_rows > 0x7fffffffLL ||
      max_blocks_per_seq > 0x7fffffff / block_size)
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
    if (D == 128) load_kv_q8_kernel<T, F, 128><<<grid, kQThreads, 0, s>>>(p);
    else load_kv_q8_kernel<T, F, 64><<<grid, kQThreads, 0, s>>>(p);
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
