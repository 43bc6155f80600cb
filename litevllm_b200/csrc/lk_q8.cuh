// 8-bit KV-cache rows: formats, quantisation constants and the conversions
// back to 16 bits, shared by the store / load kernels (kv_q8.cu) and the
// attention kernels that read the cache (paged_tree.cuh).
//
// A row x[0..D) (one token, one KV head) is held as D bytes q and one fp32
// scale s:   a = max(max|x|, 2^-100), s = RN(a / M), r = RN(M / a),
//   int8 (M = 127): q = rint(x r), one rounding of the exact product;
//   e4m3 (M = 448): q = RN_e4m3(RN32(x r)).
// The floor 2^-100 keeps r finite; a row with an infinity or a NaN is held as
// q = 0, s = NaN, so the bytes themselves never hold a special value and a
// masked token's row cannot leak one through a zero weight.
#pragma once

#include <cuda_fp8.h>

#include "lk_common.cuh"

namespace lk {

template <int FMT> struct Q8;

template <> struct Q8<LK_KV_INT8> {
  static constexpr float kMax = 127.f;
  // Four values to four bytes. Adding 1.5 * 2^23 leaves the rounded integer in
  // the low byte, in two's complement; the fused product is rounded once.
  LK_DEVINL static uint32_t pack4(const float (&x)[4], float r) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(fmaf(x[i], r, 12582912.f));
    return __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
  }
  // Four bytes to fp32: 2^23 + (q + 128) has its integer in the low byte.
  LK_DEVINL static void unpack4(uint32_t w, float (&x)[4]) {
    w ^= 0x80808080u;
    x[0] = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440)) - 8388736.f;
    x[1] = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7441)) - 8388736.f;
    x[2] = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7442)) - 8388736.f;
    x[3] = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7443)) - 8388736.f;
  }
  // Bytes (0, 1) and (2, 3) to packed f16 pairs, exactly: 0x64xx is 1024 + xx.
  LK_DEVINL static void halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
    w ^= 0x80808080u;
    lo = sub1152(__byte_perm(w, 0x64646464u, 0x4140));
    hi = sub1152(__byte_perm(w, 0x64646464u, 0x4342));
  }
  // Bytes (0, 2) and (1, 3): the pairs of a transposed 8 x 8 matrix of byte pairs.
  LK_DEVINL static void halves_t(uint32_t w, uint32_t& even, uint32_t& odd) {
    w ^= 0x80808080u;
    even = sub1152(__byte_perm(w, 0x64646464u, 0x4240));
    odd = sub1152(__byte_perm(w, 0x64646464u, 0x4341));
  }

 private:
  LK_DEVINL static uint32_t sub1152(uint32_t h) {
    const uint32_t c = 0x64806480u;  // 1024 + 128, twice
    __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&h), *reinterpret_cast<const __half2*>(&c));
    return *reinterpret_cast<uint32_t*>(&d);
  }
};

template <> struct Q8<LK_KV_E4M3> {
  static constexpr float kMax = 448.f;
  LK_DEVINL static uint32_t pack4(const float (&x)[4], float r) {
    const uint32_t a = __nv_cvt_float2_to_fp8x2(
        make_float2(__fmul_rn(x[0], r), __fmul_rn(x[1], r)), __NV_SATFINITE, __NV_E4M3);
    const uint32_t b = __nv_cvt_float2_to_fp8x2(
        make_float2(__fmul_rn(x[2], r), __fmul_rn(x[3], r)), __NV_SATFINITE, __NV_E4M3);
    return a | (b << 16);
  }
  LK_DEVINL static void unpack4(uint32_t w, float (&x)[4]) {
    uint32_t lo, hi;
    halves(w, lo, hi);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    x[0] = a.x;
    x[1] = a.y;
    x[2] = b.x;
    x[3] = b.y;
  }
  LK_DEVINL static void halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
    lo = cvt2(static_cast<uint16_t>(w));
    hi = cvt2(static_cast<uint16_t>(w >> 16));
  }
  LK_DEVINL static void halves_t(uint32_t w, uint32_t& even, uint32_t& odd) {
    halves(__byte_perm(w, 0u, 0x3120), even, odd);
  }

 private:
  LK_DEVINL static uint32_t cvt2(uint16_t w) {  // every e4m3 value is an f16 value
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(w));
    return h;
  }
};

}  // namespace lk
