// Attention of a few query tokens per sequence over the paged cache: a tree of
// drafted tokens (16-bit or 8-bit cache) and single-token decode over an 8-bit
// cache.
//
// Sequence b has n query tokens at the end of its context of ctx tokens, all
// already stored; token i sees every key j < ctx - n and key ctx - n + j where
// bit j of its mask row is set (no mask: j <= i). For its query heads,
//   out = sum_j p_j s_v[j] v[j] / sum_j p_j,  p_j = exp(scale s_k[j] q.k[j]),
// s = 1 for 16-bit caches. GQA: the n * G query rows of a KV head share its keys.
//
// The keys are read once for up to 32 query rows and 4 H D operations a key, so
// HBM bounds it while n * G is small (with many rows paged_tree_tc.cuh runs). Layout:
//  * CTA = (KV head, 8 NT query rows, split of the context, sequence), four
//    warps. Each warp streams its own stages of kTok keys (warp w takes stages
//    w, w + 4, ...) with 16-byte cp.async through a private ring: no barrier
//    between warps until the end, any block size, rows past the split are
//    zero-filled and never read.
//  * S^T = K Q^T (16 keys x 8 query rows) and O^T += V^T P^T on mma.sync
//    m16n8k16 with fp32 accumulators. 8-bit rows become f16 in registers, exactly:
//    a 16-byte piece of a K row is one k-step whose slots are permuted the same
//    way in Q, and ldmatrix.trans on byte pairs gives V^T tiles whose rows are
//    the even and the odd d of the pair. The scales stay out of the products:
//    s_k multiplies the score, log2 s_v joins the exponent of the weight, so
//    the weights keep f16's 11 bits whatever the rows' sizes. Q is scaled by a
//    power of two per row into f16's range.
//  * The weights are rounded to the operand type for P V (the denominator sums them
//    before): f16 over 8-bit caches; over a 16-bit cache its own type, since both
//    operands of mma.sync have one. bf16's 8 bits make the error of a chain's result
//    against 64 bits 1.9e-3 instead of the 1.6e-3 of fp32 weights.
//  * Online softmax in base 2, with the running maximum raised only when some
//    score exceeds it by 2^8 (weights up to 256 are as exact as weights up to
//    1, and the vote costs one instruction where the maximum costs six shuffles).
//    8-bit caches hold two: m for the sum of p, M for the weights p s_v, which
//    are rounded to f16 relative to their own maximum. Sums stay in fp32.
//  * Up to eight splits of a context are a thread-block cluster that cuts every
//    context evenly and joins its (m, l, M, O) over distributed shared memory:
//    one launch, no workspace. More splits write partials to the workspace and a
//    second small kernel joins them; a context in one split is written directly.
#pragma once

#include <cooperative_groups.h>

#include <atomic>
#include <type_traits>

#include "lk_q8.cuh"
#include "paged_tree.h"

namespace lk {
namespace tree {

constexpr int kWarps = 4;
constexpr float kRaise = 8.f;  // log2 of the largest weight

template <int FMT, typename T> struct MmaType { using type = __half; };
template <typename T> struct MmaType<LK_KV_16BIT, T> { using type = T; };

template <int FMT, int D, int NT> struct Shape {
  static constexpr int kEsz = FMT == LK_KV_16BIT ? 2 : 1;
  static constexpr int kRow = D * kEsz;       // bytes of a key row
  static constexpr int kCpr = kRow / 16;      // 16-byte pieces of a row
  // Keys per stage and stages per ring: 16 KB of a warp's rows in flight or in use
  // at D = 128. Two m-tiles per stage share a vote and hide each other's
  // latency, where the accumulators leave registers for them.
  static constexpr int kTok = kEsz == 1 && NT == 1 ? 32 : 16;
  static constexpr int kMt = kTok / 16;
  static constexpr int kNst = (NT == 1 ? 2 : 3) * (D == 64 ? 2 : 1);
  static constexpr int kTile = kTok * kRow;
  static constexpr int kScales = kEsz == 1 ? 2 * kTok * 4 : 0;
  static constexpr int kStage = 2 * kTile + kScales;
  static constexpr int kRing = kWarps * kNst * kStage;
};

// Byte offset of piece `c` of row `r`: XOR-swizzled so that the eight rows of an
// ldmatrix at one piece fall into different 16-byte bank groups.
template <int CPR> LK_DEVINL uint32_t piece(uint32_t r, uint32_t c) {
  const uint32_t f = CPR >= 8 ? (r & 7u) : ((r >> 1) & 3u);
  return (r * CPR + (c ^ f)) << 4;
}

// Whether a 16-bit value, or either half of a pair, is an infinity or a NaN.
template <typename T> LK_DEVINL bool has_special(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (w & e) == e || (w & (e << 16)) == (e << 16);
}
template <typename T> LK_DEVINL float from_16(uint32_t b) {
  const uint16_t h = static_cast<uint16_t>(b);
  return Elem<T>::to_f(*reinterpret_cast<const T*>(&h));
}

template <typename T> LK_DEVINL T round_to(float x);
template <> LK_DEVINL __nv_bfloat16 round_to<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> LK_DEVINL __half round_to<__half>(float x) { return __float2half_rn(x); }

template <int FMT, typename T, int D, int NT> struct Smem {
  static constexpr int kCols = 8 * NT;
  static constexpr int kQStride = D * 2 + 16;  // bytes; rows shift by 16 bytes: no bank conflicts
  // the warps' partials, then the CTA's for its cluster
  static constexpr int kMerge = (kWarps + 1) * kCols * ((D + 4) * 4 + 16);
  static constexpr int kRing = Shape<FMT, D, NT>::kRing;
  static constexpr int kMain = kRing > kMerge ? kRing : kMerge;
  static constexpr int kBytes = kMain + kCols * kQStride + kCols * 12;
};

template <int FMT, typename T, int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 3 : 2)
paged_tree_kernel(const TreeParams p) {
  using S = Shape<FMT, D, NT>;
  using SM = Smem<FMT, T, D, NT>;
  using MT = typename MmaType<FMT, T>::type;
  constexpr bool Q8B = FMT != LK_KV_16BIT;
  constexpr int COLS = 8 * NT;
  constexpr int KS = D / 16;
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t* q_smem = smem + SM::kMain;
  float* col_scale = reinterpret_cast<float*>(q_smem + COLS * SM::kQStride);
  int* col_token = reinterpret_cast<int*>(col_scale + COLS);  // query token of a column, -1: none
  int* col_head = col_token + COLS;

  // Waits for the kernel ahead (the store of this step's rows). Global memory is read
  // after it and by ordinary loads: the read-only path is for data that nothing writes
  // during the kernel's lifetime, which begins while the kernel ahead still runs.
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;

  const int col_groups = (p.max_q * p.G + COLS - 1) / COLS;
  unsigned u = blockIdx.x;
  int sp = 0;
  if (p.cluster > 1) {
    sp = u % p.cluster;
    u /= p.cluster;
  }
  const int cg = u % col_groups;
  u /= col_groups;
  const int kvh = u % p.H_kv;
  u /= p.H_kv;
  const int b = u % p.B;
  if (p.cluster == 1) sp = u / p.B;
  auto quotient = [&](int key) { return tree_quotient(p, key); };
  const int32_t* bt = p.block_tables + static_cast<int64_t>(b) * p.bt_stride;
  // Where the split's start does not depend on the context's length, the first
  // stage's block is read beside that length, not after it.
  int early = 0;
  if (p.cluster == 1)
    early = bt[min(quotient(sp * p.chunk + warp * S::kTok + lane), p.max_blocks - 1)];

  int row0;
  const int n = tree_tokens(p, b, &row0);
  const int rows = n * p.G;  // query rows of this KV head
  if (cg * COLS >= rows) return;
  int ctx = p.context_lens[b];
  if (ctx > p.max_blocks * p.bs || ctx < (p.cu_seqlens_q ? n : 0)) {
    if (threadIdx.x == 0 && p.status) atomicOr(p.status, LK_STATUS_CTX_OOB);
    ctx = max(min(ctx, p.max_blocks * p.bs), 0);
  }
  // A cluster cuts every context into even pieces; its CTAs all stay.
  const int chunk =
      p.cluster > 1 ? ((ctx + S::kTok - 1) / S::kTok + p.cluster - 1) / p.cluster * S::kTok
                    : p.chunk;
  const int key0 = min(sp * chunk, ctx);
  if (p.cluster == 1 && sp * chunk >= ctx && sp > 0) return;
  const int key1 = min(ctx, key0 + chunk);
  // keys below `open` are seen by every row
  const int open = p.cu_seqlens_q ? max(ctx - n, 0) : ctx;

  // ------------------------------------------------------------ the ring ---
  const uint32_t width = p.H_kv * S::kRow;  // bytes of a slot
  const int pc = lane % S::kCpr;            // the lane's piece of the rows it copies
  const uint8_t* kbase = static_cast<const uint8_t*>(p.k) + kvh * S::kRow + pc * 16;
  const uint8_t* vbase = static_cast<const uint8_t*>(p.v) + kvh * S::kRow + pc * 16;
  uint8_t* ring = smem + warp * (S::kNst * S::kStage);
  const int nstage = (key1 - key0 + S::kTok - 1) / S::kTok;
  const int mine = nstage > warp ? (nstage - warp + kWarps - 1) / kWarps : 0;
  auto first_key = [&](int i) { return key0 + (warp + i * kWarps) * S::kTok; };
  // Block of the lane's key of stage i: looked up one stage before its copies.
  auto block_of = [&](int i) {
    const int key = first_key(i) + lane;
    if (i >= mine || lane >= S::kTok || key >= key1) return -1;
    const int blk = i == 0 && p.cluster == 1 ? early : bt[quotient(key)];
    if (blk < 0 || blk >= p.num_blocks) {
      if (p.status) atomicOr(p.status, LK_STATUS_BLOCK_OOB);
      return -1;
    }
    return blk;
  };
  auto load_stage = [&](int i, int blk) {
    uint8_t* st = ring + (i % S::kNst) * S::kStage;
    const int key = first_key(i) + lane;
    const int off = key - quotient(key) * p.bs;
    const int slot = blk < 0 ? -1 : blk * p.bs + off;
    constexpr int RPI = 32 / S::kCpr;  // rows per copy instruction
#pragma unroll
    for (int j = 0; j < S::kTok / RPI; ++j) {
      const int r = j * RPI + lane / S::kCpr;
      const int sl = __shfl_sync(0xffffffffu, slot, r);
      const uint64_t at = static_cast<uint64_t>(static_cast<uint32_t>(max(sl, 0))) * width;
      const uint32_t to = piece<S::kCpr>(r, pc);
      cp_async16(st + to, kbase + at, sl >= 0);
      cp_async16(st + S::kTile + to, vbase + at, sl >= 0);
    }
    if constexpr (Q8B) {
      if (lane < S::kTok) {
        float* sc = reinterpret_cast<float*>(st + 2 * S::kTile);
        const int64_t at = slot < 0 ? 0 : (static_cast<int64_t>(blk) * p.H_kv + kvh) * p.bs + off;
        cp_async4(sc + lane, p.k_scale + at, slot >= 0);
        cp_async4(sc + S::kTok + lane, p.v_scale + at, slot >= 0);
      }
    }
  };
  int next = block_of(0);
#pragma unroll
  for (int i = 0; i < S::kNst - 1; ++i) {
    const int blk = next;
    next = block_of(i + 1);
    if (i < mine) load_stage(i, blk);
    cp_async_commit();
  }

  // ------------------------------------------------------ queries to smem ---
  for (int j = warp; j < COLS; j += kWarps) {
    const int r = cg * COLS + j;
    const int tok = tree_token(p, r);
    const int token = r < rows ? tok : -1;
    const int head = kvh * p.G + r - tok * p.G;
    const T* src = static_cast<const T*>(p.q) +
                   static_cast<int64_t>(row0 + max(token, 0)) * p.q_stride +
                   static_cast<int64_t>(head) * D;
    float x[D / 32], top = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      x[i] = token >= 0 ? Elem<T>::to_f(src[lane + 32 * i]) : 0.f;
      top = fmaxf(top, fabsf(x[i]));
    }
    float up = 1.f, down = 1.f;
    if constexpr (Q8B) {
      top = warp_max(top);
      // 2^k that brings the row's largest value into [2^14, 2^15); at most 2^126
      const int e = __float_as_int(top) >> 23;
      if (e > 0 && e < 255) {
        const int f = min(268 - e, 253);
        up = __int_as_float(f << 23);
        down = __int_as_float((254 - f) << 23);
      }
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const int d = lane + 32 * i;
      int at = d;
      if constexpr (Q8B) {  // bytes 4c..4c+3 of a piece feed slots 2c, 2c+1, 2c+8, 2c+9
        const int e = d & 3, cc = (d & 15) >> 2;
        at = (d & ~15) + (e < 2 ? 2 * cc + e : 8 + 2 * cc + (e - 2));
      }
      reinterpret_cast<MT*>(q_smem + j * SM::kQStride)[at] = round_to<MT>(x[i] * up);
    }
    if (lane == 0) {
      col_scale[j] = p.scale_log2 * down;
      col_token[j] = token;
      col_head[j] = head;
    }
  }
  __syncthreads();

  // Q^T operand: registers while they fit, else read from smem per stage
  constexpr bool QREG = NT <= 2;
  uint32_t qf[QREG ? NT : 1][QREG ? KS : 1][2];
  const uint32_t q_addr = smem_u32(q_smem) + (lane & 7) * SM::kQStride + (lane >> 3) * 16;
  if constexpr (QREG) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < KS / 2; ++i)
        ldsm_x4(q_addr + nt * 8 * SM::kQStride + i * 64, qf[nt][2 * i][0], qf[nt][2 * i][1],
                qf[nt][2 * i + 1][0], qf[nt][2 * i + 1][1]);
  }
  float cs[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    cs[nt][0] = col_scale[nt * 8 + 2 * c];
    cs[nt][1] = col_scale[nt * 8 + 2 * c + 1];
  }

  float o[KS][NT][4];
#pragma unroll
  for (int i = 0; i < KS; ++i)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
  // Start of the running maxima: finite, so that a masked score (-inf) less it
  // is -inf and never NaN.
  float m[NT][2], l[NT][2], M[NT][2], dm[NT][2];  // dm = m - M
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m[nt][h] = M[nt][h] = -3.402823466e38f;
      l[nt][h] = dm[nt][h] = 0.f;
    }

  // Which of the keys t0 .. t0 + 31 column j sees, one bit each: all below
  // `open`, drafted key d = key - open by the mask, none from key1 on.
  auto window = [&](int j, int t0) {
    const int s = t0 - open;  // > -32 where drafts matter
    uint32_t bits = 0xffffffffu;
    if (s > -32) {
      const int token = col_token[j];
      const int lo = max(s, 0);
      uint32_t w = 0u;
      if (token >= 0) {
        if (p.mask == nullptr) {
          const int k = token + 1 - lo;  // drafts lo .. token
          w = k <= 0 ? 0u : k >= 32 ? 0xffffffffu : (1u << k) - 1u;
        } else {
          const int64_t* row = p.mask + static_cast<int64_t>(row0 + token) * p.mask_stride;
          const int at = lo >> 6, sh = lo & 63;
          const uint64_t a = at < p.mask_words ? static_cast<uint64_t>(row[at]) : 0ull;
          const uint64_t n = sh > 32 && at + 1 < p.mask_words
                                 ? static_cast<uint64_t>(row[at + 1]) << (64 - sh)
                                 : 0ull;
          w = static_cast<uint32_t>((a >> sh) | n);
        }
      }
      bits = s >= 0 ? w : (w << -s) | ((1u << -s) - 1u);
    }
    const int left = key1 - t0;
    return left >= 32 ? bits : bits & ((1u << left) - 1u);
  };

  const int lj = lane >> 3;
  for (int i = 0; i < mine; ++i) {
    {
      const int ahead = i + S::kNst - 1;
      const int blk = next;
      next = block_of(ahead + 1);
      __syncwarp();  // every lane has read the slot that is filled now
      if (ahead < mine) load_stage(ahead, blk);
      cp_async_commit();
    }
    cp_async_wait<S::kNst - 1>();
    __syncwarp();
    uint8_t* st = ring + (i % S::kNst) * S::kStage;
    const uint32_t kb = smem_u32(st), vb = kb + S::kTile;
    const float* sc_s = reinterpret_cast<const float*>(st + 2 * S::kTile);

    // S^T = K Q^T
    float x[S::kMt][NT][4];
#pragma unroll
    for (int mt = 0; mt < S::kMt; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        x[mt][nt][0] = x[mt][nt][1] = x[mt][nt][2] = x[mt][nt][3] = 0.f;
    const uint32_t krow = (lane & 7) + ((lj & 1) << 3);
#pragma unroll
    for (int kk = 0; kk < KS / 2; ++kk) {  // two k-steps
      uint32_t qs[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if constexpr (QREG) {
          qs[nt][0] = qf[nt][2 * kk][0];
          qs[nt][1] = qf[nt][2 * kk][1];
          qs[nt][2] = qf[nt][2 * kk + 1][0];
          qs[nt][3] = qf[nt][2 * kk + 1][1];
        } else {
          ldsm_x4(q_addr + nt * 8 * SM::kQStride + kk * 64, qs[nt][0], qs[nt][1], qs[nt][2],
                  qs[nt][3]);
        }
      }
#pragma unroll
      for (int mt = 0; mt < S::kMt; ++mt) {
        uint32_t a0[4], a1[4];
        if constexpr (Q8B) {
          uint32_t r[4];
          ldsm_x4(kb + piece<S::kCpr>(mt * 16 + krow, 2 * kk + (lj >> 1)), r[0], r[1], r[2], r[3]);
          Q8<FMT>::halves(r[0], a0[0], a0[2]);
          Q8<FMT>::halves(r[1], a0[1], a0[3]);
          Q8<FMT>::halves(r[2], a1[0], a1[2]);
          Q8<FMT>::halves(r[3], a1[1], a1[3]);
        } else {
          ldsm_x4(kb + piece<S::kCpr>(mt * 16 + krow, 4 * kk + (lj >> 1)), a0[0], a0[1], a0[2],
                  a0[3]);
          ldsm_x4(kb + piece<S::kCpr>(mt * 16 + krow, 4 * kk + 2 + (lj >> 1)), a1[0], a1[1], a1[2],
                  a1[3]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma16816<MT>(x[mt][nt], a0, qs[nt][0], qs[nt][1]);
          mma16816<MT>(x[mt][nt], a1, qs[nt][2], qs[nt][3]);
        }
      }
    }

    // Scores in base 2, less the running maxima: elements 0, 1 are key g and
    // columns 2c, 2c + 1; elements 2, 3 key g + 8.
    const int t0 = first_key(i);
    const bool drafts = min(t0 + S::kTok, key1) > open;
    const bool masked = t0 + S::kTok > key1 || drafts;
    float f[S::kMt][NT][4], lsv[S::kMt][2];
#pragma unroll
    for (int mt = 0; mt < S::kMt; ++mt) {
      float s0 = 1.f, s1 = 1.f;
      if constexpr (Q8B) {
        s0 = sc_s[mt * 16 + g];
        s1 = sc_s[mt * 16 + g + 8];
        lsv[mt][0] = __log2f(sc_s[S::kTok + mt * 16 + g]);
        lsv[mt][1] = __log2f(sc_s[S::kTok + mt * 16 + g + 8]);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        f[mt][nt][0] = s0 * cs[nt][0];
        f[mt][nt][1] = s0 * cs[nt][1];
        f[mt][nt][2] = s1 * cs[nt][0];
        f[mt][nt][3] = s1 * cs[nt][1];
      }
    }
    if (masked) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t bits = window(nt * 8 + 2 * c + h, t0) >> g;
#pragma unroll
          for (int mt = 0; mt < S::kMt; ++mt)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int e = 2 * k + h;
              x[mt][nt][e] = (bits >> (mt * 16 + 8 * k)) & 1u ? x[mt][nt][e] * f[mt][nt][e]
                                                              : -INFINITY;
              f[mt][nt][e] = 1.f;
            }
        }
    }
    float d[S::kMt][NT][4], d2[S::kMt][NT][4];
    auto scores = [&]() {
      float top = -INFINITY;
#pragma unroll
      for (int mt = 0; mt < S::kMt; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            d[mt][nt][e] = fmaf(x[mt][nt][e], f[mt][nt][e], -m[nt][e & 1]);
            if constexpr (Q8B) {
              d2[mt][nt][e] = d[mt][nt][e] + (lsv[mt][e >> 1] + dm[nt][e & 1]);
              // a masked weight is zero even where its row's scale is NaN
              if (masked && d[mt][nt][e] == -INFINITY) d2[mt][nt][e] = -INFINITY;
              top = fmax3(top, d[mt][nt][e], d2[mt][nt][e]);
            } else {
              top = fmaxf(top, d[mt][nt][e]);
            }
          }
      return top;
    };
    // raise the maxima where a weight would pass 2^kRaise
    if (__any_sync(0xffffffffu, scores() > kRaise)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float a = m[nt][h], w = M[nt][h];
#pragma unroll
          for (int mt = 0; mt < S::kMt; ++mt)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float y = x[mt][nt][2 * k + h] * f[mt][nt][2 * k + h];
              a = fmaxf(a, y);
              if constexpr (Q8B) w = fmaxf(w, y == -INFINITY ? y : y + lsv[mt][k]);
            }
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) {
            a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, off));
            if constexpr (Q8B) w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, off));
          }
          if constexpr (!Q8B) w = a;
          l[nt][h] *= ex2_mufu(m[nt][h] - a);
          const float al = ex2_mufu(M[nt][h] - w);
          m[nt][h] = a;
          M[nt][h] = w;
          if constexpr (Q8B) dm[nt][h] = a - w;
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            o[k][nt][h] *= al;
            o[k][nt][2 + h] *= al;
          }
        }
      scores();
    }

    // weights
    uint32_t pb[S::kMt][NT][2];
#pragma unroll
    for (int mt = 0; mt < S::kMt; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = ex2_mufu(d[mt][nt][e]);
          l[nt][e & 1] += w[e];
          if constexpr (Q8B) w[e] = ex2_mufu(d2[mt][nt][e]);
        }
        pb[mt][nt][0] = pack2<MT>(w[0], w[1]);
        pb[mt][nt][1] = pack2<MT>(w[2], w[3]);
      }

    if constexpr (!Q8B) {
      // A drafted token that some row does not see must not reach it through
      // 0 * inf: rows of V with special values are taken out of the tile here
      // and added to the rows that see them one by one (rare).
      if (drafts) {
        bool special = false;
#pragma unroll
        for (int k = 0; k < S::kTile / 512; ++k) {
          const uint4 w = reinterpret_cast<const uint4*>(st + S::kTile)[lane + 32 * k];
          special |= has_special<T>(w.x) | has_special<T>(w.y) | has_special<T>(w.z) |
                     has_special<T>(w.w);
        }
        if (__any_sync(0xffffffffu, special)) {
          for (int t = 0; t < S::kTok; ++t) {
            uint16_t* vr = reinterpret_cast<uint16_t*>(st + S::kTile);
            auto at = [&](int d) { return (piece<S::kCpr>(t, d >> 3) >> 1) + (d & 7); };
            bool here = false;
            for (int d = lane; d < D; d += 32) here |= has_special<T>(vr[at(d)]);
            if (!__any_sync(0xffffffffu, here)) continue;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              // the weights of key t sit in the lanes with g = t & 7
              const uint32_t pw =
                  __shfl_sync(0xffffffffu, t < 8 ? pb[0][nt][0] : pb[0][nt][1], ((t & 7) << 2) | c);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                if (!((window(nt * 8 + 2 * c + h, t0) >> t) & 1u)) continue;
                const float w = from_16<T>(h ? pw >> 16 : pw & 0xffffu);
                // the weight is positive even where it is rounded to zero
                auto part = [&](int d) {
                  const uint16_t v = vr[at(d)];
                  return has_special<T>(v) ? from_16<T>(v) : w * from_16<T>(v);
                };
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                  o[k][nt][h] += part(k * 16 + g);
                  o[k][nt][2 + h] += part(k * 16 + g + 8);
                }
              }
            }
            __syncwarp();
            for (int d = lane; d < D; d += 32) vr[at(d)] = 0;
            __syncwarp();
          }
        }
      }
    }

    // O^T += V^T P^T
#pragma unroll
    for (int mt = 0; mt < S::kMt; ++mt) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        pb[mt][nt][0] = movmatrix_t(pb[mt][nt][0]);
        pb[mt][nt][1] = movmatrix_t(pb[mt][nt][1]);
      }
      if constexpr (Q8B) {
        const uint32_t vrow = mt * 16 + (lane & 7) + ((lj & 1) << 3);
#pragma unroll
        for (int k2 = 0; k2 < KS / 2; ++k2) {
          uint32_t r[4], a[4];
          ldsm_x4_t(vb + piece<S::kCpr>(vrow, 2 * k2 + (lj >> 1)), r[0], r[1], r[2], r[3]);
          Q8<FMT>::halves_t(r[0], a[0], a[1]);
          Q8<FMT>::halves_t(r[1], a[2], a[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816<MT>(o[2 * k2][nt], a, pb[mt][nt][0], pb[mt][nt][1]);
          Q8<FMT>::halves_t(r[2], a[0], a[1]);
          Q8<FMT>::halves_t(r[3], a[2], a[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816<MT>(o[2 * k2 + 1][nt], a, pb[mt][nt][0], pb[mt][nt][1]);
        }
      } else {
        const uint32_t vrow = mt * 16 + (lane & 7) + ((lj >> 1) << 3);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t a[4];
          ldsm_x4_t(vb + piece<S::kCpr>(vrow, 2 * k + (lj & 1)), a[0], a[1], a[2], a[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816<MT>(o[k][nt], a, pb[mt][nt][0], pb[mt][nt][1]);
        }
      }
    }
  }
  pdl_launch_dependents();

  // -------------------------------------------------------- join the warps ---
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int off = 4; off < 32; off <<= 1)
        l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], off);
  cp_async_wait<0>();
  __syncthreads();  // the rings are idle: their space holds the partials
  constexpr int OS = D + 4;
  float* po = reinterpret_cast<float*>(smem);                        // [warp][col][OS]
  float4* pm = reinterpret_cast<float4*>(po + kWarps * COLS * OS);   // [warp][col]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int col = nt * 8 + 2 * c + h;
      float* dst = po + (warp * COLS + col) * OS;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        if constexpr (Q8B) {  // rows g and g + 8 are d = 2 g and 2 g + 1
          *reinterpret_cast<float2*>(dst + k * 16 + 2 * g) =
              make_float2(o[k][nt][h], o[k][nt][2 + h]);
        } else {
          dst[k * 16 + g] = o[k][nt][h];
          dst[k * 16 + g + 8] = o[k][nt][2 + h];
        }
      }
      if (g == 0)
        pm[warp * COLS + col] = make_float4(m[nt][h], l[nt][h], Q8B ? M[nt][h] : m[nt][h], 0.f);
    }
  __syncthreads();
  const int H = p.H_kv * p.G;
  const bool whole = p.cluster == 1 && key0 == 0 && key1 == ctx;
  // the CTA's own partials, for its cluster: [col][OS], [col]
  float* co = reinterpret_cast<float*>(pm + kWarps * COLS);
  float4* cm = reinterpret_cast<float4*>(co + COLS * OS);
  for (int j = warp; j < COLS; j += kWarps) {
    const int token = col_token[j];
    if (token < 0) continue;
    float4 w[kWarps];
    float a = -3.402823466e38f, A = a;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      w[i] = pm[i * COLS + j];
      a = fmaxf(a, w[i].x);
      A = fmaxf(A, w[i].z);
    }
    float L = 0.f, f[kWarps];
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      L += w[i].y * ex2_mufu(w[i].x - a);
      f[i] = ex2_mufu(w[i].z - A);
    }
    const int64_t row = static_cast<int64_t>(row0 + token);
    // no visible key: L = 0 and the row is 0 / 0 = NaN
    const float fin = (Q8B ? exp2f(A - a) : 1.f) / L;
    const int64_t part = (row * H + col_head[j]) * p.nsplit + sp;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const int d = lane + 32 * i;
      float acc = 0.f;
#pragma unroll
      for (int t = 0; t < kWarps; ++t) acc += po[(t * COLS + j) * OS + d] * f[t];
      if (whole)
        static_cast<T*>(p.out)[row * p.out_stride + col_head[j] * D + d] = round_to<T>(acc * fin);
      else if (p.cluster > 1)
        co[j * OS + d] = acc;
      else
        p.part_o[part * D + d] = acc;
    }
    if (!whole && lane == 0)
      *(p.cluster > 1 ? cm + j : p.part_ml + part) = make_float4(a, L, A, 0.f);
  }
  if (p.cluster == 1) return;

  // ------------------------------------------------------ join the cluster ---
  // CTA r of the cluster joins columns r, r + n, ..., in split order.
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  cluster.sync();
  const int n_cta = min(p.cluster, max(1, (ctx + chunk - 1) / max(chunk, 1)));  // that held keys
  for (int j = sp + warp * p.cluster; j < COLS; j += kWarps * p.cluster) {
    const int token = col_token[j];
    if (token < 0) continue;
    float a = -3.402823466e38f, A = a;
    for (int i = 0; i < n_cta; ++i) {
      const float4 w = *cluster.map_shared_rank(cm + j, i);
      a = fmaxf(a, w.x);
      A = fmaxf(A, w.z);
    }
    float L = 0.f, acc[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
#pragma unroll 4
    for (int i = 0; i < n_cta; ++i) {
      const float4 w = *cluster.map_shared_rank(cm + j, i);
      const float* src = cluster.map_shared_rank(co + j * OS, i);
      const float f = ex2_mufu(w.z - A);
      L += w.y * ex2_mufu(w.x - a);
#pragma unroll
      for (int k = 0; k < D / 32; ++k) acc[k] += src[lane + 32 * k] * f;
    }
    const float fin = (Q8B ? exp2f(A - a) : 1.f) / L;
    T* dst = static_cast<T*>(p.out) + static_cast<int64_t>(row0 + token) * p.out_stride +
             col_head[j] * D;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) dst[lane + 32 * k] = round_to<T>(acc[k] * fin);
  }
  cluster.sync();  // no CTA leaves while another reads its partials
}

template <int FMT, typename T, int D, int NT>
int launch(const TreeParams& p, unsigned grid, cudaStream_t s) {
  constexpr int bytes = Smem<FMT, T, D, NT>::kBytes;
  auto* kernel = paged_tree_kernel<FMT, T, D, NT>;
  static std::atomic<uint64_t> ready{0};  // devices whose function attribute is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return LK_ERR_CUDA;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
        cudaSuccess)
      return LK_ERR_CUDA;
    if (dev < 64) ready.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  if (pdl_enabled()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (p.cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = p.cluster;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? check_launch() : LK_ERR_CUDA;
}

template <int FMT, typename T, int D>
int by_rows(const TreeParams& p, int NT, unsigned grid, cudaStream_t s) {
  switch (NT) {
    case 1: return launch<FMT, T, D, 1>(p, grid, s);
    case 2: return launch<FMT, T, D, 2>(p, grid, s);
    default: return launch<FMT, T, D, 4>(p, grid, s);
  }
}

template <int FMT>
int by_type(const TreeParams& p, int dtype, int D, int NT, unsigned grid, cudaStream_t s) {
  if (dtype == LK_DTYPE_BF16)
    return D == 128 ? by_rows<FMT, __nv_bfloat16, 128>(p, NT, grid, s)
                    : by_rows<FMT, __nv_bfloat16, 64>(p, NT, grid, s);
  return D == 128 ? by_rows<FMT, __half, 128>(p, NT, grid, s)
                  : by_rows<FMT, __half, 64>(p, NT, grid, s);
}

}  // namespace tree
}  // namespace lk
