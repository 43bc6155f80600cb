// Drafted-tree attention on the fifth-generation tensor cores, for calls with
// many query rows per KV head (n * G; paged_tree.cuh has the formulas and takes
// the small ones). A row of keys is then used by so many query rows that
// mma.sync, not HBM, is the limit there.
//
// CTA = (128 query rows of one KV head of one sequence, split of its keys), two
// CTAs per SM, keys in chunks of 64:
//  * one warp issues S = Q K^T (128 x 64, tcgen05, both operands in shared memory)
//    into two TMEM buffers in turn and O += P V with P from TMEM, over the first
//    half of its own S. S of the next chunk is issued before P V of this one, so
//    the tensor core works during the softmax; the SM's other CTA fills the rest,
//    set-up and tail among it.
//  * warps 0-3: softmax, one query row per thread, no shuffles. One pass over a
//    chunk's scores: weights are taken relative to a running maximum that is raised
//    (and O rescaled in TMEM, the chunk's weights redone) only where one would pass
//    2^8. Warps whose rows are all padding only keep the barriers going.
//  * K and V come with TMA (boxes of 16 slots through the block table, so block sizes
//    are multiples of 16), two stages deep. 16-bit rows land in the swizzled operand
//    tiles; a warp waits for K's tiles and another for V's.
//  * 8-bit rows land as bytes in the upper half of their operand tile; one warp copies
//    both, looking in turn which tile is free; two warps for K and two for V take the
//    bytes into registers and widen them to f16 (exactly) into the tile.
// Latencies bound its loop, not the tensor pipe: a chunk is 3500 cycles from copy to use,
// 900 S, 1500 the softmax, 900 P V, and two stages in each of two CTAs overlap them to
// 2300 (16 bits) and 3200 cycles a chunk (8). 32 trees of 20-32 nodes over 64-2048
// tokens, bf16, G = 4: 47 us (151 MB, 3.2 TB/s), the 32 chunks of the longest trees one
// after the other, as one wave of CTAs leaves no room to cut them. 16 trees of 48-64
// over 1K-8K, int8: 200 us (337 TFLOP/s). The loop is half of that: 62 chunks a resident
// CTA are 100 us, pieces of unequal length in the order of their start and 4 us of set-up
// each make it 128, the join is 17, and what the other 50 go to is not known (the tensor
// pipe is 22 % busy over all, 46 % would go with 3200 cycles a chunk throughout). With
// the bytes of one chunk of K at a time in a buffer of their own the int8 case took 254,
// with suspending waits for the copies 230, with one thread alone in the MMA warp's
// loop 212.
// The weights are rounded to the operand type for P V, as the tensor core takes it (the
// denominator sums them before): f16, 11 bits, over 8-bit caches; over a bf16 cache 8
// bits, each weight off by up to 2^-8 of itself, as in the other attention kernels here.
// In that case the result's error against 64 bits is 2.1e-3 where fp32 weights and
// the rounding of the result alone make 1.7e-3.
// Scales as in paged_tree.cuh, but with one running maximum, M, of the weights
// p s_v: the special-function unit (16 a clock) limits the softmax, so the weight is
// the product of 2^(x - M), which the denominator sums, and s_v. That costs nothing
// while the rows' scales stay within 2^-100 and 2^100 of one another's order: a
// smaller s_v counts as 2^-100 for M, and denominators of 2^-102 and less, where
// all scales are above 2^100, lose bits.
#pragma once

#include <atomic>
#include <type_traits>

#include "lk_q8.cuh"
#include "paged_tree.h"

namespace lk {
namespace treetc {

constexpr int kChunk = 64;     // keys per softmax step and per P V
constexpr int kRows = 128;     // query rows per CTA
constexpr float kRaise = 8.f;  // log2 of the largest weight
constexpr float kLow = -3.402823466e38f;

template <int FMT, int D> struct Shape {
  static constexpr bool kQ8 = FMT != LK_KV_16BIT;
  static constexpr int kHalves = D / 64;               // 128-byte column blocks of a 16-bit row
  static constexpr int kQHalf = kRows * 128;
  static constexpr int kQ = kHalves * kQHalf;
  static constexpr int kTHalf = kChunk * 128;
  static constexpr int kT = kHalves * kTHalf;          // operand tile of a K or V chunk
  static constexpr int kRaw = kQ8 ? kChunk * D : 0;    // a chunk's bytes, K or V
  static constexpr int kSmem = 1024 + kQ + 4 * kT;     // two tiles of each
  // warps: 0-3 softmax; 8-bit: 4, 5 widening K, 6, 7 V; 16-bit: 4 looking through V;
  // then one that issues MMAs and one copying (16-bit: one for each of K and V)
  static constexpr int kMma = kQ8 ? 8 : 5;
  static constexpr int kThreads = 32 * (kQ8 ? 10 : 8);
};

// 8-bit: the softmax takes registers from the widening warps. 128 x kSoftmaxRegs +
// 128 x kWidenRegs + 64 x 96 is the 320 x 96 the CTA is launched with.
constexpr int kSoftmaxRegs = 128, kWidenRegs = 64;
template <int N> LK_DEVINL void setmaxnreg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N> LK_DEVINL void setmaxnreg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <typename T> LK_DEVINL bool special16(uint32_t h) {  // infinity or NaN
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (h & e) == e;
}
template <typename T> LK_DEVINL float half_of(uint32_t w, int h) {
  const uint16_t v = static_cast<uint16_t>(h ? w >> 16 : w);
  return Elem<T>::to_f(*reinterpret_cast<const T*>(&v));
}

template <int FMT, typename T, int D>
__global__ void __launch_bounds__(Shape<FMT, D>::kThreads, 2)
paged_tree_tc_kernel(const __grid_constant__ CUtensorMap kmap,
                     const __grid_constant__ CUtensorMap vmap, const TreeParams p) {
  using S = Shape<FMT, D>;
  using MT = std::conditional_t<S::kQ8, __half, T>;  // operand type
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2],
      v_clean[2], s_full[2], p_full[2], o_done[2], sc_full[4], raw[2][2];
  __shared__ uint32_t tmem_slot;
  __shared__ __align__(16) float s_scale[S::kQ8 ? 4 : 1][2][kChunk];  // s_k, s_v of a chunk
  __shared__ float q_down[kRows];       // 8-bit: what undoes a row's scaling of Q
  __shared__ uint32_t v_special;        // some drafted V row has a special value
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + S::kQ;               // tile st at st * kT
  uint8_t* sV = sK + 2 * S::kT;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // Set-up before the wait for the kernel ahead (the store of this step's rows); global
  // memory is read after it, by ordinary loads (paged_tree.cuh says why).
  if (threadIdx.x == 0) {
    mbar_init(&q_full, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], S::kQ8 ? 1 : 2);  // P V done; looked through
      mbar_init(&v_clean[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
      mbar_init(&raw[0][i], 1);
      mbar_init(&raw[1][i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&sc_full[i], 1);
    fence_barrier_init();
    v_special = 0u;
  }
  if (warp == S::kMma) {
    __syncwarp();
    tc::alloc(&tmem_slot, 256);
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = tmem_slot;  // S buffers at columns 0 and 64, O from 128
  pdl_wait();

  // ------------------------------------------------------------- the work ---
  const int row_tiles = (p.max_q * p.G + kRows - 1) / kRows;
  unsigned rest = blockIdx.x;
  const int tile = rest % row_tiles;
  rest /= row_tiles;
  const int kvh = rest % p.H_kv;
  rest /= p.H_kv;
  const int b = rest % p.B;
  const int sp = rest / p.B;
  int row0;
  const int n = tree_tokens(p, b, &row0);
  int ctx = p.context_lens[b];
  if (ctx > p.max_blocks * p.bs || ctx < (p.cu_seqlens_q ? n : 0)) {
    if (threadIdx.x == 0 && p.status) atomicOr(p.status, LK_STATUS_CTX_OOB);
    ctx = max(min(ctx, p.max_blocks * p.bs), 0);
  }
  const int rows = n * p.G - tile * kRows;  // of this CTA's, may pass kRows
  const int key0 = sp * p.chunk;
  const bool live = rows > 0 && (key0 < ctx || sp == 0);
  const int key1 = min(ctx, key0 + p.chunk);
  const int open = max(ctx - n, 0);  // keys below are seen by every row
  const int chunks = live ? (key1 - key0 + kChunk - 1) / kChunk : 0;
  // 16-bit V chunks that are looked through before use: drafted keys, and rows
  // behind the context in its last block. They are the last chunks of a context.
  auto unclean = [&](int k) {
    const int end = key0 + (k + 1) * kChunk;
    return !S::kQ8 && (end > open || end > key1);
  };

  // Copies of a warp: chunk k of K or V as TMA boxes of 16 slots. A lane holds the
  // first slot of one of the boxes of eight chunks, and of the eight after them.
  const int32_t* bt = p.block_tables + static_cast<int64_t>(b) * p.bt_stride;
  const int none = max(static_cast<int>(p.num_blocks) * p.bs, 1);  // TMA reads zeros there
  auto boxes_of = [&](int k0) {
    const int key = key0 + k0 * kChunk + lane * 16;
    if (chunks == 0 || key >= key1) return none;
    const int q = tree_quotient(p, key);
    const int blk = bt[q];
    if (blk < 0 || blk >= p.num_blocks) {
      if (p.status) atomicOr(p.status, LK_STATUS_BLOCK_OOB);
      return none;
    }
    return blk * p.bs + (key - q * p.bs);
  };
  int boxes[2] = {none, none}, ahead[2] = {none, none};  // K's, V's
  auto copy = [&](int k, int is_v, const CUtensorMap* map, uint64_t* full, uint8_t* dst) {
    if ((k & 7) == 0) {
      boxes[is_v] = k == 0 ? boxes_of(0) : ahead[is_v];
      ahead[is_v] = boxes_of(k + 8);
    }
    int slot[kChunk / 16];
#pragma unroll
    for (int i = 0; i < kChunk / 16; ++i)
      slot[i] = __shfl_sync(0xffffffffu, boxes[is_v], (k & 7) * 4 + i);
    if (lane == 0) {
      mbar_arrive_expect_tx(full, S::kQ8 ? S::kRaw : S::kT);
#pragma unroll
      for (int i = 0; i < kChunk / 16; ++i) {
        if constexpr (S::kQ8) {
          tma_load_3d(dst + i * 16 * D, map, full, 0, slot[i], kvh);
        } else {
#pragma unroll
          for (int c = 0; c < S::kHalves; ++c)
            tma_load_3d(dst + c * S::kTHalf + i * 2048, map, full, c * 64, slot[i], kvh);
        }
      }
    }
    __syncwarp();
  };

  if (warp == S::kMma) {
    // ---------------------------------------------------------- MMA issue ---
    if (chunks > 0) {
      constexpr int fmt = std::is_same<MT, __nv_bfloat16>::value ? 1 : 0;
      constexpr uint32_t idS = tc::idesc_f16(fmt, 0, 0, kRows, kChunk);
      constexpr uint32_t idO = tc::idesc_f16(fmt, 0, 1, kRows, D);
      // descriptors differ in their address field alone: bytes / 16
      const uint64_t dq = tc::smem_desc_sw128(smem_u32(sQ), 16, 1024);
      const uint64_t dk = tc::smem_desc_sw128(smem_u32(sK), 16, 1024);
      const uint64_t dv = tc::smem_desc_sw128(smem_u32(sV), S::kTHalf, 1024);
      bool ok = __all_sync(0xffffffffu, mbar_wait(&q_full, 0));
      const bool one = tc::elect();  // the thread that issues; all take part in the waits
      auto issue_s = [&](int k) {
        const int st = k & 1;
        ok = ok && __all_sync(0xffffffffu, mbar_wait(&k_full[st], (k >> 1) & 1));
        if (!ok) return;
        tc::fence_after();
        const uint64_t dks = dk + st * (S::kT / 16);
        if (one) {
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks)
            tc::mma_f16(tmem + 64 * st, dq + ((ks >> 2) * S::kQHalf + (ks & 3) * 32) / 16,
                        dks + ((ks >> 2) * S::kTHalf + (ks & 3) * 32) / 16, idS, ks > 0 ? 1u : 0u);
          tc::commit(&s_full[st]);
          tc::commit(&k_empty[st]);
        }
        __syncwarp();
      };
      issue_s(0);
      int cleaned = 0;  // unclean chunks so far
      for (int k = 0; k < chunks && ok; ++k) {
        const int vs = k & 1;
        if (k + 1 < chunks) issue_s(k + 1);  // over S and P of chunk k - 1, whose P V was issued
        ok = ok && __all_sync(0xffffffffu, mbar_wait(&v_full[vs], (k >> 1) & 1));
        if (ok && unclean(k)) {
          ok = __all_sync(0xffffffffu, mbar_wait(&v_clean[cleaned & 1], (cleaned >> 1) & 1));
          ++cleaned;
        }
        ok = ok && __all_sync(0xffffffffu, mbar_wait(&p_full[k & 1], (k >> 1) & 1));
        if (!ok) break;
        tc::fence_after();
        const uint64_t dvs = dv + vs * (S::kT / 16);
        if (one) {
#pragma unroll
          for (int kk = 0; kk < kChunk / 16; ++kk)
            tc::mma_f16_ts(tmem + 128, tmem + 64 * (k & 1) + kk * 8, dvs + kk * (2048 / 16), idO,
                           (k > 0 || kk > 0) ? 1u : 0u);
          tc::commit(&v_empty[vs]);
          tc::commit(&o_done[k & 1]);
        }
        __syncwarp();
      }
      if (!ok && p.status && one) atomicOr(p.status, LK_STATUS_WAIT_TIMEOUT);
    }
  } else if (warp > S::kMma) {
    // -------------------------------------------------------------- copies ---
    // 16-bit: a warp waits for the tiles of K, another for V's; 8-bit: one looks at both
    constexpr bool both = S::kQ8;
    const bool does_k = both || warp == S::kMma + 1, does_v = both || !does_k;
    if (lane < 2) prefetch_tensormap(lane ? &vmap : &kmap);
    int next_k = does_k ? 0 : chunks, next_v = does_v ? 0 : chunks;  // chunks to start
    auto ready = [&](uint64_t* bar, uint32_t parity) {
      return both ? mbar_test(bar, parity) : mbar_try_wait(bar, parity);
    };
    uint64_t t0 = globaltimer_ns();
    while (next_k < chunks || next_v < chunks) {
      bool moved = false;
      if (next_k < chunks) {
        const int st = next_k & 1;
        if (__all_sync(0xffffffffu, ready(&k_empty[st], ((next_k >> 1) & 1) ^ 1))) {
          copy(next_k, 0, &kmap, S::kQ8 ? &raw[0][st] : &k_full[st], sK + st * S::kT + S::kRaw);
          ++next_k;
          moved = true;
        }
      }
      if (next_v < chunks) {
        const int st = next_v & 1;
        if (__all_sync(0xffffffffu, ready(&v_empty[st], ((next_v >> 1) & 1) ^ 1))) {
          copy(next_v, 1, &vmap, S::kQ8 ? &raw[1][st] : &v_full[st], sV + st * S::kT + S::kRaw);
          ++next_v;
          moved = true;
        }
      }
      if (moved) {
        t0 = globaltimer_ns();
      } else if (__any_sync(0xffffffffu, globaltimer_ns() - t0 > kWaitTimeoutNs)) {
        if (p.status && lane == 0) atomicOr(p.status, LK_STATUS_WAIT_TIMEOUT);
        break;
      }
    }
  } else if (warp >= 4) {
    bool ok = true;
    if constexpr (!S::kQ8) {
      // ------------------------------------------------ looking through V ---
      // Special values of drafted tokens would reach rows that do not see them
      // through 0 * inf, and so would what is left behind the context in its last
      // block: they are zeroed in the tile, and the epilogue gives the drafted ones
      // to the rows that see them. Rows below `open` are seen by all. This warp
      // takes part in every stage's release, so it never misses a phase.
      int cleaned = 0;
      for (int k = 0; k < chunks; ++k) {
        const int st = k & 1;
        ok = mbar_wait(&v_full[st], (k >> 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (unclean(k)) {
          const int t0 = key0 + k * kChunk;
          const int last = min(kChunk, (key1 - t0 + 15) / 16 * 16);
          for (int r = max(open - t0, 0) + lane / 8; r < last; r += 4) {
#pragma unroll
            for (int c = 0; c < S::kHalves; ++c) {
              uint4* at = reinterpret_cast<uint4*>(sV + st * S::kT + c * S::kTHalf +
                                                   swz128(r, lane & 7));
              uint4 v = *at;
              uint32_t* w = &v.x;
              bool hit = false;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const bool lo = special16<T>(w[e]), hi = special16<T>(w[e] >> 16);
                hit |= lo | hi;
                w[e] = (lo ? 0u : w[e] & 0xffffu) | (hi ? 0u : w[e] & 0xffff0000u);
              }
              if (hit) {
                *at = v;
                if (t0 + r < key1) atomicOr(&v_special, 1u);
              }
            }
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_clean[cleaned & 1]);
          ++cleaned;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_empty[st]);
      }
    } else {
      // ------------------------------------------------------ 8-bit widening ---
      __syncwarp();  // all 32 lanes issue it together
      setmaxnreg_dec<kWidenRegs>();
      const bool is_v = warp >= 6;
      const int g = threadIdx.x & 63;
      constexpr int kPieces = S::kRaw / 1024;  // 16-byte pieces of a chunk per thread
      // Of a piece, 16 columns c of row r, a thread takes the same c in every (1024 / D)th
      // row, so its swizzled places are steps of one. In the columns' second half rows
      // are swapped in pairs: eight lanes write to eight different banks.
      constexpr int kStep = 1024 / D;
      const int c = g % (D / 16), r0 = (g / (D / 16)) ^ (c >> 2);
      const int from = S::kRaw + r0 * D + c * 16;
      const int to0 = (c >> 2) * S::kTHalf + swz128(r0, (2 * c) & 7);
      const int to1 = (c >> 2) * S::kTHalf + swz128(r0, (2 * c + 1) & 7);
      // K side: the scales of key g, loaded one chunk ahead, its block two
      int blk = -1;
      float2 cur, nxt = make_float2(0.f, 0.f);
      auto block_at = [&](int k) {
        const int key = key0 + k * kChunk + g;
        blk = k < chunks && key < key1 ? bt[tree_quotient(p, key)] : -1;
        if (blk >= p.num_blocks) blk = -1;  // flagged by the copies
      };
      auto scales = [&](int k) {
        const int key = key0 + k * kChunk + g;
        const int64_t at = (static_cast<int64_t>(blk) * p.H_kv + kvh) * p.bs +
                           (key - tree_quotient(p, key) * p.bs);
        nxt = blk < 0 ? make_float2(0.f, 0.f) : make_float2(p.k_scale[at], p.v_scale[at]);
      };
      if (!is_v) {
        block_at(0);
        scales(0);
        block_at(1);
      }
      for (int k = 0; k < chunks; ++k) {
        if (!is_v) {
          cur = nxt;
          scales(k + 1);
          block_at(k + 2);
        }
        const int st = k & 1;
        uint8_t* tile_at = (is_v ? sV : sK) + st * S::kT;
        ok = mbar_wait(&raw[is_v][st], (k >> 1) & 1);
        uint4 w[kPieces];
        if (ok) {
#pragma unroll
          for (int i = 0; i < kPieces; ++i)
            w[i] = *reinterpret_cast<const uint4*>(tile_at + from + i * 1024);
        }
        // all 64 threads have their bytes: the tile may be written
        ok = is_v ? named_sync_and(2, 64, ok) : named_sync_and(1, 64, ok);
        if (!ok) break;
        {
          const int left = key1 - (key0 + k * kChunk);
          if (left < kChunk) {  // rows behind the context may hold anything
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
              if (r0 + i * kStep >= left) w[i] = make_uint4(0u, 0u, 0u, 0u);
          }
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            uint4 x, y;
            Q8<FMT>::halves(w[i].x, x.x, x.y);
            Q8<FMT>::halves(w[i].y, x.z, x.w);
            Q8<FMT>::halves(w[i].z, y.x, y.y);
            Q8<FMT>::halves(w[i].w, y.z, y.w);
            *reinterpret_cast<uint4*>(tile_at + to0 + i * kStep * 128) = x;
            *reinterpret_cast<uint4*>(tile_at + to1 + i * kStep * 128) = y;
          }
          if (!is_v) {
            s_scale[k & 3][0][g] = cur.x;
            s_scale[k & 3][1][g] = cur.y;
          }
          fence_proxy_async();
        }
        ok = is_v ? named_sync_and(2, 64, ok) : named_sync_and(1, 64, ok);
        if (!ok) break;
        if (g == 0) {
          mbar_arrive(is_v ? &v_full[st] : &k_full[st]);
          if (!is_v) mbar_arrive(&sc_full[k & 3]);
        }
      }
    }
    if (!ok && p.status && lane == 0) atomicOr(p.status, LK_STATUS_WAIT_TIMEOUT);
  } else {
    // ------------------------------------------------------------- softmax ---
    // Waits, masks and special values part the lanes of a warp: before each of the
    // instructions that all 32 have to issue together (register split, TMEM loads and
    // stores) they are brought together again.
    __syncwarp();
    if constexpr (S::kQ8) setmaxnreg_inc<kSoftmaxRegs>();
   if (live) {
    const int t = threadIdx.x;                           // row of the CTA
    const int wrow = warp * 32;
    const bool row_ok = t < rows;
    const bool warp_ok = wrow < rows;                    // some row of the warp is real
    const int r = tile * kRows + t;
    const int token = row_ok ? tree_token(p, r) : 0;
    const int head = kvh * p.G + (row_ok ? r - token * p.G : 0);
    const uint32_t lanes = static_cast<uint32_t>(wrow) << 16;
    const uint32_t tO = tmem + 128;
    const int64_t qrow = row0 + token;
    // mask words of the row: those that its first drafted chunk here needs
    const int word0 = max(key0 - open, 0) >> 6;
    uint64_t mask_a = 0ull, mask_b = 0ull;
    const int64_t* mask = p.mask ? p.mask + qrow * p.mask_stride : nullptr;
    if (mask) {
      if (word0 < p.mask_words) mask_a = mask[word0];
      if (word0 + 1 < p.mask_words) mask_b = mask[word0 + 1];
    }
    float cs = p.scale_log2;
    if (warp_ok) {
      // the warp's 32 rows of Q, 16 bytes a lane
      constexpr int LPR = D / 8;                 // lanes per row
      const int c = lane % LPR;
      const T* qb = static_cast<const T*>(p.q) + static_cast<int64_t>(kvh) * p.G * D + 8 * c;
      const bool vec = (reinterpret_cast<uintptr_t>(p.q) & 15u) == 0 && (p.q_stride & 7) == 0;
      auto row_of = [&](int i) { return wrow + i * (32 / LPR) + lane / LPR; };
      auto load8 = [&](int i) {  // LPR steps of 32 / LPR rows
        const int rr = row_of(i);
        if (rr >= rows) return make_uint4(0u, 0u, 0u, 0u);
        const int rg = tile * kRows + rr;
        const int tok = tree_token(p, rg);
        const T* src = qb + static_cast<int64_t>(row0 + tok) * p.q_stride + (rg - tok * p.G) * D;
        if (vec) return *reinterpret_cast<const uint4*>(src);
        const uint16_t* s = reinterpret_cast<const uint16_t*>(src);
        return make_uint4(s[0] | (s[1] << 16), s[2] | (s[3] << 16), s[4] | (s[5] << 16),
                          s[6] | (s[7] << 16));
      };
      auto put8 = [&](int i, uint4 x) {
        const int rr = row_of(i);
        if constexpr (S::kQ8) {
          float f[8];
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
          float top = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            f[e] = half_of<T>(w[e >> 1], e & 1);
            top = fmaxf(top, fabsf(f[e]));
          }
#pragma unroll
          for (int o = LPR / 2; o > 0; o >>= 1)
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          // the power of two that brings the row's largest value into [2^14, 2^15)
          const int e = __float_as_int(top) >> 23;
          float up = 1.f, down = 1.f;
          if (e > 0 && e < 255) {
            const int q = min(268 - e, 253);
            up = __int_as_float(q << 23);
            down = __int_as_float((254 - q) << 23);
          }
          x = make_uint4(pack2<__half>(f[0] * up, f[1] * up), pack2<__half>(f[2] * up, f[3] * up),
                         pack2<__half>(f[4] * up, f[5] * up), pack2<__half>(f[6] * up, f[7] * up));
          if (c == 0) q_down[rr] = down;
        }
        *reinterpret_cast<uint4*>(sQ + (c >> 3) * S::kQHalf + swz128(rr, c & 7)) = x;
      };
      if (vec) {
        uint4 x[LPR];
#pragma unroll
        for (int i = 0; i < LPR; ++i) x[i] = load8(i);
#pragma unroll
        for (int i = 0; i < LPR; ++i) put8(i, x[i]);
      } else {
#pragma unroll 1
        for (int i = 0; i < LPR; ++i) put8(i, load8(i));
      }
      fence_proxy_async();
    }
    __syncwarp();
    if (S::kQ8 && warp_ok) cs *= q_down[t];
    if (lane == 0) mbar_arrive(&q_full);

    // The keys t0 .. t0 + 63 that this row sees, one bit each.
    auto window = [&](int t0) {
      const int s = t0 - open;
      uint64_t bits = ~0ull;
      if (s > -kChunk) {
        const int lo = max(s, 0);
        uint64_t w = 0ull;
        if (mask == nullptr) {
          const int k = token + 1 - lo;
          w = k <= 0 ? 0ull : k >= 64 ? ~0ull : (1ull << k) - 1;
        } else {
          const int at = lo >> 6, sh = lo & 63;
          uint64_t a = mask_a, c = mask_b;
          if (at != word0) {
            a = at < p.mask_words ? static_cast<uint64_t>(mask[at]) : 0ull;
            c = at + 1 < p.mask_words ? static_cast<uint64_t>(mask[at + 1]) : 0ull;
          }
          w = a >> sh;
          if (sh) w |= c << (64 - sh);
        }
        bits = s >= 0 ? w : (w << -s) | ((1ull << -s) - 1);
      }
      const int left = key1 - t0;
      return left >= 64 ? bits : bits & ((1ull << left) - 1);
    };

    float m = kLow, l = 0.f;  // 8-bit: m is the maximum of the weights p s_v
    bool ok = true;
    for (int k = 0; k < chunks; ++k) {
      ok = mbar_wait(&s_full[k & 1], (k >> 1) & 1);
      if constexpr (S::kQ8) ok = ok && mbar_wait(&sc_full[k & 3], (k >> 2) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (warp_ok) {
        tc::fence_after();
        const uint32_t tS = tmem + lanes + 64 * (k & 1);
        const int t0 = key0 + k * kChunk;
        const bool masked = t0 + kChunk > min(key1, open);
        const uint64_t bits = masked ? window(t0) : ~0ull;
        const float* sk = s_scale[S::kQ8 ? k & 3 : 0][0];
        const float* sv_ = s_scale[S::kQ8 ? k & 3 : 0][1];
        uint32_t pw[kChunk / 2];
        float sum0, sum1;
        bool up = k == 0;
        // The chunk's weights for the present maxima: pw, their sum, the
        // largest; again after the maxima are raised.
        bool raise = k == 0;
        for (;;) {
          if (raise) {
            // new maxima of the rows that need them, from the scores themselves
            float a = m;
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
              uint32_t sv[32];
              __syncwarp();
              tc::ld32(tS + 32 * c, sv);
              tc::wait_ld();
              const uint32_t seen = static_cast<uint32_t>(bits >> (32 * c));
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                float y = __uint_as_float(sv[i]) * cs;
                if constexpr (S::kQ8)
                  y = fmaf(y, sk[32 * c + i], fmaxf(__log2f(sv_[32 * c + i]), -100.f));
                if ((seen >> i) & 1u) a = fmaxf(a, y);
              }
            }
            if (!up) a = m;
            const float alpha = ex2_mufu(m - a);
            l *= alpha;
            m = a;
            if (k > 0) {
              // O is stable once P V of chunk k - 1 has completed; P V of chunk k
              // waits for this warp's P
              ok = __all_sync(0xffffffffu, mbar_wait(&o_done[(k - 1) & 1], ((k - 1) >> 1) & 1));
              if (!ok) break;
              tc::fence_after();
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t ov[32];
                tc::ld32(tO + lanes + 32 * c, ov);
                tc::wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
                tc::st32(tO + lanes + 32 * c, ov);
              }
              tc::wait_st();
            }
          }
          __syncwarp();  // inside weigh() it costs 84 bytes of spills
          float top = -INFINITY;  // of the exponents (8-bit: of the weights)
          sum0 = sum1 = 0.f;
          auto weigh = [&](auto with_mask) {
            uint32_t sv[64];
            tc::ld32(tS, *reinterpret_cast<uint32_t(*)[32]>(sv));
            tc::ld32(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(sv + 32));
            tc::wait_ld();
#pragma unroll
            for (int i = 0; i < 64; i += 4) {
              float e[4];
              [[maybe_unused]] float ks[4], vs[4];
              if constexpr (S::kQ8) {
                const float4 a = *reinterpret_cast<const float4*>(sk + i);
                const float4 c = *reinterpret_cast<const float4*>(sv_ + i);
                ks[0] = a.x; ks[1] = a.y; ks[2] = a.z; ks[3] = a.w;
                vs[0] = c.x; vs[1] = c.y; vs[2] = c.z; vs[3] = c.w;
              }
              float d[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float x = __uint_as_float(sv[i + j]);
                d[j] = S::kQ8 ? fmaf(x * ks[j], cs, -m) : fmaf(x, cs, -m);
                if (decltype(with_mask)::value && !((bits >> (i + j)) & 1ull)) d[j] = -INFINITY;
                e[j] = ex2_mufu(d[j]);
              }
              if constexpr (!S::kQ8) {
                top = fmax3(top, d[0], d[1]);
                top = fmax3(top, d[2], d[3]);
              }
              sum0 += e[0];
              sum1 += e[1];
              sum0 += e[2];
              sum1 += e[3];
              if constexpr (S::kQ8) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  e[j] *= vs[j];
                  // zero even where the hidden row's scale is NaN
                  if (decltype(with_mask)::value && !((bits >> (i + j)) & 1ull)) e[j] = 0.f;
                }
                top = fmax3(top, e[0], e[1]);
                top = fmax3(top, e[2], e[3]);
              }
              pw[i >> 1] = pack2<MT>(e[0], e[1]);
              pw[(i >> 1) + 1] = pack2<MT>(e[2], e[3]);
            }
          };
          if (masked) weigh(std::true_type());
          else weigh(std::false_type());
          if (raise) break;
          // 8-bit: a weight is small, or 0 times infinity, where s_v is, while its 2^(x - M)
          // in the denominator passes all bounds; raised maxima keep the sum below 2^106
          up = S::kQ8 ? top > 256.f || sum0 + sum1 > 0x1p110f : top > kRaise;
          raise = __any_sync(0xffffffffu, up);
          if (!raise) break;
        }
        if (!ok) break;  // alike in all lanes
        l += sum0 + sum1;
        __syncwarp();
        tc::st32(tS, pw);
        tc::wait_st();
        tc::fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[k & 1]);
    }
    if (!ok && p.status && lane == 0) atomicOr(p.status, LK_STATUS_WAIT_TIMEOUT);
    pdl_launch_dependents();

    // ------------------------------------------------------------ epilogue ---
    if (ok && warp_ok) {
      if (chunks > 0) {
        // two barriers: with one, the phase before the last could pass for the last
        ok = mbar_wait(&o_done[(chunks - 1) & 1], ((chunks - 1) >> 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        tc::fence_after();
      }
      const int H = p.H_kv * p.G;
      const bool whole = key0 == 0 && key1 == ctx;
      // no visible key: l = 0 and the row is 0 / 0 = NaN
      const float fin = whole ? 1.f / l : 1.f;
      const int64_t part = (qrow * H + head) * p.nsplit + sp;
      T* out = static_cast<T*>(p.out) + qrow * p.out_stride + static_cast<int64_t>(head) * D;
      const bool vec = ((reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
      const bool special = !S::kQ8 && v_special != 0u;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t ov[32];
        if (chunks > 0) {
          __syncwarp();  // lanes part below
          tc::ld32(tO + lanes + 32 * c, ov);
          tc::wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) ov[i] = 0u;
        }
        if (special) {
          // special values of drafted tokens that this row sees (their weight is
          // positive: it only gives them their place in the sum)
          for (int key = max(key0, open); key < key1; ++key) {
            if (!(window(key) & 1ull)) continue;
            const int q = key / p.bs;
            const int blk = p.block_tables[b * p.bt_stride + q];
            if (blk < 0 || blk >= p.num_blocks) continue;
            const T* vr = static_cast<const T*>(p.v) +
                          (static_cast<int64_t>(blk) * p.bs + key % p.bs) * p.H_kv * D +
                          static_cast<int64_t>(kvh) * D + 32 * c;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float v = Elem<T>::to_f(vr[i]);
              if (!(fabsf(v) <= -kLow)) ov[i] = __float_as_uint(__uint_as_float(ov[i]) + v);
            }
          }
        }
        if (row_ok && whole) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = pack2<T>(__uint_as_float(ov[i + 2 * e]) * fin,
                              __uint_as_float(ov[i + 2 * e + 1]) * fin);
            if (vec) {
              *reinterpret_cast<uint4*>(out + 32 * c + i) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
              uint16_t* o16 = reinterpret_cast<uint16_t*>(out) + 32 * c + i;
#pragma unroll
              for (int e = 0; e < 8; ++e)
                o16[e] = static_cast<uint16_t>(w[e >> 1] >> ((e & 1) * 16));
            }
          }
        } else if (row_ok) {
          float4* po = reinterpret_cast<float4*>(p.part_o + part * D + 32 * c);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            po[i] = make_float4(__uint_as_float(ov[4 * i]), __uint_as_float(ov[4 * i + 1]),
                                __uint_as_float(ov[4 * i + 2]), __uint_as_float(ov[4 * i + 3]));
        }
      }
      if (row_ok && !whole) p.part_ml[part] = make_float4(m, l, m, 0.f);
    }
   }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  __syncwarp();
  if (warp == S::kMma) tc::dealloc(tmem, 256);
}

template <int FMT, typename T, int D>
int launch(const TreeParams& p, unsigned grid, cudaStream_t s) {
  constexpr int bytes = Shape<FMT, D>::kSmem;
  auto* kernel = paged_tree_tc_kernel<FMT, T, D>;
  static std::atomic<uint64_t> ready{0};  // devices whose function attribute is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return LK_ERR_CUDA;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
        cudaSuccess)
      return LK_ERR_CUDA;
    if (Shape<FMT, D>::kQ8) {  // a build whose registers do not add up must not wait for them
      cudaFuncAttributes a;
      if (cudaFuncGetAttributes(&a, kernel) != cudaSuccess) return LK_ERR_CUDA;
      if (128 * (kSoftmaxRegs + kWidenRegs) > 256 * a.numRegs) return LK_ERR_UNSUPPORTED;
    }
    if (dev < 64) ready.fetch_or(bit, std::memory_order_relaxed);
  }
  CUtensorMap km, vm;
  const int kind = FMT != LK_KV_16BIT ? kMapBytes : Elem<T>::code;
  const int64_t slots = p.num_blocks > 0 ? p.num_blocks * p.bs : 1;  // a map is never empty
  int rc = make_kv_tensor_map(&km, p.k, slots, p.H_kv, D, kind, 16, 1);
  if (rc == LK_OK) rc = make_kv_tensor_map(&vm, p.v, slots, p.H_kv, D, kind, 16, 1);
  if (rc != LK_OK) return rc;
  if (launch_after_previous(kernel, dim3(grid), dim3(Shape<FMT, D>::kThreads), bytes, s, km, vm, p) != cudaSuccess)
    return LK_ERR_CUDA;
  return check_launch();
}

template <int FMT>
int by_type(const TreeParams& p, int dtype, int D, unsigned grid, cudaStream_t s) {
  if (dtype == LK_DTYPE_BF16)
    return D == 128 ? launch<FMT, __nv_bfloat16, 128>(p, grid, s)
                    : launch<FMT, __nv_bfloat16, 64>(p, grid, s);
  return D == 128 ? launch<FMT, __half, 128>(p, grid, s) : launch<FMT, __half, 64>(p, grid, s);
}

}  // namespace treetc
}  // namespace lk
