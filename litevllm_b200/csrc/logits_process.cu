// Processing of a step's logits before sampling, in one pass over [B, V]: for
// token v of row b, with c = how often v occurs in the row's output tokens,
//   x = logits[b, v]
//   v in prompt or output: x = x > 0 ? x / rep_b : x * rep_b
//   x = x - (freq_b * c + pres_b * [c > 0])
//   x = x + the sum of the row's biases for v, in list order
//   v not allowed: x = -inf
// in fp32, each operation rounded as written, and once more to the logits'
// type. The repetition step is the reference's _apply_repetition_penalty
// (litevllm/layers/sampler.py:190-201); the others have no counterpart there.
//
// Bytes bound it: B * V logits in, B * V out, the mask's bits and the
// histories. CTA = (part of the vocabulary, row). Its logits go from global memory
// through registers and back with the mask applied, a dense pass that knows
// nothing of tokens; a vector that the mask closes is not read, and in place only
// closed tokens are written. Then the CTA counts the row's history tokens of its
// part in shared memory (so no [B, V] count tensor exists) and lists them, and
// computes those few tokens, and the biased ones, again from their logits, while
// other CTAs of the SM are in their dense pass. 128 x 151936 bf16 with 16 biases,
// histories of up to 1024 + 512 tokens and every fourth row under a mask that
// closes most of it (72 MB: closed vectors are not read): 24 us (3.0 TB/s; a bare
// copy 11); with the counts read for every vector it took 40. Every part looks
// through its row's whole history: 8192 + 2048 tokens take 62 us. 8 rows of 128256
// fp32: 4.9 us, a launch and one CTA's chain of dependent steps.
// Seven CTAs per SM leave 32 registers: the aligned forms spill 84 to 148 bytes, which
// the batch gains more than it costs; a few rows would not need so many CTAs.
// Rows whose addresses are not multiples of 16 bytes keep 16-byte accesses:
// tokens are indexed from the aligned address in front of the row.
#include "lk_common.cuh"
#include "lk_host.h"

namespace {

constexpr int kLThreads = 256;
constexpr int kLVecs = 4;        // 16-byte vectors per thread
constexpr int kLCtas = 7;        // CTAs per SM (5: 28.0 us, 7: 24.0; with the stores after the history 28.5)
constexpr int kLMaxBias = 1024;  // bias entries per row
constexpr int kLList = 2048;     // listed history tokens of a part; more: all counts are looked at

// What is known of a token, in C bits: in the prompt (top bit), biased (the next),
// occurrences in the output. 16 bits, two tokens a word, for outputs of up to 16383
// tokens: half the shared memory.
template <int C> struct Marks {
  static constexpr uint32_t kInPrompt = 1u << (C - 1), kBiased = 1u << (C - 2),
                            kCount = kBiased - 1u;
  LK_DEVINL static uint32_t get(const uint32_t* s, int at) {
    return C == 32 ? s[at] : (s[at >> 1] >> ((at & 1) * 16)) & 0xffffu;
  }
  // both return what was there before
  LK_DEVINL static uint32_t set(uint32_t* s, int at, uint32_t bits) {
    if (C == 32) return atomicOr(&s[at], bits);
    return (atomicOr(&s[at >> 1], bits << ((at & 1) * 16)) >> ((at & 1) * 16)) & 0xffffu;
  }
  LK_DEVINL static uint32_t count(uint32_t* s, int at) {
    if (C == 32) return atomicAdd(&s[at], 1u);
    return (atomicAdd(&s[at >> 1], 1u << ((at & 1) * 16)) >> ((at & 1) * 16)) & 0xffffu;
  }
};

struct LogitsParams {
  const void* logits;
  int64_t ld;
  void* out;
  int64_t out_ld;
  int V;
  const int64_t* prompt_ids;   // [B, prompt_ld]
  int64_t prompt_ld;
  const int32_t* prompt_lens;
  int prompt_max;
  const int64_t* output_ids;
  int64_t output_ld;
  const int32_t* output_lens;
  int output_max;
  const float* repetition;     // [B] or NULL
  const float* presence;
  const float* frequency;
  const int64_t* bias_ids;     // [B, nbias]
  const float* bias;
  int nbias;
  const uint32_t* allowed;     // [B, allowed_ld] bit words or NULL
  int64_t allowed_ld;
  int32_t* status;
};

template <typename T> struct Raw;
template <> struct Raw<float> {
  static constexpr int kVe = 4;
  // v where bit i of `open` allows its tokens, -inf elsewhere
  LK_DEVINL static uint4 masked(uint4 v, uint32_t open) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (!((open >> i) & 1u)) (&v.x)[i] = 0xff800000u;
    return v;
  }
  LK_DEVINL static float get(const uint4& v, int i) { return __uint_as_float((&v.x)[i]); }
  LK_DEVINL static void put(uint4& v, int i, float x) { (&v.x)[i] = __float_as_uint(x); }
  LK_DEVINL static float round(float x) { return x; }
};
template <typename T> struct Raw16 {
  static constexpr int kVe = 8;
  LK_DEVINL static uint4 masked(uint4 v, uint32_t open) {
    constexpr uint32_t inf = lk::Elem<T>::code == LK_DTYPE_BF16 ? 0xff80ff80u : 0xfc00fc00u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = ((open >> (2 * i)) & 1u ? 0x0000ffffu : 0u) |
                         ((open >> (2 * i)) & 2u ? 0xffff0000u : 0u);
      (&v.x)[i] = ((&v.x)[i] & m) | (inf & ~m);
    }
    return v;
  }
  LK_DEVINL static float get(const uint4& v, int i) {
    const uint16_t h = static_cast<uint16_t>((&v.x)[i >> 1] >> ((i & 1) * 16));
    return lk::Elem<T>::to_f(*reinterpret_cast<const T*>(&h));
  }
  LK_DEVINL static void put(uint4& v, int i, float x) {
    const T h = round(x);
    const uint32_t b = *reinterpret_cast<const uint16_t*>(&h);
    uint32_t& w = (&v.x)[i >> 1];
    w = (i & 1) ? (w & 0x0000ffffu) | (b << 16) : (w & 0xffff0000u) | b;
  }
  LK_DEVINL static T round(float x);
};
template <> LK_DEVINL __nv_bfloat16 Raw16<__nv_bfloat16>::round(float x) { return __float2bfloat16_rn(x); }
template <> LK_DEVINL __half Raw16<__half>::round(float x) { return __float2half_rn(x); }
template <> struct Raw<__nv_bfloat16> : Raw16<__nv_bfloat16> {};
template <> struct Raw<__half> : Raw16<__half> {};

struct RowTerms {
  float rep, pres, freq;
};

template <int C> LK_DEVINL float process(float x, uint32_t seen, const RowTerms& r) {
  if ((seen & ~Marks<C>::kBiased) == 0u) return x;
  x = x > 0.f ? __fdiv_rn(x, r.rep) : __fmul_rn(x, r.rep);
  const uint32_t c = seen & Marks<C>::kCount;
  const float p = c ? __fadd_rn(__fmul_rn(r.freq, static_cast<float>(c)), r.pres) : 0.f;
  return __fsub_rn(x, p);
}

template <typename T, bool VEC, int C>
__global__ void __launch_bounds__(kLThreads, kLCtas) logits_process_kernel(const LogitsParams p) {
  constexpr int VE = Raw<T>::kVe;
  constexpr int CH = kLThreads * kLVecs * VE;  // tokens per CTA
  constexpr uint32_t kAll = (1u << VE) - 1u;
  using Mk = Marks<C>;
  extern __shared__ __align__(16) uint32_t seen[];            // [CH] marks, only with sparse terms
  uint16_t* list = reinterpret_cast<uint16_t*>(seen + CH * C / 32);  // [kLList] seen tokens
  float* bias_v = reinterpret_cast<float*>(list + kLList);    // [nbias]
  int* bias_t = reinterpret_cast<int*>(bias_v + p.nbias);     // [nbias] token or -1
  __shared__ int listed;
  const int b = blockIdx.y, tid = threadIdx.x;
  const T* in = static_cast<const T*>(p.logits) + b * p.ld;
  T* out = static_cast<T*>(p.out) + b * p.out_ld;
  const bool in_place = static_cast<const void*>(in) == static_cast<const void*>(out);
  // token v sits at index v + shift from a 16-byte boundary
  const int shift = VEC ? static_cast<int>((reinterpret_cast<uintptr_t>(in) & 15u) / sizeof(T)) : 0;
  const int a0 = blockIdx.x * CH;
  const int a1 = min(a0 + CH, p.V + shift);
  if (a0 >= a1) return;
  const uint32_t* allowed = p.allowed ? p.allowed + b * p.allowed_ld : nullptr;

  RowTerms r;
  r.rep = p.repetition ? p.repetition[b] : 1.f;
  r.pres = p.presence ? p.presence[b] : 0.f;
  r.freq = p.frequency ? p.frequency[b] : 0.f;
  const bool past = r.pres != 0.f || r.freq != 0.f || r.rep != 1.f;
  const bool sparse = past || p.nbias > 0;
  // ------------------------------------------------ dense: loads under way ---
  // which tokens of each vector exist (live) and are allowed (open), a bit each
  uint32_t live[kLVecs], open[kLVecs];
  uint4 x[kLVecs];
  const bool inner = VEC && a0 >= shift && a0 + CH - shift <= p.V;  // every vector whole
  if (inner) {
    const int v0 = a0 - shift + tid * VE;
#pragma unroll
    for (int k = 0; k < kLVecs; ++k) {
      live[k] = open[k] = kAll;
      if (allowed) {
        const int v = v0 + k * kLThreads * VE;
        if (shift == 0) {  // a vector's bits are a byte or half of one
          open[k] = (__ldg(reinterpret_cast<const uint8_t*>(allowed) + (v >> 3)) >> (v & 7)) & kAll;
        } else {
          const uint32_t lo = __ldg(allowed + (v >> 5));
          const uint32_t hi = (v & 31) + VE > 32 ? __ldg(allowed + (v >> 5) + 1) : 0u;
          open[k] = __funnelshift_r(lo, hi, v & 31) & kAll;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kLVecs; ++k)
      x[k] = open[k] ? *reinterpret_cast<const uint4*>(in + v0 + k * kLThreads * VE)
                     : make_uint4(0u, 0u, 0u, 0u);
  } else {
    const int words = (p.V + 31) >> 5;
#pragma unroll
    for (int k = 0; k < kLVecs; ++k) {
      const int v = a0 + (k * kLThreads + tid) * VE - shift;
      const int skip = max(-v, 0), left = min(max(p.V - v, 0), VE);
      live[k] = left > skip ? ((1u << left) - 1u) & ~((1u << skip) - 1u) : 0u;
      open[k] = live[k];
      if (allowed && live[k]) {
        const int at = max(v, 0) >> 5, sh = max(v, 0) & 31;
        const uint32_t lo = __ldg(allowed + at);
        const uint32_t hi = sh + VE > 32 && at + 1 < words ? __ldg(allowed + at + 1) : 0u;
        open[k] &= __funnelshift_r(lo, hi, sh) << skip;
      }
      x[k] = make_uint4(0u, 0u, 0u, 0u);
      if (VEC && open[k] && live[k] == kAll) {
        x[k] = *reinterpret_cast<const uint4*>(in + v);
      } else if (open[k]) {
#pragma unroll
        for (int i = 0; i < VE; ++i)
          if ((live[k] >> i) & 1u) Raw<T>::put(x[k], i, lk::Elem<T>::to_f(in[v + i]));
      }
    }
  }

  // ---------------------------------------------------------- dense: stores ---
#pragma unroll
  for (int k = 0; k < kLVecs; ++k) {
    if (!live[k]) continue;
    const int v = a0 + (k * kLThreads + tid) * VE - shift;
    if (open[k] != live[k]) x[k] = Raw<T>::masked(x[k], open[k]);
    else if (in_place) continue;
    if (VEC && (inner || live[k] == kAll)) {
      *reinterpret_cast<uint4*>(out + v) = x[k];
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i)
        if ((live[k] >> i) & 1u) out[v + i] = Raw<T>::round(Raw<T>::get(x[k], i));
    }
  }
  if (!sparse) return;

  // ------------------------------------- the part's history and its biases ---
  for (int i = tid; i < CH * C / 128; i += kLThreads)
    reinterpret_cast<uint4*>(seen)[i] = make_uint4(0u, 0u, 0u, 0u);
  if (tid == 0) listed = 0;
  for (int j = tid; j < p.nbias; j += kLThreads) {
    const int64_t id = p.bias_ids[static_cast<int64_t>(b) * p.nbias + j];
    if (id >= p.V && p.status && blockIdx.x == 0) atomicOr(p.status, LK_STATUS_TOKEN_OOB);
    bias_t[j] = id < 0 || id >= p.V ? -1 : static_cast<int>(id);
    bias_v[j] = p.bias[static_cast<int64_t>(b) * p.nbias + j];
  }
  __syncthreads();
  auto note = [&](int64_t id, bool prompt) {
    if (id >= p.V && p.status && blockIdx.x == 0) atomicOr(p.status, LK_STATUS_TOKEN_OOB);
    if (id < 0 || id >= p.V) return;
    const int at = static_cast<int>(id) + shift - a0;
    if (at < 0 || at >= CH) return;
    const uint32_t was = prompt ? Mk::set(seen, at, Mk::kInPrompt) : Mk::count(seen, at);
    if ((was & ~Mk::kBiased) == 0u) {  // its first occurrence
      const int n = atomicAdd(&listed, 1);
      if (n < kLList) list[n] = static_cast<uint16_t>(at);
    }
  };
  if (past) {
    if (p.prompt_ids && r.rep != 1.f) {
      const int64_t* ids = p.prompt_ids + b * p.prompt_ld;
      const int n = p.prompt_lens ? min(p.prompt_lens[b], p.prompt_max) : p.prompt_max;
#pragma unroll 4
      for (int i = tid; i < n; i += kLThreads) note(__ldg(ids + i), true);
    }
    if (p.output_ids) {
      const int64_t* ids = p.output_ids + b * p.output_ld;
      const int n = p.output_lens ? min(p.output_lens[b], p.output_max) : p.output_max;
#pragma unroll 4
      for (int i = tid; i < n; i += kLThreads) note(__ldg(ids + i), false);
    }
  }
  for (int j = tid; j < p.nbias; j += kLThreads) {
    const int at = bias_t[j] + shift - a0;
    if (bias_t[j] >= 0 && at >= 0 && at < CH) Mk::set(seen, at, Mk::kBiased);
  }

  // ---------------------------------- sparse: after the vectors around them ---
  __syncthreads();
  auto is_open = [&](int v) { return !allowed || ((allowed[v >> 5] >> (v & 31)) & 1u); };
  auto one = [&](int at) {  // a history token without a bias
    const uint32_t s = Mk::get(seen, at);
    const int v = at + a0 - shift;
    if (s == 0u || (s & Mk::kBiased) || !is_open(v)) return;
    out[v] = Raw<T>::round(process<C>(lk::Elem<T>::to_f(in[v]), s, r));
  };
  if (listed <= kLList) {
    for (int i = tid; i < listed; i += kLThreads) one(list[i]);
  } else {
    for (int i = tid; i < a1 - a0; i += kLThreads) one(i);
  }
  for (int j = tid; j < p.nbias; j += kLThreads) {
    const int v = bias_t[j];
    const int at = v + shift - a0;
    if (v < 0 || at < 0 || at >= CH || !is_open(v)) continue;
    bool first = true;  // the first entry of a token adds up all of them, in list order
    float sum = 0.f;
#pragma unroll 8
    for (int i = 0; i < p.nbias; ++i) {
      const bool same = bias_t[i] == v;
      first &= !same || i >= j;
      sum = same ? __fadd_rn(sum, bias_v[i]) : sum;
    }
    if (!first) continue;
    out[v] = Raw<T>::round(__fadd_rn(process<C>(lk::Elem<T>::to_f(in[v]), Mk::get(seen, at), r), sum));
  }
}

template <typename T>
int launch_logits(const LogitsParams& p, int B, cudaStream_t s) {
  constexpr int CH = kLThreads * kLVecs * Raw<T>::kVe;
  const int parts = (p.V + 15 + CH - 1) / CH;  // room for the shift
  const bool sparse = p.repetition || p.presence || p.frequency || p.nbias > 0;
  const bool small = !p.output_ids || p.output_max <= static_cast<int>(Marks<16>::kCount);
  const size_t smem = sparse ? CH * (small ? 2 : 4) + kLList * 2 + static_cast<size_t>(p.nbias) * 8 : 0;
  const bool vec =
      ((reinterpret_cast<uintptr_t>(p.logits) ^ reinterpret_cast<uintptr_t>(p.out)) & 15u) == 0 &&
      (((p.ld - p.out_ld) * static_cast<int64_t>(sizeof(T))) & 15) == 0;
  static_assert(CH * 4 + kLList * 2 + kLMaxBias * 8 <= 48 * 1024, "no launch asks for more than the default");
  auto go = [&](auto* kernel) -> int {
    kernel<<<dim3(parts, B), kLThreads, smem, s>>>(p);
    return lk::check_launch();
  };
  if (small)
    return vec ? go(logits_process_kernel<T, true, 16>) : go(logits_process_kernel<T, false, 16>);
  return vec ? go(logits_process_kernel<T, true, 32>) : go(logits_process_kernel<T, false, 32>);
}

}  // namespace

extern "C" int lk_process_logits(
    void* out, int64_t out_ld, const void* logits, int32_t B, int32_t V, int64_t ld,
    const int64_t* prompt_ids, int64_t prompt_ld, const int32_t* prompt_lens, int32_t prompt_max,
    const int64_t* output_ids, int64_t output_ld, const int32_t* output_lens, int32_t output_max,
    const float* repetition, const float* presence, const float* frequency,
    const int64_t* bias_ids, const float* bias, int32_t num_bias, const int32_t* allowed,
    int64_t allowed_ld, int32_t dtype, int32_t* status, void* stream) {
  if (B < 0 || V <= 0 || ld < V || out_ld < V || prompt_max < 0 || output_max < 0 || num_bias < 0)
    return LK_ERR_INVALID_ARG;
  if (B == 0) return LK_OK;
  if (!out || !logits || (out == logits && out_ld != ld) || (prompt_max > 0 && !prompt_ids) ||
      (output_max > 0 && !output_ids) || (prompt_max > 0 && prompt_ld < prompt_max) ||
      (output_max > 0 && output_ld < output_max) || (num_bias > 0 && (!bias_ids || !bias)) ||
      (allowed && allowed_ld < (V + 31) / 32))
    return LK_ERR_INVALID_ARG;
  if (num_bias > kLMaxBias || B > 65535 || V > 0x7fff0000) return LK_ERR_UNSUPPORTED;
  LogitsParams p;
  p.logits = logits;
  p.ld = ld;
  p.out = out;
  p.out_ld = out_ld;
  p.V = V;
  p.prompt_ids = prompt_max > 0 ? prompt_ids : nullptr;
  p.prompt_ld = prompt_ld;
  p.prompt_lens = prompt_lens;
  p.prompt_max = prompt_max;
  p.output_ids = output_max > 0 ? output_ids : nullptr;
  p.output_ld = output_ld;
  p.output_lens = output_lens;
  p.output_max = output_max;
  p.repetition = repetition;
  p.presence = presence;
  p.frequency = frequency;
  p.bias_ids = bias_ids;
  p.bias = bias;
  p.nbias = num_bias;
  p.allowed = reinterpret_cast<const uint32_t*>(allowed);
  p.allowed_ld = allowed_ld;
  p.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case LK_DTYPE_BF16: return launch_logits<__nv_bfloat16>(p, B, s);
    case LK_DTYPE_F16: return launch_logits<__half>(p, B, s);
    case LK_DTYPE_F32: return launch_logits<float>(p, B, s);
    default: return LK_ERR_UNSUPPORTED;
  }
}
