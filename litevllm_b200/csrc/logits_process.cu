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
// histories. CTA = (part of the vocabulary, row): it counts the row's history
// tokens that fall into its part in shared memory (top bit: in the prompt, the
// rest: occurrences in the output), so no [B, V] count tensor exists, while
// its logits are already on their way to registers. A part that the mask
// closes is not read, and in place only what changes is written.
// Rows whose addresses are not multiples of 16 bytes keep 16-byte accesses:
// tokens are indexed from the aligned address in front of the row.
#include "lk_common.cuh"
#include "lk_host.h"

namespace {

constexpr int kLThreads = 256;
constexpr int kLVecs = 4;        // 16-byte vectors per thread
constexpr int kLMaxBias = 1024;  // bias entries per row
constexpr uint32_t kInPrompt = 0x80000000u;

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
  LK_DEVINL static float get(const uint4& v, int i) { return __uint_as_float((&v.x)[i]); }
  LK_DEVINL static void put(uint4& v, int i, float x) { (&v.x)[i] = __float_as_uint(x); }
  LK_DEVINL static float round(float x) { return x; }
};
template <typename T> struct Raw16 {
  static constexpr int kVe = 8;
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

LK_DEVINL float process(float x, uint32_t seen, const RowTerms& r) {
  if (seen == 0u) return x;
  x = x > 0.f ? __fdiv_rn(x, r.rep) : __fmul_rn(x, r.rep);
  const uint32_t c = seen & ~kInPrompt;
  const float p = c ? __fadd_rn(__fmul_rn(r.freq, static_cast<float>(c)), r.pres) : 0.f;
  return __fsub_rn(x, p);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kLThreads) logits_process_kernel(const LogitsParams p) {
  constexpr int VE = Raw<T>::kVe;
  constexpr int CH = kLThreads * kLVecs * VE;  // tokens per CTA
  extern __shared__ uint32_t seen[];           // [CH], then the biases
  float* bias_x = reinterpret_cast<float*>(seen + CH);        // [nbias] results
  float* bias_v = bias_x + p.nbias;                            // [nbias]
  int* bias_t = reinterpret_cast<int*>(bias_v + p.nbias);      // [nbias] token or -1
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
  const int words = (p.V + 31) >> 5;

  RowTerms r;
  r.rep = p.repetition ? p.repetition[b] : 1.f;
  r.pres = p.presence ? p.presence[b] : 0.f;
  r.freq = p.frequency ? p.frequency[b] : 0.f;
  const bool counts = r.pres != 0.f || r.freq != 0.f;
  const bool past = counts || r.rep != 1.f;

  // which tokens of each vector exist (bits 0..VE-1) and are allowed
  uint32_t live[kLVecs], open[kLVecs];
  uint4 x[kLVecs];
#pragma unroll
  for (int k = 0; k < kLVecs; ++k) {
    const int v = a0 + (k * kLThreads + tid) * VE - shift;
    const int skip = max(-v, 0), left = min(max(p.V - v, 0), VE);
    live[k] = left > skip ? ((1u << left) - 1u) & ~((1u << skip) - 1u) : 0u;
    open[k] = live[k];
    if (allowed && live[k]) {
      const int at = max(v, 0) >> 5, sh = max(v, 0) & 31;
      uint64_t w = __ldg(allowed + at);
      if (sh + VE > 32 && at + 1 < words) w |= static_cast<uint64_t>(__ldg(allowed + at + 1)) << 32;
      open[k] &= static_cast<uint32_t>(w >> sh) << skip;
    }
    x[k] = make_uint4(0u, 0u, 0u, 0u);
    if (open[k]) {
      if (VEC && live[k] == (1u << VE) - 1u) {
        x[k] = *reinterpret_cast<const uint4*>(in + v);
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i)
          if ((live[k] >> i) & 1u) Raw<T>::put(x[k], i, lk::Elem<T>::to_f(in[v + i]));
      }
    }
  }

  if (past) {
    for (int i = tid; i < CH; i += kLThreads) seen[i] = 0u;
    __syncthreads();
    auto scan = [&](const int64_t* ids, int n, bool prompt) {
      for (int i = tid; i < n; i += kLThreads) {
        const int64_t id = ids[i];
        if (id >= p.V && p.status && blockIdx.x == 0) atomicOr(p.status, LK_STATUS_TOKEN_OOB);
        const int64_t at = id + shift - a0;
        if (id < 0 || id >= p.V || at < 0 || at >= CH) continue;
        if (prompt) atomicOr(&seen[at], kInPrompt);
        else atomicAdd(&seen[at], 1u);
      }
    };
    if (p.prompt_ids && r.rep != 1.f)
      scan(p.prompt_ids + b * p.prompt_ld, p.prompt_lens ? min(p.prompt_lens[b], p.prompt_max) : p.prompt_max, true);
    if (p.output_ids)
      scan(p.output_ids + b * p.output_ld, p.output_lens ? min(p.output_lens[b], p.output_max) : p.output_max, false);
    __syncthreads();
  }
  auto seen_at = [&](int v) { return past ? seen[v + shift - a0] : 0u; };

  // Biased tokens of this part: computed before anything is overwritten.
  if (p.nbias > 0) {
    for (int j = tid; j < p.nbias; j += kLThreads) {
      const int64_t id = p.bias_ids[static_cast<int64_t>(b) * p.nbias + j];
      if (id >= p.V && p.status && blockIdx.x == 0) atomicOr(p.status, LK_STATUS_TOKEN_OOB);
      bias_t[j] = id < 0 || id >= p.V ? -1 : static_cast<int>(id);
      bias_v[j] = p.bias[static_cast<int64_t>(b) * p.nbias + j];
    }
    __syncthreads();
    for (int j = tid; j < p.nbias; j += kLThreads) {
      const int v = bias_t[j];
      if (v < 0 || v + shift < a0 || v + shift >= a1) continue;
      bool first = true;
      for (int i = 0; i < j && first; ++i) first = bias_t[i] != v;
      if (!first) continue;
      float sum = 0.f;
      for (int i = j; i < p.nbias; ++i)
        if (bias_t[i] == v) sum = __fadd_rn(sum, bias_v[i]);
      bias_x[j] = __fadd_rn(process(lk::Elem<T>::to_f(in[v]), seen_at(v), r), sum);
    }
    __syncthreads();
  }

#pragma unroll
  for (int k = 0; k < kLVecs; ++k) {
    if (!live[k]) continue;
    const int at = (k * kLThreads + tid) * VE;
    const int v = a0 + at - shift;
    bool change = open[k] != live[k];
    if (past && open[k]) {
#pragma unroll
      for (int i = 0; i < VE; i += 4) {
        const uint4 s = *reinterpret_cast<const uint4*>(seen + at + i);
        if ((s.x | s.y | s.z | s.w) == 0u) continue;
        change = true;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if ((&s.x)[j]) Raw<T>::put(x[k], i + j, process(Raw<T>::get(x[k], i + j), (&s.x)[j], r));
      }
    }
    if (open[k] != live[k]) {
#pragma unroll
      for (int i = 0; i < VE; ++i)
        if (!((open[k] >> i) & 1u)) Raw<T>::put(x[k], i, -INFINITY);
    }
    if (in_place && !change) continue;
    if (VEC && live[k] == (1u << VE) - 1u) {
      *reinterpret_cast<uint4*>(out + v) = x[k];
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i)
        if ((live[k] >> i) & 1u) out[v + i] = Raw<T>::round(Raw<T>::get(x[k], i));
    }
  }

  if (p.nbias > 0) {
    __syncthreads();  // after the vectors that hold the same tokens
    for (int j = tid; j < p.nbias; j += kLThreads) {
      const int v = bias_t[j];
      if (v < 0 || v + shift < a0 || v + shift >= a1) continue;
      bool first = true;
      for (int i = 0; i < j && first; ++i) first = bias_t[i] != v;
      if (!first) continue;
      const bool ok = !allowed || ((allowed[v >> 5] >> (v & 31)) & 1u);
      out[v] = Raw<T>::round(ok ? bias_x[j] : -INFINITY);
    }
  }
}

template <typename T>
int launch_logits(const LogitsParams& p, int B, cudaStream_t s) {
  constexpr int CH = kLThreads * kLVecs * Raw<T>::kVe;
  const int parts = (p.V + 15 + CH - 1) / CH;  // room for the shift
  const size_t smem = CH * 4 + static_cast<size_t>(p.nbias) * 12;
  const bool vec =
      ((reinterpret_cast<uintptr_t>(p.logits) ^ reinterpret_cast<uintptr_t>(p.out)) & 15u) == 0 &&
      (((p.ld - p.out_ld) * static_cast<int64_t>(sizeof(T))) & 15) == 0;
  auto go = [&](auto* kernel) -> int {
    if (smem > 48 * 1024 &&
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(smem)) != cudaSuccess)
      return LK_ERR_CUDA;
    kernel<<<dim3(parts, B), kLThreads, smem, s>>>(p);
    return lk::check_launch();
  };
  return vec ? go(logits_process_kernel<T, true>) : go(logits_process_kernel<T, false>);
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
