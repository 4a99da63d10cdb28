// Log probabilities of given tokens, the entropy of each row's distribution and its k likeliest
// tokens, from logits [N, V] (fp32 or bf16, any row stride), and the gradient of the first two.
//
// With m the row's maximum, S = sum e^(x - m), W = sum e^(x - m) (x - m):
//   log p_t = (x_t - m) - log S,      H = log S - W / S,
// one pass over the logits: each thread keeps (m, S, W) of what it has read, the threads' are joined.
// Differences x - m are taken before anything is multiplied, so a token that is alone has log p
// exactly 0 and large logits lose nothing. Minus infinity, and anything far below m, adds exact
// zeros; a row of minus infinities alone has log p = -inf, H = 0 and a zero gradient. A NaN or
// plus infinity makes the row's values NaN. A token of -100 has log p = 0, any other outside the
// vocabulary NaN.
//
// The k likeliest (k <= 64, larger first, the lowest index first among equals): the largest
// value of each of 64 groups of 8 threads comes with the pass above. k groups hold a value of at
// least the k-th largest of these 64, so that value bounds the answer from below: a second
// look at the row (in L2) collects the few values at or above it, which are ranked by counting. Rows
// with more of them than fit (long runs of equal values) are searched k times instead.
//
// Gradient: dx_j = g_lp (1[j = t] - p_j) - g_H p_j (log p_j + H), one read and one write.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/types.h>

#include "common.cuh"
#include "device_setup.h"

namespace hrm {
namespace {

constexpr int kThreads = 512;
constexpr int kGroups = 64;         // of 8 threads: the largest k
constexpr int kCandidates = 1024;   // values that are ranked by counting
constexpr int64_t kIgnore = -100;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGone = -1e4f;  // e^kGone is 0; keeps 0 * (x - m) finite

template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
};

__device__ __forceinline__ float value(float v) { return v; }
__device__ __forceinline__ float value(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void store(float* p, float v) { *p = v; }
__device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ void load_vec(const float* p, float (&v)[4]) {
  const float4 w = *reinterpret_cast<const float4*>(p);
  v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
}
__device__ __forceinline__ void load_vec(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const float2 a = unpack_bf16x2(w.x), b = unpack_bf16x2(w.y), c = unpack_bf16x2(w.z), d = unpack_bf16x2(w.w);
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
}
__device__ __forceinline__ void store_vec(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                            pack_bf16x2(v[6], v[7]));
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// A (value, index) as one number that orders larger values first and, among equals, lower
// indices first; NaN above everything.
__device__ __forceinline__ unsigned long long rank_key(float v, int j) {
  if (v == 0.f) v = 0.f;  // -0 and 0 are equal
  uint32_t b = v != v ? 0x7fffffffu : __float_as_uint(v);
  b = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (unsigned long long)b << 32 | (uint32_t)~j;
}
__device__ __forceinline__ int key_index(unsigned long long k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

struct Sums {
  float m, s, w;
};
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  const float m = fmaxf(a.m, b.m);
  const float da = a.m == m ? 0.f : a.m - m, db = b.m == m ? 0.f : b.m - m;
  const float fa = fast_exp2(da * kLog2e), fb = fast_exp2(db * kLog2e);
  // W under another m: sum e^(x - m) (x - m) with x - m = (x - m_a) + (m_a - m)
  return Sums{m, a.s * fa + b.s * fb, fa * fmaf(a.s, fmaxf(da, kGone), a.w) + fb * fmaf(b.s, fmaxf(db, kGone), b.w)};
}

// Calls f(index, n values, first) for the row's elements: single ones up to a 16-byte boundary, vectors,
// single ones at the end.
template <typename T, typename One, typename Many>
__device__ __forceinline__ void for_row(const T* x, int V, One one, Many many) {
  constexpr int N = Vec<T>::N;
  const int head = min(V, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T));
  const int vecs = (V - head) / N, tail = head + vecs * N;
  if ((int)threadIdx.x < head) one((int)threadIdx.x);
  for (int i = threadIdx.x; i < vecs; i += kThreads) many(head + i * N);
  if (tail + (int)threadIdx.x < V) one(tail + (int)threadIdx.x);
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    logprobs_kernel(const T* __restrict__ logits, long ld, int V, const int64_t* __restrict__ tokens, int k,
                    float* __restrict__ logprob, float* __restrict__ entropy, float* __restrict__ stats,
                    int64_t* __restrict__ top_ids, float* __restrict__ top_lp) {
  constexpr int N = Vec<T>::N;
  const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* x = logits + row * ld;
  Sums acc{-INFINITY, 0.f, 0.f};
  float ref = 0.f;  // acc.m where there is one
  float best = -INFINITY;
  int best_j = 0x7fffffff;

  const auto take = [&](const float* v, int n, int j0) {
    float top = v[0];
#pragma unroll
    for (int i = 1; i < n; ++i) top = max_nan(top, v[i]);
    if (!(top <= best) || best_j == 0x7fffffff) {  // rare after the first few
      if (best == best) {
#pragma unroll
        for (int i = n - 1; i >= 0; --i)
          if (v[i] == top || v[i] != v[i]) best_j = j0 + i;
        best = top;
      }
      if (top > acc.m) {
        const float d = acc.m - top, f = fast_exp2(d * kLog2e);
        acc.w = f * fmaf(acc.s, fmaxf(d, kGone), acc.w);
        acc.s *= f;
        acc.m = ref = top;
      }
    }
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float d = v[i] - ref, e = fast_exp2(d * kLog2e);
      acc.s += e;
      acc.w = fmaf(e, fmaxf(d, kGone), acc.w);
    }
  };
  for_row(
      x, V,
      [&](int j) {
        const float v[1] = {value(x[j])};
        take(v, 1, j);
      },
      [&](int j) {
        float v[N];
        load_vec(x + j, v);
        take(v, N, j);
      });

  unsigned long long key = best_j == 0x7fffffff ? 0 : rank_key(best, best_j);
  __shared__ Sums s_sum[kThreads / 32];
  __shared__ unsigned long long s_group[kGroups], s_best[kGroups], s_cand[kCandidates];
  __shared__ int s_count;
  __shared__ unsigned long long s_bound;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    acc = join(acc, Sums{__shfl_xor_sync(~0u, acc.m, off), __shfl_xor_sync(~0u, acc.s, off), __shfl_xor_sync(~0u, acc.w, off)});
    if (off < 8) key = max(key, __shfl_xor_sync(~0u, key, off));
  }
  if (lane == 0) s_sum[warp] = acc;
  if ((lane & 7) == 0) s_group[tid >> 3] = key;
  if (tid == 0) s_count = 0;
  __syncthreads();
  acc = s_sum[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) acc = join(acc, s_sum[w]);
  const float log_s = logf(acc.s);

  // the groups' values in order: thread i < 64 ranks group i
  if (tid < kGroups) {
    const unsigned long long mine = s_group[tid];
    int r = 0;
    for (int i = 0; i < kGroups; ++i) r += s_group[i] > mine || (s_group[i] == mine && i < tid);
    if (r < kGroups) s_best[r] = mine;
    if (r == k - 1) s_bound = mine;
  }
  __syncthreads();
  const float top = key_value(s_best[0]);
  const bool empty = top == -INFINITY;
  const auto logp = [&](float v) {  // of a logit of this row
    return empty ? -INFINITY : (v - acc.m) - log_s;
  };
  if (tid == 0) {
    const int64_t t = tokens[row];
    logprob[row] = t == kIgnore ? 0.f : t < 0 || t >= V ? NAN : logp(value(x[t]));
    const float h = empty ? 0.f : log_s - acc.w / acc.s;
    entropy[row] = h;
    if (stats != nullptr) {
      stats[row * 3] = empty ? 0.f : acc.m;
      stats[row * 3 + 1] = empty ? INFINITY : log_s;  // no probability, so no gradient
      stats[row * 3 + 2] = h;
    }
  }
  if (k == 0) return;
  int64_t* ids = top_ids + (long)row * k;
  float* lps = top_lp + (long)row * k;
  if (k == 1) {
    if (tid == 0) {
      ids[0] = key_index(s_best[0]);
      lps[0] = logp(top);
    }
    return;
  }
  const unsigned long long bound = s_bound;
  const auto offer = [&](float v, int j) {
    const unsigned long long c = rank_key(v, j);
    if (c >= bound) {
      const int n = atomicAdd(&s_count, 1);
      if (n < kCandidates) s_cand[n] = c;
    }
  };
  const float bound_v = key_value(bound);
  for_row(
      x, V, [&](int j) { offer(value(x[j]), j); },
      [&](int j) {
        float v[N];
        load_vec(x + j, v);
        float m = v[0];
#pragma unroll
        for (int i = 1; i < N; ++i) m = max_nan(m, v[i]);
        if (!(m < bound_v)) {
#pragma unroll
          for (int i = 0; i < N; ++i) offer(v[i], j + i);
        }
      });
  __syncthreads();
  const int n = s_count;
  if (n <= kCandidates) {
    for (int c = tid; c < n; c += kThreads) {
      const unsigned long long mine = s_cand[c];
      int r = 0;
      for (int i = 0; i < n; ++i) r += s_cand[i] > mine;
      if (r < k) {
        ids[r] = key_index(mine);
        lps[r] = logp(key_value(mine));
      }
    }
    return;
  }
  // too many at the bound: the largest below the last one found, k times
  unsigned long long last = ~0ull;
  for (int r = 0; r < k; ++r) {
    unsigned long long mine = 0;
    for (int j = tid; j < V; j += kThreads) {
      const unsigned long long c = rank_key(value(x[j]), j);
      if (c < last && c > mine) mine = c;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mine = max(mine, __shfl_xor_sync(~0u, mine, off));
    __syncthreads();
    if (lane == 0) s_best[warp] = mine;
    __syncthreads();
    last = s_best[0];
    for (int w = 1; w < kThreads / 32; ++w) last = max(last, s_best[w]);
    if (tid == 0) {
      ids[r] = key_index(last);
      lps[r] = logp(key_value(last));
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    logprobs_bwd_kernel(const T* __restrict__ logits, long ld, int V, const int64_t* __restrict__ tokens,
                        const float* __restrict__ stats, const float* __restrict__ g_lp,
                        const float* __restrict__ g_h, T* __restrict__ grad, long ldg) {
  constexpr int N = Vec<T>::N;
  const int row = blockIdx.x;
  const T* x = logits + row * ld;
  T* out = grad + row * ldg;
  const int64_t t = tokens[row];
  const float m = stats[row * 3], log_s = stats[row * 3 + 1], h = stats[row * 3 + 2];
  float glp = g_lp != nullptr && t != kIgnore ? g_lp[row] : 0.f;
  if (t != kIgnore && (t < 0 || t >= V)) glp = NAN;
  if (log_s == INFINITY) glp = 0.f;  // a row of nothing
  const float gh = g_h != nullptr ? g_h[row] : 0.f;
  const float a = -(glp + gh * h);
  // dx = p (a - g_H log p) (+ g_lp at the token)
  const auto one = [&](float v, int j) {
    const float d = (v - m) - log_s;
    const float p = fast_exp2(d * kLog2e);
    float r = p * fmaf(-gh, fmaxf(d, kGone), a);
    if (p == 0.f) r = 0.f;
    return j == t ? r + glp : r;
  };
  if (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(out)) & 15) != 0) {
    for (int j = threadIdx.x; j < V; j += kThreads) store(out + j, one(value(x[j]), j));
    return;
  }
  for_row(
      x, V, [&](int j) { store(out + j, one(value(x[j]), j)); },
      [&](int j) {
        float v[N];
        load_vec(x + j, v);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = one(v[i], j + i);
        store_vec(out + j, v);
      });
}

void check_logits(const at::Tensor& logits, const at::Tensor& tokens) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.numel() == 0 || logits.stride(1) == 1) &&
                  (logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16),
              "token_logprobs: logits CUDA [rows, vocabulary], fp32 or bf16, rows contiguous");
  TORCH_CHECK(logits.size(1) >= 1 && logits.size(1) < (1LL << 31) - 16, "token_logprobs: vocabulary size");
  TORCH_CHECK(logits.size(0) < (1LL << 31), "token_logprobs: too many rows");
  TORCH_CHECK(tokens.device() == logits.device() && tokens.scalar_type() == at::kLong && tokens.is_contiguous() &&
                  tokens.numel() == logits.size(0),
              "token_logprobs: int64 tokens, one for each row");
}

}  // namespace

int64_t logprobs_max_top() { return kGroups; }

// logprob, entropy [N] fp32; stats [N, 3] fp32 or none (for the gradient); top_ids int64 and
// top_lp fp32 [N, k].
void token_logprobs_fwd(const at::Tensor& logits, const at::Tensor& tokens, int64_t k, const at::Tensor& logprob,
                        const at::Tensor& entropy, const c10::optional<at::Tensor>& stats, const at::Tensor& top_ids,
                        const at::Tensor& top_lp) {
  check_logits(logits, tokens);
  const int64_t N = logits.size(0), V = logits.size(1);
  TORCH_CHECK(k >= 0 && k <= kGroups && k <= V, "token_logprobs: top_k is 0 to ", kGroups, " and at most the vocabulary");
  for (const at::Tensor* o : {&logprob, &entropy, &top_lp})
    TORCH_CHECK(o->device() == logits.device() && o->scalar_type() == at::kFloat && o->is_contiguous(), "token_logprobs: outputs");
  TORCH_CHECK(logprob.numel() == N && entropy.numel() == N && top_lp.numel() == N * k && top_ids.numel() == N * k &&
                  top_ids.scalar_type() == at::kLong && top_ids.is_contiguous() && top_ids.device() == logits.device() &&
                  (!stats || (stats->numel() == 3 * N && stats->scalar_type() == at::kFloat && stats->is_contiguous() &&
                              stats->device() == logits.device())),
              "token_logprobs: outputs");
  if (N == 0) return;
  c10::cuda::CUDAGuard guard(logits.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  float* st = stats ? stats->data_ptr<float>() : nullptr;
  const auto run = [&](auto* x) {
    using T = std::remove_pointer_t<decltype(x)>;
    logprobs_kernel<T><<<(unsigned)N, kThreads, 0, stream>>>(x, logits.stride(0), (int)V, tokens.data_ptr<int64_t>(), (int)k,
                                                             logprob.data_ptr<float>(), entropy.data_ptr<float>(), st,
                                                             top_ids.data_ptr<int64_t>(), top_lp.data_ptr<float>());
  };
  if (logits.scalar_type() == at::kFloat)
    run(logits.data_ptr<float>());
  else
    run(reinterpret_cast<__nv_bfloat16*>(logits.data_ptr()));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// grad [N, V] like logits from the gradients of logprob and entropy ([N] fp32, either may be none).
void token_logprobs_bwd(const at::Tensor& logits, const at::Tensor& tokens, const at::Tensor& stats,
                        const c10::optional<at::Tensor>& g_lp, const c10::optional<at::Tensor>& g_h,
                        const at::Tensor& grad) {
  check_logits(logits, tokens);
  const int64_t N = logits.size(0), V = logits.size(1);
  for (const auto* g : {&g_lp, &g_h})
    TORCH_CHECK(!*g || ((*g)->device() == logits.device() && (*g)->scalar_type() == at::kFloat && (*g)->is_contiguous() &&
                        (*g)->numel() == N),
                "token_logprobs: gradients fp32, one for each row");
  TORCH_CHECK(stats.numel() == 3 * N && stats.scalar_type() == at::kFloat && stats.is_contiguous() &&
                  stats.device() == logits.device(),
              "token_logprobs: statistics of the forward pass");
  TORCH_CHECK(grad.sizes() == logits.sizes() && grad.scalar_type() == logits.scalar_type() &&
                  grad.device() == logits.device() && (grad.numel() == 0 || grad.stride(1) == 1),
              "token_logprobs: gradient like the logits");
  if (N == 0) return;
  c10::cuda::CUDAGuard guard(logits.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const float* a = g_lp ? g_lp->data_ptr<float>() : nullptr;
  const float* b = g_h ? g_h->data_ptr<float>() : nullptr;
  const auto run = [&](auto* x, auto* g) {
    using T = std::remove_pointer_t<decltype(x)>;
    logprobs_bwd_kernel<T><<<(unsigned)N, kThreads, 0, stream>>>(x, logits.stride(0), (int)V, tokens.data_ptr<int64_t>(),
                                                                 stats.data_ptr<float>(), a, b, g, grad.stride(0));
  };
  if (logits.scalar_type() == at::kFloat)
    run(logits.data_ptr<float>(), grad.data_ptr<float>());
  else
    run(reinterpret_cast<__nv_bfloat16*>(logits.data_ptr()), reinterpret_cast<__nv_bfloat16*>(grad.data_ptr()));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace hrm
