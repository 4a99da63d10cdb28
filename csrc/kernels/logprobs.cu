// Log probabilities of given tokens, the entropy of each row's distribution and its k likeliest
// tokens, from logits [N, V] (fp32 or bf16, any row stride), and the gradient of the first two.
//
// With m the row's maximum, S = sum e^(x - m), W = sum e^(x - m) (x - m):
//   log p_t = (x_t - m) - log S,      H = log S - W / S,
// one pass over the logits: each thread keeps (m, S, W) of what it has read, the threads' are joined.
// Differences x - m are taken before anything is multiplied, so a token that is alone has log p
// exactly 0 and large logits lose nothing. Minus infinity, and anything far below m, adds exact
// zeros; a row of minus infinities alone has log p = -inf, H = 0 and a zero gradient. A NaN or
// plus infinity makes the row's values NaN. A token of -100 has log p = 0 and no gradient of it, any other outside
// the vocabulary NaN for both; the row's entropy and its gradient do not depend on the token.
//
// The k likeliest (k <= 64, larger first, the lowest index first among equals): the threads are 64
// groups, and k groups hold a value of at least the k-th largest of the groups' largest values, so
// that value bounds the answer from below. The pass has noted the largest value of every 64 bytes:
// those that reach the bound, few more than k, are read again, and their values at or above it
// are ranked by counting. Rows with more such values than fit are searched k times instead: long runs of equal
// values, and, because the bound is then minus infinity, rows above 12288 bf16 or 6144 fp32 logits in which a mask
// leaves fewer than k of the groups a finite value (33 rows of 32768 bf16 with 30 tokens left, twenty
// alternatives: 123 us, 6.6 unmasked).
//
// Gradient: dx_j = g_lp (1[j = t] - p_j) - g_H p_j (log p_j + H), one read and one write.
//
// Measured (one B200, copy rate 6.54 TB/s, L2 cold): 8192 rows of 32768 bf16 90 to 92 us forward (91 to 89 % of the copy
// rate; 104 us with the likeliest token, 107 with five, 116 with twenty) and 175 us backward (94 %); 4096
// rows of 32003 fp32 83 to 88 us (97 to 91 %; 90 to 95 us with the likeliest). Long rows are bound by memory, bf16
// ones nearly as much by instructions (issue slots 80 % used: an element costs an exponential, a
// difference, a product, two sums and a maximum); short rows by what each row's end costs (20000 rows of
// 4096 bf16 41 us, 61 %), a few rows by latency (33 rows of 32768 bf16 with five alternatives 6.3 us). Some hundreds of long
// rows leave SMs short of loads (300 rows of 32768 bf16 11.5 us for 3 us of bytes, 600 13), and a gradient of few long
// rows has one CTA a row (33 rows of 150000 fp32 57 us for 6).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/types.h>

#include "common.cuh"
#include "device_setup.h"
#include "launch_early.h"

namespace hrm {
namespace {

constexpr int kGroups = 64;         // groups of threads: the largest k
constexpr int kCandidates = 512;    // values that are ranked by counting
constexpr int kBatch = 4;           // 16-byte loads of a thread that are in flight together
constexpr int kBatchBwd = 2;        // the same of the backward pass, which stores as many
constexpr int kNoted = 16384;       // batches of a row whose largest value is kept in shared memory
constexpr int kAgain = 384;         // of them, those that are read again
constexpr int64_t kIgnore = -100;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGone = -1e4f;  // e^kGone is 0; keeps 0 * (x - m) finite

__device__ __forceinline__ float value(float v) { return v; }
__device__ __forceinline__ float value(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void store(float* p, float v) { *p = v; }
__device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 16 bytes of logits
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static constexpr uint32_t kNothing = 0xff800000u;  // minus infinity in every place
  static __device__ __forceinline__ void unpack(const uint4& w, float (&v)[4]) {
    v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y); v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ float last_max(uint32_t a) { return __uint_as_float(a); }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr uint32_t kNothing = 0xff80ff80u;
  static __device__ __forceinline__ void unpack(const uint4& w, float (&v)[8]) {
    const float2 a = unpack_bf16x2(w.x), b = unpack_bf16x2(w.y), c = unpack_bf16x2(w.z), d = unpack_bf16x2(w.w);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
    return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float last_max(uint32_t a) {
    const float2 v = unpack_bf16x2(a);
    return max_nan(v.x, v.y);
  }
};
// the largest of a vector's values, NaN if one is
template <typename T>
__device__ __forceinline__ uint32_t vec_max(const uint4& w) {
  return Vec<T>::max2(Vec<T>::max2(w.x, w.y), Vec<T>::max2(w.z, w.w));
}

// A value as a number that orders like it; NaN above everything, 0 below.
__device__ __forceinline__ uint32_t order_of(float v) {
  if (v == 0.f) v = 0.f;  // -0 and 0 are equal
  const uint32_t b = v != v ? 0x7fffffffu : __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t b) { return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b); }
constexpr uint32_t kMasked = 0x007fffffu;  // order_of(-infinity)
// A (value, index) as one number: larger values first, among equals lower indices first.
__device__ __forceinline__ unsigned long long rank_key(float v, int j) {
  return (unsigned long long)order_of(v) << 32 | (uint32_t)~j;
}
__device__ __forceinline__ int key_index(unsigned long long k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float key_value(unsigned long long k) { return value_of((uint32_t)(k >> 32)); }

struct Sums {
  float m, s, w;
  // to another m, not below this one: with x - m' = (x - m) + (m - m')
  __device__ __forceinline__ void move(float to) {
    const float d = m == to ? 0.f : m - to, f = fast_exp2(d * kLog2e);
    w = f * fmaf(s, fmaxf(d, kGone), w);
    s *= f;
    m = to;
  }
};
// the lanes' sums in every lane
__device__ __forceinline__ Sums warp_join(Sums a) {
  float m = a.m;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, off));
  a.move(m);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    a.s += __shfl_xor_sync(~0u, a.s, off);
    a.w += __shfl_xor_sync(~0u, a.w, off);
  }
  return a;
}

// A row: single elements up to a 16-byte boundary, vectors, single ones at the end.
template <typename T>
struct Row {
  int head, vecs, tail;
  __device__ __forceinline__ Row(const T* x, int V) {
    head = min(V, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T));
    vecs = (V - head) / Vec<T>::N;
    tail = head + vecs * Vec<T>::N;
  }
  // loads the thread's vectors i, i + THREADS, ... of those from `base` on, i = base + thread; STREAM marks
  // them for early eviction (forward, fp32 rows: 100 -> 88 us; the backward pass is slower with it, 177 -> 190)
  template <int THREADS, int BATCH, bool STREAM>
  __device__ __forceinline__ void load(const T* x, int base, int i, uint4 (&raw)[BATCH]) const {
    const uint4* p = reinterpret_cast<const uint4*>(x + head) + i;
    const auto get = [](const uint4* q) { return STREAM ? __ldcs(q) : *q; };
    if (base + THREADS * BATCH <= vecs) {  // the CTA's batches are whole: nothing to compare or to fill
#pragma unroll
      for (int u = 0; u < BATCH; ++u) raw[u] = get(p + u * THREADS);
    } else {
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const uint32_t z = Vec<T>::kNothing;
        raw[u] = i + u * THREADS < vecs ? get(p + u * THREADS) : make_uint4(z, z, z, z);
      }
    }
  }
};

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS)
    logprobs_kernel(const T* __restrict__ logits, long ld, int V, const int64_t* __restrict__ tokens, int k,
                    float* __restrict__ logprob, float* __restrict__ entropy, float* __restrict__ stats,
                    int64_t* __restrict__ top_ids, float* __restrict__ top_lp) {
  constexpr int N = Vec<T>::N, WARPS = THREADS / 32;
  __shared__ Sums s_sum[WARPS];
  __shared__ __align__(16) uint32_t s_group[kGroups];
  __shared__ float s_m, s_log_s;
  __shared__ uint16_t s_again[kAgain];
  __shared__ int s_count, s_again_count;
  __shared__ uint32_t s_bound;
  // for k > 0: largest values of the batches, rounded up, [min(batches of the row, kNoted)]; when those have
  // been looked through, the candidates, [kCandidates]. Shared memory is kept small because what is left of
  // it as L1 bounds the loads in flight.
  extern __shared__ __align__(8) uint8_t s_more[];
  __nv_bfloat16* s_noted = reinterpret_cast<__nv_bfloat16*>(s_more);
  unsigned long long* s_cand = reinterpret_cast<unsigned long long*>(s_more);
  const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* x = logits + row * ld;
  const Row<T> r(x, V);

  int64_t t = kIgnore;  // thread 0 has the row's token and its logit
  float xt = 0.f;
  if (tid == 0) {
    t = tokens[row];
    if (t != kIgnore) xt = t < 0 || t >= V ? NAN : value(x[t]);
  }
  Sums acc{-INFINITY, 0.f, 0.f};
  float ref = 0.f;  // acc.m once a finite value was seen
  if (tid < kGroups) s_group[tid] = 0;
  float best = -INFINITY;  // the thread's largest value, NaN above all
  const auto raise = [&](float top) {
    if (!(top <= best)) {
      if (best == best) best = top;
      if (top > acc.m) {
        acc.move(top);
        ref = top;
      }
    }
  };
  const auto add = [&](float v, float& s, float& w) {
    const float d = v - ref, e = fast_exp2(d * kLog2e);
    s += e;
    w = fmaf(e, fmaxf(d, kGone), w);
  };
  if (tid < r.head) {
    const float v = value(x[tid]);
    raise(v);
    add(v, acc.s, acc.w);
  }
  for (int base = 0; base < r.vecs; base += THREADS * kBatch) {
    uint4 raw[kBatch];
    r.template load<THREADS, kBatch, true>(x, base, base + tid, raw);
    uint32_t most = vec_max<T>(raw[0]);
#pragma unroll
    for (int u = 1; u < kBatch; ++u) most = Vec<T>::max2(most, vec_max<T>(raw[u]));
    const float top = Vec<T>::last_max(most);
    raise(top);
    if (k > 0) {
      const int b = base / kBatch + tid;
      if (b < kNoted) s_noted[b] = __float2bfloat16_ru(top);
    }
    float s2 = 0.f, w2 = 0.f;  // every second element: two chains of sums
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      float v[N];
      Vec<T>::unpack(raw[u], v);
#pragma unroll
      for (int n = 0; n < N; n += 2) {
        add(v[n], acc.s, acc.w);
        add(v[n + 1], s2, w2);
      }
    }
    acc.s += s2;
    acc.w += w2;
  }
  if (r.tail + tid < V) {
    const float v = value(x[r.tail + tid]);
    raise(v);
    add(v, acc.s, acc.w);
  }

  acc = warp_join(acc);
  if (lane == 0) s_sum[warp] = acc;
  if (k > 0) {
    __syncthreads();  // the groups are cleared
    const bool any = tid < r.head || tid < r.vecs || r.tail + tid < V;
    if (any) atomicMax(&s_group[tid % kGroups], order_of(best));
  }
  __syncthreads();
  if (warp == 0) {
    acc = warp_join(lane < WARPS ? s_sum[lane] : Sums{-INFINITY, 0.f, 0.f});
    if (lane == 0) {
      // nothing but minus infinities: m and S such that every logit's log p is -inf
      const bool empty = acc.m == -INFINITY && acc.s == 0.f;
      const float m = empty ? 0.f : acc.m, log_s = empty ? INFINITY : logf(acc.s);
      logprob[row] = t == kIgnore ? 0.f : (xt - m) - log_s;
      const float h = empty ? 0.f : log_s - acc.w / acc.s;
      entropy[row] = h;
      if (stats != nullptr) {
        stats[(long)row * 3] = m;
        stats[(long)row * 3 + 1] = log_s;
        stats[(long)row * 3 + 2] = h;
      }
      s_m = m;
      s_log_s = log_s;
      s_count = s_again_count = 0;
    }
  }
  if (k == 0) return;
  // the bound: the k-th largest of the groups' values, by the last two warps
  if (tid >= THREADS - kGroups) {
    const int g = tid - (THREADS - kGroups);
    const uint32_t mine = s_group[g];
    int rank = 0;
#pragma unroll
    for (int i = 0; i < kGroups; i += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(&s_group[i]);
      rank += (o.x > mine || (o.x == mine && i < g)) + (o.y > mine || (o.y == mine && i + 1 < g)) +
              (o.z > mine || (o.z == mine && i + 2 < g)) + (o.w > mine || (o.w == mine && i + 3 < g));
    }
    if (rank == k - 1) s_bound = mine;
  }
  __syncthreads();
  const float m = s_m, log_s = s_log_s;
  const uint32_t bound = s_bound;
  int64_t* ids = top_ids + (long)row * k;
  float* lps = top_lp + (long)row * k;
  const auto write = [&](int at, unsigned long long key) {
    ids[at] = key_index(key);
    lps[at] = (key_value(key) - m) - log_s;
  };
  // Minus infinities, of which a mask leaves many, are of use only where fewer than k values are
  // larger, and then the first k places hold enough of them.
  const auto offer = [&](float v, int j) {
    const uint32_t o = order_of(v);
    if (o >= bound && (o != kMasked || j < k)) {
      const int n = atomicAdd(&s_count, 1);
      if (n < kCandidates) s_cand[n] = rank_key(v, j);
    }
  };
  const float bound_v = bound == 0 ? -INFINITY : value_of(bound);
  const auto offer_vec = [&](int i) {
    const uint4 raw = reinterpret_cast<const uint4*>(x + r.head)[i];
    if (Vec<T>::last_max(vec_max<T>(raw)) < bound_v) return;
    float v[N];
    Vec<T>::unpack(raw, v);
#pragma unroll
    for (int n = 0; n < N; ++n) offer(v[n], r.head + i * N + n);
  };
  // the batches to read again, first as a list, so that all of them are on their way together
  if (!(best < bound_v)) {
    for (int i = tid, b = tid; i < r.vecs && b < kNoted; i += THREADS * kBatch, b += THREADS) {
      if (!(__bfloat162float(s_noted[b]) < bound_v)) {
        const int n = atomicAdd(&s_again_count, 1);
        if (n < kAgain) s_again[n] = (uint16_t)b;
      }
    }
  }
  __syncthreads();
  const int again = s_again_count;
  if (again <= kAgain) {
    for (int e = tid; e < again * kBatch; e += THREADS) {
      const int b = s_again[e / kBatch], i = (b / THREADS * kBatch + e % kBatch) * THREADS + b % THREADS;
      if (i < r.vecs) offer_vec(i);
    }
    for (int i = tid + kNoted * kBatch; i < r.vecs; i += THREADS) offer_vec(i);  // batches that were not noted
  }
  if (tid < r.head) offer(value(x[tid]), tid);
  if (r.tail + tid < V) offer(value(x[r.tail + tid]), r.tail + tid);
  __syncthreads();
  const int n = s_count;
  if (n <= kCandidates && again <= kAgain) {
    for (int c = tid; c < n; c += THREADS) {
      const unsigned long long mine = s_cand[c];
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += s_cand[i] > mine;
      if (rank < k) write(rank, mine);
    }
    return;
  }
  // too many at the bound: the largest, then the largest below the last one found; the key of a NaN at id 0 is
  // all ones, so nothing is below a start from there
  __syncthreads();
  unsigned long long last = 0;
  for (int at = 0; at < k; ++at) {
    unsigned long long mine = 0;
    for (int j = tid; j < V; j += THREADS) {
      const unsigned long long c = rank_key(value(x[j]), j);
      if ((at == 0 || c < last) && c > mine) mine = c;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mine = max(mine, __shfl_xor_sync(~0u, mine, off));
    __syncthreads();
    if (lane == 0) s_cand[warp] = mine;
    __syncthreads();
    last = s_cand[0];
    for (int w = 1; w < WARPS; ++w) last = max(last, s_cand[w]);
    if (tid == 0) write(at, last);
  }
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS)
    logprobs_bwd_kernel(const T* __restrict__ logits, long ld, int V, const int64_t* __restrict__ tokens,
                        const float* __restrict__ stats, const float* __restrict__ g_lp,
                        const float* __restrict__ g_h, T* __restrict__ grad, long ldg) {
  constexpr int N = Vec<T>::N;
  const int row = blockIdx.x, tid = threadIdx.x;
  const T* x = logits + row * ld;
  T* out = grad + row * ldg;
  const int64_t t = tokens[row];
  const float m = stats[(long)row * 3], log_s = stats[(long)row * 3 + 1], h = stats[(long)row * 3 + 2];
  float glp = g_lp != nullptr && t != kIgnore ? g_lp[row] : 0.f;
  if (g_lp != nullptr && t != kIgnore && (t < 0 || t >= V)) glp = NAN;  // the entropy does not depend on the token
  if (log_s == INFINITY) glp = 0.f;  // a row of nothing
  const float gh = g_h != nullptr ? g_h[row] : 0.f;
  const float a = -(glp + gh * h);
  // dx = p (a - g_H log p), and g_lp more at the token
  const auto slope = [&](float v) {
    const float d = (v - m) - log_s;
    return fast_exp2(d * kLog2e) * fmaf(-gh, fmaxf(d, kGone), a);
  };
  const auto single = [&](int j) { store(out + j, slope(value(x[j])) + (j == t ? glp : 0.f)); };
  if (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(out)) & 15) != 0) {
    for (int j = tid; j < V; j += THREADS) single(j);
    return;
  }
  const Row<T> r(x, V);
  if (tid < r.head) single(tid);
  for (int base = 0; base < r.vecs; base += THREADS * kBatchBwd) {
    const int i = base + tid;
    uint4 raw[kBatchBwd];
    r.template load<THREADS, kBatchBwd, false>(x, base, i, raw);
#pragma unroll
    for (int u = 0; u < kBatchBwd; ++u) {
      const int j = r.head + (i + u * THREADS) * N;
      float v[N];
      Vec<T>::unpack(raw[u], v);
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] = slope(v[n]);
      if (t >= j && t < j + N) {
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] += j + n == t ? glp : 0.f;
      }
      if (i + u * THREADS < r.vecs) *reinterpret_cast<uint4*>(out + j) = Vec<T>::pack(v);
    }
  }
  if (r.tail + tid < V) single(r.tail + tid);
}

// Threads for a row, forward. Few rows: many threads each (33 rows of 32768 bf16: 1024 threads).
// Many rows: small CTAs, of which an SM holds many, so that one's loads run under another's
// reductions (8192 such rows: 128 threads 92 us, 256 97, 512 140); for rows under 8 KB, which 128
// threads would not fill, 64 (50000 rows of 2000 bf16: 66 us, 99 with 128; even at 8 KB).
int row_threads(int64_t N, int64_t row_bytes) {
  return N <= 2 * device_sm_count() ? 1024 : row_bytes < 8192 ? 64 : 128;
}

void check_logits(const at::Tensor& logits, const at::Tensor& tokens) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.numel() == 0 || logits.size(1) == 1 || logits.stride(1) == 1) &&
                  (logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16),
              "token_logprobs: logits CUDA [rows, vocabulary], fp32 or bf16, rows contiguous");
  TORCH_CHECK(logits.size(1) >= 1 && logits.size(1) < (1LL << 31) - 16, "token_logprobs: vocabulary size");
  TORCH_CHECK(logits.size(0) < (1LL << 31), "token_logprobs: too many rows");
  TORCH_CHECK(tokens.device() == logits.device() && tokens.scalar_type() == at::kLong && tokens.is_contiguous() &&
                  tokens.numel() == logits.size(0),
              "token_logprobs: int64 tokens, one for each row");
}

}  // namespace

// Returns logprob and entropy [N] fp32; for k > 0 top_ids int64 and top_lp fp32 [N, k]; with `keep` last the
// statistics [N, 3] fp32 that the gradient needs.
std::vector<at::Tensor> token_logprobs_fwd(const at::Tensor& logits, const at::Tensor& tokens, int64_t k, bool keep) {
  check_logits(logits, tokens);
  const int64_t N = logits.size(0), V = logits.size(1);
  TORCH_CHECK(k >= 0 && k <= kGroups && k <= V, "token_logprobs: top_k is 0 to ", kGroups, " and at most the vocabulary");
  c10::cuda::CUDAGuard guard(logits.device());
  Outputs make(logits.options());
  make.plan({N}, at::kFloat).plan({N}, at::kFloat).plan({N, k}, at::kLong).plan({N, k}, at::kFloat);
  std::vector<at::Tensor> out;
  out.reserve(5);
  out.push_back(make.next({N}, at::kFloat));
  out.push_back(make.next({N}, at::kFloat));
  if (k > 0) {
    out.push_back(make.next({N, k}, at::kLong));
    out.push_back(make.next({N, k}, at::kFloat));
  }
  if (keep) out.push_back(at::empty({N, 3}, logits.options().dtype(at::kFloat)));
  if (N == 0) return out;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  float* st = keep ? out.back().data_ptr<float>() : nullptr;
  int64_t* ids = k > 0 ? out[2].data_ptr<int64_t>() : nullptr;
  float* lps = k > 0 ? out[3].data_ptr<float>() : nullptr;
  const auto run = [&](auto* x) {
    using T = std::remove_pointer_t<decltype(x)>;
    const int threads = row_threads(N, V * (int64_t)sizeof(T));
    auto* kernel = threads == 1024 ? logprobs_kernel<T, 1024> : threads == 128 ? logprobs_kernel<T, 128> : logprobs_kernel<T, 64>;
    // every thread's last batch may be short
    const int64_t batches = V * (int64_t)sizeof(T) / (16 * kBatch) + 2 * threads;
    const int more = k > 0 ? (int)std::max<int64_t>(std::min<int64_t>(batches, kNoted) * 2, kCandidates * 8) : 0;
    kernel<<<(unsigned)N, threads, more, stream>>>(x, logits.stride(0), (int)V, tokens.data_ptr<int64_t>(), (int)k,
                                                            out[0].data_ptr<float>(), out[1].data_ptr<float>(), st, ids, lps);
  };
  if (logits.scalar_type() == at::kFloat)
    run(logits.data_ptr<float>());
  else
    run(reinterpret_cast<__nv_bfloat16*>(logits.data_ptr()));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
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
                  grad.device() == logits.device() && (grad.numel() == 0 || grad.size(1) == 1 || grad.stride(1) == 1),
              "token_logprobs: gradient like the logits");
  if (N == 0) return;
  c10::cuda::CUDAGuard guard(logits.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const float* a = g_lp ? g_lp->data_ptr<float>() : nullptr;
  const float* b = g_h ? g_h->data_ptr<float>() : nullptr;
  const auto run = [&](auto* x, auto* g) {
    using T = std::remove_pointer_t<decltype(x)>;
    // nothing is reduced here: 256 threads for rows of 64 KB and more (4096 rows of 32003 fp32: 179 us, 190 with
    // 128), 128 for shorter ones (20000 of 4096 bf16: 64 us, 88 with 256)
    const bool wide = V * (int64_t)sizeof(T) >= 64 * 1024;
    auto* kernel = wide ? logprobs_bwd_kernel<T, 256> : logprobs_bwd_kernel<T, 128>;
    kernel<<<(unsigned)N, wide ? 256 : 128, 0, stream>>>(x, logits.stride(0), (int)V, tokens.data_ptr<int64_t>(),
                                                         stats.data_ptr<float>(), a, b, g, grad.stride(0));
  };
  if (logits.scalar_type() == at::kFloat)
    run(logits.data_ptr<float>(), grad.data_ptr<float>());
  else
    run(reinterpret_cast<__nv_bfloat16*>(logits.data_ptr()), reinterpret_cast<__nv_bfloat16*>(grad.data_ptr()));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace hrm
