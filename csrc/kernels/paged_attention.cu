// Attention of new tokens over a paged KV cache held in 8 bits (paged_kv8.cu), one scale for each
// block of tokens and head.
//
// Query row (token j of request i, query head hq), kv head h = hq / G, at position
// p = L_i - n_i + j, sees keys k <= p (causal) or all L_i keys:
//   a_k = (q . c_k) * Sk[b(k), h] / sqrt(128),   o = sum_k softmax(a)_k * c'_k * Sv[b(k), h],
//   y = sigmoid(gate) * o   (when a gate is given).
//
// Work split. A unit is 128 keys of one (request, kv head); the units of all pairs, laid end to
// end with a fixed cost before each pair, are cut into equal ranges, one for each CTA (the prefix
// sums come with the step, see paged_tables.cu). A long sequence is thus spread over many CTAs
// and short ones share a CTA, whatever the mix of lengths. A pair inside one CTA is finished
// there; the parts of a pair that spans CTAs go to a workspace and a second kernel joins them in
// order (no atomics: the same inputs give the same bits).
//
// In a CTA each of 8 warps takes 16 keys of a unit and keeps its own running maximum, sum and
// output for up to 8 * NT query rows (G query heads times the request's new tokens); the
// warps are merged through shared memory once per pair. Each warp copies its own codes ahead into
// its own ring of shared memory (cp.async, 4 KB a stage), across the ends of pairs, so that it
// waits for no other warp and a pair's first loads run under the work before it.
// A warp's 16 keys are
//   S^T [16 keys x 8 rows] = C [16 x 128] Q^T,   O^T [128 dims x 8 rows] += C'^T [128 x 16] P^T
// in mma.m16n8k16 with the keys as the M side: 8 rows, the smallest N, waste the least of a
// matrix instruction on the one or few rows a decode step has. The kernel is bound by reading the
// codes (256 bytes a key and head for 4 * 128 * rows flops), so warp-level matrix instructions
// on codes converted in registers are far from their limit:
//   * the k index of S = C Q^T may be permuted as one likes if Q is permuted alike, so a lane
//     owns 32 dims of two keys as four 16-byte words, and a 32-bit word of codes is the lane's
//     part of one k step;
//   * the m index of O^T likewise: a lane owns 16 dims of four keys, pairs of keys are
//     interleaved by byte permutes before they are widened;
//   * P^T is S^T transposed 8x8 by movmatrix.
// Codes are exact in f16 (int8: 1024 + 128 + c by a byte permute, minus 1152; e4m3: one cvt).
// Queries are scaled by a power of two to a row maximum in [1, 2) before they are rounded to f16:
// a bf16 value keeps all its bits unless it is 2^-14 of the row's largest. P is rounded to f16 (11
// bits, against 8 of bf16), sums stay fp32. The key scale multiplies the fp32 score; the value
// scale is kept as the unit of the accumulators: O is held in multiples of the current
// block's scale and multiplied by (old unit / new unit) where it changes.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>
#include <torch/types.h>

#include "common.cuh"
#include "device_setup.h"
#include "paged.h"

namespace hrm {
namespace {

constexpr int D = 128;
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kStage = 2 * 16 * D;  // bytes of a warp's 16 keys: codes of keys, then of values
constexpr float kLazy = 8.f;        // a running maximum may lag by 2^8: P stays below 256 in f16
constexpr float kMinUnit = 0x1p-64f;  // a unit is at least this part of the one before it

struct AttnArgs {
  const __nv_bfloat16* q;
  long q_st, q_sh;
  const uint8_t* kc;
  const uint8_t* vc;
  const float* ks;
  const float* vs;
  const int* tables;
  long table_ld;
  const int* kv_len;
  const int* cu_new;
  const int* cu_units;
  int R, Hkv, G, size_log2, causal, T, num_blocks;
  float scale_log2;
  const __nv_bfloat16* gate;
  long g_st, g_sh;
  __nv_bfloat16* out;  // [T, Hq, 128]
  long o_st;
  float* part;  // [2 * workers][tiles][8 * NT][130]: output, maximum, sum
};

// The request whose part of the costs laid end to end holds position `x`; every thread of the CTA
// calls it.
__device__ __forceinline__ int find_request(const AttnArgs& a, long x) {
  int i = 0;
  for (int base = 0; base < a.R; base += kThreads) {
    const int j = base + (int)threadIdx.x;
    const int c = __syncthreads_count(j < a.R && (long)a.cu_units[j + 1] * a.Hkv <= x);
    i += c;
    if (c < kThreads) break;
  }
  return i;
}

// A CTA's range of positions, walked pair by pair.
struct Walk {
  long x, x_end;
  int i, c0, c1;      // a request, its first position / Hkv and its end's
  int h, u0, u1, nu;  // units [u0, u1) of nu of a pair (i, h)
  int row_t, n, len;  // the request's first packed row, new tokens, tokens

  __device__ __forceinline__ void start(const AttnArgs& a, long from, long to, int request) {
    x = from;
    x_end = to;
    i = request;
    enter(a);
  }
  __device__ __forceinline__ void enter(const AttnArgs& a) {
    c0 = a.cu_units[i];
    c1 = a.cu_units[i + 1];
    row_t = a.cu_new[i];
    n = a.cu_new[i + 1] - row_t;
    len = a.kv_len[i];
  }
  // The next piece of a pair with rows in tile `first_row`; false at the end.
  __device__ __forceinline__ bool next(const AttnArgs& a, int first_row) {
    while (x < x_end) {
      while (x >= (long)c1 * a.Hkv) {
        ++i;
        enter(a);
      }
      const int cost = c1 - c0;
      const long in = x - (long)c0 * a.Hkv;
      h = (int)(in / cost);
      const int p0 = (int)(in - (long)h * cost), p1 = (int)min((long)cost, p0 + (x_end - x));
      x += p1 - p0;
      u0 = max(0, p0 - kPairCost);
      u1 = max(0, p1 - kPairCost);
      nu = cost - kPairCost;
      if (u1 > u0 && n * a.G > first_row) return true;
    }
    return false;
  }
  // keys that a row of the tile can see at most
  __device__ __forceinline__ int most(const AttnArgs& a, int first_row, int rows) const {
    return a.causal ? len - n + (first_row + rows - 1) / a.G + 1 : len;
  }
};

__device__ __forceinline__ void copy16(void* smem, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(global) : "memory");
}
__device__ __forceinline__ void copy4(void* smem, const void* global) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(smem)), "l"(global) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <bool FP8>
__device__ __forceinline__ uint32_t widen(uint32_t two) {  // two codes in the low 16 bits -> f16x2
  if constexpr (FP8) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)two));
    return r;
  } else {
    uint32_t r = __byte_perm(two, 0x64646464u, 0x4140);
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152
    const __half2 v = __hsub2(*reinterpret_cast<__half2*>(&r), bias);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <bool FP8>
__device__ __forceinline__ uint32_t widen_hi(uint32_t w) {  // the codes in the high 16 bits
  if constexpr (FP8) {
    return widen<true>(w >> 16);
  } else {
    uint32_t r = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));
    const __half2 v = __hsub2(*reinterpret_cast<__half2*>(&r), bias);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
// int8 codes are widened from code + 128
template <bool FP8>
__device__ __forceinline__ uint32_t biased(uint32_t w) {
  return FP8 ? w : w ^ 0x80808080u;
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t word(const uint4& v, int j) {
  return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w;
}

__device__ __forceinline__ void write_row(const AttnArgs& a, int t, int hq, int d, float o) {
  if (a.gate != nullptr) o *= sigmoidf_(__bfloat162float(a.gate[t * a.g_st + hq * a.g_sh + d]));
  a.out[t * a.o_st + (long)hq * D + d] = __float2bfloat16_rn(o);
}

// A warp's copies ahead: the codes and scales of its 16 keys of every unit of the CTA's range, in order,
// one unit a stage.
template <int STAGES>
struct Ahead {
  Walk w;
  bool live;
  int u, most, block, first;  // next unit; this lane's block, of unit first + lane
  uint8_t* ring;
  float* scales;

  __device__ __forceinline__ void segment(const AttnArgs& a, int first_row, int tile_rows) {
    live = w.next(a, first_row);
    if (live) {
      u = w.u0;
      most = w.most(a, first_row, min(w.n * a.G - first_row, tile_rows));
      first = u - 32;
    }
  }
  __device__ __forceinline__ void copy(const AttnArgs& a, int stage, int warp, int lane, int first_row, int tile_rows) {
    while (live && (u >= w.u1 || u * kUnitKeys + warp * 16 >= most)) segment(a, first_row, tile_rows);
    if (live) {
      if (u - first == 32) {
        first = u;
        const int kb = (u + lane) * kUnitKeys + warp * 16;
        block = 0;
        if (u + lane < w.u1 && kb < w.len) block = a.tables[w.i * a.table_ld + (kb >> a.size_log2)];
        if (block < 0 || block >= a.num_blocks) block = 0;  // not a table of this cache
      }
      const long bh = (long)__shfl_sync(~0u, block, u - first) * a.Hkv + w.h;
      const int kb = u * kUnitKeys + warp * 16;
      const long base = ((bh << a.size_log2) + (kb & ((1 << a.size_log2) - 1))) * D + lane * 16;
      uint8_t* to = ring + stage * kStage;
      // four rows of 128 bytes an instruction; the 16-byte pieces of a row change places so that the
      // reads below meet no bank twice
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = j * 4 + (lane >> 3), c = lane & 7;
        copy16(to + r * D + ((c ^ ((r & 1) * 4)) << 4), a.kc + base + j * 4 * D);
        copy16(to + kStage / 2 + r * D + ((c ^ (r & 6)) << 4), a.vc + base + j * 4 * D);
      }
      if (lane < 2) copy4(scales + stage * 2 + lane, (lane ? a.vs : a.ks) + bh);
      ++u;
    }
    copy_commit();
  }
};

template <bool FP8, int NT, int STAGES>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1) paged_attention_kernel(const AttnArgs a) {
  constexpr int ROWS = 8 * NT;
  extern __shared__ __align__(128) uint8_t s_ring[];  // [kWarps][STAGES][kStage], then the merge's
  float* s_o = reinterpret_cast<float*>(s_ring + kWarps * STAGES * kStage);  // [kWarps][rows of the tile][D]
  __shared__ float s_scales[kWarps][STAGES][2];
  __shared__ float s_m[kWarps][ROWS], s_l[kWarps][ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tg = lane & 3;
  const int worker = blockIdx.x, tile = blockIdx.y, r0 = tile * ROWS, Hq = a.Hkv * a.G;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join may take its places; it waits for the end

  if (tile == 0)  // rows of no request
    for (long t = a.cu_new[a.R] + worker; t < a.T; t += gridDim.x)
      for (int c = threadIdx.x; c < Hq * D / 8; c += kThreads)
        *reinterpret_cast<uint4*>(a.out + t * a.o_st + c * 8) = make_uint4(0, 0, 0, 0);

  const long total = (long)a.cu_units[a.R] * a.Hkv, per = (total + gridDim.x - 1) / gridDim.x;
  if (per * worker >= total) return;
  Walk at;
  at.start(a, per * worker, min(total, per * (worker + 1)), find_request(a, per * worker));
  Ahead<STAGES> ahead;
  ahead.w = at;
  ahead.ring = s_ring + warp * STAGES * kStage;
  ahead.scales = s_scales[warp][0];
  ahead.segment(a, r0, ROWS);
#pragma unroll
  for (int st = 0; st < STAGES - 1; ++st) ahead.copy(a, st, warp, lane, r0, ROWS);
  int stage = 0;

  while (at.next(a, r0)) {
    const int row_t = at.row_t, n = at.n, len = at.len, u0 = at.u0, u1 = at.u1;
    const int rows = min(n * a.G - r0, ROWS);

    // queries as the B operand, scaled to f16; limits and logit factors of this lane's columns
    uint32_t qf[NT][8][2];
    float factor[NT][2];
    int limit[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 8 + g;
      uint4 raw[4] = {};
      if (r < rows) {
        const int rr = r0 + r;
        const __nv_bfloat16* p = a.q + (row_t + rr / a.G) * a.q_st + (at.h * a.G + rr % a.G) * a.q_sh + tg * 16;
        raw[0] = *reinterpret_cast<const uint4*>(p);
        raw[1] = *reinterpret_cast<const uint4*>(p + 8);
        raw[2] = *reinterpret_cast<const uint4*>(p + 64);
        raw[3] = *reinterpret_cast<const uint4*>(p + 72);
      }
      uint32_t top = 0;
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) top = __vmaxu2(top, word(raw[c], j) & 0x7fff7fffu);
      top = max(top & 0xffffu, top >> 16);
      top = max(top, __shfl_xor_sync(~0u, top, 1));
      top = max(top, __shfl_xor_sync(~0u, top, 2));
      // 2^-e with e the exponent of the largest magnitude (within what a float can hold)
      const int e = min(126, max(-126, (int)(top >> 7) - 127));
      const float down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 lo = unpack_bf16x2(word(raw[j / 2], (j & 1) * 2)), hi = unpack_bf16x2(word(raw[j / 2], (j & 1) * 2 + 1));
        qf[nt][j][0] = pack_f16x2(lo.x * down, lo.y * down);
        qf[nt][j][1] = pack_f16x2(hi.x * down, hi.y * down);
      }
      const float up = __uint_as_float((uint32_t)(127 + e) << 23) * a.scale_log2;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        factor[nt][c] = __shfl_sync(~0u, up, (2 * tg + c) * 4);
        const int rc = nt * 8 + 2 * tg + c;
        limit[nt][c] = rc >= rows ? 0 : a.causal ? len - n + (r0 + rc) / a.G + 1 : len;
      }
    }
    const int most = at.most(a, r0, rows);
    const int least = a.causal ? len - n + r0 / a.G + 1 : len;

    float o[NT][8][4] = {}, m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        m[nt][c] = -INFINITY;
        l[nt][c] = 0.f;
      }
    float unit = 0.f;  // O is held in multiples of this

    for (int u = u0; u < u1; ++u) {
      const int kb = u * kUnitKeys + warp * 16;
      if (kb >= most) break;
      copy_wait<STAGES - 2>();
      __syncwarp();  // this stage is there, and the stage before it was read by every lane
      ahead.copy(a, stage == 0 ? STAGES - 1 : stage - 1, warp, lane, r0, ROWS);
      const uint8_t* kp = s_ring + (warp * STAGES + stage) * kStage + g * D + ((tg ^ ((g & 1) * 4)) << 4);
      const uint8_t* vp = s_ring + (warp * STAGES + stage) * kStage + kStage / 2 + 2 * tg * D + ((g ^ (2 * tg)) << 4);
      const float ks = s_scales[warp][stage][0], vs = s_scales[warp][stage][1];
      stage = stage == STAGES - 1 ? 0 : stage + 1;
      const auto codes = [](const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); };
      // rows g and g + 8 of the keys (pieces tg and tg + 4), rows 2 tg, 2 tg + 1 and those 8 below of the values
      const uint8_t* kp1 = s_ring + (kp - s_ring ^ 64);
      const uint4 k0 = codes(kp), k1 = codes(kp1), k2 = codes(kp + 8 * D), k3 = codes(kp1 + 8 * D);
      const uint4 v0 = codes(vp), v1 = codes(vp + D), v2 = codes(vp + 8 * D), v3 = codes(vp + 9 * D);

      float s[NT][4] = {};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t lo = biased<FP8>(word(j < 4 ? k0 : k1, j & 3)), hi = biased<FP8>(word(j < 4 ? k2 : k3, j & 3));
        const uint32_t a0 = widen<FP8>(lo), a2 = widen_hi<FP8>(lo), a1 = widen<FP8>(hi), a3 = widen_hi<FP8>(hi);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816(s[nt], a0, a1, a2, a3, qf[nt][j][0], qf[nt][j][1]);
      }

      bool raise = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float f0 = factor[nt][0] * ks, f1 = factor[nt][1] * ks;
        s[nt][0] *= f0;
        s[nt][1] *= f1;
        s[nt][2] *= f0;
        s[nt][3] *= f1;
        if (kb + 16 > least) {
          if (kb + g >= limit[nt][0]) s[nt][0] = -INFINITY;
          if (kb + g >= limit[nt][1]) s[nt][1] = -INFINITY;
          if (kb + g + 8 >= limit[nt][0]) s[nt][2] = -INFINITY;
          if (kb + g + 8 >= limit[nt][1]) s[nt][3] = -INFINITY;
        }
        raise |= fmaxf(s[nt][0], s[nt][2]) > m[nt][0] + kLazy || fmaxf(s[nt][1], s[nt][3]) > m[nt][1] + kLazy;
      }
      // accumulators to the new block's unit, and under the new maximum where one has risen
      const float next = vs == 0.f ? unit : fmaxf(vs, unit * kMinUnit) + (vs - vs);  // NaN stays NaN
      const float ratio = next == unit ? 1.f : unit / next;
      const float shrink = vs == next || vs == 0.f ? 1.f : vs / next;
      unit = next;
      raise = __any_sync(~0u, raise);
      if (raise || ratio != 1.f) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float f[2] = {ratio, ratio};
          if (raise) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float top = fmaxf(s[nt][c], s[nt][c + 2]);
              top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
              top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
              top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
              const float now = fmaxf(m[nt][c], top);
              const float alpha = now == m[nt][c] ? 1.f : fast_exp2(m[nt][c] - now);
              m[nt][c] = now;
              l[nt][c] *= alpha;
              f[c] *= alpha;
            }
          }
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {
            o[nt][mt][0] *= f[0];
            o[nt][mt][1] *= f[1];
            o[nt][mt][2] *= f[0];
            o[nt][mt][3] *= f[1];
          }
        }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float m0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], m1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
        float p0 = fast_exp2(s[nt][0] - m0), p1 = fast_exp2(s[nt][1] - m1);
        float p2 = fast_exp2(s[nt][2] - m0), p3 = fast_exp2(s[nt][3] - m1);
        l[nt][0] += p0 + p2;
        l[nt][1] += p1 + p3;
        if (shrink != 1.f) {
          p0 *= shrink;
          p1 *= shrink;
          p2 *= shrink;
          p3 *= shrink;
        }
        pb[nt][0] = transpose8x8(pack_f16x2(p0, p1));
        pb[nt][1] = transpose8x8(pack_f16x2(p2, p3));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w0 = biased<FP8>(word(v0, j)), w1 = biased<FP8>(word(v1, j)), w2 = biased<FP8>(word(v2, j)),
                       w3 = biased<FP8>(word(v3, j));
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // two of the word's four dims
          const uint32_t lo = __byte_perm(w0, w1, half ? 0x7362 : 0x5140), hi = __byte_perm(w2, w3, half ? 0x7362 : 0x5140);
          const uint32_t a0 = widen<FP8>(lo), a1 = widen_hi<FP8>(lo), a2 = widen<FP8>(hi), a3 = widen_hi<FP8>(hi);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][2 * j + half], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
        }
      }
    }

    // the warps' parts: this lane has dims 16 g + 2 mt (+ 1) of rows 2 tg and 2 tg + 1 of each 8
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float sum = l[nt][c];
        sum += __shfl_xor_sync(~0u, sum, 4);
        sum += __shfl_xor_sync(~0u, sum, 8);
        sum += __shfl_xor_sync(~0u, sum, 16);
        const int r = nt * 8 + 2 * tg + c;
        if (r < rows) {
          if (g == 0) {
            s_m[warp][r] = m[nt][c];
            s_l[warp][r] = sum;
          }
          float4* to = reinterpret_cast<float4*>(s_o + ((long)warp * rows + r) * D + g * 16);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            to[k] = make_float4(o[nt][2 * k][c] * unit, o[nt][2 * k][c + 2] * unit, o[nt][2 * k + 1][c] * unit,
                                o[nt][2 * k + 1][c + 2] * unit);
        }
      }
    __syncthreads();
    const bool whole = u0 == 0 && u1 == at.nu;
    // the part of a pair that starts here but ends elsewhere has the worker's second place
    float* part = a.part + ((long)(2 * worker + (u0 == 0 ? 1 : 0)) * gridDim.y + tile) * ROWS * (D + 2);
    for (int idx = threadIdx.x; idx < rows * D; idx += kThreads) {
      const int r = idx / D, d = idx % D;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w][r]);
      const float ref = top == -INFINITY ? 0.f : top;
      float sum = 0.f, out = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = fast_exp2(s_m[w][r] - ref);
        sum += s_l[w][r] * f;
        out += s_o[((long)w * rows + r) * D + d] * f;
      }
      if (whole) {
        write_row(a, row_t + (r0 + r) / a.G, at.h * a.G + (r0 + r) % a.G, d, sum == 0.f ? 0.f : out / sum);
      } else {
        part[r * (D + 2) + d] = out;
        if (d == 0) {
          part[r * (D + 2) + D] = top;
          part[r * (D + 2) + D + 1] = sum;
        }
      }
    }
    __syncthreads();
  }
}

// Joins the pairs that span workers: the worker in whose range such a pair ends does it.
template <int NT>
__global__ void __launch_bounds__(kThreads) paged_attention_join_kernel(const AttnArgs a) {
  constexpr int ROWS = 8 * NT;
  const long total = (long)a.cu_units[a.R] * a.Hkv, per = (total + gridDim.x - 1) / gridDim.x;
  const int worker = blockIdx.x, tile = blockIdx.y, r0 = tile * ROWS;
  const long x = per * worker, x_end = min(total, x + per);
  if (x >= x_end) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const int i = find_request(a, x), c0 = a.cu_units[i], cost = a.cu_units[i + 1] - c0;
  const long in = x - (long)c0 * a.Hkv;
  const int h = (int)(in / cost), p = (int)(in - (long)h * cost);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the parts are written; in every CTA, so this grid ends last
  if (p <= kPairCost || x + (cost - p) > x_end) return;  // starts here, or goes on in the next range
  const int row_t = a.cu_new[i], n = a.cu_new[i + 1] - row_t;
  const int rows = min(n * a.G - r0, ROWS);
  const int first = (int)((x - p + kPairCost) / per);
  const auto place = [&](int w) {  // the first worker may start with the pair or before it
    return a.part + ((long)(2 * w + (w == first ? 1 : 0)) * gridDim.y + tile) * ROWS * (D + 2);
  };
  for (int idx = threadIdx.x; idx < rows * D; idx += kThreads) {
    const int r = idx / D, d = idx % D;
    float top = -INFINITY;
    for (int w = first; w <= worker; ++w) top = fmaxf(top, place(w)[r * (D + 2) + D]);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f, out = 0.f;
    for (int w = first; w <= worker; ++w) {
      const float* p = place(w) + r * (D + 2);
      const float f = fast_exp2(p[D] - ref);
      sum += p[D + 1] * f;
      out += p[d] * f;
    }
    write_row(a, row_t + (r0 + r) / a.G, h * a.G + (r0 + r) % a.G, d, sum == 0.f ? 0.f : out / sum);
  }
}

template <bool FP8, int NT, int STAGES>
void launch(AttnArgs a, int max_rows, const at::TensorOptions& opts, cudaStream_t stream) {
  constexpr int ROWS = 8 * NT;
  const int tiles = (max_rows + ROWS - 1) / ROWS;
  TORCH_CHECK(tiles <= 65535, "paged_attention: too many new tokens for one request");
  const int smem = kWarps * (STAGES * kStage + std::min(max_rows, ROWS) * D * 4);
  C10_CUDA_CHECK(ensure_dynamic_smem((const void*)paged_attention_kernel<FP8, NT, STAGES>,
                                     kWarps * (STAGES * kStage + ROWS * D * 4)));
  const int workers = device_sm_count() * (NT == 1 ? 2 : 1);
  const at::Tensor part = at::empty({2L * workers * tiles * ROWS * (D + 2)}, opts.dtype(at::kFloat));
  a.part = part.data_ptr<float>();
  const dim3 grid(workers, tiles);
  paged_attention_kernel<FP8, NT, STAGES><<<grid, kThreads, smem, stream>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  // the join is launched while the first kernel runs and waits for its end itself
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(kThreads);
  config.stream = stream;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early;
  config.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&config, paged_attention_join_kernel<NT>, a));
}

template <bool FP8>
void launch_rows(const AttnArgs& a, int max_rows, const at::TensorOptions& opts, cudaStream_t stream) {
  if (max_rows <= 4)
    launch<FP8, 1, 3>(a, max_rows, opts, stream);
  else if (max_rows <= 8)
    launch<FP8, 1, 2>(a, max_rows, opts, stream);
  else if (max_rows <= 16)
    launch<FP8, 2, 4>(a, max_rows, opts, stream);
  else
    launch<FP8, 4, 3>(a, max_rows, opts, stream);
}

}  // namespace

// query [T, Hq, 128] bf16 (row and head strides of whole 16 bytes); the cache of one layer
// (paged_kv8.cu); tables and meta of the step (paged_tables.cu); max_new bounds the new tokens of a
// request; gate [T, Hq, 128] bf16 or none. Returns [T, Hq, 128] bf16.
at::Tensor paged_attention(const at::Tensor& query, const at::Tensor& keys, const at::Tensor& values,
                     const at::Tensor& key_scales, const at::Tensor& value_scales, const at::Tensor& tables,
                     const at::Tensor& meta, int64_t max_new, bool causal, const c10::optional<at::Tensor>& gate) {
  TORCH_CHECK(keys.is_cuda() && keys.dim() == 4 && keys.size(3) == D && keys.is_contiguous() &&
                  (keys.scalar_type() == at::kChar || keys.scalar_type() == at::kFloat8_e4m3fn) &&
                  values.sizes() == keys.sizes() && values.scalar_type() == keys.scalar_type() && values.is_contiguous() &&
                  values.device() == keys.device(),
              "paged_attention: contiguous CUDA codes [blocks, heads, block size, 128], int8 or float8_e4m3fn");
  const int64_t T = query.size(0), H = keys.size(1), R = tables.size(0), s = keys.size(2);
  TORCH_CHECK(s == 16 || s == 32 || s == 64 || s == 128, "block size must be 16, 32, 64 or 128");
  for (const at::Tensor* t : {&key_scales, &value_scales})
    TORCH_CHECK(t->dim() == 2 && t->size(0) == keys.size(0) && t->size(1) == H && t->is_contiguous() &&
                    t->scalar_type() == at::kFloat && t->device() == keys.device(),
                "paged_attention: fp32 scales [blocks, heads]");
  const auto rows_ok = [&](const at::Tensor& t) {
    return t.device() == keys.device() && t.scalar_type() == at::kBFloat16 && t.dim() == 3 && t.size(2) == D &&
           (t.numel() == 0 || t.stride(2) == 1) && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 &&
           reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  };
  TORCH_CHECK(rows_ok(query) && query.size(1) % H == 0 && query.size(1) > 0,
              "paged_attention: query [T, heads, 128] bf16 on the cache's device, with 16-byte aligned rows and a "
              "multiple of the cache's heads");
  TORCH_CHECK(!gate || (rows_ok(*gate) && gate->sizes() == query.sizes()), "paged_attention: gate like query");
  TORCH_CHECK(tables.device() == keys.device() && tables.scalar_type() == at::kInt && tables.dim() == 2 &&
                  tables.stride(1) == 1,
              "paged_attention: block tables int32 [requests, blocks]");
  TORCH_CHECK(meta.device() == keys.device() && meta.scalar_type() == at::kInt && meta.is_contiguous() &&
                  meta.numel() == 3 * R + 3,
              "paged_attention: a step of these tables");
  c10::cuda::CUDAGuard guard(keys.device());
  const at::Tensor out = at::empty({T, query.size(1), D}, query.options());
  if (T == 0) return out;
  AttnArgs a{};
  a.q = reinterpret_cast<const __nv_bfloat16*>(query.data_ptr());
  a.q_st = query.stride(0);
  a.q_sh = query.stride(1);
  a.kc = reinterpret_cast<const uint8_t*>(keys.data_ptr());
  a.vc = reinterpret_cast<const uint8_t*>(values.data_ptr());
  a.ks = key_scales.data_ptr<float>();
  a.vs = value_scales.data_ptr<float>();
  a.tables = tables.data_ptr<int>();
  a.table_ld = tables.stride(0);
  a.cu_new = meta.data_ptr<int>();
  a.cu_units = a.cu_new + R + 1;
  a.kv_len = a.cu_units + R + 1;
  a.R = (int)R;
  a.Hkv = (int)H;
  a.G = (int)(query.size(1) / H);
  a.size_log2 = s == 16 ? 4 : s == 32 ? 5 : s == 64 ? 6 : 7;
  a.causal = causal;
  a.T = (int)T;
  a.num_blocks = (int)keys.size(0);
  a.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)D));
  if (gate) {
    a.gate = reinterpret_cast<const __nv_bfloat16*>(gate->data_ptr());
    a.g_st = gate->stride(0);
    a.g_sh = gate->stride(1);
  }
  a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  a.o_st = out.stride(0);
  const int64_t max_rows = std::min<int64_t>(max_new, T) * a.G;
  TORCH_CHECK(max_rows < (1LL << 30), "paged_attention: too many rows");
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  if (keys.scalar_type() == at::kFloat8_e4m3fn)
    launch_rows<true>(a, (int)std::max<int64_t>(max_rows, 1), query.options(), stream);
  else
    launch_rows<false>(a, (int)std::max<int64_t>(max_rows, 1), query.options(), stream);
  return out;
}

}  // namespace hrm
