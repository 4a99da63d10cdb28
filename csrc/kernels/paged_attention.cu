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
// In a CTA each of 4 warps takes 32 keys of a unit and keeps its own running maximum, sum and
// output for up to 8 * NT query rows (G query heads times the request's new tokens; requests with
// more rows take several tiles). The warps are merged through shared memory once per pair. Each
// warp copies its own codes ahead into its own ring of shared memory (cp.async, 8 KB a stage), across
// the ends of pairs, so that it waits for no other warp and a pair's first loads run under the
// work before it. 16 of a warp's keys are
//   S^T [16 keys x 8 rows] = C [16 x 128] Q^T,   O^T [128 dims x 8 rows] += C'^T [128 x 16] P^T
// in mma.m16n8k16 with the keys as the M side: 8 rows, the smallest N, waste the least of a
// matrix instruction on the one or few rows a decode step has. The kernel reads 256 bytes a key
// and head for 4 * 128 * rows flops, so warp-level matrix instructions are far from their limit; what
// counts is how few instructions a byte of codes takes:
//   * the k index of S = C Q^T may be permuted as one likes if Q is permuted alike, so a lane
//     owns 32 dims of two keys as four 16-byte words, and a 32-bit word of codes is the lane's
//     part of one k step;
//   * the m index of O^T likewise: a lane owns 16 dims of four keys, pairs of keys are
//     interleaved by byte permutes before they are widened;
//   * P^T is S^T transposed 8x8 by movmatrix.
// Codes are exact in f16: e4m3 by one cvt, int8 as 1152 + c by one byte permute, less 1152. Queries are
// scaled by a power of two to a row maximum in [1, 2) before they are rounded to f16: a bf16 value keeps all its bits
// unless it is 2^-14 of the row's largest. P is rounded to f16 (11 bits, against 8 of bf16), sums
// stay fp32. The key scale multiplies the fp32 score. What is rounded is the product of P and the block's value scale, in
// multiples of a unit of the row's own: a second running maximum, of score + log2(value scale), which moves like
// the first (of the scores, for the sum of P). So each product keeps its 11 bits whatever ranges the row's blocks have, and
// one that is lost is below 2^-24 of the row's largest.
//
// Measured (one B200, copy rate 6.54 TB/s, L2 cold): 16 requests of 4000 to 40000 tokens, 8 kv heads, 4 query
// heads each, int8: 98 us for 632 MB (99 % of the copy rate); 100 requests of 1 to 4096 tokens, 12 heads,
// e4m3: 102 us for 663 MB (99 %). Small calls are bound by dependent loads and launches: one
// request of 777 tokens 6.3 us, 33 requests around 600 tokens 16 us (e4m3: 15) for 46 MB, of which about 5 us
// pass before the first codes arrive; the join ends some 2 us later. With 8 to 16 rows (12 requests of 300 to 6000
// tokens, up to 7 new ones, 2 query heads) 26 us (int8: 27) for 96 MB: the latency of a step's chains (11 warps an SM,
// 49 % of the issue slots used). Many new tokens read and widen the codes again for each 16 rows: 2048 on 2048
// cached, 10 heads, 214 us (e4m3: 196), of which the products at the bf16 rate would be 26. 3 CTAs an SM (168
// registers) hold 12 warps with 8 KB each in flight; 2 CTAs of 8 warps with 4 KB steps were 6 and 18 % slower on the
// first two cases.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>
#include <torch/types.h>

#include "common.cuh"
#include "device_setup.h"
#include "launch_early.h"
#include "paged.h"

namespace hrm {
namespace {

constexpr int D = 128;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kJoin = 256;  // threads of the joining kernel
constexpr int kKeys = kUnitKeys / kWarps;  // a warp's keys of a unit: two halves of 16
constexpr int kHalf = 2 * 16 * D;          // bytes of 16 keys: codes of keys, then of values
constexpr int kStage = 2 * kHalf;
constexpr int kStages = 2;      // one is read while the other is filled
constexpr int kPart = D + 4;    // floats of a row's part, in whole 16 bytes
constexpr int kFewTiles = 4;    // up to these the grid has each nominal tile's workers
constexpr float kLazy = 8.f;    // a running maximum may lag by 2^8: P stays below 256 in f16
constexpr float kNoUnit = 1e30f;  // in place of log2(2^m / O's unit) before a value was met: O is 0
constexpr float kMostRatio = 126.f;  // where 2^m / unit * scale is larger, P is 0

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
  float* part;  // [tiles][workers][2][8 * NT][kPart]: output, maximum, sum
  int split;    // 0: the grid is workers x tiles; else CTAs that the step's tiles are given
};

struct Found {
  int i, c0, c1;      // a request, its first position / Hkv and its end's
  int row_t, n, len;  // its first packed row, new tokens, tokens
};
// What this thread knows of request `j`, loaded before the position is known.
__device__ __forceinline__ Found request_of(const AttnArgs& a, int j) {
  if (j >= a.R) return Found{j, 0, 0, 0, 0, 0};
  const int row_t = a.cu_new[j];
  return Found{j, a.cu_units[j], a.cu_units[j + 1], row_t, a.cu_new[j + 1] - row_t, a.kv_len[j]};
}
// Which of a tile's workers a CTA is. Few tiles: the grid says so. Otherwise the host knows only a bound of the tiles,
// which may be far above what the step's largest request has: that is read here, and the workers of a tile follow.
struct Place {
  int workers, worker, tile;
  bool none;
};
template <int ROWS>
__device__ __forceinline__ Place place_of(const AttnArgs& a, const Found& mine) {
  Place p{(int)gridDim.x, (int)blockIdx.x, (int)blockIdx.y, false};
  if (a.split > 0) {
    __shared__ int s_most[32];
    int n = mine.n;
    for (int j = threadIdx.x + blockDim.x; j < a.R; j += blockDim.x) n = max(n, a.cu_new[j + 1] - a.cu_new[j]);
    n = __reduce_max_sync(~0u, n);
    if ((threadIdx.x & 31) == 0) s_most[threadIdx.x >> 5] = n;
    __syncthreads();
    for (int w = 0; w < (int)blockDim.x / 32; ++w) n = max(n, s_most[w]);
    const int tiles = max(1, (int)(((long)n * a.G + ROWS - 1) / ROWS));
    p.workers = max(1, a.split / max(tiles, kFewTiles));  // few: as with a grid that says so
    p.worker = blockIdx.x % p.workers;
    p.tile = blockIdx.x / p.workers;
    p.none = p.tile >= tiles;
  }
  return p;
}
// The request whose part of the costs laid end to end holds position `x`; every thread of the CTA
// calls it. `mine` is request_of(threadIdx.x).
__device__ __forceinline__ Found find_request(const AttnArgs& a, long x, Found mine) {
  __shared__ Found s_found;
  for (;;) {
    const int c = __syncthreads_count(mine.i < a.R && (long)mine.c1 * a.Hkv <= x);
    if (c < (int)blockDim.x) {
      if ((int)threadIdx.x == c) s_found = mine;
      break;
    }
    mine = request_of(a, mine.i + (int)blockDim.x);
  }
  __syncthreads();
  return s_found;
}

// A CTA's range of positions, walked pair by pair.
struct Walk {
  long x, x_end;
  Found at;           // a request
  int h, u0, u1, nu;  // units [u0, u1) of nu of a pair (at.i, h)

  // The next piece of a pair with rows in tile `first_row`; false at the end.
  __device__ __forceinline__ bool next(const AttnArgs& a, int first_row) {
    while (x < x_end) {
      while (x >= (long)at.c1 * a.Hkv) at = request_of(a, at.i + 1);
      const int cost = at.c1 - at.c0;
      const uint32_t in = (uint32_t)(x - (long)at.c0 * a.Hkv);  // the host checked that this fits
      h = (int)(in / (uint32_t)cost);
      const int p0 = (int)(in - (uint32_t)h * cost), p1 = (int)min((long)cost, p0 + (x_end - x));
      x += p1 - p0;
      u0 = max(0, p0 - kPairCost);
      u1 = max(0, p1 - kPairCost);
      nu = cost - kPairCost;
      if (u1 > u0 && at.n * a.G > first_row) return true;
    }
    return false;
  }
  // keys that a row of the tile can see at most
  __device__ __forceinline__ int most(const AttnArgs& a, int first_row, int rows) const {
    return a.causal ? at.len - at.n + (first_row + rows - 1) / a.G + 1 : at.len;
  }
};

__device__ __forceinline__ void copy16(void* smem, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(global) : "memory");
}
__device__ __forceinline__ void copy4(void* smem, const void* global) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(smem)), "l"(global) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// Two codes, in bytes 0 and 1 (HI: 2 and 3) of a word, as f16x2: e4m3 themselves; int8, given as code + 128,
// as 1024 + that, less 1152.
template <bool FP8, bool HI>
__device__ __forceinline__ uint32_t widen(uint32_t w) {
  uint32_t r;
  if constexpr (FP8) {
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)(HI ? w >> 16 : w)));
  } else {
    r = __byte_perm(w, 0x64646464u, HI ? 0x4342 : 0x4140);
    const __half2 v = __hsub2(*reinterpret_cast<__half2*>(&r), __half2half2(__ushort_as_half(0x6480)));
    r = *reinterpret_cast<const uint32_t*>(&v);
  }
  return r;
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
__device__ __forceinline__ float log2_of(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t word(const uint4& v, int j) {
  return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w;
}

// Four dims of a finished row: o / l, times the gate's sigmoid.
__device__ __forceinline__ void write_row(const AttnArgs& a, int t, int hq, int d, const float (&o)[4], float l, uint2 gate) {
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float v[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  if (a.gate != nullptr) {
    const float2 lo = unpack_bf16x2(gate.x), hi = unpack_bf16x2(gate.y);
    v[0] *= sigmoidf_(lo.x);
    v[1] *= sigmoidf_(lo.y);
    v[2] *= sigmoidf_(hi.x);
    v[3] *= sigmoidf_(hi.y);
  }
  *reinterpret_cast<uint2*>(a.out + t * a.o_st + (long)hq * D + d) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

// A warp's copies ahead: the codes and scales of its keys of every unit of the CTA's range, in order,
// one unit a stage.
struct Ahead {
  Walk w;
  bool live;
  int u, most, first, block;  // next unit; this lane's block: of unit first + lane / 2, half lane % 2
  uint8_t* ring;
  float* scales;  // [kStages][2 halves][keys, values]

  __device__ __forceinline__ void segment(const AttnArgs& a, int first_row, int tile_rows) {
    live = w.next(a, first_row);
    if (live) {
      u = w.u0;
      most = w.most(a, first_row, min(w.at.n * a.G - first_row, tile_rows));
      first = u - 16;
    }
  }
  __device__ __forceinline__ void copy(const AttnArgs& a, int stage, int warp, int lane, int first_row, int tile_rows) {
    while (live && (u >= w.u1 || u * kUnitKeys + warp * kKeys >= most)) segment(a, first_row, tile_rows);
    if (live) {
      if (u - first == 16) {
        first = u;
        // a half after the last token takes the block, and so the scales, of the half before it
        const int kb = (u + (lane >> 1)) * kUnitKeys + warp * kKeys + (lane & 1) * 16;
        block = 0;
        if (u + (lane >> 1) < w.u1) block = a.tables[w.at.i * a.table_ld + (min(kb, w.at.len - 1) >> a.size_log2)];
        if (block < 0 || block >= a.num_blocks) block = 0;  // not a table of this cache
      }
      // lane's row of each four and its 16-byte piece; the pieces of a row change places so that the
      // reads meet no bank twice: by 4 in odd rows of keys, by (row & 6) in rows of values
      const int q = lane >> 3, c = lane & 7;
      uint8_t* kto = ring + stage * kStage + q * D + ((c ^ ((q & 1) * 4)) << 4);
      uint8_t* vto = ring + stage * kStage + kHalf / 2 + q * D + ((c ^ (q & 2)) << 4);
      const int odd = ((c ^ (q & 2) ^ 4) - (c ^ (q & 2))) * 16;  // to the place in rows 4 to 7 and 12 to 15
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int kb = u * kUnitKeys + warp * kKeys + half * 16;
        const long bh = (long)__shfl_sync(~0u, block, 2 * (u - first) + half) * a.Hkv + w.h;
        const long base = ((bh << a.size_log2) + (kb & ((1 << a.size_log2) - 1))) * D + lane * 16;
        const uint8_t *kp = a.kc + base, *vp = a.vc + base;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          copy16(kto + half * kHalf + j * 4 * D, kp + j * 4 * D);
          copy16(vto + half * kHalf + j * 4 * D + (j & 1) * odd, vp + j * 4 * D);
        }
        if (lane < 2) copy4(scales + stage * 4 + half * 2 + lane, (lane ? a.vs : a.ks) + bh);
      }
      ++u;
    }
    copy_commit();
  }
};

template <bool FP8, int NT>
__global__ void __launch_bounds__(kThreads, 3) paged_attention_kernel(const AttnArgs a) {
  constexpr int ROWS = 8 * NT;
  static_assert(ROWS * D * 4 <= kStage, "a stage holds a warp's part of the merge");
  extern __shared__ __align__(128) uint8_t s_ring[];  // [kWarps][kStages][kStage]
  __shared__ __align__(16) float s_scales[kWarps][kStages][2][2];
  __shared__ float s_m[kWarps][ROWS], s_l[kWarps][ROWS];
  __shared__ __align__(16) uint32_t s_q[NT == 1 ? 1 : 8][32][NT * 2];  // queries, where registers are short
  __shared__ int s_part[kWarps];  // where in s_ring a warp's part of the merge is, -1: it has none
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tg = lane & 3;
  const int Hq = a.Hkv * a.G;
  asm volatile("griddepcontrol.wait;" ::: "memory");               // this grid starts while the kernel before it ends
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join may take its places; it waits for the end

  const Found mine = request_of(a, threadIdx.x);
  const int units = a.cu_units[a.R], real_rows = a.cu_new[a.R];
  const Place place = place_of<ROWS>(a, mine);
  if (place.none) return;
  const int r0 = place.tile * ROWS;
  if (r0 == 0)  // rows of no request
    for (long t = real_rows + place.worker; t < a.T; t += place.workers)
      for (int c = threadIdx.x; c < Hq * D / 8; c += kThreads)
        *reinterpret_cast<uint4*>(a.out + t * a.o_st + c * 8) = make_uint4(0, 0, 0, 0);
  const long total = (long)units * a.Hkv, per = (total + place.workers - 1) / place.workers;
  if (per * place.worker >= total) return;
  const int slot = (place.tile * place.workers + place.worker) * 2;  // this CTA's two places in the workspace
  Walk walk;
  walk.x = per * place.worker;
  walk.x_end = min(total, walk.x + per);
  walk.at = find_request(a, walk.x, mine);
  Ahead ahead;
  ahead.w = walk;
  ahead.ring = s_ring + warp * kStages * kStage;
  ahead.scales = s_scales[warp][0][0];
  ahead.segment(a, r0, ROWS);
  int stage = 0;
  bool begun = false;
  // this lane's pieces: rows g and g + 8 of the keys, pieces tg and tg + 4; rows 2 tg, 2 tg + 1 and those 8
  // below of the values, piece g
  const uint8_t* k_lane = ahead.ring + g * D + ((tg ^ ((g & 1) * 4)) << 4);
  const int k_more = ((tg ^ ((g & 1) * 4) ^ 4) - (tg ^ ((g & 1) * 4))) * 16;
  const uint8_t* v_lane = ahead.ring + kHalf / 2 + 2 * tg * D + ((g ^ (2 * tg)) << 4);
  const auto codes = [](const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); };

  while (walk.next(a, r0)) {
    const int row_t = walk.at.row_t, n = walk.at.n, len = walk.at.len, u0 = walk.u0, u1 = walk.u1, h = walk.h;
    const int rows = min(n * a.G - r0, ROWS);

    // queries as the B operand, scaled to f16; limits and logit factors of this lane's columns
    uint4 raws[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int rr = r0 + nt * 8 + g;
      const __nv_bfloat16* p = a.q + (row_t + rr / a.G) * a.q_st + (h * a.G + rr % a.G) * a.q_sh + tg * 16;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        raws[nt][c] = rr < n * a.G ? *reinterpret_cast<const uint4*>(p + (c >> 1) * 64 + (c & 1) * 8) : make_uint4(0, 0, 0, 0);
    }
    if (!begun) ahead.copy(a, 0, warp, lane, r0, ROWS);  // the first codes, while the queries are on their way
    begun = true;
    uint32_t qf[NT][8][2];
    float factor[NT][2];
    int limit[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint4(&raw)[4] = raws[nt];
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
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float2 v = unpack_bf16x2(word(raw[j / 2], (j & 1) * 2 + c));
          qf[nt][j][c] = pack_f16x2(v.x * down, v.y * down);
        }
      }
      const float up = __uint_as_float((uint32_t)(127 + e) << 23) * a.scale_log2;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        factor[nt][c] = __shfl_sync(~0u, up, (2 * tg + c) * 4);
        const int rc = nt * 8 + 2 * tg + c;
        limit[nt][c] = rc >= rows ? 0 : a.causal ? len - n + (r0 + rc) / a.G + 1 : len;
      }
    }
    if constexpr (NT > 1) {  // the same in every warp: each writes its share
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j / 2 == warp)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            s_q[j][lane][nt * 2] = qf[nt][j][0];
            s_q[j][lane][nt * 2 + 1] = qf[nt][j][1];
          }
      __syncthreads();
    }
    const int most = walk.most(a, r0, rows);
    const int least = a.causal ? len - n + r0 / a.G + 1 : len;

    float o[NT][8][4] = {}, m[NT][2] = {}, l[NT][2] = {};
    float to_unit[NT][2];          // log2(2^m / unit), O of a column held in multiples of its unit
    int none = (1 << 2 * NT) - 1;  // columns that have no maximum yet
    int last = -1;                 // the stage read last
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) to_unit[nt][0] = to_unit[nt][1] = kNoUnit;

    for (int u = u0; u < u1; ++u) {
      const int kb = u * kUnitKeys + warp * kKeys;
      if (kb >= most) break;
      copy_wait();
      __syncwarp();  // this stage is there, and the other one was read by every lane
      ahead.copy(a, stage ^ 1, warp, lane, r0, ROWS);
      last = stage;
      const float4 scale = *reinterpret_cast<const float4*>(s_scales[warp][stage][0]);  // halves: keys, values
      const uint8_t *kp = k_lane + stage * kStage, *vp = v_lane + stage * kStage;
      stage ^= 1;

      float s[2][NT][4] = {};
      uint4 k[2][4];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        k[half][0] = codes(kp + half * kHalf);
        k[half][1] = codes(kp + half * kHalf + k_more);
        k[half][2] = codes(kp + half * kHalf + 8 * D);
        k[half][3] = codes(kp + half * kHalf + 8 * D + k_more);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t q[NT][2];
        if constexpr (NT == 1) {
          q[0][0] = qf[0][j][0];
          q[0][1] = qf[0][j][1];
        } else {
          const uint4 v = *reinterpret_cast<const uint4*>(s_q[j][lane]);
          q[0][0] = v.x;
          q[0][1] = v.y;
          q[NT - 1][0] = v.z;
          q[NT - 1][1] = v.w;
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t lo = biased<FP8>(word(k[half][j / 4], j & 3)), hi = biased<FP8>(word(k[half][2 + j / 4], j & 3));
          const uint32_t a0 = widen<FP8, false>(lo), a2 = widen<FP8, true>(lo);
          const uint32_t a1 = widen<FP8, false>(hi), a3 = widen<FP8, true>(hi);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816(s[half][nt], a0, a1, a2, a3, q[nt][0], q[nt][1]);
        }
      }

      // scores under the running maximum, which moves when one passes it by kLazy, and to a first one
      bool raise = none != 0;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float ks = half ? scale.z : scale.x;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float f[2] = {factor[nt][0] * ks, factor[nt][1] * ks};
#pragma unroll
          for (int c = 0; c < 4; ++c) s[half][nt][c] = fmaf(s[half][nt][c], f[c & 1], -m[nt][c & 1]);
        }
      }
      if (kb + kKeys > least) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (kb + half * 16 + g + (c >> 1) * 8 >= limit[nt][c & 1]) s[half][nt][c] = -INFINITY;
      }
      const float vlog[2] = {log2_of(scale.y), log2_of(scale.w)};
      float up[2][NT][2];
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            up[half][nt][c] = fmaxf(s[half][nt][c], s[half][nt][c + 2]);
            raise |= fmaxf(up[half][nt][c], up[half][nt][c] + (vlog[half] + to_unit[nt][c])) > kLazy;
          }
      if (__any_sync(~0u, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float alpha[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float by = fmaxf(up[0][nt][c], up[1][nt][c]);
            float most_v = fmaxf(up[0][nt][c] + vlog[0], up[1][nt][c] + vlog[1]);
#pragma unroll
            for (int off = 4; off < 32; off *= 2) {
              by = fmaxf(by, __shfl_xor_sync(~0u, by, off));
              most_v = fmaxf(most_v, __shfl_xor_sync(~0u, most_v, off));
            }
            const int bit = 1 << (nt * 2 + c);
            if (none & bit ? by > -INFINITY : by > 0.f) {
              if (!(none & bit)) l[nt][c] *= fast_exp2(-by);
              none &= ~bit;
              m[nt][c] += by;
              to_unit[nt][c] += by;
              most_v -= by;
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                s[half][nt][c] -= by;
                s[half][nt][c + 2] -= by;
              }
            }
            alpha[c] = 1.f;
            if (most_v > -INFINITY && most_v + to_unit[nt][c] > 0.f) {  // the unit becomes the largest product
              alpha[c] = fast_exp2(-most_v - to_unit[nt][c]);
              to_unit[nt][c] = -most_v;
            }
          }
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {
            o[nt][mt][0] *= alpha[0];
            o[nt][mt][1] *= alpha[1];
            o[nt][mt][2] *= alpha[0];
            o[nt][mt][3] *= alpha[1];
          }
        }
      }

#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t pb[NT][2];
        const bool poisoned = vlog[half] != vlog[half];  // a block whose value scale is NaN
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float p[4], ratio[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) ratio[c] = fast_exp2(min_nan(vlog[half] + to_unit[nt][c], kMostRatio));
#pragma unroll
          for (int c = 0; c < 4; ++c) p[c] = fast_exp2(s[half][nt][c]);
          l[nt][0] += p[0] + p[2];
          l[nt][1] += p[1] + p[3];
#pragma unroll
          for (int c = 0; c < 4; ++c) p[c] *= ratio[c & 1];
          if (poisoned) {  // not for the rows that do not see it
#pragma unroll
            for (int c = 0; c < 4; ++c) p[c] = s[half][nt][c] == -INFINITY ? 0.f : NAN;
          }
          pb[nt][0] = transpose8x8(pack_f16x2(p[0], p[1]));
          pb[nt][1] = transpose8x8(pack_f16x2(p[2], p[3]));
        }
        const uint4 v0 = codes(vp + half * kHalf), v1 = codes(vp + half * kHalf + D), v2 = codes(vp + half * kHalf + 8 * D),
                    v3 = codes(vp + half * kHalf + 9 * D);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t w0 = biased<FP8>(word(v0, j)), w1 = biased<FP8>(word(v1, j)), w2 = biased<FP8>(word(v2, j)),
                         w3 = biased<FP8>(word(v3, j));
#pragma unroll
          for (int two = 0; two < 2; ++two) {  // two of the word's four dims
            const uint32_t lo = __byte_perm(w0, w1, two ? 0x7362 : 0x5140), hi = __byte_perm(w2, w3, two ? 0x7362 : 0x5140);
            const uint32_t a0 = widen<FP8, false>(lo), a1 = widen<FP8, true>(lo);
            const uint32_t a2 = widen<FP8, false>(hi), a3 = widen<FP8, true>(hi);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][2 * j + two], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
          }
        }
      }
    }

    // the warps' parts, each in the stage that its warp read last: this lane has dims 16 g + 2 mt (+ 1) of
    // rows 2 tg and 2 tg + 1 of each 8
    __syncwarp();
    float* mine = reinterpret_cast<float*>(ahead.ring + max(last, 0) * kStage);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float sum = l[nt][c];
        sum += __shfl_xor_sync(~0u, sum, 4);
        sum += __shfl_xor_sync(~0u, sum, 8);
        sum += __shfl_xor_sync(~0u, sum, 16);
        const int r = nt * 8 + 2 * tg + c;
        if (r < rows && last >= 0) {
          if (g == 0) {
            s_m[warp][r] = none >> (nt * 2 + c) & 1 ? -INFINITY : m[nt][c];
            s_l[warp][r] = sum;
          }
          const float unit = fast_exp2(-to_unit[nt][c]);
          float4* to = reinterpret_cast<float4*>(mine + r * D + g * 16);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            to[k] = make_float4(o[nt][2 * k][c] * unit, o[nt][2 * k][c + 2] * unit, o[nt][2 * k + 1][c] * unit,
                                o[nt][2 * k + 1][c + 2] * unit);
        }
      }
    if (lane == 0) s_part[warp] = last < 0 ? -1 : (warp * kStages + last) * kStage;
    __syncthreads();
    const bool whole = u0 == 0 && u1 == walk.nu;
    // the part of a pair that starts here but ends elsewhere has the worker's second place
    float* part = a.part + (long)(slot + (u0 == 0 ? 1 : 0)) * ROWS * kPart;
    int from[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) from[w] = s_part[w];
#pragma unroll 2
    for (int idx = threadIdx.x; idx < rows * (D / 4); idx += kThreads) {  // a thread has four dims of a row
      const int r = idx / (D / 4), d = idx % (D / 4) * 4;
      const int t = row_t + (r0 + r) / a.G, hq = h * a.G + (r0 + r) % a.G;
      uint2 gate = make_uint2(0, 0);
      if (whole && a.gate != nullptr) gate = *reinterpret_cast<const uint2*>(a.gate + t * a.g_st + hq * a.g_sh + d);
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        if (from[w] >= 0) top = fmaxf(top, s_m[w][r]);
      const float ref = top == -INFINITY ? 0.f : top;
      float sum = 0.f, out[4] = {};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (from[w] >= 0) {
          const float f = fast_exp2(s_m[w][r] - ref);
          const float4 v = *reinterpret_cast<const float4*>(s_ring + from[w] + (r * D + d) * 4);
          sum += s_l[w][r] * f;
          out[0] = fmaf(v.x, f, out[0]);
          out[1] = fmaf(v.y, f, out[1]);
          out[2] = fmaf(v.z, f, out[2]);
          out[3] = fmaf(v.w, f, out[3]);
        }
      }
      if (whole) {
        write_row(a, t, hq, d, out, sum, gate);
      } else {
        *reinterpret_cast<float4*>(part + r * kPart + d) = make_float4(out[0], out[1], out[2], out[3]);
        if (d == 0) *reinterpret_cast<float2*>(part + r * kPart + D) = make_float2(top, sum);
      }
    }
    __syncthreads();
  }
}

// Joins the parts of the pairs that span workers. Up to kFew parts: the worker in whose range the pair
// ends has them all, a thread four dims of a row. More (a long context and few pairs): each of
// the pair's workers takes every so many-th row, and its warps share the row's parts.
template <int NT>
struct Join {
  static constexpr int ROWS = 8 * NT, kFew = 8, JW = kJoin / 32;
  const AttnArgs& a;
  long per;
  int base, r0;  // the tile's first place in the workspace, its first row
  int h, first, parts, rows, row_t;

  __device__ __forceinline__ const float* part(int w, int r) const {  // the first worker may start with the pair or before
    return a.part + ((long)(base + 2 * (first + w) + (w == 0 ? 1 : 0)) * ROWS + r) * kPart;
  }
  // parts w0, w0 + step, ... of row r, four dims from d on, added under a common maximum
  template <int N>
  __device__ __forceinline__ void add(int r, int d, int w0, int step, float& top, float& sum, float (&out)[4]) const {
    float4 v[N];
    float2 ml[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      ml[k] = make_float2(-INFINITY, 0.f);
      if (w0 + k * step < parts) {
        const float* p = part(w0 + k * step, r);
        v[k] = *reinterpret_cast<const float4*>(p + d);
        ml[k] = *reinterpret_cast<const float2*>(p + D);
      }
    }
    float now = top;
#pragma unroll
    for (int k = 0; k < N; ++k) now = fmaxf(now, ml[k].x);
    const float ref = now == -INFINITY ? 0.f : now, old = fast_exp2(top - ref);
    sum *= old;
#pragma unroll
    for (int c = 0; c < 4; ++c) out[c] *= old;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float f = fast_exp2(ml[k].x - ref);
      sum = fmaf(ml[k].y, f, sum);
      out[0] = fmaf(v[k].x, f, out[0]);
      out[1] = fmaf(v[k].y, f, out[1]);
      out[2] = fmaf(v[k].z, f, out[2]);
      out[3] = fmaf(v[k].w, f, out[3]);
    }
    top = now;
  }
  __device__ __forceinline__ void write(int r, int d, const float (&o)[4], float l) const {
    const int t = row_t + (r0 + r) / a.G, hq = h * a.G + (r0 + r) % a.G;
    uint2 gate = make_uint2(0, 0);
    if (a.gate != nullptr) gate = *reinterpret_cast<const uint2*>(a.gate + t * a.g_st + hq * a.g_sh + d);
    write_row(a, t, hq, d, o, l, gate);
  }
  // the pair at position x, for this worker
  __device__ __forceinline__ void pair(const Found& at, long x, int worker) {
    const int cost = at.c1 - at.c0;
    h = (int)((uint32_t)(x - (long)at.c0 * a.Hkv) / (uint32_t)cost);
    const long begin = (long)at.c0 * a.Hkv + (long)h * cost;
    first = (int)((begin + kPairCost) / per);
    const int last = (int)((begin + cost - 1) / per);
    parts = last - first + 1;
    if (parts == 1 || worker < first || (parts <= kFew && worker != last)) return;
    row_t = at.row_t;
    rows = min(at.n * a.G - r0, ROWS);
    if (parts <= kFew) {
      for (int idx = threadIdx.x; idx < rows * (D / 4); idx += kJoin) {
        const int r = idx / (D / 4), d = idx % (D / 4) * 4;
        float top = -INFINITY, sum = 0.f, out[4] = {};
        add<kFew>(r, d, 0, 1, top, sum, out);
        write(r, d, out, sum);
      }
      return;
    }
    __shared__ __align__(16) float s_out[JW][D];
    __shared__ float s_ml[JW][2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int r = worker - first; r < rows; r += parts) {
      float top = -INFINITY, sum = 0.f, out[4] = {};
      for (int w0 = warp; w0 < parts; w0 += 4 * JW) add<4>(r, lane * 4, w0, JW, top, sum, out);
      *reinterpret_cast<float4*>(&s_out[warp][lane * 4]) = make_float4(out[0], out[1], out[2], out[3]);
      if (lane == 0) {
        s_ml[warp][0] = top;
        s_ml[warp][1] = sum;
      }
      __syncthreads();
      if (warp == 0) {
        float most = -INFINITY, l = 0.f, o[4] = {};
#pragma unroll
        for (int w = 0; w < JW; ++w) most = fmaxf(most, s_ml[w][0]);
        const float ref = most == -INFINITY ? 0.f : most;
#pragma unroll
        for (int w = 0; w < JW; ++w) {
          const float f = fast_exp2(s_ml[w][0] - ref);
          const float4 v = *reinterpret_cast<const float4*>(&s_out[w][lane * 4]);
          l += s_ml[w][1] * f;
          o[0] = fmaf(v.x, f, o[0]);
          o[1] = fmaf(v.y, f, o[1]);
          o[2] = fmaf(v.z, f, o[2]);
          o[3] = fmaf(v.w, f, o[3]);
        }
        write(r, lane * 4, o, l);
      }
      __syncthreads();
    }
  }
};

template <int NT>
__global__ void __launch_bounds__(kJoin) paged_attention_join_kernel(const AttnArgs a) {
  const Found mine = request_of(a, threadIdx.x);
  const Place place = place_of<8 * NT>(a, mine);
  const int worker = place.worker;
  const long total = (long)a.cu_units[a.R] * a.Hkv, per = (total + place.workers - 1) / place.workers;
  const long x = per * worker, x_end = min(total, x + per);
  const bool some = x < x_end && !place.none && place.workers > 1;  // one worker's pairs are whole
  Found at{}, end{};
  if (some) {  // the pairs at both ends of the range; those between are whole
    at = find_request(a, x, mine);
    end = find_request(a, x_end - 1, mine);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the parts are written; in every CTA, so this grid ends last
  if (!some) return;
  Join<NT> join{a, per};
  join.base = place.tile * place.workers * 2;
  join.r0 = place.tile * Join<NT>::ROWS;
  join.pair(at, x, worker);
  const int cost = at.c1 - at.c0;
  const long in = x - (long)at.c0 * a.Hkv;
  if (in / cost != (x_end - 1 - (long)at.c0 * a.Hkv) / cost || end.i != at.i) join.pair(end, x_end - 1, worker);
}

template <bool FP8, int NT>
void launch(AttnArgs a, int max_rows, const at::TensorOptions& opts) {
  constexpr int ROWS = 8 * NT, smem = kWarps * kStages * kStage;
  const int tiles = (max_rows + ROWS - 1) / ROWS;
  C10_CUDA_CHECK(ensure_dynamic_smem((const void*)paged_attention_kernel<FP8, NT>, smem));
  // up to kFewTiles tiles: each is cut among as many CTAs as fit the SMs. More (a request with many new tokens, or a step
  // that does not say how many one may have): four waves of CTAs among the tiles that the step turns out to have, at
  // least one a tile. The workspace is under 32 MB either way.
  const int resident = device_sm_count() * 3;
  a.split = tiles <= kFewTiles ? 0 : kFewTiles * resident;
  const at::Tensor part = at::empty({2L * (a.split ? a.split : resident * tiles) * ROWS * kPart}, opts.dtype(at::kFloat));
  a.part = part.data_ptr<float>();
  const dim3 grid = a.split ? dim3(std::max(a.split, tiles)) : dim3(resident, tiles);
  launch_early(paged_attention_kernel<FP8, NT>, grid, kThreads, smem, a);
  launch_early(paged_attention_join_kernel<NT>, grid, kJoin, 0, a);
}

template <bool FP8>
void launch_rows(const AttnArgs& a, int max_rows, const at::TensorOptions& opts) {
  if (max_rows <= 8)
    launch<FP8, 1>(a, max_rows, opts);
  else
    launch<FP8, 2>(a, max_rows, opts);
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
           (t.numel() == 0 || t.stride(2) == 1) && (t.size(0) <= 1 || t.stride(0) % 8 == 0) &&
           (t.size(1) <= 1 || t.stride(1) % 8 == 0) &&
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
  // a request's new tokens fit its table
  const int64_t max_rows = std::min<int64_t>({max_new, T, tables.size(1) * s}) * a.G;
  TORCH_CHECK(max_rows < (1LL << 30), "paged_attention: too many query rows of a request for one call");
  TORCH_CHECK((tables.size(1) * s / kUnitKeys + kPairCost + 1) * H < (1LL << 31), "paged_attention: tables too wide");
  if (keys.scalar_type() == at::kFloat8_e4m3fn)
    launch_rows<true>(a, (int)std::max<int64_t>(max_rows, 1), query.options());
  else
    launch_rows<false>(a, (int)std::max<int64_t>(max_rows, 1), query.options());
  return out;
}

}  // namespace hrm
