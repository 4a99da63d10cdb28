// The 8-bit paged KV cache: quantising new tokens into their blocks, and reading tokens back.
//
// One layer's cache is, for keys and for values, codes [num_blocks, H, s, 128] (int8 or e4m3)
// and scales [num_blocks, H] fp32: a (block, head) holds s tokens whose values are code * scale,
// so a head's tokens of one block are s * 128 consecutive bytes.
//
// Append. The new tokens of one block are consecutive (a "run" of paged_tables.cu). With S the
// scale so far (0 for a block that was empty) and q the largest code (127, 448):
//   S' = max(S, amax(new) * (1/q)),  code = round(x * (1/S')),
// and where S' > S the block's older codes are rounded again, code' = round(code * (S * (1/S'))).
// A block's scale only grows while it fills, so an older value is rounded again only when a
// larger one arrives. 1/q and 1/S' are correctly rounded fp32 and every product rounds once.
// A block that gets an infinity or a NaN gets the scale NaN and codes 0: attention over it
// is NaN, as over the tokens themselves, but its codes stay finite, so that rows of a reused block
// that its new owner has not written yet contribute exact zeros when they are masked.
// Scales of non-zero tokens are at least 2^-100: 1/S' is finite, and ratios of two scales are.
//
// One CTA takes the keys and the values of one (run, head): 16 lanes hold a row of 128
// values as 16-byte loads, the run stays in registers between the maximum and the rounding, so
// tokens are read once and codes written once. Bound by memory for prompts: 14800 tokens of 12
// heads, e4m3, 91 MB read and 45 MB written, 21 us (int8 26; with keys and values in CTAs of their own 26 % more); by launch and load
// latency for a decode step: 33 tokens of 10 heads 4.1 us.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp8.h>
#include <torch/types.h>

#include "common.cuh"
#include "launch_early.h"

namespace hrm {
namespace {

constexpr int D = 128;

template <bool FP8>
struct Code {
  static constexpr float kMax = FP8 ? 448.f : 127.f;
};

__device__ __forceinline__ void unpack8(const uint4& w, float (&v)[8]) {
  const float2 a = unpack_bf16x2(w.x), b = unpack_bf16x2(w.y), c = unpack_bf16x2(w.z), d = unpack_bf16x2(w.w);
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
}

// 8 values, already divided by the scale, to 8 codes (round to nearest even, saturating)
template <bool FP8>
__device__ __forceinline__ uint2 to_codes(const float (&x)[8]) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (FP8) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * h], x[4 * h + 1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * h + 2], x[4 * h + 3]), __NV_SATFINITE, __NV_E4M3);
      w[h] = lo | hi << 16;
    } else {
      w[h] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = max(-127, min(127, __float2int_rn(x[4 * h + i])));
        w[h] |= (uint32_t)(c & 0xff) << (8 * i);
      }
    }
  }
  return make_uint2(w[0], w[1]);
}

template <bool FP8>
__device__ __forceinline__ void from_codes(const uint2& w, float (&x)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t v = h ? w.y : w.x;
    if constexpr (FP8) {
      const float2 a = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(v & 0xffff), __NV_E4M3)));
      const float2 b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(v >> 16), __NV_E4M3)));
      x[4 * h] = a.x; x[4 * h + 1] = a.y; x[4 * h + 2] = b.x; x[4 * h + 3] = b.y;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * h + i] = (float)(int8_t)(v >> (8 * i));
    }
  }
}

struct AppendArgs {
  const __nv_bfloat16* x[2];  // keys, values: rows of H * 128
  long x_st[2], x_sh[2];
  uint8_t* codes[2];
  float* scales[2];
  const int4* runs;
  const int* num_runs;
  int H, size, T, num_blocks;
};

template <bool FP8, int THREADS, int ROWS>  // ROWS: rows of a run that a thread holds, size * 16 / THREADS
__global__ void __launch_bounds__(THREADS) paged_append_kernel(const AppendArgs a) {
  constexpr int kRowsAtOnce = THREADS / 16, kWarps = THREADS / 32;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 run = a.runs[blockIdx.x];  // block, first offset, tokens, first row
  if ((int)blockIdx.x >= a.num_runs[0]) return;
  const int h = blockIdx.y;
  const int lane = threadIdx.x & 15, row0 = threadIdx.x >> 4;
  // a plan of another cache or another number of rows: nothing outside the tensors is touched
  if (run.x < 0 || run.x >= a.num_blocks || run.w < 0 || run.w + run.z > a.T || run.y + run.z > a.size) return;

  const long bh = (long)run.x * a.H + h;
  uint4 held[2][ROWS];
  float before[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const long st = c ? a.x_st[1] : a.x_st[0];
    const __nv_bfloat16* x = (c ? a.x[1] : a.x[0]) + run.w * st + h * (c ? a.x_sh[1] : a.x_sh[0]) + lane * 8;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int r = row0 + i * kRowsAtOnce;
      held[c][i] = r < run.z ? *reinterpret_cast<const uint4*>(x + r * st) : make_uint4(0, 0, 0, 0);
    }
    before[c] = run.y > 0 ? (c ? a.scales[1] : a.scales[0])[bh] : 0.f;
  }
  __shared__ uint32_t s_top[2][kWarps];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t top = 0;  // bf16 magnitudes order as integers; at least 0x7f80 is not finite
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const uint4 v = held[c][i];
      top = __vmaxu2(top, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu),
                                   __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
    }
    top = max(top & 0xffffu, top >> 16);
    top = __reduce_max_sync(~0u, top);
    if ((threadIdx.x & 31) == 0) s_top[c][threadIdx.x >> 5] = top;
  }
  __syncthreads();  // also: every thread has read the scales
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t top = s_top[c][0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) top = max(top, s_top[c][w]);
    const bool finite = top < 0x7f80u && before[c] == before[c];
    float now = __uint_as_float(top << 16) * (1.f / Code<FP8>::kMax);
    if (top > 0) now = fmaxf(now, 0x1p-100f);
    now = finite ? fmaxf(now, before[c]) : __int_as_float(0x7fc00000);
    const float inv = now > 0.f ? __frcp_rn(now) : 0.f;
    uint8_t* codes = (c ? a.codes[1] : a.codes[0]) + bh * a.size * D + lane * 8;
    if (threadIdx.x == 0) (c ? a.scales[1] : a.scales[0])[bh] = now;

    if (finite && before[c] > 0.f && now != before[c]) {  // the block's older tokens, to the wider range
      const float ratio = before[c] * inv;
      for (int r = row0; r < run.y; r += kRowsAtOnce) {
        uint2* p = reinterpret_cast<uint2*>(codes + r * D);
        float v[8];
        from_codes<FP8>(*p, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= ratio;
        *p = to_codes<FP8>(v);
      }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int r = row0 + i * kRowsAtOnce;
      if (r < run.z) {
        uint2 out = make_uint2(0, 0);
        if (finite) {
          float v[8];
          unpack8(held[c][i], v);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] *= inv;
          out = to_codes<FP8>(v);
        }
        *reinterpret_cast<uint2*>(codes + (run.y + r) * D) = out;
      }
    }
  }
}

// Tokens back as bf16: 16 threads a slot and kReadHeads heads, keys and values; slot -1 (or one outside
// the cache) gives zeros. 14800 tokens of 12 heads, 136 MB: 20 us (27 us with one head a thread).
constexpr int kReadHeads = 4;
template <bool FP8>
__global__ void __launch_bounds__(128)
    paged_read_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc, const float* __restrict__ ks,
                      const float* __restrict__ vs, const int* __restrict__ slots, int N, int H, int size_log2,
                      int num_blocks, __nv_bfloat16* __restrict__ keys, __nv_bfloat16* __restrict__ values) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 15, n = blockIdx.x * 8 + (threadIdx.x >> 4), h0 = blockIdx.y * kReadHeads;
  if (n >= N) return;
  const int slot = slots[n], block = slot >> size_log2;
  const bool held = slot >= 0 && block < num_blocks;
  uint2 w[kReadHeads][2];
  float s[kReadHeads][2];
#pragma unroll
  for (int i = 0; i < kReadHeads; ++i) {
    w[i][0] = w[i][1] = make_uint2(0, 0);
    s[i][0] = s[i][1] = 0.f;
    if (held && h0 + i < H) {
      const long bh = (long)block * H + h0 + i;
      const long at = ((bh << size_log2) + (slot & ((1 << size_log2) - 1))) * D + lane * 8;
      w[i][0] = *reinterpret_cast<const uint2*>(kc + at);
      w[i][1] = *reinterpret_cast<const uint2*>(vc + at);
      s[i][0] = ks[bh];
      s[i][1] = vs[bh];
    }
  }
#pragma unroll
  for (int i = 0; i < kReadHeads; ++i) {
    if (h0 + i >= H) break;
    const long to = ((long)n * H + h0 + i) * 16 + lane;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float v[8];
      from_codes<FP8>(w[i][c], v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= s[i][c];
      reinterpret_cast<uint4*>(c ? values : keys)[to] = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                                                  pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    }
  }
}

// Checks one layer's cache; returns true for e4m3 codes.
bool check_cache(const at::Tensor& keys, const at::Tensor& values, const at::Tensor& key_scales,
                 const at::Tensor& value_scales) {
  TORCH_CHECK(keys.is_cuda() && keys.dim() == 4 && keys.size(3) == D && keys.is_contiguous() &&
                  (keys.scalar_type() == at::kChar || keys.scalar_type() == at::kFloat8_e4m3fn),
              "cache: contiguous CUDA codes [blocks, heads, block size, 128], int8 or float8_e4m3fn");
  TORCH_CHECK(values.sizes() == keys.sizes() && values.scalar_type() == keys.scalar_type() && values.is_contiguous() &&
                  values.device() == keys.device(),
              "cache: keys and values of one shape and type");
  const int64_t s = keys.size(2);
  TORCH_CHECK(s == 16 || s == 32 || s == 64 || s == 128, "block size must be 16, 32, 64 or 128");
  for (const at::Tensor* t : {&key_scales, &value_scales})
    TORCH_CHECK(t->dim() == 2 && t->size(0) == keys.size(0) && t->size(1) == keys.size(1) && t->is_contiguous() &&
                    t->scalar_type() == at::kFloat && t->device() == keys.device(),
                "cache: fp32 scales [blocks, heads]");
  TORCH_CHECK(keys.size(0) * s < (1LL << 31), "cache: slots are int32");
  return keys.scalar_type() == at::kFloat8_e4m3fn;
}

template <bool FP8>
void launch_append(const AppendArgs& a, dim3 grid) {
  // 4 to 8 rows a thread: enough loads in flight, and registers for several CTAs an SM
  switch (a.size) {
    case 16: return launch_early(paged_append_kernel<FP8, 128, 2>, grid, 128, 0, a);
    case 32: return launch_early(paged_append_kernel<FP8, 128, 4>, grid, 128, 0, a);
    case 64: return launch_early(paged_append_kernel<FP8, 256, 4>, grid, 256, 0, a);
    default: return launch_early(paged_append_kernel<FP8, 256, 8>, grid, 256, 0, a);
  }
}

}  // namespace

// key, value [T, H, 128] bf16 (any row and head strides of whole 16 bytes) into the blocks of the
// step that made `runs` and `meta` (whose last element is the number of runs).
void paged_append(const at::Tensor& key, const at::Tensor& value, const at::Tensor& keys, const at::Tensor& values,
                  const at::Tensor& key_scales, const at::Tensor& value_scales, const at::Tensor& runs,
                  const at::Tensor& meta) {
  const bool fp8 = check_cache(keys, values, key_scales, value_scales);
  const int64_t H = keys.size(1), T = key.size(0);
  for (const at::Tensor* t : {&key, &value})
    TORCH_CHECK(t->device() == keys.device() && t->scalar_type() == at::kBFloat16 && t->dim() == 3 && t->size(0) == T &&
                    t->size(1) == H && t->size(2) == D && (t->numel() == 0 || t->stride(2) == 1) &&
                    (T <= 1 || t->stride(0) % 8 == 0) && (H <= 1 || t->stride(1) % 8 == 0) &&
                    reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                "paged_append: key and value [T, heads, 128] bf16 on the cache's device, with 16-byte aligned rows");
  TORCH_CHECK(runs.device() == keys.device() && runs.scalar_type() == at::kInt && runs.dim() == 2 && runs.size(1) == 4 &&
                  runs.is_contiguous() && meta.device() == keys.device() && meta.scalar_type() == at::kInt &&
                  meta.is_contiguous() && meta.numel() >= 6,
              "paged_append: the step's runs");
  TORCH_CHECK(H <= 65535, "paged_append: too many heads");
  if (runs.size(0) == 0 || T == 0) return;
  c10::cuda::CUDAGuard guard(keys.device());
  AppendArgs a{};
  const at::Tensor* x[2] = {&key, &value};
  const at::Tensor* c[2] = {&keys, &values};
  const at::Tensor* s[2] = {&key_scales, &value_scales};
  for (int i = 0; i < 2; ++i) {
    a.x[i] = reinterpret_cast<const __nv_bfloat16*>(x[i]->data_ptr());
    a.x_st[i] = x[i]->stride(0);
    a.x_sh[i] = x[i]->stride(1);
    a.codes[i] = reinterpret_cast<uint8_t*>(c[i]->data_ptr());
    a.scales[i] = s[i]->data_ptr<float>();
  }
  a.runs = reinterpret_cast<const int4*>(runs.data_ptr<int>());
  a.num_runs = meta.data_ptr<int>() + meta.numel() - 1;
  a.H = (int)H;
  a.size = (int)keys.size(2);
  a.T = (int)T;
  a.num_blocks = (int)keys.size(0);
  const dim3 grid((unsigned)runs.size(0), (unsigned)H);
  if (fp8)
    launch_append<true>(a, grid);
  else
    launch_append<false>(a, grid);
}

// slots [N] int32 -> keys, values [N, H, 128] bf16.
std::tuple<at::Tensor, at::Tensor> paged_read(const at::Tensor& keys, const at::Tensor& values, const at::Tensor& key_scales,
                                              const at::Tensor& value_scales, const at::Tensor& slots) {
  const bool fp8 = check_cache(keys, values, key_scales, value_scales);
  const int64_t N = slots.numel(), H = keys.size(1);
  TORCH_CHECK(slots.device() == keys.device() && slots.scalar_type() == at::kInt && slots.is_contiguous(),
              "paged_read: contiguous int32 slots on the cache's device");
  Outputs make(key_scales.options());
  make.plan({N, H, D}, at::kBFloat16).plan({N, H, D}, at::kBFloat16);
  const at::Tensor out_keys = make.next({N, H, D}, at::kBFloat16), out_values = make.next({N, H, D}, at::kBFloat16);
  if (N == 0) return {out_keys, out_values};
  c10::cuda::CUDAGuard guard(keys.device());
  int size_log2 = 4;
  while ((1 << size_log2) < keys.size(2)) ++size_log2;
  TORCH_CHECK(N < (1LL << 31) - 8 && H <= 65535LL * kReadHeads, "paged_read: too many slots or heads");
  const dim3 grid((unsigned)((N + 7) / 8), (unsigned)((H + kReadHeads - 1) / kReadHeads));
  const auto* kc = reinterpret_cast<const uint8_t*>(keys.data_ptr());
  const auto* vc = reinterpret_cast<const uint8_t*>(values.data_ptr());
  auto* ok = reinterpret_cast<__nv_bfloat16*>(out_keys.data_ptr());
  auto* ov = reinterpret_cast<__nv_bfloat16*>(out_values.data_ptr());
  launch_early(fp8 ? paged_read_kernel<true> : paged_read_kernel<false>, grid, 128, 0, kc, vc, key_scales.data_ptr<float>(),
               value_scales.data_ptr<float>(), slots.data_ptr<int>(), (int)N, (int)H, size_log2, (int)keys.size(0), ok, ov);
  return {out_keys, out_values};
}

}  // namespace hrm
