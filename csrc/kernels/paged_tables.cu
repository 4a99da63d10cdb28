// Block tables and slot maps of a paged KV cache, built on the device from request lengths.
//
// State (device): tables [R, MB] int32 (block ids, -1 where none), lengths [R] cached tokens,
// free [num_blocks] a stack of block ids whose first num_free[0] entries are free.
//
//   step(new)       have_i = ceil(L_i / s), need_i = ceil((L_i + n_i) / s) - have_i,
//                   rank_i = sum of need over the requests before i; the j-th new block of
//                   request i is free[num_free - 1 - (rank_i + j)]. Packed row t of request i at
//                   position p gets slot tables[i, p / s] * s + p % s. All or nothing: when a
//                   request or the pool cannot hold its tokens, nothing changes, the step is
//                   empty and status[0] says why.
//   truncate(keep)  L_i = min(L_i, keep_i); surplus blocks go back in the reverse order of
//                   ranks, so a truncate to the lengths before a step undoes that step exactly.
//
// The state may have been restored or changed from outside: lengths outside the table and counts outside the stack
// are a failure of either call, which then changes nothing; block ids are checked where the cache is read.
//
// Both are one launch and read no host value, so a captured decode step crosses block
// boundaries by itself. Every CTA computes the prefix sums over the requests for itself (a few
// loads a thread, in L2) instead of waiting for another kernel or CTA; the rows are spread over
// the CTAs and find their request by binary search in shared memory. The CTA that finishes last
// (a counter that it puts back to zero) moves lengths and num_free, after every CTA has read
// them. These calls are bound by launch and dependent-load latency, not by bytes: a truncate and a
// decode step of 25 requests take 8 us together, a truncate and the step of 512 prompts of half a million tokens
// 11 us (15 us with one row a thread; 8 CTAs an SM instead of 2 were 2.5 us slower, the prefix sums again in
// each).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/types.h>

#include "common.cuh"
#include "device_setup.h"
#include "launch_early.h"
#include "paged.h"

namespace hrm {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kRows = 4;            // rows of a step that a thread takes together
constexpr int kMaxRequests = 8192;  // three prefix arrays of this many int32 in shared memory

// status codes; the Python side names them
enum StepStatus : int { kStepOk = 0, kStepPool = 1, kStepRows = 2, kStepLong = 3, kStepNegative = 4, kStepMaxNew = 5, kStepState = 6 };

struct Sums {
  long long a, b, c, d;
};

// Exclusive prefix of `v` over the CTA's threads; `total` is the sum over all of them.
__device__ Sums block_exclusive(Sums v, Sums& total) {
  __shared__ Sums warp_sum[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Sums inc = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long a = __shfl_up_sync(~0u, inc.a, off), b = __shfl_up_sync(~0u, inc.b, off);
    const long long c = __shfl_up_sync(~0u, inc.c, off), d = __shfl_up_sync(~0u, inc.d, off);
    if (lane >= off) {
      inc.a += a;
      inc.b += b;
      inc.c += c;
      inc.d += d;
    }
  }
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  Sums base{0, 0, 0, 0};
  total = base;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const Sums s = warp_sum[w];
    if (w < warp) {
      base.a += s.a;
      base.b += s.b;
      base.c += s.c;
      base.d += s.d;
    }
    total.a += s.a;
    total.b += s.b;
    total.c += s.c;
    total.d += s.d;
  }
  __syncthreads();
  return Sums{base.a + inc.a - v.a, base.b + inc.b - v.b, base.c + inc.c - v.c, base.d + inc.d - v.d};
}

// True in every thread of the CTA that arrives last of `gridDim.x`; puts the counter back to 0.
__device__ bool last_cta(int* done) {
  __shared__ int is_last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    is_last = atomicAdd(done, 1) == (int)gridDim.x - 1;
    if (is_last) *done = 0;
  }
  __syncthreads();
  return is_last != 0;
}

struct StepArgs {
  int* tables;
  long table_ld;
  int* lengths;
  const int* fresh;  // new tokens of each request
  const int* free_stack;
  int* num_free;
  int* status;  // [code, request]
  int* done;
  int R, MB, F, size_log2, rows, max_new, max_runs;  // F: places of the stack
  int* slots;
  int* positions;
  int* cu_new;
  int* kv_lengths;
  int* cu_units;
  int4* runs;
  int* num_runs;
};

__global__ void __launch_bounds__(kThreads) paged_step_kernel(const StepArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ int sm[];
  int* s_cu = sm;              // [R + 1] first packed row of each request
  int* s_rank = s_cu + a.R + 1;  // [R] rank of its first new block
  int* s_run = s_rank + a.R;   // [R] its first run
  const int size = 1 << a.size_log2, tid = threadIdx.x;
  const int per = (a.R + kThreads - 1) / kThreads, i0 = min(a.R, tid * per), i1 = min(a.R, i0 + per);
  const int free_top = a.num_free[0];
  const auto blocks = [&](long long n) { return (n + size - 1) >> a.size_log2; };

  Sums mine{0, 0, 0, 0}, total;
  int bad = kStepOk, bad_at = 0;
  for (int i = i0; i < i1; ++i) {
    const long long len = a.lengths[i], n = a.fresh[i];
    const long long most = (long long)a.MB << a.size_log2;
    const int code = len < 0 || len > most ? kStepState
                     : n < 0               ? kStepNegative
                     : n > a.max_new       ? kStepMaxNew
                     : len + n > most      ? kStepLong
                                           : kStepOk;
    if (code != kStepOk && bad == kStepOk) {
      bad = code;
      bad_at = i;
    }
    if (n > 0) {
      mine.a += n;
      mine.b += blocks(len + n) - blocks(len);
      mine.c += blocks(len + n) - (len >> a.size_log2);
      mine.d += (len + n + kUnitKeys - 1) / kUnitKeys + kPairCost;
    }
  }
  const Sums first = block_exclusive(mine, total);
  // the same verdict in every CTA: a request's own fault before the whole step's
  __shared__ int s_bad, s_bad_at;
  if (tid == 0) {
    s_bad = free_top < 0 || free_top > a.F ? kStepState : total.a > a.rows ? kStepRows : total.b > free_top ? kStepPool : kStepOk;
    s_bad_at = -1;
  }
  __syncthreads();
  if (bad != kStepOk) atomicMax(&s_bad_at, a.R - 1 - bad_at);  // the lowest request
  __syncthreads();
  if (bad != kStepOk && s_bad_at == a.R - 1 - bad_at) s_bad = bad;
  __syncthreads();
  const int failed = s_bad, failed_at = s_bad_at < 0 ? -1 : a.R - 1 - s_bad_at;

  Sums at = first;
  for (int i = i0; i < i1; ++i) {
    const long long len = a.lengths[i], n = failed ? 0 : a.fresh[i];
    s_cu[i] = failed ? 0 : (int)at.a;
    s_rank[i] = (int)at.b;
    s_run[i] = (int)at.c;
    if (blockIdx.x == 0) {
      a.cu_new[i] = s_cu[i];
      a.kv_lengths[i] = (int)(len + n);
      a.cu_units[i] = failed ? 0 : (int)at.d;
    }
    if (n > 0) {
      at.a += n;
      at.b += blocks(len + n) - blocks(len);
      at.c += blocks(len + n) - (len >> a.size_log2);
      at.d += (len + n + kUnitKeys - 1) / kUnitKeys + kPairCost;
    }
  }
  const int used = failed ? 0 : (int)total.a;
  if (tid == 0) {
    s_cu[a.R] = used;
    if (blockIdx.x == 0) {
      a.cu_new[a.R] = used;
      a.cu_units[a.R] = failed ? 0 : (int)total.d;
      a.num_runs[0] = failed ? 0 : (int)total.c;
    }
  }
  __syncthreads();

  // four rows a thread: one search, and mostly one block, serves them
  const bool wide = ((reinterpret_cast<uintptr_t>(a.slots) | reinterpret_cast<uintptr_t>(a.positions)) & 15) == 0;
  for (int t0 = (blockIdx.x * kThreads + tid) * kRows; t0 < a.rows; t0 += gridDim.x * kThreads * kRows) {
    int lo = 0, hi = a.R;  // the last request whose first row is at or before t0
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_cu[mid] <= t0)
        lo = mid;
      else
        hi = mid;
    }
    int i = lo, len = a.lengths[i], id = -1, held_block = -1;
    int slot[kRows], pos[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const int t = t0 + k;
      slot[k] = -1;
      pos[k] = 0;
      if (t < used) {
        if (t >= s_cu[i + 1]) {
          do ++i;
          while (t >= s_cu[i + 1]);
          len = a.lengths[i];
          held_block = -1;
        }
        const int row = t - s_cu[i], n = s_cu[i + 1] - s_cu[i];
        pos[k] = len + row;
        const int block = pos[k] >> a.size_log2, off = pos[k] & (size - 1), have = (int)blocks(len);
        if (block != held_block) {
          held_block = block;
          id = block < have ? a.tables[i * a.table_ld + block] : a.free_stack[free_top - 1 - (s_rank[i] + block - have)];
        }
        if (off == 0 && block >= have) a.tables[i * a.table_ld + block] = id;  // a new block's first row is new
        slot[k] = (id << a.size_log2) + off;
        if (row == 0 || off == 0) {
          const int r = s_run[i] + block - (len >> a.size_log2);
          if (r < a.max_runs) a.runs[r] = make_int4(id, off, min(size - off, n - row), t);
        }
      }
    }
    if (wide && t0 + kRows <= a.rows) {
      *reinterpret_cast<int4*>(a.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      *reinterpret_cast<int4*>(a.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        if (t0 + k < a.rows) {
          a.slots[t0 + k] = slot[k];
          a.positions[t0 + k] = pos[k];
        }
      }
    }
  }

  if (last_cta(a.done)) {
    if (failed) {
      if (tid == 0 && a.status[0] == kStepOk) {  // the first failure stays until it is read
        a.status[0] = failed;
        a.status[1] = failed_at;
      }
    } else {
      for (int i = tid; i < a.R; i += kThreads) a.lengths[i] += a.fresh[i];
      if (tid == 0) a.num_free[0] = free_top - (int)total.b;
    }
  }
}

__global__ void __launch_bounds__(kThreads)
    paged_truncate_kernel(int* tables, long table_ld, int* lengths, const int* __restrict__ keep, int* free_stack,
                          int* num_free, int* status, int* done, int R, int MB, int F, int size_log2) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ int s_rank[];  // [R] freed blocks of the requests before
  const int size = 1 << size_log2, tid = threadIdx.x;
  const int per = (R + kThreads - 1) / kThreads, i0 = min(R, tid * per), i1 = min(R, i0 + per);
  const int top = num_free[0];
  const auto blocks = [&](int n) { return (int)(((long long)n + size - 1) >> size_log2); };
  const auto kept = [&](int i) { return min(lengths[i], max(keep[i], 0)); };
  Sums mine{0, 0, 0, 0}, total;
  int bad_at = R;
  for (int i = i0; i < i1; ++i) {
    mine.a += blocks(lengths[i]) - blocks(kept(i));
    if (lengths[i] < 0 || lengths[i] > ((long long)MB << size_log2)) bad_at = min(bad_at, i);
  }
  Sums at = block_exclusive(mine, total);
  __shared__ int s_bad_at;  // R: no request is at fault
  if (tid == 0) s_bad_at = R;
  __syncthreads();
  if (bad_at < R) atomicMin(&s_bad_at, bad_at);
  __syncthreads();
  // the same verdict in every CTA
  const bool failed = s_bad_at < R || top < 0 || top > F || total.a > F - top;
  if (failed) {
    if (last_cta(done) && tid == 0 && status[0] == kStepOk) {
      status[0] = kStepState;
      status[1] = s_bad_at < R ? s_bad_at : -1;
    }
    return;
  }
  for (int i = i0; i < i1; ++i) {
    s_rank[i] = (int)at.a;
    at.a += blocks(lengths[i]) - blocks(kept(i));
  }
  __syncthreads();
  const int freed = (int)total.a;
  for (int i = blockIdx.x * kWarps + (tid >> 5); i < R; i += gridDim.x * kWarps) {
    const int b0 = blocks(kept(i)), b1 = blocks(lengths[i]);
    for (int b = b0 + (tid & 31); b < b1; b += 32) {
      free_stack[top + freed - 1 - (s_rank[i] + b - b0)] = tables[i * table_ld + b];
      tables[i * table_ld + b] = -1;
    }
  }
  if (last_cta(done)) {
    for (int i = tid; i < R; i += kThreads) lengths[i] = kept(i);
    if (tid == 0) num_free[0] = top + freed;
  }
}

void check_state(const at::Tensor& tables, const at::Tensor& lengths, const at::Tensor& free_stack,
                 const at::Tensor& num_free, const at::Tensor& status, const at::Tensor& done, int64_t block_size) {
  TORCH_CHECK(tables.is_cuda() && tables.dim() == 2 && tables.scalar_type() == at::kInt && tables.stride(1) == 1,
              "block tables: CUDA int32 [requests, blocks]");
  for (const at::Tensor* t : {&lengths, &free_stack, &num_free, &status, &done})
    TORCH_CHECK(t->device() == tables.device() && t->scalar_type() == at::kInt && t->is_contiguous(),
                "block tables: the state's tensors are contiguous int32 on one device");
  TORCH_CHECK(lengths.numel() == tables.size(0) && num_free.numel() == 1 && status.numel() == 2 && done.numel() == 1,
              "block tables: state sizes");
  TORCH_CHECK(tables.size(0) >= 1 && tables.size(0) <= kMaxRequests, "block tables: 1 to ", kMaxRequests, " requests");
  TORCH_CHECK(block_size == 16 || block_size == 32 || block_size == 64 || block_size == 128,
              "block size must be 16, 32, 64 or 128");
  TORCH_CHECK(free_stack.numel() * block_size < (1LL << 31) && tables.size(1) * block_size < (1LL << 31),
              "block tables: slots and positions are int32");
}

int log2_of(int64_t v) {
  int n = 0;
  while ((int64_t(1) << n) < v) ++n;
  return n;
}

}  // namespace

// One step: see the head of this file. Returns int32 tensors: slots and positions [rows]; runs
// [max_runs, 4] (block, first offset, tokens, first row); meta, which is cu_new [R + 1], cu_units
// [R + 1], kv_lengths [R] and the number of runs, one after the other.
std::vector<at::Tensor> paged_step(const at::Tensor& tables, const at::Tensor& lengths, const at::Tensor& free_stack,
                                   const at::Tensor& num_free, const at::Tensor& status, const at::Tensor& done,
                                   int64_t block_size, const at::Tensor& fresh, int64_t rows, int64_t max_new) {
  check_state(tables, lengths, free_stack, num_free, status, done, block_size);
  const int64_t R = tables.size(0);
  TORCH_CHECK(fresh.device() == tables.device() && fresh.scalar_type() == at::kInt && fresh.is_contiguous() &&
                  fresh.numel() == R,
              "paged_step: new_tokens contiguous int32 [", R, "] on the tables' device");
  TORCH_CHECK(rows >= 0 && rows < (1LL << 31) - kThreads * 1024 * kRows, "paged_step: num_tokens ", rows);
  c10::cuda::CUDAGuard guard(tables.device());
  const int64_t max_runs = std::min(rows, rows / block_size + 2 * R);
  Outputs make(tables.options());
  make.plan({rows}, at::kInt).plan({rows}, at::kInt).plan({max_runs, 4}, at::kInt).plan({3 * R + 3}, at::kInt);
  std::vector<at::Tensor> out;
  out.reserve(4);
  out.push_back(make.next({rows}, at::kInt));
  out.push_back(make.next({rows}, at::kInt));
  out.push_back(make.next({max_runs, 4}, at::kInt));
  out.push_back(make.next({3 * R + 3}, at::kInt));
  int* meta = out[3].data_ptr<int>();
  StepArgs a{};
  a.tables = tables.data_ptr<int>();
  a.table_ld = tables.stride(0);
  a.lengths = lengths.data_ptr<int>();
  a.fresh = fresh.data_ptr<int>();
  a.free_stack = free_stack.data_ptr<int>();
  a.num_free = num_free.data_ptr<int>();
  a.status = status.data_ptr<int>();
  a.done = done.data_ptr<int>();
  a.R = (int)R;
  a.MB = (int)tables.size(1);
  a.F = (int)free_stack.numel();
  a.size_log2 = log2_of(block_size);
  a.rows = (int)rows;
  a.max_new = (int)std::min<int64_t>(max_new, INT32_MAX);
  a.max_runs = (int)max_runs;
  a.slots = out[0].data_ptr<int>();
  a.positions = out[1].data_ptr<int>();
  a.runs = reinterpret_cast<int4*>(out[2].data_ptr<int>());
  a.cu_new = meta;
  a.cu_units = meta + R + 1;
  a.kv_lengths = meta + 2 * R + 2;
  a.num_runs = meta + 3 * R + 2;
  const int smem = (int)(3 * R + 1) * 4;
  C10_CUDA_CHECK(ensure_dynamic_smem((const void*)paged_step_kernel, (3 * kMaxRequests + 1) * 4));
  // a CTA for each 1024 rows, at most two for an SM: more would only repeat the prefix sums
  const int64_t most = 2 * device_sm_count(), per = kThreads * kRows;
  const int64_t grid = std::max<int64_t>(1, std::min<int64_t>((rows + per - 1) / per, most));
  launch_early(paged_step_kernel, dim3((unsigned)grid), kThreads, smem, a);
  return out;
}

void paged_truncate(const at::Tensor& tables, const at::Tensor& lengths, const at::Tensor& free_stack,
                    const at::Tensor& num_free, const at::Tensor& status, const at::Tensor& done, int64_t block_size,
                    const at::Tensor& keep) {
  check_state(tables, lengths, free_stack, num_free, status, done, block_size);
  TORCH_CHECK(keep.device() == tables.device() && keep.scalar_type() == at::kInt && keep.is_contiguous() &&
                  keep.numel() == lengths.numel(),
              "paged_truncate: keep contiguous int32 [", lengths.numel(), "] on the tables' device");
  c10::cuda::CUDAGuard guard(tables.device());
  const int R = (int)tables.size(0);
  C10_CUDA_CHECK(ensure_dynamic_smem((const void*)paged_truncate_kernel, kMaxRequests * 4));
  const int grid = std::max(1, std::min((R + kWarps - 1) / kWarps, 2 * device_sm_count()));
  launch_early(paged_truncate_kernel, dim3(grid), kThreads, R * 4, tables.data_ptr<int>(), tables.stride(0),
               lengths.data_ptr<int>(), keep.data_ptr<int>(), free_stack.data_ptr<int>(), num_free.data_ptr<int>(),
               status.data_ptr<int>(), done.data_ptr<int>(), R, (int)tables.size(1), (int)free_stack.numel(),
               log2_of(block_size));
}

}  // namespace hrm
