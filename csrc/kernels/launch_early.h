// Host helpers of kernels whose calls are short next to their launch.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <torch/types.h>

namespace hrm {

// Launches `kernel` on the current stream while the kernel before it ends; the kernel itself waits for that
// end (griddepcontrol.wait) before it touches memory.
template <typename... P, typename... A>
inline void launch_early(void (*kernel)(P...), dim3 grid, int threads, int smem, A... args) {
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = at::cuda::getCurrentCUDAStream();
  config.attrs = &early;
  config.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, P(args)...));
}

// Uninitialised tensors of one allocation, each on a 256-byte boundary: a step's or a sampled token's
// outputs are a few hundred bytes, and an allocation of its own cost each more than the kernel's launch
// configuration does (0.65 us of host time).
class Outputs {
 public:
  explicit Outputs(const at::TensorOptions& like) : like_(like) {}
  // how many bytes a tensor takes; call for all of them before the first `next`
  Outputs& plan(at::IntArrayRef sizes, at::ScalarType type) {
    bytes_ += room(sizes, type);
    return *this;
  }
  at::Tensor next(at::IntArrayRef sizes, at::ScalarType type) {
    if (!buffer_.defined()) buffer_ = at::empty({bytes_}, like_.dtype(at::kByte));
    auto impl = c10::make_intrusive<at::TensorImpl>(c10::Storage(buffer_.storage()), buffer_.key_set(),
                                                    c10::scalarTypeToTypeMeta(type));
    impl->set_storage_offset(at_ / (int64_t)c10::elementSize(type));
    impl->set_sizes_contiguous(sizes);
    at_ += room(sizes, type);
    return at::Tensor(std::move(impl));
  }

 private:
  static int64_t room(at::IntArrayRef sizes, at::ScalarType type) {
    int64_t n = (int64_t)c10::elementSize(type);
    for (const int64_t s : sizes) n *= s;
    return (n + 255) / 256 * 256;
  }
  at::TensorOptions like_;
  at::Tensor buffer_;
  int64_t bytes_ = 0, at_ = 0;
};

}  // namespace hrm
