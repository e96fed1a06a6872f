// The status words that bounded waits inside kernels write to.
#include <torch/extension.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

namespace sb {

// Zeros that are there when this returns, whatever the caller's stream does.  The first call of a process may be one that a
// graph captures: on its stream the words would come from the graph's memory and be cleared by every replay, errors that other
// kernels reported with them.  So they are made on a stream that captures nothing, and waited for.
static at::Tensor fresh_words(int64_t device, int64_t n) {
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
  const c10::cuda::CUDAStreamCaptureModeGuard relaxed{cudaStreamCaptureModeRelaxed};
  auto stream = c10::cuda::getStreamFromPool(false, static_cast<c10::DeviceIndex>(device));
  for (int i = 0; i < 64; ++i) {                     // streams of the pool are handed out in turn
    cudaStreamCaptureStatus status;
    C10_CUDA_CHECK(cudaStreamIsCapturing(stream, &status));
    if (status == cudaStreamCaptureStatusNone) break;
    stream = c10::cuda::getStreamFromPool(false, static_cast<c10::DeviceIndex>(device));
  }
  const c10::cuda::CUDAStreamGuard on(stream);
  auto words = at::zeros({n}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, static_cast<c10::DeviceIndex>(device)));
  C10_CUDA_CHECK(cudaStreamSynchronize(stream));
  return words;
}

}  // namespace sb

void bind_status(pybind11::module& m) {
  m.def("fresh_words", &sb::fresh_words, "int32 zeros made apart from the current stream and its capture");
}
