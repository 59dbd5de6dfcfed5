// Library-level entry points of libxgb.so (version, status names, error word).
#include "xgb_common.cuh"

// One on every device, zero when the library is loaded there.
static __device__ int device_error_word;

XGB_API int xgb_version(void) { return 100; }

XGB_API const char* xgb_status_string(int status) {
  switch (status) {
    case XGB_OK: return "ok";
    case XGB_ERR_ARG: return "invalid argument";
    case XGB_ERR_SHAPE: return "unsupported shape";
    case XGB_ERR_STRIDE: return "unsupported stride";
    case XGB_ERR_ALIGN: return "misaligned pointer or stride";
    case XGB_ERR_LAUNCH: return "CUDA launch error";
    case XGB_ERR_DEVICE: return "device is not an sm_100 GPU";
    case XGB_ERR_WORKSPACE: return "workspace missing or too small";
    default: return "unknown status";
  }
}

XGB_API int* xgb_error_word(void) {
  // The first use on a device may load the module, also while a stream of this
  // thread is being captured.
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) {
    cudaGetLastError();
    return nullptr;
  }
  void* word = nullptr;
  const cudaError_t rc = cudaGetSymbolAddress(&word, device_error_word);
  cudaThreadExchangeStreamCaptureMode(&mode);
  if (rc != cudaSuccess) {
    cudaGetLastError();
    return nullptr;
  }
  return static_cast<int*>(word);
}
