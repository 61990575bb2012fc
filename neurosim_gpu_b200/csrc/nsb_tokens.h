// nsb_tokens.h -- host-side launchers of the token operators, shared with their C ABI (capi_tokens.cu).
#pragma once

#include "nsb_launch.h"
#include "nsb_values.cuh"

namespace nsb {

// Records `message` for nsb_last_error() (capi.cu) and returns `code`; never throws.
int set_error(int code, const char* message) noexcept;
int set_cuda_error(cudaError_t err, const char* where) noexcept;

// Raises a kernel's limit of dynamic shared memory once per device.
struct SharedLimit {
  bool raised[64] = {};
  template <typename K>
  cudaError_t raise(K* kernel, int bytes) {
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess || raised[device & 63]) return err;
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    raised[device & 63] = err == cudaSuccess;
    return err;
  }
};

// How many clusters of a kernel's CTAs run at once on the current device, asked once per device.
struct ClusterLimit {
  int known[64] = {};
  template <typename K>
  cudaError_t most(K* kernel, int cluster, int threads, int shared, int* clusters) {
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess) return err;
    if (known[device & 63] == 0) {
      cudaLaunchConfig_t config{};
      config.gridDim = dim3(static_cast<unsigned>(cluster));
      config.blockDim = dim3(static_cast<unsigned>(threads));
      config.dynamicSmemBytes = static_cast<size_t>(shared);
      cudaLaunchAttribute attribute{};
      attribute.id = cudaLaunchAttributeClusterDimension;
      attribute.val.clusterDim = {static_cast<unsigned>(cluster), 1, 1};
      config.attrs = &attribute;
      config.numAttrs = 1;
      int found = 0;
      if ((err = cudaOccupancyMaxActiveClusters(&found, kernel, &config)) != cudaSuccess) return err;
      known[device & 63] = found;
    }
    *clusters = known[device & 63];
    return cudaSuccess;
  }
};

// stimulus.cu
cudaError_t launch_stimulus_drive(const void* tokens, int token_bytes, int64_t n, const Dense& table,
                                  float scale, const Dense& out, cudaStream_t stream);
size_t stimulus_gradient_workspace_bytes(int64_t n, int64_t cols);
cudaError_t launch_stimulus_gradient(const void* tokens, int token_bytes, const Dense& grad,
                                     float scale, const Dense& out, void* workspace,
                                     cudaStream_t stream);

// microscale.cu
struct Nvfp4 {
  int64_t rows, cols;
  uint8_t* codes;         // [rows, pitch]
  int64_t pitch;          // bytes: 16 * ceil(cols / 32)
  uint8_t* block_scales;  // [ceil(rows / 128), 4 * ceil(cols / 256), 512]
  float* scale;           // [rows] or [1]
  bool per_row;
};
size_t nvfp4_quantize_workspace_bytes(const Nvfp4& out, bool transpose);
cudaError_t launch_nvfp4_quantize(const Dense& value, bool transpose, const Nvfp4& out, unsigned int* amax,
                                  bool amax_given, void* workspace, cudaStream_t stream);
cudaError_t launch_nvfp4_dequantize(const Nvfp4& in, const Dense& out, cudaStream_t stream);
size_t column_sums_workspace_bytes(int64_t rows, int64_t cols);
cudaError_t launch_column_sums(const Dense& value, float* out, void* workspace, cudaStream_t stream);

// microscale_product.cu
// b_ready: b was complete before the kernel ahead in the stream started.
cudaError_t launch_nvfp4_product(const Nvfp4& a, const Nvfp4& b, const float* bias, const Dense& out,
                                 bool b_ready, int* status, cudaStream_t stream);
void set_product_polls(int polls);
cudaError_t take_product_status(int* code, cudaStream_t stream);

// logits.cu
struct LogitsArgs {
  Dense logits, out;
  const int32_t* history;  // [rows, history_length], stride history_stride
  int64_t history_length, history_stride;
  const int32_t* lengths;         // [rows] or null: all history_length
  const int32_t* prompt_lengths;  // [rows] or null: none
  nsb_row_values repetition, presence, frequency;
  const float* bias;              // [rows or 1, vocabulary]
  int64_t bias_stride;            // 0: the same for all rows
  const int32_t* mask;            // [rows or 1, ceil(vocabulary / 32)]
  int64_t mask_stride;
  int64_t* choice;                // [rows] or null
};
cudaError_t launch_adjust_logits(const LogitsArgs& args, cudaStream_t stream);

}  // namespace nsb
