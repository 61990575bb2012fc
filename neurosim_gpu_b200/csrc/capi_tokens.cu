// capi_tokens.cu -- extern "C" entry points of the token operators (see include/neurosim_b200.h).
//
// As in capi.cu, arguments are checked completely before anything is enqueued; a failed check
// returns a negative status and leaves a message for nsb_last_error().  Nothing here throws.
#include <algorithm>

#include "nsb_tokens.h"

namespace {

constexpr int64_t kMost = int64_t{1} << 31;  // rows, columns and tokens are below this
constexpr int64_t kMostProduct = kMost - 256;  // ... a product's rows below this: its tiles are counted in 32 bits

bool fail(const char* message) { return nsb::set_error(NSB_ERR_ARGUMENT, message), false; }

bool type_ok(int32_t type) {
  return type == NSB_VALUE_F32 || type == NSB_VALUE_F16 || type == NSB_VALUE_BF16;
}

bool check_matrix(const nsb_matrix* m, nsb::Dense* d, const char* shape, const char* data) {
  if (!m || m->rows < 0 || m->cols < 1 || m->rows >= kMost || m->cols >= kMost || m->row_stride < m->cols ||
      !type_ok(m->type))
    return fail(shape);
  if (m->rows > 0 && (!m->data || reinterpret_cast<uintptr_t>(m->data) % nsb::value_bytes(m->type) != 0))
    return fail(data);
  *d = {m->data, m->rows, m->cols, m->row_stride, m->type};
  return true;
}

// Whether two matrices of one element size share no element: apart in memory, or columns side by side in rows that
// are the same distance apart.
bool apart(const nsb::Dense& a, const nsb::Dense& b) {
  if (a.rows == 0 || b.rows == 0) return true;
  const auto bytes = [](const nsb::Dense& m, int64_t elements) { return static_cast<uintptr_t>(elements) * nsb::value_bytes(m.type); };
  const auto from_a = reinterpret_cast<uintptr_t>(a.data), from_b = reinterpret_cast<uintptr_t>(b.data);
  if (from_a + bytes(a, (a.rows - 1) * a.stride + a.cols) <= from_b || from_b + bytes(b, (b.rows - 1) * b.stride + b.cols) <= from_a)
    return true;
  const uintptr_t pitch = bytes(a, a.stride);
  if (pitch != bytes(b, b.stride)) return false;
  const uintptr_t ahead = from_b >= from_a ? (from_b - from_a) % pitch : (pitch - (from_a - from_b) % pitch) % pitch;
  return ahead >= bytes(a, a.cols) && ahead + bytes(b, b.cols) <= pitch;
}

bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

bool check_status(const int* status) { return aligned(status, 4) ? true : fail("the status word must be 4-byte aligned"); }

bool check_tokens(const void* tokens, int32_t bytes, int64_t n) {
  if (bytes != 4 && bytes != 8) return fail("tokens must be int32 or int64");
  if (n > 0 && (!tokens || reinterpret_cast<uintptr_t>(tokens) % bytes != 0)) return fail("tokens are required, aligned to their size");
  return true;
}

bool check_nvfp4(const nsb_nvfp4* m, nsb::Nvfp4* d) {
  if (!m || m->rows < 0 || m->cols < 1 || m->rows >= kMost || m->cols >= kMost)
    return fail("an NVFP4 matrix is [rows >= 0, cols >= 1], each below 2^31");
  if (m->code_stride != (m->cols + 31) / 32 * 16) return fail("NVFP4 codes: rows must be 16 * ceil(cols / 32) bytes apart");
  if (m->scale_count != m->rows && m->scale_count != 1) return fail("NVFP4 scale: one value per row, or one");
  if (m->rows > 0 && (!m->codes || !m->block_scales || !m->scale)) return fail("NVFP4 codes, block scales and scale are required");
  if (reinterpret_cast<uintptr_t>(m->codes) % 16 != 0 || reinterpret_cast<uintptr_t>(m->block_scales) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(m->scale) % 4 != 0)
    return fail("NVFP4 codes and block scales must be 16-byte aligned, the scale 4-byte aligned");
  *d = {m->rows, m->cols, m->codes, m->code_stride, m->block_scales, m->scale, m->scale_count == m->rows};
  return true;
}

bool check_workspace(const void* workspace, size_t have, size_t need, size_t align) {
  if (need == 0) return true;
  if (workspace && have >= need && reinterpret_cast<uintptr_t>(workspace) % align == 0) return true;
  nsb::set_error(NSB_ERR_WORKSPACE, "workspace missing, misaligned or too small");
  return false;
}

int done(cudaError_t err, const char* where) {
  return err == cudaSuccess ? NSB_OK : nsb::set_cuda_error(err, where);
}

// A packed matrix in a workspace; moves `at` past it.
nsb::Nvfp4 carve(uint8_t** at, int64_t rows, int64_t cols, bool per_row) {
  const int64_t pitch = (cols + 31) / 32 * 16, scales = (rows + 127) / 128 * ((cols + 255) / 256) * 2048;
  uint8_t* bytes = *at;
  *at += (rows * pitch + scales + 4 * rows + 255) / 256 * 256;
  return {rows, cols, bytes, pitch, bytes + rows * pitch, reinterpret_cast<float*>(bytes + rows * pitch + scales), per_row};
}

size_t packed_bytes(int64_t rows, int64_t cols) {
  uint8_t* at = nullptr;
  carve(&at, rows, cols, true);
  return reinterpret_cast<uintptr_t>(at);
}

bool sizes_ok(int64_t rows, int64_t cols, int64_t outputs) {
  return rows >= 1 && cols >= 1 && outputs >= 1 && rows < kMost && cols < kMost && outputs < kMost;
}

bool product_ok(int64_t a_rows, int64_t b_rows) {
  return a_rows < kMostProduct && b_rows < kMostProduct ? true : fail("a product's matrices must have fewer than 2^31 - 256 rows");
}

}  // namespace

extern "C" {

int nsb_stimulus_drive(const void* tokens, int32_t token_bytes, const nsb_matrix* table, float scale,
                       const nsb_matrix* out, void* stream) {
  nsb::Dense t, o;
  if (!check_matrix(table, &t, "the stimulus table must be a [rows, neurons] matrix of float32, float16 or bfloat16", "the stimulus table is required") ||
      !check_matrix(out, &o, "the drive must be a [tokens, neurons] matrix of float32, float16 or bfloat16", "the drive output is required"))
    return NSB_ERR_ARGUMENT;
  if (o.cols != t.cols) return nsb::set_error(NSB_ERR_ARGUMENT, "drive and table must have the same number of neurons");
  if (o.type != t.type && o.type != NSB_VALUE_F32) return nsb::set_error(NSB_ERR_ARGUMENT, "the drive has the table's type or float32");
  if (!apart(t, o)) return nsb::set_error(NSB_ERR_ARGUMENT, "the drive must not overlap with the table");
  if (!check_tokens(tokens, token_bytes, o.rows)) return NSB_ERR_ARGUMENT;
  nsb::set_error(NSB_OK, "");
  if (o.rows == 0) return NSB_OK;
  return done(nsb::launch_stimulus_drive(tokens, token_bytes, o.rows, t, scale, o, static_cast<cudaStream_t>(stream)),
              "nsb_stimulus_drive launch");
}

size_t nsb_stimulus_gradient_workspace_size(int64_t tokens, int64_t cols) {
  if (tokens <= 0 || cols < 1 || tokens >= kMost || cols >= kMost) return 0;
  return nsb::stimulus_gradient_workspace_bytes(tokens, cols);
}

int nsb_stimulus_gradient(const void* tokens, int32_t token_bytes, const nsb_matrix* grad, float scale,
                          const nsb_matrix* out, void* workspace, size_t workspace_bytes, void* stream) {
  nsb::Dense g, o;
  if (!check_matrix(grad, &g, "the drive's gradient must be a [tokens, neurons] matrix of float32, float16 or bfloat16", "the drive's gradient is required") ||
      !check_matrix(out, &o, "the table's gradient must be a [rows, neurons] matrix of float32, float16 or bfloat16", "the table's gradient is required"))
    return NSB_ERR_ARGUMENT;
  if (o.cols != g.cols) return nsb::set_error(NSB_ERR_ARGUMENT, "the gradients must have the same number of neurons");
  if (o.type != g.type && o.type != NSB_VALUE_F32 && g.type != NSB_VALUE_F32)
    return nsb::set_error(NSB_ERR_ARGUMENT, "one of the gradients must be float32 where their types differ");
  if (!check_tokens(tokens, token_bytes, g.rows)) return NSB_ERR_ARGUMENT;
  if (!check_workspace(workspace, workspace_bytes, nsb_stimulus_gradient_workspace_size(g.rows, g.cols), 16)) return NSB_ERR_WORKSPACE;
  nsb::set_error(NSB_OK, "");
  if (o.rows == 0) return NSB_OK;
  return done(nsb::launch_stimulus_gradient(tokens, token_bytes, g, scale, o, workspace, static_cast<cudaStream_t>(stream)),
              "nsb_stimulus_gradient launch");
}

size_t nsb_nvfp4_quantize_workspace_size(int64_t rows, int64_t cols, int32_t transpose, int64_t scale_count) {
  if (rows < 1 || cols < 1 || rows >= kMost || cols >= kMost) return 0;
  const nsb::Nvfp4 out{transpose ? cols : rows, transpose ? rows : cols, nullptr, 0, nullptr, nullptr, scale_count == (transpose ? cols : rows)};
  return nsb::nvfp4_quantize_workspace_bytes(out, transpose != 0);
}

int nsb_nvfp4_quantize(const nsb_matrix* value, int32_t transpose, const nsb_nvfp4* out, float* amax,
                       int32_t amax_given, void* workspace, size_t workspace_bytes, void* stream) {
  nsb::Dense v;
  nsb::Nvfp4 o;
  if (!check_matrix(value, &v, "the value must be a matrix of float32, float16 or bfloat16", "the value is required") ||
      !check_nvfp4(out, &o))
    return NSB_ERR_ARGUMENT;
  if (o.rows != (transpose ? v.cols : v.rows) || o.cols != (transpose ? v.rows : v.cols))
    return nsb::set_error(NSB_ERR_ARGUMENT, "the NVFP4 matrix must have the value's shape, or the transposed one");
  if (reinterpret_cast<uintptr_t>(amax) % 4 != 0 || (amax_given && !amax))
    return nsb::set_error(NSB_ERR_ARGUMENT, "a given amax is required, 4-byte aligned");
  const size_t need = nsb_nvfp4_quantize_workspace_size(v.rows, v.cols, transpose, out->scale_count);
  if (!check_workspace(workspace, workspace_bytes, need, 4)) return NSB_ERR_WORKSPACE;
  nsb::set_error(NSB_OK, "");
  if (v.rows == 0) return NSB_OK;
  return done(nsb::launch_nvfp4_quantize(v, transpose != 0, o, reinterpret_cast<unsigned int*>(amax), amax_given != 0, workspace, static_cast<cudaStream_t>(stream)),
              "nsb_nvfp4_quantize launch");
}

int nsb_nvfp4_dequantize(const nsb_nvfp4* value, const nsb_matrix* out, void* stream) {
  nsb::Nvfp4 v;
  nsb::Dense o;
  if (!check_nvfp4(value, &v) ||
      !check_matrix(out, &o, "the output must be a matrix of float32, float16 or bfloat16", "the output is required"))
    return NSB_ERR_ARGUMENT;
  if (o.rows != v.rows || o.cols != v.cols) return nsb::set_error(NSB_ERR_ARGUMENT, "the output must have the NVFP4 matrix's shape");
  nsb::set_error(NSB_OK, "");
  if (v.rows == 0) return NSB_OK;
  return done(nsb::launch_nvfp4_dequantize(v, o, static_cast<cudaStream_t>(stream)), "nsb_nvfp4_dequantize launch");
}

int nsb_nvfp4_product(const nsb_nvfp4* a, const nsb_nvfp4* b, const float* bias, const nsb_matrix* out,
                      int* status, void* stream) {
  nsb::Nvfp4 x, y;
  nsb::Dense o;
  if (!check_nvfp4(a, &x) || !check_nvfp4(b, &y) ||
      !check_matrix(out, &o, "the product must be a matrix of float32, float16 or bfloat16", "the product is required"))
    return NSB_ERR_ARGUMENT;
  if (x.cols != y.cols) return nsb::set_error(NSB_ERR_ARGUMENT, "the operands must have the same number of columns");
  if (y.rows < 1 || o.rows != x.rows || o.cols != y.rows)
    return nsb::set_error(NSB_ERR_ARGUMENT, "the product must be [a.rows, b.rows], b.rows >= 1");
  if (!product_ok(x.rows, y.rows) || !check_status(status)) return NSB_ERR_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(bias) % 4 != 0) return nsb::set_error(NSB_ERR_ARGUMENT, "the bias must be 4-byte aligned");
  nsb::set_error(NSB_OK, "");
  if (x.rows == 0) return NSB_OK;
  return done(nsb::launch_nvfp4_product(x, y, bias, o, false, status, static_cast<cudaStream_t>(stream)),
              "nsb_nvfp4_product launch");
}

void nsb_nvfp4_product_wait_limit(int32_t polls) { nsb::set_product_polls(polls); }

int nsb_nvfp4_product_status(int32_t* code, void* stream) {
  if (!code) return nsb::set_error(NSB_ERR_ARGUMENT, "a place for the code is required");
  nsb::set_error(NSB_OK, "");
  return done(nsb::take_product_status(code, static_cast<cudaStream_t>(stream)), "nsb_nvfp4_product_status");
}

size_t nsb_nvfp4_readout_workspace_size(int64_t rows, int64_t cols) {
  return sizes_ok(rows, cols, 1) ? packed_bytes(rows, cols) : 0;
}

int nsb_nvfp4_readout(const nsb_matrix* state, const nsb_nvfp4* weight, const float* bias, const nsb_matrix* out,
                      void* workspace, size_t workspace_bytes, int* status, void* stream) {
  nsb::Dense x, o;
  nsb::Nvfp4 w;
  if (!check_matrix(state, &x, "states must be a matrix of float32, float16 or bfloat16", "states are required") || !check_nvfp4(weight, &w) ||
      !check_matrix(out, &o, "the output must be a matrix of float32, float16 or bfloat16", "the output is required"))
    return NSB_ERR_ARGUMENT;
  if (x.cols != w.cols) return nsb::set_error(NSB_ERR_ARGUMENT, "states and weights must have the same number of columns");
  if (w.rows < 1 || o.rows != x.rows || o.cols != w.rows)
    return nsb::set_error(NSB_ERR_ARGUMENT, "the output must be [state.rows, weight.rows], weight.rows >= 1");
  if (!product_ok(x.rows, w.rows) || !check_status(status)) return NSB_ERR_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(bias) % 4 != 0) return nsb::set_error(NSB_ERR_ARGUMENT, "the bias must be 4-byte aligned");
  if (!check_workspace(workspace, workspace_bytes, nsb_nvfp4_readout_workspace_size(x.rows, x.cols), 16)) return NSB_ERR_WORKSPACE;
  nsb::set_error(NSB_OK, "");
  if (x.rows == 0) return NSB_OK;
  auto* bytes = static_cast<uint8_t*>(workspace);
  const nsb::Nvfp4 q = carve(&bytes, x.rows, x.cols, true);
  const cudaError_t err = nsb::launch_nvfp4_quantize(x, false, q, nullptr, false, nullptr, static_cast<cudaStream_t>(stream));
  if (err != cudaSuccess) return done(err, "nsb_nvfp4_readout launch");
  return done(nsb::launch_nvfp4_product(q, w, bias, o, true, status, static_cast<cudaStream_t>(stream)), "nsb_nvfp4_readout launch");
}

// Forward: the packed states and weights; backward: the operands of one product at a time, and the sums
// of the bias; 256 bytes for the largest sizes.
size_t nsb_nvfp4_train_workspace_size(int64_t rows, int64_t cols, int64_t outputs) {
  if (!sizes_ok(rows, cols, outputs)) return 0;
  const size_t forward = packed_bytes(rows, cols) + packed_bytes(outputs, cols);
  const size_t state = packed_bytes(rows, outputs) + packed_bytes(cols, outputs);
  const size_t weight = packed_bytes(outputs, rows) + packed_bytes(cols, rows);
  return 256 + std::max({forward, state, weight, nsb::column_sums_workspace_bytes(rows, outputs)});
}

int nsb_nvfp4_train_forward(const nsb_matrix* state, const nsb_matrix* weight, const float* bias, const nsb_matrix* out,
                            float* largest, void* workspace, size_t workspace_bytes, int* status, void* stream) {
  nsb::Dense x, w, o;
  if (!check_matrix(state, &x, "states must be a matrix of float32, float16 or bfloat16", "states are required") ||
      !check_matrix(weight, &w, "weights must be a matrix of float32, float16 or bfloat16", "weights are required") ||
      !check_matrix(out, &o, "the output must be a matrix of float32, float16 or bfloat16", "the output is required"))
    return NSB_ERR_ARGUMENT;
  if (x.cols != w.cols || w.rows < 1 || o.rows != x.rows || o.cols != w.rows)
    return nsb::set_error(NSB_ERR_ARGUMENT, "states [M, K], weights [N >= 1, K] and output [M, N] do not fit together");
  if (!product_ok(x.rows, w.rows) || !check_status(status)) return NSB_ERR_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(bias) % 4 != 0 || !largest || reinterpret_cast<uintptr_t>(largest) % 4 != 0)
    return nsb::set_error(NSB_ERR_ARGUMENT, "two words for the largest sizes are required; they and the bias must be 4-byte aligned");
  if (!check_workspace(workspace, workspace_bytes, nsb_nvfp4_train_workspace_size(x.rows, x.cols, w.rows), 16)) return NSB_ERR_WORKSPACE;
  nsb::set_error(NSB_OK, "");
  if (x.rows == 0) return NSB_OK;
  const auto s = static_cast<cudaStream_t>(stream);
  auto* most = reinterpret_cast<unsigned int*>(largest);
  auto* at = static_cast<uint8_t*>(workspace) + 256;
  const nsb::Nvfp4 qx = carve(&at, x.rows, x.cols, true), qw = carve(&at, w.rows, w.cols, false);
  cudaError_t err = nsb::launch_nvfp4_quantize(w, false, qw, most + 1, false, nullptr, s);
  if (err == cudaSuccess) err = nsb::launch_nvfp4_quantize(x, false, qx, most, false, nullptr, s);
  if (err == cudaSuccess) err = nsb::launch_nvfp4_product(qx, qw, bias, o, true, status, s);
  return done(err, "nsb_nvfp4_train_forward launch");
}

int nsb_nvfp4_train_backward(const nsb_matrix* state, const nsb_matrix* weight, const nsb_matrix* grad, const float* largest,
                             const nsb_matrix* state_grad, const nsb_matrix* weight_grad, float* bias_grad, void* workspace,
                             size_t workspace_bytes, int* status, void* stream) {
  nsb::Dense x, w, d, dx, dw;
  if (!check_matrix(state, &x, "states must be a matrix of float32, float16 or bfloat16", "states are required") ||
      !check_matrix(weight, &w, "weights must be a matrix of float32, float16 or bfloat16", "weights are required") ||
      !check_matrix(grad, &d, "the output's gradient must be a matrix of float32, float16 or bfloat16", "the output's gradient is required") ||
      (state_grad && !check_matrix(state_grad, &dx, "the states' gradient must be a matrix of float32, float16 or bfloat16", "the states' gradient has no data")) ||
      (weight_grad && !check_matrix(weight_grad, &dw, "the weights' gradient must be a matrix of float32, float16 or bfloat16", "the weights' gradient has no data")))
    return NSB_ERR_ARGUMENT;
  if (x.rows < 1 || w.rows < 1 || x.cols != w.cols || d.rows != x.rows || d.cols != w.rows ||
      (state_grad && (dx.rows != x.rows || dx.cols != x.cols)) || (weight_grad && (dw.rows != w.rows || dw.cols != w.cols)))
    return nsb::set_error(NSB_ERR_ARGUMENT, "states [M >= 1, K], weights [N >= 1, K], the output's gradient [M, N] and the gradients do not fit together");
  if (!product_ok(x.rows, w.rows) || !product_ok(x.cols, x.cols) || !check_status(status)) return NSB_ERR_ARGUMENT;
  if (!largest || reinterpret_cast<uintptr_t>(largest) % 4 != 0 || reinterpret_cast<uintptr_t>(bias_grad) % 4 != 0)
    return nsb::set_error(NSB_ERR_ARGUMENT, "the largest sizes of the forward call are required; they and the bias's gradient must be 4-byte aligned");
  if (!check_workspace(workspace, workspace_bytes, nsb_nvfp4_train_workspace_size(x.rows, x.cols, w.rows), 16)) return NSB_ERR_WORKSPACE;
  nsb::set_error(NSB_OK, "");
  const auto s = static_cast<cudaStream_t>(stream);
  auto* most = reinterpret_cast<unsigned int*>(const_cast<float*>(largest));
  auto* grad_most = static_cast<unsigned int*>(workspace);
  auto* const first = static_cast<uint8_t*>(workspace) + 256;
  cudaError_t err = cudaSuccess;
  if (state_grad) {
    uint8_t* at = first;
    const nsb::Nvfp4 qd = carve(&at, d.rows, d.cols, true), qw = carve(&at, w.cols, w.rows, false);
    err = nsb::launch_nvfp4_quantize(w, true, qw, most + 1, true, nullptr, s);
    if (err == cudaSuccess) err = nsb::launch_nvfp4_quantize(d, false, qd, grad_most, false, nullptr, s);
    if (err == cudaSuccess) err = nsb::launch_nvfp4_product(qd, qw, nullptr, dx, true, status, s);
  }
  if (weight_grad && err == cudaSuccess) {
    uint8_t* at = first;
    const nsb::Nvfp4 qd = carve(&at, d.cols, d.rows, false), qx = carve(&at, x.cols, x.rows, false);
    err = nsb::launch_nvfp4_quantize(d, true, qd, grad_most, state_grad != nullptr, nullptr, s);
    if (err == cudaSuccess) err = nsb::launch_nvfp4_quantize(x, true, qx, most, true, nullptr, s);
    if (err == cudaSuccess) err = nsb::launch_nvfp4_product(qd, qx, nullptr, dw, false, status, s);
  }
  if (bias_grad && err == cudaSuccess) err = nsb::launch_column_sums(d, bias_grad, first, s);
  return done(err, "nsb_nvfp4_train_backward launch");
}

size_t nsb_column_sums_workspace_size(int64_t rows, int64_t cols) {
  if (rows < 1 || cols < 1 || rows >= kMost || cols >= kMost) return 0;
  return nsb::column_sums_workspace_bytes(rows, cols);
}

int nsb_column_sums(const nsb_matrix* value, float* out, void* workspace, size_t workspace_bytes,
                    void* stream) {
  nsb::Dense v;
  if (!check_matrix(value, &v, "the value must be a matrix of float32, float16 or bfloat16", "the value is required"))
    return NSB_ERR_ARGUMENT;
  if (!out || reinterpret_cast<uintptr_t>(out) % 4 != 0) return nsb::set_error(NSB_ERR_ARGUMENT, "the sums are required, 4-byte aligned");
  if (!check_workspace(workspace, workspace_bytes, nsb_column_sums_workspace_size(v.rows, v.cols), 4)) return NSB_ERR_WORKSPACE;
  nsb::set_error(NSB_OK, "");
  return done(nsb::launch_column_sums(v, out, workspace, static_cast<cudaStream_t>(stream)), "nsb_column_sums launch");
}

int nsb_adjust_logits(const nsb_logits* args, void* stream) {
  if (!args) return nsb::set_error(NSB_ERR_ARGUMENT, "logit arguments are required");
  nsb::LogitsArgs a{};
  if (!check_matrix(&args->logits, &a.logits, "logits must be a [rows, vocabulary] matrix of float32, float16 or bfloat16", "logits are required") ||
      !check_matrix(&args->out, &a.out, "the output must be a [rows, vocabulary] matrix of the logits' type", "the output is required"))
    return NSB_ERR_ARGUMENT;
  if (a.out.rows != a.logits.rows || a.out.cols != a.logits.cols || a.out.type != a.logits.type)
    return nsb::set_error(NSB_ERR_ARGUMENT, "the output must have the logits' shape and type");
  if (!(a.out.data == a.logits.data && (a.out.rows <= 1 || a.out.stride == a.logits.stride)) && !apart(a.logits, a.out))
    return nsb::set_error(NSB_ERR_ARGUMENT, "the output must be the logits themselves, or not overlap with them");
  if (a.logits.cols >= kMost / 2) return nsb::set_error(NSB_ERR_ARGUMENT, "the vocabulary must be below 2^30");
  if (args->history_length < 0 || args->history_length >= kMost || (args->history_length > 0 && a.logits.rows > 0 && (!args->history || args->history_stride < 0)))
    return nsb::set_error(NSB_ERR_ARGUMENT, "the history must be [rows, length] int32");
  if ((args->bias && args->bias_stride < 0) || (args->mask && args->mask_stride < 0) ||
      args->repetition.stride < 0 || args->presence.stride < 0 || args->frequency.stride < 0)
    return nsb::set_error(NSB_ERR_ARGUMENT, "strides must not be negative");
  if (!aligned(args->history, 4) || !aligned(args->lengths, 4) || !aligned(args->prompt_lengths, 4) || !aligned(args->bias, 4) ||
      !aligned(args->mask, 4) || !aligned(args->choice, 8) || !aligned(args->repetition.data, 4) ||
      !aligned(args->presence.data, 4) || !aligned(args->frequency.data, 4))
    return nsb::set_error(NSB_ERR_ARGUMENT, "history, lengths, penalties, bias, mask and choice must be aligned to their elements");
  if (!args->repetition.data && !(args->repetition.scalar > 0.0f))
    return nsb::set_error(NSB_ERR_ARGUMENT, "the repetition penalty must be above 0");
  a.history = args->history;
  a.history_length = args->history_length;
  a.history_stride = args->history_stride;
  a.lengths = args->lengths;
  a.prompt_lengths = args->prompt_lengths;
  a.repetition = args->repetition;
  a.presence = args->presence;
  a.frequency = args->frequency;
  a.bias = args->bias;
  a.bias_stride = args->bias_stride;
  a.mask = args->mask;
  a.mask_stride = args->mask_stride;
  a.choice = args->choice;
  nsb::set_error(NSB_OK, "");
  if (a.logits.rows == 0) return NSB_OK;
  return done(nsb::launch_adjust_logits(a, static_cast<cudaStream_t>(stream)), "nsb_adjust_logits launch");
}

}  // extern "C"
