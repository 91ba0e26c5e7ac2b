// dropout and layer norm with their gradients.
#include "encoder.cuh"

#include <algorithm>

namespace nvtext_amd {
namespace {

constexpr int kThreads = 256;

inline unsigned grid_for(int64_t work, int64_t per_cu) { return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(work, per_cu * device_cus()))); }

// ------------------------------------------------------------------ dropout
// A thread takes eight values with one counter.  It divides once to find its row and column and steps from there.
template <typename T>
__global__ void __launch_bounds__(kThreads) dropout_kernel(Rows<const T> x, Rows<T> out, int64_t rows, int64_t cols, int64_t blocks, Dropout d)
{
  int64_t const threads = static_cast<int64_t>(gridDim.x) * kThreads;
  int64_t const first   = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  int64_t i = first / blocks, b = first % blocks;
  int64_t const di = threads / blocks, db = threads % blocks;
  while (i < rows) {
    float f[8];
    load8(f, x.row(i) + b * 8, cols - b * 8);
    d.apply(f, i, b);
    store8(out.row(i) + b * 8, f, cols - b * 8);
    i += di;
    b += db;
    if (b >= blocks) {
      b -= blocks;
      ++i;
    }
  }
}

// ------------------------------------------------------------------ layer norm
// A vector of weights, of the tensors' type or of 32 bits.
struct Weights {
  const void* data;
  int32_t type;
  template <typename T>
  __device__ __forceinline__ void load(float (&f)[8], int64_t at, int64_t n) const
  {
    if (type == NVTEXT_AMD_TYPE_FLOAT32)
      load8(f, static_cast<const float*>(data) + at, n);
    else
      load8(f, static_cast<const T*>(data) + at, n);
  }
};

template <typename T>
__device__ __forceinline__ void load_sum(float (&f)[8], Rows<const T> x, Rows<const T> residual, int64_t i, int64_t b, int64_t cols, Dropout const& d)
{
  load8(f, x.row(i) + b * 8, cols - b * 8);
  if (d.dropped) d.apply(f, i, b);
  if (residual) {
    float r[8];
    load8(r, residual.row(i) + b * 8, cols - b * 8);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] += r[k];
  }
}

// A workgroup a row, which it goes through three times.
template <typename T>
__global__ void __launch_bounds__(kThreads) layer_norm_kernel(Rows<const T> x, Rows<const T> residual, Weights weight, Weights bias, float eps, Dropout d,
                                                              Rows<T> out, Rows<T> sum, float* mean_out, float* rstd_out, int64_t rows, int64_t cols)
{
  __shared__ float lds[kThreads / kWave];
  int64_t const blocks = (cols + 7) / 8;
  for (int64_t i = blockIdx.x; i < rows; i += gridDim.x) {
    float s = 0.f;
    for (int64_t b = threadIdx.x; b < blocks; b += kThreads) {
      float f[8];
      load_sum(f, x, residual, i, b, cols, d);
#pragma unroll
      for (int k = 0; k < 8; ++k) s += f[k];
    }
    float const mean = block_sum<kThreads>(s, lds) / static_cast<float>(cols);
    s                = 0.f;
    for (int64_t b = threadIdx.x; b < blocks; b += kThreads) {
      float f[8];
      load_sum(f, x, residual, i, b, cols, d);
#pragma unroll
      for (int k = 0; k < 8; ++k) s += b * 8 + k < cols ? (f[k] - mean) * (f[k] - mean) : 0.f;
    }
    float const rstd = 1.f / sqrtf(block_sum<kThreads>(s, lds) / static_cast<float>(cols) + eps);
    for (int64_t b = threadIdx.x; b < blocks; b += kThreads) {
      float f[8], w[8], c[8];
      load_sum(f, x, residual, i, b, cols, d);
      weight.load<T>(w, b * 8, cols - b * 8);
      bias.load<T>(c, b * 8, cols - b * 8);
      if (sum) store8(sum.row(i) + b * 8, f, cols - b * 8);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = (f[k] - mean) * rstd * w[k] + c[k];
      store8(out.row(i) + b * 8, f, cols - b * 8);
    }
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[i] = mean;
      if (rstd_out) rstd_out[i] = rstd;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
layer_norm_rows_backward_kernel(Rows<const T> grad, Rows<const T> sum, const float* mean_in, const float* rstd_in, Weights weight, Rows<const T> sum_grad,
                                Dropout d, Rows<T> x_grad, Rows<T> residual_grad, int64_t rows, int64_t cols)
{
  __shared__ float lds[kThreads / kWave];
  int64_t const blocks = (cols + 7) / 8;
  for (int64_t i = blockIdx.x; i < rows; i += gridDim.x) {
    float const mean = mean_in[i], rstd = rstd_in[i];
    float sa = 0.f, sh = 0.f;
    for (int64_t b = threadIdx.x; b < blocks; b += kThreads) {
      float g[8], s[8], w[8];
      load8(g, grad.row(i) + b * 8, cols - b * 8);
      load8(s, sum.row(i) + b * 8, cols - b * 8);
      weight.load<T>(w, b * 8, cols - b * 8);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        sa += g[k] * w[k];
        sh += g[k] * w[k] * ((s[k] - mean) * rstd);
      }
    }
    float const ma = block_sum<kThreads>(sa, lds) / static_cast<float>(cols);
    float const mh = block_sum<kThreads>(sh, lds) / static_cast<float>(cols);
    for (int64_t b = threadIdx.x; b < blocks; b += kThreads) {
      float g[8], s[8], w[8], e[8];
      load8(g, grad.row(i) + b * 8, cols - b * 8);
      load8(s, sum.row(i) + b * 8, cols - b * 8);
      weight.load<T>(w, b * 8, cols - b * 8);
      if (sum_grad) load8(e, sum_grad.row(i) + b * 8, cols - b * 8);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        s[k] = rstd * (g[k] * w[k] - ma - (s[k] - mean) * rstd * mh);
        if (sum_grad) s[k] += e[k];
      }
      store8(residual_grad.row(i) + b * 8, s, cols - b * 8);
      if (x_grad) {
        if (d.dropped) d.apply(s, i, b);
        store8(x_grad.row(i) + b * 8, s, cols - b * 8);
      }
    }
  }
}

// parts[part] and parts[count + part]: the sums over every count-th row of grad * h and of grad.  (Reads sum and grad before
// the kernel above, which may write over them.)
template <typename T>
__global__ void __launch_bounds__(kThreads)
layer_norm_weights_backward_kernel(Rows<const T> grad, Rows<const T> sum, const float* mean_in, const float* rstd_in, int64_t rows, int64_t cols, float* parts)
{
  int64_t const b = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (b * 8 >= cols) return;
  float dw[8] = {}, db[8] = {};
  for (int64_t i = blockIdx.y; i < rows; i += gridDim.y) {
    float const mean = mean_in[i], rstd = rstd_in[i];
    float g[8], s[8];
    load8(g, grad.row(i) + b * 8, cols - b * 8);
    load8(s, sum.row(i) + b * 8, cols - b * 8);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      dw[k] += g[k] * ((s[k] - mean) * rstd);
      db[k] += g[k];
    }
  }
  store8(parts + blockIdx.y * cols + b * 8, dw, cols - b * 8);
  store8(parts + (gridDim.y + static_cast<int64_t>(blockIdx.y)) * cols + b * 8, db, cols - b * 8);
}

bool is_weights(const nvtext_amd_matrix* w, const nvtext_amd_matrix* x) { return is_shape(w, 1, x->cols) && (w->type == x->type || w->type == NVTEXT_AMD_TYPE_FLOAT32); }
bool is_like(const nvtext_amd_matrix* m, const nvtext_amd_matrix* x) { return is_shape(m, x->rows, x->cols) && m->type == x->type; }

}  // namespace
}  // namespace nvtext_amd

extern "C" {

nvtext_amd_status nvtext_amd_dropout(const nvtext_amd_matrix* x, double p, uint64_t seed, uint32_t offset, void* stream_, const nvtext_amd_matrix* out)
{
  using namespace nvtext_amd;
  EntryScope const entry("nvtext_amd_dropout");
  if (!x || !out) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  for (auto* m : {x, out})
    if (const char* bad = bad_matrix(m)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  if (!is_like(out, x)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "out must be of the size and type of x");
  if (!is_probability(p)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "p must be between 0 and 1");
  if (x->rows == 0 || x->cols == 0) return NVTEXT_AMD_SUCCESS;
  hipStream_t stream   = static_cast<hipStream_t>(stream_);
  Dropout const d      = make_dropout(p, seed, offset);
  int64_t const blocks = (x->cols + 7) / 8;
  with_type(x->type, [&](auto zero) {
    using T = decltype(zero);
    ProfileScope const scope("dropout", stream);
    hipLaunchKernelGGL(dropout_kernel<T>, dim3(grid_for((x->rows * blocks + kThreads - 1) / kThreads, 16)), dim3(kThreads), 0, stream, rows_of<const T>(x), rows_of<T>(out),
                       x->rows, x->cols, blocks, d);
  });
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

nvtext_amd_status nvtext_amd_layer_norm(const nvtext_amd_matrix* x, const nvtext_amd_matrix* residual, const nvtext_amd_matrix* weight,
                                        const nvtext_amd_matrix* bias, double eps, double p, uint64_t seed, uint32_t offset, void* stream_,
                                        const nvtext_amd_matrix* out, const nvtext_amd_matrix* sum, float* mean, float* rstd)
{
  using namespace nvtext_amd;
  EntryScope const entry("nvtext_amd_layer_norm");
  if (!x || !weight || !bias || !out) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  for (auto* m : {x, residual, weight, bias, out, sum})
    if (const char* bad = m ? bad_matrix(m) : nullptr) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  if (x->cols == 0) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "a layer norm needs a width of 1 or more");
  for (auto* m : {residual, out, sum})
    if (m && !is_like(m, x)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "residual, out and sum must be of the size and type of x");
  if (!is_weights(weight, x) || !is_weights(bias, x) || weight->type != bias->type)
    return fail(NVTEXT_AMD_INVALID_ARGUMENT, "weight and bias must be vectors of x's width, both of x's type or both FLOAT32");
  if (!(eps >= 0)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "eps must not be negative");
  if (!is_probability(p)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "p must be between 0 and 1");
  if (x->rows == 0) return NVTEXT_AMD_SUCCESS;
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  Dropout const d    = make_dropout(p, seed, offset);
  with_type(x->type, [&](auto zero) {
    using T = decltype(zero);
    ProfileScope const scope("layer_norm", stream);
    hipLaunchKernelGGL(layer_norm_kernel<T>, dim3(grid_for(x->rows, 8)), dim3(kThreads), 0, stream, rows_of<const T>(x), rows_of<const T>(residual),
                       Weights{weight->data, weight->type}, Weights{bias->data, bias->type}, static_cast<float>(eps), d, rows_of<T>(out), rows_of<T>(sum), mean, rstd,
                       x->rows, x->cols);
  });
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

nvtext_amd_status nvtext_amd_layer_norm_backward(const nvtext_amd_matrix* grad, const nvtext_amd_matrix* sum, const float* mean, const float* rstd,
                                                 const nvtext_amd_matrix* weight, const nvtext_amd_matrix* sum_grad, double p, uint64_t seed, uint32_t offset,
                                                 void* stream_, const nvtext_amd_allocator* mr_, const nvtext_amd_matrix* x_grad,
                                                 const nvtext_amd_matrix* residual_grad, const nvtext_amd_matrix* weight_grad, const nvtext_amd_matrix* bias_grad)
{
  using namespace nvtext_amd;
  EntryScope const entry("nvtext_amd_layer_norm_backward");
  if (!grad || !sum || !weight || !residual_grad) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  for (auto* m : {grad, sum, weight, sum_grad, x_grad, residual_grad, weight_grad, bias_grad})
    if (const char* bad = m ? bad_matrix(m) : nullptr) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  if (grad->cols == 0) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "a layer norm needs a width of 1 or more");
  for (auto* m : {sum, sum_grad, x_grad, residual_grad})
    if (m && !is_like(m, grad)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "sum, sum_grad, x_grad and residual_grad must be of the size and type of grad");
  if (!is_weights(weight, grad)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "weight must be a vector of grad's width, of its type or FLOAT32");
  if (!weight_grad != !bias_grad) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "weight_grad and bias_grad come together");
  for (auto* m : {weight_grad, bias_grad})
    if (m && !is_like(m, weight)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "weight_grad and bias_grad must be of weight's size and type");
  if (!is_probability(p)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "p must be between 0 and 1");
  if (p > 0 && !x_grad) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "with dropout x_grad is a result of its own");
  if (grad->rows > 0 && (!mean || !rstd)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  Mr const mr{mr_, stream};
  Dropout const d    = make_dropout(p, seed, offset);
  int64_t const rows = grad->rows, cols = grad->cols;
  // rows = 0: the sums of the weights' gradients are zeros, of one part
  int64_t const parts = std::max<int64_t>(1, std::min<int64_t>(rows, 256));
  Temp const sums(mr, weight_grad ? static_cast<size_t>(2 * parts * cols) * sizeof(float) : 0);
  if (!sums.ok()) return fail(NVTEXT_AMD_ALLOC_FAILED, "temporary allocation failed");
  with_type(grad->type, [&](auto zero) {
    using T = decltype(zero);
    if (weight_grad) {
      ProfileScope const scope("layer_norm_weights_backward", stream);
      hipLaunchKernelGGL(layer_norm_weights_backward_kernel<T>, dim3(static_cast<unsigned>((cols + 8 * kThreads - 1) / (8 * kThreads)), static_cast<unsigned>(parts)), dim3(kThreads),
                         0, stream, rows_of<const T>(grad), rows_of<const T>(sum), mean, rstd, rows, cols, sums.as<float>());
    }
    if (rows > 0) {
      ProfileScope const scope("layer_norm_rows_backward", stream);
      hipLaunchKernelGGL(layer_norm_rows_backward_kernel<T>, dim3(grid_for(rows, 8)), dim3(kThreads), 0, stream, rows_of<const T>(grad), rows_of<const T>(sum), mean, rstd,
                         Weights{weight->data, weight->type}, rows_of<const T>(sum_grad), d, rows_of<T>(x_grad), rows_of<T>(residual_grad), rows, cols);
    }
  });
  if (weight_grad)
    with_type(weight->type, [&](auto zero) {
      using W = decltype(zero);
      ProfileScope const scope("layer_norm_add_parts", stream);
      launch_add_parts(sums.as<float>(), parts, cols, static_cast<W*>(weight_grad->data), stream);
      launch_add_parts(sums.as<float>() + parts * cols, parts, cols, static_cast<W*>(bias_grad->data), stream);
    });
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

}  // extern "C"
