// The matrix product of a layer with bias, activation and residual, and its gradients.
#include "encoder.cuh"

#include <algorithm>

namespace nvtext_amd {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float activate(float z, int activation)
{
  switch (activation) {
    case NVTEXT_AMD_ACTIVATION_RELU: return z > 0.f ? z : 0.f;
    case NVTEXT_AMD_ACTIVATION_GELU: return z * (0.5f + 0.5f * erff(z * 0.70710678118654752f));
    case NVTEXT_AMD_ACTIVATION_GELU_TANH: return z * (0.5f + 0.5f * tanhf(0.79788456080286536f * (z + 0.044715f * z * z * z)));
    case NVTEXT_AMD_ACTIVATION_SILU: return z / (1.f + expf(-z));
    default: return z;
  }
}

__device__ __forceinline__ float slope(float z, int activation)
{
  switch (activation) {
    case NVTEXT_AMD_ACTIVATION_RELU: return z > 0.f ? 1.f : 0.f;
    case NVTEXT_AMD_ACTIVATION_GELU: return 0.5f + 0.5f * erff(z * 0.70710678118654752f) + z * expf(-0.5f * z * z) * 0.39894228040143268f;
    case NVTEXT_AMD_ACTIVATION_GELU_TANH: {
      float const t = tanhf(0.79788456080286536f * (z + 0.044715f * z * z * z));
      return 0.5f + 0.5f * t + 0.5f * z * (1.f - t * t) * 0.79788456080286536f * (1.f + 0.134145f * z * z);
    }
    case NVTEXT_AMD_ACTIVATION_SILU: {
      float const s = 1.f / (1.f + expf(-z));
      return s * (1.f + z * (1.f - s));
    }
    default: return 1.f;
  }
}

// An operand of a product: value (i, k) is data[i * of_i + k * of_k].
template <typename T>
struct Operand {
  const T* data;
  int64_t of_i, of_k;
  __device__ __forceinline__ float at(int64_t i, int64_t k) const { return static_cast<float>(data[i * of_i + k * of_k]); }
};

// What becomes of a sum over k.
template <typename T>
struct Epilogue {
  Rows<const T> bias, residual;
  Rows<T> out, preactivation;
  int activation;
  __device__ __forceinline__ void finish(float z, int64_t i, int64_t j) const
  {
    if (bias) z += static_cast<float>(bias.data[j]);
    if (preactivation) preactivation.row(i)[j] = static_cast<T>(z);
    z = activate(z, activation);
    if (residual) z += static_cast<float>(residual.row(i)[j]);
    out.row(i)[j] = static_cast<T>(z);
  }
};

// out (i, j) = sum over k of a (i, k) * b (j, k).  A workgroup a tile of 64 x 64, a thread 4 x 4 of it.
constexpr int kTile = 64, kDepth = 16;

template <typename T>
__global__ void __launch_bounds__(kThreads) product_kernel(Operand<T> a, Operand<T> b, int64_t m, int64_t n, int64_t depth, Epilogue<T> end)
{
  __shared__ float la[kDepth][kTile + 4], lb[kDepth][kTile + 4];
  int64_t const i0 = static_cast<int64_t>(blockIdx.y) * kTile, j0 = static_cast<int64_t>(blockIdx.x) * kTile;
  int const ti = threadIdx.x / 16 * 4, tj = threadIdx.x % 16 * 4;
  float sum[4][4] = {};
  for (int64_t k0 = 0; k0 < depth; k0 += kDepth) {
    for (int x = threadIdx.x; x < kTile * kDepth; x += kThreads) {
      // neighbouring threads read neighbouring values
      int const ia = a.of_k == 1 ? x / kDepth : x % kTile, ka = a.of_k == 1 ? x % kDepth : x / kTile;
      int const ib = b.of_k == 1 ? x / kDepth : x % kTile, kb = b.of_k == 1 ? x % kDepth : x / kTile;
      la[ka][ia] = i0 + ia < m && k0 + ka < depth ? a.at(i0 + ia, k0 + ka) : 0.f;
      lb[kb][ib] = j0 + ib < n && k0 + kb < depth ? b.at(j0 + ib, k0 + kb) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] += la[k][ti + i] * lb[k][tj + j];
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + ti + i < m && j0 + tj + j < n) end.finish(sum[i][j], i0 + ti + i, j0 + tj + j);
}

// d = grad * activation'(z) where it is wanted, and the sums of the columns of it: a workgroup 2048 columns and every
// gridDim.y-th row.
template <typename T>
__global__ void __launch_bounds__(kThreads)
activation_backward_kernel(Rows<const T> grad, Rows<const T> z, int activation, int64_t rows, int64_t cols, Rows<T> d, float* parts)
{
  int64_t const j = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * 8;
  if (j >= cols) return;
  float sum[8] = {};
  for (int64_t i = blockIdx.y; i < rows; i += gridDim.y) {
    float g[8], v[8];
    load8(g, grad.row(i) + j, cols - j);
    if (z) {
      load8(v, z.row(i) + j, cols - j);
#pragma unroll
      for (int k = 0; k < 8; ++k) g[k] *= slope(v[k], activation);
      if (d) store8(d.row(i) + j, g, cols - j);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) sum[k] += g[k];
  }
  if (parts) store8(parts + blockIdx.y * cols + j, sum, cols - j);
}

template <typename T>
void launch_product(Operand<T> const& a, Operand<T> const& b, int64_t m, int64_t n, int64_t depth, Epilogue<T> const& end, hipStream_t stream)
{
  hipLaunchKernelGGL(product_kernel<T>, dim3(static_cast<unsigned>((n + kTile - 1) / kTile), static_cast<unsigned>((m + kTile - 1) / kTile)), dim3(kThreads), 0, stream, a, b, m, n,
                     depth, end);
}

bool is_activation(int32_t a) { return a >= NVTEXT_AMD_ACTIVATION_NONE && a <= NVTEXT_AMD_ACTIVATION_SILU; }

// What the shapes of linear's matrices have in common with those of its gradients; nullptr if it holds.
const char* bad_shapes(const nvtext_amd_matrix* x, const nvtext_amd_matrix* weight)
{
  if (weight->cols != x->cols) return "x and weight must have the same number of inputs";
  if (weight->rows > INT32_MAX) return "invalid matrix sizes";
  return nullptr;
}

}  // namespace
}  // namespace nvtext_amd

extern "C" {

nvtext_amd_status nvtext_amd_linear(const nvtext_amd_matrix* x, const nvtext_amd_matrix* weight, const nvtext_amd_matrix* bias, int32_t activation,
                                    const nvtext_amd_matrix* residual, void* stream_, const nvtext_amd_allocator* mr_, const nvtext_amd_matrix* out,
                                    const nvtext_amd_matrix* preactivation)
{
  using namespace nvtext_amd;
  EntryScope const entry("nvtext_amd_linear");
  if (!x || !weight || !out) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  for (auto* m : {x, weight, bias, residual, out, preactivation}) {
    if (const char* bad = m ? bad_matrix(m) : nullptr) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
    if (m && m->type != x->type) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "all matrices must be of one type");
  }
  if (const char* bad = bad_shapes(x, weight)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  int64_t const m = x->rows, n = weight->rows, depth = x->cols;
  if (bias && !is_shape(bias, 1, n)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "bias must be a vector of a value for each output");
  for (auto* o : {residual, out, preactivation})
    if (o && !is_shape(o, m, n)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "out, residual and preactivation must have x's rows and weight's outputs");
  if (!is_activation(activation)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "unknown activation");
  if (m == 0 || n == 0) return NVTEXT_AMD_SUCCESS;
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  with_type(x->type, [&](auto zero) {
    using T        = decltype(zero);
    auto const xs  = rows_of<const T>(x);
    auto const ws  = rows_of<const T>(weight);
    ProfileScope const scope("linear", stream);
    launch_product<T>({xs.data, xs.stride, 1}, {ws.data, ws.stride, 1}, m, n, depth,
                      {rows_of<const T>(bias), rows_of<const T>(residual), rows_of<T>(out), rows_of<T>(preactivation), activation}, stream);
  });
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

nvtext_amd_status nvtext_amd_linear_backward(const nvtext_amd_matrix* grad, const nvtext_amd_matrix* x, const nvtext_amd_matrix* weight, int32_t activation,
                                             const nvtext_amd_matrix* preactivation, void* stream_, const nvtext_amd_allocator* mr_,
                                             const nvtext_amd_matrix* x_grad, const nvtext_amd_matrix* weight_grad, const nvtext_amd_matrix* bias_grad)
{
  using namespace nvtext_amd;
  EntryScope const entry("nvtext_amd_linear_backward");
  if (!grad || !x || !weight) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  for (auto* m : {grad, x, weight, preactivation, x_grad, weight_grad, bias_grad}) {
    if (const char* bad = m ? bad_matrix(m) : nullptr) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
    if (m && m->type != x->type) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "all matrices must be of one type");
  }
  if (const char* bad = bad_shapes(x, weight)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  int64_t const m = x->rows, n = weight->rows, depth = x->cols;
  for (auto* o : {grad, preactivation})
    if (o && !is_shape(o, m, n)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "grad and preactivation must have x's rows and weight's outputs");
  if (x_grad && !is_shape(x_grad, m, depth)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "x_grad must be of x's size");
  if (weight_grad && !is_shape(weight_grad, n, depth)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "weight_grad must be of weight's size");
  if (bias_grad && !is_shape(bias_grad, 1, n)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "bias_grad must be a vector of a value for each output");
  if (!is_activation(activation)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "unknown activation");
  if (activation != NVTEXT_AMD_ACTIVATION_NONE && !preactivation) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "the gradient of an activation needs what it was applied to");
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  Mr const mr{mr_, stream};
  bool const slopes   = activation != NVTEXT_AMD_ACTIVATION_NONE;
  int64_t const parts = std::max<int64_t>(1, std::min<int64_t>(m, 256));
  TempParts<2> const temp(mr, {slopes ? static_cast<size_t>(m * n) * type_bytes(x->type) : 0, bias_grad ? static_cast<size_t>(parts * n) * sizeof(float) : 0});
  if (!temp.ok()) return fail(NVTEXT_AMD_ALLOC_FAILED, "temporary allocation failed");
  with_type(x->type, [&](auto zero) {
    using T       = decltype(zero);
    auto const xs = rows_of<const T>(x), ws = rows_of<const T>(weight), gs = rows_of<const T>(grad);
    Rows<T> const d = slopes ? Rows<T>{temp.part<T>(0), n} : Rows<T>{nullptr, 0};
    float* const sums = bias_grad ? temp.part<float>(1) : nullptr;
    if (n > 0 && (slopes || bias_grad)) {
      ProfileScope const scope("linear_activation_backward", stream);
      hipLaunchKernelGGL(activation_backward_kernel<T>, dim3(static_cast<unsigned>((n + 8 * kThreads - 1) / (8 * kThreads)), static_cast<unsigned>(parts)), dim3(kThreads), 0, stream, gs,
                         slopes ? rows_of<const T>(preactivation) : Rows<const T>{nullptr, 0}, activation, m, n, d, sums);
      if (bias_grad) launch_add_parts(sums, parts, n, static_cast<T*>(bias_grad->data), stream);
    }
    Rows<const T> const ds = slopes ? Rows<const T>{d.data, d.stride} : gs;
    auto const plain = [](const nvtext_amd_matrix* o) { return Epilogue<T>{{nullptr, 0}, {nullptr, 0}, rows_of<T>(o), {nullptr, 0}, NVTEXT_AMD_ACTIVATION_NONE}; };
    if (x_grad && m > 0 && depth > 0) {
      ProfileScope const scope("linear_x_backward", stream);
      launch_product<T>({ds.data, ds.stride, 1}, {ws.data, 1, ws.stride}, m, depth, n, plain(x_grad), stream);
    }
    if (weight_grad && n > 0 && depth > 0) {
      ProfileScope const scope("linear_weight_backward", stream);
      launch_product<T>({ds.data, 1, ds.stride}, {xs.data, 1, xs.stride}, n, depth, m, plain(weight_grad), stream);
    }
  });
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

}  // extern "C"
