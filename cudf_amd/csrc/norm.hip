// dropout and layer norm with their gradients.
#include "encoder.cuh"

#include <algorithm>
#include <type_traits>

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

// The sum over the lanes of a row's WAVES wavefronts.  lds: a value a wavefront, which two calls in turn do not share: that one
// barrier a call is enough.
template <int WAVES>
__device__ __forceinline__ float row_sum(float v, float* lds)
{
  v = wave_sum(v);
  if constexpr (WAVES > 1) {
    int const wave = threadIdx.x / kWave % WAVES;
    if (lane_id() == 0) lds[wave] = v;
    lds_barrier();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v += lds[w];
  }
  return v;
}

// Rows that fit into registers: WAVES wavefronts a row, BLOCKS times eight values a lane, each read once; the mean first, then the
// squares around it.  A workgroup takes several rows one after the other and keeps the weights.
template <typename T, int WAVES, int BLOCKS>
__global__ void __launch_bounds__(WAVES > 4 ? WAVES * kWave : kThreads)
layer_norm_kernel(Rows<const T> x, Rows<const T> residual, Weights weight, Weights bias, float eps, Dropout d, Rows<T> out, Rows<T> sum, float* mean_out,
                  float* rstd_out, int64_t rows, int64_t cols)
{
  constexpr int kThreadsHere = WAVES > 4 ? WAVES * kWave : kThreads, kRows = kThreadsHere / (WAVES * kWave);
  __shared__ float lds[2][kRows][WAVES];
  int const place = threadIdx.x / (WAVES * kWave), lane = threadIdx.x % (WAVES * kWave);  // the row of the workgroup, the lane of the row
  float const width = static_cast<float>(cols);
  float w[BLOCKS][8], c[BLOCKS][8];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b) {
    int64_t const j = (static_cast<int64_t>(b) * WAVES * kWave + lane) * 8;
    weight.load<T>(w[b], j, cols - j);
    bias.load<T>(c[b], j, cols - j);
  }
  // (all wavefronts of a workgroup go round equally often, for the barriers)
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kRows; first < rows; first += static_cast<int64_t>(gridDim.x) * kRows) {
    int64_t const i = first + place < rows ? first + place : rows - 1;  // (behind the last: the last once more)
    typename Eight<T>::type vx[BLOCKS], vr[BLOCKS];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      int64_t const j = (static_cast<int64_t>(b) * WAVES * kWave + lane) * 8;
      vx[b]           = load_raw8<T>(x.row(i) + j, cols - j);
      if (residual) vr[b] = load_raw8<T>(residual.row(i) + j, cols - j);
    }
    float f[BLOCKS][8], s = 0.f;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      widen<T>(f[b], vx[b]);
      if (d.dropped) d.apply(f[b], i, static_cast<int64_t>(b) * WAVES * kWave + lane);
      if (residual) {
        float r[8];
        widen<T>(r, vr[b]);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[b][k] += r[k];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) s += f[b][k];
    }
    float const mean = row_sum<WAVES>(s, lds[0][place]) / width;  // (not times 1 / width: the mean of equal values is that value)
    s                = 0.f;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      int64_t const left = cols - (static_cast<int64_t>(b) * WAVES * kWave + lane) * 8;
#pragma unroll
      for (int k = 0; k < 8; ++k) s += k < left ? (f[b][k] - mean) * (f[b][k] - mean) : 0.f;
    }
    float const rstd = 1.f / sqrtf(row_sum<WAVES>(s, lds[1][place]) / width + eps);
    if (first + place < rows) {
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        int64_t const j = (static_cast<int64_t>(b) * WAVES * kWave + lane) * 8;
        if (sum) store8(sum.row(i) + j, f[b], cols - j);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[b][k] = (f[b][k] - mean) * rstd * w[b][k] + c[b][k];
        store8(out.row(i) + j, f[b], cols - j);
      }
      if (lane == 0) {
        if (mean_out) mean_out[i] = mean;
        if (rstd_out) rstd_out[i] = rstd;
      }
    }
  }
}

// Wider ones: a workgroup a row, which it goes through three times.
template <typename T>
__global__ void __launch_bounds__(kThreads) wide_layer_norm_kernel(Rows<const T> x, Rows<const T> residual, Weights weight, Weights bias, float eps, Dropout d,
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

// The gradient of rows that fit into registers, read once.  The workgroup's sums over its rows of grad * h and of grad go to parts
// [workgroup] and [number of workgroups + workgroup]: a lane adds them up for its columns, and the workgroup's rows are added up in
// order in the end.
template <typename T, int WAVES, int BLOCKS>
__global__ void __launch_bounds__(WAVES > 4 ? WAVES * kWave : kThreads)
layer_norm_backward_kernel(Rows<const T> grad, Rows<const T> sum, const float* mean_in, const float* rstd_in, Weights weight, Rows<const T> sum_grad, Dropout d, Rows<T> x_grad,
                           Rows<T> residual_grad, float* parts, int64_t rows, int64_t cols)
{
  constexpr int kThreadsHere = WAVES > 4 ? WAVES * kWave : kThreads, kRows = kThreadsHere / (WAVES * kWave), kCols = WAVES * BLOCKS * kWave * 8;
  __shared__ float lds[2][kRows][WAVES];
  __shared__ float joined[kRows > 1 ? 2 : 1][kRows > 1 ? kCols : 1];
  int const place = threadIdx.x / (WAVES * kWave), lane = threadIdx.x % (WAVES * kWave);
  float const width = static_cast<float>(cols);
  float w[BLOCKS][8], dw[BLOCKS][8], db[BLOCKS][8];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b) {
    int64_t const j = (static_cast<int64_t>(b) * WAVES * kWave + lane) * 8;
    weight.load<T>(w[b], j, cols - j);
#pragma unroll
    for (int k = 0; k < 8; ++k) dw[b][k] = db[b][k] = 0.f;
  }
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kRows; first < rows; first += static_cast<int64_t>(gridDim.x) * kRows) {
    bool const here  = first + place < rows;
    int64_t const i  = here ? first + place : rows - 1;
    float const mean = mean_in[i], rstd = rstd_in[i];
    typename Eight<T>::type vg[BLOCKS], vs[BLOCKS], ve[BLOCKS];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      int64_t const j = (static_cast<int64_t>(b) * WAVES * kWave + lane) * 8;
      vg[b]           = load_raw8<T>(grad.row(i) + j, cols - j);
      vs[b]           = load_raw8<T>(sum.row(i) + j, cols - j);
      if (sum_grad) ve[b] = load_raw8<T>(sum_grad.row(i) + j, cols - j);
    }
    float sa = 0.f, sh = 0.f;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      float g[8], s[8];
      widen<T>(g, vg[b]);
      widen<T>(s, vs[b]);
#pragma unroll
      for (int k = 0; k < 8; ++k) {  // (behind the last column grad is 0)
        float const h = (s[k] - mean) * rstd, gh = g[k] * h;
        sa += g[k] * w[b][k];
        sh += gh * w[b][k];
        if (here) {
          dw[b][k] += gh;
          db[b][k] += g[k];
        }
      }
    }
    float const ma = row_sum<WAVES>(sa, lds[0][place]) / width, mh = row_sum<WAVES>(sh, lds[1][place]) / width;
    if (here) {
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        int64_t const j = (static_cast<int64_t>(b) * WAVES * kWave + lane) * 8;
        float g[8], s[8], e[8];
        widen<T>(g, vg[b]);
        widen<T>(s, vs[b]);
        if (sum_grad) widen<T>(e, ve[b]);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          s[k] = rstd * (g[k] * w[b][k] - ma - (s[k] - mean) * rstd * mh);
          if (sum_grad) s[k] += e[k];
        }
        store8(residual_grad.row(i) + j, s, cols - j);
        if (x_grad) {
          if (d.dropped) d.apply(s, i, static_cast<int64_t>(b) * WAVES * kWave + lane);
          store8(x_grad.row(i) + j, s, cols - j);
        }
      }
    }
  }
  if (!parts) return;
  float* const out[2] = {parts + blockIdx.x * cols, parts + (static_cast<int64_t>(gridDim.x) + blockIdx.x) * cols};
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if constexpr (kRows > 1) __syncthreads();
    if (place != r) continue;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      int const j = (b * WAVES * kWave + lane) * 8;
      if constexpr (kRows > 1) {
        if (r > 0) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            dw[b][k] += joined[0][j + k];
            db[b][k] += joined[1][j + k];
          }
        }
        if (r + 1 < kRows) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            joined[0][j + k] = dw[b][k];
            joined[1][j + k] = db[b][k];
          }
          continue;
        }
      }
      store8(out[0] + j, dw[b], cols - j);
      store8(out[1] + j, db[b], cols - j);
    }
  }
}

// The gradient of wider rows, in two kernels.
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

// Calls f with the wavefronts a row and the blocks of eight values a lane that hold a row of `cols` values, or with none: up to 2048
// values one wavefront, which needs no barrier.
template <typename F>
void with_shape(int64_t cols, F&& f)
{
  using std::integral_constant;
  if (cols <= 512) f(integral_constant<int, 1>{}, integral_constant<int, 1>{});
  else if (cols <= 1024) f(integral_constant<int, 1>{}, integral_constant<int, 2>{});
  else if (cols <= 1536) f(integral_constant<int, 1>{}, integral_constant<int, 3>{});
  else if (cols <= 2048) f(integral_constant<int, 1>{}, integral_constant<int, 4>{});
  else if (cols <= 4096) f(integral_constant<int, 4>{}, integral_constant<int, 2>{});
  else if (cols <= 8192) f(integral_constant<int, 4>{}, integral_constant<int, 4>{});
  else if (cols <= 16384) f(integral_constant<int, 16>{}, integral_constant<int, 2>{});
  else f(integral_constant<int, 0>{}, integral_constant<int, 0>{});
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
    with_shape(x->cols, [&](auto waves, auto blocks) {
      constexpr int W = decltype(waves)::value, B = decltype(blocks)::value;
      auto const launch = [&](auto kernel, int threads, int64_t groups) {
        hipLaunchKernelGGL(kernel, dim3(grid_for(groups, 2048 / threads)), dim3(threads), 0, stream, rows_of<const T>(x), rows_of<const T>(residual), Weights{weight->data, weight->type},
                           Weights{bias->data, bias->type}, static_cast<float>(eps), d, rows_of<T>(out), rows_of<T>(sum), mean, rstd, x->rows, x->cols);
      };
      if constexpr (W == 0)
        launch(wide_layer_norm_kernel<T>, kThreads, x->rows);
      else if constexpr (W > 4)
        launch(layer_norm_kernel<T, W, B>, W * kWave, x->rows);
      else
        launch(layer_norm_kernel<T, W, B>, kThreads, (x->rows * W + 3) / 4);
    });
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
  int64_t parts      = 0;
  with_shape(cols, [&](auto waves, auto) {
    constexpr int W = decltype(waves)::value;
    // rows = 0: the sums of the weights' gradients are zeros, of one part
    parts = W == 0 ? std::max<int64_t>(1, std::min<int64_t>(rows, 256)) : grid_for(W > 4 ? rows : (rows * W + 3) / 4, W > 4 ? 1 : 4);
  });
  Temp const sums(mr, weight_grad ? static_cast<size_t>(2 * parts * cols) * sizeof(float) : 0);
  if (!sums.ok()) return fail(NVTEXT_AMD_ALLOC_FAILED, "temporary allocation failed");
  Weights const w{weight->data, weight->type};
  with_type(grad->type, [&](auto zero) {
    using T = decltype(zero);
    with_shape(cols, [&](auto waves, auto blocks) {
      constexpr int W = decltype(waves)::value, B = decltype(blocks)::value;
      if constexpr (W > 0) {
        ProfileScope const scope("layer_norm_backward", stream);
        hipLaunchKernelGGL(HIP_KERNEL_NAME(layer_norm_backward_kernel<T, W, B>), dim3(static_cast<unsigned>(parts)), dim3(W > 4 ? W * kWave : kThreads), 0, stream, rows_of<const T>(grad),
                           rows_of<const T>(sum), mean, rstd, w, rows_of<const T>(sum_grad), d, rows_of<T>(x_grad), rows_of<T>(residual_grad), weight_grad ? sums.as<float>() : nullptr,
                           rows, cols);
      } else {
        if (weight_grad) {
          ProfileScope const scope("layer_norm_weights_backward", stream);
          hipLaunchKernelGGL(layer_norm_weights_backward_kernel<T>, dim3(static_cast<unsigned>((cols + 8 * kThreads - 1) / (8 * kThreads)), static_cast<unsigned>(parts)),
                             dim3(kThreads), 0, stream, rows_of<const T>(grad), rows_of<const T>(sum), mean, rstd, rows, cols, sums.as<float>());
        }
        if (rows > 0) {
          ProfileScope const scope("layer_norm_rows_backward", stream);
          hipLaunchKernelGGL(layer_norm_rows_backward_kernel<T>, dim3(grid_for(rows, 8)), dim3(kThreads), 0, stream, rows_of<const T>(grad), rows_of<const T>(sum), mean, rstd, w,
                             rows_of<const T>(sum_grad), d, rows_of<T>(x_grad), rows_of<T>(residual_grad), rows, cols);
        }
      }
    });
  });
  if (weight_grad)
    with_type(weight->type, [&](auto zero) {
      using W = decltype(zero);
      ProfileScope const scope("layer_norm_add_parts", stream);
      launch_add_parts(sums.as<float>(), parts, cols, static_cast<W*>(weight_grad->data), static_cast<W*>(bias_grad->data), stream);
    });
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

}  // extern "C"
