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
    auto v = load_row8<T>(x.row(i), b * 8, cols);
    settle_row8<T>(v, b * 8, cols);
    widen<T>(f, v);
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
  __device__ __forceinline__ void load(float (&f)[8], int64_t j, int64_t cols) const
  {
    if (type == NVTEXT_AMD_TYPE_FLOAT32)
      load_of(f, static_cast<const float*>(data), j, cols);
    else
      load_of(f, static_cast<const T*>(data), j, cols);
  }
  template <typename W>
  static __device__ __forceinline__ void load_of(float (&f)[8], const W* w, int64_t j, int64_t cols)
  {
    auto v = load_row8<W>(w, j, cols);
    settle_row8<W>(v, j, cols);
    widen<W>(f, v);
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

// The sum over the LANES lanes of a row: neighbours of a wavefront, or whole wavefronts.  lds (of several wavefronts): a value each,
// which two calls in turn do not share: that one barrier a call is enough.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* lds)
{
  if constexpr (LANES < kWave) {
    v += dpp_zero_f<0xB1, 0xf>(v);   // quad_perm 1 0 3 2
    v += dpp_zero_f<0x4E, 0xf>(v);   // quad_perm 2 3 0 1
    v += dpp_zero_f<0x141, 0xf>(v);  // row_half_mirror
    v += dpp_zero_f<0x140, 0xf>(v);  // row_mirror
    if constexpr (LANES == 32) v += __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, v), 0x401F));  // the other 16
    return v;
  } else {
    v = wave_sum(v);
    if constexpr (LANES > kWave) {
      constexpr int kWaves = LANES / kWave;
      if (lane_id() == 0) lds[threadIdx.x / kWave % kWaves] = v;
      lds_barrier();
      v = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) v += lds[w];
    }
    return v;
  }
}

// A row of `cols` values over LANES lanes with BLOCKS times eight values each.
constexpr int threads_of(int lanes, int threads) { return lanes > threads ? lanes : threads; }

template <int LANES, int BLOCKS, int THREADS = kThreads>
struct Shape {
  static constexpr int kThreadsHere = threads_of(LANES, THREADS);
  static constexpr int kRows        = kThreadsHere / LANES;  // that a workgroup has at a time
  static constexpr int kCols        = LANES * BLOCKS * 8;        // at most
  static constexpr int kWaves       = LANES > kWave ? LANES / kWave : 1;
  static __device__ __forceinline__ unsigned block(int b, int lane) { return b * LANES + lane; }
  // the row of the workgroup that a lane works on: known to be one for a wavefront, where it is, so that addresses are scalars
  static __device__ __forceinline__ int place()
  {
    int const p = threadIdx.x / LANES;
    return LANES < kWave ? p : __builtin_amdgcn_readfirstlane(p);
  }
};

// Rows that fit into registers, each read once; the mean first, then the squares around it.  A workgroup takes several rows one
// after the other and keeps the weights.  Bound by memory: 32768 rows of 1024 16-bit values with dropout and residual 48 us,
// 5.6 TB/s; the generator's 60 instructions for eight values are hidden.
template <typename T, int LANES, int BLOCKS>
__global__ void __launch_bounds__(threads_of(LANES, kThreads))
layer_norm_kernel(Rows<const T> x, Rows<const T> residual, Weights weight, Weights bias, float eps, Dropout d, Rows<T> out, Rows<T> sum, float* mean_out,
                  float* rstd_out, int64_t rows, int64_t cols)
{
  using S = Shape<LANES, BLOCKS>;
  __shared__ float lds[2][S::kRows][S::kWaves];
  int const place = S::place(), lane = threadIdx.x % LANES;  // the row of the workgroup, the lane of the row
  float const width = static_cast<float>(cols);
  float w[BLOCKS][8], c[BLOCKS][8];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b) {
    unsigned const j = S::block(b, lane) * 8;
    weight.load<T>(w[b], j, cols);
    bias.load<T>(c[b], j, cols);
  }
  // (all wavefronts of a workgroup go round equally often, for the barriers)
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * S::kRows; first < rows; first += static_cast<int64_t>(gridDim.x) * S::kRows) {
    int64_t const i = first + place < rows ? first + place : rows - 1;  // (behind the last: the last once more)
    typename Eight<T>::type vx[BLOCKS], vr[BLOCKS];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      unsigned const j = S::block(b, lane) * 8;
      vx[b]           = load_row8<T>(x.row(i), j, cols);
      if (residual) vr[b] = load_row8<T>(residual.row(i), j, cols);
    }
    if (cols != S::kCols) {
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        unsigned const j = S::block(b, lane) * 8;
        settle_row8<T>(vx[b], j, cols);
        if (residual) settle_row8<T>(vr[b], j, cols);
      }
    }
    float f[BLOCKS][8], s = 0.f;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      widen<T>(f[b], vx[b]);
      if (d.dropped) d.apply(f[b], i, S::block(b, lane));
      if (residual) {
        float r[8];
        widen<T>(r, vr[b]);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[b][k] += r[k];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) s += f[b][k];
    }
    float const mean = row_sum<LANES>(s, lds[0][place]) / width;  // (not times 1 / width: the mean of equal values is that value)
    s                = 0.f;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      int64_t const left = cols - static_cast<int64_t>(S::block(b, lane) * 8);
#pragma unroll
      for (int k = 0; k < 8; ++k) s += k < left ? (f[b][k] - mean) * (f[b][k] - mean) : 0.f;
    }
    float const rstd = 1.f / sqrtf(row_sum<LANES>(s, lds[1][place]) / width + eps);
    if (first + place < rows) {
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        unsigned const j = S::block(b, lane) * 8;
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
      weight.load<T>(w, b * 8, cols);
      bias.load<T>(c, b * 8, cols);
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

// Where the weights' gradients go.
struct WeightGrads {
  float* parts;  // of several workgroups: [workgroup] and [number of workgroups + workgroup]
  void *weight, *bias;
  int32_t type;
  template <typename T>
  __device__ __forceinline__ void store(int which, float const (&f)[8], int64_t j, int64_t cols) const
  {
    if (gridDim.x > 1) {
      store8(parts + (which * static_cast<int64_t>(gridDim.x) + blockIdx.x) * cols + j, f, cols - j);
    } else if (type == NVTEXT_AMD_TYPE_FLOAT32) {
      store8(static_cast<float*>(which == 0 ? weight : bias) + j, f, cols - j);
    } else {
      store8(static_cast<T*>(which == 0 ? weight : bias) + j, f, cols - j);
    }
  }
  template <typename T>
  __device__ __forceinline__ void store_one(int which, float f, int64_t j, int64_t cols) const
  {
    if (gridDim.x > 1)
      parts[(which * static_cast<int64_t>(gridDim.x) + blockIdx.x) * cols + j] = f;
    else if (type == NVTEXT_AMD_TYPE_FLOAT32)
      static_cast<float*>(which == 0 ? weight : bias)[j] = f;
    else
      static_cast<T*>(which == 0 ? weight : bias)[j] = static_cast<T>(f);
  }
};

// The gradient of rows that fit into registers, read once.  A lane adds up grad * h and grad for its columns, the workgroup's rows
// are added up in order in the end.  Bound by memory: 20011 rows of 1536 16-bit values with dropout 56 us, 4.4 TB/s, and 5 us
// for the parts of 512 workgroups.
template <typename T, int LANES, int BLOCKS, int THREADS>
__global__ void __launch_bounds__(threads_of(LANES, THREADS))
layer_norm_backward_kernel(Rows<const T> grad, Rows<const T> sum, const float* mean_in, const float* rstd_in, Weights weight, Rows<const T> sum_grad, Dropout d, Rows<T> x_grad,
                           Rows<T> residual_grad, WeightGrads weights, int64_t rows, int64_t cols)
{
  using S             = Shape<LANES, BLOCKS, THREADS>;
  constexpr int kRows = S::kRows;
  __shared__ float lds[2][kRows][S::kWaves];
  __shared__ float joined[kRows > 1 ? kRows * S::kCols : 1];
  int const place = S::place(), lane = threadIdx.x % LANES;
  float const width = static_cast<float>(cols);
  float w[BLOCKS][8], dw[BLOCKS][8], db[BLOCKS][8];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b) {
    unsigned const j = S::block(b, lane) * 8;
    weight.load<T>(w[b], j, cols);
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
      unsigned const j = S::block(b, lane) * 8;
      vg[b]           = load_row8<T>(grad.row(i), j, cols);
      vs[b]           = load_row8<T>(sum.row(i), j, cols);
      if (sum_grad) ve[b] = load_row8<T>(sum_grad.row(i), j, cols);
    }
    if (cols != S::kCols) {
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        unsigned const j = S::block(b, lane) * 8;
        settle_row8<T>(vg[b], j, cols);
        settle_row8<T>(vs[b], j, cols);
        if (sum_grad) settle_row8<T>(ve[b], j, cols);
      }
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
    float const ma = row_sum<LANES>(sa, lds[0][place]) / width, mh = row_sum<LANES>(sh, lds[1][place]) / width;
    if (here) {
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        unsigned const j = S::block(b, lane) * 8;
        asm volatile("" : "+v"(vg[b]), "+v"(vs[b]));  // (widened once more: kept as floats they took 285 registers instead of 211)
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
          if (d.dropped) d.apply(s, i, S::block(b, lane));
          store8(x_grad.row(i) + j, s, cols - j);
        }
      }
    }
  }
  if (!weights.weight) return;
  if constexpr (kRows == 1) {
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      unsigned const j = S::block(b, lane) * 8;
      weights.store<T>(0, dw[b], j, cols);
      weights.store<T>(1, db[b], j, cols);
    }
  } else {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int k = 0; k < 8; ++k) joined[place * S::kCols + S::block(b, lane) * 8 + k] = which == 0 ? dw[b][k] : db[b][k];
      __syncthreads();
      for (int j = threadIdx.x; j < cols; j += S::kThreadsHere) {
        float all = joined[j];
#pragma unroll
        for (int r = 1; r < kRows; ++r) all += joined[r * S::kCols + j];
        weights.store_one<T>(which, all, j, cols);
      }
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
      weight.load<T>(w, b * 8, cols);
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
      weight.load<T>(w, b * 8, cols);
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

// Calls f with the lanes a row and the blocks of eight values a lane that hold a row of `cols` values, or with none: up to 2048
// values one wavefront, which needs no barrier; a quarter or half of one up to 128 or 256 (40,000 rows of 100 values, one to a
// wavefront: 36 us).
template <typename F>
void with_shape(int64_t cols, F&& f)
{
  using std::integral_constant;
  if (cols <= 128) f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  else if (cols <= 256) f(integral_constant<int, 32>{}, integral_constant<int, 1>{});
  else if (cols <= 512) f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (cols <= 1024) f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  else if (cols <= 1536) f(integral_constant<int, 64>{}, integral_constant<int, 3>{});
  else if (cols <= 2048) f(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  else if (cols <= 4096) f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  else if (cols <= 8192) f(integral_constant<int, 256>{}, integral_constant<int, 4>{});
  else if (cols <= 16384) f(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
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
    with_shape(x->cols, [&](auto lanes, auto blocks) {
      constexpr int L = decltype(lanes)::value, B = decltype(blocks)::value;
      auto const launch = [&](auto kernel, int threads, int64_t groups) {
        hipLaunchKernelGGL(kernel, dim3(grid_for(groups, 2048 / threads)), dim3(threads), 0, stream, rows_of<const T>(x), rows_of<const T>(residual), Weights{weight->data, weight->type},
                           Weights{bias->data, bias->type}, static_cast<float>(eps), d, rows_of<T>(out), rows_of<T>(sum), mean, rstd, x->rows, x->cols);
      };
      if constexpr (L == 0)
        launch(wide_layer_norm_kernel<T>, kThreads, x->rows);
      else
        launch(layer_norm_kernel<T, L, B>, Shape<L, B>::kThreadsHere, (x->rows + Shape<L, B>::kRows - 1) / Shape<L, B>::kRows);
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
  // the workgroups: as many as the registers let run at a time (32768 rows of 1024 16-bit values, 3 a CU: 73 us; 4: 83), and one
  // alone, of twice the wavefronts, for rows that it goes through in kAlone rounds: it needs no parts and no second launch (54 rows
  // of 192 values: 14 us for the call instead of 20)
  constexpr int kMany = 2 * kThreads, kAlone = 6;
  int64_t groups      = 0;
  bool wide = false, alone = false;
  with_shape(cols, [&](auto lanes, auto blocks) {
    constexpr int L = decltype(lanes)::value, B = decltype(blocks)::value;
    wide            = L == 0;
    if constexpr (L > 0) {
      groups = (rows + Shape<L, B>::kRows - 1) / Shape<L, B>::kRows;
      alone  = rows <= kAlone * Shape<L, B, kMany>::kRows;
    } else {
      groups = std::min<int64_t>(rows, 256);
    }
    groups = alone ? 1 : grid_for(groups, L > kThreads ? 1 : B <= 1 ? 4 : B == 2 && grad->type != NVTEXT_AMD_TYPE_FLOAT32 ? 3 : 2);
  });
  bool const parts = weight_grad && (wide || groups > 1);
  Temp const sums(mr, parts ? static_cast<size_t>(2 * groups * cols) * sizeof(float) : 0);
  if (!sums.ok()) return fail(NVTEXT_AMD_ALLOC_FAILED, "temporary allocation failed");
  Weights const w{weight->data, weight->type};
  WeightGrads const grads{sums.as<float>(), weight_grad ? weight_grad->data : nullptr, bias_grad ? bias_grad->data : nullptr, weight->type};
  with_type(grad->type, [&](auto zero) {
    using T = decltype(zero);
    with_shape(cols, [&](auto lanes, auto blocks) {
      constexpr int L = decltype(lanes)::value, B = decltype(blocks)::value;
      if constexpr (L > 0) {
        ProfileScope const scope("layer_norm_backward", stream);
        auto const launch = [&](auto kernel, int threads) {
          hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(groups)), dim3(threads), 0, stream, rows_of<const T>(grad), rows_of<const T>(sum), mean, rstd, w, rows_of<const T>(sum_grad), d,
                             rows_of<T>(x_grad), rows_of<T>(residual_grad), grads, rows, cols);
        };
        constexpr int kMost = L < kMany ? kMany : kThreads;
        if (alone)
          launch(layer_norm_backward_kernel<T, L, B, kMost>, Shape<L, B, kMost>::kThreadsHere);
        else
          launch(layer_norm_backward_kernel<T, L, B, kThreads>, Shape<L, B>::kThreadsHere);
      } else {
        if (weight_grad) {
          ProfileScope const scope("layer_norm_weights_backward", stream);
          hipLaunchKernelGGL(layer_norm_weights_backward_kernel<T>, dim3(static_cast<unsigned>((cols + 8 * kThreads - 1) / (8 * kThreads)), static_cast<unsigned>(groups)),
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
  if (parts)
    with_type(weight->type, [&](auto zero) {
      using W = decltype(zero);
      ProfileScope const scope("layer_norm_add_parts", stream);
      launch_add_parts(sums.as<float>(), groups, cols, static_cast<W*>(weight_grad->data), static_cast<W*>(bias_grad->data), stream);
    });
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

}  // extern "C"
