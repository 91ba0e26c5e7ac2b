// Shared by the encoder operators (embedding, dropout, layer norm, linear): element types, eight values at a time, the
// dropout's generator, sums over a wavefront and over columns, and the checks of matrices.
#pragma once

#include "../../include/nvtext_amd_encoder.h"
#include "common.cuh"

#include <algorithm>

namespace nvtext_amd {

using half_t = _Float16;
using bf16_t = __bf16;

// calls f with a value of the element type
template <typename F>
inline auto with_type(int32_t type, F&& f)
{
  if (type == NVTEXT_AMD_TYPE_FLOAT16) return f(half_t{});
  if (type == NVTEXT_AMD_TYPE_BFLOAT16) return f(bf16_t{});
  return f(float{});
}

inline size_t type_bytes(int32_t type) { return type == NVTEXT_AMD_TYPE_FLOAT32 ? 4 : 2; }

// What a kernel is given of a matrix.
template <typename T>
struct Rows {
  T* data;
  int64_t stride;
  __device__ __forceinline__ T* row(int64_t i) const { return data + i * stride; }
  __host__ __device__ __forceinline__ explicit operator bool() const { return data != nullptr; }
};

template <typename T>
inline Rows<T> rows_of(const nvtext_amd_matrix* m)
{
  return m ? Rows<T>{static_cast<T*>(m->data), m->rows < 2 ? m->cols : m->stride} : Rows<T>{nullptr, 0};
}

// ------------------------------------------------------------------ checks
// nullptr if `m` can be used, else what is wrong with it
inline const char* bad_matrix(const nvtext_amd_matrix* m)
{
  if (m->type != NVTEXT_AMD_TYPE_FLOAT32 && m->type != NVTEXT_AMD_TYPE_FLOAT16 && m->type != NVTEXT_AMD_TYPE_BFLOAT16)
    return "matrices must be of FLOAT32, FLOAT16 or BFLOAT16";
  if (m->rows < 0 || m->cols < 0 || m->rows > (int64_t{1} << 40) || m->cols > INT32_MAX) return "invalid matrix sizes";
  if (m->rows >= 2 && (m->stride < m->cols || m->stride > (int64_t{1} << 40))) return "a matrix' stride must not be less than its width";
  if (m->rows > 0 && m->cols > 0) {
    if (!m->data) return "a matrix has no data";
    if (reinterpret_cast<uintptr_t>(m->data) % type_bytes(m->type) != 0) return "a matrix must be aligned to its type";
  }
  return nullptr;
}

inline bool is_shape(const nvtext_amd_matrix* m, int64_t rows, int64_t cols) { return m->rows == rows && m->cols == cols; }

// ------------------------------------------------------------------ workgroups
// A dimension of a launch counts threads in 32 bits: of 2^32 and more the runtime starts what is left modulo 2^32, without an error.
// Workgroups beyond 2^31 threads lie in several rows of the second dimension, whose last one may go on past the end.
inline dim3 grid_of(int64_t blocks, int threads)
{
  int64_t const most = (int64_t{1} << 31) / threads, rows = std::max<int64_t>(1, (blocks + most - 1) / most);
  return dim3(static_cast<unsigned>((blocks + rows - 1) / rows), static_cast<unsigned>(rows));
}

__device__ __forceinline__ int64_t block_number() { return static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x; }

// ------------------------------------------------------------------ eight values
// Rows need not begin at multiples of 16 bytes: global loads and stores of four words take any address of the element
// type's alignment, at a cost only where they cross a cache line.
template <typename T>
struct Eight {
  typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

// values p[0 .. n), zeros from n on
template <typename T>
__device__ __forceinline__ void load8(float (&f)[8], const T* p, int64_t n)
{
  if (n >= 8) {
    auto const v = *reinterpret_cast<const typename Eight<T>::type*>(p);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = static_cast<float>(v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = k < n ? static_cast<float>(p[k]) : 0.f;
  }
}

// PAST: past the caches
template <bool PAST = false, typename T>
__device__ __forceinline__ void store8(T* p, float const (&f)[8], int64_t n)
{
  if (n >= 8) {
    typename Eight<T>::type v;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = static_cast<T>(f[k]);
    if constexpr (PAST)
      __builtin_nontemporal_store(v, reinterpret_cast<typename Eight<T>::type*>(p));
    else
      *reinterpret_cast<typename Eight<T>::type*>(p) = v;
  } else if (n > 0) {
    // four, two and one of them
    typedef T V4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    typedef T V2 __attribute__((ext_vector_type(2), aligned(sizeof(T))));
    T v[4] = {static_cast<T>(f[0]), static_cast<T>(f[1]), static_cast<T>(f[2]), static_cast<T>(f[3])};
    if (n & 4) {
      *reinterpret_cast<V4*>(p) = V4{v[0], v[1], v[2], v[3]};
      p += 4;
#pragma unroll
      for (int k = 0; k < 3; ++k) v[k] = static_cast<T>(f[4 + k]);
    }
    if (n & 2) {
      *reinterpret_cast<V2*>(p) = V2{v[0], v[1]};
      p += 2;
      v[0] = v[2];
    }
    if (n & 1) *p = v[0];
  }
}

// values p[0 .. n) as they are, zeros from n on
template <typename T>
__device__ __forceinline__ typename Eight<T>::type load_raw8(const T* p, int64_t n)
{
  typename Eight<T>::type v{};
  if (n >= 8) {
    v = *reinterpret_cast<const typename Eight<T>::type*>(p);
  } else if (n > 0) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) v[k] = p[k];
  }
  return v;
}

// Values j .. j + 7 of a row of `cols`, in two steps, so that several loads are on their way before the first is waited for, and
// without a condition on any of them: a lane behind the last eight values loads these, and the second step moves its own to the
// front and puts zeros behind them.  (Loaded one by one under conditions, what was left of rows of 1023 values doubled the time of
// a layer norm.)
template <typename T>
__device__ __forceinline__ typename Eight<T>::type load_row8(const T* row, int64_t j, int64_t cols)
{
  if (cols >= 8) return *reinterpret_cast<const typename Eight<T>::type*>(row + (j + 8 <= cols ? j : cols - 8));
  return load_raw8<T>(row + j, cols - j);
}

template <typename T>
__device__ __forceinline__ void settle_row8(typename Eight<T>::type& v, int64_t j, int64_t cols)
{
  if (cols < 8) return;
  constexpr int kWords = 8 * sizeof(T) / 4, kEach = 4 / sizeof(T);  // 32-bit words, and values in one
  typedef uint32_t W __attribute__((ext_vector_type(kWords)));
  W w             = __builtin_bit_cast(W, v);
  int const ahead = j + 8 > cols ? static_cast<int>(j + 8 - cols) : 0;
  if (cols % 8 != 0) {  // (the same for all lanes: no width is left to a branch of single lanes)
    if constexpr (kEach == 2) {
#pragma unroll
      for (int k = 0; k < kWords; ++k) w[k] = ahead & 1 ? __builtin_amdgcn_alignbit(k + 1 < kWords ? w[k + 1] : 0u, w[k], 16) : w[k];
    }
#pragma unroll
    for (int by = 1; by < kWords; by *= 2) {
#pragma unroll
      for (int k = 0; k < kWords; ++k) w[k] = !(ahead & by * kEach) ? w[k] : k + by < kWords ? w[k + by] : 0u;
    }
  }
#pragma unroll
  for (int k = 0; k < kWords; ++k) w[k] = ahead >= 8 ? 0u : w[k];
  v = __builtin_bit_cast(typename Eight<T>::type, w);
}

template <typename T>
__device__ __forceinline__ void widen(float (&f)[8], typename Eight<T>::type const& v)
{
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = static_cast<float>(v[k]);
}

// ------------------------------------------------------------------ dropout
// Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011): ten rounds
// of two 32 x 32 -> 64 bit products each, one instruction apiece here.  A counter gives four words, eight draws of 16 bits.
__device__ __forceinline__ uint4 philox4x32(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1)
{
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    uint64_t const a = static_cast<uint64_t>(c0) * 0xD2511F53u;
    uint64_t const b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// The probability rounded to 1/65536, and the reciprocal of what is left of it: what is kept is multiplied by exactly the
// reciprocal of the share that is kept on average.
struct Dropout {
  uint32_t dropped;  // draws below are dropped; 0: none, 65536: all
  float scale;
  uint32_t k0, k1, offset;

  // values 8 * block .. 8 * block + 7 of row `row`
  __device__ __forceinline__ void apply(float (&f)[8], int64_t row, int64_t block) const
  {
    uint4 const r = philox4x32(static_cast<uint32_t>(block), static_cast<uint32_t>(row), static_cast<uint32_t>(row >> 32), offset, k0, k1);
    uint32_t const w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint32_t const draw = k % 2 ? w[k / 2] >> 16 : w[k / 2] & 0xffffu;
      f[k]                = draw >= dropped ? f[k] * scale : 0.f;  // (chosen, not multiplied: what is dropped may be NaN)
    }
  }
};

inline Dropout make_dropout(double p, uint64_t seed, uint32_t offset)
{
  uint32_t const dropped = static_cast<uint32_t>(p * 65536 + 0.5);
  float const scale      = dropped >= 65536 ? 0.f : static_cast<float>(65536.0 / (65536 - dropped));
  return Dropout{dropped, scale, static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32), offset};
}

inline bool is_probability(double p) { return p >= 0 && p <= 1; }  // (not NaN)

// ------------------------------------------------------------------ sums
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ float dpp_zero_f(float v)
{
  return __builtin_bit_cast(float, dpp_zero<CTRL, ROW_MASK>(__builtin_bit_cast(uint32_t, v)));
}

// the sum over the wavefront, in every lane
__device__ __forceinline__ float wave_sum(float v)
{
  v += dpp_zero_f<0x111, 0xf>(v);
  v += dpp_zero_f<0x112, 0xf>(v);
  v += dpp_zero_f<0x114, 0xf>(v);
  v += dpp_zero_f<0x118, 0xf>(v);
  v += dpp_zero_f<0x142, 0xa>(v);
  v += dpp_zero_f<0x143, 0xc>(v);
  return __builtin_bit_cast(float, wave_bcast(__builtin_bit_cast(uint32_t, v), kWave - 1));
}

// the sum over the workgroup, in every thread; `lds` needs a value a wavefront
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* lds)
{
  v = wave_sum(v);
  __syncthreads();  // lds may still be read from the call before
  if (lane_id() == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) sum += lds[w];
  return sum;
}

// Sums over the rows of a matrix: parts [count, cols] of them are added up into a row of type T, by a workgroup for 64 columns,
// whose wavefronts take a run of parts each.  Of two such arrays one after the other the second becomes `second`.
template <typename T>
__global__ void __launch_bounds__(512) add_parts_kernel(const float* parts, int64_t count, int64_t cols, T* out, T* second)
{
  constexpr int kWaves = 512 / kWave;
  __shared__ float lds[kWaves][kWave];
  int const wave = threadIdx.x / kWave, lane = lane_id();
  int64_t const j = block_number() * kWave + lane;
  int64_t const each = (count + kWaves - 1) / kWaves, first = wave * each, last = first + each < count ? first + each : count;
  parts += blockIdx.z * count * cols;
  float sum = 0.f;
  if (j < cols) {
#pragma unroll 8
    for (int64_t i = first; i < last; ++i) sum += parts[i * cols + j];
  }
  lds[wave][lane] = sum;
  __syncthreads();
  if (wave != 0 || j >= cols) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) sum += lds[w][lane];
  (blockIdx.z == 0 ? out : second)[j] = static_cast<T>(sum);
}

template <typename T>
inline void launch_add_parts(const float* parts, int64_t count, int64_t cols, T* out, T* second, hipStream_t stream)
{
  dim3 grid = grid_of((cols + kWave - 1) / kWave, 512);
  grid.z    = second ? 2 : 1;
  hipLaunchKernelGGL(add_parts_kernel<T>, grid, dim3(512), 0, stream, parts, count, cols, out, second);
}

}  // namespace nvtext_amd
