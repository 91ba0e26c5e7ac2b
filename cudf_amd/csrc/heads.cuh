// Shared by the operators that look at the heads of a row's tokens (rotary positions, attention): what a kernel is given of them, the
// rows' bounds, and the checks.
#pragma once

#include "encoder.cuh"

namespace nvtext_amd {

// What a kernel is given of heads: value j of head h of token t at data[t * stride + h * head_stride + j].
template <typename T>
struct Heads {
  T* data;
  int64_t stride, head_stride;
  __device__ __forceinline__ T* at(int64_t t, int64_t h) const { return data + t * stride + h * head_stride; }
};

template <typename T>
inline Heads<T> heads_of(const nvtext_amd_heads* x)
{
  return {static_cast<T*>(x->data), x->tokens < 2 ? 0 : x->stride, x->heads < 2 ? 0 : x->head_stride};
}

// ------------------------------------------------------------------ checks
constexpr int64_t kMostStride = int64_t{1} << 40;

// nullptr if `x` can be read, else what is wrong with it
inline const char* bad_heads(const nvtext_amd_heads* x)
{
  if (x->type != NVTEXT_AMD_TYPE_FLOAT32 && x->type != NVTEXT_AMD_TYPE_FLOAT16 && x->type != NVTEXT_AMD_TYPE_BFLOAT16)
    return "heads must be of FLOAT32, FLOAT16 or BFLOAT16";
  if (x->tokens < 0 || x->tokens > INT32_MAX || x->heads < 0 || x->heads > INT32_MAX || x->width < 0 || x->width > INT32_MAX) return "invalid sizes of heads";
  if ((x->tokens >= 2 && (x->stride < 0 || x->stride > kMostStride)) || (x->heads >= 2 && (x->head_stride < 0 || x->head_stride > kMostStride)))
    return "the strides of heads must not be negative";
  if (x->tokens > 0 && x->heads > 0 && x->width > 0) {
    if (!x->data) return "heads have no data";
    if (reinterpret_cast<uintptr_t>(x->data) % type_bytes(x->type) != 0) return "heads must be aligned to their type";
  }
  return nullptr;
}

// the same for one that is written: no two of its values may lie at one place
inline const char* bad_result(const nvtext_amd_heads* x)
{
  if (const char* bad = bad_heads(x)) return bad;
  int64_t const tokens = x->tokens, heads = x->heads, width = x->width;
  if (tokens == 0 || heads == 0 || width == 0) return nullptr;
  bool const inside = heads < 2 || x->head_stride >= width, apart = tokens < 2 || x->stride >= width;
  // heads within tokens, or tokens within heads (strides are at most 2^40, counts 2^31: no product of them passes 2^71)
  bool const ordered = heads < 2 || tokens < 2 || static_cast<__int128>(heads - 1) * x->head_stride + width <= x->stride ||
                       static_cast<__int128>(tokens - 1) * x->stride + width <= x->head_stride;
  return inside && apart && ordered ? nullptr : "the values of a result must not overlap";
}

inline bool is_like(const nvtext_amd_heads* x, const nvtext_amd_heads* like) { return x->tokens == like->tokens && x->heads == like->heads && x->width == like->width; }

// ------------------------------------------------------------------ rows
// Tokens in runs: row r is offsets[r] .. offsets[r + 1].  Whatever the offsets hold, what comes out of here lies within the tokens.
// Counted with the rows are two runs of tokens that belong to none: run 0 in front of the first row, run r + 1 is row r, run rows + 1
// lies behind the last.
struct Runs {
  const int32_t* offsets;
  int32_t rows;
  int32_t tokens;

  __device__ __forceinline__ int32_t clamped(int32_t t) const { return t < 0 ? 0 : t > tokens ? tokens : t; }
  // where run i begins, i up to rows + 2
  __device__ __forceinline__ int32_t begin(int32_t i) const { return i <= 0 || rows == 0 ? (i <= 1 ? 0 : tokens) : i >= rows + 2 ? tokens : clamped(offsets[i - 1]); }

  // Runs are cut into blocks of 2^shift tokens, each run from its own begin.  A run's blocks have numbers from
  // begin / 2^shift + its own number on: as many as it needs or one more, so no block is two runs' and nobody has to count
  // blocks before the kernel.  Block numbers are below blocks().
  __host__ __device__ __forceinline__ int64_t blocks(int shift) const { return (static_cast<int64_t>(tokens) >> shift) + rows + 2; }
  __device__ __forceinline__ int64_t first_block(int32_t i, int shift) const { return (static_cast<int64_t>(begin(i)) >> shift) + i; }
  // The run that block `b` is one of, the same in all lanes of the (whole) wavefront: the last whose first block is not behind b.
  // The lanes look at 64 runs at once: two rounds of reads for 4,000 rows, where halving takes twelve, one after the other.
  __device__ __forceinline__ int32_t run_of(int64_t b, int shift) const
  {
    int32_t lo = 0, count = rows + 2;  // the run is one of lo .. lo + count - 1, and lo's first block is not behind b
    while (count > 1) {
      int32_t const each = (count + kWave - 1) / kWave;
      int32_t const i    = lane_id() * each;
      bool const reached = i < count && first_block(lo + i, shift) <= b;
      uint64_t const all = __ballot(reached) | 1;
      int32_t const last = 63 - __clzll(static_cast<long long>(all));
      lo += last * each;
      count = count - last * each < each ? count - last * each : each;
    }
    return __builtin_amdgcn_readfirstlane(lo);
  }
};

inline const char* bad_rows(int32_t rows, const int32_t* offsets)
{
  if (rows < 0 || rows > INT32_MAX - 8) return "invalid number of rows";
  if (rows > 0 && !offsets) return "rows need offsets";
  return nullptr;
}

}  // namespace nvtext_amd
