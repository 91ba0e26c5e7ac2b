// Embedding of a LIST<INT32> column of token ids, and the gradients of its tables.
#include "encoder.cuh"

#include <algorithm>

namespace nvtext_amd {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves   = kThreads / kWave;

inline unsigned grid_for(int64_t work, int64_t per_cu) { return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(work, per_cu * device_cus()))); }

struct Tokens {
  const int32_t* offsets;
  const int32_t* ids;
  int32_t rows;
  int32_t count;

  // where in its row token t is, or -1: it belongs to none.  (The last row that does not begin behind t: empty rows in front of it
  // begin where it does.)
  __device__ __forceinline__ int64_t place(int32_t t) const
  {
    if (rows == 0 || t >= offsets[rows]) return -1;
    int32_t lo = 0, hi = rows;  // offsets[lo - 1] <= t < offsets[hi]
    while (lo < hi) {
      int32_t const mid = lo + (hi - lo) / 2;
      if (offsets[mid] <= t)
        lo = mid + 1;
      else
        hi = mid;
    }
    return lo == 0 ? -1 : static_cast<int64_t>(t) - offsets[lo - 1];
  }
};

// A wavefront a token.
template <typename T>
__global__ void __launch_bounds__(kThreads)
embedding_kernel(Tokens tokens, Rows<const T> table, int64_t vocabulary, Rows<const T> positions, int64_t places, int64_t cols, Rows<T> out)
{
  int const lane = lane_id();
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / kWave; t < tokens.count; t += static_cast<int64_t>(gridDim.x) * kWaves) {
    int64_t const at = tokens.place(static_cast<int32_t>(t));
    int64_t const id = tokens.ids[t];
    bool const known = at >= 0 && id >= 0 && id < vocabulary, placed = at >= 0 && at < places;
    for (int64_t j = lane * 8; j < cols; j += kWave * 8) {
      float f[8] = {}, g[8] = {};
      if (known) load8(f, table.row(id) + j, cols - j);
      if (placed) load8(g, positions.row(at) + j, cols - j);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] += g[k];
      store8(out.row(t) + j, f, cols - j);
    }
  }
}

// ------------------------------------------------------------------ tokens in the order of their ids
// A stable sort: tokens of one id stay in their order, so that sums over them are added in one order at every call.  Least
// significant digit first, eight bits a pass: count the digits of every tile, add the counts up digit by digit, place.
constexpr int kDigitBits = 8;
constexpr int kDigits    = 1 << kDigitBits;
constexpr int kTile      = 2048;
constexpr int kRounds    = kTile / kThreads;

struct Sorted {
  uint32_t* keys;  // id, or the size of the vocabulary for what belongs to no entry
  uint32_t* tokens;
};

__global__ void __launch_bounds__(kThreads) token_keys_kernel(Tokens tokens, uint32_t vocabulary, Sorted out)
{
  int64_t const t = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (t >= tokens.count) return;
  uint32_t const id = static_cast<uint32_t>(tokens.ids[t]);
  bool const inside = tokens.rows > 0 && t >= tokens.offsets[0] && t < tokens.offsets[tokens.rows];
  out.keys[t]       = inside && id < vocabulary ? id : vocabulary;
  out.tokens[t]     = static_cast<uint32_t>(t);
}

__global__ void __launch_bounds__(kThreads) digit_counts_kernel(const uint32_t* keys, int32_t n, int shift, int32_t tiles, uint32_t* counts)
{
  __shared__ uint32_t lds[kDigits];
  lds[threadIdx.x] = 0;
  __syncthreads();
  for (int r = 0; r < kRounds; ++r) {
    int64_t const i = static_cast<int64_t>(blockIdx.x) * kTile + r * kThreads + threadIdx.x;
    if (i < n) atomicAdd(&lds[(keys[i] >> shift) & (kDigits - 1)], 1u);
  }
  __syncthreads();
  counts[static_cast<int64_t>(threadIdx.x) * tiles + blockIdx.x] = lds[threadIdx.x];
}

__global__ void __launch_bounds__(kThreads) digit_place_kernel(Sorted in, int32_t n, int shift, int32_t tiles, const uint32_t* places, Sorted out)
{
  __shared__ uint32_t lds[kWaves][kDigits];
  int const wave = threadIdx.x / kWave, lane = lane_id();
  for (int w = 0; w < kWaves; ++w) lds[w][threadIdx.x] = 0;
  __syncthreads();
  // a wavefront's keys are consecutive, 64 a round
  uint32_t key[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    int64_t const i = static_cast<int64_t>(blockIdx.x) * kTile + (wave * kRounds + r) * kWave + lane;
    key[r]          = i < n ? in.keys[i] : 0;
    if (i < n) atomicAdd(&lds[wave][(key[r] >> shift) & (kDigits - 1)], 1u);
  }
  __syncthreads();
  uint32_t place = places[static_cast<int64_t>(threadIdx.x) * tiles + blockIdx.x];
  for (int w = 0; w < kWaves; ++w) {
    uint32_t const count = lds[w][threadIdx.x];
    lds[w][threadIdx.x]  = place;
    place += count;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    int64_t const i      = static_cast<int64_t>(blockIdx.x) * kTile + (wave * kRounds + r) * kWave + lane;
    bool const here      = i < n;
    uint32_t const digit = (key[r] >> shift) & (kDigits - 1);
    uint64_t same        = ballot64(here);
#pragma unroll
    for (int bit = 0; bit < kDigitBits; ++bit) {
      bool const set        = (digit >> bit) & 1u;
      uint64_t const others = ballot64(set);
      same &= set ? others : ~others;
    }
    uint32_t at = 0;
    if (here) at = lds[wave][digit] + lanes_below(same);
    wave_lds_fence();
    if (here && lanes_below(same) == 0) lds[wave][digit] += static_cast<uint32_t>(__builtin_popcountll(same));
    wave_lds_fence();
    if (here) {
      out.keys[at]   = key[r];
      out.tokens[at] = in.tokens[i];
    }
  }
}

struct Counts {
  const uint32_t* counts;
  __device__ uint64_t operator()(int64_t i) const { return counts[i]; }
};

// ------------------------------------------------------------------ the table's gradient
// The sorted tokens are cut into chunks of kChunk.  A wavefront adds up the gradients of a chunk, id by id, 512 columns at a
// time; an id whose tokens all lie in the chunk is done then, the sums of others go to the chunk's two places: the first for
// an id that began in a chunk before, the second for one that begins here and goes on.
constexpr int kChunk = 32;

template <typename T, typename G>
__global__ void __launch_bounds__(kThreads)
chunk_sums_kernel(Sorted sorted, int32_t n, uint32_t vocabulary, Rows<const T> grad, int64_t cols, float* parts, Rows<G> out)
{
  int32_t const chunk = static_cast<int32_t>(blockIdx.x) * kWaves + static_cast<int32_t>(threadIdx.x) / kWave;
  int64_t const first = static_cast<int64_t>(chunk) * kChunk;
  if (first >= n) return;
  int64_t const last = std::min<int64_t>(first + kChunk, n);
  int64_t const j    = (static_cast<int64_t>(blockIdx.y) * kWave + lane_id()) * 8;
  float f[8]         = {};
  bool begun         = first == 0 || sorted.keys[first - 1] != sorted.keys[first];
  for (int64_t i = first; i < last; ++i) {
    uint32_t const id = sorted.keys[i];
    if (id >= vocabulary) break;
    float g[8];
    if (j < cols) {
      load8(g, grad.row(sorted.tokens[i]) + j, cols - j);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] += g[k];
    }
    bool const ends = i + 1 == n || sorted.keys[i + 1] != id;
    if (!ends && i + 1 < last) continue;
    if (j < cols) {
      if (begun && ends)
        store8(out.row(id) + j, f, cols - j);
      else
        store8(parts + (2 * static_cast<int64_t>(chunk) + (begun ? 1 : 0)) * cols + j, f, cols - j);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = 0.f;
    begun = true;
  }
}

// A wavefront a chunk: if an id begins in it and goes on into the next, its parts are added up, chunk after chunk.
template <typename G>
__global__ void __launch_bounds__(kThreads) join_chunks_kernel(Sorted sorted, int32_t n, uint32_t vocabulary, int64_t cols, const float* parts, Rows<G> out)
{
  int32_t const chunk = static_cast<int32_t>(blockIdx.x) * kWaves + static_cast<int32_t>(threadIdx.x) / kWave;
  int64_t const first = static_cast<int64_t>(chunk) * kChunk, last = first + kChunk;
  if (last >= n) return;
  uint32_t const id = sorted.keys[last];
  if (id >= vocabulary || sorted.keys[last - 1] != id) return;
  if (sorted.keys[first] == id && first > 0 && sorted.keys[first - 1] == id) return;  // it began before
  int64_t const j = (static_cast<int64_t>(blockIdx.y) * kWave + lane_id()) * 8;
  if (j >= cols) return;
  float f[8];
  load8(f, parts + (2 * static_cast<int64_t>(chunk) + 1) * cols + j, cols - j);
  for (int64_t c = chunk + 1; c * kChunk < n && sorted.keys[c * kChunk] == id; ++c) {
    float g[8];
    load8(g, parts + 2 * c * cols + j, cols - j);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] += g[k];
  }
  store8(out.row(id) + j, f, cols - j);
}

// Zeros for the entries that do not occur: a wavefront looks 64 of them up in the sorted ids.
template <typename G>
__global__ void __launch_bounds__(kThreads) absent_rows_kernel(Sorted sorted, int32_t n, uint32_t vocabulary, int64_t cols, Rows<G> out)
{
  int64_t const first = (static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / kWave) * kWave;
  if (first >= vocabulary) return;
  uint32_t const id = static_cast<uint32_t>(first) + lane_id();
  int32_t lo = 0, hi = n;
  while (lo < hi) {
    int32_t const mid = lo + (hi - lo) / 2;
    if (sorted.keys[mid] < id)
      lo = mid + 1;
    else
      hi = mid;
  }
  uint64_t absent     = ballot64(id < vocabulary && (lo >= n || sorted.keys[lo] != id));
  float const zero[8] = {};
  for (; absent; absent &= absent - 1) {
    int64_t const row = first + __builtin_ctzll(absent);
    for (int64_t j = lane_id() * 8; j < cols; j += kWave * 8) store8(out.row(row) + j, zero, cols - j);
  }
}

// ------------------------------------------------------------------ the positions' gradient
// A workgroup a place and 512 columns: its wavefronts share the rows that are long enough, and add up what they found in the end.
template <typename T, typename G>
__global__ void __launch_bounds__(kThreads) position_sums_kernel(Tokens tokens, Rows<const T> grad, int64_t places, int64_t cols, Rows<G> out)
{
  __shared__ float lds[kWaves][8 * kWave];
  int const wave = threadIdx.x / kWave, lane = lane_id();
  int64_t const at = blockIdx.x;
  int64_t const j  = (static_cast<int64_t>(blockIdx.y) * kWave + lane) * 8;
  float f[8]       = {};
  for (int64_t base = wave * kWave; base < tokens.rows; base += kThreads) {
    int64_t const r   = base + lane;
    int64_t const t   = r < tokens.rows ? tokens.offsets[r] + at : 0;
    uint64_t enough   = ballot64(r < tokens.rows && t >= 0 && t < tokens.offsets[r + 1] && t < tokens.count);
    for (; enough; enough &= enough - 1) {
      int64_t const token = wave_bcast(static_cast<uint32_t>(t), __builtin_ctzll(enough));
      float g[8];
      if (j < cols) {
        load8(g, grad.row(token) + j, cols - j);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] += g[k];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) lds[wave][k * kWave + lane] = f[k];
  __syncthreads();
  if (wave == 0 && j < cols) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      for (int w = 1; w < kWaves; ++w) f[k] += lds[w][k * kWave + lane];
    store8(out.row(at) + j, f, cols - j);
  }
}

const char* bad_tokens(const nvtext_amd_list_column* t)
{
  if (t->child_type != NVTEXT_AMD_TYPE_INT32) return "tokens must be a LIST<INT32> column";
  if (t->size < 0 || t->child_size < 0) return "invalid column sizes";
  if ((t->size > 0 && !t->offsets) || (t->child_size > 0 && !t->child)) return "the column of tokens has no data";
  return nullptr;
}

Tokens view_of(const nvtext_amd_list_column* t)
{
  return Tokens{t->offsets, static_cast<const int32_t*>(t->child), t->size, static_cast<int32_t>(t->child_size)};
}

}  // namespace
}  // namespace nvtext_amd

extern "C" {

nvtext_amd_status nvtext_amd_embedding(const nvtext_amd_list_column* tokens, const nvtext_amd_matrix* token_table, const nvtext_amd_matrix* position_table,
                                       void* stream_, const nvtext_amd_matrix* out)
{
  using namespace nvtext_amd;
  EntryScope const entry("nvtext_amd_embedding");
  if (!tokens || !token_table || !out) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  if (const char* bad = bad_tokens(tokens)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  if (tokens->child_size > INT32_MAX) return fail(NVTEXT_AMD_OVERFLOW, "the column has too many tokens");
  for (auto* m : {token_table, position_table, out})
    if (const char* bad = m ? bad_matrix(m) : nullptr) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  if (token_table->type != out->type || token_table->cols != out->cols || (position_table && (position_table->type != out->type || position_table->cols != out->cols)))
    return fail(NVTEXT_AMD_INVALID_ARGUMENT, "the tables and out must be of one type and width");
  if (out->rows != tokens->child_size) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "out must have a row for every token");
  if (out->rows == 0 || out->cols == 0) return NVTEXT_AMD_SUCCESS;
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  with_type(out->type, [&](auto zero) {
    using T = decltype(zero);
    ProfileScope const scope("embedding", stream);
    hipLaunchKernelGGL(embedding_kernel<T>, dim3(grid_for((out->rows + kWaves - 1) / kWaves, 16)), dim3(kThreads), 0, stream, view_of(tokens), rows_of<const T>(token_table),
                       token_table->rows, rows_of<const T>(position_table), position_table ? position_table->rows : 0, out->cols, rows_of<T>(out));
  });
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

nvtext_amd_status nvtext_amd_embedding_backward(const nvtext_amd_list_column* tokens, const nvtext_amd_matrix* grad, void* stream_, const nvtext_amd_allocator* mr_,
                                                const nvtext_amd_matrix* token_grad, const nvtext_amd_matrix* position_grad)
{
  using namespace nvtext_amd;
  EntryScope const entry("nvtext_amd_embedding_backward");
  if (!tokens || !grad || !token_grad) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  if (const char* bad = bad_tokens(tokens)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  if (tokens->child_size > INT32_MAX) return fail(NVTEXT_AMD_OVERFLOW, "the column has too many tokens");
  for (auto* m : {grad, token_grad, position_grad})
    if (const char* bad = m ? bad_matrix(m) : nullptr) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  if (grad->rows != tokens->child_size) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "grad must have a row for every token");
  for (auto* m : {token_grad, position_grad})
    if (m && (m->cols != grad->cols || (m->type != grad->type && m->type != NVTEXT_AMD_TYPE_FLOAT32) || m->type != token_grad->type))
      return fail(NVTEXT_AMD_INVALID_ARGUMENT, "the tables' gradients must be of grad's width, both of its type or both FLOAT32");
  if (token_grad->rows > INT32_MAX || (position_grad && position_grad->rows > INT32_MAX)) return fail(NVTEXT_AMD_OVERFLOW, "a table has too many rows");
  if (grad->cols == 0) return NVTEXT_AMD_SUCCESS;
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  Mr const mr{mr_, stream};
  Tokens const view         = view_of(tokens);
  uint32_t const vocabulary = static_cast<uint32_t>(token_grad->rows);
  int32_t const n           = view.count;
  int64_t const cols        = grad->cols;
  int32_t const tiles       = (n + kTile - 1) / kTile;
  int64_t const chunks      = (static_cast<int64_t>(n) + kChunk - 1) / kChunk;
  int64_t const counts      = static_cast<int64_t>(tiles) * kDigits;
  unsigned const slices     = static_cast<unsigned>((cols + 8 * kWave - 1) / (8 * kWave));
  size_t const list         = static_cast<size_t>(n) * sizeof(uint32_t);
  TempParts<7> const temp(mr, {list, list, list, list, static_cast<size_t>(counts + 1) * sizeof(uint32_t), scan_temp_bytes(counts), static_cast<size_t>(2 * chunks * cols) * sizeof(float)});
  if (!temp.ok()) return fail(NVTEXT_AMD_ALLOC_FAILED, "temporary allocation failed");
  Sorted sorted{temp.part<uint32_t>(0), temp.part<uint32_t>(1)}, other{temp.part<uint32_t>(2), temp.part<uint32_t>(3)};
  if (n > 0 && vocabulary > 0) {
    ProfileScope const scope("embedding_sort", stream);
    hipLaunchKernelGGL(token_keys_kernel, dim3((n + kThreads - 1) / kThreads), dim3(kThreads), 0, stream, view, vocabulary, sorted);
    for (int shift = 0; shift < 32 && (vocabulary >> shift) != 0; shift += kDigitBits) {
      uint32_t* const places = temp.part<uint32_t>(4);
      hipLaunchKernelGGL(digit_counts_kernel, dim3(tiles), dim3(kThreads), 0, stream, sorted.keys, n, shift, tiles, places);
      device_exclusive_scan(Counts{places}, counts, places, temp.part<uint64_t>(5), stream, TellNobody{});
      hipLaunchKernelGGL(digit_place_kernel, dim3(tiles), dim3(kThreads), 0, stream, sorted, n, shift, tiles, places, other);
      std::swap(sorted, other);
    }
  }
  with_type(grad->type, [&](auto zero) {
    using T         = decltype(zero);
    auto const sums = [&](auto result) {
      using G            = decltype(result);
      float* const parts = temp.part<float>(6);
      dim3 const by_chunk(static_cast<unsigned>((chunks + kWaves - 1) / kWaves), slices);
      if (n > 0 && vocabulary > 0) {
        ProfileScope const scope("embedding_token_sums", stream);
        hipLaunchKernelGGL(HIP_KERNEL_NAME(chunk_sums_kernel<T, G>), by_chunk, dim3(kThreads), 0, stream, sorted, n, vocabulary, rows_of<const T>(grad), cols, parts, rows_of<G>(token_grad));
        hipLaunchKernelGGL(join_chunks_kernel<G>, by_chunk, dim3(kThreads), 0, stream, sorted, n, vocabulary, cols, parts, rows_of<G>(token_grad));
      }
      if (vocabulary > 0) {
        ProfileScope const scope("embedding_absent_rows", stream);
        hipLaunchKernelGGL(absent_rows_kernel<G>, dim3((vocabulary + kThreads - 1) / kThreads), dim3(kThreads), 0, stream, sorted, n, vocabulary, cols, rows_of<G>(token_grad));
      }
      if (position_grad && position_grad->rows > 0) {
        ProfileScope const scope("embedding_position_sums", stream);
        hipLaunchKernelGGL(HIP_KERNEL_NAME(position_sums_kernel<T, G>), dim3(static_cast<unsigned>(position_grad->rows), slices), dim3(kThreads), 0, stream, view, rows_of<const T>(grad),
                           position_grad->rows, cols, rows_of<G>(position_grad));
      }
    };
    if (token_grad->type == NVTEXT_AMD_TYPE_FLOAT32)
      sums(float{});
    else
      sums(zero);
  });
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

}  // extern "C"
