// Attention of a row's tokens over its keys, and its gradient.
#include "heads.cuh"

#include <cmath>

namespace nvtext_amd {
namespace {

constexpr int kThreads    = 256;
constexpr int kMostWidth  = 256;
constexpr float kLog2e    = 1.4426950408889634f;
constexpr float kLn2      = 0.6931471805599453f;

// What the kernels of both directions are given.
template <typename T>
struct Problem {
  Heads<const T> q, k, v;
  int32_t heads, kv_heads, width;
  Runs runs, key_runs;
  const int32_t* key_lengths;
  bool causal;
  float scale;

  // The keys of run `i` (a row's), of which there are `length`, from token `first` on.
  __device__ __forceinline__ void keys_of(int32_t i, int32_t& first, int32_t& length) const
  {
    first  = key_runs.begin(i);
    length = key_runs.begin(i + 1) - first;
    if (key_lengths) {
      int32_t const l = key_lengths[i - 1];
      length          = l < length ? l : length;
    }
    length = length > 0 ? length : 0;
  }
  __device__ __forceinline__ bool is_row(int32_t i) const { return i > 0 && i <= runs.rows; }
  // How many keys token `i` of a row of `tokens` sees, of `keys`.
  __device__ __forceinline__ int32_t seen(int32_t i, int32_t tokens, int32_t keys) const
  {
    int64_t const n = causal ? static_cast<int64_t>(i) + 1 + keys - tokens : keys;
    return static_cast<int32_t>(n < 0 ? 0 : n < keys ? n : keys);
  }
};

// ------------------------------------------------------------------ a row at a time
// The formulas as they stand, a wavefront for a token and a head, 64 keys at a time: a lane for a key in the scores, a lane for a column in the
// sums.  Nothing that a token does not see is multiplied by anything.

template <typename T>
__device__ __forceinline__ float dot(const T* a, const T* b, int32_t width)
{
  float sum = 0.f;
  for (int32_t j = 0; j < width; ++j) sum = fmaf(static_cast<float>(a[j]), static_cast<float>(b[j]), sum);
  return sum;
}

__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
  for (int by = 32; by > 0; by /= 2) v = fmaxf(v, __shfl_xor(v, by));
  return v;
}

template <typename T>
struct Forward : Problem<T> {
  Heads<T> out;
  float* logsum;
};

// The run that token t is in.
__device__ __forceinline__ int32_t run_with(Runs const& runs, int32_t t)
{
  int32_t lo = 0, hi = runs.rows + 2;
  while (hi - lo > 1) {
    int32_t const mid = lo + (hi - lo) / 2;
    if (runs.begin(mid) <= t)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

template <typename T>
__device__ void attend_row(Forward<T> const& f, int32_t t, int32_t h)
{
  int const lane    = lane_id();
  int32_t const run = run_with(f.runs, t);
  int32_t first = 0, keys = 0, seen = 0;
  if (f.is_row(run)) {
    f.keys_of(run, first, keys);
    seen = f.seen(t - f.runs.begin(run), f.runs.begin(run + 1) - f.runs.begin(run), keys);
  }
  int32_t const kh   = h / (f.heads / f.kv_heads);
  float const scale  = f.scale * kLog2e;
  const T* const q   = f.q.at(t, h);
  float top = -INFINITY, sum = 0.f, o[kMostWidth / kWave] = {};
  for (int32_t base = 0; base < seen; base += kWave) {
    int32_t const n = seen - base < kWave ? seen - base : kWave;
    float const s   = lane < n ? dot(q, f.k.at(first + base + lane, kh), f.width) * scale : -INFINITY;
    float const now = fmaxf(top, wave_max(s));
    float const p   = lane < n ? __builtin_amdgcn_exp2f(s - now) : 0.f, fade = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - now);
    sum = sum * fade + wave_sum(p);
#pragma unroll
    for (int c = 0; c < kMostWidth / kWave; ++c) o[c] *= fade;
    for (int32_t j = 0; j < n; ++j) {
      float const pj = __shfl(p, j);
#pragma unroll
      for (int c = 0; c < kMostWidth / kWave; ++c)
        if (c * kWave + lane < f.width) o[c] = fmaf(pj, static_cast<float>(f.v.at(first + base + j, kh)[c * kWave + lane]), o[c]);
    }
    top = now;
  }
#pragma unroll
  for (int c = 0; c < kMostWidth / kWave; ++c)
    if (c * kWave + lane < f.width) f.out.at(t, h)[c * kWave + lane] = static_cast<T>(seen > 0 ? o[c] / sum : 0.f);
  if (f.logsum && lane == 0) f.logsum[static_cast<int64_t>(h) * f.runs.tokens + t] = seen > 0 ? (top + __builtin_amdgcn_logf(sum)) * kLn2 : -INFINITY;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) attend_rows_kernel(Forward<T> f)
{
  int64_t const w = block_number() * (kThreads / kWave) + threadIdx.x / kWave;
  if (w >= static_cast<int64_t>(f.runs.tokens) * f.heads) return;
  attend_row(f, static_cast<int32_t>(w / f.heads), static_cast<int32_t>(w % f.heads));
}

template <typename T>
struct Backward : Problem<T> {
  Heads<const T> grad, out;
  const float* logsum;
  float* deltas;  // [heads, tokens]: grad . out
  Heads<T> q_grad, k_grad, v_grad;
};

// The gradient of token t's head h of q, and its delta.
template <typename T>
__device__ void query_gradient_row(Backward<T> const& f, int32_t t, int32_t h)
{
  int const lane    = lane_id();
  int32_t const run = run_with(f.runs, t);
  int32_t first = 0, keys = 0, seen = 0;
  if (f.is_row(run)) {
    f.keys_of(run, first, keys);
    seen = f.seen(t - f.runs.begin(run), f.runs.begin(run + 1) - f.runs.begin(run), keys);
  }
  int32_t const kh = h / (f.heads / f.kv_heads);
  const T *const q = f.q.at(t, h), *const g = f.grad.at(t, h);
  int64_t const at  = static_cast<int64_t>(h) * f.runs.tokens + t;
  float const log   = f.logsum[at] * kLog2e, scale = f.scale * kLog2e;
  float const delta = seen > 0 ? dot(g, f.out.at(t, h), f.width) : 0.f;
  if (lane == 0) f.deltas[at] = delta;
  float d[kMostWidth / kWave] = {};
  for (int32_t base = 0; base < seen; base += kWave) {
    int32_t const n = seen - base < kWave ? seen - base : kWave;
    float ds        = 0.f;
    if (lane < n) {
      float const p = __builtin_amdgcn_exp2f(dot(q, f.k.at(first + base + lane, kh), f.width) * scale - log);
      ds            = p * (dot(g, f.v.at(first + base + lane, kh), f.width) - delta) * f.scale;
    }
    for (int32_t j = 0; j < n; ++j) {
      float const dj = __shfl(ds, j);
#pragma unroll
      for (int c = 0; c < kMostWidth / kWave; ++c)
        if (c * kWave + lane < f.width) d[c] = fmaf(dj, static_cast<float>(f.k.at(first + base + j, kh)[c * kWave + lane]), d[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < kMostWidth / kWave; ++c)
    if (c * kWave + lane < f.width) f.q_grad.at(t, h)[c * kWave + lane] = static_cast<T>(d[c]);
}

// The gradients of key token t's head kh of k and v.
template <typename T>
__device__ void key_gradient_row(Backward<T> const& f, int32_t t, int32_t kh)
{
  int const lane    = lane_id();
  int32_t const run = run_with(f.key_runs, t), each = f.heads / f.kv_heads;
  float dk[kMostWidth / kWave] = {}, dv[kMostWidth / kWave] = {};
  int32_t first = 0, keys = 0;
  if (f.is_row(run)) f.keys_of(run, first, keys);
  int32_t const j = t - first;
  if (f.is_row(run) && j < keys) {
    int32_t const begin = f.runs.begin(run), tokens = f.runs.begin(run + 1) - begin;
    // token i sees key j from i = j + tokens - keys on
    int64_t const from = f.causal ? static_cast<int64_t>(j) + tokens - keys : 0;
    const T *const k = f.k.at(t, kh), *const v = f.v.at(t, kh);
    float const scale = f.scale * kLog2e;
    for (int32_t h = kh * each; h < (kh + 1) * each; ++h) {
      for (int64_t base = from < 0 ? 0 : from; base < tokens; base += kWave) {
        int32_t const n = static_cast<int32_t>(tokens - base < kWave ? tokens - base : kWave), token = static_cast<int32_t>(begin + base);
        float p = 0.f, ds = 0.f;
        if (lane < n) {
          int64_t const at = static_cast<int64_t>(h) * f.runs.tokens + token + lane;
          p                = __builtin_amdgcn_exp2f(dot(f.q.at(token + lane, h), k, f.width) * scale - f.logsum[at] * kLog2e);
          ds               = p * (dot(f.grad.at(token + lane, h), v, f.width) - f.deltas[at]) * f.scale;
        }
        for (int32_t i = 0; i < n; ++i) {
          float const pi = __shfl(p, i), di = __shfl(ds, i);
#pragma unroll
          for (int c = 0; c < kMostWidth / kWave; ++c)
            if (c * kWave + lane < f.width) {
              dv[c] = fmaf(pi, static_cast<float>(f.grad.at(token + i, h)[c * kWave + lane]), dv[c]);
              dk[c] = fmaf(di, static_cast<float>(f.q.at(token + i, h)[c * kWave + lane]), dk[c]);
            }
        }
      }
    }
  }
#pragma unroll
  for (int c = 0; c < kMostWidth / kWave; ++c)
    if (c * kWave + lane < f.width) {
      f.k_grad.at(t, kh)[c * kWave + lane] = static_cast<T>(dk[c]);
      f.v_grad.at(t, kh)[c * kWave + lane] = static_cast<T>(dv[c]);
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) query_gradient_rows_kernel(Backward<T> f)
{
  int64_t const w = block_number() * (kThreads / kWave) + threadIdx.x / kWave;
  if (w >= static_cast<int64_t>(f.runs.tokens) * f.heads) return;
  query_gradient_row(f, static_cast<int32_t>(w / f.heads), static_cast<int32_t>(w % f.heads));
}

template <typename T>
__global__ void __launch_bounds__(kThreads) key_gradient_rows_kernel(Backward<T> f)
{
  int64_t const w = block_number() * (kThreads / kWave) + threadIdx.x / kWave;
  if (w >= static_cast<int64_t>(f.key_runs.tokens) * f.kv_heads) return;
  key_gradient_row(f, static_cast<int32_t>(w / f.kv_heads), static_cast<int32_t>(w % f.kv_heads));
}

// ------------------------------------------------------------------ launches
template <typename T>
nvtext_amd_status attention(Forward<T> const& f, Mr const&, hipStream_t stream)
{
  ProfileScope const scope("attention_rows", stream);
  hipLaunchKernelGGL(attend_rows_kernel<T>, grid_of((static_cast<int64_t>(f.runs.tokens) * f.heads + 3) / 4, kThreads), dim3(kThreads), 0, stream, f);
  return NVTEXT_AMD_SUCCESS;
}

template <typename T>
nvtext_amd_status attention_backward(Backward<T> f, Mr const& mr, hipStream_t stream)
{
  Temp const deltas(mr, static_cast<size_t>(f.heads) * static_cast<size_t>(f.runs.tokens) * sizeof(float));
  if (!deltas.ok()) return fail(NVTEXT_AMD_ALLOC_FAILED, "temporary allocation failed");
  f.deltas = deltas.template as<float>();
  if (f.runs.tokens > 0) {
    ProfileScope const scope("attention_query_gradient", stream);
    hipLaunchKernelGGL(query_gradient_rows_kernel<T>, grid_of((static_cast<int64_t>(f.runs.tokens) * f.heads + 3) / 4, kThreads), dim3(kThreads), 0, stream, f);
  }
  if (f.key_runs.tokens > 0) {
    ProfileScope const scope("attention_key_gradient", stream);
    hipLaunchKernelGGL(key_gradient_rows_kernel<T>, grid_of((static_cast<int64_t>(f.key_runs.tokens) * f.kv_heads + 3) / 4, kThreads), dim3(kThreads), 0, stream, f);
  }
  return NVTEXT_AMD_SUCCESS;
}

// What both directions ask of their arguments; nullptr if it holds.
const char* bad_attention(const nvtext_amd_heads* q, const nvtext_amd_heads* k, const nvtext_amd_heads* v, int32_t rows, const int32_t* offsets, const int32_t* key_offsets,
                          const int32_t* key_lengths, double scale)
{
  for (auto* x : {q, k, v})
    if (const char* bad = bad_heads(x)) return bad;
  if (k->type != q->type || v->type != q->type) return "q, k and v must be of one type";
  if (!is_like(v, k)) return "v must be of k's size";
  if (k->width != q->width) return "k and v must be of q's width";
  if (q->width > kMostWidth) return "heads may have 256 values at most";
  if (q->heads > 0 ? k->heads == 0 || q->heads % k->heads != 0 : k->heads != 0) return "the heads of k and v must be a divisor of q's";
  if (const char* bad = bad_rows(rows, offsets)) return bad;
  if (key_lengths && !key_offsets) return "key_lengths need key_offsets";
  if (!key_offsets && k->tokens != q->tokens) return "without offsets of their own, k and v must have q's tokens";
  if (!(scale >= 0) || !std::isfinite(static_cast<float>(scale))) return "scale must be finite and not negative";
  return nullptr;
}

template <typename T>
Problem<T> problem_of(const nvtext_amd_heads* q, const nvtext_amd_heads* k, const nvtext_amd_heads* v, int32_t rows, const int32_t* offsets, const int32_t* key_offsets,
                      const int32_t* key_lengths, int32_t causal, double scale)
{
  return {heads_of<const T>(q), heads_of<const T>(k), heads_of<const T>(v), static_cast<int32_t>(q->heads), static_cast<int32_t>(k->heads), static_cast<int32_t>(q->width),
          Runs{offsets, rows, static_cast<int32_t>(q->tokens)}, Runs{key_offsets ? key_offsets : offsets, rows, static_cast<int32_t>(k->tokens)}, key_lengths, causal != 0,
          static_cast<float>(scale)};
}

}  // namespace
}  // namespace nvtext_amd

extern "C" {

nvtext_amd_status nvtext_amd_attention(const nvtext_amd_heads* q, const nvtext_amd_heads* k, const nvtext_amd_heads* v, int32_t rows, const int32_t* offsets, const int32_t* key_offsets,
                                       const int32_t* key_lengths, int32_t causal, double scale, void* stream_, const nvtext_amd_allocator* mr_, const nvtext_amd_heads* out, float* logsum)
{
  using namespace nvtext_amd;
  EntryScope const entry("nvtext_amd_attention");
  if (!q || !k || !v || !out) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  if (const char* bad = bad_attention(q, k, v, rows, offsets, key_offsets, key_lengths, scale)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  if (const char* bad = bad_result(out)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  if (out->type != q->type || !is_like(out, q)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "out must be of q's size and type");
  if (q->tokens == 0 || q->heads == 0) return NVTEXT_AMD_SUCCESS;
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  Mr const mr{mr_, stream};
  nvtext_amd_status st = NVTEXT_AMD_SUCCESS;
  with_type(q->type, [&](auto zero) {
    using T = decltype(zero);
    st      = attention<T>({problem_of<T>(q, k, v, rows, offsets, key_offsets, key_lengths, causal, scale), heads_of<T>(out), logsum}, mr, stream);
  });
  if (st != NVTEXT_AMD_SUCCESS) return st;
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

nvtext_amd_status nvtext_amd_attention_backward(const nvtext_amd_heads* grad, const nvtext_amd_heads* q, const nvtext_amd_heads* k, const nvtext_amd_heads* v, const nvtext_amd_heads* out,
                                                const float* logsum, int32_t rows, const int32_t* offsets, const int32_t* key_offsets, const int32_t* key_lengths, int32_t causal,
                                                double scale, void* stream_, const nvtext_amd_allocator* mr_, const nvtext_amd_heads* q_grad, const nvtext_amd_heads* k_grad,
                                                const nvtext_amd_heads* v_grad)
{
  using namespace nvtext_amd;
  EntryScope const entry("nvtext_amd_attention_backward");
  if (!grad || !q || !k || !v || !out || !q_grad || !k_grad || !v_grad) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  if (const char* bad = bad_attention(q, k, v, rows, offsets, key_offsets, key_lengths, scale)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  for (auto* x : {grad, out}) {
    if (const char* bad = bad_heads(x)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
    if (x->type != q->type || !is_like(x, q)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "grad and out must be of q's size and type");
  }
  for (auto* x : {q_grad, k_grad, v_grad}) {
    if (const char* bad = bad_result(x)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
    if (x->type != q->type || !is_like(x, x == q_grad ? q : k)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "the gradients must be of the size and type of what they are those of");
  }
  if (q->heads == 0 || (q->tokens == 0 && k->tokens == 0)) return NVTEXT_AMD_SUCCESS;
  if (q->tokens > 0 && !logsum) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  Mr const mr{mr_, stream};
  nvtext_amd_status st = NVTEXT_AMD_SUCCESS;
  with_type(q->type, [&](auto zero) {
    using T = decltype(zero);
    Backward<T> b{problem_of<T>(q, k, v, rows, offsets, key_offsets, key_lengths, causal, scale)};
    b.grad   = heads_of<const T>(grad);
    b.out    = heads_of<const T>(out);
    b.logsum = logsum;
    b.q_grad = heads_of<T>(q_grad);
    b.k_grad = heads_of<T>(k_grad);
    b.v_grad = heads_of<T>(v_grad);
    st       = attention_backward<T>(b, mr, stream);
  });
  if (st != NVTEXT_AMD_SUCCESS) return st;
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

}  // extern "C"
