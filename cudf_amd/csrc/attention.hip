// Attention of a row's tokens over its keys, and its gradient.
#include "attention.cuh"

#include <cmath>

namespace nvtext_amd {
namespace {

constexpr int kThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kThreads) attend_rows_kernel(Forward<T> f)
{
  int64_t const w = block_number() * (kThreads / kWave) + threadIdx.x / kWave;
  if (w >= static_cast<int64_t>(f.runs.tokens) * f.heads) return;
  attend_row(f, static_cast<int32_t>(w / f.heads), static_cast<int32_t>(w % f.heads));
}

// ------------------------------------------------------------------ forward, in tiles
// The work of a launch: blocks of tokens, of every head.  The heads that share a key head come one after the other on one XCD (workgroups go to
// the eight XCDs in turn), and so do, where the number of key heads allows, the blocks of a key head: its keys come from that XCD's L2.  The last
// blocks come first: of a long row they are those with the most keys to see.
struct Work {
  int64_t block;
  int32_t kv_head, head;
};
constexpr int kXcds = 8;
inline int64_t work_items(int64_t blocks, int32_t kv_heads, int32_t each) { return (blocks * kv_heads + kXcds - 1) / kXcds * kXcds * each; }
// false: nothing to do
__device__ __forceinline__ bool work_of(int64_t item, int64_t blocks, int32_t kv_heads, int32_t each, Work& w)
{
  int64_t const n = item / kXcds, unit = n / each * kXcds + item % kXcds;
  if (unit >= blocks * kv_heads) return false;
  w.block   = blocks - 1 - unit / kv_heads;
  w.kv_head = static_cast<int32_t>(unit % kv_heads);
  w.head    = w.kv_head * each + static_cast<int32_t>(n % each);
  return true;
}

template <int D, int WAVES, int NQ>
struct ForwardShape {
  static constexpr int kTokens = 32 * WAVES * NQ, kShift = __builtin_ctz(kTokens), kLds = 4 * Tile<D>::kBytes;
};

// A workgroup has kTokens tokens of a head, a wavefront 32 * NQ of them, in its registers: q, and the sums of out, transposed.  Keys come through LDS, 64 at a
// time, the next ones while these are multiplied.  Scores are products with the keys as rows, so a lane has all of a token's scores (with the
// one 32 further on), and exponentials are in its registers as the second product takes them: no lane needs another's but for the maximum.
// Sums are kept in proportion to 2^top, where top is a maximum that may be 8 too small: only then are they multiplied anew.
template <typename T, int D, int WAVES, int NQ>
__global__ void __launch_bounds__(WAVES * kWave, 2) attend_tiles_kernel(Forward<T> f)
{
  using Shape = ForwardShape<D, WAVES, NQ>;
  extern __shared__ __align__(16) char lds_[];
  LdsBytes const lds = (LdsBytes)lds_;
  constexpr int kSteps = D / 16, kColumns = D / 32;
  constexpr float kSlack = 8.f;
  Work w;
  int32_t const each = f.heads / f.kv_heads;
  if (!work_of(block_number(), f.runs.template blocks<Shape::kShift>(), f.kv_heads, each, w)) return;
  int32_t const run   = f.runs.template run_of<Shape::kShift>(w.block);
  int32_t const begin = uniform(f.runs.begin(run)), tokens = uniform(f.runs.begin(run + 1)) - begin;
  int64_t const in_run = (w.block - f.runs.template first_block<Shape::kShift>(run)) << Shape::kShift;
  if (in_run >= tokens) return;
  int const wave = uniform(threadIdx.x / kWave), lane = lane_id(), column = lane % 32, half = lane / 32;
  int32_t const block0 = static_cast<int32_t>(in_run), rest = uniform(tokens - block0);  // the first token in the run, tokens from there on
  int32_t first = 0, keys = 0;
  if (f.is_row(run)) f.keys_of(run, first, keys);
  first = uniform(first);
  keys  = uniform(keys);
  // keys that the workgroup's last token sees, and the wavefront's first and last
  int32_t const wave0 = wave * 32 * NQ, wave1 = wave0 + 32 * NQ < rest ? wave0 + 32 * NQ : rest;
  int32_t const all  = uniform(f.seen(block0 + (rest < Shape::kTokens ? rest : Shape::kTokens) - 1, tokens, keys));
  int32_t const least = uniform(wave0 < rest ? f.seen(block0 + wave0, tokens, keys) : 0), most = uniform(wave0 < rest ? f.seen(block0 + wave1 - 1, tokens, keys) : 0);

  Fragment<T> q[NQ][kSteps];
  int32_t seen[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    int32_t const i = wave0 + n * 32 + column;
    seen[n]         = i < rest ? f.seen(block0 + i, tokens, keys) : 0;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) q[n][s] = fragment_of(f.q.at(static_cast<int64_t>(begin) + block0 + (i < rest ? i : 0), w.head), 16 * s + 8 * half, f.width, i < rest);
  }
  TileLoader<D, WAVES> load_k, load_v;
  load_k.aim(f.k, first, w.kv_head, f.width, wave, lane);
  load_v.aim(f.v, first, w.kv_head, f.width, wave, lane);
  TileReader<T, D> const read(lane);
  float const scale = f.scale * kLog2e;
  f32x16_t o[NQ][kColumns];
  float top[NQ], sum[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    top[n] = -INFINITY;
    sum[n] = 0.f;
#pragma unroll
    for (int c = 0; c < kColumns; ++c) o[n][c] = f32x16_t{};
  }
  int32_t const tiles = (all + kTile - 1) / kTile;
  if (tiles > 0) {
    load_k.load(lds, keys, wave);
    load_v.load(lds + Tile<D>::kBytes, keys, wave);
  }
  for (int32_t tile = 0; tile < tiles; ++tile) {
    LdsBytes const k_tile = lds + (tile & 1) * 2 * Tile<D>::kBytes, v_tile = k_tile + Tile<D>::kBytes;
    stage_barrier<0>();
    if (tile + 1 < tiles) {
      LdsBytes const next = lds + (~tile & 1) * 2 * Tile<D>::kBytes;
      load_k.load(next, keys - (tile + 1) * kTile, wave);
      load_v.load(next + Tile<D>::kBytes, keys - (tile + 1) * kTile, wave);
    }
    int32_t const key0 = tile * kTile;
    if (key0 >= most) continue;
    f32x16_t s[NQ][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) s[n][b] = f32x16_t{};
#pragma unroll
      for (int step = 0; step < kSteps; ++step) {
        Fragment<T> const k = read.rows(k_tile, b, step);
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[n][b] = multiply32(k, q[n][step], s[n][b]);
      }
    }
    if (key0 + kTile > least) {
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[n][b][r] = key0 + 32 * b + 8 * (r / 4) + 4 * half + r % 4 < seen[n] ? s[n][b][r] : -INFINITY;
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float high = s[n][0][0];
#pragma unroll
      for (int r = 1; r < 32; ++r) high = fmaxf(high, s[n][r / 16][r % 16]);
      Halves const both = halves(high);
      high              = fmaxf(both.low, both.high) * scale;
      // (a token that sees nothing yet keeps top at -infinity; NaN in a score is found in out at the end)
      if (__ballot(high > top[n] + kSlack || top[n] == -INFINITY)) {
        float const now  = fmaxf(top[n], high);
        float const fade = now == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top[n] - now);
        top[n]           = now;
        sum[n] *= fade;
#pragma unroll
        for (int c = 0; c < kColumns; ++c)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[n][c][r] *= fade;
      }
      float const base = top[n] == -INFINITY ? 0.f : top[n];
#pragma unroll
      for (int r = 0; r < 32; ++r) {
        float const p       = __builtin_amdgcn_exp2f(fmaf(s[n][r / 16][r % 16], scale, -base));
        s[n][r / 16][r % 16] = p;
        sum[n] += p;
      }
    }
    Fragment<T> p[NQ][4];
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int step = 0; step < 4; ++step) p[n][step] = rounded<T>(s[n][step / 2], step % 2);
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        Fragment<T> const v = read.columns(v_tile, c, step);
#pragma unroll
        for (int n = 0; n < NQ; ++n) o[n][c] = multiply32(v, p[n][step], o[n][c]);
      }
  }
  if (wave0 >= rest) return;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    int32_t const i   = wave0 + n * 32 + column;
    int64_t const t   = static_cast<int64_t>(begin) + block0 + i;
    Halves const both = halves(sum[n]);
    float const total = both.low + both.high, part = seen[n] > 0 ? 1.f / total : 0.f;
    bool finite       = true;
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        o[n][c][r] *= part;
        finite = finite && fabsf(o[n][c][r]) < INFINITY;
      }
    // What is not finite may come from keys that the token does not see, whose exponentials of 0 were multiplied: such tokens are done once more, by themselves.
    uint64_t odd = __ballot(i < rest && seen[n] > 0 && !finite);
    odd          = (odd | odd >> 32) & 0xffffffffu;
    if (i < rest && !(odd >> column & 1)) {
      T* const out = f.out.at(t, w.head);
#pragma unroll
      for (int c = 0; c < kColumns; ++c)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          int32_t const j = 32 * c + 8 * g + 4 * half;
          typedef T Four __attribute__((ext_vector_type(4)));
          Four const four = {static_cast<T>(o[n][c][4 * g]), static_cast<T>(o[n][c][4 * g + 1]), static_cast<T>(o[n][c][4 * g + 2]), static_cast<T>(o[n][c][4 * g + 3])};
          if (j < f.width) *reinterpret_cast<Four*>(out + j) = four;
        }
      if (f.logsum && half == 0) f.logsum[static_cast<int64_t>(w.head) * f.runs.tokens + t] = seen[n] > 0 ? (top[n] + __builtin_amdgcn_logf(total)) * kLn2 : -INFINITY;
    }
    while (odd) {
      int const which = __builtin_ctzll(odd);
      odd &= odd - 1;
      attend_row(f, static_cast<int32_t>(begin + block0 + wave0 + n * 32 + which), w.head);
    }
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
// Whether the tiles' loads can read heads as they lie: pieces of 16 bytes, and lines of a tile within the 31 bits of their offsets.
template <typename T>
bool reads_as_it_lies(Heads<const T> const& x, int32_t width)
{
  constexpr int kEach = 16 / sizeof(T);
  return width % kEach == 0 && x.stride % kEach == 0 && x.head_stride % kEach == 0 && reinterpret_cast<uintptr_t>(x.data) % 16 == 0 && x.stride < (int64_t{1} << 23);
}

template <typename T, int D, int WAVES, int NQ>
nvtext_amd_status attend_tiles(Forward<T> const& f, hipStream_t stream)
{
  using Shape = ForwardShape<D, WAVES, NQ>;
  ProfileScope const scope("attention_tiles", stream);
  if constexpr (Shape::kLds > 65536) {
    NVTEXT_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(attend_tiles_kernel<T, D, WAVES, NQ>), hipFuncAttributeMaxDynamicSharedMemorySize, Shape::kLds));
  }
  int64_t const items = work_items(f.runs.template blocks<Shape::kShift>(), f.kv_heads, f.heads / f.kv_heads);
  hipLaunchKernelGGL(HIP_KERNEL_NAME(attend_tiles_kernel<T, D, WAVES, NQ>), grid_of(items, WAVES * kWave), dim3(WAVES * kWave), Shape::kLds, stream, f);
  return NVTEXT_AMD_SUCCESS;
}

template <typename T>
nvtext_amd_status attention(Forward<T> const& f, Mr const&, hipStream_t stream)
{
  if constexpr (sizeof(T) == 2) {
    bool const four = f.out.stride % 4 == 0 && f.out.head_stride % 4 == 0 && reinterpret_cast<uintptr_t>(f.out.data) % 8 == 0;  // (as they are written)
    if (f.width > 0 && four && reads_as_it_lies(f.q, f.width) && reads_as_it_lies(f.k, f.width) && reads_as_it_lies(f.v, f.width)) {
      if (f.width <= 64) return attend_tiles<T, 64, 4, 1>(f, stream);
      if (f.width <= 128) return attend_tiles<T, 128, 4, 1>(f, stream);
      return attend_tiles<T, 256, 4, 1>(f, stream);
    }
  }
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
