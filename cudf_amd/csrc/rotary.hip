// Rotary positions: the first values of every head, in pairs, turned by an angle that follows from the token's position.
#include "heads.cuh"

#include <cmath>

namespace nvtext_amd {
namespace {

constexpr int kThreads = 256;
constexpr int kAngles  = 2048;  // sines and cosines that a workgroup has room for: 16 KB
constexpr double kTurn = 0.15915494309189534;  // 1 / (2 pi)

// Sine and cosine of 2 pi * turns.  The quarter turns are taken off in 64 bits, where nothing is lost; what is left, at most an eighth of a turn either
// way, fits 32 bits with an error of 2^-26 of a quarter, and the Taylor series of both at pi / 4 end with terms of 1.7e-9 and 2.5e-8 and less.
__device__ __forceinline__ void sine_cosine(double turns, float& sine, float& cosine)
{
  double const quarters = 4.0 * turns, whole = rint(quarters);
  float const a  = static_cast<float>(quarters - whole) * 1.5707963267948966f, b = a * a;
  int const turn = static_cast<int>(static_cast<int64_t>(whole) & 3);
  float s = 2.7557319e-6f, c = -2.7557319e-7f;
  s = fmaf(s, b, -1.9841270e-4f);
  s = fmaf(s, b, 8.3333333e-3f);
  s = fmaf(s, b, -1.6666667e-1f);
  s = fmaf(s * b, a, a);
  c = fmaf(c, b, 2.4801587e-5f);
  c = fmaf(c, b, -1.3888889e-3f);
  c = fmaf(c, b, 4.1666667e-2f);
  c = fmaf(c, b, -0.5f);
  c = fmaf(c, b, 1.f);
  float const p = turn & 1 ? c : s, q = turn & 1 ? s : c;
  sine   = turn & 2 ? -p : p;
  cosine = (turn + 1) & 2 ? -q : q;
}

template <typename T>
struct Rotary {
  Heads<const T> x;
  Heads<T> out;
  int32_t heads, width, pairs;
  Runs runs;
  const int32_t* starts;
  const double* frequencies;
  bool inverse;
  float magnitude;
  bool copy;  // the values that are not turned: out is another memory than x
  int32_t each;  // tokens of a workgroup; each * pairs angles at most kAngles
};

constexpr int64_t kNoRow = INT64_MIN;

// The position of a token, or kNoRow.
__device__ __forceinline__ int64_t position(Runs const& runs, const int32_t* starts, int32_t t)
{
  int32_t lo = 0, hi = runs.rows + 1;  // run lo begins at t or before, run hi behind it (as far as offsets ascend)
  while (hi - lo > 1) {
    int32_t const mid = lo + (hi - lo) / 2;
    if (runs.begin(mid) <= t)
      lo = mid;
    else
      hi = mid;
  }
  if (lo == 0 || t >= runs.begin(lo + 1)) return kNoRow;
  return static_cast<int64_t>(t) - runs.begin(lo) + (starts ? starts[lo - 1] : 0);
}

// A workgroup takes `each` tokens: it computes their angles' sines and cosines into LDS, once for all heads, then goes through their values
// as they lie, a thread with VEC pairs at a time.  Bound by memory: 65536 tokens of 32 heads of 64, bfloat16, 109 us, 4.9 TB/s, what a large copy reaches; halves of 20011 x 24 heads of 80
// in float32 79 us, 3.9 TB/s (what is not turned is 160 bytes of a head's 320); 32 single tokens 5 us.
template <typename T, int VEC, bool HALF>
__global__ void __launch_bounds__(kThreads) rotary_kernel(Rotary<T> r)
{
  __shared__ float2 angles[kAngles];  // cosine, sine
  __shared__ int64_t at[kThreads];
  typedef T Vec __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
  typedef T Vec2 __attribute__((ext_vector_type(2 * VEC), aligned(sizeof(T))));
  int64_t const first = block_number() * r.each;
  if (first >= r.runs.tokens) return;
  int32_t const count = static_cast<int32_t>(r.runs.tokens - first < r.each ? r.runs.tokens - first : r.each), tid = threadIdx.x;
  if (tid < count) at[tid] = position(r.runs, r.starts, static_cast<int32_t>(first) + tid);
  __syncthreads();
  for (int32_t i = tid; i < count * r.pairs; i += kThreads) {
    int32_t const t = i / r.pairs, n = i - t * r.pairs;
    int64_t const place = at[t];
    float s = 0.f, c = 1.f;
    if (place != kNoRow) {
      sine_cosine(static_cast<double>(place) * (r.frequencies[n] * kTurn), s, c);
      s *= r.inverse ? -r.magnitude : r.magnitude;
      c *= r.magnitude;
    }
    angles[i] = make_float2(c, s);
  }
  __syncthreads();
  int32_t const steps = (r.pairs + VEC - 1) / VEC, rest = r.copy ? r.width - 2 * r.pairs : 0, rests = (rest + 2 * VEC - 1) / (2 * VEC), of_head = steps + rests;
  int32_t const of_token = of_head * r.heads;
  for (int32_t i = tid; i < count * of_token; i += kThreads) {
    int32_t const t = i / of_token, u = i - t * of_token, h = u / of_head, step = u - h * of_head;
    const T* const from = r.x.at(first + t, h);
    T* const to         = r.out.at(first + t, h);
    if (step >= steps) {
      int32_t const j = 2 * r.pairs + (step - steps) * 2 * VEC, n = r.width - j;
      if (n >= 2 * VEC) {
        *reinterpret_cast<Vec2*>(to + j) = *reinterpret_cast<const Vec2*>(from + j);
      } else {
        for (int k = 0; k < n; ++k) to[j + k] = from[j + k];
      }
      continue;
    }
    // (a token of no row keeps its bits: cosine 1 and sine 0 would not keep an infinity or what NaN holds)
    if (at[t] == kNoRow && !r.copy) continue;
    bool const turn = at[t] != kNoRow;
    int32_t const n = step * VEC;  // the first pair
    const float2* const angle = angles + t * r.pairs + n;
    if (n + VEC <= r.pairs) {
      Vec a, b;
      if constexpr (HALF) {
        a = *reinterpret_cast<const Vec*>(from + n);
        b = *reinterpret_cast<const Vec*>(from + n + r.pairs);
      } else {
        Vec2 const both = *reinterpret_cast<const Vec2*>(from + 2 * n);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          a[k] = both[2 * k];
          b[k] = both[2 * k + 1];
        }
      }
      if (turn) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          float const p = static_cast<float>(a[k]), q = static_cast<float>(b[k]), c = angle[k].x, s = angle[k].y;
          a[k] = static_cast<T>(p * c - q * s);
          b[k] = static_cast<T>(p * s + q * c);
        }
      }
      if constexpr (HALF) {
        *reinterpret_cast<Vec*>(to + n)           = a;
        *reinterpret_cast<Vec*>(to + n + r.pairs) = b;
      } else {
        Vec2 both;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          both[2 * k]     = a[k];
          both[2 * k + 1] = b[k];
        }
        *reinterpret_cast<Vec2*>(to + 2 * n) = both;
      }
    } else {
      for (int k = 0; n + k < r.pairs; ++k) {
        int32_t const i0 = HALF ? n + k : 2 * (n + k), i1 = HALF ? n + k + r.pairs : 2 * (n + k) + 1;
        T const a = from[i0], b = from[i1];
        float const p = static_cast<float>(a), q = static_cast<float>(b), c = angle[k].x, s = angle[k].y;
        to[i0] = turn ? static_cast<T>(p * c - q * s) : a;
        to[i1] = turn ? static_cast<T>(p * s + q * c) : b;
      }
    }
  }
}

template <typename T>
void launch(Rotary<T> r, bool half, hipStream_t stream)
{
  // As many tokens as there is room for the angles of, but not so many that CUs have nothing to do, nor more than a thread each.
  int64_t const most = std::max<int64_t>(1, std::min<int64_t>(kAngles / std::max(r.pairs, 1), kThreads));
  r.each             = static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>({most, 8, r.runs.tokens / (4 * device_cus())})));
  ProfileScope const scope("rotary", stream);
  dim3 const grid = grid_of((static_cast<int64_t>(r.runs.tokens) + r.each - 1) / r.each, kThreads);
  constexpr int kVec = 16 / sizeof(T);  // (pairs of a thread at a time: two loads of 16 bytes)
  if (half)
    hipLaunchKernelGGL(HIP_KERNEL_NAME(rotary_kernel<T, kVec, true>), grid, dim3(kThreads), 0, stream, r);
  else
    hipLaunchKernelGGL(HIP_KERNEL_NAME(rotary_kernel<T, kVec, false>), grid, dim3(kThreads), 0, stream, r);
}

}  // namespace
}  // namespace nvtext_amd

extern "C" {

nvtext_amd_status nvtext_amd_rotary(const nvtext_amd_heads* x, int32_t rows, const int32_t* offsets, const int32_t* starts, const double* frequencies, int64_t pairs, int32_t layout,
                                    int32_t inverse, double magnitude, void* stream_, const nvtext_amd_heads* out)
{
  using namespace nvtext_amd;
  EntryScope const entry("nvtext_amd_rotary");
  if (!x || !out) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  if (const char* bad = bad_heads(x)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  if (const char* bad = bad_result(out)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  if (const char* bad = bad_rows(rows, offsets)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  if (x->type != out->type || !is_like(out, x)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "out must be of x's size and type");
  if (x->data == out->data && ((x->tokens >= 2 && x->stride != out->stride) || (x->heads >= 2 && x->head_stride != out->head_stride)))
    return fail(NVTEXT_AMD_INVALID_ARGUMENT, "out may be x, but not lie over it in another order");
  if (pairs < 0 || pairs > x->width / 2) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "there must not be more frequencies than pairs of values in a head");
  if (pairs > kAngles) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "there may be 2048 frequencies at most");
  if (pairs > 0 && !frequencies) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "frequencies have no data");
  if (layout != NVTEXT_AMD_ROTARY_HALF && layout != NVTEXT_AMD_ROTARY_INTERLEAVED) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "unknown layout");
  if (!std::isfinite(magnitude)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "magnitude must be finite");
  // a thread's steps over a workgroup's values are counted in 32 bits
  if (x->heads * ((x->width + 1) / 2 + 1) > INT32_MAX / 16) return fail(NVTEXT_AMD_OVERFLOW, "a token has too many values");
  if (x->tokens == 0 || x->heads == 0 || x->width == 0) return NVTEXT_AMD_SUCCESS;
  with_type(x->type, [&](auto zero) {
    using T = decltype(zero);
    launch<T>({heads_of<const T>(x), heads_of<T>(out), static_cast<int32_t>(x->heads), static_cast<int32_t>(x->width), static_cast<int32_t>(pairs),
               {offsets, rows, static_cast<int32_t>(x->tokens)}, starts, frequencies, inverse != 0, static_cast<float>(magnitude), x->data != out->data, 1},
              layout == NVTEXT_AMD_ROTARY_HALF, static_cast<hipStream_t>(stream_));
  });
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

}  // extern "C"
