// Exercises nvtext::encoder's rotary positions and attention (cudf_amd/include/nvtext/encoder.hpp) on the GPU: small heads of float32 against plain loops
// in double, keys in places with room, and the exceptions.  Prints one line per case, exits non-zero if a check failed.
#include <hip/hip_runtime.h>
#include <nvtext/encoder.hpp>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <vector>

#define HIP_OK(x)                                                                            \
  do {                                                                                       \
    hipError_t e_ = (x);                                                                     \
    if (e_ != hipSuccess) {                                                                  \
      std::printf("HIP error %s at %s:%d\n", hipGetErrorString(e_), __FILE__, __LINE__);     \
      std::exit(2);                                                                          \
    }                                                                                        \
  } while (0)

static int g_failures = 0;
#define CHECK(cond)                                                     \
  do {                                                                  \
    if (!(cond)) {                                                      \
      std::printf("  FAILED: %s (%s:%d)\n", #cond, __FILE__, __LINE__); \
      ++g_failures;                                                     \
    }                                                                   \
  } while (0)
#define EXPECT_THROW(stmt, type)                                                     \
  do {                                                                               \
    bool thrown_ = false;                                                            \
    try { stmt; } catch (type const&) { thrown_ = true; } catch (...) {}             \
    if (!thrown_) { std::printf("  FAILED: expected " #type " from " #stmt "\n"); ++g_failures; } \
  } while (0)

namespace enc = nvtext::encoder;

template <typename T>
struct Buffer {
  T* data{nullptr};
  size_t size;
  explicit Buffer(std::vector<T> const& h) : size(h.size())
  {
    HIP_OK(hipMalloc(&data, std::max<size_t>(size, 1) * sizeof(T)));
    if (size) HIP_OK(hipMemcpy(data, h.data(), size * sizeof(T), hipMemcpyHostToDevice));
  }
  explicit Buffer(size_t n) : Buffer(std::vector<T>(n)) {}
  Buffer(Buffer const&) = delete;
  ~Buffer() { (void)hipFree(data); }
  std::vector<T> host() const
  {
    std::vector<T> h(size);
    HIP_OK(hipDeviceSynchronize());
    if (size) HIP_OK(hipMemcpy(h.data(), data, size * sizeof(T), hipMemcpyDeviceToHost));
    return h;
  }
};

enc::heads view(Buffer<float> const& b, int64_t tokens, int64_t count, int64_t width) { return {b.data, enc::element::FLOAT32, tokens, count, width}; }

enc::rows of(Buffer<int32_t> const& offsets) { return {{offsets.data, offsets.size}, {}}; }

std::vector<float> values(size_t n, int seed)
{
  std::vector<float> v(n);
  uint32_t state = 12345u + static_cast<uint32_t>(seed);
  for (auto& x : v) {
    state = state * 1664525u + 1013904223u;
    x     = static_cast<float>(state >> 8) / 8388608.f - 1.f;
  }
  return v;
}

bool near(std::vector<float> const& got, std::vector<double> const& expected, double tolerance)
{
  if (got.size() != expected.size()) return false;
  for (size_t i = 0; i < got.size(); ++i)
    if (!(std::fabs(got[i] - expected[i]) <= tolerance)) return false;
  return true;
}

void test_rotary()
{
  std::printf("rotary positions\n");
  int const tokens = 5, heads = 2, width = 6, pairs = 2;
  std::vector<int32_t> const offsets{0, 2, 5}, starts{7, 0};
  std::vector<double> const frequencies{1.0, 0.03};
  auto const x = values(tokens * heads * width, 1);
  Buffer<int32_t> doffsets(offsets), dstarts(starts);
  Buffer<double> df(frequencies);
  Buffer<float> dx(x), out(x.size());
  for (bool half : {true, false}) {
    enc::rotary(view(dx, tokens, heads, width), of(doffsets), {df.data, df.size}, half ? enc::rotary_layout::HALF : enc::rotary_layout::INTERLEAVED, view(out, tokens, heads, width),
                {dstarts.data, dstarts.size}, false, 1.5);
    std::vector<double> expected(x.begin(), x.end());
    for (int r = 0; r < 2; ++r)
      for (int t = offsets[r]; t < offsets[r + 1]; ++t)
        for (int h = 0; h < heads; ++h)
          for (int n = 0; n < pairs; ++n) {
            int const first = (t * heads + h) * width, i = first + (half ? n : 2 * n), j = first + (half ? n + pairs : 2 * n + 1);
            double const angle = (starts[r] + t - offsets[r]) * frequencies[n];
            expected[i]        = 1.5 * (x[i] * std::cos(angle) - x[j] * std::sin(angle));
            expected[j]        = 1.5 * (x[i] * std::sin(angle) + x[j] * std::cos(angle));
          }
    CHECK(near(out.host(), expected, 2e-6));
  }
  // in place, and back
  enc::rotary(view(dx, tokens, heads, width), of(doffsets), {df.data, df.size}, enc::rotary_layout::HALF, view(dx, tokens, heads, width));
  enc::rotary(view(dx, tokens, heads, width), of(doffsets), {df.data, df.size}, enc::rotary_layout::HALF, view(dx, tokens, heads, width), {}, true);
  CHECK(near(dx.host(), {x.begin(), x.end()}, 2e-6));
  EXPECT_THROW(enc::rotary(view(dx, tokens, heads, width), {}, {df.data, df.size}, enc::rotary_layout::HALF, view(out, tokens, heads, width)), std::invalid_argument);
  EXPECT_THROW(enc::rotary(view(dx, tokens, heads, width), of(doffsets), {df.data, df.size}, enc::rotary_layout::HALF, view(out, tokens, heads, width), {dstarts.data, 1}),
               std::invalid_argument);
  EXPECT_THROW(enc::rotary(view(dx, tokens, heads, 2), of(doffsets), {df.data, df.size}, enc::rotary_layout::HALF, view(out, tokens, heads, 2)), std::invalid_argument);
}

// the formulas, a token and a head at a time, for keys first .. first + count - 1 of a row and its tokens; gradients are added up
struct Attention {
  int heads, kv_heads, width;
  double scale;
  std::vector<float> q, k, v, grad;
  std::vector<double> out, logsum, dq, dk, dv;
  void row(int begin, int tokens, int first, int count, bool causal, int all_tokens)
  {
    for (int i = 0; i < tokens; ++i)
      for (int h = 0; h < heads; ++h) {
        int const seen = causal ? std::max(0, std::min(count, i + 1 + count - tokens)) : count, kh = h / (heads / kv_heads);
        int const at = ((begin + i) * heads + h) * width;
        auto const key = [&](int j) { return ((first + j) * kv_heads + kh) * width; };
        std::vector<double> s(seen);
        double sum = 0, delta = 0;
        for (int j = 0; j < seen; ++j) {
          for (int d = 0; d < width; ++d) s[j] += scale * q[at + d] * k[key(j) + d];
          sum += std::exp(s[j]);
        }
        logsum[h * all_tokens + begin + i] = std::log(sum);
        for (int j = 0; j < seen; ++j)
          for (int d = 0; d < width; ++d) out[at + d] += std::exp(s[j]) / sum * v[key(j) + d];
        for (int d = 0; d < width; ++d) delta += grad[at + d] * out[at + d];
        for (int j = 0; j < seen; ++j) {
          double dp = 0;
          for (int d = 0; d < width; ++d) dp += static_cast<double>(grad[at + d]) * v[key(j) + d];
          double const p = std::exp(s[j]) / sum, ds = p * (dp - delta) * scale;
          for (int d = 0; d < width; ++d) {
            dq[at + d] += ds * k[key(j) + d];
            dk[key(j) + d] += ds * q[at + d];
            dv[key(j) + d] += p * grad[at + d];
          }
        }
      }
  }
};

void test_attention()
{
  std::printf("attention\n");
  int const tokens = 7, places = 12, heads = 4, kv_heads = 2, width = 8;
  std::vector<int32_t> const offsets{0, 3, 7}, key_offsets{1, 6, 12}, key_lengths{4, 6};
  Attention a{heads, kv_heads, width, 0.5, values(tokens * heads * width, 2), values(places * kv_heads * width, 3), values(places * kv_heads * width, 4), values(tokens * heads * width, 5),
              std::vector<double>(tokens * heads * width), std::vector<double>(heads * tokens), std::vector<double>(tokens * heads * width), std::vector<double>(places * kv_heads * width),
              std::vector<double>(places * kv_heads * width)};
  for (int r = 0; r < 2; ++r) a.row(offsets[r], offsets[r + 1] - offsets[r], key_offsets[r], key_lengths[r], true, tokens);
  Buffer<int32_t> doffsets(offsets), dkey(key_offsets), dlengths(key_lengths);
  Buffer<float> q(a.q), k(a.k), v(a.v), grad(a.grad), out(a.out.size()), logsum(a.logsum.size()), dq(a.dq.size()), dk(a.dk.size()), dv(a.dv.size());
  enc::rows const keys{{dkey.data, dkey.size}, {dlengths.data, dlengths.size}};
  enc::attention(view(q, tokens, heads, width), view(k, places, kv_heads, width), view(v, places, kv_heads, width), of(doffsets), keys, true, 0.5, view(out, tokens, heads, width),
                 {logsum.data, logsum.size});
  CHECK(near(out.host(), a.out, 1e-5));
  CHECK(near(logsum.host(), a.logsum, 1e-5));
  enc::attention_backward(view(grad, tokens, heads, width), view(q, tokens, heads, width), view(k, places, kv_heads, width), view(v, places, kv_heads, width), view(out, tokens, heads, width),
                          {logsum.data, logsum.size}, {}, of(doffsets), keys, true, 0.5, view(dq, tokens, heads, width), view(dk, places, kv_heads, width), view(dv, places, kv_heads, width));
  CHECK(near(dq.host(), a.dq, 1e-5));
  CHECK(near(dk.host(), a.dk, 1e-5));
  CHECK(near(dv.host(), a.dv, 1e-5));
  // the tokens' own keys; wrong sizes
  Buffer<float> same(a.out.size());
  enc::attention(view(q, tokens, heads, width), view(q, tokens, heads, width), view(grad, tokens, heads, width), of(doffsets), {}, false, 0.5, view(same, tokens, heads, width));
  EXPECT_THROW(enc::attention(view(q, tokens, heads, width), view(k, places, kv_heads, width), view(v, places, kv_heads, width), of(doffsets), {}, true, 0.5, view(out, tokens, heads, width)),
               std::invalid_argument);
  EXPECT_THROW(enc::attention(view(q, tokens, heads, width), view(k, places, kv_heads, width), view(v, places, kv_heads, width), of(doffsets), keys, true, 0.5,
                              view(out, tokens, heads, width), {logsum.data, 3}),
               std::invalid_argument);
  EXPECT_THROW(enc::attention(view(q, tokens, heads, width), view(k, places, kv_heads, width), view(v, places, kv_heads, width), keys, keys, true, 0.5, view(out, tokens, heads, width)),
               std::invalid_argument);
}

int main()
{
  int devices = 0;
  if (hipGetDeviceCount(&devices) != hipSuccess || devices == 0) {
    std::printf("no GPU\n");
    return 77;
  }
  test_rotary();
  test_attention();
  std::printf(g_failures ? "FAILED (%d checks)\n" : "ALL PASSED\n", g_failures);
  return g_failures ? 1 : 0;
}
