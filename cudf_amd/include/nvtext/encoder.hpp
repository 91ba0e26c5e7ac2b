// nvtext::encoder: the operators between wordpiece_tokenize's column of ids and a model that learns from it, over the C ABI in
// include/nvtext_amd_encoder.h, which says what each computes.  Matrices are views of memory that the caller owns; errors are
// thrown as by the other nvtext calls.
#pragma once
#include <cudf/lists/lists_column_view.hpp>
#include <cudf/utilities/span.hpp>
#include <nvtext/detail_result.hpp>
#include <nvtext_amd_encoder.h>
#include <rmm/resource_ref.hpp>

#include <cstdint>

namespace nvtext::encoder {

enum class element : int32_t { FLOAT32 = NVTEXT_AMD_TYPE_FLOAT32, FLOAT16 = NVTEXT_AMD_TYPE_FLOAT16, BFLOAT16 = NVTEXT_AMD_TYPE_BFLOAT16 };

enum class activation : int32_t {
  NONE      = NVTEXT_AMD_ACTIVATION_NONE,
  RELU      = NVTEXT_AMD_ACTIVATION_RELU,
  GELU      = NVTEXT_AMD_ACTIVATION_GELU,
  GELU_TANH = NVTEXT_AMD_ACTIVATION_GELU_TANH,
  SILU      = NVTEXT_AMD_ACTIVATION_SILU
};

// `rows` rows of `cols` values, one every `stride` values (0: every `cols`); without data, no matrix: an argument left out.
class matrix {
 public:
  matrix() = default;
  matrix(void* data, element type, int64_t rows, int64_t cols, int64_t stride = 0)
    : _there{true}, _m{data, rows, cols, stride == 0 ? cols : stride, static_cast<int32_t>(type)}
  {
  }
  [[nodiscard]] nvtext_amd_matrix const* c_view() const { return _there ? &_m : nullptr; }

 private:
  bool _there{false};
  nvtext_amd_matrix _m{};
};

// What is dropped: each value with probability p, by the draws of a seed and a call's own number under it.
struct dropped {
  double p{0};
  uint64_t seed{0};
  uint32_t offset{0};
};

namespace detail {
// a LIST<INT32> column, sliced or not, as the C ABI takes it (a null row holds no tokens)
inline nvtext_amd_list_column tokens_view(cudf::lists_column_view const& tokens)
{
  nvtext_amd_list_column c{};
  c.size       = tokens.size();
  c.child_type = NVTEXT_AMD_TYPE_INT32;
  if (tokens.num_children() > 1) {
    CUDF_EXPECTS(tokens.offsets().type().id() == cudf::type_id::INT32, "list offsets must be INT32");
    c.child_type   = static_cast<int32_t>(tokens.child().type().id());
    c.offsets_size = tokens.size() + 1;
    c.offsets      = const_cast<int32_t*>(tokens.offsets().head<int32_t>() + tokens.offset());
    c.child        = const_cast<int32_t*>(tokens.child().data<int32_t>());
    c.child_size   = tokens.child().size();
  } else {
    CUDF_EXPECTS(tokens.size() == 0, "a lists column with rows needs offsets and a child");
  }
  return c;
}
}  // namespace detail

inline void embedding(cudf::lists_column_view const& tokens, matrix const& token_table, matrix const& position_table, matrix const& out,
                      cuda::stream_ref stream = cudf::get_default_stream())
{
  auto const c = detail::tokens_view(tokens);
  nvtext::detail::throw_on_error(nvtext_amd_embedding(&c, token_table.c_view(), position_table.c_view(), stream.get(), out.c_view()));
}

inline void embedding_backward(cudf::lists_column_view const& tokens, matrix const& grad, matrix const& token_grad, matrix const& position_grad,
                               cuda::stream_ref stream = cudf::get_default_stream(), rmm::device_async_resource_ref mr = cudf::get_current_device_resource_ref())
{
  auto const c = detail::tokens_view(tokens);
  nvtext_amd_allocator storage{};
  nvtext::detail::throw_on_error(nvtext_amd_embedding_backward(&c, grad.c_view(), stream.get(), mr.c_allocator(storage), token_grad.c_view(), position_grad.c_view()));
}

inline void dropout(matrix const& x, dropped const& d, matrix const& out, cuda::stream_ref stream = cudf::get_default_stream())
{
  nvtext::detail::throw_on_error(nvtext_amd_dropout(x.c_view(), d.p, d.seed, d.offset, stream.get(), out.c_view()));
}

inline void layer_norm(matrix const& x, matrix const& residual, matrix const& weight, matrix const& bias, double eps, dropped const& d, matrix const& out,
                       matrix const& sum = {}, cudf::device_span<float> mean = {}, cudf::device_span<float> rstd = {},
                       cuda::stream_ref stream = cudf::get_default_stream())
{
  for (auto const& s : {mean, rstd})
    if (s.data() && x.c_view() && static_cast<int64_t>(s.size()) != x.c_view()->rows) throw std::invalid_argument("mean and rstd hold a value a row");
  nvtext::detail::throw_on_error(nvtext_amd_layer_norm(x.c_view(), residual.c_view(), weight.c_view(), bias.c_view(), eps, d.p, d.seed, d.offset, stream.get(),
                                                       out.c_view(), sum.c_view(), mean.data(), rstd.data()));
}

inline void layer_norm_backward(matrix const& grad, matrix const& sum, cudf::device_span<float const> mean, cudf::device_span<float const> rstd, matrix const& weight,
                                matrix const& sum_grad, dropped const& d, matrix const& x_grad, matrix const& residual_grad, matrix const& weight_grad,
                                matrix const& bias_grad, cuda::stream_ref stream = cudf::get_default_stream(),
                                rmm::device_async_resource_ref mr = cudf::get_current_device_resource_ref())
{
  for (auto const& s : {mean, rstd})
    if (grad.c_view() && static_cast<int64_t>(s.size()) != grad.c_view()->rows) throw std::invalid_argument("mean and rstd hold a value a row");
  nvtext_amd_allocator storage{};
  nvtext::detail::throw_on_error(nvtext_amd_layer_norm_backward(grad.c_view(), sum.c_view(), mean.data(), rstd.data(), weight.c_view(), sum_grad.c_view(), d.p, d.seed,
                                                                d.offset, stream.get(), mr.c_allocator(storage), x_grad.c_view(), residual_grad.c_view(),
                                                                weight_grad.c_view(), bias_grad.c_view()));
}

inline void linear(matrix const& x, matrix const& weight, matrix const& bias, activation act, matrix const& residual, matrix const& out,
                   matrix const& preactivation = {}, cuda::stream_ref stream = cudf::get_default_stream(),
                   rmm::device_async_resource_ref mr = cudf::get_current_device_resource_ref())
{
  nvtext_amd_allocator storage{};
  nvtext::detail::throw_on_error(nvtext_amd_linear(x.c_view(), weight.c_view(), bias.c_view(), static_cast<int32_t>(act), residual.c_view(), stream.get(),
                                                   mr.c_allocator(storage), out.c_view(), preactivation.c_view()));
}

inline void linear_backward(matrix const& grad, matrix const& x, matrix const& weight, activation act, matrix const& preactivation, matrix const& x_grad,
                            matrix const& weight_grad, matrix const& bias_grad, cuda::stream_ref stream = cudf::get_default_stream(),
                            rmm::device_async_resource_ref mr = cudf::get_current_device_resource_ref())
{
  nvtext_amd_allocator storage{};
  nvtext::detail::throw_on_error(nvtext_amd_linear_backward(grad.c_view(), x.c_view(), weight.c_view(), static_cast<int32_t>(act), preactivation.c_view(), stream.get(),
                                                            mr.c_allocator(storage), x_grad.c_view(), weight_grad.c_view(), bias_grad.c_view()));
}

enum class rotary_layout : int32_t { HALF = NVTEXT_AMD_ROTARY_HALF, INTERLEAVED = NVTEXT_AMD_ROTARY_INTERLEAVED };

// The heads of `tokens` tokens, `count` of `width` values each, one token every `stride` values (0: every count * width) and one head every
// `head_stride` (0: every width).
class heads {
 public:
  heads() = default;
  heads(void* data, element type, int64_t tokens, int64_t count, int64_t width, int64_t stride = 0, int64_t head_stride = 0)
    : _there{true}, _h{data, tokens, count, width, stride == 0 ? count * width : stride, head_stride == 0 ? width : head_stride, static_cast<int32_t>(type)}
  {
  }
  [[nodiscard]] nvtext_amd_heads const* c_view() const { return _there ? &_h : nullptr; }

 private:
  bool _there{false};
  nvtext_amd_heads _h{};
};

// Which tokens make up a row: offsets, one more than there are rows; of keys with room behind a row's, how many there are, too.
struct rows {
  cudf::device_span<int32_t const> offsets{};
  cudf::device_span<int32_t const> lengths{};
  [[nodiscard]] int32_t size() const
  {
    if (offsets.size() == 0) throw std::invalid_argument("offsets must have a value more than there are rows");
    return static_cast<int32_t>(offsets.size() - 1);
  }
};

namespace detail {
// (offsets and lengths of the keys; neither where they are those of the tokens)
inline rows keys_of(rows const& tokens, rows const& keys)
{
  if (tokens.lengths.data()) throw std::invalid_argument("only keys have lengths");
  if (keys.offsets.size() != 0 && keys.size() != tokens.size()) throw std::invalid_argument("there must be as many rows of keys as of tokens");
  if (keys.lengths.data() && static_cast<int64_t>(keys.lengths.size()) != tokens.size()) throw std::invalid_argument("there must be a length for every row");
  return keys;
}
}  // namespace detail

inline void rotary(heads const& x, rows const& tokens, cudf::device_span<double const> frequencies, rotary_layout layout, heads const& out,
                   cudf::device_span<int32_t const> starts = {}, bool inverse = false, double magnitude = 1.0, cuda::stream_ref stream = cudf::get_default_stream())
{
  if (starts.data() && static_cast<int64_t>(starts.size()) != tokens.size()) throw std::invalid_argument("there must be a start for every row");
  nvtext::detail::throw_on_error(nvtext_amd_rotary(x.c_view(), tokens.size(), tokens.offsets.data(), starts.data(), frequencies.data(), static_cast<int64_t>(frequencies.size()),
                                                   static_cast<int32_t>(layout), inverse, magnitude, stream.get(), out.c_view()));
}

// keys: left out where they are the tokens' own
inline void attention(heads const& q, heads const& k, heads const& v, rows const& tokens, rows const& keys, bool causal, double scale, heads const& out,
                      cudf::device_span<float> logsum = {}, cudf::device_span<int8_t> rest = {}, cuda::stream_ref stream = cudf::get_default_stream(),
                      rmm::device_async_resource_ref mr = cudf::get_current_device_resource_ref())
{
  auto const* c = q.c_view();
  if (c && logsum.data() && static_cast<int64_t>(logsum.size()) != c->heads * c->tokens) throw std::invalid_argument("logsum holds a value a head of a token");
  if (c && rest.data() && static_cast<int64_t>(rest.size()) != c->heads * c->tokens * c->width) throw std::invalid_argument("rest holds a value for each of q's");
  rows const of_keys = detail::keys_of(tokens, keys);
  nvtext_amd_allocator storage{};
  nvtext::detail::throw_on_error(nvtext_amd_attention(q.c_view(), k.c_view(), v.c_view(), tokens.size(), tokens.offsets.data(), of_keys.offsets.data(), of_keys.lengths.data(), causal,
                                                      scale, stream.get(), mr.c_allocator(storage), out.c_view(), logsum.data(), rest.data()));
}

inline void attention_backward(heads const& grad, heads const& q, heads const& k, heads const& v, heads const& out, cudf::device_span<float const> logsum,
                               cudf::device_span<int8_t const> rest, rows const& tokens, rows const& keys, bool causal, double scale, heads const& q_grad, heads const& k_grad,
                               heads const& v_grad, cuda::stream_ref stream = cudf::get_default_stream(),
                               rmm::device_async_resource_ref mr = cudf::get_current_device_resource_ref())
{
  auto const* c = q.c_view();
  if (c && static_cast<int64_t>(logsum.size()) != c->heads * c->tokens) throw std::invalid_argument("logsum holds a value a head of a token");
  if (c && rest.data() && static_cast<int64_t>(rest.size()) != c->heads * c->tokens * c->width) throw std::invalid_argument("rest holds a value for each of q's");
  rows const of_keys = detail::keys_of(tokens, keys);
  nvtext_amd_allocator storage{};
  nvtext::detail::throw_on_error(nvtext_amd_attention_backward(grad.c_view(), q.c_view(), k.c_view(), v.c_view(), out.c_view(), logsum.data(), rest.data(), tokens.size(),
                                                               tokens.offsets.data(), of_keys.offsets.data(), of_keys.lengths.data(), causal, scale, stream.get(),
                                                               mr.c_allocator(storage), q_grad.c_view(), k_grad.c_view(), v_grad.c_view()));
}

}  // namespace nvtext::encoder
