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

}  // namespace nvtext::encoder
