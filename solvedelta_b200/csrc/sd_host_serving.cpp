// Host side of the serving operators: 8-bit projections and token sampling.  Checks, tensors, one C call each.
#include "sd_host.h"

#include <cmath>

namespace {

int element_type(const Tensor& t) { return t.scalar_type() == at::kFloat ? SD_F32 : SD_BF16; }
bool is_real(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }

// The calls record nothing, and skip autograd's part of every tensor operation (about a tenth of a short call each).
using NoAutograd = at::AutoDispatchBelowADInplaceOrView;

// [..., K] as rows with unit channel stride and one stride between them; a view where the layout has that.
Tensor as_rows(const Tensor& t) {
    const int64_t K = t.size(-1);
    Tensor r = t.dim() == 2 ? t : t.reshape({-1, K});
    return r.stride(1) == 1 || K == 1 ? r : r.contiguous();
}
int64_t row_stride(const Tensor& rows) { return rows.size(0) > 1 ? rows.stride(0) : std::max<int64_t>(rows.stride(0), rows.size(1)); }

// Rows that quantize_rows made are read in place; others are copied.
Tensor readable(const Tensor& rows) {
    if (int8_readable(rows)) return rows;
    Tensor copy = at::empty({rows.size(0), int8_padded(rows.size(1))}, rows.options()).narrow(1, 0, rows.size(1));
    copy.copy_(rows);
    return copy;
}

void require_no_gradient(std::initializer_list<const Tensor*> tensors) {
    for (const Tensor* t : tensors)   // tangents pass whether gradients are recorded or not
        if (t->defined() && t->_fw_grad(0).defined())
            throw std::runtime_error("8-bit projections have no forward-mode derivative: call them on tensors without tangents");
    if (!at::GradMode::is_enabled()) return;
    for (const Tensor* t : tensors)
        if (t->defined() && t->requires_grad())
            throw std::runtime_error("8-bit projections have no reverse pass: call them under torch.no_grad(), or on detached tensors");
}

void check_width(int64_t K) {
    value_error(K < 1, "rows must have at least one entry");
    value_error(K > 131072, "rows longer than 131072 entries are not supported: their sums may leave 32 bits");
}

py::tuple quantize_rows(const Tensor& x) {
    type_error(!x.is_cuda() || !is_real(x), "x must be a BF16 or FP32 CUDA tensor");
    value_error(x.dim() < 1, "x must be [...,K]");
    const int64_t K = x.size(-1);
    check_width(K);
    const c10::cuda::CUDAGuard guard(x.device());
    const NoAutograd below;
    const Tensor rows = as_rows(x);
    const int64_t M = rows.size(0);
    value_error(M > 0x7fffffffLL, "too many rows");
    const int64_t pitch = int8_padded(K);
    std::vector<int64_t> shape = x.sizes().vec();
    const bool dense = pitch == K;   // else the rows' padding is cut off below
    Tensor q = dense ? at::empty(shape, x.options().dtype(at::kChar)) : at::empty({M, pitch}, x.options().dtype(at::kChar));
    Tensor scale = f32_like(x, x.sizes().slice(0, x.dim() - 1));
    if (M > 0) {
        sd_quantize_rows_args a{};
        a.rows = M; a.K = (int32_t)K; a.x_type = element_type(rows); a.x = rows.data_ptr(); a.x_stride = row_stride(rows);
        a.q = q.data_ptr(); a.q_stride = pitch; a.scale = f32(scale);
        check(sd_quantize_rows(&a, stream_of(x)));
    }
    if (!dense) {
        std::vector<int64_t> stride(shape.size(), 1);
        int64_t step = pitch;
        for (int64_t d = (int64_t)shape.size() - 2; d >= 0; --d) {
            stride[d] = step;
            step *= std::max<int64_t>(shape[d], 1);
        }
        q = q.as_strided(shape, stride);
    }
    return py::make_tuple(q, scale);
}

at::ScalarType output_type(const py::object& dtype) {
    type_error(!THPDtype_Check(dtype.ptr()), "out_dtype must be torch.bfloat16 or torch.float32");
    const at::ScalarType type = reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type;
    type_error(type != at::kBFloat16 && type != at::kFloat, "out_dtype must be torch.bfloat16 or torch.float32");
    return type;
}

// x: BF16 / FP32 rows, or int8 rows with their scales.  `chained`: the kernel before is this library's, launched behind
// everything that may have written the weight.
Tensor product(const Tensor& x, const Tensor& scale_in, const Tensor& weight_in, const Tensor& weight_scale_in,
               const OptTensor& bias_in, bool swiglu, at::ScalarType out_type, bool chained = false) {
    const Tensor bias = given(bias_in);
    const bool quantized = scale_in.defined();
    type_error(!weight_in.is_cuda() || weight_in.scalar_type() != at::kChar, "weight must be an int8 CUDA tensor");
    value_error(weight_in.dim() != 2, "weight must be [N,K]");
    const int64_t N = weight_in.size(0), K = weight_in.size(1);
    value_error(x.dim() < 1 || x.size(-1) != K, "the last axis of the rows must be as long as the weight's");
    check_width(K);
    value_error(N < 1 || N > 0x7fffff00LL, "weight must have at least one row, and fewer than 2^31");
    value_error(swiglu && N % 2 != 0, "with swiglu the weight holds gate rows and as many value rows");
    type_error(weight_scale_in.scalar_type() != at::kFloat, "weight_scale must be FP32");
    value_error(!is_shape(weight_scale_in, {N}), "weight_scale must be [N]");
    if (bias.defined()) {
        type_error(!is_real(bias), "bias must be BF16 or FP32");
        value_error(!is_shape(bias, {N}), "bias must be [N]");
    }
    for (const Tensor* t : {&weight_in, &weight_scale_in, &bias, &scale_in})
        value_error(t->defined() && t->device() != x.device(), "all tensors must be on the device of the rows");
    require_no_gradient({&x, &scale_in, &weight_scale_in, &bias});

    const c10::cuda::CUDAGuard guard(x.device());
    const NoAutograd below;
    std::vector<int64_t> shape = x.sizes().vec();
    if (quantized) {
        type_error(scale_in.scalar_type() != at::kFloat, "scale must be FP32");
        value_error(!is_shape(scale_in, x.sizes().slice(0, x.dim() - 1)), "scale must have the shape of the rows without their last axis");
    }
    Tensor rows = as_rows(x);
    const int64_t M = rows.size(0);
    value_error(M > 0x7fffff00LL, "too many rows");
    shape.back() = swiglu ? N / 2 : N;
    Tensor y = at::empty(shape, x.options().dtype(out_type));
    if (M == 0) return y;
    if (quantized) rows = readable(rows);
    const Tensor weight = readable(weight_in), weight_scale = weight_scale_in.contiguous();
    const Tensor scale = !quantized ? Tensor() : scale_in.is_contiguous() ? scale_in : scale_in.contiguous();
    const Tensor b = bias.defined() ? bias.contiguous() : Tensor();
    // a copy made here is written by the kernel before
    chained = chained && weight.data_ptr() == weight_in.data_ptr() && weight_scale.data_ptr() == weight_scale_in.data_ptr() &&
              (!b.defined() || b.data_ptr() == bias.data_ptr());
    sd_int8_linear_args a{};
    a.rows = M; a.N = (int32_t)N; a.K = (int32_t)K; a.swiglu = swiglu ? 1 : 0;
    a.x_type = quantized ? SD_I8 : element_type(rows); a.y_type = out_type == at::kFloat ? SD_F32 : SD_BF16;
    a.x = rows.data_ptr(); a.x_stride = quantized ? int8_stride(rows) : row_stride(rows); a.x_scale = f32(scale);
    a.weight = weight.data_ptr(); a.weight_stride = int8_stride(weight); a.weight_scale = f32(weight_scale);
    a.bias = raw(b); a.bias_type = b.defined() ? element_type(b) : SD_BF16;
    a.y = y.data_ptr(); a.y_stride = shape.back();
    const size_t need = sd_int8_linear_scratch_bytes(&a);
    const Tensor scratch = need > 0 ? workspace(x, need) : Tensor();
    a.scratch = raw(scratch); a.scratch_bytes = need; a.chained = chained ? 1 : 0;
    check(sd_int8_linear(&a, stream_of(x)));
    return y;
}

Tensor int8_linear(const Tensor& x, const Tensor& weight, const Tensor& weight_scale, const OptTensor& bias, bool swiglu,
                   const py::object& out_dtype) {
    type_error(!x.is_cuda() || !is_real(x), "x must be a BF16 or FP32 CUDA tensor");
    return product(x, Tensor(), weight, weight_scale, bias, swiglu, output_type(out_dtype));
}
Tensor int8_matmul(const Tensor& q, const Tensor& scale, const Tensor& weight, const Tensor& weight_scale, const OptTensor& bias,
                   bool swiglu, const py::object& out_dtype) {
    type_error(!q.is_cuda() || q.scalar_type() != at::kChar, "q must be an int8 CUDA tensor");
    return product(q, scale, weight, weight_scale, bias, swiglu, output_type(out_dtype));
}

// The gated MLP: its second product is chained to the first.
Tensor int8_gated_mlp(const Tensor& x, const Tensor& up, const Tensor& up_scale, const OptTensor& up_bias, const Tensor& down,
                      const Tensor& down_scale, const OptTensor& down_bias) {
    type_error(!x.is_cuda() || !is_real(x), "x must be a BF16 or FP32 CUDA tensor");
    const Tensor act = product(x, Tensor(), up, up_scale, up_bias, true, at::kBFloat16);
    return product(act, Tensor(), down, down_scale, down_bias, false, at::kBFloat16, true);
}

// ---- sampling -----------------------------------------------------------------------------------------------
// A setting: one number for all rows, or a tensor with one for each.
Tensor row_setting(const py::object& value, const char* name, const Tensor& logits, at::ScalarType type) {
    if (!THPVariable_Check(value.ptr())) return {};
    const Tensor t = value.cast<Tensor>();
    if (!is_shape(t, {logits.size(0)})) throw py::value_error(std::string(name) + " must be a number or a tensor [B]");
    if (t.device() != logits.device()) throw py::value_error(std::string(name) + " must be on the device of the logits");
    if (type == at::kInt ? !at::isIntegralType(t.scalar_type(), false) : !at::isFloatingType(t.scalar_type()))
        throw py::type_error(std::string(name) + (type == at::kInt ? " must hold whole numbers" : " must hold real numbers"));
    if (type == at::kInt && t.scalar_type() == at::kLong) return t.clamp(0, 0x7fffffff).to(type).contiguous();
    return t.to(type).contiguous();
}

Tensor sample_tokens(const Tensor& logits_in, const Tensor& uniform, const py::object& temperature, const py::object& top_k,
                     const py::object& top_p, const py::object& min_p, int64_t empty_token) {
    type_error(!logits_in.is_cuda() || !is_real(logits_in), "logits must be a BF16 or FP32 CUDA tensor");
    value_error(logits_in.dim() != 2 || logits_in.size(1) < 1, "logits must be [B,V]");
    value_error(logits_in.size(1) > 262144, "vocabularies of more than 262144 entries are not supported");
    const int64_t B = logits_in.size(0), V = logits_in.size(1);
    type_error(uniform.scalar_type() != at::kFloat, "uniform must be FP32");
    value_error(!is_shape(uniform, {B}) || uniform.device() != logits_in.device(), "uniform must be [B] on the device of the logits");
    const c10::cuda::CUDAGuard guard(logits_in.device());
    const NoAutograd below;
    const Tensor logits = as_rows(logits_in), u = uniform.contiguous();
    const Tensor t = row_setting(temperature, "temperature", logits, at::kFloat), k = row_setting(top_k, "top_k", logits, at::kInt),
                 tp = row_setting(top_p, "top_p", logits, at::kFloat), mp = row_setting(min_p, "min_p", logits, at::kFloat);
    sd_sample_tokens_args a{};
    a.temperature = t.defined() ? 0.0 : temperature.cast<double>();
    a.top_p = tp.defined() ? 1.0 : top_p.cast<double>();
    a.min_p = mp.defined() ? 0.0 : min_p.cast<double>();
    const int64_t whole_k = k.defined() ? 0 : top_k.cast<int64_t>();
    value_error(!std::isfinite(a.temperature) || a.temperature < 0, "temperature must be finite and not negative");
    value_error(!(a.top_p >= 0 && a.top_p <= 1), "top_p must be between 0 and 1");
    value_error(!(a.min_p >= 0 && a.min_p <= 1), "min_p must be between 0 and 1");
    value_error(whole_k < 0, "top_k must not be negative");
    a.top_k = (int32_t)std::min<int64_t>(whole_k, 0x7fffffff);
    Tensor tokens = at::empty({B}, logits.options().dtype(at::kLong));
    if (B == 0) return tokens;
    a.rows = B; a.V = (int32_t)V; a.logits_type = element_type(logits); a.logits = logits.data_ptr(); a.stride = row_stride(logits);
    a.uniform = f32(u);
    a.temperature_row = f32(t); a.top_p_row = f32(tp); a.min_p_row = f32(mp);
    a.top_k_row = k.defined() ? k.data_ptr<int32_t>() : nullptr;
    a.empty_token = empty_token;
    a.tokens = tokens.data_ptr<int64_t>();
    check(sd_sample_tokens(&a, stream_of(logits)));
    return tokens;
}

}  // namespace

void register_serving(py::module_& m) {
    m.def("quantize_rows", &quantize_rows);
    m.def("int8_linear", &int8_linear);
    m.def("int8_matmul", &int8_matmul);
    m.def("int8_gated_mlp", &int8_gated_mlp);
    m.def("sample_tokens", &sample_tokens);
}
