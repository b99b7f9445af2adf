// Tensor front ends of the experts' feed-forward operators, as front.cpp has those of the others: contiguous operands of one
// type on the current device; nothing for any other form, which hip_ops.py converts, copies or refuses.
#include "front.h"

#include <c10/hip/HIPFunctions.h>

namespace ddl_front {
namespace {

bool here(const Tensor& t) { return plain(t) && t.device().index() == c10::hip::current_device(); }
bool alike(const MaybeTensor& t, const Tensor& x) { return !t || (here(*t) && t->scalar_type() == x.scalar_type() && t->sizes() == x.sizes()); }
bool int32(const Tensor& t) { return here(t) && t.scalar_type() == at::kInt; }
bool floats_of(const Tensor& t, at::IntArrayRef shape) { return here(t) && t.scalar_type() == at::kFloat && t.sizes() == shape; }

// [..., cols] rows that the norm takes, with a weight of their own.
bool norm_rows(const Tensor& x, const MaybeTensor& weight) {
    return here(x) && float_code(x) && x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 16384 &&
           (!weight || (here(*weight) && weight->scalar_type() == x.scalar_type() && weight->numel() == x.size(-1)));
}
Tensor floats(const Tensor& like, at::IntArrayRef shape) { return at::empty(shape, like.options().dtype(at::kFloat)); }

bool plan_tensors(const Tensor& place, const Tensor& offsets) { return int32(place) && place.dim() == 2 && int32(offsets) && offsets.dim() == 1 && offsets.numel() >= 1; }
const int32_t* held_of(const Tensor& offsets) { return offsets.data_ptr<int32_t>() + offsets.numel() - 1; }
bool rows_of(const Tensor& t, int64_t count) { return here(t) && t.dim() == 2 && t.size(0) == count && t.size(1) >= 1; }

// [rows, k], [experts, n, k] and [experts + 1]
bool expert_operands(const Tensor& x, const Tensor& w, const Tensor& offsets) {
    return here(x) && here(w) && x.dim() == 2 && w.dim() == 3 && x.size(1) == w.size(2) && x.size(1) >= 1 && w.size(1) >= 1 && x.scalar_type() == w.scalar_type() && int32(offsets) &&
           offsets.dim() == 1 && offsets.size(0) == w.size(0) + 1;
}

}  // namespace

std::optional<Normed> rms_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& residual, double eps, bool eight_bit) {
    if (!norm_rows(x, weight) || !alike(residual, x) || !(eps >= 0)) return std::nullopt;
    const int64_t cols = x.size(-1), rows = x.numel() / cols;
    Normed res;
    if (residual) res.h = at::empty(x.sizes(), x.options());
    res.y = eight_bit ? at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn)) : at::empty(x.sizes(), x.options());
    if (eight_bit) res.scales = floats(x, x.sizes().slice(0, x.dim() - 1));
    check(ddl_rms_norm(x.data_ptr(), pointer(residual), pointer(weight), float_code(x), rows, cols, cols, cols, static_cast<float>(eps), pointer(res.h),
                       eight_bit ? nullptr : res.y.data_ptr(), eight_bit ? res.y.data_ptr() : nullptr, static_cast<float*>(pointer(res.scales)), nullptr, nullptr, 0, cols,
                       current_stream()),
          "ddl_rms_norm");
    return res;
}

std::optional<std::tuple<Tensor, Tensor>> quantize_rows(const Tensor& x) {
    if (!norm_rows(x, std::nullopt)) return std::nullopt;
    const int64_t cols = x.size(-1);
    Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn)), scales = floats(x, x.sizes().slice(0, x.dim() - 1));
    check(ddl_quantize_rows(x.data_ptr(), float_code(x), x.numel() / cols, cols, cols, codes.data_ptr(), scales.data_ptr<float>(), current_stream()), "ddl_quantize_rows");
    return std::make_tuple(codes, scales);
}

std::optional<Two> rms_norm_backward(const Tensor& dy, const Tensor& h, const MaybeTensor& weight, const MaybeTensor& dh, double eps, bool want_input, bool want_weight) {
    if (!norm_rows(h, weight) || !alike(dy, h) || !alike(dh, h)) return std::nullopt;
    const int64_t cols = h.size(-1), rows = h.numel() / cols;
    Tensor dx, dw, work;
    if (want_input) dx = at::empty(h.sizes(), h.options());
    int64_t elems = 0;
    if (want_weight && weight) {
        dw = at::empty(weight->sizes(), weight->options());
        elems = ddl_rms_norm_backward_workspace(rows, cols);
        work = floats(h, {elems});
    }
    check(ddl_rms_norm_backward(dy.data_ptr(), h.data_ptr(), pointer(dh), pointer(weight), float_code(h), rows, cols, cols, cols, cols, static_cast<float>(eps), pointer(dx),
                                pointer(dw), static_cast<float*>(pointer(work)), elems, nullptr, nullptr, nullptr, 0, cols, current_stream()),
          "ddl_rms_norm_backward");
    return Two(dx.defined() ? MaybeTensor(dx) : std::nullopt, dw.defined() ? MaybeTensor(dw) : std::nullopt);
}

std::optional<std::tuple<Tensor, Tensor>> expert_plan(const Tensor& ids, int64_t low, int64_t high) {
    if (!here(ids) || ids.dim() != 2 || (ids.scalar_type() != at::kLong && ids.scalar_type() != at::kInt) || high < low) return std::nullopt;
    const int64_t tokens = ids.size(0), chosen = ids.size(1), elems = ddl_expert_plan_workspace(tokens * chosen, high - low);
    const auto ints = ids.options().dtype(at::kInt);
    Tensor place = at::empty({tokens, chosen}, ints), offsets = at::empty({high - low + 1}, ints), work;
    if (elems) work = at::empty({elems}, ints);
    check(ddl_expert_plan(ids.data_ptr(), static_cast<int>(ids.element_size()), tokens, chosen, chosen, low, high, place.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(),
                          static_cast<int32_t*>(pointer(work)), elems, current_stream()),
          "ddl_expert_plan");
    return std::make_tuple(place, offsets);
}

std::optional<Two> expert_sort(const Tensor& x, const Tensor& place, const Tensor& offsets, const MaybeTensor& scales) {
    if (!plan_tensors(place, offsets) || !rows_of(x, place.size(0)) || (x.element_size() != 1 && x.element_size() != 2 && x.element_size() != 4) || x.is_complex() ||
        (scales && !floats_of(*scales, {place.size(0)})))
        return std::nullopt;
    const int64_t tokens = place.size(0), chosen = place.size(1), cols = x.size(1);
    Tensor out = at::empty({tokens * chosen, cols}, x.options()), out_scales;
    if (scales) out_scales = floats(x, {tokens * chosen});
    check(ddl_expert_sort(x.data_ptr(), static_cast<int>(x.element_size()), tokens, chosen, cols, cols, place.data_ptr<int32_t>(), held_of(offsets), out.data_ptr(),
                          static_cast<const float*>(pointer(scales)), static_cast<float*>(pointer(out_scales)), current_stream()),
          "ddl_expert_sort");
    return Two(out, scales ? MaybeTensor(out_scales) : std::nullopt);
}

MaybeTensor expert_combine(const Tensor& y, const Tensor& place, const Tensor& offsets, const MaybeTensor& weights) {
    if (!plan_tensors(place, offsets) || !rows_of(y, place.numel()) || !float_code(y) || (weights && !floats_of(*weights, place.sizes()))) return std::nullopt;
    const int64_t tokens = place.size(0), cols = y.size(1);
    Tensor out = at::empty({tokens, cols}, y.options());
    check(ddl_expert_combine(y.data_ptr(), float_code(y), tokens, place.size(1), cols, cols, place.data_ptr<int32_t>(), held_of(offsets),
                             static_cast<const float*>(pointer(weights)), out.data_ptr(), current_stream()),
          "ddl_expert_combine");
    return out;
}

std::optional<Two> expert_combine_backward(const Tensor& dout, const MaybeTensor& y, const Tensor& place, const Tensor& offsets, const Tensor& weights, bool want_rows,
                                           bool want_weights) {
    if (!plan_tensors(place, offsets) || !rows_of(dout, place.size(0)) || !float_code(dout) || !floats_of(weights, place.sizes()) ||
        (want_weights && (!y || !rows_of(*y, place.numel()) || y->size(1) != dout.size(1) || y->scalar_type() != dout.scalar_type())))
        return std::nullopt;
    const int64_t cols = dout.size(1);
    Tensor dy, dweights;
    if (want_rows) dy = at::empty({place.numel(), cols}, dout.options());
    if (want_weights) dweights = floats(dout, place.sizes());
    check(ddl_expert_combine_backward(dout.data_ptr(), want_weights ? pointer(y) : nullptr, float_code(dout), place.size(0), place.size(1), cols, cols, cols, place.data_ptr<int32_t>(),
                                      held_of(offsets), weights.data_ptr<float>(), pointer(dy), static_cast<float*>(pointer(dweights)), current_stream()),
          "ddl_expert_combine_backward");
    return Two(want_rows ? MaybeTensor(dy) : std::nullopt, want_weights ? MaybeTensor(dweights) : std::nullopt);
}

MaybeTensor expert_linear(const Tensor& x, const Tensor& w, const Tensor& offsets) {
    if (!expert_operands(x, w, offsets) || !float_code(x)) return std::nullopt;
    const int64_t rows = x.size(0), n = w.size(1), k = w.size(2);
    Tensor y = at::empty({rows, n}, x.options());
    check(ddl_expert_linear(x.data_ptr(), w.data_ptr(), float_code(x), offsets.data_ptr<int32_t>(), w.size(0), rows, n, k, k, y.data_ptr(), current_stream()),
          "ddl_expert_linear");
    return y;
}

MaybeTensor expert_linear_8bit(const Tensor& x, const Tensor& w, const Tensor& offsets, const Tensor& x_scales, const Tensor& w_scales, at::ScalarType dtype) {
    const int code = dtype == at::kFloat ? DDL_DT_F32 : dtype == at::kBFloat16 ? DDL_DT_BF16 : dtype == at::kHalf ? DDL_DT_F16 : 0;
    if (!expert_operands(x, w, offsets) || x.scalar_type() != at::kFloat8_e4m3fn || !code || !multiple(x.data_ptr(), 16) || !multiple(w.data_ptr(), 16) || !floats_of(x_scales, {x.size(0)}) || !floats_of(w_scales, {w.size(0), w.size(1)}))
        return std::nullopt;
    const int64_t rows = x.size(0), n = w.size(1), k = w.size(2);
    Tensor y = at::empty({rows, n}, x.options().dtype(dtype));
    check(ddl_expert_linear_8bit(x.data_ptr(), x_scales.data_ptr<float>(), w.data_ptr(), w_scales.data_ptr<float>(), offsets.data_ptr<int32_t>(), w.size(0), rows, n, k, k,
                                 y.data_ptr(), code, current_stream()),
          "ddl_expert_linear_8bit");
    return y;
}

std::optional<Two> expert_linear_backward(const Tensor& dy, const Tensor& x, const Tensor& w, const Tensor& offsets, bool want_input, bool want_weight) {
    if (!expert_operands(x, w, offsets) || !float_code(x) || !rows_of(dy, x.size(0)) || dy.size(1) != w.size(1) || dy.scalar_type() != x.scalar_type()) return std::nullopt;
    const int64_t rows = x.size(0), n = w.size(1), k = w.size(2);
    Tensor dx, dw;
    if (want_input) dx = at::empty(x.sizes(), x.options());
    if (want_weight) dw = at::empty(w.sizes(), w.options());
    check(ddl_expert_linear_backward_long(dy.data_ptr(), x.data_ptr(), w.data_ptr(), float_code(x), offsets.data_ptr<int32_t>(), w.size(0), rows, n, k, n, k, pointer(dx),
                                     pointer(dw), current_stream()),
          "ddl_expert_linear_backward_long");
    return Two(want_input ? MaybeTensor(dx) : std::nullopt, want_weight ? MaybeTensor(dw) : std::nullopt);
}

}  // namespace ddl_front
