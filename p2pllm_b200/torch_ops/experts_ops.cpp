// The 4-bit products and the token shuffle around routed experts as torch custom operators (namespace p2p_b200). The
// products are for inference: an x that is differentiated, in either mode, is refused. The shuffle's two directions are
// differentiable in reverse mode; their gradients are the library's own kernels, one level deep (second derivatives of the
// weighted sum are refused, and inputs with a forward-mode tangent).
#include <torch/csrc/autograd/custom_function.h>

#include <algorithm>

#include "op_common.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kPickTokens = 8;                    // items of up to here pick x's rows by the order

// Places of one item, what one pass over an expert's weights takes: somewhat more than experts have on average, so that
// few take two passes and no tile is mostly empty; at most what leaves the accumulators room. Both sides of every step, us
// of the product alone at a mean number of pairs (128 experts, ids evenly drawn; 1536 x 2048 gated, bf16, groups of 128 |
// 2048 x 768, f16, groups of 32, zero points):
//   mean   4: items of   8:  56 |  40, of  16:  58 |  44      mean   5: of   8:  60 |  45, of  16:  62 |  48
//   mean  10: items of  16:  67 |  51, of  32:  81 |  61      mean  12: of  16:  70 |  54, of  32:  85 |  63
//   mean  24: items of  32: 113 |  80, of  64: 124 | 139      mean  26: of  32: 116 |  81, of  64: 123 | 138
//   mean  48: items of  64: 130 | 142, of 128: 158 | 180      mean  52: of  64: 141 | 153, of 128: 176 | 198
//   mean 100: items of 128: 201 | 226, of 160: 203 | 228      mean 118: of 128: 238 | 273, of 160: 225 | 254
//   mean 130: items of 160: 227 | 255, of 256: 262 | 326      mean 134: of 160: 226 | 256, of 256: 261 | 327
//                                                             mean 200: of 160: 384 | 454, of 256: 311 | 387
// The smaller size holds on a little past most steps (to a mean of 5, 12, 26, 52, 104 and between 134 and 160); with skewed
// ids some experts are past theirs, and the steps are early for them.
int64_t item_tokens(int64_t pairs, int64_t experts) {
    const double mean = (double)pairs / experts;
    if (pairs <= kPickTokens || mean <= 4) return kPickTokens;
    return mean <= 10 ? 16 : mean <= 24 ? 32 : mean <= 48 ? 64 : mean <= 100 ? 128 : mean <= 130 ? 160 : 256;
}

// t [rows, cols] with unit column stride and rows that do not overlap (an expanded gradient's do).
at::Tensor rows2d(const at::Tensor& t) {
    const bool cols_ok = t.size(1) <= 1 || t.stride(1) == 1, rows_ok = t.size(0) <= 1 || t.stride(0) >= t.size(1);
    return cols_ok && rows_ok ? t : t.contiguous();
}
// t with rows that start on 16-byte boundaries; the columns that a copy's stride adds are never read.
at::Tensor aligned_rows(const at::Tensor& t) {
    const at::Tensor r = rows2d(t);
    if (reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 == 0 && (r.size(0) <= 1 || r.stride(0) % 8 == 0)) return r;
    at::Tensor copy = at::empty({r.size(0), (r.size(1) + 7) / 8 * 8}, r.options()).narrow(1, 0, r.size(1));
    copy.copy_(r);
    return copy;
}
int64_t row_stride(const at::Tensor& t) { return std::max(t.size(0) <= 1 ? (int64_t)0 : t.stride(0), t.size(1)); }
// The same, rounded up to 8 elements where one row stands alone.
int64_t aligned_stride(const at::Tensor& t) { return t.size(0) <= 1 ? (t.size(1) + 7) / 8 * 8 : t.stride(0); }

void check_matrix(const at::Tensor& t, const char* what) {
    TORCH_CHECK(t.is_cuda(), "p2p_b200: ", what, ": CUDA tensors only (the replica path has no CPU fallback)");
    TORCH_CHECK(t.dim() == 2, "p2p_b200: ", what, " of ", t.sizes(), " is not a matrix");
}

const int32_t* ints(const at::Tensor& t, const at::Tensor& like, int64_t n, const char* what) {
    TORCH_CHECK(t.device() == like.device() && t.scalar_type() == at::kInt && t.is_contiguous() && t.numel() >= n,
                "p2p_b200: ", what, " is not a contiguous int32 tensor of ", n, " on ", like.device());
    return t.data_ptr<int32_t>();
}

at::Tensor moe_spread(const at::Tensor& x_in, const at::Tensor& where, const at::Tensor& offsets, int64_t topk);

// ---- 4-bit products --------------------------------------------------------------------------------------------------

void check_int4(const at::Tensor& x, const at::Tensor& layout, bool zeros, int64_t experts, int64_t rows, int64_t cols,
                int64_t group, bool gated) {
    check_matrix(x, "x");
    TORCH_CHECK(x.size(1) == cols, "p2p_b200: x of ", x.sizes(), " does not have ", cols, " columns");
    TORCH_CHECK(group == 32 || group == 64 || group == 128, "p2p_b200: groups of ", group, " columns, not 32, 64 or 128");
    const int64_t need = p2p_int4_layout_bytes(experts, rows, cols, (int)group, zeros, gated);
    // the layout's bytes do not say what their scales are, its tensor's dtype does
    TORCH_CHECK(layout.scalar_type() == x.scalar_type(), "p2p_b200: x is ", x.scalar_type(), ", the 4-bit layout's weights ",
                layout.scalar_type());
    TORCH_CHECK(need > 0 && layout.device() == x.device() && layout.is_contiguous() && (int64_t)layout.nbytes() >= need,
                "p2p_b200: the 4-bit layout does not hold ", rows, " x ", cols, " weights");
}

void check_rows_out(const at::Tensor& out, const at::Tensor& x, int64_t rows, int64_t cols) {
    TORCH_CHECK(out.device() == x.device() && out.scalar_type() == x.scalar_type() && out.dim() == 2 &&
                    out.size(0) == rows && out.size(1) == cols &&
                    (out.numel() == 0 || ((cols == 1 || out.stride(1) == 1) && (rows == 1 || out.stride(0) >= cols))),
                "p2p_b200: out of ", out.sizes(), " ", out.scalar_type(), " does not take y [", rows, ", ", cols, "] ",
                x.scalar_type());
}

void int4_mm_into(const at::Tensor& x_in, const at::Tensor& layout, bool zeros, int64_t rows, int64_t cols, int64_t group, bool gated,
                  const at::Tensor& out) {
    check_int4(x_in, layout, zeros, 1, rows, cols, group, gated);
    check_rows_out(out, x_in, x_in.size(0), gated ? rows / 2 : rows);
    const c10::cuda::CUDAGuard guard(x_in.device());
    const at::Tensor x = aligned_rows(x_in);
    const size_t need = p2p_int4_workspace(x.size(0), rows, cols, gated);
    const at::Tensor ws = need ? at::empty({(int64_t)need}, x.options().dtype(at::kByte)) : at::Tensor();
    check(p2p_int4_mm(x.data_ptr(), dtype_code(x), x.size(0), cols, aligned_stride(x),
                      layout.data_ptr(), zeros, rows, (int)group, gated, out.data_ptr(),
                      row_stride(out), need ? ws.data_ptr() : nullptr, need, stream_of(x)),
          "p2p_int4_mm");
}

at::Tensor int4_mm(const at::Tensor& x, const at::Tensor& layout, bool zeros, int64_t rows, int64_t cols, int64_t group, bool gated) {
    check_matrix(x, "x");
    at::Tensor out = at::empty({x.size(0), gated ? rows / 2 : rows}, x.options());
    int4_mm_into(x, layout, zeros, rows, cols, group, gated, out);
    return out;
}

void int4_grouped_run(const at::Tensor& x_in, const at::Tensor& layout, bool zeros, int64_t experts, int64_t rows, int64_t cols,
                      int64_t group, bool gated, const at::Tensor& order, const at::Tensor& where, const at::Tensor& offsets,
                      const at::Tensor& items, const at::Tensor& n_items, int64_t topk, bool gather,
                      const at::Tensor& out, bool zero_behind) {
    check_int4(x_in, layout, zeros, experts, rows, cols, group, gated);
    const int64_t pairs = order.numel();
    TORCH_CHECK(topk >= 1 && x_in.size(0) == (gather ? pairs / topk : pairs) && pairs % topk == 0, "p2p_b200: x has ",
                x_in.size(0), " rows, the order is of ", pairs, " pairs, ", topk, " a token");
    check_rows_out(out, x_in, pairs, gated ? rows / 2 : rows);
    const c10::cuda::CUDAGuard guard(x_in.device());
    const int32_t* at_order = ints(order, x_in, pairs, "order");
    const int32_t* at_offsets = ints(offsets, x_in, experts + 1, "offsets");
    TORCH_CHECK(offsets.numel() == experts + 1, "p2p_b200: the order is of ", offsets.numel() - 1, " experts, the weights of ",
                experts);
    if (pairs == 0) return;
    const int64_t most = item_tokens(pairs, experts);
    // few pairs: the product picks x's rows itself
    const bool pick = gather && most <= kPickTokens;
    const at::Tensor x = aligned_rows(gather && !pick ? moe_spread(x_in, where, offsets, topk) : x_in);
    const size_t need = p2p_int4_grouped_workspace(items.numel() / 4, most, rows, cols, gated);
    const at::Tensor ws = need ? at::empty({(int64_t)need}, x.options().dtype(at::kByte)) : at::Tensor();
    check(p2p_int4_grouped(x.data_ptr(), dtype_code(x), cols, aligned_stride(x), layout.data_ptr(), zeros, rows, (int)group,
                           gated, ints(items, x, 0, "items"), ints(n_items, x, 1, "n_items"), items.numel() / 4, most,
                           pick ? at_order : nullptr, (int)topk, zero_behind ? at_offsets + experts : nullptr, pairs,
                           out.data_ptr(), row_stride(out), need ? ws.data_ptr() : nullptr, need, stream_of(x)),
          "p2p_int4_grouped");
}

void int4_grouped_into(const at::Tensor& x, const at::Tensor& layout, bool zeros, int64_t experts, int64_t rows, int64_t cols,
                       int64_t group, bool gated, const at::Tensor& order, const at::Tensor& where, const at::Tensor& offsets,
                       const at::Tensor& items, const at::Tensor& n_items, int64_t topk, bool gather,
                       const at::Tensor& out) {
    int4_grouped_run(x, layout, zeros, experts, rows, cols, group, gated, order, where, offsets, items, n_items, topk,
                     gather, out, false);
}

at::Tensor int4_grouped(const at::Tensor& x, const at::Tensor& layout, bool zeros, int64_t experts, int64_t rows, int64_t cols,
                        int64_t group, bool gated, const at::Tensor& order, const at::Tensor& where, const at::Tensor& offsets,
                        const at::Tensor& items, const at::Tensor& n_items, int64_t topk, bool gather) {
    check_matrix(x, "x");
    at::Tensor out = at::empty({order.numel(), gated ? rows / 2 : rows}, x.options());
    int4_grouped_run(x, layout, zeros, experts, rows, cols, group, gated, order, where, offsets, items, n_items, topk,
                     gather, out, true);
    return out;
}

// ---- tokens sorted by expert and back --------------------------------------------------------------------------------

int64_t max_items(int64_t pairs, int64_t experts) {
    const int64_t most = item_tokens(pairs, experts);
    return std::min(pairs, (pairs + most - 1) / most + experts);
}

// all[begin .. begin + n) as a tensor of its own on the same storage, without a trip through the dispatcher.
at::Tensor part(const at::Tensor& all, int64_t begin, int64_t n) {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(all.storage_offset() + begin);
    t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    return t;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> moe_sort(const at::Tensor& ids_in, int64_t experts) {
    TORCH_CHECK(ids_in.is_cuda(), "p2p_b200: CUDA tensors only (the replica path has no CPU fallback)");
    TORCH_CHECK(ids_in.scalar_type() == at::kInt || ids_in.scalar_type() == at::kLong, "p2p_b200: ids are int32 or int64");
    TORCH_CHECK(experts >= 1 && experts <= 1024, "p2p_b200: ", experts, " experts, 1 to 1024");
    const c10::cuda::CUDAGuard guard(ids_in.device());
    const at::Tensor ids = ids_in.contiguous();
    const int64_t n = ids.numel(), most = std::max<int64_t>(max_items(n, experts), 1);
    // one allocation: items (16-byte aligned), order, where, offsets, n_items
    at::Tensor all = at::empty({4 * most + 2 * n + experts + 2}, ids.options().dtype(at::kInt));
    at::Tensor items = part(all, 0, 4 * most), order = part(all, 4 * most, n), where = part(all, 4 * most + n, n),
               offsets = part(all, 4 * most + 2 * n, experts + 1),
               n_items = part(all, 4 * most + 2 * n + experts + 1, 1);
    check(p2p_moe_sort(ids.data_ptr(), (int)ids.element_size(), n, (int)experts, order.data_ptr<int32_t>(),
                       where.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(), items.data_ptr<int32_t>(), most,
                       (int)item_tokens(n, experts), n_items.data_ptr<int32_t>(), stream_of(ids)),
          "p2p_moe_sort");
    return {order, where, offsets, items, n_items};
}

const int32_t* routed_of(const at::Tensor& offsets, const at::Tensor& like) {
    return ints(offsets, like, 1, "offsets") + offsets.numel() - 1;
}

at::Tensor moe_spread(const at::Tensor& x_in, const at::Tensor& where, const at::Tensor& offsets, int64_t topk) {
    check_matrix(x_in, "x");
    const c10::cuda::CUDAGuard guard(x_in.device());
    const at::Tensor x = rows2d(x_in);
    TORCH_CHECK(topk >= 1 && where.numel() == x.size(0) * topk, "p2p_b200: x has ", x.size(0), " rows, the order is of ",
                where.numel(), " pairs, ", topk, " a token");
    at::Tensor out = at::empty({where.numel(), x.size(1)}, x.options());
    if (out.numel() == 0) return out;
    check(p2p_moe_spread(x.data_ptr(), dtype_code(x), x.size(0), (int)topk, x.size(1), row_stride(x),
                         ints(where, x, where.numel(), "where"), routed_of(offsets, x), out.data_ptr(), out.size(1),
                         stream_of(x)),
          "p2p_moe_spread");
    return out;
}

void check_sum(const at::Tensor& y, const at::Tensor& where, const std::optional<at::Tensor>& weights, int64_t topk) {
    check_matrix(y, "y");
    TORCH_CHECK(topk >= 1 && where.numel() % topk == 0 && y.size(0) == where.numel(), "p2p_b200: y has ", y.size(0),
                " rows, the order is of ", where.numel(), " pairs, ", topk, " a token");
    TORCH_CHECK(!weights || (weights->device() == y.device() && weights->dim() == 2 && weights->size(1) == topk &&
                             weights->numel() == where.numel()),
                "p2p_b200: weights are not [", where.numel() / topk, ", ", topk, "] on ", y.device());
}

at::Tensor moe_sum(const at::Tensor& y_in, const at::Tensor& where, const at::Tensor&,
                   const std::optional<at::Tensor>& weights, int64_t topk) {
    check_sum(y_in, where, weights, topk);
    const c10::cuda::CUDAGuard guard(y_in.device());
    const at::Tensor y = rows2d(y_in);
    at::Tensor out = at::empty({where.numel() / topk, y.size(1)}, y.options());
    if (out.numel() == 0) return out;
    const at::Tensor w = weights ? weights->contiguous() : at::Tensor();
    check(p2p_moe_sum(y.data_ptr(), dtype_code(y), out.size(0), (int)topk, y.size(1), row_stride(y),
                      ints(where, y, where.numel(), "where"), weights ? w.data_ptr() : nullptr,
                      weights ? dtype_code(w) : P2P_F32, out.data_ptr(), out.size(1), stream_of(y)),
          "p2p_moe_sum");
    return out;
}

std::tuple<at::Tensor, at::Tensor> moe_sum_back(const at::Tensor& dout_in, const at::Tensor& y_in,
                                                const at::Tensor& where, const at::Tensor& offsets,
                                                const at::Tensor& weights_in, int64_t topk) {
    check_sum(y_in, where, weights_in, topk);
    check_matrix(dout_in, "the gradient");
    TORCH_CHECK(dout_in.device() == y_in.device() && dout_in.scalar_type() == y_in.scalar_type() &&
                    dout_in.size(0) == where.numel() / topk && dout_in.size(1) == y_in.size(1),
                "p2p_b200: a gradient of ", dout_in.sizes(), " ", dout_in.scalar_type(), " for rows of ", y_in.sizes(), " ",
                y_in.scalar_type());
    const c10::cuda::CUDAGuard guard(y_in.device());
    const at::Tensor y = rows2d(y_in), dout = rows2d(dout_in), w = weights_in.contiguous();
    at::Tensor dy = at::empty({y.size(0), y.size(1)}, y.options()), dw = at::empty(weights_in.sizes(), w.options());
    if (y.size(0) == 0) return {dy, dw};
    if (y.size(1) == 0) return {dy, dw.zero_()};
    check(p2p_moe_sum_back(dout.data_ptr(), y.data_ptr(), dtype_code(y), dout.size(0), (int)topk, y.size(1),
                           row_stride(dout), row_stride(y), ints(where, y, where.numel(), "where"),
                           routed_of(offsets, y), w.data_ptr(), dtype_code(w), dy.data_ptr(), y.size(1), dw.data_ptr(),
                           stream_of(y)),
          "p2p_moe_sum_back");
    return {dy, dw};
}

// The operators as the dispatcher sees them, for the gradients below.
at::Tensor call_spread(const at::Tensor& x, const at::Tensor& where, const at::Tensor& offsets, int64_t topk) {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("p2p_b200::moe_spread", "").typed<decltype(moe_spread)>();
    return op.call(x, where, offsets, topk);
}
at::Tensor call_sum(const at::Tensor& y, const at::Tensor& where, const at::Tensor& offsets,
                    const std::optional<at::Tensor>& weights, int64_t topk) {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("p2p_b200::moe_sum", "").typed<decltype(moe_sum)>();
    return op.call(y, where, offsets, weights, topk);
}
std::tuple<at::Tensor, at::Tensor> call_sum_back(const at::Tensor& dout, const at::Tensor& y, const at::Tensor& where,
                                                 const at::Tensor& offsets, const at::Tensor& weights, int64_t topk) {
    static const auto op =
        c10::Dispatcher::singleton().findSchemaOrThrow("p2p_b200::moe_sum_back", "").typed<decltype(moe_sum_back)>();
    return op.call(dout, y, where, offsets, weights, topk);
}

bool needs_grad(const at::Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }
// Whether t carries a tangent, which a call below autograd would lose without a word.
bool has_tangent(const at::Tensor& t) { return t._fw_grad(0).defined(); }
void check_tangents(bool any) {
    TORCH_CHECK(!any, "p2p_b200: forward-mode derivatives of the token shuffle are not offered");
}

struct Spread : torch::autograd::Function<Spread> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& where,
                              const at::Tensor& offsets, int64_t topk) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({where, offsets});
        ctx->saved_data["topk"] = topk;
        return call_spread(x, where, offsets, topk);
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const variable_list s = ctx->get_saved_variables();
        at::Tensor dx;
        if (grads[0].defined()) dx = call_sum(grads[0], s[0], s[1], std::nullopt, ctx->saved_data["topk"].toInt());
        return {dx, at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

struct Sum : torch::autograd::Function<Sum> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& y, const at::Tensor& where,
                              const at::Tensor& offsets, const std::optional<at::Tensor>& weights, int64_t topk) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->saved_data["topk"] = topk;
        ctx->saved_data["weighted"] = weights.has_value();
        if (weights) ctx->save_for_backward({where, offsets, y, *weights});
        else ctx->save_for_backward({where, offsets});
        return call_sum(y, where, offsets, weights, topk);
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const variable_list s = ctx->get_saved_variables();
        const int64_t topk = ctx->saved_data["topk"].toInt();
        at::Tensor dy, dw;
        if (grads[0].defined()) {
            if (!ctx->saved_data["weighted"].toBool()) dy = call_spread(grads[0], s[0], s[1], topk);
            else std::tie(dy, dw) = call_sum_back(grads[0], s[2], s[0], s[1], s[3], topk);
        }
        return {dy, at::Tensor(), at::Tensor(), dw, at::Tensor()};
    }
};

at::Tensor moe_spread_grad(const at::Tensor& x, const at::Tensor& where, const at::Tensor& offsets, int64_t topk) {
    check_tangents(has_tangent(x));
    if (needs_grad(x)) return Spread::apply(x, where, offsets, topk);
    at::AutoDispatchBelowADInplaceOrView below;
    return call_spread(x, where, offsets, topk);
}
at::Tensor moe_sum_grad(const at::Tensor& y, const at::Tensor& where, const at::Tensor& offsets,
                        const std::optional<at::Tensor>& weights, int64_t topk) {
    check_tangents(has_tangent(y) || (weights && has_tangent(*weights)));
    if (needs_grad(y) || (weights && needs_grad(*weights))) return Sum::apply(y, where, offsets, weights, topk);
    at::AutoDispatchBelowADInplaceOrView below;
    return call_sum(y, where, offsets, weights, topk);
}
std::tuple<at::Tensor, at::Tensor> moe_sum_back_grad(const at::Tensor& dout, const at::Tensor& y,
                                                     const at::Tensor& where, const at::Tensor& offsets,
                                                     const at::Tensor& weights, int64_t topk) {
    check_tangents(has_tangent(dout) || has_tangent(y) || has_tangent(weights));
    TORCH_CHECK(!(needs_grad(dout) || needs_grad(y) || needs_grad(weights)),
                "p2p_b200: second derivatives of the weighted sum are not offered");
    at::AutoDispatchBelowADInplaceOrView below;
    return call_sum_back(dout, y, where, offsets, weights, topk);
}

// The products as autograd sees them: an input that is differentiated in either mode, under torch.func too, is refused.

void check_inference(const at::Tensor& x) {
    TORCH_CHECK(!needs_grad(x) && !has_tangent(x), "p2p_b200: 4-bit weights are for inference: x must not need a gradient");
}
void check_inference(const at::Tensor& x, const at::Tensor& out) {
    check_inference(x);
    TORCH_CHECK(!needs_grad(out) && !has_tangent(out),
                "p2p_b200: 4-bit weights are for inference: out must not need a gradient");
}

at::Tensor int4_mm_grad(const at::Tensor& x, const at::Tensor& layout, bool zeros, int64_t rows, int64_t cols,
                        int64_t group, bool gated) {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("p2p_b200::int4_mm", "").typed<decltype(int4_mm)>();
    check_inference(x);
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(x, layout, zeros, rows, cols, group, gated);
}
void int4_mm_into_grad(const at::Tensor& x, const at::Tensor& layout, bool zeros, int64_t rows, int64_t cols, int64_t group,
                       bool gated, const at::Tensor& out) {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("p2p_b200::int4_mm_into", "").typed<decltype(int4_mm_into)>();
    check_inference(x, out);
    at::AutoDispatchBelowADInplaceOrView below;
    op.call(x, layout, zeros, rows, cols, group, gated, out);
}
at::Tensor int4_grouped_grad(const at::Tensor& x, const at::Tensor& layout, bool zeros, int64_t experts, int64_t rows, int64_t cols,
                             int64_t group, bool gated, const at::Tensor& order, const at::Tensor& where, const at::Tensor& offsets,
                             const at::Tensor& items, const at::Tensor& n_items, int64_t topk, bool gather) {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("p2p_b200::int4_grouped", "").typed<decltype(int4_grouped)>();
    check_inference(x);
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(x, layout, zeros, experts, rows, cols, group, gated, order, where, offsets, items, n_items, topk, gather);
}
void int4_grouped_into_grad(const at::Tensor& x, const at::Tensor& layout, bool zeros, int64_t experts, int64_t rows, int64_t cols,
                            int64_t group, bool gated, const at::Tensor& order, const at::Tensor& where, const at::Tensor& offsets,
                            const at::Tensor& items, const at::Tensor& n_items, int64_t topk, bool gather,
                            const at::Tensor& out) {
    static const auto op =
        c10::Dispatcher::singleton().findSchemaOrThrow("p2p_b200::int4_grouped_into", "").typed<decltype(int4_grouped_into)>();
    check_inference(x, out);
    at::AutoDispatchBelowADInplaceOrView below;
    op.call(x, layout, zeros, experts, rows, cols, group, gated, order, where, offsets, items, n_items, topk, gather, out);
}

// ---- shapes ----------------------------------------------------------------------------------------------------------

at::Tensor int4_mm_meta(const at::Tensor& x, const at::Tensor&, bool, int64_t rows, int64_t, int64_t, bool gated) {
    return at::empty({x.size(0), gated ? rows / 2 : rows}, x.options());
}
void int4_mm_into_meta(const at::Tensor&, const at::Tensor&, bool, int64_t, int64_t, int64_t, bool, const at::Tensor&) {}
at::Tensor int4_grouped_meta(const at::Tensor& x, const at::Tensor&, bool, int64_t, int64_t rows, int64_t, int64_t,
                             bool gated, const at::Tensor& order, const at::Tensor&, const at::Tensor&,
                             const at::Tensor&, const at::Tensor&, int64_t, bool) {
    return at::empty({order.numel(), gated ? rows / 2 : rows}, x.options());
}
void int4_grouped_into_meta(const at::Tensor&, const at::Tensor&, bool, int64_t, int64_t, int64_t, int64_t, bool,
                            const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                            const at::Tensor&, int64_t, bool, const at::Tensor&) {}
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> moe_sort_meta(const at::Tensor& ids, int64_t experts) {
    const auto o = ids.options().dtype(at::kInt);
    const int64_t n = ids.numel();
    return {at::empty({n}, o), at::empty({n}, o), at::empty({experts + 1}, o),
            at::empty({4 * std::max<int64_t>(max_items(n, experts), 1)}, o), at::empty({1}, o)};
}
at::Tensor moe_spread_meta(const at::Tensor& x, const at::Tensor& where, const at::Tensor&, int64_t) {
    return at::empty({where.numel(), x.size(1)}, x.options());
}
at::Tensor moe_sum_meta(const at::Tensor& y, const at::Tensor& where, const at::Tensor&, const std::optional<at::Tensor>&,
                        int64_t topk) {
    return at::empty({where.numel() / topk, y.size(1)}, y.options());
}
std::tuple<at::Tensor, at::Tensor> moe_sum_back_meta(const at::Tensor&, const at::Tensor& y, const at::Tensor&,
                                                     const at::Tensor&, const at::Tensor& weights, int64_t) {
    return {at::empty(y.sizes(), y.options()), at::empty(weights.sizes(), weights.options())};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(p2p_b200, m) {
    m.def("int4_mm(Tensor x, Tensor layout, bool zeros, int rows, int cols, int group, bool gated) -> Tensor");
    m.def("int4_mm_into(Tensor x, Tensor layout, bool zeros, int rows, int cols, int group, bool gated, "
          "Tensor(a!) out) -> ()");
    m.def("int4_grouped(Tensor x, Tensor layout, bool zeros, int experts, int rows, int cols, int group, "
          "bool gated, Tensor order, Tensor where, Tensor offsets, Tensor items, Tensor n_items, int topk, bool gather) -> Tensor");
    m.def("int4_grouped_into(Tensor x, Tensor layout, bool zeros, int experts, int rows, int cols, "
          "int group, bool gated, Tensor order, Tensor where, Tensor offsets, Tensor items, Tensor n_items, int topk, bool gather, "
          "Tensor(a!) out) -> ()");
    m.def("moe_sort(Tensor ids, int experts) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("moe_spread(Tensor x, Tensor where, Tensor offsets, int topk) -> Tensor");
    m.def("moe_sum(Tensor y, Tensor where, Tensor offsets, Tensor? weights, int topk) -> Tensor");
    m.def("moe_sum_back(Tensor dout, Tensor y, Tensor where, Tensor offsets, Tensor weights, int topk) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(p2p_b200, CUDA, m) {
    m.impl("int4_mm", &int4_mm);
    m.impl("int4_mm_into", &int4_mm_into);
    m.impl("int4_grouped", &int4_grouped);
    m.impl("int4_grouped_into", &int4_grouped_into);
    m.impl("moe_sort", &moe_sort);
    m.impl("moe_spread", &moe_spread);
    m.impl("moe_sum", &moe_sum);
    m.impl("moe_sum_back", &moe_sum_back);
}

TORCH_LIBRARY_IMPL(p2p_b200, Autograd, m) {
    m.impl("int4_mm", &int4_mm_grad);
    m.impl("int4_mm_into", &int4_mm_into_grad);
    m.impl("int4_grouped", &int4_grouped_grad);
    m.impl("int4_grouped_into", &int4_grouped_into_grad);
    m.impl("moe_spread", &moe_spread_grad);
    m.impl("moe_sum", &moe_sum_grad);
    m.impl("moe_sum_back", &moe_sum_back_grad);
}

TORCH_LIBRARY_IMPL(p2p_b200, Meta, m) {
    m.impl("int4_mm", &int4_mm_meta);
    m.impl("int4_mm_into", &int4_mm_into_meta);
    m.impl("int4_grouped", &int4_grouped_meta);
    m.impl("int4_grouped_into", &int4_grouped_into_meta);
    m.impl("moe_sort", &moe_sort_meta);
    m.impl("moe_spread", &moe_spread_meta);
    m.impl("moe_sum", &moe_sum_meta);
    m.impl("moe_sum_back", &moe_sum_back_meta);
}
