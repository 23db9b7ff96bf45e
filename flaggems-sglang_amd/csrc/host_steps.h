// Host side of the routed layer's steps and their gradients (flaggems_sglang.ops.
// steps, .linear): part of host_ext.cpp, whose helpers it uses.

struct StepsLibrary {
  decltype(&fgs_moe_permute_workspace_bytes) permute_workspace_bytes;
  decltype(&fgs_moe_permute) permute;
  decltype(&fgs_moe_permute_rows) permute_rows;
  decltype(&fgs_moe_unpermute) unpermute;
  decltype(&fgs_moe_unpermute_grad) unpermute_grad;
  decltype(&fgs_moe_topk_gating) topk_gating;
  decltype(&fgs_moe_topk_gating_grad) topk_gating_grad;
  decltype(&fgs_moe_linear) linear;
  decltype(&fgs_moe_linear_act_grad) linear_act_grad;
  decltype(&fgs_moe_linear_input_grad) linear_input_grad;
  decltype(&fgs_moe_linear_weight_grad) linear_weight_grad;
  decltype(&fgs_moe_linear_bias_grad_workspace_bytes) linear_bias_grad_workspace_bytes;
  decltype(&fgs_moe_linear_bias_grad) linear_bias_grad;
};
StepsLibrary g_steps{};

constexpr int64_t kMaxLinearStride = int64_t{1} << 21;  // of the products' rows

const int32_t* ints(const at::Tensor& t) { return static_cast<const int32_t*>(ptr(t)); }
int32_t* ints_out(const at::Tensor& t) { return static_cast<int32_t*>(ptr(t)); }
at::Tensor contiguous(const at::Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }
at::Tensor bytes_for(int64_t n, const at::Tensor& like) {  // workspace, or none
  return n > 0 ? make({n}, at::kByte, like) : at::Tensor();
}

// ------------------------------------------------------- rows and tokens ---
bool movable(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16:
    case at::kHalf:
    case at::kFloat:
    case at::kFloat8_e4m3fn:
    case at::kFloat8_e5m2:
    case at::kChar:
    case at::kByte:
    case at::kInt:
    case at::kLong: return true;
    default: return false;
  }
}

void check_order(const at::Tensor& row_of_slot, const at::Tensor* slot_of_row) {
  require(row_of_slot.dim() == 2 && row_of_slot.scalar_type() == at::kInt && row_of_slot.size(1) > 0,
          "row_of_slot must be int32 [tokens, topk]");
  require(!slot_of_row || (slot_of_row->dim() == 1 && slot_of_row->scalar_type() == at::kInt),
          "slot_of_row must be int32 [rows]");
}

void check_movable(const at::Tensor& x) {
  require(x.dim() == 2 && x.size(1) > 0, "x must be [tokens, cols]");
  require(movable(x.scalar_type()), "x must be of a 8- to 64-bit integer or a 8- to 32-bit float type");
}

struct Permuted {
  at::Tensor rows, counts, row_of_slot, slot_of_row;
};
Permuted permute_of(const Arg& xa, const Arg& ia, int64_t experts) {
  const int index = check_inputs({xa, ia});
  const at::Tensor& x = *xa.t;
  check_movable(x);
  require(ia.t->dim() == 2 && ia.t->size(0) == x.size(0) && ia.t->size(1) > 0 &&
              ia.t->scalar_type() == at::kInt,
          "topk_ids must be int32 [tokens, topk]");
  if (experts < 1 || experts > 1022)
    refuse(PyExc_ValueError, "moe_permute: num_experts must be in [1, 1022]");
  const int64_t m = x.size(0), topk = ia.t->size(1), slots = m * topk, size = x.element_size();
  const Rows xr = rows_of(x, x.size(1));
  const at::Tensor ids = contiguous(*ia.t);
  const int64_t need = g_steps.permute_workspace_bytes(slots, static_cast<int32_t>(experts));
  if (need < 0) refuse(PyExc_NotImplementedError, "moe_permute: more than 2^30 slots");
  const Permuted p{make({slots, x.size(1)}, x.scalar_type(), x), make({experts}, at::kInt, x),
                   make({m, topk}, at::kInt, x), make({slots}, at::kInt, x)};
  const at::Tensor ws = bytes_for(need, x);
  void* stream = stream_of(index);
  call(index, "moe_permute", g_steps.permute, ptr(xr.t), xr.stride * size, m, x.size(1) * size,
       ints(ids), static_cast<int32_t>(topk), static_cast<int32_t>(experts), ptr(p.rows),
       ints_out(p.counts), ints_out(p.row_of_slot), ints_out(p.slot_of_row), ptr(ws), need, stream);
  return p;
}

at::Tensor permute_rows_of(const Arg& xa, const Arg& ra, const Arg& sa) {
  const int index = check_inputs({xa, ra, sa});
  const at::Tensor& x = *xa.t;
  check_movable(x);
  check_order(*ra.t, sa.t);
  require(ra.t->size(0) == x.size(0) && sa.t->size(0) == ra.t->numel(),
          "the order is one of other tokens");
  const int64_t size = x.element_size();
  const Rows xr = rows_of(x, x.size(1));
  const at::Tensor row_of_slot = contiguous(*ra.t), slot_of_row = contiguous(*sa.t);
  const at::Tensor rows = make({slot_of_row.size(0), x.size(1)}, x.scalar_type(), x);
  void* stream = stream_of(index);
  call(index, "moe_permute", g_steps.permute_rows, ptr(xr.t), xr.stride * size, x.size(0),
       x.size(1) * size, ints(row_of_slot), static_cast<int32_t>(row_of_slot.size(1)),
       ints(slot_of_row), ptr(rows), stream);
  return rows;
}

void check_weights(const Arg& wa, const at::Tensor& row_of_slot) {
  require(!wa.t || (wa.t->sizes() == row_of_slot.sizes() && wa.t->scalar_type() == at::kFloat),
          "topk_weights must be float32 [tokens, topk]");
}

at::Tensor unpermute_of(const Arg& ra, const Arg& oa, const Arg& wa) {
  const int index = check_inputs({ra, oa, wa});
  const at::Tensor& rows = *ra.t;
  const int type = type_code(rows);
  require(type >= 0, "rows must be bfloat16, float16 or float32");
  require(rows.dim() == 2 && rows.size(1) > 0, "rows must be [rows, cols]");
  check_order(*oa.t, nullptr);
  check_weights(wa, *oa.t);
  const int64_t m = oa.t->size(0), cols = rows.size(1);
  const Rows rr = rows_of(rows, cols);
  const at::Tensor order = contiguous(*oa.t);
  const at::Tensor weights = wa.t ? contiguous(*wa.t) : at::Tensor();
  const at::Tensor out = make({m, cols}, rows.scalar_type(), rows);
  void* stream = stream_of(index);
  call(index, "moe_unpermute", g_steps.unpermute, ptr(rr.t), rr.stride, rows.size(0), ints(order),
       floats(weights), m, static_cast<int32_t>(order.size(1)), cols, type, ptr(out), stream);
  return out;
}

// (drows, dweights), those asked for; rows only for dweights.
std::array<at::Tensor, 2> unpermute_grad_of(const Arg& da, const Arg& ra, const Arg& oa,
                                            const Arg& sa, const Arg& wa, bool with_drows,
                                            bool with_dweights) {
  const int index = check_inputs({da, ra, oa, sa, wa});
  const at::Tensor& dout = *da.t;
  const int type = type_code(dout);
  require(type >= 0, "dout must be bfloat16, float16 or float32");
  check_order(*oa.t, sa.t);
  check_weights(wa, *oa.t);
  const int64_t m = oa.t->size(0), n_rows = sa.t->size(0);
  require(dout.dim() == 2 && dout.size(0) == m && dout.size(1) > 0, "dout must be [tokens, cols]");
  const int64_t cols = dout.size(1);
  require(!with_dweights || ra.t, "the weights' gradient needs the rows");
  Rows rr{{}, 0};
  if (ra.t) {
    require(ra.t->dim() == 2 && ra.t->size(0) == n_rows && ra.t->size(1) == cols &&
                ra.t->scalar_type() == dout.scalar_type(),
            "rows must be [rows, cols] of dout's type");
    rr = rows_of(*ra.t, cols);
  }
  const Rows dr = rows_of(dout, cols);
  const at::Tensor order = contiguous(*oa.t), slot_of_row = contiguous(*sa.t);
  const at::Tensor weights = wa.t ? contiguous(*wa.t) : at::Tensor();
  at::Tensor drows, dweights;
  if (with_drows) drows = make({n_rows, cols}, dout.scalar_type(), dout);
  if (with_dweights) dweights = make(order.sizes(), at::kFloat, dout);
  void* stream = stream_of(index);
  call(index, "moe_unpermute", g_steps.unpermute_grad, ptr(dr.t), dr.stride, ptr(rr.t), rr.stride,
       n_rows, ints(order), ints(slot_of_row), floats(weights), m,
       static_cast<int32_t>(order.size(1)), cols, type, ptr(drows), floats(dweights), stream);
  return {drows, dweights};
}

// ----------------------------------------------------------------- router ---
void check_logits(const at::Tensor& l, int64_t topk) {
  require(l.dim() == 2 && (l.scalar_type() == at::kFloat || l.scalar_type() == at::kBFloat16),
          "logits must be float32 or bfloat16 [tokens, experts]");
  if (topk < 0 || topk > 64) refuse(PyExc_ValueError, "fused_topk: topk must be in [1, 64]");
}

// (weights, ids)
std::array<at::Tensor, 2> topk_gating_of(const Arg& la, int64_t topk, int32_t scoring,
                                         bool renormalize) {
  const int index = check_inputs({la});
  const at::Tensor& l = *la.t;
  check_logits(l, topk);
  const at::Tensor logits = contiguous(l);
  const at::Tensor weights = make({l.size(0), topk}, at::kFloat, l);
  const at::Tensor ids = make({l.size(0), topk}, at::kInt, l);
  void* stream = stream_of(index);
  call(index, "fused_topk", g_steps.topk_gating, ptr(logits),
       static_cast<int32_t>(l.scalar_type() == at::kBFloat16), l.size(0),
       static_cast<int32_t>(l.size(1)), static_cast<int32_t>(topk), scoring,
       static_cast<int32_t>(renormalize), floats(weights), ints_out(ids), stream);
  return {weights, ids};
}

// The logits' gradient is one of the weights alone where they are the picks' own
// softmax, or sigmoids that are not renormalised.
bool topk_grad_reads_logits(int32_t scoring, bool renormalize) {
  return (scoring == FGS_SCORING_SIGMOID) == renormalize;
}

// (la: not given where they are not read)
at::Tensor topk_gating_grad_of(const Arg& wa, const Arg& ia, const Arg& da, const Arg& la,
                               int64_t experts, at::ScalarType type, int32_t scoring,
                               bool renormalize) {
  const int index = check_inputs({wa, ia, da, la});
  require(ia.t->dim() == 2 && ia.t->scalar_type() == at::kInt, "ids must be int32 [tokens, topk]");
  require(wa.t->sizes() == ia.t->sizes() && da.t->sizes() == ia.t->sizes() &&
              wa.t->scalar_type() == at::kFloat && da.t->scalar_type() == at::kFloat,
          "the weights and their gradient must be float32 [tokens, topk]");
  require(la.t || !topk_grad_reads_logits(scoring, renormalize), "the logits are read");
  require(!la.t || (la.t->dim() == 2 && la.t->size(0) == ia.t->size(0) && la.t->size(1) == experts &&
                    la.t->scalar_type() == type),
          "logits must be of the forward pass's shape and type");
  const at::Tensor weights = contiguous(*wa.t), ids = contiguous(*ia.t), d = contiguous(*da.t),
                   logits = la.t ? contiguous(*la.t) : at::Tensor();
  const int64_t m = ids.size(0);
  const at::Tensor out = make({m, experts}, type, ids);
  void* stream = stream_of(index);
  call(index, "fused_topk", g_steps.topk_gating_grad, ptr(logits),
       static_cast<int32_t>(type == at::kBFloat16), m, static_cast<int32_t>(experts),
       static_cast<int32_t>(ids.size(1)), scoring, static_cast<int32_t>(renormalize),
       floats(weights), ints(ids), floats(d), ptr(out), stream);
  return out;
}

// --------------------------------------------------------------- products ---
// A 16-bit matrix (or several) with adjacent columns, 16-byte aligned rows and a row
// stride of at least `least`: where it is, or copied. (Products whose sums run across
// its rows take a row for the end of the one before it.)
struct Matrix {
  at::Tensor t;
  int64_t row, group;  // strides
};
Matrix matrix(const at::Tensor& t, int64_t rows, int64_t cols, int64_t least = 0) {
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && cols % 8 == 0) {
    if (t.is_contiguous()) return {t, cols, rows * cols};
    const int64_t d = t.dim();
    if ((d == 2 || d == 3) && t.stride(d - 1) == 1 &&
        (rows <= 1 || (t.stride(d - 2) % 8 == 0 && t.stride(d - 2) <= kMaxLinearStride &&
                       t.stride(d - 2) >= least)) &&
        (d == 2 || t.size(0) <= 1 || t.stride(0) % 8 == 0))
      return {t, rows <= 1 ? cols : t.stride(d - 2), d == 3 ? t.stride(0) : 0};
  }
  return {t.clone(at::MemoryFormat::Contiguous), cols, rows * cols};
}

struct LinearSizes {
  int64_t groups, rows, wide, k;
  const at::Tensor* counts;
};
// Types and shapes of x [..., k] (grouped: [rows, k]) and w [wide, k] (grouped:
// [groups, wide, k]), counts [groups].
LinearSizes check_product(const at::Tensor& x, const at::Tensor& w, const Arg& ca) {
  const int type = type_code(x);
  require(type == FGS_DTYPE_BF16 || type == FGS_DTYPE_FP16, "x must be bfloat16 or float16");
  require(w.scalar_type() == x.scalar_type(), "weight must be of x's type");
  LinearSizes s{1, 0, 0, 0, ca.t};
  if (ca.t) {
    require(w.dim() == 3 && x.dim() == 2 && x.size(1) == w.size(2),
            "x must be [rows, k] and weight [groups, n, k]");
    require(ca.t->dim() == 1 && ca.t->size(0) == w.size(0) && ca.t->scalar_type() == at::kInt,
            "counts must be int32 [groups]");
    s.groups = w.size(0);
  } else {
    require(w.dim() == 2 && x.dim() >= 1 && x.size(-1) == w.size(1),
            "x must be [..., k] and weight [n, k]");
  }
  s.wide = w.size(-2);
  s.k = w.size(-1);
  require(s.groups > 0 && s.wide > 0 && s.k > 0, "weight must not be empty");
  s.rows = x.numel() / s.k;
  return s;
}
at::Tensor flat(const at::Tensor& x, int64_t rows, int64_t cols) {
  return x.dim() == 2 ? x : x.reshape({rows, cols});
}

struct LinearHow {
  int32_t act;
  bool gated;
  int32_t flags;  // a byte each of the forward product, the input's gradient, the weights'
  int32_t of(int pass) const { return (flags >> (8 * pass)) & 0xff; }
};

// (out, z)
std::array<at::Tensor, 2> linear_of(const Arg& xa, const Arg& wa, const Arg& ca, const Arg& ba,
                                    const Arg& ra, LinearHow how, bool with_z) {
  const int index = check_inputs({xa, wa, ca, ba, ra});
  const at::Tensor &x = *xa.t, &w = *wa.t;
  const LinearSizes s = check_product(x, w, ca);
  require(!how.gated || s.wide % 2 == 0, "a gated weight must hold gate rows and up rows");
  const int64_t n = how.gated ? s.wide / 2 : s.wide;
  at::DimVector shape(x.sizes().begin(), x.sizes().end());
  shape.back() = n;
  at::Tensor bias;
  if (ba.t) {
    require(ba.t->scalar_type() == x.scalar_type() && ba.t->dim() == w.dim() - 1 &&
                ba.t->size(-1) == s.wide && (!ca.t || ba.t->size(0) == s.groups),
            "bias must be [n] (grouped: [groups, n]) of x's type");
    bias = contiguous(*ba.t);
  }
  Matrix res{{}, 0, 0};
  if (ra.t) {
    require(ra.t->sizes() == shape && ra.t->scalar_type() == x.scalar_type(),
            "residual must be of the output's shape and type");
    res = matrix(flat(*ra.t, s.rows, n), s.rows, n);
  }
  const Matrix xm = matrix(flat(x, s.rows, s.k), s.rows, s.k), wm = matrix(w, s.wide, s.k);
  const at::Tensor counts = ca.t ? contiguous(*ca.t) : at::Tensor();
  const at::Tensor out = make(shape, x.scalar_type(), x);
  at::Tensor z;
  if (with_z) z = make({s.rows, s.wide}, at::kFloat, x);
  void* stream = stream_of(index);
  call(index, ca.t ? "grouped_linear" : "fused_linear", g_steps.linear, ptr(xm.t), xm.row,
       ptr(wm.t), wm.row, wm.group, ptr(bias), ptr(res.t), res.row, ints(counts),
       static_cast<int32_t>(s.groups), s.rows, n, s.k, static_cast<int32_t>(type_code(x)),
       how.act, static_cast<int32_t>(how.gated), how.of(0), floats(z), ptr(out), stream);
  return {out, z};
}

// (dx, dweight, dbias), those asked for; w only for dx, x only for dweight.
std::array<at::Tensor, 3> linear_grad_of(const Arg& da, const Arg& xa, const Arg& wa,
                                         const Arg& ca, const Arg& za, LinearHow how,
                                         bool with_dx, bool with_dw, bool with_db) {
  const int index = check_inputs({da, xa, wa, ca, za});
  const at::Tensor& dout = *da.t;
  const char* what = ca.t ? "grouped_linear" : "fused_linear";
  const int32_t type = static_cast<int32_t>(type_code(dout));
  require((type == FGS_DTYPE_BF16 || type == FGS_DTYPE_FP16) && dout.dim() >= 1 && dout.size(-1) > 0,
          "dout must be of the output's shape and type");
  const int64_t n = dout.size(-1);
  LinearSizes s{ca.t ? ca.t->size(0) : 1, dout.numel() / n, how.gated ? 2 * n : n, 0, ca.t};
  require(!ca.t || (ca.t->dim() == 1 && ca.t->scalar_type() == at::kInt), "counts must be int32 [groups]");
  require((wa.t || !with_dx) && (xa.t || !with_dw), "dx needs the weight, dweight x");
  if (with_dw) s.k = xa.t->size(-1);
  if (with_dx) s.k = wa.t->size(-1);
  require(!with_dx || (wa.t->dim() == (ca.t ? 3 : 2) && wa.t->size(-2) == s.wide &&
                       wa.t->numel() == s.groups * s.wide * s.k &&
                       wa.t->scalar_type() == dout.scalar_type()),
          "weight must be of the forward pass's shape and type");
  require(!with_dw || (xa.t->size(-1) == s.k && xa.t->numel() == s.rows * s.k &&
                       xa.t->scalar_type() == dout.scalar_type()),
          "x must be of the forward pass's shape and type");
  require(za.t || (how.act == FGS_ACT_NONE && !how.gated), "an activation's gradient needs z");
  require(!za.t || (za.t->dim() == 2 && za.t->size(0) == s.rows && za.t->size(1) == s.wide &&
                    za.t->scalar_type() == at::kFloat && za.t->is_contiguous()),
          "z must be float32 [rows, n], contiguous");
  const int32_t groups = static_cast<int32_t>(s.groups);
  const at::Tensor counts = ca.t ? contiguous(*ca.t) : at::Tensor();
  void* stream = stream_of(index);
  Matrix dz = matrix(flat(dout, s.rows, n), s.rows, n, with_dw && !za.t ? n : 0);
  if (za.t) {
    // (the products take dz rounded; the bias's sums with what that leaves, a matrix more)
    const at::Tensor t = make({s.rows * (with_db ? 2 : 1), s.wide}, dout.scalar_type(), dout);
    call(index, what, g_steps.linear_act_grad, ptr(dz.t), dz.row, floats(*za.t), s.rows, n,
         with_db ? type | FGS_DZ_REST : type, how.act, static_cast<int32_t>(how.gated), ptr(t), stream);
    dz = {t, s.wide, 0};
  }
  at::Tensor dx, dw, db;
  if (with_dx) {
    const Matrix wm = matrix(*wa.t, s.wide, s.k, s.k);
    at::DimVector shape(dout.sizes().begin(), dout.sizes().end());
    shape.back() = s.k;
    dx = make(shape, dout.scalar_type(), dout);
    call(index, what, g_steps.linear_input_grad, ptr(dz.t), dz.row, ptr(wm.t), wm.row, wm.group,
         ints(counts), groups, s.rows, s.wide, s.k, type, how.of(1), ptr(dx), stream);
  }
  if (with_dw) {
    const Matrix xm = matrix(flat(*xa.t, s.rows, s.k), s.rows, s.k, s.k);
    at::DimVector shape{s.groups, s.wide, s.k};
    if (!ca.t) shape.erase(shape.begin());
    dw = make(shape, dout.scalar_type(), dout);
    call(index, what, g_steps.linear_weight_grad, ptr(dz.t), dz.row, ptr(xm.t), xm.row,
         ints(counts), groups, s.rows, s.wide, s.k, type, how.of(2), ptr(dw), stream);
  }
  if (with_db) {
    const int64_t need = g_steps.linear_bias_grad_workspace_bytes(groups, s.rows, s.wide);
    const at::Tensor ws = bytes_for(need, dout);
    at::DimVector shape{s.groups, s.wide};
    if (!ca.t) shape.erase(shape.begin());
    db = make(shape, dout.scalar_type(), dout);
    call(index, what, g_steps.linear_bias_grad, ptr(dz.t), dz.row, ints(counts), groups, s.rows,
         s.wide, za.t ? type | FGS_DZ_REST : type, ptr(ws), need, ptr(db), stream);
  }
  return {dx, dw, db};
}

// -------------------------------------------------------------- gradients ---
// The operators as autograd functions. (As Python ones a forward and backward call
// of the router took 75 us, 8 of them the GPU's.)
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

Arg optional_arg(const at::Tensor& t, const char* name) { return {name, t.defined() ? &t : nullptr}; }
// (An undefined tensor is no argument of an autograd function; an absent optional one has
// no place among its edges either.)
std::optional<at::Tensor> given(const Arg& a) {
  return a.t ? std::optional<at::Tensor>(*a.t) : std::nullopt;
}
at::Tensor or_undefined(const std::optional<at::Tensor>& t) { return t ? *t : at::Tensor(); }

// A backward pass: `f` of gradients that are there, without gradients of its own;
// where a derivative of the result is asked for (create_graph), taking it raises.
template <class F>
variable_list backward_of(const char* what, const variable_list& grads, size_t count, F&& f) {
  variable_list out(count);
  if (!grads[0].defined()) return out;
  const bool again = c10::GradMode::is_enabled();
  {
    const at::AutoGradMode off(false);
    try {
      f(out);
    } catch (const Refusal& r) {  // (as what the engine hands on to the caller)
      TORCH_CHECK(false, r.text);
    }
  }
  if (!again) return out;
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string(what) + " has no second derivative", 1);
  for (at::Tensor& t : out)
    if (t.defined() && !t.is_same(grads[0])) t = (*error)({t.set_requires_grad(true)})[0];
  return out;
}

struct PermuteFunction : torch::autograd::Function<PermuteFunction> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& ids,
                               int64_t experts) {
    const Permuted p = permute_of({"x", &x}, {"topk_ids", &ids}, experts);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({p.counts, p.row_of_slot, p.slot_of_row});
    ctx->save_for_backward({p.row_of_slot});
    return {p.rows, p.counts, p.row_of_slot, p.slot_of_row};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return backward_of("moe_permute", grads, 3, [&](variable_list& out) {
      const at::Tensor order = ctx->get_saved_variables()[0];
      out[0] = unpermute_of({"rows", &grads[0]}, {"row_of_slot", &order}, {"topk_weights", nullptr});
    });
  }
};

struct PermuteRowsFunction : torch::autograd::Function<PermuteRowsFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& row_of_slot,
                            const at::Tensor& slot_of_row) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({row_of_slot});
    return permute_rows_of({"x", &x}, {"row_of_slot", &row_of_slot}, {"slot_of_row", &slot_of_row});
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return backward_of("moe_permute", grads, 3, [&](variable_list& out) {
      const at::Tensor order = ctx->get_saved_variables()[0];
      out[0] = unpermute_of({"rows", &grads[0]}, {"row_of_slot", &order}, {"topk_weights", nullptr});
    });
  }
};

struct UnpermuteFunction : torch::autograd::Function<UnpermuteFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& rows,
                            const std::optional<at::Tensor>& given_weights,
                            const at::Tensor& row_of_slot, const at::Tensor& slot_of_row,
                            bool with_dweights) {
    const at::Tensor weights = or_undefined(given_weights);
    ctx->set_materialize_grads(false);
    const at::Tensor none;
    ctx->save_for_backward({with_dweights ? rows : none, rows.requires_grad() ? weights : none,
                            row_of_slot, slot_of_row});
    return unpermute_of({"rows", &rows}, {"row_of_slot", &row_of_slot},
                        optional_arg(weights, "topk_weights"));
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return backward_of("moe_unpermute", grads, 5, [&](variable_list& out) {
      const variable_list saved = ctx->get_saved_variables();
      const auto g = unpermute_grad_of(
          {"dout", &grads[0]}, optional_arg(saved[0], "rows"), {"row_of_slot", &saved[2]},
          {"slot_of_row", &saved[3]}, optional_arg(saved[1], "topk_weights"),
          ctx->needs_input_grad(0), saved[0].defined() && ctx->needs_input_grad(1));
      out[0] = g[0];
      out[1] = g[1];
    });
  }
};

struct TopkFunction : torch::autograd::Function<TopkFunction> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, int64_t topk,
                               int64_t scoring, bool renormalize) {
    const auto r = topk_gating_of({"gating_output", &logits}, topk, static_cast<int32_t>(scoring),
                                  renormalize);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({r[1]});
    const bool read = topk_grad_reads_logits(static_cast<int32_t>(scoring), renormalize);
    ctx->save_for_backward({read ? logits : at::Tensor(), r[0], r[1]});
    ctx->saved_data["how"] = int64_t{renormalize} | scoring << 1 |
                             int64_t{logits.scalar_type() == at::kBFloat16} << 2 | logits.size(1) << 3;
    return {r[0], r[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return backward_of("fused_topk", grads, 4, [&](variable_list& out) {
      const variable_list saved = ctx->get_saved_variables();
      const int64_t how = ctx->saved_data["how"].toInt();
      out[0] = topk_gating_grad_of({"weights", &saved[1]}, {"ids", &saved[2]}, {"dweights", &grads[0]},
                                   optional_arg(saved[0], "logits"), how >> 3,
                                   how & 4 ? at::kBFloat16 : at::kFloat, how >> 1 & 1, how & 1);
    });
  }
};

struct LinearFunction : torch::autograd::Function<LinearFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w,
                            const std::optional<at::Tensor>& given_bias,
                            const std::optional<at::Tensor>& given_residual,
                            const std::optional<at::Tensor>& given_counts, int64_t act, bool gated,
                            int64_t flags, bool with_z) {
    const at::Tensor bias = or_undefined(given_bias), residual = or_undefined(given_residual),
                     counts = or_undefined(given_counts);
    const LinearHow how{static_cast<int32_t>(act), gated, static_cast<int32_t>(flags)};
    const auto r = linear_of({"x", &x}, {"weight", &w}, optional_arg(counts, "counts"),
                             optional_arg(bias, "bias"), optional_arg(residual, "residual"), how,
                             with_z);
    ctx->set_materialize_grads(false);
    // (what the gradients read that are asked for, and no more)
    const bool dx = x.requires_grad(), dw = w.requires_grad(),
               db = bias.defined() && bias.requires_grad();
    const at::Tensor none;
    ctx->save_for_backward({dw ? x : none, dx ? w : none, dx || dw || db ? counts : none, r[1]});
    // (one entry: each is a look-up by name, 0.4 us)
    ctx->saved_data["how"] = act | int64_t{gated} << 8 | int64_t{bias.defined()} << 9 |
                             int64_t{residual.defined()} << 10 | (flags & 0xffffff) << 16;
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return backward_of("this product", grads, 9, [&](variable_list& out) {
      const int64_t saved_how = ctx->saved_data["how"].toInt();
      const bool bias = saved_how >> 9 & 1, residual = saved_how >> 10 & 1;
      const bool dx = ctx->needs_input_grad(0), dw = ctx->needs_input_grad(1),
                 db = bias && ctx->needs_input_grad(2);
      if (dx || dw || db) {
        const variable_list saved = ctx->get_saved_variables();
        const LinearHow how{static_cast<int32_t>(saved_how & 0xff), (saved_how >> 8 & 1) != 0,
                            static_cast<int32_t>(saved_how >> 16)};
        const auto g = linear_grad_of({"dout", &grads[0]}, optional_arg(saved[0], "x"),
                                      optional_arg(saved[1], "weight"),
                                      optional_arg(saved[2], "counts"), optional_arg(saved[3], "z"),
                                      how, dx, dw, db);
        for (int i = 0; i < 3; ++i) out[i] = g[i];
      }
      if (residual && ctx->needs_input_grad(2 + bias)) out[3] = grads[0];
    });
  }
};

// ------------------------------------------------------------ Python's calls ---
// permute(x, topk_ids, num_experts, with_grad) -> (rows, counts, row_of_slot,
// slot_of_row)
PyObject* permute(PyObject* const* args) {
  const Arg x = tensor_arg(args[0], "x"), ids = tensor_arg(args[1], "topk_ids");
  const int64_t experts = whole(args[2]);
  if (truth(args[3])) {
    const variable_list r = PermuteFunction::apply(*x.t, *ids.t, experts);
    return wrap_all<4>({r[0], r[1], r[2], r[3]});
  }
  const Permuted p = permute_of(x, ids, experts);
  return wrap_all<4>({p.rows, p.counts, p.row_of_slot, p.slot_of_row});
}

// permute_rows(x, row_of_slot, slot_of_row, with_grad) -> rows
PyObject* permute_rows(PyObject* const* args) {
  const Arg x = tensor_arg(args[0], "x"), row_of_slot = tensor_arg(args[1], "row_of_slot"),
            slot_of_row = tensor_arg(args[2], "slot_of_row");
  if (truth(args[3])) return wrap(PermuteRowsFunction::apply(*x.t, *row_of_slot.t, *slot_of_row.t));
  return wrap(permute_rows_of(x, row_of_slot, slot_of_row));
}

// unpermute(rows, row_of_slot, slot_of_row, topk_weights, with_grad) -> out
PyObject* unpermute(PyObject* const* args) {
  const Arg rows = tensor_arg(args[0], "rows"), row_of_slot = tensor_arg(args[1], "row_of_slot"),
            slot_of_row = tensor_arg(args[2], "slot_of_row"),
            weights = tensor_arg(args[3], "topk_weights", true);
  if (truth(args[4])) {
    check_inputs({{"row_of_slot", row_of_slot.t}, {"slot_of_row", slot_of_row.t}});
    check_order(*row_of_slot.t, slot_of_row.t);
    return wrap(UnpermuteFunction::apply(*rows.t, given(weights), *row_of_slot.t, *slot_of_row.t,
                                         weights.t && weights.t->requires_grad()));
  }
  return wrap(unpermute_of(rows, row_of_slot, weights));
}

// topk_gating(logits, topk, scoring, renormalize) -> (weights, ids), with the
// weights' gradient
PyObject* topk_gating(PyObject* const* args) {
  const Arg logits = tensor_arg(args[0], "gating_output");
  const variable_list r =
      TopkFunction::apply(*logits.t, whole(args[1]), whole(args[2]), truth(args[3]));
  return wrap_all<2>({r[0], r[1]});
}

// linear(x, weight, counts, bias, act, gated, residual, with_grad, flags) -> out
PyObject* linear(PyObject* const* args) {
  const Arg x = tensor_arg(args[0], "x"), w = tensor_arg(args[1], "weight"),
            counts = tensor_arg(args[2], "counts", true), bias = tensor_arg(args[3], "bias", true),
            residual = tensor_arg(args[6], "residual", true);
  const LinearHow how{static_cast<int32_t>(whole(args[4])), truth(args[5]),
                      static_cast<int32_t>(whole(args[8]))};
  if (!truth(args[7])) return wrap(linear_of(x, w, counts, bias, residual, how, false)[0]);
  // what the activation is taken of is kept where a gradient goes through it
  bool through = false;
  for (const Arg* a : {&x, &w, &bias}) through = through || (a->t && a->t->requires_grad());
  const bool with_z = through && (how.act != FGS_ACT_NONE || how.gated);
  return wrap(LinearFunction::apply(*x.t, *w.t, given(bias), given(residual), given(counts),
                                    static_cast<int64_t>(how.act), how.gated,
                                    static_cast<int64_t>(how.flags), with_z));
}

// foreign_leaf(tensor) -> whether autograd holds the tensor's gradient node for
// another stream than the current one.
PyObject* foreign_leaf(PyObject* const* args) {
  const Arg a = tensor_arg(args[0], "tensor");
  bool foreign = false;
  if (a.t->is_cuda() && a.t->requires_grad() && a.t->is_leaf()) {
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*a.t);
    if (node) {
      const auto stream = node->stream();
      const c10::Stream now = c10::impl::VirtualGuardImpl(a.t->device().type()).getStream(a.t->device());
      foreign = stream && *stream != now;
    }
  }
  return PyBool_FromLong(foreign);
}

// bind_steps(addresses of the entries, in StepsLibrary's order)
PyObject* bind_steps(PyObject* const* args) {
  auto set = [&](int i, auto& entry) {
    entry = reinterpret_cast<std::decay_t<decltype(entry)>>(reinterpret_cast<void*>(whole(args[i])));
  };
  set(0, g_steps.permute_workspace_bytes);
  set(1, g_steps.permute);
  set(2, g_steps.permute_rows);
  set(3, g_steps.unpermute);
  set(4, g_steps.unpermute_grad);
  set(5, g_steps.topk_gating);
  set(6, g_steps.topk_gating_grad);
  set(7, g_steps.linear);
  set(8, g_steps.linear_act_grad);
  set(9, g_steps.linear_input_grad);
  set(10, g_steps.linear_weight_grad);
  set(11, g_steps.linear_bias_grad_workspace_bytes);
  set(12, g_steps.linear_bias_grad);
  Py_RETURN_NONE;
}
