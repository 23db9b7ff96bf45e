// Host side of the routed layer's steps and their gradients (flaggems_sglang.ops.
// steps, .linear): part of host_ext.cpp, whose helpers it uses.

struct StepsLibrary {
  decltype(&fgs_moe_permute_workspace_bytes) permute_workspace_bytes;
  decltype(&fgs_moe_permute) permute;
  decltype(&fgs_moe_permute_rows) permute_rows;
  decltype(&fgs_moe_unpermute) unpermute;
  decltype(&fgs_moe_unpermute_grad) unpermute_grad;
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

// permute(x, topk_ids, num_experts) -> (rows, counts, row_of_slot, slot_of_row)
PyObject* permute(PyObject* const* args) {
  const Arg xa = tensor_arg(args[0], "x"), ia = tensor_arg(args[1], "topk_ids");
  const int index = check_inputs({xa, ia});
  const int64_t experts = whole(args[2]);
  const at::Tensor& x = *xa.t;
  require(x.dim() == 2 && x.size(1) > 0, "x must be [tokens, cols]");
  require(movable(x.scalar_type()), "x must be of a 8- to 64-bit integer or a 8- to 32-bit float type");
  require(ia.t->dim() == 2 && ia.t->size(0) == x.size(0) && ia.t->size(1) > 0 &&
              ia.t->scalar_type() == at::kInt,
          "topk_ids must be int32 [tokens, topk]");
  if (experts < 1 || experts > 1022)
    refuse(PyExc_ValueError, "moe_permute: num_experts must be in [1, 1022]");
  const int64_t m = x.size(0), topk = ia.t->size(1), slots = m * topk, size = x.element_size();
  const Rows xr = rows_of(x, x.size(1));
  const at::Tensor ids = contiguous(*ia.t);
  const at::Tensor rows = make({slots, x.size(1)}, x.scalar_type(), x);
  const at::Tensor counts = make({experts}, at::kInt, x);
  const at::Tensor row_of_slot = make({m, topk}, at::kInt, x);
  const at::Tensor slot_of_row = make({slots}, at::kInt, x);
  const int64_t need = g_steps.permute_workspace_bytes(slots, static_cast<int32_t>(experts));
  if (need < 0) refuse(PyExc_NotImplementedError, "moe_permute: more than 2^30 slots");
  const at::Tensor ws = bytes_for(need, x);
  void* stream = stream_of(index);
  call(index, "moe_permute", g_steps.permute, ptr(xr.t), xr.stride * size, m, x.size(1) * size,
       ints(ids), static_cast<int32_t>(topk), static_cast<int32_t>(experts), ptr(rows),
       ints_out(counts), ints_out(row_of_slot), ints_out(slot_of_row), ptr(ws), need, stream);
  return wrap_all<4>({rows, counts, row_of_slot, slot_of_row});
}

// permute_rows(x, row_of_slot, slot_of_row) -> rows
PyObject* permute_rows(PyObject* const* args) {
  const Arg xa = tensor_arg(args[0], "x"), ra = tensor_arg(args[1], "row_of_slot"),
            sa = tensor_arg(args[2], "slot_of_row");
  const int index = check_inputs({xa, ra, sa});
  const at::Tensor& x = *xa.t;
  require(x.dim() == 2 && x.size(1) > 0, "x must be [tokens, cols]");
  require(movable(x.scalar_type()), "x must be of a 8- to 64-bit integer or a 8- to 32-bit float type");
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
  return wrap(rows);
}

void check_weights(const Arg& wa, const at::Tensor& row_of_slot) {
  require(!wa.t || (wa.t->sizes() == row_of_slot.sizes() && wa.t->scalar_type() == at::kFloat),
          "topk_weights must be float32 [tokens, topk]");
}

// unpermute(rows, row_of_slot, topk_weights) -> out
PyObject* unpermute(PyObject* const* args) {
  const Arg ra = tensor_arg(args[0], "rows"), oa = tensor_arg(args[1], "row_of_slot"),
            wa = tensor_arg(args[2], "topk_weights", true);
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
  return wrap(out);
}

// unpermute_grad(dout, rows, row_of_slot, slot_of_row, topk_weights, with_drows,
// with_dweights) -> (drows, dweights); rows may be None without dweights
PyObject* unpermute_grad(PyObject* const* args) {
  const Arg da = tensor_arg(args[0], "dout"), ra = tensor_arg(args[1], "rows", true),
            oa = tensor_arg(args[2], "row_of_slot"), sa = tensor_arg(args[3], "slot_of_row"),
            wa = tensor_arg(args[4], "topk_weights", true);
  const int index = check_inputs({da, ra, oa, sa, wa});
  const bool with_drows = truth(args[5]), with_dweights = truth(args[6]);
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
  return wrap_all<2>({drows, dweights});
}

// topk_gating_grad(logits, weights, ids, dweights, scoring, renormalize) -> dlogits
PyObject* topk_gating_grad(PyObject* const* args) {
  const Arg la = tensor_arg(args[0], "logits"), wa = tensor_arg(args[1], "weights"),
            ia = tensor_arg(args[2], "ids"), da = tensor_arg(args[3], "dweights");
  const int index = check_inputs({la, wa, ia, da});
  const int32_t scoring = static_cast<int32_t>(whole(args[4]));
  const bool renormalize = truth(args[5]);
  const at::Tensor& l = *la.t;
  require(l.dim() == 2 && (l.scalar_type() == at::kFloat || l.scalar_type() == at::kBFloat16),
          "logits must be float32 or bfloat16 [tokens, experts]");
  require(ia.t->dim() == 2 && ia.t->size(0) == l.size(0) && ia.t->scalar_type() == at::kInt,
          "ids must be int32 [tokens, topk]");
  require(wa.t->sizes() == ia.t->sizes() && da.t->sizes() == ia.t->sizes() &&
              wa.t->scalar_type() == at::kFloat && da.t->scalar_type() == at::kFloat,
          "the weights and their gradient must be float32 [tokens, topk]");
  const at::Tensor logits = contiguous(l), weights = contiguous(*wa.t), ids = contiguous(*ia.t),
                   d = contiguous(*da.t);
  const at::Tensor out = make(l.sizes(), l.scalar_type(), l);
  void* stream = stream_of(index);
  call(index, "fused_topk", g_steps.topk_gating_grad, ptr(logits),
       static_cast<int32_t>(l.scalar_type() == at::kBFloat16), l.size(0),
       static_cast<int32_t>(l.size(1)), static_cast<int32_t>(ids.size(1)), scoring,
       static_cast<int32_t>(renormalize), floats(weights), ints(ids), floats(d), ptr(out), stream);
  return wrap(out);
}

// --------------------------------------------------------------- products ---
// A 16-bit matrix (or several) with adjacent columns and 16-byte aligned rows:
// where it is, or copied.
struct Matrix {
  at::Tensor t;
  int64_t row, group;  // strides
};
Matrix matrix(const at::Tensor& t, int64_t rows, int64_t cols) {
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && cols % 8 == 0) {
    if (t.is_contiguous()) return {t, cols, rows * cols};
    const int64_t d = t.dim();
    if ((d == 2 || d == 3) && t.stride(d - 1) == 1 &&
        (rows <= 1 || (t.stride(d - 2) % 8 == 0 && t.stride(d - 2) <= kMaxLinearStride)) &&
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

// linear(x, weight, counts, bias, act, gated, residual, with_z, flags) -> (out, z)
PyObject* linear(PyObject* const* args) {
  const Arg xa = tensor_arg(args[0], "x"), wa = tensor_arg(args[1], "weight"),
            ca = tensor_arg(args[2], "counts", true), ba = tensor_arg(args[3], "bias", true),
            ra = tensor_arg(args[6], "residual", true);
  const int index = check_inputs({xa, wa, ca, ba, ra});
  const int32_t act = static_cast<int32_t>(whole(args[4]));
  const bool gated = truth(args[5]), with_z = truth(args[7]);
  const int32_t flags = static_cast<int32_t>(whole(args[8]));
  const at::Tensor &x = *xa.t, &w = *wa.t;
  const LinearSizes s = check_product(x, w, ca);
  require(!gated || s.wide % 2 == 0, "a gated weight must hold gate rows and up rows");
  const int64_t n = gated ? s.wide / 2 : s.wide;
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
  if (with_z) z = make({s.rows, s.wide}, x.scalar_type(), x);
  void* stream = stream_of(index);
  call(index, ca.t ? "grouped_linear" : "fused_linear", g_steps.linear, ptr(xm.t), xm.row,
       ptr(wm.t), wm.row, wm.group, ptr(bias), ptr(res.t), res.row, ints(counts),
       static_cast<int32_t>(s.groups), s.rows, n, s.k, static_cast<int32_t>(type_code(x)), act,
       static_cast<int32_t>(gated), flags, ptr(z), ptr(out), stream);
  return wrap_all<2>({out, z});
}

// linear_grad(dout, x, weight, counts, z, act, gated, with_dx, with_dweight,
// with_dbias, flags) -> (dx, dweight, dbias)
PyObject* linear_grad(PyObject* const* args) {
  const Arg da = tensor_arg(args[0], "dout"), xa = tensor_arg(args[1], "x"),
            wa = tensor_arg(args[2], "weight"), ca = tensor_arg(args[3], "counts", true),
            za = tensor_arg(args[4], "z", true);
  const int index = check_inputs({da, xa, wa, ca, za});
  const int32_t act = static_cast<int32_t>(whole(args[5]));
  const bool gated = truth(args[6]), with_dx = truth(args[7]), with_dw = truth(args[8]),
             with_db = truth(args[9]);
  const int32_t flags = static_cast<int32_t>(whole(args[10]));
  const at::Tensor &x = *xa.t, &w = *wa.t;
  const char* what = ca.t ? "grouped_linear" : "fused_linear";
  const LinearSizes s = check_product(x, w, ca);
  require(!gated || s.wide % 2 == 0, "a gated weight must hold gate rows and up rows");
  const int64_t n = gated ? s.wide / 2 : s.wide;
  at::DimVector shape(x.sizes().begin(), x.sizes().end());
  shape.back() = n;
  require(da.t->sizes() == shape && da.t->scalar_type() == x.scalar_type(),
          "dout must be of the output's shape and type");
  require(za.t || (act == FGS_ACT_NONE && !gated), "an activation's gradient needs z");
  require(!za.t || (za.t->dim() == 2 && za.t->size(0) == s.rows && za.t->size(1) == s.wide &&
                    za.t->scalar_type() == x.scalar_type() && za.t->is_contiguous()),
          "z must be [rows, n] of x's type, contiguous");
  const int32_t type = static_cast<int32_t>(type_code(x)), groups = static_cast<int32_t>(s.groups);
  const at::Tensor counts = ca.t ? contiguous(*ca.t) : at::Tensor();
  void* stream = stream_of(index);
  Matrix dz = matrix(flat(*da.t, s.rows, n), s.rows, n);
  if (za.t) {
    const at::Tensor t = make({s.rows, s.wide}, x.scalar_type(), x);
    call(index, what, g_steps.linear_act_grad, ptr(dz.t), dz.row, ptr(*za.t), s.rows, n, type, act,
         static_cast<int32_t>(gated), ptr(t), stream);
    dz = {t, s.wide, 0};
  }
  at::Tensor dx, dw, db;
  if (with_dx) {
    const Matrix wm = matrix(w, s.wide, s.k);
    dx = make(x.sizes(), x.scalar_type(), x);
    call(index, what, g_steps.linear_input_grad, ptr(dz.t), dz.row, ptr(wm.t), wm.row, wm.group,
         ints(counts), groups, s.rows, s.wide, s.k, type, flags, ptr(dx), stream);
  }
  if (with_dw) {
    const Matrix xm = matrix(flat(x, s.rows, s.k), s.rows, s.k);
    dw = make(w.sizes(), x.scalar_type(), x);
    call(index, what, g_steps.linear_weight_grad, ptr(dz.t), dz.row, ptr(xm.t), xm.row,
         ints(counts), groups, s.rows, s.wide, s.k, type, flags, ptr(dw), stream);
  }
  if (with_db) {
    const int64_t need = g_steps.linear_bias_grad_workspace_bytes(groups, s.rows, s.wide);
    const at::Tensor ws = bytes_for(need, x);
    db = ca.t ? make({s.groups, s.wide}, x.scalar_type(), x) : make({s.wide}, x.scalar_type(), x);
    call(index, what, g_steps.linear_bias_grad, ptr(dz.t), dz.row, ints(counts), groups, s.rows,
         s.wide, type, ptr(ws), need, ptr(db), stream);
  }
  return wrap_all<3>({dx, dw, db});
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
  set(5, g_steps.topk_gating_grad);
  set(6, g_steps.linear);
  set(7, g_steps.linear_act_grad);
  set(8, g_steps.linear_input_grad);
  set(9, g_steps.linear_weight_grad);
  set(10, g_steps.linear_bias_grad_workspace_bytes);
  set(11, g_steps.linear_bias_grad);
  Py_RETURN_NONE;
}
