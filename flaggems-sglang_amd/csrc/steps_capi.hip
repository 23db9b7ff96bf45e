// C entries of the routed layer's steps and their gradients (include/fgs_moe.h):
// what the arguments are checked for, and the launches.
#include <string.h>

#include <algorithm>
#include <string>

#include "fgs_moe_kernels.h"

namespace fgs {
namespace {

hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }
bool misaligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }
int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }

constexpr int kMaxPermuteExperts = 1022;  // (a class more: slots of no expert)
constexpr int64_t kMaxSlots = 1 << 30;
constexpr int kMaxGroups = 4096;

int check_slots(int64_t m, int32_t topk) {
  if (m < 0 || topk < 1) return fail(FGS_EINVAL, "m >= 0 and topk >= 1 required");
  if (m > kMaxSlots / topk) return fail(FGS_EUNSUPPORTED, "more than 2^30 slots");
  return FGS_OK;
}
int check_moved_rows(int64_t row_bytes, int64_t x_stride) {
  if (row_bytes < 1) return fail(FGS_EINVAL, "row_bytes must be >= 1");
  if (row_bytes > (int64_t{1} << 24)) return fail(FGS_EUNSUPPORTED, "rows of more than 2^24 bytes");
  if (x_stride < 0) return fail(FGS_EINVAL, "row strides must be >= 0");
  return FGS_OK;
}
int check_float_type(int32_t dtype) {
  if (dtype != FGS_DTYPE_BF16 && dtype != FGS_DTYPE_FP16 && dtype != FGS_DTYPE_FP32)
    return fail(FGS_EINVAL, "unknown element type");
  return FGS_OK;
}
uintptr_t element(int32_t dtype) { return dtype == FGS_DTYPE_FP32 ? 4 : 2; }

int check_unpermute(int64_t m, int32_t topk, int64_t n_rows, int64_t cols, int32_t dtype) {
  int rc = check_slots(m, topk);
  if (rc) return rc;
  if ((rc = check_float_type(dtype))) return rc;
  if (n_rows < 0 || cols < 1) return fail(FGS_EINVAL, "n_rows >= 0 and cols >= 1 required");
  if (n_rows > kMaxSlots) return fail(FGS_EUNSUPPORTED, "more than 2^30 rows");
  if (cols > (int64_t{1} << 22)) return fail(FGS_EUNSUPPORTED, "rows of more than 2^22 columns");
  return FGS_OK;
}

// Sizes of a product (`wide`: rows of a matrix of w).
int check_linear(int64_t groups, int64_t rows, int64_t wide, int64_t k, int32_t dtype) {
  if (dtype != FGS_DTYPE_BF16 && dtype != FGS_DTYPE_FP16)
    return fail(dtype == FGS_DTYPE_FP32 ? FGS_EUNSUPPORTED : FGS_EINVAL,
                "the matrices must be bf16 or fp16");
  if (groups < 1 || rows < 0 || wide < 1 || k < 1)
    return fail(FGS_EINVAL, "rows >= 0, groups >= 1, n >= 1 and k >= 1 required");
  if (wide % 8 || k % 8) return fail(FGS_EUNSUPPORTED, "n and k must be multiples of 8");
  if (groups > kMaxGroups || rows > kLinearMaxRows || wide > kLinearMaxCols || k > kLinearMaxCols)
    return fail(FGS_EUNSUPPORTED, "sizes too large for the kernels' grids");
  return FGS_OK;
}
int check_act(int32_t act) {
  if (act < FGS_ACT_NONE || act > FGS_ACT_GELU) return fail(FGS_EINVAL, "unknown activation");
  return FGS_OK;
}
// A matrix whose rows the kernels read in whole vectors.
int check_rows(const char* name, const void* p, int64_t rows, int64_t ld) {
  if (misaligned(p, 16) || (rows > 1 && ld % 8))
    return fail(FGS_EUNSUPPORTED, std::string("rows of ") + name + " must be 16-byte aligned");
  if (rows > 1 && (ld < 0 || ld > kLinearMaxStride))
    return fail(FGS_EUNSUPPORTED, std::string("row stride of ") + name + " negative or too large");
  return FGS_OK;
}

}  // namespace
}  // namespace fgs

using namespace fgs;

extern "C" {

int32_t fgs_moe_topk_gating_grad(const void* logits, int32_t logits_bf16, int64_t m,
                                 int32_t num_experts, int32_t topk, int32_t scoring,
                                 int32_t renormalize, const float* topk_weights,
                                 const int32_t* topk_ids, const float* dweights, void* dlogits,
                                 void* stream) {
  if (m < 0) return fail(FGS_EINVAL, "m must be >= 0");
  if (num_experts < 1 || num_experts > 1024)
    return fail(FGS_EINVAL, "num_experts must be in [1, 1024]");
  if (topk < 1 || topk > num_experts || topk > 64)
    return fail(FGS_EINVAL, "topk must be in [1, min(num_experts, 64)]");
  if (scoring != FGS_SCORING_SOFTMAX && scoring != FGS_SCORING_SIGMOID)
    return fail(FGS_EINVAL, "unknown scoring function");
  const bool reads_logits = (scoring == FGS_SCORING_SIGMOID) == (renormalize != 0);
  if (m > 0 && ((reads_logits && !logits) || !topk_weights || !topk_ids || !dweights || !dlogits))
    return fail(FGS_EINVAL, "null pointer argument");
  return launch_topk_gating_grad(logits, logits_bf16 != 0, m, num_experts, topk,
                                 scoring == FGS_SCORING_SIGMOID, renormalize != 0, topk_weights,
                                 topk_ids, dweights, dlogits, as_stream(stream));
}

// each slot's place, the class of each place, the number of places; the
// alignment's counts
int64_t fgs_moe_permute_workspace_bytes(int64_t numel, int32_t num_experts) {
  if (numel < 0 || numel > kMaxSlots || num_experts < 1 || num_experts > kMaxPermuteExperts)
    return -1;
  return 3 * up256(numel * 4) + 256 + align_scratch_bytes(numel, num_experts + 1);
}

int32_t fgs_moe_permute(const void* x, int64_t x_stride, int64_t m, int64_t row_bytes,
                        const int32_t* topk_ids, int32_t topk, int32_t num_experts, void* rows,
                        int32_t* counts, int32_t* row_of_slot, int32_t* slot_of_row,
                        void* workspace, int64_t ws_bytes, void* stream) {
  int rc = check_slots(m, topk);
  if (rc) return rc;
  if ((rc = check_moved_rows(row_bytes, x_stride))) return rc;
  if (num_experts < 1 || num_experts > kMaxPermuteExperts)
    return fail(FGS_EINVAL, "num_experts must be in [1, 1022]");
  const int64_t numel = m * topk;
  if (!counts || (numel > 0 && (!x || !topk_ids || !rows || !row_of_slot || !slot_of_row)))
    return fail(FGS_EINVAL, "null pointer argument");
  if (!workspace || ws_bytes < fgs_moe_permute_workspace_bytes(numel, num_experts))
    return fail(FGS_EINVAL, "workspace too small");
  if (misaligned(workspace, 256)) return fail(FGS_EINVAL, "workspace must be 256-byte aligned");
  if (misaligned(topk_ids, 4) || misaligned(counts, 4) || misaligned(row_of_slot, 4) ||
      misaligned(slot_of_row, 4))
    return fail(FGS_EINVAL, "tensors must be aligned to their elements");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int64_t part = up256(numel * 4);
  int32_t* place = reinterpret_cast<int32_t*>(ws);
  int32_t* sorted = reinterpret_cast<int32_t*>(ws + part);
  int32_t* classes = reinterpret_cast<int32_t*>(ws + 2 * part);
  int32_t* npp = reinterpret_cast<int32_t*>(ws + 3 * part);
  int32_t* scratch = align_scratch_bytes(numel, num_experts + 1) > 0 ? npp + 64 : nullptr;
  PermuteParams p{};
  p.x = static_cast<const uint8_t*>(x);
  p.x_stride = x_stride;
  p.bytes = row_bytes;
  p.m = m;
  p.topk = topk;
  p.experts = num_experts;
  p.ids = topk_ids;
  p.place = place;
  p.row_of_slot = row_of_slot;
  p.slot_of_row = slot_of_row;
  p.rows = static_cast<uint8_t*>(rows);
  p.counts = counts;
  if (numel > 0 && numel <= kPermuteFew) return launch_permute_few(p, as_stream(stream));
  rc = launch_align(topk_ids, numel, num_experts + 1, 1, sorted, classes, npp, numel,
                    as_stream(stream), scratch, nullptr, nullptr, num_experts, counts, place);
  if (rc || numel == 0) return rc;
  return launch_permute(p, as_stream(stream));
}

int32_t fgs_moe_permute_rows(const void* x, int64_t x_stride, int64_t m, int64_t row_bytes,
                             const int32_t* row_of_slot, int32_t topk, const int32_t* slot_of_row,
                             void* rows, void* stream) {
  int rc = check_slots(m, topk);
  if (rc) return rc;
  if ((rc = check_moved_rows(row_bytes, x_stride))) return rc;
  if (m == 0) return FGS_OK;
  if (!x || !row_of_slot || !slot_of_row || !rows) return fail(FGS_EINVAL, "null pointer argument");
  if (misaligned(row_of_slot, 4) || misaligned(slot_of_row, 4))
    return fail(FGS_EINVAL, "tensors must be aligned to their elements");
  PermuteParams p{};
  p.x = static_cast<const uint8_t*>(x);
  p.x_stride = x_stride;
  p.bytes = row_bytes;
  p.m = m;
  p.topk = topk;
  p.row_of_slot = const_cast<int32_t*>(row_of_slot);  // (read where there are no ids)
  p.slot_of_row = const_cast<int32_t*>(slot_of_row);
  p.rows = static_cast<uint8_t*>(rows);
  return launch_permute(p, as_stream(stream));
}

int32_t fgs_moe_unpermute(const void* rows, int64_t ld, int64_t n_rows,
                          const int32_t* row_of_slot, const float* topk_weights, int64_t m,
                          int32_t topk, int64_t cols, int32_t dtype, void* out, void* stream) {
  int rc = check_unpermute(m, topk, n_rows, cols, dtype);
  if (rc || m == 0) return rc;
  if (!row_of_slot || !out || (n_rows > 0 && !rows))
    return fail(FGS_EINVAL, "null pointer argument");
  if (n_rows > 1 && ld < 0) return fail(FGS_EINVAL, "row strides must be >= 0");
  if (misaligned(rows, element(dtype)) || misaligned(out, element(dtype)) ||
      misaligned(row_of_slot, 4) || misaligned(topk_weights, 4))
    return fail(FGS_EINVAL, "tensors must be aligned to their elements");
  UnpermuteParams p{};
  p.rows = rows;
  p.ld = ld;
  p.n_rows = n_rows;
  p.cols = cols;
  p.m = m;
  p.topk = topk;
  p.row_of_slot = row_of_slot;
  p.weights = topk_weights;
  p.out = out;
  return launch_unpermute(p, dtype, as_stream(stream));
}

int32_t fgs_moe_unpermute_grad(const void* dout, int64_t ldd, const void* rows, int64_t ld,
                               int64_t n_rows, const int32_t* row_of_slot,
                               const int32_t* slot_of_row, const float* topk_weights, int64_t m,
                               int32_t topk, int64_t cols, int32_t dtype, void* drows,
                               float* dweights, void* stream) {
  int rc = check_unpermute(m, topk, n_rows, cols, dtype);
  if (rc) return rc;
  if (m == 0 && n_rows == 0) return FGS_OK;
  if (!drows && !dweights) return fail(FGS_EINVAL, "no output was asked for");
  if ((m > 0 && (!dout || !row_of_slot)) || (drows && n_rows > 0 && !slot_of_row) ||
      (dweights && m > 0 && n_rows > 0 && !rows))
    return fail(FGS_EINVAL, "null pointer argument");
  if ((n_rows > 1 && ld < 0) || (m > 1 && ldd < 0))
    return fail(FGS_EINVAL, "row strides must be >= 0");
  for (const void* t : {dout, rows, static_cast<const void*>(drows)})
    if (misaligned(t, element(dtype)))
      return fail(FGS_EINVAL, "tensors must be aligned to their elements");
  for (const void* t : {static_cast<const void*>(row_of_slot), static_cast<const void*>(slot_of_row),
                        static_cast<const void*>(topk_weights), static_cast<const void*>(dweights)})
    if (misaligned(t, 4)) return fail(FGS_EINVAL, "tensors must be aligned to their elements");
  UnpermuteParams p{};
  p.rows = rows;
  p.ld = ld;
  p.n_rows = n_rows;
  p.cols = cols;
  p.m = m;
  p.topk = topk;
  p.row_of_slot = row_of_slot;
  p.weights = topk_weights;
  p.dout = dout;
  p.ldd = ldd;
  p.slot_of_row = slot_of_row;
  p.drows = drows;
  p.dweights = dweights;
  return launch_unpermute(p, dtype, as_stream(stream));
}

int32_t fgs_moe_linear(const void* x, int64_t ldx, const void* w, int64_t ldw,
                       int64_t w_group_stride, const void* bias, const void* residual,
                       int64_t ldr, const int32_t* counts, int32_t groups, int64_t rows,
                       int64_t n, int64_t k, int32_t dtype, int32_t act, int32_t gated,
                       int32_t flags, float* z, void* out, void* stream) {
  int rc = check_linear(groups, rows, n, k, dtype);
  if (rc || (gated && (rc = check_linear(groups, rows, 2 * n, k, dtype)))) return rc;
  if ((rc = check_act(act))) return rc;
  if (!linear_flags_ok(gated ? kLinearGated : kLinearForward, flags)) return fail(FGS_EINVAL, "unknown flags");
  if (!counts && groups != 1) return fail(FGS_EINVAL, "counts are needed for several groups");
  if (rows == 0) return FGS_OK;
  if (!x || !w || !out) return fail(FGS_EINVAL, "null pointer argument");
  if ((rc = check_rows("x", x, rows, ldx)) || (rc = check_rows("w", w, 2, ldw)) ||
      (rc = check_rows("the residual", residual, residual ? rows : 0, ldr)) ||
      (rc = check_rows("out", out, 0, 0)) || (rc = check_rows("z", z, 0, 0)))
    return rc;
  if (groups > 1 && (w_group_stride < 0 || w_group_stride % 8))
    return fail(FGS_EUNSUPPORTED, "matrices of w must be 16-byte aligned");
  if (misaligned(bias, 2) || misaligned(counts, 4))
    return fail(FGS_EINVAL, "tensors must be aligned to their elements");
  LinearParams p{};
  p.q = x;
  p.ldq = rows > 1 ? ldx : k;
  p.p = w;
  p.ldp = ldw;
  p.p_group = w_group_stride;
  p.out = out;
  p.bias = bias;
  p.residual = residual;
  p.ldr = ldr;
  p.z = z;
  p.counts = counts;
  p.groups = groups;
  p.rows = static_cast<int32_t>(rows);
  p.red = static_cast<int32_t>(k);
  p.n = static_cast<int32_t>(n);
  p.act = act;
  const int mode = gated ? kLinearGated : kLinearForward;
  return launch_linear(p, mode, dtype, linear_form(mode, groups, rows, 0, n, k, flags),
                       as_stream(stream));
}

int32_t fgs_moe_linear_act_grad(const void* dout, int64_t ldd, const float* z, int64_t rows,
                                int64_t n, int32_t dtype, int32_t act, int32_t gated, void* dz,
                                void* stream) {
  const bool with_rest = (dtype & FGS_DZ_REST) != 0;
  dtype &= ~FGS_DZ_REST;
  int rc = check_linear(1, rows, n, 8, dtype);
  if (rc || (gated && (rc = check_linear(1, rows, 2 * n, 8, dtype)))) return rc;
  if ((rc = check_act(act))) return rc;
  if (rows == 0) return FGS_OK;
  if (!dout || !z || !dz) return fail(FGS_EINVAL, "null pointer argument");
  if ((rc = check_rows("dout", dout, rows, ldd)) || (rc = check_rows("z", z, 0, 0)) ||
      (rc = check_rows("dz", dz, 0, 0)))
    return rc;
  LinearActGradParams p{};
  p.dout = dout;
  p.ldd = ldd;
  p.z = z;
  p.dz = dz;
  if (with_rest) p.rest = static_cast<uint16_t*>(dz) + rows * (gated ? 2 * n : n);
  p.rows = rows;
  p.n = n;
  p.act = act;
  p.gated = gated != 0;
  return launch_linear_act_grad(p, dtype, as_stream(stream));
}

int32_t fgs_moe_linear_input_grad(const void* dz, int64_t ldz, const void* w, int64_t ldw,
                                  int64_t w_group_stride, const int32_t* counts, int32_t groups,
                                  int64_t rows, int64_t wide, int64_t k, int32_t dtype,
                                  int32_t flags, void* dx, void* stream) {
  int rc = check_linear(groups, rows, wide, k, dtype);
  if (rc) return rc;
  if (!linear_flags_ok(kLinearDgrad, flags)) return fail(FGS_EINVAL, "unknown flags");
  if (!counts && groups != 1) return fail(FGS_EINVAL, "counts are needed for several groups");
  if (rows == 0) return FGS_OK;
  if (!dz || !w || !dx) return fail(FGS_EINVAL, "null pointer argument");
  if ((rc = check_rows("dz", dz, rows, ldz)) || (rc = check_rows("w", w, 2, ldw)) ||
      (rc = check_rows("dx", dx, 0, 0)))
    return rc;
  if (groups > 1 && (w_group_stride < 0 || w_group_stride % 8))
    return fail(FGS_EUNSUPPORTED, "matrices of w must be 16-byte aligned");
  if (misaligned(counts, 4)) return fail(FGS_EINVAL, "tensors must be aligned to their elements");
  LinearParams p{};
  p.q = dz;
  p.ldq = rows > 1 ? ldz : wide;
  p.p = w;
  p.ldp = ldw;
  p.p_group = w_group_stride;
  p.out = dx;
  p.counts = counts;
  p.groups = groups;
  p.rows = static_cast<int32_t>(rows);
  p.red = static_cast<int32_t>(wide);
  p.n = static_cast<int32_t>(k);
  return launch_linear(p, kLinearDgrad, dtype,
                       linear_form(kLinearDgrad, groups, rows, 0, k, wide, flags),
                       as_stream(stream));
}

int32_t fgs_moe_linear_weight_grad(const void* dz, int64_t ldz, const void* x, int64_t ldx,
                                   const int32_t* counts, int32_t groups, int64_t rows,
                                   int64_t wide, int64_t k, int32_t dtype, int32_t flags,
                                   void* dw, void* stream) {
  int rc = check_linear(groups, rows, wide, k, dtype);
  if (rc) return rc;
  if (!linear_flags_ok(kLinearWgrad, flags)) return fail(FGS_EINVAL, "unknown flags");
  if (!counts && groups != 1) return fail(FGS_EINVAL, "counts are needed for several groups");
  if (!dw || (rows > 0 && (!dz || !x))) return fail(FGS_EINVAL, "null pointer argument");
  if ((rc = check_rows("dz", dz, rows, ldz)) || (rc = check_rows("x", x, rows, ldx)) ||
      (rc = check_rows("dw", dw, 0, 0)))
    return rc;
  if (misaligned(counts, 4)) return fail(FGS_EINVAL, "tensors must be aligned to their elements");
  LinearParams p{};
  p.q = dz;
  p.ldq = rows > 1 ? ldz : wide;
  p.p = x;
  p.ldp = rows > 1 ? ldx : k;
  p.out = dw;
  p.counts = counts;
  p.groups = groups;
  p.rows = static_cast<int32_t>(rows);
  p.m = static_cast<int32_t>(wide);
  p.n = static_cast<int32_t>(k);
  return launch_linear(p, kLinearWgrad, dtype,
                       linear_form(kLinearWgrad, groups, rows, wide, k, rows, flags),
                       as_stream(stream));
}

int64_t fgs_moe_linear_bias_grad_workspace_bytes(int32_t groups, int64_t rows, int64_t wide) {
  if (groups < 1 || rows < 0 || wide < 1 || groups > kMaxGroups || rows > kLinearMaxRows ||
      wide > kLinearMaxCols)
    return -1;
  const int64_t parts = linear_bias_parts(groups, rows, wide);
  return parts > 1 ? parts * groups * wide * 4 : 0;
}

int32_t fgs_moe_linear_bias_grad(const void* dz, int64_t ldz, const int32_t* counts,
                                 int32_t groups, int64_t rows, int64_t wide, int32_t dtype,
                                 void* workspace, int64_t ws_bytes, void* dbias, void* stream) {
  const bool with_rest = (dtype & FGS_DZ_REST) != 0;
  dtype &= ~FGS_DZ_REST;
  int rc = check_linear(groups, rows, wide, 8, dtype);
  if (rc) return rc;
  if (!counts && groups != 1) return fail(FGS_EINVAL, "counts are needed for several groups");
  if (!dbias || (rows > 0 && !dz)) return fail(FGS_EINVAL, "null pointer argument");
  if ((rc = check_rows("dz", dz, rows, ldz))) return rc;
  const int64_t need = fgs_moe_linear_bias_grad_workspace_bytes(groups, rows, wide);
  if (need > 0 && (!workspace || ws_bytes < need)) return fail(FGS_EINVAL, "workspace too small");
  if (misaligned(dbias, 2) || misaligned(counts, 4) || misaligned(workspace, 4))
    return fail(FGS_EINVAL, "tensors must be aligned to their elements");
  if (with_rest && rows > 1 && ldz != wide) return fail(FGS_EINVAL, "dz must be contiguous");
  LinearBiasGradParams p{};
  p.dz = dz;
  if (with_rest) p.rest = static_cast<const uint16_t*>(dz) + rows * wide;
  p.ldd = rows > 1 ? ldz : wide;
  p.counts = counts;
  p.groups = groups;
  p.rows = static_cast<int32_t>(rows);
  p.n = wide;
  p.part = static_cast<float*>(workspace);
  p.parts = linear_bias_parts(groups, rows, wide);
  p.out = dbias;
  return launch_linear_bias_grad(p, dtype, as_stream(stream));
}

int32_t fgs_moe_linear_schedule(int32_t pass, int32_t groups, int64_t rows, int64_t n, int64_t k,
                                int32_t gated, int32_t flags, char* buf, int32_t len) {
  if (pass < 0 || pass > 2) return fail(FGS_EINVAL, "pass must be 0, 1 or 2");
  const int64_t wide = gated ? 2 * n : n;
  int rc = check_linear(groups, rows, pass ? wide : n, k, FGS_DTYPE_BF16);
  if (rc || (rc = check_linear(groups, rows, wide, k, FGS_DTYPE_BF16))) return rc;
  if (!buf || len < 1) return fail(FGS_EINVAL, "buf must hold at least one byte");
  const int mode = pass == 1 ? kLinearDgrad : pass == 2 ? kLinearWgrad
                                                        : gated ? kLinearGated : kLinearForward;
  if (!linear_flags_ok(mode, flags)) return fail(FGS_EINVAL, "unknown flags");
  const int form = pass == 1   ? linear_form(mode, groups, rows, 0, k, wide, flags)
                   : pass == 2 ? linear_form(mode, groups, rows, wide, k, rows, flags)
                               : linear_form(mode, groups, rows, 0, n, k, flags);
  const std::string s = linear_form_name(mode, form);
  const size_t used = std::min(s.size(), static_cast<size_t>(len - 1));
  memcpy(buf, s.data(), used);
  buf[used] = 0;
  return FGS_OK;
}

}  // extern "C"
