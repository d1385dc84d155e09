// C ABI of the label operators (declared in include/euclid_b200.h): argument checks, then
// the launches of k_scores.cu, k_groups.cu and k_codebook.cu.
#include "engine.h"
#include "../../include/euclid_b200.h"

#include <cmath>
#include <string>

namespace euc {

constexpr int64_t kMaxIndex = 0x7ffffffell;  // sorted positions, slots and labels are int32
constexpr int64_t kMaxScores = 1ll << 30;    // a row's elements and vectors are counted in int32,
constexpr int64_t kMaxDim = 1ll << 30;       // in every operator
constexpr int kMaxTop = 32;

static int done(cudaError_t e, const char* where) {
  if (e == cudaSuccess) return EUC_OK;
  return set_error(EUC_ERR_LAUNCH, (std::string(where) + ": " + cudaGetErrorString(e)).c_str());
}

static int type_size(int t) { return t == EUC_ROW_F64 ? 8 : t == EUC_ROW_F32 ? 4 : 2; }

static int bad_type(int t) {
  return t < EUC_ROW_F32 || t > EUC_ROW_BF16 ? set_error(EUC_ERR_DTYPE, "unknown row type") : EUC_OK;
}

static int no_device() {
  return device_is_sm100() ? EUC_OK : set_error(EUC_ERR_DEVICE, "euclid_b200 requires an sm_100 (B200) device");
}

static int rows_shape(int64_t n, int64_t p, int64_t dim) {
  if (n < 0 || p < 0 || dim < 0) return set_error(EUC_ERR_SHAPE, "negative size");
  if (n > kMaxIndex || p > kMaxIndex || (p > 0 && n > kMaxIndex / p)) return set_error(EUC_ERR_SHAPE, "too many slots");
  if (dim > kMaxDim) return set_error(EUC_ERR_SHAPE, "dim too large");
  return EUC_OK;
}

using Pointers = std::initializer_list<const void*>;

// whether a pointer is off its elements: rows of the row type, fp32 or fp64 values, int32
// indexes, labels of either type
static bool off(size_t bytes, Pointers ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % bytes) return true;
  return false;
}
static bool misaligned(int t, Pointers rows, Pointers values, Pointers indexes, const void* labels, bool labels_i64) {
  return off(type_size(t), rows) || off(t == EUC_ROW_F64 ? 8 : 4, values) || off(4, indexes) ||
         off(labels_i64 ? 8 : 4, {labels});
}

static int scores_shape(int row_type, int64_t ld, int64_t n, int64_t m, double scale) {
  if (n < 0 || n > kMaxIndex || m < 1 || m > kMaxScores) return set_error(EUC_ERR_SHAPE, "scores: bad size");
  if (ld < m && n > 1) return set_error(EUC_ERR_SHAPE, "scores: row stride below the row's length");
  if (!std::isfinite(scale) || scale == 0.0) return set_error(EUC_ERR_ARG, "scale must be finite and not 0");
  // the arithmetic holds |scale|, twice it and its multiple of log2(e) as normal numbers; scores
  // with the exponents of fp32 or fp64 may differ by more than their type holds, by 2^128 or
  // 2^1024, and times |scale| that is 256 or 1024 at least: exp of minus that is 0
  const double least = row_type == EUC_ROW_F64 ? 0x1p-1014 : row_type == EUC_ROW_F16 ? 0x1p-126 : 0x1p-120;
  const double most = row_type == EUC_ROW_F64 ? 0x1p1022 : 0x1p126;
  if (!(std::fabs(scale) >= least && std::fabs(scale) <= most))
    return set_error(EUC_ERR_ARG, "scale is outside the range of the scores' type");
  return EUC_OK;
}

}  // namespace euc

using namespace euc;

extern "C" {

int euc_label_log_probs(int row_type, const void* scores, int64_t ld, int64_t n, int64_t m, const void* labels,
                        int labels_are_i64, double scale, int top, void* log_probs, void* entropy, void* row_stats,
                        void* top_log_probs, int64_t* top_labels, void* stream) {
  if (int rc = bad_type(row_type)) return rc;
  if (int rc = scores_shape(row_type, ld, n, m, scale)) return rc;
  if (top < 0 || top > kMaxTop || top > m) return set_error(EUC_ERR_UNSUPPORTED, "top must be in [0, min(m, 32)]");
  if (int rc = no_device()) return rc;
  if (n == 0) return EUC_OK;
  if (!scores || (log_probs && !labels) || (top > 0 && (!top_log_probs || !top_labels)))
    return set_error(EUC_ERR_ARG, "null pointer");
  if (misaligned(row_type, {scores}, {log_probs, entropy, row_stats, top_log_probs}, {}, labels, labels_are_i64 != 0) ||
      off(8, {top_labels}))
    return set_error(EUC_ERR_ARG, "misaligned pointer");
  ScoreJob j{};
  j.x = scores;
  j.ld = ld;
  j.n = n;
  j.m = m;
  j.labels = labels;
  j.labels_i64 = labels_are_i64 != 0;
  j.scale = scale;
  j.top = top;
  j.log_probs = log_probs;
  j.entropy = entropy;
  j.stats = row_stats;
  j.top_log_probs = top_log_probs;
  j.top_labels = top_labels;
  return done(launch_label_log_probs(static_cast<RowType>(row_type), j, static_cast<cudaStream_t>(stream)),
              "label_log_probs");
}

int euc_label_log_probs_grad(int row_type, const void* scores, int64_t ld, int64_t n, int64_t m, const void* labels,
                             int labels_are_i64, double scale, const void* row_stats, const void* grad_log_probs,
                             const void* grad_entropy, void* grad, void* stream) {
  if (int rc = bad_type(row_type)) return rc;
  if (int rc = scores_shape(row_type, ld, n, m, scale)) return rc;
  if (int rc = no_device()) return rc;
  if (n == 0) return EUC_OK;
  if (!scores || !row_stats || !grad || (grad_log_probs && !labels)) return set_error(EUC_ERR_ARG, "null pointer");
  if (misaligned(row_type, {scores, grad}, {row_stats, grad_log_probs, grad_entropy}, {}, labels, labels_are_i64 != 0))
    return set_error(EUC_ERR_ARG, "misaligned pointer");
  ScoreGradJob j{};
  j.x = scores;
  j.ld = ld;
  j.n = n;
  j.m = m;
  j.labels = labels;
  j.labels_i64 = labels_are_i64 != 0;
  j.scale = scale;
  j.stats = row_stats;
  j.g_log_probs = grad_log_probs;
  j.g_entropy = grad_entropy;
  j.grad = grad;
  return done(launch_label_log_probs_grad(static_cast<RowType>(row_type), j, static_cast<cudaStream_t>(stream)),
              "label_log_probs_grad");
}

size_t euc_group_rows_workspace_bytes(int64_t slots, int64_t k) {
  if (slots <= 0 || k < 0 || slots > kMaxIndex || k > kMaxIndex) return 0;
  return group_ws_bytes(slots, k);
}

int euc_group_rows(const void* labels, int labels_are_i64, int64_t slots, int64_t k, int32_t* offsets, int32_t* order,
                   int32_t* position, int32_t* sorted_labels, void* ws, size_t ws_bytes, void* stream) {
  if (slots < 0 || k < 0) return set_error(EUC_ERR_SHAPE, "negative size");
  if (slots > kMaxIndex || k > kMaxIndex) return set_error(EUC_ERR_SHAPE, "too many slots or labels");
  if (int rc = no_device()) return rc;
  if (!offsets || (slots > 0 && (!labels || !order || !position || !sorted_labels)))
    return set_error(EUC_ERR_ARG, "null pointer");
  if (misaligned(EUC_ROW_F32, {}, {}, {offsets, order, position, sorted_labels}, labels, labels_are_i64 != 0))
    return set_error(EUC_ERR_ARG, "misaligned pointer");
  const size_t need = group_ws_bytes(slots, k);
  if (need > 0 && (!ws || ws_bytes < need))
    return set_error(EUC_ERR_WORKSPACE,
                     ("group_rows: workspace of " + std::to_string(need) + " bytes required").c_str());
  if (need > 0 && off(16, {ws}))
    return set_error(EUC_ERR_ARG, "group_rows: the workspace must start on a 16-byte boundary");
  return done(launch_group_rows(labels, labels_are_i64 != 0, slots, k, offsets, order, position, sorted_labels, ws,
                                static_cast<cudaStream_t>(stream)),
              "group_rows");
}

int euc_rows_to_groups(int row_type, const void* X, const int32_t* position, const int32_t* kept, int64_t n, int64_t p,
                       int64_t dim, void* Y, void* stream) {
  if (int rc = bad_type(row_type)) return rc;
  if (int rc = rows_shape(n, p, dim)) return rc;
  if (int rc = no_device()) return rc;
  if (n == 0 || p == 0 || dim == 0) return EUC_OK;
  if (!X || !position || !kept || !Y) return set_error(EUC_ERR_ARG, "null pointer");
  if (misaligned(row_type, {X, Y}, {}, {position, kept}, nullptr, false))
    return set_error(EUC_ERR_ARG, "misaligned pointer");
  return done(launch_rows_to_groups(type_size(row_type), X, position, kept, n, static_cast<int>(p), dim, Y,
                                    static_cast<cudaStream_t>(stream)),
              "rows_to_groups");
}

int euc_rows_from_groups(int row_type, const void* Y, const int32_t* position, const void* weights, int64_t n, int64_t p,
                         int64_t dim, void* out, void* stream) {
  if (int rc = bad_type(row_type)) return rc;
  if (int rc = rows_shape(n, p, dim)) return rc;
  if (int rc = no_device()) return rc;
  if (n == 0 || dim == 0) return EUC_OK;
  if (!out || (p > 0 && (!Y || !position))) return set_error(EUC_ERR_ARG, "null pointer");
  if (misaligned(row_type, {Y, out}, {weights}, {position}, nullptr, false))
    return set_error(EUC_ERR_ARG, "misaligned pointer");
  return done(launch_rows_from_groups(static_cast<RowType>(row_type), Y, position, weights, n, static_cast<int>(p), dim,
                                      out, static_cast<cudaStream_t>(stream)),
              "rows_from_groups");
}

int euc_rows_from_groups_grad(int row_type, const void* grad_out, const void* Y, const int32_t* position,
                              const void* weights, const int32_t* kept, int64_t n, int64_t p, int64_t dim, void* grad_Y,
                              void* grad_weights, void* stream) {
  if (int rc = bad_type(row_type)) return rc;
  if (int rc = rows_shape(n, p, dim)) return rc;
  if (int rc = no_device()) return rc;
  if (n == 0 || p == 0 || (!grad_Y && !grad_weights)) return EUC_OK;
  if (!position || !kept || (dim > 0 && (!grad_out || (grad_weights && !Y))))
    return set_error(EUC_ERR_ARG, "null pointer");
  if (misaligned(row_type, {grad_out, Y, grad_Y}, {weights, grad_weights}, {position, kept}, nullptr, false))
    return set_error(EUC_ERR_ARG, "misaligned pointer");
  if (dim == 0) {  // empty products
    if (!grad_weights) return EUC_OK;
    return done(cudaMemsetAsync(grad_weights, 0, static_cast<size_t>(n) * p * (row_type == EUC_ROW_F64 ? 8 : 4),
                                static_cast<cudaStream_t>(stream)),
                "rows_from_groups_grad");
  }
  return done(launch_rows_from_groups_grad(static_cast<RowType>(row_type), grad_out, Y, position, weights, kept, n,
                                           static_cast<int>(p), dim, grad_Y, grad_weights,
                                           static_cast<cudaStream_t>(stream)),
              "rows_from_groups_grad");
}

int euc_codebook_lookup(int row_type, const void* C, int64_t k, const void* labels, int labels_are_i64, int64_t n,
                        int64_t dim, double scale, void* out, void* stream) {
  if (int rc = bad_type(row_type)) return rc;
  if (n < 0 || k < 0 || dim < 0) return set_error(EUC_ERR_SHAPE, "negative size");
  if (dim > kMaxDim || (dim > 0 && n > (int64_t(1) << 62) / dim)) return set_error(EUC_ERR_SHAPE, "shape too large");
  if (int rc = no_device()) return rc;
  if (n == 0 || dim == 0) return EUC_OK;
  if (!labels || !out || (k > 0 && !C)) return set_error(EUC_ERR_ARG, "null pointer");
  if (misaligned(row_type, {C, out}, {}, {}, labels, labels_are_i64 != 0))
    return set_error(EUC_ERR_ARG, "misaligned pointer");
  return done(launch_codebook_lookup(static_cast<RowType>(row_type), C, k, labels, labels_are_i64 != 0, n, dim, scale,
                                     out, static_cast<cudaStream_t>(stream)),
              "codebook_lookup");
}

size_t euc_codebook_grad_workspace_bytes(int row_type, int64_t n, int64_t dim) {
  if (row_type < EUC_ROW_F32 || row_type > EUC_ROW_BF16 || n <= 0 || dim <= 0) return 0;
  return codebook_grad_ws_bytes(static_cast<RowType>(row_type), n, dim);
}

int euc_codebook_grad(int row_type, const void* grad_out, const int32_t* offsets, const int32_t* order,
                      const int32_t* sorted_labels, int64_t n, int64_t k, int64_t dim, double scale, void* grad_C,
                      void* ws, size_t ws_bytes, void* stream) {
  if (int rc = bad_type(row_type)) return rc;
  if (int rc = rows_shape(n, 1, dim)) return rc;
  if (k < 0 || k > kMaxIndex) return set_error(EUC_ERR_SHAPE, "bad number of labels");
  if (int rc = no_device()) return rc;
  if (k == 0 || dim == 0) return EUC_OK;
  if (!offsets || !grad_C || (n > 0 && (!grad_out || !order || !sorted_labels)))
    return set_error(EUC_ERR_ARG, "null pointer");
  if (misaligned(row_type, {grad_out, grad_C}, {ws}, {offsets, order, sorted_labels}, nullptr, false))
    return set_error(EUC_ERR_ARG, "misaligned pointer");
  const size_t need = euc_codebook_grad_workspace_bytes(row_type, n, dim);
  if (need > 0 && (!ws || ws_bytes < need))
    return set_error(EUC_ERR_WORKSPACE,
                     ("codebook_grad: workspace of " + std::to_string(need) + " bytes required").c_str());
  return done(launch_codebook_grad(static_cast<RowType>(row_type), grad_out, offsets, order, sorted_labels, n, k, dim,
                                   scale, grad_C, ws, static_cast<cudaStream_t>(stream)),
              "codebook_grad");
}

}  // extern "C"
