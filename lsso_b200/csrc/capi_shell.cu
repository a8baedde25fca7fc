// C entry points of the token shell's operators: argument checks and launches.
#include <cmath>
#include <initializer_list>

#include "capi_util.h"
#include "ffn.h"
#include "shell_ops.h"

namespace {

using lsso::capi::aligned;
using lsso::capi::invalid;

constexpr int64_t kMostRows = int64_t(1) << 30;

bool is_16bit(int type) { return type == LSSO_TYPE_BF16 || type == LSSO_TYPE_FP16; }
bool is_type(int type) { return is_16bit(type) || type == LSSO_TYPE_FP32; }
size_t type_bytes(int type) { return type == LSSO_TYPE_FP32 ? 4 : 2; }

int check_ffn_sizes(const char* who, int64_t T, int64_t D, int64_t H) {
  if (T <= 0 || D <= 0 || H <= 0 || D % 8 != 0 || H % 8 != 0) {
    return invalid("%s: T must be positive, D and H positive multiples of 8", who);
  }
  if (T > kMostRows || D > (1 << 20) || H > (1 << 20)) return invalid("%s: shape exceeds the supported launch range", who);
  return LSSO_OK;
}

int check_embedding(const char* who, int64_t T, int64_t V, int64_t D) {
  if (T <= 0 || V <= 0 || D <= 0) return invalid("%s: T, V and D must be positive", who);
  if (T > kMostRows || V > kMostRows || D > (1 << 20)) return invalid("%s: shape exceeds the supported launch range", who);
  return LSSO_OK;
}

int check_dropout(const char* who, int branch_type, int out_type, int64_t rows, int64_t width, double p,
                  const void* state) {
  if (state == nullptr) return invalid("%s: a required pointer is NULL", who);
  if (!is_type(branch_type) || (out_type != branch_type && out_type != LSSO_TYPE_FP32)) {
    return invalid("%s: out_type must be branch_type or FP32", who);
  }
  if (rows <= 0 || width <= 0 || rows > (int64_t(1) << 40) || width > (int64_t(1) << 31) ||
      rows > (int64_t(1) << 46) / width) {
    return invalid("%s: rows and width must be positive and within the supported range", who);
  }
  if (!(p >= 0.0 && p <= 1.0)) return invalid("%s: p must be in [0, 1], got %g", who, p);
  return LSSO_OK;
}

void set_rate(lsso::DropoutCall* c, double p) {
  const double threshold = std::nearbyint(p * 4294967296.0);
  c->drop_all = threshold >= 4294967296.0 ? 1 : 0;
  c->threshold = c->drop_all ? 1u : static_cast<uint32_t>(threshold);  // p = 1: the kernel's words are zero
  c->scale = c->drop_all ? 0.0f : static_cast<float>(1.0 / (1.0 - p));
}

int ffn_backward(const char* who, const void* dy, const void* x, const void* kept, const void* h, const void* w_in,
                 const void* w_out, int type, int64_t T, int64_t D, int64_t H, int activation, int grad_type,
                 int bias_grad_type, void* dx, void* dw_in, void* dw_out, void* db_in, void* db_out, void* workspace,
                 size_t workspace_bytes, void* stream) {
  lsso::capi::clear_error();
  if (dy == nullptr || x == nullptr || kept == nullptr || h == nullptr || w_in == nullptr || w_out == nullptr ||
      workspace == nullptr) {
    return invalid("%s: a required pointer is NULL", who);
  }
  int rc = check_ffn_sizes(who, T, D, H);
  if (rc != LSSO_OK) return rc;
  if (!is_16bit(type) || !is_type(grad_type) || !is_type(bias_grad_type)) return invalid("%s: unknown type", who);
  if (activation != LSSO_FFN_SILU && activation != LSSO_FFN_GELU) return invalid("%s: unknown activation", who);
  for (const void* p : {dy, x, kept, h, w_in, w_out, static_cast<const void*>(dx), static_cast<const void*>(dw_in),
                        static_cast<const void*>(dw_out), static_cast<const void*>(db_in),
                        static_cast<const void*>(db_out), static_cast<const void*>(workspace)}) {
    if (!aligned(p, 16)) return invalid("%s: every array must be 16-byte aligned", who);
  }
  int sms = 0;
  int* status = nullptr;
  rc = lsso::capi::device(&sms, &status);
  if (rc != LSSO_OK) return rc;
  const size_t need = lsso::ffn_backward_workspace(T, D, H, sms);
  if (workspace_bytes < need) return lsso::capi::workspace_too_small(who, workspace_bytes, need);
  const lsso::FfnBackwardCall c{dy, x,  kept,  h,      w_in,  w_out, T, D, H, type, activation, grad_type, bias_grad_type,
                                dx, dw_in, dw_out, db_in, db_out, static_cast<uint8_t*>(workspace), status};
  return lsso::capi::launched(lsso::launch_ffn_backward(c, sms, static_cast<cudaStream_t>(stream)), who);
}

}  // namespace

extern "C" {

int lsso_ffn_streams_weights(int64_t T, int64_t D, int64_t H) {
  return T > 0 && D > 0 && H > 0 && lsso::ffn_streams_weights(T, D, H, true) ? 1 : 0;
}

int lsso_ffn_forward(const void* x, int type, int64_t T, int64_t D, int64_t H, const void* w_in, const void* w_out,
                     int weight_type, const void* b_in, const void* b_out, int bias_type, int activation, void* kept,
                     void* h, void* y, void* stream) {
  lsso::capi::clear_error();
  const char* who = "lsso_ffn_forward";
  if (x == nullptr || w_in == nullptr || w_out == nullptr || h == nullptr || y == nullptr) {
    return invalid("%s: a required pointer is NULL", who);
  }
  int rc = check_ffn_sizes(who, T, D, H);
  if (rc != LSSO_OK) return rc;
  if (!is_16bit(type)) return invalid("%s: type must be BF16 or FP16", who);
  if (weight_type != type &&
      !(weight_type == LSSO_TYPE_FP32 && kept == nullptr && lsso::ffn_streams_weights(T, D, H, true))) {
    return invalid("%s: the weights must have x's type (FP32 only where lsso_ffn_streams_weights says so)", who);
  }
  if ((b_in != nullptr || b_out != nullptr) && !is_type(bias_type)) return invalid("%s: unknown bias type", who);
  if (activation != LSSO_FFN_SILU && activation != LSSO_FFN_GELU) return invalid("%s: unknown activation", who);
  if (!aligned(x, 16) || !aligned(w_in, 16) || !aligned(w_out, 16) || !aligned(kept, 16) || !aligned(h, 16) ||
      !aligned(y, 16)) {
    return invalid("%s: matrices must be 16-byte aligned", who);
  }
  int sms = 0;
  int* status = nullptr;
  rc = lsso::capi::device(&sms, &status);
  if (rc != LSSO_OK) return rc;
  const lsso::FfnForwardCall c{x,           w_in,      w_out,      b_in, b_out, T, D, H,     type,
                               weight_type, bias_type, activation, kept, h,     y, status};
  return lsso::capi::launched(lsso::launch_ffn_forward(c, sms, static_cast<cudaStream_t>(stream)), who);
}

size_t lsso_ffn_backward_workspace_size(int64_t T, int64_t D, int64_t H) {
  lsso::capi::clear_error();
  if (check_ffn_sizes("lsso_ffn_backward", T, D, H) != LSSO_OK) return 0;
  int sms = 0;
  int* status = nullptr;
  if (lsso::capi::device(&sms, &status) != LSSO_OK) return 0;
  return lsso::ffn_backward_workspace(T, D, H, sms);
}

int lsso_ffn_backward(const void* dy, const void* x, const void* kept, const void* h, const void* w_in,
                      const void* w_out, int type, int64_t T, int64_t D, int64_t H, int activation, int grad_type,
                      void* dx, void* dw_in, void* dw_out, void* db_in, void* db_out, void* workspace,
                      size_t workspace_bytes, void* stream) {
  return ffn_backward("lsso_ffn_backward", dy, x, kept, h, w_in, w_out, type, T, D, H, activation, grad_type, grad_type,
                      dx, dw_in, dw_out, db_in, db_out, workspace, workspace_bytes, stream);
}

int lsso_ffn_backward_mixed(const void* dy, const void* x, const void* kept, const void* h, const void* w_in,
                            const void* w_out, int type, int64_t T, int64_t D, int64_t H, int activation,
                            int grad_type, int bias_grad_type, void* dx, void* dw_in, void* dw_out, void* db_in,
                            void* db_out, void* workspace, size_t workspace_bytes, void* stream) {
  return ffn_backward("lsso_ffn_backward_mixed", dy, x, kept, h, w_in, w_out, type, T, D, H, activation, grad_type,
                      bias_grad_type, dx, dw_in, dw_out, db_in, db_out, workspace, workspace_bytes, stream);
}

int lsso_ffn_cast(const float* w_in, void* w_in_out, int64_t w_in_count, const float* w_out, void* w_out_out,
                  int64_t w_out_count, int type, void* stream) {
  lsso::capi::clear_error();
  const char* who = "lsso_ffn_cast";
  if (w_in == nullptr || w_in_out == nullptr || w_out == nullptr || w_out_out == nullptr) {
    return invalid("%s: a required pointer is NULL", who);
  }
  if (w_in_count <= 0 || w_out_count <= 0 || w_in_count % 8 != 0 || w_out_count % 8 != 0) {
    return invalid("%s: counts must be positive multiples of 8", who);
  }
  if (!is_16bit(type)) return invalid("%s: type must be BF16 or FP16", who);
  if (!aligned(w_in, 16) || !aligned(w_in_out, 16) || !aligned(w_out, 16) || !aligned(w_out_out, 16)) {
    return invalid("%s: every array must be 16-byte aligned", who);
  }
  int sms = 0;
  int* status = nullptr;
  const int rc = lsso::capi::device(&sms, &status);
  if (rc != LSSO_OK) return rc;
  const float* const src[2] = {w_in, w_out};
  void* const dst[2] = {w_in_out, w_out_out};
  const int64_t count[2] = {w_in_count, w_out_count};
  return lsso::capi::launched(lsso::launch_ffn_cast(src, dst, count, type, sms, static_cast<cudaStream_t>(stream)), who);
}

int lsso_embedding_forward(const void* ids, int ids_int64, const uint8_t* row_mask, int64_t T, const void* weight,
                           int weight_type, int64_t V, int64_t D, float scale, void* y, int out_type, void* stream) {
  lsso::capi::clear_error();
  const char* who = "lsso_embedding_forward";
  if (ids == nullptr || weight == nullptr || y == nullptr) return invalid("%s: a required pointer is NULL", who);
  int rc = check_embedding(who, T, V, D);
  if (rc != LSSO_OK) return rc;
  if (!is_type(weight_type) || !is_type(out_type)) return invalid("%s: unknown type", who);
  if (!aligned(ids, ids_int64 ? 8 : 4) || !aligned(weight, type_bytes(weight_type)) || !aligned(y, type_bytes(out_type))) {
    return invalid("%s: an array is not aligned to its elements", who);
  }
  int sms = 0;
  int* status = nullptr;
  rc = lsso::capi::device(&sms, &status);
  if (rc != LSSO_OK) return rc;
  lsso::EmbeddingCall c{};
  c.ids = ids;
  c.ids64 = ids_int64 != 0 ? 1 : 0;
  c.weight = weight;
  c.out = y;
  c.row_mask = row_mask;
  c.tokens = T;
  c.vocab = V;
  c.width = D;
  c.padding = -1;
  c.scale = scale;
  c.weight_type = weight_type;
  c.out_type = out_type;
  c.status = status;
  return lsso::capi::launched(lsso::launch_embedding_forward(c, sms, static_cast<cudaStream_t>(stream)), who);
}

size_t lsso_embedding_backward_workspace_size(int64_t T, int64_t V, int64_t D) {
  lsso::capi::clear_error();
  if (check_embedding("lsso_embedding_backward", T, V, D) != LSSO_OK) return 0;
  int sms = 0;
  int* status = nullptr;
  if (lsso::capi::device(&sms, &status) != LSSO_OK) return 0;
  return lsso::make_embedding_grad_plan(T, V, D, sms).total;
}

int lsso_embedding_backward(const void* ids, int ids_int64, const uint8_t* row_mask, int64_t T, const void* dy,
                            int dy_type, int64_t V, int64_t D, int64_t padding, float scale, void* dweight,
                            int weight_type, void* workspace, size_t workspace_bytes, void* stream) {
  lsso::capi::clear_error();
  const char* who = "lsso_embedding_backward";
  if (ids == nullptr || dy == nullptr || dweight == nullptr || workspace == nullptr) {
    return invalid("%s: a required pointer is NULL", who);
  }
  int rc = check_embedding(who, T, V, D);
  if (rc != LSSO_OK) return rc;
  if (!is_type(weight_type) || !is_type(dy_type)) return invalid("%s: unknown type", who);
  if (padding < -1 || padding >= V) return invalid("%s: padding must be -1 or a row of the table", who);
  if (!aligned(ids, ids_int64 ? 8 : 4) || !aligned(dy, type_bytes(dy_type))) {
    return invalid("%s: an array is not aligned to its elements", who);
  }
  if (!aligned(dweight, 16) || !aligned(workspace, 16)) {
    return invalid("%s: dweight and workspace must be 16-byte aligned", who);
  }
  int sms = 0;
  int* status = nullptr;
  rc = lsso::capi::device(&sms, &status);
  if (rc != LSSO_OK) return rc;
  const lsso::EmbeddingGradPlan plan = lsso::make_embedding_grad_plan(T, V, D, sms);
  if (workspace_bytes < plan.total) return lsso::capi::workspace_too_small(who, workspace_bytes, plan.total);
  lsso::EmbeddingCall c{};
  c.ids = ids;
  c.ids64 = ids_int64 != 0 ? 1 : 0;
  c.grad = dy;
  c.out = dweight;
  c.row_mask = row_mask;
  c.tokens = T;
  c.vocab = V;
  c.width = D;
  c.padding = padding;
  c.scale = scale;
  c.weight_type = weight_type;
  c.out_type = dy_type;
  c.status = status;
  return lsso::capi::launched(lsso::launch_embedding_backward(plan, c, static_cast<uint8_t*>(workspace), sms,
                                                              static_cast<cudaStream_t>(stream)),
                              who);
}

int lsso_dropout_forward(const void* branch, int branch_type, const void* residual, int out_type,
                         const uint8_t* row_mask, int64_t rows, int64_t width, double p, const int64_t* state,
                         uint32_t site, int64_t* used_state, void* y, void* stream) {
  lsso::capi::clear_error();
  const char* who = "lsso_dropout_forward";
  if (branch == nullptr || y == nullptr) return invalid("%s: a required pointer is NULL", who);
  int rc = check_dropout(who, branch_type, out_type, rows, width, p, state);
  if (rc != LSSO_OK) return rc;
  if (!aligned(branch, type_bytes(branch_type)) || !aligned(residual, type_bytes(out_type)) ||
      !aligned(y, type_bytes(out_type)) || !aligned(state, 8) || !aligned(used_state, 8)) {
    return invalid("%s: an array is not aligned to its elements", who);
  }
  int sms = 0;
  int* status = nullptr;
  rc = lsso::capi::device(&sms, &status);
  if (rc != LSSO_OK) return rc;
  lsso::DropoutCall c{};
  c.in = branch;
  c.residual = residual;
  c.out = y;
  c.row_mask = row_mask;
  c.state = state;
  c.used_state = used_state;
  c.rows = rows;
  c.width = width;
  c.site = site;
  c.branch_type = branch_type;
  c.out_type = out_type;
  set_rate(&c, p);
  return lsso::capi::launched(lsso::launch_dropout_forward(c, sms, static_cast<cudaStream_t>(stream)), who);
}

int lsso_dropout_backward(const void* dy, int out_type, int branch_type, const uint8_t* row_mask, int64_t rows,
                          int64_t width, double p, const int64_t* state, uint32_t site, void* dbranch,
                          void* dresidual, void* stream) {
  lsso::capi::clear_error();
  const char* who = "lsso_dropout_backward";
  if (dy == nullptr || (dbranch == nullptr && dresidual == nullptr)) {
    return invalid("%s: a required pointer is NULL", who);
  }
  int rc = check_dropout(who, branch_type, out_type, rows, width, p, state);
  if (rc != LSSO_OK) return rc;
  if (!aligned(dy, type_bytes(out_type)) || !aligned(dbranch, type_bytes(branch_type)) ||
      !aligned(dresidual, type_bytes(out_type)) || !aligned(state, 8)) {
    return invalid("%s: an array is not aligned to its elements", who);
  }
  int sms = 0;
  int* status = nullptr;
  rc = lsso::capi::device(&sms, &status);
  if (rc != LSSO_OK) return rc;
  lsso::DropoutCall c{};
  c.in = dy;
  c.out = dbranch;
  c.residual_grad = dresidual;
  c.row_mask = row_mask;
  c.state = state;
  c.rows = rows;
  c.width = width;
  c.site = site;
  c.branch_type = branch_type;
  c.out_type = out_type;
  set_rate(&c, p);
  return lsso::capi::launched(lsso::launch_dropout_backward(c, sms, static_cast<cudaStream_t>(stream)), who);
}

}  // extern "C"
