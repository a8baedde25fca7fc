// C entry points of the causal mixer's operators: argument checks and launches.
#include <initializer_list>

#include "capi_util.h"
#include "shell_ops.h"

namespace {

using lsso::capi::aligned;
using lsso::capi::invalid;

size_t type_bytes(int type) { return type == LSSO_TYPE_FP32 ? 4 : 2; }

int check_decay_sizes(const char* who, int64_t B, int64_t N, int64_t H, int64_t DK, int64_t DV) {
  if (B <= 0 || N <= 0 || H <= 0) return invalid("%s: B, N and H must be positive", who);
  if (DK < 8 || DV < 8 || DK > 128 || DV > 128 || DK % 8 != 0 || DV % 8 != 0) {
    return invalid("%s: head widths must be multiples of 8 from 8 to 128, got %lld and %lld", who,
                   static_cast<long long>(DK), static_cast<long long>(DV));
  }
  if (H > (1 << 16) || B > (1 << 24) || B * H > (int64_t(1) << 24) || N > (int64_t(1) << 30)) {
    return invalid("%s: shape exceeds the supported launch range", who);
  }
  return LSSO_OK;
}

// Strides (elements) of [B, N, H, D] as tensor maps take them: the arrays start on 16 bytes and so does every row.
int check_tensor(const char* who, const char* name, const void* p, const int64_t* strides) {
  if (p == nullptr || strides == nullptr) return invalid("%s: a required pointer is NULL", who);
  bool good = aligned(p, 16);
  for (int i = 0; i < 3; ++i) good = good && strides[i] > 0 && strides[i] % 8 == 0 && strides[i] < (int64_t(1) << 38);
  if (!good) return invalid("%s: %s needs 16-byte alignment and positive strides that are multiples of 8 elements", who, name);
  return LSSO_OK;
}

lsso::TokenTensor tensor(const void* p, const int64_t* s) { return lsso::TokenTensor{p, s[0], s[1], s[2]}; }

}  // namespace

extern "C" {

size_t lsso_decay_workspace_size(int64_t B, int64_t N, int64_t H, int64_t DK, int64_t DV, int backward) {
  lsso::capi::clear_error();
  if (check_decay_sizes("lsso_decay", B, N, H, DK, DV) != LSSO_OK) return 0;
  int sms = 0;
  int* status = nullptr;
  if (lsso::capi::device(&sms, &status) != LSSO_OK) return 0;
  return lsso::decay_workspace(B, N, static_cast<int>(H), static_cast<int>(DK), static_cast<int>(DV), backward != 0, sms);
}

int lsso_decay_forward(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                       const int64_t* v_strides, int type, const float* log_decay, const uint8_t* mask, int64_t B,
                       int64_t N, int64_t H, int64_t DK, int64_t DV, float scale, const float* state, float* last,
                       void* y, const int64_t* y_strides, void* workspace, size_t workspace_bytes, void* stream) {
  lsso::capi::clear_error();
  const char* who = "lsso_decay_forward";
  int rc = check_decay_sizes(who, B, N, H, DK, DV);
  if (rc == LSSO_OK) rc = check_tensor(who, "q", q, q_strides);
  if (rc == LSSO_OK) rc = check_tensor(who, "k", k, k_strides);
  if (rc == LSSO_OK) rc = check_tensor(who, "v", v, v_strides);
  if (rc == LSSO_OK) rc = check_tensor(who, "y", y, y_strides);
  if (rc != LSSO_OK) return rc;
  if (log_decay == nullptr) return invalid("%s: a required pointer is NULL", who);
  if (type != LSSO_TYPE_BF16 && type != LSSO_TYPE_FP16) return invalid("%s: type must be BF16 or FP16", who);
  if (!aligned(log_decay, 4) || !aligned(state, 16) || !aligned(last, 16) || !aligned(workspace, 16)) {
    return invalid("%s: states and workspace must be 16-byte aligned", who);
  }
  int sms = 0;
  lsso::DecayCall c{};
  rc = lsso::capi::device(&sms, &c.status);
  if (rc != LSSO_OK) return rc;
  const size_t need = lsso::decay_workspace(B, N, static_cast<int>(H), static_cast<int>(DK), static_cast<int>(DV), false, sms);
  if (need > 16 && (workspace == nullptr || workspace_bytes < need)) {
    return lsso::capi::workspace_too_small(who, workspace == nullptr ? 0 : workspace_bytes, need);
  }
  c.q = tensor(q, q_strides);
  c.k = tensor(k, k_strides);
  c.v = tensor(v, v_strides);
  c.y = tensor(y, y_strides);
  c.log_decay = log_decay;
  c.mask = mask;
  c.state = state;
  c.last = last;
  c.batch = B;
  c.length = N;
  c.heads = static_cast<int>(H);
  c.key = static_cast<int>(DK);
  c.value = static_cast<int>(DV);
  c.type = type;
  c.scale = scale;
  return lsso::capi::launched(
      lsso::launch_decay_forward(c, static_cast<uint8_t*>(workspace), sms, static_cast<cudaStream_t>(stream)), who);
}

int lsso_decay_backward(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                        const int64_t* v_strides, const void* dy, const int64_t* dy_strides, int type,
                        const float* log_decay, const uint8_t* mask, int64_t B, int64_t N, int64_t H, int64_t DK,
                        int64_t DV, float scale, const float* state, const float* dlast, void* dq,
                        const int64_t* dq_strides, void* dk, const int64_t* dk_strides, void* dv,
                        const int64_t* dv_strides, float* dstate, void* workspace, size_t workspace_bytes,
                        void* stream) {
  lsso::capi::clear_error();
  const char* who = "lsso_decay_backward";
  int rc = check_decay_sizes(who, B, N, H, DK, DV);
  if (rc == LSSO_OK) rc = check_tensor(who, "q", q, q_strides);
  if (rc == LSSO_OK) rc = check_tensor(who, "k", k, k_strides);
  if (rc == LSSO_OK) rc = check_tensor(who, "v", v, v_strides);
  if (rc == LSSO_OK) rc = check_tensor(who, "dy", dy, dy_strides);
  if (rc == LSSO_OK) rc = check_tensor(who, "dq", dq, dq_strides);
  if (rc == LSSO_OK) rc = check_tensor(who, "dk", dk, dk_strides);
  if (rc == LSSO_OK) rc = check_tensor(who, "dv", dv, dv_strides);
  if (rc != LSSO_OK) return rc;
  if (log_decay == nullptr) return invalid("%s: a required pointer is NULL", who);
  if (type != LSSO_TYPE_BF16 && type != LSSO_TYPE_FP16) return invalid("%s: type must be BF16 or FP16", who);
  if (!aligned(log_decay, 4) || !aligned(state, 16) || !aligned(dlast, 16) || !aligned(dstate, 16) || !aligned(workspace, 16)) {
    return invalid("%s: states and workspace must be 16-byte aligned", who);
  }
  int sms = 0;
  lsso::DecayCall c{};
  rc = lsso::capi::device(&sms, &c.status);
  if (rc != LSSO_OK) return rc;
  const size_t need = lsso::decay_workspace(B, N, static_cast<int>(H), static_cast<int>(DK), static_cast<int>(DV), true, sms);
  if (need > 16 && (workspace == nullptr || workspace_bytes < need)) {
    return lsso::capi::workspace_too_small(who, workspace == nullptr ? 0 : workspace_bytes, need);
  }
  c.q = tensor(q, q_strides);
  c.k = tensor(k, k_strides);
  c.v = tensor(v, v_strides);
  c.y = tensor(dy, dy_strides);
  c.dq = tensor(dq, dq_strides);
  c.dk = tensor(dk, dk_strides);
  c.dv = tensor(dv, dv_strides);
  c.log_decay = log_decay;
  c.mask = mask;
  c.state = state;
  c.dlast = dlast;
  c.dstate = dstate;
  c.batch = B;
  c.length = N;
  c.heads = static_cast<int>(H);
  c.key = static_cast<int>(DK);
  c.value = static_cast<int>(DV);
  c.type = type;
  c.scale = scale;
  return lsso::capi::launched(
      lsso::launch_decay_backward(c, static_cast<uint8_t*>(workspace), sms, static_cast<cudaStream_t>(stream)), who);
}

int lsso_decay_step(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                    const int64_t* v_strides, int type, const float* log_decay, const uint8_t* active, int64_t B,
                    int64_t H, int64_t DK, int64_t DV, float scale, const float* state, float* new_state, void* y,
                    void* stream) {
  lsso::capi::clear_error();
  const char* who = "lsso_decay_step";
  int rc = check_decay_sizes(who, B, 1, H, DK, DV);
  if (rc != LSSO_OK) return rc;
  if (q == nullptr || k == nullptr || v == nullptr || q_strides == nullptr || k_strides == nullptr ||
      v_strides == nullptr || log_decay == nullptr || state == nullptr || new_state == nullptr || y == nullptr) {
    return invalid("%s: a required pointer is NULL", who);
  }
  if (type != LSSO_TYPE_BF16 && type != LSSO_TYPE_FP16 && type != LSSO_TYPE_FP32) return invalid("%s: unknown type", who);
  for (const void* p : {q, k, v, static_cast<const void*>(y)}) {
    if (!aligned(p, type_bytes(type))) return invalid("%s: an array is not aligned to its elements", who);
  }
  if (!aligned(log_decay, 4) || !aligned(state, 16) || !aligned(new_state, 16)) {
    return invalid("%s: states must be 16-byte aligned", who);
  }
  const int64_t bytes = B * H * DK * DV * 4;
  const uintptr_t from = reinterpret_cast<uintptr_t>(state), to = reinterpret_cast<uintptr_t>(new_state);
  if (from != to && from < to + bytes && to < from + bytes) return invalid("%s: new_state overlaps state in part", who);
  int sms = 0;
  int* status = nullptr;
  rc = lsso::capi::device(&sms, &status);
  if (rc != LSSO_OK) return rc;
  lsso::DecayStepCall c{};
  c.q = q;
  c.k = k;
  c.v = v;
  for (int i = 0; i < 2; ++i) {
    c.q_strides[i] = q_strides[i];
    c.k_strides[i] = k_strides[i];
    c.v_strides[i] = v_strides[i];
  }
  c.y = y;
  c.log_decay = log_decay;
  c.active = active;
  c.state = state;
  c.new_state = new_state;
  c.batch = B;
  c.heads = static_cast<int>(H);
  c.key = static_cast<int>(DK);
  c.value = static_cast<int>(DV);
  c.type = type;
  c.scale = scale;
  return lsso::capi::launched(lsso::launch_decay_step(c, static_cast<cudaStream_t>(stream)), who);
}

int lsso_rotary(const void* x, const int64_t* strides, int type, int64_t B, int64_t N, int64_t H, int64_t D,
                int64_t pairs, const void* frequencies, int frequencies_fp64, const void* positions, int position_type,
                int positions_batched, int interleaved, int backward, float magnitude, void* y, void* stream) {
  lsso::capi::clear_error();
  const char* who = "lsso_rotary";
  if (x == nullptr || strides == nullptr || y == nullptr || frequencies == nullptr) {
    return invalid("%s: a required pointer is NULL", who);
  }
  if (B <= 0 || N <= 0 || H <= 0 || D <= 0 || D % 2 != 0 || pairs <= 0 || 2 * pairs > D) {
    return invalid("%s: B, N and H must be positive, D even, and 2 * pairs in [2, D]", who);
  }
  if (pairs > 2048 || D > (1 << 16) || H > (1 << 16) || N > (int64_t(1) << 31) || B > (int64_t(1) << 31) / N) {
    return invalid("%s: shape exceeds the supported launch range", who);
  }
  if (type != LSSO_TYPE_BF16 && type != LSSO_TYPE_FP16 && type != LSSO_TYPE_FP32) return invalid("%s: unknown type", who);
  if (positions != nullptr && (position_type < LSSO_POSITION_INT64 || position_type > LSSO_POSITION_FP64)) {
    return invalid("%s: unknown position type", who);
  }
  const bool wide_position = position_type == LSSO_POSITION_INT64 || position_type == LSSO_POSITION_FP64;
  if (!aligned(x, 2 * type_bytes(type)) || !aligned(y, 2 * type_bytes(type)) ||
      !aligned(frequencies, frequencies_fp64 ? 8 : 4) || !aligned(positions, wide_position ? 8 : 4)) {
    return invalid("%s: x and y must be aligned to two elements, frequencies and positions to one", who);
  }
  for (int i = 0; i < 3; ++i) {
    if (strides[i] < 0 || strides[i] % 2 != 0) return invalid("%s: strides must be even and not negative", who);
  }
  int sms = 0;
  int* status = nullptr;
  const int rc = lsso::capi::device(&sms, &status);
  if (rc != LSSO_OK) return rc;
  lsso::RotaryCall c{};
  c.x = x;
  c.y = y;
  c.batch = B;
  c.length = N;
  c.stride_batch = strides[0];
  c.stride_token = strides[1];
  c.stride_head = strides[2];
  c.heads = static_cast<int>(H);
  c.dim = static_cast<int>(D);
  c.pairs = static_cast<int>(pairs);
  c.frequencies = frequencies;
  c.frequency64 = frequencies_fp64 != 0 ? 1 : 0;
  c.positions = positions;
  c.position_type = position_type;
  c.positions_batched = positions_batched != 0 ? 1 : 0;
  c.interleaved = interleaved != 0 ? 1 : 0;
  c.backward = backward != 0 ? 1 : 0;
  c.magnitude = magnitude;
  c.type = type;
  return lsso::capi::launched(lsso::launch_rotary(c, sms, static_cast<cudaStream_t>(stream)), who);
}

}  // extern "C"
