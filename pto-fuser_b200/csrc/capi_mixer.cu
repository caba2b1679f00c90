// C entry points of the operators around a recurrent token mixer: argument validation and
// dispatch. Nothing here allocates, synchronises or touches the device before a launch.
#include "capi_internal.h"

namespace ptof {
namespace {

bool dtype_ok(int d) { return d == PTOF_F32 || d == PTOF_F16 || d == PTOF_BF16; }
bool own_or_f32(int d, int dtype) { return d == dtype || d == PTOF_F32; }
bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
// token indexes are 32-bit and run a few tiles past the last token
constexpr int kMaxTokens = 0x7fffffff - 4096;
// as are channel indexes, past the last block of channels
constexpr int kMaxChannels = 1 << 30;
int elem_bytes(int d) { return d == PTOF_F32 ? 4 : 2; }

struct Ptr {
  const void* p;
  const char* name;
  int bytes;      // element alignment
  bool required;
};
int check_tensors(const char* what, std::initializer_list<Ptr> ptrs) {
  for (const Ptr& q : ptrs) {
    if (!q.p && q.required) return fail(PTOF_EINVAL, "%s: %s is NULL", what, q.name);
    if (!aligned(q.p, q.bytes))
      return fail(PTOF_EALIGN, "%s: %s not aligned to its elements", what, q.name);
  }
  return PTOF_OK;
}
int check_strides(const char* what, std::initializer_list<int64_t> strides) {
  for (int64_t s : strides)
    if (s < 0) return fail(PTOF_EINVAL, "%s: negative stride", what);
  return PTOF_OK;
}

int validate(const ptof_ssm_scan_params* p) {
  if (!p) return fail(PTOF_EINVAL, "ssm_scan: null params");
  if (p->N < 0 || p->T < 0 || p->D < 1 || p->D > kMaxChannels || p->G < 1 || p->D % p->G)
    return fail(PTOF_EINVAL, "ssm_scan: N=%d T=%d D=%d G=%d (D a multiple of G)", p->N, p->T, p->D,
                p->G);
  if (p->T > kMaxTokens) return fail(PTOF_EUNSUPPORTED, "ssm_scan: T=%d tokens", p->T);
  if (p->n < 1 || p->n > 128) return fail(PTOF_EUNSUPPORTED, "ssm_scan: n=%d (1 to 128 states)", p->n);
  if (!dtype_ok(p->dtype)) return fail(PTOF_EINVAL, "ssm_scan: bad dtype code");
  if (p->max_len < 0) return fail(PTOF_EINVAL, "ssm_scan: max_len=%d", p->max_len);
  return check_strides("ssm_scan",
                       {p->x_batch_stride, p->x_token_stride, p->dt_batch_stride,
                        p->dt_token_stride, p->z_batch_stride, p->z_token_stride,
                        p->y_batch_stride, p->y_token_stride, p->B_batch_stride,
                        p->B_token_stride, p->B_group_stride, p->C_batch_stride,
                        p->C_token_stride, p->C_group_stride});
}

}  // namespace
}  // namespace ptof

using namespace ptof;

extern "C" {

int ptof_short_conv_exec(const ptof_short_conv_params* p, const void* x, const void* w,
                         const void* bias, const int* cu, const void* initial, void* y,
                         void* final_state, void* stream) {
  if (!p) return fail(PTOF_EINVAL, "short_conv: null params");
  if (p->N < 0 || p->T < 0 || p->D < 1 || p->D > kMaxChannels)
    return fail(PTOF_EINVAL, "short_conv: N=%d T=%d D=%d", p->N, p->T, p->D);
  if (p->T > kMaxTokens) return fail(PTOF_EUNSUPPORTED, "short_conv: T=%d tokens", p->T);
  if (p->width < 2 || p->width > 4)
    return fail(PTOF_EUNSUPPORTED, "short_conv: width=%d (2 to 4 taps)", p->width);
  if (!dtype_ok(p->dtype) || !own_or_f32(p->w_dtype, p->dtype))
    return fail(PTOF_EINVAL, "short_conv: bad dtype code");
  const int b = elem_bytes(p->dtype), wb = elem_bytes(p->w_dtype);
  const bool any = p->T > 0 && (p->packed || p->N > 0);
  int rc = check_tensors("short_conv", {{x, "x", b, any},
                                        {w, "w", wb, true},
                                        {bias, "bias", wb, false},
                                        {cu, "cu_seqlens", 4, p->packed != 0},
                                        {initial, "initial", b, false},
                                        {y, "y", b, any},
                                        {final_state, "final_state", b, false}});
  if (!rc)
    rc = check_strides("short_conv", {p->x_batch_stride, p->x_token_stride, p->y_batch_stride,
                                      p->y_token_stride});
  if (rc) return rc;
  return launch_short_conv(*p, x, w, bias, p->packed ? cu : nullptr, initial, y, final_state,
                           static_cast<cudaStream_t>(stream));
}

int ptof_short_conv_step_exec(const ptof_short_conv_step_params* p, const void* x, void* state,
                              const void* w, const void* bias, const int* slots, void* y,
                              void* stream) {
  if (!p) return fail(PTOF_EINVAL, "short_conv_step: null params");
  if (p->M < 0 || p->slots < 0 || p->D < 1 || p->D > kMaxChannels)
    return fail(PTOF_EINVAL, "short_conv_step: M=%d slots=%d D=%d", p->M, p->slots, p->D);
  if (p->width < 2 || p->width > 4)
    return fail(PTOF_EUNSUPPORTED, "short_conv_step: width=%d (2 to 4 taps)", p->width);
  if (!dtype_ok(p->dtype) || !own_or_f32(p->w_dtype, p->dtype))
    return fail(PTOF_EINVAL, "short_conv_step: bad dtype code");
  const int b = elem_bytes(p->dtype), wb = elem_bytes(p->w_dtype);
  int rc = check_tensors("short_conv_step", {{x, "x", b, p->M > 0},
                                             {state, "state", b, p->slots > 0},
                                             {w, "w", wb, true},
                                             {bias, "bias", wb, false},
                                             {slots, "slots", 4, false},
                                             {y, "y", b, p->M > 0}});
  if (!rc)
    rc = check_strides("short_conv_step", {p->x_row_stride, p->y_row_stride, p->state_slot_stride,
                                           p->state_tap_stride});
  if (rc) return rc;
  return launch_short_conv_step(*p, x, state, w, bias, slots, y, static_cast<cudaStream_t>(stream));
}

int64_t ptof_ssm_scan_ws_bytes(const ptof_ssm_scan_params* p) {
  if (validate(p) != PTOF_OK) return -1;
  return static_cast<int64_t>(ssm_scan_ws_bytes(*p));
}

int ptof_ssm_scan_exec(const ptof_ssm_scan_params* p, const void* x, const void* dt,
                       const float* A, const void* B, const void* C, const float* Dskip,
                       const void* z, const float* dt_bias, const int* cu, const float* initial,
                       void* y, float* final_state, void* ws, int64_t ws_bytes, void* stream) {
  int rc = validate(p);
  if (rc) return rc;
  const int b = elem_bytes(p->dtype);
  const bool any = p->T > 0 && p->N > 0, fill = p->T > 0 && p->packed && p->zero_fill;
  rc = check_tensors("ssm_scan", {{x, "x", b, any},
                                  {dt, "dt", b, any},
                                  {A, "A", 4, true},
                                  {B, "B", b, any},
                                  {C, "C", b, any},
                                  {Dskip, "Dskip", 4, false},
                                  {z, "z", b, false},
                                  {dt_bias, "dt_bias", 4, false},
                                  {cu, "cu_seqlens", 4, p->packed != 0},
                                  {initial, "initial", 4, false},
                                  {y, "y", b, any || fill},
                                  {final_state, "final_state", 4, false},
                                  {ws, "ws", 16, false}});
  if (rc) return rc;
  const int64_t need = static_cast<int64_t>(ssm_scan_ws_bytes(*p));
  if (need > 0 && (!ws || ws_bytes < need))
    return fail(PTOF_EINVAL, "ssm_scan: %lld bytes of scratch, %lld needed", (long long)ws_bytes,
                (long long)need);
  return launch_ssm_scan(*p, x, dt, A, B, C, Dskip, z, dt_bias, p->packed ? cu : nullptr, initial,
                         y, final_state, ws, static_cast<cudaStream_t>(stream));
}

int ptof_ssm_scan_step_exec(const ptof_ssm_scan_step_params* p, const void* x, const void* dt,
                            const float* A, const void* B, const void* C, const float* Dskip,
                            const void* z, const float* dt_bias, const int* slots, float* state,
                            void* y, void* stream) {
  if (!p) return fail(PTOF_EINVAL, "ssm_scan_step: null params");
  if (p->M < 0 || p->slots < 0 || p->D < 1 || p->D > kMaxChannels || p->G < 1 || p->D % p->G)
    return fail(PTOF_EINVAL, "ssm_scan_step: M=%d slots=%d D=%d G=%d (D a multiple of G)", p->M,
                p->slots, p->D, p->G);
  if (p->n < 1 || p->n > 128)
    return fail(PTOF_EUNSUPPORTED, "ssm_scan_step: n=%d (1 to 128 states)", p->n);
  if (!dtype_ok(p->dtype)) return fail(PTOF_EINVAL, "ssm_scan_step: bad dtype code");
  const int b = elem_bytes(p->dtype);
  const bool any = p->M > 0;
  int rc = check_tensors("ssm_scan_step", {{x, "x", b, any},
                                           {dt, "dt", b, any},
                                           {A, "A", 4, true},
                                           {B, "B", b, any},
                                           {C, "C", b, any},
                                           {Dskip, "Dskip", 4, false},
                                           {z, "z", b, false},
                                           {dt_bias, "dt_bias", 4, false},
                                           {slots, "slots", 4, false},
                                           {state, "state", 4, p->slots > 0},
                                           {y, "y", b, any}});
  if (!rc)
    rc = check_strides("ssm_scan_step",
                       {p->x_row_stride, p->dt_row_stride, p->z_row_stride, p->y_row_stride,
                        p->B_row_stride, p->B_group_stride, p->C_row_stride, p->C_group_stride,
                        p->state_slot_stride});
  if (rc) return rc;
  return launch_ssm_scan_step(*p, x, dt, A, B, C, Dskip, z, dt_bias, slots, state, y,
                              static_cast<cudaStream_t>(stream));
}

int ptof_add_rms_norm_exec(const ptof_add_rms_norm_params* p, const void* x, const void* residual,
                           const void* w, void* y, void* sum, float* scale, void* stream) {
  if (!p) return fail(PTOF_EINVAL, "add_rms_norm: null params");
  if (p->rows < 0 || p->rows > 0x7fffffffLL || p->D < 1 || p->D > kMaxChannels)
    return fail(PTOF_EINVAL, "add_rms_norm: rows=%lld D=%d", (long long)p->rows, p->D);
  if (!dtype_ok(p->dtype) || !own_or_f32(p->w_dtype, p->dtype) ||
      (residual && !own_or_f32(p->residual_dtype, p->dtype)))
    return fail(PTOF_EINVAL, "add_rms_norm: bad dtype code");
  if (p->fp8 ? (p->group != 0 && p->group != 32 && p->group != 64 && p->group != 128) : p->group != 0)
    return fail(PTOF_EUNSUPPORTED, "add_rms_norm: group=%d (8-bit output: 0, 32, 64 or 128)",
                p->group);
  if (!residual != !sum) return fail(PTOF_EINVAL, "add_rms_norm: residual and sum come together");
  const int b = elem_bytes(p->dtype), rb = elem_bytes(p->residual_dtype);
  const bool any = p->rows > 0;
  int rc = check_tensors("add_rms_norm", {{x, "x", b, any},
                                          {residual, "residual", rb, false},
                                          {w, "w", elem_bytes(p->w_dtype), true},
                                          {y, "y", p->fp8 ? 1 : b, any},
                                          {sum, "sum", rb, false},
                                          {scale, "scale", 4, any && p->fp8 != 0}});
  if (!rc)
    rc = check_strides("add_rms_norm", {p->x_row_stride, p->residual_row_stride, p->y_row_stride,
                                        p->sum_row_stride});
  if (rc) return rc;
  return launch_add_rms_norm(*p, x, residual, w, y, sum, scale, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
