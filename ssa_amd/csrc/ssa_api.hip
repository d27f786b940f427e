// Status plumbing shared by every entry point of libssa_hip.
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <utility>

#include "ssa_common.h"

namespace ssa {

static thread_local char g_last_error[512] = "";

int fail(int status, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
  return status;
}

int check_launch(const char* what) {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(SSA_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
  return SSA_OK;
}

int reserve_lds(const void* kernel, size_t bytes, const char* what) {
  if (bytes <= 64 * 1024) return SSA_OK;
  int dev = 0, max_lds = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&max_lds, hipDeviceAttributeMaxSharedMemoryPerBlock, dev) != hipSuccess)
    return fail(SSA_ERR_HIP, "%s: cannot query the LDS limit", what);
  if (bytes > static_cast<size_t>(max_lds))
    return fail(SSA_ERR_UNSUPPORTED, "%s: needs %zu bytes of LDS, device allows %d", what, bytes,
                max_lds);
  if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                          static_cast<int>(bytes)) != hipSuccess)
    return fail(SSA_ERR_HIP, "%s: cannot reserve %zu bytes of LDS", what, bytes);
  return SSA_OK;
}

}  // namespace ssa

extern "C" int ssa_version(void) { return 1; }

extern "C" const char* ssa_status_str(int status) {
  switch (status) {
    case SSA_OK: return "ok";
    case SSA_ERR_INVALID_ARGUMENT: return "invalid argument";
    case SSA_ERR_UNSUPPORTED: return "unsupported shape or type";
    case SSA_ERR_WORKSPACE: return "workspace too small";
    case SSA_ERR_HIP: return "HIP runtime error";
    default: return "unknown status";
  }
}

extern "C" const char* ssa_last_error(void) { return ssa::g_last_error; }

// ssa_call: a slot of eight bytes as an argument of type T.
namespace {

template <typename T>
T argument(int64_t slot) {
  if constexpr (std::is_pointer_v<T>) {
    return reinterpret_cast<T>(static_cast<uintptr_t>(slot));
  } else if constexpr (std::is_floating_point_v<T>) {
    double x;
    memcpy(&x, &slot, sizeof(x));
    return static_cast<T>(x);
  } else {
    return static_cast<T>(slot);
  }
}

template <typename... A, size_t... I>
int spread(int (*f)(A...), const int64_t* a, std::index_sequence<I...>) {
  return f(argument<A>(a[I])...);
}
template <typename... A>
int spread(int (*f)(A...), const int64_t* a) {
  return spread(f, a, std::make_index_sequence<sizeof...(A)>());
}

}  // namespace

extern "C" int ssa_call(int function, const int64_t* arguments) {
  if (arguments == nullptr) return ssa::fail(SSA_ERR_INVALID_ARGUMENT, "ssa_call: null pointer");
  switch (function) {
    case SSA_CALL_MASK_SPANS: return spread(ssa_mask_spans, arguments);
    case SSA_CALL_MASK_SPANS_WINDOW: return spread(ssa_mask_spans_window, arguments);
    case SSA_CALL_MASKED_ATTENTION: return spread(ssa_masked_attention, arguments);
    case SSA_CALL_MASKED_ATTENTION_TWO: return spread(ssa_masked_attention_two, arguments);
    case SSA_CALL_MASKED_ATTENTION_BACKWARD: return spread(ssa_masked_attention_backward, arguments);
    case SSA_CALL_MASKED_ATTENTION_TWO_BACKWARD: return spread(ssa_masked_attention_two_backward, arguments);
    case SSA_CALL_PAGED_STEP: return spread(ssa_paged_step, arguments);
    case SSA_CALL_PAGED_STEP_ZEROED: return spread(ssa_paged_step_zeroed, arguments);
    case SSA_CALL_PAGED_STEP_GENERAL: return spread(ssa_paged_step_general, arguments);
    case SSA_CALL_PAGED_READ: return spread(ssa_paged_read, arguments);
    case SSA_CALL_PAGED_KEEP: return spread(ssa_paged_keep, arguments);
    default: return ssa::fail(SSA_ERR_INVALID_ARGUMENT, "ssa_call: no function %d", function);
  }
}
