// seq_common.cu -- messages of the sequence operators, which take no context.
#include "seq_common.cuh"

#include <stdarg.h>
#include <stdio.h>

namespace zrl {
namespace {
thread_local char g_msg[256] = {0};
}

zrl_status seq_fail(zrl_status s, const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_msg, sizeof(g_msg), fmt, ap);
  va_end(ap);
  return s;
}

zrl_status seq_launched(const char *what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return ZRL_OK;
  return seq_fail(ZRL_CUDA_ERROR, "%s: %s", what, cudaGetErrorString(e));
}

const char *seq_last_error() { return g_msg; }
void seq_clear_error() { g_msg[0] = 0; }

}  // namespace zrl
