// Library-wide C-ABI entry points: version, error reporting, the device error word.
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <tuple>
#include <type_traits>

#include "qp_api_internal.h"
#include "qp_common.cuh"

namespace qp {
__device__ int g_device_error = 0;
}

static thread_local char g_last_error[512] = "";

int set_error(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
  return code;
}

int check_launch(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(QP_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return QP_OK;
}

int device_sm_count() {
  static int counts[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (counts[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    counts[dev] = n;
  }
  return counts[dev];
}

extern "C" int qp_version(void) { return 100; }

extern "C" const char* qp_last_error(void) { return g_last_error; }

// Reads and clears the device error word of the current device (synchronous). *code = 0 when no kernel gave up a
// bounded wait since the last call.
extern "C" int qp_device_error(int* code) {
  if (!code) return set_error(QP_ERR_INVALID, "qp_device_error: null pointer");
  int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(code, qp::g_device_error, sizeof(int));
  if (e == cudaSuccess) e = cudaMemcpyToSymbol(qp::g_device_error, &zero, sizeof(int));
  if (e != cudaSuccess) return set_error(QP_ERR_CUDA, "qp_device_error: %s", cudaGetErrorString(e));
  return QP_OK;
}

// ---------------------------------------------------------------------------------------------------------------
// The entry points with the longest argument lists, from a block of 64-bit words.
#include "../../include/quantpack_b200.h"

namespace {
struct Words {
  const char* at;
  template <class T>
  T take() {
    if constexpr (std::is_same<T, float>::value) {
      double v;
      memcpy(&v, at, 8);
      at += 8;
      return static_cast<float>(v);
    } else {
      int64_t v;
      memcpy(&v, at, 8);
      at += 8;
      if constexpr (std::is_pointer<T>::value) return reinterpret_cast<T>(static_cast<uintptr_t>(v));
      else return static_cast<T>(v);
    }
  }
};

// braces: the words are taken in the order of the parameters
template <class... A>
struct Call {
  std::tuple<A...> args;
  explicit Call(Words w) : args{w.take<A>()...} {}
};
template <class... A>
int invoke(int (*fn)(A...), const void* words, int count) {
  if (count != static_cast<int>(sizeof...(A)))
    return set_error(QP_ERR_INVALID, "invoke: %d arguments, expected %d", count, static_cast<int>(sizeof...(A)));
  return std::apply(fn, Call<A...>(Words{static_cast<const char*>(words)}).args);
}
}  // namespace

extern "C" int qp_invoke(int entry, const void* words, int count) {
  if (!words) return set_error(QP_ERR_INVALID, "invoke: null pointer");
  switch (entry) {
    case 0: return invoke(qp_paged_decode, words, count);
    case 1: return invoke(qp_accumulate_attn_weights, words, count);
    case 2: return invoke(qp_evict_cache, words, count);
    default: return set_error(QP_ERR_INVALID, "invoke: entry %d", entry);
  }
}
