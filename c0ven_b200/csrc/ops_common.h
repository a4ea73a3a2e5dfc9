// What the operators without a layer (include/moe_layer.h) share on the host: the message a call leaves, what a device pointer
// has to be, and the place every C entry turns an exception into a status.
#pragma once

#include <cuda_runtime.h>

#include <initializer_list>
#include <new>
#include <string>

#include "cuda_rt.h"
#include "moe_layer.h"

namespace moe {

std::string &ops_error();  // the calling thread's

inline void need(bool ok, const char *what) {
  if (!ok) throw BadArgument(what);
}

// A buffer's address: on the current device (what the driver knows of it says so), aligned. A null pointer passes where it may be null.
struct DevicePtr {
  const void *p;
  const char *name;
  uint32_t align;
  bool optional = false;
};

inline void need_device(std::initializer_list<DevicePtr> ptrs) {
  int device = 0;
  CUDA_OK(cudaGetDevice(&device));
  for (const DevicePtr &d : ptrs) {
    if (!d.p) {
      if (!d.optional) throw BadArgument(std::string(d.name) + " is required");
      continue;
    }
    if ((uintptr_t)d.p % d.align) throw BadArgument(std::string(d.name) + " must be " + std::to_string(d.align) + "-byte aligned");
    cudaPointerAttributes at{};
    CUDA_OK(cudaPointerGetAttributes(&at, d.p));
    if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) throw BadArgument(std::string(d.name) + " is not device memory");
    if (at.type == cudaMemoryTypeDevice && at.device != device) throw BadArgument(std::string(d.name) + " is another device's than the current one");
  }
}

// The body of a C entry: no exception leaves it.
template <class Body>
inline moe_status ops_call(Body &&body) noexcept {
  try {
    body();
    return MOE_OK;
  } catch (const BadArgument &e) {
    try {
      ops_error() = e.what();
    } catch (...) {
    }
    return MOE_BAD_ARGUMENT;
  } catch (const Timeout &e) {
    try {
      ops_error() = e.what();
    } catch (...) {
    }
    return MOE_TIMEOUT;
  } catch (const std::exception &e) {
    try {
      ops_error() = e.what();
    } catch (...) {
    }
    return MOE_ERROR;
  } catch (...) {
    return MOE_ERROR;
  }
}

// One value of a row as f32, by ggml's type number.
inline uint32_t row_type_bytes(uint32_t type) { return type == MOE_TYPE_F32 ? 4u : type == MOE_TYPE_F16 || type == MOE_TYPE_BF16 ? 2u : 0u; }

}  // namespace moe
