// b2g_internal.h — helpers shared between the library's translation units
// (not part of the C ABI; hidden symbols).
#pragma once

#include <cuda.h>

namespace b2g {

// Device address of the current device's error word (the one
// b2g_read_device_error reports), created on first use; nullptr when no
// sm_100 device is current.
int* current_error_word();

// The current device: its SMs and its error word.  B2G_ERR_NO_DEVICE when no
// sm_100 device is current.
struct Device {
  int num_sms = 0;
  int* error_word = nullptr;
};
int current_device(Device* out);

// cuTensorMapEncodeTiled (through the runtime's entry point), without
// interleave, 256-byte L2 promotion, zeros outside.  false: not to be had, or
// the driver refuses the layout.
bool encode_tiled(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base,
                  const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
                  const cuuint32_t* element_strides, CUtensorMapSwizzle swizzle);

// Bound on every device-side wait, in ns (B2G_WAIT_LIMIT_MS, default 2 s).
long long current_wait_limit_ns();

// Launch with programmatic stream serialization (0 when built without it).
bool pdl_enabled();

}  // namespace b2g
