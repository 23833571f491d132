// What the files of the C entry points share: the error of this thread, the device check, alignment.
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace fa {

// FLASH_OK, or FLASH_ELAUNCH with the text of the HIP error kept for flash_last_hip_error()
int record_hip(int e);
// FLASH_OK on a gfx950, FLASH_ENODEVICE elsewhere
int device_usable();

inline bool misaligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

}  // namespace fa
