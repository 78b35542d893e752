// What the translation units of the library share on the host side (defined in svb_api.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#define SVB_HIDDEN __attribute__((visibility("hidden")))

namespace svb {
namespace host {

SVB_HIDDEN bool device_ok();          // the current device is a gfx950
SVB_HIDDEN int device_cus();          // its compute units (0: unknown)
SVB_HIDDEN int fail_hip(hipError_t);  // remembers the error for svbgpu_strerror, returns SVBGPU_EHIP
SVB_HIDDEN int fill_u32(void* ptr, uint32_t value, size_t bytes, hipStream_t st);
// Before and after the kernels of an encoder that places its tiles by look-back: the workspace is checked, the call
// gets its tag (or a clearing launch), and a captured call puts the tickets back (svbgpu_workspace_init).
SVB_HIDDEN int begin_lookback(uint32_t count, void* ws, size_t ws_bytes, hipStream_t st, unsigned* tag2);
SVB_HIDDEN int end_lookback(void* ws, hipStream_t st, unsigned tag2);
// Non-temporal policy of a call that reads and writes that many bytes once each (bit 0 loads, bit 1 stores).
SVB_HIDDEN int nt_policy(unsigned long long load_bytes, unsigned long long store_bytes);

}  // namespace host
}  // namespace svb
