// llmk_host.h — what the library's entry points share on the host: the handle,
// the calling thread's error message and the check of HIP calls.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "llmk_device.h"

struct llmk_sampler {
  int device;
  uint32_t max_batch, max_vocab;
  llmk::Ws ws;
  void* mem;
  size_t mem_bytes;
  void* stage;         // aligned copies of rows passed at any offset (allocated on demand)
  size_t stage_bytes;
  uint32_t epoch;      // calls made (their parity picks the job count)
  uint32_t ncu;        // the device's compute units
  uint32_t xs_spin;    // phase 1's wait limit (LLMK_TEST_XS_SPIN at create, for tests)
};

namespace llmk {

// Sets the calling thread's error message (llmk_last_error) and returns code.
__attribute__((visibility("hidden"))) int fail(int code, const std::string& msg);

#define HIPCHK(expr)                                                        \
  do {                                                                      \
    hipError_t e_ = (expr);                                                 \
    if (e_ != hipSuccess)                                                   \
      return fail(LLMK_ERR_HIP, std::string(#expr " failed: ") +            \
                                    hipGetErrorString(e_));                 \
  } while (0)

}  // namespace llmk
