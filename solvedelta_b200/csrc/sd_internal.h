// What the translation units of the library share on the host side.
#pragma once
#include <cuda.h>   // CUtensorMap (types only)
#include <cuda_runtime.h>

namespace sd {

typedef CUresult (*TensorMapEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                      const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                      CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// cuTensorMapEncodeTiled, reached through the runtime; null when the driver has none.
__attribute__((visibility("hidden"))) TensorMapEncodeFn map_encoder();
// The fault word of the current device (see sd_device_fault); null when there is no device.
__attribute__((visibility("hidden"))) int* fault_word();

}  // namespace sd
