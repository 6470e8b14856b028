// Host-side helpers that the library's two translation units share (defined in kvskip_b200.cu).
#pragma once
#include <cuda.h>

namespace kvb_host {

int fail(int code, const char* fmt, ...);          // records the calling thread's message, returns code
int ensure_smem(const void* func, int bytes);      // dynamic shared-memory opt-in, once per (device, kernel)
bool use_pdl();                                    // the "pdl" option
int num_sms();                                     // SMs of the current device
// cuTensorMapEncodeTiled, or null
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled();
// status word of the second translation unit (cache8.cu): reads it, and clears it if it is set
int cache8_status(unsigned int* status);

}  // namespace kvb_host
