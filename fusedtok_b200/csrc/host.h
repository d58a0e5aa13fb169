// What the library's translation units share on the host side: the error message of the last failing call, launch
// bookkeeping and the TMA descriptor encoder. Defined in fusedtok_b200.cu.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <string>

namespace ftk {
namespace host {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                  CUtensorMapFloatOOBfill);

// records the message of a failing call and returns `code`
int fail(int code, const std::string& msg);
// after a kernel launch: counts it, and turns a launch error into a status
int launched(const char* what);
// SM count of the current device
int current_sm_count(int* count);
// cuTensorMapEncodeTiled of the installed driver
int encoder(EncodeTiledFn* fn);

// Status word of the 8-bit decode kernels on the current device, read and cleared (decode_q8 has no workspace of the
// library's to keep it in). Defined in serving_q8.cu.
int q8_status(int* status);

}  // namespace host
}  // namespace ftk
