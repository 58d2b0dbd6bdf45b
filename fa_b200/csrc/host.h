// host.h -- what the host sides of the library's translation units share: the
// calling thread's last error (b200fa_last_error_string) and the driver's
// tensor-map encoder.  Defined in b200fa.cu.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

namespace b200fa {

void clear_error();
int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* where);
PFN_cuTensorMapEncodeTiled_v12000 encode_fn();  // NULL when the driver has none

}  // namespace b200fa
