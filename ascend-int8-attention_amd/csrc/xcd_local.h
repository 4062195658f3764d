// Whether work-groups whose blockIdx agree modulo 8 run on one XCD of the
// current device (a one-time probe, run by the first eager launch; never
// during capture).  Defined in sharedkv_c8.hip.
#pragma once
#include <hip/hip_runtime.h>
namespace sharedkv {
bool xcd_local(hipStream_t stream);
}
