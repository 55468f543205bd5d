// fa4d_host.h — host helpers of fa4d_api.cu shared with the library's other C ABI files:
// error messages, the owning device of a pointer, the device status word, tensor maps.
#pragma once

#include <cstdint>
#include <cuda.h>

namespace fa4d {

int host_fail(int code, const char* message);  // records the message, returns code
int host_ok();
int host_bind_device_of(const void* ptr, const char* name);
int* host_status_word();
int host_sm_count();
int host_encode_bthd(CUtensorMap* m, const void* ptr, int B, int T, int H, int D, const int64_t st[3], int rows,
                     bool bf16, const char* name);

}  // namespace fa4d
