// What translation units outside tenmo_hip.hip need of the library's state: where a call enqueues its work and how it
// reports a failure.  Internal to libtenmo_hip.so (hidden symbols).
#ifndef TENMO_LIBRARY_STATE_HPP
#define TENMO_LIBRARY_STATE_HPP
#include <hip/hip_runtime.h>

namespace tenmo {

struct LibraryState {
    hipStream_t stream; // the stream of tenmo_hip_get_stream
    int device;         // the device of tenmo_hip_init
    int cus;            // its compute units
};

// 0 and *out filled in, or TENMO_ERR_NOT_INITIALIZED with the message set
__attribute__((visibility("hidden"))) int library_state(LibraryState* out);
// sets the message that tenmo_hip_last_error returns and gives `code` back
__attribute__((visibility("hidden"))) int library_error(int code, const char* message);

} // namespace tenmo
#endif
