// The stream and event handles of the C ABI, for the entry points that take them.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/tatara_hip.h"

struct TataraStream {
    hipStream_t s;
    int device;
    bool wrapped;  // another library's stream
};

struct TataraEvent {
    hipEvent_t e;
    int device;
};

namespace tatara {

// NULL is the device's null stream.
inline hipStream_t raw(TataraStream* s) { return s ? s->s : nullptr; }

}  // namespace tatara
