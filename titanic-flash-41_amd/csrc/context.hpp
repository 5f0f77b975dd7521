// What ca_primitives_open* returns a handle to; shared by the library's translation units.
#pragma once
#include "../../include/titanic_moe.h"
#include <hip/hip_runtime.h>

struct Context {
    ca_geometry g;
    int cus;
    int stream_wgs;    // persistent workgroups of the streaming kernels
    hipEvent_t marks[7];   // profiling aid: see ca_primitives_marks
    bool marking;
    bool kernel_marks;     // marks[5], marks[6]: begin and end of the FC1 + SwiGLU kernel itself
    int spin_limit;        // polls a wait inside the front-end launch may take before the waiter does the work itself
    int shared_reserve;    // CUs the shared expert's many-row first projection leaves without a workgroup (0: none)
    int device;            // the device the context was opened on
    uint8_t* static_scratch;   // that device's copy of `scratch`
};
