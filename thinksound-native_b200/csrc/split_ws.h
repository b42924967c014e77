// split_ws.h — the workspace of attention calls that split their keys over several CTAs, and the encoder of tensor maps.
#pragma once
#include <cudaTypedefs.h>

#include "runtime.h"

namespace tsn {

// Groups of rows whose parts can meet in a handle's workspace, and its bytes for their sums.
constexpr size_t SPLIT_GROUPS = 4096, SPLIT_BYTES = (size_t) 32 << 20;

struct SplitUse {
    unsigned int * count = nullptr;   // [groups], zero before and after a call
    float * part = nullptr;
    bool captured = false;
    unsigned long long stream = 0;
};
// Before a call's launch: counters of `groups` (at most SPLIT_GROUPS) and `bytes` (at most SPLIT_BYTES) for its parts. An eager
// call takes the handle's workspace in turn with the others, a captured one memory that its graph owns. `name`: of the entry point.
int split_begin(DeviceCtx & c, const char * name, size_t groups, size_t bytes, SplitUse & u);
cudaError_t split_end(DeviceCtx & c, const SplitUse & u);   // after the launch
void release_split(int ordinal);   // with the device: workspaces of graphs that are gone

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();   // null where the driver has none

} // namespace tsn
