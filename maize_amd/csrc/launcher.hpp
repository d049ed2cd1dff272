// What the launcher (shim.cpp) gives to entry points in other files, and the code object that such a file brings along.
// The launcher knows no such file by name: a program built without it has no further code object and needs none.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "maize_hip.h"

namespace maize __attribute__((visibility("hidden"))) {

constexpr uint32_t kMaxMoreKernels = 48;

// Loaded into every context behind the launcher's own code objects; a context that cannot load it is not made.
struct MoreKernels {
    const unsigned char* image;
    const char* what;                          // for the error message
    uint32_t count;
    const char* (*name)(uint32_t index);       // NULL: no kernel of this index
};
// Called while the library is loaded, before any context exists; there is one such code object.
int add_kernels(const MoreKernels* more);

// The text of maize_hip_last_error, and `code` back.
__attribute__((format(printf, 2, 3))) int32_t report(int32_t code, const char* fmt, ...);

uint32_t compute_units(const maize_ctx_t* ctx);
// The stream's scratch memory: as for the split products, zero where a launch leaves it zero.  false: it cannot be had (no device memory, or
// too many are kept for graphs); no error of the runtime is left behind, so that a launch that needs none can follow.
bool stream_workspace(maize_ctx_t* ctx, void* stream, size_t bytes, void** out);
// One kernel of the further code object on a grid of `grid` workgroups.
int32_t launch_more(maize_ctx_t* ctx, uint32_t index, uint32_t grid, uint32_t block, void* stream, const void* args, size_t nbytes);

}  // namespace maize
