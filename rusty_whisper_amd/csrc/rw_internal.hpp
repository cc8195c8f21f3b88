// rw_internal.hpp -- what the library's translation units share: the calling
// thread's error text, the device check and the per-(device, stream)
// workspaces.  Defined in rw_rocm.hip.
#pragma once
#include <stddef.h>

// sets the calling thread's error text and returns `code`
int rw_internal_fail(int code, const char *msg);
// the calling thread's current device (gfx950, or RW_ENODEV)
int rw_internal_current_device(int *dev);
// takes the workspace of (device, stream) until `slot` is released
int rw_internal_workspace(int device, void *stream, size_t bytes, void **slot, void **out);
void rw_internal_workspace_release(void *slot);
