// moe_launch.hpp — error reporting that the kernel files of libprefree_kernels.so share (text behind pfk_last_error).
#pragma once

// Records `what` as this thread's last error and returns `status`.
__attribute__((visibility("hidden"))) int pfk_internal_fail(int status, const char *what);
// PF_OK, or PF_ERR_HIP with the runtime's message when the launch before it failed.
__attribute__((visibility("hidden"))) int pfk_internal_launched(const char *what);
