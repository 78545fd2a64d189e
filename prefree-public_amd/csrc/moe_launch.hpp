// moe_launch.hpp — error reporting and launch limits that the kernel files of libprefree_kernels.so share.
#pragma once

// Workgroups of `threads` that one launch may have: a grid's work items are counted in 32 bits, and a launch of more reports
// success and leaves out all but the remainder.  A multiple of the XCDs.
constexpr long long most_workgroups(int threads) { return 0xffffffffLL / threads / 8 * 8; }

// launch(first, count) over [0, total), no more than `most` at a time.
template <typename F>
void in_launches(long long total, long long most, F launch)
{
    for (long long first = 0; first < total; first += most) launch(first, total - first < most ? total - first : most);
}

// Records `what` as this thread's last error (the text behind pfk_last_error) and returns `status`.
__attribute__((visibility("hidden"))) int pfk_internal_fail(int status, const char *what);
// PF_OK, or PF_ERR_HIP with the runtime's message when the launch before it failed.
__attribute__((visibility("hidden"))) int pfk_internal_launched(const char *what);
