// error.h — the text behind pf_last_error(), for the other files of the C ABI.
#pragma once

#include <string>

// Records msg as this thread's last error and returns `status`.
__attribute__((visibility("hidden"))) int pf_internal_fail(int status, const std::string &msg);
