// The library's last error message (cfh_last_error), set from any of its source files.
#pragma once

namespace cfh {

__attribute__((visibility("hidden"), format(printf, 2, 3))) int fail(int code, const char* fmt, ...);   // returns code
__attribute__((visibility("hidden"))) int finish_launch(const char* what);     // CFH_OK, or CFH_ELAUNCH with HIP's message

}  // namespace cfh
