// Host-side helpers shared by the translation units of libsad.
#pragma once
#include <hip/hip_runtime.h>

namespace sad {

// stores the message sad_last_error() returns to the calling thread and gives back `code`; defined in sad_api.hip
__attribute__((visibility("hidden"), format(printf, 2, 3))) int set_error(int code, const char* fmt, ...);

}  // namespace sad
