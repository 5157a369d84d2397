// dsk_host.h — what the library's translation units share on the host: the text of the last error.
#pragma once

#include <cstdarg>

namespace dsk {
// Writes dsk_last_error()'s text of this thread and returns `code`.
__attribute__((visibility("hidden"))) int fail_text(int code, const char* fmt, va_list ap);
}  // namespace dsk
