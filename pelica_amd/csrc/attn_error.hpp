// The calling thread's last error, shared by the files that hold entry points.
#pragma once

namespace pelica {

void clear_error();
// records the message, returns `code`
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

}  // namespace pelica
