// The calling thread's error text (internal to the library).
#pragma once

namespace pto {
// writes the text that pto_last_error() returns, and gives `code` back
int fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
}  // namespace pto
