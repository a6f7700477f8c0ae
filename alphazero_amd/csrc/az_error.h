// How entry points without an engine handle report why they failed (az_last_error(NULL), per calling thread).
#pragma once

// keeps `message` for az_last_error(NULL) and returns `code`
int az_fail(int code, const char *message) noexcept;
