// errors.h -- the thread's last error of calls without an engine (camelid_hip_last_error(NULL)),
// for the translation units beside engine.hip.
#pragma once

namespace cm {
// Records the message; returns 1, the status of a failed call.
int fail_global(const char* what, const char* why) noexcept;
}  // namespace cm
