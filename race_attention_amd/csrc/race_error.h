// race_error.h -- the status codes' messages, shared by the library's translation units.
#pragma once

#define RACE_INTERNAL __attribute__((visibility("hidden")))

namespace race {

// Store the thread's message (race_last_error) and return the code / clear it and return RACE_OK.
RACE_INTERNAL int fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
RACE_INTERNAL int ok();
// The status of the launches since the last one: RACE_OK or RACE_E_LAUNCH.
RACE_INTERNAL int launched(const char *what);

}  // namespace race
