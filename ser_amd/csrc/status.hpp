// What the translation units of libserhip.so share: the thread-local error message and the device of a context
// (both defined in serhip.hip).
#pragma once

#include <string>

struct serhip_ctx;

namespace serhip {

// records `msg` for serhip_last_error() and returns `code`
int set_error(int code, const std::string& msg);
int context_device(const serhip_ctx* ctx);

}  // namespace serhip
