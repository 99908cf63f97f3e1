// Status of a C ABI call, shared by the sources that define entry points.
#pragma once

#include <string>

namespace mfh {

// Leaves `msg` for mfh_last_error() on this thread and returns `code`.
int SetError(int code, const std::string &msg);

}  // namespace mfh
