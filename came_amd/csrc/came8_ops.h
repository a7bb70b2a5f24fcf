// What the translation units of libcame8 share on the host beside the CAME step: the calling thread's error message
// and the check after a launch (both defined in came8.hip).
#pragma once

#include <string>

namespace came8 {

// keeps msg for came8_last_error() and returns code
int op_fail(int code, const std::string& msg);

// CAME8_OK, or CAME8_EHIP with the launch's error
int op_check_launch(const char* what);

}  // namespace came8
