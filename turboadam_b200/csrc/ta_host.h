// ta_host.h -- what the library's host sources share.
#pragma once

#include <string>

#include "../../include/turboadam_b200.h"

// Sets the calling thread's ta_last_error message and returns s.
ta_status ta_fail(ta_status s, const std::string& message);
