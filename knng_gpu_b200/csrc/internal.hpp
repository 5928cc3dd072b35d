// internal.hpp -- what the translation units of libknng_gpu.so share: the
// thread's last error message (knng_gpu_last_error).
#pragma once
#include <string>

#include "knng_gpu.h"

namespace knng_b200 {
knng_gpu_status set_last_error(knng_gpu_status s, const std::string& msg);
void clear_last_error();
}  // namespace knng_b200
