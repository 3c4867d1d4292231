// launches.h — kernels launched by the bindings whose number of launches depends on their arguments.
#pragma once
#include <atomic>
#include <cstdint>

namespace bd {

extern std::atomic<int64_t> counted_launches;  // bindings.cpp

}  // namespace bd
