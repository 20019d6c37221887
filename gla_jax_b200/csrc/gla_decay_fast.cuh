#pragma once
#include "gla_decay.cuh"
namespace gla {
namespace decay {
int tc_walk(cudaStream_t, const Walk&, int kind, const char* name);
unsigned int tc_walk_bad_offsets();
unsigned int tc_walk_timeouts();
}  // namespace decay
}  // namespace gla
