// The walks of gla_decay.cuh in mode "state" (a file each, so that they compile side by side).
#include "gla_decay.cuh"

namespace gla {
namespace decay {
int walk_state(cudaStream_t stream, const Walks& p, int n, bool out, const char* name) { return walk_mode<M_STATE>(stream, p, n, out, name); }
}  // namespace decay
}  // namespace gla
