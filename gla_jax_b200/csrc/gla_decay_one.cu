// The walks of gla_decay.cuh in mode "one" (a file each, so that they compile side by side).
#include "gla_decay.cuh"

namespace gla {
namespace decay {
int walk_one(cudaStream_t stream, const Walks& p, int n, bool out, const char* name) { return walk_mode<M_ONE>(stream, p, n, out, name); }
}  // namespace decay
}  // namespace gla
