// The walks of gla_decay_bf16.cuh and gla_decay_tc.cuh.
#include "gla_decay_bf16.cuh"
#include "gla_decay_fast.cuh"

namespace gla {
namespace decay {

int fast_walk(cudaStream_t stream, const Walk& p, int kind, const char* name) {
  switch (kind) {
    case F_FINE:
      if (p.kd <= 64) return p.vd <= 64 ? launch_fast<64, 1, 2, 2, true>(stream, p, name) : launch_fast<64, 2, 2, 2, true>(stream, p, name);
      return p.vd <= 64 ? launch_fast<128, 1, 2, 2, true>(stream, p, name) : launch_fast<128, 2, 2, 2, true>(stream, p, name);
    default: return tc_walk(stream, p, kind, name);
  }
}
unsigned int bad_offsets_fast() { return read_bad_offsets() + tc_walk_bad_offsets(); }

}  // namespace decay
}  // namespace gla
