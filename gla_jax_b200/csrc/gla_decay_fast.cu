// The walks of gla_decay_bf16.cuh.
#include <type_traits>
#include "gla_decay_bf16.cuh"

namespace gla {
namespace decay {

template <int NU, int NS, bool OUT>
static int walk_sizes(cudaStream_t stream, const Walk& p, const char* name) {
  if (p.kd <= 64) return p.vd <= 64 ? launch_fast<64, 1, NU, NS, OUT>(stream, p, name) : launch_fast<64, 2, NU, NS, OUT>(stream, p, name);
  return p.vd <= 64 ? launch_fast<128, 1, NU, NS, OUT>(stream, p, name) : launch_fast<128, 2, NU, NS, OUT>(stream, p, name);
}
int fast_walk(cudaStream_t stream, const Walk& p, int kind, const char* name) {
  switch (kind) {
    case F_ONE: return walk_sizes<2, 1, true>(stream, p, name);
    case F_STATE: return walk_sizes<3, 1, true>(stream, p, name);
    case F_FINE: return walk_sizes<2, 2, true>(stream, p, name);
    case F_SUMS: return walk_sizes<2, 1, false>(stream, p, name);
    default: return walk_sizes<3, 1, false>(stream, p, name);
  }
}
unsigned int bad_offsets_fast() { return read_bad_offsets(); }

}  // namespace decay
}  // namespace gla
