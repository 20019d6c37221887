// The walks of gla_decay_tc.cuh.
#include "gla_decay_tc.cuh"
#include "gla_decay_fast.cuh"

namespace gla {
namespace decay {

static_assert(WALK_COLS == TC_COLS, "partial sums of rdot");

template <int NU, int NS, bool OUT>
static int sizes(cudaStream_t stream, const Walk& p, const char* name) {
  if (p.kd <= 64) return p.vd <= 64 ? launch_tc<64, 64, NU, NS, OUT>(stream, p, name) : launch_tc<64, 128, NU, NS, OUT>(stream, p, name);
  return p.vd <= 64 ? launch_tc<128, 64, NU, NS, OUT>(stream, p, name) : launch_tc<128, 128, NU, NS, OUT>(stream, p, name);
}
int fast_walk(cudaStream_t stream, const Walk& p, int kind, const char* name) {
  switch (kind) {
    case F_ONE: return sizes<2, 1, true>(stream, p, name);
    case F_STATE: return sizes<3, 1, true>(stream, p, name);
    case F_FINE: return sizes<2, 2, true>(stream, p, name);
    case F_SUMS: return sizes<2, 1, false>(stream, p, name);
    default: return sizes<3, 1, false>(stream, p, name);
  }
}
unsigned int tc_walk_timeouts() { return read_wait_timeouts(); }

}  // namespace decay
}  // namespace gla
