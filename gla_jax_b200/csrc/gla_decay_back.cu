// The backward walk of gla_decay_tcb.cuh.
#include <type_traits>
#include "gla_decay_tcb.cuh"
#include "gla_decay_fast.cuh"

namespace gla {
namespace decay {

template <int DK, int DV>
static int back_gate(cudaStream_t stream, TcBack& b, const void* dout, bool gate) {
  return gate ? launch_tc_back<DK, DV, true>(stream, b, dout) : launch_tc_back<DK, DV, false>(stream, b, dout);
}
int fast_back(cudaStream_t stream, const Back& x, bool gate) {
  TcBack b;
  b.w = x.w;
  b.a = x.a; b.S_runs = x.S_runs; b.S_end = x.S_end; b.S_init = x.S_init; b.dk = x.dk; b.dv = x.dv; b.dk_f32 = x.dk_f32; b.dg = x.dg;
  if (b.w.kd <= 64) return b.w.vd <= 64 ? back_gate<64, 64>(stream, b, x.dout, gate) : back_gate<64, 128>(stream, b, x.dout, gate);
  return b.w.vd <= 64 ? back_gate<128, 64>(stream, b, x.dout, gate) : back_gate<128, 128>(stream, b, x.dout, gate);
}
unsigned int tc_back_timeouts() { return read_wait_timeouts(); }

}  // namespace decay
}  // namespace gla
