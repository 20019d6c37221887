// The backward walk of gla_decay_bf16.cuh.
#include <type_traits>
#include "gla_decay_bf16.cuh"

namespace gla {
namespace decay {

template <int DK, int DV>
static int back_gate(cudaStream_t stream, const Back& b, bool gate) {
  return gate ? launch_back<DK, DV, true>(stream, b) : launch_back<DK, DV, false>(stream, b);
}
int fast_back(cudaStream_t stream, const Back& b, bool gate) {
  if (b.w.kd <= 64) return b.w.vd <= 64 ? back_gate<64, 64>(stream, b, gate) : back_gate<64, 128>(stream, b, gate);
  return b.w.vd <= 64 ? back_gate<128, 64>(stream, b, gate) : back_gate<128, 128>(stream, b, gate);
}

}  // namespace decay
}  // namespace gla
