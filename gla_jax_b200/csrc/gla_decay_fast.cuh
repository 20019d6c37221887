// The tensor-core walks as the rest of decay attention calls them: bf16, head sizes up to 128.
#pragma once
#include "gla_decay.cuh"

namespace gla {
namespace decay {

constexpr int WALK_COLS = 2;               // partial sums that a walk leaves in rdot

// A backward walk: dk, dv, the gates (dg, with `gate`) and the first state's gradient (w.fin).
struct Back {
  Walk w;                                  // k, q, v; H, sizes, gates, runs; seg_state: gradients that enter each run backwards
  const void* dout;
  const float* a;                          // [WALK_COLS][token][H], with gates: what the walk for dq leaves in rdot
  const float *S_runs, *S_end;             // entering states of the runs [slot][H][vd][kd] (NULL: one run each), final states
  const void* S_init;                      // the sequences' first states, in the type of w.init
  void *dk, *dv;
  int dk_f32;
  float* dg;
};
// planes of the weighted keys and of the state: 2, 1 | 3, 1 (a state that leaves in float32) | 2, 2 (with the gates' gradient);
// sums only: 2 | 3
enum FastKind { F_ONE = 0, F_STATE = 1, F_FINE = 2, F_SUMS = 3, F_SUMS_STATE = 4 };
int fast_walk(cudaStream_t, const Walk&, int kind, const char* name);
int fast_back(cudaStream_t, const Back&, bool gate);
unsigned int tc_walk_timeouts();
unsigned int tc_back_timeouts();

}  // namespace decay
}  // namespace gla
