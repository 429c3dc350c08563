// decay_attention_f32.hip — K14's passes for fp32 q, k and v (pm_decay.h).

#include "pm_decay.h"

namespace pm {

hipError_t decay_pass_f32(const DecayPasses& a, int kind, hipStream_t st) { return run_pass<3>(a, kind, st); }
hipError_t decay_near_f32(const DecayNear& a, hipStream_t st) { return run_near<3>(a, st); }

}  // namespace pm
