// Decay attention, exact fp32 (v_mfma_f32_16x16x4_f32).
#include <atomic>

#include "decay_kernel.h"

namespace evfly {
int decay_pass_f32(const DecayPass &p, const DecayPlan &pl, bool vec, hipStream_t st) { return decay::launch_all<float>(p, pl, vec, st); }
}  // namespace evfly
