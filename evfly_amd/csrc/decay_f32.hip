// Decay attention, exact fp32 (v_mfma_f32_16x16x4_f32).
#include <atomic>

#include "decay_kernel.h"

namespace evfly {
int decay_passes_f32(const DecayPasses &p, bool state, hipStream_t st) { return decay::launch_all<float>(p, state, st); }
}  // namespace evfly
