// Decay attention, bf16 tokens (v_mfma_f32_16x16x32_bf16, fp32 accumulate and state).
#include <atomic>

#include "decay_kernel.h"

namespace evfly {
int decay_passes_bf16(const DecayPasses &p, bool state, hipStream_t st) { return decay::launch_all<bf16_t>(p, state, st); }
}  // namespace evfly
