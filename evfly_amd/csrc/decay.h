// Decay attention (decay.hip, decay_f32.hip, decay_bf16.hip): one pass o_t = s_out e^{..} a_t S + s_intra sum e^{g (t - s)} (a_t . b_s) c_s over a
// sequence, forwards or backwards in time. Forward and all three gradients of the operator are such passes with their roles exchanged:
//   out     a = q,     b = k,     c = v       forwards   (state S  [dk][dv])
//   dq      a = d_out, b = v,     c = k       forwards   (state S  transposed)
//   dk      a = v,     b = d_out, c = q       backwards  (state dS transposed)
//   dv      a = k,     b = q,     c = d_out   backwards  (state dS [dk][dv])
#pragma once
#include "common.h"

namespace evfly {

constexpr int DECAY_CHUNK = 64;      // tokens per chunk: four waves of 16 token columns each

struct DecayPass {
    const void *a, *b, *c;
    int64_t as[3], bs[3], cs[3];     // element strides: stream, token, head
    int ra, rb, rc;                  // head h of the pass reads head h / r of the tensor (shared key / value heads)
    void *out;                       // contiguous (stream, token, head, dc), in the tokens' type, or fp32 with out_f32
    int out_f32;
    const float *log_decay;
    const int32_t *lengths;          // NULL: every stream has T tokens
    const float *s_in;               // state the pass starts from (NULL: zeros)
    float *s_fin;                    // state behind the pass (NULL: not wanted); may be s_in
    int64_t s_a, s_c;                // element strides of the state's a and c dimension
    float *seg;                      // states the segments start from, [stream, head][segment][dk][dv] (nseg > 1)
    int n, T, H, da, dc, nseg, seg_len;
    int rev;                         // token order: 0 first to last, 1 last to first
    float f_intra, f_out, f_upd;     // where the operator's scale enters: pair products, state read, state update
};

// Passes of one launch (the same tiles): neighbouring blocks run the passes of one place, so that rows that several of them read come from L2.
struct DecayPasses {
    DecayPass p[3];
    int np;
};

// Split of the sequence into segments that run side by side.
struct DecaySplit { int nseg, seg_len; };
DecaySplit decay_split(int n, int T, int H, int dk, int dv, int dtype, bool backward);

// All passes have the same da and dc classes. STATE: the segments' own states only (into slot segment + 1 of seg), no output.
int decay_passes_f32(const DecayPasses &p, bool state, hipStream_t st);
int decay_passes_bf16(const DecayPasses &p, bool state, hipStream_t st);

inline int decay_tile_a(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }      // the a dimension whole (its rows are summed in registers)
inline int decay_tile_c(int d) { return d <= 32 ? 32 : 64; }                       // columns of c per block

}  // namespace evfly
