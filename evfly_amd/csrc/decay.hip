// Decay attention: entry points, the plan of the chunked passes, the recurrent kernel for few tokens and the sum over shared heads.
#include <cmath>

#include "bf16.h"
#include "decay.h"

namespace evfly {
namespace {

// ---------------------------------------------------------------------------------------- recurrence, few tokens
// S_t = e^g S_{t-1} + k_t v_t^T, out_t = scale q_t S_t with the state in registers from its one read to its one write: a call for one
// window moves 8 bytes per state element and little else. One block per (stream, head); a thread holds VW neighbouring columns of the rows
// m R + rg; the tokens' q and k wait in LDS as fp32; column sums meet by lane exchange, then over the waves in LDS, once per call.

struct StepArgs {
    const void *q, *k, *v;
    int64_t qs[3], ks[3], vs[3];
    const float *log_decay, *s_in;
    float *s_out;
    const int32_t *lengths;
    void *out;
    int T, H, rep, dk, dv;
    float scale;
};

template <typename T, int VW, int CG> __global__ __launch_bounds__(256) void k_decay_step(StepArgs p) {
    constexpr int R = 256 / CG, RT = EVFLY_DECAY_MAX_DIM / R;          // rows side by side; rows per thread
    constexpr int NPART = CG <= 64 ? 4 : 2;                              // partial column sums per token
    extern __shared__ __align__(16) float sm[];
    const int tid = threadIdx.x, cg = tid % CG, rg = tid / CG, c = cg * VW;
    const int h = blockIdx.x % p.H;
    const int64_t n = blockIdx.x / p.H;
    const int len = p.lengths ? min(max(p.lengths[n], 0), p.T) : p.T;
    const int64_t sb = (n * p.H + h) * p.dk * p.dv;
    float *const qk = sm, *const part = sm + 2 * p.T * p.dk;

    float S[RT][VW];
#pragma unroll
    for (int m = 0; m < RT; ++m) {
        const int row = m * R + rg;
#pragma unroll
        for (int e = 0; e < VW; ++e) S[m][e] = 0.f;
        if (p.s_in && row < p.dk && c < p.dv) {
            const float *s = p.s_in + sb + (int64_t)row * p.dv + c;
            if constexpr (VW == 4) Elem<float>::load(s, S[m]);
            else S[m][0] = *s;
        }
    }
    const T *const qp = static_cast<const T *>(p.q) + n * p.qs[0] + h * p.qs[2];
    const T *const kp = static_cast<const T *>(p.k) + n * p.ks[0] + (h / p.rep) * p.ks[2];
    const T *const vp = static_cast<const T *>(p.v) + n * p.vs[0] + (h / p.rep) * p.vs[2];
    for (int i = tid; i < 2 * len * p.dk; i += 256) {
        const int t = i / (2 * p.dk), r = i % (2 * p.dk);
        qk[i] = r < p.dk ? Elem<T>::ld1(qp + t * p.qs[1] + r) : Elem<T>::ld1(kp + t * p.ks[1] + (r - p.dk));
    }
    const float keep = expf(p.log_decay[h]);
    __syncthreads();
    for (int t = 0; t < len; ++t) {
        float v[VW], o[VW];
#pragma unroll
        for (int e = 0; e < VW; ++e) {
            v[e] = c < p.dv ? Elem<T>::ld1(vp + t * p.vs[1] + c + e) : 0.f;
            o[e] = 0.f;
        }
        const float *qt = qk + 2 * t * p.dk, *kt = qt + p.dk;
#pragma unroll
        for (int m = 0; m < RT; ++m) {
            const int row = m * R + rg;
            if (row < p.dk) {
                const float kk = kt[row], qq = qt[row];
#pragma unroll
                for (int e = 0; e < VW; ++e) {
                    S[m][e] = fmaf(kk, v[e], keep * S[m][e]);
                    o[e] = fmaf(qq, S[m][e], o[e]);
                }
            }
        }
#pragma unroll
        for (int d = CG; d < 64; d *= 2)
#pragma unroll
            for (int e = 0; e < VW; ++e) o[e] += __shfl_xor(o[e], d);
        if (CG >= 64 || (tid & 63) < CG)
#pragma unroll
            for (int e = 0; e < VW; ++e) part[(t * NPART + (CG <= 64 ? tid >> 6 : rg)) * (CG * VW) + c + e] = o[e];
    }
    if (p.s_out)
#pragma unroll
        for (int m = 0; m < RT; ++m) {
            const int row = m * R + rg;
            if (row < p.dk && c < p.dv) {
                float *s = p.s_out + sb + (int64_t)row * p.dv + c;
                if constexpr (VW == 4) Elem<float>::store(s, S[m]);
                else *s = S[m][0];
            }
        }
    __syncthreads();
    for (int i = tid; i < p.T * p.dv; i += 256) {
        const int t = i / p.dv, col = i % p.dv;
        float o = 0.f;
        if (t < len)
#pragma unroll
            for (int w = 0; w < NPART; ++w) o += part[(t * NPART + w) * (CG * VW) + col];
        Elem<T>::st1(static_cast<T *>(p.out) + ((n * p.T + t) * p.H + h) * p.dv + col, t < len ? o * p.scale : 0.f);
    }
}

template <typename T, int VW, int CG> int step_launch(const StepArgs &a, int n, hipStream_t st) {
    const size_t lds = sizeof(float) * a.T * (2 * a.dk + (CG <= 64 ? 4 : 2) * CG * VW);
    hipLaunchKernelGGL((k_decay_step<T, VW, CG>), dim3((unsigned)((int64_t)n * a.H)), dim3(256), lds, st, a);
    EVFLY_LAUNCH_CHECK();
    return 0;
}
template <typename T> int step_all(const StepArgs &a, int n, hipStream_t st) {
    const bool v4 = a.dv % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.s_in) | reinterpret_cast<uintptr_t>(a.s_out)) & 15) == 0;
    if (v4) return a.dv <= 32 ? step_launch<T, 4, 8>(a, n, st) : a.dv <= 64 ? step_launch<T, 4, 16>(a, n, st) : step_launch<T, 4, 32>(a, n, st);
    return a.dv <= 32 ? step_launch<T, 1, 32>(a, n, st) : a.dv <= 64 ? step_launch<T, 1, 64>(a, n, st) : step_launch<T, 1, 128>(a, n, st);
}

// ---------------------------------------------------------------------------------------- sum over the heads that share a key / value head
// in (rows, kv, rep, d) fp32 -> out (rows, kv, d), added in head order
template <typename T> __global__ __launch_bounds__(256) void k_decay_head_sum(const float *in, int64_t n, int rep, int d, T *out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / d;
        const float *s = in + row * rep * d + i % d;
        float a = 0.f;
        for (int r = 0; r < rep; ++r) a += s[(int64_t)r * d];
        Elem<T>::st1(out + i, a);
    }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct Tokens {              // one token tensor: pointer, element strides, heads per head of the pass, width
    const void *p;
    int64_t s[3];
    int r, d;
};
bool vec_ok(const Tokens &t, int vec) {
    return aligned16(t.p) && t.d % vec == 0 && t.s[0] % vec == 0 && t.s[1] % vec == 0 && t.s[2] % vec == 0;
}

int run_pass(DecayPass p, const Tokens &a, const Tokens &b, const Tokens &c, int dtype, float *seg, hipStream_t st) {
    p.a = a.p; p.b = b.p; p.c = c.p;
    for (int i = 0; i < 3; ++i) { p.as[i] = a.s[i]; p.bs[i] = b.s[i]; p.cs[i] = c.s[i]; }
    p.ra = a.r; p.rb = b.r; p.rc = c.r;
    p.da = a.d; p.dc = c.d;
    const DecayPlan pl = decay_plan(p.n, p.T, p.H, p.da, p.dc);
    p.nseg = pl.nseg; p.seg_len = pl.seg_len; p.seg = seg;
    const int vec = dtype == EVFLY_DTYPE_F32 ? 4 : 8;
    const bool v = vec_ok(a, vec) && vec_ok(b, vec) && vec_ok(c, vec) && aligned16(p.out);
    return dtype == EVFLY_DTYPE_F32 ? decay_pass_f32(p, pl, v, st) : decay_pass_bf16(p, pl, v, st);
}

struct Ws { int64_t seg, part, bytes; };      // offsets in bytes
Ws decay_ws(int n, int T, int H, int KV, int dk, int dv, bool backward) {
    auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    Ws w{0, 0, 0};
    int64_t seg = 0;
    if (T > EVFLY_DECAY_STEP_TOKENS || backward) {
        seg = decay_plan(n, T, H, dk, dv).seg_floats;
        if (backward) {
            const int64_t t = decay_plan(n, T, H, dv, dk).seg_floats;
            seg = seg > t ? seg : t;
        }
    }
    w.part = up(seg * 4);
    w.bytes = w.part + (backward && H != KV ? up((int64_t)n * T * H * (dk > dv ? dk : dv) * 4) : 0);
    return w;
}

int check_shape(const char *who, int n, int T, int H, int KV, int dk, int dv, int dtype, float scale) {
    EVFLY_REQUIRE(n >= 0 && T >= 0 && T <= (1 << 30), "%s: %d streams of %d tokens", who, n, T);
    EVFLY_REQUIRE(H > 0 && KV > 0 && H % KV == 0, "%s: %d heads do not share %d key / value heads evenly", who, H, KV);
    EVFLY_REQUIRE(dk > 0 && dv > 0 && dk <= EVFLY_DECAY_MAX_DIM && dv <= EVFLY_DECAY_MAX_DIM, "%s: head sizes %d, %d are not in 1 .. %d", who, dk, dv, EVFLY_DECAY_MAX_DIM);
    EVFLY_REQUIRE(dtype == EVFLY_DTYPE_F32 || dtype == EVFLY_DTYPE_BF16, "%s: dtype %d (EVFLY_DTYPE_F32 or EVFLY_DTYPE_BF16)", who, dtype);
    EVFLY_REQUIRE(std::isfinite(scale), "%s: scale is not finite", who);
    EVFLY_REQUIRE((int64_t)n * H <= INT32_MAX, "%s: %d streams of %d heads", who, n, H);
    return 0;
}

void token_strides(const int64_t *s, int T, int heads, int d, int64_t (&out)[3]) {
    if (s) { out[0] = s[0]; out[1] = s[1]; out[2] = s[2]; }
    else { out[0] = (int64_t)T * heads * d; out[1] = (int64_t)heads * d; out[2] = d; }
}

}  // namespace

// Tiles: the a dimension whole (its rows are summed in registers), 64 columns of c per block (32 if there are no more). Segments: the sequence is cut where there are
// fewer than four blocks per CU, into pieces of at least four chunks -- a cut costs the rows b and c a second read and the state a round trip.
DecayPlan decay_plan(int n, int T, int H, int da, int dc) {
    DecayPlan p;
    p.DA = da <= 32 ? 32 : da <= 64 ? 64 : 128;
    p.DC = dc <= 32 ? 32 : 64;
    p.ndc = (dc + p.DC - 1) / p.DC;
    const int64_t base = (int64_t)n * H * p.ndc;
    int64_t nseg = base > 0 ? (4 * kNumCU + base - 1) / base : 1;
    const int64_t most = (T + 4 * DECAY_CHUNK - 1) / (4 * DECAY_CHUNK);
    nseg = nseg < most ? nseg : most;
    nseg = nseg > 1 ? nseg : 1;
    int64_t len = (T + nseg - 1) / nseg;
    len = (len + DECAY_CHUNK - 1) / DECAY_CHUNK * DECAY_CHUNK;
    if (len < DECAY_CHUNK) len = DECAY_CHUNK;
    p.seg_len = (int)len;
    p.nseg = (int)((T + len - 1) / len);
    if (p.nseg < 1) p.nseg = 1;
    p.seg_floats = p.nseg > 1 ? base * p.nseg * p.DA * p.DC : 0;
    return p;
}

}  // namespace evfly

using namespace evfly;

extern "C" int64_t evfly_decay_attention_workspace_bytes(int n_streams, int tokens, int heads, int kv_heads, int dk, int dv, int dtype,
                                                         int backward) {
    if (check_shape("decay_attention_workspace_bytes", n_streams, tokens, heads, kv_heads, dk, dv, dtype, 1.f)) return -1;
    return decay_ws(n_streams, tokens, heads, kv_heads, dk, dv, backward != 0).bytes;
}

extern "C" int evfly_decay_attention_forward(const void *q, const void *k, const void *v, const int64_t *strides_host,
                                             const float *log_decay, const float *state_in, const int32_t *lengths, int n_streams,
                                             int tokens, int heads, int kv_heads, int dk, int dv, float scale, int dtype, void *out,
                                             float *state_out, void *workspace, int64_t workspace_bytes, void *stream) {
    if (int rc = check_shape("decay_attention_forward", n_streams, tokens, heads, kv_heads, dk, dv, dtype, scale)) return rc;
    if (n_streams == 0) return 0;
    EVFLY_REQUIRE(log_decay && (tokens == 0 || (q && k && v && out)), "decay_attention_forward: null argument");
    const Ws ws = decay_ws(n_streams, tokens, heads, kv_heads, dk, dv, false);
    EVFLY_REQUIRE(workspace_bytes >= ws.bytes && (ws.bytes == 0 || (workspace && aligned16(workspace))),
                  "decay_attention_forward: workspace smaller than evfly_decay_attention_workspace_bytes, or not 16-byte aligned");
    hipStream_t st = as_stream(stream);
    const int rep = heads / kv_heads;
    Tokens tq{q, {}, 1, dk}, tk{k, {}, rep, dk}, tv{v, {}, rep, dv};
    token_strides(strides_host, tokens, heads, dk, tq.s);
    token_strides(strides_host ? strides_host + 3 : nullptr, tokens, kv_heads, dk, tk.s);
    token_strides(strides_host ? strides_host + 6 : nullptr, tokens, kv_heads, dv, tv.s);
    if (tokens <= EVFLY_DECAY_STEP_TOKENS) {
        StepArgs a;
        a.q = q; a.k = k; a.v = v;
        for (int i = 0; i < 3; ++i) { a.qs[i] = tq.s[i]; a.ks[i] = tk.s[i]; a.vs[i] = tv.s[i]; }
        a.log_decay = log_decay; a.s_in = state_in; a.s_out = state_out; a.lengths = lengths; a.out = out;
        a.T = tokens; a.H = heads; a.rep = rep; a.dk = dk; a.dv = dv; a.scale = scale;
        return dtype == EVFLY_DTYPE_F32 ? step_all<float>(a, n_streams, st) : step_all<bf16_t>(a, n_streams, st);
    }
    DecayPass p{};
    p.out = out; p.log_decay = log_decay; p.lengths = lengths; p.n = n_streams; p.T = tokens; p.H = heads;
    p.s_in = state_in; p.s_fin = state_out; p.s_a = dv; p.s_c = 1;
    p.f_intra = scale; p.f_out = scale; p.f_upd = 1.f;
    return run_pass(p, tq, tk, tv, dtype, static_cast<float *>(workspace), st);
}

extern "C" int evfly_decay_attention_backward(const void *q, const void *k, const void *v, const int64_t *strides_host,
                                              const float *log_decay, const float *state_in, const int32_t *lengths, const void *d_out,
                                              const float *d_state_out, int n_streams, int tokens, int heads, int kv_heads, int dk, int dv,
                                              float scale, int dtype, void *dq, void *dk_out, void *dv_out, float *d_state_in, void *workspace,
                                              int64_t workspace_bytes, void *stream) {
    if (int rc = check_shape("decay_attention_backward", n_streams, tokens, heads, kv_heads, dk, dv, dtype, scale)) return rc;
    if (n_streams == 0) return 0;
    EVFLY_REQUIRE(log_decay && (tokens == 0 || (q && k && v && d_out && dq && dk_out && dv_out)), "decay_attention_backward: null argument");
    const Ws ws = decay_ws(n_streams, tokens, heads, kv_heads, dk, dv, true);
    EVFLY_REQUIRE(workspace_bytes >= ws.bytes && (ws.bytes == 0 || (workspace && aligned16(workspace))),
                  "decay_attention_backward: workspace smaller than evfly_decay_attention_workspace_bytes, or not 16-byte aligned");
    hipStream_t st = as_stream(stream);
    const int rep = heads / kv_heads;
    Tokens tq{q, {}, 1, dk}, tk{k, {}, rep, dk}, tv{v, {}, rep, dv}, to{d_out, {}, 1, dv};
    token_strides(strides_host, tokens, heads, dk, tq.s);
    token_strides(strides_host ? strides_host + 3 : nullptr, tokens, kv_heads, dk, tk.s);
    token_strides(strides_host ? strides_host + 6 : nullptr, tokens, kv_heads, dv, tv.s);
    token_strides(nullptr, tokens, heads, dv, to.s);
    char *const w = static_cast<char *>(workspace);
    float *const seg = reinterpret_cast<float *>(w), *const part = reinterpret_cast<float *>(w + ws.part);

    DecayPass p{};
    p.log_decay = log_decay; p.lengths = lengths; p.n = n_streams; p.T = tokens; p.H = heads;
    // dq_t = scale sum_{s <= t} e^{g (t - s)} (d_out_t . v_s) k_s + scale e^{g (t + 1)} S_in d_out_t
    DecayPass a = p;
    a.out = dq; a.s_in = state_in; a.s_a = 1; a.s_c = dv; a.f_intra = scale; a.f_out = scale; a.f_upd = 1.f;
    if (tokens > 0)
        if (int rc = run_pass(a, to, tv, tk, dtype, seg, st)) return rc;
    // dk_s = scale sum_{t >= s} e^{g (t - s)} (v_s . d_out_t) q_t + e^{g (T - 1 - s)} d_state_out v_s
    DecayPass b = p;
    b.rev = 1; b.out = rep > 1 ? static_cast<void *>(part) : dk_out; b.out_f32 = rep > 1;
    b.s_in = d_state_out; b.s_a = 1; b.s_c = dv; b.f_intra = scale; b.f_out = 1.f; b.f_upd = scale;
    auto head_sum = [&](void *out, int d) {
        const int64_t rows = (int64_t)n_streams * tokens * kv_heads, m = rows * d;
        const unsigned blocks = (unsigned)(m / 256 + 1 < 8 * kNumCU ? m / 256 + 1 : 8 * kNumCU);
        if (dtype == EVFLY_DTYPE_F32) hipLaunchKernelGGL(k_decay_head_sum<float>, dim3(blocks), dim3(256), 0, st, part, m, rep, d, static_cast<float *>(out));
        else hipLaunchKernelGGL(k_decay_head_sum<bf16_t>, dim3(blocks), dim3(256), 0, st, part, m, rep, d, static_cast<bf16_t *>(out));
    };
    if (tokens > 0) {
        if (int rc = run_pass(b, tv, to, tq, dtype, seg, st)) return rc;
        if (rep > 1) head_sum(dk_out, dk);
    }
    // dv_s = scale sum_{t >= s} e^{g (t - s)} (k_s . q_t) d_out_t + e^{g (T - 1 - s)} d_state_out^T k_s; the state that this pass ends with is the
    // gradient of state_in
    DecayPass c = p;
    c.rev = 1; c.out = rep > 1 ? static_cast<void *>(part) : dv_out; c.out_f32 = rep > 1;
    c.s_in = d_state_out; c.s_fin = d_state_in; c.s_a = dv; c.s_c = 1; c.f_intra = scale; c.f_out = 1.f; c.f_upd = scale;
    if (int rc = run_pass(c, tk, tq, to, dtype, seg, st)) return rc;
    if (rep > 1 && tokens > 0) head_sum(dv_out, dv);
    EVFLY_LAUNCH_CHECK();
    return 0;
}
