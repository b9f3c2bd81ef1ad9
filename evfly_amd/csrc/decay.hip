// Decay attention: entry points, the plan of the chunked passes, the recurrent kernel for few tokens and the sum over shared heads.
#include <cmath>
#include <type_traits>

#include "bf16.h"
#include "decay.h"

namespace evfly {
namespace {

// ---------------------------------------------------------------------------------------- recurrence, few tokens
// S_t = e^g S_{t-1} + k_t v_t^T, out_t = scale q_t S_t with the state in registers from its one read to its one write: a call for one
// window moves 8 bytes per state element and little else (256 streams x 16 heads x 64 x 64: 134 MB in 23 us). One block per (stream, head) of four waves, or of
// one for several tokens on a state of up to 32 x 32 (256 streams x 10 windows x 8 heads of 32: 12.4 us against 14.6 for four waves that exchange column sums, 10.4
// since the tokens' loads overlap; one token, 64 streams x 4 heads: 4.3 against 3.7). A thread holds four neighbouring columns (16 bytes at any address) of
// neighbouring rows; the tokens wait in LDS as fp32; column sums meet by lane exchange, then over the waves in LDS, once per call.
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

template <typename T, int CG, int DK, int NW> __global__ __launch_bounds__(64 * NW) void k_decay_step(StepArgs p) {
    constexpr int VW = 4, R = 64 * NW / CG, RT = DK / R;                             // groups of rows side by side; rows per thread
    static_assert(RT >= 1, "every group has rows");
    extern __shared__ __align__(16) float sm[];
    const int tid = threadIdx.x, cg = tid % CG, rg = tid / CG, c = cg * VW;
    const int h = blockIdx.x % p.H;
    const int64_t n = blockIdx.x / p.H;
    const int len = p.lengths ? min(max(p.lengths[n], 0), p.T) : p.T;
    const int64_t sb = (n * p.H + h) * p.dk * p.dv;
    constexpr int tw = 2 * DK + CG * VW;                                 // a token's q, k and v, padded with zeros to the threads' rows and columns
    float *const tok = sm, *const part = sm + p.T * tw;

    float S[RT][VW];
    auto read_state = [&](auto tail) {                                   // (a width of whole pieces: every load free of the others' branches)
#pragma unroll
        for (int m = 0; m < RT; ++m) {
            const int row = rg * RT + m;
            uint4 u = make_uint4(0, 0, 0, 0);
            if (row < p.dk) u = load_piece<float, decltype(tail)::value>(p.s_in + sb + (int64_t)row * p.dv + c, p.dv - c);
            S[m][0] = __uint_as_float(u.x); S[m][1] = __uint_as_float(u.y); S[m][2] = __uint_as_float(u.z); S[m][3] = __uint_as_float(u.w);
        }
    };
    if (!p.s_in)
#pragma unroll
        for (int m = 0; m < RT; ++m)
#pragma unroll
            for (int e = 0; e < VW; ++e) S[m][e] = 0.f;
    else if (p.dv % VW == 0) read_state(std::false_type{});
    else read_state(std::true_type{});
    const T *const qp = static_cast<const T *>(p.q) + n * p.qs[0] + h * p.qs[2];
    const T *const kp = static_cast<const T *>(p.k) + n * p.ks[0] + (h / p.rep) * p.ks[2];
    const T *const vp = static_cast<const T *>(p.v) + n * p.vs[0] + (h / p.rep) * p.vs[2];
    // (unrolled: the loads of several tokens are in flight before the first one is needed)
#pragma unroll 4
    for (int i = tid; i < len * DK; i += 64 * NW) {
        const int t = i / DK, r = i % DK;
        tok[t * tw + r] = r < p.dk ? Elem<T>::ld1(qp + t * p.qs[1] + r) : 0.f;
        tok[t * tw + DK + r] = r < p.dk ? Elem<T>::ld1(kp + t * p.ks[1] + r) : 0.f;
    }
#pragma unroll 4
    for (int i = tid; i < len * (CG * VW); i += 64 * NW) {
        const int t = i / (CG * VW), r = i % (CG * VW);
        tok[t * tw + 2 * DK + r] = r < p.dv ? Elem<T>::ld1(vp + t * p.vs[1] + r) : 0.f;
    }
    const float keep = expf(p.log_decay[h]);
    __syncthreads();
    for (int t = 0; t < len; ++t) {
        float v[VW], o[VW], qq[RT], kk[RT];
        const float *at = tok + t * tw;
#pragma unroll
        for (int e = 0; e < VW; ++e) { v[e] = at[2 * DK + c + e]; o[e] = 0.f; }
#pragma unroll
        for (int m = 0; m < RT; ++m) { qq[m] = at[rg * RT + m]; kk[m] = at[DK + rg * RT + m]; }
#pragma unroll
        for (int m = 0; m < RT; ++m)
#pragma unroll
            for (int e = 0; e < VW; ++e) {
                S[m][e] = fmaf(kk[m], v[e], keep * S[m][e]);
                o[e] = fmaf(qq[m], S[m][e], o[e]);
            }
#pragma unroll
        for (int e = 0; e < VW; ++e) {
            if (CG <= 8) o[e] += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(o[e]), 0x128, 0xf, 0xf, true));      // row_ror:8
            if (CG <= 16) o[e] = sum_xor16(o[e]);
            o[e] = sum_xor32(o[e]);
        }
        if ((tid & 63) < CG)
#pragma unroll
            for (int e = 0; e < VW; ++e) part[(t * NW + (tid >> 6)) * (CG * VW) + c + e] = o[e];
    }
    if (p.s_out)
#pragma unroll
        for (int m = 0; m < RT; ++m) {
            const int row = rg * RT + m;
            if (row >= p.dk) continue;
            float *s = p.s_out + sb + (int64_t)row * p.dv + c;
            if (c + 4 <= p.dv) store16_any(s, make_uint4(__float_as_uint(S[m][0]), __float_as_uint(S[m][1]), __float_as_uint(S[m][2]), __float_as_uint(S[m][3])));
            else
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    if (c + e < p.dv) s[e] = S[m][e];
        }
    __syncthreads();
    for (int t = tid >> 6; t < p.T; t += NW)
        for (int col = tid & 63; col < p.dv; col += 64) {
            float o = 0.f;
            if (t < len)
#pragma unroll
                for (int w = 0; w < NW; ++w) o += part[(t * NW + w) * (CG * VW) + col];
            Elem<T>::st1(static_cast<T *>(p.out) + ((n * p.T + t) * p.H + h) * p.dv + col, t < len ? o * p.scale : 0.f);
        }
}

template <typename T, int CG, int DK, int NW> int step_launch(const StepArgs &a, int n, hipStream_t st) {
    const size_t lds = sizeof(float) * a.T * (2 * DK + CG * 4 + NW * CG * 4);      // at most 56 KB
    hipLaunchKernelGGL((k_decay_step<T, CG, DK, NW>), dim3((unsigned)((int64_t)n * a.H)), dim3(64 * NW), lds, st, a);
    EVFLY_LAUNCH_CHECK();
    return 0;
}
template <typename T, int CG> int step_rows(const StepArgs &a, int n, hipStream_t st) {
    return a.dk <= 32 ? step_launch<T, CG, 32, 4>(a, n, st) : a.dk <= 64 ? step_launch<T, CG, 64, 4>(a, n, st) : step_launch<T, CG, 128, 4>(a, n, st);
}
template <typename T> int step_all(const StepArgs &a, int n, hipStream_t st) {
    if (a.T > 1 && a.dv <= 32 && a.dk <= 32) return step_launch<T, 8, 32, 1>(a, n, st);
    return a.dv <= 32 ? step_rows<T, 8>(a, n, st) : a.dv <= 64 ? step_rows<T, 16>(a, n, st) : step_rows<T, 32>(a, n, st);
}

// ---------------------------------------------------------------------------------------- states at the segment borders
// slot s + 1 holds segment s's own state (the tokens of that segment alone); slot s receives the state that segment s starts from,
//     start_{s+1} = e^{g cnt_s} start_s + own_s,    start_0 = s_in
// (start_0 as well: the last segment may write its final state over s_in while the first one runs). Segments count in the pass's own order of time.
struct ScanArgs {
    float *slots[2];
    const float *s_in[2];
    const float *log_decay;
    const int32_t *lengths;
    int T, H, nseg, seg_len, elems;       // elems = dk * dv
};
__global__ __launch_bounds__(256) void k_decay_scan(ScanArgs p) {
    const int i = blockIdx.y * 256 + threadIdx.x, nh = blockIdx.x, z = blockIdx.z;
    if (i >= p.elems) return;
    const int len = p.lengths ? min(max(p.lengths[nh / p.H], 0), p.T) : p.T;
    const float gl = p.log_decay[nh % p.H];
    float *slot = p.slots[z] + (int64_t)nh * p.nseg * p.elems + i;
    float S = p.s_in[z] ? p.s_in[z][(int64_t)nh * p.elems + i] : 0.f;
    slot[0] = S;
    const float full = expf(gl * (float)p.seg_len);
#pragma unroll 8
    for (int s = 1; s < p.nseg; ++s) {
        const int cnt = min(max(len - (s - 1) * p.seg_len, 0), p.seg_len);
        const float keep = cnt == p.seg_len ? full : cnt == 0 ? 1.f : expf(gl * (float)cnt);
        S = fmaf(keep, S, slot[(int64_t)s * p.elems]);
        slot[(int64_t)s * p.elems] = S;
    }
}

// ---------------------------------------------------------------------------------------- sum over the heads that share a key / value head
// in (rows, kv, rep, d) fp32 -> out (rows, kv, d), added in head order; blockIdx.y: dk or dv
struct HeadSum {
    const float *in[2];
    void *out[2];
    int d[2];
    int64_t heads;                         // rows * kv
    int rep;
};
template <typename T> __global__ __launch_bounds__(256) void k_decay_head_sum(HeadSum p) {
    const int y = blockIdx.y, d = p.d[y];
    const int64_t n = p.heads * d;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t head = i / d;
        const float *s = p.in[y] + head * p.rep * d + (i - head * d);
        float a = 0.f;
        for (int r = 0; r < p.rep; ++r) a += s[(int64_t)r * d];
        Elem<T>::st1(static_cast<T *>(p.out[y]) + i, a);
    }
}

// The recurrence costs a step per token, a chunk of 64 the same for one token as for all. Forward, us, recurrence against chunk, bf16: 256 streams x 8 heads x 64, 8 tokens
// 20 / 28, 11 tokens 24 / 28, 13 tokens 28 / 28; 16 x 8 x 128, 11 tokens 13.6 / 13.5, 16 tokens 17 / 13.5; 64 x 16 x 128, 12 tokens 45 / 52, 16 tokens 54 / 51. So the
// crossing lies between 11 and 16 tokens, earliest where few blocks run; from 11 on the side not taken is up to a fifth better on large batches. 256 x 8 x 32, bf16, 16 tokens
// 15.0 / 15.9; fp32, 16 tokens, 256 x 8 x 64 32 / 34, 64 x 16 x 128 56 / 106, 16 x 8 x 128 16.7 / 16.4.
bool recurrent(int tokens, int dk, int dv, int dtype) {
    const bool quick_chunk = dtype == EVFLY_DTYPE_BF16 && (dk > 32 || dv > 32);
    return tokens <= (quick_chunk ? 11 : EVFLY_DECAY_STEP_TOKENS);
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// a buffer of states that shares some of its bytes with another one: a block would write what another still reads
bool overlaps(const float *a, const float *b, int64_t floats) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && (x < y ? y - x : x - y) < (uintptr_t)floats * 4;
}

struct Tokens {              // one token tensor: pointer, element strides, heads of the pass per head of it, width
    const void *p;
    int64_t s[3];
    int r, d;
};

// One call's passes: roles filled in, tiles chosen, launched together where the tiles agree.
struct Run {
    int dtype;
    hipStream_t st;
    DecayPass base;                        // what all passes share

    DecayPass pass(const Tokens &a, const Tokens &b, const Tokens &c) const {
        DecayPass p = base;
        p.a = a.p; p.b = b.p; p.c = c.p;
        for (int i = 0; i < 3; ++i) { p.as[i] = a.s[i]; p.bs[i] = b.s[i]; p.cs[i] = c.s[i]; }
        p.ra = a.r; p.rb = b.r; p.rc = c.r;
        p.da = a.d; p.dc = c.d;
        return p;
    }
    int launch(const DecayPasses &ps, bool state) const {
        return dtype == EVFLY_DTYPE_F32 ? decay_passes_f32(ps, state, st) : decay_passes_bf16(ps, state, st);
    }
    // slots of up to two state sequences [dk][dv], each from its own state pass
    int segment_states(const DecayPass *own, int np, int dk, int dv) const {
        DecayPasses ps{};
        ScanArgs sc{};
        ps.np = np;
        for (int i = 0; i < np; ++i) { ps.p[i] = own[i]; sc.slots[i] = own[i].seg; sc.s_in[i] = own[i].s_in; }
        if (int rc = launch(ps, true)) return rc;
        sc.log_decay = base.log_decay; sc.lengths = base.lengths; sc.T = base.T; sc.H = base.H; sc.nseg = base.nseg; sc.seg_len = base.seg_len; sc.elems = dk * dv;
        hipLaunchKernelGGL(k_decay_scan, dim3((unsigned)(base.n * base.H), (dk * dv + 255) / 256, np), dim3(256), 0, st, sc);
        EVFLY_LAUNCH_CHECK();
        return 0;
    }
};

struct Ws { int64_t seg_floats, part_k, part_v, bytes; };      // part_*: offsets in bytes
Ws decay_ws(int n, int T, int H, int KV, int dk, int dv, int dtype, bool backward) {
    auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    Ws w{0, 0, 0, 0};
    if (T > EVFLY_DECAY_STEP_TOKENS || backward) {
        const DecaySplit sp = decay_split(n, T, H, dk, dv, dtype, backward);
        if (sp.nseg > 1) w.seg_floats = up((int64_t)n * H * sp.nseg * dk * dv * 4) / 4;
    }
    w.part_k = w.seg_floats * 4 * (backward ? 2 : 1);
    w.part_v = w.part_k + (backward && H != KV ? up((int64_t)n * T * H * dk * 4) : 0);
    w.bytes = w.part_v + (backward && H != KV ? up((int64_t)n * T * H * dv * 4) : 0);
    return w;
}

int check_shape(const char *who, int n, int T, int H, int KV, int dk, int dv, int dtype, float scale) {
    EVFLY_REQUIRE(n >= 0 && T >= 0 && T <= (1 << 30), "%s: %d streams of %d tokens", who, n, T);
    EVFLY_REQUIRE(H > 0 && KV > 0 && H % KV == 0, "%s: %d heads do not share %d key / value heads evenly", who, H, KV);
    EVFLY_REQUIRE(dk > 0 && dv > 0 && dk <= EVFLY_DECAY_MAX_DIM && dv <= EVFLY_DECAY_MAX_DIM, "%s: head sizes %d, %d are not in 1 .. %d", who, dk, dv, EVFLY_DECAY_MAX_DIM);
    EVFLY_REQUIRE(dtype == EVFLY_DTYPE_F32 || dtype == EVFLY_DTYPE_BF16, "%s: dtype %d (EVFLY_DTYPE_F32 or EVFLY_DTYPE_BF16)", who, dtype);
    EVFLY_REQUIRE(std::isfinite(scale), "%s: scale is not finite", who);
    EVFLY_REQUIRE((int64_t)n * H <= UINT32_MAX / 256, "%s: %d streams of %d heads", who, n, H);      // (a launch counts its threads in 32 bits)
    return 0;
}

void token_strides(const int64_t *s, int T, int heads, int d, int64_t (&out)[3]) {
    if (s) { out[0] = s[0]; out[1] = s[1]; out[2] = s[2]; }
    else { out[0] = (int64_t)T * heads * d; out[1] = (int64_t)heads * d; out[2] = d; }
}

}  // namespace

// Segments of a sequence. More of them fill the CUs and shorten the longest chain of chunks, but each cut makes two of the token tensors read twice (the state
// pass, 0.4 of a chunk's work) and adds two launches. The split with the smallest estimate, in us, is taken:
//     (chunks per segment + 1/2) * t * max(1, share * blocks per CU)      for each launch of the pass and, at 0.4 t, for the state pass
//     + 5 + 0.15 * segments                                               if it is cut at all (the scan over the borders)
// with t the time of a lone block's chunk (by type and a dimension) and `share` what a block uses of its CU. It ranks the splits, it does not tell their times (30 and 317 where 49 and
// 276 are measured). Against sweeps of 1 .. 64 segments on thirteen shapes, forward and backward (profiles/temporal_segments.txt), the choice is within 4 % of the best in 24
// of 26 and 11 and 15 % off in two; us forward / backward, chosen and neighbours: 8 x 4096 tokens x 16 heads x 64 bf16, four 100 forward (two 133, eight 110), two 212
// backward (one 228, four 219); 1 x 16384 x 4 x 64 bf16, 64 segments 49 forward (16: 73); 1 x 32768 x 16 x 128 bf16, 16 segments 271-281 (8: 372, 32: 288); 6 x
// 500 x 8 x 40 / 72 fp32, eight 33 / 84 (four 37 / 90, one 53 / 131); 16 x 1000 x 8 x 32 bf16, four 26 forward (one 30), one 36 backward (two 40).
namespace {
int col_tiles(int c) { return (c + decay_tile_c(c) - 1) / decay_tile_c(c); }
// the gradients' passes have their roles exchanged: one launch serves all three if both head sizes have the same tiles
bool decay_one_launch(int dk, int dv) {
    return decay_tile_a(dk) == decay_tile_a(dv) && decay_tile_c(dk) == decay_tile_c(dv) && col_tiles(dk) == col_tiles(dv);
}
}  // namespace
DecaySplit decay_split(int n, int T, int H, int dk, int dv, int dtype, bool backward) {
    const bool f32 = dtype == EVFLY_DTYPE_F32;
    const double rows = (double)n * H, share = f32 ? 0.7 : 0.8;
    const int chunks = (T + DECAY_CHUNK - 1) / DECAY_CHUNK;
    auto launch_cost = [&](int a, double blocks) {
        const int DA = decay_tile_a(a);
        const double busy = std::ceil(blocks / kNumCU) * share;
        return (f32 ? 4.0 : 2.5) * (DA == 128 ? 1.7 : DA == 64 ? 1.0 : 0.6) * (busy > 1.0 ? busy : 1.0);
    };
    DecaySplit best{1, DECAY_CHUNK * (chunks > 0 ? chunks : 1)};
    double least = INFINITY;
    for (int want = 1; want <= chunks && (want == 1 || rows * want <= 16 * kNumCU); want += want < 32 ? 1 : want / 8) {
        const int per = (chunks + want - 1) / want, nseg = (chunks + per - 1) / per;
        double cost;
        if (!backward) cost = launch_cost(dk, rows * nseg * col_tiles(dv));
        else if (decay_one_launch(dk, dv)) cost = launch_cost(dk, rows * nseg * col_tiles(dv) * 3);
        else cost = launch_cost(dv, rows * nseg * col_tiles(dk) * 2) + launch_cost(dk, rows * nseg * col_tiles(dv));
        if (nseg > 1) cost += 0.4 * launch_cost(dk, rows * (nseg - 1) * col_tiles(dv) * (backward ? 2 : 1));
        cost = cost * (per + 0.5) + (nseg > 1 ? 5.0 + 0.15 * nseg : 0.0);
        if (cost < 0.99 * least) {
            least = cost;
            best = DecaySplit{nseg, per * DECAY_CHUNK};
        }
    }
    return best;
}

}  // namespace evfly

using namespace evfly;

extern "C" int64_t evfly_decay_attention_workspace_bytes(int n_streams, int tokens, int heads, int kv_heads, int dk, int dv, int dtype,
                                                         int backward) {
    if (check_shape("decay_attention_workspace_bytes", n_streams, tokens, heads, kv_heads, dk, dv, dtype, 1.f)) return -1;
    return decay_ws(n_streams, tokens, heads, kv_heads, dk, dv, dtype, backward != 0).bytes;
}

extern "C" int evfly_decay_attention_forward(const void *q, const void *k, const void *v, const int64_t *strides_host,
                                             const float *log_decay, const float *state_in, const int32_t *lengths, int n_streams,
                                             int tokens, int heads, int kv_heads, int dk, int dv, float scale, int dtype, void *out,
                                             float *state_out, void *workspace, int64_t workspace_bytes, void *stream) {
    if (int rc = check_shape("decay_attention_forward", n_streams, tokens, heads, kv_heads, dk, dv, dtype, scale)) return rc;
    if (n_streams == 0) return 0;
    EVFLY_REQUIRE(log_decay && (tokens == 0 || (q && k && v && out)), "decay_attention_forward: null argument");
    const Ws ws = decay_ws(n_streams, tokens, heads, kv_heads, dk, dv, dtype, false);
    EVFLY_REQUIRE(workspace_bytes >= ws.bytes && (ws.bytes == 0 || (workspace && aligned16(workspace))),
                  "decay_attention_forward: workspace smaller than evfly_decay_attention_workspace_bytes, or not 16-byte aligned");
    EVFLY_REQUIRE(state_in == state_out || !overlaps(state_in, state_out, (int64_t)n_streams * heads * dk * dv),
                  "decay_attention_forward: state_in and state_out overlap in part");
    hipStream_t st = as_stream(stream);
    const int rep = heads / kv_heads;
    Tokens tq{q, {}, 1, dk}, tk{k, {}, rep, dk}, tv{v, {}, rep, dv};
    token_strides(strides_host, tokens, heads, dk, tq.s);
    token_strides(strides_host ? strides_host + 3 : nullptr, tokens, kv_heads, dk, tk.s);
    token_strides(strides_host ? strides_host + 6 : nullptr, tokens, kv_heads, dv, tv.s);
    if (recurrent(tokens, dk, dv, dtype)) {
        StepArgs a;
        a.q = q; a.k = k; a.v = v;
        for (int i = 0; i < 3; ++i) { a.qs[i] = tq.s[i]; a.ks[i] = tk.s[i]; a.vs[i] = tv.s[i]; }
        a.log_decay = log_decay; a.s_in = state_in; a.s_out = state_out; a.lengths = lengths; a.out = out;
        a.T = tokens; a.H = heads; a.rep = rep; a.dk = dk; a.dv = dv; a.scale = scale;
        return dtype == EVFLY_DTYPE_F32 ? step_all<float>(a, n_streams, st) : step_all<bf16_t>(a, n_streams, st);
    }
    Run run{dtype, st, DecayPass{}};
    const DecaySplit sp = decay_split(n_streams, tokens, heads, dk, dv, dtype, false);
    DecayPass &b = run.base;
    b.log_decay = log_decay; b.lengths = lengths; b.n = n_streams; b.T = tokens; b.H = heads; b.nseg = sp.nseg; b.seg_len = sp.seg_len;
    b.seg = static_cast<float *>(workspace); b.s_in = state_in; b.s_a = dv; b.s_c = 1;
    DecayPasses ps{};
    ps.np = 1;
    ps.p[0] = run.pass(tq, tk, tv);
    ps.p[0].out = out; ps.p[0].s_fin = state_out; ps.p[0].f_intra = scale; ps.p[0].f_out = scale; ps.p[0].f_upd = 1.f;
    if (sp.nseg > 1)
        if (int rc = run.segment_states(ps.p, 1, dk, dv)) return rc;
    return run.launch(ps, false);
}

extern "C" int evfly_decay_attention_backward(const void *q, const void *k, const void *v, const int64_t *strides_host,
                                              const float *log_decay, const float *state_in, const int32_t *lengths, const void *d_out,
                                              const float *d_state_out, int n_streams, int tokens, int heads, int kv_heads, int dk, int dv,
                                              float scale, int dtype, void *dq, void *dk_out, void *dv_out, float *d_state_in, void *workspace,
                                              int64_t workspace_bytes, void *stream) {
    if (int rc = check_shape("decay_attention_backward", n_streams, tokens, heads, kv_heads, dk, dv, dtype, scale)) return rc;
    if (n_streams == 0) return 0;
    EVFLY_REQUIRE(log_decay && (tokens == 0 || (q && k && v && d_out && dq && dk_out && dv_out)), "decay_attention_backward: null argument");
    const Ws ws = decay_ws(n_streams, tokens, heads, kv_heads, dk, dv, dtype, true);
    EVFLY_REQUIRE(workspace_bytes >= ws.bytes && (ws.bytes == 0 || (workspace && aligned16(workspace))),
                  "decay_attention_backward: workspace smaller than evfly_decay_attention_workspace_bytes, or not 16-byte aligned");
    hipStream_t st = as_stream(stream);
    const int rep = heads / kv_heads;
    Tokens tq{q, {}, 1, dk}, tk{k, {}, rep, dk}, tv{v, {}, rep, dv}, to{d_out, {}, 1, dv};
    token_strides(strides_host, tokens, heads, dk, tq.s);
    token_strides(strides_host ? strides_host + 3 : nullptr, tokens, kv_heads, dk, tk.s);
    token_strides(strides_host ? strides_host + 6 : nullptr, tokens, kv_heads, dv, tv.s);
    token_strides(nullptr, tokens, heads, dv, to.s);
    const int64_t states = (int64_t)n_streams * heads * dk * dv;
    EVFLY_REQUIRE(!overlaps(d_state_in, state_in, states) && !overlaps(d_state_in, d_state_out, states),
                  "decay_attention_backward: d_state_in shares memory with state_in or d_state_out");
    Run run{dtype, st, DecayPass{}};
    const DecaySplit sp = decay_split(n_streams, tokens, heads, dk, dv, dtype, true);
    char *const w = static_cast<char *>(workspace);
    float *const seg = reinterpret_cast<float *>(w), *const part_k = reinterpret_cast<float *>(w + ws.part_k), *const part_v = reinterpret_cast<float *>(w + ws.part_v);
    DecayPass &b = run.base;
    b.log_decay = log_decay; b.lengths = lengths; b.n = n_streams; b.T = tokens; b.H = heads; b.nseg = sp.nseg; b.seg_len = sp.seg_len;
    b.f_intra = scale;

    // dq_t = scale sum_{s <= t} e^{g (t - s)} (d_out_t . v_s) k_s + scale e^{g (t + 1)} S_in d_out_t: the state's own sequence, read transposed
    DecayPass pq = run.pass(to, tv, tk);
    pq.out = dq; pq.seg = seg; pq.s_in = state_in; pq.s_a = 1; pq.s_c = dv; pq.f_out = scale; pq.f_upd = 1.f;
    // dk_s = scale sum_{t >= s} e^{g (t - s)} (v_s . d_out_t) q_t + e^{g (T - 1 - s)} d_state_out v_s: backwards over the state's gradient, read transposed
    DecayPass pk = run.pass(tv, to, tq);
    pk.rev = 1; pk.out = rep > 1 ? static_cast<void *>(part_k) : dk_out; pk.out_f32 = rep > 1;
    pk.seg = seg + ws.seg_floats; pk.s_in = d_state_out; pk.s_a = 1; pk.s_c = dv; pk.f_out = 1.f; pk.f_upd = scale;
    // dv_s = scale sum_{t >= s} e^{g (t - s)} (k_s . q_t) d_out_t + e^{g (T - 1 - s)} d_state_out^T k_s; the state it ends with is state_in's gradient
    DecayPass pv = run.pass(tk, tq, to);
    pv.rev = 1; pv.out = rep > 1 ? static_cast<void *>(part_v) : dv_out; pv.out_f32 = rep > 1;
    pv.seg = seg + ws.seg_floats; pv.s_in = d_state_out; pv.s_fin = d_state_in; pv.s_a = dv; pv.s_c = 1; pv.f_out = 1.f; pv.f_upd = scale;
    if (sp.nseg > 1) {
        // the state k v^T and its gradient q d_out^T, both [dk][dv]
        DecayPass own[2] = {run.pass(tk, tk, tv), pv};
        own[0].seg = seg; own[0].s_in = state_in; own[0].s_a = dv; own[0].s_c = 1; own[0].f_upd = 1.f;
        if (int rc = run.segment_states(own, 2, dk, dv)) return rc;
    }
    DecayPasses ps{};
    ps.p[0] = pq; ps.p[1] = pk; ps.p[2] = pv;
    if (decay_one_launch(dk, dv)) {
        ps.np = 3;
        if (int rc = run.launch(ps, false)) return rc;
    } else {
        ps.np = 2;
        if (int rc = run.launch(ps, false)) return rc;
        ps.np = 1;
        ps.p[0] = pv;
        if (int rc = run.launch(ps, false)) return rc;
    }
    if (rep > 1 && tokens > 0) {
        HeadSum h{{part_k, part_v}, {dk_out, dv_out}, {dk, dv}, (int64_t)n_streams * tokens * kv_heads, rep};
        const int64_t need = (h.heads * (dk > dv ? dk : dv) + 255) / 256;
        const dim3 grid((unsigned)(need < 8 * kNumCU ? need : 8 * kNumCU), 2);
        if (dtype == EVFLY_DTYPE_F32) hipLaunchKernelGGL(k_decay_head_sum<float>, grid, dim3(256), 0, st, h);
        else hipLaunchKernelGGL(k_decay_head_sum<bf16_t>, grid, dim3(256), 0, st, h);
    }
    EVFLY_LAUNCH_CHECK();
    return 0;
}
