// The chunked kernel of decay attention for one element type (included by decay_f32.hip and decay_bf16.hip).
//
// A chunk of 64 tokens (local index i = t - t0) against the state S that the chunks before it left:
//     out_i = f_out e^{g (i + o)} a_i S  +  sum_{j <= i} f_intra e^{g (i - j)} (a_i . b_j) c_j
//     S'    = e^{g cnt} S  +  sum_j f_upd e^{g (cnt - j - o)} b_j c_j^T                 cnt tokens in the chunk; o = 1 forwards, 0 backwards
// Every exponent is a whole number of steps in [0, 64], so one table of 65 powers per head serves all of them and no weight is the quotient of two
// others. All four products run on 16x16 MFMAs with token columns: P^T = b a^T leaves, in a lane, pair weights of one token i against
// four neighbouring j, which is the operand layout of out^T = c^T P^T -- the pair products never leave registers.
//
// Work: one block of four waves per (stream, head, tile of DC columns of c, segment); wave w owns 16 of the chunk's tokens of the output and a share of
// the state's a-rows. The a rows go from memory to the wave's registers, b and c through LDS (read as rows for P, as columns for the other two
// products), S lives in the accumulators and is copied to LDS once per chunk as an operand of a_i S. The next chunk's rows are in flight during the products.
//
// Bounds (medians under the profiler). bf16, 64 wide (8 x 4096 tokens x 16 heads): a pass moves 268 MB in 76 us, 3.5 TB/s of the 4.9 that a copy reaches here. bf16,
// 128 wide (1 x 32768 x 16): 220 us; counted busy are the matrix pipes 35 %, vector issue 57 %, LDS 61 % of the time (46 % of its cycles conflicts): two waves per SIMD
// (78 KB of LDS a block, 51 of them the state's three parts) overlap them only in part. fp32: the 16x16x4 products, 45 % of their pipe's time at 48 / 96 wide with two blocks a CU.
#pragma once
#include "bf16.h"
#include "decay.h"

namespace evfly {
namespace decay {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

// Element-type side: a fragment is 16 bytes per lane = KB / 4 values of the summed index (KB per MFMA step over the four lane groups).
template <typename T> struct Mm;

template <> struct Mm<float> {
    static constexpr int KB = 16;       // values of the summed index per fragment
    static constexpr int TILES = 1;     // 16-row tiles of it
    static constexpr int NP = 1;        // parts of an fp32 value as an operand
    typedef f32x4 frag;
    __device__ static __forceinline__ frag load(const char *lds) { return *reinterpret_cast<const frag *>(lds); }
    __device__ static __forceinline__ f32x4 mma(frag a, frag b, f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
    // column `col` of rows 16 kb + 4 g .. + 3 of a row-major tile (row stride rsb bytes)
    __device__ static __forceinline__ frag load_col(const char *tile, int rsb, int kb, int g, int col) {
        frag f;
        const char *p = tile + (16 * kb + 4 * g) * rsb + col * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = *reinterpret_cast<const float *>(p + i * rsb);
        return f;
    }
    __device__ static __forceinline__ void weigh(frag b, const float *w, frag (&o)[NP]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[0][i] = b[i] * w[i];
    }
    __device__ static __forceinline__ void split(const f32x4 *acc, frag (&o)[NP]) { o[0] = acc[0]; }
    __device__ static __forceinline__ void put_state(char *p, int, f32x4 s) { *reinterpret_cast<f32x4 *>(p) = s; }
};

// hi + mid + lo of an fp32 value as bf16 (8 + 8 + 8 significant bits, each part the rounding of what the parts before it left): all of its 24 bits, so that pair
// products, state and update enter the products as the fp32 values they are. (Two parts carry 17 bits: the 2-norm distance of bf16 results from those of a form
// in fp32 is then 9.6e-5 of theirs instead of 3.3e-5, 8 x 4096 tokens x 16 heads x 64 with gradients, 300 us against 322; 1 x 32768 x 16 x 128 forward, 9.5e-5
// instead of 3.6e-5, 270 us against 297.) An infinity, or a value within 2^-9 of the largest float, leaves NaN to the next part.
template <> struct Mm<bf16_t> {
    static constexpr int KB = 32;
    static constexpr int TILES = 2;
    static constexpr int NP = 3;
    typedef bf16x8 frag;
    union U { uint4 u; frag f; i16x4 h[2]; };
    __device__ static __forceinline__ frag load(const char *lds) { return *reinterpret_cast<const frag *>(lds); }
    __device__ static __forceinline__ f32x4 mma(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    // summed index in the order of two accumulator tiles: values 0..3 = rows 32 kb + 4 g + e, values 4..7 = rows 32 kb + 16 + 4 g + e. The transposed LDS
    // read takes, for 16 lanes, the addresses of four rows of four 8-byte pieces and hands lane l column l of the four rows.
    __device__ static __forceinline__ frag load_col(const char *tile, int rsb, int kb, int g, int col) {
        const int l = col & 15, c0 = col & ~15;
        const char *p = tile + (32 * kb + 4 * g + (l >> 2)) * rsb + (c0 + 4 * (l & 3)) * 2;
        U r;
        typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
        r.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(p));
        r.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(p + 16 * rsb));
        return r.f;
    }
    __device__ static __forceinline__ void parts(const float (&x)[8], frag (&o)[NP]) {
        float r[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = x[e];
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            unsigned w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[e] = pack_bf2(r[2 * e], r[2 * e + 1]);
                if (k + 1 < NP) {
                    r[2 * e] -= bf_lo(w[e]);
                    r[2 * e + 1] -= bf_hi(w[e]);
                }
            }
            U u;
            u.u = make_uint4(w[0], w[1], w[2], w[3]);
            o[k] = u.f;
        }
    }
    __device__ static __forceinline__ void weigh(frag b, const float *w, frag (&o)[NP]) {
        U u;
        u.f = b;
        const unsigned d[4] = {u.u.x, u.u.y, u.u.z, u.u.w};
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[2 * e] = bf_lo(d[e]) * w[2 * e];
            x[2 * e + 1] = bf_hi(d[e]) * w[2 * e + 1];
        }
        parts(x, o);
    }
    __device__ static __forceinline__ void split(const f32x4 *acc, frag (&o)[NP]) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) { x[e] = acc[0][e]; x[4 + e] = acc[1][e]; }
        parts(x, o);
    }
    // four neighbouring a-values of one column of S, a bf16 plane for each part
    __device__ static __forceinline__ void put_state(char *p, int plane, f32x4 s) {
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const unsigned h0 = pack_bf2(s[0], s[1]), h1 = pack_bf2(s[2], s[3]);
            *reinterpret_cast<uint2 *>(p + k * plane) = make_uint2(h0, h1);
            if (k + 1 < NP) s -= f32x4{bf_lo(h0), bf_hi(h0), bf_lo(h1), bf_hi(h1)};
        }
    }
};

template <typename T, int DA, int DC> struct Lds {
    static constexpr int RB = DA * (int)sizeof(T) + 16;        // row strides in bytes: 16 more than the row, so that 16 rows read at one column
    static constexpr int RC = DC * (int)sizeof(T) + 16;        // spread over the banks
    static constexpr int RS = DA * (int)sizeof(T) + 16;
    static constexpr int PW = 0, UW = 272, B = 1024, C = B + DECAY_CHUNK * RB, S = C + DECAY_CHUNK * RC;
    static constexpr int PLANE = DC * RS;
    static constexpr int STATE_BYTES = S, BYTES = S + PLANE * Mm<T>::NP;      // (a pass for the state alone has no use for S as an operand)
};

// Blocks that share a CU: as many as LDS and registers hold without spills.
template <typename T, int DA, int DC, bool STATE> constexpr int blocks_per_cu() {
    constexpr int regs = DA == 128 ? (sizeof(T) == 4 ? 2 : 3) : sizeof(T) == 4 ? 3 : 4;
    constexpr int fit = kMaxLds / (STATE ? Lds<T, DA, DC>::STATE_BYTES : Lds<T, DA, DC>::BYTES);
    return fit < regs ? fit : regs;
}

// STATE: the segment's own state only (no output), for the sequences that are split into segments. TAIL: a head size that is no whole number of 16-byte
// pieces (without it the loop is free of the branches of partial pieces: 8 x 4096 x 16 heads x 64, bf16, measured with two parts a value: 70 us a pass against 76).
template <typename T, int DA, int DC, bool STATE, bool TAIL>
__global__ __launch_bounds__(256, (blocks_per_cu<T, DA, DC, STATE>())) void k_decay_chunk(DecayPasses ps) {
    typedef Mm<T> M;
    typedef typename M::frag frag;
    typedef Lds<T, DA, DC> L;
    constexpr int C = DECAY_CHUNK, V = 16 / sizeof(T);
    constexpr int KA = DA / M::KB;                   // fragments along a
    constexpr int KS = C / M::KB;                    // fragments along the chunk
    constexpr int NC = DC / 16;                      // 16-column tiles of c
    constexpr int NA = DA >= 64 ? DA / 64 : 1;       // the wave's share of the state: NA a-tiles by NCW c-tiles
    constexpr int NCW = DA >= 64 ? NC : NC / 2;
    // products with nothing but zeros (pairs with later tokens, tiles behind the head size): fp32, bound by its products, leaves them out; in bf16 the
    // branches around them cost more
    constexpr bool SKIP = sizeof(T) == 4;
    constexpr int NB = C * DA / V / 256, NV = C * DC / V / 256;      // 16-byte pieces per thread of a chunk of b and c
    static_assert(NB >= 1 && NV >= 1, "a chunk is at least one piece per thread");
    extern __shared__ __align__(16) char lds[];
    float *const pw = reinterpret_cast<float *>(lds + L::PW), *const uw = reinterpret_cast<float *>(lds + L::UW);

    // (the waves' shares of the tokens turn with the block: later tokens have more pairs, and a last chunk may have only early ones)
    const int tid = threadIdx.x, lane = tid & 63, l = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), wt = (w + blockIdx.x / kNumXCD) & 3;
    // blocks of one XCD (block index mod 8) take neighbouring work: the heads of a token share cache lines, shared heads and column tiles share rows
    const int total = gridDim.x, q8 = total / kNumXCD, r8 = total % kNumXCD, xcd = blockIdx.x % kNumXCD;
    int id = xcd * q8 + min(xcd, r8) + blockIdx.x / kNumXCD;
    const DecayPass &p = ps.p[id % ps.np]; id /= ps.np;
    const int nseg = STATE ? p.nseg - 1 : p.nseg, ndc = (p.dc + DC - 1) / DC;
    const int wide = ((p.dc + ndc - 1) / ndc + 15) / 16 * 16;            // columns per block, evenly shared (96: 48 and 48)
    const int c0 = (id % ndc) * wide; id /= ndc;
    const int h = id % p.H; id /= p.H;
    const int seg = id % nseg;
    const int n = id / nseg;

    const int len = p.lengths ? min(max(p.lengths[n], 0), p.T) : p.T;
    const int u_lo = seg * p.seg_len, u_hi = min(u_lo + p.seg_len, p.T), u_end = min(u_hi, len);
    const int dcw = max(0, min(p.dc - c0, wide));    // columns of this tile
    const int o = p.rev ? 0 : 1;
    const T *const ap = static_cast<const T *>(p.a) + n * p.as[0] + (h / p.ra) * p.as[2];
    const T *const bp = static_cast<const T *>(p.b) + n * p.bs[0] + (h / p.rb) * p.bs[2];
    const T *const cp = static_cast<const T *>(p.c) + n * p.cs[0] + (h / p.rc) * p.cs[2] + c0;
    const int64_t st_base = ((int64_t)n * p.H + h) * p.da * p.dc;
    const int64_t ot = (int64_t)p.H * p.dc;          // output elements per token
    const int64_t ob = ((int64_t)n * p.T * p.H + h) * p.dc + c0;

    // pw[m] = e^{g m}; uw[x] = the state update's weight of a row that is followed by 63 - x others (0: there is no such row)
    if (tid <= C) pw[tid] = tid == 0 ? 1.f : expf(p.log_decay[h] * (float)tid);
    if (tid < 2 * C) {
        const int m = C - tid - o;
        uw[tid] = tid >= C ? 0.f : m == 0 ? p.f_upd : p.f_upd * expf(p.log_decay[h] * (float)m);
    }

    // ---- the state: rows a = 16 (a-tile) + 4 g + i, column c = 16 (c-tile) + l
    const int a_t0 = DA >= 64 ? w * NA : w & 1, c_t0 = DA >= 64 ? 0 : (w >> 1) * NCW;
    f32x4 S[NA][NCW];
    float *const slots = p.seg + st_base * p.nseg;                           // (nseg > 1)
    const int64_t state_n = (int64_t)p.da * p.dc;
    const float *const start = STATE ? nullptr : p.nseg > 1 ? slots + seg * state_n : p.s_in ? p.s_in + st_base : nullptr;
    auto each_state = [&](auto fn) {
#pragma unroll
        for (int x = 0; x < NA; ++x)
#pragma unroll
            for (int y = 0; y < NCW; ++y)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int a = 16 * (a_t0 + x) + 4 * g + i, c = 16 * (c_t0 + y) + l;
                    S[x][y][i] = fn(S[x][y][i], a < p.da && c < dcw, a * p.s_a + (c0 + c) * p.s_c);
                }
    };
    each_state([&](float, bool in, int64_t at) { return start && in ? start[at] : 0.f; });

    // rows of the next chunk: this thread's piece of b and c (16-byte pieces RPB, RPC rows apart) and its token's a row. Row pointers step by a whole chunk
    constexpr int RPB = 256 / (DA / V), RPC = 256 / (DC / V);
    uint4 rb[NB], rc[NV];
    frag fa[KA], fa_next[KA];
    const int dir = p.rev ? -1 : 1, first = p.rev ? len - 1 - u_lo : u_lo;
    const int br = tid / (DA / V), bcol = tid % (DA / V) * V, cr = tid / (DC / V), ccol = tid % (DC / V) * V, ar = 16 * wt + l;
    const T *bq = bp + (int64_t)(first + dir * br) * p.bs[1] + bcol, *cq = cp + (int64_t)(first + dir * cr) * p.cs[1] + ccol;
    const T *aq = ap + (int64_t)(first + dir * ar) * p.as[1] + g * V;
    const int64_t bstep = dir * RPB * p.bs[1], cstep = dir * RPC * p.cs[1], astep = dir * C * p.as[1];
    auto fetch = [&](int u0) {
        const int left = u_end - u0;                 // rows of the chunk that are there
#pragma unroll
        for (int x = 0; x < NB; ++x, bq += bstep) {
            rb[x] = make_uint4(0, 0, 0, 0);
            if (br + x * RPB < left) rb[x] = load_piece<T, TAIL>(bq, p.da - bcol);
        }
#pragma unroll
        for (int x = 0; x < NV; ++x, cq += cstep) {
            rc[x] = make_uint4(0, 0, 0, 0);
            if (cr + x * RPC < left) rc[x] = load_piece<T, TAIL>(cq, dcw - ccol);
        }
        if (!STATE) {
#pragma unroll
            for (int k = 0; k < KA; ++k) {
                union { uint4 u4; frag f; } t;
                t.u4 = make_uint4(0, 0, 0, 0);
                if (ar < left) t.u4 = load_piece<T, TAIL>(aq + k * M::KB, p.da - k * M::KB - g * V);
                fa_next[k] = t.f;
            }
            aq += astep;
        }
    };
    int64_t oi = ob + (int64_t)(first + dir * ar) * ot;
    const int64_t ostep = dir * C * ot;
    if (u_lo < u_end) fetch(u_lo);
    __syncthreads();

    // ---- weights of the pairs of token i = 16 wt + l with j = 16 st + 4 g + e, the same in every chunk
    float wp[4][4];
#pragma unroll
    for (int st = 0; st < 4; ++st)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = 16 * st + 4 * g + e, d = 16 * wt + l - j;
            wp[st][e] = d >= 0 ? p.f_intra * pw[max(d, 0)] : 0.f;
        }
    const float w_out = p.f_out * pw[16 * wt + l + o];

    // fp32: a chunk's sum is formed apart and joined to the state behind the barrier, one rounding at the state's size instead of one per product of four tokens (4 x
    // 2777 tokens x 8 heads x 48 / 96: error of the state 3.0e-7 -> 1.6e-7 of it, of the output 3.4e-7 -> 2.4e-7, 82 -> 83 us; joined in front of the barrier 89: the last
    // products are waited for there). bf16 has two products of 32 tokens for each part: 2.2e-7 as it is, 1.5e-7 apart (a form in fp32 1.8e-7), for 1.5 % of the time.
    constexpr bool APART = sizeof(T) == 4;
    f32x4 U[NA][NCW];
    f32x4 (&to)[NA][NCW] = APART ? U : S;
    float keep = 1.f;
    auto join = [&]() {
        if (APART)
#pragma unroll
            for (int x = 0; x < NA; ++x)
#pragma unroll
                for (int y = 0; y < NCW; ++y)
#pragma unroll
                    for (int e = 0; e < 4; ++e) S[x][y][e] = fmaf(keep, S[x][y][e], U[x][y][e]);
    };

    for (int u0 = u_lo; u0 < u_end; u0 += C) {
        const int cnt = min(C, u_end - u0);
        if (u0 > u_lo) {
            __syncthreads();                         // the products of the chunk before have read their tiles
            join();
        }
#pragma unroll
        for (int x = 0; x < NB; ++x)
            *reinterpret_cast<uint4 *>(lds + L::B + (br + x * RPB) * L::RB + bcol * (int)sizeof(T)) = rb[x];
#pragma unroll
        for (int x = 0; x < NV; ++x)
            *reinterpret_cast<uint4 *>(lds + L::C + (cr + x * RPC) * L::RC + ccol * (int)sizeof(T)) = rc[x];
        if (!STATE) {
#pragma unroll
            for (int x = 0; x < NA; ++x)
#pragma unroll
                for (int y = 0; y < NCW; ++y)
                    M::put_state(lds + L::S + (16 * (c_t0 + y) + l) * L::RS + (16 * (a_t0 + x) + 4 * g) * (int)sizeof(T), L::PLANE, S[x][y]);
#pragma unroll
            for (int k = 0; k < KA; ++k) fa[k] = fa_next[k];
        }
        __syncthreads();
        if (u0 + C < u_end) fetch(u0 + C);

        // (a wave that forms its output goes ahead of one that updates its state: of two waves on a SIMD one then feeds the matrix pipe while the other does
        // its vector work; 32768 x 16 heads x 128, bf16, 282 -> 273 us, 8 x 4096 x 16 x 64 with gradients 311 -> 304)
        __builtin_amdgcn_s_setprio(1);
        if (!STATE && 16 * wt < cnt) {
            // ---- P^T tiles of this wave's tokens (j-tiles up to its own), weighted, as operand parts
            frag P[KS][M::NP];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (SKIP && ks * M::TILES > wt) continue;
                f32x4 acc[M::TILES];
#pragma unroll
                for (int x = 0; x < M::TILES; ++x) {
                    const int st = ks * M::TILES + x;
                    acc[x] = f32x4{0.f, 0.f, 0.f, 0.f};
                    if (SKIP && st > wt) continue;
#pragma unroll
                    for (int k = 0; k < KA; ++k)
                        if (!SKIP || k * M::KB < p.da) acc[x] = M::mma(M::load(lds + L::B + (16 * st + l) * L::RB + k * 64 + g * 16), fa[k], acc[x]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[x][e] *= wp[st][e];
                }
                M::split(acc, P[ks]);
            }
            // ---- out^T = w_out S^T a^T + c^T P^T
            const bool there = u0 + ar < u_end;
#pragma unroll
            for (int y = 0; y < NC; ++y) {
                if (SKIP && 16 * y >= dcw) continue;
                f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KA; ++k)
#pragma unroll
                    for (int x = 0; x < M::NP; ++x)
                        if (!SKIP || k * M::KB < p.da) acc = M::mma(M::load(lds + L::S + x * L::PLANE + (16 * y + l) * L::RS + k * 64 + g * 16), fa[k], acc);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] *= w_out;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    if (SKIP && ks * M::TILES > wt) continue;
                    const frag fc = M::load_col(lds + L::C, L::RC, ks, g, 16 * y + l);
#pragma unroll
                    for (int x = 0; x < M::NP; ++x) acc = M::mma(fc, P[ks][x], acc);
                }
                const int c = 16 * y + 4 * g;
                if (there && c < dcw) {
                    const uint4 w4 = make_uint4(__float_as_uint(acc[0]), __float_as_uint(acc[1]), __float_as_uint(acc[2]), __float_as_uint(acc[3]));
                    if (sizeof(T) == 4 || p.out_f32) {
                        float *d = static_cast<float *>(p.out) + oi + c;
                        if (!TAIL || c + 4 <= dcw) store16_any(d, w4);
                        else
#pragma unroll
                            for (int e = 0; e < 3; ++e)
                                if (c + e < dcw) d[e] = acc[e];
                    } else {
                        T *d = static_cast<T *>(p.out) + oi + c;
                        if (!TAIL || c + 4 <= dcw) store8_any(d, make_uint2(pack_bf2(acc[0], acc[1]), pack_bf2(acc[2], acc[3])));
                        else
#pragma unroll
                            for (int e = 0; e < 3; ++e)
                                if (c + e < dcw) Elem<T>::st1(d + e, acc[e]);
                    }
                }
            }
        }
        __builtin_amdgcn_s_setprio(0);
        if (!STATE) oi += ostep;

        // ---- S = e^{g cnt} S + (w b)^T c
        keep = pw[cnt];
#pragma unroll
        for (int x = 0; x < NA; ++x)
#pragma unroll
            for (int y = 0; y < NCW; ++y)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (APART) U[x][y][e] = 0.f;
                    else S[x][y][e] *= keep;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            if (SKIP && ks * M::KB >= cnt) continue;
            float wu[M::TILES * 4];
#pragma unroll
            for (int e = 0; e < M::TILES * 4; ++e) wu[e] = uw[C - cnt + 16 * (ks * M::TILES + e / 4) + 4 * g + e % 4];
            frag fb[NA][M::NP];
#pragma unroll
            for (int x = 0; x < NA; ++x) M::weigh(M::load_col(lds + L::B, L::RB, ks, g, 16 * (a_t0 + x) + l), wu, fb[x]);
#pragma unroll
            for (int y = 0; y < NCW; ++y) {
                if (SKIP && 16 * (c_t0 + y) >= dcw) continue;
                const frag fc = M::load_col(lds + L::C, L::RC, ks, g, 16 * (c_t0 + y) + l);
#pragma unroll
                for (int x = 0; x < NA; ++x)
#pragma unroll
                    for (int z = 0; z < M::NP; ++z) to[x][y] = M::mma(fb[x][z], fc, to[x][y]);
            }
        }
    }

    if (u_lo < u_end) join();
    if (STATE) {
        float *const own = slots + (seg + 1) * state_n;
        each_state([&](float v, bool in, int64_t at) { if (in) own[at] = v; return v; });
        return;
    }
    // ---- rows behind the sequence are zero; the last segment ends with the state behind the whole sequence
    for (int64_t i = tid; i < (int64_t)max(0, u_hi - max(u_lo, len)) * dcw; i += 256) {
        const int64_t at = ob + (max(u_lo, len) + i / dcw) * ot + i % dcw;
        if (p.out_f32) static_cast<float *>(p.out)[at] = 0.f;
        else static_cast<T *>(p.out)[at] = T(0);
    }
    if (p.s_fin && seg == p.nseg - 1) each_state([&](float v, bool in, int64_t at) { if (in) p.s_fin[st_base + at] = v; return v; });
}

template <typename T, int DA, int DC, bool STATE, bool TAIL> int launch(const DecayPasses &ps, hipStream_t st) {
    constexpr int bytes = STATE ? Lds<T, DA, DC>::STATE_BYTES : Lds<T, DA, DC>::BYTES;
    static_assert(bytes <= kMaxLds, "LDS of one CU");
    const DecayPass &p = ps.p[0];
    const int64_t blocks = (int64_t)p.n * p.H * ((p.dc + DC - 1) / DC) * (STATE ? p.nseg - 1 : p.nseg) * ps.np;
    EVFLY_REQUIRE(blocks <= UINT32_MAX / 256, "decay_attention: %lld tiles of work", (long long)blocks);
    const auto kern = k_decay_chunk<T, DA, DC, STATE, TAIL>;
    static std::atomic<bool> attr_set[64];
    int dev = 0;
    EVFLY_HIP(hipGetDevice(&dev));
    EVFLY_REQUIRE(dev >= 0 && dev < 64, "device index %d out of range", dev);
    if (!attr_set[dev].load(std::memory_order_acquire)) {
        EVFLY_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        attr_set[dev].store(true, std::memory_order_release);
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), bytes, st, ps);
    EVFLY_LAUNCH_CHECK();
    return 0;
}

template <typename T, int DA, int DC> int launch_s(const DecayPasses &p, bool state, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    if (p.p[0].da % V || p.p[0].dc % V) return state ? launch<T, DA, DC, true, true>(p, st) : launch<T, DA, DC, false, true>(p, st);
    return state ? launch<T, DA, DC, true, false>(p, st) : launch<T, DA, DC, false, false>(p, st);
}
template <typename T> int launch_all(const DecayPasses &p, bool state, hipStream_t st) {
    const int DA = decay_tile_a(p.p[0].da);
    if (decay_tile_c(p.p[0].dc) == 32)
        return DA == 32 ? launch_s<T, 32, 32>(p, state, st) : DA == 64 ? launch_s<T, 64, 32>(p, state, st) : launch_s<T, 128, 32>(p, state, st);
    return DA == 32 ? launch_s<T, 32, 64>(p, state, st) : DA == 64 ? launch_s<T, 64, 64>(p, state, st) : launch_s<T, 128, 64>(p, state, st);
}

}  // namespace decay
}  // namespace evfly
