// Block norm: y = res_scale x + act(gate) norm_post(f), h = norm_pre(y), and its gradients. Bound by HBM: forward reads x, f (gate) and writes y, h once;
// backward reads x, f (gate), dy, dh, forms the forward's row again in registers and writes dx, df (d_gate) once, beside the column sums.
//
// A row is held by a group of G lanes in registers from its load to its stores, eight values per lane (one 16-byte piece of bf16, two of fp32, at
// any alignment), so G is the smallest power of two that covers the channels: rows of up to 512
// channels share waves, longer ones take a block of up to 1024 threads. Each group keeps its columns of every weight vector in registers over all the rows it
// visits. Mean and variance are two passes over the registers, fp32.
//
// Column sums (weights, biases, residual scale, a broadcast gate) are kept per lane over the block's rows, added over the block's groups in LDS, written
// as one partial row per block and added in block order by k_bn_columns: no atomics, the same bits on every call.
#include <atomic>
#include <cmath>

#include "bf16.h"
#include "common.h"

namespace evfly {
namespace {

constexpr int E = 8;                     // values per lane
constexpr int BN_MAX_BLOCKS = 2 * kNumCU;      // backward: blocks that carry column sums (each leaves one partial row per vector)

struct BnArgs {
    const void *f, *x, *gate;
    const float *alpha, *w1, *b1, *w2, *b2;
    void *y, *h;
    int post, pre, act, gate_f32, C;
    uint32_t rows, rpg;                  // rows, rows per gate row
    uint32_t span;                       // backward: rows that `parts` units share (those of a gate row, or all)
    float eps, inv_c;
    // backward
    const void *dy, *dh;
    void *df, *dx, *dgate;
    float *cols;                         // partial column sums [block][kind][C]: kinds alpha, w1, b1, w2, b2, gate
    float *gate_part;                    // partial gate rows [gate row][part][C] (parts > 1)
    int want;                            // bit per kind
    uint32_t unit_rows, parts, units;    // work units: contiguous rows of one gate row
};
enum { K_ALPHA, K_W1, K_B1, K_W2, K_B2, K_GATE, K_N };

// A lane's eight values are 16-byte pieces of VS neighbouring ones: value j lies in column ((j / VS) G + gl) VS + j % VS. Columns behind C read as zero. A
// row is fetched as it lies in memory (one row ahead of its use) and widened when its turn comes.
template <typename T> constexpr int VS = 16 / sizeof(T);
template <typename T, int G> __device__ __forceinline__ int column(int gl, int j) { return (j / VS<T> * G + gl) * VS<T> + j % VS<T>; }

template <typename T, int G> struct Row {
    uint4 raw[E / VS<T>];
    __device__ __forceinline__ void fetch(const T *row, int gl, int C) {
#pragma unroll
        for (int k = 0; k < E / VS<T>; ++k) {
            const int c = (k * G + gl) * VS<T>;
            raw[k] = load_piece<T, true>(row + c, C - c);
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int k = 0; k < E / VS<T>; ++k) raw[k] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void widen(float (&v)[E]) const {
#pragma unroll
        for (int k = 0; k < E / VS<T>; ++k) {
            float t[VS<T>];
            Elem<T>::load(reinterpret_cast<const T *>(&raw[k]), t);
#pragma unroll
            for (int i = 0; i < VS<T>; ++i) v[k * VS<T> + i] = t[i];
        }
    }
};
template <typename T, int G> __device__ __forceinline__ void store_row(T *row, int gl, int C, const float (&v)[E]) {
#pragma unroll
    for (int k = 0; k < E / VS<T>; ++k) {
        const int c = (k * G + gl) * VS<T>;
        float t[VS<T>];
#pragma unroll
        for (int i = 0; i < VS<T>; ++i) t[i] = v[k * VS<T> + i];
        if (c + VS<T> <= C) {
            uint4 u;
            Elem<T>::store(reinterpret_cast<T *>(&u), t);
            store16_any(row + c, u);
        } else if (c < C) {
#pragma unroll
            for (int i = 0; i < VS<T> - 1; ++i)
                if (c + i < C) Elem<T>::st1(row + c + i, t[i]);
        }
    }
}
// the same columns of an fp32 vector (`other` where there is none, and behind C)
template <typename T, int G> __device__ __forceinline__ void load_vec(const float *p, int gl, int C, float other, float (&v)[E]) {
#pragma unroll
    for (int j = 0; j < E; j += 4) {
        const int c = column<T, G>(gl, j);
        if (p && c + 4 <= C) {
            const uint4 u = load16_any(p + c);
            v[j] = __uint_as_float(u.x); v[j + 1] = __uint_as_float(u.y); v[j + 2] = __uint_as_float(u.z); v[j + 3] = __uint_as_float(u.w);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[j + i] = p && c + i < C ? p[c + i] : other;
        }
    }
}
// a gate row in its own type (the tokens' or fp32)
template <typename T, int G> __device__ __forceinline__ void load_gate(const BnArgs &p, int64_t row, int gl, float (&v)[E]) {
    if (p.gate_f32) {
        load_vec<T, G>(static_cast<const float *>(p.gate) + row * p.C, gl, p.C, 0.f, v);
    } else {
        Row<T, G> t;
        t.fetch(static_cast<const T *>(p.gate) + row * p.C, gl, p.C);
        t.widen(v);
    }
}
// e^x to about an ulp in nine instructions: 2^t with t = x log2(e) rounded, plus (what t's rounding dropped) ln 2 of it. From 80 on either way (1e35) the
// correction, up to 80 * 2^-24, is left out: infinities have none.
__device__ __forceinline__ float exp_ulp(float x) {
    const float t = x * 1.44269504f, lost = fmaf(x, 1.44269504f, -t) + x * 1.92596303e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    return fabsf(x) < 80.f ? fmaf(e, lost * 0.693147182f, e) : e;
}
// act(z) in place of z; slope = act'(z). (The reciprocal instruction's one ulp instead of a rounded division: with the square root's below 53 -> 43 us on 524288 gated rows of 64,
// bf16, where the arithmetic of a row costs as much as its bytes.)
__device__ __forceinline__ void activate(int act, float z, float &a, float &slope) {
    a = z;
    slope = 1.f;
    if (act == EVFLY_ACT_SIGMOID) {
        a = __builtin_amdgcn_rcpf(1.f + exp_ulp(-z));
        slope = a * (1.f - a);
    } else if (act == EVFLY_ACT_TANH) {
        a = tanhf(z);
        slope = 1.f - a * a;
    }
}

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// sum over aligned groups of G <= 64 lanes, in every lane
template <int G> __device__ __forceinline__ float lane_sum(float v) {
    if (G >= 2) v += dpp<0xB1>(v);          // quad_perm 1,0,3,2
    if (G >= 4) v += dpp<0x4E>(v);          // quad_perm 2,3,0,1
    if (G >= 8) v += dpp<0x141>(v);         // row_half_mirror
    if (G >= 16) v += dpp<0x140>(v);        // row_mirror
    if (G >= 32) v = sum_xor16(v);
    if (G >= 64) v = sum_xor32(v);
    return v;
}
// sums of N values over the G lanes of a row. G > 64: over the group's waves through `red` (two buffers in turn: one barrier per sum; every thread of the block comes here)
template <int G, int N> __device__ __forceinline__ void row_sum(float (&v)[N], float *red, int &turn) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lane_sum<(G > 64 ? 64 : G)>(v[i]);
    if constexpr (G > 64) {
        const int w = threadIdx.x >> 6;
        float *buf = red + (turn & 1) * 32;
        ++turn;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) buf[i * 16 + w] = v[i];
        __syncthreads();
        const int w0 = w / (G / 64) * (G / 64);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = 0.f;
#pragma unroll
            for (int k = 0; k < G / 64; ++k) v[i] += buf[i * 16 + w0 + k];
        }
    }
}
// v -> (v - mean) / sqrt(var + eps) in place (EVFLY_NORM_RMS: mean = 0); columns behind C stay zero. Returns 1 / sqrt(..).
template <typename T, int G> __device__ __forceinline__ float normalise(float (&v)[E], int kind, int gl, int C, float inv_c, float eps, float *red, int &turn) {
    float mu = 0.f;
    if (kind == EVFLY_NORM_LAYER) {
        float s[1] = {0.f};
#pragma unroll
        for (int j = 0; j < E; ++j) s[0] += v[j];
        row_sum<G>(s, red, turn);
        mu = s[0] * inv_c;
    }
    float q[1] = {0.f};
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const int c = column<T, G>(gl, j);
        v[j] = c < C ? v[j] - mu : 0.f;
        q[0] = fmaf(v[j], v[j], q[0]);
    }
    row_sum<G>(q, red, turn);
    // (the instruction takes a subnormal for zero: such a mean square is brought into the normal numbers and its root back)
    const float ms = fmaf(q[0], inv_c, eps);
    const bool tiny = ms < 0x1p-126f;
    const float r = __builtin_amdgcn_rsqf(tiny ? ms * 0x1p32f : ms) * (tiny ? 0x1p16f : 1.f);
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] *= r;
    return r;
}

template <typename T, int G> __global__ __launch_bounds__(G > 256 ? G : 256) void k_bn_fwd(BnArgs p) {
    constexpr int NT = G > 256 ? G : 256, GR = NT / G;
    __shared__ float red[64];
    int turn = 0;
    const int gl = threadIdx.x % G, gi = threadIdx.x / G;
    float w1[E], b1[E], w2[E], b2[E], al[E], a[E];
    load_vec<T, G>(p.w1, gl, p.C, 1.f, w1);
    load_vec<T, G>(p.b1, gl, p.C, 0.f, b1);
    load_vec<T, G>(p.w2, gl, p.C, 1.f, w2);
    load_vec<T, G>(p.b2, gl, p.C, 0.f, b2);
    load_vec<T, G>(p.alpha, gl, p.C, 1.f, al);
    int64_t held = -1;                               // gate row in a[]
    const bool token_gate = p.gate && p.rpg == 1 && !p.gate_f32;
    Row<T, G> nf, nx, ng;
    nf.clear(); nx.clear(); ng.clear();
    auto fetch = [&](int64_t r) {
        if (r >= p.rows) return;
        nf.fetch(static_cast<const T *>(p.f) + r * p.C, gl, p.C);
        if (p.x) nx.fetch(static_cast<const T *>(p.x) + r * p.C, gl, p.C);
        if (token_gate) ng.fetch(static_cast<const T *>(p.gate) + r * p.C, gl, p.C);
    };
    fetch((int64_t)blockIdx.x * GR + gi);
    for (int64_t r0 = (int64_t)blockIdx.x * GR; r0 < p.rows; r0 += (int64_t)gridDim.x * GR) {
        const int64_t r = r0 + gi;
        const bool live = r < p.rows;
        float v[E], x[E];
        nf.widen(v);
        nx.widen(x);
        if (p.gate && live) {
            const int64_t gr = p.rpg == 1 ? r : (uint32_t)r / p.rpg;
            if (gr != held) {
                if (token_gate) ng.widen(a);
                else load_gate<T, G>(p, gr, gl, a);
                held = gr;
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    float slope;
                    activate(p.act, a[j], a[j], slope);
                }
            }
        }
        fetch(r + (int64_t)gridDim.x * GR);
        if (p.post != EVFLY_NORM_NONE) {
            normalise<T, G>(v, p.post, gl, p.C, p.inv_c, p.eps, red, turn);
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] = fmaf(v[j], w1[j], b1[j]);
        }
        if (p.gate)
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] *= a[j];
        if (p.x)
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] = fmaf(al[j], x[j], v[j]);
        if (live && p.y) store_row<T, G>(static_cast<T *>(p.y) + r * p.C, gl, p.C, v);
        if (p.pre != EVFLY_NORM_NONE) {
            normalise<T, G>(v, p.pre, gl, p.C, p.inv_c, p.eps, red, turn);
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] = fmaf(v[j], w2[j], b2[j]);
            if (live) store_row<T, G>(static_cast<T *>(p.h) + r * p.C, gl, p.C, v);
        }
    }
}

// Sum of one value array over the block's groups; group 0's lanes hold the result (after the wave exchange: lanes < G of wave 0 for G <= 64).
template <int G, int NT> __device__ __forceinline__ void block_columns(float (&v)[E], float *lds, int gl, int gi) {
    if constexpr (G < 64)
#pragma unroll
        for (int d = G; d < 64; d *= 2)
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] += __shfl_xor(v[j], d);
    constexpr int GW = G < 64 ? 64 : G, NG = NT / GW;           // groups that are left, one per GW threads
    if constexpr (NG > 1) {
        const int k = threadIdx.x / GW;
        __syncthreads();
        if (threadIdx.x % GW < G)
#pragma unroll
            for (int j = 0; j < E; ++j) lds[(k * E + j) * G + gl] = v[j];
        __syncthreads();
        if (gi == 0)
#pragma unroll
            for (int j = 0; j < E; ++j) {
                v[j] = 0.f;
#pragma unroll
                for (int i = 0; i < NG; ++i) v[j] += lds[(i * E + j) * G + gl];
            }
    }
}
template <typename T, int G> __device__ __forceinline__ void store_columns(float *out, int gl, int C, const float (&v)[E]) {
#pragma unroll
    for (int j = 0; j < E; j += 4) {
        const int c = column<T, G>(gl, j);
        if (c + 4 <= C) store16_any(out + c, make_uint4(__float_as_uint(v[j]), __float_as_uint(v[j + 1]), __float_as_uint(v[j + 2]), __float_as_uint(v[j + 3])));
        else
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + i < C) out[c + i] = v[j + i];
    }
}

template <typename T, int G> __global__ __launch_bounds__(G > 256 ? G : 256) void k_bn_bwd(BnArgs p) {
    constexpr int NT = G > 256 ? G : 256, GR = NT / G, GW = G < 64 ? 64 : G;
    __shared__ float red[64];
    __shared__ float lds[NT / GW > 1 ? NT / GW * E * G : 1];
    int turn = 0;
    const int gl = threadIdx.x % G, gi = threadIdx.x / G;
    // A block of 1024 threads has 128 registers per thread: it reads weights and rows when it needs them and keeps four of the column sums in LDS (8192
    // channels, bf16, 4096 rows: 144 us; 466 with everything in registers, spilled, on half as many blocks)
    constexpr bool KEEP = G < 1024;
    float w1[E], b1[E], w2[E], al[E];
    if (KEEP) {
        load_vec<T, G>(p.w1, gl, p.C, 1.f, w1);
        load_vec<T, G>(p.b1, gl, p.C, 0.f, b1);
        load_vec<T, G>(p.w2, gl, p.C, 1.f, w2);
        load_vec<T, G>(p.alpha, gl, p.C, 1.f, al);
    }
    float sa[KEEP ? E : 1], sw1[KEEP ? E : 1], sb1[KEEP ? E : 1], sw2[KEEP ? E : 1], sb2[E], sg[E];
    extern __shared__ float held[];                   // !KEEP: w1, b1, w2 and alpha sums, [kind][value][thread]
    auto sum = [&](float *reg, int kind, int j) -> float & {
        if constexpr (KEEP) return reg[j];
        else return held[(kind * E + j) * NT + threadIdx.x];
    };
#pragma unroll
    for (int j = 0; j < E; ++j) sum(sa, 3, j) = sum(sw1, 0, j) = sum(sb1, 1, j) = sum(sw2, 2, j) = sb2[j] = sg[j] = 0.f;
    const bool gate_rows = p.dgate && p.rpg > 1 && p.rpg < p.rows;        // a gate row for several rows, not for all
    for (uint32_t unit = blockIdx.x; unit < p.units; unit += gridDim.x) {
        // unit = (gate row, part); its rows lie in one gate row (one gate row for everything: parts of all rows)
        const uint32_t grow = unit / p.parts, part = unit % p.parts;
        const int64_t base = (int64_t)grow * p.span, lo = base + (int64_t)part * p.unit_rows;
        const int64_t hi = min(lo + (int64_t)p.unit_rows, base + (int64_t)p.span);
        float a[E], slope[E];
        auto load_act = [&](int64_t row) {
            load_gate<T, G>(p, row, gl, a);
#pragma unroll
            for (int j = 0; j < E; ++j) activate(p.act, a[j], a[j], slope[j]);
        };
#pragma unroll
        for (int j = 0; j < E; ++j) a[j] = slope[j] = 1.f;
        if (p.gate && p.rpg > 1) load_act(lo / p.rpg);
        Row<T, G> nf, nx, ny, nh;
        nf.clear(); nx.clear(); ny.clear(); nh.clear();
        auto fetch = [&](int64_t r) {
            if (r >= hi) return;
            nf.fetch(static_cast<const T *>(p.f) + r * p.C, gl, p.C);
            if (p.x) nx.fetch(static_cast<const T *>(p.x) + r * p.C, gl, p.C);
            if (p.dy) ny.fetch(static_cast<const T *>(p.dy) + r * p.C, gl, p.C);
            if (p.dh) nh.fetch(static_cast<const T *>(p.dh) + r * p.C, gl, p.C);
        };
        if (KEEP) fetch(lo + gi);
        for (int64_t r0 = lo; r0 < hi; r0 += GR) {
            const int64_t r = r0 + gi;
            const bool live = r < hi;
            float f[E], x[E], dy[E], dh[E];
            if (!KEEP) {
                nf.clear(); nx.clear(); ny.clear(); nh.clear();
                fetch(r);
            }
            nf.widen(f);
            nx.widen(x);
            ny.widen(dy);
            nh.widen(dh);
            if (live && p.gate && p.rpg == 1) load_act(r);
            if (KEEP) fetch(r + GR);
            // forward again: fh = normalised f, u = its affine form
            float r1 = 1.f, u[E];
            if (p.post != EVFLY_NORM_NONE) r1 = normalise<T, G>(f, p.post, gl, p.C, p.inv_c, p.eps, red, turn);
            if (!KEEP) {
                load_vec<T, G>(p.w1, gl, p.C, 1.f, w1);
                load_vec<T, G>(p.b1, gl, p.C, 0.f, b1);
            }
#pragma unroll
            for (int j = 0; j < E; ++j) u[j] = p.post != EVFLY_NORM_NONE ? fmaf(f[j], w1[j], b1[j]) : f[j];
            if (p.pre != EVFLY_NORM_NONE) {
                float y[E];
                if (!KEEP) load_vec<T, G>(p.alpha, gl, p.C, 1.f, al);
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    y[j] = a[j] * u[j];
                    if (p.x) y[j] = fmaf(al[j], x[j], y[j]);
                }
                const float r2 = normalise<T, G>(y, p.pre, gl, p.C, p.inv_c, p.eps, red, turn);
                float s[2] = {0.f, 0.f};
                if (!KEEP) load_vec<T, G>(p.w2, gl, p.C, 1.f, w2);
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    if (live) {                          // (a row that is not there may normalise to NaN: its zeros are not enough)
                        sb2[j] += dh[j];
                        sum(sw2, 2, j) = fmaf(dh[j], y[j], sum(sw2, 2, j));
                    }
                    dh[j] *= w2[j];
                    s[0] += dh[j];
                    s[1] = fmaf(dh[j], y[j], s[1]);
                }
                row_sum<G>(s, red, turn);
                const float m0 = p.pre == EVFLY_NORM_LAYER ? s[0] * p.inv_c : 0.f, m1 = s[1] * p.inv_c;
#pragma unroll
                for (int j = 0; j < E; ++j) dy[j] = fmaf(r2, dh[j] - m0 - y[j] * m1, dy[j]);
            }
            // dy is now the gradient of y from both outputs
            if (!KEEP) load_vec<T, G>(p.alpha, gl, p.C, 1.f, al);
            float t[E];
            if (p.x) {
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    if (live) sum(sa, 3, j) = fmaf(dy[j], x[j], sum(sa, 3, j));
                    t[j] = al[j] * dy[j];
                }
                if (live && p.dx) store_row<T, G>(static_cast<T *>(p.dx) + r * p.C, gl, p.C, t);
            }
            if (p.gate) {
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    t[j] = dy[j] * u[j] * slope[j];
                    if (live) sg[j] += t[j];
                    dy[j] *= a[j];
                }
                if (live && p.dgate && p.rpg == 1) {
                    if (p.gate_f32) store_columns<T, G>(static_cast<float *>(p.dgate) + r * p.C, gl, p.C, t);
                    else store_row<T, G>(static_cast<T *>(p.dgate) + r * p.C, gl, p.C, t);
                }
            }
            if (p.post != EVFLY_NORM_NONE) {
                if (!KEEP) load_vec<T, G>(p.w1, gl, p.C, 1.f, w1);
                float s[2] = {0.f, 0.f};
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    if (live) {
                        sum(sb1, 1, j) += dy[j];
                        sum(sw1, 0, j) = fmaf(dy[j], f[j], sum(sw1, 0, j));
                    }
                    dy[j] *= w1[j];
                    const float in = column<T, G>(gl, j) < p.C ? dy[j] : 0.f;
                    s[0] += in;
                    s[1] = fmaf(in, f[j], s[1]);
                }
                row_sum<G>(s, red, turn);
                const float m0 = p.post == EVFLY_NORM_LAYER ? s[0] * p.inv_c : 0.f, m1 = s[1] * p.inv_c;
#pragma unroll
                for (int j = 0; j < E; ++j) dy[j] = r1 * (dy[j] - m0 - f[j] * m1);
            }
            if (live) store_row<T, G>(static_cast<T *>(p.df) + r * p.C, gl, p.C, dy);
        }
        if (gate_rows) {
            block_columns<G, NT>(sg, lds, gl, gi);
            if (gi == 0) {
                if (p.parts > 1) store_columns<T, G>(p.gate_part + (int64_t)unit * p.C, gl, p.C, sg);
                else if (p.gate_f32) store_columns<T, G>(static_cast<float *>(p.dgate) + (int64_t)grow * p.C, gl, p.C, sg);
                else store_row<T, G>(static_cast<T *>(p.dgate) + (int64_t)grow * p.C, gl, p.C, sg);
            }
#pragma unroll
            for (int j = 0; j < E; ++j) sg[j] = 0.f;
        }
    }
    float *const out = p.cols + (int64_t)blockIdx.x * K_N * p.C;
    auto flush = [&](int kind, float (&v)[E]) {
        if (!(p.want >> kind & 1)) return;
        block_columns<G, NT>(v, lds, gl, gi);
        if (gi == 0) store_columns<T, G>(out + kind * p.C, gl, p.C, v);
    };
    flush(K_B2, sb2); flush(K_GATE, sg);
    auto flush_sum = [&](int kind, float *reg, int at) {
        float v[E];
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = sum(reg, at, j);
        flush(kind, v);
    };
    flush_sum(K_W1, sw1, 0); flush_sum(K_B1, sb1, 1); flush_sum(K_W2, sw2, 2); flush_sum(K_ALPHA, sa, 3);
}

// out_k[c] = sum over partial rows in order: 16 runs of rows per column, then the runs. blockIdx.y: the vector; in: [row][stride], column offset kind * C.
struct BnSums {
    const float *in[K_N];
    void *out[K_N];
    int bf16[K_N];
    int64_t row_stride;                // floats between partial rows
    int64_t group_stride;              // floats between outputs' groups (blockIdx.z)
    int n, C;
};
__global__ __launch_bounds__(1024) void k_bn_columns(BnSums p) {
    __shared__ float s[16][64];
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6, c = blockIdx.x * 64 + l, k = blockIdx.y;
    const float *in = p.in[k] + (int64_t)blockIdx.z * p.group_stride;
    const int per = (p.n + 15) / 16, lo = w * per, hi = min(lo + per, p.n);
    float a = 0.f;
    if (c < p.C)
#pragma unroll 8
        for (int i = lo; i < hi; ++i) a += in[i * p.row_stride + c];
    s[w][l] = a;
    __syncthreads();
    if (w == 0 && c < p.C) {
        a = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) a += s[i][l];
        const int64_t at = (int64_t)blockIdx.z * p.C + c;
        if (p.bf16[k]) static_cast<bf16_t *>(p.out[k])[at] = f2bf_dev(a);
        else static_cast<float *>(p.out[k])[at] = a;
    }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, int G> int bn_launch(const BnArgs &p, bool backward, unsigned blocks, hipStream_t st) {
    constexpr int NT = G > 256 ? G : 256;
    if (backward) {
        constexpr int held = G < 1024 ? 0 : 4 * E * NT * (int)sizeof(float);
        if (held > 0) {
            static std::atomic<bool> attr_set[64];
            int dev = 0;
            EVFLY_HIP(hipGetDevice(&dev));
            EVFLY_REQUIRE(dev >= 0 && dev < 64, "device index %d out of range", dev);
            if (!attr_set[dev].load(std::memory_order_acquire)) {
                EVFLY_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(k_bn_bwd<T, G>), hipFuncAttributeMaxDynamicSharedMemorySize, held));
                attr_set[dev].store(true, std::memory_order_release);
            }
        }
        hipLaunchKernelGGL((k_bn_bwd<T, G>), dim3(blocks), dim3(NT), held, st, p);
    }
    else hipLaunchKernelGGL((k_bn_fwd<T, G>), dim3(blocks), dim3(NT), 0, st, p);
    EVFLY_LAUNCH_CHECK();
    return 0;
}
template <typename T> int bn_group(const BnArgs &p, int G, bool backward, unsigned blocks, hipStream_t st) {
    switch (G) {
    case 4: return bn_launch<T, 4>(p, backward, blocks, st);
    case 8: return bn_launch<T, 8>(p, backward, blocks, st);
    case 16: return bn_launch<T, 16>(p, backward, blocks, st);
    case 32: return bn_launch<T, 32>(p, backward, blocks, st);
    case 64: return bn_launch<T, 64>(p, backward, blocks, st);
    case 128: return bn_launch<T, 128>(p, backward, blocks, st);
    case 256: return bn_launch<T, 256>(p, backward, blocks, st);
    case 512: return bn_launch<T, 512>(p, backward, blocks, st);
    default: return bn_launch<T, 1024>(p, backward, blocks, st);
    }
}
int bn_run(const BnArgs &p, int dtype, int G, bool backward, unsigned blocks, hipStream_t st) {
    return dtype == EVFLY_DTYPE_F32 ? bn_group<float>(p, G, backward, blocks, st) : bn_group<bf16_t>(p, G, backward, blocks, st);
}

int lanes_for(int C) {
    int g = 4;
    while (g * E < C) g *= 2;
    return g;
}

struct BnPlan {
    int G, GR;
    uint32_t unit_rows, parts, units;
    unsigned blocks;
    int64_t o_gate, bytes;
};
// Backward: units of rows that share a gate row. One gate row for everything (or none, or one per row): one unit per block, of equal rows; a gate row
// per stream: enough parts of each stream that every block has work. At least two rows per group in either.
BnPlan bn_plan(int64_t rows, int C, int64_t rpg) {
    BnPlan b{};
    b.G = lanes_for(C);
    b.GR = (b.G > 256 ? b.G : 256) / b.G;
    const bool streams = rpg > 1 && rpg < rows;
    const int64_t span = streams ? rpg : rows, groups = streams ? rows / rpg : 1;
    const int max_blocks = b.G > 256 ? kNumCU : BN_MAX_BLOCKS;
    int64_t parts = (max_blocks + groups - 1) / groups;
    const int64_t most = (span + 2 * b.GR - 1) / (2 * b.GR);
    if (parts > most) parts = most;
    if (parts < 1) parts = 1;
    const int64_t ur = (span + parts - 1) / parts;
    b.unit_rows = (uint32_t)((ur + b.GR - 1) / b.GR * b.GR);
    b.parts = (uint32_t)((span + b.unit_rows - 1) / b.unit_rows);
    b.units = (uint32_t)(groups * b.parts);
    b.blocks = b.units < (uint32_t)max_blocks ? b.units : (uint32_t)max_blocks;
    b.o_gate = ((int64_t)b.blocks * K_N * C * 4 + 255) / 256 * 256;
    b.bytes = b.o_gate + (streams && b.parts > 1 ? (int64_t)b.units * C * 4 : 0);
    return b;
}

int bn_check(const char *who, const void *f, const void *x, const void *gate, int64_t rpg, int gate_act, const float *alpha, int post, int pre, float eps,
             int64_t rows, int C, int dtype) {
    EVFLY_REQUIRE(rows >= 0 && rows <= INT32_MAX && C > 0 && C <= EVFLY_BLOCK_NORM_MAX_CHANNELS, "%s: %lld rows of %d channels (1 .. %d)", who, (long long)rows, C,
                  EVFLY_BLOCK_NORM_MAX_CHANNELS);
    EVFLY_REQUIRE(dtype == EVFLY_DTYPE_F32 || dtype == EVFLY_DTYPE_BF16, "%s: dtype %d (EVFLY_DTYPE_F32 or EVFLY_DTYPE_BF16)", who, dtype);
    EVFLY_REQUIRE(post >= EVFLY_NORM_NONE && post <= EVFLY_NORM_RMS && pre >= EVFLY_NORM_NONE && pre <= EVFLY_NORM_RMS, "%s: norm kinds %d, %d", who, post, pre);
    EVFLY_REQUIRE(std::isfinite(eps) && eps >= 0.f, "%s: eps is negative or not finite", who);
    EVFLY_REQUIRE(!alpha || x, "%s: res_scale without a residual", who);
    EVFLY_REQUIRE(rows == 0 || f, "%s: null argument", who);
    if (gate) {
        EVFLY_REQUIRE(gate_act == EVFLY_ACT_NONE || gate_act == EVFLY_ACT_TANH || gate_act == EVFLY_ACT_SIGMOID, "%s: gate activation %d", who, gate_act);
        EVFLY_REQUIRE(rows == 0 || (rpg >= 1 && rpg <= rows && rows % rpg == 0), "%s: %lld rows per gate row do not divide %lld rows", who, (long long)rpg, (long long)rows);
    }
    return 0;
}

}  // namespace
}  // namespace evfly

using namespace evfly;

extern "C" int evfly_block_norm_forward(const void *f, const void *x, const void *gate, int64_t rows_per_gate, int gate_f32, int gate_act,
                                        const float *res_scale, int post_kind, const float *post_weight, const float *post_bias,
                                        int pre_kind, const float *pre_weight, const float *pre_bias, float eps, int64_t rows, int channels,
                                        int dtype, void *y, void *h, void *stream) {
    if (int rc = bn_check("block_norm_forward", f, x, gate, rows_per_gate, gate_act, res_scale, post_kind, pre_kind, eps, rows, channels, dtype)) return rc;
    if (rows == 0) return 0;
    EVFLY_REQUIRE(y || (pre_kind != EVFLY_NORM_NONE && h), "block_norm_forward: no output");
    EVFLY_REQUIRE(pre_kind == EVFLY_NORM_NONE || h, "block_norm_forward: a pre norm without h");
    BnArgs p{};
    p.f = f; p.x = x; p.gate = gate; p.alpha = res_scale; p.w1 = post_weight; p.b1 = post_bias; p.w2 = pre_weight; p.b2 = pre_bias;
    p.y = y; p.h = h; p.post = post_kind; p.pre = pre_kind; p.act = gate_act; p.gate_f32 = gate_f32; p.C = channels;
    p.rows = (uint32_t)rows; p.rpg = gate ? (uint32_t)rows_per_gate : 1u; p.eps = eps; p.inv_c = 1.f / (float)channels;
    const int G = lanes_for(channels), GR = (G > 256 ? G : 256) / G;
    const int64_t need = (rows + GR - 1) / GR, most = 8 * kNumCU;
    return bn_run(p, dtype, G, false, (unsigned)(need < most ? need : most), as_stream(stream));
}

extern "C" int64_t evfly_block_norm_workspace_bytes(int64_t rows, int channels, int64_t rows_per_gate, int dtype) {
    if (bn_check("block_norm_workspace_bytes", &rows, nullptr, nullptr, 1, 0, nullptr, 0, 0, 0.f, rows, channels, dtype)) return -1;
    return rows == 0 ? 0 : bn_plan(rows, channels, rows_per_gate < 1 ? 1 : rows_per_gate).bytes;
}

extern "C" int evfly_block_norm_backward(const void *f, const void *x, const void *gate, int64_t rows_per_gate, int gate_f32, int gate_act,
                                         const float *res_scale, int post_kind, const float *post_weight, const float *post_bias,
                                         int pre_kind, const float *pre_weight, const float *pre_bias, float eps, const void *dy, const void *dh,
                                         int64_t rows, int channels, int dtype, void *df, void *dx, void *d_gate, float *d_res_scale,
                                         float *d_post_weight, float *d_post_bias, float *d_pre_weight, float *d_pre_bias, void *workspace,
                                         int64_t workspace_bytes, void *stream) {
    if (int rc = bn_check("block_norm_backward", f, x, gate, rows_per_gate, gate_act, res_scale, post_kind, pre_kind, eps, rows, channels, dtype)) return rc;
    EVFLY_REQUIRE(rows == 0 || df, "block_norm_backward: null argument");
    EVFLY_REQUIRE((x || (!dx && !d_res_scale)) && (gate || !d_gate), "block_norm_backward: the gradient of an input that is not there");
    EVFLY_REQUIRE(post_kind != EVFLY_NORM_NONE || (!d_post_weight && !d_post_bias), "block_norm_backward: post norm gradients without a post norm");
    EVFLY_REQUIRE(pre_kind != EVFLY_NORM_NONE || (!d_pre_weight && !d_pre_bias && !dh), "block_norm_backward: dh or pre norm gradients without a pre norm");
    hipStream_t st = as_stream(stream);
    const int64_t rpg = gate ? rows_per_gate : 1;
    const BnPlan b = rows > 0 ? bn_plan(rows, channels, rpg) : BnPlan{};
    EVFLY_REQUIRE(rows == 0 || (workspace && aligned16(workspace) && workspace_bytes >= b.bytes), "block_norm_backward: workspace smaller than evfly_block_norm_workspace_bytes, or not 16-byte aligned");
    BnArgs p{};
    p.f = f; p.x = x; p.gate = gate; p.alpha = res_scale; p.w1 = post_weight; p.b1 = post_bias; p.w2 = pre_weight; p.b2 = pre_bias;
    p.post = post_kind; p.pre = pre_kind; p.act = gate_act; p.gate_f32 = gate_f32; p.C = channels;
    p.rows = (uint32_t)rows; p.rpg = (uint32_t)rpg; p.eps = eps; p.inv_c = 1.f / (float)channels;
    p.dy = dy; p.dh = dh; p.df = df; p.dx = dx; p.dgate = d_gate;
    p.cols = static_cast<float *>(workspace);
    p.gate_part = reinterpret_cast<float *>(static_cast<char *>(workspace) + b.o_gate);
    const bool streams = rpg > 1 && rpg < rows;
    p.unit_rows = b.unit_rows; p.parts = b.parts; p.units = b.units; p.span = (uint32_t)(streams ? rpg : rows);
    float *const vecs[K_N] = {d_res_scale, d_post_weight, d_post_bias, d_pre_weight, d_pre_bias, nullptr};
    BnSums s{};
    s.n = (int)b.blocks; s.C = channels; s.row_stride = (int64_t)K_N * channels;
    int m = 0;
    for (int k = 0; k < K_N; ++k) {
        void *o = vecs[k];
        if (k == K_GATE) o = gate && rpg == rows && rows > 1 ? d_gate : nullptr;
        if (!o) continue;
        p.want |= 1 << k;
        s.in[m] = p.cols + (int64_t)k * channels;
        s.out[m] = o;
        s.bf16[m] = k == K_GATE && !gate_f32 && dtype == EVFLY_DTYPE_BF16;
        ++m;
    }
    if (rows > 0)
        if (int rc = bn_run(p, dtype, b.G, true, b.blocks, st)) return rc;
    if (m) hipLaunchKernelGGL(k_bn_columns, dim3((channels + 63) / 64, m, 1), dim3(1024), 0, st, s);
    if (streams && d_gate && b.parts > 1) {
        BnSums g{};
        g.in[0] = p.gate_part; g.out[0] = d_gate; g.bf16[0] = !gate_f32 && dtype == EVFLY_DTYPE_BF16;
        g.n = (int)b.parts; g.C = channels; g.row_stride = channels; g.group_stride = (int64_t)b.parts * channels;
        hipLaunchKernelGGL(k_bn_columns, dim3((channels + 63) / 64, 1, (unsigned)(rows / rpg)), dim3(1024), 0, st, g);
    }
    EVFLY_LAUNCH_CHECK();
    return 0;
}
