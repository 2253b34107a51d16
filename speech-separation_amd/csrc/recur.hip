// Gated linear recurrence over long sequences:  h_t = a_t h_{t-1} + (1 - a_t) x_t,  a_t = sigmoid(f_t),  y_t = h_t,
// channel by channel, forwards or backwards in time, over items of unequal lengths.  Its backward runs the same kind of
// recurrence the other way:  s_t = a_t g_t,  g_t = dy_t + s_{t+1};  dx_t = (1 - a_t) g_t,  df_t = a_t (1 - a_t) g_t
// (h_{t-1} - x_t).
//
// Bound: HBM (forward reads x, f and writes y; backward reads x, f, dy and writes dx, df; about 5 and 14 operations per
// element).  Both maps are affine in the state, so steps compose as (A, H): h -> A h + H, and the composition is
// associative: a thread folds TC consecutive steps of VEC channels in registers, TS threads cover one tile of TS * TC
// steps and combine by shuffles and one LDS exchange, and the tile is finished from the same registers -- x and f are
// read once.  States are fp32 throughout.  The forward pass keeps the state at every tile's start; the backward
// pass recomputes the tile's states from it (in fp32: the rounded y would not do for h_{t-1} - x_t) instead of reading y.
// Measured, bf16: 1040 x 47 x 1024 75 us forward (4.0 TB/s), 104 backward (4.8 TB/s); 2 x 15001 x 1024, cut into
// segments whose maps a launch of its own finds first: 41 + 35 and 25 + 58 us.
#include "common.h"
#include "../../include/dtt_hip.h"

namespace {
constexpr int NTH = 256, TC = 8;                 // threads of a workgroup, steps a thread folds per tile
constexpr int TSPLIT = 8;                        // time lanes of the split form

template <typename T, int VEC> struct Raw;       // VEC consecutive channels as loaded
template <> struct Raw<float, 4> {
    float4 v;
    __device__ __forceinline__ float get(int i) const { return (&v.x)[i]; }
    __device__ __forceinline__ void put(const float (&f)[4]) { v = make_float4(f[0], f[1], f[2], f[3]); }
};
template <> struct Raw<float, 2> {
    float2 v;
    __device__ __forceinline__ float get(int i) const { return (&v.x)[i]; }
    __device__ __forceinline__ void put(const float (&f)[2]) { v = make_float2(f[0], f[1]); }
};
template <> struct Raw<float, 1> {
    float v;
    __device__ __forceinline__ float get(int) const { return v; }
    __device__ __forceinline__ void put(const float (&f)[1]) { v = f[0]; }
};
template <> struct Raw<bf16, 4> {
    uint2 v;
    __device__ __forceinline__ float get(int i) const {
        const uint32_t w = (&v.x)[i >> 1];
        return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
    }
    __device__ __forceinline__ void put(const float (&f)[4]) { v = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])); }
};
template <> struct Raw<bf16, 2> {
    uint32_t v;
    __device__ __forceinline__ float get(int i) const { return __uint_as_float(i ? (v & 0xffff0000u) : (v << 16)); }
    __device__ __forceinline__ void put(const float (&f)[2]) { v = pack_bf16x2(f[0], f[1]); }
};
template <> struct Raw<bf16, 1> {
    unsigned short v;
    __device__ __forceinline__ float get(int) const { return bf2f(v); }
    __device__ __forceinline__ void put(const float (&f)[1]) { v = f2bf(f[0]); }
};
template <typename T, int VEC> __device__ __forceinline__ Raw<T, VEC> ldr(const T* p) {
    Raw<T, VEC> r;
    r.v = *reinterpret_cast<const decltype(r.v)*>(p);
    return r;
}
template <typename T, int VEC> __device__ __forceinline__ void str(T* p, const Raw<T, VEC>& r) {
    *reinterpret_cast<decltype(r.v)*>(p) = r.v;
}

// a = sigmoid(f) and i = 1 - a = sigmoid(-f), both to the last bits, from e = exp(-f): 1 / (1 + e) and e / (1 + e).  e is
// held below 2^126 (no inf * 0); NaN passes.  fp32: the rounding of f log2(e) is carried along (|f| up to 80 would lose 6
// bits); bf16 does not show it.
template <typename T> __device__ __forceinline__ void gate(float f, float& a, float& i) {
    float e;
    if constexpr (sizeof(T) == 4) {
        f = f < -87.f ? -87.f : f;
        f = f > 104.f ? 104.f : f;
        const float t = f * -1.4426950408889634f;
        const float lo = fmaf(f, -1.4426950408889634f, -t) + f * -1.925963033500e-8f;
        e = __builtin_amdgcn_exp2f(t);
        e = fmaf(e * 0.6931471805599453f, lo, e);
    } else {
        const float t = f * -1.4426950408889634f;
        e = __builtin_amdgcn_exp2f(t > 126.f ? 126.f : t);
    }
    a = __builtin_amdgcn_rcpf(1.0f + e);
    i = e * a;
}

struct RecP {
    const void* x; const void* f; const void* dy;
    void* y; void* dx; void* df;
    const float* h0; const float* dlast;         // [N][D] or null
    float* last; float* dh0;                     // [N][D]
    float* st;                                   // [tiles][N][D]: state at every tile's start (forward writes, backward reads)
    float* agg;                                  // [nseg][2][N][D]: (A, H) of every segment
    const int* len;                              // [N] or null
    int64_t x_so, x_si, x_sl, f_so, f_si, f_sl, g_so, g_si, g_sl;
    int64_t cols;                                // N * ceil(D / VEC)
    int N, NI, L, D, dv, reverse, nseg, seg;     // seg: steps of a segment, a multiple of the tile
};

// one thread's place: a column (item, VEC channels) and a time lane
template <int VEC, int TS> struct Place {
    int cl, ts, n, d0, len;
    bool ok;
    int64_t nd;                                  // offset of the column in [N][D]
    __device__ __forceinline__ explicit Place(const RecP& p) {
        constexpr int CL = NTH / TS;
        cl = threadIdx.x % CL, ts = threadIdx.x / CL;
        const int64_t col = (int64_t)blockIdx.x * CL + cl;
        ok = col < p.cols;
        const int64_t c = ok ? col : p.cols - 1;
        n = (int)(c / p.dv);
        d0 = (int)(c - (int64_t)n * p.dv) * VEC;
        nd = (int64_t)n * p.D + d0;
        len = p.len ? min(max(p.len[n], 0), p.L) : p.L;
    }
    // logical step t (0 .. L-1, in the order of the recurrence) -> row; the rows behind an item's length stay in place
    __device__ __forceinline__ int row(const RecP& p, int t) const { return p.reverse && t < len ? len - 1 - t : t; }
    // TC rows from logical step t on.  all: every one is live for every lane of the wave (one pointer that walks); otherwise
    // dead rows read row 0 instead, whose values are not used
    template <typename T> __device__ __forceinline__ void load(const RecP& p, const T* base, int64_t sl, int t, bool all, Raw<T, VEC> (&r)[TC]) const {
        if (all) {
            const T* q = base + (int64_t)row(p, t) * sl;
            const int64_t step = p.reverse ? -sl : sl;
#pragma unroll
            for (int i = 0; i < TC; ++i) r[i] = ldr<T, VEC>(q + i * step);
        } else {
#pragma unroll
            for (int i = 0; i < TC; ++i) r[i] = ldr<T, VEC>(base + (int64_t)(t + i < len ? row(p, t + i) : 0) * sl);
        }
    }
    template <typename T> __device__ __forceinline__ void store(const RecP& p, T* base, int t, int te, bool all, const Raw<T, VEC> (&r)[TC]) const {
        if (!ok) return;
        if (all) {
            T* q = base + (int64_t)row(p, t) * p.D;
            const int64_t step = p.reverse ? -p.D : p.D;
#pragma unroll
            for (int i = 0; i < TC; ++i) str<T, VEC>(q + i * step, r[i]);
        } else {
#pragma unroll
            for (int i = 0; i < TC; ++i)
                if (t + i < te) str<T, VEC>(base + (int64_t)row(p, t + i) * p.D, r[i]);
        }
    }
};

// Combines the TS time lanes' maps (A, H) of one column and returns the state that this lane starts from, given the
// state `carry` that the tile starts from (of all lanes); carry becomes the state behind the tile.  BACK: later lanes
// first.  tot: LDS of [waves][CL][2][VEC], two copies used in turn so that one barrier a tile is enough.
template <int VEC, int TS, bool BACK>
__device__ __forceinline__ void combine(float (&A)[VEC], float (&H)[VEC], float (&carry)[VEC], float (&in)[VEC], int ts, int cl,
                                        float* tot) {
    constexpr int CL = NTH / TS, TW = 64 / CL, NW = NTH / 64;       // time lanes of a wave, waves
    static_assert(TW == 2, "two time lanes a wave: one exchange between its halves");
    const int wave = threadIdx.x >> 6, tw = ts % TW, pt = BACK ? TW - 1 - tw : tw;
    float ea[VEC], eh[VEC];                                          // the other half's map, where it comes first
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        const float a = __shfl_xor(A[v], 32, 64), h = __shfl_xor(H[v], 32, 64);
        ea[v] = pt ? a : 1.f;
        eh[v] = pt ? h : 0.f;
        H[v] = fmaf(A[v], eh[v], H[v]);
        A[v] *= ea[v];
    }
    if (pt)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            tot[((wave * CL + cl) * 2 + 0) * VEC + v] = A[v];
            tot[((wave * CL + cl) * 2 + 1) * VEC + v] = H[v];
        }
    __syncthreads();
    float mine[VEC];
#pragma unroll
    for (int k = 0; k < NW; ++k) {
        const int w = BACK ? NW - 1 - k : k;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            if (w == wave) mine[v] = carry[v];
            carry[v] = fmaf(tot[((w * CL + cl) * 2 + 0) * VEC + v], carry[v], tot[((w * CL + cl) * 2 + 1) * VEC + v]);
        }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) in[v] = fmaf(ea[v], mine[v], eh[v]);
}

// State ahead of this segment from the maps of the segments before it (BACK: behind it): every time lane folds a part of
// them, in a few round trips to memory, and the parts are combined like a tile's (one thread after the other through 118
// segments took 9 of the 48 us of an fp32 forward pass over 37501 x 512).
template <int VEC, int TS, bool BACK>
__device__ __forceinline__ void fold_segments(const RecP& p, int64_t nd, const float* start, float (&c)[VEC], int ts, int cl, float* tot) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) c[v] = start ? start[nd + v] : 0.f;
    if constexpr (TS > 1) {
        const int cnt = BACK ? p.nseg - 1 - (int)blockIdx.y : (int)blockIdx.y;
        if (cnt == 0) return;                                            // (the same for the whole workgroup)
        const int64_t ND = (int64_t)p.N * p.D;
        const int per = (cnt + TS - 1) / TS, k0 = (BACK ? TS - 1 - ts : ts) * per, k1 = min(cnt, k0 + per);
        float A[VEC], H[VEC], in[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) A[v] = 1.f, H[v] = 0.f;
#pragma unroll 4
        for (int k = k0; k < k1; ++k) {
            const float* g = p.agg + (int64_t)(BACK ? p.nseg - 1 - k : k) * 2 * ND + nd;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                H[v] = fmaf(g[v], H[v], g[ND + v]);
                A[v] *= g[v];
            }
        }
        combine<VEC, TS, BACK>(A, H, c, in, ts, cl, tot);
    }
}

// (A, H) of every segment: a time lane folds seg / TS consecutive steps.  BACK: the map of s over the segment, from its
// last step to its first, with dy in x's place.
template <typename T, int VEC, int TS, bool BACK>
__global__ __launch_bounds__(NTH) void rec_agg_kernel(const RecP p) {
    constexpr int CL = NTH / TS;
    __shared__ float tot[NTH / 64 * CL * 2 * VEC];
    const Place<VEC, TS> w(p);
    const T* f = (const T*)p.f + (int64_t)(w.n / p.NI) * p.f_so + (int64_t)(w.n % p.NI) * p.f_si + w.d0;
    const T* x = BACK ? (const T*)p.dy + (int64_t)(w.n / p.NI) * p.g_so + (int64_t)(w.n % p.NI) * p.g_si + w.d0
                      : (const T*)p.x + (int64_t)(w.n / p.NI) * p.x_so + (int64_t)(w.n % p.NI) * p.x_si + w.d0;
    const int64_t xl = BACK ? p.g_sl : p.x_sl;
    const int per = p.seg / TS, nb = per / TC, t0 = blockIdx.y * p.seg + w.ts * per;      // (seg is a multiple of TS * TC)
    float A[VEC], H[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) A[v] = 1.f, H[v] = 0.f;
    Raw<T, VEC> rf[TC], rx[TC];
    bool all = false;
    auto load = [&](int k) {
        const int t = t0 + (BACK ? nb - 1 - k : k) * TC;
        all = __all(t + TC <= w.len);
        if (__all(t >= w.len)) return;
        w.load(p, f, p.f_sl, t, all, rf);
        w.load(p, x, xl, t, all, rx);
    };
    load(0);
    for (int k = 0; k < nb; ++k) {
        const int t = t0 + (BACK ? nb - 1 - k : k) * TC;
        const bool full = all;
        Raw<T, VEC> cf[TC], cx[TC];
#pragma unroll
        for (int i = 0; i < TC; ++i) cf[i] = rf[i], cx[i] = rx[i];
        if (k + 1 < nb) load(k + 1);
        if (__all(t >= w.len)) continue;
#pragma unroll
        for (int j = 0; j < TC; ++j) {
            const int i = BACK ? TC - 1 - j : j;
            const bool on = full || t + i < w.len;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float a, im;
                gate<T>(cf[i].get(v), a, im);
                const float h = BACK ? a * (cx[i].get(v) + H[v]) : fmaf(a, H[v], im * cx[i].get(v));
                H[v] = on ? h : H[v];
                A[v] = on ? A[v] * a : A[v];
            }
        }
    }
    // the whole segment's map: where the states 0 and (with H left out) 1 go
    float c[VEC], in[VEC], A2[VEC], H2[VEC], z[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) c[v] = 0.f, A2[v] = A[v], H2[v] = 0.f, z[v] = 1.f;
    combine<VEC, TS, BACK>(A, H, c, in, w.ts, w.cl, tot);
    __syncthreads();
    combine<VEC, TS, BACK>(A2, H2, z, in, w.ts, w.cl, tot);
    if (w.ok && w.ts == 0) {
        float* g = p.agg + (int64_t)blockIdx.y * 2 * p.N * p.D + w.nd;
#pragma unroll
        for (int v = 0; v < VEC; ++v) g[v] = z[v], g[(int64_t)p.N * p.D + v] = c[v];
    }
}

template <typename T, int VEC, int TS>
__global__ __launch_bounds__(NTH) void rec_fwd_kernel(const RecP p) {
    constexpr int CL = NTH / TS, TILE = TS * TC;
    __shared__ float tot[2][NTH / 64 * CL * 2 * VEC];
    const Place<VEC, TS> w(p);
    const T* x = (const T*)p.x + (int64_t)(w.n / p.NI) * p.x_so + (int64_t)(w.n % p.NI) * p.x_si + w.d0;
    const T* f = (const T*)p.f + (int64_t)(w.n / p.NI) * p.f_so + (int64_t)(w.n % p.NI) * p.f_si + w.d0;
    T* y = (T*)p.y + (int64_t)w.n * p.L * p.D + w.d0;
    const int ta = blockIdx.y * p.seg, te = min(p.L, ta + p.seg);
    float c[VEC];
    fold_segments<VEC, TS, false>(p, w.nd, p.h0, c, w.ts, w.cl, tot[1]);
    Raw<T, VEC> nx[TC], nf[TC];
    bool all;
    auto load = [&](int tb) {
        const int t = tb + w.ts * TC;
        all = __all(t + TC <= w.len);
        w.load(p, x, p.x_sl, t, all, nx);
        w.load(p, f, p.f_sl, t, all, nf);
    };
    load(ta);
    int buf = 0;
    for (int tb = ta; tb < te; tb += TILE) {
        const int t = tb + w.ts * TC;
        const bool full = all;
        if (p.st && tb > 0 && w.ok && w.ts == 0) {
            float* s = p.st + (int64_t)(tb / TILE) * p.N * p.D + w.nd;
#pragma unroll
            for (int v = 0; v < VEC; ++v) s[v] = c[v];
        }
        float a[TC][VEC], b[TC][VEC], A[VEC], H[VEC];
#pragma unroll
        for (int i = 0; i < TC; ++i)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                gate<T>(nf[i].get(v), a[i][v], b[i][v]);
                b[i][v] *= nx[i].get(v);
            }
        if (tb + TILE < te) load(tb + TILE);
        if (!full)
#pragma unroll
            for (int i = 0; i < TC; ++i)
#pragma unroll
                for (int v = 0; v < VEC; ++v) {                       // padding: the state passes
                    a[i][v] = t + i < w.len ? a[i][v] : 1.f;
                    b[i][v] = t + i < w.len ? b[i][v] : 0.f;
                }
        float h[VEC];
        if constexpr (TS > 1) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) A[v] = a[0][v], H[v] = b[0][v];
#pragma unroll
            for (int i = 1; i < TC; ++i)
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    H[v] = fmaf(a[i][v], H[v], b[i][v]);
                    A[v] *= a[i][v];
                }
            combine<VEC, TS, false>(A, H, c, h, w.ts, w.cl, tot[buf]);
            buf ^= 1;
        } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) h[v] = c[v];
        }
        Raw<T, VEC> o[TC];
#pragma unroll
        for (int i = 0; i < TC; ++i) {
            float out[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                h[v] = fmaf(a[i][v], h[v], b[i][v]);
                out[v] = full || t + i < w.len ? h[v] : 0.f;
            }
            o[i].put(out);
        }
        w.store(p, y, t, te, full, o);
        if constexpr (TS == 1)
#pragma unroll
            for (int v = 0; v < VEC; ++v) c[v] = h[v];
    }
    if (p.last && blockIdx.y == p.nseg - 1 && w.ok && w.ts == 0)
#pragma unroll
        for (int v = 0; v < VEC; ++v) p.last[w.nd + v] = c[v];
}

template <typename T, int VEC, int TS>
__global__ __launch_bounds__(NTH) void rec_bwd_kernel(const RecP p) {
    constexpr int CL = NTH / TS, TILE = TS * TC;
    __shared__ float tot[2][NTH / 64 * CL * 2 * VEC];
    const Place<VEC, TS> w(p);
    const T* x = (const T*)p.x + (int64_t)(w.n / p.NI) * p.x_so + (int64_t)(w.n % p.NI) * p.x_si + w.d0;
    const T* f = (const T*)p.f + (int64_t)(w.n / p.NI) * p.f_so + (int64_t)(w.n % p.NI) * p.f_si + w.d0;
    const T* dy = (const T*)p.dy + (int64_t)(w.n / p.NI) * p.g_so + (int64_t)(w.n % p.NI) * p.g_si + w.d0;
    T* dx = (T*)p.dx + (int64_t)w.n * p.L * p.D + w.d0;
    T* df = (T*)p.df + (int64_t)w.n * p.L * p.D + w.d0;
    const int ta = blockIdx.y * p.seg, te = min(p.L, ta + p.seg);
    float s[VEC];                                                    // s_{t+1} of the step behind the tile
    fold_segments<VEC, TS, true>(p, w.nd, p.dlast, s, w.ts, w.cl, tot[1]);
    Raw<T, VEC> nx[TC], nf[TC], ng[TC];
    float nc[VEC];
    bool all;
    auto load = [&](int tb) {
        const int t = tb + w.ts * TC;
        all = __all(t + TC <= w.len);
        w.load(p, x, p.x_sl, t, all, nx);
        w.load(p, f, p.f_sl, t, all, nf);
        w.load(p, dy, p.g_sl, t, all, ng);
        const float* st = tb > 0 ? p.st + (int64_t)(tb / TILE) * p.N * p.D : p.h0;
#pragma unroll
        for (int v = 0; v < VEC; ++v) nc[v] = st ? st[w.nd + v] : 0.f;
    };
    const int tl = ta + (te - ta - 1) / TILE * TILE;
    load(tl);
    for (int tb = tl; tb >= ta; tb -= TILE) {
        const int t = tb + w.ts * TC;
        const bool full = all;
        // im: 1 - a; d: x, then h_{t-1} - x; g: dy
        float a[TC][VEC], im[TC][VEC], d[TC][VEC], g[TC][VEC], A[VEC], H[VEC], c[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) A[v] = 1.f, H[v] = 0.f, c[v] = nc[v];
#pragma unroll
        for (int i = 0; i < TC; ++i)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                gate<T>(nf[i].get(v), a[i][v], im[i][v]);
                d[i][v] = nx[i].get(v);
                g[i][v] = ng[i].get(v);
            }
        if (tb > ta) load(tb - TILE);
        if (!full)
#pragma unroll
            for (int i = 0; i < TC; ++i)
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const bool live = t + i < w.len;
                    a[i][v] = live ? a[i][v] : 1.f;
                    im[i][v] = live ? im[i][v] : 0.f;
                    d[i][v] = live ? d[i][v] : 0.f;
                    g[i][v] = live ? g[i][v] : 0.f;
                }
        float h[VEC];
        if constexpr (TS > 1) {
#pragma unroll
            for (int i = 0; i < TC; ++i)
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    H[v] = fmaf(a[i][v], H[v], im[i][v] * d[i][v]);
                    A[v] *= a[i][v];
                }
            combine<VEC, TS, false>(A, H, c, h, w.ts, w.cl, tot[0]);
        } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) h[v] = c[v];
        }
#pragma unroll
        for (int i = 0; i < TC; ++i)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float xv = d[i][v];
                d[i][v] = h[v] - xv;
                h[v] = fmaf(a[i][v], h[v], im[i][v] * xv);
            }
        float sn[VEC];
        if constexpr (TS > 1) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) A[v] = 1.f, H[v] = 0.f;
#pragma unroll
            for (int i = TC - 1; i >= 0; --i)
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    H[v] = a[i][v] * (g[i][v] + H[v]);
                    A[v] *= a[i][v];
                }
            combine<VEC, TS, true>(A, H, s, sn, w.ts, w.cl, tot[1]);
        } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) sn[v] = s[v];
        }
        Raw<T, VEC> ox[TC], of[TC];
#pragma unroll
        for (int i = TC - 1; i >= 0; --i) {
            float vx[VEC], vf[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float gt = g[i][v] + sn[v];
                sn[v] = a[i][v] * gt;
                vx[v] = im[i][v] * gt;
                vf[v] = im[i][v] * d[i][v] * sn[v];
            }
            ox[i].put(vx);
            of[i].put(vf);
        }
        if (!full) {                                                  // behind the length 0, also where im = 0 met a state or dlast that is not finite
            const float zero[VEC] = {};
#pragma unroll
            for (int i = 0; i < TC; ++i)
                if (t + i >= w.len) ox[i].put(zero), of[i].put(zero);
        }
        w.store(p, dx, t, te, full, ox);
        w.store(p, df, t, te, full, of);
        if constexpr (TS == 1)
#pragma unroll
            for (int v = 0; v < VEC; ++v) s[v] = sn[v];
    }
    if (p.dh0 && blockIdx.y == 0 && w.ok && w.ts == 0)
#pragma unroll
        for (int v = 0; v < VEC; ++v) p.dh0[w.nd + v] = s[v];
}

template <typename T, int VEC>
__global__ __launch_bounds__(NTH) void rec_step_kernel(const T* __restrict__ x, const T* __restrict__ f, float* __restrict__ st,
                                                       T* __restrict__ y, int64_t cols, int dv, int64_t xs, int64_t fs, int D) {
    const int64_t col = (int64_t)blockIdx.x * NTH + threadIdx.x;
    if (col >= cols) return;
    const int64_t n = col / dv, d = (col - n * dv) * VEC;
    const Raw<T, VEC> rx = ldr<T, VEC>(x + n * xs + d), rf = ldr<T, VEC>(f + n * fs + d);
    Raw<float, VEC> h = ldr<float, VEC>(st + n * D + d);
    Raw<T, VEC> o;
    float hv[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        float a, i;
        gate<T>(rf.get(v), a, i);
        hv[v] = fmaf(a, h.get(v), i * rx.get(v));
    }
    h.put(hv);
    o.put(hv);
    str<float, VEC>(st + n * D + d, h);
    str<T, VEC>(y + n * D + d, o);
}

// VEC = 2 needs every row of every operand on a 2-element boundary
bool is_wide(const DttRecurrence* g) {
    const int e = g->dtype ? 2 : 4;
    int64_t s = g->D;                             // (strides of axes of one element do not count)
    if (g->N > g->NI) s |= g->x_so | g->f_so | g->g_so;
    if (g->NI > 1) s |= g->x_si | g->f_si | g->g_si;
    if (g->L > 1) s |= g->x_sl | g->f_sl | g->g_sl;
    const uintptr_t a = (uintptr_t)g->x | (uintptr_t)g->f | (uintptr_t)g->dy | (uintptr_t)g->y | (uintptr_t)g->dx | (uintptr_t)g->df;
    return s % 2 == 0 && a % (2 * e) == 0;
}
// How a call is cut: one time lane per column where the columns alone give every CU its eight waves (a tile then is TC
// steps), else 8 time lanes; and, where that leaves CUs empty, segments of the time axis (of four tiles at least) whose maps
// a first launch folds: as many as fill one round of resident workgroups.  Residence goes by registers: four workgroups a
// CU forward, three backward (two in fp32); 30 segments instead of 24, a quarter into a second round, took 65 instead of
// 57 us in a backward pass over 2 x 15001 x 1024.
struct Plan { int ts, vec, nseg, seg, tiles; int64_t cols, groups; };
Plan plan_of(const DttRecurrence* g) {
    const int64_t N = g->N;
    const int L = g->L, D = g->D, slots = g->dy ? g->dtype ? 768 : 512 : 1024;
    Plan q;
    q.vec = is_wide(g) ? 2 : 1;
    q.cols = N * ((D + q.vec - 1) / q.vec);
    q.ts = N * ((D + 1) / 2) >= 256 * 8 * 64 ? 1 : TSPLIT;    // (not by vec: the backward call has to cut the tiles as its forward did)
    const int tile = q.ts * TC;
    q.tiles = (L + tile - 1) / tile;
    const int CL = NTH / q.ts;
    q.groups = (q.cols + CL - 1) / CL;
    q.nseg = 1;
    if (q.ts > 1) {
        const int64_t want = slots / q.groups, most = q.tiles / 4;
        q.nseg = (int)(want < 1 ? 1 : want > most ? (most < 1 ? 1 : most) : want);
    }
    q.seg = (q.tiles + q.nseg - 1) / q.nseg * tile;
    q.nseg = (L + q.seg - 1) / q.seg;
    return q;
}

int fill(RecP& p, const DttRecurrence* g, Plan& q, const char* what) {
    DTT_CHECK(g, "%s: null argument", what);
    DTT_CHECK(g->N > 0 && g->L > 0 && g->D > 0 && g->NI > 0 && g->N % g->NI == 0, "%s: bad sizes N=%d NI=%d L=%d D=%d", what, g->N,
              g->NI, g->L, g->D);
    q = plan_of(g);
    DTT_CHECK(g->L <= (1 << 30), "%s: L=%d, at most 2^30", what, g->L);
    DTT_CHECK(g->dtype == 0 || g->dtype == 1, "%s: dtype must be 0 (float32) or 1 (bfloat16)", what);
    DTT_CHECK(g->x && g->f, "%s: null buffer", what);
    DTT_CHECK(q.groups * NTH < DTT_MAX_THREADS, "%s: too many columns", what);
    const int64_t need = q.nseg > 1 ? (int64_t)q.nseg * 2 * g->N * g->D * 4 : 0;
    DTT_CHECK(need == 0 || (g->ws && g->ws_bytes >= need), "%s: workspace of %lld bytes, %lld given", what, (long long)need,
              (long long)g->ws_bytes);
    p = RecP{};
    p.x = g->x; p.f = g->f; p.dy = g->dy; p.y = g->y; p.dx = g->dx; p.df = g->df;
    p.h0 = g->h0; p.dlast = g->dlast; p.last = g->last; p.dh0 = g->dh0; p.st = g->states; p.agg = (float*)g->ws; p.len = g->lengths;
    p.x_so = g->x_so; p.x_si = g->x_si; p.x_sl = g->x_sl;
    p.f_so = g->f_so; p.f_si = g->f_si; p.f_sl = g->f_sl;
    p.g_so = g->g_so; p.g_si = g->g_si; p.g_sl = g->g_sl;
    p.cols = q.cols; p.N = g->N; p.NI = g->NI; p.L = g->L; p.D = g->D; p.dv = (g->D + q.vec - 1) / q.vec;
    p.reverse = g->reverse; p.nseg = q.nseg; p.seg = q.seg;
    return 0;
}
template <typename T, int VEC, int TS> void launch_fwd(const RecP& p, const Plan& q, hipStream_t s) {
    const dim3 grid((unsigned)q.groups, q.nseg);
    if constexpr (TS > 1)
        if (q.nseg > 1) hipLaunchKernelGGL((rec_agg_kernel<T, VEC, TS, false>), grid, dim3(NTH), 0, s, p);
    hipLaunchKernelGGL((rec_fwd_kernel<T, VEC, TS>), grid, dim3(NTH), 0, s, p);
}
template <typename T, int VEC, int TS> void launch_bwd(const RecP& p, const Plan& q, hipStream_t s) {
    const dim3 grid((unsigned)q.groups, q.nseg);
    if constexpr (TS > 1)
        if (q.nseg > 1) hipLaunchKernelGGL((rec_agg_kernel<T, VEC, TS, true>), grid, dim3(NTH), 0, s, p);
    hipLaunchKernelGGL((rec_bwd_kernel<T, VEC, TS>), grid, dim3(NTH), 0, s, p);
}
#define REC_DISPATCH(FN)                                                                                                   \
    do {                                                                                                                   \
        if (g->dtype == 0) {                                                                                               \
            if (q.vec == 2) { if (q.ts == 1) FN<float, 2, 1>(p, q, s); else FN<float, 2, TSPLIT>(p, q, s); }               \
            else { if (q.ts == 1) FN<float, 1, 1>(p, q, s); else FN<float, 1, TSPLIT>(p, q, s); }                          \
        } else {                                                                                                           \
            if (q.vec == 2) { if (q.ts == 1) FN<bf16, 2, 1>(p, q, s); else FN<bf16, 2, TSPLIT>(p, q, s); }                 \
            else { if (q.ts == 1) FN<bf16, 1, 1>(p, q, s); else FN<bf16, 1, TSPLIT>(p, q, s); }                            \
        }                                                                                                                  \
    } while (0)
}  // namespace

extern "C" int64_t dtt_recurrence_ws_bytes(const DttRecurrence* g) {
    if (!g || g->N <= 0 || g->L <= 0 || g->D <= 0) return 0;
    const Plan q = plan_of(g);
    return q.nseg > 1 ? (int64_t)q.nseg * 2 * g->N * g->D * 4 : 0;
}

extern "C" int64_t dtt_recurrence_states(const DttRecurrence* g) {
    if (!g || g->N <= 0 || g->L <= 0 || g->D <= 0) return 0;
    return (int64_t)plan_of(g).tiles * g->N * g->D;
}

extern "C" int dtt_recurrence_fwd(const DttRecurrence* g, void* stream) {
    Plan q;
    RecP p;
    if (int rc = fill(p, g, q, "dtt_recurrence_fwd")) return rc;
    DTT_CHECK(g->y, "dtt_recurrence_fwd: null buffer");
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    REC_DISPATCH(launch_fwd);
    DTT_LAUNCH_CHECK();
    return 0;
}

extern "C" int dtt_recurrence_bwd(const DttRecurrence* g, void* stream) {
    Plan q;
    RecP p;
    if (int rc = fill(p, g, q, "dtt_recurrence_bwd")) return rc;
    DTT_CHECK(g->dy && g->dx && g->df && (g->states || q.tiles == 1), "dtt_recurrence_bwd: null buffer");
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    REC_DISPATCH(launch_bwd);
    DTT_LAUNCH_CHECK();
    return 0;
}

extern "C" int dtt_recurrence_step(const void* x, const void* f, float* state, void* y, int N, int D, int64_t x_sn, int64_t f_sn,
                                   int dtype, void* stream) {
    DTT_CHECK(x && f && state && y, "dtt_recurrence_step: null buffer");
    DTT_CHECK(N > 0 && D > 0 && (dtype == 0 || dtype == 1), "dtt_recurrence_step: bad arguments N=%d D=%d dtype=%d", N, D, dtype);
    const int e = dtype ? 2 : 4;
    const bool wide = (x_sn | f_sn | D) % 4 == 0 && ((uintptr_t)x | (uintptr_t)f | (uintptr_t)y) % (4 * e) == 0 &&
                      (uintptr_t)state % 16 == 0;
    const int dv = wide ? D / 4 : D;
    const int64_t cols = (int64_t)N * dv;
    DTT_CHECK(cols + NTH < DTT_MAX_THREADS, "dtt_recurrence_step: too many columns");
    const dim3 grid((unsigned)((cols + NTH - 1) / NTH));
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define STEP(T, V) hipLaunchKernelGGL((rec_step_kernel<T, V>), grid, dim3(NTH), 0, s, (const T*)x, (const T*)f, state, (T*)y, cols, dv, x_sn, f_sn, D)
    if (dtype == 0) { if (wide) STEP(float, 4); else STEP(float, 1); }
    else { if (wide) STEP(bf16, 4); else STEP(bf16, 1); }
#undef STEP
    DTT_LAUNCH_CHECK();
    return 0;
}
