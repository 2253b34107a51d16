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
#include "common.h"
#include "../../include/dtt_hip.h"

namespace {
constexpr int NTH = 256, TC = 4;                 // threads of a workgroup, steps a thread folds per tile

template <typename T, int VEC> struct Raw;       // VEC consecutive channels as loaded
template <> struct Raw<float, 4> {
    float4 v;
    __device__ __forceinline__ float get(int i) const { return (&v.x)[i]; }
    __device__ __forceinline__ void set(int i, float f) { (&v.x)[i] = f; }
};
template <> struct Raw<float, 1> {
    float v;
    __device__ __forceinline__ float get(int) const { return v; }
    __device__ __forceinline__ void set(int, float f) { v = f; }
};
template <> struct Raw<bf16, 4> {
    uint2 v;
    __device__ __forceinline__ float get(int i) const {
        const uint32_t w = (&v.x)[i >> 1];
        return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
    }
    __device__ __forceinline__ void set(int i, float f) {
        uint32_t& w = (&v.x)[i >> 1];
        const uint32_t b = f2bf(f);
        w = (i & 1) ? ((w & 0xffffu) | (b << 16)) : ((w & 0xffff0000u) | b);
    }
};
template <> struct Raw<bf16, 1> {
    unsigned short v;
    __device__ __forceinline__ float get(int) const { return bf2f(v); }
    __device__ __forceinline__ void set(int, float f) { v = f2bf(f); }
};
template <typename T, int VEC> __device__ __forceinline__ Raw<T, VEC> ldr(const T* p) {
    Raw<T, VEC> r;
    r.v = *reinterpret_cast<const decltype(r.v)*>(p);
    return r;
}
template <typename T, int VEC> __device__ __forceinline__ void str(T* p, const Raw<T, VEC>& r) {
    *reinterpret_cast<decltype(r.v)*>(p) = r.v;
}

// a = sigmoid(f) and i = 1 - a, both to the last bits: the smaller of the two from the exponential, the larger as one
// minus it.  fp32: the rounding of |f| log2(e) is carried along (|f| up to 80 would lose 6 bits); bf16 does not show it.
template <typename T> __device__ __forceinline__ void gate(float f, float& a, float& i) {
    float m = fabsf(f), e;
    if constexpr (sizeof(T) == 4) {
        m = m > 127.f ? 127.f : m;                // infinities too; NaN stays
        const float t = m * -1.4426950408889634f;
        const float lo = fmaf(m, -1.4426950408889634f, -t) + m * -1.925963033500e-8f;
        e = __builtin_amdgcn_exp2f(t);
        e = fmaf(e * 0.6931471805599453f, lo, e);
    } else {
        e = __builtin_amdgcn_exp2f(m * -1.4426950408889634f);
    }
    const float sm = e * __builtin_amdgcn_rcpf(1.0f + e), lg = 1.0f - sm;
    a = f >= 0.f ? lg : sm;
    i = f >= 0.f ? sm : lg;
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
};

// Combines the TS time lanes' maps (A, H) of one column and returns the state that this lane starts from, given the
// state `carry` that the tile starts from (of all lanes); carry becomes the state behind the tile.  BACK: later lanes
// first.  tot: LDS of [waves][CL][2][VEC], two copies used in turn so that one barrier a tile is enough.
template <int VEC, int TS, bool BACK>
__device__ __forceinline__ void combine(float (&A)[VEC], float (&H)[VEC], float (&carry)[VEC], float (&in)[VEC], int ts, int cl,
                                        float* tot) {
    constexpr int CL = NTH / TS, TW = 64 / CL, NW = NTH / 64;       // time lanes of a wave, waves
    const int wave = threadIdx.x >> 6, tw = ts % TW, pt = BACK ? TW - 1 - tw : tw;
#pragma unroll
    for (int o = 1; o < TW; o <<= 1) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float a = BACK ? __shfl_down(A[v], o * CL, 64) : __shfl_up(A[v], o * CL, 64);
            const float h = BACK ? __shfl_down(H[v], o * CL, 64) : __shfl_up(H[v], o * CL, 64);
            H[v] = pt >= o ? fmaf(A[v], h, H[v]) : H[v];
            A[v] = pt >= o ? A[v] * a : A[v];
        }
    }
    if (pt == TW - 1)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            tot[((wave * CL + cl) * 2 + 0) * VEC + v] = A[v];
            tot[((wave * CL + cl) * 2 + 1) * VEC + v] = H[v];
        }
    float ea[VEC], eh[VEC];                                          // the lanes of this wave ahead of this one
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        const float a = BACK ? __shfl_down(A[v], CL, 64) : __shfl_up(A[v], CL, 64);
        const float h = BACK ? __shfl_down(H[v], CL, 64) : __shfl_up(H[v], CL, 64);
        ea[v] = pt ? a : 1.f;
        eh[v] = pt ? h : 0.f;
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

// state ahead of segment `seg` from the maps of the segments before it (BACK: behind it)
template <int VEC, bool BACK>
__device__ __forceinline__ void fold_segments(const RecP& p, int64_t nd, const float* start, float (&c)[VEC]) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) c[v] = start ? start[nd + v] : 0.f;
    const int seg = blockIdx.y, cnt = BACK ? p.nseg - 1 - seg : seg;
    const int64_t ND = (int64_t)p.N * p.D;
    for (int k = 0; k < cnt; ++k) {
        const float* g = p.agg + (int64_t)(BACK ? p.nseg - 1 - k : k) * 2 * ND + nd;
#pragma unroll
        for (int v = 0; v < VEC; ++v) c[v] = fmaf(g[v], c[v], g[ND + v]);
    }
}

// (A, H) of every segment: a time lane folds seg / TS consecutive steps.  BACK: the map of s over the segment, from its
// last step to its first, with dy in x's place.
template <typename T, int VEC, int TS, bool BACK>
__global__ __launch_bounds__(NTH) void rec_agg_kernel(const RecP p) {
    constexpr int CL = NTH / TS, UN = 8;
    __shared__ float tot[NTH / 64 * CL * 2 * VEC];
    const Place<VEC, TS> w(p);
    const T* f = (const T*)p.f + (int64_t)(w.n / p.NI) * p.f_so + (int64_t)(w.n % p.NI) * p.f_si + w.d0;
    const T* x = BACK ? (const T*)p.dy + (int64_t)(w.n / p.NI) * p.g_so + (int64_t)(w.n % p.NI) * p.g_si + w.d0
                      : (const T*)p.x + (int64_t)(w.n / p.NI) * p.x_so + (int64_t)(w.n % p.NI) * p.x_si + w.d0;
    const int64_t xl = BACK ? p.g_sl : p.x_sl;
    const int per = p.seg / TS, t0 = blockIdx.y * p.seg + w.ts * per, t1 = min(t0 + per, w.len);
    float A[VEC], H[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) A[v] = 1.f, H[v] = 0.f;
    for (int tb = t0; tb < t1; tb += UN) {
        Raw<T, VEC> rf[UN], rx[UN];
#pragma unroll
        for (int i = 0; i < UN; ++i) {
            const int k = min(tb + i, t1 - 1), t = BACK ? t0 + t1 - 1 - k : k, r = w.row(p, t);
            rf[i] = ldr<T, VEC>(f + (int64_t)r * p.f_sl);
            rx[i] = ldr<T, VEC>(x + (int64_t)r * xl);
        }
#pragma unroll
        for (int i = 0; i < UN; ++i) {
            const bool on = tb + i < t1;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float a, im;
                gate<T>(rf[i].get(v), a, im);
                const float h = BACK ? a * (rx[i].get(v) + H[v]) : fmaf(a, H[v], im * rx[i].get(v));
                H[v] = on ? h : H[v];
                A[v] = on ? A[v] * a : A[v];
            }
        }
    }
    // the whole segment's map: start from the two unit states (A: 1 -> with H's left out, H: 0)
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
    fold_segments<VEC, false>(p, w.nd, p.h0, c);
    Raw<T, VEC> nx[TC], nf[TC];
    auto load = [&](int tb) {
#pragma unroll
        for (int i = 0; i < TC; ++i) {
            const int t = tb + w.ts * TC + i, r = t < w.len ? w.row(p, t) : 0;
            nx[i] = ldr<T, VEC>(x + (int64_t)r * p.x_sl);
            nf[i] = ldr<T, VEC>(f + (int64_t)r * p.f_sl);
        }
    };
    load(ta);
    int buf = 0;
    for (int tb = ta; tb < te; tb += TILE) {
        if (p.st && tb > 0 && w.ok && w.ts == 0) {
            float* s = p.st + (int64_t)(tb / TILE) * p.N * p.D + w.nd;
#pragma unroll
            for (int v = 0; v < VEC; ++v) s[v] = c[v];
        }
        float a[TC][VEC], b[TC][VEC], A[VEC], H[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) A[v] = 1.f, H[v] = 0.f;
#pragma unroll
        for (int i = 0; i < TC; ++i) {
            const bool live = tb + w.ts * TC + i < w.len;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float im;
                gate<T>(nf[i].get(v), a[i][v], im);
                a[i][v] = live ? a[i][v] : 1.f;                 // padding: the state passes
                b[i][v] = live ? im * nx[i].get(v) : 0.f;
                if constexpr (TS > 1) {
                    H[v] = fmaf(a[i][v], H[v], b[i][v]);
                    A[v] *= a[i][v];
                }
            }
        }
        if (tb + TILE < te) load(tb + TILE);
        float h[VEC];
        if constexpr (TS > 1) {
            combine<VEC, TS, false>(A, H, c, h, w.ts, w.cl, tot[buf]);
            buf ^= 1;
        } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) h[v] = c[v];
        }
#pragma unroll
        for (int i = 0; i < TC; ++i) {
            const int t = tb + w.ts * TC + i;
            Raw<T, VEC> o;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                h[v] = fmaf(a[i][v], h[v], b[i][v]);
                o.set(v, t < w.len ? h[v] : 0.f);
            }
            if (w.ok && t < te) str<T, VEC>(y + (int64_t)w.row(p, t) * p.D, o);
        }
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
    fold_segments<VEC, true>(p, w.nd, p.dlast, s);
    Raw<T, VEC> nx[TC], nf[TC], ng[TC];
    float nc[VEC];
    auto load = [&](int tb) {
#pragma unroll
        for (int i = 0; i < TC; ++i) {
            const int t = tb + w.ts * TC + i, r = t < w.len ? w.row(p, t) : 0;
            nx[i] = ldr<T, VEC>(x + (int64_t)r * p.x_sl);
            nf[i] = ldr<T, VEC>(f + (int64_t)r * p.f_sl);
            ng[i] = ldr<T, VEC>(dy + (int64_t)r * p.g_sl);
        }
        const float* st = tb > 0 ? p.st + (int64_t)(tb / TILE) * p.N * p.D : p.h0;
#pragma unroll
        for (int v = 0; v < VEC; ++v) nc[v] = st ? st[w.nd + v] : 0.f;
    };
    const int tl = ta + (te - ta - 1) / TILE * TILE;
    load(tl);
    int buf = 0;
    for (int tb = tl; tb >= ta; tb -= TILE) {
        float a[TC][VEC], im[TC][VEC], d[TC][VEC], g[TC][VEC], A[VEC], H[VEC], c[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) A[v] = 1.f, H[v] = 0.f, c[v] = nc[v];
#pragma unroll
        for (int i = 0; i < TC; ++i) {
            const bool live = tb + w.ts * TC + i < w.len;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                gate<T>(nf[i].get(v), a[i][v], im[i][v]);
                a[i][v] = live ? a[i][v] : 1.f;
                im[i][v] = live ? im[i][v] : 0.f;
                d[i][v] = live ? nx[i].get(v) : 0.f;                  // x, then h_{t-1} - x
                g[i][v] = live ? ng[i].get(v) : 0.f;
                if constexpr (TS > 1) {
                    H[v] = fmaf(a[i][v], H[v], im[i][v] * d[i][v]);
                    A[v] *= a[i][v];
                }
            }
        }
        if (tb > ta) load(tb - TILE);
        float h[VEC];
        if constexpr (TS > 1) {
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
#pragma unroll
        for (int i = TC - 1; i >= 0; --i) {
            const int t = tb + w.ts * TC + i;
            Raw<T, VEC> ox, of;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float gt = g[i][v] + sn[v], gx = im[i][v] * gt;
                ox.set(v, gx);                                        // (0 behind the length: im = 0)
                of.set(v, gx * a[i][v] * d[i][v]);
                sn[v] = a[i][v] * gt;
            }
            if (w.ok && t < te) {
                const int64_t r = (int64_t)w.row(p, t) * p.D;
                str<T, VEC>(dx + r, ox);
                str<T, VEC>(df + r, of);
            }
        }
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
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        float a, i;
        gate<T>(rf.get(v), a, i);
        const float hv = fmaf(a, h.get(v), i * rx.get(v));
        h.set(v, hv);
        o.set(v, hv);
    }
    str<float, VEC>(st + n * D + d, h);
    str<T, VEC>(y + n * D + d, o);
}

constexpr int TSPLIT = 16;                       // time lanes of the split form

// How a call is cut: one time lane per column where the columns alone give every CU its eight waves (a tile then is TC
// steps), else 16 time lanes; and, while that leaves fewer than four workgroups a CU, segments of the time axis whose
// maps a first launch folds.
struct Plan { int ts, vec, nseg, seg, tiles; int64_t cols, groups; };
Plan plan_of(int64_t N, int L, int D, bool wide) {
    Plan q;
    q.vec = wide ? 4 : 1;
    q.cols = N * ((D + q.vec - 1) / q.vec);
    q.ts = N * ((D + 3) / 4) >= 256 * 8 * 64 ? 1 : TSPLIT;    // (not by vec: the backward call has to cut the tiles as its forward did)
    const int tile = q.ts * TC;
    q.tiles = (L + tile - 1) / tile;
    const int CL = NTH / q.ts;
    q.groups = (q.cols + CL - 1) / CL;
    q.nseg = 1;
    if (q.ts > 1) {
        const int64_t want = 1024 / q.groups, most = q.tiles / 4;     // segments of four tiles at least
        q.nseg = (int)(want < 1 ? 1 : want > most ? (most < 1 ? 1 : most) : want);
    }
    q.seg = (q.tiles + q.nseg - 1) / q.nseg * tile;
    q.nseg = (L + q.seg - 1) / q.seg;
    return q;
}

// VEC = 4 needs every row of every operand on a 4-element boundary
bool is_wide(const DttRecurrence* g) {
    const int e = g->dtype ? 2 : 4;
    int64_t s = g->D;                             // (strides of axes of one element do not count)
    if (g->N > g->NI) s |= g->x_so | g->f_so | g->g_so;
    if (g->NI > 1) s |= g->x_si | g->f_si | g->g_si;
    if (g->L > 1) s |= g->x_sl | g->f_sl | g->g_sl;
    const uintptr_t a = (uintptr_t)g->x | (uintptr_t)g->f | (uintptr_t)g->dy | (uintptr_t)g->y | (uintptr_t)g->dx | (uintptr_t)g->df;
    return s % 4 == 0 && a % (4 * e) == 0;
}
int fill(RecP& p, const DttRecurrence* g, Plan& q, const char* what) {
    DTT_CHECK(g, "%s: null argument", what);
    DTT_CHECK(g->N > 0 && g->L > 0 && g->D > 0 && g->NI > 0 && g->N % g->NI == 0, "%s: bad sizes N=%d NI=%d L=%d D=%d", what, g->N,
              g->NI, g->L, g->D);
    q = plan_of(g->N, g->L, g->D, is_wide(g));
    DTT_CHECK(g->L <= (1 << 30), "%s: L=%d, at most 2^30", what, g->L);
    DTT_CHECK(g->dtype == 0 || g->dtype == 1, "%s: dtype must be 0 (float32) or 1 (bfloat16)", what);
    DTT_CHECK(g->x && g->f, "%s: null buffer", what);
    DTT_CHECK(q.groups < (1ll << 31), "%s: too many columns", what);
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
            if (q.vec == 4) { if (q.ts == 1) FN<float, 4, 1>(p, q, s); else FN<float, 4, TSPLIT>(p, q, s); }               \
            else { if (q.ts == 1) FN<float, 1, 1>(p, q, s); else FN<float, 1, TSPLIT>(p, q, s); }                          \
        } else {                                                                                                           \
            if (q.vec == 4) { if (q.ts == 1) FN<bf16, 4, 1>(p, q, s); else FN<bf16, 4, TSPLIT>(p, q, s); }                 \
            else { if (q.ts == 1) FN<bf16, 1, 1>(p, q, s); else FN<bf16, 1, TSPLIT>(p, q, s); }                            \
        }                                                                                                                  \
    } while (0)
}  // namespace

extern "C" int64_t dtt_recurrence_ws_bytes(const DttRecurrence* g) {
    if (!g || g->N <= 0 || g->L <= 0 || g->D <= 0) return 0;
    const Plan q = plan_of(g->N, g->L, g->D, is_wide(g));
    return q.nseg > 1 ? (int64_t)q.nseg * 2 * g->N * g->D * 4 : 0;
}

extern "C" int64_t dtt_recurrence_states(const DttRecurrence* g) {
    if (!g || g->N <= 0 || g->L <= 0 || g->D <= 0) return 0;
    return (int64_t)plan_of(g->N, g->L, g->D, is_wide(g)).tiles * g->N * g->D;
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
    DTT_CHECK(cols < (1ll << 38), "dtt_recurrence_step: too many columns");
    const dim3 grid((unsigned)((cols + NTH - 1) / NTH));
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define STEP(T, V) hipLaunchKernelGGL((rec_step_kernel<T, V>), grid, dim3(NTH), 0, s, (const T*)x, (const T*)f, state, (T*)y, cols, dv, x_sn, f_sn, D)
    if (dtype == 0) { if (wide) STEP(float, 4); else STEP(float, 1); }
    else { if (wide) STEP(bf16, 4); else STEP(bf16, 1); }
#undef STEP
    DTT_LAUNCH_CHECK();
    return 0;
}
