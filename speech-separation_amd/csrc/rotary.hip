// Rotary positions: every pair (u, v) of the first r channels of a query or key head is turned by the angle
// position * frequency and scaled by `amplitude`; the channels behind r are copied.  Half layout: pair i is (i, i + r/2);
// interleaved: (2i, 2i + 1).  Turning back (sign = -1) is the backward pass.
//
// Bound: HBM (q and k read and written once).  Angles: a position far into a stream times a frequency needs more than 24
// bits, so the product and its reduction to a fraction of a turn are done in fp64, and sine and cosine of that fraction
// in fp32, with what the fraction's rounding left off as a first-order correction (without it results were 1.3 times as far from
// the exact ones as with exact angles).  A workgroup takes the (token, pair) angles of a few tokens once into LDS and uses them for all heads of q and k.
// Measured: 4 x 4096 tokens, 16 + 4 heads of 128, bf16: 39 us (4.3 TB/s); 3 x 5001, 8 + 8 heads of 64, fp32: 25 us (4.9 TB/s).
#include "common.h"
#include "../../include/dtt_hip.h"

namespace {
constexpr int NTH = 256;

struct RotP {
    const void* x[2]; void* y[2];
    int64_t sb[2], st[2], sh[2];                 // element strides of q, k
    int H[2];
    const void* pos; const double* freq;
    int64_t pb, pt;
    int pos64, T, dh, r, tok;                    // tok: tokens of a workgroup
    int64_t n;                                   // tokens
    float sign, amp;
};

template <typename T, int VEC> struct alignas(VEC * sizeof(T)) RVec { T e[VEC]; };

template <typename T, int VEC, bool INTER>
__global__ __launch_bounds__(NTH) void rotary_kernel(const RotP p) {
    extern __shared__ float2 cs[];               // [tok][r / 2]
    const int half = p.r / 2;
    const int64_t t0 = (int64_t)blockIdx.x * p.tok;
    const int nt = (int)min((int64_t)p.tok, p.n - t0);
    for (int i = threadIdx.x; i < nt * half; i += NTH) {
        const int64_t tok = t0 + i / half;
        const int64_t at = tok / p.T * p.pb + tok % p.T * p.pt;
        const double pos = p.pos64 ? (double)((const int64_t*)p.pos)[at] : (double)((const int*)p.pos)[at];
        const double turns = pos * (p.freq[i % half] * 0.15915494309189533577);
        const double part = turns - rint(turns);
        const float near = (float)part, d = (float)(part - near) * 6.283185307f;
        float s, c;
        sincospif(2.0f * near, &s, &c);
        cs[i] = make_float2(fmaf(-s, d, c) * p.amp, fmaf(c, d, s) * p.amp * p.sign);
    }
    __syncthreads();
    // items of a head: pairs of vectors (half layout) or vectors (interleaved) of the turned part, then copied vectors
    // (interleaved with VEC = 1, for rows at odd elements: a pair by its two elements)
    const int nr = (INTER && VEC > 1 ? p.r : half) / VEC, ni = nr + (p.dh - p.r) / VEC, heads = p.H[0] + p.H[1];
    typedef RVec<T, VEC> V;
    for (int i = threadIdx.x; i < nt * heads * ni; i += NTH) {
        const int tk = i / (heads * ni), hi = i / ni % heads, it = i % ni, w = hi >= p.H[0], h = w ? hi - p.H[0] : hi;
        const int64_t tok = t0 + tk;
        const T* x = (const T*)p.x[w] + tok / p.T * p.sb[w] + tok % p.T * p.st[w] + h * p.sh[w];
        T* y = (T*)p.y[w] + (tok * p.H[w] + h) * p.dh;
        if (it >= nr) {
            const int d = p.r + (it - nr) * VEC;
            *(V*)(y + d) = *(const V*)(x + d);
        } else if constexpr (INTER && VEC == 1) {
            const float2 t = cs[tk * half + it];
            const float u = ldf(x + 2 * it), v = ldf(x + 2 * it + 1);
            stf(y + 2 * it, u * t.x - v * t.y);
            stf(y + 2 * it + 1, u * t.y + v * t.x);
        } else if constexpr (INTER) {
            V a = *(const V*)(x + it * VEC);
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
                const float2 t = cs[tk * half + (it * VEC + e) / 2];
                const float u = ldf(&a.e[e]), v = ldf(&a.e[e + 1]);
                stf(&a.e[e], u * t.x - v * t.y);
                stf(&a.e[e + 1], u * t.y + v * t.x);
            }
            *(V*)(y + it * VEC) = a;
        } else {
            V a = *(const V*)(x + it * VEC), b = *(const V*)(x + half + it * VEC);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float2 t = cs[tk * half + it * VEC + e];
                const float u = ldf(&a.e[e]), v = ldf(&b.e[e]);
                stf(&a.e[e], u * t.x - v * t.y);
                stf(&b.e[e], u * t.y + v * t.x);
            }
            *(V*)(y + it * VEC) = a;
            *(V*)(y + half + it * VEC) = b;
        }
    }
}
}  // namespace

extern "C" int dtt_rotary(const DttRotary* g, void* stream) {
    DTT_CHECK(g, "dtt_rotary: null argument");
    DTT_CHECK(g->dtype == 0 || g->dtype == 1, "dtt_rotary: dtype must be 0 (float32) or 1 (bfloat16)");
    DTT_CHECK(g->B > 0 && g->T > 0 && g->Hq > 0 && g->Hk >= 0 && g->dh > 0 && g->r > 0 && g->r % 2 == 0 && g->r <= g->dh,
              "dtt_rotary: bad sizes B=%d T=%d Hq=%d Hk=%d dh=%d r=%d", g->B, g->T, g->Hq, g->Hk, g->dh, g->r);
    DTT_CHECK(g->r <= 4096, "dtt_rotary: r=%d, at most 4096", g->r);
    DTT_CHECK(g->q && g->qo && g->positions && g->freq && (g->Hk == 0 || (g->k && g->ko)), "dtt_rotary: null buffer");
    RotP p{};
    p.x[0] = g->q; p.x[1] = g->k; p.y[0] = g->qo; p.y[1] = g->ko;
    // (strides of axes of one element do not count)
    p.sb[0] = g->B > 1 ? g->q_sb : 0; p.st[0] = g->T > 1 ? g->q_st : 0; p.sh[0] = g->Hq > 1 ? g->q_sh : 0;
    p.sb[1] = g->B > 1 ? g->k_sb : 0; p.st[1] = g->T > 1 ? g->k_st : 0; p.sh[1] = g->Hk > 1 ? g->k_sh : 0;
    p.H[0] = g->Hq; p.H[1] = g->Hk;
    p.pos = g->positions; p.freq = g->freq; p.pb = g->p_sb; p.pt = g->p_st; p.pos64 = g->pos64;
    p.T = g->T; p.dh = g->dh; p.r = g->r; p.n = (int64_t)g->B * g->T;
    p.sign = g->back ? -1.f : 1.f; p.amp = g->amplitude;
    // widest vector that divides every part of a head and that every row starts on
    const int e = g->dtype ? 2 : 4, part = g->interleaved ? g->r : g->r / 2;
    int64_t str = p.sb[0] | p.st[0] | p.sh[0] | part | (g->dh - g->r) | g->dh;
    uintptr_t ad = (uintptr_t)g->q | (uintptr_t)g->qo;
    if (g->Hk) str |= p.sb[1] | p.st[1] | p.sh[1], ad |= (uintptr_t)g->k | (uintptr_t)g->ko;
    int vec = 16 / e;
    while (vec > 1 && (str % vec || ad % (vec * e))) vec /= 2;
    // tokens of a workgroup: about four passes of the threads over its items, no more than leaves four workgroups a CU
    const int64_t items = ((int64_t)g->Hq + g->Hk) * ((g->interleaved ? g->r : g->r / 2) + g->dh - g->r) / vec;
    int64_t tok = (4 * NTH + items - 1) / items;
    if (tok > p.n / 1024) tok = p.n / 1024;
    if (tok > 4096 / p.r) tok = 4096 / p.r;
    p.tok = tok < 1 ? 1 : (int)tok;
    const int64_t grid = (p.n + p.tok - 1) / p.tok;
    DTT_CHECK(grid * NTH < DTT_MAX_THREADS, "dtt_rotary: too many tokens");
    DTT_CHECK(items * p.tok < (1ll << 31) - NTH, "dtt_rotary: too many heads");        // (a workgroup counts its items in 32 bits)
    const size_t lds = (size_t)p.tok * (p.r / 2) * sizeof(float2);
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define ROT(T, V, I) hipLaunchKernelGGL((rotary_kernel<T, V, I>), dim3((unsigned)grid), dim3(NTH), lds, s, p)
    if (g->dtype == 0) {
        if (g->interleaved) { if (vec == 4) ROT(float, 4, true); else if (vec == 2) ROT(float, 2, true); else ROT(float, 1, true); }
        else { if (vec == 4) ROT(float, 4, false); else if (vec == 2) ROT(float, 2, false); else ROT(float, 1, false); }
    } else {
        if (g->interleaved) {
            if (vec == 8) ROT(bf16, 8, true);
            else if (vec == 4) ROT(bf16, 4, true);
            else if (vec == 2) ROT(bf16, 2, true);
            else ROT(bf16, 1, true);
        } else {
            if (vec == 8) ROT(bf16, 8, false);
            else if (vec == 4) ROT(bf16, 4, false);
            else if (vec == 2) ROT(bf16, 2, false);
            else ROT(bf16, 1, false);
        }
    }
#undef ROT
    DTT_LAUNCH_CHECK();
    return 0;
}
