// Windowed attention with first tokens that stay visible.  The query at position p = offset + i sees the key at position j
// where  j <= p + right  and  (j >= p - left  or  j < sinks)  and  j < len;  positions from len on are padding (rows of
// zeros, no gradient); a row that sees nothing is a row of zeros.  q [B][Tq][Hq][DH], k, v [B][Tk][Hk][DH] by strides, Hq a
// multiple of Hk (query head h reads key head h / (Hq / Hk)), bf16 or fp32.
//
// One pass over the visible key tiles with the running maximum and sum of the softmax in fp32 (base 2: one v_exp_f32 a
// score).  Scores are formed transposed, S^T = K Q^T on 32x32 matrix tiles: a lane then owns one query (column lane & 31),
// so that the softmax statistics are per-lane scalars and one exchange with lane ^ 32, and the tile's accumulator
// registers, packed to the compute type, already are the B operand of O^T += V^T P^T: register r of a 16-key chunk holds key
// (r & 3) + 8 (r >> 2) + 4 (lane >> 5), and V^T's fragments are read from LDS in that order of keys.
// In bf16 the weights P and dS enter their products as two operands, the rounded value and what that left off (2^-16 of it in
// all): with the first alone (2^-8) results were 1.4 times as far from the exact ones as their own rounding puts them,
// whatever the window (o 2.22e-3 against 1.63e-3 relative, dv 2.33e-3 and dq 2.42e-3 against 1.66e-3).  Statistics,
// accumulators, D = sum(dO O) and first tokens' partial sums stay fp32.
//
// Bound: the matrix cores (4 DH flops per visible pair forward, 10 DH backward; in bf16 the second operands add 2 and 6 that the
// formulas do not have) for windows beyond a few hundred keys, HBM below.  Measured, bf16, 2 x 4096 rows, 16 / 4 heads of 128,
// window 512 + 4 first tokens (114 GF, 92 us at the rate of a large matrix product): forward 77 us (85 with what the backward pass
// wants of it), dq 103, dk / dv 156, the first tokens' sums 5; matrix cores busy 26 to 30 % of the time.  What keeps them from the
// rate are latencies in series (staging, Q K^T, exponentials, the pieces, P V) at the two waves a SIMD that the accumulators leave room for.
#include "common.h"
#include "../../include/dtt_hip.h"
#include <algorithm>

namespace {
constexpr int NTH = 256, BN = 64;                // threads (dk / dv: up to twice that); keys of a staged tile (forward, dq)
constexpr int QN = 64, MAX_SINKS = 128;          // dk / dv: query rows of a staged tile
constexpr float LOG2E = 1.4426950408889634f;

struct WaP {
    const void* q; const void* k; const void* v; const void* o; const void* dout;
    void* out; void* rest; void* dq; void* dk; void* dv;
    float* lse; float* dd; float* part;
    const int* len;
    int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh, g_sb, g_st, g_sh;
    int B, Tq, Tk, Hq, Hk, G, left, right, sinks, offset;
    int nt, nchunk, chunk, npart, edge;          // tiles along the row axis; chunks of the rows from edge on (first tokens' gradients)
    float scale;
};

// LDS image of rows of DH elements in 16-byte pieces; piece c of row r is stored at c ^ swz(r).  Rows are a power of two of
// pieces.  swz spreads both reads over all 64 banks: the natural fragment read (16 rows, one piece each) and the
// transposing read (four consecutive rows, four neighbouring pieces).
template <typename T, int DH> struct Img {
    static constexpr int EPP = 16 / sizeof(T), NP = DH / EPP;
    static constexpr int RP = NP <= 4 ? 4 : NP <= 8 ? 8 : NP <= 16 ? 16 : NP <= 32 ? 32 : 64, LD = RP * EPP;
    static __device__ __forceinline__ int swz(int r) {
        if constexpr (RP >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
        else if constexpr (RP == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
        else return (r >> 2) & 3;
    }
    static __device__ __forceinline__ int at(int r, int piece) { return r * LD + (piece ^ swz(r)) * EPP; }
};

// natural fragment: row r, the 8 elements from 16 c + 8 lh on
template <typename T, int DH> __device__ __forceinline__ typename MM<T>::Frag nat_frag(const T* img, int r, int c, int lh) {
    if constexpr (sizeof(T) == 2) {
        return MM<T>::ldfrag(img + Img<T, DH>::at(r, 2 * c + lh));
    } else {
        typename MM<T>::Frag f;
        f.lo = *reinterpret_cast<const float4*>(img + Img<T, DH>::at(r, 4 * c + 2 * lh));
        f.hi = *reinterpret_cast<const float4*>(img + Img<T, DH>::at(r, 4 * c + 2 * lh + 1));
        return f;
    }
}
// transposed fragment: column c0 + (lane & 31), rows kb + (e & 3) + 8 (e >> 2) + 4 lh for e = 0 .. 7
template <typename T, int DH> __device__ __forceinline__ typename MM<T>::Frag tr_frag_of(const T* img, int kb, int c0) {
    const int lane = threadIdx.x & 63, lh = lane >> 5;
    if constexpr (sizeof(T) == 2) {
        const int g = (lane >> 4) & 1, q = (lane & 15) >> 2, p = lane & 3, piece = c0 / 8 + 2 * g + (p >> 1), r = kb + 4 * lh + q;
        return tr_frag(img + Img<T, DH>::at(r, piece) + 4 * (p & 1), img + Img<T, DH>::at(r + 8, piece) + 4 * (p & 1));
    } else {
        const int d = c0 + (lane & 31);
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = img[Img<T, DH>::at(kb + (i & 3) + 8 * (i >> 2) + 4 * lh, d >> 2) + (d & 3)];
        typename MM<T>::Frag f;
        f.lo = make_float4(e[0], e[1], e[2], e[3]);
        f.hi = make_float4(e[4], e[5], e[6], e[7]);
        return f;
    }
}
// accumulator registers 8 c .. 8 c + 7 as an operand fragment
template <typename T> __device__ __forceinline__ typename MM<T>::Frag acc_frag(const f32x16_t& s, int c) {
    if constexpr (sizeof(T) == 2) {
        uint4 u = make_uint4(pack_bf16x2(s[8 * c], s[8 * c + 1]), pack_bf16x2(s[8 * c + 2], s[8 * c + 3]),
                             pack_bf16x2(s[8 * c + 4], s[8 * c + 5]), pack_bf16x2(s[8 * c + 6], s[8 * c + 7]));
        return __builtin_bit_cast(s16x8_t, u);
    } else {
        typename MM<T>::Frag f;
        f.lo = make_float4(s[8 * c], s[8 * c + 1], s[8 * c + 2], s[8 * c + 3]);
        f.hi = make_float4(s[8 * c + 4], s[8 * c + 5], s[8 * c + 6], s[8 * c + 7]);
        return f;
    }
}
// what the rounding of acc_frag left off registers 8 c .. 8 c + 7 (bf16), as a second operand fragment: the two pieces hold a
// value to 2^-16 of it
__device__ __forceinline__ s16x8_t rest_frag(const f32x16_t& s, int c, const s16x8_t& first) {
    const uint4 u = __builtin_bit_cast(uint4, first);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t w = (&u.x)[e >> 1];
        v[e] = s[8 * c + e] - __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
    }
    return __builtin_bit_cast(s16x8_t, make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])));
}
__device__ __forceinline__ f32x16_t zero_acc() {
    f32x16_t z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}
__device__ __forceinline__ int acc_row(int r, int lh) { return (r & 3) + 8 * (r >> 2) + 4 * lh; }

// R rows (row stride rs elements) into registers and on into an LDS image.  The tile's rows are a buffer of their own whose
// size ends with the last valid row, so that rows behind it read as zeros without a predicate, and a lane's offsets are
// the same 32-bit numbers for every tile (address arithmetic per lane was a quarter of
// the forward kernel's vector instructions).  Needs DH <= rs <= 2^22 (checked on the host).
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;
template <typename T, int DH, int R, int NT = NTH> struct Stage {
    typedef Img<T, DH> I;
    static constexpr int N = (R * I::RP + NT - 1) / NT;
    u32x4_t v[N];
    static constexpr int ROWS = NT / I::RP;       // rows between a lane's pieces
    uint32_t off, step;
    int at[2];
    __device__ __forceinline__ explicit Stage(int64_t rs) {
        const int r = threadIdx.x / I::RP, pc = threadIdx.x % I::RP;
        // (a lane without a piece of its own: beyond every buffer)
        off = pc < I::NP && r < R ? (uint32_t)(r * (int)rs + pc * I::EPP) * sizeof(T) : 0x80000000u;
        step = (uint32_t)(ROWS * (int)rs) * sizeof(T);
        at[0] = I::at(r, pc);                     // (the swizzle repeats every 16 rows: one place, or two in turn)
        at[1] = I::at(r + ROWS, pc) - ROWS * I::LD;
        static_assert(N == 1 || ROWS % 8 == 0, "");
    }
    __device__ __forceinline__ void load(const T* src, int64_t rs, int r0, int n) {
        const int rows = min(n - r0, R);
        const int bytes = rows > 0 ? ((rows - 1) * (int)rs + DH) * (int)sizeof(T) : 0;
        const __amdgpu_buffer_rsrc_t b = __builtin_amdgcn_make_buffer_rsrc((void*)(src + (int64_t)r0 * rs), 0, bytes, 0x00027000);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __builtin_amdgcn_raw_buffer_load_b128(b, off + i * step, 0, 0);
    }
    __device__ __forceinline__ void store(T* img) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (R * I::RP % NT == 0 || threadIdx.x < R * I::RP) *reinterpret_cast<u32x4_t*>(img + at[ROWS % 16 ? i & 1 : 0] + i * ROWS * I::LD) = v[i];
    }
};

// consecutive logical workgroups on one XCD (workgroup id % 8): the heads of a group and neighbouring tiles share keys
__device__ __forceinline__ int xcd_order(int id, int n) {
    const int per = n / 8;
    return id < per * 8 ? (id & 7) * per + (id >> 3) : id;
}

// 4 consecutive channels per register group of an O^T-shaped accumulator: row pointer + 32 ct + 8 q + 4 lh.  rest (bf16, may be
// null): the same row's place for what the rounding left off
template <typename T, int DH>
__device__ __forceinline__ void store_rows(T* row, const f32x16_t (&acc)[DH / 32], float mul, int lh, T* rest = nullptr) {
#pragma unroll
    for (int ct = 0; ct < DH / 32; ++ct)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            T* o = row + 32 * ct + 8 * q + 4 * lh;
            const float a = acc[ct][4 * q] * mul, b = acc[ct][4 * q + 1] * mul, c = acc[ct][4 * q + 2] * mul, d = acc[ct][4 * q + 3] * mul;
            if constexpr (sizeof(T) == 2) {
                const uint32_t u = pack_bf16x2(a, b), w = pack_bf16x2(c, d);
                *reinterpret_cast<uint2*>(o) = make_uint2(u, w);
                if (rest)
                    *reinterpret_cast<uint2*>(rest + (o - row)) =
                        make_uint2(pack_bf16x2(a - __uint_as_float(u << 16), b - __uint_as_float(u & 0xffff0000u)),
                                   pack_bf16x2(c - __uint_as_float(w << 16), d - __uint_as_float(w & 0xffff0000u)));
            } else {
                *reinterpret_cast<float4*>(o) = make_float4(a, b, c, d);
            }
        }
}

// The value of lane ^ 32 combined with this lane's: one exchange of the register file's halves (no LDS round trip)
__device__ __forceinline__ float both_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float both_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Raw scores x of 32 NX keys -> weights 2^(sc x - m), with the running reference m and sum l of this lane's query.  The
// reference need not be the maximum: it follows it only when a row's maximum has grown by more than 2^8 over it (weights up
// to 256 keep all their relative precision in fp32 and bf16), so that the accumulators are hardly ever rescaled.
template <int DH, int NX>
__device__ __forceinline__ void softmax_tile(f32x16_t (&x)[NX], float& m, float& l, f32x16_t (&o)[DH / 32], float sc) {
    float top = x[0][0];
#pragma unroll
    for (int n = 0; n < NX; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, x[n][r]);
    top = both_max(top) * sc;
    if (__any(top > m + 8.f)) {
        const float mn = fmaxf(m, top), al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        l *= al;
        m = mn;
#pragma unroll
        for (int c = 0; c < DH / 32; ++c)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[c][r] *= al;
    }
    const float mu = m == -INFINITY ? 0.f : m;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NX; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            x[n][r] = __builtin_amdgcn_exp2f(fmaf(x[n][r], sc, -mu));
            sum[r & 3] += x[n][r];
        }
    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// A wave's accumulators to and from LDS, [register][lane]: waves that share rows add up their halves there
template <int N> __device__ __forceinline__ void park(float* at, const f32x16_t (&a)[N], int lane) {
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) at[(c * 16 + r) * 64 + lane] = a[c][r];
}
template <int N> __device__ __forceinline__ void unpark(const float* at, f32x16_t (&a)[N], int lane, float mine, float theirs) {
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) a[c][r] = fmaf(at[(c * 16 + r) * 64 + lane], theirs, a[c][r] * mine);
}

// The key tiles (of N keys) that the query rows at positions p0 .. p1 see: [0, a) holds first tokens only, [b, c] the window.
struct Tiles { int a, b, c; };
template <int N> __device__ __forceinline__ Tiles key_tiles(const WaP& p, int p0, int p1, int klen) {
    Tiles t{0, 0, -1};
    if (p1 < p0 || klen <= 0) return t;
    const int jmax = min(p1 + p.right, klen - 1), jmin = max(0, p0 - p.left), ns = min(p.sinks, jmax + 1);
    if (jmax < 0) return t;
    t.a = (ns + N - 1) / N;
    if (jmin <= jmax) t.b = jmin / N, t.c = jmax / N, t.a = min(t.a, t.b);
    else t.b = t.a, t.c = t.a - 1;
    return t;
}

// How many keys the query at pos sees.  A softmax over one key is 1 whatever the score is: such a row has no gradient through
// its weights, which dP - D would give only up to rounding.
__device__ __forceinline__ int seen_keys(const WaP& p, int pos, int klen) {
    const int hi = min(pos + p.right, klen - 1), lo = max(0, pos - p.left);
    return max(0, hi - lo + 1) + max(0, min(min(p.sinks, lo), hi + 1));
}

// Scores of the keys j0 + acc_row(r, 0) that the query at pos does not see -> -inf.  The window is one comparison of the
// distance from its first key; tiles with first tokens add theirs.
__device__ __forceinline__ void hide_keys(const WaP& p, f32x16_t& x, int j0, int pos, int klen) {
    const int lo = pos - p.left, hi = min(pos + p.right, klen - 1);
    const uint32_t at = (uint32_t)(j0 - lo), span = (uint32_t)max(0, hi - lo + 1);
    if (j0 < p.sinks) {
        const int s = min(p.sinks - 1, hi) - j0;
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = at + acc_row(r, 0) < span || acc_row(r, 0) <= s ? x[r] : -INFINITY;
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = at + acc_row(r, 0) < span ? x[r] : -INFINITY;
    }
}

// RG row groups of 32 a workgroup, each by SP waves that take its 32-key tiles in turn and join at the end
template <typename T, int DH, int RG, int SP>
__global__ __launch_bounds__(NTH, sizeof(T) == 2 ? 2 : 1) void wattn_fwd_kernel(const WaP p) {
    typedef Img<T, DH> I;
    typedef typename MM<T>::Frag Frag;
    constexpr int BM = 32 * RG, NX = 1;
    __shared__ __align__(16) T img[2 * BN * I::LD];
    __shared__ float ml[SP > 1 ? RG : 1][2][32];
    static_assert(RG * SP * 64 == NTH && (SP == 1 || (SP == 2 && RG * DH * 128 <= (int)sizeof(img))), "");
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lr = lane & 31, lh = lane >> 5, rg = SP > 1 ? wave % RG : wave, sp = SP > 1 ? wave / RG : 0;
    int id = xcd_order(blockIdx.x, gridDim.x);
    const int g = id % p.G; id /= p.G;
    const int qt = id % p.nt; id /= p.nt;
    const int hk = id % p.Hk, b = id / p.Hk, h = hk * p.G + g;
    const int qlen = p.len ? p.len[b] : INT_MAX, klen = min(p.Tk, qlen);
    const int i = qt * BM + rg * 32 + lr, pos = p.offset + i, pw = p.offset + qt * BM + rg * 32;
    const T* q = (const T*)p.q + b * p.q_sb + (int64_t)min(i, p.Tq - 1) * p.q_st + h * p.q_sh;
    const T* kp = (const T*)p.k + b * p.k_sb + hk * p.k_sh;
    const T* v = (const T*)p.v + b * p.v_sb + hk * p.v_sh;
    Frag qf[DH / 16];
#pragma unroll
    for (int c = 0; c < DH / 16; ++c) qf[c] = MM<T>::ldfrag(q + 16 * c + 8 * lh);
    f32x16_t o[DH / 32];
#pragma unroll
    for (int c = 0; c < DH / 32; ++c) o[c] = zero_acc();
    float m = -INFINITY, l = 0.f;
    const float sc = p.scale * LOG2E;

    const int p0 = p.offset + qt * BM, p1 = min(p.offset + min(qt * BM + BM, p.Tq), qlen) - 1;
    const Tiles tl = key_tiles<BN>(p, p0, p1, klen);
    Stage<T, DH, BN> sk(p.k_st), sv(p.v_st);
    const int count = tl.a + tl.c - tl.b + 1;
    T* ks = img;
    T* vs = img + BN * I::LD;
    auto load = [&](int n) {
        const int r0 = (n < tl.a ? n : tl.b + (n - tl.a)) * BN;
        sk.load(kp, p.k_st, r0, klen);
        sv.load(v, p.v_st, r0, klen);
    };
    if (count > 0) load(0);
    for (int n = 0; n < count; ++n) {
        __syncthreads();
        sk.store(ks);
        sv.store(vs);
        __syncthreads();
        const int j0 = (n < tl.a ? n : tl.b + (n - tl.a)) * BN;
        if (n + 1 < count) load(n + 1);
#pragma unroll
        for (int k = 0; k < BN / 32 / SP; ++k) {
            const int sub = k * SP + sp, ja = j0 + 32 * sub, jb = ja + 31;
            // nothing of this 32 x 32 tile is visible
            if (ja > pw + 31 + p.right || (jb < pw - p.left && ja >= p.sinks) || ja >= klen) continue;
            f32x16_t x[NX];
#pragma unroll
            for (int n = 0; n < NX; ++n) x[n] = zero_acc();
#pragma unroll
            for (int c = 0; c < DH / 16; ++c)
#pragma unroll
                for (int n = 0; n < NX; ++n) MM<T>::mma(nat_frag<T, DH>(ks, 32 * (sub + n) + lr, c, lh), qf[c], x[n]);
            if (!(jb <= pw + p.right && (ja >= pw + 31 - p.left || jb < p.sinks) && jb < klen)) {
#pragma unroll
                for (int n = 0; n < NX; ++n) hide_keys(p, x[n], ja + 32 * n + 4 * lh, pos, klen);
            }
            softmax_tile<DH, NX>(x, m, l, o, sc);
#pragma unroll
            for (int n = 0; n < NX; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const Frag pf = acc_frag<T>(x[n], c);
                    Frag pr;
                    if constexpr (sizeof(T) == 2) pr = rest_frag(x[n], c, pf);
#pragma unroll
                    for (int ct = 0; ct < DH / 32; ++ct) {
                        const Frag vt = tr_frag_of<T, DH>(vs, 32 * (sub + n) + 16 * c, 32 * ct);
                        MM<T>::mma(vt, pf, o[ct]);
                        if constexpr (sizeof(T) == 2) MM<T>::mma(vt, pr, o[ct]);
                    }
                }
        }
    }
    l = both_sum(l);
    if constexpr (SP > 1) {
        float* at = reinterpret_cast<float*>(img) + rg * DH * 32;
        __syncthreads();
        if (sp) {
            park(at, o, lane);
            if (lh == 0) ml[rg][0][lr] = m, ml[rg][1][lr] = l;
        }
        __syncthreads();
        if (sp) return;
        const float m1 = ml[rg][0][lr], mn = fmaxf(m, m1), mu = mn == -INFINITY ? 0.f : mn;
        const float a0 = __builtin_amdgcn_exp2f(m - mu), a1 = __builtin_amdgcn_exp2f(m1 - mu);
        l = fmaf(ml[rg][1][lr], a1, l * a0);
        m = mn;
        unpark(at, o, lane, a0, a1);
    }
    if (i >= p.Tq) return;
    const bool live = pos < qlen && l != 0.f;         // (l is at least 1 where anything is visible; NaN passes)
    const int64_t row = (((int64_t)b * p.Tq + i) * p.Hq + h) * DH;
    if (!live) {
#pragma unroll
        for (int c = 0; c < DH / 32; ++c) o[c] = zero_acc();
    }
    store_rows<T, DH>((T*)p.out + row, o, live ? 1.f / l : 0.f, lh, p.rest ? (T*)p.rest + row : nullptr);
    if (p.lse && lh == 0) {
        // (reference and log of the sum apart: their sum as one float would cost the weights 2^-24 of its size)
        float* s = p.lse + ((int64_t)b * p.Hq + h) * p.Tq + i;
        s[0] = live ? m : INFINITY, s[(int64_t)p.B * p.Hq * p.Tq] = live ? log2f(l) : 0.f;
    }
}

// dq, and D per row for the dk / dv launch behind it.  D = sum(dO O) = sum(P dP).  The first, by the matrix cores as the diagonal of
// O dO^T, costs nothing; bf16 takes O with what its rounding left off, since D cancels against dP, which is not rounded to 8 bits.
// It does not cancel as the second does (two sums in different orders, and O's own errors, which show where one key has nearly all
// the weight: fp32 dq of rows of two or three keys came out 2 to 6 times as far from the exact one as plain arithmetic in 32 bits),
// so workgroups in which a row sees no more than WALK_KEYS keys walk their keys, a few tiles, once more ahead for D = sum(P dP).
constexpr int WALK_KEYS = 32;
template <typename T, int DH, int RG, int SP>
__global__ __launch_bounds__(NTH, SP == 1 && (sizeof(T) == 2 || DH <= 64) ? 2 : 1) void wattn_dq_kernel(const WaP p) {
    typedef Img<T, DH> I;
    typedef typename MM<T>::Frag Frag;
    constexpr int BM = 32 * RG, BN = SP == 1 ? 32 : 64;
    __shared__ __align__(16) T img[2 * BN * I::LD];
    __shared__ float half[SP > 1 ? NTH / 64 : 1][32];
    static_assert(RG * SP * 64 == NTH && (SP == 1 || (SP == 2 && RG * DH * 128 <= (int)sizeof(img))), "");
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lr = lane & 31, lh = lane >> 5, rg = SP > 1 ? wave % RG : wave, sp = SP > 1 ? wave / RG : 0;
    int id = xcd_order(blockIdx.x, gridDim.x);
    const int g = id % p.G; id /= p.G;
    const int qt = id % p.nt; id /= p.nt;
    const int hk = id % p.Hk, b = id / p.Hk, h = hk * p.G + g;
    const int qlen = p.len ? p.len[b] : INT_MAX, klen = min(p.Tk, qlen);
    const int i = qt * BM + rg * 32 + lr, ic = min(i, p.Tq - 1), pos = p.offset + i, pw = p.offset + qt * BM + rg * 32;
    const bool live = i < p.Tq && pos < qlen;
    const T* q = (const T*)p.q + b * p.q_sb + (int64_t)ic * p.q_st + h * p.q_sh;
    const T* go = (const T*)p.dout + b * p.g_sb + (int64_t)ic * p.g_st + h * p.g_sh;
    const int64_t row = (((int64_t)b * p.Tq + ic) * p.Hq + h) * DH;
    const T* kp = (const T*)p.k + b * p.k_sb + hk * p.k_sh;
    const T* v = (const T*)p.v + b * p.v_sb + hk * p.v_sh;
    Frag qf[DH / 16], gf[DH / 16];
#pragma unroll
    for (int c = 0; c < DH / 16; ++c) {
        qf[c] = MM<T>::ldfrag(q + 16 * c + 8 * lh);
        gf[c] = MM<T>::ldfrag(go + 16 * c + 8 * lh);
    }
    const bool walk = __syncthreads_or(live && seen_keys(p, pos, klen) <= WALK_KEYS);
    float dd = 0.f;
    if (!walk) {
        f32x16_t t = zero_acc();
#pragma unroll
        for (int c = 0; c < DH / 16; ++c) {
            MM<T>::mma(MM<T>::ldfrag((const T*)p.o + row + 16 * c + 8 * lh), gf[c], t);
            if constexpr (sizeof(T) == 2) MM<T>::mma(MM<T>::ldfrag((const T*)p.rest + row + 16 * c + 8 * lh), gf[c], t);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) dd += acc_row(r, lh) == lr ? t[r] : 0.f;
        dd = both_sum(dd);
    }
    const int64_t at = ((int64_t)b * p.Hq + h) * p.Tq + ic;
    const float lse = p.lse[at], lsum = p.lse[at + (int64_t)p.B * p.Hq * p.Tq];
    f32x16_t dq[DH / 32];
#pragma unroll
    for (int c = 0; c < DH / 32; ++c) dq[c] = zero_acc();
    const float sc = p.scale * LOG2E;
    const int p0 = p.offset + qt * BM, p1 = min(p.offset + min(qt * BM + BM, p.Tq), qlen) - 1;
    const Tiles tl = key_tiles<BN>(p, p0, p1, klen);
    Stage<T, DH, BN> sk(p.k_st), sv(p.v_st);
    const int count = tl.a + tl.c - tl.b + 1;
    T* ks = img;
    T* vs = img + BN * I::LD;
    auto load = [&](int n) {
        const int r0 = (n < tl.a ? n : tl.b + (n - tl.a)) * BN;
        sk.load(kp, p.k_st, r0, klen);
        sv.load(v, p.v_st, r0, klen);
    };
    // tile n into LDS, the next one on its way; returns its first key
    auto stage = [&](int n, int next) {
        __syncthreads();
        sk.store(ks);
        sv.store(vs);
        __syncthreads();
        if (next < count) load(next);
        return (n < tl.a ? n : tl.b + (n - tl.a)) * BN;
    };
    // any of the 32 keys from js on is visible
    auto seen = [&](int js) { return !(js > pw + 31 + p.right || (js + 31 < pw - p.left && js >= p.sinks) || js >= klen); };
    // adds raw scores (hidden ones -inf) and dP of the staged 32 keys from 32 s on, key js the first
    auto scores = [&](int s, int js, f32x16_t& x, f32x16_t& y) {
#pragma unroll
        for (int c = 0; c < DH / 16; ++c) {
            MM<T>::mma(nat_frag<T, DH>(ks, 32 * s + lr, c, lh), qf[c], x);
            MM<T>::mma(nat_frag<T, DH>(vs, 32 * s + lr, c, lh), gf[c], y);
        }
        const bool full = js + 31 <= pw + p.right && (js >= pw + 31 - p.left || js + 31 < p.sinks) && js + 31 < klen;
        if (!full) hide_keys(p, x, js + 4 * lh, pos, klen);
    };
    if (count > 0) load(0);
    if (walk) {
        for (int n = 0; n < count; ++n) {
            const int j0 = stage(n, n + 1 < count ? n + 1 : 0);             // (and the first tile again for the loop below)
#pragma unroll
            for (int k = 0; k < BN / 32 / SP; ++k) {
                const int s = k * SP + sp;
                if (!seen(j0 + 32 * s)) continue;
                f32x16_t x = zero_acc(), y = zero_acc();
                scores(s, j0 + 32 * s, x, y);
#pragma unroll
                for (int r = 0; r < 16; ++r) dd = fmaf(__builtin_amdgcn_exp2f(fmaf(x[r], sc, -lse) - lsum), y[r], dd);
            }
        }
        dd = both_sum(dd);
        if constexpr (SP > 1) {                                             // both waves' halves
            half[wave][lr] = dd;
            __syncthreads();
            dd = half[rg][lr] + half[(rg + RG) % (NTH / 64)][lr];
        }
    }
    for (int n = 0; n < count; ++n) {
        const int j0 = stage(n, n + 1);
#pragma unroll
        for (int k = 0; k < BN / 32 / SP; ++k) {
            const int s = k * SP + sp;
            if (!seen(j0 + 32 * s)) continue;
            f32x16_t x = zero_acc(), y = zero_acc();
            scores(s, j0 + 32 * s, x, y);
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_exp2f(fmaf(x[r], sc, -lse) - lsum) * (y[r] - dd);
            const Frag pf[2] = {acc_frag<T>(x, 0), acc_frag<T>(x, 1)};
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int ct = 0; ct < DH / 32; ++ct) {
                    const Frag kt = tr_frag_of<T, DH>(ks, 32 * s + 16 * c, 32 * ct);
                    MM<T>::mma(kt, pf[c], dq[ct]);
                    if constexpr (sizeof(T) == 2) MM<T>::mma(kt, rest_frag(x, c, pf[c]), dq[ct]);
                }
        }
    }
    if (live && lh == 0 && sp == 0) p.dd[at] = dd;
    if constexpr (SP > 1) {
        float* mem = reinterpret_cast<float*>(img) + rg * DH * 32;
        __syncthreads();
        if (sp) park(mem, dq, lane);
        __syncthreads();
        if (sp) return;
        unpark(mem, dq, lane, 1.f, 1.f);
    }
    if (i >= p.Tq) return;
    if (!live || seen_keys(p, pos, klen) <= 1) {
#pragma unroll
        for (int c = 0; c < DH / 32; ++c) dq[c] = zero_acc();
    }
    store_rows<T, DH>((T*)p.dq + (((int64_t)b * p.Tq + i) * p.Hq + h) * DH, dq, p.scale, lh);
}

// dk, dv: a workgroup owns 32 KG keys of one key head (32 a wave) and walks the query rows that see them, over the heads of
// its group: no atomics, one order of additions.  SP waves share the same keys and take the 32-row tiles in turn; their
// sums meet in LDS at the end.  First tokens are seen by every later row: the rows from p.edge on are left out of the
// walk of the key tiles that hold them and cut into chunks, each a workgroup of its own (blockIdx.x >= main) whose waves 0
// and 1 take every other 32-row tile against the first tokens' rows; those and the key tiles' own sums go to fp32 partials
// that wattn_sink_sum_kernel adds in order.
template <typename T, int DH, int KG, int SP>
__global__ __launch_bounds__(KG * SP * 64, sizeof(T) == 2 && (DH <= 64 || KG * SP == 8) ? 2 : 1) void wattn_dkv_kernel(const WaP p, int main) {
    typedef Img<T, DH> I;
    typedef typename MM<T>::Frag Frag;
    // V's fragments (and K's) are read from LDS where with both sums, both tiles and the next rows on their way they would
    // exceed the registers of two waves a SIMD (fp32: of one)
    constexpr int KM = 32 * KG, NT = KG * SP * 64;
    constexpr bool VL = DH >= 96, KL = DH == 128 && sizeof(T) == 2 && KG * SP == 8;
    constexpr int TILE = QN * I::LD, OWN = KM * I::LD, N = 2 * TILE + (VL ? OWN : 0) + (KL ? OWN : 0);
    constexpr int PARK = SP > 1 ? KG * DH * 128 / (int)sizeof(T) : 0;
    static_assert(SP <= QN / 32, "a 32-row tile of a staged one for every wave that shares keys");
    __shared__ __align__(16) T mem[N > PARK ? N : PARK];
    __shared__ __align__(16) float st[sizeof(T) == 4 ? 4 : 3][QN];        // per row: reference, D, 1 (0 where one key is seen: no gradient of weights), log of the sum
    T* qs = mem;
    T* gs = mem + TILE;
    T* vimg = mem + 2 * TILE;
    T* kimg = vimg + OWN;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lr = lane & 31, lh = lane >> 5, kg = SP > 1 ? wave % KG : wave, sp = SP > 1 ? wave / KG : 0;
    const bool far = (int)blockIdx.x >= main;
    int id = far ? blockIdx.x - main : xcd_order(blockIdx.x, main);
    const int ns32 = (p.sinks + 31) / 32;
    int kt = 0, ch = 0, kw;                       // key tile; chunk; first key of this wave
    if (far) {
        ch = id % p.nchunk; id /= p.nchunk;
        kw = id % ns32 * 32; id /= ns32;
    } else {
        kt = id % p.nt; id /= p.nt;
        kw = kt * KM + kg * 32;
    }
    const int hk = id % p.Hk, b = id / p.Hk;
    const int qlen = p.len ? p.len[b] : INT_MAX, klen = min(p.Tk, qlen);
    const int qrows = min(p.Tq, qlen < INT_MAX ? max(0, qlen - p.offset) : p.Tq);       // live query rows
    // query rows of this workgroup: [r0, r1)
    int r0, r1;
    if (far) {
        r0 = p.edge + ch * p.chunk;
        r1 = min(r0 + p.chunk, qrows);
    } else {
        r0 = max(0, kt * KM - p.right - p.offset);
        r1 = min(qrows, max(0, kt * KM + KM + p.left - p.offset));
        if (kt * KM < p.sinks) r1 = min(qrows, p.edge);                  // (and no chunks: all rows)
    }
    const int j = kw + lr, jc = min(j, p.Tk - 1);
    const uint32_t span = j >= klen ? 0u : j < p.sinks ? 0x7fffffffu : (uint32_t)(p.left + p.right + 1);
    const T* k = (const T*)p.k + b * p.k_sb + hk * p.k_sh;
    const T* v = (const T*)p.v + b * p.v_sb + hk * p.v_sh;
    Frag kf[KL ? 1 : DH / 16], vf[VL ? 1 : DH / 16];
#pragma unroll
    for (int c = 0; c < DH / 16; ++c) {
        if constexpr (!KL) kf[c] = MM<T>::ldfrag(k + (int64_t)jc * p.k_st + 16 * c + 8 * lh);
        if constexpr (!VL) vf[c] = MM<T>::ldfrag(v + (int64_t)jc * p.v_st + 16 * c + 8 * lh);
    }
    if constexpr (VL) {                           // (rows behind the keys: zeros; seen by the barrier ahead of the first tile)
        for (int e = threadIdx.x; e < KM * I::NP; e += NT) {
            const int r = e / I::NP, pc = e % I::NP, jv = (far ? kw : kt * KM) + r;
            st16<T>(vimg + I::at(r, pc), ld16_pred<T>(v + (int64_t)jv * p.v_st + pc * I::EPP, v, jv < klen));
            if constexpr (KL) st16<T>(kimg + I::at(r, pc), ld16_pred<T>(k + (int64_t)jv * p.k_st + pc * I::EPP, k, jv < klen));
        }
    }
    const int vrow = (far ? 0 : kg * 32) + lr;    // this lane's row there
    f32x16_t dk[DH / 32], dv[DH / 32];
#pragma unroll
    for (int c = 0; c < DH / 32; ++c) dk[c] = zero_acc(), dv[c] = zero_acc();
    const float sc = p.scale * LOG2E;
    Stage<T, DH, QN, NT> sq(p.q_st), sg(p.g_st);
    const int per = r1 > r0 ? (r1 - r0 + QN - 1) / QN : 0, count = per * p.G;
    float sl = 0.f, sd = 0.f, sw = 0.f, ss = 0.f;
    auto load = [&](int n) {
        const int h = hk * p.G + n / per, r = r0 + n % per * QN;
        sq.load((const T*)p.q + b * p.q_sb + h * p.q_sh, p.q_st, r, r1);
        sg.load((const T*)p.dout + b * p.g_sb + h * p.g_sh, p.g_st, r, r1);
        if (threadIdx.x < QN) {
            const int i = r + threadIdx.x;
            const int64_t at = ((int64_t)b * p.Hq + h) * p.Tq + min(i, p.Tq - 1);
            const float lv = p.lse[at], dvv = p.dd[at];
            ss = p.lse[at + (int64_t)p.B * p.Hq * p.Tq];
            sl = i < r1 ? lv : INFINITY;
            sw = i < r1 && seen_keys(p, p.offset + i, klen) > 1 ? 1.f : 0.f;
            sd = sw != 0.f ? dvv : 0.f;
        }
    };
    if (count > 0) load(0);
    for (int n = 0; n < count; ++n) {
        __syncthreads();
        sq.store(qs);
        sg.store(gs);
        if (threadIdx.x < QN) {
            // (bf16: the two as one float; D is formed already, and a weight's own 2^-24 of that is far below its pieces)
            st[0][threadIdx.x] = sizeof(T) == 4 ? sl : sl + ss, st[1][threadIdx.x] = sd, st[2][threadIdx.x] = sw;
            if constexpr (sizeof(T) == 4) st[3][threadIdx.x] = ss;
        }
        __syncthreads();
        const int i0 = r0 + n % per * QN;
        if (n + 1 < count) load(n + 1);
#pragma unroll
        for (int it = 0; it < (SP > 1 ? 1 : QN / 32); ++it) {
            const int s = far ? wave : SP > 1 ? sp : it;                  // far: waves 0 and 1, one tile each
            if (far && (it || wave >= QN / 32)) continue;
            const int pr = p.offset + i0 + 32 * s;                        // position of the tile's first row
            if (kw > pr + 31 + p.right || (kw + 31 < pr - p.left && kw >= p.sinks) || kw >= klen || i0 + 32 * s >= r1) continue;
            int vr = vrow, qr = 32 * s + lr;
            // (the addresses of these fragments are formed anew for every tile: kept in registers they were spilled)
            if constexpr (VL) asm volatile("" : "+v"(vr));
            if constexpr (VL && !KL) asm volatile("" : "+v"(qr));
            f32x16_t x = zero_acc(), y = zero_acc();
#pragma unroll
            for (int c = 0; c < DH / 16; ++c) {
                if constexpr (KL) MM<T>::mma(nat_frag<T, DH>(qs, qr, c, lh), nat_frag<T, DH>(kimg, vr, c, lh), x);
                else MM<T>::mma(nat_frag<T, DH>(qs, qr, c, lh), kf[c], x);
            }
#pragma unroll
            for (int c = 0; c < DH / 16; ++c) {
                if constexpr (VL) MM<T>::mma(nat_frag<T, DH>(gs, qr, c, lh), nat_frag<T, DH>(vimg, vr, c, lh), y);
                else MM<T>::mma(nat_frag<T, DH>(gs, qr, c, lh), vf[c], y);
            }
            const bool full = kw + 31 <= pr + p.right && (kw >= pr + 31 - p.left || kw + 31 < p.sinks) && kw + 31 < klen;
            if (!full) {                          // rows p with j - right <= p <= j + left (a first token: no end), one comparison
                const uint32_t at = (uint32_t)(pr + 4 * lh - (j - p.right));
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = at + acc_row(r, 0) < span ? x[r] : -INFINITY;
            }
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const float4 ls = *reinterpret_cast<const float4*>(&st[0][32 * s + 8 * r4 + 4 * lh]);
                const float4 ds = *reinterpret_cast<const float4*>(&st[1][32 * s + 8 * r4 + 4 * lh]);
                const float4 ws = *reinterpret_cast<const float4*>(&st[2][32 * s + 8 * r4 + 4 * lh]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 4 * r4 + e;
                    x[r] = fmaf(x[r], sc, -(&ls.x)[e]);
                    if constexpr (sizeof(T) == 4) x[r] -= st[3][32 * s + 8 * r4 + 4 * lh + e];
                    x[r] = __builtin_amdgcn_exp2f(x[r]);
                    y[r] = x[r] * fmaf(y[r], (&ws.x)[e], -(&ds.x)[e]);
                }
            }
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const Frag pf = acc_frag<T>(x, c), pr = rest_frag(x, c, pf);
                    const Frag df = acc_frag<T>(y, c), dr = rest_frag(y, c, df);
#pragma unroll
                    for (int ct = 0; ct < DH / 32; ++ct) {
                        const Frag gt = tr_frag_of<T, DH>(gs, 32 * s + 16 * c, 32 * ct);
                        MM<T>::mma(gt, pf, dv[ct]);
                        MM<T>::mma(gt, pr, dv[ct]);
                        const Frag qt = tr_frag_of<T, DH>(qs, 32 * s + 16 * c, 32 * ct);
                        MM<T>::mma(qt, df, dk[ct]);
                        MM<T>::mma(qt, dr, dk[ct]);
                    }
                }
            } else {
                const Frag pf[2] = {acc_frag<T>(x, 0), acc_frag<T>(x, 1)};
                const Frag df[2] = {acc_frag<T>(y, 0), acc_frag<T>(y, 1)};
#pragma unroll
                for (int ct = 0; ct < DH / 32; ++ct)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        MM<T>::mma(tr_frag_of<T, DH>(gs, 32 * s + 16 * c, 32 * ct), pf[c], dv[ct]);
                        MM<T>::mma(tr_frag_of<T, DH>(qs, 32 * s + 16 * c, 32 * ct), df[c], dk[ct]);
                    }
            }
        }
    }
    if (SP > 1 && !far) {
        float* at = reinterpret_cast<float*>(mem) + kg * DH * 32;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            __syncthreads();
            if (sp) park(at, w ? dv : dk, lane);
            __syncthreads();
            if (!sp) unpark(at, w ? dv : dk, lane, 1.f, 1.f);
        }
        if (sp) return;
    }
    if (j >= klen) {                                                      // padding: what was read of it stays out
#pragma unroll
        for (int c = 0; c < DH / 32; ++c) dk[c] = zero_acc(), dv[c] = zero_acc();
    }
    if (p.nchunk > 0 && j < p.sinks && (!far || wave < QN / 32)) {              // first tokens: fp32 partials, summed in order behind
        const int at = far ? 1 + 2 * ch + wave : 0;
        float* d = p.part + ((((int64_t)b * p.Hk + hk) * p.npart + at) * p.sinks + j) * 2 * DH;
        store_rows<float, DH>(d, dk, p.scale, lh);
        store_rows<float, DH>(d + DH, dv, 1.f, lh);
    }
    if (far || j >= p.Tk || (p.nchunk > 0 && j < p.sinks)) return;
    const int64_t row = (((int64_t)b * p.Tk + j) * p.Hk + hk) * DH;
    store_rows<T, DH>((T*)p.dk + row, dk, p.scale, lh);
    store_rows<T, DH>((T*)p.dv + row, dv, 1.f, lh);
}

// first tokens' dk, dv: the partials in one order (four slices of them side by side, then the four sums)
template <typename T>
__global__ __launch_bounds__(NTH) void wattn_sink_sum_kernel(const WaP p, int dh, int64_t n) {
    __shared__ float part[4][64];
    const int e = threadIdx.x & 63, sl = threadIdx.x >> 6;
    const int64_t id = (int64_t)blockIdx.x * 64 + e;
    const int64_t c = id < n ? id : n - 1;
    const int d = (int)(c % (2 * dh));
    const int64_t bj = c / (2 * dh), bh = bj / p.sinks, step = (int64_t)p.sinks * 2 * dh;
    const int j = (int)(bj % p.sinks), per = (p.npart + 3) / 4, k1 = min(p.npart, (sl + 1) * per);
    const float* s = p.part + (bh * p.npart * p.sinks + j) * 2 * dh + d;
    float sum = 0.f;
#pragma unroll 8
    for (int k = sl * per; k < k1; ++k) sum += s[k * step];
    part[sl][e] = sum;
    __syncthreads();
    if (sl || id >= n) return;
    sum = (part[0][e] + part[1][e]) + (part[2][e] + part[3][e]);
    const int64_t row = ((bh / p.Hk * p.Tk + j) * p.Hk + bh % p.Hk) * dh;
    if (d < dh) stf((T*)p.dk + row + d, sum);
    else stf((T*)p.dv + row + d - dh, sum);
}

// ---- one token against a rolling cache -------------------------------------------------------------------------------
struct WsP {
    const void* q; const void* k; const void* v; void* kc; void* vc; void* out;
    const int64_t* pos;
    float* part;                                  // [B][Hk][ngrp][nsplit][32][DH + 2]: o (unnormalised), m, l
    int64_t q_sb, q_sh, k_sb, k_sh, v_sb, v_sh, kc_sb, kc_st, kc_sh, vc_sb, vc_st, vc_sh;
    int B, Hq, Hk, G, ngrp, S, W, nsplit, per;    // per: slots of a split (a multiple of 128)
    float scale;
};

__device__ __forceinline__ int slot_of(int64_t pos, int S, int W) { return pos < S ? (int)pos : S + (int)((pos - S) % W); }

// A workgroup takes one item, one key head (all its query heads at once: the columns of the matrix tile) and one range of
// slots; a wave takes every fourth 32-slot tile of it.  K is read from memory in fragment order; V goes through
// a wave's own LDS image for the transposing read.
template <typename T, int DH>
__global__ __launch_bounds__(NTH, sizeof(T) == 2 ? 2 : 1) void wattn_step_kernel(const WsP p) {
    typedef Img<T, DH> I;
    typedef typename MM<T>::Frag Frag;
    constexpr int NV = (32 * I::NP + 63) / 64;
    __shared__ __align__(16) T vs[4][32 * I::LD];
    __shared__ float ml[4][2][32];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lr = lane & 31, lh = lane >> 5;
    int id = blockIdx.x;
    const int split = id % p.nsplit; id /= p.nsplit;
    const int grp = id % p.ngrp; id /= p.ngrp;
    const int hk = id % p.Hk, b = id / p.Hk;
    const int64_t pos = p.pos[b];
    const int M = p.S + p.W;
    const int valid = pos < 0 ? 0 : pos >= M ? M : (int)pos + 1, cur = pos < 0 ? -1 : slot_of(pos, p.S, p.W);
    const int hg = grp * 32 + lr, h = hk * p.G + min(hg, p.G - 1);
    const T* q = (const T*)p.q + b * p.q_sb + h * p.q_sh;
    const T* kn = (const T*)p.k + b * p.k_sb + hk * p.k_sh;
    const T* vn = (const T*)p.v + b * p.v_sb + hk * p.v_sh;
    T* kc = (T*)p.kc + b * p.kc_sb + hk * p.kc_sh;
    T* vc = (T*)p.vc + b * p.vc_sb + hk * p.vc_sh;
    const int s0 = split * p.per, s1 = min(valid, s0 + p.per);
    if (grp == 0 && cur >= s0 && cur < s0 + p.per && wave == 3 && lane < I::NP) {
        // the new token's rows; every reader of this slot takes them from k, v instead
        st16<T>(kc + (int64_t)cur * p.kc_st + lane * I::EPP, ld16<T>(kn + lane * I::EPP));
        st16<T>(vc + (int64_t)cur * p.vc_st + lane * I::EPP, ld16<T>(vn + lane * I::EPP));
    }
    Frag qf[DH / 16];
#pragma unroll
    for (int c = 0; c < DH / 16; ++c) qf[c] = MM<T>::ldfrag(q + 16 * c + 8 * lh);
    f32x16_t o[DH / 32];
#pragma unroll
    for (int c = 0; c < DH / 32; ++c) o[c] = zero_acc();
    float m = -INFINITY, l = 0.f;
    const float sc = p.scale * LOG2E;
    Frag kf[DH / 16];
    Vec16<T> vv[NV];
    auto load = [&](int js) {
        const int j = js + lr;
        const T* kr = j == cur ? kn : kc + (int64_t)min(j, M - 1) * p.kc_st;
#pragma unroll
        for (int c = 0; c < DH / 16; ++c) kf[c] = MM<T>::ldfrag(kr + 16 * c + 8 * lh);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = lane + 64 * i, r = e / I::NP, jj = js + r, pc = e % I::NP * I::EPP;
            vv[i] = ld16_pred<T>(jj == cur ? vn + pc : vc + (int64_t)jj * p.vc_st + pc, vn, r < 32 && jj < valid);
        }
    };
    int js = s0 + wave * 32;
    if (js < s1) load(js);
    for (; js < s1; js += 128) {
        f32x16_t xs[1] = {zero_acc()};
        f32x16_t& x = xs[0];
#pragma unroll
        for (int c = 0; c < DH / 16; ++c) MM<T>::mma(kf[c], qf[c], x);
        T* img = vs[wave];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = lane + 64 * i;
            if (32 * I::NP % 64 == 0 || e < 32 * I::NP) st16<T>(img + I::at(e / I::NP, e % I::NP), vv[i]);
        }
        if (js + 128 < s1) load(js + 128);
        if (js + 31 >= valid) {
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = js + acc_row(r, lh) < valid ? x[r] : -INFINITY;
        }
        softmax_tile<DH, 1>(xs, m, l, o, sc);
        const Frag pf[2] = {acc_frag<T>(x, 0), acc_frag<T>(x, 1)};
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");          // the image's writes ahead of its reads (one wave)
#pragma unroll
        for (int ct = 0; ct < DH / 32; ++ct)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const Frag vt = tr_frag_of<T, DH>(img, 16 * c, 32 * ct);
                MM<T>::mma(vt, pf[c], o[ct]);
                if constexpr (sizeof(T) == 2) MM<T>::mma(vt, rest_frag(x, c, pf[c]), o[ct]);
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");          // and its reads ahead of the next writes
    }
    l = both_sum(l);
    // the four waves' states into one: weights 2^(m_w - m), channels of a column summed over the waves through LDS
    if (lh == 0) ml[wave][0][lr] = m, ml[wave][1][lr] = l;
    __syncthreads();
    float mt = -INFINITY, lt = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mt = fmaxf(mt, ml[w][0][lr]);
    const float mu = mt == -INFINITY ? 0.f : mt;
#pragma unroll
    for (int w = 0; w < 4; ++w) lt = fmaf(ml[w][1][lr], __builtin_amdgcn_exp2f(ml[w][0][lr] - mu), lt);
    const float wt = __builtin_amdgcn_exp2f(m - mu);
    float* acc = reinterpret_cast<float*>(&vs[0][0]);                    // [G' columns][DH], G' = min(32, heads of this block)
    const int cols = min(32, p.G - grp * 32);
    constexpr int FIT = (int)(sizeof(T) * 4 * 32 * I::LD / (4 * DH));    // columns that fit: at least 32 (4 images of 32 rows)
    static_assert(FIT >= 32, "the image holds one fp32 row per column");
    for (int w = 0; w < 4; ++w) {
        __syncthreads();
        if (wave == w && lr < cols) {
#pragma unroll
            for (int ct = 0; ct < DH / 32; ++ct)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float* d = acc + lr * DH + 32 * ct + acc_row(r, lh);
                    const float add = o[ct][r] * wt;
                    *d = w ? *d + add : add;
                }
        }
    }
    __syncthreads();
    const int64_t bh = (int64_t)b * p.Hk + hk;
    if (wave == 0 && lh == 0) ml[0][0][lr] = mt, ml[0][1][lr] = lt;
    __syncthreads();
    for (int e = threadIdx.x; e < cols * DH; e += NTH) {
        const int c = e / DH, d = e % DH;
        if (p.nsplit == 1) {
            const float lv = ml[0][1][c];
            stf((T*)p.out + ((int64_t)b * p.Hq + hk * p.G + grp * 32 + c) * DH + d, lv != 0.f ? acc[e] / lv : 0.f);
        } else {
            float* w = p.part + (((bh * p.ngrp + grp) * p.nsplit + split) * 32 + c) * (DH + 2);
            w[d] = acc[e];
            if (d < 2) w[DH + d] = ml[0][d][c];
        }
    }
}

// The same in fp32 for at most 4 query heads a key head, by vector arithmetic: an fp32 matrix tile computes 32 columns for 8192
// cycles per 32 keys of 128 channels however few heads there are, this some 1000 per head (one frame of one stream, 256
// slots, 2 heads of 128: 18.6 -> 7.0 us).  A row lies across LP lanes of 16 bytes; every such group of lanes keeps a
// softmax of its own over the rows it reads, and the groups of the eight waves join at the end.
template <int DH, int G>
__global__ __launch_bounds__(512) void wattn_step_few_kernel(const WsP p) {
    constexpr int NW = 8, LP = DH <= 32 ? 8 : DH <= 64 ? 16 : 32, RW = 64 / LP, U = 8, KB = RW * U, NG = NW * RW;
    __shared__ float acc[NG][G][DH];
    __shared__ float ml[NG][G][2];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, sub = lane / LP, d0 = lane % LP * 4;
    const bool in = d0 < DH;
    int id = blockIdx.x;
    const int split = id % p.nsplit; id /= p.nsplit;
    const int hk = id % p.Hk, b = id / p.Hk;
    const int64_t pos = p.pos[b];
    const int M = p.S + p.W, dl = in ? d0 : 0;
    const int valid = pos < 0 ? 0 : pos >= M ? M : (int)pos + 1, cur = pos < 0 ? -1 : slot_of(pos, p.S, p.W);
    const float* kn = (const float*)p.k + b * p.k_sb + hk * p.k_sh + dl;
    const float* vn = (const float*)p.v + b * p.v_sb + hk * p.v_sh + dl;
    float* kc = (float*)p.kc + b * p.kc_sb + hk * p.kc_sh + dl;
    float* vc = (float*)p.vc + b * p.vc_sb + hk * p.vc_sh + dl;
    const int s0 = split * p.per, s1 = min(valid, s0 + p.per);
    if (cur >= s0 && cur < s0 + p.per && wave == 3 && sub == 0 && in) {
        // the new token's rows; every reader of this slot takes them from k, v instead
        *reinterpret_cast<float4*>(kc + (int64_t)cur * p.kc_st) = *reinterpret_cast<const float4*>(kn);
        *reinterpret_cast<float4*>(vc + (int64_t)cur * p.vc_st) = *reinterpret_cast<const float4*>(vn);
    }
    const float sc = p.scale * LOG2E;
    float4 q[G], o[G];
    float m[G], l[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        q[g] = *reinterpret_cast<const float4*>((const float*)p.q + b * p.q_sb + (hk * G + g) * p.q_sh + dl);
        if (!in) q[g] = make_float4(0.f, 0.f, 0.f, 0.f);
        q[g].x *= sc, q[g].y *= sc, q[g].z *= sc, q[g].w *= sc;
        o[g] = make_float4(0.f, 0.f, 0.f, 0.f);
        m[g] = -INFINITY, l[g] = 0.f;
    }
    Vec16<float> nk[U], nv[U];
    auto load = [&](int js) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = js + u * RW + sub;
            nk[u] = ld16_pred<float>(j == cur ? kn : kc + (int64_t)j * p.kc_st, kn, j < s1);
            nv[u] = ld16_pred<float>(j == cur ? vn : vc + (int64_t)j * p.vc_st, vn, j < s1);
        }
    };
    int js = s0 + wave * KB;
    if (js < s1) load(js);
    for (; js < s1; js += NW * KB) {
        Vec16<float> k[U], v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) k[u] = nk[u], v[u] = nv[u];
        if (js + NW * KB < s1) load(js + NW * KB);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float x[U], top = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float4 a = k[u].v;
                x[u] = fmaf(a.w, q[g].w, fmaf(a.z, q[g].z, fmaf(a.y, q[g].y, a.x * q[g].x)));
#pragma unroll
                for (int w = 1; w < LP; w <<= 1) x[u] += __shfl_xor(x[u], w, 64);
                x[u] = js + u * RW + sub < s1 ? x[u] : -INFINITY;
                top = fmaxf(top, x[u]);
            }
            if (__any(top > m[g] + 8.f)) {                              // (see softmax_tile)
                const float mn = fmaxf(m[g], top), al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[g] - mn);
                m[g] = mn, l[g] *= al;
                o[g].x *= al, o[g].y *= al, o[g].z *= al, o[g].w *= al;
            }
            const float mu = m[g] == -INFINITY ? 0.f : m[g];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float e = __builtin_amdgcn_exp2f(x[u] - mu);
                l[g] += e;
                o[g].x = fmaf(e, v[u].v.x, o[g].x), o[g].y = fmaf(e, v[u].v.y, o[g].y);
                o[g].z = fmaf(e, v[u].v.z, o[g].z), o[g].w = fmaf(e, v[u].v.w, o[g].w);
            }
        }
    }
    const int grp = wave * RW + sub;
#pragma unroll
    for (int g = 0; g < G; ++g) {
        if (in) *reinterpret_cast<float4*>(&acc[grp][g][d0]) = o[g];
        if (d0 == 0) ml[grp][g][0] = m[g], ml[grp][g][1] = l[g];
    }
    __syncthreads();
    const int64_t bh = (int64_t)b * p.Hk + hk;
    for (int e = threadIdx.x; e < G * DH; e += NW * 64) {
        const int g = e / DH, d = e % DH;
        float mt = -INFINITY, lt = 0.f, ot = 0.f;
#pragma unroll
        for (int n = 0; n < NG; ++n) mt = fmaxf(mt, ml[n][g][0]);
        const float mu = mt == -INFINITY ? 0.f : mt;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            const float w = __builtin_amdgcn_exp2f(ml[n][g][0] - mu);
            lt = fmaf(ml[n][g][1], w, lt);
            ot = fmaf(acc[n][g][d], w, ot);
        }
        if (p.nsplit == 1) {
            ((float*)p.out)[((int64_t)b * p.Hq + hk * G + g) * DH + d] = lt != 0.f ? ot / lt : 0.f;
        } else {
            float* w = p.part + ((bh * p.nsplit + split) * 32 + g) * (DH + 2);
            w[d] = ot;
            if (d < 2) w[DH + d] = d ? lt : mt;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(NTH) void wattn_step_join_kernel(const WsP p, int dh) {
    const int64_t id = (int64_t)blockIdx.x * NTH + threadIdx.x;
    if (id >= (int64_t)p.B * p.Hq * dh) return;
    const int d = (int)(id % dh), h = (int)(id / dh % p.Hq);
    const int64_t b = id / dh / p.Hq;
    const int hk = h / p.G, g = h % p.G;
    const float* w = p.part + (((b * p.Hk + hk) * p.ngrp + g / 32) * p.nsplit * 32 + g % 32) * (dh + 2);
    const int64_t ss = 32ll * (dh + 2);
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (int s = 0; s < p.nsplit; ++s) m = fmaxf(m, w[s * ss + dh]);
    const float mu = m == -INFINITY ? 0.f : m;
    for (int s = 0; s < p.nsplit; ++s) {
        const float e = __builtin_amdgcn_exp2f(w[s * ss + dh] - mu);
        l = fmaf(w[s * ss + dh + 1], e, l);
        o = fmaf(w[s * ss + d], e, o);
    }
    stf((T*)p.out + id, l != 0.f ? o / l : 0.f);
}

// rows of a whole sequence that its cache holds after position len - 1: the first S and the last W
template <typename T>
__global__ __launch_bounds__(NTH) void wattn_fill_kernel(const WsP p, const int* len, int Tn, int64_t k_st, int64_t v_st, int np, int64_t n) {
    constexpr int EPP = 16 / sizeof(T);
    const int64_t id = (int64_t)blockIdx.x * NTH + threadIdx.x;
    if (id >= n) return;
    const int pc = (int)(id % np) * EPP, M = p.S + p.W;
    int64_t r = id / np;
    const int hk = (int)(r % p.Hk);
    r /= p.Hk;
    const int slot = (int)(r % M), b = (int)(r / M), L = len ? min(max(len[b], 0), Tn) : Tn;
    int64_t t = slot;                             // the last position that lives in this slot
    if (slot >= p.S && L > slot) t = slot + (int64_t)(L - 1 - slot) / p.W * p.W;
    if (t >= L) return;                           // never written: left as it was
    st16<T>((T*)p.kc + b * p.kc_sb + slot * p.kc_st + hk * p.kc_sh + pc, ld16<T>((const T*)p.k + b * p.k_sb + t * k_st + hk * p.k_sh + pc));
    st16<T>((T*)p.vc + b * p.vc_sb + slot * p.vc_st + hk * p.vc_sh + pc, ld16<T>((const T*)p.v + b * p.v_sb + t * v_st + hk * p.v_sh + pc));
}

// ---- host ------------------------------------------------------------------------------------------------------------
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int wa_check(const DttWattn* g, WaP& p, const char* what) {
    DTT_CHECK(g->dtype == 0 || g->dtype == 1, "%s: dtype must be 0 (float32) or 1 (bfloat16)", what);
    DTT_CHECK(g->B > 0 && g->Tq > 0 && g->Tk > 0 && g->Hk > 0 && g->Hq > 0 && g->Hq % g->Hk == 0,
              "%s: bad sizes B=%d Tq=%d Tk=%d Hq=%d Hk=%d (Hq a multiple of Hk)", what, g->B, g->Tq, g->Tk, g->Hq, g->Hk);
    DTT_CHECK(g->DH == 32 || g->DH == 64 || g->DH == 96 || g->DH == 128, "%s: head width %d (32, 64, 96 or 128)", what, g->DH);
    DTT_CHECK(g->left >= 0 && g->right >= 0 && g->offset >= 0 && g->left < (1 << 29) && g->right < (1 << 29) && g->offset < (1 << 29) &&
              g->Tq < (1 << 29) && g->Tk < (1 << 29), "%s: window, offset and lengths must be in [0, 2^29)", what);
    DTT_CHECK(g->sinks >= 0 && g->sinks <= MAX_SINKS, "%s: sinks=%d (0 to %d)", what, g->sinks, MAX_SINKS);
    DTT_CHECK(g->scale > 0.f && g->scale < INFINITY, "%s: scale=%g must be positive", what, g->scale);
    DTT_CHECK(g->q && g->k && g->v, "%s: null buffer", what);
    p = WaP{};
    p.q = g->q; p.k = g->k; p.v = g->v; p.o = g->out; p.out = g->out; p.dout = g->dout; p.dq = g->dq; p.dk = g->dk; p.dv = g->dv;
    p.rest = g->dtype ? g->rest : nullptr; p.lse = g->lse; p.dd = g->dd; p.len = g->lengths;
    // (strides of axes of one element do not count)
    const bool b = g->B > 1, tq = g->Tq > 1, tk = g->Tk > 1, hq = g->Hq > 1, hk = g->Hk > 1;
    p.q_sb = b ? g->q_sb : 0; p.q_st = tq ? g->q_st : g->DH; p.q_sh = hq ? g->q_sh : 0;
    p.k_sb = b ? g->k_sb : 0; p.k_st = tk ? g->k_st : g->DH; p.k_sh = hk ? g->k_sh : 0;
    p.v_sb = b ? g->v_sb : 0; p.v_st = tk ? g->v_st : g->DH; p.v_sh = hk ? g->v_sh : 0;
    p.g_sb = b ? g->g_sb : 0; p.g_st = tq && g->dout ? g->g_st : g->DH; p.g_sh = hq ? g->g_sh : 0;
    const auto row_ok = [&](int64_t st) { return st >= g->DH && st <= (1 << 22); };
    DTT_CHECK(row_ok(p.q_st) && row_ok(p.k_st) && row_ok(p.v_st) && row_ok(p.g_st), "%s: row strides must be DH to 2^22 elements", what);
    DTT_CHECK((p.q_sb | p.q_st | p.q_sh | p.k_sb | p.k_st | p.k_sh | p.v_sb | p.v_st | p.v_sh) % (g->dtype ? 8 : 4) == 0 && aligned16(g->q) &&
              aligned16(g->k) && aligned16(g->v), "%s: rows must start on 16 bytes", what);
    p.B = g->B; p.Tq = g->Tq; p.Tk = g->Tk; p.Hq = g->Hq; p.Hk = g->Hk; p.G = g->Hq / g->Hk;
    p.left = g->left; p.right = g->right; p.sinks = g->sinks < g->Tk ? g->sinks : g->Tk; p.offset = g->offset; p.scale = g->scale;
    return 0;
}

// The rows that see first tokens from beyond the windows of their key tiles, and the chunks they are cut into.  Short ones
// keep the chunks' workgroups below the time of a key tile's.
void far_chunks(WaP& p) {
    const int64_t edge = (int64_t)MAX_SINKS + p.left - p.offset;          // behind the window of every tile with first tokens
    p.edge = p.sinks == 0 || edge >= p.Tq ? p.Tq : edge > 0 ? (int)edge : 0;
    p.chunk = std::max(128, (p.Tq - p.edge + 511) / 512 / 64 * 64 + 64);  // (512 chunks at most, or the partials outgrow the gradients)
    p.nchunk = p.sinks ? (p.Tq - p.edge + p.chunk - 1) / p.chunk : 0;
    p.npart = 1 + 2 * p.nchunk;
}
int64_t part_bytes(const WaP& p, int dh) { return p.nchunk ? (int64_t)p.B * p.Hk * p.npart * p.sinks * 2 * dh * 4 : 0; }

// Few rows: half of them a workgroup, two waves on each (the walk over its keys half as long): fp32 training over 16 clips of
// 376 frames, 2 heads of 128: forward 44 -> 23 us, dq 67 -> 37, dk / dv 77 -> 38; with 1024 workgroups, two to four a CU,
// the other way: 2 x 4096 rows, 16 / 4 heads, bf16: forward 85 -> 98 us, dq 104 -> 198, dk / dv 157 -> 204.  512 workgroups are two a CU.
bool split_rows(const WaP& p) { return (int64_t)p.B * p.Hq * ((p.Tq + 127) / 128) < 512; }
bool split_keys(const WaP& p) { return (int64_t)p.B * p.Hk * ((p.Tk + 127) / 128) < 256; }
// Windows of at most 32 keys: of the rows that a tile of 128 keys walks a wave's 32 keys are seen by few; tiles of 64: dk / dv
// 91 -> 68 us at 8 x 4096 rows, 8 heads of 64, 8 keys, bf16 (fp32, half as many: 132 -> 126).
bool narrow(const WaP& p) { return std::min<int64_t>((int64_t)p.left + p.right + 1 + p.sinks, p.Tk) <= 32; }

#define WA_DH(FN, T)                                                              \
    do {                                                                          \
        if (g->DH == 32) FN(T, 32);                                               \
        else if (g->DH == 64) FN(T, 64);                                          \
        else if (g->DH == 96) FN(T, 96);                                          \
        else FN(T, 128);                                                          \
    } while (0)
#define WA_DISPATCH(FN) do { if (g->dtype) WA_DH(FN, bf16); else WA_DH(FN, float); } while (0)
}  // namespace

extern "C" int dtt_wattn_fwd(const DttWattn* g, void* stream) {
    DTT_CHECK(g, "dtt_wattn_fwd: null argument");
    WaP p;
    if (int rc = wa_check(g, p, "dtt_wattn_fwd")) return rc;
    DTT_CHECK(g->out && aligned16(g->out) && aligned16(p.rest), "dtt_wattn_fwd: null or unaligned output");
    const bool split = split_rows(p);
    const int bm = split ? 64 : 128;
    p.nt = (p.Tq + bm - 1) / bm;
    const int64_t grid = (int64_t)p.B * p.Hq * p.nt;
    DTT_CHECK(grid * NTH < DTT_MAX_THREADS, "dtt_wattn_fwd: too many rows");
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define FWD(T, D)                                                                                                      \
    do {                                                                                                               \
        if (split) hipLaunchKernelGGL((wattn_fwd_kernel<T, D, 2, 2>), dim3((unsigned)grid), dim3(NTH), 0, s, p);       \
        else hipLaunchKernelGGL((wattn_fwd_kernel<T, D, 4, 1>), dim3((unsigned)grid), dim3(NTH), 0, s, p);             \
    } while (0)
    WA_DISPATCH(FWD);
#undef FWD
    DTT_LAUNCH_CHECK();
    return 0;
}

extern "C" int64_t dtt_wattn_bwd_ws_bytes(const DttWattn* g) {
    WaP p;
    if (!g || wa_check(g, p, "dtt_wattn_bwd_ws_bytes")) return 0;
    far_chunks(p);
    return part_bytes(p, g->DH);
}

extern "C" int dtt_wattn_bwd(const DttWattn* g, void* stream) {
    DTT_CHECK(g, "dtt_wattn_bwd: null argument");
    WaP p;
    if (int rc = wa_check(g, p, "dtt_wattn_bwd")) return rc;
    DTT_CHECK(g->out && (p.rest || g->dtype == 0) && g->dout && g->lse && g->dd && g->dq && g->dk && g->dv, "dtt_wattn_bwd: null buffer");
    DTT_CHECK((p.g_sb | p.g_st | p.g_sh) % (g->dtype ? 8 : 4) == 0 && aligned16(g->out) && aligned16(p.rest) && aligned16(g->dout) && aligned16(g->dq) &&
              aligned16(g->dk) && aligned16(g->dv), "dtt_wattn_bwd: rows must start on 16 bytes");
    far_chunks(p);
    const int64_t need = part_bytes(p, g->DH);
    DTT_CHECK(need == 0 || (g->ws && aligned16(g->ws) && g->ws_bytes >= need), "dtt_wattn_bwd: workspace of %lld bytes, %lld given",
              (long long)need, (long long)g->ws_bytes);
    p.part = (float*)g->ws;
    const bool split = split_rows(p), splitk = split_keys(p) || narrow(p);
    const int bm = split ? 64 : 128, km = splitk ? 64 : 128;
    p.nt = (p.Tq + bm - 1) / bm;
    WaP pk = p;
    pk.nt = (p.Tk + km - 1) / km;
    const int64_t gq = (int64_t)p.B * p.Hq * p.nt, gk = (int64_t)p.B * p.Hk * pk.nt;
    const int64_t gf = (int64_t)p.B * p.Hk * p.nchunk * ((p.sinks + 31) / 32), n = (int64_t)p.B * p.Hk * p.sinks * 2 * g->DH;
    DTT_CHECK(gq * NTH < DTT_MAX_THREADS && (gk + gf) * (splitk || g->dtype == 0 ? NTH : 2 * NTH) < DTT_MAX_THREADS && (n + 63) / 64 * NTH < DTT_MAX_THREADS,
              "dtt_wattn_bwd: too many rows");
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const dim3 dq((unsigned)gq), dkv((unsigned)(gk + gf));
#define BWD(T, D)                                                                                                                  \
    do {                                                                                                                           \
        constexpr int SP = sizeof(T) == 2 ? 2 : 1;                                                                                 \
        if (split) hipLaunchKernelGGL((wattn_dq_kernel<T, D, 2, 2>), dq, dim3(NTH), 0, s, p);                                      \
        else hipLaunchKernelGGL((wattn_dq_kernel<T, D, 4, 1>), dq, dim3(NTH), 0, s, p);                                            \
        if (splitk) hipLaunchKernelGGL((wattn_dkv_kernel<T, D, 2, 2>), dkv, dim3(NTH), 0, s, pk, (int)gk);                         \
        else hipLaunchKernelGGL((wattn_dkv_kernel<T, D, 4, SP>), dkv, dim3(NTH * SP), 0, s, pk, (int)gk);                          \
        if (p.nchunk)                                                                                                              \
            hipLaunchKernelGGL((wattn_sink_sum_kernel<T>), dim3((unsigned)((n + 63) / 64)), dim3(NTH), 0, s, p, g->DH, n);   \
    } while (0)
    WA_DISPATCH(BWD);
#undef BWD
    DTT_LAUNCH_CHECK();
    return 0;
}

namespace {
int ws_check(const DttWattnStep* g, WsP& p, const char* what) {
    DTT_CHECK(g->dtype == 0 || g->dtype == 1, "%s: dtype must be 0 (float32) or 1 (bfloat16)", what);
    DTT_CHECK(g->B > 0 && g->Hk > 0 && g->Hq > 0 && g->Hq % g->Hk == 0 && g->S >= 0 && g->W > 0 && (int64_t)g->S + g->W < (1 << 30),
              "%s: bad sizes B=%d Hq=%d Hk=%d sinks=%d window=%d", what, g->B, g->Hq, g->Hk, g->S, g->W);
    DTT_CHECK(g->DH == 32 || g->DH == 64 || g->DH == 96 || g->DH == 128, "%s: head width %d (32, 64, 96 or 128)", what, g->DH);
    DTT_CHECK(g->scale > 0.f && g->scale < INFINITY, "%s: scale=%g must be positive", what, g->scale);
    DTT_CHECK(g->k && g->v && g->kc && g->vc, "%s: null buffer", what);
    p = WsP{};
    p.q = g->q; p.k = g->k; p.v = g->v; p.kc = g->kc; p.vc = g->vc; p.out = g->out; p.pos = g->positions;
    const bool b = g->B > 1, hq = g->Hq > 1, hk = g->Hk > 1, m = g->S + g->W > 1;
    p.q_sb = b ? g->q_sb : 0; p.q_sh = hq ? g->q_sh : 0;
    p.k_sb = b ? g->k_sb : 0; p.k_sh = hk ? g->k_sh : 0; p.v_sb = b ? g->v_sb : 0; p.v_sh = hk ? g->v_sh : 0;
    p.kc_sb = b ? g->kc_sb : 0; p.kc_st = m ? g->kc_st : 0; p.kc_sh = hk ? g->kc_sh : 0;
    p.vc_sb = b ? g->vc_sb : 0; p.vc_st = m ? g->vc_st : 0; p.vc_sh = hk ? g->vc_sh : 0;
    DTT_CHECK((p.q_sb | p.q_sh | p.k_sb | p.k_sh | p.v_sb | p.v_sh | p.kc_sb | p.kc_st | p.kc_sh | p.vc_sb | p.vc_st | p.vc_sh) %
              (g->dtype ? 8 : 4) == 0 && aligned16(g->q) && aligned16(g->k) && aligned16(g->v) && aligned16(g->kc) && aligned16(g->vc),
              "%s: rows must start on 16 bytes", what);
    p.B = g->B; p.Hq = g->Hq; p.Hk = g->Hk; p.G = g->Hq / g->Hk; p.ngrp = (p.G + 31) / 32; p.S = g->S; p.W = g->W; p.scale = g->scale;
    // Splits of the slots, in ranges of 512 at least (four tiles a wave).  One workgroup a CU reads at the full rate: 64 streams over
    // 4016 slots, 16 / 4 heads of 128, 93 us, with four splits 99 + 6.  Up to half as many (item, key head) pairs as CUs are split
    // until that is reached.  Above, the busiest CU decides: it has ceil(rows n / 256) of n parts, and two or three are
    // taken where that is less by a fifth, the join and the shorter ranges costing as much (same heads, us: 132 pairs 78 whole, 85 in two,
    // 63 in three; 160: 80, 89, 70; 192: 83, 93, 91; 264: 158, 132, 116; 384: 175, 154; 416: 180, 184; 512: 204, 203).  The fp32
    // kernel, twice the waves a workgroup, gains from parts of less than 1024 slots only above 256 pairs (2016 slots, heads of 64: 132
    // pairs 42 whole, 45 in three; 264: 90, 75).
    const int M = g->S + g->W;
    const int64_t rows = (int64_t)p.B * p.Hk * p.ngrp, most = (M + 511) / 512;
    int64_t ns = std::min(256 / rows, most);
    if (ns < 2) {
        const auto busiest = [&](int64_t n) { return (rows * n + 255) / 256 * (6 / n); };        // in sixths of a row
        const int64_t least = g->dtype || rows > 256 ? 512 : 1024;
        ns = 1;
        for (int64_t n = 2; n <= 3 && n <= (M + least - 1) / least; ++n)
            if (busiest(n) * 5 <= busiest(1) * 4 && busiest(n) < busiest(ns)) ns = n;
    }
    p.per = (int)(((M + ns - 1) / ns + 127) / 128 * 128);
    p.nsplit = (M + p.per - 1) / p.per;
    return 0;
}
int64_t step_bytes(const WsP& p, int dh) { return p.nsplit > 1 ? (int64_t)p.B * p.Hk * p.ngrp * p.nsplit * 32 * (dh + 2) * 4 : 0; }
}  // namespace

extern "C" int64_t dtt_wattn_step_ws_bytes(const DttWattnStep* g) {
    WsP p;
    if (!g || ws_check(g, p, "dtt_wattn_step_ws_bytes")) return 0;
    return step_bytes(p, g->DH);
}

extern "C" int dtt_wattn_step(const DttWattnStep* g, void* stream) {
    DTT_CHECK(g, "dtt_wattn_step: null argument");
    WsP p;
    if (int rc = ws_check(g, p, "dtt_wattn_step")) return rc;
    DTT_CHECK(g->q && g->out && g->positions, "dtt_wattn_step: null buffer");
    const int64_t need = step_bytes(p, g->DH);
    DTT_CHECK(need == 0 || (g->ws && g->ws_bytes >= need), "dtt_wattn_step: workspace of %lld bytes, %lld given", (long long)need,
              (long long)g->ws_bytes);
    p.part = (float*)g->ws;
    const int64_t grid = (int64_t)p.B * p.Hk * p.ngrp * p.nsplit, n = (int64_t)p.B * p.Hq * g->DH;
    DTT_CHECK(grid * (g->dtype == 0 && p.G <= 4 ? 512 : NTH) < DTT_MAX_THREADS && (p.nsplit == 1 || n + NTH < DTT_MAX_THREADS),
              "dtt_wattn_step: too many rows");
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define STEP(T, D) hipLaunchKernelGGL((wattn_step_kernel<T, D>), dim3((unsigned)grid), dim3(NTH), 0, s, p)
#define FEW1(D, N) hipLaunchKernelGGL((wattn_step_few_kernel<D, N>), dim3((unsigned)grid), dim3(512), 0, s, p)
#define FEW(T, D)                                                                                                   \
    do {                                                                                                            \
        if (p.G == 1) FEW1(D, 1); else if (p.G == 2) FEW1(D, 2); else if (p.G == 3) FEW1(D, 3); else FEW1(D, 4);     \
    } while (0)
    if (g->dtype) WA_DH(STEP, bf16);
    else if (p.G <= 4) WA_DH(FEW, float);
    else WA_DH(STEP, float);
#undef FEW
#undef FEW1
#undef STEP
    if (p.nsplit > 1) {
        const dim3 gj((unsigned)((n + NTH - 1) / NTH));
        if (g->dtype) hipLaunchKernelGGL((wattn_step_join_kernel<bf16>), gj, dim3(NTH), 0, s, p, g->DH);
        else hipLaunchKernelGGL((wattn_step_join_kernel<float>), gj, dim3(NTH), 0, s, p, g->DH);
    }
    DTT_LAUNCH_CHECK();
    return 0;
}

extern "C" int dtt_wattn_cache_fill(const DttWattnStep* g, const int32_t* lengths, int Tn, void* stream) {
    DTT_CHECK(g, "dtt_wattn_cache_fill: null argument");
    WsP p;
    if (int rc = ws_check(g, p, "dtt_wattn_cache_fill")) return rc;
    DTT_CHECK(Tn > 0, "dtt_wattn_cache_fill: T=%d", Tn);
    DTT_CHECK(Tn == 1 || (g->k_st | g->v_st) % (g->dtype ? 8 : 4) == 0, "dtt_wattn_cache_fill: rows must start on 16 bytes");
    const int np = g->DH / (g->dtype ? 8 : 4);
    const int64_t n = (int64_t)p.B * (p.S + p.W) * p.Hk * np, grid = (n + NTH - 1) / NTH;
    DTT_CHECK(grid * NTH < DTT_MAX_THREADS, "dtt_wattn_cache_fill: too many rows");
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (g->dtype) hipLaunchKernelGGL((wattn_fill_kernel<bf16>), dim3((unsigned)grid), dim3(NTH), 0, s, p, lengths, Tn, g->k_st, g->v_st, np, n);
    else hipLaunchKernelGGL((wattn_fill_kernel<float>), dim3((unsigned)grid), dim3(NTH), 0, s, p, lengths, Tn, g->k_st, g->v_st, np, n);
    DTT_LAUNCH_CHECK();
    return 0;
}
