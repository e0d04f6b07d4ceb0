// Drawing a token from a row of logits: temperature, top-k, top-p, min-p, one given uniform number a row.
//
// The mathematics.  z = l / T ranks like l itself, so every filter keeps a PREFIX of one order: value descending, index ascending.
// That order is the ascending order of the 64-bit word  rank = (~monotone(l) << 32) | index  (unique per token), and "what is kept"
// is  rank <= cut  (top-k and top-p) together with  z - z_max >= log(min_p).
// Masses are WHOLE NUMBERS: w_i = round(2^F exp(z_i - z_max)), F = min(50, 62 - ceil(log2 V)), the exponential in double precision;
// what lies 32 or more below the maximum (e^-32 = 1.3e-14) weighs nothing.  Integer sums do not depend on their order: any order of
// atomics gives the same sums, the same cut and the same token, bit for bit; the draw itself not on the split of the row either (what
// top_p is a share of does in long rows, by 6e-12: k_sample_hist).  fp32 sums would not do: over a flat vocabulary of 128 k tokens the
// borders between tokens lie 8e-6 of the whole apart and 6e-8 of rounding moves the answer of one row in a hundred.
// fp64 multiply-adds run at the rate of unpacked fp32 ones on this chip, and the exponential takes a table entry and a short polynomial.
//
// Finding the cut.  A histogram (counts and masses; 512 or 1024 bins over the row's spread, or bins of 1/32 in z) says in which bin the k-th token, or
// p of the mass, lies; only that bin's tokens are ranked among themselves.
//
// Rows up to SMP_ROW_MAX tokens: one workgroup a row, the row in registers, one launch (k_sample_row).  Longer rows: four launches, the row
// spread over many workgroups (k_sample_hist, _zone, _gather, _draw).
#include "common.h"
#include "ecog2txt_hip.h"
#include <math.h>

typedef unsigned long long u64;
#define ST ((hipStream_t)stream)

#define SMP_BINS 2048
#define SMP_TILE 4096               // long rows: tokens of a tile (256 threads x 16)
#define SMP_CHUNK_TILES 12          // tiles of a workgroup of k_sample_hist at most (the packed word's bits)
#define SMP_LIST 8192               // long rows: tokens around the cut that are kept in a list (more: k_sample_draw)

struct SampleArgs {
    const void* logits; long long ldl; int V, frac;            // frac = F
    const float* u;
    float t0, p0, m0; int k0;                                  // settings of all rows ...
    const float* t; const int* k; const float* p; const float* m;   // ... or [B] each
    int* token; float* logprob;
    // bookkeeping of a decoder step (done == NULL: none)
    int l, Lmax, eos, pad; int *done, *out, *next_tok; float* score;
    char* ws; int G, tiles;                                    // long rows: workspace, chunks and tiles of a row
};
struct Settings { float T, P, M; int k; bool use_k, use_p, use_m, greedy; };
// (all loads leave together: where there is no array, the row's u stands in as a readable place)
__device__ __forceinline__ Settings settings_of(const SampleArgs& a, int b) {
    const float t = *(a.t ? a.t + b : a.u + b), p = *(a.p ? a.p + b : a.u + b), m = *(a.m ? a.m + b : a.u + b);
    const int k = *(a.k ? a.k + b : (const int*)a.u + b);
    Settings s;
    s.T = a.t ? t : a.t0; s.P = a.p ? p : a.p0; s.M = a.m ? m : a.m0; s.k = a.k ? k : a.k0;
    s.use_p = s.P < 1.0f; s.use_k = s.k > 0 && s.k < a.V; s.use_m = s.M > 0.0f; s.greedy = !(s.T > 0.0f);
    return s;
}

// ---- logits -------------------------------------------------------------------------------------------------------------------------
// NaN is never drawn, +inf is the largest finite number, -0 ties with +0
__device__ __forceinline__ float clean(float v) { if (!(v == v)) v = -INFINITY; return fminf(v, 3.402823466e+38f) + 0.0f; }
// 16-byte groups of a row: group q holds elements q * E - o .. + E - 1 (E = 4 fp32, 8 bf16; o = the row's offset from a 16-byte boundary).
// Only groups that lie wholly inside the row are loaded whole.
template <bool BF16> struct Row {
    static constexpr int E = BF16 ? 8 : 4;
    const char* row; int V, o;
    __device__ __forceinline__ Row(const SampleArgs& a, int b) {
        row = (const char*)a.logits + (size_t)b * a.ldl * (BF16 ? 2 : 4); V = a.V;
        o = (int)(((uintptr_t)row & 15) / (BF16 ? 2 : 4));
    }
    __device__ __forceinline__ float at(int i) const { return clean(BF16 ? bf2f(((const bf16_t*)row)[i]) : ((const float*)row)[i]); }
    // n groups q0, q0 + step, ... as they lie (-inf outside the row); all loads leave before the first is looked at
    template <int N> __device__ __forceinline__ void load(int q0, int step, uint4 (&w)[N]) const {
        const int first = q0 * E - o, last = (q0 + (N - 1) * step) * E - o;
        if (__all(first >= 0 && last + E <= V)) {
#pragma unroll
            for (int n = 0; n < N; ++n) w[n] = *(const uint4*)(row + (long long)(first + n * step * E) * (BF16 ? 2 : 4));
            return;
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = first + n * step * E;
            unsigned x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (BF16) {
                    const int k = i + 2 * e;
                    const unsigned lo = k >= 0 && k < V ? ((const bf16_t*)row)[k] : 0xFF80u, hi = k + 1 >= 0 && k + 1 < V ? ((const bf16_t*)row)[k + 1] : 0xFF80u;
                    x[e] = lo | (hi << 16);
                } else x[e] = i + e >= 0 && i + e < V ? ((const unsigned*)row)[i + e] : 0xFF800000u;
            }
            w[n] = make_uint4(x[0], x[1], x[2], x[3]);
        }
    }
    static __device__ __forceinline__ void unpack(const uint4& w, float* v) {
        const unsigned x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (BF16) { v[2 * e] = clean(__uint_as_float(x[e] << 16)); v[2 * e + 1] = clean(__uint_as_float(x[e] & 0xFFFF0000u)); }
            else v[e] = clean(__uint_as_float(x[e]));
        }
    }
};
__device__ __forceinline__ unsigned mono(float v) { const unsigned b = __float_as_uint(v); return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u); }
__device__ __forceinline__ float unmono(unsigned o) { return __uint_as_float((o >> 31) ? (o ^ 0x80000000u) : ~o); }
__device__ __forceinline__ u64 rank_of(float v, int i) { return ((u64)(~mono(v)) << 32) | (unsigned)i; }
__device__ __forceinline__ float rank_value(u64 c) { return unmono(~(unsigned)(c >> 32)); }

// ---- reductions over a workgroup of NT threads (red: NT / 64 words of LDS; a call starts with a barrier, unless red is its own) ----
// Within a wave by data-parallel moves (shifts by 1, 2, 4, 8 inside a row of 16 lanes, then the rows' last lanes handed on): six dependent
// steps of a few cycles instead of six trips through LDS.  The whole wave's result is in lane 63.
template <int CTRL, int ROWS> __device__ __forceinline__ u64 dpp_u64(u64 other, u64 v) {       // `other` where there is no source lane
    const unsigned lo = __builtin_amdgcn_update_dpp((unsigned)other, (unsigned)v, CTRL, ROWS, 0xF, false);
    const unsigned hi = __builtin_amdgcn_update_dpp((unsigned)(other >> 32), (unsigned)(v >> 32), CTRL, ROWS, 0xF, false);
    return ((u64)hi << 32) | lo;
}
__device__ __forceinline__ u64 wave_scan(u64 v) {              // inclusive
    v += dpp_u64<0x111, 0xF>(0, v); v += dpp_u64<0x112, 0xF>(0, v); v += dpp_u64<0x114, 0xF>(0, v); v += dpp_u64<0x118, 0xF>(0, v);
    v += dpp_u64<0x142, 0xA>(0, v); v += dpp_u64<0x143, 0xC>(0, v);
    return v;
}
__device__ __forceinline__ u64 wave_min_63(u64 v) {
    u64 x;
    x = dpp_u64<0x111, 0xF>(~0ull, v); v = x < v ? x : v; x = dpp_u64<0x112, 0xF>(~0ull, v); v = x < v ? x : v;
    x = dpp_u64<0x114, 0xF>(~0ull, v); v = x < v ? x : v; x = dpp_u64<0x118, 0xF>(~0ull, v); v = x < v ? x : v;
    x = dpp_u64<0x142, 0xA>(~0ull, v); v = x < v ? x : v; x = dpp_u64<0x143, 0xC>(~0ull, v); v = x < v ? x : v;
    return v;
}
template <int CTRL, int ROWS> __device__ __forceinline__ float dpp_max(float v) {
    return fmaxf(v, __uint_as_float(__builtin_amdgcn_update_dpp(0xFF800000u, __float_as_uint(v), CTRL, ROWS, 0xF, false)));
}
__device__ __forceinline__ float wave_max_63(float v) {
    v = dpp_max<0x111, 0xF>(v); v = dpp_max<0x112, 0xF>(v); v = dpp_max<0x114, 0xF>(v); v = dpp_max<0x118, 0xF>(v);
    v = dpp_max<0x142, 0xA>(v); return dpp_max<0x143, 0xC>(v);
}
__device__ __forceinline__ u64 lane_u64(u64 v, int i) {         // lane i's (i the same in all lanes)
    return ((u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), i) << 32) | (unsigned)__builtin_amdgcn_readlane((int)v, i);
}
template <int NT> __device__ __forceinline__ u64 block_min(u64 v, u64* red) {
    v = wave_min_63(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) v = red[i] < v ? red[i] : v;
    return v;
}
template <int NT, bool OWN = false> __device__ __forceinline__ float block_max(float v, u64* red, float* wave_top = nullptr) {
    v = wave_max_63(v);
    float* r = (float*)red;
    if (!OWN) __syncthreads();
    if ((threadIdx.x & 63) == 63) { r[threadIdx.x >> 6] = v; if (wave_top) wave_top[threadIdx.x >> 6] = v; }
    __syncthreads();
    v = r[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) v = fmaxf(v, r[i]);
    return v;
}
// exclusive prefix over the threads; total = sum of all
template <int NT, bool OWN = false> __device__ __forceinline__ u64 block_scan(u64 v, u64* red, u64& total) {
    const u64 s = wave_scan(v);
    if (!OWN) __syncthreads();
    if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = s;
    __syncthreads();
    u64 before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) { if (i < (int)(threadIdx.x >> 6)) before += red[i]; all += red[i]; }
    total = all;
    return before + s - v;
}
// two of them with one pair of barriers (red: twice as long)
template <int NT, bool OWN = false> __device__ __forceinline__ void block_scan2(u64& v, u64& w, u64* red, u64& total_v, u64& total_w) {
    const u64 s = wave_scan(v), t = wave_scan(w);
    if (!OWN) __syncthreads();
    if ((threadIdx.x & 63) == 63) { red[threadIdx.x >> 6] = s; red[NT / 64 + (threadIdx.x >> 6)] = t; }
    __syncthreads();
    u64 bv = 0, bw = 0, av = 0, aw = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
        const u64 x = red[i], y = red[NT / 64 + i];
        if (i < (int)(threadIdx.x >> 6)) { bv += x; bw += y; }
        av += x; aw += y;
    }
    total_v = av; total_w = aw;
    v = bv + s - v; w = bw + t - w;
}

// ---- weights ------------------------------------------------------------------------------------------------------------------------
// 2^F exp(-at / 64), at >= 0: the nearest whole number's from a table in LDS (made as the product of two short ones; what lies 2048
// or further down weighs nothing), the rest from a polynomial: about 18 instructions a token, and no branch between the tokens of
// a thread, so that their chains interleave.
// exp(-n) and exp(-n / 64), rounded to the nearest: loads that travel with the logits', where exp() itself would take 0.5 us
__device__ const double smp_exp_a[32] = {
    0x1.0000000000000p+0, 0x1.78b56362cef38p-2, 0x1.152aaa3bf81ccp-3, 0x1.97db0ccceb0afp-5, 0x1.2c155b8213cf4p-6, 0x1.b993fe00d5376p-8,
    0x1.44e51f113d4d6p-9, 0x1.de16b9c24a98fp-11, 0x1.5fc21041027adp-12, 0x1.02cf22526545ap-13, 0x1.7cd79b5647c9bp-15, 0x1.18354238f6764p-16,
    0x1.9c54c3b43bc8bp-18, 0x1.2f6053b981d98p-19, 0x1.be6c6fdb01612p-21, 0x1.4875ca227ec38p-22, 0x1.e355bbaee85cbp-24, 0x1.639e3175a689dp-25,
    0x1.05a628c699fa1p-26, 0x1.81056ff2c5772p-28, 0x1.1b48655f37267p-29, 0x1.a0db0d0ddb3ecp-31, 0x1.32b48bf117da2p-32, 0x1.c3527e433fab1p-34,
    0x1.4c1078fe9228ap-35, 0x1.e8a37a45fc32ep-37, 0x1.67852a7007e42p-38, 0x1.0885298767e9ap-39, 0x1.853f01d6d53bap-41, 0x1.1e642baeb84a0p-42,
    0x1.a56e0c2ac7f75p-44, 0x1.36121e24d3bbap-45};
__device__ const double smp_exp_b[64] = {
    0x1.0000000000000p+0, 0x1.f80feabfeefa5p-1, 0x1.f03f56a88b5d8p-1, 0x1.e88dc6afecfc0p-1, 0x1.e0fabfbc702a4p-1, 0x1.d985c89d041a3p-1,
    0x1.d22e6a0197c03p-1, 0x1.caf42e73a4c7ep-1, 0x1.c3d6a24ed8222p-1, 0x1.bcd553b9d7b62p-1, 0x1.b5efd29f24c26p-1, 0x1.af25b0a61a7b5p-1,
    0x1.a876812c0877cp-1, 0x1.a1e1d93d687d0p-1, 0x1.9b674f8f2f3d8p-1, 0x1.95067c78379f2p-1, 0x1.8ebef9eac820bp-1, 0x1.8890636e31f54p-1,
    0x1.827a561889716p-1, 0x1.7c7c70887763cp-1, 0x1.769652df22f7ep-1, 0x1.70c79eba33c07p-1, 0x1.6b0ff72deb89dp-1, 0x1.656f00bf5796ap-1,
    0x1.5fe4615e98e8fp-1, 0x1.5a6fc061433c8p-1, 0x1.5510c67cd2591p-1, 0x1.4fc71dc135627p-1, 0x1.4a9271936fd09p-1, 0x1.45726ea84fb88p-1,
    0x1.4066c2ff39127p-1, 0x1.3b6f1ddd05a92p-1, 0x1.368b2fc6f960ap-1, 0x1.31baaa7dca843p-1, 0x1.2cfd40f8bdcaep-1, 0x1.2852a760d5c59p-1,
    0x1.23ba930c1568bp-1, 0x1.1f34ba78d5666p-1, 0x1.1ac0d5492c0dcp-1, 0x1.165e9c3e67663p-1, 0x1.120dc934993e8p-1, 0x1.0dce171e34e7fp-1,
    0x1.099f41ffbe580p-1, 0x1.058106eb8a6aap-1, 0x1.017323fd90020p-1, 0x1.faeab0ae9381dp-2, 0x1.f30ec8375038bp-2, 0x1.eb5210d6270b7p-2,
    0x1.e3b40ebefcd7ep-2, 0x1.dc3448110daaep-2, 0x1.d4d244cf4ea9ep-2, 0x1.cd8d8ed8ee386p-2, 0x1.c665b1e1f1e0dp-2, 0x1.bf5a3b6bf18b7p-2,
    0x1.b86ababeef8dfp-2, 0x1.b196c0e24d229p-2, 0x1.aadde095dad4bp-2, 0x1.a43fae4b0474ep-2, 0x1.9dbbc01e18268p-2, 0x1.9751adcfa81c1p-2,
    0x1.910110be06976p-2, 0x1.8ac983dedbc65p-2, 0x1.84aaa3b8d514ep-2, 0x1.7ea40e5d6d8fap-2};
struct ExpTab { double e[SMP_BINS + 1]; };
template <int NT> __device__ __forceinline__ void exp_tab_fill(ExpTab& t, int frac) {          // (a barrier before the first use)
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const double b = smp_exp_b[threadIdx.x & 63] * (double)(1ull << frac);
#pragma unroll
    for (int j = 0; j < SMP_BINS / NT; ++j) t.e[j * NT + threadIdx.x] = smp_exp_a[j * (NT / 64) + wave] * b;
    if (threadIdx.x == 0) t.e[SMP_BINS] = 0.0;
}
// 2^37 (exp(f / 32) - 1), 0 <= f < 1, rounded to a whole number, as the low bits of 2^52 + x: f times the polynomial of degree 3 through
// four Chebyshev nodes of [0, 1] (off by at most 0.3)
__device__ __forceinline__ u64 excess37(double f) {
    double p = 5530.091479314363;
    p = __builtin_fma(p, f, 699007.5976518993); p = __builtin_fma(p, f, 67108872.62136903); p = __builtin_fma(p, f, 4294967295.7305384);
    return (u64)__double_as_longlong(__builtin_fma(p, f, 4503599627370496.0)) - 0x4330000000000000ull;
}
// exp(-f / 64), -1/2 <= f <= 1/2: the polynomial of degree 4 through the Chebyshev nodes (off by at most 1.5e-14)
__device__ __forceinline__ double exp64(double f) {
    double p = 2.483533181583589e-09;
    p = __builtin_fma(p, f, -6.357853029268959e-07); p = __builtin_fma(p, f, 0.00012207031249960526); p = __builtin_fma(p, f, -0.015624999999848418);
    return __builtin_fma(p, f, 1.0);
}
struct Weigh {
    const ExpTab* tab; double top, s, scale, amax;             // s = 64 / T; amax: min-p as a bound of at
    __device__ __forceinline__ Weigh(const ExpTab* t, float top_, const Settings& st, int frac) {
        tab = t; top = top_; s = 64.0 / (double)st.T; scale = (double)(1ull << frac);
        amax = st.use_m ? -64.0 * log((double)fminf(st.M, 1.0f)) : INFINITY;
    }
    __device__ __forceinline__ Weigh(const ExpTab* t, double top_, double s_, double amax_, int frac) : tab(t), top(top_), s(s_), scale((double)(1ull << frac)), amax(amax_) {}
    // 64 (z_max - z); SMP_BINS and more: no weight
    __device__ __forceinline__ double at(float v) const { return v == -INFINITY ? 1e300 : (top - (double)v) * s; }
    __device__ __forceinline__ u64 mass(double at) const {
        const double c = fmin(at, (double)SMP_BINS), t = c + 6755399441055744.0;          // (1.5 * 2^52: the low word is the nearest whole number)
        const double f = c - (t - 6755399441055744.0);
        return (u64)__double_as_longlong(__builtin_fma(tab->e[(int)(unsigned)__double_as_longlong(t)], exp64(f), 4503599627370496.0)) - 0x4330000000000000ull;
    }
    // what counts in the draw
    __device__ __forceinline__ u64 kept(float v, int i, u64 cut) const {
        const double x = at(v);
        return x <= amax && rank_of(v, i) <= cut ? mass(x) : 0;
    }
};
// floor(u * all), exact; u outside [0, 1) is moved to its nearest end
__device__ __forceinline__ u64 u_times(float u, u64 all) {
    if (!(u > 0.0f)) u = 0.0f;
    u = fminf(u, 0x1.fffffep-1f);
    const u64 U = (u64)((double)u * 0x1p63);
    return (__umul64hi(all, U) << 1) | ((all * U) >> 63);
}
// p of a mass, as the smallest whole number that a prefix has to reach (at least one token is kept)
__device__ __forceinline__ u64 p_need(float P, u64 mass) {
    const u64 n = (u64)ceil(P > 0.0f ? (double)P * (double)mass : 0.0);
    return n < 1 ? 1 : n;
}
__device__ __forceinline__ void sample_store(const SampleArgs& a, int b, int token, float lp) {
    if (a.done) {
        const int dn = a.done[b], tk = token < 0 ? a.eos : token;      // a row with nothing to draw from ends its sentence
        a.out[(size_t)b * a.Lmax + a.l] = dn ? a.pad : tk;
        a.done[b] = dn | (tk == a.eos);
        if (a.next_tok) a.next_tok[b] = tk;
        if (a.score && !dn) a.score[b] += lp;
    } else {
        a.token[b] = token;
        if (a.logprob) a.logprob[b] = lp;
    }
}
__device__ __forceinline__ float log_prob(const Weigh& w, double at, u64 all) { return (float)(at * (-1.0 / 64.0) - log((double)all / w.scale)); }

// ---- ranking a few tokens among themselves -----------------------------------------------------------------------------------------
// Of the tokens with rank <= hi that `each` enumerates (at most n, each by exactly one thread): the need-th by count (by_mass false; there are
// as many), or the first at which the running mass reaches need -- the last one where the whole does not; `mass_to`: the mass up to
// and with it.  While there are more than 64: a histogram over the eight highest bits in which they differ.  The rest lie in a list, a lane
// each, and every wave ranks them for itself against the lanes' values: no barrier behind the one that completes the list (as one
// list for the workgroup with n^2 comparisons spread over it: 2.2 us a call, most of it barriers and LDS round trips).
// One call each of either kind in a kernel, from one place (inlined twice, the code of a kernel grows by a third, and between other kernels it is
// fetched anew each time); L.n is zero at the first.
struct Found { u64 before, mass; int bin, count; };            // the bin that holds a cut: tokens and mass in front of it, tokens in it
template <int NT> struct SelectLds {
    u64 m[256]; unsigned c[256];
    u64 list[2][64];
    unsigned n[2];
    u64 out[3];
};
template <int NT, class Each> __device__ __forceinline__ u64 select_rank(Each each, u64 hi, int n, u64 need, bool by_mass, const Weigh& w, SelectLds<NT>& L, u64* red,
                                                                        u64& mass_to) {
    u64 lo = 0, before_m = 0, before_c = 0;
    while (__builtin_expect(n > 64, 0)) {
        u64 mn = ~0ull, mx = ~0ull;
        each([&](u64 r) { if (r >= lo && r <= hi) { mn = r < mn ? r : mn; mx = ~r < mx ? ~r : mx; } });
        mn = block_min<NT>(mn, red); mx = ~block_min<NT>(mx, red);
        if (mn > mx) { mass_to = before_m; return ~0ull; }                 // (nothing there)
        const int shift = max(0, 56 - (mn == mx ? 64 : (int)__clzll((long long)(mn ^ mx))));
        for (int i = threadIdx.x; i < 256; i += NT) { L.m[i] = 0; L.c[i] = 0; }
        __syncthreads();
        const u64 first = mn >> shift;
        each([&](u64 r) {
            asm volatile("" : "+v"(r));                    // (else the masses of all of the thread's tokens are worked out in front of the loop, 0.5 us for nothing)
            if (r >= lo && r <= hi) { const int d = (int)((r >> shift) - first); atomicAdd(&L.c[d], 1u); atomicAdd(&L.m[d], w.mass(w.at(rank_value(r)))); }
        });
        __syncthreads();
        const u64 mc = threadIdx.x < 256 ? L.c[threadIdx.x] : 0, mm = threadIdx.x < 256 ? L.m[threadIdx.x] : 0;
        u64 tc, tm, bc = mc, bm = mm;
        block_scan2<NT>(bc, bm, red, tc, tm);
        bc += before_c; bm += before_m;
        const u64 b = by_mass ? bm : bc, x = by_mass ? mm : mc, most = by_mass ? before_m + tm : before_c + tc, nd = need < most ? need : most;
        if (threadIdx.x < 256 && b < nd && b + x >= nd) { L.out[0] = threadIdx.x; L.out[1] = bc; L.out[2] = bm; }
        __syncthreads();
        const u64 d = L.out[0];
        before_c = L.out[1]; before_m = L.out[2];
        const u64 l2 = (first + d) << shift, h2 = l2 + ((1ull << shift) - 1);
        lo = l2 > lo ? l2 : lo; hi = h2 < hi ? h2 : hi;
        n = (int)L.c[d];
        __syncthreads();
    }
    u64* list = L.list[by_mass];
    each([&](u64 r) { if (r >= lo && r <= hi) { const unsigned k = atomicAdd(&L.n[by_mass], 1u); if (k < 64) list[k] = r; } });
    __syncthreads();
    n = __builtin_amdgcn_readfirstlane((int)L.n[by_mass]);
    if (n == 0) { mass_to = before_m; return ~0ull; }
    const int lane = threadIdx.x & 63;
    const u64 r = lane < n ? list[lane] : ~0ull, own = lane < n ? w.mass(w.at(rank_value(r))) : 0;
    u64 m = before_m;
    unsigned c = 0;
    for (int i = 0; i < n; i += 4) {                       // (lanes from n on: rank ~0, mass 0)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const u64 ri = lane_u64(r, i + e), mi = lane_u64(own, i + e);
            c += ri <= r; m += ri <= r ? mi : 0;
        }
    }
    const int last = __ffsll((unsigned long long)__ballot(lane < n && c == (unsigned)n)) - 1;
    const u64 most = lane_u64(m, last), nd = by_mass && need > most ? most : need;
    const u64 x = by_mass ? m : before_c + c, b = by_mass ? x - own : x - 1;
    const u64 hit = __ballot(lane < n && b < nd && x >= nd);
    const int at = hit ? __ffsll(hit) - 1 : last;
    mass_to = lane_u64(m, at);
    return lane_u64(r, at);
}

// ---- one workgroup a row ---------------------------------------------------------------------------------------------------------------
// (The histogram here is of 512 or 1024 bins over the row's spread, counts and masses apart -- masses for top-k alone, too, where the counts would
// do --: two bins a thread or one, no conversions, and up to 8185 tokens the masses stay in registers for the draw: 1806 tokens with all four
// settings in 7.2 us, 256 such rows in 8.5.  It is a chain of dependent steps: load 0.7, maximum 0.3, masses and bins 1.3, each cut 1.5, draw
// and logarithm 1.4.)
template <bool BF16, int NT, int VPT> __global__ __launch_bounds__(NT) void k_sample_row(SampleArgs a) {
    constexpr int E = Row<BF16>::E, NG = VPT / E, NB = VPT <= 8 ? 512 : 1024, PER = NB / NT, NW = NT / 64;
    // masses in registers up to 16 tokens a thread; 32 are worked out again where they are needed (that instance takes all 256 registers as it
    // is, and 44 bytes of scratch a lane)
    constexpr bool HOLD = VPT <= 16;
    __shared__ u64 red[6 * NW];                            // (a place for each reduction)
    __shared__ ExpTab tab;
    __shared__ u64 hist_m[NB];
    __shared__ unsigned hist_c[NB];
    __shared__ SelectLds<NT> L;
    __shared__ Found found[2];
    const int b = blockIdx.x, tid = threadIdx.x;
    const Row<BF16> row(a, b);
    // thread t holds tokens t * VPT - o .. + VPT - 1
    uint4 raw[NG];
    row.load(tid * NG, 1, raw);
    const int i0 = tid * VPT - row.o;
    const Settings st = settings_of(a, b);
    const float u = a.u[b];
    exp_tab_fill<NT>(tab, a.frac);
#pragma unroll
    for (int j = 0; j < PER; ++j) { hist_m[tid + j * NT] = 0; hist_c[tid + j * NT] = 0; }
    if (tid == 0) L.n[0] = L.n[1] = 0;
    float v[VPT];
#pragma unroll
    for (int q = 0; q < NG; ++q) row.unpack(raw[q], v + q * E);
    float top = -INFINITY, low = -INFINITY;                // the largest, and minus the smallest that can be drawn
#pragma unroll
    for (int j = 0; j < VPT; ++j) { top = fmaxf(top, v[j]); low = fmaxf(low, v[j] == -INFINITY ? -INFINITY : -v[j]); }
    top = wave_max_63(top); low = wave_max_63(low);
    float* tops = (float*)red;
    if ((tid & 63) == 63) { tops[2 * (tid >> 6)] = top; tops[2 * (tid >> 6) + 1] = low; }
    __syncthreads();                                       // (publishes the table and the empty histogram, too)
    top = tops[0]; low = tops[1];
#pragma unroll
    for (int i = 1; i < NW; ++i) { top = fmaxf(top, tops[2 * i]); low = fmaxf(low, tops[2 * i + 1]); }
    if (top == -INFINITY) { if (tid == 0) sample_store(a, b, -1, -INFINITY); return; }
    if (st.greedy) {
        u64 best = ~0ull;
#pragma unroll
        for (int j = VPT - 1; j >= 0; --j) if (v[j] == top) best = (u64)(unsigned)(i0 + j);
        best = block_min<NT>(best, red);
        if (tid == 0) sample_store(a, b, (int)best, 0.0f);
        return;
    }
    const Weigh w(&tab, top, st, a.frac);
    u64 tm[HOLD ? VPT : 1];
    auto mass_of = [&](int j) { return HOLD ? tm[HOLD ? j : 0] : w.mass(w.at(v[j])); };
    if (HOLD) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) tm[HOLD ? j : 0] = w.mass(w.at(v[j]));
    }
    float cv = -INFINITY;                                  // kept: logit above cv, or equal and index up to ci
    int ci = 0x7FFFFFFF;
    if (st.use_k || st.use_p) {
        short bin[VPT];
        const double spread = fmin(w.at(-low), (double)SMP_BINS), fine = spread > 0.0 ? 0.999999 * NB / spread : 0.0;      // (a flat row's tokens in few bins: 15 us instead of 7.6)
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const double at = w.at(v[j]);
            const int n = at < (double)SMP_BINS ? (int)(at * fine) : NB;
            bin[j] = (short)n;
            if (n < NB) { atomicAdd(&hist_c[n], 1u); atomicAdd(&hist_m[n], mass_of(j)); }
        }
        __syncthreads();
        u64 c[PER], m[PER], cs = 0, ms = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) { c[j] = hist_c[tid * PER + j]; m[j] = hist_m[tid * PER + j]; cs += c[j]; ms += m[j]; }
        u64 call, mass, cb = cs, mb = ms, cut = ~0ull;
        block_scan2<NT, true>(cb, mb, red + NW, call, mass);
        const bool cut_k = st.use_k && (u64)st.k < call;
#pragma clang loop unroll(disable)
        for (int by_mass = 0; by_mass < 2; ++by_mass) {    // top-k, then top-p of what it leaves
            if (by_mass ? !st.use_p : !cut_k) continue;
            const u64 need = by_mass ? p_need(st.P, mass) : (u64)st.k;       // (at most the mass, or the count: a bin holds it)
            u64 cc = cb, mm = mb;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const u64 b = by_mass ? mm : cc, x = by_mass ? m[j] : c[j];
                if (b < need && b + x >= need) found[by_mass] = {cc, mm, tid * PER + j, (int)c[j]};
                cc += c[j]; mm += m[j];
            }
            __syncthreads();
            const Found f = found[by_mass];
            auto in_bin = [&](auto g) {                    // its tokens, by rank
#pragma unroll
                for (int j = 0; j < VPT; ++j) {
                    if (bin[j] != f.bin) continue;
                    float x = v[j];
                    asm volatile("" : "+v"(x));            // (the few that are there; not all ranks ahead of the loop)
                    g(rank_of(x, i0 + j));
                }
            };
            u64 to;
            cut = select_rank<NT>(in_bin, cut, f.count, need - (by_mass ? f.mass : f.before), by_mass, w, L, red + 3 * NW, to);
            mass = f.mass + to;
        }
        if (cut != ~0ull) { cv = rank_value(cut); ci = (int)(unsigned)cut; }
    }
    // the draw: running sums in the order of the vocabulary
    auto kept = [&](int j) {
        const bool in = v[j] > cv || (v[j] == cv && i0 + j <= ci);
        return in && (!st.use_m || w.at(v[j]) <= w.amax) ? mass_of(j) : 0;
    };
    u64 s = 0;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        asm volatile("" : "+v"(v[j]));                     // (nothing kept from above but logits and masses)
        const u64 m = kept(j);
        if (HOLD) tm[HOLD ? j : 0] = m;
        s += m;
    }
    u64 all;
    u64 before = block_scan<NT, true>(s, red + 5 * NW, all);
    const u64 r = u_times(u, all);
    if (before <= r && r < before + s) {
        int pick = -1; float pv = 0.f;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const u64 m = HOLD ? tm[HOLD ? j : 0] : kept(j);
            if (pick < 0 && r < before + m) { pick = i0 + j; pv = v[j]; }
            before += m;
        }
        sample_store(a, b, pick, log_prob(w, w.at(pv), all));
    }
}

// ---- long rows ----------------------------------------------------------------------------------------------------------------------
// Four launches: k_sample_hist (a pass over the whole row: chunks' histograms, tile maxima), k_sample_zone (which bins hold the cut),
// k_sample_gather (mass above the cut of every tile that reaches it, and a list of the tokens in the cut's bins), k_sample_draw (the cut, the
// tile, the token).  Quarter tiles (1024 tokens) whose maximum lies below the cut are not read again; where the kept tokens lie anywhere in the row,
// 100 of 128003, say, nearly every quarter holds one and the second pass is a whole read, too.
//
// A chunk counts before the row's maximum is known (a pass over the logits less): its bins are whole parts of (l - ref) 32 / T from a
// reference of its own, so they lie across the row's bins floor(32 (z_max - z)).  A token of chunk bin y -- in the row's units -- belongs to
// the row's bin y - 1 or y; entered at y - 1 throughout, the running sums bound the true ones from above, and one bin on from below:
// the cut's bin is one of two.  Where a chunk's bins lie on the row's to 1e-9 of a bin (integer logits, say) and its reference is not the
// row's maximum, the rounding of either side may shift a token on a border by one bin more either way (all of it is below 1e-10 of a bin):
// then the cut's bin is one of four.  The masses themselves are good to 6e-12: bin edge times (count + what the tokens exceed it by).
#define SMP_LBINS 1024
struct ZoneRec {
    u64 best;                 // rank of the row's first token (~0: none)
    u64 whole;                // mass of all tokens
    double top, s, amax;      // the row's Weigh
    float P; int k, greedy;   // and settings
    float v_front, v_zone, v_min;   // as bounds of the logits: in front of b0; not behind b1; what min-p leaves
    int b0, b1;               // bins whose tokens are ranked one by one; in front of b0 everything is kept, behind b1 nothing
    int cut_k, cut_p;         // what is to be found in them
    unsigned n;               // tokens in them
    u64 above, above_c;       // mass and count of the tokens in front of them
};
struct Chunk { double ref, g_top; u64 best; };                 // bin 0 holds tokens with floor((l - ref) 32 / T) = g_top
struct Tile { u64 kept; float top[4]; };                       // mass in front of b0 that min-p leaves; largest logit of each quarter (a wave's)
struct RowWs { u64* hist; Chunk* chunk; Tile* tile; ZoneRec* rec; u64* list; };
static inline __host__ __device__ size_t ws_up(size_t n) { return (n + 15) & ~(size_t)15; }
static inline __host__ __device__ size_t row_ws_bytes(int G, int tiles) {
    return (size_t)G * SMP_LBINS * 8 + ws_up(G * sizeof(Chunk)) + ws_up(tiles * sizeof(Tile)) + ws_up(sizeof(ZoneRec)) + (size_t)SMP_LIST * 8;
}
__device__ __forceinline__ RowWs row_ws(const SampleArgs& a, int b) {
    RowWs r;
    char* p = a.ws + (size_t)b * row_ws_bytes(a.G, a.tiles);
    r.hist = (u64*)p; p += (size_t)a.G * SMP_LBINS * 8;
    r.chunk = (Chunk*)p; p += ws_up(a.G * sizeof(Chunk));
    r.tile = (Tile*)p; p += ws_up(a.tiles * sizeof(Tile));
    r.rec = (ZoneRec*)p; p += ws_up(sizeof(ZoneRec));
    r.list = (u64*)p;
    return r;
}
// the lowest float whose at is below `bound` (or, closed, at most that): from the quotient's float by doubling steps, then halving ones.
// (Two or three steps as a rule; where the border lies near zero, floats are far closer together than `at` resolves.)
__device__ __forceinline__ float lowest_float(const Weigh& w, double bound, bool closed) {
    auto in = [&](unsigned o) { const double x = w.at(unmono(o)); return closed ? x <= bound : x < bound; };
    const unsigned least = mono(-3.402823466e+38f), most = mono((float)w.top);
    if (!in(most)) return INFINITY;                        // (no token at all)
    if (in(least)) return unmono(least);
    unsigned o = mono((float)fmax(w.top - bound / w.s, -3.402823466e+38));
    o = o > most ? most : o;
    unsigned out = least, yes = most, step = 1;            // out does not hold, yes does
    if (in(o)) {
        yes = o;
        while (yes - least > step) { const unsigned n = yes - step; if (!in(n)) { out = n; break; } yes = n; step *= 2; }
    } else {
        out = o;
        while (most - out > step) { const unsigned n = out + step; if (in(n)) { yes = n; break; } out = n; step *= 2; }
    }
    while (yes - out > 1) { const unsigned n = out + (yes - out) / 2; if (in(n)) yes = n; else out = n; }
    return unmono(yes);
}
template <bool BF16> __global__ __launch_bounds__(256) void k_sample_hist(SampleArgs a) {
    constexpr int NT = 256, E = Row<BF16>::E, TG = SMP_TILE / E, NQ = TG / NT;
    __shared__ u64 red[2 * (NT / 64)];
    __shared__ u64 ring[SMP_LBINS];
    const int chunk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const Row<BF16> row(a, b);
    const Settings st = settings_of(a, b);
    const bool bins = !st.greedy && (st.use_k || st.use_p);
    const RowWs ws = row_ws(a, b);
    const int t0 = (int)((long long)chunk * a.tiles / a.G), t1 = (int)((long long)(chunk + 1) * a.tiles / a.G);
    const double sc = 32.0 / (double)st.T;
    double ref = 0.0, g_top = -INFINITY;                   // bin 0 of the ring, at place `head`; lower bins lie in front of it
    int head = 0;
    float bv = -INFINITY; int bi = 0;
    const int place = (tid >> 6) * (TG / 4) + (tid & 63);   // a wave's quarter of the tile, 64 groups at a time
    uint4 raw[NQ];                                         // (the next tile is on its way while one is counted)
    row.load(t0 * TG + place, 64, raw);
    for (int t = t0; t < t1; ++t) {
        float v[NQ * E];
#pragma unroll
        for (int q = 0; q < NQ; ++q) row.unpack(raw[q], v + q * E);
        if (t + 1 < t1) row.load((t + 1) * TG + place, 64, raw);
        float mx = -INFINITY;
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float x = v[q * E + e];
                mx = fmaxf(mx, x);
                if (x > bv) { bv = x; bi = (t * TG + place + q * 64) * E - row.o + e; }     // (a thread's places ascend: the first of equals stays)
            }
        mx = block_max<NT>(mx, red, ws.tile[t].top);
        if (!bins || mx == -INFINITY) continue;
        const double g = floor(((double)mx - ref) * sc);
        if (!(g - g_top < (double)SMP_LBINS)) {             // the first tokens, or all before lie below the window: start anew from here
            ref = (double)mx; g_top = 0.0; head = 0;
            for (int i = tid; i < SMP_LBINS; i += NT) ring[i] = 0;
            __syncthreads();
        } else if (g > g_top) {                            // the window moves up: its new bins start empty
            const int nz = (int)(g - g_top);
            for (int i = tid; i < nz; i += NT) ring[(head + 1 + i) & (SMP_LBINS - 1)] = 0;
            head = (head + nz) & (SMP_LBINS - 1);
            g_top = g;
            __syncthreads();
        }
        // one word a token: 1 << 48 for the count, and 2^37 (exp(rest / 32) - 1) of what it exceeds the bin's edge by (49152 tokens: below 2^48)
#pragma unroll
        for (int j = 0; j < NQ * E; ++j) {
            const double x = ((double)v[j] - ref) * sc, fl = floor(x), rel = g_top - fl;
            if (rel < (double)SMP_LBINS) atomicAdd(&ring[(head - (int)rel) & (SMP_LBINS - 1)], (1ull << 48) + excess37(x - fl));
        }
    }
    const u64 best = block_min<NT>(bv == -INFINITY ? ~0ull : rank_of(bv, bi), red);
    if (tid == 0) { ws.chunk[chunk].best = best; ws.chunk[chunk].ref = ref; ws.chunk[chunk].g_top = g_top; }
    if (bins && best != ~0ull) for (int i = tid; i < SMP_LBINS; i += NT) ws.hist[(size_t)chunk * SMP_LBINS + i] = ring[(head - i) & (SMP_LBINS - 1)];
}

#define SMP_TILES_MAX (E2T_SAMPLE_MAX_V / SMP_TILE + 1)
__global__ __launch_bounds__(512) void k_sample_zone(SampleArgs a) {
    constexpr int NT = 512, PER = SMP_LBINS / NT;
    __shared__ u64 red[3 * (NT / 64)];
    __shared__ ExpTab tab;
    __shared__ u64 zs[4];
    __shared__ double edge[SMP_TILES_MAX];
    __shared__ u64 bin_m[SMP_LBINS], first_m;
    __shared__ unsigned bin_c[SMP_LBINS], first_c;
    __shared__ int shift[SMP_TILES_MAX], wide;
    const int b = blockIdx.x, tid = threadIdx.x;
    const RowWs ws = row_ws(a, b);
    const Chunk mine = ws.chunk[min(tid, a.G - 1)];
    const Settings st = settings_of(a, b);
    ZoneRec& rec = *ws.rec;
    exp_tab_fill<NT>(tab, a.frac);
    if (tid == 0) { wide = 0; zs[0] = zs[1] = ~0ull; first_m = 0; first_c = 0; }
    const u64 best = block_min<NT>(mine.best, red);        // (the last chunk's many times)
    const Weigh w(&tab, rank_value(best), st, a.frac);
    const bool none = best == ~0ull, cuts = !none && !st.greedy && (st.use_k || st.use_p);
    if (tid == 0) {
        rec.best = best; rec.n = 0; rec.above = rec.above_c = 0; rec.whole = 0; rec.cut_k = rec.cut_p = 0; rec.b0 = SMP_LBINS + 1; rec.b1 = SMP_LBINS;
        rec.top = w.top; rec.s = w.s; rec.amax = w.amax; rec.P = st.P; rec.k = st.k; rec.greedy = st.greedy;
    }
    if (tid == 192 && !none && !st.greedy) rec.v_min = w.amax < (double)SMP_BINS ? lowest_float(w, w.amax, true) : lowest_float(w, (double)SMP_BINS, false);
    if (!cuts) {
        if (tid == 64 && !none && !st.greedy) rec.v_front = rec.v_zone = lowest_float(w, (double)SMP_BINS, false);
        return;
    }
    if (tid < a.G) {
        // the chunk's bin 0 lies at d .. of the row's units (>= 0: the row's largest is no smaller than the chunk's)
        const double d = mine.best == ~0ull ? 1e300 : fmax(((double)rank_value(best) - mine.ref) * (32.0 / (double)st.T) - mine.g_top, 0.0), fl = floor(d);
        if (mine.ref != (double)rank_value(best) && fabs(d - rint(d)) < 1e-9 && fl <= (double)SMP_LBINS) wide = 1;
        shift[tid] = fl < (double)SMP_LBINS ? (int)fl : SMP_LBINS;
        const double g = 2.0 * (d - fl), n = rint(g);      // (0, 1 or 2)
        edge[tid] = fl < (double)SMP_LBINS ? exp64(g - n) * smp_exp_b[(int)n] : 0.0;
    }
    __syncthreads();
    // bin x: the chunks' bins that cover the row's bins x and x + 1, and in front the one that covers bin 0 alone
    auto value = [](u64 w) {                               // count + excess of a word
        return __builtin_fma((double)(unsigned)((w >> 32) & 0xFFFFu), 0x1p-5, __builtin_fma((double)(unsigned)w, 0x1p-37, (double)(unsigned)(w >> 48)));
    };
    unsigned cn[PER] = {};
    double ms0[PER] = {};
    constexpr int UN = 8;
    for (int k0 = 0; k0 < a.G; k0 += UN) {                 // (loads of eight chunks together)
        u64 w[UN][PER];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int k = min(k0 + u, a.G - 1);
#pragma unroll
            for (int j = 0; j < PER; ++j) w[u][j] = ws.hist[(size_t)k * SMP_LBINS + min(max(j * NT + tid + 1 - shift[k], 0), SMP_LBINS - 1)];
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int k = min(k0 + u, a.G - 1);
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int x = j * NT + tid, r = x + 1 - shift[k];
                const bool on = k0 + u < a.G && r >= 0 && x + 1 < SMP_LBINS;
                cn[j] += on ? (unsigned)(w[u][j] >> 48) : 0;
                ms0[j] = __builtin_fma(value(w[u][j]), on ? edge[k] : 0.0, ms0[j]);
            }
        }
    }
    if (tid < a.G && shift[tid] == 0) {
        const u64 w = ws.hist[(size_t)tid * SMP_LBINS];
        atomicAdd(&first_c, (unsigned)(w >> 48));
        atomicAdd(&first_m, (u64)(value(w) * edge[tid] * tab.e[0] + 0.5));
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) { bin_c[j * NT + tid] = cn[j]; bin_m[j * NT + tid] = (u64)(ms0[j] * tab.e[2 * (j * NT + tid + 1)] + 0.5); }
    __syncthreads();
    u64 c[PER], m[PER], cs = 0, ms = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        c[j] = bin_c[tid * PER + j]; m[j] = bin_m[tid * PER + j];
        if (tid == 0 && j == 0) { c[j] += first_c; m[j] += first_m; }
        cs += c[j]; ms += m[j];
    }
    u64 call, mall, cb = cs, mb = ms;
    block_scan2<NT, true>(cb, mb, red + NT / 64, call, mall);
    int bk = SMP_LBINS;
    u64 least = mall;                                      // the top-k's mass is at least this
    const bool cut_k = st.use_k && (u64)st.k < call;
    if (cut_k) {
        u64 cc = cb;
#pragma unroll
        for (int j = 0; j < PER; ++j) { if (cc < (u64)st.k && cc + c[j] >= (u64)st.k) zs[0] = (u64)(tid * PER + j); cc += c[j]; }
        __syncthreads();
        bk = (int)zs[0];
        // bins in front of bk (bk - 1) lie in the top-k; their mass is at least what is entered in front of bk - 1 (bk - 3)
        const int sure = bk - (wide ? 3 : 1);
        if (st.use_p && sure >= 0) {
            if (sure / PER == tid) { u64 mm = mb; for (int j = 0; j < PER; ++j) mm += j < sure % PER ? m[j] : 0; zs[2] = mm; }
            __syncthreads();
        }
        least = st.use_p && sure >= 0 ? zs[2] : 0;
    }
    int b0 = bk;
    if (st.use_p) {
        const u64 need = p_need(st.P, least);
        u64 mm = mb;
#pragma unroll
        for (int j = 0; j < PER; ++j) { if (mm < need && mm + m[j] >= need) zs[1] = (u64)(tid * PER + j); mm += m[j]; }
        __syncthreads();
        if (zs[1] != ~0ull) b0 = min(bk, (int)zs[1]);
    }
    const bool found = b0 < SMP_LBINS;                     // (not where top-k keeps every token that weighs something)
    const int b1 = (cut_k ? bk : b0) + 1 + wide;
    b0 = max(b0 - wide, 0);
    if (tid == 64) rec.v_front = lowest_float(w, found ? 2.0 * b0 : (double)SMP_BINS, false);
    if (tid == 128) rec.v_zone = lowest_float(w, found ? 2.0 * (b1 + 1) : (double)SMP_BINS, false);
    if (tid == 0 && found) { rec.whole = mall; rec.b0 = b0; rec.b1 = b1; rec.cut_k = cut_k; rec.cut_p = st.use_p; }
}

template <bool BF16> __global__ __launch_bounds__(256, 6) void k_sample_gather(SampleArgs a) {
    constexpr int NT = 256, E = Row<BF16>::E, TG = SMP_TILE / E, NQ = TG / NT;
    __shared__ u64 red[2 * (NT / 64)];
    __shared__ ExpTab tab;
    __shared__ unsigned base;
    const int t = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const RowWs ws = row_ws(a, b);
    ZoneRec& rec = *ws.rec;
    Tile& tile = ws.tile[t];
    const float mx = fmaxf(fmaxf(tile.top[0], tile.top[1]), fmaxf(tile.top[2], tile.top[3]));
    if (rec.greedy || rec.best == ~0ull) return;
    const Row<BF16> row(a, b);
    const Weigh w(&tab, rec.top, rec.s, rec.amax, a.frac);
    const float v_front = rec.v_front, v_zone = rec.v_zone, v_min = rec.v_min;
    if (!(mx >= v_zone)) { if (tid == 0) tile.kept = 0; return; }
    const int place = (tid >> 6) * (TG / 4) + (tid & 63);
    const bool some = tile.top[tid >> 6] >= v_zone;        // (of this wave's quarter)
    uint4 raw[NQ];
    if (some) row.load(t * TG + place, 64, raw);
    exp_tab_fill<NT>(tab, a.frac);
    __syncthreads();
    u64 s = 0, sk = 0, cnt = 0;                            // cnt: tokens in front of the zone, and 2^32 for each in it
    unsigned in = 0;
    const bool cuts = rec.cut_k || rec.cut_p, mp = rec.amax < INFINITY;
    if (some) {
        float v[NQ * E];
#pragma unroll
        for (int q = 0; q < NQ; ++q) row.unpack(raw[q], v + q * E);
        if (!cuts && !mp) {
#pragma unroll
            for (int j = 0; j < NQ * E; ++j) s += w.mass(w.at(v[j]));
        } else {
#pragma unroll
            for (int j0 = 0; j0 < NQ * E; j0 += 4) {
                bool any = false;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float x = v[j0 + c];
                    const bool front = x >= v_front;
                    if (x >= v_zone && !front) { in |= 1u << (j0 + c); cnt += 1ull << 32; }
                    cnt += front;
                    any |= front;
                }
                if (__any(any)) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float x = v[j0 + c];
                        const u64 m = x >= v_front ? w.mass(w.at(x)) : 0;
                        s += m; sk += x >= v_min ? m : 0;
                    }
                }
            }
        }
    }
    if (!mp) sk = s;
    u64 all, kept, count;
    const u64 before = block_scan<NT>(cnt, red, count);
    if (tid == 0) base = count >> 32 ? atomicAdd(&rec.n, (unsigned)(count >> 32)) : 0;
    block_scan2<NT>(s, sk, red, all, kept);                // (its barriers publish `base`)
    unsigned k = base + (unsigned)(before >> 32);
    for (; in; in &= in - 1, ++k) {
        const int j = __ffs(in) - 1;
        const int i = (t * TG + place + (j / E) * 64) * E - row.o + j % E;
        if (k < SMP_LIST) ws.list[k] = rank_of(row.at(i), i);
    }
    if (tid == 0) {
        tile.kept = kept;
        if (cuts && (unsigned)count) { atomicAdd(&rec.above, all); atomicAdd(&rec.above_c, (u64)(unsigned)count); }
    }
}

// The tokens of the zone once more by finer bins, SMP_SUB over its width, counted and weighed in one go: one of these holds the k-th token
// and one the token that reaches p, and what is left to rank is a handful.
#define SMP_SUB 1024
template <bool BF16> __global__ __launch_bounds__(512) void k_sample_draw(SampleArgs a) {
    constexpr int NT = 512, E = Row<BF16>::E, NG = SMP_TILE / NT / E, PER = SMP_SUB / NT, KEEP = 4;
    __shared__ u64 red[7 * (NT / 64)];                     // (a place for each reduction)
    __shared__ ExpTab tab;
    __shared__ SelectLds<NT> L;
    __shared__ u64 tsum[SMP_TILES_MAX];
    __shared__ u64 sub_m[SMP_SUB];
    __shared__ unsigned sub_c[SMP_SUB];
    __shared__ Found found[2];
    __shared__ u64 zs[2];
    const int b = blockIdx.x, tid = threadIdx.x;
    const RowWs ws = row_ws(a, b);
    const ZoneRec rec = *ws.rec;
    const float u = a.u[b];
    const u64 tile_kept = ws.tile[min(tid, a.tiles - 1)].kept;
    u64 mine[KEEP], mass_of[KEEP] = {};                    // this thread's part of the list (on its way before it is known how long it is)
#pragma unroll
    for (int k = 0; k < KEEP; ++k) mine[k] = ws.list[tid + k * NT];
    if (rec.best == ~0ull) { if (tid == 0) sample_store(a, b, -1, -INFINITY); return; }
    if (rec.greedy) { if (tid == 0) sample_store(a, b, (int)(unsigned)rec.best, 0.0f); return; }
    const bool cuts = rec.cut_k || rec.cut_p, in_list = rec.n <= SMP_LIST;
#pragma unroll
    for (int k = 0; k < KEEP; ++k) if (!cuts || !in_list || tid + k * NT >= (int)rec.n) mine[k] = ~0ull;
    const Row<BF16> row(a, b);
    exp_tab_fill<NT>(tab, a.frac);
    if (tid == 0) L.n[0] = L.n[1] = 0;
    const Weigh w(&tab, rec.top, rec.s, rec.amax, a.frac);
    if (tid < a.tiles) tsum[tid] = tile_kept;
    if (cuts) for (int i = tid; i < SMP_SUB; i += NT) { sub_m[i] = 0; sub_c[i] = 0; }
    if (tid == 0) found[1].bin = -1;
    __syncthreads();
    u64 cut = ~0ull;
    if (cuts) {
        const u64 above = rec.above, above_c = rec.above_c;
        // the tokens of the zone: from the list, or, where they are more than it holds, from the row itself, by this one workgroup in several
        // passes (4 x 131072 normal logits of sd 2: 30 us, so 213).  The zone reaches from the first cut to the last and is a sixteenth of a
        // nat or two wide at least: more than the list are a flat row's tokens, those between a top-p and a far top-k (p 0.5, k 20000), and two
        // bins of a vocabulary of half a million and more (sd 2, T 1.4, p 0.9: 549 us at 524288, 1058 at 1048576; T 1, p 0.95: 58 and 980)
        auto each = [&](auto f) {
            if (in_list) {
#pragma unroll
                for (int k = 0; k < KEEP; ++k) if (mine[k] != ~0ull) f(mine[k]);
                for (int i = KEEP * NT + tid; i < (int)rec.n; i += NT) f(ws.list[i]);
            } else {
                for (int q = tid; q < a.tiles * (SMP_TILE / E); q += NT) {
                    uint4 raw[1];
                    float v[E];
                    row.load(q, 0, raw);
                    row.unpack(raw[0], v);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        if (v[e] >= rec.v_zone && v[e] < rec.v_front) f(rank_of(v[e], q * E - row.o + e));
                    }
                }
            }
        };
        const double fine = 0.5 * SMP_SUB / (double)(rec.b1 + 1 - rec.b0);
        auto sub_of = [&](u64 r) { return min((int)((w.at(rank_value(r)) - 2.0 * rec.b0) * fine), SMP_SUB - 1); };
        int my_sub[KEEP];
#pragma unroll
        for (int k = 0; k < KEEP; ++k) my_sub[k] = mine[k] != ~0ull ? sub_of(mine[k]) : -1;
        auto in_sub = [&](int i) {
            return [&, i](auto f) {
                if (rec.n <= KEEP * NT) {
#pragma unroll
                    for (int k = 0; k < KEEP; ++k) if (my_sub[k] == i) f(mine[k]);
                } else each([&](u64 r) { if (sub_of(r) == i) f(r); });
            };
        };
        auto count_in = [&](int i, u64 m) { atomicAdd(&sub_c[i], 1u); atomicAdd(&sub_m[i], m); };
        if (rec.n <= KEEP * NT) {
#pragma unroll
            for (int k = 0; k < KEEP; ++k) if (my_sub[k] >= 0) { mass_of[k] = w.mass(w.at(rank_value(mine[k]))); count_in(my_sub[k], mass_of[k]); }
        } else each([&](u64 r) { count_in(sub_of(r), w.mass(w.at(rank_value(r)))); });
        __syncthreads();
        u64 c[PER], m[PER], cs = 0, ms = 0, x;
#pragma unroll
        for (int j = 0; j < PER; ++j) { c[j] = sub_c[tid * PER + j]; m[j] = sub_m[tid * PER + j]; cs += c[j]; ms += m[j]; }
        u64 cb = cs, mb = ms, xc;
        block_scan2<NT, true>(cb, mb, red, xc, x);
        cb += above_c; mb += above;
        u64 mass = rec.whole;
        const u64 most = above + x;
#pragma clang loop unroll(disable)
        for (int by_mass = 0; by_mass < 2; ++by_mass) {    // top-k, then top-p of what it leaves
            if (by_mass ? !rec.cut_p : !rec.cut_k) continue;
            const u64 nd = by_mass ? p_need(rec.P, mass) : 0;
            const u64 need = !by_mass ? (u64)rec.k : nd > most ? most : nd > above ? nd : above + 1;
            u64 cc = cb, mm = mb;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const u64 b = by_mass ? mm : cc, y = by_mass ? m[j] : c[j];
                if (b < need && b + y >= need) found[by_mass] = {cc, mm, tid * PER + j, (int)c[j]};
                cc += c[j]; mm += m[j];
            }
            __syncthreads();
            const Found f = found[by_mass];
            if (f.bin < 0) break;                          // (the zone's tokens weigh nothing: no matter which are kept)
            u64 to;
            cut = select_rank<NT>(in_sub(f.bin), cut, f.count, need - (by_mass ? f.mass : f.before), by_mass, w, L, red + 2 * (NT / 64), to);
            mass = f.mass + to;
        }
        auto keep = [&](u64 r, u64 m) { if (r <= cut && w.at(rank_value(r)) <= w.amax) atomicAdd(&tsum[((int)(unsigned)r + row.o) / SMP_TILE], m); };
        if (rec.n <= KEEP * NT) {
#pragma unroll
            for (int k = 0; k < KEEP; ++k) if (my_sub[k] >= 0) keep(mine[k], mass_of[k]);
        } else each([&](u64 r) { keep(r, w.mass(w.at(rank_value(r)))); });
    }
    __syncthreads();
    const u64 s = tid < a.tiles ? tsum[tid] : 0;
    u64 all;
    const u64 before = block_scan<NT, true>(s, red + 5 * (NT / 64), all);
    const u64 r = u_times(u, all);
    if (before <= r && r < before + s) { zs[0] = (u64)tid; zs[1] = before; }
    __syncthreads();
    const int t = (int)zs[0];
    const u64 in_front = zs[1];
    // the tile's tokens, in order: 8 a thread
    uint4 raw[NG];
    float v[NG * E];
    const int q = (t * NT + tid) * NG, i0 = q * E - row.o;
    row.load(q, 1, raw);
    u64 ms = 0;
#pragma unroll
    for (int n = 0; n < NG; ++n) row.unpack(raw[n], v + n * E);
#pragma unroll
    for (int e = 0; e < NG * E; ++e) ms += w.kept(v[e], i0 + e, cut);
    u64 x;
    u64 at = in_front + block_scan<NT, true>(ms, red + 6 * (NT / 64), x);
    if (at <= r && r < at + ms) {
        int pick = -1; float pv = 0.f;
#pragma unroll
        for (int e = 0; e < NG * E; ++e) {
            const u64 m = w.kept(v[e], i0 + e, cut);
            if (pick < 0 && r < at + m) { pick = i0 + e; pv = v[e]; }
            at += m;
        }
        sample_store(a, b, pick, log_prob(w, w.at(pv), all));
    }
}

// ---- entry points -----------------------------------------------------------------------------------------------------------------------
// (a row may start up to seven elements behind a 16-byte boundary.)  Top-k and top-p in one launch / four: 9000 tokens 20.3 / 27 us, 256 such rows 22.5 / 35;
// 15000 20.8 / 28, 24.6 / 37; half as many in one launch 11 to 12
#define SMP_ROW_MAX (16384 - 7)
static int frac_bits(int V) { int c = 0; while ((1ll << c) < V) ++c; return 62 - c < 50 ? 62 - c : 50; }
static int long_tiles(int V) { return (V + 7 + SMP_TILE - 1) / SMP_TILE; }
// chunks of a long row: enough workgroups for the chip (1024 in all) but no more than k_sample_zone merges quickly (16, 8 KB each), at most
// SMP_CHUNK_TILES tiles in one
static int long_chunks(int B, int V) {
    const int tiles = long_tiles(V), least = (tiles + SMP_CHUNK_TILES - 1) / SMP_CHUNK_TILES;
    int want = (1024 + B - 1) / B;
    if (want > 16) want = 16;
    return want < least ? least : want > tiles ? tiles : want;
}
// rows of one launch: in grid.y for long rows, in grid.x (below 2^32 threads) for others; larger batches run in pieces, one behind the other in the
// same workspace
static int rows_a_launch(int B, int V) { const int most = V > SMP_ROW_MAX ? 65535 : 1 << 22; return B < most ? B : most; }
extern "C" size_t e2t_sample_ws_bytes(int B, int V) {
    if (B <= 0 || V <= SMP_ROW_MAX || V > E2T_SAMPLE_MAX_V) return 0;
    const int n = rows_a_launch(B, V);
    return (size_t)n * row_ws_bytes(long_chunks(n, V), long_tiles(V));
}
template <bool BF16> static void sample_go(SampleArgs& a, int B, void* stream) {
    if (a.V <= 2048 - 7) hipLaunchKernelGGL((k_sample_row<BF16, 256, 8>), dim3(B), dim3(256), 0, ST, a);
    else if (a.V <= 8192 - 7) hipLaunchKernelGGL((k_sample_row<BF16, 512, 16>), dim3(B), dim3(512), 0, ST, a);
    else if (a.V <= SMP_ROW_MAX) hipLaunchKernelGGL((k_sample_row<BF16, 512, 32>), dim3(B), dim3(512), 0, ST, a);
    else {
        hipLaunchKernelGGL((k_sample_hist<BF16>), dim3(a.G, B), dim3(256), 0, ST, a);
        hipLaunchKernelGGL(k_sample_zone, dim3(B), dim3(512), 0, ST, a);
        hipLaunchKernelGGL((k_sample_gather<BF16>), dim3(a.tiles, B), dim3(256), 0, ST, a);
        hipLaunchKernelGGL((k_sample_draw<BF16>), dim3(B), dim3(512), 0, ST, a);
    }
}
static int sample_launch(SampleArgs& a, int dtype, int B, const e2t_sample_cfg* cfg, void* ws, size_t ws_bytes, void* stream) {
    E2T_CHECK_ARG(a.logits && a.u && cfg && B > 0 && a.V > 0 && a.V <= E2T_SAMPLE_MAX_V && a.ldl >= a.V);
    E2T_CHECK_ARG(dtype == E2T_DT_F32 || dtype == E2T_DT_BF16);
    E2T_CHECK_ARG(((uintptr_t)a.logits & (dtype == E2T_DT_F32 ? 3 : 1)) == 0);
    const size_t need = e2t_sample_ws_bytes(B, a.V);
    E2T_CHECK_ARG(ws_bytes >= need && (ws || !need) && ((uintptr_t)ws & 15) == 0);
    a.frac = frac_bits(a.V);
    a.t0 = cfg->temperature; a.k0 = cfg->top_k; a.p0 = cfg->top_p; a.m0 = cfg->min_p;
    a.t = cfg->temperature_rows; a.k = cfg->top_k_rows; a.p = cfg->top_p_rows; a.m = cfg->min_p_rows;
    const int n = rows_a_launch(B, a.V);
    a.ws = (char*)ws; a.G = long_chunks(n, a.V); a.tiles = long_tiles(a.V);
    for (long long b0 = 0; b0 < B; b0 += n) {
        SampleArgs s = a;
        auto from = [&](auto*& p, long long step) { if (p) p += b0 * step; };
        s.logits = (const char*)a.logits + (size_t)b0 * a.ldl * (dtype == E2T_DT_BF16 ? 2 : 4);
        from(s.u, 1); from(s.t, 1); from(s.k, 1); from(s.p, 1); from(s.m, 1); from(s.token, 1); from(s.logprob, 1);
        from(s.done, 1); from(s.out, a.Lmax); from(s.next_tok, 1); from(s.score, 1);
        const int rows = (int)(B - b0 < n ? B - b0 : n);
        if (dtype == E2T_DT_BF16) sample_go<true>(s, rows, stream); else sample_go<false>(s, rows, stream);
        E2T_LAUNCH_CHECK();
    }
    return E2T_OK;
}
extern "C" int e2t_sample_rows(const void* logits, int dtype, long long ldl, int B, int V, const float* u, const e2t_sample_cfg* cfg,
                               int32_t* token, float* logprob, void* ws, size_t ws_bytes, void* stream) {
    E2T_CHECK_ARG(token);
    SampleArgs a{};
    a.logits = logits; a.ldl = ldl; a.V = V; a.u = u; a.token = token; a.logprob = logprob;
    return sample_launch(a, dtype, B, cfg, ws, ws_bytes, stream);
}
extern "C" int e2t_sample_step(const void* logits, int dtype, long long ldl, int B, int V, const float* u, const e2t_sample_cfg* cfg, int l,
                               int Lmax, int eos, int pad, int32_t* done, int32_t* out, int32_t* next_tok, float* score, void* ws,
                               size_t ws_bytes, void* stream) {
    E2T_CHECK_ARG(done && out && l >= 0 && l < Lmax);
    SampleArgs a{};
    a.logits = logits; a.ldl = ldl; a.V = V; a.u = u;
    a.l = l; a.Lmax = Lmax; a.eos = eos; a.pad = pad; a.done = done; a.out = out; a.next_tok = next_tok; a.score = score;
    return sample_launch(a, dtype, B, cfg, ws, ws_bytes, stream);
}
