// Drawing a token from a row of logits: temperature, top-k, top-p, min-p, one given uniform number a row.
//
// The mathematics.  z = l / T ranks like l itself, so every filter keeps a PREFIX of one order: value descending, index ascending.
// That order is the ascending order of the 64-bit word  rank = (~monotone(l) << 32) | index  (unique per token), and "what is kept"
// is  rank <= cut  (top-k and top-p) together with  z - z_max >= log(min_p).
// Masses are WHOLE NUMBERS: w_i = round(2^F exp(z_i - z_max)), F = min(50, 62 - ceil(log2 V)), the exponential in double precision.
// Integer sums do not depend on their order: any split of a row over threads, waves or workgroups, and any order of atomics, gives
// the same sums, the same cut and the same token, bit for bit.  (A token below 2^-F of the largest weighs nothing: V of them
// together are below 2^-12 of the resolution of u.)  fp32 sums would not do: over a flat vocabulary of 128 k tokens the borders
// between tokens lie 8e-6 of the whole apart and 6e-8 of rounding moves the answer of one row in a hundred.
#include "common.h"
#include "ecog2txt_hip.h"
#include <math.h>

typedef unsigned long long u64;
#define ST ((hipStream_t)stream)

#define SMP_NT 1024                 // threads of the one-workgroup-per-row kernel
#define SMP_BINS 2048               // level-1 histogram: bins of 1/64 in z below the maximum (window 32: e^-32 = 1.3e-14)
#define SMP_PER_Z 64.0

struct SampleArgs {
    const void* logits; long long ldl; int V, frac;            // frac = F
    const float* u;
    float t0, p0, m0; int k0;                                  // settings of all rows ...
    const float* t; const int* k; const float* p; const float* m;   // ... or [B] each
    int* token; float* logprob;
    u64* list;                                                 // [B][V] ranks of the tokens around the cut (workspace)
    // bookkeeping of a decoder step (done == NULL: none)
    int l, Lmax, eos, pad; int *done, *out, *next_tok; float* score;
};

template <bool BF16> __device__ __forceinline__ float logit_at(const void* row, int i) {
    float v = BF16 ? bf2f(((const bf16_t*)row)[i]) : ((const float*)row)[i];
    if (!(v == v)) v = -INFINITY;                              // NaN: never drawn
    v = fminf(v, 3.402823466e+38f);                            // +inf: the largest finite number
    return v + 0.0f;                                           // (-0 ties with +0)
}
__device__ __forceinline__ unsigned mono(float v) { const unsigned b = __float_as_uint(v); return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u); }
__device__ __forceinline__ float unmono(unsigned o) { return __uint_as_float((o >> 31) ? (o ^ 0x80000000u) : ~o); }
__device__ __forceinline__ u64 rank_of(float v, int i) { return ((u64)(~mono(v)) << 32) | (unsigned)i; }
__device__ __forceinline__ float rank_value(u64 c) { return unmono(~(unsigned)(c >> 32)); }

__device__ __forceinline__ u64 shfl_xor_u64(u64 v, int o) {
    const unsigned lo = __shfl_xor((unsigned)v, o, 64), hi = __shfl_xor((unsigned)(v >> 32), o, 64);
    return ((u64)hi << 32) | lo;
}
__device__ __forceinline__ u64 shfl_up_u64(u64 v, int o) {
    const unsigned lo = __shfl_up((unsigned)v, o, 64), hi = __shfl_up((unsigned)(v >> 32), o, 64);
    return ((u64)hi << 32) | lo;
}
// smallest of all threads' values
template <int NT> __device__ __forceinline__ u64 block_min(u64 v, u64* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { const u64 x = shfl_xor_u64(v, o); v = x < v ? x : v; }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (int i = 1; i < NT / 64; ++i) v = red[i] < v ? red[i] : v;
    return v;
}
// exclusive prefix over the threads; *total = sum of all
template <int NT> __device__ __forceinline__ u64 block_scan(u64 v, u64* red, u64* total) {
    u64 s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const u64 x = shfl_up_u64(s, o); if ((int)(threadIdx.x & 63) >= o) s += x; }
    __syncthreads();
    if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = s;
    __syncthreads();
    u64 before = 0, all = 0;
    for (int i = 0; i < NT / 64; ++i) { if (i < (int)(threadIdx.x >> 6)) before += red[i]; all += red[i]; }
    *total = all;
    return before + s - v;
}

// z - z_max of a value, and its mass
struct Weigh {
    double top, inv_t; double scale;
    __device__ __forceinline__ double x(float v) const { return v == -INFINITY ? -INFINITY : ((double)v - top) * inv_t; }
    __device__ __forceinline__ u64 mass(double x) const { return x < -50.0 ? 0ull : (u64)__builtin_fma(exp(x), scale, 0.5); }   // (spelled out: the same bits at every place that weighs a token)
};

// the rank-th smallest entry of the list by COUNT (need = how many, >= 1), or the smallest entry at which the running MASS reaches
// `need`; ~0 if the whole list does not.  Eight passes of eight bits from the top.
template <int NT> __device__ u64 select_rank(const u64* list, int n, bool by_mass, u64 need, const Weigh& w, u64* hist /*[256]*/, u64* red) {
    u64 prefix = 0, got = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
        __syncthreads();
        if (threadIdx.x < 256) hist[threadIdx.x] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += NT) {
            const u64 c = list[i];
            if (shift < 56 && (c >> (shift + 8)) != (prefix >> (shift + 8))) continue;
            const u64 a = by_mass ? w.mass(w.x(rank_value(c))) : 1ull;
            atomicAdd(&hist[(c >> shift) & 255], a);
        }
        __syncthreads();
        u64 total;
        const u64 mine = threadIdx.x < 256 ? hist[threadIdx.x] : 0ull;
        const u64 before = got + block_scan<NT>(mine, red, &total);
        // the first digit whose running sum reaches `need`
        const bool hit = threadIdx.x < 256 && before < need && before + mine >= need;
        const u64 d = block_min<NT>(hit ? ((u64)threadIdx.x) : ~0ull, red);
        if (d == ~0ull) return ~0ull;
        const u64 b = block_min<NT>(threadIdx.x == d ? before : ~0ull, red);
        prefix |= d << shift;
        got = b;
    }
    return prefix;
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

template <bool BF16> __global__ __launch_bounds__(SMP_NT) void k_sample_row(SampleArgs a) {
    constexpr int NT = SMP_NT;
    __shared__ u64 red[NT / 64];
    __shared__ u64 mass[SMP_BINS];
    __shared__ unsigned cnt[SMP_BINS];
    __shared__ u64 hist[256];
    __shared__ unsigned nlist;
    __shared__ u64 zone_s[4];
    const int b = blockIdx.x, tid = threadIdx.x, V = a.V;
    const char* row = (const char*)a.logits + (size_t)b * a.ldl * (BF16 ? 2 : 4);
    const float T = a.t ? a.t[b] : a.t0;
    const float P = a.p ? a.p[b] : a.p0, Mp = a.m ? a.m[b] : a.m0;
    const int k = a.k ? a.k[b] : a.k0;
    const bool use_p = P < 1.0f, use_k = k > 0 && k < V, use_m = Mp > 0.0f;
    u64 best = ~0ull;
    for (int i = tid; i < V; i += NT) { const u64 c = rank_of(logit_at<BF16>(row, i), i); best = c < best ? c : best; }
    best = block_min<NT>(best, red);
    const float top = rank_value(best);
    if (top == -INFINITY) { if (tid == 0) sample_store(a, b, -1, -INFINITY); return; }
    if (!(T > 0.0f)) { if (tid == 0) sample_store(a, b, (int)(unsigned)best, 0.0f); return; }
    Weigh w;
    w.top = top; w.inv_t = 1.0 / (double)T; w.scale = (double)(1ull << a.frac);
    const double xmin = use_m ? log((double)fminf(Mp, 1.0f)) : -INFINITY;
    u64 cut = ~0ull;
    if (use_k || use_p) {
        for (int i = tid; i < SMP_BINS; i += NT) { mass[i] = 0; cnt[i] = 0; }
        if (tid == 0) { nlist = 0; zone_s[0] = zone_s[1] = ~0ull; }
        __syncthreads();
        for (int i = tid; i < V; i += NT) {
            const double x = w.x(logit_at<BF16>(row, i));
            const double at = -x * SMP_PER_Z;
            if (at < (double)SMP_BINS) { const int q = (int)at; atomicAdd(&cnt[q], 1u); atomicAdd(&mass[q], w.mass(x)); }
        }
        __syncthreads();
        constexpr int PER = SMP_BINS / NT;
        u64 c[PER], m[PER], cs = 0, ms = 0;
        for (int j = 0; j < PER; ++j) { c[j] = cnt[tid * PER + j]; m[j] = mass[tid * PER + j]; cs += c[j]; ms += m[j]; }
        u64 call, mall;
        const u64 cb = block_scan<NT>(cs, red, &call), mb = block_scan<NT>(ms, red, &mall);
        // the bin that holds the k-th token, the mass in front of it and with it
        int bk = SMP_BINS;
        u64 zlo = mall, zhi = mall;
        const bool cut_k = use_k && (u64)k < call;
        if (cut_k) {
            u64 cc = cb, mm = mb;
            for (int j = 0; j < PER; ++j) {
                if (cc < (u64)k && cc + c[j] >= (u64)k) { zone_s[0] = (u64)(tid * PER + j); zone_s[2] = mm; zone_s[3] = mm + m[j]; }
                cc += c[j]; mm += m[j];
            }
            __syncthreads();
            bk = (int)zone_s[0]; zlo = zone_s[2]; zhi = zone_s[3];
        }
        // the first bin in which the running mass can reach p of the whole (whose mass is zlo .. zhi until the k-th token is known)
        int b0 = bk;
        if (use_p) {
            const double need = P > 0.0f ? (double)P * (double)zlo : 0.0;
            u64 nd = (u64)ceil(need); if (nd < 1) nd = 1;
            u64 mm = mb;
            for (int j = 0; j < PER; ++j) { if (mm < nd && mm + m[j] >= nd) zone_s[1] = (u64)(tid * PER + j); mm += m[j]; }
            __syncthreads();
            if (zone_s[1] != ~0ull) b0 = min(bk, (int)zone_s[1]);
        }
        int b1 = cut_k ? bk : b0;
        __syncthreads();
        if (b0 < SMP_BINS) {
            // count and mass in front of the zone
            if (tid * PER <= b0 && b0 < (tid + 1) * PER) {
                u64 cc = cb, mm = mb;
                for (int j = 0; tid * PER + j < b0; ++j) { cc += c[j]; mm += m[j]; }
                zone_s[2] = cc; zone_s[3] = mm;
            }
            u64* list = a.list + (size_t)b * V;
            for (int i = tid; i < V; i += NT) {
                const float v = logit_at<BF16>(row, i);
                const double at = -w.x(v) * SMP_PER_Z;
                if (at < (double)(b1 + 1) && at >= (double)b0) list[atomicAdd(&nlist, 1u)] = rank_of(v, i);
            }
            __threadfence_block();
            __syncthreads();
            const int n = (int)nlist;
            const u64 nabove = zone_s[2], above = zone_s[3];
            u64 whole = mall;
            if (cut_k) {
                cut = select_rank<NT>(list, n, false, (u64)k - nabove, w, hist, red);
                u64 s = 0;
                for (int i = tid; i < n; i += NT) if (list[i] <= cut) s += w.mass(w.x(rank_value(list[i])));
                block_scan<NT>(s, red, &whole);
                whole += above;
            }
            if (use_p) {
                u64 nd = (u64)ceil(P > 0.0f ? (double)P * (double)whole : 0.0); if (nd < 1) nd = 1;
                if (nd > above) { const u64 cp = select_rank<NT>(list, n, true, nd - above, w, hist, red); cut = cp < cut ? cp : cut; }
            }
        }
    }
    // the draw: running sums in the order of the vocabulary
    const int per = (V + NT - 1) / NT;
    const int i0 = min(V, tid * per), i1 = min(V, i0 + per);
    u64 s = 0;
    for (int i = i0; i < i1; ++i) {
        const float v = logit_at<BF16>(row, i);
        const double x = w.x(v);
        if (x >= xmin && rank_of(v, i) <= cut) s += w.mass(x);
    }
    u64 all;
    u64 before = block_scan<NT>(s, red, &all);
    float u = a.u[b];
    if (!(u > 0.0f)) u = 0.0f;
    u = fminf(u, 0x1.fffffep-1f);
    const u64 U = (u64)((double)u * 0x1p63);
    const u64 r = (__umul64hi(all, U) << 1) | ((all * U) >> 63);          // floor(u * all), exact
    if (before <= r && r < before + s) {
        for (int i = i0; i < i1; ++i) {
            const float v = logit_at<BF16>(row, i);
            const double x = w.x(v);
            if (x >= xmin && rank_of(v, i) <= cut) {
                const u64 m = w.mass(x);
                if (r < before + m) { sample_store(a, b, i, (float)(x - log((double)all / w.scale))); break; }
                before += m;
            }
        }
    }
}

static int frac_bits(int V) { int c = 0; while ((1ll << c) < V) ++c; return 62 - c < 50 ? 62 - c : 50; }

extern "C" size_t e2t_sample_ws_bytes(int B, int V) { return B > 0 && V > 0 ? (size_t)B * (size_t)V * sizeof(u64) : 0; }

static int sample_launch(SampleArgs& a, int dtype, int B, const e2t_sample_cfg* cfg, void* ws, size_t ws_bytes, void* stream) {
    E2T_CHECK_ARG(a.logits && a.u && cfg && B > 0 && a.V > 0 && a.V <= E2T_SAMPLE_MAX_V && a.ldl >= a.V);
    E2T_CHECK_ARG(dtype == E2T_DT_F32 || dtype == E2T_DT_BF16);
    E2T_CHECK_ARG(((uintptr_t)a.logits & (dtype == E2T_DT_F32 ? 3 : 1)) == 0);
    E2T_CHECK_ARG(ws_bytes >= e2t_sample_ws_bytes(B, a.V) && (ws || !e2t_sample_ws_bytes(B, a.V)) && ((uintptr_t)ws & 15) == 0);
    a.frac = frac_bits(a.V);
    a.t0 = cfg->temperature; a.k0 = cfg->top_k; a.p0 = cfg->top_p; a.m0 = cfg->min_p;
    a.t = cfg->temperature_rows; a.k = cfg->top_k_rows; a.p = cfg->top_p_rows; a.m = cfg->min_p_rows;
    a.list = (u64*)ws;
    if (dtype == E2T_DT_BF16) hipLaunchKernelGGL((k_sample_row<true>), dim3(B), dim3(SMP_NT), 0, ST, a);
    else hipLaunchKernelGGL((k_sample_row<false>), dim3(B), dim3(SMP_NT), 0, ST, a);
    E2T_LAUNCH_CHECK(); return E2T_OK;
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
