// Products of 8-bit integers with a scale for each row of either operand, and the quantisation that makes such operands.
//
//   y[m][n] = sa[m] * sb[n] * sum_k a[m][k] * b[n][k]  (+ bias[n])
//
// The sum is exact (int32, K <= 131071); it is rounded once to fp32, scaled, biased and rounded to the output type.
#include "common.h"
#include "ecog2txt_hip.h"
#include <atomic>
#include <type_traits>
#include <math.h>

#define ST ((hipStream_t)stream)
typedef int i32x4 __attribute__((ext_vector_type(4)));

// q = round-to-nearest-even(127 x / top), decided exactly: the fp32 quotient where it is clear of a border, else in double
// precision, where 127 x is exact and the quotient's rounding (2^-53) cannot put it ON a border that the true one misses: with
// 24-bit x and top the two are at least 2^-33 apart
__device__ __forceinline__ int quant1(float x, float top, float inv) {
    if (!(x == x)) return 0;                               // NaN
    if (fabsf(x) >= top) return x > 0.f ? 127 : (x < 0.f ? -127 : 0);   // the largest itself, and +-inf; a row of zeros (top = 0)
    const float t = x * inv;
    float r = rintf(t);                                    // (|t - 127 x / top| <= 127 * 2^-23; a subnormal top makes inv infinite: t - r is NaN)
    if (!(fabsf(t - r) <= 0.4995f)) r = (float)rint((double)x * 127.0 / (double)top);
    return (int)r;
}
struct f8 { float v[8]; };
// elements i .. i + 7 of a row of K; zeros behind its end.  vec: the row starts on a 16-byte boundary
template <bool BF16> __device__ __forceinline__ f8 act8(const void* row, int i, int K, int vec) {
    f8 r;
    if (vec && i + 8 <= K) {
        if (BF16) {
            const uint4 w = *(const uint4*)((const bf16_t*)row + i);
            const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) { r.v[2 * e] = __uint_as_float(u[e] << 16); r.v[2 * e + 1] = __uint_as_float(u[e] & 0xFFFF0000u); }
        } else {
            const float4 a = *(const float4*)((const float*)row + i), b = *(const float4*)((const float*)row + i + 4);
            r.v[0] = a.x; r.v[1] = a.y; r.v[2] = a.z; r.v[3] = a.w; r.v[4] = b.x; r.v[5] = b.y; r.v[6] = b.z; r.v[7] = b.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) r.v[e] = i + e < K ? (BF16 ? bf2f(((const bf16_t*)row)[i + e]) : ((const float*)row)[i + e]) : 0.f;
    }
    return r;
}
__device__ __forceinline__ float top8(const f8& x, float top) {
#pragma unroll
    for (int e = 0; e < 8; ++e) { const float v = fabsf(x.v[e]); top = fmaxf(top, v < INFINITY ? v : 0.f); }
    return top;
}
__device__ __forceinline__ uint2 quant8(const f8& x, float top, float inv) {
    unsigned w[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e >> 2] |= (unsigned)(quant1(x.v[e], top, inv) & 255) << (8 * (e & 3));
    return make_uint2(w[0], w[1]);
}

// Rows to 8 bits: T threads a row, NC groups of eight elements a thread in registers between the maximum and the rounding (longer rows
// come from the cache a second time).  Bound by its bytes: fp32 4099 x 4104 from memory in 20.7 us = 4.1 TB/s (a large copy 4.7, a large
// read 4.0).
template <bool BF16, int T, int NC> __global__ __launch_bounds__(256) void k_quant_rows(const void* x, long long ldx, int M, int K, int vec, int8_t* q,
                                                                                       long long ldq, float* scale) {
    __shared__ float red[4];
    const int t = threadIdx.x % T, m = blockIdx.x * (256 / T) + threadIdx.x / T;
    const bool in = m < M;                                 // (T < 256: whole waves share a row)
    const char* row = (const char*)x + (size_t)(in ? m : 0) * ldx * (BF16 ? 2 : 4);
    const int K64 = (K + 63) & ~63;
    f8 v[NC];
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) { const int i = (c * T + t) * 8; if (i < K64) v[c] = act8<BF16>(row, i, K, vec); }
#pragma unroll
    for (int c = 0; c < NC; ++c) { const int i = (c * T + t) * 8; if (i < K64) top = top8(v[c], top); }
    for (int i = (NC * T + t) * 8; i < K64; i += T * 8) top = top8(act8<BF16>(row, i, K, vec), top);
    top = wave_max(top);
    if (T == 256) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
        __syncthreads();
        top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    }
    if (!in) return;
    if (t == 0) scale[m] = top / 127.0f;
    const float inv = 127.0f / top;
    int8_t* qr = q + (size_t)m * ldq;
#pragma unroll
    for (int c = 0; c < NC; ++c) { const int i = (c * T + t) * 8; if (i < K64) *(uint2*)(qr + i) = quant8(v[c], top, inv); }
    for (int i = (NC * T + t) * 8; i < K64; i += T * 8) *(uint2*)(qr + i) = quant8(act8<BF16>(row, i, K, vec), top, inv);
}

// ---- the store: y = fl32(sum) * sa * sb + bias, ReLU, output type ------------------------------------------------------------------
struct I8Args {
    const int8_t* A; const int8_t* B; const float* sa; const float* sb; const float* bias; void* C;
    long long lda, ldb, ldc;
    int M, N, S;                  // S: 64-byte k-blocks
    int relu, out_bf16, vec;      // vec: every row of the output starts on a boundary of 16, 8 or 4 bytes (0: of less)
    int full;                     // tiles of the launch that are whole; the workgroups behind them own quarters of one (k_gemm_i8_tile)
    const void* x; long long ldx; int K, xvec, xbf16;     // activations to quantise in the kernel (fused form)
};
__device__ __forceinline__ float i8_scale(int acc, float sa, float sb, float bias, int relu) {
    float y = (float)acc * sa * sb + bias;
    return relu && y < 0.f ? 0.f : y;                      // (fmaxf would turn a NaN of a scale or bias into 0)
}
// ---- tiled product -----------------------------------------------------------------------------------------------------------------
// BM x BN tile, WM x WN waves, v_mfma_i32_16x16x64_i8 (16 B of k a lane: operands lie in memory as the instruction wants them).
// One LDS stage = one 64-byte k-block of the tile's A and B rows, four stages, filled by direct-to-LDS DMA (16 B a lane, 1 KiB = 16 rows
// an instruction).  The fragments of block s + 1 are read, and the DMA of block s + 4 is issued, BETWEEN the MFMA rows of block s,
// whose own fragments already lie in registers: one barrier a block, three blocks in flight.
// LDS image: rows of 64 B, chunk c of row r at chunk position c ^ f(r), f(r) = (r >> 1 & 3) ^ (r >> 3 & 1): any 8 rows of a read hit eight
// different 16-B slots of 128 B and any 16 rows sixteen of 256 B (the DMA writes linearly, so f is applied to the source chunk).
// Rows beyond M / N are clamped to the last one; what they give is never stored.
extern __shared__ __attribute__((aligned(16))) char i8_smem[];
__device__ __forceinline__ int i8_swz(int r) { return ((r >> 1) & 3) ^ ((r >> 3) & 1); }

// tile (m0, n0) of BM x BN by KS groups of WM x WN waves, each group with an equal share of the k-blocks and stages of its own: where a
// product has few tiles, a CU's one workgroup is bound by the latency of a step (64 x 64: 0.21 us), and KS steps run side by side
template <int BM, int BN, int WM, int WN, int NS, int KS>
__device__ __forceinline__ void i8_tile(const I8Args& p, int m0, int n0) {
    constexpr int NW = WM * WN, NT = 64 * NW * KS, STAGE = (BM + BN) * 64, RING = NS * STAGE;
    constexpr int TI = BM / WM / 16, TJ = BN / WN / 16, PIECES = (BM + BN) / 16, NP = PIECES / NW;
    static_assert(PIECES % NW == 0 && TI >= 1 && TJ >= 1, "tile");
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int grp = KS > 1 ? wv / NW : 0, wave = KS > 1 ? wv % NW : wv;
    const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
    const int per = KS > 1 ? (p.S + KS - 1) / KS : p.S, kb0 = KS > 1 ? min(p.S, grp * per) : 0;
    const int S = KS > 1 ? min(per, p.S - kb0) : p.S;     // k-blocks of this group: kb0 .. kb0 + S - 1 (the barriers are those of `per`)
    // DMA piece q of this wave: 16 rows of the stage's [A rows | B rows]
    const int8_t* base[NP]; unsigned off[NP];
#pragma unroll
    for (int q = 0; q < NP; ++q) {
        const int row0 = (wave * NP + q) * 16, r = row0 + (lane >> 2);
        const int c = (lane & 3) ^ i8_swz(r);
        if (row0 < BM) { base[q] = p.A + (size_t)m0 * p.lda + kb0 * 64; off[q] = (unsigned)((min(m0 + r, p.M - 1) - m0) * p.lda + c * 16); }
        else { base[q] = p.B + (size_t)n0 * p.ldb + kb0 * 64; off[q] = (unsigned)((min(n0 + r - BM, p.N - 1) - n0) * p.ldb + c * 16); }
    }
    char* ring = i8_smem + grp * RING;
    const unsigned lds0 = lds_addr_of(ring);
    auto issue1 = [&](int s, int q) { dma16_to_lds_sbase(base[q] + (size_t)s * 64, off[q], lds0 + (NS == 4 ? (s & 3) : s % NS) * STAGE + (wave * NP + q) * 1024); };
    const int frow = lane & 15, fq = lane >> 4;
    const int fc = (fq ^ i8_swz(frow)) * 16;              // (row bases are multiples of 16: f depends on frow only)
    const char* ra = ring + (wm + frow) * 64 + fc;
    const char* rb = ring + (BM + wn + frow) * 64 + fc;
    i32x4 acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[i][j] = (i32x4){0, 0, 0, 0};
    i32x4 f[2][TI + TJ];
    auto read1 = [&](int s, int q) -> i32x4 {              // fragment q of block s: the A rows' first, then the B rows'
        const int st = (NS == 4 ? (s & 3) : s % NS) * STAGE;
        return q < TI ? *(const i32x4*)(ra + st + q * 1024) : *(const i32x4*)(rb + st + (q - TI) * 1024);
    };
    auto wait_stages = [&](int left) {                     // at most `left` stages of this wave's DMA still in flight
        if (left >= 3) dma_wait_but<3 * NP>(); else if (left == 2) dma_wait_but<2 * NP>(); else if (left == 1) dma_wait_but<NP>(); else dma_wait_but<0>();
    };
    for (int s = 0; s < NS && s < S; ++s) for (int q = 0; q < NP; ++q) issue1(s, q);
    // the tile's scales and bias wait in LDS for the epilogue: [sa: BM | sb: BN | bias: BN]
    float* sc = (float*)(i8_smem + KS * RING);
    for (int i = threadIdx.x; i < BM + BN; i += NT) {
        if (i < BM) sc[i] = p.sa[min(m0 + i, p.M - 1)];
        else {
            const int n = min(n0 + i - BM, p.N - 1);
            sc[i] = p.sb[n]; sc[i + BN] = p.bias ? p.bias[n] : 0.f;
        }
    }
    wait_stages(min(NS, S) - 1);
    __syncthreads();
    if (KS == 1 || S > 0) {
#pragma unroll
        for (int q = 0; q < TI + TJ; ++q) f[0][q] = read1(0, q);
    }
    auto step = [&](int s, i32x4 (&cur)[TI + TJ], i32x4 (&nxt)[TI + TJ]) {
        // block s's fragments are in registers (every wave's: its stage is free behind the barrier), block s + 1 has landed
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (s + 1 < S) wait_stages(min(NS - 2, S - 2 - s));
        __syncthreads();
        if (KS > 1 && s >= S) return;
        const bool more = s + 1 < S, far = s + NS < S;
        constexpr int RPR = (TI + TJ + TI - 1) / TI, PPR = (NP + TI - 1) / TI;   // fragment reads and DMA pieces per MFMA row
#pragma unroll
        for (int i = 0; i < TI; ++i) {
#pragma unroll
            for (int q = i * RPR; q < (i + 1) * RPR && q < TI + TJ; ++q) if (more) nxt[q] = read1(s + 1, q);
#pragma unroll
            for (int q = i * PPR; q < (i + 1) * PPR && q < NP; ++q) if (far) issue1(s + NS, q);
#pragma unroll
            for (int j = 0; j < TJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(cur[TI + j], cur[i], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    int s = 0;
    for (; s + 1 < per; s += 2) { step(s, f[0], f[1]); step(s + 1, f[1], f[0]); }
    if (s < per) step(s, f[0], f[1]);
    if constexpr (KS > 1) {
        // row i of the sub-tiles is finished by group i % KS: the others hand it their sums
        auto slot = [&](int i, int j, int src) { return (i32x4*)i8_smem + (((i * TJ + j) * (KS - 1) + (src < i % KS ? src : src - 1)) * NW + wave) * 64 + lane; };
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TI; ++i)
#pragma unroll
            for (int j = 0; j < TJ; ++j) if (i % KS != grp) *slot(i, j, grp) = acc[i][j];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TI; ++i)
#pragma unroll
            for (int j = 0; j < TJ; ++j)
#pragma unroll
                for (int g = 0; g < KS; ++g) if (i % KS == grp && g != grp) acc[i][j] += *slot(i, j, g);
    }
    // Epilogue.  A lane holds row frow of a sub-tile and four consecutive columns of each; 16 rows x CW columns of the wave go through
    // LDS (the stages are free: the last block's fragments were read in front of the last barrier) and out in whole rows, as many bytes a
    // lane as their alignment allows, consecutive lanes in consecutive places.
    constexpr int CW = TJ * 16, RBMAX = CW * 4 + 16;
    constexpr int OB0 = KS > 1 ? (KS - 1) * BM * BN * 4 : 0;
    static_assert(OB0 + NW * KS * 16 * RBMAX <= KS * RING, "the waves' output rows fit the stages");
    char* ob = i8_smem + OB0 + wv * 16 * RBMAX;
    const int es = p.out_bf16 ? 2 : 4, RB = CW * es + 16;
    const int ncols = min(CW, p.N - (n0 + wn));            // (may be <= 0: a wave beyond the last column)
#pragma unroll
    for (int i = 0; i < TI; ++i) {
        const int mt = m0 + wm + i * 16, nrows = min(16, p.M - mt);
        if (nrows <= 0 || ncols <= 0) break;
        if (KS > 1 && i % KS != grp) continue;
        const float sa = sc[wm + i * 16 + frow];
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
            const float4 sb = *(const float4*)(sc + BM + wn + j * 16 + fq * 4), bi = *(const float4*)(sc + BM + BN + wn + j * 16 + fq * 4);
            const float y0 = i8_scale(acc[i][j][0], sa, sb.x, bi.x, p.relu), y1 = i8_scale(acc[i][j][1], sa, sb.y, bi.y, p.relu);
            const float y2 = i8_scale(acc[i][j][2], sa, sb.z, bi.z, p.relu), y3 = i8_scale(acc[i][j][3], sa, sb.w, bi.w, p.relu);
            char* o = ob + frow * RB + (j * 16 + fq * 4) * es;
            if (p.out_bf16) *(uint2*)o = make_uint2(f2bf_pk(y0, y1), f2bf_pk(y2, y3));
            else *(float4*)o = make_float4(y0, y1, y2, y3);
        }
        char* c = (char*)p.C + ((size_t)mt * p.ldc + n0 + wn) * es;
        const size_t cs = (size_t)p.ldc * es;
        const int nb = ncols * es;                         // bytes of a row
        // as many bytes a lane as the rows' alignment allows; all of the wave's rows are read before the first is stored (with a loop in which each
        // store waited for its own LDS read, 7398 x 4337 x 812 took 70 us by elements, so 51; in whole 16 bytes (4336) 49, so 45)
        auto put = [&](auto type, auto places) {
            using T = decltype(type);
            constexpr int PER = decltype(places)::value, RPI = 64 / PER, N = 16 / RPI;          // places of a row, rows an instruction
            const int rr = lane / PER, k = (lane % PER) * (int)sizeof(T);
            T v[N];
#pragma unroll
            for (int n = 0; n < N; ++n) v[n] = *(const T*)(ob + (rr + n * RPI) * RB + k);
#pragma unroll
            for (int n = 0; n < N; ++n) if (rr + n * RPI < nrows && k < nb) *(T*)(c + (rr + n * RPI) * cs + k) = v[n];
        };
        const int vec = ncols == CW ? p.vec : p.vec >= 4 && (nb & 3) == 0 ? 4 : 0;
        if (es == 4) {
            if (vec == 16) put(make_uint4(0, 0, 0, 0), std::integral_constant<int, CW / 4>{});
            else if (vec == 8) put(make_uint2(0, 0), std::integral_constant<int, CW / 2>{});
            else put(0u, std::integral_constant<int, CW>{});
        } else {
            if (vec == 16) put(make_uint4(0, 0, 0, 0), std::integral_constant<int, CW / 8>{});
            else if (vec == 8) put(make_uint2(0, 0), std::integral_constant<int, CW / 4>{});
            else if (vec == 4) put(0u, std::integral_constant<int, CW / 2>{});
            else put((unsigned short)0, std::integral_constant<int, CW>{});
        }
    }
}

// the last round's tiles leave as quarters up to this many (each then takes about 0.27 of a round of whole tiles)
#define I8_QUARTERED 96
// workgroup L of W runs on XCD L % 8: each XCD takes a contiguous eighth of the list
__device__ __forceinline__ int xcd_order(int L, int W) {
    const int q = W >> 3, r = W & 7, xcd = L & 7, idx = L >> 3;
    return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
}
// tile w of ntm x ntn, in blocks of eight tile rows: the tiles an XCD has in flight (32 of 256 x 256) share few panels of either operand
// (8192^3: 475 us in columns of the whole height, 446 in blocks; 8704 x 8192 x 2048 166 and 157: the panels then stay in the XCD's 4 MB of L2.
// Where a dimension ends just behind a tile its edge strips count like whole tiles: 4099 x 4100 has 17 x 17, of which eight strips go into
// the full round and eight whole tiles into the quartered rest)
__device__ __forceinline__ void tile_of(int w, int ntm, int ntn, int& tm, int& tn) {
    constexpr int GM = 8;
    const int g = w / (GM * ntn), gr = min(GM, ntm - g * GM), o = w - g * GM * ntn;
    tn = o / gr; tm = g * GM + (o - tn * gr);
}
// QUARTERS: workgroups from p.full on own a quarter (BM / 2 x BN / 2) of one of the remaining tiles -- the last, partly filled round of
// the chip in four times as many pieces
template <int BM, int BN, int WM, int WN, int NS, int KS, int WGS, bool QUARTERS>
__global__ __launch_bounds__(64 * WM * WN * KS, WM * WN * KS * WGS / 4) void k_gemm_i8_tile(I8Args p) {
    const int ntm = (p.M + BM - 1) / BM, ntn = (p.N + BN - 1) / BN, L = blockIdx.x;
    int tm, tn;
    if constexpr (QUARTERS) {
        if (L >= p.full) {
            const int w = xcd_order(L - p.full, (ntm * ntn - p.full) * 4), q = w & 3;
            tile_of(p.full + (w >> 2), ntm, ntn, tm, tn);
            const int m0 = tm * BM + (q & 1) * (BM / 2), n0 = tn * BN + (q >> 1) * (BN / 2);
            if (m0 < p.M && n0 < p.N) i8_tile<BM / 2, BN / 2, WM, WN, NS, KS>(p, m0, n0);
            return;
        }
    }
    tile_of(xcd_order(L, p.full), ntm, ntn, tm, tn);
    i8_tile<BM, BN, WM, WN, NS, KS>(p, tm * BM, tn * BN);
}

// ---- few rows: the weights' bytes are what there is to move ------------------------------------------------------------------------
// A workgroup owns NTL * 16 output columns of MT * 16 rows, its NWV waves split K.  Every wave streams its share through a ring of D
// k-blocks of its own in LDS (DMA, no barrier: it waits for its own loads) and multiplies from there.  Straight to registers the same
// loads run at 36 GB/s a CU whatever the shape -- in MFMA order neighbouring lanes belong to different rows, four cache lines a
// quad of lanes --, through LDS a quad reads one 64-byte line.  The waves' partial sums meet in LDS (integer adds: their order
// does not matter).
// FUSED: the activations are x (fp32 / bf16, up to 8 rows), quantised by every workgroup for itself into LDS while its first weights are on
// their way.
template <int MT, int NTL, int NWV, int D, int FUSED /* 0 no, 1 fp32, 2 bf16 */>
__global__ __launch_bounds__(64 * NWV) void k_gemm_i8_rows(I8Args p) {
    static_assert(!FUSED || NWV == 8, "a wave for each of the rows");
    constexpr int NT = 64 * NWV, MR = MT * 16, NC = NTL * 16, NP = (FUSED ? 0 : MT) + NTL, RING = D * NP * 1024;
    __shared__ int part[MR * NC];
    __shared__ float red[NWV], sxs[FUSED ? MR : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n0 = blockIdx.x * NC, m0 = blockIdx.y * MR, frow = lane & 15, fq = lane >> 4;
    const int per = (p.S + NWV - 1) / NWV, s0 = min(p.S, wave * per), n = min(per, p.S - s0);     // this wave's k-blocks: s0 .. s0 + n - 1
    const int8_t* base[NP]; unsigned off[NP];
    {   // DMA piece q: 16 rows of 64 B; chunk c of row r lies at chunk position c ^ f(r)
        const int r = lane >> 2, c = ((lane & 3) ^ i8_swz(r)) * 16;
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            if (q < NTL) { base[q] = p.B + (size_t)n0 * p.ldb + s0 * 64; off[q] = (unsigned)((min(n0 + q * 16 + r, p.N - 1) - n0) * p.ldb + c); }
            else { base[q] = p.A + (size_t)m0 * p.lda + s0 * 64; off[q] = (unsigned)((min(m0 + (q - NTL) * 16 + r, p.M - 1) - m0) * p.lda + c); }
        }
    }
    const char* ring = i8_smem + wave * RING;
    const unsigned lds0 = lds_addr_of(ring);
    auto issue = [&](int s) {
#pragma unroll
        for (int q = 0; q < NP; ++q) dma16_to_lds_sbase(base[q] + (size_t)s * 64, off[q], lds0 + ((s % D) * NP + q) * 1024);
    };
    for (int s = 0; s < D && s < n; ++s) issue(s);
    for (int i = tid; i < MR * NC; i += NT) part[i] = 0;
    const int ldq = p.S * 64 + 16;                         // (FUSED: rows 16 B apart from a multiple of 64: sixteen rows of a read share no bank)
    char* xq = i8_smem + NWV * RING;
    i32x4 acc[MT][NTL];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j) acc[i][j] = (i32x4){0, 0, 0, 0};
    if (FUSED) {
        // up to NWV rows, each by as many waves as there are for it (a power of two)
        const int tpr = NT >> (p.M > 4 ? 3 : p.M > 2 ? 2 : p.M > 1 ? 1 : 0), wpr = tpr >> 6, t = tid & (tpr - 1), m = tid / tpr;
        const bool in = m < p.M;
        const char* row = (const char*)p.x + (size_t)(in ? m : 0) * p.ldx * (FUSED == 2 ? 2 : 4);
        f8 v[2];                                           // (two groups of eight a thread stay in registers; more come from the cache again)
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < 2; ++c) { const int i = (c * tpr + t) * 8; if (i < p.S * 64) { v[c] = act8<FUSED == 2>(row, i, p.K, p.xvec); top = top8(v[c], top); } }
        for (int i = (2 * tpr + t) * 8; i < p.S * 64; i += tpr * 8) top = top8(act8<FUSED == 2>(row, i, p.K, p.xvec), top);
        top = wave_max(top);
        if (wpr > 1) {                                     // (uniform over the workgroup)
            if (lane == 0) red[wave] = top;
            __syncthreads();
            const int w0 = wave & ~(wpr - 1);
            for (int w = 0; w < wpr; ++w) top = fmaxf(top, red[w0 + w]);
        }
        if (in) {
            if (t == 0) sxs[m] = top / 127.0f;
            const float inv = 127.0f / top;
            char* q = xq + m * ldq;
#pragma unroll
            for (int c = 0; c < 2; ++c) { const int i = (c * tpr + t) * 8; if (i < p.S * 64) *(uint2*)(q + i) = quant8(v[c], top, inv); }
            for (int i = (2 * tpr + t) * 8; i < p.S * 64; i += tpr * 8) *(uint2*)(q + i) = quant8(act8<FUSED == 2>(row, i, p.K, p.xvec), top, inv);
        }
    }
    __syncthreads();
    const char* fr = ring + frow * 64 + (fq ^ i8_swz(frow)) * 16;
    for (int s = 0; s < n; ++s) {
        // at most the later blocks' loads still in flight: block s has landed
        const int left = min(D - 1, n - 1 - s);
        if (left >= 3 && D > 3) dma_wait_but<(D > 3 ? 3 * NP : 0)>(); else if (left == 2 && D > 2) dma_wait_but<(D > 2 ? 2 * NP : 0)>();
        else if (left == 1) dma_wait_but<NP>(); else dma_wait_but<0>();
        i32x4 a[MT], b[NTL];
#pragma unroll
        for (int j = 0; j < NTL; ++j) b[j] = *(const i32x4*)(fr + ((s % D) * NP + j) * 1024);
#pragma unroll
        for (int i = 0; i < MT; ++i)
            a[i] = FUSED ? *(const i32x4*)(xq + min(i * 16 + frow, p.M - 1) * ldq + (s0 + s) * 64 + fq * 16) : *(const i32x4*)(fr + ((s % D) * NP + NTL + i) * 1024);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (read: the block's place may be filled again)
        if (s + D < n) issue(s + D);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NTL; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[j], a[i], acc[i][j], 0, 0, 0);
    }
    if (n > 0) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NTL; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) atomicAdd(&part[(i * 16 + frow) * NC + j * 16 + fq * 4 + r], acc[i][j][r]);
    }
    __syncthreads();
    for (int e = tid; e < MR * NC; e += NT) {
        const int ml = e / NC, c = n0 + (e - ml * NC), m = m0 + ml;
        if (m >= p.M || c >= p.N) continue;
        // (f2bf_pk: a NaN stays one whatever its low bits; f2bf's addition carries them into the sign)
        const float y = i8_scale(part[e], FUSED ? sxs[ml] : p.sa[m], p.sb[c], p.bias ? p.bias[c] : 0.f, p.relu);
        if (p.out_bf16) ((bf16_t*)p.C)[(size_t)m * p.ldc + c] = (bf16_t)f2bf_pk(y, y); else ((float*)p.C)[(size_t)m * p.ldc + c] = y;
    }
}

// Kernels above 64 KiB of LDS ask for it before their first launch on each device (`done`: a bit a device; a race sets the same attribute twice).
static int i8_lds(const void* kern, size_t lds, size_t most, std::atomic<unsigned long long>& done) {
    if (lds <= 65536) return E2T_OK;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) { e2t_set_error("%s:%d: no current device", __FILE__, __LINE__); return E2T_ERR_HIP; }
    const unsigned long long bit = 1ull << (dev & 63);
    if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return E2T_OK;
    if (hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)most) != hipSuccess) { e2t_set_error("%s:%d: LDS size", __FILE__, __LINE__); return E2T_ERR_HIP; }
    done.fetch_or(bit, std::memory_order_relaxed);
    return E2T_OK;
}
template <int BM, int BN, int WM, int WN, int NS, int KS, int WGS, bool QUARTERS> static int i8_tile_launch(I8Args p, void* stream) {
    constexpr int lds = (BM + BN) * 64 * NS * KS + (BM + 2 * BN) * 4;
    static_assert(lds * WGS <= 160 * 1024, "LDS");
    const long long W = (long long)((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN);
    E2T_CHECK_ARG(W < (1ll << 24));
    p.full = (int)W;
    if (QUARTERS) { const int left = (int)(W % 256); if (W > 256 && left <= I8_QUARTERED) p.full = (int)W - left; }
    const unsigned grid = (unsigned)(p.full + (W - p.full) * 4);
    auto kern = k_gemm_i8_tile<BM, BN, WM, WN, NS, KS, WGS, QUARTERS>;
    static std::atomic<unsigned long long> done;
    if (int rc = i8_lds((const void*)kern, lds, lds, done)) return rc;
    hipLaunchKernelGGL(kern, dim3(grid), dim3(64 * WM * WN * KS), lds, ST, p);
    E2T_LAUNCH_CHECK(); return E2T_OK;
}
template <int MT, int NTL, int NWV, int D> static int i8_rows_launch(const I8Args& p, void* stream) {
    const dim3 grid((p.N + NTL * 16 - 1) / (NTL * 16), (p.M + MT * 16 - 1) / (MT * 16));
    E2T_CHECK_ARG(grid.y <= 65535);
    constexpr size_t lds = NWV * D * (MT + NTL) * 1024;
    static std::atomic<unsigned long long> done;
    auto kern = k_gemm_i8_rows<MT, NTL, NWV, D, 0>;
    if (int rc = i8_lds((const void*)kern, lds, lds, done)) return rc;
    hipLaunchKernelGGL(kern, grid, dim3(64 * NWV), lds, ST, p);
    E2T_LAUNCH_CHECK(); return E2T_OK;
}
// Which instance: the one whose predicted time is the shortest.  The predictions (microseconds; S = 64-byte k-blocks, W = tiles) are straight
// lines through measured times of every instance at 120 shapes, M 16 .. 8704, N 100 .. 16384, K 64 .. 16384.  The chosen instance takes 3 % more
// than the best one on average, there and over 110 other shapes (M from 1); on those it is 29 % off at most, on the fitted ones 51 % at
// 512 x 512 x 16384 (30.1 us, 20.0), 32 % at 501 x 347 x 13543 and 20 % elsewhere.  Both sides of the larger steps:
//   M = 16, 4096 x 4096: rows 4.8, 64 x 64 tiles 13.8;   M = 128: rows 11.2, tiles in two K groups 12.0;   M = 256: rows 20.6, tiles 12.5
//   M = 1024, 4096 x 4096: 64 x 64 41, 128 x 128 31, 128 x 128 in two K groups 27, 256 x 256 52;   M = 4096: 128 x 128 84, 256 x 256 63
// No instance splits K over workgroups: few tiles of a long K take two to ten times their floor (464 x 4103 x 11997 58 us, floor 21).
static int i8_instance(int M, int N, int K) {
    const double S = (K + 63) / 64, K64 = 64.0 * S, bytes = N * K64;
    auto cdiv = [](long long a, long long b) { return (double)((a + b - 1) / b); };
    struct { double us; int kind; } best = {1e30, 0};
    auto take = [&](double us, int kind) { if (us < best.us) { best.us = us; best.kind = kind; } };
    // few rows: start and reduction, then the longest of a wave's chain of steps, the workgroups' reads (12 TB/s) and the weights' from memory
    auto rows = [&](int mt, int ntl, int nwv, double step, int kind) {
        const double mb = cdiv(M, mt * 16), blocks = cdiv(N, ntl * 16) * mb, am = M < mt * 16 ? M : mt * 16;
        const double l2 = blocks * (am + ntl * 16) * K64 / 1.2e7, mem = bytes / 5e6 * (bytes > 3e7 ? mb : 1);
        take(2.2 + 0.5 * mt * ntl + (nwv == 8 ? 0.2 : 0) + fmax(fmax(l2, mem), S / nwv * step), kind);
    };
    if (M <= 512) {
        rows(1, 1, 4, 0.125, 0); rows(1, 1, 8, 0.144, 1); rows(1, 2, 4, 0.14, 2); rows(2, 1, 4, 0.14, 3); rows(2, 2, 4, 0.16, 4); rows(2, 4, 4, 0.18, 5);
    }
    // tiles: the latency of one tile, or the chip's throughput where they queue up
    auto tiles = [&](int t, double step, double fill, double per_step, double per_tile, double base, int kind) {
        const double W = cdiv(M, t) * cdiv(N, t), even = W + 0.66 * (256.0 * ceil(W / 256) - W);      // (some CUs have a tile more than others)
        take(fmax(fmax(step * S + fill, per_step * even * S + per_tile * W + base), 2.7 + bytes / 5e6), kind);
        return W;
    };
    if (tiles(64, 0.20, 4.2, 0.0006, 0.0012, 4.0, 6) <= 256) take(fmax(0.13 * S + 5.0, 2.7 + bytes / 5e6), 7);
    if (tiles(128, 0.36, 7.5, 0.0011, 0.0064, 5.0, 8) <= 256) take(fmax(0.27 * S + 8.5, 2.7 + bytes / 5e6), 9);
    {
        const double W = cdiv(M, 256) * cdiv(N, 256), left = W < 256 ? 0 : W - 256 * floor(W / 256);
        const double round = W < 256 ? 0.7 * S + 11 : 0.85 * S + 13;
        take((W < 256 ? 1 : floor(W / 256)) * round + (left == 0 ? 0 : left <= I8_QUARTERED ? 0.27 * round : round), 10);
    }
    return best.kind;
}
static int i8_launch(const I8Args& p, void* stream) {
    switch (i8_instance(p.M, p.N, p.K)) {
    case 0: return i8_rows_launch<1, 1, 4, 4>(p, stream);
    case 1: return i8_rows_launch<1, 1, 8, 4>(p, stream);
    case 2: return i8_rows_launch<1, 2, 4, 4>(p, stream);
    case 3: return i8_rows_launch<2, 1, 4, 4>(p, stream);
    case 4: return i8_rows_launch<2, 2, 4, 4>(p, stream);
    case 5: return i8_rows_launch<2, 4, 4, 4>(p, stream);
    case 6: return i8_tile_launch<64, 64, 2, 2, 4, 1, 4, false>(p, stream);
    case 7: return i8_tile_launch<64, 64, 2, 2, 4, 2, 2, false>(p, stream);
    case 8: return i8_tile_launch<128, 128, 2, 2, 3, 1, 3, false>(p, stream);
    case 9: return i8_tile_launch<128, 128, 2, 2, 4, 2, 1, false>(p, stream);
    default: return i8_tile_launch<256, 256, 2, 4, 4, 1, 1, true>(p, stream);
    }
}
template <int NTL, int NWV, int D> static int i8_fused_launch(const I8Args& p, void* stream) {
    const dim3 grid((p.N + NTL * 16 - 1) / (NTL * 16));
    const size_t lds = NWV * D * NTL * 1024 + (size_t)p.M * (p.S * 64 + 16);
    static std::atomic<unsigned long long> done[2];
    auto kern = p.xbf16 ? k_gemm_i8_rows<1, NTL, NWV, D, 2> : k_gemm_i8_rows<1, NTL, NWV, D, 1>;
    if (int rc = i8_lds((const void*)kern, lds, 140 * 1024, done[p.xbf16])) return rc;
    hipLaunchKernelGGL(kern, grid, dim3(64 * NWV), lds, ST, p);
    E2T_LAUNCH_CHECK(); return E2T_OK;
}

// A launch has fewer than 2^32 threads.  What needs more runs in pieces: rows to quantise (256 threads each at most), columns of a product (at
// most 512 threads for sixteen), and as many of its rows as then make fewer than 2^24 tiles of 64 x 64 (256 threads each).
#define I8_QUANT_ROWS (1 << 22)
#define I8_COLS (1 << 20)
extern "C" int e2t_quant_rows_i8(const void* x, int dtype, long long ldx, int M, int K, int8_t* q, long long ldq, float* scale, void* stream) {
    E2T_CHECK_ARG(x && q && scale && M > 0 && M <= E2T_I8_MAX_ROWS && K > 0 && K < (1 << 30) && ldx >= K && (dtype == E2T_DT_F32 || dtype == E2T_DT_BF16));
    E2T_CHECK_ARG(ldq >= ((K + 63) & ~63) && (ldq & 15) == 0 && ((uintptr_t)q & 15) == 0 && ((uintptr_t)x & (dtype == E2T_DT_F32 ? 3 : 1)) == 0);
    const int vec = (((uintptr_t)x | (unsigned long long)(ldx * (dtype == E2T_DT_F32 ? 4 : 2))) & 15) == 0;
#define QL(T, NC)                                                                                                                             \
    do {                                                                                                                                      \
        const dim3 g((rows + 256 / T - 1) / (256 / T));                                                                                       \
        if (dtype == E2T_DT_BF16) hipLaunchKernelGGL((k_quant_rows<true, T, NC>), g, dim3(256), 0, ST, xs, ldx, rows, K, vec, qs, ldq, scale + m0);  \
        else hipLaunchKernelGGL((k_quant_rows<false, T, NC>), g, dim3(256), 0, ST, xs, ldx, rows, K, vec, qs, ldq, scale + m0);                      \
    } while (0)
    for (int m0 = 0; m0 < M; m0 += I8_QUANT_ROWS) {
        const int rows = M - m0 < I8_QUANT_ROWS ? M - m0 : I8_QUANT_ROWS;
        const void* xs = (const char*)x + (size_t)m0 * ldx * (dtype == E2T_DT_F32 ? 4 : 2);
        int8_t* qs = q + (size_t)m0 * ldq;
        if (K <= 1024 && M >= 512) QL(64, 2);
        else if (K <= 4096) QL(256, 2);
        else QL(256, 4);
        E2T_LAUNCH_CHECK();
    }
#undef QL
    return E2T_OK;
}

static int gemm_i8_check(const void* B, long long ldb, const float* sb, const void* C, long long ldc, int M, int N, int K, int flags) {
    E2T_CHECK_ARG(B && sb && C && M > 0 && M <= E2T_I8_MAX_ROWS && N > 0 && N <= E2T_I8_MAX_ROWS && K > 0 && K <= E2T_I8_MAX_K);
    const long long K64 = ((long long)K + 63) & ~63ll;
    E2T_CHECK_ARG(ldb <= E2T_I8_MAX_LD && ldb >= K64 && (ldb & 15) == 0 && ldc >= N && ((uintptr_t)B & 15) == 0);
    E2T_CHECK_ARG((flags & ~(E2T_GEMM_RELU | E2T_GEMM_OUT_BF16)) == 0 && ((uintptr_t)C & ((flags & E2T_GEMM_OUT_BF16) ? 1 : 3)) == 0);
    return E2T_OK;
}
static I8Args i8_args(const int8_t* B, long long ldb, const float* sb, const float* bias, void* C, long long ldc, int M, int N, int K, int flags) {
    I8Args p{};
    p.B = B; p.sb = sb; p.bias = bias; p.C = C; p.ldb = ldb; p.ldc = ldc;
    p.M = M; p.N = N; p.K = K; p.S = (K + 63) / 64; p.relu = (flags & E2T_GEMM_RELU) != 0; p.out_bf16 = (flags & E2T_GEMM_OUT_BF16) != 0;
    const unsigned long long al = (unsigned long long)(ldc * (p.out_bf16 ? 2 : 4)) | (uintptr_t)C;
    p.vec = (al & 15) == 0 ? 16 : (al & 7) == 0 ? 8 : (al & 3) == 0 ? 4 : 0;
    return p;
}
extern "C" int e2t_gemm_nt_i8(const int8_t* A, long long lda, const float* sa, const int8_t* B, long long ldb, const float* sb,
                              const float* bias, void* C, long long ldc, int M, int N, int K, int flags, void* stream) {
    if (int rc = gemm_i8_check(B, ldb, sb, C, ldc, M, N, K, flags)) return rc;
    E2T_CHECK_ARG(A && sa && lda <= E2T_I8_MAX_LD && lda >= (((long long)K + 63) & ~63ll) && (lda & 15) == 0 && ((uintptr_t)A & 15) == 0);
    const int nn = N < I8_COLS ? N : I8_COLS;
    const long long fit = (((1ll << 24) / ((nn + 63) / 64) - 1) * 64) & ~255ll;
    const int mm = M < fit ? M : (int)fit;
    const size_t es = flags & E2T_GEMM_OUT_BF16 ? 2 : 4;
    for (int n0 = 0; n0 < N; n0 += nn)
        for (long long m0 = 0; m0 < M; m0 += mm) {
            I8Args p = i8_args(B + (size_t)n0 * ldb, ldb, sb + n0, bias ? bias + n0 : nullptr, (char*)C + ((size_t)m0 * ldc + n0) * es, ldc,
                               M - m0 < mm ? (int)(M - m0) : mm, N - n0 < nn ? N - n0 : nn, K, flags);
            p.A = A + (size_t)m0 * lda; p.sa = sa + m0; p.lda = lda;
            if (int rc = i8_launch(p, stream)) return rc;
        }
    return E2T_OK;
}

extern "C" int e2t_gemm_i8_instance(int M, int N, int K) {
    return M > 0 && M <= E2T_I8_MAX_ROWS && N > 0 && N <= E2T_I8_MAX_ROWS && K > 0 && K <= E2T_I8_MAX_K ? i8_instance(M, N, K) : -1;
}

static inline size_t lin_q_bytes(int M, int K) { return ((size_t)M * (size_t)((K + 63) & ~63) + 255) & ~(size_t)255; }
// One launch where quantising again in every workgroup (16 outputs each) costs less than a launch of its own.  us for one / two launches,
// N = 1806 .. 4096: M = 1, K = 4096 5.2 / 7.8; M = 2, K = 8192 10 / 12; M = 4, K = 2048 6.0 / 6.4, K = 4096 9.1 / 8.3; M = 8, K = 1024 5.6 / 6.2,
// K = 2048 8.3 / 6.6.  Many outputs: N = 9000, M = 1, K = 2048 6.1 / 7.6, M = 2 6.9 / 7.8, M = 4 8.4 / 7.8; N = 16384, M = 1, K = 4096 12.6 / 16.2,
// M = 2 17.5 / 16.2.  (In one launch M = 1 gains at every N measured: above 12288 outputs and below K = 4096 the rule still takes two, 9.0 us for
// 7.6 at 16384 x 2048.)
static bool lin_fused(int M, int N, int K) {
    if ((size_t)M * (((K + 63) & ~63) + 16) > 100 * 1024) return false;
    return N > 8192 ? M == 1 && (K >= 4096 || N <= 12288) : M <= 2 || (M <= 8 && M * K <= 8192);
}
extern "C" size_t e2t_linear_i8_ws_bytes(int M, int N, int K) {
    return M > 0 && N > 0 && K > 0 && K <= E2T_I8_MAX_K && !lin_fused(M, N, K) ? lin_q_bytes(M, K) + (size_t)M * sizeof(float) : 0;
}
extern "C" int e2t_linear_i8(const void* x, int dtype, long long ldx, const int8_t* W, long long ldw, const float* sw, const float* bias, void* y,
                             long long ldy, int M, int N, int K, int flags, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = gemm_i8_check(W, ldw, sw, y, ldy, M, N, K, flags)) return rc;
    E2T_CHECK_ARG((ws || lin_fused(M, N, K)) && ws_bytes >= e2t_linear_i8_ws_bytes(M, N, K) && ((uintptr_t)ws & 15) == 0);
    E2T_CHECK_ARG(x && ldx >= K && (dtype == E2T_DT_F32 || dtype == E2T_DT_BF16) && ((uintptr_t)x & (dtype == E2T_DT_F32 ? 3 : 1)) == 0);
    if (lin_fused(M, N, K)) {
        for (int n0 = 0; n0 < N; n0 += I8_COLS) {
            I8Args p = i8_args(W + (size_t)n0 * ldw, ldw, sw + n0, bias ? bias + n0 : nullptr, (char*)y + n0 * (size_t)(flags & E2T_GEMM_OUT_BF16 ? 2 : 4), ldy, M,
                               N - n0 < I8_COLS ? N - n0 : I8_COLS, K, flags);
            p.x = x; p.ldx = ldx; p.xbf16 = dtype == E2T_DT_BF16; p.xvec = (((uintptr_t)x | (unsigned long long)(ldx * (p.xbf16 ? 2 : 4))) & 15) == 0;
            if (int rc = i8_fused_launch<1, 8, 4>(p, stream)) return rc;
        }
        return E2T_OK;
    }
    const long long ldq = (K + 63) & ~63;
    float* sx = (float*)((char*)ws + lin_q_bytes(M, K));
    if (int rc = e2t_quant_rows_i8(x, dtype, ldx, M, K, (int8_t*)ws, ldq, sx, stream)) return rc;
    return e2t_gemm_nt_i8((const int8_t*)ws, ldq, sx, W, ldw, sw, bias, y, ldy, M, N, K, flags, stream);
}
