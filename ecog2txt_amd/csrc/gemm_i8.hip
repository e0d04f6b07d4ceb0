// Products of 8-bit integers with a scale for each row of either operand, and the quantisation that makes such operands.
//
//   y[m][n] = sa[m] * sb[n] * sum_k a[m][k] * b[n][k]  (+ bias[n])
//
// The sum is exact (int32, K <= 131071); it is rounded once to fp32, scaled, biased and rounded to the output type.
#include "common.h"
#include "ecog2txt_hip.h"
#include <math.h>

#define ST ((hipStream_t)stream)
typedef int i32x4 __attribute__((ext_vector_type(4)));

template <bool BF16> __device__ __forceinline__ float act_at(const void* row, int i) { return BF16 ? bf2f(((const bf16_t*)row)[i]) : ((const float*)row)[i]; }

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

template <bool BF16> __global__ __launch_bounds__(256) void k_quant_rows(const void* x, long long ldx, int K, int8_t* q, long long ldq, float* scale) {
    __shared__ float red[4];
    const int m = blockIdx.x;
    const char* row = (const char*)x + (size_t)m * ldx * (BF16 ? 2 : 4);
    float top = 0.f;
    for (int i = threadIdx.x; i < K; i += 256) { const float v = fabsf(act_at<BF16>(row, i)); if (v < INFINITY) top = fmaxf(top, v); }
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    if (threadIdx.x == 0) scale[m] = top / 127.0f;
    const float inv = 127.0f / top;
    const int K64 = (K + 63) & ~63;
    int8_t* qr = q + (size_t)m * ldq;
    for (int i = threadIdx.x; i < K64; i += 256) qr[i] = i < K ? (int8_t)quant1(act_at<BF16>(row, i), top, inv) : (int8_t)0;
}

// 64 x 64 tile, four waves of 32 x 32, operands straight from global memory in MFMA order (lane = row % 16, 16 bytes of k)
template <bool OUTBF> __global__ __launch_bounds__(256) void k_gemm_i8_simple(const int8_t* A, long long lda, const float* sa, const int8_t* B,
                                                                              long long ldb, const float* sb, const float* bias, void* C,
                                                                              long long ldc, int M, int N, int K64, int relu) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int m0 = blockIdx.y * 64 + (wave >> 1) * 32, n0 = blockIdx.x * 64 + (wave & 1) * 32;
    const int8_t *ap[2], *bp[2];
    for (int i = 0; i < 2; ++i) {
        ap[i] = A + (size_t)min(m0 + i * 16 + (lane & 15), M - 1) * lda + (lane >> 4) * 16;
        bp[i] = B + (size_t)min(n0 + i * 16 + (lane & 15), N - 1) * ldb + (lane >> 4) * 16;
    }
    i32x4 acc[2][2] = {};
    for (int k = 0; k < K64; k += 64) {
        i32x4 a[2], b[2];
        for (int i = 0; i < 2; ++i) { a[i] = *(const i32x4*)(ap[i] + k); b[i] = *(const i32x4*)(bp[i] + k); }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[i], b[j], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int m = m0 + i * 16 + (lane >> 4) * 4 + r, n = n0 + j * 16 + (lane & 15);
                if (m >= M || n >= N) continue;
                float y = (float)acc[i][j][r] * sa[m] * sb[n];
                if (bias) y += bias[n];
                if (relu) y = fmaxf(y, 0.f);
                if (OUTBF) ((bf16_t*)C)[(size_t)m * ldc + n] = f2bf(y); else ((float*)C)[(size_t)m * ldc + n] = y;
            }
}

extern "C" int e2t_quant_rows_i8(const void* x, int dtype, long long ldx, int M, int K, int8_t* q, long long ldq, float* scale, void* stream) {
    E2T_CHECK_ARG(x && q && scale && M > 0 && K > 0 && ldx >= K && (dtype == E2T_DT_F32 || dtype == E2T_DT_BF16));
    E2T_CHECK_ARG(ldq >= ((K + 63) & ~63) && (ldq & 15) == 0 && ((uintptr_t)q & 15) == 0 && ((uintptr_t)x & (dtype == E2T_DT_F32 ? 3 : 1)) == 0);
    if (dtype == E2T_DT_BF16) hipLaunchKernelGGL((k_quant_rows<true>), dim3(M), dim3(256), 0, ST, x, ldx, K, q, ldq, scale);
    else hipLaunchKernelGGL((k_quant_rows<false>), dim3(M), dim3(256), 0, ST, x, ldx, K, q, ldq, scale);
    E2T_LAUNCH_CHECK(); return E2T_OK;
}

static int gemm_i8_check(const void* B, long long ldb, const float* sb, const void* C, long long ldc, int M, int N, int K, int flags) {
    E2T_CHECK_ARG(B && sb && C && M > 0 && N > 0 && K > 0 && K <= E2T_I8_MAX_K);
    const long long K64 = ((long long)K + 63) & ~63ll;
    E2T_CHECK_ARG(ldb >= K64 && (ldb & 15) == 0 && ldc >= N && ((uintptr_t)B & 15) == 0);
    E2T_CHECK_ARG((flags & ~(E2T_GEMM_RELU | E2T_GEMM_OUT_BF16)) == 0 && ((uintptr_t)C & ((flags & E2T_GEMM_OUT_BF16) ? 1 : 3)) == 0);
    return E2T_OK;
}
extern "C" int e2t_gemm_nt_i8(const int8_t* A, long long lda, const float* sa, const int8_t* B, long long ldb, const float* sb,
                              const float* bias, void* C, long long ldc, int M, int N, int K, int flags, void* stream) {
    if (int rc = gemm_i8_check(B, ldb, sb, C, ldc, M, N, K, flags)) return rc;
    E2T_CHECK_ARG(A && sa && lda >= (((long long)K + 63) & ~63ll) && (lda & 15) == 0 && ((uintptr_t)A & 15) == 0);
    const int K64 = (K + 63) & ~63;
    const dim3 grid((N + 63) / 64, (M + 63) / 64);
    E2T_CHECK_ARG(grid.y <= 65535);
    if (flags & E2T_GEMM_OUT_BF16) hipLaunchKernelGGL((k_gemm_i8_simple<true>), grid, dim3(256), 0, ST, A, lda, sa, B, ldb, sb, bias, C, ldc, M, N, K64, flags & E2T_GEMM_RELU);
    else hipLaunchKernelGGL((k_gemm_i8_simple<false>), grid, dim3(256), 0, ST, A, lda, sa, B, ldb, sb, bias, C, ldc, M, N, K64, flags & E2T_GEMM_RELU);
    E2T_LAUNCH_CHECK(); return E2T_OK;
}

static inline size_t lin_q_bytes(int M, int K) { return ((size_t)M * (size_t)((K + 63) & ~63) + 255) & ~(size_t)255; }
extern "C" size_t e2t_linear_i8_ws_bytes(int M, int K) { return M > 0 && K > 0 ? lin_q_bytes(M, K) + (size_t)M * sizeof(float) : 0; }
extern "C" int e2t_linear_i8(const void* x, int dtype, long long ldx, const int8_t* W, long long ldw, const float* sw, const float* bias, void* y,
                             long long ldy, int M, int N, int K, int flags, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = gemm_i8_check(W, ldw, sw, y, ldy, M, N, K, flags)) return rc;
    E2T_CHECK_ARG(ws && ws_bytes >= e2t_linear_i8_ws_bytes(M, K) && ((uintptr_t)ws & 15) == 0);
    const long long ldq = (K + 63) & ~63;
    float* sx = (float*)((char*)ws + lin_q_bytes(M, K));
    if (int rc = e2t_quant_rows_i8(x, dtype, ldx, M, K, (int8_t*)ws, ldq, sx, stream)) return rc;
    return e2t_gemm_nt_i8((const int8_t*)ws, ldq, sx, W, ldw, sw, bias, y, ldy, M, N, K, flags, stream);
}
