// Matrix product in 8-bit integers with a scale per token and per output channel, and the row quantisation
// that feeds it (eg2_quantize_rows, eg2_gemm_i8 in include/eg2.h).
#include "common.cuh"
#include "kernels.h"

namespace eg2 {

// ---------------------------------------------------------------------------------------------
// q[r, c] = rint(x[r, c] * (127 / max_c |x[r, c]|)), scale[r] = max / 127. One warp per row, two passes over
// the row (the second from L1). A row of zeros gets scale 0; a row that holds a NaN or an infinity gets zeros
// and scale NaN, so every product with it is NaN.
// ---------------------------------------------------------------------------------------------
template <typename T>
__global__ void quantize_rows_kernel(const T* __restrict__ x, long ldx, int8_t* __restrict__ q, long ldq,
                                     float* __restrict__ scale, long rows, int k) {
    const long row = (long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int lane = threadIdx.x & 31;
    const T* xr = x + row * ldx;
    float top = 0.f;
    bool bad = false;
    for (int c = lane; c < k; c += 32) {
        const float v = fabsf(ldf(xr, c));
        bad |= !(v < INFINITY);
        top = fmaxf(top, v);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    bad = __any_sync(0xffffffffu, bad);
    const float inv = (bad || top == 0.f) ? 0.f : __fdiv_rn(127.f, top);
    for (int c = lane; c < k; c += 32) q[row * ldq + c] = bad ? (int8_t)0 : (int8_t)__float2int_rn(__fmul_rn(ldf(xr, c), inv));
    if (lane == 0) scale[row] = bad ? __int_as_float(0x7fc00000) : __fdiv_rn(top, 127.f);
}

// ---------------------------------------------------------------------------------------------
// C[m, n] = (sum_k A[m, k] W[n, k]) * sa[m] * sw[n] + bias[n]. 64 x 64 outputs per block, dp4a over 32-byte K
// blocks staged in shared memory.
// ---------------------------------------------------------------------------------------------
template <typename TO>
__global__ void __launch_bounds__(256) gemm_i8_kernel(const int8_t* __restrict__ A, long lda, const float* __restrict__ sa,
                                                      const int8_t* __restrict__ W, long ldw, const float* __restrict__ sw,
                                                      const float* __restrict__ bias, TO* __restrict__ C, long ldc, int M,
                                                      int N, int K) {
    __shared__ int as[64][9], ws[64][9];
    const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < K; k0 += 32) {
        for (int i = threadIdx.x; i < 64 * 32; i += 256) {
            const int r = i >> 5, c = i & 31;
            reinterpret_cast<int8_t*>(as[r])[c] = (m0 + r < M && k0 + c < K) ? A[(long)(m0 + r) * lda + k0 + c] : (int8_t)0;
            reinterpret_cast<int8_t*>(ws[r])[c] = (n0 + r < N && k0 + c < K) ? W[(long)(n0 + r) * ldw + k0 + c] : (int8_t)0;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 8; c++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __dp4a(as[4 * ty + i][c], ws[4 * tx + j][c], acc[i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int m = m0 + 4 * ty + i, n = n0 + 4 * tx + j;
            if (m < M && n < N) stf(C + (long)m * ldc, n, (float)acc[i][j] * sa[m] * sw[n] + (bias ? bias[n] : 0.f));
        }
}

}  // namespace eg2

extern "C" {

int eg2_quantize_rows(int kind, const void* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t rows, int k,
                      void* stream) {
    if ((kind != EG2_F32 && kind != EG2_BF16) || rows < 0 || k <= 0 || ldx < k || ldq < k) return EG2_ERR_INVALID;
    if (rows == 0) return EG2_OK;
    if (!x || !q || !scale || rows > (1L << 31)) return EG2_ERR_INVALID;
    cudaStream_t s = (cudaStream_t)stream;
    const unsigned blocks = (unsigned)((rows + 3) / 4);
    if (kind == EG2_F32)
        eg2::quantize_rows_kernel<float><<<blocks, 128, 0, s>>>((const float*)x, ldx, q, ldq, scale, rows, k);
    else
        eg2::quantize_rows_kernel<bf16_t><<<blocks, 128, 0, s>>>((const bf16_t*)x, ldx, q, ldq, scale, rows, k);
    if (cudaGetLastError() != cudaSuccess) return EG2_ERR_CUDA;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return EG2_OK;
}

int eg2_gemm_i8(const int8_t* A, int64_t lda, const float* a_scale, const int8_t* W, int64_t ldw, const float* w_scale,
                const float* bias, void* C, int64_t ldc, int64_t M, int N, int K, int out_f32, void* stream) {
    if (M < 0 || N <= 0 || K <= 0 || K > EG2_I8_MAX_K || lda < K || ldw < K || ldc < N || lda % 16 || ldw % 16) return EG2_ERR_INVALID;
    if (M == 0) return EG2_OK;
    if (!A || !W || !a_scale || !w_scale || !C || M > (1L << 30) || ((uintptr_t)A | (uintptr_t)W) % 16) return EG2_ERR_INVALID;
    cudaStream_t s = (cudaStream_t)stream;
    const dim3 grid((unsigned)((N + 63) / 64), (unsigned)((M + 63) / 64));
    if (grid.y > 65535) return EG2_ERR_INVALID;
    if (out_f32)
        eg2::gemm_i8_kernel<float><<<grid, 256, 0, s>>>(A, lda, a_scale, W, ldw, w_scale, bias, (float*)C, ldc, (int)M, N, K);
    else
        eg2::gemm_i8_kernel<bf16_t><<<grid, 256, 0, s>>>(A, lda, a_scale, W, ldw, w_scale, bias, (bf16_t*)C, ldc, (int)M, N, K);
    if (cudaGetLastError() != cudaSuccess) return EG2_ERR_CUDA;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return EG2_OK;
}

}  // extern "C"
