// Matrix product in 8-bit integers with a scale per token and per output channel, and the row quantisation
// that feeds it (eg2_quantize_rows, eg2_gemm_i8 in include/eg2.h).
#include "common.cuh"
#include "kernels.h"

namespace eg2 {

// ---------------------------------------------------------------------------------------------
// q[r, c] = rint(x[r, c] * (127 / max_c |x[r, c]|)), scale[r] = max / 127, each operation one IEEE rounding. A row
// of zeros gets scale 0; a row that holds a NaN or an infinity gets zeros and scale NaN, so every product with it
// is NaN. Bound by HBM: a row is read once into registers (TPR threads, NV chunks of 8 elements each), reduced and
// written.
// ---------------------------------------------------------------------------------------------
struct QuantRow {
    float inv, scale;
};
EG2_DEV QuantRow quant_row(float top, bool bad) {
    QuantRow q;
    q.inv = (bad || top == 0.f) ? 0.f : __fdiv_rn(127.f, top);
    q.scale = bad ? __int_as_float(0x7fc00000) : __fdiv_rn(top, 127.f);
    return q;
}
EG2_DEV int quant_one(float x, const QuantRow& q, bool bad) { return bad ? 0 : __float2int_rn(__fmul_rn(x, q.inv)); }

template <typename T>
EG2_DEV void quant_load8(const T* p, int n, float (&v)[8]) {  // n of them exist; p is 16-byte aligned
    if (n >= 8) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
            const uint4 a = *reinterpret_cast<const uint4*>(p);
            const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v[2 * i] = __uint_as_float(u[i] << 16);
                v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < n ? ldf(p, i) : 0.f;
    }
}

template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR)
    quantize_rows_kernel(const T* __restrict__ x, long ldx, int8_t* __restrict__ q, long ldq, float* __restrict__ scale,
                         long rows, int k) {
    grid_dep_launch();
    const long row = TPR == 32 ? (long)blockIdx.x * 4 + (threadIdx.x >> 5) : (long)blockIdx.x;
    if (row >= rows) return;
    const int t = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
    const T* xr = x + row * ldx;
    float v[NV][8];
    float top = 0.f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < NV; i++) quant_load8(xr + 8l * (t + i * TPR), k - 8 * (t + i * TPR), v[i]);
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int y = 0; y < 8; y++) {
            const float a = fabsf(v[i][y]);
            bad |= !(a < INFINITY);
            top = fmaxf(top, a);
        }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    bad = __any_sync(0xffffffffu, bad);
    if constexpr (TPR > 32) {
        __shared__ float part[TPR / 32];
        if ((t & 31) == 0) part[t >> 5] = bad ? INFINITY : top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TPR / 32; i++) top = fmaxf(top, part[i]);
        bad = top == INFINITY;
    }
    const QuantRow qr = quant_row(top, bad);
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = 8 * (t + i * TPR);
        if (c >= k) continue;
        uint32_t u[2] = {0, 0};
#pragma unroll
        for (int y = 0; y < 8; y++) u[y >> 2] |= (uint32_t)(quant_one(v[i][y], qr, bad) & 0xff) << (8 * (y & 3));
        int8_t* to = q + row * ldq + c;
        if (c + 8 <= k) {
            *reinterpret_cast<uint2*>(to) = make_uint2(u[0], u[1]);
        } else {
            for (int y = 0; c + y < k; y++) to[y] = (int8_t)(u[y >> 2] >> (8 * (y & 3)));
        }
    }
    if (t == 0) scale[row] = qr.scale;
}

// Any alignment and length: a block per row, two passes over it (the second from L1 / L2).
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_any_kernel(const T* __restrict__ x, long ldx, int8_t* __restrict__ q,
                                                                long ldq, float* __restrict__ scale, int k) {
    grid_dep_launch();
    const long row = blockIdx.x;
    const T* xr = x + row * ldx;
    float top = 0.f;
    for (int c = threadIdx.x; c < k; c += 256) {
        const float a = fabsf(ldf(xr, c));
        top = fmaxf(top, a < INFINITY ? a : INFINITY);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    __shared__ float part[8];
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) top = fmaxf(top, part[i]);
    const bool bad = top == INFINITY;
    const QuantRow qr = quant_row(top, bad);
    for (int c = threadIdx.x; c < k; c += 256) q[row * ldq + c] = (int8_t)quant_one(ldf(xr, c), qr, bad);
    if (threadIdx.x == 0) scale[row] = qr.scale;
}

template <typename T>
static int quantize_rows(const T* x, long ldx, int8_t* q, long ldq, float* scale, long rows, int k, cudaStream_t s) {
    const bool vec = (uintptr_t)x % 16 == 0 && ldx * sizeof(T) % 16 == 0 && (uintptr_t)q % 8 == 0 && ldq % 8 == 0;
    const unsigned quarter = (unsigned)((rows + 3) / 4), each = (unsigned)rows;
    if (!vec || k > 16384)
        quantize_rows_any_kernel<T><<<each, 256, 0, s>>>(x, ldx, q, ldq, scale, k);
    else if (k <= 256)
        quantize_rows_kernel<T, 32, 1><<<quarter, 128, 0, s>>>(x, ldx, q, ldq, scale, rows, k);
    else if (k <= 512)
        quantize_rows_kernel<T, 32, 2><<<quarter, 128, 0, s>>>(x, ldx, q, ldq, scale, rows, k);
    else if (k <= 1024)
        quantize_rows_kernel<T, 32, 4><<<quarter, 128, 0, s>>>(x, ldx, q, ldq, scale, rows, k);
    else if (k <= 2048)
        quantize_rows_kernel<T, 128, 2><<<each, 128, 0, s>>>(x, ldx, q, ldq, scale, rows, k);
    else if (k <= 4096)
        quantize_rows_kernel<T, 256, 2><<<each, 256, 0, s>>>(x, ldx, q, ldq, scale, rows, k);
    else if (k <= 8192)
        quantize_rows_kernel<T, 256, 4><<<each, 256, 0, s>>>(x, ldx, q, ldq, scale, rows, k);
    else
        quantize_rows_kernel<T, 512, 4><<<each, 512, 0, s>>>(x, ldx, q, ldq, scale, rows, k);
    return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

// ---------------------------------------------------------------------------------------------
// C[m, n] = (sum_k A[m, k] W[n, k]) * a_scale[m] * w_scale[n] + bias[n] on the tensor cores: tcgen05 kind::i8, both
// operands K-major, exact 32-bit sums in TMEM, the scales, the bias and the rounding in the epilogue.
//
// PAIR: clusters of two CTAs on 256 x 256 tiles (M = 256 MMAs; each CTA loads its 128 rows of A and half of W), for
// calls with a tile for every pair of SMs. Otherwise single CTAs on 128 x 64 tiles, which spread the weights of a call
// of few rows over four times as many SMs. Persistent over output tiles, two accumulators:
//   warp 0      TMA producer, 128 bytes of K per stage (past K, M and N the tensor maps read zeros)
//   warp 1      TMEM allocation; lane 0 issues the MMAs (32 bytes of K each) and commits
//   warps 2..9  two epilogue sets of four warps (one per TMEM lane quadrant): set s takes the tiles of parity s
// The result leaves by TMA stores where its rows start at multiples of 16 bytes, else in 64- or 128-byte pieces of
// a row from a staging tile.
// ---------------------------------------------------------------------------------------------
constexpr int I8_THREADS = 320;
template <bool PAIR>
struct I8Cfg {
    static constexpr int BN = PAIR ? 256 : 64;
    static constexpr int A_BYTES = 128 * 128;
    static constexpr int B_BYTES = PAIR ? 128 * 128 : 64 * 128;
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGES = PAIR ? 5 : 6;
    static constexpr int OFF_OUT = STAGES * STAGE;          // per epilogue warp: two 2 KB slots
    static constexpr int OFF_SC = OFF_OUT + 8 * 4096;       // per epilogue warp: the tile's scales and biases
    static constexpr int OFF_BAR = OFF_SC + 8 * 8 * BN;
    static constexpr int N_BARS = 2 * STAGES + 5;
    static constexpr int SMEM = 1024 + OFF_BAR + N_BARS * 8 + 16;
    static constexpr uint32_t TMEM_COLS = 2 * BN;
};
static_assert(I8Cfg<true>::SMEM <= 227 * 1024 && I8Cfg<false>::SMEM <= 227 * 1024, "8-bit product: shared memory");

// Instruction descriptor of kind::i8: D s32, A and B signed, both K-major.
constexpr uint32_t i8_idesc(int M, int N) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
template <bool PAIR>
EG2_DEV void mma_i8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

// int to float on the integer and FMA pipes, rounded once like the conversion instruction: x = 65536 h + l with both
// halves placed in the mantissa of 2^23. The epilogue converts every other value this way, since the conversion unit alone
// (16 a cycle) would take as long as the MMAs of a product over K = 512.
EG2_DEV float i32_to_f32(uint32_t x) {
    const float l = __uint_as_float(__byte_perm(x, 0x4b000000u, 0x7410)) - 8388608.f;
    const float h = __uint_as_float(__byte_perm(x ^ 0x80000000u, 0x4b000000u, 0x7432)) - 8421376.f;  // 2^23 + 2^15
    return fmaf(h, 65536.f, l);
}

struct I8Params {
    const float *sa, *sw, *bias;
    void* C;
    long ldc;
    int M, N, K;
    int tma_out;
};

template <bool PAIR, typename TO>
__global__ void __launch_bounds__(I8_THREADS, 1)
    gemm_i8_tc_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                      const __grid_constant__ CUtensorMap tmC, const I8Params p) {
    using Cfg = I8Cfg<PAIR>;
    constexpr int STAGES = Cfg::STAGES, BN = Cfg::BN, BM = PAIR ? 256 : 128;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
    uint64_t* empty = full + STAGES;
    uint64_t* tfull = empty + STAGES;
    uint64_t* tempty = tfull + 2;
    uint64_t* drain = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
    const bool lead = rank == 0;
    const int tiles_n = (p.N + BN - 1) / BN, tiles = ((p.M + BM - 1) / BM) * tiles_n;
    const int t_first = (int)(blockIdx.x / (PAIR ? 2 : 1)), t_step = (int)(gridDim.x / (PAIR ? 2 : 1));
    const int kblocks = (p.K + 127) / 128;

    if (threadIdx.x == 0) {
        for (int x = 0; x < STAGES; x++) {
            mbar_init(&full[x], 1);
            mbar_init(&empty[x], 1);
        }
        for (int x = 0; x < 2; x++) {
            mbar_init(&tfull[x], 1);
            mbar_init(&tempty[x], PAIR ? 8 : 4);  // the set's warps (of both CTAs)
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbarrier_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmW);
        if (p.tma_out) tma_prefetch_desc(&tmC);
    }
    if (warp == 1) {
        if constexpr (PAIR)
            tmem_alloc_pair(tmem_slot, Cfg::TMEM_COLS);
        else
            tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    if constexpr (PAIR) cluster_sync();  // the peer's barriers are initialised
    grid_dep_launch();
    grid_dep_wait();

    if (warp == 0) {
        if (lane == 0) {
            int loads = 0;
            bool ok = true;
            for (int t = t_first; ok && t < tiles; t += t_step) {
                const int m0 = (t / tiles_n) * BM + 128 * (int)rank, n0 = (t % tiles_n) * BN + (PAIR ? 128 * (int)rank : 0);
                for (int kb = 0; kb < kblocks; kb++, loads++) {
                    const int st = loads % STAGES;
                    if (!(ok = mbar_wait(&empty[st], ((loads / STAGES) & 1) ^ 1, EG2_DEV_TIMEOUT_GEMM, abort_flag))) break;
                    uint8_t* sa = smem + st * Cfg::STAGE;
                    if constexpr (PAIR) {
                        // Both CTAs' bytes complete on the even CTA's barrier.
                        if (lead) mbar_arrive_expect_tx(&full[st], 2 * Cfg::STAGE);
                        const uint32_t bar = mapa_shared(smem_u32(&full[st]), 0);
                        tma_load_2d_pair(sa, &tmA, bar, kb * 128, m0);
                        tma_load_2d_pair(sa + Cfg::A_BYTES, &tmW, bar, kb * 128, n0);
                    } else {
                        mbar_arrive_expect_tx(&full[st], Cfg::STAGE);
                        tma_load_2d(sa, &tmA, &full[st], kb * 128, m0);
                        tma_load_2d(sa + Cfg::A_BYTES, &tmW, &full[st], kb * 128, n0);
                    }
                }
            }
            // Every load has landed before the CTA may end (on the error path too; a pair's barriers are the even CTA's,
            // which the cluster's last meeting keeps).
            if (!PAIR || lead)
                for (int x = max(0, loads - STAGES); x < loads; x++) mbar_drain(&full[x % STAGES], (x / STAGES) & 1, 200000000ull);
        }
    } else if (warp == 1) {
        if (lane == 0 && lead) {
            constexpr uint32_t idesc = i8_idesc(BM, BN);
            const uint64_t d0 = umma_desc_sw128(smem_u32(smem), 16, 1024);
            int taken = 0, local = 0;
            bool ok = true;
            for (int t = t_first; ok && t < tiles; t += t_step, local++) {
                const int acc = local & 1;
                if (!(ok = mbar_wait(&tempty[acc], ((local >> 1) & 1) ^ 1, EG2_DEV_TIMEOUT_GEMM, abort_flag))) break;
                tc_fence_after();
                for (int kb = 0; kb < kblocks; kb++, taken++) {
                    const int st = taken % STAGES;
                    if (!(ok = mbar_wait(&full[st], (taken / STAGES) & 1, EG2_DEV_TIMEOUT_GEMM, abort_flag))) break;
                    tc_fence_after();
                    const uint64_t ad = d0 + (uint64_t)(st * (Cfg::STAGE >> 4)), bd = ad + (uint64_t)(Cfg::A_BYTES >> 4);
#pragma unroll
                    for (int kk = 0; kk < 4; kk++) mma_i8<PAIR>(tmem + acc * BN, ad + 2 * kk, bd + 2 * kk, idesc, (kb | kk) != 0);
                    if constexpr (PAIR)
                        mma_commit_pair_both(&empty[st]);
                    else
                        mma_commit(&empty[st]);
                }
                if (!ok) break;
                if constexpr (PAIR)
                    mma_commit_pair_both(&tfull[acc]);
                else
                    mma_commit(&tfull[acc]);
            }
        }
    } else {
        const int w = warp - 2, set = w >> 2, e = warp & 3;
        uint8_t* slots = smem + Cfg::OFF_OUT + w * 4096;
        float* sc = reinterpret_cast<float*>(smem + Cfg::OFF_SC + w * 8 * BN);
        int local = 0, nst = 0;
        for (int t = t_first; t < tiles; t += t_step, local++) {
            if ((local & 1) != set) continue;
            const int row0 = (t / tiles_n) * BM + 128 * (int)rank + 32 * e, n0 = (t % tiles_n) * BN;
            const int row = row0 + lane;
            // Scales and biases of the tile's columns, requested before the sums are there.
            const float sa = row < p.M ? p.sa[row] : 0.f;
#pragma unroll
            for (int c = 0; c < BN; c += 32) {
                const int n = n0 + c + lane;
                sc[c + lane] = n < p.N ? p.sw[n] : 0.f;
                sc[BN + c + lane] = (p.bias && n < p.N) ? p.bias[n] : 0.f;
            }
            __syncwarp();
            if (!mbar_wait(&tfull[set], (local >> 1) & 1, EG2_DEV_TIMEOUT_GEMM, abort_flag)) break;
            tc_fence_after();
            const uint32_t base = tmem + set * BN + ((uint32_t)(32 * e) << 16);
            const int chunks = row0 < p.M ? min(BN / 32, (p.N - n0 + 31) / 32) : 0;
            auto chunk = [&](int c, uint32_t (&r)[32]) -> bool {
                float v[32];
#pragma unroll
                for (int q = 0; q < 32; q += 4) {
                    const float4 s4 = *reinterpret_cast<const float4*>(sc + 32 * c + q), b4 = *reinterpret_cast<const float4*>(sc + BN + 32 * c + q);
                    v[q] = fmaf((float)(int)r[q] * sa, s4.x, b4.x);
                    v[q + 1] = fmaf(i32_to_f32(r[q + 1]) * sa, s4.y, b4.y);
                    v[q + 2] = fmaf((float)(int)r[q + 2] * sa, s4.z, b4.z);
                    v[q + 3] = fmaf(i32_to_f32(r[q + 3]) * sa, s4.w, b4.w);
                }
                if (p.tma_out) {
                    if constexpr (sizeof(TO) == 2) {
                        tio_store32<2>(&tmC, slots, nst++, v, n0 + 32 * c, row0);
                    } else {
                        // 16 columns per 2 KB slot, 64-byte swizzle.
                        const uint32_t swz = (uint32_t)((lane >> 1) & 3);
#pragma unroll
                        for (int hh = 0; hh < 2; hh++, nst++) {
                            uint8_t* slot = slots + (nst & 1) * 2048;
                            if (lane == 0) bulk_wait_read<1>();
                            __syncwarp();
#pragma unroll
                            for (int q = 0; q < 4; q++)
                                *reinterpret_cast<float4*>(slot + lane * 64 + ((q ^ swz) << 4)) =
                                    make_float4(v[16 * hh + 4 * q], v[16 * hh + 4 * q + 1], v[16 * hh + 4 * q + 2], v[16 * hh + 4 * q + 3]);
                            fence_proxy_async();
                            __syncwarp();
                            if (lane == 0) {
                                if (n0 + 32 * c + 16 * hh < p.N) tma_store_2d(&tmC, slot, n0 + 32 * c + 16 * hh, row0);
                                bulk_commit();
                            }
                        }
                    }
                } else {
                    // 16 columns at a time through a padded tile, then lanes 0..15 and 16..31 write two rows' pieces.
                    float* tile = reinterpret_cast<float*>(slots);  // [32][17]
#pragma unroll
                    for (int hh = 0; hh < 2; hh++) {
#pragma unroll
                        for (int q = 0; q < 16; q++) tile[lane * 17 + q] = v[16 * hh + q];
                        __syncwarp();
                        const int n = n0 + 32 * c + 16 * hh + (lane & 15);
#pragma unroll 4
                        for (int rr = lane >> 4; rr < 32; rr += 2)
                            if (row0 + rr < p.M && n < p.N)
                                stf((TO*)p.C + (long)(row0 + rr) * p.ldc, n, tile[rr * 17 + (lane & 15)]);
                        __syncwarp();
                    }
                }
                return true;
            };
            if (chunks > 0) tmem_pipelined<32>(base, chunks, chunk);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR)
                    mbar_arrive_remote(mapa_shared(smem_u32(&tempty[set]), 0));
                else
                    mbar_arrive(&tempty[set]);
            }
        }
        if (lane == 0) bulk_wait_all();
        __syncwarp();
    }
    // Every MMA has completed before either CTA frees its TMEM.
    if (warp == 1 && lane == 0 && lead) {
        if constexpr (PAIR)
            mma_commit_pair(smem_u32(drain));
        else
            mma_commit(drain);
        mbar_wait(drain, 0, EG2_DEV_TIMEOUT_GEMM, nullptr);
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        if constexpr (PAIR)
            tmem_dealloc_pair(tmem, Cfg::TMEM_COLS);
        else
            tmem_dealloc(tmem, Cfg::TMEM_COLS);
    }
}

template <bool PAIR, typename TO>
static int launch_i8(const int8_t* A, long lda, const int8_t* W, long ldw, const I8Params& p, cudaStream_t s) {
    using Cfg = I8Cfg<PAIR>;
    auto kern = gemm_i8_tc_kernel<PAIR, TO>;
    static int clusters_max[64] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    int n_attr = 0;
    if (PAIR) {
        attr[n_attr].id = cudaLaunchAttributeClusterDimension;
        attr[n_attr].val.clusterDim.x = 2;
        attr[n_attr].val.clusterDim.y = 1;
        attr[n_attr++].val.clusterDim.z = 1;
    }
    cfg.blockDim = dim3(I8_THREADS, 1, 1);
    cfg.dynamicSmemBytes = Cfg::SMEM;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = n_attr;  // the occupancy query takes the cluster shape only
    if (!clusters_max[dev]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM) != cudaSuccess) return -3;
        int n = num_sms();
        cfg.gridDim = dim3(2 * num_sms(), 1, 1);
        if (PAIR && (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0)) return -3;
        clusters_max[dev] = n;
    }
    CUtensorMap ma, mw, mc;
    if (make_tmap_2d(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, A, p.K, p.M, lda, 128, 128) ||
        make_tmap_2d(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, W, p.K, p.N, ldw, 128, PAIR ? 128 : 64))
        return -1;
    constexpr bool F32 = sizeof(TO) == 4;
    mc = ma;  // unused without tma_out
    if (p.tma_out && make_tmap_2d(&mc, F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.C, p.N, p.M,
                                  p.ldc * sizeof(TO), F32 ? 16 : 32, 32, CU_TENSOR_MAP_SWIZZLE_64B))
        return -1;
    const long tiles = (((long)p.M + (PAIR ? 255 : 127)) / (PAIR ? 256 : 128)) * ((p.N + Cfg::BN - 1) / Cfg::BN);
    if (tiles > 0x7fffffffL) return -1;
    const int n = tiles < clusters_max[dev] ? (int)tiles : clusters_max[dev];
    cfg.gridDim = dim3((PAIR ? 2 : 1) * n, 1, 1);
    attr[n_attr].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n_attr].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = n_attr + (pdl_enabled() ? 1 : 0);
    return cudaLaunchKernelEx(&cfg, kern, ma, mw, mc, p) == cudaSuccess ? 0 : -3;
}

template <typename TO>
static int gemm_i8(const int8_t* A, long lda, const int8_t* W, long ldw, I8Params& p, cudaStream_t s) {
    p.tma_out = (uintptr_t)p.C % 16 == 0 && p.ldc * sizeof(TO) % 16 == 0;
    // Pairs where their 256 x 256 tiles fill at least half of the SM pairs.
    const long pair_tiles = (((long)p.M + 255) / 256) * ((p.N + 255) / 256);
    return pair_tiles >= num_sms() / 4 ? launch_i8<true, TO>(A, lda, W, ldw, p, s) : launch_i8<false, TO>(A, lda, W, ldw, p, s);
}

}  // namespace eg2

extern "C" {

int eg2_quantize_rows(int kind, const void* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t rows, int k,
                      void* stream) {
    if ((kind != EG2_F32 && kind != EG2_BF16) || rows < 0 || k <= 0 || ldx < k || ldq < k) return EG2_ERR_INVALID;
    if (rows == 0) return EG2_OK;
    if (!x || !q || !scale || rows >= (1L << 31)) return EG2_ERR_INVALID;
    cudaStream_t s = (cudaStream_t)stream;
    if (kind == EG2_F32 ? eg2::quantize_rows((const float*)x, ldx, q, ldq, scale, rows, k, s)
                        : eg2::quantize_rows((const bf16_t*)x, ldx, q, ldq, scale, rows, k, s))
        return EG2_ERR_CUDA;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return EG2_OK;
}

int eg2_gemm_i8(const int8_t* A, int64_t lda, const float* a_scale, const int8_t* W, int64_t ldw, const float* w_scale,
                const float* bias, void* C, int64_t ldc, int64_t M, int N, int K, int out_f32, void* stream) {
    if (M < 0 || N <= 0 || K <= 0 || K > EG2_I8_MAX_K || lda < K || ldw < K || ldc < N || lda % 16 || ldw % 16) return EG2_ERR_INVALID;
    if (M == 0) return EG2_OK;
    if (!A || !W || !a_scale || !w_scale || !C || M > (1L << 30) || ((uintptr_t)A | (uintptr_t)W) % 16) return EG2_ERR_INVALID;
    eg2::I8Params p{a_scale, w_scale, bias, C, ldc, (int)M, N, K, 0};
    const int rc = out_f32 ? eg2::gemm_i8<float>(A, lda, W, ldw, p, (cudaStream_t)stream)
                           : eg2::gemm_i8<bf16_t>(A, lda, W, ldw, p, (cudaStream_t)stream);
    if (rc == -1) return EG2_ERR_INVALID;
    if (rc) return EG2_ERR_CUDA;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return EG2_OK;
}

}  // extern "C"
