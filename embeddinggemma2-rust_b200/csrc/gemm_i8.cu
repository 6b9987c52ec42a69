// Matrix product in 8-bit integers with a scale per token and per output channel, and the row quantisation
// that feeds it (eg2_quantize_rows, eg2_gemm_i8 in include/eg2.h).
#include "common.cuh"
#include "kernels.h"

namespace eg2 {

// ---------------------------------------------------------------------------------------------
// q[r, c] = rint(x[r, c] * (127 / max_c |x[r, c]|)), scale[r] = max / 127, each operation one IEEE rounding; where 127 / max does not
// fit 32 bits (max below 3.74e-37) x and max are taken 2^100 times as large first, which is exact. A row
// of zeros gets scale 0; a row that holds a NaN or an infinity gets zeros and scale NaN, so every product with it
// is NaN. Bound by HBM: TPR threads hold a row in registers, reduce and write it, with the next row's loads already
// out (16,384 rows of 8,192 bf16, 402 MB: 71 to 85 us, 4.7 to 5.7 TB/s). The maximum is taken over the bits of |x|, which order like the numbers and put
// infinities and NaN above all.
// ---------------------------------------------------------------------------------------------
EG2_DEV uint32_t quant_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
struct QuantRow {
    float inv, scale;
    bool bad, tiny;  // tiny: inv is for QUANT_UP x
};
constexpr float QUANT_UP = 1.2676506002282294e30f;  // 2^100
EG2_DEV QuantRow quant_row(uint32_t top) {
    const float t = __uint_as_float(top);
    QuantRow q;
    q.bad = top >= 0x7f800000u;
    q.tiny = t < 3.74e-37f;
    q.inv = (q.bad || top == 0u) ? 0.f : __fdiv_rn(127.f, q.tiny ? t * QUANT_UP : t);
    q.scale = q.bad ? __int_as_float(0x7fc00000) : __fdiv_rn(t, 127.f);
    return q;
}
// rint(x * inv) in the low byte: adding 1.5 * 2^23 rounds to whole numbers, ties to even, and leaves them in the low bits of
// the mantissa (the conversion instruction runs at an eighth of the rate).
EG2_DEV uint32_t quant_one(float x, float inv) { return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.f)); }
EG2_DEV uint32_t quant_four(const float* v, float inv) {
    const uint32_t a = __byte_perm(quant_one(v[0], inv), quant_one(v[1], inv), 0x0040);
    const uint32_t b = __byte_perm(quant_one(v[2], inv), quant_one(v[3], inv), 0x0040);
    return __byte_perm(a, b, 0x5410);
}
// The maximum over the TPR threads of a row; slot: shared memory that the last call did not use.
template <int TPR>
EG2_DEV uint32_t quant_max(uint32_t top, uint32_t* slot) {
    top = __reduce_max_sync(0xffffffffu, top);
    if constexpr (TPR > 32) {
        if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TPR / 32; i++) top = max(top, slot[i]);
    }
    return top;
}

// Eight elements as they are in memory.
template <typename T>
struct Quant8 {
    uint4 u[sizeof(T) / 2];
    EG2_DEV void load(const T* p, int n) {  // n of them exist; p is 16-byte aligned
        if (n >= 8) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; i++) u[i] = reinterpret_cast<const uint4*>(p)[i];
        } else {
            uint32_t w[4 * sizeof(T) / 2] = {};
            for (int i = 0; i < n; i++) {
                if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(p[i]);
                else w[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
            }
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; i++) u[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        }
    }
    EG2_DEV uint32_t top() const {
        uint32_t r = 0;
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) {
            const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int y = 0; y < 4; y++) r = max(r, w[y] & 0x7fffffffu);
            } else {  // two 16-bit maxima side by side
#pragma unroll
                for (int y = 0; y < 4; y++) r = __vmaxu2(r, w[y] & 0x7fff7fffu);
            }
        }
        if constexpr (sizeof(T) == 2) r = max(r & 0xffff0000u, r << 16);
        return r;
    }
    EG2_DEV void up() {  // exact in either type
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) {
            uint32_t* w = reinterpret_cast<uint32_t*>(&u[i]);
#pragma unroll
            for (int y = 0; y < 4; y++) {
                if constexpr (sizeof(T) == 4)
                    w[y] = __float_as_uint(__uint_as_float(w[y]) * QUANT_UP);
                else
                    w[y] = bf16x2_bits(__uint_as_float(w[y] << 16) * QUANT_UP, __uint_as_float(w[y] & 0xffff0000u) * QUANT_UP);
            }
        }
    }
    EG2_DEV uint2 quant(float inv) const {
        float v[8];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) {
            const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
            for (int y = 0; y < 4; y++) {
                if constexpr (sizeof(T) == 4) {
                    v[4 * i + y] = __uint_as_float(w[y]);
                } else {
                    v[2 * y] = __uint_as_float(w[y] << 16);
                    v[2 * y + 1] = __uint_as_float(w[y] & 0xffff0000u);
                }
            }
        }
        return make_uint2(quant_four(v, inv), quant_four(v + 4, inv));
    }
};

template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR)
    quantize_rows_kernel(const T* __restrict__ x, long ldx, int8_t* __restrict__ q, long ldq, float* __restrict__ scale,
                         long rows, int k) {
    grid_dep_launch();
    grid_dep_wait();
    __shared__ uint32_t slots[2][TPR / 32];
    const int t = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
    const long step = TPR == 32 ? (long)gridDim.x * 4 : (long)gridDim.x;
    Quant8<T> now[NV], next[NV];
    auto load = [&](Quant8<T> (&v)[NV], long row) {
#pragma unroll
        for (int i = 0; i < NV; i++) v[i].load(x + row * ldx + 8l * (t + i * TPR), k - 8 * (t + i * TPR));
    };
    long row = TPR == 32 ? (long)blockIdx.x * 4 + (threadIdx.x >> 5) : (long)blockIdx.x;
    if (row < rows) load(now, row);
    for (int n = 0; row < rows; row += step, n++) {
        if (row + step < rows) load(next, row + step);
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < NV; i++) top = max(top, now[i].top());
        const QuantRow qr = quant_row(quant_max<TPR>(top, slots[n & 1]));
        if (qr.tiny) {
#pragma unroll
            for (int i = 0; i < NV; i++) now[i].up();
        }
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = 8 * (t + i * TPR);
            if (c >= k) continue;
            const uint2 u = qr.bad ? make_uint2(0u, 0u) : now[i].quant(qr.inv);
            int8_t* to = q + row * ldq + c;
            if (c + 8 <= k) {
                *reinterpret_cast<uint2*>(to) = u;
            } else {
                for (int y = 0; c + y < k; y++) to[y] = (int8_t)((y < 4 ? u.x : u.y) >> (8 * (y & 3)));
            }
        }
        if (t == 0) scale[row] = qr.scale;
#pragma unroll
        for (int i = 0; i < NV; i++) now[i] = next[i];
    }
}

// Any alignment: TPR threads hold up to 32 single elements each (16,384 x 8,192 bf16: 254 us, 85 by 16-byte units on the same box).
template <typename T, int TPR>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR)
    quantize_rows_any_kernel(const T* __restrict__ x, long ldx, int8_t* __restrict__ q, long ldq, float* __restrict__ scale,
                             long rows, int k) {
    grid_dep_launch();
    grid_dep_wait();
    __shared__ uint32_t slot[TPR / 32];
    const long row = TPR == 32 ? (long)blockIdx.x * 4 + (threadIdx.x >> 5) : (long)blockIdx.x;
    if (row >= rows) return;
    const int t = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
    const T* xr = x + row * ldx;
    float v[32];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = t + i * TPR < k ? ldf(xr, t + i * TPR) : 0.f;
#pragma unroll
    for (int i = 0; i < 32; i++) top = max(top, quant_bits(v[i]));
    const QuantRow qr = quant_row(quant_max<TPR>(top, slot));
    if (qr.tiny) {
#pragma unroll
        for (int i = 0; i < 32; i++) v[i] *= QUANT_UP;
    }
#pragma unroll
    for (int i = 0; i < 32; i++)
        if (t + i * TPR < k) q[row * ldq + t + i * TPR] = qr.bad ? (int8_t)0 : (int8_t)(quant_one(v[i], qr.inv) & 0xff);
    if (t == 0) scale[row] = qr.scale;
}

// Longer rows: a block per row, two passes over it (the second from L2). Columns are unsigned: k may be 2^31 - 1, and c ends above it.
template <typename T>
__global__ void __launch_bounds__(512) quantize_rows_long_kernel(const T* __restrict__ x, long ldx, int8_t* __restrict__ q,
                                                                 long ldq, float* __restrict__ scale, int k) {
    grid_dep_launch();
    grid_dep_wait();
    __shared__ uint32_t slot[16];
    const long row = blockIdx.x;
    const T* xr = x + row * ldx;
    uint32_t top = 0;
#pragma unroll 4
    for (unsigned c = threadIdx.x; c < (unsigned)k; c += 512) top = max(top, quant_bits(ldf(xr, c)));
    const QuantRow qr = quant_row(quant_max<512>(top, slot));
    if (qr.tiny) {
        for (unsigned c = threadIdx.x; c < (unsigned)k; c += 512) q[row * ldq + c] = (int8_t)(quant_one(ldf(xr, c) * QUANT_UP, qr.inv) & 0xff);
    } else {
#pragma unroll 4
        for (unsigned c = threadIdx.x; c < (unsigned)k; c += 512) q[row * ldq + c] = qr.bad ? (int8_t)0 : (int8_t)(quant_one(ldf(xr, c), qr.inv) & 0xff);
    }
    if (threadIdx.x == 0) scale[row] = qr.scale;
}

template <typename T>
static int quantize_rows(const T* x, long ldx, int8_t* q, long ldq, float* scale, long rows, int k, cudaStream_t s) {
    const bool vec = (uintptr_t)x % 16 == 0 && ldx * sizeof(T) % 16 == 0 && (uintptr_t)q % 8 == 0 && ldq % 8 == 0;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    auto run = [&](auto kern, int tpr, bool walk, auto... args) {
        // Walking kernels: as many threads as are resident, 1,024 to 2,048 an SM by their registers.
        const long units = tpr == 32 ? (rows + 3) / 4 : rows, most = (long)num_sms() * 2048 / (tpr == 32 ? 128 : tpr);
        cfg.gridDim = dim3((unsigned)(walk && units > most ? most : units), 1, 1);
        cfg.blockDim = dim3(tpr == 32 ? 128 : tpr, 1, 1);
        return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? 0 : -3;
    };
    if (vec && k <= 256) return run(quantize_rows_kernel<T, 32, 1>, 32, true, x, ldx, q, ldq, scale, rows, k);
    if (vec && k <= 512) return run(quantize_rows_kernel<T, 32, 2>, 32, true, x, ldx, q, ldq, scale, rows, k);
    if (vec && k <= 1024) return run(quantize_rows_kernel<T, 32, 4>, 32, true, x, ldx, q, ldq, scale, rows, k);
    if (vec && k <= 2048) return run(quantize_rows_kernel<T, 128, 2>, 128, true, x, ldx, q, ldq, scale, rows, k);
    if (vec && k <= 4096) return run(quantize_rows_kernel<T, 256, 2>, 256, true, x, ldx, q, ldq, scale, rows, k);
    if (vec && k <= 8192) return run(quantize_rows_kernel<T, 256, 4>, 256, true, x, ldx, q, ldq, scale, rows, k);
    if (vec && k <= 16384) return run(quantize_rows_kernel<T, 512, 4>, 512, true, x, ldx, q, ldq, scale, rows, k);
    if (k <= 1024) return run(quantize_rows_any_kernel<T, 32>, 32, false, x, ldx, q, ldq, scale, rows, k);
    if (k <= 4096) return run(quantize_rows_any_kernel<T, 128>, 128, false, x, ldx, q, ldq, scale, rows, k);
    if (k <= 16384) return run(quantize_rows_any_kernel<T, 512>, 512, false, x, ldx, q, ldq, scale, rows, k);
    return run(quantize_rows_long_kernel<T>, 512, false, x, ldx, q, ldq, scale, k);
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
// The result passes through a staging tile per warp, 128 bytes of a row at a time, so that every store writes whole
// lines (35,328 x 4,096 x 512 to bf16: 102 us, 111 with TMA stores of 64-byte rows; writing alone runs at 3.9 TB/s).
// Tiles are taken in panels of columns whose weights stay in L2 while the rows go by. Integer sums do not depend on
// their order, so a single CTA begins its K range at a place of its own: weights with rows of a large power of two
// bytes would otherwise be read at the same few memory channels by all CTAs at once.
// ---------------------------------------------------------------------------------------------
constexpr int I8_THREADS = 320;
template <bool PAIR>
struct I8Cfg {
    static constexpr int BN = PAIR ? 256 : 64;
    static constexpr int A_BYTES = 128 * 128;
    static constexpr int B_BYTES = PAIR ? 128 * 128 : 64 * 128;
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGES = PAIR ? 5 : 6;
    static constexpr int OFF_OUT = STAGES * STAGE;          // per epilogue warp: 32 rows of 128 + 16 bytes
    static constexpr int OFF_SC = OFF_OUT + 8 * 32 * 144;      // per epilogue warp: the tile's scales and biases
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

struct I8Params {
    const float *sa, *sw, *bias;
    void* C;
    long ldc;
    int M, N, K;
    int panel;    // column tiles per panel of the tile order
    int aligned;  // rows of C start at multiples of 16 bytes
};

template <bool PAIR, typename TO>
__global__ void __launch_bounds__(I8_THREADS, 1)
    gemm_i8_tc_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                      const I8Params p) {
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
    const int kblocks = (p.K + 127) / 128, tiles_m = (p.M + BM - 1) / BM;
    // Tile t: panels of p.panel column tiles, rows within a panel, columns within a row.
    auto place = [&](int t, int& m0, int& n0) {
        const int per = tiles_m * p.panel, pan = t / per, left = t - pan * per;
        const int width = min(p.panel, tiles_n - pan * p.panel);
        m0 = (left / width) * BM + 128 * (int)rank;
        n0 = (pan * p.panel + left % width) * BN;
    };

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
                int m0, n0;
                place(t, m0, n0);
                if (PAIR) n0 += 128 * (int)rank;
                int kb = PAIR ? 0 : (int)((unsigned)(n0 / BN) * 13u % (unsigned)kblocks);
                for (int i = 0; i < kblocks; i++, loads++, kb = kb + 1 == kblocks ? 0 : kb + 1) {
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
        uint8_t* stage = smem + Cfg::OFF_OUT + w * 32 * 144;
        float* sc = reinterpret_cast<float*>(smem + Cfg::OFF_SC + w * 8 * BN);
        int local = 0;
        for (int t = t_first; t < tiles; t += t_step, local++) {
            if ((local & 1) != set) continue;
            int row0, n0;
            place(t, row0, n0);
            row0 += 32 * e;
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
            constexpr int COLS = 128 / (int)sizeof(TO);  // columns of a staged row: two chunks of bf16, one of f32
            TO* out = (TO*)p.C + (long)row0 * p.ldc + n0;
            const int rows = min(32, p.M - row0);
            auto chunk = [&](int c, uint32_t (&r)[32]) -> bool {
                // A sum of the most columns, all -128 on both sides, is 2^31 and wraps to the one value that no other sum has; the
                // number below it in 32 bits, 2^31 - 1, becomes 2^31 as f32.
                if (p.K == EG2_I8_MAX_K) {
#pragma unroll
                    for (int q = 0; q < 32; q++) r[q] -= r[q] == 0x80000000u;
                }
                uint8_t* mine = stage + lane * 144 + (sizeof(TO) == 2 ? (c & 1) * 64 : 0);
#pragma unroll
                for (int q = 0; q < 32; q += 8) {
                    float v[8];
#pragma unroll
                    for (int y = 0; y < 8; y += 4) {
                        const float4 s4 = *reinterpret_cast<const float4*>(sc + 32 * c + q + y);
                        const float4 b4 = *reinterpret_cast<const float4*>(sc + BN + 32 * c + q + y);
                        v[y] = fmaf((float)(int)r[q + y] * sa, s4.x, b4.x);
                        v[y + 1] = fmaf((float)(int)r[q + y + 1] * sa, s4.y, b4.y);
                        v[y + 2] = fmaf((float)(int)r[q + y + 2] * sa, s4.z, b4.z);
                        v[y + 3] = fmaf((float)(int)r[q + y + 3] * sa, s4.w, b4.w);
                    }
                    if constexpr (sizeof(TO) == 2) {
                        *reinterpret_cast<uint4*>(mine + 2 * q) = make_uint4(bf16x2_bits(v[0], v[1]), bf16x2_bits(v[2], v[3]),
                                                                             bf16x2_bits(v[4], v[5]), bf16x2_bits(v[6], v[7]));
                    } else {
                        *reinterpret_cast<float4*>(mine + 4 * q) = make_float4(v[0], v[1], v[2], v[3]);
                        *reinterpret_cast<float4*>(mine + 4 * q + 16) = make_float4(v[4], v[5], v[6], v[7]);
                    }
                }
                if (sizeof(TO) == 2 && !(c & 1) && c + 1 < chunks) return true;
                __syncwarp();
                const int first = sizeof(TO) == 2 ? 32 * (c & ~1) : 32 * c;  // the staged columns start here in the tile
                const int width = min(p.N - n0 - first, COLS);
                if (p.aligned && width == COLS && (sizeof(TO) == 4 || (c & 1))) {
                    // 8 lanes a row, 4 rows an instruction: whole 128-byte pieces.
                    const int at = (lane & 7) * 16;
#pragma unroll
                    for (int y = 0; y < 8; y++) {
                        const int rr = 4 * y + (lane >> 3);
                        const uint4 x = *reinterpret_cast<const uint4*>(stage + rr * 144 + at);
                        if (rr < rows) *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(out + (long)rr * p.ldc + first) + at) = x;
                    }
                } else {
                    for (int rr = 0; rr < rows; rr++)
                        for (int y = lane; y < width; y += 32)
                            out[(long)rr * p.ldc + first + y] = reinterpret_cast<const TO*>(stage + rr * 144)[y];
                }
                __syncwarp();
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
static int launch_i8(const int8_t* A, long lda, const int8_t* W, long ldw, I8Params p, cudaStream_t s) {
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
    CUtensorMap ma, mw;
    if (make_tmap_2d(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, A, p.K, p.M, lda, 128, 128) ||
        make_tmap_2d(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, W, p.K, p.N, ldw, 128, PAIR ? 128 : 64))
        return -1;
    const long tiles = (((long)p.M + (PAIR ? 255 : 127)) / (PAIR ? 256 : 128)) * ((p.N + Cfg::BN - 1) / Cfg::BN);
    if (tiles > 0x7fffffffL) return -1;
    // 24 MB of weights per panel: a fifth of L2, which also holds the rows passing by (16,384 x 8,192 x 8,192: 673 us, 721 in one
    // panel; 8,192 x 16,384 x 8,192: 775 and 1,013; 12 to 48 MB are within the 10 % that runs at the power limit differ by).
    const long per_panel = (24L << 20) / ((long)Cfg::BN * p.K);
    const long tiles_n = ((long)p.N + Cfg::BN - 1) / Cfg::BN;
    p.panel = per_panel < 1 ? 1 : per_panel > tiles_n ? (int)tiles_n : (int)per_panel;
    const int n = tiles < clusters_max[dev] ? (int)tiles : clusters_max[dev];
    cfg.gridDim = dim3((PAIR ? 2 : 1) * n, 1, 1);
    attr[n_attr].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n_attr].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = n_attr + (pdl_enabled() ? 1 : 0);
    return cudaLaunchKernelEx(&cfg, kern, ma, mw, p) == cudaSuccess ? 0 : -3;
}

template <typename TO>
static int gemm_i8(const int8_t* A, long lda, const int8_t* W, long ldw, I8Params& p, cudaStream_t s) {
    p.aligned = (uintptr_t)p.C % 16 == 0 && p.ldc * sizeof(TO) % 16 == 0;
    // Pairs where their 256 x 256 tiles fill at least half of the SM pairs (pairs / single CTAs: 2,208 x 2,048 x 512, 72 tiles,
    // 7.8 / 9.7 us; 300 x 8,192 x 8,192, 64 tiles, 26 / 59; 1,024 x 2,048 x 512, 32 tiles, 6.9 / 6.2; 17 x 2,048 x 512 6.4 / 4.1).
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
    if (M < 0 || M > (1L << 30) || N <= 0 || N > (1 << 30) || K <= 0 || K > EG2_I8_MAX_K) return EG2_ERR_INVALID;
    if (lda < K || ldw < K || ldc < N || lda % 16 || ldw % 16) return EG2_ERR_INVALID;
    if (M == 0) return EG2_OK;
    if (!A || !W || !a_scale || !w_scale || !C || ((uintptr_t)A | (uintptr_t)W) % 16) return EG2_ERR_INVALID;
    eg2::I8Params p{a_scale, w_scale, bias, C, ldc, (int)M, N, K, 0, 0};
    const int rc = out_f32 ? eg2::gemm_i8<float>(A, lda, W, ldw, p, (cudaStream_t)stream)
                           : eg2::gemm_i8<bf16_t>(A, lda, W, ldw, p, (cudaStream_t)stream);
    if (rc == -1) return EG2_ERR_INVALID;
    if (rc) return EG2_ERR_CUDA;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return EG2_OK;
}

}  // extern "C"
