// Rotary positions of q and k in one call (eg2_rotary in include/eg2.h).
//
// A pair (a, b) of channels at position p becomes m (a cos t - b sin t, b cos t + a sin t), t = p f for the
// pair's frequency f and a factor m common to all. t is needed modulo a full turn only, so f comes as a 64-bit
// whole number of 2^-64 turns: the product with the position wraps at full turns exactly, and its top 32 bits
// are the reduced angle to 2^-32 of a turn at any position (an f32 product p f is off by 0.008 rad at
// p = 131,072).
//
// Bound by HBM: every channel is read and written once, the angle is computed once per (row, pair) and used for
// all heads of q and k.
#include "common.cuh"
#include "kernels.h"

#include <cmath>

namespace eg2 {

struct RotaryParams {
    const void *q, *k;
    void *qo, *ko;
    long ldq, ldk, ldqo, ldko;
    const int* pos;
    const unsigned long long* steps;
    long rows;
    int nh, nkv, hd, rot, inverse;
    float magnitude;
};

EG2_DEV void rotary_angle(int pos, unsigned long long step, float magnitude, float& s, float& c) {
    const unsigned long long phase = (unsigned long long)(long long)pos * step;
    sincospif((float)(int)(phase >> 32) * 4.656612873077393e-10f, &s, &c);  // 2^-31: half turns
    s *= magnitude;
    c *= magnitude;
}

// Any alignment: one thread per (row, pair), then per channel past `rot`, which is copied.
template <typename T>
__global__ void rotary_any_kernel(const RotaryParams p, int half_layout) {
    grid_dep_launch();
    grid_dep_wait();
    const int half = p.rot / 2, items = half + (p.hd - p.rot);
    const long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
    const long row = i / items;
    if (row >= p.rows) return;
    const int c = (int)(i - row * items);
    const bool copy = c >= half;
    const int a = copy ? p.rot + c - half : half_layout ? c : 2 * c;
    const int b = half_layout ? a + half : a + 1;
    float sn = 0.f, cs = 1.f;
    if (!copy) {
        rotary_angle(p.pos[row], p.steps[c], p.magnitude, sn, cs);
        if (p.inverse) sn = -sn;
    }
    for (int h = 0; h < p.nh + p.nkv; h++) {
        const bool isq = h < p.nh;
        const T* x = isq ? (const T*)p.q + row * p.ldq + (long)h * p.hd : (const T*)p.k + row * p.ldk + (long)(h - p.nh) * p.hd;
        T* y = isq ? (T*)p.qo + row * p.ldqo + (long)h * p.hd : (T*)p.ko + row * p.ldko + (long)(h - p.nh) * p.hd;
        if (copy) {
            y[a] = x[a];
        } else {
            const float u = ldf(x, a), v = ldf(x, b);
            stf(y, a, u * cs - v * sn);
            stf(y, b, v * cs + u * sn);
        }
    }
}

// 16 bytes of T as f32, and back.
template <typename T>
struct RotVec;
template <>
struct RotVec<float> {
    static constexpr int N = 4;
    EG2_DEV static void get(const uint4& u, float (&v)[4]) {
        v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
    }
    EG2_DEV static uint4 put(const float (&v)[4]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};
template <>
struct RotVec<bf16_t> {
    static constexpr int N = 8;
    EG2_DEV static void get(const uint4& u, float (&v)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    EG2_DEV static uint4 put(const float (&v)[8]) {
        return make_uint4(bf16x2_bits(v[0], v[1]), bf16x2_bits(v[2], v[3]), bf16x2_bits(v[4], v[5]), bf16x2_bits(v[6], v[7]));
    }
};

// 16-byte loads and stores. One thread takes two units of 16 bytes of a row in every head: in the half layout unit c and
// its partner rot / 2 further on, in the interleaved one units 2 c and 2 c + 1, past `rot` two units to copy. The loads of
// up to four heads are in flight together (131,071 rows of 12 + 12 heads of 64, f32: 257 us, 6.3 TB/s).
template <typename T, bool HALF>
__global__ void __launch_bounds__(256) rotary_vec_kernel(const RotaryParams p) {
    using V = RotVec<T>;
    constexpr int N = V::N, PAIRS = HALF ? N : N / 2;  // pairs per unit
    grid_dep_launch();
    grid_dep_wait();
    const int turn = HALF ? p.rot / (2 * N) : (p.rot / N + 1) / 2, rest = (p.hd - p.rot) / N;
    const unsigned items = turn + (rest + 1) / 2;
    const long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
    long row;
    int c;
    if (p.rows * (long)items < (1L << 31)) {
        row = (unsigned)i / items;
        c = (int)((unsigned)i % items);
    } else {
        row = i / items;
        c = (int)(i % items);
    }
    if (row >= p.rows) return;
    const bool copy = c >= turn;
    // This thread's units; the second may be missing at the end of an odd count.
    const int a = copy ? p.rot + 2 * N * (c - turn) : HALF ? N * c : 2 * N * c;
    const int b = copy || !HALF ? a + N : a + p.rot / 2;
    const bool two = copy ? b < p.hd : HALF || b < p.rot;
    float sn[N], cs[N];  // HALF: of the unit's N pairs; else of the N / 2 pairs of either unit
    if (!copy) {
        const int pos = p.pos[row];
        const int first = N * c;  // two units of N / 2 pairs, or one of N
#pragma unroll
        for (int y = 0; y < N; y++) {
            sn[y] = 0.f, cs[y] = 1.f;
            if (HALF || y < PAIRS || two) {
                rotary_angle(pos, p.steps[first + y], p.magnitude, sn[y], cs[y]);
                if (p.inverse) sn[y] = -sn[y];
            }
        }
    }
    const int heads = p.nh + p.nkv;
    auto src = [&](int h) {
        return h < p.nh ? (const T*)p.q + row * p.ldq + (long)h * p.hd : (const T*)p.k + row * p.ldk + (long)(h - p.nh) * p.hd;
    };
    auto dst = [&](int h) {
        return h < p.nh ? (T*)p.qo + row * p.ldqo + (long)h * p.hd : (T*)p.ko + row * p.ldko + (long)(h - p.nh) * p.hd;
    };
    for (int h0 = 0; h0 < heads; h0 += 4) {
        uint4 u[4], v[4];
#pragma unroll
        for (int y = 0; y < 4; y++) {
            if (h0 + y < heads) {
                const T* x = src(h0 + y);
                u[y] = *reinterpret_cast<const uint4*>(x + a);
                if (two) v[y] = *reinterpret_cast<const uint4*>(x + b);
            }
        }
#pragma unroll
        for (int y = 0; y < 4; y++) {
            if (h0 + y >= heads) break;
            if (!copy) {
                float f[N], g[N];
                V::get(u[y], f);
                if (two) V::get(v[y], g);
                if constexpr (HALF) {
#pragma unroll
                    for (int z = 0; z < N; z++) {
                        const float x0 = f[z], x1 = g[z];
                        f[z] = x0 * cs[z] - x1 * sn[z];
                        g[z] = x1 * cs[z] + x0 * sn[z];
                    }
                } else {
#pragma unroll
                    for (int z = 0; z < PAIRS; z++) {
                        float x0 = f[2 * z], x1 = f[2 * z + 1];
                        f[2 * z] = x0 * cs[z] - x1 * sn[z];
                        f[2 * z + 1] = x1 * cs[z] + x0 * sn[z];
                        if (two) {
                            x0 = g[2 * z], x1 = g[2 * z + 1];
                            g[2 * z] = x0 * cs[PAIRS + z] - x1 * sn[PAIRS + z];
                            g[2 * z + 1] = x1 * cs[PAIRS + z] + x0 * sn[PAIRS + z];
                        }
                    }
                }
                u[y] = V::put(f);
                if (two) v[y] = V::put(g);
            }
            T* to = dst(h0 + y);
            *reinterpret_cast<uint4*>(to + a) = u[y];
            if (two) *reinterpret_cast<uint4*>(to + b) = v[y];
        }
    }
}

// The vector form takes whole 16-byte units: heads, the rotated part (its halves in the half layout), row strides and
// pointers in multiples of them (35,328 rows of 4 + 1 heads of 512, bf16: 64 us, 163 channel by channel).
template <typename T>
static int rotary(const RotaryParams& p, int layout, cudaStream_t s) {
    constexpr int N = RotVec<T>::N;
    const bool half = layout == EG2_ROTARY_HALF;
    const uintptr_t at = (p.nh ? (uintptr_t)p.q | (uintptr_t)p.qo : 0) | (p.nkv ? (uintptr_t)p.k | (uintptr_t)p.ko : 0);
    const long ld = (p.nh ? p.ldq | p.ldqo : 0) | (p.nkv ? p.ldk | p.ldko : 0);
    const bool vec = at % 16 == 0 && (ld | p.hd) % N == 0 && p.rot % (half ? 2 * N : N) == 0;
    const long per_row = vec ? (half ? p.rot / (2 * N) : (p.rot / N + 1) / 2) + ((p.hd - p.rot) / N + 1) / 2 : p.rot / 2 + p.hd - p.rot;
    const long blocks = (p.rows * per_row + 255) / 256;
    if (blocks > 0x7fffffffL) return -1;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)blocks, 1, 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    const cudaError_t e = !vec ? cudaLaunchKernelEx(&cfg, rotary_any_kernel<T>, p, (int)half)
                          : half ? cudaLaunchKernelEx(&cfg, rotary_vec_kernel<T, true>, p) : cudaLaunchKernelEx(&cfg, rotary_vec_kernel<T, false>, p);
    return e == cudaSuccess ? 0 : -3;
}

}  // namespace eg2

extern "C" {

int eg2_rotary_steps(int rot_dim, double theta, int scaling, double factor, double original_len, uint64_t* steps,
                     float* magnitude) {
    if (!steps || !magnitude || rot_dim <= 0 || rot_dim % 2 || !(theta > 1.0) || !std::isfinite(theta)) return EG2_ERR_INVALID;
    if (scaling < EG2_SCALING_NONE || scaling > EG2_SCALING_YARN) return EG2_ERR_INVALID;
    if (scaling != EG2_SCALING_NONE && (!(factor >= 1.0) || !std::isfinite(factor))) return EG2_ERR_INVALID;
    if (scaling == EG2_SCALING_YARN && (!(original_len >= 1.0) || !std::isfinite(original_len))) return EG2_ERR_INVALID;
    const double two_pi = 6.283185307179586476925286766559;
    const int half = rot_dim / 2;
    *magnitude = 1.f;
    if (scaling == EG2_SCALING_NTK) theta *= std::pow(factor, (double)rot_dim / (rot_dim > 2 ? rot_dim - 2 : 1));
    double low = 0, high = 0;
    if (scaling == EG2_SCALING_YARN) {
        // The pair that turns `t` times over the original length.
        auto pair = [&](double t) { return rot_dim * std::log(original_len / (t * two_pi)) / (2.0 * std::log(theta)); };
        low = std::fmax(0.0, std::floor(pair(32.0)));
        high = std::fmin(rot_dim - 1.0, std::ceil(pair(1.0)));
        *magnitude = (float)(0.1 * std::log(factor) + 1.0);
    }
    for (int i = 0; i < half; i++) {
        double f = std::pow(theta, -2.0 * i / rot_dim);
        if (scaling == EG2_SCALING_LINEAR) f /= factor;
        if (scaling == EG2_SCALING_YARN) {
            const double r = std::fmin(1.0, std::fmax(0.0, (i - low) / std::fmax(high - low, 0.001)));
            f = f * (1.0 - r) + f / factor * r;
        }
        steps[i] = (uint64_t)std::nearbyint(std::ldexp(f / two_pi, 64));
    }
    return EG2_OK;
}

int eg2_rotary(int kind, int layout, int inverse, const void* q, int64_t ldq, int nh, const void* k, int64_t ldk, int nkv,
               void* q_out, int64_t ldqo, void* k_out, int64_t ldko, const int32_t* pos, int64_t rows, int hd, int rot_dim,
               const uint64_t* steps, float magnitude, void* stream) {
    if (kind != EG2_F32 && kind != EG2_BF16) return EG2_ERR_INVALID;
    if (layout != EG2_ROTARY_HALF && layout != EG2_ROTARY_INTERLEAVED) return EG2_ERR_INVALID;
    if (rows < 0 || nh < 0 || nkv < 0 || nh + nkv <= 0 || hd <= 0 || rot_dim <= 0 || rot_dim > hd || rot_dim % 2)
        return EG2_ERR_INVALID;
    // A channel's number and a few units of 16 bytes stay below 2^31.
    if (hd > (1 << 30) || (long)nh * hd > 0x7fffffffL || (long)nkv * hd > 0x7fffffffL || rows > (1L << 40) / hd) return EG2_ERR_INVALID;
    if (nh && (!q || !q_out || ldq < (long)nh * hd || ldqo < (long)nh * hd)) return EG2_ERR_INVALID;
    if (nkv && (!k || !k_out || ldk < (long)nkv * hd || ldko < (long)nkv * hd)) return EG2_ERR_INVALID;
    if (rows == 0) return EG2_OK;
    if (!pos || !steps) return EG2_ERR_INVALID;
    RotaryParams p{q, k, q_out, k_out, ldq, ldk, ldqo, ldko, pos, (const unsigned long long*)steps, rows, nh, nkv, hd, rot_dim,
                   inverse != 0, magnitude};
    const int rc = kind == EG2_F32 ? rotary<float>(p, layout, (cudaStream_t)stream) : rotary<bf16_t>(p, layout, (cudaStream_t)stream);
    if (rc == -1) return EG2_ERR_INVALID;
    if (rc) return EG2_ERR_CUDA;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return EG2_OK;
}

}  // extern "C"
