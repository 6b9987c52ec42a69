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

// One thread per (row, channel): pairs are handled by the thread of their first channel, channels past `rot`
// are copied.
template <typename T>
__global__ void rotary_kernel(const RotaryParams p, int half_layout) {
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

template <typename T>
static int rotary(const RotaryParams& p, int layout, cudaStream_t s) {
    const long items = p.rows * (p.rot / 2 + p.hd - p.rot);
    const long blocks = (items + 255) / 256;
    if (blocks > 0x7fffffffL) return -1;
    rotary_kernel<T><<<(unsigned)blocks, 256, 0, s>>>(p, layout == EG2_ROTARY_HALF);
    return cudaGetLastError() == cudaSuccess ? 0 : -3;
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
    if ((long)nh * hd > 0x7fffffffL || (long)nkv * hd > 0x7fffffffL || rows > (1L << 40) / hd) return EG2_ERR_INVALID;
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
