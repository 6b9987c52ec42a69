// Attention with capped and biased scores under document, prefix, causal and window masks
// (eg2_attention_masked in include/eg2.h).
//
//   x(i, j) = cap * tanh(scale * q_i . k_j / cap)  (or scale * q_i . k_j)  + bias(j - i)
//   out_i   = sum_j softmax_j(x(i, j)) v_j over the keys j that i may see,  lse_i = log sum_j exp x(i, j)
//
// i and j are places within the sequence; the queries are its last places. What i may see is an interval
// [lo, hi) of keys -- the window and the causal or prefix bound -- less the keys of other documents and those with a
// bias of -infinity. A row that sees nothing gets out = 0, lse = -inf. Keys that a row may not see contribute nothing whatever they hold.
#include "common.cuh"
#include "kernels.h"

#include <climits>
#include <cmath>
#include <type_traits>

namespace eg2 {

struct MaskedParams {
    const void *q, *k, *v;
    void* out;
    float* lse;
    long ldq, ldk, ldv, ldo;
    const int *q_off, *k_off, *prefix, *q_doc, *k_doc;
    const float *slopes, *table;
    long q_rows, k_rows;
    int n_seq, max_q, max_k, nh, nkv, hd, G, window, causal, radius;
    int nsplit, part;  // the key axis in nsplit parts of `part` key tiles each
    float scale, softcap;
    float* part_o;   // nsplit > 1: [nsplit][q_rows][nh][hd]
    float2* part_ml; // and [nsplit][q_rows][nh]: a part's maximum and its sum in units of that
    int log2_parts;  // maxima in the log2 domain (the forms for bf16)
};

// One sequence: its rows, clamped to the buffers and to the stated maxima whatever the offsets hold.
struct MaskedSeq {
    long q0, k0;
    int nq, nk, prefix;
};
EG2_DEV MaskedSeq masked_seq(const MaskedParams& p, int b) {
    MaskedSeq s;
    auto bound = [](long x, long lo, long hi) { return x < lo ? lo : x > hi ? hi : x; };
    s.q0 = bound(p.q_off[b], 0, p.q_rows);
    s.k0 = bound(p.k_off[b], 0, p.k_rows);
    s.nq = (int)min(bound(p.q_off[b + 1], s.q0, p.q_rows) - s.q0, (long)p.max_q);
    s.nk = (int)min(bound(p.k_off[b + 1], s.k0, p.k_rows) - s.k0, (long)p.max_k);
    s.prefix = p.prefix ? p.prefix[b] : 0;
    return s;
}
// Keys [lo, hi) of the query at place i (before the document mask).
EG2_DEV void masked_range(const MaskedParams& p, const MaskedSeq& s, int i, int& lo, int& hi) {
    lo = 0;
    hi = s.nk;
    if (p.window >= 0) {
        // In 64 bits on both sides: places of queries beyond the keys are negative, windows any int.
        lo = (int)max(0l, (long)i - p.window);
        hi = min(hi, (int)min((long)i + p.window + 1, (long)s.nk));
    }
    if (p.causal) hi = min(hi, max(i + 1, s.prefix));
}

// A distance bias as it is used: finite ones are at least -1e30, so that a row whose keys all have the type's lowest value
// keeps its softmax (the log2 domain of the tensor-core form would overflow). -infinity is a mask: it is not added but tested,
// since a key that it hides may have a score that is not finite.
EG2_DEV float masked_bias(float b) { return b < -1e30f && b > -INFINITY ? -1e30f : b; }
EG2_DEV float masked_table(const MaskedParams& p, int head, int apart) {
    return masked_bias(p.table[(long)head * (2 * p.radius + 1) + p.radius + min(max(apart, -p.radius), p.radius)]);
}

// ---------------------------------------------------------------------------------------------
// CUDA cores, f32 arithmetic. A block takes 16 RPT rows (row r = token r / G, head r % G of the K/V head's G
// query heads) and walks 64-key tiles; thread (ty, tx) holds RPT x 4 scores and RPT x 4 channels of each
// 64-channel chunk of the output. K and V pass through shared memory in chunks of 64 keys x 64 channels, the
// next chunk's loads in flight (in registers) while one is used. For f32, and for bf16 that TMA cannot address.
// Bound by the shared-memory reads that feed the FMAs (4,096 tokens, 4 heads over 1 of 128, f32: 1.47 ms,
// 23 TFLOP/s), in small calls by the latency of few tiles.
// ---------------------------------------------------------------------------------------------
constexpr int AMS_LD = 68;  // floats per staged row: 16-byte units of neighbouring rows in different banks

template <typename T>
EG2_DEV float4 ams_load4(const T* p, int n, bool vec) {  // n valid elements
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
    if (n >= 4 && vec) {
        if constexpr (sizeof(T) == 4) {
            r = *reinterpret_cast<const float4*>(p);
        } else {
            const uint2 u = *reinterpret_cast<const uint2*>(p);
            r = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                            __uint_as_float(u.y & 0xffff0000u));
        }
    } else {
        if (n > 0) r.x = ldf(p, 0);
        if (n > 1) r.y = ldf(p, 1);
        if (n > 2) r.z = ldf(p, 2);
        if (n > 3) r.w = ldf(p, 3);
    }
    return r;
}

template <typename T, int NCH, int RPT>
__global__ void __launch_bounds__(256, RPT == 2 && NCH <= 4 ? 2 : 1) attention_masked_simt_kernel(const MaskedParams p, int q_tiles, int vec) {
    constexpr int TR = 16 * RPT, QLD = 64 * NCH + 4;
    extern __shared__ float ams_smem[];
    float* qs = ams_smem;                 // [TR][QLD]
    float* kv = qs + TR * QLD;            // [64][AMS_LD]
    float* ps = kv + 64 * AMS_LD;         // [TR][AMS_LD]
    int* docs = (int*)(ps + TR * AMS_LD); // [64]
    uint32_t* marked = (uint32_t*)(docs + 64);  // [part]: with documents, the key tiles that hold a key of some row's
    __shared__ int doc_range[2];
    const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
    // Heavy tiles first: under a causal mask the last queries see the most keys.
    long id = blockIdx.x;
    const int g = (int)(id % p.nkv);
    id /= p.nkv;
    const int b = (int)(id % p.n_seq);
    const int tile = q_tiles - 1 - (int)(id / p.n_seq);
    const MaskedSeq sq = masked_seq(p, b);
    const int r0 = tile * TR, n_rows = sq.nq * p.G;  // nq * G < 2^31: checked on the host
    if (r0 >= n_rows) return;
    const int split = blockIdx.y;
    const T* Q = (const T*)p.q;
    const T* K = (const T*)p.k;
    const T* V = (const T*)p.v;

    for (int i = tid; i < TR * NCH * 16; i += 256) {
        const int r = i / (NCH * 16), c = (i % (NCH * 16)) * 4;
        const int rr = r0 + r;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (rr < n_rows) x = ams_load4(Q + (sq.q0 + rr / p.G) * p.ldq + (long)(g * p.G + rr % p.G) * p.hd + c, p.hd - c, vec);
        *reinterpret_cast<float4*>(qs + r * QLD + c) = x;
    }
    int lo[RPT], hi[RPT], place[RPT], qdoc[RPT], head[RPT];
#pragma unroll
    for (int i = 0; i < RPT; i++) {
        const int rr = r0 + ty * RPT + i;
        const int t = rr < n_rows ? rr / p.G : 0;
        place[i] = sq.nk - sq.nq + t;
        head[i] = g * p.G + rr % p.G;
        masked_range(p, sq, place[i], lo[i], hi[i]);
        if (rr >= n_rows) lo[i] = hi[i] = 0;
        qdoc[i] = p.q_doc ? p.q_doc[sq.q0 + t] : 0;
    }
    // The union of the rows' ranges, and the documents that they belong to.
    const int t_first = r0 / p.G, t_last = (min(n_rows, r0 + TR) - 1) / p.G;
    int k_lo, k_hi, tmp;
    masked_range(p, sq, sq.nk - sq.nq + t_first, k_lo, tmp);
    masked_range(p, sq, sq.nk - sq.nq + t_last, tmp, k_hi);
    const int first = k_lo / 64, tiles = k_hi > k_lo ? (k_hi + 63) / 64 - first : 0;
    const int j_first = first + min(tiles, split * p.part), j_last = min(first + tiles, j_first + p.part);
    if (p.q_doc) {
        if (tid < 2) doc_range[tid] = tid ? INT_MIN : INT_MAX;
        for (int x = tid; x < (j_last - j_first + 31) / 32; x += 256) marked[x] = 0u;
        __syncthreads();
        if (tid <= t_last - t_first) {
            const int d = p.q_doc[sq.q0 + t_first + tid];
            atomicMin(&doc_range[0], d);
            atomicMax(&doc_range[1], d);
        }
        __syncthreads();
        const int doc_lo = doc_range[0], doc_hi = doc_range[1];
        for (int x = tid; x < (j_last - j_first) * 64; x += 256) {
            const int key = j_first * 64 + x;
            if (key < sq.nk) {
                const int d = p.k_doc[sq.k0 + key];
                if (d >= doc_lo && d <= doc_hi) atomicOr(&marked[x >> 11], 1u << ((x >> 6) & 31));
            }
        }
        __syncthreads();
    }


    float m[RPT], l[RPT], o[NCH][RPT][4];
#pragma unroll
    for (int i = 0; i < RPT; i++) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; c++)
#pragma unroll
            for (int x = 0; x < 4; x++) o[c][i][x] = 0.f;
    }
    const float inv_cap = p.softcap > 0.f ? p.scale / p.softcap : 0.f;
    const int lr = tid >> 4, lc = (tid & 15) * 4;  // staged element: rows lr + 16 x, channels lc ..
    float4 st[4];
    for (int j = j_first; j < j_last; j++) {
        const int key0 = j * 64;
        auto fetch = [&](const T* base, long ld, int ch) {
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const int key = key0 + lr + 16 * x;
                st[x] = key < sq.nk ? ams_load4(base + (sq.k0 + key) * ld + (long)g * p.hd + ch * 64 + lc, p.hd - ch * 64 - lc, vec)
                                    : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        };
        auto stage = [&] {
#pragma unroll
            for (int x = 0; x < 4; x++) *reinterpret_cast<float4*>(kv + (lr + 16 * x) * AMS_LD + lc) = st[x];
        };
        if (p.k_doc && !((marked[(j - j_first) >> 5] >> ((j - j_first) & 31)) & 1u)) continue;
        __syncthreads();  // the previous tile's V and documents are done with
        if (p.k_doc && tid < 64) docs[tid] = key0 + tid < sq.nk ? p.k_doc[sq.k0 + key0 + tid] : 0;
        fetch(K, p.ldk, 0);
        float s[RPT][4];
#pragma unroll
        for (int i = 0; i < RPT; i++)
#pragma unroll
            for (int x = 0; x < 4; x++) s[i][x] = 0.f;
#pragma unroll
        for (int ch = 0; ch < NCH; ch++) {
            if (ch) __syncthreads();
            stage();
            __syncthreads();
            if (ch + 1 < NCH)
                fetch(K, p.ldk, ch + 1);
            else
                fetch(V, p.ldv, 0);
#pragma unroll 4
            for (int d = 0; d < 64; d += 4) {
                float4 a[RPT], w[4];
#pragma unroll
                for (int i = 0; i < RPT; i++) a[i] = *reinterpret_cast<const float4*>(qs + (ty * RPT + i) * QLD + ch * 64 + d);
#pragma unroll
                for (int x = 0; x < 4; x++) w[x] = *reinterpret_cast<const float4*>(kv + (tx + 16 * x) * AMS_LD + d);
#pragma unroll
                for (int i = 0; i < RPT; i++)
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        s[i][x] = fmaf(a[i].x, w[x].x, s[i][x]);
                        s[i][x] = fmaf(a[i].y, w[x].y, s[i][x]);
                        s[i][x] = fmaf(a[i].z, w[x].z, s[i][x]);
                        s[i][x] = fmaf(a[i].w, w[x].w, s[i][x]);
                    }
            }
        }
        // Scores of keys key0 + tx + 16 x.
        bool hidden = false;
#pragma unroll
        for (int i = 0; i < RPT; i++) {
            uint32_t unseen = 0u;
            float top = -INFINITY;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const int key = key0 + tx + 16 * x;
                float v = p.softcap > 0.f ? p.softcap * tanhf(s[i][x] * inv_cap) : s[i][x] * p.scale;
                const int apart = key - place[i];
                if (p.slopes) v -= p.slopes[head[i]] * fabsf((float)apart);
                bool seen = key >= lo[i] && key < hi[i] && (!p.k_doc || docs[tx + 16 * x] == qdoc[i]);
                if (p.table) {
                    const float bias = masked_table(p, head[i], apart);
                    seen = seen && bias != -INFINITY;
                    v += bias;
                }
                unseen |= seen ? 0u : 1u << x;
                s[i][x] = seen ? v : -INFINITY;
                top = fmaxf(top, s[i][x]);
            }
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float mn = fmaxf(m[i], top);
            const float base = mn == -INFINITY ? 0.f : mn;
            const float corr = expf(m[i] - base);
            float sum = 0.f;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const float e = expf(s[i][x] - base);
                sum += e;
                ps[(ty * RPT + i) * AMS_LD + tx + 16 * x] = e;
            }
            if (unseen) {  // -0 marks a hidden key: a weight that has vanished is +0
                hidden = true;
#pragma unroll
                for (int x = 0; x < 4; x++)
                    if ((unseen >> x) & 1u) ps[(ty * RPT + i) * AMS_LD + tx + 16 * x] = -0.f;
            }
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            l[i] = l[i] * corr + sum;
            m[i] = mn;
#pragma unroll
            for (int c = 0; c < NCH; c++)
#pragma unroll
                for (int x = 0; x < 4; x++) o[c][i][x] *= corr;
        }
        hidden = __syncthreads_or(hidden);  // also: K is done with, P is written
#pragma unroll
        for (int ch = 0; ch < NCH; ch++) {
            if (ch) __syncthreads();
            stage();
            __syncthreads();
            if (ch + 1 < NCH) fetch(V, p.ldv, ch + 1);
            auto accumulate = [&](auto guard) {
#pragma unroll 2
                for (int d = 0; d < 64; d += 4) {
                    float4 a[RPT];
#pragma unroll
                    for (int i = 0; i < RPT; i++) a[i] = *reinterpret_cast<const float4*>(ps + (ty * RPT + i) * AMS_LD + d);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float4 w = *reinterpret_cast<const float4*>(kv + (d + e) * AMS_LD + tx * 4);
#pragma unroll
                        for (int i = 0; i < RPT; i++) {
                            const float pe = e == 0 ? a[i].x : e == 1 ? a[i].y : e == 2 ? a[i].z : a[i].w;
                            // A hidden key's value may be anything: 0 x NaN must not reach the sum, of a key that the row sees it must.
                            if (!decltype(guard)::value || __float_as_uint(pe) != 0x80000000u) {
                                o[ch][i][0] = fmaf(pe, w.x, o[ch][i][0]);
                                o[ch][i][1] = fmaf(pe, w.y, o[ch][i][1]);
                                o[ch][i][2] = fmaf(pe, w.z, o[ch][i][2]);
                                o[ch][i][3] = fmaf(pe, w.w, o[ch][i][3]);
                            }
                        }
                    }
                }
            };
            if (hidden)
                accumulate(std::true_type{});
            else
                accumulate(std::false_type{});
        }
    }
#pragma unroll
    for (int i = 0; i < RPT; i++) {
        const int rr = r0 + ty * RPT + i;
        if (rr >= n_rows) continue;
        const long row = sq.q0 + rr / p.G;
        const float inv = l[i] > 0.f ? 1.f / l[i] : l[i] == 0.f ? 0.f : l[i];  // NaN stays
        if (p.nsplit > 1) {
            const long at = ((long)split * p.q_rows + row) * p.nh + head[i];
            if (tx == 0) p.part_ml[at] = make_float2(m[i], l[i]);
#pragma unroll
            for (int c = 0; c < NCH; c++)
#pragma unroll
                for (int x = 0; x < 4; x++)
                    if (c * 64 + tx * 4 + x < p.hd) p.part_o[at * p.hd + c * 64 + tx * 4 + x] = o[c][i][x] * inv;
        } else {
            if (tx == 0 && p.lse) p.lse[row * p.nh + head[i]] = l[i] == 0.f ? -INFINITY : m[i] + logf(l[i]);
            T* orow = (T*)p.out + row * p.ldo + (long)head[i] * p.hd;
#pragma unroll
            for (int c = 0; c < NCH; c++)
#pragma unroll
                for (int x = 0; x < 4; x++)
                    if (c * 64 + tx * 4 + x < p.hd) stf(orow, c * 64 + tx * 4 + x, o[c][i][x] * inv);
        }
    }
}

#include "attention_masked_tc.cuh"
#include "attention_masked_few.cuh"

// A part that has seen nothing weighs -0 and may hold anything; one whose weight has vanished counts all the same, as its sum may not
// be finite.
EG2_DEV bool masked_part_counts(float w) { return __float_as_uint(w) != 0x80000000u; }
EG2_DEV float masked_part_weight(const MaskedParams& p, float2 ml, float base) {
    return ml.y == 0.f ? -0.f : ml.y * (p.log2_parts ? ex2_approx(ml.x - base) : expf(ml.x - base));
}
EG2_DEV float masked_part_lse(const MaskedParams& p, float base, float total) {
    return total == 0.f ? -INFINITY : p.log2_parts ? (base + log2f(total)) * 0.6931471805599453f : base + logf(total);
}

// Joins the parts of a split key axis: out = sum_s w_s o_s / sum_s w_s with w_s = l_s exp(m_s - max m), in part order. Maximum and sum
// come apart: of m + log l in 32 bits little is left of the sum where the maximum is large. A block per (sequence, query, head),
// two groups of 128 threads that take every other part; the parts' results are on their way while the weights are
// worked out. Bound by latency: few rows, their parts read once.
template <typename T>
__global__ void __launch_bounds__(256) attention_masked_join_kernel(const MaskedParams p) {
    extern __shared__ float weight[];  // [nsplit] (-0: nothing seen), then [hd] of the second group
    __shared__ float red[8];
    grid_dep_launch();
    grid_dep_wait();
    long id = blockIdx.x;
    const int h = (int)(id % p.nh);
    id /= p.nh;
    const int t = (int)(id % p.max_q), b = (int)(id / p.max_q);
    const MaskedSeq sq = masked_seq(p, b);
    if (t >= sq.nq) return;
    const long row = sq.q0 + t, item = row * p.nh + h, step = p.q_rows * p.nh;
    const int group = threadIdx.x >> 7, c0 = threadIdx.x & 127;
    constexpr int AHEAD = 16;  // parts on their way, of the thread's first channel
    float early[AHEAD];
#pragma unroll
    for (int y = 0; y < AHEAD; y++) {
        const int s = group + 2 * y;
        early[y] = s < p.nsplit && c0 < p.hd ? p.part_o[(s * step + item) * p.hd + c0] : 0.f;
    }
    float top = -INFINITY;
    for (int s = threadIdx.x; s < p.nsplit; s += 256) {
        const float2 ml = p.part_ml[s * step + item];
        top = fmaxf(top, ml.y == 0.f ? -INFINITY : ml.x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 8; x++) top = fmaxf(top, red[x]);
    const float base = top == -INFINITY ? 0.f : top;
    for (int s = threadIdx.x; s < p.nsplit; s += 256) weight[s] = masked_part_weight(p, p.part_ml[s * step + item], base);
    __syncthreads();
    float total = 0.f;
    for (int s = 0; s < p.nsplit; s++) total += weight[s];  // the same sum in every thread
    const float inv = total == 0.f ? 0.f : 1.f / total;
    float* second = weight + p.nsplit;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};  // hd is at most 512
#pragma unroll
    for (int x = 0; x < 4; x++) {
        const int c = c0 + 128 * x;
        if (c >= p.hd) break;
        int s = group;
        if (x == 0) {
#pragma unroll
            for (int y = 0; y < AHEAD; y++, s += 2)
                if (s < p.nsplit && masked_part_counts(weight[s])) sum[x] = fmaf(weight[s], early[y], sum[x]);
        }
#pragma unroll 8
        for (; s < p.nsplit; s += 2) {
            const float w = weight[s];
            const float o = masked_part_counts(w) ? p.part_o[(s * step + item) * p.hd + c] : 0.f;
            sum[x] = fmaf(w, o, sum[x]);
        }
        if (group) second[c] = sum[x];
    }
    __syncthreads();
    if (group == 0) {
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const int c = c0 + 128 * x;
            if (c < p.hd) stf((T*)p.out + row * p.ldo + (long)h * p.hd, c, (sum[x] + second[c]) * inv);
        }
        if (c0 == 0 && p.lse) p.lse[item] = masked_part_lse(p, base, total);
    }
}

// The same for up to JOIN_PARTS parts, a warp per row: many rows with few parts each are bound by reading the parts, and a
// block per row is mostly waiting (call of 1,000 queries, 4 heads over 2 of 256, 8,192 keys in 4 parts: 59 us with it, 83 with
// a block per row; of 32 queries in 8 parts: 38 and 34).
constexpr int JOIN_PARTS = 8;
template <typename T>
__global__ void __launch_bounds__(256) attention_masked_join_rows_kernel(const MaskedParams p) {
    grid_dep_launch();
    grid_dep_wait();
    const int lane = threadIdx.x & 31;
    long id = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (id >= (long)p.n_seq * p.max_q * p.nh) return;
    const int h = (int)(id % p.nh);
    id /= p.nh;
    const int t = (int)(id % p.max_q), b = (int)(id / p.max_q);
    const MaskedSeq sq = masked_seq(p, b);
    if (t >= sq.nq) return;
    const long row = sq.q0 + t, item = row * p.nh + h, step = p.q_rows * p.nh;
    const float2 ml = lane < p.nsplit ? p.part_ml[lane * step + item] : make_float2(0.f, 0.f);
    float top = ml.y == 0.f ? -INFINITY : ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float base = top == -INFINITY ? 0.f : top, mine = masked_part_weight(p, ml, base);
    float w[JOIN_PARTS], total = 0.f;
#pragma unroll
    for (int s = 0; s < JOIN_PARTS; s++) total += w[s] = __shfl_sync(0xffffffffu, mine, s);
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll 4
    for (int c = lane; c < p.hd; c += 32) {
        float o[JOIN_PARTS], sum = 0.f;
#pragma unroll
        for (int s = 0; s < JOIN_PARTS; s++) o[s] = masked_part_counts(w[s]) ? p.part_o[(s * step + item) * p.hd + c] : 0.f;
#pragma unroll
        for (int s = 0; s < JOIN_PARTS; s++) sum = fmaf(w[s], o[s], sum);
        stf((T*)p.out + row * p.ldo + (long)h * p.hd, c, sum * inv);
    }
    if (lane == 0 && p.lse) p.lse[item] = masked_part_lse(p, base, total);
}

template <typename T, int NCH, int RPT>
static int launch_masked_simt(const MaskedParams& p, int vec, cudaStream_t s) {
    constexpr int TR = 16 * RPT;
    constexpr int FIXED = (TR * (64 * NCH + 4) + 64 * AMS_LD + TR * AMS_LD + 64) * 4;
    const int smem = FIXED + (p.q_doc ? (p.part + 31) / 32 * 4 : 0);
    static bool attr_set[64] = {false};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
    auto kern = attention_masked_simt_kernel<T, NCH, RPT>;
    if (!attr_set[dev]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, FIXED + EG2_MASKED_MAX_LEN / 64 / 8) != cudaSuccess) return -3;
        attr_set[dev] = true;
    }
    const int q_tiles = (int)(((long)p.max_q * p.G + TR - 1) / TR);
    const long blocks = (long)q_tiles * p.n_seq * p.nkv;
    if (blocks > 0x7fffffffL) return -1;
    kern<<<dim3((unsigned)blocks, (unsigned)p.nsplit), 256, smem, s>>>(p, q_tiles, vec);
    return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

template <typename T, int RPT>
static int attention_masked_simt(const MaskedParams& p, int vec, cudaStream_t s) {
    if (p.hd <= 64) return launch_masked_simt<T, 1, RPT>(p, vec, s);
    if (p.hd <= 128) return launch_masked_simt<T, 2, RPT>(p, vec, s);
    if (p.hd <= 256) return launch_masked_simt<T, 4, RPT>(p, vec, s);
    return launch_masked_simt<T, 8, RPT>(p, vec, s);
}
// Rows of a query tile on the CUDA cores: 64 use shared memory best, 32 fill the SMs of a call with few tiles (f32, 64 / 32
// rows: 256 tiles of 64, 4,096 tokens, 4 heads over 1 of 128: 1,471 / 1,732 us; 192 tiles, 1,000 tokens, 12 heads of 64:
// 226 / 196; 32 tiles, 500 tokens, 4 heads over 2 of 256: 174 / 132).
static int masked_simt_rows(const eg2_masked_attention* a) {
    const long tiles = ((long)a->max_q * (a->nh / a->nkv) + 63) / 64 * a->n_seq * a->nkv;
    return tiles >= num_sms() * 3L / 2 ? 64 : 32;
}

template <typename T>
static int attention_masked_join(const MaskedParams& p, cudaStream_t s) {
    const long items = (long)p.n_seq * p.max_q * p.nh;
    const bool by_rows = p.nsplit <= JOIN_PARTS && items > 4L * num_sms();
    const long blocks = by_rows ? (items + 7) / 8 : items;
    if (blocks > 0x7fffffffL) return -1;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)blocks, 1, 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.dynamicSmemBytes = by_rows ? 0 : (p.nsplit + p.hd) * 4;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, by_rows ? attention_masked_join_rows_kernel<T> : attention_masked_join_kernel<T>, p) == cudaSuccess ? 0 : -3;
}

// How a call runs. The tensor cores take bf16 whose rows and heads TMA can address (16-byte multiples) and G query
// heads that divide a 128-row tile are packed into it, unless their bias tables together pass the shared memory
// kept for them; the rest runs on the CUDA cores. Calls whose query tiles would be at most an eighth full -- 16 rows --
// are bound by reading K and V and take the form made for that (4 heads over 2 of 256, 8 x up to 11,774 keys: 1 query each 42 us,
// 75 in 128-row tiles, both with L2 flushed and one call at a time (33 among other calls); 8 queries each 54 and 77; 64 x 512 keys, 12 heads
// of 64: 53 and 57; only at a few hundred keys and all 16 rows do the tiles win: 8 queries over 300, 28 and 21). Packing: 256 sequences of 17 tokens, 4 heads over 1 of 256, 24 us, 64
// with a tile per head.
struct MaskedPlan {
    bool tc, few;
    int Gt, nsplit, part;
};
static MaskedPlan masked_plan(const eg2_masked_attention* a) {
    MaskedPlan r;
    const int G = a->nh / a->nkv;
    r.tc = a->kind == EG2_BF16 && a->hd % 8 == 0 && (a->ldq | a->ldk | a->ldv | a->ldo) % 8 == 0 &&
           ((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out) % 16 == 0 && a->k_rows > 0 &&
           a->q_rows < (1L << 31) && a->k_rows < (1L << 31) - 128;
    r.Gt = G;
    if (r.tc && (128 % G || (a->dist_bias && G * (2L * a->dist_radius + 257) > AMT_TABLE))) r.Gt = 1;
    r.few = r.tc && (long)a->max_q * G <= 16;
    if (r.few) r.Gt = G;
    // The key axis is split into parts of a fixed number of key tiles when the query tiles alone leave SMs idle, so many that
    // the parts of all sequences are resident at once: their count is at most the key tiles there are (k_rows) over the part,
    // and one more per sequence and head. A part pays for its partial result, 128 rows of it more than one: at least 8 tiles,
    // or 2 where a query tile is mostly empty (each with as much again to share), or a block of 16 keys for each warp of the form
    // for few rows (two at head 512). Split and whole: 2,000 queries, 4 heads over 2 of 256, 8,192 keys 90 / 129 us; 256 queries,
    // 12 heads of 64, 2,048 keys 21 / 22; 1,200 over as many in two parts of 5 tiles 35 / 29 (hence the 8); 1 query over 2,208
    // keys 14 / 55.
    const int rows = r.few ? 16 : r.tc ? 128 : masked_simt_rows(a), keys = r.few ? 16 : r.tc ? 128 : 64;
    const int halves = r.tc && a->hd > 256 ? 2 : 1;
    const long tile_rows = (long)a->max_q * r.Gt;
    const long base = (tile_rows + rows - 1) / rows * a->n_seq * (a->nh / r.Gt) * halves;
    const long longest = a->max_k < a->k_rows ? a->max_k : a->k_rows;
    const long key_tiles = (longest + keys - 1) / keys;
    const long slots = num_sms() * (r.few && halves == 1 ? 2L : 1L);
    long all = base * key_tiles;
    if (a->n_seq > 0 && base / a->n_seq * ((a->k_rows + keys - 1) / keys + a->n_seq) < all) all = base / a->n_seq * ((a->k_rows + keys - 1) / keys + a->n_seq);
    long part = base < slots ? (all + slots - base - 1) / (slots - base) : key_tiles;
    const long least = r.few ? (a->hd > 256 ? 8 : 4) : tile_rows > rows / 4 ? 8 : 2;
    if (part < least) part = least;
    r.nsplit = base >= slots || part >= key_tiles || (!r.few && key_tiles < 2 * least) ? 1 : (int)((key_tiles + part - 1) / part);
    if (r.nsplit > 1 && base * r.nsplit <= slots) part = (key_tiles + r.nsplit - 1) / r.nsplit;
    r.part = r.nsplit > 1 ? (int)part : (int)(key_tiles > 0 ? key_tiles : 1);
    return r;
}

// Workspace: the parts' results, then their maxima and sums, at an even number of floats.
static int64_t masked_part_ml_at(const eg2_masked_attention* a, int nsplit) {
    return ((int64_t)nsplit * a->q_rows * a->nh * a->hd + 1) / 2 * 2;
}

static bool masked_valid(const eg2_masked_attention* a) {
    if (!a || (a->kind != EG2_F32 && a->kind != EG2_BF16)) return false;
    if (a->n_seq < 0 || a->max_q < 0 || a->max_k < 0 || a->q_rows < 0 || a->k_rows < 0) return false;
    if (a->nh <= 0 || a->nkv <= 0 || a->nh % a->nkv || a->hd <= 0 || a->hd > 512 || a->nh > 4096) return false;
    if (a->max_q > EG2_MASKED_MAX_LEN || a->max_k > EG2_MASKED_MAX_LEN) return false;
    if (a->ldq < (int64_t)a->nh * a->hd || a->ldo < (int64_t)a->nh * a->hd || a->ldk < (int64_t)a->nkv * a->hd ||
        a->ldv < (int64_t)a->nkv * a->hd)
        return false;
    if (!std::isfinite(a->scale) || !(a->softcap >= 0.f) || !std::isfinite(a->softcap)) return false;
    if ((a->q_doc == nullptr) != (a->k_doc == nullptr)) return false;
    if (a->prefix_len && !a->causal) return false;
    if (a->dist_bias && (a->dist_radius < 0 || a->dist_radius > EG2_MASKED_MAX_RADIUS)) return false;
    if ((long)a->max_q * (a->nh / a->nkv) > 0x7fffffffL - 256) return false;
    return true;
}

}  // namespace eg2

extern "C" {

int64_t eg2_attention_masked_workspace(const eg2_masked_attention* a) {
    if (!eg2::masked_valid(a)) return EG2_ERR_INVALID;
    const int n = eg2::masked_plan(a).nsplit;
    return n > 1 ? eg2::masked_part_ml_at(a, n) * 4 + (int64_t)n * a->q_rows * a->nh * 8 : 0;
}

int eg2_attention_masked(const eg2_masked_attention* a, void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace eg2;
    if (!masked_valid(a)) return EG2_ERR_INVALID;
    if (a->q_rows == 0 || a->n_seq == 0 || a->max_q == 0) return EG2_OK;
    if (!a->q || !a->out || !a->q_off || !a->k_off || (a->k_rows > 0 && (!a->k || !a->v))) return EG2_ERR_INVALID;
    MaskedParams p{a->q, a->k, a->v, a->out, a->lse, a->ldq, a->ldk, a->ldv, a->ldo, a->q_off, a->k_off, a->prefix_len, a->q_doc,
                   a->k_doc, a->slopes, a->dist_bias, a->q_rows, a->k_rows, a->n_seq, a->max_q, a->max_k, a->nh, a->nkv, a->hd,
                   a->nh / a->nkv, a->window, a->causal, a->dist_radius, 1, 0, a->scale, a->softcap, nullptr, nullptr, 0};
    // Numbers whose products with log2 e or with one another would leave f32: a scale or a cap past 1e38 acts as 1e38 does (scores
    // differ only where they pass it), and under a cap of less than 1e-30 of the scale every score but zero is the cap.
    p.scale = std::fmax(-1e38f, std::fmin(1e38f, p.scale));
    p.softcap = std::fmin(1e38f, p.softcap);
    if (p.softcap > 0.f && std::fabs(p.scale) > 1e30f * p.softcap) p.scale = std::copysign(1e30f * p.softcap, p.scale);
    cudaStream_t s = (cudaStream_t)stream;
    const MaskedPlan plan = masked_plan(a);
    p.nsplit = plan.nsplit;
    p.part = plan.part;
    if (p.nsplit > 1) {
        if (!workspace || workspace_bytes < eg2_attention_masked_workspace(a) || (uintptr_t)workspace % 16) return EG2_ERR_INVALID;
        p.part_o = (float*)workspace;
        p.part_ml = (float2*)(p.part_o + masked_part_ml_at(a, p.nsplit));
        p.log2_parts = plan.tc;
    }
    int rc;
    if (plan.few) {
        rc = a->hd <= 64 ? launch_masked_few<64>(p, s) : a->hd <= 128 ? launch_masked_few<128>(p, s)
             : a->hd <= 256 ? launch_masked_few<256>(p, s) : launch_masked_few<512>(p, s);
    } else if (plan.tc) {
        rc = a->hd <= 64 ? launch_masked_tc<64>(p, plan.Gt, s) : a->hd <= 128 ? launch_masked_tc<128>(p, plan.Gt, s)
             : a->hd <= 256 ? launch_masked_tc<256>(p, plan.Gt, s) : launch_masked_tc<512>(p, plan.Gt, s);
    } else {
        const int unit = a->kind == EG2_F32 ? 16 : 8;  // bytes of four elements
        const int vec = ((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v) % unit == 0 && (a->ldq | a->ldk | a->ldv | a->hd) % 4 == 0;
        if (masked_simt_rows(a) == 64)
            rc = a->kind == EG2_F32 ? attention_masked_simt<float, 4>(p, vec, s) : attention_masked_simt<bf16_t, 4>(p, vec, s);
        else
            rc = a->kind == EG2_F32 ? attention_masked_simt<float, 2>(p, vec, s) : attention_masked_simt<bf16_t, 2>(p, vec, s);
    }
    if (!rc && p.nsplit > 1) rc = a->kind == EG2_F32 ? attention_masked_join<float>(p, s) : attention_masked_join<bf16_t>(p, s);
    if (rc == -1) return EG2_ERR_INVALID;
    if (rc) return EG2_ERR_CUDA;
    g_launches.fetch_add(p.nsplit > 1 ? 2 : 1, std::memory_order_relaxed);
    return EG2_OK;
}

}  // extern "C"
