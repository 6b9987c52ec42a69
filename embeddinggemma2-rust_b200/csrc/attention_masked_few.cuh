// The form of masked attention for few query rows over many keys (bf16), included by attention_masked.cu.
//
// At most 16 rows (query tokens x the G heads of a K/V head): the work is to read K and V once, so the design is for
// bytes in flight and a short path per byte, not for tensor throughput -- warp-level mma.sync with the 16 rows as M.
// (The 128-row tile of the tcgen05 form spends 40,000 cycles on its first tiles here: its softmax is thousands of
// instructions long, and nothing repeats to amortise their fetch.)
//
// A CTA takes one part of the keys of one (sequence, K/V head, 256-channel half of O); each of its warps walks blocks
// of 16 keys on its own, with a ring of its own that one lane fills by TMA, 16 keys x 64 channels a box, and its own
// running maximum, sum and O in registers. The warps' results are joined through shared memory at the end. Blocks that
// no row may see, by range or by document, are not loaded.

template <int HD>
struct AmfCfg {
    static constexpr int DV = HD < 256 ? HD : 256, HALVES = HD / DV;
    static constexpr int WARPS = HD <= 128 ? 8 : 4;
    static constexpr int STAGES = HD == 64 ? 6 : HD == 512 ? 2 : 3;
    static constexpr int K_BYTES = 16 * HD * 2, STAGE = 16 * (HD + DV) * 2;
    static constexpr int OFF_RING = 16 * HD * 2;  // after Q
    static constexpr int OFF_BAR = OFF_RING + WARPS * STAGES * STAGE;
    static constexpr int OFF_BLOCKS = OFF_BAR + WARPS * STAGES * 8;  // bit mask of the part's blocks
    static constexpr int MAX_WORDS = EG2_MASKED_MAX_LEN / 16 / 32;
    static constexpr int SMEM = 1024 + OFF_BLOCKS;  // + the mask of the call's part
};

EG2_DEV void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
EG2_DEV void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
EG2_DEV void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Byte offset of (row, channel) in chunks of [16 rows x 64 channels] with the 128-byte swizzle.
EG2_DEV uint32_t amf_at(int row, int ch) {
    return (uint32_t)((ch >> 6) * 2048 + row * 128 + ((((ch >> 3) & 7) ^ (row & 7)) << 4) + (ch & 7) * 2);
}

template <int HD>
__global__ void __launch_bounds__(32 * AmfCfg<HD>::WARPS, 1)
    attention_masked_few_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                                const __grid_constant__ MaskedParams p) {
    using Cfg = AmfCfg<HD>;
    constexpr int DV = Cfg::DV, WARPS = Cfg::WARPS, STAGES = Cfg::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
    uint32_t* blocks = reinterpret_cast<uint32_t*>(smem + Cfg::OFF_BLOCKS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dep_launch();
    grid_dep_wait();
    int id = blockIdx.x;
    const int half = id % Cfg::HALVES;
    id /= Cfg::HALVES;
    const int g = id % p.nkv, b = id / p.nkv;
    const int split = blockIdx.y;
    const MaskedSeq sq = masked_seq(p, b);
    const int rows = sq.nq * p.G;  // at most 16: the host's max_q says so
    if (rows == 0) return;
    int k_lo, k_hi, tmp;
    masked_range(p, sq, sq.nk - sq.nq, k_lo, tmp);
    masked_range(p, sq, sq.nk - 1, tmp, k_hi);
    // Blocks of 16 keys [first, last) of this part.
    const int all_first = k_lo / 16, all_last = k_hi > k_lo ? (k_hi + 15) / 16 : all_first;
    const int first = min(all_last, all_first + split * p.part), last = min(all_last, first + p.part);
    const int words = (last - first + 31) / 32;

    // This thread's rows r0 and r0 + 8, and its columns of a block: 2 (lane % 4) + {0, 1} and 8 more.
    int lo[2], hi[2], place[2], qdoc[2], head[2];
    float slope[2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int r = (lane >> 2) + 8 * x, t = r < rows ? r / p.G : 0;
        place[x] = sq.nk - sq.nq + t;
        head[x] = g * p.G + r % p.G;
        masked_range(p, sq, place[x], lo[x], hi[x]);
        if (r >= rows) lo[x] = hi[x] = 0;
        qdoc[x] = p.q_doc ? p.q_doc[sq.q0 + t] : 0;
        slope[x] = p.slopes ? p.slopes[head[x]] * AMT_LOG2E : 0.f;
    }
    if (threadIdx.x == 0) {
        for (int x = 0; x < WARPS * STAGES; x++) mbar_init(&bars[x], 1);
        fence_mbarrier_init();
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    for (int w = threadIdx.x; w < words; w += blockDim.x) blocks[w] = p.q_doc ? 0u : w + 1 < words || !((last - first) & 31) ? ~0u : (1u << ((last - first) & 31)) - 1u;
    for (int x = threadIdx.x; x < 16 * HD / 8; x += blockDim.x) {
        const int r = x / (HD / 8), c = x % (HD / 8) * 8;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (r < rows && c < p.hd)
            v = *reinterpret_cast<const uint4*>((const bf16_t*)p.q + (sq.q0 + r / p.G) * p.ldq + (long)(g * p.G + r % p.G) * p.hd + c);
        *reinterpret_cast<uint4*>(smem + amf_at(r, c)) = v;
    }
    __syncthreads();
    if (p.q_doc) {
        // Blocks with a key of some query's document (of their range of ids: the rows mask exactly).
        int dlo = INT_MAX, dhi = INT_MIN;
        for (int t = 0; t < sq.nq; t++) {
            const int d = p.q_doc[sq.q0 + t];
            dlo = min(dlo, d);
            dhi = max(dhi, d);
        }
        for (int x = threadIdx.x; x < (last - first) * 16; x += blockDim.x) {
            const int key = first * 16 + x;
            if (key < sq.nk) {
                const int d = p.k_doc[sq.k0 + key];
                if (d >= dlo && d <= dhi) atomicOr(&blocks[x >> 9], 1u << ((x >> 4) & 31));
            }
        }
        __syncthreads();
    }
    // This warp takes every WARPS-th of the marked blocks, the warp-th first.
    int at_word = 0;
    uint32_t left = words ? blocks[0] : 0u;
    auto next_block = [&]() -> int {  // -1: none
        while (!left) {
            if (++at_word >= words) return -1;
            left = blocks[at_word];
        }
        const int bit = __ffs(left) - 1;
        left &= left - 1u;
        return first + at_word * 32 + bit;
    };
    auto my_next = [&](int skip) -> int {
        int blk = words ? next_block() : -1;
        for (int x = 0; x < skip && blk >= 0; x++) blk = next_block();
        return blk;
    };
    uint8_t* ring = smem + Cfg::OFF_RING + warp * STAGES * Cfg::STAGE;
    uint64_t* full = bars + warp * STAGES;
    int queue[STAGES], issued = 0;  // the blocks under way, by stage
    auto issue = [&](int blk) {
        const int st = issued % STAGES;
        if (lane == 0) {
            mbar_arrive_expect_tx(&full[st], Cfg::STAGE);
            for (int c = 0; c < HD / 64; c++) tma_load_3d(ring + st * Cfg::STAGE + c * 2048, &tmK, &full[st], 64 * c, g, (int)sq.k0 + blk * 16);
            for (int c = 0; c < DV / 64; c++)
                tma_load_3d(ring + st * Cfg::STAGE + Cfg::K_BYTES + c * 2048, &tmV, &full[st], half * 256 + 64 * c, g, (int)sq.k0 + blk * 16);
        }
        issued++;
    };
    int blk = my_next(warp);
#pragma unroll
    for (int st = 0; st < STAGES; st++) {
        queue[st] = blk;
        if (blk >= 0) {
            issue(blk);
            blk = my_next(WARPS - 1);
        }
    }

    const bool capped = p.softcap > 0.f;
    const float in_scale = capped ? p.scale / p.softcap : p.scale * AMT_LOG2E, cap2 = p.softcap * AMT_LOG2E;
    float m[2] = {AMT_NONE, AMT_NONE}, l[2] = {0.f, 0.f};
    float o[DV / 8][4];
#pragma unroll
    for (int c = 0; c < DV / 8; c++)
#pragma unroll
        for (int x = 0; x < 4; x++) o[c][x] = 0.f;
    const uint32_t q_addr = smem_u32(smem);
    bool ok = true;
    int taken = 0;
    while (true) {
        const int st = taken % STAGES;
        int now = queue[0];
#pragma unroll
        for (int x = 1; x < STAGES; x++)
            if (st == x) now = queue[x];
        if (now < 0) break;
        const int key0 = now * 16;
        // Document ids of this thread's four columns, under the latency of the block.
        int ids[4];
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const int key = key0 + 8 * (x >> 1) + 2 * (lane & 3) + (x & 1);
            ids[x] = p.k_doc && key < sq.nk ? p.k_doc[sq.k0 + key] : 0;
        }
        if (!(ok = mbar_wait(&full[st], (taken / STAGES) & 1, EG2_DEV_TIMEOUT_ATTN, nullptr))) break;
        uint8_t* kb = ring + st * Cfg::STAGE;
        uint8_t* vb = kb + Cfg::K_BYTES;
        const uint32_t k_addr = smem_u32(kb), v_addr = smem_u32(vb);
        float s[2][4] = {};
#pragma unroll
        for (int c = 0; c < HD / 16; c++) {
            uint32_t qa[4], kf[4];
            // Q: rows 0-7 / 8-15 x channels 0-7, then the same x channels 8-15; K: keys 0-7 x both, keys 8-15 x both.
            ldmatrix4(q_addr + amf_at((lane & 7) + 8 * ((lane >> 3) & 1), 16 * c + 8 * (lane >> 4)), qa);
            ldmatrix4(k_addr + amf_at((lane & 7) + 8 * (lane >> 4), 16 * c + 8 * ((lane >> 3) & 1)), kf);
            mma_16816(s[0], qa, kf[0], kf[1]);
            mma_16816(s[1], qa, kf[2], kf[3]);
        }
        bool hidden = false;  // some key is hidden from some row of this thread
        float top[2] = {AMT_NONE, AMT_NONE};
#pragma unroll
        for (int x = 0; x < 2; x++)  // row
#pragma unroll
            for (int y = 0; y < 4; y++) {  // column
                float& v = s[y >> 1][2 * x + (y & 1)];
                const int key = key0 + 8 * (y >> 1) + 2 * (lane & 3) + (y & 1), apart = key - place[x];
                v = capped ? cap2 * tanh_any(v * in_scale) : v * in_scale;
                if (p.slopes) v = fmaf(-slope[x], fabsf((float)apart), v);
                if (p.table)
                    v += masked_bias(p.table[(long)head[x] * (2 * p.radius + 1) + p.radius + min(max(apart, -p.radius), p.radius)]) * AMT_LOG2E;
                const bool seen = key >= lo[x] && key < hi[x] && (!p.k_doc || ids[y] == qdoc[x]);
                hidden |= !seen && (lane >> 2) + 8 * x < rows;
                v = seen ? v : -INFINITY;
                top[x] = fmaxf(top[x], v);
            }
        float factor[2];
        uint32_t pa[4];
#pragma unroll
        for (int x = 0; x < 2; x++) {
            top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
            top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
            const float mn = fmaxf(m[x], top[x]);
            factor[x] = ex2_approx(m[x] - mn);
            m[x] = mn;
            l[x] *= factor[x];
#pragma unroll
            for (int y = 0; y < 4; y++) {
                float& v = s[y >> 1][2 * x + (y & 1)];
                v = ex2_approx(v - mn);
                l[x] += v;
            }
            pa[x] = bf16x2_bits(s[0][2 * x], s[0][2 * x + 1]);
            pa[2 + x] = bf16x2_bits(s[1][2 * x], s[1][2 * x + 1]);
        }
        if (__any_sync(0xffffffffu, factor[0] != 1.f || factor[1] != 1.f)) {
#pragma unroll
            for (int c = 0; c < DV / 8; c++) {
                o[c][0] *= factor[0];
                o[c][1] *= factor[0];
                o[c][2] *= factor[1];
                o[c][3] *= factor[1];
            }
        }
        if (__any_sync(0xffffffffu, hidden)) {
            // A hidden key's value may be anything, and 0 x NaN must not reach the sum: elements that are not finite become
            // zero, after the rows that do see the key have taken them.
            uint32_t bad = 0;  // keys
            for (int x = lane; x < 16 * DV / 8; x += 32) {
                const int key = x / (DV / 8), c = x % (DV / 8) * 8;
                const uint4 v = *reinterpret_cast<const uint4*>(vb + amf_at(key, c));
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int y = 0; y < 4; y++)
                    if ((w[y] & 0x7f80u) == 0x7f80u || (w[y] & 0x7f800000u) == 0x7f800000u) bad |= 1u << key;
            }
            bad = __reduce_or_sync(0xffffffffu, bad);
            for (; bad; bad &= bad - 1u) {
                const int key = __ffs(bad) - 1;
                const int src = (lane & ~3) + ((key & 7) >> 1);  // who holds this key's weights of my rows
                const float a0 = __shfl_sync(0xffffffffu, s[0][key & 1 ? 1 : 0], src), a1 = __shfl_sync(0xffffffffu, s[0][key & 1 ? 3 : 2], src);
                const float b0 = __shfl_sync(0xffffffffu, s[1][key & 1 ? 1 : 0], src), b1 = __shfl_sync(0xffffffffu, s[1][key & 1 ? 3 : 2], src);
                const float w0 = key < 8 ? a0 : b0, w1 = key < 8 ? a1 : b1;
#pragma unroll
                for (int c = 0; c < DV / 8; c++)
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        const float v = bf16_to_f32(*reinterpret_cast<const bf16_t*>(vb + amf_at(key, 8 * c + 2 * (lane & 3) + y)));
                        if (!(fabsf(v) < INFINITY)) {
                            if (w0 != 0.f) o[c][y] = fmaf(w0, v, o[c][y]);
                            if (w1 != 0.f) o[c][2 + y] = fmaf(w1, v, o[c][2 + y]);
                        }
                    }
                __syncwarp();
                for (int c = lane; c < DV; c += 32) {
                    bf16_t* v = reinterpret_cast<bf16_t*>(vb + amf_at(key, c));
                    if ((*v & 0x7f80u) == 0x7f80u) *v = 0;
                }
                __syncwarp();
            }
        }
#pragma unroll
        for (int c = 0; c < DV / 16; c++) {
            uint32_t vf[4];
            // V transposed: keys 0-7 and 8-15 x channels 0-7, then x channels 8-15.
            ldmatrix4_trans(v_addr + amf_at((lane & 7) + 8 * ((lane >> 3) & 1), 16 * c + 8 * (lane >> 4)), vf);
            mma_16816(o[2 * c], pa, vf[0], vf[1]);
            mma_16816(o[2 * c + 1], pa, vf[2], vf[3]);
        }
        fence_proxy_async();  // the cleaning's writes come before the next load's
        __syncwarp();         // the stage has been read
        taken++;
#pragma unroll
        for (int x = 0; x < STAGES; x++)
            if (st == x) queue[x] = blk;
        if (blk >= 0) {
            issue(blk);
            blk = my_next(WARPS - 1);
        }
    }
    // No load may land after the CTA has ended (on the error path; else all have been waited for).
    if (!ok && lane == 0)
        for (int x = taken; x < issued; x++) mbar_drain(&full[x % STAGES], (x / STAGES) & 1, 200000000ull);
#pragma unroll
    for (int x = 0; x < 2; x++) {
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    }
    // ---- the warps' results, joined in warp order ----
    __syncthreads();
    float* mo = reinterpret_cast<float*>(smem + Cfg::OFF_RING);  // [WARPS][16][DV]
    float* ml = reinterpret_cast<float*>(smem);                  // [WARPS][16][2]: over Q
    static_assert(WARPS * 16 * DV * 4 <= WARPS * STAGES * Cfg::STAGE && WARPS * 16 * 8 <= 16 * HD * 2, "few rows: shared memory of the join");
    {
        const int r = lane >> 2;
        if ((lane & 3) == 0)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                ml[(warp * 16 + r + 8 * x) * 2] = m[x];
                ml[(warp * 16 + r + 8 * x) * 2 + 1] = l[x];
            }
#pragma unroll
        for (int c = 0; c < DV / 8; c++)
#pragma unroll
            for (int x = 0; x < 2; x++)
                *reinterpret_cast<float2*>(mo + (warp * 16 + r + 8 * x) * DV + 8 * c + 2 * (lane & 3)) = make_float2(o[c][2 * x], o[c][2 * x + 1]);
    }
    __syncthreads();
    for (int x = threadIdx.x; x < rows * DV; x += blockDim.x) {
        const int r = x / DV, c = x % DV, ch = half * 256 + c;
        float mm = AMT_NONE;
#pragma unroll
        for (int w = 0; w < WARPS; w++) mm = fmaxf(mm, ml[(w * 16 + r) * 2]);
        float ll = 0.f, a = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const float f = ex2_approx(ml[(w * 16 + r) * 2] - mm);
            ll = fmaf(ml[(w * 16 + r) * 2 + 1], f, ll);
            if (f != 0.f) a = fmaf(mo[(w * 16 + r) * DV + c], f, a);
        }
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        const long row = sq.q0 + r / p.G;
        const int h = g * p.G + r % p.G;
        const long at = row * p.nh + h;
        if (p.nsplit > 1) {
            if (ch < p.hd) p.part_o[((long)split * p.q_rows * p.nh + at) * p.hd + ch] = ll == 0.f ? 0.f : a * inv;
        } else {
            if (ch < p.hd) stf((bf16_t*)p.out + row * p.ldo + (long)h * p.hd, ch, ll == 0.f ? 0.f : a * inv);
        }
        if (c == 0 && half == 0) {
            const float lse = ll == 0.f ? -INFINITY : (mm + log2f(ll)) * 0.6931471805599453f;
            if (p.nsplit > 1)
                p.part_lse[(long)split * p.q_rows * p.nh + at] = lse;
            else if (p.lse)
                p.lse[at] = lse;
        }
    }
}

template <int HD>
static int launch_masked_few(const MaskedParams& p, cudaStream_t s) {
    using Cfg = AmfCfg<HD>;
    auto kern = attention_masked_few_kernel<HD>;
    const int smem = Cfg::SMEM + (p.part + 31) / 32 * 4;
    if (smem > 227 * 1024) return -1;
    static bool attr_set[64] = {false};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
    if (!attr_set[dev]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess) return -3;
        attr_set[dev] = true;
    }
    CUtensorMap mk, mv;
    const CUtensorMapDataType dt = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    if (make_tmap_3d(&mk, dt, p.k, p.hd, p.nkv, p.k_rows, (uint64_t)p.hd * 2, (uint64_t)p.ldk * 2, 64, 1, 16) ||
        make_tmap_3d(&mv, dt, p.v, p.hd, p.nkv, p.k_rows, (uint64_t)p.hd * 2, (uint64_t)p.ldv * 2, 64, 1, 16))
        return -1;
    const long units = (long)p.n_seq * p.nkv * Cfg::HALVES;
    if (units > 0x7fffffffL || p.nsplit > 65535) return -1;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)units, (unsigned)p.nsplit, 1);
    cfg.blockDim = dim3(32 * Cfg::WARPS, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, mk, mv, p) == cudaSuccess ? 0 : -3;
}
