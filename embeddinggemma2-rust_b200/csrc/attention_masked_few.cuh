// The form of masked attention for few query rows over many keys (bf16), included by attention_masked.cu.
//
// At most 16 rows (query tokens x the G heads of a K/V head): the work is to read K and V once, so the design is for
// bytes in flight and a short path per byte, not for tensor throughput -- warp-level mma.sync with the 16 rows as M.
// (One token of 4 heads over 2 of 256 for each of 8 documents of up to 11,774 cached keys: 33 us, 3.4 TB/s; 4 queries over
// 30,000 keys, 4 heads over 2 of 128, a window of 20,000: 26 us, 30 in the 128-row tiles of the tcgen05 form, whose first tiles wait for
// their instructions.)
//
// A CTA takes one part of the keys of one (sequence, K/V head, 256-channel half of O); each of its warps walks blocks
// of 16 keys on its own, with a ring of its own that one lane fills by TMA, 16 keys x 64 channels a box, and its own
// running maximum, sum and O in registers. The warps' results are joined through shared memory at the end. Blocks that
// no row may see, by range or by document, are not loaded.

template <int HD>
struct AmfCfg {
    static constexpr int DV = HD < 256 ? HD : 256, HALVES = HD / DV;
    static constexpr int WARPS = 4, CTAS = HD == 512 ? 1 : 2;  // CTAs per SM
    // Slots of 16 keys per warp; two CTAs of an SM then have about 128 KB under way.
    static constexpr int KS = HD == 64 ? 6 : HD == 128 ? 3 : 2, VS = HD == 256 ? 1 : KS;
    static constexpr int K_BYTES = 16 * HD * 2, V_BYTES = 16 * DV * 2, RING = KS * K_BYTES + VS * V_BYTES;
    static constexpr int OFF_RING = 16 * HD * 2;  // after Q
    static constexpr int OFF_BAR = OFF_RING + WARPS * RING;
    static constexpr int OFF_BLOCKS = OFF_BAR + WARPS * (KS + VS) * 8;  // bit mask of the part's blocks
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
__global__ void __launch_bounds__(32 * AmfCfg<HD>::WARPS, AmfCfg<HD>::CTAS)
    attention_masked_few_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                                const __grid_constant__ MaskedParams p) {
    using Cfg = AmfCfg<HD>;
    constexpr int DV = Cfg::DV, WARPS = Cfg::WARPS, KS = Cfg::KS, VS = Cfg::VS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
    uint32_t* blocks = reinterpret_cast<uint32_t*>(smem + Cfg::OFF_BLOCKS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int x = 0; x < WARPS * (KS + VS); x++) mbar_init(&bars[x], 1);
        fence_mbarrier_init();
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    __syncthreads();
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
    if (p.nsplit > 1 && first == last) {  // a short sequence's later parts: their slot on the SM is wanted
        if (half == 0 && (int)threadIdx.x < rows)
            p.part_ml[((long)split * p.q_rows + sq.q0 + threadIdx.x / p.G) * p.nh + g * p.G + threadIdx.x % p.G] = make_float2(AMT_NONE, 0.f);
        return;
    }

    if (p.q_doc)
        for (int w = threadIdx.x; w < words; w += blockDim.x) blocks[w] = 0u;
    if (p.q_doc) __syncthreads();
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
    // This warp takes every WARPS-th block, with documents of the marked ones, the warp-th first. -1: none is left.
    int at_word = 0, at_block = first + warp - WARPS;
    uint32_t left = p.q_doc && words ? blocks[0] : 0u;
    auto next_block = [&](int skip) -> int {
        if (!p.q_doc) {
            at_block += WARPS;
            return at_block < last ? at_block : -1;
        }
        for (; words; skip--) {
            while (!left) {
                if (++at_word >= words) return -1;
                left = blocks[at_word];
            }
            const int bit = __ffs(left) - 1;
            left &= left - 1u;
            if (!skip) return first + at_word * 32 + bit;
        }
        return -1;
    };
    uint8_t* k_ring = smem + Cfg::OFF_RING + warp * Cfg::RING;
    uint8_t* v_ring = k_ring + KS * Cfg::K_BYTES;
    uint64_t* k_full = bars + warp * (KS + VS);
    uint64_t* v_full = k_full + KS;
    int queue[KS], k_issued = 0, v_issued = 0;  // the warp's n-th block, at n % KS
    auto issue_k = [&](int blk) {
        const int st = k_issued % KS;
        if (lane == 0) {
            mbar_arrive_expect_tx(&k_full[st], Cfg::K_BYTES);
            for (int c = 0; c < HD / 64; c++) tma_load_3d(k_ring + st * Cfg::K_BYTES + c * 2048, &tmK, &k_full[st], 64 * c, g, (int)sq.k0 + blk * 16);
        }
        k_issued++;
    };
    auto issue_v = [&](int blk) {
        const int st = v_issued % VS;
        if (lane == 0) {
            mbar_arrive_expect_tx(&v_full[st], Cfg::V_BYTES);
            for (int c = 0; c < DV / 64; c++)
                tma_load_3d(v_ring + st * Cfg::V_BYTES + c * 2048, &tmV, &v_full[st], half * 256 + 64 * c, g, (int)sq.k0 + blk * 16);
        }
        v_issued++;
    };
    auto queued = [&](int n) -> int {
        int blk = queue[0];
#pragma unroll
        for (int x = 1; x < KS; x++)
            if (n % KS == x) blk = queue[x];
        return blk;
    };
    int blk = next_block(warp);
#pragma unroll
    for (int st = 0; st < KS; st++) {
        queue[st] = blk;
        if (blk >= 0) {
            issue_k(blk);
            if (st < VS) issue_v(blk);
            blk = next_block(WARPS - 1);
        }
    }

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
    // Q, while the first blocks are under way.
    for (int x = threadIdx.x; x < 16 * HD / 8; x += blockDim.x) {
        const int r = x / (HD / 8), c = x % (HD / 8) * 8;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (r < rows && c < p.hd)
            v = *reinterpret_cast<const uint4*>((const bf16_t*)p.q + (sq.q0 + r / p.G) * p.ldq + (long)(g * p.G + r % p.G) * p.hd + c);
        *reinterpret_cast<uint4*>(smem + amf_at(r, c)) = v;
    }
    __syncthreads();

    const bool capped = p.softcap > 0.f;
    const float in_scale = capped ? p.scale / p.softcap : p.scale * AMT_LOG2E, cap2 = p.softcap * AMT_LOG2E;
    float m[2] = {AMT_NONE, AMT_NONE}, l[2] = {0.f, 0.f};
    float o[DV / 8][4];
#pragma unroll
    for (int c = 0; c < DV / 8; c++)
#pragma unroll
        for (int x = 0; x < 4; x++) o[c][x] = 0.f;
    // ldmatrix addresses within a 64-channel chunk, by step of 16 channels: Q and V take rows (or keys) 0-7 / 8-15 by bit 3 of the
    // lane and channels 0-7 / 8-15 by bit 4, K the other way round.
    uint32_t q_off[4], k_off[4];
#pragma unroll
    for (int c = 0; c < 4; c++) {
        q_off[c] = amf_at((lane & 7) + 8 * ((lane >> 3) & 1), 16 * c + 8 * (lane >> 4));
        k_off[c] = amf_at((lane & 7) + 8 * (lane >> 4), 16 * c + 8 * ((lane >> 3) & 1));
    }
    const uint32_t q_addr = smem_u32(smem);
    // Keys that every row sees.
    int all_lo = 0, all_hi = sq.nk;
    masked_range(p, sq, sq.nk - 1, all_lo, tmp);
    masked_range(p, sq, sq.nk - sq.nq, tmp, all_hi);
    bool ok = true;
    int taken = 0;
    while (true) {
        const int now = queued(taken);
        if (now < 0) break;
        const int key0 = now * 16;
        // Document ids of this thread's four columns, under the latency of the block.
        int ids[4] = {0, 0, 0, 0};
        if (p.k_doc) {
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const int key = key0 + 8 * (x >> 1) + 2 * (lane & 3) + (x & 1);
                ids[x] = key < sq.nk ? p.k_doc[sq.k0 + key] : 0;
            }
        }
        if (!(ok = mbar_wait(&k_full[taken % KS], (taken / KS) & 1, EG2_DEV_TIMEOUT_ATTN, nullptr))) break;
        const uint32_t k_addr = smem_u32(k_ring + (taken % KS) * Cfg::K_BYTES);
        uint8_t* vb = v_ring + (taken % VS) * Cfg::V_BYTES;
        const uint32_t v_addr = smem_u32(vb);
        float s[2][4] = {};
#pragma unroll 1
        for (int c0 = 0; c0 < HD / 64; c0++) {
            // Four steps of 16 channels: their eight loads are under way together.
            uint32_t qa[4][4], kf[4][4];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                ldmatrix4(q_addr + c0 * 2048 + q_off[c], qa[c]);
                ldmatrix4(k_addr + c0 * 2048 + k_off[c], kf[c]);
            }
#pragma unroll
            for (int c = 0; c < 4; c++) {
                mma_16816(s[0], qa[c], kf[c][0], kf[c][1]);
                mma_16816(s[1], qa[c], kf[c][2], kf[c][3]);
            }
        }
        __syncwarp();  // the K slot has been read
#pragma unroll
        for (int x = 0; x < KS; x++)
            if (taken % KS == x) queue[x] = blk;
        if (blk >= 0) {
            issue_k(blk);
            blk = next_block(WARPS - 1);
        }
        // Scores in the log2 domain: s[y / 2][2 x + y % 2] is row x, column y of this thread's.
        float v[8];
#pragma unroll
        for (int x = 0; x < 8; x++) v[x] = s[(x >> 1) & 1][2 * (x >> 2) + (x & 1)] * in_scale;
        if (capped) {
#pragma unroll
            for (int x = 0; x < 8; x++) v[x] = cap2 * tanh_any(v[x]);
        }
        const int col0 = key0 + 2 * (lane & 3);
        if (p.slopes) {
#pragma unroll
            for (int x = 0; x < 8; x++) v[x] = fmaf(-slope[x >> 2], fabsf((float)(col0 + 8 * ((x >> 1) & 1) + (x & 1) - place[x >> 2])), v[x]);
        }
        uint32_t unseen = 0u;  // of this thread's eight scores
        if (p.table) {
#pragma unroll
            for (int x = 0; x < 8; x++) {
                const float bias = masked_table(p, head[x >> 2], col0 + 8 * ((x >> 1) & 1) + (x & 1) - place[x >> 2]);
                v[x] = fmaf(bias, AMT_LOG2E, v[x]);
                unseen |= bias == -INFINITY ? 1u << x : 0u;
            }
        }
        if (p.k_doc || key0 < all_lo || key0 + 16 > all_hi) {
#pragma unroll
            for (int x = 0; x < 8; x++) {
                const int key = col0 + 8 * ((x >> 1) & 1) + (x & 1), y = x >> 2;
                const bool seen = key >= lo[y] && key < hi[y] && (!p.k_doc || ids[x & 3] == qdoc[y]);
                unseen |= seen ? 0u : 1u << x;
            }
        }
        bool hidden = false;  // some key is hidden from some row
        if (unseen) {
#pragma unroll
            for (int x = 0; x < 8; x++) {
                if ((unseen >> x) & 1u) {
                    v[x] = -INFINITY;
                    hidden |= (lane >> 2) + 8 * (x >> 2) < rows;
                }
            }
        }
        float top[2];
#pragma unroll
        for (int x = 0; x < 2; x++) top[x] = fmaxf(fmaxf(fmaxf(v[4 * x], v[4 * x + 1]), fmaxf(v[4 * x + 2], v[4 * x + 3])), AMT_NONE);
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
                v[4 * x + y] = ex2_approx(v[4 * x + y] - mn);
                l[x] += v[4 * x + y];
            }
            pa[x] = bf16x2_bits(v[4 * x], v[4 * x + 1]);
            pa[2 + x] = bf16x2_bits(v[4 * x + 2], v[4 * x + 3]);
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
        if (!(ok = mbar_wait(&v_full[taken % VS], (taken / VS) & 1, EG2_DEV_TIMEOUT_ATTN, nullptr))) break;
        if (__any_sync(0xffffffffu, hidden)) {
            // A hidden key's value may be anything, and 0 x NaN must not reach the sum: elements that are not finite become
            // zero, after the rows that do see the key have taken them.
            uint32_t bad = 0;  // keys
            for (int x = lane; x < 16 * DV / 8; x += 32) {
                const int key = x / (DV / 8), c = x % (DV / 8) * 8;
                const uint4 e = *reinterpret_cast<const uint4*>(vb + amf_at(key, c));
                const uint32_t w[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
                for (int y = 0; y < 4; y++)
                    if ((w[y] & 0x7f80u) == 0x7f80u || (w[y] & 0x7f800000u) == 0x7f800000u) bad |= 1u << key;
            }
            bad = __reduce_or_sync(0xffffffffu, bad);
            for (; bad; bad &= bad - 1u) {
                const int key = __ffs(bad) - 1;
                const int src = (lane & ~3) + ((key & 7) >> 1);  // who holds this key's weights of my rows
                float w0 = 0.f, w1 = 0.f;
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    const float a0 = __shfl_sync(0xffffffffu, v[y], src), a1 = __shfl_sync(0xffffffffu, v[4 + y], src);
                    if (y == 2 * (key >> 3) + (key & 1)) w0 = a0, w1 = a1;
                }
                const uint32_t not_seen = __shfl_sync(0xffffffffu, unseen, src) >> (2 * (key >> 3) + (key & 1));
#pragma unroll
                for (int c = 0; c < DV / 8; c++)
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        const float e = bf16_to_f32(*reinterpret_cast<const bf16_t*>(vb + amf_at(key, 8 * c + 2 * (lane & 3) + y)));
                        if (!(fabsf(e) < INFINITY)) {
                            if (!(not_seen & 1u)) o[c][y] = fmaf(w0, e, o[c][y]);
                            if (!(not_seen & 16u)) o[c][2 + y] = fmaf(w1, e, o[c][2 + y]);
                        }
                    }
                __syncwarp();
                for (int c = lane; c < DV; c += 32) {
                    bf16_t* e = reinterpret_cast<bf16_t*>(vb + amf_at(key, c));
                    if ((*e & 0x7f80u) == 0x7f80u) *e = 0;
                }
                __syncwarp();
            }
        }
#pragma unroll
        for (int c0 = 0; c0 < DV / 64; c0++) {
            uint32_t vf[4][4];
#pragma unroll
            for (int c = 0; c < 4; c++) ldmatrix4_trans(v_addr + c0 * 2048 + q_off[c], vf[c]);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                mma_16816(o[8 * c0 + 2 * c], pa, vf[c][0], vf[c][1]);
                mma_16816(o[8 * c0 + 2 * c + 1], pa, vf[c][2], vf[c][3]);
            }
        }
        fence_proxy_async();  // the cleaning's writes come before the next load's
        __syncwarp();         // the V slot has been read
        const int then = queued(taken + VS);
        taken++;
        if (then >= 0) issue_v(then);
    }
    // No load may land after the CTA has ended (on the error path; else all have been waited for).
    if (!ok && lane == 0) {
        for (int x = max(0, k_issued - KS); x < k_issued; x++) mbar_drain(&k_full[x % KS], (x / KS) & 1, 200000000ull);
        for (int x = max(0, v_issued - VS); x < v_issued; x++) mbar_drain(&v_full[x % VS], (x / VS) & 1, 200000000ull);
    }
#pragma unroll
    for (int x = 0; x < 2; x++) {
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    }
    // ---- the warps' results, joined in warp order ----
    __syncthreads();
    float* mo = reinterpret_cast<float*>(smem + Cfg::OFF_RING);  // [WARPS][16][DV]
    float* ml = reinterpret_cast<float*>(smem);                  // [WARPS][16][2]: over Q
    static_assert(WARPS * 16 * DV * 4 <= WARPS * Cfg::RING && WARPS * 16 * 8 <= 16 * HD * 2, "few rows: shared memory of the join");
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
            const float f = ex2_approx(ml[(w * 16 + r) * 2] - mm), lw = ml[(w * 16 + r) * 2 + 1];
            ll = fmaf(lw, f, ll);
            if (lw != 0.f) a = fmaf(mo[(w * 16 + r) * DV + c], f, a);  // also where f has vanished: the sum may not be finite
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
            if (p.nsplit > 1)
                p.part_ml[(long)split * p.q_rows * p.nh + at] = make_float2(mm, ll);
            else if (p.lse)
                p.lse[at] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) * 0.6931471805599453f;
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
