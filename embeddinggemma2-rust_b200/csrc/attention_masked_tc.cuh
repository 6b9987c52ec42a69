// The tensor-core form of masked attention (bf16), included by attention_masked.cu.
//
// A CTA holds a query tile of 128 rows -- row r is token r / G, head r % G of the G query heads that share a K/V
// head, so a K/V tile serves all of them -- and walks 128-key tiles: S = Q K^T into TMEM, a softmax warpgroup turns
// S into P (bf16, written over its S), O += P V. Two softmax warpgroups take turns, one key tile each: while one
// turns scores into weights (ex2 on the XU pipe, 8 cycles a warp) the other caps, biases and masks its tile (FMA
// and ALU pipes). A thread holds one row; the running maximum of the row goes from one group to the other through
// shared memory as soon as it is known. Persistent: one CTA per SM takes units (query tile, sequence, K/V head,
// 256-channel half of O, part of the key axis), the heavy ones (last queries under a causal mask) first.
//
// TMEM: NS S buffers of 128 columns by tile, then O. Heads up to 128 have room for three, so S(T + 2) does not wait
// for P(T) V; 256 and 512 for two (O takes 256 columns, at 512 channels by halves, each half with the whole S).
//
//   warp 0      TMA producer: Q, then K(0), K(1), V(0), K(2), V(1), ... into a ring of K and one of V units (one
//               consumer each: a wait names only the parity of a barrier's phase, so whoever waits for a unit must
//               have taken the one before it in its slot)
//   warp 1      TMEM allocation; lane 0 issues S = Q K^T
//   warp 2      lane 0 issues O += P V; the warp cleans V tiles (below)
//   warp 3      scout: describes the next unit (double-buffered): the key tiles that some row may see, and those
//               that need the document ids row by row, from the ranges of ids in the tile
//   warps 4-11  softmax and the O / l epilogue
//
// Bound by the latency of the softmax at heads 64 and 128 (two warps a scheduler, which issue in 43 % of the cycles and wait for fixed
// latencies, TMEM and instructions in the rest; no pipe is past 55 %), by products and their loads at 256 and 512, whose rings hold two
// units and less than a tile: 12,001 tokens under a causal mask with a prefix, capped, with slopes, 8 heads over 2 of 128: 622 us; 8,192
// tokens without a mask 290 us, 948 TFLOP/s.
//
// The score of a pair lives in the log2 domain (scale, cap and biases carry log2 e), so a weight is one FMA and
// one ex2. O is rescaled only when a row's maximum grows by more than 2^8: a stale maximum is exact. l sums the
// weights in f32 as they are, P rounds them to bf16: the product with V takes 16-bit operands, and 2^-8 of a weight
// is what the 16-bit result carries anyway.
//
// Hidden keys are masked by selection, so what K holds there is harmless, but a NaN or infinity in a hidden V row
// would reach the sum as 0 x NaN. Rows past the sequence's end are zeroed in shared memory by the P V warp. Other
// hidden rows are taken to be finite; a unit with masked tiles whose result is not finite is run again in stages
// (AmtUnit::stage): once with the elements of V that are not finite set to 0, which gives every row its finite sum, then
// twice over the tiles that held such elements, with 1 for each of them in V and 1 for each visible key in P: where this
// product is positive the row sees an infinity of that sign, or a NaN, in that channel, and takes it. So no visible bit
// depends on what hidden keys hold, at no cost while all is finite; where it is not, a unit's time grows by its one
// repetition and the tiles concerned, whatever their number, never by rows taken one by one (8,192 tokens, 8 heads over 2 of 128: causal 139 us, with
// one NaN 728, with NaN alone 3,011; with 40 NaN rows of a hidden document 322 and 1,140).

constexpr int AMT_THREADS = 384;
constexpr int AMT_MASK_WORDS = EG2_MASKED_MAX_LEN / 128 / 32;
constexpr int AMT_TABLE = 4096;  // floats of distance bias in shared memory
constexpr float AMT_LOG2E = 1.4426950408889634f;
constexpr float AMT_NONE = -3e38f;  // the maximum of a row that has seen nothing

struct alignas(16) AmtUnit {
    MaskedSeq sq;
    int t0, rows;     // first token of the tile; rows with a query
    int g, head0;     // K/V head; first query head
    int split, half;  // part of the key axis; 256-channel half of O
    int n, first;     // key tiles to visit; the first (without documents they are consecutive,
    int down;         // and the first `down` of them are visited backwards)
    int sparse;       // the tiles are those of `visit`
    int stop;         // no further unit
    int stage;        // 0 as it is; 1 elements of V that are not finite count as 0; 2, 3 as 1 if +infinity (2), -infinity (3)
                      // or NaN, else 0, under weights of 1
    int retry;        // (set by the softmax in stage 0) run again
    int masked;       // (set by the softmax) some tile was masked
    int found;        // (set by the P V warp in stage 1) some element was not finite: in the tiles of `bad`
    uint32_t visit[AMT_MASK_WORDS], docs[AMT_MASK_WORDS], bad[AMT_MASK_WORDS];
};

struct AmtParams {
    MaskedParams p;
    int Gt;              // query heads packed into a tile (G or 1)
    int q_tiles, heads;  // tiles per sequence; K/V heads x (G / Gt)
    int n_units;
    int out32;           // rows of out start at multiples of 32 bytes, heads are multiples of 16 channels
};

template <int HD>
struct AmtCfg {
    static constexpr int R_AUX = HD <= 128 ? 56 : 72, R_SOFT = HD <= 128 ? 224 : 216;  // registers (measured: 2 % to 8 % either way)
    static constexpr int QCH = HD / 64;                   // 16 KB chunks of Q
    static constexpr int QBUF = HD <= 128 ? 2 : 1;        // Q buffers: the next unit's Q lands under this one
    static constexpr int UCH = HD == 128 || HD == 256 ? 2 : 1;  // 64-channel chunks per ring unit (128 keys each)
    static constexpr int UNIT = UCH * 16384;
    static constexpr int DV = HD < 256 ? HD : 256;        // O channels per CTA
    static constexpr int HALVES = HD / DV;
    static constexpr int KU = HD / (64 * UCH), VU = DV / (64 * UCH);  // ring units per K / V tile
    static constexpr int RING = HD == 64 ? 4 : 2;         // units of the K ring, and of the V ring
    static constexpr int NS = HD <= 128 ? 3 : 2;          // S buffers
    // The producer of head 512, whose rings hold a fraction of a tile, loads whichever of K and V has room (954 us against
    // 1,254 for 8,192 tokens, 4 heads); elsewhere it waits in order: its polling took issue slots from the softmax (320 -> 350 us
    // at head 128).
    static constexpr bool POLL = HD == 512;
    static constexpr int T_O = 128 * NS;
    static constexpr int OC = DV / 2;                     // O columns per thread in the epilogue
    static constexpr int OFF_R = QBUF * QCH * 16384;
    static constexpr int OFF_V = OFF_R + RING * UNIT;
    static constexpr int OFF_UNIT = OFF_V + RING * UNIT;
    static constexpr int OFF_X = OFF_UNIT + 2 * (int)sizeof(AmtUnit);  // running maxima [2 groups][128]; (maximum, sum) [2][2 groups][128]
    static constexpr int OFF_TAB = OFF_X + 2048 + 4096;
    static constexpr int OFF_BAR = OFF_TAB + AMT_TABLE * 4;
    static constexpr int N_BARS = 4 + 2 * QBUF + 4 * RING + 3 * NS + 1 + 4 + 2 + 2;
    static constexpr int SMEM = 1024 + OFF_BAR + N_BARS * 8 + 16;
};
static_assert(AmtCfg<64>::SMEM <= 227 * 1024 && AmtCfg<128>::SMEM <= 227 * 1024 && AmtCfg<256>::SMEM <= 227 * 1024 &&
                  AmtCfg<512>::SMEM <= 227 * 1024,
              "masked attention: shared memory");

EG2_DEV uint64_t f2_pack(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
EG2_DEV void f2_unpack(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
EG2_DEV uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
EG2_DEV uint64_t f2_mul(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
EG2_DEV uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// tanh on |x| <= 0.5: x P(x^2), minimax in relative error (3e-8 with these coefficients in f32), found by reweighted
// least squares. Relative, because a small score's cap must not cost it digits.
constexpr float AMT_TANH_MAX = 0.5f;
constexpr float AMT_T0 = 1.f, AMT_T1 = -0.3333306908607483f, AMT_T2 = 0.13324779272079468f, AMT_T3 = -0.05298607423901558f,
                AMT_T4 = 0.017135003581643105f;
// Arrive on `bar` from one lane of a converged warp, without a branch.
EG2_DEV void mbar_arrive_if(uint64_t* bar, bool pred) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 st;\n\tsetp.ne.b32 p, %1, 0;\n\t"
        "@p mbarrier.arrive.shared::cta.b64 st, [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"((int)pred)
        : "memory");
}
EG2_DEV bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
EG2_DEV float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// tanh past 0.5 as 1 - 2 / (1 + e^2x), good to 2^-21 there (1 where e^2x overflows); anywhere.
EG2_DEV float tanh_far(float x) { return 1.f - __fdividef(2.f, 1.f + ex2_approx(2.f * AMT_LOG2E * x)); }
EG2_DEV float tanh_any(float x) {
    const float y = x * x;
    const float near = x * fmaf(fmaf(fmaf(fmaf(AMT_T4, y, AMT_T3), y, AMT_T2), y, AMT_T1), y, AMT_T0);
    return fabsf(x) <= AMT_TANH_MAX ? near : tanh_far(x);
}

// The set bits of a mask, in order.
struct BitWalk {
    const uint32_t* w;
    int at;
    uint32_t cur;
    EG2_DEV explicit BitWalk(const uint32_t* words) : w(words), at(0), cur(words ? words[0] : 0u) {}
    EG2_DEV int next() {  // there is one
        while (!cur && at + 1 < AMT_MASK_WORDS) cur = w[++at];
        const int b = __ffs(cur) - 1;
        cur &= cur - 1;
        return at * 32 + b;
    }
};

// A unit's key tiles in the order all roles take them.
struct TileWalk {
    BitWalk bits;
    bool sparse;
    int first, down, j;
    EG2_DEV TileWalk() : bits(nullptr), sparse(false), first(0), down(0), j(0) {}
    EG2_DEV explicit TileWalk(const AmtUnit& u) : bits(u.visit), sparse(u.sparse != 0), first(u.first), down(u.down), j(0) {}
    EG2_DEV int next() {
        const int i = j++;
        return sparse ? bits.next() : first + (i < down ? down - 1 - i : i);
    }
};

// Prepares one 16 KB chunk of a V tile (128 keys of 128 bytes, whatever the order of the 16-byte units in a row) for the
// unit's stage; rows from `live` on become zero. Whether some other element was not finite, in the whole warp. Looks before it writes:
// most chunks have none, and loads alone are under way together.
EG2_DEV bool guard_chunk(uint8_t* chunk, int live, int stage) {
    const int lane = threadIdx.x & 31;
    uint4* const units = reinterpret_cast<uint4*>(chunk);
    // Top bits of the halves whose exponent is full.
    auto odd_halves = [](uint32_t w) -> uint32_t { return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; };
    const int end = 8 * max(min(live, 128), 0);
    bool hit = false;
    if (stage) {
        uint32_t odd = 0u;
#pragma unroll 4
        for (int x = lane; x < 1024; x += 32) {
            const uint4 v = units[x];
            const uint32_t o = odd_halves(v.x) | odd_halves(v.y) | odd_halves(v.z) | odd_halves(v.w);
            odd |= x < end ? o : 0u;
        }
        hit = __any_sync(0xffffffffu, odd != 0u);
    }
    if (hit || stage > 1) {
#pragma unroll 1
        for (int x = lane; x < end; x += 32) {
            const uint4 v = units[x];
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
            // Past stage 1 an infinity of the other sign is not meant.
            const uint32_t other = stage == 2 ? 0xff80u : 0x7f80u;
#pragma unroll
            for (int y = 0; y < 4; y++) {
                uint32_t odd = odd_halves(w[y]);
                if (stage > 1) odd &= ((w[y] & 0xffffu) == other ? 0u : 0x8000u) | ((w[y] >> 16) == other ? 0u : 0x80000000u);
                const uint32_t ones = odd >> 15;  // 1 in each half that counts
                w[y] = stage == 1 ? w[y] & ~(ones * 0xffffu) : ones * 0x3f80u;
            }
            units[x] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    for (int x = end + lane; x < 1024; x += 32) units[x] = make_uint4(0u, 0u, 0u, 0u);
    return hit;
}

// The columns of a tile that the staged table hides; a call, since it is rare and the loop over scores is faster without its code.
__device__ __noinline__ uint4 masked_hidden_columns(const float* table) {
    uint4 h = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 1
    for (int c = 0; c < 32; c++) {
        if (table[c] == -INFINITY) h.x |= 1u << c;
        if (table[32 + c] == -INFINITY) h.y |= 1u << c;
        if (table[64 + c] == -INFINITY) h.z |= 1u << c;
        if (table[96 + c] == -INFINITY) h.w |= 1u << c;
    }
    return h;
}

// A softmax warp's part of a unit in stages 2 and 3: weights of 1 for the visible keys of its group's tiles, then, where the
// product is positive, the infinity to the sums that stage 1 wrote (of both signs, or with a NaN, they make NaN). False where a
// wait ran out.
template <int HD, bool TABLES>
EG2_DEV bool masked_count_unit(const AmtParams& ap, const AmtUnit& u, uint32_t tmem, int T, int U, uint64_t* s_full, uint64_t* p_full,
                               uint64_t* pv_done, uint64_t* o_empty, uint64_t* e_bar, volatile int* abort_flag) {
    using Cfg = AmtCfg<HD>;
    constexpr int NS = Cfg::NS;
    const MaskedParams& p = ap.p;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, e = warp & 3, wg = (warp - 4) >> 2, r = 32 * e + lane;
    const uint32_t mine = tmem + ((uint32_t)(32 * e) << 16);
    const bool live = r < u.rows;
    const int t = u.t0 + r / ap.Gt, head = u.head0 + r % ap.Gt;
    const long row = u.sq.q0 + t;
    int lo = 0, hi = 0;
    const int place = u.sq.nk - u.sq.nq + t;
    if (live) masked_range(p, u.sq, place, lo, hi);
    const int qdoc = live && p.q_doc ? p.q_doc[row] : 0;
    TileWalk walk(u);
    bool ok = true;
    for (int j = 0; j < u.n; j++) {
        const int kbase = walk.next() * 128, buf = (T + j) % NS;
        if (((T + j) & 1) != wg) continue;
        ok = mbar_wait(&s_full[buf], ((T + j) / NS) & 1, EG2_DEV_TIMEOUT_ATTN, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) return false;
        tc_fence_after();
        const bool docs = p.q_doc && ((u.docs[kbase >> 12] >> ((kbase >> 7) & 31)) & 1u);
#pragma unroll 1
        for (int x = 0; x < 128; x += 32) {
            const int a = min(max(lo - kbase - x, 0), 32), z = min(max(hi - kbase - x, 0), 32);
            uint32_t seen = z > a ? (0xffffffffu >> (32 - z)) & (0xffffffffu << a) : 0u, pk[16];
            if (docs || (TABLES && p.table))
                for (uint32_t left = seen; left; left &= left - 1u) {
                    const int key = kbase + x + __ffs(left) - 1;
                    if ((docs && p.k_doc[u.sq.k0 + key] != qdoc) || (TABLES && p.table && masked_table(p, head, key - place) == -INFINITY))
                        seen &= ~(left & (~left + 1u));
                }
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 16; q++) pk[q] = ((seen >> (2 * q)) & 1u ? 0x3f80u : 0u) | ((seen >> (2 * q + 1)) & 1u ? 0x3f800000u : 0u);
            tmem_st16(mine + 128 * buf + x / 2, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        mbar_arrive_if(&p_full[buf], lane == 0);
    }
    // The group of the last tile has seen its S, so that pv_done below is in that tile's phase or past it.
    const int last = T + u.n - 1;
    mbar_arrive_if(&e_bar[e], lane == 0);
    ok = mbar_wait(&e_bar[e], U & 1, EG2_DEV_TIMEOUT_ATTN, abort_flag);
    if (!__all_sync(0xffffffffu, ok)) return false;
    ok = mbar_wait(&pv_done[last % NS], (last / NS) & 1, EG2_DEV_TIMEOUT_ATTN, abort_flag);
    if (!__all_sync(0xffffffffu, ok)) return false;
    tc_fence_after();
    const float inf = u.stage == 2 ? INFINITY : -INFINITY;
    const long at = row * p.nh + head + (p.nsplit > 1 ? (long)u.split * p.q_rows * p.nh : 0);
#pragma unroll 1
    for (int c = 0; c < Cfg::OC; c += 16) {
        uint32_t o[16], hit = 0u;
        tmem_ld16(mine + Cfg::T_O + wg * Cfg::OC + c, o);
        tmem_ld_wait();
        reg_fence<16>(o);
#pragma unroll
        for (int q = 0; q < 16; q++) hit |= live && __uint_as_float(o[q]) > 0.f ? 1u << q : 0u;
        for (; hit; hit &= hit - 1u) {
            const int ch = u.half * 256 + wg * Cfg::OC + c + __ffs(hit) - 1;
            if (p.nsplit > 1) {
                p.part_o[at * p.hd + ch] += inf;
            } else {
                bf16_t* out = (bf16_t*)p.out + row * p.ldo + (long)head * p.hd;
                stf(out, ch, ldf(out, ch) + inf);
            }
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncwarp();
    mbar_arrive_if(o_empty, lane == 0);
    return true;
}

// The same as a call or as code of the kernel: the loop over scores does not use it, but its speed goes by what else is compiled into the
// kernel. 8,192 tokens, as a call / inlined (12 heads of 64, 8 over 2 of 128, 4 over 2 of 256): plain 420 / 389, 352 / 291 and 285 / 293 us,
// a table 561 / 594, 442 / 498 and 377 / 348, capped 633 / 655, 483 / 483 and 348 / 367. As a branch inside the loop 372 at head 128, plain.
template <int HD, bool TABLES>
__device__ __noinline__ bool masked_count_call(const AmtParams& ap, const AmtUnit& u, uint32_t tmem, int T, int U, uint64_t* s_full,
                                               uint64_t* p_full, uint64_t* pv_done, uint64_t* o_empty, uint64_t* e_bar, volatile int* abort_flag) {
    return masked_count_unit<HD, TABLES>(ap, u, tmem, T, U, s_full, p_full, pv_done, o_empty, e_bar, abort_flag);
}
template <int HD, bool TABLES>
EG2_DEV bool masked_count(const AmtParams& ap, const AmtUnit& u, uint32_t tmem, int T, int U, uint64_t* s_full, uint64_t* p_full,
                          uint64_t* pv_done, uint64_t* o_empty, uint64_t* e_bar, volatile int* abort_flag) {
    if constexpr (HD == 512 || (HD <= 128 && !TABLES))
        return masked_count_unit<HD, TABLES>(ap, u, tmem, T, U, s_full, p_full, pv_done, o_empty, e_bar, abort_flag);
    else
        return masked_count_call<HD, TABLES>(ap, u, tmem, T, U, s_full, p_full, pv_done, o_empty, e_bar, abort_flag);
}

// The score's parts that a kernel is compiled for; AMT_ANY decides at run time. The softmax is long straight code, and what
// a call does not need costs it instruction fetches. 8,192 tokens, 12 heads of 64 / 8 over 2 of 128 / 4 over 2
// of 256, decided at run time and compiled for the call: plain 471 / 373 / 301 and 393 / 295 / 287 us, capped 743 / 543 / 381 and 655 / 489 / 352, slopes
// 619 / 455 / 358 and 526 / 414 / 328, a table 652 / 496 / 395 and 571 / 432 / 345. `raw` below stays a test at run time in
// each: with it known, the compiler mixes the parts with the mask's code and spills (table 588 / 560 / 378 us).
constexpr int AMT_CAP = 1, AMT_SLOPES = 2, AMT_TAB = 4, AMT_ANY = 8;

template <int HD, int PARTS>
__global__ void __launch_bounds__(AMT_THREADS, 1)
    attention_masked_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                               const __grid_constant__ CUtensorMap tmV, const __grid_constant__ AmtParams ap) {
    using Cfg = AmtCfg<HD>;
    constexpr int RING = Cfg::RING, KU = Cfg::KU, VU = Cfg::VU, NS = Cfg::NS, QBUF = Cfg::QBUF;
    const MaskedParams& p = ap.p;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    AmtUnit* units = reinterpret_cast<AmtUnit*>(smem + Cfg::OFF_UNIT);
    uint64_t* unit_full = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
    uint64_t* unit_empty = unit_full + 2;
    uint64_t* q_full = unit_empty + 2;
    uint64_t* q_empty = q_full + QBUF;
    uint64_t* k_full = q_empty + QBUF;
    uint64_t* k_empty = k_full + RING;
    uint64_t* v_full = k_empty + RING;
    uint64_t* v_empty = v_full + RING;
    uint64_t* s_full = v_empty + RING;  // [NS]
    uint64_t* p_full = s_full + NS;
    uint64_t* pv_done = p_full + NS;
    uint64_t* o_empty = pv_done + NS;
    uint64_t* e_bar = o_empty + 1;  // [4 lane quadrants]: the groups' maxima and sums of a unit
    uint64_t* t_bar = e_bar + 4;    // [2]: the bias table may be rewritten; is written
    uint64_t* drain = t_bar + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* table_hides = abort_flag + 1;  // [2], by build: the staged table holds -infinity

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int x = 0; x < 2; x++) {
            mbar_init(&unit_full[x], 32);
            mbar_init(&unit_empty[x], Cfg::POLL ? 12 : 11);  // TMA (both of its walks), both MMA issuers, 8 softmax warps
            mbar_init(&t_bar[x], 8);
            mbar_init(&drain[x], 1);
        }
        for (int x = 0; x < NS; x++) {
            mbar_init(&s_full[x], 1);
            mbar_init(&p_full[x], 4);
            mbar_init(&pv_done[x], 1);
        }
        mbar_init(o_empty, 8);
        for (int x = 0; x < 4; x++) mbar_init(&e_bar[x], 2);
        for (int x = 0; x < QBUF; x++) {
            mbar_init(&q_full[x], 1);
            mbar_init(&q_empty[x], 1);
        }
        for (int x = 0; x < RING; x++) {
            mbar_init(&k_full[x], 1);
            mbar_init(&k_empty[x], 1);
            mbar_init(&v_full[x], 1);
            mbar_init(&v_empty[x], 1);
        }
        *abort_flag = 0;
        table_hides[0] = table_hides[1] = 0;
        fence_mbarrier_init();
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    if (warp == 1) tmem_alloc(tmem_slot, 512);
    // Running maxima, each with the number of its tile in the upper half: none yet.
    if (threadIdx.x >= 128) reinterpret_cast<unsigned long long*>(smem + Cfg::OFF_X)[threadIdx.x - 128] = ~0ull;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    grid_dep_launch();
    grid_dep_wait();

    // Every role walks the scout's units; unit i's description is in units[i & 1] once unit_full says so. A role
    // ends its walk at the last unit, or when one of its waits ran out.
    auto unit_at = [&](int i) -> AmtUnit* {
        if (!mbar_wait(&unit_full[i & 1], (i >> 1) & 1, EG2_DEV_TIMEOUT_ATTN, abort_flag)) return nullptr;
        return units[i & 1].stop ? nullptr : &units[i & 1];
    };
    // Whether V of key tile kt of a unit is prepared: rows past the sequence's end that are other sequences' (past the
    // buffer TMA reads zeros), or a later stage.
    auto guarded = [&](const AmtUnit& u, int kt) {
        return u.stage != 0 || (kt * 128 + 128 > u.sq.nk && u.sq.k0 + u.sq.nk < p.k_rows);
    };

    if (warp < 4) {
        // The block starts with 168 registers a thread: 3 x 168 = R_AUX + 2 R_SOFT.
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::R_AUX));
        if (warp == 0 && lane == 0) {
            int k_loads = 0, v_loads = 0, q_loads = 0;
            if constexpr (!Cfg::POLL) {
            bool ok = true;
            for (int i = 0; ok; i++) {
                const AmtUnit* un = unit_at(i);
                if (!un) break;
                const int n = un->n, g = un->g, half = un->half;
                const int qrow = (int)(un->sq.q0 + un->t0), krow = (int)un->sq.k0, head0 = un->head0;
                if (n > 0) {
                    const int qb = q_loads % QBUF;
                    if (!mbar_wait(&q_empty[qb], ((q_loads / QBUF) & 1) ^ 1, EG2_DEV_TIMEOUT_ATTN, abort_flag)) break;
                    mbar_arrive_expect_tx(&q_full[qb], Cfg::QCH * 16384);
                    for (int c = 0; c < Cfg::QCH; c++)
                        tma_load_3d(smem + (qb * Cfg::QCH + c) * 16384, &tmQ, &q_full[qb], 64 * c, head0, qrow);
                    q_loads++;
                    auto load = [&](const CUtensorMap* m, uint64_t* full, uint64_t* empty, int off, int& loads, int ch, int kt) -> bool {
                        const int u = loads % RING;
                        if (!mbar_wait(&empty[u], ((loads / RING) & 1) ^ 1, EG2_DEV_TIMEOUT_ATTN, abort_flag)) return false;
                        mbar_arrive_expect_tx(&full[u], Cfg::UNIT);
                        for (int c = 0; c < Cfg::UCH; c++)
                            tma_load_3d(smem + off + u * Cfg::UNIT + c * 16384, m, &full[u], ch + 64 * c, g, krow + kt * 128);
                        loads++;
                        return true;
                    };
                    auto load_k = [&](int x, int kt) { return load(&tmK, k_full, k_empty, Cfg::OFF_R, k_loads, x * 64 * Cfg::UCH, kt); };
                    auto load_v = [&](int x, int kt) { return load(&tmV, v_full, v_empty, Cfg::OFF_V, v_loads, half * 256 + x * 64 * Cfg::UCH, kt); };
                    TileWalk walk(*un);
                    int kt = walk.next();
                    for (int x = 0; ok && x < KU; x++) ok = load_k(x, kt);
                    for (int j = 0; ok && j < n; j++) {
                        int kn = 0;
                        if (j + 1 < n) {
                            kn = walk.next();
                            for (int x = 0; ok && x < KU; x++) ok = load_k(x, kn);
                        }
                        for (int x = 0; ok && x < VU; x++) ok = load_v(x, kt);
                        kt = kn;
                    }
                }
                mbar_arrive(&unit_empty[i & 1]);
            }
            } else {
            // Two walks over the units, one loading Q and K, one V; a step does what there is room for, or nothing.
            struct Side {
                int i = 0, j = 0, x = 0, kt = 0;  // unit, tile, ring unit of the tile, key tile
                bool q = false, done = false;     // Q is loaded; no further unit
                AmtUnit* un = nullptr;
                TileWalk walk;
            } ks, vs;
            // Steps into the next unit with tiles. True where it moved.
            auto enter = [&](Side& d) -> bool {
                if (!mbar_test(&unit_full[d.i & 1], (d.i >> 1) & 1)) return false;
                AmtUnit* un = &units[d.i & 1];
                if (un->stop) {
                    d.done = true;
                } else if (un->n == 0) {
                    mbar_arrive(&unit_empty[d.i & 1]);
                    d.i++;
                } else {
                    d.un = un;
                    d.j = d.x = 0;
                    d.q = false;
                    d.walk = TileWalk(*un);
                    d.kt = d.walk.next();
                }
                return true;
            };
            auto load = [&](Side& d, const CUtensorMap* m, uint64_t* full, uint64_t* empty, int off, int& loads, int per, int ch0) -> bool {
                const int u = loads % RING;
                if (!mbar_test(&empty[u], ((loads / RING) & 1) ^ 1)) return false;
                mbar_arrive_expect_tx(&full[u], Cfg::UNIT);
                for (int c = 0; c < Cfg::UCH; c++)
                    tma_load_3d(smem + off + u * Cfg::UNIT + c * 16384, m, &full[u], ch0 + (d.x * Cfg::UCH + c) * 64, d.un->g,
                                (int)d.un->sq.k0 + d.kt * 128);
                loads++;
                if (++d.x == per) {
                    d.x = 0;
                    if (++d.j == d.un->n) {
                        mbar_arrive(&unit_empty[d.i & 1]);
                        d.i++;
                        d.un = nullptr;
                    } else {
                        d.kt = d.walk.next();
                    }
                }
                return true;
            };
            uint64_t since = 0;
            for (uint32_t idle = 0; !(ks.done && vs.done);) {
                bool moved = false;
                if (!ks.done) {
                    if (!ks.un) {
                        moved = enter(ks);
                    } else if (!ks.q) {
                        const int qb = q_loads % QBUF;
                        if (mbar_test(&q_empty[qb], ((q_loads / QBUF) & 1) ^ 1)) {
                            mbar_arrive_expect_tx(&q_full[qb], Cfg::QCH * 16384);
                            for (int c = 0; c < Cfg::QCH; c++)
                                tma_load_3d(smem + (qb * Cfg::QCH + c) * 16384, &tmQ, &q_full[qb], 64 * c, ks.un->head0, (int)(ks.un->sq.q0 + ks.un->t0));
                            q_loads++;
                            moved = ks.q = true;
                        }
                    } else {
                        moved = load(ks, &tmK, k_full, k_empty, Cfg::OFF_R, k_loads, KU, 0);
                    }
                }
                if (!vs.done) moved |= vs.un ? load(vs, &tmV, v_full, v_empty, Cfg::OFF_V, v_loads, VU, vs.un->half * 256) : enter(vs);
                if (moved) {
                    idle = 0;
                    continue;
                }
                __nanosleep(40);  // the softmax warps of this scheduler have the use of its issue slots
                if ((++idle & 63u) == 0u) {  // the bounded wait of mbar_wait
                    const uint64_t now = globaltimer_ns();
                    if (idle == 64u) since = now;
                    if (*abort_flag || *(volatile int*)&eg2_dev_status != 0 || now - since > EG2_WAIT_LIMIT_NS) {
                        if (!*abort_flag) eg2_record_error(EG2_DEV_TIMEOUT_ATTN);
                        *abort_flag = 1;
                        break;
                    }
                }
            }
            }
            // Every load has landed before the CTA may end (on the error path too).
            for (int x = max(0, q_loads - QBUF); x < q_loads; x++) mbar_drain(&q_full[x % QBUF], (x / QBUF) & 1, 200000000ull);
            for (int x = max(0, k_loads - RING); x < k_loads; x++) mbar_drain(&k_full[x % RING], (x / RING) & 1, 200000000ull);
            for (int x = max(0, v_loads - RING); x < v_loads; x++) mbar_drain(&v_full[x % RING], (x / RING) & 1, 200000000ull);
        } else if (warp == 1 && lane == 0) {
            constexpr uint32_t idesc = umma_idesc(128, 128, 1);
            const uint64_t dq0 = umma_desc_sw128(smem_u32(smem), 16, 1024);
            const uint64_t dk0 = umma_desc_sw128(smem_u32(smem + Cfg::OFF_R), 16, 1024);
            int at = 0, q_seen = 0, T = 0;  // K units, Q tiles and key tiles taken
            bool ok = true;
            for (int i = 0; ok; i++) {
                const AmtUnit* un = unit_at(i);
                if (!un) break;
                const int n = un->n, qb = q_seen % QBUF;
                if (n > 0) {
                    ok = mbar_wait(&q_full[qb], (q_seen / QBUF) & 1, EG2_DEV_TIMEOUT_ATTN, abort_flag);
                    q_seen++;
                    for (int j = 0; ok && j < n; j++, T++) {
                        const int buf = T % NS;
                        // The buffer's last P has been multiplied with V.
                        if (T >= NS && !(ok = mbar_wait(&pv_done[buf], (T / NS - 1) & 1, EG2_DEV_TIMEOUT_ATTN, abort_flag))) break;
                        for (int x = 0; x < KU; x++, at++) {
                            if (!(ok = mbar_wait(&k_full[at % RING], (at / RING) & 1, EG2_DEV_TIMEOUT_ATTN, abort_flag))) break;
                            tc_fence_after();
#pragma unroll
                            for (int c = 0; c < Cfg::UCH; c++)
#pragma unroll
                                for (int kk = 0; kk < 4; kk++)
                                    mma_bf16(tmem + 128 * buf, dq0 + (uint64_t)((qb * Cfg::QCH + x * Cfg::UCH + c) * 1024 + 2 * kk),
                                             dk0 + (uint64_t)((at % RING) * (Cfg::UNIT >> 4) + c * 1024 + 2 * kk), idesc,
                                             (x | c | kk) != 0);
                            mma_commit(&k_empty[at % RING]);
                        }
                        if (!ok) break;
                        mma_commit(&s_full[buf]);
                    }
                    if (!ok) break;
                    mma_commit(&q_empty[qb]);
                }
                mbar_arrive(&unit_empty[i & 1]);
            }
            mma_commit(&drain[0]);
            mbar_wait(&drain[0], 0, EG2_DEV_TIMEOUT_ATTN, nullptr);
        } else if (warp == 2) {
            constexpr int N = 64 * Cfg::UCH;
            constexpr uint32_t idesc = umma_idesc(128, N, 1, /*b_mn_major=*/true);
            const uint64_t dv0 = umma_desc_sw128(smem_u32(smem + Cfg::OFF_V), 16384, 1024);
            int at = 0, T = 0, U = 0;  // V units, key tiles, and units with any taken
            bool ok = true;
            for (int i = 0; ok; i++) {
                AmtUnit* un = unit_at(i);
                if (!un) break;
                const int n = un->n;
                TileWalk walk(*un);
                for (int j = 0; ok && j < n; j++, T++) {
                    const int kt = walk.next(), buf = T % NS;
                    const bool clean = guarded(*un, kt);
                    for (int x = 0; ok && x < VU; x++, at++) {
                        const int u = at % RING;
                        if (!(ok = mbar_wait(&v_full[u], (at / RING) & 1, EG2_DEV_TIMEOUT_ATTN, abort_flag))) break;
                        if (clean) {
                            bool hit = false;
                            for (int c = 0; c < Cfg::UCH; c++)
                                hit |= guard_chunk(smem + Cfg::OFF_V + u * Cfg::UNIT + c * 16384, un->sq.nk - kt * 128, un->stage);
                            if (un->stage == 1 && hit && lane == 0) {
                                un->bad[kt >> 5] |= 1u << (kt & 31);
                                un->found = 1;
                            }
                            fence_proxy_async();
                            __syncwarp();
                        }
                        if (x == 0) {
                            // The unit before has been read out of O.
                            if (j == 0 && U >= 1 && !(ok = mbar_wait(o_empty, (U - 1) & 1, EG2_DEV_TIMEOUT_ATTN, abort_flag))) break;
                            if (!(ok = mbar_wait(&p_full[buf], (T / NS) & 1, EG2_DEV_TIMEOUT_ATTN, abort_flag))) break;
                        }
                        tc_fence_after();
                        if (lane == 0) {
                            // 16 keys per MMA: 8 packed P columns, 16 V rows (2,048 bytes).
#pragma unroll
                            for (int kk = 0; kk < 8; kk++)
                                mma_bf16_ts(tmem + Cfg::T_O + x * N, tmem + 128 * buf + 8 * kk,
                                            dv0 + (uint64_t)(u * (Cfg::UNIT >> 4) + kk * 128), idesc, (j | kk) != 0);
                            mma_commit(&v_empty[u]);
                            if (x + 1 == VU) mma_commit(&pv_done[buf]);
                        }
                        __syncwarp();
                    }
                }
                if (!ok) break;
                if (n > 0) U++;
                if (lane == 0) mbar_arrive(&unit_empty[i & 1]);
            }
            if (lane == 0) {
                mma_commit(&drain[1]);
                mbar_wait(&drain[1], 0, EG2_DEV_TIMEOUT_ATTN, nullptr);
            }
        } else if (warp == 3) {
            int id = blockIdx.x;
            bool idle = false;
            int round = 0;
            for (int i = 0;; i++) {
                if (i >= 2 && !mbar_wait(&unit_empty[i & 1], ((i >> 1) & 1) ^ 1, EG2_DEV_TIMEOUT_ATTN, abort_flag)) break;
                AmtUnit& un = units[i & 1];
                int stage = 0;
                if (i >= 2) {
                    const volatile AmtUnit& was = un;
                    stage = was.stage == 0 ? was.retry : was.stage == 1 ? (was.found ? 2 : 0) : was.stage == 2 ? 3 : 0;
                }
                const bool again = stage != 0;
                __syncwarp();
                if (again || id >= ap.n_units) {
                    // A unit that met a value that is not finite runs again as it is described, then over the tiles that hold
                    // some; when there is none and none is left, an empty unit first, since the other buffer's may still
                    // have to run again.
                    int n = 0;
                    if (stage == 1)
                        for (int w = lane; w < AMT_MASK_WORDS; w += 32) un.bad[w] = 0u;
                    if (stage == 2) {
                        for (int w = lane; w < AMT_MASK_WORDS; w += 32) {
                            const uint32_t v = un.bad[w] ? un.visit[w] & un.bad[w] : 0u;
                            un.visit[w] = v;
                            n += __popc(v);
                        }
                        n = __reduce_add_sync(0xffffffffu, n);
                    }
                    if (lane == 0) {
                        un.stop = !again && idle;
                        un.stage = stage;
                        un.retry = un.masked = un.found = 0;
                        if (stage == 2) un.n = n, un.sparse = 1;
                        if (!again) un.n = un.rows = 0;
                        if (!again && !idle) un.visit[0] = 0u;
                    }
                    __syncwarp();
                    mbar_arrive(&unit_full[i & 1]);
                    if (!again && idle) break;
                    idle = !again;
                    continue;
                }
                idle = false;
                int x = id;
                // Round robin, every other round backwards: under a causal mask units shrink along the list.
                round++;
                id = round * gridDim.x + ((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
                const int split = x % p.nsplit;
                x /= p.nsplit;
                const int half = x % Cfg::HALVES;
                x /= Cfg::HALVES;
                const int hg = x % ap.heads;
                x /= ap.heads;
                const int b = x % p.n_seq;
                const int tile = ap.q_tiles - 1 - x / p.n_seq;
                const MaskedSeq sq = masked_seq(p, b);
                const int per = 128 / ap.Gt, t0 = tile * per;
                const int tokens = min(per, sq.nq - t0);
                int n = 0, first_tile = 0, down_to = -1;
                if (tokens > 0) {
                    int lo, hi, tmp;
                    masked_range(p, sq, sq.nk - sq.nq + t0, lo, tmp);
                    masked_range(p, sq, sq.nk - sq.nq + t0 + tokens - 1, tmp, hi);
                    const int first = lo / 128, last = hi > lo ? (hi + 127) / 128 : first;  // key tiles [first, last)
                    int dlo = INT_MAX, dhi = INT_MIN;
                    if (p.q_doc) {
                        for (int t = lane; t < tokens; t += 32) {
                            const int d = p.q_doc[sq.q0 + t0 + t];
                            dlo = min(dlo, d);
                            dhi = max(dhi, d);
                        }
                        dlo = __reduce_min_sync(0xffffffffu, dlo);
                        dhi = __reduce_max_sync(0xffffffffu, dhi);
                    }
                    const int w_end = (last + 31) / 32;
                    for (int w = lane; w <= w_end && w < AMT_MASK_WORDS; w += 32) {
                        // bits of tiles [first, last)
                        const int a = max(first - 32 * w, 0), z = min(last - 32 * w, 32);
                        un.visit[w] = z > a ? (z == 32 ? 0xffffffffu : (1u << z) - 1u) & ~((1u << a) - 1u) : 0u;
                        un.docs[w] = 0u;
                    }
                    __syncwarp();
                    n = last - first;
                    first_tile = first;
                    // Distance penalties: from the last query's place backwards, then on, so that the largest scores come
                    // first and O is hardly ever rescaled.
                    if (p.slopes) down_to = max(sq.nk - sq.nq + t0 + tokens - 1, 0) / 128;
                    if (p.q_doc && n > 0) {
                        n = 0;
                        for (int w = first / 32; w < w_end; w++) {
                            const uint32_t in = un.visit[w];
                            uint32_t visit = 0, docs = 0;
                            // The ids of four tiles in flight at a time.
                            for (int t0_ = 0; t0_ < 32; t0_ += 4) {
                                if (!((in >> t0_) & 15u)) continue;
                                int klo[4], khi[4];
#pragma unroll
                                for (int t = 0; t < 4; t++) {
                                    klo[t] = INT_MAX;
                                    khi[t] = INT_MIN;
#pragma unroll
                                    for (int y = 0; y < 4; y++) {
                                        const int key = (32 * w + t0_ + t) * 128 + 32 * y + lane;
                                        if (key < sq.nk) {
                                            const int d = p.k_doc[sq.k0 + key];
                                            klo[t] = min(klo[t], d);
                                            khi[t] = max(khi[t], d);
                                        }
                                    }
                                }
#pragma unroll
                                for (int t = 0; t < 4; t++) {
                                    const int a = __reduce_min_sync(0xffffffffu, klo[t]), z = __reduce_max_sync(0xffffffffu, khi[t]);
                                    const uint32_t bit = 1u << (t0_ + t);
                                    if (!(in & bit) || z < dlo || a > dhi) continue;
                                    visit |= bit;
                                    if (a != z || dlo != dhi || a != dlo) docs |= bit;
                                }
                            }
                            __syncwarp();
                            if (lane == 0) {
                                un.visit[w] = visit;
                                un.docs[w] = docs;
                            }
                            n += __popc(visit);
                        }
                        __syncwarp();
                    }
                    if (p.nsplit > 1) {
                        // This part's share of the tiles: the a-th to the z-th of them.
                        const int a = min(n, split * p.part), z = min(n, a + p.part);
                        int before = 0;
                        for (int w0 = 0; w0 < w_end; w0 += 32) {
                            const int w = w0 + lane;
                            uint32_t v = w < w_end ? un.visit[w] : 0u;
                            const int c = __popc(v);
                            int sum = c;
#pragma unroll
                            for (int o = 1; o < 32; o <<= 1) {
                                const int y = __shfl_up_sync(0xffffffffu, sum, o);
                                if (lane >= o) sum += y;
                            }
                            int at = before + sum - c;
                            before += __shfl_sync(0xffffffffu, sum, 31);
                            for (uint32_t left = v; left; left &= left - 1u, at++)
                                if (at < a || at >= z) v &= ~(left & (~left + 1u));
                            if (w < w_end) un.visit[w] = v;
                        }
                        n = z - a;
                        first_tile += a;
                        __syncwarp();
                    }
                }
                if (lane == 0) {
                    un.sq = sq;
                    un.t0 = t0;
                    un.rows = max(tokens, 0) * ap.Gt;
                    un.head0 = hg * ap.Gt;
                    un.g = un.head0 / p.G;
                    un.split = split;
                    un.half = half;
                    un.n = n;
                    un.first = first_tile;
                    un.down = min(max(down_to + 1 - first_tile, 0), n);
                    un.sparse = p.q_doc != nullptr;
                    un.stop = un.stage = un.retry = un.masked = un.found = 0;
                }
                __syncwarp();
                mbar_arrive(&unit_full[i & 1]);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::R_SOFT));
        const int e = warp & 3, wg = (warp - 4) >> 2;
        const int r = 32 * e + lane;
        const uint32_t lane_off = (uint32_t)(32 * e) << 16;
        constexpr int NC = 128;
        volatile unsigned long long* xm = reinterpret_cast<unsigned long long*>(smem + Cfg::OFF_X);  // [2 groups][128]
        float* xe = reinterpret_cast<float*>(smem + Cfg::OFF_X + 2048);                              // [2][2 groups][128][2]
        // The row's maximum after the other group's tile `tile`: the same thread of that group writes value and number at once,
        // and writes its next only after it has read this group's answer.
        auto maximum_after = [&](int tile, bool& ok) -> float {
            unsigned long long v = xm[(wg ^ 1) * 128 + r];
            if ((int)(v >> 32) != tile) {
                const uint64_t t0 = globaltimer_ns();
                for (uint32_t it = 1; ok && (int)((v = xm[(wg ^ 1) * 128 + r]) >> 32) != tile; it++)
                    if ((it & 255u) == 0u && (*abort_flag || *(volatile int*)&eg2_dev_status != 0 || globaltimer_ns() - t0 > EG2_WAIT_LIMIT_NS)) {
                        if (!*abort_flag) eg2_record_error(EG2_DEV_TIMEOUT_ATTN);
                        *abort_flag = 1;
                        ok = false;
                    }
            }
            return __uint_as_float((uint32_t)v);
        };
        float* table = reinterpret_cast<float*>(smem + Cfg::OFF_TAB);
        const int tab_ld = 2 * p.radius + 1 + 256;  // 128 copies of either end around the table
        // Scores are kept as v with the score (log2 domain) v * sc: the scale is left to the exponent's FMA where nothing
        // needs it before (sc > 0, so the order is kept).
        const bool capped = PARTS == AMT_ANY ? p.softcap > 0.f : (PARTS & AMT_CAP) != 0;
        const bool slopes = PARTS == AMT_ANY ? p.slopes != nullptr : (PARTS & AMT_SLOPES) != 0;
        const bool tables = PARTS == AMT_ANY ? p.table != nullptr : (PARTS & AMT_TAB) != 0;
        const float cap2 = p.softcap * AMT_LOG2E;
        const float a = capped ? p.scale / p.softcap : p.scale * AMT_LOG2E;
        const bool raw = !(p.softcap > 0.f) && !p.slopes && !p.table && a > 0.f;
        const float sc = raw ? a : 1.f;
        // cap2 tanh(a s) = s (c0 + c1 s^2 + ...) where |a s| <= 1/2, as long as the powers of a stay in range: of scale / softcap between
        // 1e-4 and 1e3, and |score| <= softcap / 2. A warp's tile with a score past that, a hidden one too, is done twice, and so is every tile outside
        // that range of a: 8,192 tokens, scores of deviation 2 under a cap of 50 / of 5: 655 / 1,300 us (12 heads of 64), 485 / 900 (8 over 2
        // of 128), 352 / 560 (4 over 2 of 256), 1,062 / 1,478 (4 over 1 of 512).
        const bool near_ok = fabsf(a) > 1e-4f && fabsf(a) < 1e3f;
        const float near_max = near_ok ? (AMT_TANH_MAX / a) * (AMT_TANH_MAX / a) : -1.f;
        const float c0 = AMT_T0 * a * cap2, c1 = AMT_T1 * a * a * a * cap2, c2 = AMT_T2 * (a * a) * (a * a) * a * cap2,
                    c3 = AMT_T3 * (a * a * a) * (a * a * a) * a * cap2, c4 = AMT_T4 * (a * a * a) * (a * a * a) * (a * a * a) * cap2;
        int T = 0, U = 0, tab_head = -1, builds = 0;
        bool ok = true, hides = false;

        for (int i = 0; ok; i++) {
            AmtUnit* un = unit_at(i);
            if (!un) break;
            const int n = un->n;
            if (un->stage >= 2) {
                if (!(ok = masked_count<HD, (PARTS & (AMT_TAB | AMT_ANY)) != 0>(ap, *un, tmem, T, U, s_full, p_full, pv_done, o_empty, e_bar, abort_flag))) break;
                T += n;
                U++;
                if (lane == 0) mbar_arrive(&unit_empty[i & 1]);
                continue;
            }
            const bool live = r < un->rows;
            const bool warp_live = 32 * e < un->rows;
            const int tok = un->t0 + r / ap.Gt, head = un->head0 + r % ap.Gt;
            const int place = un->sq.nk - un->sq.nq + tok;
            int lo = 0, hi = 0, qdoc = 0;
            if (live) {
                masked_range(p, un->sq, place, lo, hi);
                if (p.q_doc) qdoc = p.q_doc[un->sq.q0 + tok];
            }
            const float slope = (slopes && live) ? p.slopes[head] * AMT_LOG2E : 0.f;
            if (tables && un->rows > 0 && tab_head != un->head0) {
                tab_head = un->head0;
                const int s_tid = threadIdx.x - 128;
                __syncwarp();
                if (lane == 0) mbar_arrive(&t_bar[0]);
                if (!(ok = mbar_wait(&t_bar[0], builds & 1, EG2_DEV_TIMEOUT_ATTN, abort_flag))) break;
                if (s_tid == 0) table_hides[(builds + 1) & 1] = 0;  // the build before has been read, the next one waits for t_bar[0]
                for (int x = s_tid; x < ap.Gt * tab_ld; x += 256) {
                    const int hh = x / tab_ld, c = min(max(x % tab_ld - 128, 0), 2 * p.radius);
                    const float b = masked_bias(p.table[(long)(tab_head + hh) * (2 * p.radius + 1) + c]);
                    table[x] = b * AMT_LOG2E;
                    if (b == -INFINITY) table_hides[builds & 1] = 1;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&t_bar[1]);
                if (!(ok = mbar_wait(&t_bar[1], builds & 1, EG2_DEV_TIMEOUT_ATTN, abort_flag))) break;
                hides = table_hides[builds & 1];
                builds++;
            }
            const float* my_table = table + (r % ap.Gt) * tab_ld;
            float m = AMT_NONE, l = 0.f;  // the row's maximum at this group's last tile, and its part of the sum in units of 2^m
            bool any_masked = false;
            if (n > 0) {
                TileWalk walk(*un);
                // The keys that some and that every row of the warp sees.
                const int some_lo = __reduce_min_sync(0xffffffffu, lo < hi ? lo : INT_MAX);
                const int some_hi = __reduce_max_sync(0xffffffffu, lo < hi ? hi : 0);
                const int all_lo = __reduce_max_sync(0xffffffffu, live ? lo : 0);
                const int all_hi = __reduce_min_sync(0xffffffffu, live ? hi : INT_MAX);
                const int mine = (wg ^ T) & 1;  // this group's tiles: mine, mine + 2, ...
                if (mine) walk.next();
                // The next tile's first key, and of its document ids those of columns lane, 32 + lane, ...
                int next_key = mine < n ? walk.next() * 128 : 0, ids[4];
                auto fetch_ids = [&] {
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        const int key = next_key + 32 * x + lane;
                        ids[x] = p.q_doc && key < un->sq.nk ? p.k_doc[un->sq.k0 + key] : 0;
                    }
                };
                if (mine < n) fetch_ids();
                int buf = (T + mine) % NS, phase = ((T + mine) / NS) & 1;
                for (int j = mine; j < n; j += 2) {
                    const int tile = T + j, kbase = next_key;
                    const uint32_t ts = tmem + 128 * buf + lane_off;
                    const bool sees = kbase < some_hi && kbase + NC > some_lo;
                    const bool docs = p.q_doc && ((un->docs[kbase >> 12] >> ((kbase >> 7) & 31)) & 1u);
                    const bool some = docs || (tables && hides);
                    const bool full = !some && kbase >= all_lo && kbase + NC <= all_hi;
                    any_masked |= !full;
                    uint32_t same[4] = {~0u, ~0u, ~0u, ~0u};  // columns of this row's document that no bias hides
                    if (some && sees) {
                        if (docs) {
                            // The rows of a warp are of few documents, mostly one: a ballot per document and 32 columns.
                            uint32_t left = __ballot_sync(0xffffffffu, lo < hi);
#pragma unroll
                            for (int x = 0; x < 4; x++) same[x] = 0u;
                            while (left) {
                                const int d = __shfl_sync(0xffffffffu, qdoc, __ffs(left) - 1);
                                left &= ~__ballot_sync(0xffffffffu, qdoc == d);
#pragma unroll
                                for (int x = 0; x < 4; x++) {
                                    const uint32_t cols = __ballot_sync(0xffffffffu, ids[x] == d);
                                    if (qdoc == d) same[x] = cols;
                                }
                            }
                        }
                        if (tables && hides) {
                            const uint4 h = masked_hidden_columns(my_table + min(max(kbase - place, -p.radius - 128), p.radius) + p.radius + 128);
                            same[0] &= ~h.x;
                            same[1] &= ~h.y;
                            same[2] &= ~h.z;
                            same[3] &= ~h.w;
                        }
                    }
                    if (j + 2 < n) {
                        walk.next();
                        next_key = walk.next() * 128;
                        fetch_ids();
                    }
                    if (ok) ok = mbar_wait(&s_full[buf], phase, EG2_DEV_TIMEOUT_ATTN, abort_flag);
                    tc_fence_after();
                    float mt = AMT_NONE;
                    uint32_t su[NC];
                    float* sv = reinterpret_cast<float*>(su);
                    auto load_s = [&] {
#pragma unroll
                        for (int c = 0; c < NC / 32; c++) tmem_ld32(ts + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(su + 32 * c));
                        tmem_ld_wait();
                        reg_fence<NC>(su);
                    };
                    if (sees) {
                        load_s();
                        if (!raw) {
                            if (capped) {
                                // The polynomial for every score, four pairs at a time; where one is out of its range the
                                // tile is done again from S, 16 columns at a time through TMEM. Each score keeps the form that its
                                // own size asks for, so its bits do not depend on its neighbours, hidden ones among them.
                                float far = 0.f;
#pragma unroll
                                for (int c = 0; c < NC; c += 8) {
                                    uint64_t x[4], y[4], r[4];
#pragma unroll
                                    for (int q = 0; q < 4; q++) {
                                        x[q] = f2_pack(sv[c + 2 * q], sv[c + 2 * q + 1]);
                                        y[q] = f2_mul(x[q], x[q]);
                                    }
#pragma unroll
                                    for (int q = 0; q < 4; q++) {
                                        float u, w;
                                        f2_unpack(y[q], u, w);
                                        far = max3(far, u, w);
                                        r[q] = f2_fma(y[q], f2_pack(c4, c4), f2_pack(c3, c3));
                                    }
#pragma unroll
                                    for (int q = 0; q < 4; q++) r[q] = f2_fma(r[q], y[q], f2_pack(c2, c2));
#pragma unroll
                                    for (int q = 0; q < 4; q++) r[q] = f2_fma(r[q], y[q], f2_pack(c1, c1));
#pragma unroll
                                    for (int q = 0; q < 4; q++) r[q] = f2_fma(r[q], y[q], f2_pack(c0, c0));
#pragma unroll
                                    for (int q = 0; q < 4; q++) f2_unpack(f2_mul(x[q], r[q]), sv[c + 2 * q], sv[c + 2 * q + 1]);
                                }
                                if (!__all_sync(0xffffffffu, far <= near_max)) {
#pragma unroll 1
                                    for (int c = 0; c < NC; c += 16) {
                                        uint32_t o[16];
                                        tmem_ld16(ts + c, o);
                                        tmem_ld_wait();
                                        reg_fence<16>(o);
                                        if (near_ok) {
#pragma unroll
                                            for (int q = 0; q < 16; q++) {
                                                const float x = __uint_as_float(o[q]), y = x * x;
                                                const float near = x * fmaf(fmaf(fmaf(fmaf(y, c4, c3), y, c2), y, c1), y, c0);
                                                o[q] = __float_as_uint(y <= near_max ? near : cap2 * tanh_far(x * a));
                                            }
                                        } else {
#pragma unroll
                                            for (int q = 0; q < 16; q++) o[q] = __float_as_uint(cap2 * tanh_any(__uint_as_float(o[q]) * a));
                                        }
                                        tmem_st16(ts + c, o);
                                    }
                                    tmem_st_wait();
                                    load_s();
                                }
                            } else {
                                const uint64_t a2 = f2_pack(a, a);
#pragma unroll
                                for (int c = 0; c < NC; c += 2) f2_unpack(f2_mul(f2_pack(sv[c], sv[c + 1]), a2), sv[c], sv[c + 1]);
                            }
                            if (slopes) {
                                const float d0 = (float)(kbase - place);
#pragma unroll
                                for (int c = 0; c < NC; c++) sv[c] = fmaf(-slope, fabsf(d0 + (float)c), sv[c]);
                            }
                            if (tables) {
                                // j - i runs over 128 consecutive values: clamped once, the copies of the ends do the rest.
                                const float* tb = my_table + min(max(kbase - place, -p.radius - 128), p.radius) + p.radius + 128;
#pragma unroll
                                for (int c = 0; c < NC; c++) sv[c] += tb[c];
                            }
                        }
                        if (!full) {
#pragma unroll
                            for (int x = 0; x < NC; x += 32) {
                                const int u = min(max(lo - kbase - x, 0), 32), z = min(max(hi - kbase - x, 0), 32);
                                uint32_t seen = z > u ? (0xffffffffu >> (32 - z)) & (0xffffffffu << u) : 0u;
                                seen &= same[x / 32];
#pragma unroll
                                for (int c = 0; c < 32; c++) sv[x + c] = (seen >> c) & 1u ? sv[x + c] : -INFINITY;
                            }
                        }
                        float mx[4] = {sv[0], sv[1], sv[2], sv[3]};
#pragma unroll
                        for (int c = 4; c + 7 < NC; c += 8)
#pragma unroll
                            for (int q = 0; q < 4; q++) mx[q] = max3(mx[q], sv[c + q], sv[c + 4 + q]);
#pragma unroll
                        for (int q = 0; q < 4; q++) mx[q] = fmaxf(mx[q], sv[NC - 4 + q]);
                        mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;
                    }
                    // The row's maximum so far comes from the other group's tile, and goes on to its next.
                    float before = AMT_NONE;
                    if (j >= 1) {
                        if (ok) before = maximum_after(tile - 1, ok);
                        ok = __all_sync(0xffffffffu, ok);
                    }
                    const float now = (mt - before > ATT_RESCALE_LOG2 || before == AMT_NONE) ? fmaxf(mt, AMT_NONE) : before;
                    xm[wg * 128 + r] = (unsigned long long)(uint32_t)tile << 32 | __float_as_uint(now);
                    l *= ex2_approx(m - now);
                    m = now;
                    if (__any_sync(0xffffffffu, now != before && before != AMT_NONE)) {
                        // O is in units of 2^before, and complete up to the tile before.
                        if (ok) ok = mbar_wait(&pv_done[(tile - 1) % NS], ((tile - 1) / NS) & 1, EG2_DEV_TIMEOUT_ATTN, abort_flag);
                        tc_fence_after();
                        const float factor = before == AMT_NONE ? 1.f : ex2_approx(before - now);
#pragma unroll 1
                        for (int c = 0; c < Cfg::DV; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(tmem + Cfg::T_O + c + lane_off, o);
                            tmem_ld_wait();
                            reg_fence<16>(o);
#pragma unroll
                            for (int q = 0; q < 16; q++) o[q] = __float_as_uint(__uint_as_float(o[q]) * factor);
                            tmem_st16(tmem + Cfg::T_O + c + lane_off, o);
                        }
                    }
                    if (sees) {
                        const float base = -m;
                        const uint64_t sc2 = f2_pack(sc, sc), base2 = f2_pack(base, base);
                        uint64_t sum0 = 0, sum1 = 0;
#pragma unroll
                        for (int c = 0; c < NC; c += 32) {
                            uint32_t pk[16];
#pragma unroll
                            for (int q = 0; q < 16; q++) {
                                float u, w;
                                f2_unpack(f2_fma(f2_pack(sv[c + 2 * q], sv[c + 2 * q + 1]), sc2, base2), u, w);
                                u = ex2_approx(u);
                                w = ex2_approx(w);
                                pk[q] = bf16x2_bits(u, w);
                                if (q & 1)
                                    sum1 = f2_add(sum1, f2_pack(u, w));
                                else
                                    sum0 = f2_add(sum0, f2_pack(u, w));
                            }
                            tmem_st16(ts + c / 2, pk);
                        }
                        float u, w;
                        f2_unpack(f2_add(sum0, sum1), u, w);
                        l += u + w;
                    } else if (warp_live) {
                        uint32_t pk[16];
#pragma unroll
                        for (int q = 0; q < 16; q++) pk[q] = 0u;
#pragma unroll
                        for (int c = 0; c < NC; c += 32) tmem_st16(ts + c / 2, pk);
                    }
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    mbar_arrive_if(&p_full[buf], lane == 0);
                    buf += 2;
                    if (buf >= NS) {
                        buf -= NS;
                        phase ^= 1;
                    }
                }
                T += n;
            }
            // ---- O / l: half of the channels by each group ----
            {
                float* mine = xe + (((U & 1) * 2 + wg) * 128 + r) * 2;
                float* other = xe + (((U & 1) * 2 + (wg ^ 1)) * 128 + r) * 2;
                if (any_masked && lane == 0) *(volatile int*)&un->masked = 1;
                mine[0] = m;
                mine[1] = l;
                __syncwarp();
                mbar_arrive_if(&e_bar[e], lane == 0);
                if (ok) ok = mbar_wait(&e_bar[e], U & 1, EG2_DEV_TIMEOUT_ATTN, abort_flag);
                U++;
                const float m2 = *(volatile float*)other, l2 = *(volatile float*)(other + 1);
                const float top = fmaxf(m, m2);
                // The same sum, in the same order, in both groups.
                const float part = l * ex2_approx(m - top), part2 = l2 * ex2_approx(m2 - top);
                l = wg == 0 ? part + part2 : part2 + part;
                m = top;
            }
            {
                if (n > 0) {
                    if (ok) ok = mbar_wait(&pv_done[(T - 1) % NS], ((T - 1) / NS) & 1, EG2_DEV_TIMEOUT_ATTN, abort_flag);
                    tc_fence_after();
                }
                const float inv = l == 0.f ? 0.f : 1.f / l;
                const long row = un->sq.q0 + tok;
                const long at = row * p.nh + head + (p.nsplit > 1 ? (long)un->split * p.q_rows * p.nh : 0);
                if (live && un->half == 0 && wg == 0) {
                    if (p.nsplit > 1)
                        p.part_ml[at] = make_float2(m, l);
                    else if (p.lse)
                        p.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
                }
                const int ch0 = un->half * 256 + wg * Cfg::OC;
                const uint32_t to = tmem + Cfg::T_O + wg * Cfg::OC + lane_off;
                const bool some = n > 0 && l != 0.f;
                float odd = 0.f;  // stays 0 while all channels are finite
#pragma unroll 1
                for (int c = 0; c < Cfg::OC; c += 32) {
                    uint32_t o[32];
                    if (n > 0 && warp_live) {
                        tmem_ld32(to + c, o);
                        tmem_ld_wait();
                        reg_fence<32>(o);
                    }
#pragma unroll
                    for (int q = 0; q < 32; q++) {
                        const float x = some ? __uint_as_float(o[q]) * inv : 0.f;
                        odd = fmaf(x, 0.f, odd);
                        o[q] = __float_as_uint(x);
                    }
                    if (live) {
#pragma unroll
                        for (int q = 0; q < 32; q += 16) {
                            const int ch = ch0 + c + q;
                            if (ch >= p.hd) break;
                            if (p.nsplit > 1) {
                                float* part = p.part_o + at * p.hd + ch;
#pragma unroll
                                for (int y = 0; y < 16; y += 4)
                                    if (ch + y < p.hd)
                                        *reinterpret_cast<uint4*>(part + y) = make_uint4(o[q + y], o[q + y + 1], o[q + y + 2], o[q + y + 3]);
                            } else {
                                uint32_t pk[8];
#pragma unroll
                                for (int y = 0; y < 8; y++)
                                    pk[y] = bf16x2_bits(__uint_as_float(o[q + 2 * y]), __uint_as_float(o[q + 2 * y + 1]));
                                bf16_t* out = (bf16_t*)p.out + row * p.ldo + (long)head * p.hd + ch;
                                if (ap.out32) {
                                    st_global_v8(out, pk);
                                } else {
                                    *reinterpret_cast<uint4*>(out) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
                                    if (ch + 8 < p.hd) *reinterpret_cast<uint4*>(out + 8) = make_uint4(pk[4], pk[5], pk[6], pk[7]);
                                }
                            }
                        }
                    }
                    __syncwarp();
                }
                if (n > 0) {
                    tc_fence_before();
                    __syncwarp();
                    mbar_arrive_if(o_empty, lane == 0);
                }
                if (un->stage == 0 && __any_sync(0xffffffffu, live && odd != 0.f) && *(volatile int*)&un->masked && lane == 0)
                    *(volatile int*)&un->retry = 1;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&unit_empty[i & 1]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int HD, int PARTS>
static int launch_masked_tc(const MaskedParams& p, int Gt, cudaStream_t s) {
    using Cfg = AmtCfg<HD>;
    auto kern = attention_masked_tc_kernel<HD, PARTS>;
    static bool attr_set[64] = {false};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
    if (!attr_set[dev]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM) != cudaSuccess) return -3;
        attr_set[dev] = true;
    }
    CUtensorMap mq, mk, mv;
    const CUtensorMapDataType dt = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    if (make_tmap_3d(&mq, dt, p.q, p.hd, p.nh, p.q_rows, (uint64_t)p.hd * 2, (uint64_t)p.ldq * 2, 64, Gt, 128 / Gt) ||
        make_tmap_3d(&mk, dt, p.k, p.hd, p.nkv, p.k_rows, (uint64_t)p.hd * 2, (uint64_t)p.ldk * 2, 64, 1, 128) ||
        make_tmap_3d(&mv, dt, p.v, p.hd, p.nkv, p.k_rows, (uint64_t)p.hd * 2, (uint64_t)p.ldv * 2, 64, 1, 128))
        return -1;
    AmtParams ap;
    ap.p = p;
    ap.Gt = Gt;
    ap.q_tiles = (int)(((long)p.max_q * Gt + 127) / 128);
    ap.heads = p.nh / Gt;
    const long units = (long)ap.q_tiles * p.n_seq * ap.heads * Cfg::HALVES * p.nsplit;
    if (units > 0x3fffffffL) return -1;
    ap.n_units = (int)units;
    ap.out32 = (uintptr_t)p.out % 32 == 0 && (p.ldo | p.hd) % 16 == 0;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)(units < num_sms() ? units : num_sms()), 1, 1);
    cfg.blockDim = dim3(AMT_THREADS, 1, 1);
    cfg.dynamicSmemBytes = Cfg::SMEM;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, mq, mk, mv, ap) == cudaSuccess ? 0 : -3;
}

// The kernel compiled for just this call's score, where there is one (the plain score keeps its scale for the exponent,
// which wants it positive).
template <int HD>
static int launch_masked_tc(const MaskedParams& p, int Gt, cudaStream_t s) {
    const int parts = (p.softcap > 0.f ? AMT_CAP : 0) | (p.slopes ? AMT_SLOPES : 0) | (p.table ? AMT_TAB : 0);
    switch (parts) {
        case 0: return p.scale > 0.f ? launch_masked_tc<HD, 0>(p, Gt, s) : launch_masked_tc<HD, AMT_ANY>(p, Gt, s);
        case AMT_CAP: return launch_masked_tc<HD, AMT_CAP>(p, Gt, s);
        case AMT_SLOPES: return launch_masked_tc<HD, AMT_SLOPES>(p, Gt, s);
        case AMT_TAB: return launch_masked_tc<HD, AMT_TAB>(p, Gt, s);
        case AMT_CAP | AMT_SLOPES: return launch_masked_tc<HD, AMT_CAP | AMT_SLOPES>(p, Gt, s);
        default: return launch_masked_tc<HD, AMT_ANY>(p, Gt, s);
    }
}
