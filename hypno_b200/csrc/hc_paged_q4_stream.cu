// Attention of few rows, or of rows with lists of pages, over a pool in 4 bits
// with heads of 64 or 128 elements and pages of whole tiles of 16 keys
// (k_paged_split takes the others).
//
// The line of units, its runs, the join and the products are k_paged_split's.  A
// fifth warp copies: a stage is 128 keys, eight tiles of 16 in a page each, so a
// page's place is worked out once a tile and the four warps that compute spend
// nothing on it.  Each takes 32 keys of a stage: two tiles whose chains of dependent
// steps (codes, products, maxima, weights, products) overlap.  16 bytes a lane and
// copy (one run a tile and pool, cp.async.bulk, took the copy engine's time: 391,000 runs
// of 128 and 1,024 bytes 49 us where the same bytes in runs of four times that took 43).
//
// A key's codes become float16 in registers (q4_pairs, 11 instructions for eight
// elements), half of the 405 instructions that 16 keys of a head of 128 cost.  Bound by
// them: shifts, logic and float16 arithmetic run at half rate, and what depends on
// what leaves a scheduler's three or four warps idle on 40% of the cycles.  8 sequences
// of up to 32,768 keys, 64 heads over 8 of 128, f16: 70 us, 3.2 TB/s (the copies alone 46;
// issue slots 59%, logic 43%, so neither is at its limit); 32 of up to 2,304, 32 heads over 8,
// f32: 31 us with the join; 32 tokens over 128 listed pages of 16 each: 39 us.  (Five warps a scheduler at 96 registers
// for the first: 73 us; eight warps of 16 keys each: 84.)
#include "hc_paged_split.cuh"

namespace hc {

namespace {

constexpr int QS_WARPS = 4, QS_ROWS = 32 * QS_WARPS, QS_THREADS = QS_ROWS + 32, QS_TILES = 2 * QS_WARPS, QS_KEYS = SP_TK * QS_TILES;

template <int HD, int NQ, bool HILO>
struct StreamShape {
    static constexpr int ROWB = HD / 2, SCB = 2 * q4_slots(HD);
    static constexpr int CODES = QS_KEYS * ROWB, SCALES = QS_KEYS * SCB;  // of K or V
    static constexpr int STAGE = 2 * (CODES + SCALES);                    // K codes, V codes, K scales, V scales
    static constexpr int STAGES = HD <= 64 ? 4 : 3;
    static constexpr int LDO = HD + 4;
    static constexpr int OUT = 8 * NQ * LDO * 4;                          // a warp's outputs
    static constexpr int QF = NQ * (HD / 16) * 32 * (HILO ? 4 : 2);       // the queries' fragments, in words
    static constexpr int SMEM = STAGES * STAGE + QS_WARPS * OUT + 128;
    static_assert(QF * 4 <= QS_WARPS * OUT, "the queries' fragments lie where the outputs go later");
};

// One CTA's share of a pair.
struct PairWork {
    int seq, r0, first, kvh, m0, mrows;
    int c0, c1;     // positions (LIST: places of the list)
    bool cut;
    int64_t slot;   // of the partial results
    int p_own;      // position of the first row's token
    const int32_t* list;
    int stages;     // -1: no more pairs
    int lost;       // its copies were given up
    int p_min, l_max, one_token;  // keys that every row sees lie in [l_max, p_min]; LIST: not used
};
template <bool LIST>
__device__ __forceinline__ bool next_pair(const SplitArgs& X, const LineTable& line, int64_t& u, int64_t u_begin, int64_t u_end, Line& at, PairWork& w) {
    const PagedAttnArgs& A = X.a;
    if (u >= u_end || !(A.p.n_seqs <= 32 ? advance_by(line, u, at) : advance<LIST>(X, u, X.whole != 0, at))) return false;
    const int64_t rem = u - at.base;
    const int pair = (int)(X.whole ? rem : quotient(rem, at.w.units));
    const int unit = X.whole ? 0 : (int)(rem - (int64_t)pair * at.w.units);
    const int nunits = X.whole ? at.w.units : (int)min((int64_t)(at.w.units - unit), u_end - u);
    w.seq = at.b;
    w.r0 = at.w.r0;
    w.first = at.w.first;
    w.cut = nunits < at.w.units;
    w.slot = 2 * (int64_t)blockIdx.x + (u == u_begin ? 0 : 1);
    u += X.whole ? 1 : nunits;
    w.kvh = pair % A.p.nkv;
    tile_rows<LIST>(X, pair / A.p.nkv, at.w.r1 - w.r0, w.m0, w.mrows);
    int begin, end;
    w.p_own = w.first + token_of(A, w.m0);
    w.list = nullptr;
    if constexpr (LIST) {
        const int row = w.r0 + token_of(A, w.m0);
        w.list = X.l.pages + row * X.l.row_stride + w.kvh * X.l.head_stride;
        begin = 0;
        end = (int)min((int64_t)min(list_count(X.l, row, w.kvh), pages_seen(A.p, w.p_own)) * A.p.page_size, (int64_t)0x7fffff00);
    } else {
        visible(A, w.first, w.m0, w.mrows, begin, end);
        begin &= ~(SP_TK - 1);
    }
    w.c0 = (int)min((int64_t)end, begin + (int64_t)unit * UNIT);
    w.c1 = (int)min((int64_t)end, w.c0 + (int64_t)nunits * UNIT);
    w.stages = (w.c1 - w.c0 + QS_KEYS - 1) / QS_KEYS;
    const int last = token_of(A, w.m0 + w.mrows - 1);
    w.p_min = w.p_own;
    w.l_max = A.window > 0 ? w.first + last - A.window + 1 : 0;
    w.one_token = LIST || token_of(A, w.m0) == last;
    return true;
}

template <int STAGES>
struct StreamBars {
    uint64_t full[STAGES], empty[STAGES];
    uint32_t in[STAGES][QS_TILES];  // which keys of a tile are there
    PairWork work[2];
    int abort;  // a wait for copies or stages ran out
};
// The copying warp tells of a pair by one barrier of the CTA, and the others that they have
// done with it by another, in turn for even and odd pairs.  (Barriers of all threads: what
// they wait for always comes, because the waits for copies and stages are bounded, and a
// warp that gave one up goes on to the CTA's last pair.)  The numbers are the instructions'
// own: taken from a register, 32 tokens over listed pages took 39.5 us in place of 39.0.
constexpr int QS_TOLD = 2, QS_READ = 4;
template <int ID>
__device__ __forceinline__ void pair_sync(bool odd) {
    if (odd) asm volatile("bar.sync %0, %1;" ::"n"(ID + 1), "n"(QS_THREADS) : "memory");
    else asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(QS_THREADS) : "memory");
}
template <int ID>
__device__ __forceinline__ void pair_arrive(bool odd) {
    if (odd) asm volatile("bar.arrive %0, %1;" ::"n"(ID + 1), "n"(QS_THREADS) : "memory");
    else asm volatile("bar.arrive %0, %1;" ::"n"(ID), "n"(QS_THREADS) : "memory");
}

// Waits a bounded time; the whole warp.  (The clock is read when the first look fails.)
__device__ __forceinline__ bool stream_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}
// Arrives at the barrier when this thread's copies so far have landed.
__device__ __forceinline__ void cp_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// The copying warp.
template <typename Sh, int HD, bool LIST>
__device__ __forceinline__ void stream_copies(const SplitArgs& X, const LineTable& line, StreamBars<Sh::STAGES>& B, uint32_t ring, int64_t u_begin, int64_t u_end) {
    constexpr int S = Sh::STAGES, CHUNKS = HD / 32, ROWS = 32 / CHUNKS;  // a row's 16-byte pieces, rows that the lanes copy at once
    const PagedAttnArgs& A = X.a;
    const PagedArgs& P = A.p;
    const int lane = threadIdx.x & 31, tile = lane & 7, kind = lane >> 3;  // what this lane works out: K, V codes, K, V scales
    const int row = lane / CHUNKS, chunk = lane % CHUNKS, srow = lane & 15;
    const bool sv = lane >= 16;  // this lane copies scales of V
    const uint32_t to = ring + lane * 16, to_s = ring + 2 * Sh::CODES + (sv ? Sh::SCALES : 0) + srow * Sh::SCB;
    int64_t u = u_begin;
    Line at = {0, 0, {}};
    PairWork w;
    uint32_t n = 0, pairs = 0;  // stages, pairs so far
    bool ok = true;  // false: a wait ran out, and the pairs from there on are told of without copies
    for (;;) {
        const bool more = next_pair<LIST>(X, line, u, u_begin, u_end, at, w);
        w.lost = !ok;
        if (!ok) w.stages = 0;
        if (!more) w.stages = -1;
        if (pairs >= 2) pair_sync<QS_READ>(pairs & 1);
        if (lane == 0) B.work[pairs & 1] = w;
        __syncwarp();
        pair_arrive<QS_TOLD>(pairs & 1);
        pairs++;
        if (!more) break;
        if (!ok) continue;
        const uint8_t* kb = (const uint8_t*)P.k + w.kvh * P.khs + row * P.kss + chunk * 16;
        const uint8_t* vb = (const uint8_t*)P.v + w.kvh * P.vhs + row * P.vss + chunk * 16;
        const uint8_t* sb = (const uint8_t*)(sv ? X.c.v + w.kvh * X.c.vhs + srow * X.c.vss : X.c.k + w.kvh * X.c.khs + srow * X.c.kss);
        // bytes from page to page and from position to position of this lane's kind
        const int64_t page_bytes = kind == 0 ? P.kps : kind == 1 ? P.vps : 2 * (kind == 2 ? X.c.kps : X.c.vps);
        const int64_t pos_bytes = kind == 0 ? P.kss : kind == 1 ? P.vss : 2 * (kind == 2 ? X.c.kss : X.c.vss);
        const int64_t k_step = ROWS * P.kss, v_step = ROWS * P.vss;
        auto entry_of = [&](int k) {  // LIST: the index that the list has for this lane's tile
            const int64_t v = w.c0 + (int64_t)k * QS_KEYS + tile * SP_TK;
            return LIST && v < w.c1 ? __ldg(w.list + page_of(P, (int)v)) : 0;
        };
        auto place_of_tile = [&](int k, int entry, uint32_t& keys) {  // bytes from the pool's start, the keys that are there
            keys = 0;
            const int64_t v = w.c0 + (int64_t)k * QS_KEYS + tile * SP_TK;
            if (v >= w.c1) return (int64_t)0;
            int x = page_of(P, (int)v), have = min(SP_TK, w.c1 - (int)v), low = 0;
            const int slot = (int)v - x * P.page_size;
            if constexpr (LIST) {
                x = entry;
                if (x >= P.max_pages) return (int64_t)0;
                const int64_t pos = (int64_t)x * P.page_size + slot;
                have = (int)min((int64_t)have, w.p_own - pos + 1);
                if (A.window > 0) low = (int)min(max(w.p_own - A.window + 1 - pos, (int64_t)0), (int64_t)SP_TK);
                if (have <= low) return (int64_t)0;
            } else if (A.window > 0 && w.one_token) {
                // (a lone token's first tile begins in front of its window: what lies there, it
                // may not be finite, is not there; tiles of several tokens look for that by themselves)
                low = min(max(w.p_own - A.window + 1 - (int)v, 0), SP_TK);
            }
            const int64_t g = __ldg(P.table + (int64_t)w.seq * P.table_stride + x);
            if ((uint64_t)g >= (uint64_t)P.n_pages) return (int64_t)0;
            keys = ((1u << have) - 1) & ~((1u << low) - 1);
            return g * page_bytes + slot * pos_bytes;
        };
        uint32_t keys;
        int64_t from = place_of_tile(0, entry_of(0), keys);
        int entry = entry_of(1);
        for (int k = 0; k < w.stages; k++, n++) {
            uint32_t next_keys;
            const int64_t next_from = place_of_tile(k + 1, entry, next_keys);
            entry = entry_of(k + 2);
            const uint32_t st = n % S;
            if (n >= S && !stream_wait(&B.empty[st], (n / S & 1) ^ 1, &B.abort)) {
                ok = false;
                break;
            }
            if (kind == 0) B.in[st][tile] = keys;
            const uint32_t base = st * Sh::STAGE, there = __ballot_sync(0xffffffffu, keys != 0);
#pragma unroll
            for (int x = 0; x < QS_TILES; x++) {
                if (!(there >> x & 1u)) continue;
                const uint8_t* kf = kb + __shfl_sync(0xffffffffu, from, x);
                const uint8_t* vf = vb + __shfl_sync(0xffffffffu, from, 8 + x);
                const uint8_t* sf = sb + __shfl_sync(0xffffffffu, from, (sv ? 24 : 16) + x);
#pragma unroll
                for (int y = 0; y < SP_TK / ROWS; y++) {
                    const uint32_t d = to + base + x * SP_TK * Sh::ROWB + y * 512;
                    cp16(d, kf + y * k_step, true);
                    cp16(d + Sh::CODES, vf + y * v_step, true);
                }
                cp_small<Sh::SCB>(to_s + base + x * SP_TK * Sh::SCB, sf, true);
            }
            cp_arrive(&B.full[st]);
            // (that arrival orders a lane's copies alone: its stores are published by one of their own)
            __syncwarp();
            if (lane == 0) mbar_arrive(&B.full[st]);
            from = next_from;
            keys = next_keys;
        }
    }
    cp_commit();
    cp_wait<0>();  // every copy has landed before the CTA ends
    if (pairs >= 2) pair_sync<QS_READ>(pairs & 1);  // (the last pair's, so that no barrier is left half full)
}

template <typename QT, int HD, int NQ, bool LIST>
__global__ void __launch_bounds__(QS_THREADS, NQ == 1 ? 3 : 2) k_paged_q4(const __grid_constant__ SplitArgs X) {
    using Sh = StreamShape<HD, NQ, sizeof(QT) == 4>;
    constexpr int R = 8 * NQ, S = Sh::STAGES, ROWB = Sh::ROWB, SCB = Sh::SCB, LDO = Sh::LDO;
    constexpr bool HILO = sizeof(QT) == 4;
    constexpr int DT = HD / 16, KS = HD / 16, LE = HD / 4, FW = HILO ? 4 : 2;
    // the maximum stays until a score passes it by 2^TAU; weights are held times
    // 2^BIAS in fp16, so that one of 2^-25 of the largest still has 11 bits
    constexpr float BIAS = 11.0f, TAU = 4.0f;
    const PagedAttnArgs& A = X.a;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 127u);
    __shared__ StreamBars<S> B;
    __shared__ LineTable line;
    __shared__ float s_m[QS_WARPS][R], s_l[QS_WARPS][R], s_cf[R];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; i++) {
            mbar_init(&B.full[i], 33);  // 32 lanes' copies, and the keys' masks
            mbar_init(&B.empty[i], QS_WARPS);
        }
        B.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1 && A.p.n_seqs <= 32) fill_table<LIST>(X, line);
    __syncthreads();
    pdl_trigger();  // the join may become resident; it waits for this grid's end
    const uint32_t ring = smem_u32(smem);
    if (warp == QS_WARPS) {
        int64_t u = blockIdx.x, u_end = u + 1;
        if (!X.whole) {
            const int64_t run = run_of(A.p.n_seqs <= 32 ? line.units : all_units<LIST>(X), X.ctas);
            u = blockIdx.x * run;
            u_end = u + run;
        }
        stream_copies<Sh, HD, LIST>(X, line, B, ring, u, u_end);
        return;
    }
    uint8_t* outs = smem + S * Sh::STAGE;
    uint32_t* qf = reinterpret_cast<uint32_t*>(outs);  // until the outputs: [tile of rows][16 elements][lane][hi, hi (, lo, lo)]
    const uint32_t qs = smem_u32(qf);
    uint32_t st = 0, phase = 0;  // the next stage and the parity of its round
    bool lost = false;
    const int c = lane & 3, col = 2 * c, k0 = q4_key(lane >> 2);
    for (uint32_t pairs = 0;; pairs++) {
        pair_sync<QS_TOLD>(pairs & 1);  // (by then the outputs before have been read, too)
        // (read where it is needed: kept in registers it would cost a warp's worth of them)
        const volatile PairWork& w = B.work[pairs & 1];
        const int stages = w.stages, c0 = w.c0;
        if (stages < 0) break;
        lost |= w.lost != 0;
        // ---- queries as B fragments, once for all warps: eight elements a thread
        constexpr int QW = HD / 8;
        for (int i = threadIdx.x; i < R * QW; i += QS_ROWS) {  // (whole warps: R QW is a multiple of 32)
            const int m = i / QW, kw = i % QW;
            const bool in = m < w.mrows;
            const int t = token_of(A, w.m0 + m);
            const QT* q = (const QT*)A.q + (in ? (int64_t)(w.r0 + t) * A.q_rs + (w.kvh * A.G + (w.m0 + m) - t * A.G) * A.q_hs : 0);
            // (a factor below zero turns the query's sign)
            float f = fabsf(A.scale) * LOG2E;
            float x[8], top = 0.0f, by = A.scale < 0.0f ? -1.0f : 1.0f;
            load_q8(q, in, A.qvec, 8 * kw, x);
            if constexpr (HILO) {
#pragma unroll
                for (int y = 0; y < 8; y++) top = fmaxf(top, fabsf(x[y]));
#pragma unroll
                for (int d = 1; d < QW; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                // 2^e <= max |q| < 2^(e + 1), e within what 2^e and 2^-e can be
                const int e = min(max((int)(__float_as_uint(top) >> 23), 2), 252);
                by *= __uint_as_float((uint32_t)(254 - e) << 23);
                f *= __uint_as_float((uint32_t)e << 23);
            }
            // Scores are masked with -inf before they are multiplied, so the factor is above zero: a
            // product with 2^-126 of a score below 2^90 is as good as zero, one that is not finite stays so.
            if (kw == 0) s_cf[m] = f < 0x1p-126f ? 0x1p-126f : f;
            const int part = kw / (LE / 8), k = kw % (LE / 8);  // word k of lane part's share of a key
            uint32_t* to = qf + ((m >> 3) * KS * 32 + (m & 7) * 4 + part) * FW;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t* z = to + (2 * k + (j >> 1)) * 32 * FW + (j & 1);
                if constexpr (HILO) split2(x[j] * by, x[4 + j] * by, z[0], z[2]);
                else z[0] = pack(x[j] * by, x[4 + j] * by);
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(QS_ROWS) : "memory");
        float cf[NQ][2];  // score factors of this thread's two columns, above zero
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int y = 0; y < 2; y++) cf[n][y] = s_cf[n * 8 + col + y];
        float o[NQ][DT][4];
        float mx[NQ][2], sum[NQ][2];  // running maximum in log2 units; sum of this thread's keys only
#pragma unroll
        for (int n = 0; n < NQ; n++) {
#pragma unroll
            for (int t = 0; t < DT; t++)
#pragma unroll
                for (int y = 0; y < 4; y++) o[n][t][y] = 0.0f;
            mx[n][0] = mx[n][1] = -INFINITY;
            sum[n][0] = sum[n][1] = 0.0f;
        }
        for (int k = 0; k < stages; k++) {
            if (!lost && !stream_wait(&B.full[st], phase, &B.abort)) lost = true;
            __syncwarp();
            const uint32_t base = ring + st * Sh::STAGE;
            const uint32_t kt = base + warp * 2 * SP_TK * ROWB, vt = kt + Sh::CODES;
            const uint32_t ksc = base + 2 * Sh::CODES + warp * 2 * SP_TK * SCB, vsc = ksc + Sh::SCALES;
            const uint2 in2 = *reinterpret_cast<const uint2*>(&B.in[st][2 * warp]);
            const uint32_t in[2] = {in2.x, in2.y};
            const int j0 = c0 + k * QS_KEYS + warp * 2 * SP_TK;
            if ((in[0] | in[1]) && !lost) {
                // ---- S^T = K Q^T: [0], [1] = key k0 and this thread's two columns, [2], [3] = key k0 + 8
                float s[2][NQ][4], sl[HILO ? 2 : 1][HILO ? NQ : 1][4];
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int n = 0; n < NQ; n++)
#pragma unroll
                        for (int y = 0; y < 4; y++) {
                            s[b][n][y] = 0.0f;
                            if constexpr (HILO) sl[b][n][y] = 0.0f;
                        }
                {
                    uint32_t w0[2][LE / 8], w1[2][LE / 8];
                    __half2 s0[2], s1[2], z0[2], z1[2];
#pragma unroll
                    for (int b = 0; b < 2; b++) {
                        q4_key_words<HD>(kt + b * SP_TK * ROWB, ksc + b * SP_TK * SCB, k0, HD, w0[b], s0 + b, z0 + b);
                        q4_key_words<HD>(kt + b * SP_TK * ROWB, ksc + b * SP_TK * SCB, k0 + 8, HD, w1[b], s1 + b, z1 + b);
                    }
#pragma unroll
                    for (int x = 0; x < LE / 8; x++) {
                        uint32_t q[NQ][2][FW];
#pragma unroll
                        for (int n = 0; n < NQ; n++)
#pragma unroll
                            for (int h = 0; h < 2; h++) lds_words<FW>(qs + ((n * KS + 2 * x + h) * 32 + lane) * FW * 4, q[n][h]);
#pragma unroll
                        for (int b = 0; b < 2; b++) {
                            uint32_t e[4], f[4];
                            q4_pairs(w0[b][x], s0[b], z0[b], e);
                            q4_pairs(w1[b][x], s1[b], z1[b], f);
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                const uint32_t a[4] = {e[2 * h], f[2 * h], e[2 * h + 1], f[2 * h + 1]};
#pragma unroll
                                for (int n = 0; n < NQ; n++) {
                                    mma16(s[b][n], a, q[n][h][0], q[n][h][1]);
                                    if constexpr (HILO) mma16(sl[b][n], a, q[n][h][2], q[n][h][3]);
                                }
                            }
                        }
                    }
                }
                if constexpr (HILO) {
#pragma unroll
                    for (int b = 0; b < 2; b++)
#pragma unroll
                        for (int n = 0; n < NQ; n++)
#pragma unroll
                            for (int y = 0; y < 4; y++) s[b][n][y] += sl[b][n][y];
                }
                // ---- weights
                const bool full = (in[0] & in[1]) == 0xffffu && (LIST || (j0 + 2 * SP_TK - 1 <= w.p_min && j0 >= w.l_max));
                // (position of a column's row, and the first one that it sees)
                auto row_of = [&](int n, int y, int& p, int& first) {
                    const int m = n * 8 + col + y;
                    p = m < w.mrows ? w.first + token_of(A, w.m0 + m) : -1;
                    first = A.window > 0 ? p - A.window + 1 : 0;
                };
                if (!full) {
#pragma unroll
                    for (int n = 0; n < NQ; n++)
#pragma unroll
                        for (int y = 0; y < 2; y++) {
                            int p = 0, lo = 0;
                            if (!LIST) row_of(n, y, p, lo);
#pragma unroll
                            for (int b = 0; b < 2; b++)
#pragma unroll
                                for (int z = 0; z < 2; z++) {
                                    const int key = k0 + z * 8, j = j0 + b * SP_TK + key;
                                    if (!(in[b] >> key & 1u) || (!LIST && (j > p || j < lo))) s[b][n][2 * z + y] = -INFINITY;
                                }
                        }
                }
#pragma unroll
                for (int n = 0; n < NQ; n++) {
                    float nm[2];
#pragma unroll
                    for (int y = 0; y < 2; y++) nm[y] = fmaxf(fmaxf(s[0][n][y], s[0][n][2 + y]), fmaxf(s[1][n][y], s[1][n][2 + y]));
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) {
                        nm[0] = fmaxf(nm[0], __shfl_xor_sync(0xffffffffu, nm[0], d));
                        nm[1] = fmaxf(nm[1], __shfl_xor_sync(0xffffffffu, nm[1], d));
                    }
                    nm[0] *= cf[n][0];
                    nm[1] *= cf[n][1];
                    if (__any_sync(0xffffffffu, nm[0] > mx[n][0] + TAU || nm[1] > mx[n][1] + TAU)) {
#pragma unroll
                        for (int y = 0; y < 2; y++) {
                            const float m = nm[y] > mx[n][y] + TAU ? nm[y] : mx[n][y];
                            const float f = m == mx[n][y] ? 1.0f : pow2<true>(mx[n][y] - m);
                            mx[n][y] = m;
                            sum[n][y] *= f;
#pragma unroll
                            for (int t = 0; t < DT; t++) {
                                o[n][t][y] *= f;
                                o[n][t][2 + y] *= f;
                            }
                        }
                    }
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        const float b = mx[n][y] == -INFINITY ? 0.0f : mx[n][y] - BIAS;
#pragma unroll
                        for (int i = 0; i < 2; i++)
#pragma unroll
                            for (int z = 0; z < 2; z++) s[i][n][2 * z + y] = pow2<true>(fmaf(s[i][n][2 * z + y], cf[n][y], -b));
                        sum[n][y] += (s[0][n][y] + s[0][n][2 + y]) + (s[1][n][y] + s[1][n][2 + y]);
                    }
                }
                // ---- O^T += V^T P^T
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    const uint32_t vt_b = vt + b * SP_TK * ROWB, vsc_b = vsc + b * SP_TK * SCB;
                    // A key that some rows of the tile see and others do not must not
                    // reach the latter through 0 * v where v is not finite: such a
                    // tile adds its products one by one, masked keys left out.
                    bool careful = false;
                    if (!LIST && !full && !w.one_token) {
                        uint32_t bad = 0;
                        for (int x = lane; x < SP_TK * SCB / 4; x += 32) bad |= (lds_u32(vsc_b + 4 * x) & 0x7C007C00u) + 0x04000400u;
                        careful = __any_sync(0xffffffffu, (bad & 0x80008000u) != 0);
                    }
                    if (!LIST && careful) {
                        for (int key = 0; key < SP_TK; key++) {
                            const int src = q4_key(key & 7) * 4 + c, j = j0 + b * SP_TK + key;
                            const bool key_in = in[b] >> key & 1u;
#pragma unroll
                            for (int n = 0; n < NQ; n++)
#pragma unroll
                                for (int y = 0; y < 2; y++) {
                                    const float p = __shfl_sync(0xffffffffu, key < 8 ? s[b][n][y] : s[b][n][2 + y], src);
                                    int row_p, row_lo;
                                    row_of(n, y, row_p, row_lo);
                                    if (!key_in || j > row_p || j < row_lo) continue;
#pragma unroll
                                    for (int t = 0; t < DT; t++)
#pragma unroll
                                        for (int z = 0; z < 2; z++)
                                            o[n][t][2 * z + y] = fmaf(p, q4_value<HD>(vt_b, vsc_b, key, (lane >> 2) * (HD / 8) + 2 * t + z), o[n][t][2 * z + y]);
                                }
                            __syncwarp();
                        }
                        continue;
                    }
                    uint32_t ph[NQ][2], pl[HILO ? NQ : 1][2];  // P^T as B fragments
#pragma unroll
                    for (int n = 0; n < NQ; n++)
#pragma unroll
                        for (int y = 0; y < 2; y++) {
                            if constexpr (HILO) {
                                split2(s[b][n][2 * y], s[b][n][2 * y + 1], ph[n][y], pl[n][y]);
                                pl[n][y] = mov_trans(pl[n][y]);
                            } else {
                                ph[n][y] = pack(s[b][n][2 * y], s[b][n][2 * y + 1]);
                            }
                            ph[n][y] = mov_trans(ph[n][y]);
                        }
                    uint32_t vw[4][LE / 16];
                    __half2 sv[2], sz[2];
                    q4_value_words<HD>(vt_b, vsc_b, in[b], vw, sv, sz);
#pragma unroll
                    for (int h = 0; h < HD / 32; h++) {  // four columns
                        uint32_t e[4], f[4];
                        q4_pairs(__byte_perm(vw[0][h / 2], vw[1][h / 2], h & 1 ? 0x7632 : 0x5410), sv[0], sz[0], e);
                        q4_pairs(__byte_perm(vw[2][h / 2], vw[3][h / 2], h & 1 ? 0x7632 : 0x5410), sv[1], sz[1], f);
#pragma unroll
                        for (int y = 0; y < 2; y++) {
                            const uint32_t a[4] = {e[2 * y], e[2 * y + 1], f[2 * y], f[2 * y + 1]};
                            const int t = 2 * h + y;
#pragma unroll
                            for (int n = 0; n < NQ; n++) {
                                if constexpr (HILO) {
                                    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                                    mma16(d, a, pl[n][0], pl[n][1]);
                                    mma16(d, a, ph[n][0], ph[n][1]);
#pragma unroll
                                    for (int z = 0; z < 4; z++) o[n][t][z] += d[z];
                                } else {
                                    mma16(o[n][t], a, ph[n][0], ph[n][1]);
                                }
                            }
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&B.empty[st]);
            if (++st == S) {
                st = 0;
                phase ^= 1;
            }
        }
        if (lost) {  // (a copy that never came: not a number, rather than a wrong one)
#pragma unroll
            for (int n = 0; n < NQ; n++) sum[n][0] = sum[n][1] = __int_as_float(0x7FC00000);
        }

        // ---- this warp's (m, l, o) to shared memory (where the queries were), the four warps' joined
        asm volatile("bar.sync 1, %0;" ::"n"(QS_ROWS) : "memory");
        float* so = reinterpret_cast<float*>(outs + warp * Sh::OUT);
#pragma unroll
        for (int n = 0; n < NQ; n++) {
#pragma unroll
            for (int y = 0; y < 2; y++) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) sum[n][y] += __shfl_xor_sync(0xffffffffu, sum[n][y], d);
                if (lane < 4) {
                    s_m[warp][n * 8 + col + y] = mx[n][y];
                    s_l[warp][n * 8 + col + y] = sum[n][y];
                }
#pragma unroll
                for (int t = 0; t < DT; t++)
                    *reinterpret_cast<float2*>(so + (n * 8 + col + y) * LDO + (lane >> 2) * (HD / 8) + 2 * t) = make_float2(o[n][t][y], o[n][t][2 + y]);
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(QS_ROWS) : "memory");
        constexpr int HQ = HD >> 2;
        for (int x = threadIdx.x; x < w.mrows * HQ; x += QS_ROWS) {
            const int m = x / HQ, d = (x - m * HQ) * 4;
            float mm = -INFINITY;
#pragma unroll
            for (int i = 0; i < QS_WARPS; i++) mm = fmaxf(mm, s_m[i][m]);
            float l = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < QS_WARPS; i++) {
                if (s_l[i][m] == 0.0f) continue;  // saw nothing
                const float f = exp2f(s_m[i][m] - mm);
                const float4 y = *reinterpret_cast<const float4*>(outs + i * Sh::OUT + (m * LDO + d) * 4);
                l = fmaf(f, s_l[i][m], l);
                v.x = fmaf(f, y.x, v.x);
                v.y = fmaf(f, y.y, v.y);
                v.z = fmaf(f, y.z, v.z);
                v.w = fmaf(f, y.w, v.w);
            }
            if (!w.cut) {
                const int t = token_of(A, w.m0 + m), row = w.r0 + t, head = w.kvh * A.G + (w.m0 + m) - t * A.G;
                store_row4<QT>(A, row, head, d, l, v);
                if (A.lse && d == 0) A.lse[(int64_t)row * A.nh + head] = l == 0.0f ? -INFINITY : (mm - BIAS + log2f(l)) / LOG2E;
            } else {
                *reinterpret_cast<float4*>(X.po + (w.slot * R + m) * HD + d) = v;
                if (d == 0) X.pml[w.slot * R + m] = make_float2(mm == -INFINITY ? mm : mm - BIAS, l);
            }
        }
        __syncwarp();
        pair_arrive<QS_READ>(pairs & 1);
    }
}

template <typename QT, int HD, int NQ, bool LIST>
int launch_stream_t(SplitArgs& X, cudaStream_t s) {
    using Sh = StreamShape<HD, NQ, sizeof(QT) == 4>;
    static std::atomic<uint64_t> asked{0};
    HC_TRY(ask_smem((const void*)k_paged_q4<QT, HD, NQ, LIST>, Sh::SMEM, asked));
    static const int resident = [] {
        int n = 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k_paged_q4<QT, HD, NQ, LIST>, QS_THREADS, Sh::SMEM) != cudaSuccess) n = 1;
        return std::min(std::max(n, 1), SP_CTAS / 148);
    }();
    X.ctas = 148 * resident;
    const int64_t pairs = pairs_bound(X);
    HC_CHECK(pairs <= 0x7fffffff, HC_ERR_INVALID, "paged attention: %d rows of %d heads", X.a.p.n_rows, X.a.nh);
    k_paged_q4<QT, HD, NQ, LIST><<<X.whole ? (unsigned)pairs : (unsigned)X.ctas, QS_THREADS, Sh::SMEM, s>>>(X);
    HC_LAUNCH_CHECK();
    return X.whole ? HC_OK : launch_join<QT, LIST>(X, pairs, s);
}

template <typename QT, bool LIST>
int launch_stream_hd(SplitArgs& X, cudaStream_t s) {
    if (X.rows == 8) return X.a.p.hd == 64 ? launch_stream_t<QT, 64, 1, LIST>(X, s) : launch_stream_t<QT, 128, 1, LIST>(X, s);
    return X.a.p.hd == 64 ? launch_stream_t<QT, 64, 2, LIST>(X, s) : launch_stream_t<QT, 128, 2, LIST>(X, s);
}

}  // namespace

int launch_q4_stream(SplitArgs& X, int q16, cudaStream_t s) {
    if (X.l.width) return q16 ? launch_stream_hd<__half, true>(X, s) : launch_stream_hd<float, true>(X, s);
    return q16 ? launch_stream_hd<__half, false>(X, s) : launch_stream_hd<float, false>(X, s);
}

}  // namespace hc
