// Attention over a paged cache for sequences with few rows (single tokens,
// short chunks): split over the keys, joined at the end.
//
// A CTA takes up to R = 8 or 16 packed (token, query head of the group) rows of
// one (sequence, KV head) and a run of its visible positions; each of its four
// warps takes every fourth tile of 16 keys, with a cp.async ring of its own
// (no barrier between warps while the keys stream).  Per tile and row
//   s_j = c q.k_j,  m' = max(m, s_j),  p_j = 2^(s_j - m'),
//   l' = l 2^(m - m') + sum p_j,  o' = o 2^(m - m') + sum p_j v_j
// with c = scale log2(e).  The warps' (m, l, o) are joined in shared memory, the
// CTAs' by k_paged_join in a fixed order.
//
// Bound by the bytes of K and V: each is read once, and R rows share it.  8
// sequences of up to 32,768 FP16 keys, 64 heads over 8 of 128: 139 us, 5.8 TB/s;
// with f32 queries by latency: twelve warps an SM wait for chains of dependent
// two-part products (32 sequences of up to 2,304 keys, 32 heads over 8: 41 us,
// 4.4 TB/s; issue slots 42%, tensor pipe 17%).  FP32 cache: likewise, with three
// products and the splitting of both operands (32 full sequences of 2,304 keys:
// 223 us, 2.7 TB/s; 512 tokens over 4,096 keys: 1.8 ms, 18 TFLOP/s).
// Products: mma.sync on S^T = K Q^T and O^T = V^T P^T, keys and head columns on
// the 16-row side and the query rows on the 8-column side (8 rows a CTA where a
// token's group fits them, 57 us, 16 rows 73: 32 full sequences of 2,304 keys, f32
// queries; a token of a group
// of 4 or 8 heads fills half or all of it; the other way round, 16 query rows
// would waste twice that, and the tcgen05 forms pad them to 64 or 128).  FP16
// cache: m16n8k16 f16 products, K and V exact; f32 queries enter as
// q = 2^e (hi + lo) with hi, lo fp16 and e the row's own (22 bits, any range),
// their weights as hi + lo too.  FP32 cache: m16n8k8 tf32 products of both
// operands split in two (hi hi + hi lo + lo hi, 22 bits, the full exponent
// range).  Over an FP16 cache weights are held times 2^14 in fp16, so that one of
// 2^-28 of the largest still has 11 bits; with 16-bit queries in one part (half
// the products; the sums take them unrounded), which adds to a result's own
// rounding less than that itself: relative error against 64 bits 2.2e-4 where f32
// weights have 2.1e-4 (single tokens over 32,768 keys).
#include "hc_paged.h"

namespace hc {

namespace {

constexpr int SP_TK = 16, SP_WARPS = 4, SP_THREADS = 128;
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t* r, uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a));
}
__device__ __forceinline__ void mma16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Transposes an 8 x 8 matrix of 16-bit values held by the warp.
__device__ __forceinline__ uint32_t mov_trans(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// x = hi + lo with both in tf32 (10 mantissa bits, rounded)
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) + 0x1000u;
}

// Work is counted in units of 64 positions (16 for each warp).  A sequence has
// tiles x nkv pairs of (row tile, KV head) and every pair of it the same
// number of units; the pairs of all sequences in order form one line of units.
// With `whole`, CTA i takes pair i.  Otherwise every CTA takes an equal run of
// the line, whatever the lengths of the sequences, and a pair that is cut
// leaves partial results to k_paged_join; a CTA cuts at most two (its first
// and its last), so it has two slots.
constexpr int UNIT = SP_WARPS * SP_TK;
constexpr int SP_CTAS = 148 * 3;  // at most: CTAs of the cut line, as many as are resident at once
constexpr int MIN_UNITS = 4;      // of a run: a CTA's start costs about as much as the stream of 256 keys

struct SplitArgs {
    PagedAttnArgs a;
    int whole;
    int ctas;     // CTAs of the line (cut)
    int rows;     // R, rows of a tile
    float* po;    // [slot][R][hd] partial outputs, slot = 2 CTA + (0: its first pair, 1: its last)
    float2* pml;  // [slot][R] (maximum in log2 units, sum)
};

struct SeqWork {
    int r0, r1, first;  // rows, position of the first row
    int units, pairs;   // units of a pair, pairs
};
__device__ __forceinline__ SeqWork seq_work(const PagedAttnArgs& A, int R, int b) {
    SeqWork w;
    seq_rows(A.p, b, w.r0, w.r1);
    const int T = w.r1 - w.r0;
    w.first = seq_len(A.p, b) - T;
    const int64_t tiles = ((int64_t)T * A.G + R - 1) / R;
    // positions seen by any tile, at most: the last tile's end from the first tile's begin, per tile no
    // more than its window and its own tokens
    int len = min(max(0, w.first + T), A.p.reach);
    if (A.window > 0) len = (int)min((int64_t)len, (int64_t)A.window + R);
    w.units = max(1, len / UNIT + (len % UNIT != 0));
    w.pairs = (int)(tiles * A.p.nkv);
    return w;
}

// A place on the line of units: sequence b, which begins at `base`.
struct Line {
    int b;
    int64_t base;
    SeqWork w;
};
// Moves on to the sequence that holds unit u (a whole warp; false past the end).
__device__ __forceinline__ bool advance(const PagedAttnArgs& A, int R, int64_t u, bool whole, Line& at) {
    const int lane = threadIdx.x & 31;
    while (at.b < A.p.n_seqs) {
        SeqWork w = {0, 0, 0, 1, 0};
        if (at.b + lane < A.p.n_seqs) w = seq_work(A, R, at.b + lane);
        const int64_t n = (int64_t)w.pairs * (whole ? 1 : w.units);
        int64_t incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t t = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += t;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, at.base + incl > u);
        if (hit) {
            const int l = __ffs(hit) - 1;
            at.b += l;
            at.base += __shfl_sync(0xffffffffu, incl, l) - __shfl_sync(0xffffffffu, n, l);
            at.w.r0 = __shfl_sync(0xffffffffu, w.r0, l);
            at.w.r1 = __shfl_sync(0xffffffffu, w.r1, l);
            at.w.first = __shfl_sync(0xffffffffu, w.first, l);
            at.w.units = __shfl_sync(0xffffffffu, w.units, l);
            at.w.pairs = __shfl_sync(0xffffffffu, w.pairs, l);
            return true;
        }
        at.base += __shfl_sync(0xffffffffu, incl, 31);
        at.b += 32;
    }
    return false;
}
// Units of all sequences, and of one CTA's run.
__device__ __forceinline__ int64_t all_units(const PagedAttnArgs& A, int R) {
    int64_t n = 0;
    for (int b = threadIdx.x & 31; b < A.p.n_seqs; b += 32) {
        const SeqWork w = seq_work(A, R, b);
        n += (int64_t)w.pairs * w.units;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
}
__device__ __forceinline__ int64_t run_of(int64_t units, int ctas) {
    return max((units + ctas - 1) / ctas, (int64_t)MIN_UNITS);
}

template <typename CT, int HD>
struct SplitShape {
    static constexpr int ROWB = HD * (int)sizeof(CT);           // bytes of a key in shared memory
    static constexpr int STAGE = 2 * SP_TK * ROWB;              // K tile, V tile
    static constexpr int STAGES = STAGE > 8192 ? 3 : (STAGE > 4096 ? 2 : 4);  // three CTAs an SM before a deeper ring
    static constexpr int WARPB = STAGES * STAGE;
    static constexpr int SMEM = SP_WARPS * WARPB + 512;         // 512: rows are aligned to their size
    static constexpr int LDO = HD + 4;                          // row of outputs: conflict-free column stores
    static_assert(WARPB >= 16 * LDO * 4, "a warp's outputs fit its ring");
};

template <typename QT, typename CT, int HD, int NQ>
__global__ void __launch_bounds__(SP_THREADS) k_paged_split(const __grid_constant__ SplitArgs X) {
    using Sh = SplitShape<CT, HD>;
    constexpr bool C16 = sizeof(CT) == 2;
    constexpr bool HILO = C16 && sizeof(QT) == 4;
    // Operands in two parts: the tensor core cuts (does not round) the low
    // bits of a running sum, so the small products get a sum of their own (or
    // a short one) and the running outputs are added to by f32 adds.
    constexpr int R = 8 * NQ;
    constexpr int S = Sh::STAGES, ROWB = Sh::ROWB, LDO = Sh::LDO;
    constexpr int EPC = 16 / (int)sizeof(CT);    // elements of a 16-byte chunk
    constexpr int CPL = HD / EPC / 4;            // chunks of a row per lane (four lanes copy a row)
    constexpr int DT = HD / 16;                  // output row tiles
    const PagedAttnArgs& A = X.a;
    const PagedArgs& P = A.p;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 511u);
    __shared__ float s_m[SP_WARPS][R], s_l[SP_WARPS][R];
    __shared__ uint32_t s_in[SP_WARPS][S];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_trigger();  // the join may become resident; it waits for this grid's end

    int64_t u, u_end;
    if (X.whole) {
        u = blockIdx.x;
        u_end = u + 1;
    } else {
        const int64_t run = run_of(all_units(A, R), X.ctas);
        u = blockIdx.x * run;
        u_end = u + run;
    }
    const int64_t u_begin = u;
    Line at = {0, 0, {}};
    while (u < u_end && advance(A, R, u, X.whole != 0, at)) {
        const int seq = at.b, r0 = at.w.r0, first = at.w.first;
        const int64_t rem = u - at.base;
        const int pair = (int)(X.whole ? rem : rem / at.w.units);
        const int unit = X.whole ? 0 : (int)(rem - (int64_t)pair * at.w.units);
        const int nunits = X.whole ? at.w.units : (int)min((int64_t)(at.w.units - unit), u_end - u);
        const bool cut = nunits < at.w.units;
        const int64_t slot = 2 * (int64_t)blockIdx.x + (u == u_begin ? 0 : 1);
        u += X.whole ? 1 : nunits;
        const int kvh = pair % P.nkv, m0 = pair / P.nkv * R;
        const int mrows = (int)min((int64_t)R, (int64_t)(at.w.r1 - r0) * A.G - m0);
        int begin, end;
        visible(A, first, m0, mrows, begin, end);
        const int c0 = (int)min((int64_t)end, begin + (int64_t)unit * UNIT);
        const int c1 = (int)min((int64_t)end, c0 + (int64_t)nunits * UNIT);

        // ---- the keys' ring: this lane copies a quarter of rows kr and kr + 8
        const uint32_t ring = smem_u32(smem) + warp * Sh::WARPB;
        const int ntiles = (c1 - c0 + SP_TK - 1) / SP_TK;
        const int mine = ntiles > warp ? (ntiles - warp + SP_WARPS - 1) / SP_WARPS : 0;
        const int kr = lane >> 2;
        const uint32_t put = (uint32_t)(kr * ROWB + (((lane & 3) ^ kr) << 4));
        int slot0, slot1, page0, page1;
        auto look = [&](int i) {
            const int j = c0 + (warp + i * SP_WARPS) * SP_TK + kr;
            page0 = page1 = -1;
            slot0 = slot1 = 0;
            if (i < mine) {
                if (j < c1) page0 = lookup(P, seq, j, slot0);
                if (j + 8 < c1) page1 = lookup(P, seq, j + 8, slot1);
            }
        };
        look(0);
        auto issue = [&](int i) {
            if (i < mine) {
                const uint32_t b0 = __ballot_sync(0xffffffffu, page0 >= 0), b1 = __ballot_sync(0xffffffffu, page1 >= 0);
                if (lane == 0) {  // one bit per key: the lanes of a row agree
                    uint32_t in = 0;
#pragma unroll
                    for (int r = 0; r < 8; r++) in |= ((b0 >> (4 * r)) & 1u) << r | ((b1 >> (4 * r)) & 1u) << (8 + r);
                    s_in[warp][i % S] = in;
                }
                const uint32_t dst = ring + (i % S) * Sh::STAGE + put;
                const int64_t e = (lane & 3) * EPC, h0 = max(page0, 0), h1 = max(page1, 0);
                const CT* k0 = (const CT*)P.k + h0 * P.kps + kvh * P.khs + slot0 * P.kss + e;
                const CT* k1 = (const CT*)P.k + h1 * P.kps + kvh * P.khs + slot1 * P.kss + e;
                const CT* v0 = (const CT*)P.v + h0 * P.vps + kvh * P.vhs + slot0 * P.vss + e;
                const CT* v1 = (const CT*)P.v + h1 * P.vps + kvh * P.vhs + slot1 * P.vss + e;
#pragma unroll
                for (int x = 0; x < CPL; x++) {
                    const bool d_in = (int)e + 4 * x * EPC < P.hd;  // elements past head_dim are zeros, not read
                    const bool in0 = d_in && page0 >= 0, in1 = d_in && page1 >= 0;
                    const uint32_t o = dst ^ (uint32_t)(x << 6);
                    cp16(o, in0 ? k0 + 4 * x * EPC : (const CT*)P.k, in0);
                    cp16(o + 8 * ROWB, in1 ? k1 + 4 * x * EPC : (const CT*)P.k, in1);
                    cp16(o + SP_TK * ROWB, in0 ? v0 + 4 * x * EPC : (const CT*)P.v, in0);
                    cp16(o + (SP_TK + 8) * ROWB, in1 ? v1 + 4 * x * EPC : (const CT*)P.v, in1);
                }
                look(i + 1);
            }
            cp_commit();
        };
#pragma unroll
        for (int i = 0; i < S - 1; i++) issue(i);

        // ---- queries as B fragments: column lane / 4 of each tile of eight rows
        constexpr int KS = C16 ? HD / 16 : HD / 8;
        uint32_t qh[NQ][KS][2];
        uint32_t ql[HILO ? NQ : 1][HILO ? KS : 1][2];
        float cf[NQ][2];                    // score factors of this thread's two columns, 2 (lane % 4) and + 1
        int ps[NQ][2], lo[NQ][2];           // their positions and first visible positions
        const int col = 2 * (lane & 3);
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            const int m = n * 8 + (lane >> 2);
            const bool in = m < mrows;
            const int t = token_of(A, m0 + m);
            const QT* q = (const QT*)A.q + (in ? (int64_t)(r0 + t) * A.q_rs + (kvh * A.G + (m0 + m) - t * A.G) * A.q_hs : 0);
            float c = A.scale * LOG2E;
            if constexpr (C16) {
                float2 f[KS][2];
#pragma unroll
                for (int k = 0; k < KS; k++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int d = k * 16 + i * 8 + col;
                        f[k][i] = make_float2(0.0f, 0.0f);
                        if (in && d < P.hd) {
                            if (A.qvec) {
                                if constexpr (sizeof(QT) == 4) f[k][i] = *reinterpret_cast<const float2*>(q + d);
                                else f[k][i] = __half22float2(*reinterpret_cast<const __half2*>(q + d));
                            } else {
                                f[k][i] = make_float2(to_f32(q[d]), to_f32(q[d + 1]));
                            }
                        }
                    }
                if constexpr (HILO) {
                    float mx = 0.0f;
#pragma unroll
                    for (int k = 0; k < KS; k++)
#pragma unroll
                        for (int i = 0; i < 2; i++) mx = fmaxf(mx, fmaxf(fabsf(f[k][i].x), fabsf(f[k][i].y)));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    // 2^e <= max |q| < 2^(e + 1), e within what 2^e and 2^-e can be
                    const int e = min(max((int)(__float_as_uint(mx) >> 23), 2), 252);
                    const float down = __uint_as_float((uint32_t)(254 - e) << 23);
                    c *= __uint_as_float((uint32_t)e << 23);
#pragma unroll
                    for (int k = 0; k < KS; k++)
#pragma unroll
                        for (int i = 0; i < 2; i++) split2(f[k][i].x * down, f[k][i].y * down, qh[n][k][i], ql[n][k][i]);
                } else {
#pragma unroll
                    for (int k = 0; k < KS; k++)
#pragma unroll
                        for (int i = 0; i < 2; i++) qh[n][k][i] = pack(f[k][i].x, f[k][i].y);
                }
            } else {
#pragma unroll
                for (int k = 0; k < KS; k++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int d = k * 8 + i * 4 + (lane & 3);
                        qh[n][k][i] = __float_as_uint(in && d < P.hd ? to_f32(q[d]) : 0.0f);
                    }
            }
#pragma unroll
            for (int x = 0; x < 2; x++) {
                cf[n][x] = __shfl_sync(0xffffffffu, c, (col + x) * 4);
                const int mm = n * 8 + col + x;
                ps[n][x] = mm < mrows ? first + token_of(A, m0 + mm) : -1;
                lo[n][x] = A.window > 0 ? ps[n][x] - A.window + 1 : 0;
            }
        }
        // keys that every row of the tile sees
        const int p_min = first + token_of(A, m0), l_max = A.window > 0 ? first + token_of(A, m0 + mrows - 1) - A.window + 1 : 0;
        const bool one_token = token_of(A, m0) == token_of(A, m0 + mrows - 1);

        float o[NQ][DT][4];
        float mx[NQ][2], sum[NQ][2];  // running maximum; sum of this thread's keys only
#pragma unroll
        for (int n = 0; n < NQ; n++) {
#pragma unroll
            for (int t = 0; t < DT; t++)
#pragma unroll
                for (int x = 0; x < 4; x++) o[n][t][x] = 0.0f;
            mx[n][0] = mx[n][1] = -INFINITY;
            sum[n][0] = sum[n][1] = 0.0f;
        }
        constexpr float BIAS = C16 ? 14.0f : 0.0f;
        const int mi = lane >> 3;
        // ldmatrix rows: K as A (keys x d), V transposed as A (d x keys)
        const int krow = (lane & 7) + (mi & 1) * 8, vrow = (lane & 7) + (mi >> 1) * 8;
        const uint32_t kget = (uint32_t)(krow * ROWB + (((mi >> 1) ^ (krow & 7)) << 4));
        const uint32_t vget = (uint32_t)(vrow * ROWB + (((mi & 1) ^ (vrow & 7)) << 4));

        for (int i = 0; i < mine; i++) {
            cp_wait<S - 2>();
            __syncwarp();
            issue(i + S - 1);
            const uint32_t kt = ring + (i % S) * Sh::STAGE, vt = kt + SP_TK * ROWB;
            const uint32_t in = s_in[warp][i % S];
            const int j0 = c0 + (warp + i * SP_WARPS) * SP_TK;
            // S^T: [0], [1] = key lane / 4 and this thread's two columns, [2], [3] = key lane / 4 + 8
            float s[NQ][4], sl[HILO ? NQ : 1][4];
#pragma unroll
            for (int n = 0; n < NQ; n++)
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    s[n][x] = 0.0f;
                    if constexpr (HILO) sl[n][x] = 0.0f;
                }
            if constexpr (C16) {
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    uint32_t a[4];
                    ldsm4(a, (kt + kget) ^ (uint32_t)(k << 5));
#pragma unroll
                    for (int n = 0; n < NQ; n++) {
                        mma16(s[n], a, qh[n][k][0], qh[n][k][1]);
                        if constexpr (HILO) mma16(sl[n], a, ql[n][k][0], ql[n][k][1]);
                    }
                }
            } else {
                const int r = lane >> 2;
                const uint32_t base = kt + r * ROWB + 4 * (lane & 3) + (r << 4);  // chunk c of row r at c ^ r
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    uint32_t ah[4], al[4];
                    const uint32_t a0 = base ^ (uint32_t)((2 * k) << 4), a1 = base ^ (uint32_t)((2 * k + 1) << 4);
                    split_tf32(lds_f32(a0), ah[0], al[0]);
                    split_tf32(lds_f32(a0 + 8 * ROWB), ah[1], al[1]);
                    split_tf32(lds_f32(a1), ah[2], al[2]);
                    split_tf32(lds_f32(a1 + 8 * ROWB), ah[3], al[3]);
#pragma unroll
                    for (int n = 0; n < NQ; n++) {
                        uint32_t h0, l0, h1, l1;
                        split_tf32(__uint_as_float(qh[n][k][0]), h0, l0);
                        split_tf32(__uint_as_float(qh[n][k][1]), h1, l1);
                        float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        mma8(d, al, h0, h1);
                        mma8(d, ah, l0, l1);
                        mma8(d, ah, h0, h1);
#pragma unroll
                        for (int x = 0; x < 4; x++) s[n][x] += d[x];
                    }
                }
            }
            // scores in log2 units, masked ones -inf; the weights
            const bool whole = in == 0xffffu && j0 + SP_TK - 1 <= p_min && j0 >= l_max;
#pragma unroll
            for (int n = 0; n < NQ; n++) {
                float nm[2];
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    if constexpr (HILO) {
                        s[n][x] += sl[n][x];
                        s[n][2 + x] += sl[n][2 + x];
                    }
                    s[n][x] *= cf[n][x];
                    s[n][2 + x] *= cf[n][x];
                    if (!whole) {
                        const int jj = lane >> 2, j = j0 + jj;
                        if (!((in >> jj) & 1u) || j > ps[n][x] || j < lo[n][x]) s[n][x] = -INFINITY;
                        if (!((in >> (jj + 8)) & 1u) || j + 8 > ps[n][x] || j + 8 < lo[n][x]) s[n][2 + x] = -INFINITY;
                    }
                    nm[x] = fmaxf(s[n][x], s[n][2 + x]);
                }
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    nm[0] = fmaxf(nm[0], __shfl_xor_sync(0xffffffffu, nm[0], d));
                    nm[1] = fmaxf(nm[1], __shfl_xor_sync(0xffffffffu, nm[1], d));
                }
                if (__any_sync(0xffffffffu, nm[0] > mx[n][0] || nm[1] > mx[n][1])) {
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        const float m = fmaxf(nm[x], mx[n][x]);
                        const float f = m == mx[n][x] ? 1.0f : exp2f(mx[n][x] - m);
                        mx[n][x] = m;
                        sum[n][x] *= f;
#pragma unroll
                        for (int t = 0; t < DT; t++) {
                            o[n][t][x] *= f;
                            o[n][t][2 + x] *= f;
                        }
                    }
                }
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const float b = mx[n][x] == -INFINITY ? 0.0f : mx[n][x] - BIAS;
                    s[n][x] = exp2f(s[n][x] - b);
                    s[n][2 + x] = exp2f(s[n][2 + x] - b);
                    sum[n][x] += s[n][x] + s[n][2 + x];
                }
            }
            // A key that some rows of the tile see and others do not must not
            // reach the latter through 0 * v where v is not finite: such a
            // tile adds its products one by one, masked keys left out.
            bool careful = false;
            if (!whole && !one_token) {
                uint32_t bad = 0;
                if constexpr (C16) {
                    for (int x = lane; x < SP_TK * HD / 2; x += 32)
                        bad |= (__float_as_uint(lds_f32(vt + 4 * x)) & 0x7C007C00u) + 0x04000400u;
                    bad &= 0x80008000u;
                } else {
                    for (int x = lane; x < SP_TK * HD; x += 32)
                        bad |= (__float_as_uint(lds_f32(vt + 4 * x)) & 0x7F800000u) + 0x00800000u;
                    bad &= 0x80000000u;
                }
                careful = __any_sync(0xffffffffu, bad != 0);
            }
            if (careful) {
                for (int jj = 0; jj < SP_TK; jj++) {
                    const int src = (jj & 7) * 4 + (lane & 3), j = j0 + jj;
                    const bool key_in = (in >> jj) & 1u;
#pragma unroll
                    for (int n = 0; n < NQ; n++)
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            const float p = __shfl_sync(0xffffffffu, jj < 8 ? s[n][x] : s[n][2 + x], src);
                            if (!key_in || j > ps[n][x] || j < lo[n][x]) continue;
#pragma unroll
                            for (int t = 0; t < DT; t++)
#pragma unroll
                                for (int y = 0; y < 2; y++) {
                                    const int d = t * 16 + y * 8 + (lane >> 2);
                                    const uint32_t ad = vt + jj * ROWB + (((d / EPC) ^ (jj & 7)) << 4) + (d % EPC) * (int)sizeof(CT);
                                    float v;
                                    if constexpr (C16) v = __half2float(lds_f16(ad));
                                    else v = lds_f32(ad);
                                    o[n][t][2 * y + x] = fmaf(p, v, o[n][t][2 * y + x]);
                                }
                        }
                    __syncwarp();
                }
            } else if constexpr (C16) {
                uint32_t ph[NQ][2], pl[HILO ? NQ : 1][2];  // P^T as B fragments
#pragma unroll
                for (int n = 0; n < NQ; n++)
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        if constexpr (HILO) {
                            split2(s[n][2 * y], s[n][2 * y + 1], ph[n][y], pl[n][y]);
                            pl[n][y] = mov_trans(pl[n][y]);
                        } else {
                            ph[n][y] = pack(s[n][2 * y], s[n][2 * y + 1]);
                        }
                        ph[n][y] = mov_trans(ph[n][y]);
                    }
#pragma unroll
                for (int t = 0; t < DT; t++) {
                    uint32_t a[4];
                    ldsm4t(a, (vt + vget) ^ (uint32_t)(t << 5));
#pragma unroll
                    for (int n = 0; n < NQ; n++) {
                        if constexpr (HILO) {
                            float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma16(d, a, pl[n][0], pl[n][1]);
                            mma16(d, a, ph[n][0], ph[n][1]);
#pragma unroll
                            for (int x = 0; x < 4; x++) o[n][t][x] += d[x];
                        } else {
                            mma16(o[n][t], a, ph[n][0], ph[n][1]);
                        }
                    }
                }
            } else {
                // P^T as B fragments: key lane % 4 (+ 4), row lane / 4, of each eight keys
                uint32_t bh[NQ][2][2], bl[NQ][2][2];
#pragma unroll
                for (int n = 0; n < NQ; n++)
#pragma unroll
                    for (int y = 0; y < 2; y++)
#pragma unroll
                        for (int z = 0; z < 2; z++) {
                            const int src = ((lane & 3) + 4 * z) * 4 + (lane >> 3);
                            const float e = __shfl_sync(0xffffffffu, s[n][2 * y], src), f = __shfl_sync(0xffffffffu, s[n][2 * y + 1], src);
                            split_tf32((lane >> 2) & 1 ? f : e, bh[n][y][z], bl[n][y][z]);
                        }
                const int ka = lane & 3;
#pragma unroll
                for (int t = 0; t < DT; t++) {
                    float d[NQ][4];
#pragma unroll
                    for (int n = 0; n < NQ; n++)
#pragma unroll
                        for (int x = 0; x < 4; x++) d[n][x] = 0.0f;
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        uint32_t ah[4], al[4];
#pragma unroll
                        for (int z = 0; z < 4; z++) {
                            const int dd = t * 16 + (z & 1) * 8 + (lane >> 2), key = y * 8 + ka + (z >> 1) * 4;
                            split_tf32(lds_f32(vt + key * ROWB + (((dd >> 2) ^ (key & 7)) << 4) + 4 * (dd & 3)), ah[z], al[z]);
                        }
#pragma unroll
                        for (int n = 0; n < NQ; n++) {
                            mma8(d[n], al, bh[n][y][0], bh[n][y][1]);
                            mma8(d[n], ah, bl[n][y][0], bl[n][y][1]);
                            mma8(d[n], ah, bh[n][y][0], bh[n][y][1]);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NQ; n++)
#pragma unroll
                        for (int x = 0; x < 4; x++) o[n][t][x] += d[n][x];
                }
            }
            __syncwarp();
        }
        cp_wait<0>();
        __syncwarp();

        // ---- this warp's (m, l, o) to shared memory (over its ring)
        float* so = reinterpret_cast<float*>(smem + warp * Sh::WARPB);
#pragma unroll
        for (int n = 0; n < NQ; n++) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) sum[n][x] += __shfl_xor_sync(0xffffffffu, sum[n][x], d);
                if (lane < 4) {
                    s_m[warp][n * 8 + col + x] = mx[n][x];
                    s_l[warp][n * 8 + col + x] = sum[n][x];
                }
#pragma unroll
                for (int t = 0; t < DT; t++)
#pragma unroll
                    for (int y = 0; y < 2; y++) so[(n * 8 + col + x) * LDO + t * 16 + y * 8 + (lane >> 2)] = o[n][t][2 * y + x];
            }
        }
        __syncthreads();
        const int hq = P.hd >> 2;  // float4 columns (head_dim is a multiple of 4 here)
        for (int x = threadIdx.x; x < mrows * hq; x += SP_THREADS) {
            const int m = x / hq, d = (x - m * hq) * 4;
            float mm = -INFINITY;
#pragma unroll
            for (int w = 0; w < SP_WARPS; w++) mm = fmaxf(mm, s_m[w][m]);
            float l = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < SP_WARPS; w++) {
                if (s_l[w][m] == 0.0f) continue;  // saw nothing
                const float f = exp2f(s_m[w][m] - mm);
                const float4 y = *reinterpret_cast<const float4*>(smem + w * Sh::WARPB + (m * LDO + d) * 4);
                l = fmaf(f, s_l[w][m], l);
                v.x = fmaf(f, y.x, v.x);
                v.y = fmaf(f, y.y, v.y);
                v.z = fmaf(f, y.z, v.z);
                v.w = fmaf(f, y.w, v.w);
            }
            if (!cut) {
                const int t = token_of(A, m0 + m), row = r0 + t, head = kvh * A.G + (m0 + m) - t * A.G;
                store_row4<QT>(A, row, head, d, l, v);
                if (A.lse && d == 0)
                    A.lse[(int64_t)row * A.nh + head] = l == 0.0f ? -INFINITY : (mm - BIAS + log2f(l)) / LOG2E;
            } else {
                *reinterpret_cast<float4*>(X.po + (slot * R + m) * P.hd + d) = v;
                if (d == 0) X.pml[slot * R + m] = make_float2(mm == -INFINITY ? mm : mm - BIAS, l);
            }
        }
        __syncthreads();
    }
}

// Joins the partial results of a pair that was cut, in the order of the CTAs.
// Bound by latency (a pair has a few KB of them), so what can be worked out from
// the batch alone is done before the wait.  The batch may be read there: the
// kernel in front is not a programmatic dependent, so all that came before it
// (and may have written the batch) had ended when it began, and it writes only
// partial results and outputs.
template <typename QT>
__global__ void __launch_bounds__(SP_THREADS) k_paged_join(const __grid_constant__ SplitArgs X) {
    const PagedAttnArgs& A = X.a;
    const PagedArgs& P = A.p;
    const int64_t run = run_of(all_units(A, X.rows), X.ctas);
    Line at = {0, 0, {}};
    const bool any = advance(A, X.rows, blockIdx.x, true, at);  // pair blockIdx.x, counted in pairs
    const int seq = at.b, pair = (int)(blockIdx.x - at.base);
    // units before this sequence
    int64_t before = 0;
    for (int b = threadIdx.x & 31; b < seq; b += 32) {
        const SeqWork w = seq_work(A, X.rows, b);
        before += (int64_t)w.pairs * w.units;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    const int64_t p0 = before + (int64_t)pair * at.w.units, p1 = p0 + at.w.units;
    const int c0 = (int)(p0 / run), c1 = (int)((p1 - 1) / run);
    pdl_wait();  // (every CTA waits: the next kernel on the stream begins when this grid has ended)
    if (!any || c0 == c1) return;  // c0 == c1: one CTA took it whole
    const int kvh = pair % P.nkv, m0 = pair / P.nkv * X.rows, r0 = at.w.r0;
    const int mrows = (int)min((int64_t)X.rows, (int64_t)(at.w.r1 - r0) * A.G - m0);
    const int hq = P.hd >> 2;
    // the first CTA has it as its last pair, unless its run begins with the pair
    const int s0 = 2 * c0 + (c0 * run < p0 ? 1 : 0);
    auto slot = [&](int c) -> int64_t { return c == c0 ? s0 : 2 * (int64_t)c; };
    for (int x = blockIdx.y * SP_THREADS + threadIdx.x; x < mrows * hq; x += SP_THREADS * gridDim.y) {
        const int m = x / hq, d = (x - m * hq) * 4;
        float mx, l;
        float4 v;
        join_runs(c1 - c0 + 1, [&](int i) { return slot(c0 + i) * X.rows + m; }, X.po, X.pml, P.hd, d, mx, l, v);
        const int t = token_of(A, m0 + m), row = r0 + t, head = kvh * A.G + (m0 + m) - t * A.G;
        store_row4<QT>(A, row, head, d, l, v);
        if (A.lse && d == 0)
            A.lse[(int64_t)row * A.nh + head] = l == 0.0f ? -INFINITY : (mx + log2f(l)) / LOG2E;
    }
}

// Pairs of all sequences, at most.
int64_t pairs_bound(const SplitArgs& X) {
    return ((int64_t)X.a.p.n_rows * X.a.G / X.rows + X.a.p.n_seqs) * X.a.p.nkv;
}

template <typename QT, typename CT, int HD, int NQ>
int launch_split_t(SplitArgs& X, cudaStream_t s) {
    using Sh = SplitShape<CT, HD>;
    HC_CUDA(cudaFuncSetAttribute(k_paged_split<QT, CT, HD, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM));
    const PagedArgs& P = X.a.p;
    static const int resident = [] {  // CTAs an SM holds: the kernel's registers and shared memory decide
        int n = 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k_paged_split<QT, CT, HD, NQ>, SP_THREADS, Sh::SMEM) != cudaSuccess) n = 1;
        return std::min(std::max(n, 1), SP_CTAS / 148);
    }();
    X.ctas = 148 * resident;
    const int64_t pairs = pairs_bound(X);
    HC_CHECK(pairs <= 0x7fffffff, HC_ERR_INVALID, "paged attention: %d rows of %d heads", P.n_rows, X.a.nh);
    k_paged_split<QT, CT, HD, NQ><<<X.whole ? (unsigned)pairs : (unsigned)X.ctas, SP_THREADS, Sh::SMEM, s>>>(X);
    HC_LAUNCH_CHECK();
    if (!X.whole) {
        const int y = (std::min(X.rows, X.a.G) * P.hd / 4 + SP_THREADS - 1) / SP_THREADS;
        HC_TRY(launch_pdl(k_paged_join<QT>, dim3((unsigned)pairs, std::max(y, 1)), dim3(SP_THREADS), 0, s, X));
        HC_LAUNCH_CHECK();
    }
    return HC_OK;
}

template <typename QT, typename CT>
int launch_split_hd(SplitArgs& X, cudaStream_t s) {
    const int hd = X.a.p.hd;
    if constexpr (sizeof(CT) == 2) {
        if (hd > 128) return launch_split_t<QT, CT, 256, 1>(X, s);
    }
    if (X.rows == 8) return hd <= 64 ? launch_split_t<QT, CT, 64, 1>(X, s) : launch_split_t<QT, CT, 128, 1>(X, s);
    return hd <= 64 ? launch_split_t<QT, CT, 64, 2>(X, s) : launch_split_t<QT, CT, 128, 2>(X, s);
}

}  // namespace

bool paged_split_ok(const PagedArgs& P, int c16) {
    const int64_t e = c16 ? 8 : 4;
    return P.hd <= (c16 ? 256 : 128) && P.hd % e == 0 && ((uintptr_t)P.k | (uintptr_t)P.v) % 16 == 0 &&
           (P.kps | P.khs | P.kss | P.vps | P.vhs | P.vss) % e == 0;
}

size_t paged_split_bytes(const PagedAttnArgs& A, int max_q_len, int max_kv_len) {
    return paged_split_whole(A, max_q_len, max_kv_len) ? 0 : (size_t)2 * SP_CTAS * 16 * ((size_t)A.p.hd * 4 + 8);
}

// One CTA per pair where no pair is long enough to be worth cutting (64 sequences
// of 256 keys, 8 KV heads: 31 us cut, 21 whole; of 512 keys: 34 cut, 38 whole), and for
// chunks with many pairs: a chunk's early row tiles see fewer keys than the
// line counts for them, and a CTA's pairs cost a start each (7 chunks of 264
// tokens, 9 heads of 64, FP32 cache: 69 us cut, 51 whole).
bool paged_split_whole(const PagedAttnArgs& A, int max_q_len, int max_kv_len) {
    if ((int64_t)max_q_len * A.G > 64 && (int64_t)A.p.n_rows * A.G / 16 * A.p.nkv >= 2 * SP_CTAS) return true;
    const int64_t len = A.window > 0 ? std::min<int64_t>(max_kv_len, (int64_t)A.window + 16) : max_kv_len;
    return len <= MIN_UNITS * UNIT;
}

int launch_paged_split(const PagedAttnArgs& A, int q16, int c16, int max_q_len, int max_kv_len, void* ws,
                       cudaStream_t s) {
    SplitArgs X;
    X.a = A;
    X.whole = paged_split_whole(A, max_q_len, max_kv_len);
    // 16 rows of more than 128 elements do not fit the registers
    X.rows = (int64_t)max_q_len * A.G <= 8 || A.p.hd > 128 ? 8 : 16;
    X.po = (float*)ws;
    X.pml = (float2*)((float*)ws + (size_t)2 * SP_CTAS * 16 * A.p.hd);
    if (q16) return c16 ? launch_split_hd<__half, __half>(X, s) : launch_split_hd<__half, float>(X, s);
    return c16 ? launch_split_hd<float, __half>(X, s) : launch_split_hd<float, float>(X, s);
}

}  // namespace hc
