// Attention over a paged cache for sequences with few rows (single tokens,
// short chunks): split over the keys, joined at the end.
//
// A CTA takes up to 16 packed (token, query head of the group) rows of one
// (sequence, KV head) and a run of its visible positions; each of its four
// warps takes every fourth tile of 16 keys, with a cp.async ring of its own
// (no barrier between warps while the keys stream).  Per tile and row
//   s_j = c q.k_j,  m' = max(m, s_j),  p_j = 2^(s_j - m'),
//   l' = l 2^(m - m') + sum p_j,  o' = o 2^(m - m') + sum p_j v_j
// with c = scale log2(e).  The warps' (m, l, o) are joined in shared memory, the
// CTAs' by k_paged_join in a fixed order.
//
// Bound by the bytes of K and V: each is read once, and 16 rows share it.
// Products: mma.sync, because a 16-row tile fits its shape and the tcgen05
// forms would pad it to 128 rows.  FP16 cache: m16n8k16 f16 products, K and V
// exact; f32 queries enter as q = 2^e (hi + lo) with hi, lo fp16 and e the
// row's own (22 bits, any range), their weights as hi + lo too.  FP32 cache:
// m16n8k8 tf32 products of both operands split in two (hi hi + hi lo + lo hi,
// 22 bits, the full exponent range).  Weights are held times 2^14 in fp16, so
// that one of 2^-28 of the largest still has 11 bits.
#include "hc_paged.h"

namespace hc {

namespace {

constexpr int SP_ROWS = 16, SP_TK = 16, SP_WARPS = 4, SP_THREADS = 128;
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
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
__device__ __forceinline__ float lds_f32(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ __half lds_f16(uint32_t a) {
    unsigned short v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
    return __ushort_as_half(v);
}
__device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// x = hi + lo with both in fp16 (two values)
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = pack(a - f.x, b - f.y);
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
constexpr int SP_CTAS = 148 * 2;  // two CTAs per SM
constexpr int MIN_UNITS = 4;      // of a run: a CTA's start costs about as much as the stream of 256 keys

struct SplitArgs {
    PagedAttnArgs a;
    int whole;
    float* po;    // [slot][16][hd] partial outputs, slot = 2 CTA + (0: its first pair, 1: its last)
    float2* pml;  // [slot][16] (maximum in log2 units, sum)
};

// Visible positions of packed rows [m0, m0 + n) of a sequence: [begin, end).
__device__ __forceinline__ void visible(const PagedAttnArgs& A, int first, int m0, int n, int& begin, int& end) {
    end = max(0, first + (m0 + n - 1) / A.G + 1);
    begin = A.window > 0 ? max(0, first + m0 / A.G - A.window + 1) : 0;
    begin = min(begin, end);
}

struct SeqWork {
    int r0, r1, first;  // rows, position of the first row
    int units, pairs;   // units of a pair, pairs
};
__device__ __forceinline__ SeqWork seq_work(const PagedAttnArgs& A, int b) {
    SeqWork w;
    seq_rows(A.p, b, w.r0, w.r1);
    const int T = w.r1 - w.r0;
    w.first = __ldg(A.p.kv_len + b) - T;
    const int64_t tiles = ((int64_t)T * A.G + SP_ROWS - 1) / SP_ROWS;
    // positions seen by any tile, at most: the last tile's end from the first tile's begin, per tile no
    // more than its window and its own tokens
    int len = max(0, w.first + T);
    if (A.window > 0) len = (int)min((int64_t)len, (int64_t)A.window + SP_ROWS);
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
__device__ __forceinline__ bool advance(const PagedAttnArgs& A, int64_t u, bool whole, Line& at) {
    const int lane = threadIdx.x & 31;
    while (at.b < A.p.n_seqs) {
        SeqWork w = {0, 0, 0, 1, 0};
        if (at.b + lane < A.p.n_seqs) w = seq_work(A, at.b + lane);
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
__device__ __forceinline__ int64_t all_units(const PagedAttnArgs& A) {
    int64_t n = 0;
    for (int b = threadIdx.x & 31; b < A.p.n_seqs; b += 32) {
        const SeqWork w = seq_work(A, b);
        n += (int64_t)w.pairs * w.units;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
}
__device__ __forceinline__ int64_t run_of(int64_t units) {
    return max((units + SP_CTAS - 1) / SP_CTAS, (int64_t)MIN_UNITS);
}

template <typename QT, typename CT, int HD>
struct SplitShape {
    static constexpr bool C16 = sizeof(CT) == 2;
    static constexpr int ROWB = HD * (int)sizeof(CT);           // bytes of a key in shared memory
    static constexpr int STAGE = 2 * SP_TK * ROWB;              // K tile, V tile
    static constexpr int STAGES = STAGE > 8192 ? 3 : (STAGE > 4096 ? 3 : 5);
    static constexpr int WARPB = STAGES * STAGE;
    static constexpr int SMEM = SP_WARPS * WARPB;
    static_assert(WARPB >= SP_ROWS * HD * 4, "a warp's outputs fit its ring");
};

template <typename QT, typename CT, int HD>
__global__ void __launch_bounds__(SP_THREADS) k_paged_split(const __grid_constant__ SplitArgs X) {
    using Sh = SplitShape<QT, CT, HD>;
    constexpr bool C16 = Sh::C16;
    constexpr bool HILO = C16 && sizeof(QT) == 4;
    // Operands in two parts: the tensor core cuts (does not round) the low
    // bits of a running sum, so the small products get a sum of their own (or
    // a short one) and the running outputs are added to by f32 adds.
    constexpr int S = Sh::STAGES, ROWB = Sh::ROWB;
    constexpr int EPC = 16 / (int)sizeof(CT);    // elements of a 16-byte chunk
    constexpr int CPR = HD / EPC;                // chunks of a row
    constexpr int NT = HD / 8;                   // output column tiles
    const PagedAttnArgs& A = X.a;
    const PagedArgs& P = A.p;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_m[SP_WARPS][SP_ROWS], s_l[SP_WARPS][SP_ROWS];
    __shared__ uint32_t s_in[SP_WARPS][S];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_trigger();  // the join may become resident; it waits for this grid's end

    int64_t u, u_end;
    if (X.whole) {
        u = blockIdx.x;
        u_end = u + 1;
    } else {
        const int64_t run = run_of(all_units(A));
        u = blockIdx.x * run;
        u_end = u + run;
    }
    const int64_t u_begin = u;
    Line at = {0, 0, {}};
    while (u < u_end && advance(A, u, X.whole != 0, at)) {
        const int seq = at.b, r0 = at.w.r0, first = at.w.first;
        const int64_t rem = u - at.base;
        const int pair = (int)(X.whole ? rem : rem / at.w.units);
        const int unit = X.whole ? 0 : (int)(rem - (int64_t)pair * at.w.units);
        const int nunits = X.whole ? at.w.units : (int)min((int64_t)(at.w.units - unit), u_end - u);
        const bool cut = nunits < at.w.units;
        const int64_t slot = 2 * (int64_t)blockIdx.x + (u == u_begin ? 0 : 1);
        u += X.whole ? 1 : nunits;
        {
            const int kvh = pair % P.nkv, m0 = pair / P.nkv * SP_ROWS;
            const int mrows = (int)min((int64_t)SP_ROWS, (int64_t)(at.w.r1 - r0) * A.G - m0);
            int begin, end;
            visible(A, first, m0, mrows, begin, end);
            const int c0 = (int)min((int64_t)end, begin + (int64_t)unit * UNIT);
            const int c1 = (int)min((int64_t)end, c0 + (int64_t)nunits * UNIT);

            // this thread's two rows
            const int ra = lane >> 2, rb = ra + 8, col = 2 * (lane & 3);
            const int ta = (m0 + ra) / A.G, tb = (m0 + rb) / A.G;
            const bool ina = ra < mrows, inb = rb < mrows;
            const int pa = ina ? first + ta : -1, pb = inb ? first + tb : -1;
            const int la = A.window > 0 ? pa - A.window + 1 : 0, lb = A.window > 0 ? pb - A.window + 1 : 0;
            const int p_min = first + m0 / A.G, l_max = A.window > 0 ? first + (m0 + mrows - 1) / A.G - A.window + 1 : 0;

            // ---- the keys' ring
            const uint32_t ring = smem_u32(smem) + warp * Sh::WARPB;
            const int ntiles = (c1 - c0 + SP_TK - 1) / SP_TK;
            const int mine = ntiles > warp ? (ntiles - warp + SP_WARPS - 1) / SP_WARPS : 0;
            auto page_at = [&](int i, int& slot) -> int {  // page of this lane's row of the warp's i-th tile
                const int j = c0 + (warp + i * SP_WARPS) * SP_TK + (lane & 15);
                slot = 0;
                return i < mine && j < c1 ? lookup(P, seq, j, slot) : -1;
            };
            int nslot, npage = page_at(0, nslot);
            auto issue = [&](int i) {
                if (i < mine) {
                    const uint32_t in = __ballot_sync(0xffffffffu, npage >= 0) & 0xffffu;
                    const CT* kp = (const CT*)P.k + (npage >= 0 ? npage * P.kps + kvh * P.khs + nslot * P.kss : 0);
                    const CT* vp = (const CT*)P.v + (npage >= 0 ? npage * P.vps + kvh * P.vhs + nslot * P.vss : 0);
                    const uint32_t dst = ring + (i % S) * Sh::STAGE;
                    if (lane == 0) s_in[warp][i % S] = in;
                    constexpr int RPI = 32 / CPR > 0 ? 32 / CPR : 1;   // rows of one warp-wide copy
                    constexpr int CPI = CPR > 32 ? CPR / 32 : 1;
#pragma unroll
                    for (int it = 0; it < SP_TK / RPI; it++) {
                        const int r = it * RPI + (CPR >= 32 ? 0 : lane / CPR);
                        const CT* k = (const CT*)__shfl_sync(0xffffffffu, (unsigned long long)kp, r);
                        const CT* v = (const CT*)__shfl_sync(0xffffffffu, (unsigned long long)vp, r);
                        const bool row_in = (in >> r) & 1u;
#pragma unroll
                        for (int x = 0; x < CPI; x++) {
                            const int c = (CPR >= 32 ? lane + 32 * x : lane % CPR);
                            const bool ok = row_in && c * EPC < P.hd;
                            const uint32_t o = (uint32_t)(r * ROWB + ((c ^ (r & 7)) << 4));
                            cp16(dst + o, ok ? k + c * EPC : (const CT*)P.k, ok);
                            cp16(dst + SP_TK * ROWB + o, ok ? v + c * EPC : (const CT*)P.v, ok);
                        }
                    }
                    npage = page_at(i + 1, nslot);
                }
                cp_commit();
            };
#pragma unroll
            for (int i = 0; i < S - 1; i++) issue(i);

            // ---- queries as A fragments
            constexpr int KS = C16 ? HD / 16 : HD / 8;
            uint32_t qh[KS][4];
            uint32_t ql[HILO ? KS : 1][4];
            float ca = A.scale * LOG2E, cb = ca;
            {
                const QT* q = (const QT*)A.q;
                const QT* qa = q + (int64_t)(r0 + ta) * A.q_rs + (kvh * A.G + (m0 + ra) - ta * A.G) * A.q_hs;
                const QT* qb = q + (int64_t)(r0 + tb) * A.q_rs + (kvh * A.G + (m0 + rb) - tb * A.G) * A.q_hs;
                auto at = [&](const QT* p, bool in, int d) -> float { return in && d < P.hd ? to_f32(p[d]) : 0.0f; };
                auto at2 = [&](const QT* p, bool in, int d) -> float2 {
                    if (!in || d >= P.hd) return make_float2(0.0f, 0.0f);
                    if (A.qvec) {
                        if constexpr (sizeof(QT) == 4) return *reinterpret_cast<const float2*>(p + d);
                        else return __half22float2(*reinterpret_cast<const __half2*>(p + d));
                    }
                    return make_float2(to_f32(p[d]), at(p, true, d + 1));
                };
                if constexpr (C16) {
                    float2 f[KS][4];
#pragma unroll
                    for (int k = 0; k < KS; k++) {
                        f[k][0] = at2(qa, ina, k * 16 + col);
                        f[k][1] = at2(qb, inb, k * 16 + col);
                        f[k][2] = at2(qa, ina, k * 16 + col + 8);
                        f[k][3] = at2(qb, inb, k * 16 + col + 8);
                    }
                    if constexpr (HILO) {
                        float xa = 0.0f, xb = 0.0f;
#pragma unroll
                        for (int k = 0; k < KS; k++) {
                            xa = fmaxf(xa, fmaxf(fmaxf(fabsf(f[k][0].x), fabsf(f[k][0].y)), fmaxf(fabsf(f[k][2].x), fabsf(f[k][2].y))));
                            xb = fmaxf(xb, fmaxf(fmaxf(fabsf(f[k][1].x), fabsf(f[k][1].y)), fmaxf(fabsf(f[k][3].x), fabsf(f[k][3].y))));
                        }
#pragma unroll
                        for (int o = 1; o < 4; o <<= 1) {
                            xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, o));
                            xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, o));
                        }
                        // 2^e <= max |q| < 2^(e + 1), e within what 2^e and 2^-e can be
                        const int ea = min(max((int)(__float_as_uint(xa) >> 23), 2), 252);
                        const int eb = min(max((int)(__float_as_uint(xb) >> 23), 2), 252);
                        const float ia = __uint_as_float((uint32_t)(254 - ea) << 23), ib = __uint_as_float((uint32_t)(254 - eb) << 23);
                        ca *= __uint_as_float((uint32_t)ea << 23);
                        cb *= __uint_as_float((uint32_t)eb << 23);
#pragma unroll
                        for (int k = 0; k < KS; k++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const float s = (i & 1) ? ib : ia;
                                split2(f[k][i].x * s, f[k][i].y * s, qh[k][i], ql[k][i]);
                            }
                    } else {
#pragma unroll
                        for (int k = 0; k < KS; k++)
#pragma unroll
                            for (int i = 0; i < 4; i++) qh[k][i] = pack(f[k][i].x, f[k][i].y);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < KS; k++) {
                        qh[k][0] = __float_as_uint(at(qa, ina, k * 8 + (lane & 3)));
                        qh[k][1] = __float_as_uint(at(qb, inb, k * 8 + (lane & 3)));
                        qh[k][2] = __float_as_uint(at(qa, ina, k * 8 + (lane & 3) + 4));
                        qh[k][3] = __float_as_uint(at(qb, inb, k * 8 + (lane & 3) + 4));
                    }
                }
            }

            float o[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[n][i] = 0.0f;
            float ma = -INFINITY, mb = -INFINITY, sa = 0.0f, sb = 0.0f;  // sums: this thread's columns only
            constexpr float BIAS = C16 ? 14.0f : 0.0f;

            for (int i = 0; i < mine; i++) {
                cp_wait<S - 2>();
                __syncwarp();
                issue(i + S - 1);
                const uint32_t kt = ring + (i % S) * Sh::STAGE, vt = kt + SP_TK * ROWB;
                const uint32_t in = s_in[warp][i % S];
                const int j0 = c0 + (warp + i * SP_WARPS) * SP_TK;
                float s[2][4], sl[HILO ? 2 : 1][4];  // sl: the low parts' products
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int x = 0; x < 4; x++) s[n][x] = 0.0f;
#pragma unroll
                for (int n = 0; n < (HILO ? 2 : 1); n++)
#pragma unroll
                    for (int x = 0; x < 4; x++) sl[n][x] = 0.0f;
                if constexpr (C16) {
#pragma unroll
                    for (int k = 0; k < KS; k++) {
                        // matrices: keys 0-7 / 8-15 x the two 8-element halves of the K step
                        uint32_t b[4];
                        const int r = (lane & 7) + ((lane >> 4) << 3), c = 2 * k + ((lane >> 3) & 1);
                        ldsm4(b, kt + r * ROWB + ((c ^ (r & 7)) << 4));
                        mma16(s[0], qh[k], b[0], b[1]);
                        mma16(s[1], qh[k], b[2], b[3]);
                        if constexpr (HILO) {
                            mma16(sl[0], ql[k], b[0], b[1]);
                            mma16(sl[1], ql[k], b[2], b[3]);
                        }
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < KS; k++) {
                        uint32_t ah[4], al[4];
#pragma unroll
                        for (int x = 0; x < 4; x++) split_tf32(__uint_as_float(qh[k][x]), ah[x], al[x]);
#pragma unroll
                        for (int n = 0; n < 2; n++) {
                            const int r = n * 8 + (lane >> 2);
                            const uint32_t base = kt + r * ROWB + 4 * (lane & 3);
                            uint32_t h0, l0, h1, l1;
                            split_tf32(lds_f32(base + (((2 * k) ^ (r & 7)) << 4)), h0, l0);
                            split_tf32(lds_f32(base + (((2 * k + 1) ^ (r & 7)) << 4)), h1, l1);
                            float d0[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma8(d0, al, h0, h1);
                            mma8(d0, ah, l0, l1);
                            mma8(d0, ah, h0, h1);
#pragma unroll
                            for (int x = 0; x < 4; x++) s[n][x] += d0[x];
                        }
                    }
                }
                if constexpr (HILO)
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int x = 0; x < 4; x++) s[n][x] += sl[n][x];
                // scores in log2 units; masked ones -inf
                const bool whole = in == 0xffffu && j0 + SP_TK - 1 <= p_min && j0 >= l_max;
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        s[n][x] *= ca;
                        s[n][2 + x] *= cb;
                        if (!whole) {
                            const int jj = n * 8 + col + x, j = j0 + jj;
                            const bool ok = (in >> jj) & 1u;
                            if (!ok || j > pa || j < la) s[n][x] = -INFINITY;
                            if (!ok || j > pb || j < lb) s[n][2 + x] = -INFINITY;
                        }
                    }
                float na = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
                float nb = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
#pragma unroll
                for (int d = 1; d < 4; d <<= 1) {
                    na = fmaxf(na, __shfl_xor_sync(0xffffffffu, na, d));
                    nb = fmaxf(nb, __shfl_xor_sync(0xffffffffu, nb, d));
                }
                na = fmaxf(na, ma);
                nb = fmaxf(nb, mb);
                if (__any_sync(0xffffffffu, na > ma || nb > mb)) {
                    const float fa = na == ma ? 1.0f : exp2f(ma - na), fb = nb == mb ? 1.0f : exp2f(mb - nb);
                    sa *= fa;
                    sb *= fb;
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        o[n][0] *= fa;
                        o[n][1] *= fa;
                        o[n][2] *= fb;
                        o[n][3] *= fb;
                    }
                    ma = na;
                    mb = nb;
                }
                const float ba = ma == -INFINITY ? 0.0f : ma - BIAS, bb = mb == -INFINITY ? 0.0f : mb - BIAS;
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        s[n][x] = exp2f(s[n][x] - ba);
                        s[n][2 + x] = exp2f(s[n][2 + x] - bb);
                        sa += s[n][x];
                        sb += s[n][2 + x];
                    }
                // A key that some rows of the tile see and others do not must not
                // reach the latter through 0 * v where v is not finite: such a
                // tile adds its products one by one, masked keys left out.
                bool careful = false;
                if (!whole && m0 / A.G != (m0 + mrows - 1) / A.G) {
                    uint32_t bad = 0;
                    if constexpr (C16) {
                        for (int x = lane; x < SP_TK * HD / 2; x += 32) {
                            uint32_t w;
                            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(vt + 4 * x));
                            bad |= (w & 0x7C007C00u) + 0x04000400u;
                        }
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
                        const int src = (lane & ~3) | ((jj & 7) >> 1), n = jj >> 3, odd = jj & 1;
                        const float xa = __shfl_sync(0xffffffffu, odd ? (n ? s[1][1] : s[0][1]) : (n ? s[1][0] : s[0][0]), src);
                        const float xb = __shfl_sync(0xffffffffu, odd ? (n ? s[1][3] : s[0][3]) : (n ? s[1][2] : s[0][2]), src);
                        const int j = j0 + jj;
                        const bool ok = (in >> jj) & 1u, oka = ok && j <= pa && j >= la, okb = ok && j <= pb && j >= lb;
#pragma unroll
                        for (int t = 0; t < NT; t++)
#pragma unroll
                            for (int x = 0; x < 2; x++) {
                                const int d = t * 8 + col + x;
                                const uint32_t ad = vt + jj * ROWB + (((d / EPC) ^ (jj & 7)) << 4) + (d % EPC) * (int)sizeof(CT);
                                float v;
                                if constexpr (C16) v = __half2float(lds_f16(ad));
                                else v = lds_f32(ad);
                                if (oka) o[t][x] = fmaf(xa, v, o[t][x]);
                                if (okb) o[t][2 + x] = fmaf(xb, v, o[t][2 + x]);
                            }
                    }
                } else if constexpr (C16) {
                    uint32_t ph[4], pl[4];
                    if constexpr (HILO) {
                        split2(s[0][0], s[0][1], ph[0], pl[0]);
                        split2(s[0][2], s[0][3], ph[1], pl[1]);
                        split2(s[1][0], s[1][1], ph[2], pl[2]);
                        split2(s[1][2], s[1][3], ph[3], pl[3]);
                    } else {
                        ph[0] = pack(s[0][0], s[0][1]);
                        ph[1] = pack(s[0][2], s[0][3]);
                        ph[2] = pack(s[1][0], s[1][1]);
                        ph[3] = pack(s[1][2], s[1][3]);
                    }
#pragma unroll
                    for (int t = 0; t < NT; t += 2) {
                        uint32_t b[4];
                        const int r = (lane & 7) + (((lane >> 3) & 1) << 3), c = t + (lane >> 4);
                        ldsm4t(b, vt + r * ROWB + ((c ^ (r & 7)) << 4));
                        if constexpr (HILO) {
                            float d0[4] = {0.0f, 0.0f, 0.0f, 0.0f}, d1[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma16(d0, pl, b[0], b[1]);
                            mma16(d1, pl, b[2], b[3]);
                            mma16(d0, ph, b[0], b[1]);
                            mma16(d1, ph, b[2], b[3]);
#pragma unroll
                            for (int x = 0; x < 4; x++) {
                                o[t][x] += d0[x];
                                o[t + 1][x] += d1[x];
                            }
                        } else {
                            mma16(o[t], ph, b[0], b[1]);
                            mma16(o[t + 1], ph, b[2], b[3]);
                        }
                    }
                } else {
                    // the products' K index: k -> key 2k, k + 4 -> key 2k + 1 of each
                    // eight, so that the scores' accumulators are the A fragment
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        uint32_t ah[4], al[4];
                        split_tf32(s[n][0], ah[0], al[0]);
                        split_tf32(s[n][2], ah[1], al[1]);
                        split_tf32(s[n][1], ah[2], al[2]);
                        split_tf32(s[n][3], ah[3], al[3]);
                        const int ka = n * 8 + 2 * (lane & 3), kb = ka + 1;
#pragma unroll
                        for (int t = 0; t < NT; t++) {
                            const int d = t * 8 + (lane >> 2);
                            uint32_t h0, l0, h1, l1;
                            split_tf32(lds_f32(vt + ka * ROWB + (((d >> 2) ^ (ka & 7)) << 4) + 4 * (d & 3)), h0, l0);
                            split_tf32(lds_f32(vt + kb * ROWB + (((d >> 2) ^ (kb & 7)) << 4) + 4 * (d & 3)), h1, l1);
                            float d0[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma8(d0, al, h0, h1);
                            mma8(d0, ah, l0, l1);
                            mma8(d0, ah, h0, h1);
#pragma unroll
                            for (int x = 0; x < 4; x++) o[t][x] += d0[x];
                        }
                    }
                }
                __syncwarp();
            }
            cp_wait<0>();
            __syncwarp();

            // ---- this warp's (m, l, o) to shared memory (over its ring)
#pragma unroll
            for (int d = 1; d < 4; d <<= 1) {
                sa += __shfl_xor_sync(0xffffffffu, sa, d);
                sb += __shfl_xor_sync(0xffffffffu, sb, d);
            }
            float* so = reinterpret_cast<float*>(smem + warp * Sh::WARPB);
#pragma unroll
            for (int t = 0; t < NT; t++) {
                *reinterpret_cast<float2*>(so + ra * HD + t * 8 + col) = make_float2(o[t][0], o[t][1]);
                *reinterpret_cast<float2*>(so + rb * HD + t * 8 + col) = make_float2(o[t][2], o[t][3]);
            }
            if ((lane & 3) == 0) {
                s_m[warp][ra] = ma;
                s_m[warp][rb] = mb;
                s_l[warp][ra] = sa;
                s_l[warp][rb] = sb;
            }
            __syncthreads();
            const int hq = P.hd >> 2;  // float4 columns (head_dim is a multiple of 4 here)
            for (int x = threadIdx.x; x < mrows * hq; x += SP_THREADS) {
                const int m = x / hq, d = (x - m * hq) * 4;
                float mx = -INFINITY;
#pragma unroll
                for (int w = 0; w < SP_WARPS; w++) mx = fmaxf(mx, s_m[w][m]);
                float l = 0.0f;
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < SP_WARPS; w++) {
                    if (s_l[w][m] == 0.0f) continue;  // saw nothing
                    const float f = exp2f(s_m[w][m] - mx);
                    const float4 y = *reinterpret_cast<const float4*>(smem + w * Sh::WARPB + (m * HD + d) * 4);
                    l = fmaf(f, s_l[w][m], l);
                    v.x = fmaf(f, y.x, v.x);
                    v.y = fmaf(f, y.y, v.y);
                    v.z = fmaf(f, y.z, v.z);
                    v.w = fmaf(f, y.w, v.w);
                }
                if (!cut) {
                    const int t = (m0 + m) / A.G, row = r0 + t, head = kvh * A.G + (m0 + m) - t * A.G;
                    store_row4<QT>(A, row, head, d, l, v);
                    if (A.lse && d == 0)
                        A.lse[(int64_t)row * A.nh + head] = l == 0.0f ? -INFINITY : (mx - BIAS + log2f(l)) / LOG2E;
                } else {
                    *reinterpret_cast<float4*>(X.po + (slot * SP_ROWS + m) * P.hd + d) = v;
                    if (d == 0) X.pml[slot * SP_ROWS + m] = make_float2(mx == -INFINITY ? mx : mx - BIAS, l);
                }
            }
            __syncthreads();
        }
    }
}

// Joins the partial results of a pair that was cut: with M = max m_s, o = sum
// 2^(m_s - M) o_s / sum 2^(m_s - M) l_s, in the order of the CTAs.
template <typename QT>
__global__ void __launch_bounds__(SP_THREADS) k_paged_join(const __grid_constant__ SplitArgs X) {
    const PagedAttnArgs& A = X.a;
    const PagedArgs& P = A.p;
    const int64_t run = run_of(all_units(A));
    Line at = {0, 0, {}};
    const bool any = advance(A, blockIdx.x, true, at);  // pair blockIdx.x, counted in pairs
    pdl_wait();
    if (!any) return;
    const int seq = at.b, pair = (int)(blockIdx.x - at.base);
    // units before this sequence
    int64_t before = 0;
    for (int b = threadIdx.x & 31; b < seq; b += 32) {
        const SeqWork w = seq_work(A, b);
        before += (int64_t)w.pairs * w.units;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    const int64_t p0 = before + (int64_t)pair * at.w.units, p1 = p0 + at.w.units;
    const int c0 = (int)(p0 / run), c1 = (int)((p1 - 1) / run);
    if (c0 == c1) return;  // one CTA took it whole
    const int kvh = pair % P.nkv, m0 = pair / P.nkv * SP_ROWS, r0 = at.w.r0;
    const int mrows = (int)min((int64_t)SP_ROWS, (int64_t)(at.w.r1 - r0) * A.G - m0);
    const int hq = P.hd >> 2;
    // the first CTA has it as its last pair, unless its run begins with the pair
    const int s0 = 2 * c0 + (c0 * run < p0 ? 1 : 0);
    auto slot = [&](int c) -> int64_t { return c == c0 ? s0 : 2 * (int64_t)c; };
    for (int x = blockIdx.y * SP_THREADS + threadIdx.x; x < mrows * hq; x += SP_THREADS * gridDim.y) {
        const int m = x / hq, d = (x - m * hq) * 4;
        float mx = -INFINITY;
        for (int c = c0; c <= c1; c++) mx = fmaxf(mx, X.pml[slot(c) * SP_ROWS + m].x);
        float l = 0.0f;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int c = c0; c <= c1; c++) {
            const float2 ml = X.pml[slot(c) * SP_ROWS + m];
            const float4 y = *reinterpret_cast<const float4*>(X.po + (slot(c) * SP_ROWS + m) * P.hd + d);
            if (ml.y == 0.0f) continue;  // saw nothing
            const float f = exp2f(ml.x - mx);
            l = fmaf(f, ml.y, l);
            v.x = fmaf(f, y.x, v.x);
            v.y = fmaf(f, y.y, v.y);
            v.z = fmaf(f, y.z, v.z);
            v.w = fmaf(f, y.w, v.w);
        }
        const int t = (m0 + m) / A.G, row = r0 + t, head = kvh * A.G + (m0 + m) - t * A.G;
        store_row4<QT>(A, row, head, d, l, v);
        if (A.lse && d == 0)
            A.lse[(int64_t)row * A.nh + head] = l == 0.0f ? -INFINITY : (mx + log2f(l)) / LOG2E;
    }
}

// Pairs of all sequences, at most.
int64_t pairs_bound(const PagedAttnArgs& A) {
    return ((int64_t)A.p.n_rows * A.G / SP_ROWS + A.p.n_seqs) * A.p.nkv;
}

template <typename QT, typename CT, int HD>
int launch_split_t(const SplitArgs& X, cudaStream_t s) {
    using Sh = SplitShape<QT, CT, HD>;
    HC_CUDA(cudaFuncSetAttribute(k_paged_split<QT, CT, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM));
    const PagedArgs& P = X.a.p;
    const int64_t pairs = pairs_bound(X.a);
    HC_CHECK(pairs <= 0x7fffffff, HC_ERR_INVALID, "paged attention: %d rows of %d heads", P.n_rows, X.a.nh);
    k_paged_split<QT, CT, HD><<<X.whole ? (unsigned)pairs : SP_CTAS, SP_THREADS, Sh::SMEM, s>>>(X);
    HC_LAUNCH_CHECK();
    if (!X.whole) {
        const int rows = std::min(SP_ROWS, X.a.G);
        const int y = (rows * P.hd / 4 + SP_THREADS - 1) / SP_THREADS;
        HC_TRY(launch_pdl(k_paged_join<QT>, dim3((unsigned)pairs, y), dim3(SP_THREADS), 0, s, X));
        HC_LAUNCH_CHECK();
    }
    return HC_OK;
}

template <typename QT, typename CT>
int launch_split_hd(const SplitArgs& X, cudaStream_t s) {
    return X.a.p.hd <= 64 ? launch_split_t<QT, CT, 64>(X, s) : launch_split_t<QT, CT, 128>(X, s);
}

}  // namespace

bool paged_split_ok(const PagedArgs& P, int c16) {
    const int64_t e = c16 ? 8 : 4;
    return P.hd <= 128 && P.hd % e == 0 && ((uintptr_t)P.k | (uintptr_t)P.v) % 16 == 0 &&
           (P.kps | P.khs | P.kss | P.vps | P.vhs | P.vss) % e == 0;
}

size_t paged_split_bytes(const PagedAttnArgs& A, int max_kv_len) {
    return paged_split_whole(A, max_kv_len) ? 0 : (size_t)2 * SP_CTAS * SP_ROWS * ((size_t)A.p.hd * 4 + 8);
}

// One CTA per pair where no pair is long enough to be worth cutting.
bool paged_split_whole(const PagedAttnArgs& A, int max_kv_len) {
    const int64_t len = A.window > 0 ? std::min<int64_t>(max_kv_len, (int64_t)A.window + SP_ROWS) : max_kv_len;
    return len <= MIN_UNITS * UNIT;
}

int launch_paged_split(const PagedAttnArgs& A, int q16, int c16, int max_kv_len, void* ws, cudaStream_t s) {
    SplitArgs X;
    X.a = A;
    X.whole = paged_split_whole(A, max_kv_len);
    X.po = (float*)ws;
    X.pml = (float2*)((float*)ws + (size_t)2 * SP_CTAS * SP_ROWS * A.p.hd);
    if (q16) return c16 ? launch_split_hd<__half, __half>(X, s) : launch_split_hd<__half, float>(X, s);
    return c16 ? launch_split_hd<float, __half>(X, s) : launch_split_hd<float, float>(X, s);
}

}  // namespace hc
