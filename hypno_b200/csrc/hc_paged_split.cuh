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
//
// A pool in 4 bits (CT = q4x): the codes stream as they are, and each lane makes
// of them the float16 operands that ldmatrix would have given it, in registers
// (q4_pairs; exact, so the rest is as over an FP16 cache).  The order of the
// elements in a product's sum is free, so a lane's part of a key is a run of its
// bytes; V needs pairs of keys, which one byte permutation per eight elements
// makes of two keys' words, and its columns are a run of its bytes again.
//
// Lists of pages (LIST): a tile holds rows of one token, whose keys are the
// positions of its listed pages one after another; in pages of whole tiles a tile's
// place is worked out once, by a lane, 16 tiles ahead.  8 tokens over 64 FP16 pages of 64
// each, 64 heads over 8 of 128: 39 us with the join, 3.4 TB/s; bound by the latency of the start
// (the list, its pages, their keys, one after another) and of the copies, which the warps
// that compute issue themselves, two tiles ahead.  FP32 pages, the caches cold: 121 us where
// FP16 ones take 47, by the three products and the splitting of both operands.
#pragma once

#include "hc_paged.h"

#include <type_traits>

namespace hc {

// Work is counted in units of 64 positions (16 for each warp).  A sequence has
// tiles x nkv pairs of (row tile, KV head) and every pair of it the same
// number of units; the pairs of all sequences in order form one line of units.
// With `whole`, CTA i takes pair i.  Otherwise every CTA takes an equal run of
// the line, whatever the lengths of the sequences, and a pair that is cut
// leaves partial results to k_paged_join; a CTA cuts at most two (its first
// and its last), so it has two slots.
struct SplitArgs {
    PagedAttnArgs a;
    PagedScales c;  // 4 bits only
    PagedList l;    // LIST only
    int tg;         // LIST: tiles of a token
    int uni;        // 4 bits, LIST: a tile of 16 keys lies in one page
    int whole;
    int ctas;     // CTAs of the line (cut)
    int rows;     // R, rows of a tile
    float* po;    // [slot][R][hd] partial outputs, slot = 2 CTA + (0: its first pair, 1: its last)
    float2* pml;  // [slot][R] (maximum in log2 units, sum)
};

constexpr int SP_TK = 16, SP_WARPS = 4, SP_THREADS = 128;
constexpr int UNIT = SP_WARPS * SP_TK;
constexpr int SP_CTAS = 148 * 3;  // at most: CTAs of the cut line, as many as are resident at once
constexpr int MIN_UNITS = 4;      // of a run: a CTA's start costs about as much as the stream of 256 keys

namespace {

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

struct SeqWork {
    int r0, r1, first;  // rows, position of the first row
    int units, pairs;   // units of a pair, pairs
};
template <bool LIST>
__device__ __forceinline__ SeqWork seq_work(const SplitArgs& X, int b) {
    const PagedAttnArgs& A = X.a;
    const int R = X.rows;
    SeqWork w;
    seq_rows(A.p, b, w.r0, w.r1);
    const int T = w.r1 - w.r0;
    w.first = seq_len(A.p, b) - T;
    if constexpr (LIST) {
        // the last row's pages, or the lists' width: no list is longer
        const int64_t keys = (int64_t)min(X.l.width, pages_seen(A.p, w.first + T - 1)) * A.p.page_size;
        w.units = (int)max((keys + UNIT - 1) / UNIT, (int64_t)1);
        w.pairs = T * X.tg * A.p.nkv;
        return w;
    }
    const int64_t tiles = ((int64_t)T * A.G + R - 1) >> (R == 8 ? 3 : 4);
    // positions seen by any tile, at most: the last tile's end from the first tile's begin, per tile no
    // more than its window and its own tokens
    int len = min(max(0, w.first + T), A.p.reach);
    if (A.window > 0) len = (int)min((int64_t)len, (int64_t)A.window + R + (X.uni ? SP_TK - 1 : 0));  // (uni: from a tile's first key on)
    w.units = max(1, len / UNIT + (len % UNIT != 0));
    w.pairs = (int)(tiles * A.p.nkv);
    return w;
}

// a / b, neither negative: a 64-bit division takes some 500 cycles.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    return (uint64_t)(a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// A place on the line of units: sequence b, which begins at `base`.
struct Line {
    int b;
    int64_t base;
    SeqWork w;
};
// Moves on to the sequence that holds unit u (a whole warp; false past the end).
template <bool LIST>
__device__ __forceinline__ bool advance(const SplitArgs& X, int64_t u, bool whole, Line& at) {
    const PagedAttnArgs& A = X.a;
    const int lane = threadIdx.x & 31;
    while (at.b < A.p.n_seqs) {
        SeqWork w = {0, 0, 0, 1, 0};
        if (at.b + lane < A.p.n_seqs) w = seq_work<LIST>(X, at.b + lane);
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
template <bool LIST>
__device__ __forceinline__ int64_t all_units(const SplitArgs& X) {
    int64_t n = 0;
    for (int b = threadIdx.x & 31; b < X.a.p.n_seqs; b += 32) {
        const SeqWork w = seq_work<LIST>(X, b);
        n += (int64_t)w.pairs * w.units;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
}
__device__ __forceinline__ int64_t run_of(int64_t units, int ctas) {
    return max(quotient(units + ctas - 1, ctas), (int64_t)MIN_UNITS);
}

// The line of up to 32 sequences, worked out once a CTA (by its first warp).
struct LineTable {
    int64_t end[32];  // units (whole: pairs) up to each sequence's last
    SeqWork w[32];
    int64_t units;    // of all sequences
};
template <bool LIST>
__device__ __forceinline__ void fill_table(const SplitArgs& X, LineTable& t) {
    const int lane = threadIdx.x & 31;
    SeqWork w = {0, 0, 0, 1, 0};
    if (lane < X.a.p.n_seqs) w = seq_work<LIST>(X, lane);
    int64_t incl = (int64_t)w.pairs * (X.whole ? 1 : w.units);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    t.end[lane] = incl;
    t.w[lane] = w;
    if (lane == 31) t.units = incl;
}
// advance() by the table.
__device__ __forceinline__ bool advance_by(const LineTable& t, int64_t u, Line& at) {
    const int lane = threadIdx.x & 31;
    const unsigned hit = __ballot_sync(0xffffffffu, t.end[lane] > u);
    if (!hit) return false;
    at.b = __ffs(hit) - 1;
    at.base = at.b ? t.end[at.b - 1] : 0;
    at.w = t.w[at.b];
    return true;
}

// The packed rows of a tile: the first, and how many.
template <bool LIST>
__device__ __forceinline__ void tile_rows(const SplitArgs& X, int tile, int T, int& m0, int& mrows) {
    const int G = X.a.G, R = X.rows;
    if constexpr (LIST) {
        const int t = tile / X.tg, g0 = (tile - t * X.tg) * R;
        m0 = t * G + g0;
        mrows = min(R, G - g0);
    } else {
        m0 = tile * R;
        mrows = (int)min((int64_t)R, (int64_t)T * G - m0);
    }
}

template <typename CT, int HD>
struct SplitShape {
    static constexpr bool Q4 = std::is_same<CT, q4x>::value;
    static constexpr int ROWB = Q4 ? HD / 2 : HD * (int)sizeof(CT);  // bytes of a key in shared memory
    static constexpr int SCB = Q4 ? 2 * q4_slots(HD) : 0;            // and of its scales, behind the tiles
    static constexpr int STAGE = 2 * SP_TK * (ROWB + SCB);           // K tile, V tile
    static constexpr int STAGES = Q4 ? 4 : STAGE > 8192 ? 3 : (STAGE > 4096 ? 2 : 4);  // three CTAs an SM before a deeper ring
    static constexpr int WARPB = STAGES * STAGE;
    static constexpr int SMEM = SP_WARPS * WARPB + 512;         // 512: rows are aligned to their size
    static constexpr int LDO = HD + 4;                          // row of outputs: conflict-free column stores
    static_assert(WARPB >= 16 * LDO * 4, "a warp's outputs fit its ring");
};

// ---- 4 bits.  Tiles lie in shared memory as in a page: a key's bytes after one
// another, the scales of all keys behind the codes.  Lane c = lane % 4 of a key's
// four lanes has a quarter of its bytes (two groups of 32 elements, 128 elements apart,
// for heads above 128), eight elements a word.  Of the values, lanes r = lane / 4
// have an eighth of a key's bytes each, of the four keys that their operands take.
// Key m of the products is key q4_key(m) of the tile: the keys 0, 3, 4, 7 that the
// four lanes c read at once lie on different banks by pairs (0, 2, 4, 6 would not),
// and so do the two keys that eight lanes read at once.
__device__ __forceinline__ int q4_key(int m) { return m ^ (m >> 1 & 1); }  // its own inverse
// First element of word w of lane c's part of a key.
template <int HD>
__device__ __forceinline__ int q4_part(int c, int w) {
    return HD > 128 ? (w >> 2) * 128 + c * 32 + (w & 3) * 8 : c * (HD / 4) + w * 8;
}
__device__ __forceinline__ uint32_t lds_u32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
template <int N>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t* v) {
    if constexpr (N == 1) v[0] = lds_u32(a);
    else if constexpr (N == 2) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(a));
    else asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a));
}
template <int BYTES>
__device__ __forceinline__ void cp_small(uint32_t dst, const void* src, bool in) {
    if constexpr (BYTES == 16) cp16(dst, src, in);
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(in ? BYTES : 0) : "memory");
}
// Copies keys r = lane / 4 and r + 8 of a tile with their scales, zeros for a page of -1.
template <int HD>
__device__ __forceinline__ void copy_q4(const SplitArgs& X, int kvh, int page0, int slot0, int page1, int slot1, uint32_t stage) {
    using Sh = SplitShape<q4x, HD>;
    const PagedArgs& P = X.a.p;
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    constexpr int ROWB = Sh::ROWB, SCB = Sh::SCB, SC = 2 * SP_TK * ROWB;
    const uint8_t *kb = (const uint8_t*)P.k, *vb = (const uint8_t*)P.v;
    auto chunk = [&](int key, int page, int slot, int x) {
        const bool in = page >= 0 && x * 32 < P.hd;  // chunks past head_dim are zeros, not read
        const int64_t g = max(page, 0);
        const uint32_t to = stage + key * ROWB + (x << 4);
        cp16(to, in ? kb + g * P.kps + kvh * P.khs + slot * P.kss + x * 16 : kb, in);
        cp16(to + SP_TK * ROWB, in ? vb + g * P.vps + kvh * P.vhs + slot * P.vss + x * 16 : vb, in);
    };
    if constexpr (HD <= 64) {
        chunk(r + (c >> 1) * 8, c >> 1 ? page1 : page0, c >> 1 ? slot1 : slot0, c & 1);
    } else {
#pragma unroll
        for (int x = 0; x < HD / 128; x++) {
            chunk(r, page0, slot0, c + 4 * x);
            chunk(r + 8, page1, slot1, c + 4 * x);
        }
    }
    // one lane a scale row: keys r, r + 8 of K, of V
    const int key = r + (c & 1) * 8, page = c & 1 ? page1 : page0, slot = c & 1 ? slot1 : slot0;
    const bool in = page >= 0;
    const int64_t g = max(page, 0);
    const __half* src = c >> 1 ? X.c.v + g * X.c.vps + kvh * X.c.vhs + slot * X.c.vss : X.c.k + g * X.c.kps + kvh * X.c.khs + slot * X.c.kss;
    cp_small<SCB>(stage + SC + ((c >> 1) * SP_TK + key) * SCB, in ? src : X.c.k, in);
}
// Lane c's words of a key and their scales s, with z = -72 s.
template <int HD>
__device__ __forceinline__ void q4_key_words(uint32_t tile, uint32_t scales, int row, int hd, uint32_t* w, __half2* s, __half2* z) {
    constexpr int ROWB = HD / 2, SCB = 2 * q4_slots(HD);
    const int c = threadIdx.x & 3;
#pragma unroll
    for (int x = 0; x < (HD > 128 ? 2 : 1); x++) {
        if constexpr (HD <= 64) lds_words<2>(tile + row * ROWB + c * 8, w);
        else lds_words<4>(tile + row * ROWB + ((c + 4 * x) << 4), w + 4 * x);
        const int g = HD <= 64 ? c >> 1 : c + 4 * x;
        // (the slots past head_dim may hold anything)
        s[x] = g * 32 < hd ? __half2half2(lds_f16(scales + row * SCB + 2 * g)) : __half2half2(__ushort_as_half(0));
        z[x] = __hmul2(s[x], __half2half2(__float2half_rn(-72.0f)));
    }
}
// This lane's words of its four keys' values, the scales of each pair of keys: zero
// for the ones that are not in, whatever their slots hold.
template <int HD>
__device__ __forceinline__ void q4_value_words(uint32_t tile, uint32_t scales, uint32_t in, uint32_t (*w)[HD / 64], __half2* s, __half2* z) {
    constexpr int ROWB = HD / 2, SCB = 2 * q4_slots(HD);
    const int r = (threadIdx.x & 31) >> 2, c = threadIdx.x & 3;
    const int key = q4_key(2 * c);  // then key ^ 1, and both + 8
    __half h[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int row = (key ^ (i & 1)) + (i >> 1) * 8;
        lds_words<HD / 64>(tile + row * ROWB + r * (HD / 16), w[i]);
        h[i] = lds_f16(scales + row * SCB + 2 * (HD <= 64 ? r >> 2 : HD <= 128 ? r >> 1 : r));
    }
    if (in != 0xffffu) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (!(in >> ((key ^ (i & 1)) + (i >> 1) * 8) & 1u)) h[i] = __ushort_as_half(0);
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        s[i] = __halves2half2(h[2 * i], h[2 * i + 1]);
        z[i] = __hmul2(s[i], __half2half2(__float2half_rn(-72.0f)));
    }
}
// One value of a tile.
template <int HD>
__device__ __forceinline__ float q4_value(uint32_t tile, uint32_t scales, int key, int d) {
    constexpr int ROWB = HD / 2, SCB = 2 * q4_slots(HD);
    const uint32_t word = lds_u32(tile + key * ROWB + (d >> 3) * 4);
    return (float)((int)(word >> (4 * (d & 7)) & 15) - 8) * __half2float(lds_f16(scales + key * SCB + 2 * (d >> 5)));
}
// 2^x; results below 2^-126 are zeros.
template <bool FAST>
__device__ __forceinline__ float pow2(float x) {
    if constexpr (FAST) {
        float y;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
        return y;
    } else {
        return exp2f(x);
    }
}
// Eight elements of a query row.
template <typename QT>
__device__ __forceinline__ void load_q8(const QT* q, bool in, int vec, int d, float* x) {
    if (in && vec) {
        if constexpr (sizeof(QT) == 4) {
            const float4 a = *reinterpret_cast<const float4*>(q + d), b = *reinterpret_cast<const float4*>(q + d + 4);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
            const uint4 a = *reinterpret_cast<const uint4*>(q + d);
            const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
                x[2 * i] = f.x, x[2 * i + 1] = f.y;
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = in ? to_f32(q[d + i]) : 0.0f;
}

// CTAs an SM is to hold at least, for the forms whose copies are planned ahead (their
// state would take the registers of the third); 0: as the compiler likes it.
template <typename CT, int HD, int NQ, bool LIST>
constexpr int split_ctas() { return (LIST || std::is_same<CT, q4x>::value) && NQ == 1 && HD <= 128 ? 3 : 0; }

template <typename QT, typename CT, int HD, int NQ, bool LIST>
__global__ void __launch_bounds__(SP_THREADS, split_ctas<CT, HD, NQ, LIST>()) k_paged_split(const __grid_constant__ SplitArgs X) {
    using Sh = SplitShape<CT, HD>;
    constexpr bool Q4 = Sh::Q4;
    constexpr bool C16 = Q4 || sizeof(CT) == 2;  // products of float16
    constexpr bool HILO = C16 && sizeof(QT) == 4;
    // Operands in two parts: the tensor core cuts (does not round) the low
    // bits of a running sum, so the small products get a sum of their own (or
    // a short one) and the running outputs are added to by f32 adds.
    constexpr int R = 8 * NQ;
    constexpr int S = Sh::STAGES, ROWB = Sh::ROWB, LDO = Sh::LDO;
    constexpr int EPC = Q4 ? 32 : 16 / (int)sizeof(CT);  // elements of a 16-byte chunk
    constexpr int CPL = HD / EPC / 4;            // chunks of a row per lane (four lanes copy a row)
    constexpr int SCB = Sh::SCB, SC = 2 * SP_TK * ROWB;  // 4 bits: scales of a key, their place in a stage
    constexpr int LE = HD / 4;                   // 4 bits: elements of a key per lane
    constexpr int DT = HD / 16;                  // output row tiles
    const PagedAttnArgs& A = X.a;
    const PagedArgs& P = A.p;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 511u);
    __shared__ float s_m[SP_WARPS][R], s_l[SP_WARPS][R];
    __shared__ uint32_t s_in[SP_WARPS][S];
    constexpr bool PLAN = Q4 || LIST;  // forms with one page a tile
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_trigger();  // the join may become resident; it waits for this grid's end

    __shared__ LineTable s_line[1];
    const bool table = PLAN && A.p.n_seqs <= 32;
    if (table) {
        if (warp == 0) fill_table<LIST>(X, s_line[0]);
        __syncthreads();
    }
    int64_t u, u_end;
    if (X.whole) {
        u = blockIdx.x;
        u_end = u + 1;
    } else {
        const int64_t run = run_of(table ? s_line[0].units : all_units<LIST>(X), X.ctas);
        u = blockIdx.x * run;
        u_end = u + run;
    }
    const int64_t u_begin = u;
    Line at = {0, 0, {}};
    while (u < u_end && (table ? advance_by(s_line[0], u, at) : advance<LIST>(X, u, X.whole != 0, at))) {
        const int seq = at.b, r0 = at.w.r0, first = at.w.first;
        const int64_t rem = u - at.base;
        const int pair = (int)(X.whole ? rem : quotient(rem, at.w.units));
        const int unit = X.whole ? 0 : (int)(rem - (int64_t)pair * at.w.units);
        const int nunits = X.whole ? at.w.units : (int)min((int64_t)(at.w.units - unit), u_end - u);
        const bool cut = nunits < at.w.units;
        const int64_t slot = 2 * (int64_t)blockIdx.x + (u == u_begin ? 0 : 1);
        u += X.whole ? 1 : nunits;
        const int kvh = pair % P.nkv;
        int m0, mrows;
        tile_rows<LIST>(X, pair / P.nkv, at.w.r1 - r0, m0, mrows);
        int begin, end;
        const int p_own = first + token_of(A, m0);  // position of the tile's first token (LIST: its only one)
        const bool one_token = token_of(A, m0) == token_of(A, m0 + mrows - 1);
        const int32_t* list = nullptr;
        if constexpr (LIST) {
            const int row = r0 + token_of(A, m0);
            list = X.l.pages + row * X.l.row_stride + kvh * X.l.head_stride;
            begin = 0;
            end = (int)min((int64_t)min(list_count(X.l, row, kvh), pages_seen(P, p_own)) * P.page_size, (int64_t)0x7fffff00);
        } else {
            visible(A, first, m0, mrows, begin, end);
            if (Q4 && X.uni) begin &= ~(SP_TK - 1);
        }
        const int c0 = (int)min((int64_t)end, begin + (int64_t)unit * UNIT);
        const int c1 = (int)min((int64_t)end, c0 + (int64_t)nunits * UNIT);

        // ---- the keys' ring: this lane copies a quarter of rows kr and kr + 8
        const uint32_t ring = smem_u32(smem) + warp * Sh::WARPB;
        const int ntiles = (c1 - c0 + SP_TK - 1) / SP_TK;
        const int mine = ntiles > warp ? (ntiles - warp + SP_WARPS - 1) / SP_WARPS : 0;
        const int kr = lane >> 2;
        const uint32_t put = Q4 ? 0 : (uint32_t)(kr * ROWB + (((lane & 3) ^ kr) << 4));
        int slot0, slot1, page0, page1;
        auto look = [&](int i) {
            const int j = c0 + (warp + i * SP_WARPS) * SP_TK + kr;
            page0 = page1 = -1;
            slot0 = slot1 = 0;
            if (i < mine) {
                if constexpr (LIST) {
                    if (j < c1) page0 = lookup_listed(A, list, seq, j, p_own, slot0);
                    if (j + 8 < c1) page1 = lookup_listed(A, list, seq, j + 8, p_own, slot1);
                } else {
                    if (j < c1) page0 = lookup(P, seq, j, slot0);
                    if (j + 8 < c1) page1 = lookup(P, seq, j + 8, slot1);
                }
            }
        };
        // One page a tile: lane l works out the places of this warp's tiles 32 n + l
        // ahead of their copies, page, slot << 16 and the keys that are there.
        [[maybe_unused]] int now_page = -1, then_page = -1, then_entry = -1;
        [[maybe_unused]] uint32_t now_place = 0, then_place = 0;
        auto find_entry = [&](int i0) {  // LIST: the index that the list has there
            const int i = i0 + lane;
            then_entry = LIST && i < mine ? __ldg(list + page_of(P, c0 + (warp + i * SP_WARPS) * SP_TK)) : 0;
        };
        auto find_page = [&](int i0) {
            const int i = i0 + lane;
            then_page = -1;
            then_place = 0;
            if (i >= mine) return;
            const int v = c0 + (warp + i * SP_WARPS) * SP_TK;
            int x = page_of(P, v), n = min(SP_TK, c1 - v), low = 0;
            const int place = v - x * P.page_size;
            if constexpr (LIST) {
                x = then_entry;
                if (x >= P.max_pages) return;
                const int64_t pos = (int64_t)x * P.page_size + place;
                n = (int)min((int64_t)n, p_own - pos + 1);
                if (A.window > 0) low = (int)min(max(p_own - A.window + 1 - pos, (int64_t)0), (int64_t)SP_TK);
                if (n <= low) return;
            } else if (A.window > 0 && one_token) {  // (begins at a tile's first key: what lies in front of the window is not there)
                low = min(max(p_own - A.window + 1 - v, 0), SP_TK);
            }
            const int g = __ldg(P.table + (int64_t)seq * P.table_stride + x);
            if ((unsigned)g >= (unsigned)P.n_pages) return;
            then_page = g;
            then_place = (uint32_t)place << 16 | (((1u << n) - 1) & ~((1u << low) - 1));
        };
        const bool plan = PLAN && X.uni;
        if (plan) {
            find_entry(0);
            find_page(0);
        } else {
            look(0);
        }
        auto issue = [&](int i) {
            if (plan) {
                if (i < mine) {
                    if ((i & 31) == 0) {
                        now_page = then_page;
                        now_place = then_place;
                        find_entry(i + 32);
                    } else if ((i & 31) == 16) {
                        find_page(i + 16);
                    }
                    const int page = __shfl_sync(0xffffffffu, now_page, i & 31);
                    const uint32_t at = __shfl_sync(0xffffffffu, now_place, i & 31), in = at & 0xffffu;
                    page0 = in >> kr & 1u ? page : -1;  // (a key that no row sees is zeros)
                    page1 = in >> (kr + 8) & 1u ? page : -1;
                    slot0 = (int)(at >> 16) + kr;
                    slot1 = slot0 + 8;
                    if (lane == 0) s_in[warp][i % S] = in;
                }
            }
            if (i < mine && !plan) {
                const uint32_t b0 = __ballot_sync(0xffffffffu, page0 >= 0), b1 = __ballot_sync(0xffffffffu, page1 >= 0);
                if (lane == 0) {  // one bit per key: the lanes of a row agree
                    uint32_t in = 0;
#pragma unroll
                    for (int r = 0; r < 8; r++) in |= ((b0 >> (4 * r)) & 1u) << r | ((b1 >> (4 * r)) & 1u) << (8 + r);
                    s_in[warp][i % S] = in;
                }
            }
            if (i < mine) {
                if constexpr (Q4) {
                    copy_q4<HD>(X, kvh, page0, slot0, page1, slot1, ring + (i % S) * Sh::STAGE);
                } else {
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
                }
                if (!plan) look(i + 1);
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
                if constexpr (Q4) {
                    // the elements of this lane's part of a key, in the order that q4_pairs gives them
#pragma unroll
                    for (int w = 0; w < LE / 8; w++) {
                        const int d = q4_part<HD>(lane & 3, w);
                        float x[8];
                        load_q8(q, in && d < P.hd, A.qvec, d, x);
#pragma unroll
                        for (int j = 0; j < 4; j++) f[(4 * w + j) / 2][j & 1] = make_float2(x[j], x[4 + j]);
                    }
                }
#pragma unroll
                for (int k = 0; k < (Q4 ? 0 : KS); k++)
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
        // Planned forms (4 bits, and lists over every pool): the maximum stays until a score
        // passes it by 2^TAU, so that the outputs are rarely scaled (a tile in three raises
        // one of its rows' maxima by a little); a weight is at most 2^(BIAS + TAU), one of
        // 2^-25 of the largest still has 11 bits (2^-28 in the dense form over FP16), a smaller
        // one is off by 2^-36 of the largest at most.  Their exponential is the special
        // function alone (2^-22 of the weight at most, as much as the two-part products
        // leave; weights below 2^-126 are zeros), over FP32 pages too.
        constexpr float BIAS = PLAN && C16 ? 11.0f : C16 ? 14.0f : 0.0f, TAU = PLAN ? 4.0f : 0.0f;
        const int mi = lane >> 3;
        // ldmatrix rows: K as A (keys x d), V transposed as A (d x keys)
        const int krow = (lane & 7) + (mi & 1) * 8, vrow = (lane & 7) + (mi >> 1) * 8;
        const uint32_t kget = (uint32_t)(krow * ROWB + (((mi >> 1) ^ (krow & 7)) << 4));
        const uint32_t vget = (uint32_t)(vrow * ROWB + (((mi & 1) ^ (vrow & 7)) << 4));

        for (int i = 0; i < mine; i++) {
            const uint32_t st = i % S;
            cp_wait<S - 2>();
            __syncwarp();
            issue(i + S - 1);
            const uint32_t kt = ring + st * Sh::STAGE, vt = kt + SP_TK * ROWB;
            const uint32_t in = s_in[warp][st];
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
            if constexpr (Q4) {
                uint32_t w0[LE / 8], w1[LE / 8];  // this lane's part of keys lane / 4 and lane / 4 + 8
                __half2 s0[HD > 128 ? 2 : 1], s1[HD > 128 ? 2 : 1], z0[HD > 128 ? 2 : 1], z1[HD > 128 ? 2 : 1];
                q4_key_words<HD>(kt, kt + SC, q4_key(lane >> 2), P.hd, w0, s0, z0);
                q4_key_words<HD>(kt, kt + SC, q4_key(lane >> 2) + 8, P.hd, w1, s1, z1);
#pragma unroll
                for (int w = 0; w < LE / 8; w++) {
                    uint32_t e[4], f[4];
                    q4_pairs(w0[w], s0[w / 4], z0[w / 4], e);
                    q4_pairs(w1[w], s1[w / 4], z1[w / 4], f);
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const uint32_t a[4] = {e[2 * k], f[2 * k], e[2 * k + 1], f[2 * k + 1]};
#pragma unroll
                        for (int n = 0; n < NQ; n++) {
                            mma16(s[n], a, qh[n][2 * w + k][0], qh[n][2 * w + k][1]);
                            if constexpr (HILO) mma16(sl[n], a, ql[n][2 * w + k][0], ql[n][2 * w + k][1]);
                        }
                    }
                }
            } else if constexpr (C16) {
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
            const bool whole = in == 0xffffu && (LIST || (j0 + SP_TK - 1 <= p_min && j0 >= l_max));
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
                        const int jj = Q4 ? q4_key(lane >> 2) : lane >> 2, j = j0 + jj;
                        if (!((in >> jj) & 1u) || (!LIST && (j > ps[n][x] || j < lo[n][x]))) s[n][x] = -INFINITY;
                        if (!((in >> (jj + 8)) & 1u) || (!LIST && (j + 8 > ps[n][x] || j + 8 < lo[n][x]))) s[n][2 + x] = -INFINITY;
                    }
                    nm[x] = fmaxf(s[n][x], s[n][2 + x]);
                }
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    nm[0] = fmaxf(nm[0], __shfl_xor_sync(0xffffffffu, nm[0], d));
                    nm[1] = fmaxf(nm[1], __shfl_xor_sync(0xffffffffu, nm[1], d));
                }
                if (__any_sync(0xffffffffu, nm[0] > mx[n][0] + TAU || nm[1] > mx[n][1] + TAU)) {
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        const float m = PLAN && !(nm[x] > mx[n][x] + TAU) ? mx[n][x] : fmaxf(nm[x], mx[n][x]);
                        const float f = m == mx[n][x] ? 1.0f : pow2<PLAN>(mx[n][x] - m);
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
                    s[n][x] = pow2<PLAN>(s[n][x] - b);
                    s[n][2 + x] = pow2<PLAN>(s[n][2 + x] - b);
                    sum[n][x] += s[n][x] + s[n][2 + x];
                }
            }
            // A key that some rows of the tile see and others do not must not
            // reach the latter through 0 * v where v is not finite: such a
            // tile adds its products one by one, masked keys left out.
            bool careful = false;
            if (!LIST && !whole && !one_token) {
                uint32_t bad = 0;
                if constexpr (Q4) {
                    for (int x = lane; x < SP_TK * SCB / 4; x += 32)
                        bad |= (lds_u32(kt + SC + SP_TK * SCB + 4 * x) & 0x7C007C00u) + 0x04000400u;
                    bad &= 0x80008000u;
                } else if constexpr (C16) {
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
            if (!LIST && careful) {
                for (int jj = 0; jj < SP_TK; jj++) {
                    const int src = (Q4 ? q4_key(jj & 7) : jj & 7) * 4 + (lane & 3), j = j0 + jj;
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
                                    float v;
                                    if constexpr (Q4) {
                                        v = q4_value<HD>(vt, kt + SC + SP_TK * SCB, jj, (lane >> 2) * (HD / 8) + 2 * t + y);
                                    } else {
                                    const int d = t * 16 + y * 8 + (lane >> 2);
                                    const uint32_t ad = vt + jj * ROWB + (((d / EPC) ^ (jj & 7)) << 4) + (d % EPC) * (int)sizeof(CT);
                                    if constexpr (C16) v = __half2float(lds_f16(ad));
                                    else v = lds_f32(ad);
                                    }
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
                auto add = [&](int t, const uint32_t* a) {  // a: 16 columns of V of 16 keys
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
                };
                if constexpr (Q4) {
                    uint32_t w[4][LE / 16];  // this lane's run of columns, of keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9
                    __half2 sv[2], sz[2];
                    q4_value_words<HD>(vt, kt + SC + SP_TK * SCB, in, w, sv, sz);
#pragma unroll
                    for (int h = 0; h < HD / 32; h++) {  // four columns
                        uint32_t e[4], f[4];
                        q4_pairs(__byte_perm(w[0][h / 2], w[1][h / 2], h & 1 ? 0x7632 : 0x5410), sv[0], sz[0], e);
                        q4_pairs(__byte_perm(w[2][h / 2], w[3][h / 2], h & 1 ? 0x7632 : 0x5410), sv[1], sz[1], f);
#pragma unroll
                        for (int y = 0; y < 2; y++) {
                            const uint32_t a[4] = {e[2 * y], e[2 * y + 1], f[2 * y], f[2 * y + 1]};
                            add(2 * h + y, a);
                        }
                    }
                } else {
#pragma unroll
                for (int t = 0; t < DT; t++) {
                    uint32_t a[4];
                    ldsm4t(a, (vt + vget) ^ (uint32_t)(t << 5));
                    add(t, a);
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
                    for (int y = 0; y < 2; y++)
                        so[(n * 8 + col + x) * LDO + (Q4 ? (lane >> 2) * (HD / 8) + 2 * t + y : t * 16 + y * 8 + (lane >> 2))] = o[n][t][2 * y + x];
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
template <typename QT, bool LIST>
__global__ void __launch_bounds__(SP_THREADS) k_paged_join(const __grid_constant__ SplitArgs X) {
    const PagedAttnArgs& A = X.a;
    const PagedArgs& P = A.p;
    const int64_t run = run_of(all_units<LIST>(X), X.ctas);
    Line at = {0, 0, {}};
    const bool any = advance<LIST>(X, blockIdx.x, true, at);  // pair blockIdx.x, counted in pairs
    const int seq = at.b, pair = (int)(blockIdx.x - at.base);
    // units before this sequence
    int64_t before = 0;
    for (int b = threadIdx.x & 31; b < seq; b += 32) {
        const SeqWork w = seq_work<LIST>(X, b);
        before += (int64_t)w.pairs * w.units;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    const int64_t p0 = before + (int64_t)pair * at.w.units, p1 = p0 + at.w.units;
    const int c0 = (int)quotient(p0, run), c1 = (int)quotient(p1 - 1, run);
    pdl_wait();  // (every CTA waits: the next kernel on the stream begins when this grid has ended)
    if (!any || c0 == c1) return;  // c0 == c1: one CTA took it whole
    const int kvh = pair % P.nkv, r0 = at.w.r0;
    int m0, mrows;
    tile_rows<LIST>(X, pair / P.nkv, at.w.r1 - r0, m0, mrows);
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
inline int64_t pairs_bound(const SplitArgs& X) {
    if (X.l.width) return (int64_t)X.a.p.n_rows * X.tg * X.a.p.nkv;
    return ((int64_t)X.a.p.n_rows * X.a.G / X.rows + X.a.p.n_seqs) * X.a.p.nkv;
}

template <typename QT, bool LIST>
int launch_join(const SplitArgs& X, int64_t pairs, cudaStream_t s) {
    const int y = (std::min(X.rows, X.a.G) * X.a.p.hd / 4 + SP_THREADS - 1) / SP_THREADS;
    HC_TRY(launch_pdl(k_paged_join<QT, LIST>, dim3((unsigned)pairs, std::max(y, 1)), dim3(SP_THREADS), 0, s, X));
    HC_LAUNCH_CHECK();
    return HC_OK;
}

template <typename QT, typename CT, int HD, int NQ, bool LIST>
int launch_split_t(SplitArgs& X, cudaStream_t s) {
    using Sh = SplitShape<CT, HD>;
    static std::atomic<uint64_t> asked{0};
    HC_TRY(ask_smem((const void*)k_paged_split<QT, CT, HD, NQ, LIST>, Sh::SMEM, asked));
    const PagedArgs& P = X.a.p;
    static const int resident = [] {  // CTAs an SM holds: the kernel's registers and shared memory decide
        int n = 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k_paged_split<QT, CT, HD, NQ, LIST>, SP_THREADS, Sh::SMEM) != cudaSuccess) n = 1;
        return std::min(std::max(n, 1), SP_CTAS / 148);
    }();
    X.ctas = 148 * resident;
    const int64_t pairs = pairs_bound(X);
    HC_CHECK(pairs <= 0x7fffffff, HC_ERR_INVALID, "paged attention: %d rows of %d heads", P.n_rows, X.a.nh);
    k_paged_split<QT, CT, HD, NQ, LIST><<<X.whole ? (unsigned)pairs : (unsigned)X.ctas, SP_THREADS, Sh::SMEM, s>>>(X);
    HC_LAUNCH_CHECK();
    return X.whole ? HC_OK : launch_join<QT, LIST>(X, pairs, s);
}

template <typename QT, typename CT, bool LIST>
int launch_split_hd(SplitArgs& X, cudaStream_t s) {
    const int hd = X.a.p.hd;
    if constexpr (!std::is_same<CT, float>::value) {
        if (hd > 128) return launch_split_t<QT, CT, 256, 1, LIST>(X, s);
    }
    if (X.rows == 8) return hd <= 64 ? launch_split_t<QT, CT, 64, 1, LIST>(X, s) : launch_split_t<QT, CT, 128, 1, LIST>(X, s);
    return hd <= 64 ? launch_split_t<QT, CT, 64, 2, LIST>(X, s) : launch_split_t<QT, CT, 128, 2, LIST>(X, s);
}

}  // namespace

// One of each for every cache type and both kinds of call, in files of their own
// (hc_paged_split.cu, hc_paged_split_q4.cu, hc_paged_split_list.cu).
int launch_split_dense(SplitArgs& X, int q16, int kv, cudaStream_t s);
int launch_split_q4(SplitArgs& X, int q16, cudaStream_t s);
int launch_split_list(SplitArgs& X, int q16, int kv, cudaStream_t s);
int launch_q4_stream(SplitArgs& X, int q16, cudaStream_t s);  // heads of 64 or 128, X.uni

}  // namespace hc
