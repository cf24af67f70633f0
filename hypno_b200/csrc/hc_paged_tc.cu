// Attention over a paged FP16 cache for sequences with many rows (prompts,
// chunks): tcgen05 products, softmax in registers, accumulators in tensor
// memory.
//
// A CTA takes 256 packed (token, query head of the group) rows of one
// (sequence, KV head) as two halves of 128, and walks key tiles of 128:
//   S_h = Q_h K^T          tcgen05.mma, Q and K in shared memory (128 x 128 f32)
//   P_h = 2^(c S_h - m)    two threads per row, 64 keys each, S read from tensor memory
//   O_h += P_h V           tcgen05.mma, P in tensor memory over S, V in shared memory
// While one half's threads work on their weights the tensor core works on
// the other half's products; S, P and O of both halves fill the 512 columns.
// A half's weights and its products wait for one another, so the time from
// S_h to P_h counts in full: two threads a row (16 warps, four a scheduler)
// halve it, where one thread a row left the schedulers idle for want of
// independent work.  The products start when each thread has 32 of its 64
// weights.
//
// 16-bit queries: the weights are fp16 for the product with V (the operand type
// that runs at the full rate; l adds them up before they are rounded), which
// adds to a result's own rounding less than that itself: relative error against
// 64 bits 2.7e-4 where f32 weights have 2.1e-4 (512 tokens over 16,384 keys).
// O adds up in tensor memory, so the running maximum m moves
// only when a row's maximum passes it by more than 2^TAU (the weights are held
// times 2^BIAS and stay below 2^15, so that one of 2^-25 of the largest still
// has 11 bits); O is rescaled in the first tiles and rarely after them.
// Bound by the exponentials as much as by the products (128 x 128 of them take
// 1024 cycles of the SM's special function units, the two products 1024 of the
// tensor core), so part of them is a polynomial on the multiply-add units.
//
// f32 queries enter as q = 2^e (hi + lo), fp16 each, e the row's own, and their
// weights as hi + lo: twice the products.  The tensor core cuts (does not
// round) the low bits of its running sums, which over many tiles is a bias
// of several f32 ulps, so a tile's outputs start from zero and the running
// ones are in registers of the row's threads, 64 columns each, added to in f32.
//
// Warps: 0-7 and 8-15 the halves' rows (load Q, softmax, output; of a half's
// eight, the first four take keys 0-63 and the low columns of O, the others the
// rest), 16 issues the products, 17 (to 19) copy K and V tiles.  Pages of a multiple of eight
// positions come by TMA, in boxes of as many positions (8 to 128) as divide the
// page: a lane looks up one box's page.  Pages of other sizes are looked up key
// by key and come by cp.async, 16 bytes a thread; that took 4,400 to 6,000
// cycles a tile pair, where the products of a pair take 2,048.  (TMA gathers of
// four rows an instruction took 78 cycles each, 10,000 a pair.)  Keys without a
// page are zeros; keys of a box that no row sees are zeroed by the rows' threads.
//
// 512 tokens over 16,384 keys, 64 heads over 8 of 128, f16: 331 us, 816 TFLOP/s
// (301 us, 899, with the GPU cool); bound by the chain from S_h to P_h of a half.
// 4 prompts of 2,048, 32 heads over 8: f32 380 us, 362 TFLOP/s of twice as many
// products (342 us with the GPU cool), f16 222 us, 619 TFLOP/s (cool); a CTA's start
// (queries to shared memory) and end, some 19,000 cycles of 55,000, overlap
// nothing.  Key by key copies in place of boxes, cool: 477, 434 and 335 us.
//
// The loop of the rows' warps is kept short (values that are not finite have a
// loop of their own): the instruction fetch of code unrolled for every case cost
// more than its arithmetic.
#include "hc_paged.h"
#include "hc_tc.cuh"

#include <type_traits>

namespace hc {

namespace {

constexpr int TC_HALF = 128, TC_ROWS = 256, TC_KEYS = 128;
constexpr int TC_THREADS = 640;  // 16 warps of rows (two threads a row), 4 of products and copies
constexpr int TC_COPY = 3;       // copying warps where keys come one by one, every third group of eight each
constexpr int TC_MASKS = 8;      // ring of the tiles' key bits
constexpr float TAU = 4.0f, BIAS = 11.0f, BIAS_EXACT = 15.0f;
constexpr int POLY_OF_8 = 2;     // of eight pairs of weights, those by the polynomial

struct TcArgs {
    PagedAttnArgs a;
    CUtensorMap kmap, vmap;  // the pools as [page][head][position][64 elements] (TMA only)
    int box;                 // positions of a box, 0: copies key by key
    int nsplit;   // runs of key tiles per row tile
    int longest;  // the host's bound of the lengths; 0: all CTAs are resident at once, any order will do
    float* po;    // [(tile * nkv + kvh) * nsplit + run][256][hd]
    float2* pml;  // [..][256] (maximum in log2 units, sum)
};

constexpr int TC_CTRL = 3 * 1024; // shared memory before the queries and the ring, which begin on a 1024-byte boundary

template <int HD, bool HILO>
struct TcShape {
    static constexpr int QH = TC_HALF * HD * 2 * (HILO ? 2 : 1);   // bytes of a half's queries: hi, lo
    static constexpr int QG = (HILO ? 2 : 1) * (HD / 64) * 1024;   // bytes of eight rows: 128-byte pieces, hi then lo
    static constexpr int TILE = TC_KEYS * HD * 2;
    static constexpr int NS = HD == 64 ? 6 : (HILO ? 3 : 5);       // key / value tiles in flight
    static constexpr int SMEM = TC_CTRL + 2 * QH + NS * TILE;
};

struct TcBarriers {
    uint64_t full[6], empty[6];
    uint64_t q_ready[2], s_full[2], o_full[2], vote[2];
    uint64_t p_ready[2][2];  // [half][keys 0-31 and 64-95, the others]
    uint64_t fin[8];         // the pairs of warps of the same rows, at the end
    uint64_t drain;
};

// The key tiles of a CTA: positions begin + 128 j for j in [ja, jb), of which
// half h is active in [ha[h], hb[h]).
struct TcRange {
    int begin, end;    // begin: a multiple of the box
    int seen;          // first position that any row sees
    int ja, jb;
    int ha[2], hb[2];
};
struct TcControl {
    TcBarriers bars;
    __align__(16) uint32_t in[TC_MASKS][4];  // which keys of a tile exist (bytes of eight)
    float pair[TC_ROWS][2];                  // what a row's two threads tell one another
    uint32_t tmem;
    int abort, skip[2], bad[2], tile[6];
    TcRange range;
};
static_assert(sizeof(TcControl) <= TC_CTRL, "the control block fits");

__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}

__device__ __forceinline__ void tmem_ld_x8(uint32_t taddr, uint32_t* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr)
                 : "memory");
}

// Waits for tensor-memory loads; the registers named are used only after it.
__device__ __forceinline__ void tmem_wait_ld16(uint32_t* v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]),
                   "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
                 :
                 : "memory");
}

// A box of a 4-D tensor map into this CTA's shared memory.
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int pos, int head, int page) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
        "[%2];" ::"r"(dst),
        "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(pos), "r"(head), "r"(page)
        : "memory");
}

// D (+)= A[smem descriptor] x B[smem descriptor], kind::f16, one CTA.
__device__ __forceinline__ void mma_f16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Descriptor of an MN-major tile (V: rows of 64 head columns by key) in the
// 128-byte swizzle layout: eight keys 1024 bytes apart, blocks of 64 columns
// one tile of 128 keys apart.
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t saddr) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr >> 4) & 0x3FFF);
    d |= (uint64_t)((TC_KEYS * 128) >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Largest of three, NaN if any is.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// Pairs of f32 in one instruction.
typedef unsigned long long f2;
__device__ __forceinline__ f2 two(float a, float b) {
    f2 y;
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ void untwo(f2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 y;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
    return y;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 y;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 y;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}
// 2^x of a pair without the special function unit: x = n + r with n the nearest
// integer (read from the low bits of x + 1.5 2^23), 2^r by the polynomial of
// degree 5 with the least relative error on [-1/2, 1/2] (Remez exchange, the
// coefficients then rounded to f32: 1.6e-7 as they stand, 2.1e-7 evaluated in
// f32; degree 3 would do for fp16 weights but not for the sums), n added to the
// exponent.  x below -126 counts as -126.
__device__ __forceinline__ void ex2_poly(f2 x, float& y0, float& y1) {
    float a, b;
    untwo(x, a, b);
    x = two(fmaxf(a, -126.0f), fmaxf(b, -126.0f));
    const f2 t = add2(x, two(12582912.0f, 12582912.0f));
    const f2 n = add2(t, two(-12582912.0f, -12582912.0f));
    const f2 r = fma2(n, two(-1.0f, -1.0f), x);
    f2 p = fma2(r, two(0.0013276472f, 0.0013276472f), two(0.009675541f, 0.009675541f));
    p = fma2(p, r, two(0.05550713f, 0.05550713f));
    p = fma2(p, r, two(0.2402212f, 0.2402212f));
    p = fma2(p, r, two(0.69314694f, 0.69314694f));
    p = fma2(p, r, two(1.0000001f, 1.0000001f));
    float ta, tb;
    untwo(t, ta, tb);
    untwo(p, a, b);
    y0 = __uint_as_float(__float_as_uint(a) + (__float_as_uint(ta) << 23));
    y1 = __uint_as_float(__float_as_uint(b) + (__float_as_uint(tb) << 23));
}

// A wait that mostly finds its phase complete: the bounded loop is off the path.
__device__ __forceinline__ bool quick_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    return mbar_try_wait(bar, parity) || mbar_wait(bar, parity, abort_flag);
}

__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ TcRange tc_range(const PagedAttnArgs& A, int first, int m0, int mtot, int run, int nsplit, int box) {
    TcRange r;
    visible(A, first, m0, min(TC_ROWS, mtot - m0), r.seen, r.end);
    r.begin = box > 0 ? r.seen & ~(box - 1) : r.seen;
    const int n = (r.end - r.begin + TC_KEYS - 1) / TC_KEYS;
    const int per = (n + nsplit - 1) / nsplit;
    r.ja = min(n, run * per);
    r.jb = min(n, r.ja + per);
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int mh = m0 + h * TC_HALF, rows = min(TC_HALF, mtot - mh);
        r.ha[h] = r.hb[h] = r.ja;
        if (rows <= 0) continue;
        int b, e;
        visible(A, first, mh, rows, b, e);
        if (e <= b) continue;
        r.ha[h] = min(max((b - r.begin) / TC_KEYS, r.ja), r.jb);
        r.hb[h] = max(min((e - r.begin + TC_KEYS - 1) / TC_KEYS, r.jb), r.ha[h]);
    }
    return r;
}

// The n-th row tile: sequences of more visible keys first, in classes of a
// sixteenth of the longest, and a sequence's later tiles, which see more of
// them, before its earlier ones (a CTA that begins last should end soon; all
// heads of a tile are next to one another; 24 ragged sequences of up to 257
// tokens over up to 4,001 keys: 164 to 169 us, 196 in the sequences' order).  Executed
// by a whole warp; false past the last tile.
__device__ __forceinline__ bool tile_at(const TcArgs& X, int n, int& seq, int& in_seq) {
    constexpr int CLASSES = 16;
    const PagedAttnArgs& A = X.a;
    const PagedArgs& P = A.p;
    const int lane = threadIdx.x & 31;
    const int span = max(A.window > 0 ? min(A.window, X.longest) : X.longest, 1);
    auto tiles_of = [&](int b, int& cls) -> int {
        cls = -1;
        if (b >= P.n_seqs) return 0;
        int r0, r1;
        seq_rows(P, b, r0, r1);
        const int len = min(max(seq_len(P, b), 1), span);
        cls = (int)((int64_t)(len - 1) * CLASSES / span);
        return (int)(((int64_t)(r1 - r0) * A.G + TC_ROWS - 1) / TC_ROWS);
    };
    int cls = X.longest > 0 ? -1 : 0, before = 0;  // (span 1: all sequences are of class 0)
    if (cls < 0) {
        int total[CLASSES];
#pragma unroll
        for (int c = 0; c < CLASSES; c++) total[c] = 0;
        for (int b0 = 0; b0 < P.n_seqs; b0 += 32) {
            int its;
            const int t = tiles_of(b0 + lane, its);
#pragma unroll
            for (int c = 0; c < CLASSES; c++) total[c] += __reduce_add_sync(0xffffffffu, its == c ? t : 0);
        }
#pragma unroll
        for (int c = CLASSES - 1; c >= 0; c--) {
            if (cls >= 0) continue;
            if (n - before < total[c]) cls = c;
            else before += total[c];
        }
        if (cls < 0) return false;
    }
    for (int b0 = 0; b0 < P.n_seqs; b0 += 32) {
        int its;
        int t = tiles_of(b0 + lane, its);
        if (its != cls) t = 0;
        int incl = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + incl > n);
        if (hit) {
            const int l = __ffs(hit) - 1;
            seq = b0 + l;
            in_seq = before + __shfl_sync(0xffffffffu, incl, l) - 1 - n;
            return true;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    return false;
}

template <typename QT, int HD, bool TMA>
__global__ void __launch_bounds__(TC_THREADS, 1) k_paged_tc(const __grid_constant__ TcArgs X) {
    constexpr bool HILO = sizeof(QT) == 4;
    using Sh = TcShape<HD, HILO>;
    constexpr int NS = Sh::NS, PL = HILO ? 2 : 1;
    // registers of a row's thread and of the others': 512 R + 128 C = 640 x 96, what the launch holds
    constexpr int REG_ROW = 104, REG_CTRL = 64;
    const PagedAttnArgs& A = X.a;
    const PagedArgs& P = A.p;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    TcControl& C = *reinterpret_cast<TcControl*>(smem_raw);
    TcBarriers& B = C.bars;
    auto& s_in = C.in;
    auto& s_pair = C.pair;
    auto& s_skip = C.skip;
    auto& s_bad = C.bad;
    auto& s_tile = C.tile;
    int& abort_flag = C.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t q_s = smem_u32(smem_raw) + TC_CTRL, ring = q_s + 2 * Sh::QH;
    pdl_trigger();  // the join may become resident; it waits for this grid's end

    if (warp == 0) {
        int seq = 0, tile = 0;
        const bool ok = tile_at(X, (int)(blockIdx.x / ((unsigned)P.nkv * X.nsplit)), seq, tile);
        if (ok && lane == 0) {
            // once for all warps: everything that follows from the tile's place
            int a, b;
            seq_rows(P, seq, a, b);
            const int at = seq_len(P, seq) - (b - a), m = tile * TC_ROWS;
            s_tile[1] = seq;
            s_tile[2] = m;
            s_tile[3] = a;
            s_tile[4] = (int)min((int64_t)(b - a) * A.G, (int64_t)m + TC_ROWS);  // rows up to this tile's end
            s_tile[5] = at;
            C.range = tc_range(A, at, m, s_tile[4], (int)(blockIdx.x / P.nkv % X.nsplit), X.nsplit, TMA ? X.box : 0);
        }
        if (lane == 0) s_tile[0] = ok;
    }
    if (threadIdx.x == 32) {
        abort_flag = 0;
        s_bad[0] = s_bad[1] = 0;
        for (int i = 0; i < NS; i++) {
            mbar_init(&B.full[i], TMA ? 1 : TC_COPY);
            mbar_init(&B.empty[i], 1);
        }
        for (int h = 0; h < 2; h++) {
            mbar_init(&B.q_ready[h], 256);
            mbar_init(&B.s_full[h], 1);
            mbar_init(&B.p_ready[h][0], 256);
            mbar_init(&B.p_ready[h][1], 256);
            mbar_init(&B.o_full[h], 1);
            mbar_init(&B.vote[h], 256);
        }
        for (int i = 0; i < 8; i++) mbar_init(&B.fin[i], 64);
        mbar_init(&B.drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&C.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = C.tmem;
    if (!s_tile[0]) {  // the grid is an upper bound
        if (warp == 16) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
        return;
    }
    const int kvh = (int)(blockIdx.x % P.nkv), at_tile = (int)(blockIdx.x / P.nkv), run = at_tile % X.nsplit;
    const int seq = s_tile[1], m0 = s_tile[2], r0 = s_tile[3], mtot = s_tile[4], first = s_tile[5];
    const TcRange rg = C.range;

    if (warp < 16) {
        // ================ the halves: queries, weights, outputs
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REG_ROW));
        const int h = warp >> 3, g = (warp >> 2) & 1, r = (warp & 3) * 32 + lane;  // half, key half, row
        const int mh = m0 + h * TC_HALF, rows = min(max(mtot - mh, 0), TC_HALF);
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
        // this thread's 64 score columns and HD / 2 output columns
        constexpr int HO = HD / 2;
        const uint32_t s_col = tmem + lane_off + (uint32_t)(h * 128 + g * 64), o_col = tmem + lane_off + 256u + (uint32_t)(h * 128 + g * HO);
        const uint32_t qs = q_s + h * Sh::QH;
        // the other warp of these rows (one that gives up arrives once more, so that nobody is left waiting)
        const int pair_id = 1 + h * 4 + (warp & 3);
        auto pair_sync = [&]() { named_sync(pair_id, 64); };
        bool ok = true;
        float up = 1.0f;  // 2^e of an f32 row
        auto row_offset = [&](int64_t rs, int64_t hs) -> int64_t {
            const int t = token_of(A, mh + r);
            return (int64_t)(r0 + t) * rs + (kvh * A.G + (mh + r) - t * A.G) * hs;
        };
        // ---- queries.  Eight rows are QG bytes, whether as they come (f32 or fp16
        // rows one after the other) or as the products take them (128-byte pieces
        // of the eight rows), so a warp copies its rows as they come and turns
        // them over eight at a time in place.
        if (rg.hb[h] > rg.ha[h]) {
            constexpr int EPL = HILO ? 4 : 8, LPR = HD / EPL, RPI = 32 / LPR;  // elements a lane, lanes a row, rows at once
            const int d = (lane % LPR) * EPL;
            const uint32_t mine = qs + (uint32_t)(((warp & 3) * 4 + g * 2) * Sh::QG);  // 16 rows
            const int row0 = (warp & 3) * 32 + g * 16;
            const int64_t at = r < rows ? row_offset(A.q_rs, A.q_hs) : 0;  // of this lane's row
#pragma unroll 4
            for (int i = 0; i < 16 / RPI; i++) {
                const int rr = i * RPI + lane / LPR, row = row0 + rr;
                const bool there = row < rows && d < P.hd;
                const QT* q = (const QT*)A.q + __shfl_sync(0xffffffffu, at, g * 16 + rr) + (there ? d : 0);
                const uint32_t dst = mine + (HILO ? (uint32_t)(rr * HD * 4 + (lane % LPR) * 16)
                                                  : (uint32_t)((rr >> 3) * Sh::QG + (d >> 6) * 1024 + (rr & 7) * 128 + ((((d & 63) >> 3) ^ (rr & 7)) << 4)));
                if (A.qvec || !there) {
                    cp16(dst, there ? (const void*)q : P.k, there);
                } else {
#pragma unroll 1
                    for (int e = 0; e < EPL; e++) {
                        if constexpr (HILO) asm volatile("st.shared.f32 [%0], %1;" ::"r"(dst + 4 * e), "f"(q[e]) : "memory");
                        else asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst + 2 * e), "h"(__half_as_ushort(q[e])) : "memory");
                    }
                }
            }
            cp_commit();
            cp_wait<0>();
            __syncwarp();
            if constexpr (HILO) {
#pragma unroll 1
                for (int e8 = 0; e8 < 2; e8++) {
                    constexpr int N = 8 / RPI;
                    float f[N][4];
#pragma unroll
                    for (int i = 0; i < N; i++)
                        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(f[i][0]), "=f"(f[i][1]), "=f"(f[i][2]), "=f"(f[i][3])
                                     : "r"(mine + (uint32_t)(e8 * Sh::QG + (i * RPI + lane / LPR) * HD * 4 + (lane % LPR) * 16)));
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const int rr = i * RPI + lane / LPR;  // of the eight
                        float mx = fmaxf(fmaxf(fabsf(f[i][0]), fabsf(f[i][1])), fmaxf(fabsf(f[i][2]), fabsf(f[i][3])));
                        if constexpr (LPR == 32) {  // |q| orders like its bits
                            mx = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mx)));
                        } else {
#pragma unroll
                            for (int o = 1; o < LPR; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                        }
                        const int e = min(max((int)(__float_as_uint(mx) >> 23), 2), 252);
                        const float down = __uint_as_float((uint32_t)(254 - e) << 23);
                        uint32_t hi[2], lo[2];
                        split2(f[i][0] * down, f[i][1] * down, hi[0], lo[0]);
                        split2(f[i][2] * down, f[i][3] * down, hi[1], lo[1]);
                        const uint32_t dst = mine + (uint32_t)(e8 * Sh::QG + (d >> 6) * 1024 + rr * 128 + ((((d & 63) >> 3) ^ rr) << 4) + (d & 7) * 2);
                        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(dst), "r"(hi[0]), "r"(hi[1]) : "memory");
                        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(dst + Sh::QG / 2), "r"(lo[0]), "r"(lo[1]) : "memory");
                        if (lane % LPR == 0) s_pair[h * TC_HALF + row0 + e8 * 8 + rr][0] = __uint_as_float((uint32_t)e << 23);
                    }
                    __syncwarp();
                }
            }
            fence_async_shared();
            if constexpr (HILO) {
                pair_sync();
                up = s_pair[h * TC_HALF + r][0];
                __syncwarp();
            }
            mbar_arrive(&B.q_ready[h]);  // (no scores, so nobody's next word in s_pair, before all have read it)
        }
        const bool in = r < rows;
        const int pos = in ? first + token_of(A, mh + r) : -1;
        const int lo_pos = A.window > 0 ? pos - A.window + 1 : 0;
        const int p_min = first + token_of(A, mh), l_max = A.window > 0 ? first + token_of(A, mh + rows - 1) - A.window + 1 : 0;
        // (never 0, which would make -inf, a masked key, NaN: a row of zeros has the least `up`)
        const float cf = fmaxf(A.scale * LOG2E * up, 1.401298464e-45f);
        float m = -INFINITY, l = 0.0f;  // running maximum (log2 units), sum of weights
        float acc[HILO ? HO : 1];       // f32 queries: the running outputs
        if constexpr (HILO) {
#pragma unroll
            for (int i = 0; i < HO; i++) acc[i] = 0.0f;
        }
        bool tile_out = false;          // f32 queries: a tile's outputs are in tensor memory
        auto add_tile = [&]() {
            if constexpr (HILO) {
#pragma unroll
                for (int c = 0; c < HO / 16; c++) {
                    uint32_t u[16];
                    tmem_ld_x16(o_col + 16u * c, u);
                    tmem_wait_ld16(u);
#pragma unroll
                    for (int i = 0; i < 16; i += 2)
                        untwo(add2(two(acc[16 * c + i], acc[16 * c + i + 1]), two(__uint_as_float(u[i]), __uint_as_float(u[i + 1]))),
                              acc[16 * c + i], acc[16 * c + i + 1]);
                }
            }
        };
        // The maximum moves to `nm` (NaN and +inf make the row NaN); returns
        // the factor of what was summed with the old one.
        auto move_max = [&](float nm, bool raise) -> float {
            float to = raise ? nm : m;
            if (!(to < INFINITY) || m != m) to = __int_as_float(0x7fffffff);
            const float f = to == m ? 1.0f : ex2(m - to);
            m = to;
            l *= f;
            return f;
        };
        // A tile's products by the row's threads, masked keys left out: from the
        // scores still in tensor memory into the half's outputs there, this
        // thread's columns of them.
        auto careful = [&](float nb, bool add, uint32_t vt, int hi_c, int lo_c, const uint32_t* bits) {
#pragma unroll 1
            for (int c1 = 0; c1 < HO; c1 += 8) {
                const int c0 = g * HO + c1;
                uint32_t u[8];
                float o[8];
                if (add) {
                    tmem_ld_x8(o_col + c1, u);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int i = 0; i < 8; i++) o[i] = add ? __uint_as_float(u[i]) : 0.0f;
#pragma unroll 1
                for (int k = 0; k < TC_KEYS; k += 8) {
                    tmem_ld_x8(s_col - (uint32_t)(g * 64) + (uint32_t)k, u);
                    tmem_wait_ld();
#pragma unroll
                    for (int y = 0; y < 8; y++) {
                        const int key = k + y;
                        if (key > hi_c || key < lo_c || !((bits[key >> 5] >> (key & 31)) & 1u)) continue;
                        const float p = ex2(fmaf(__uint_as_float(u[y]), cf, nb));
                        uint32_t w[4];
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                                     : "r"(vt + (c0 >> 6) * (TC_KEYS * 128) + key * 128 + ((((c0 & 63) >> 3) ^ (key & 7)) << 4)));
#pragma unroll
                        for (int z = 0; z < 4; z++) {
                            const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&w[z]));
                            o[2 * z] = fmaf(p, g.x, o[2 * z]);
                            o[2 * z + 1] = fmaf(p, g.y, o[2 * z + 1]);
                        }
                    }
                    __syncwarp();
                }
#pragma unroll
                for (int i = 0; i < 8; i++) u[i] = __float_as_uint(o[i]);
                tmem_st_x8(o_col + c1, u);
            }
            tmem_wait_st();
            pair_sync();  // both have read the scores that the weights will overwrite
        };
        uint32_t done = 0, votes = 0;
        for (int j = rg.ha[h]; j < rg.hb[h]; j++, done++) {
            ok = quick_wait(&B.s_full[h], done & 1u, &abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tmem_fence_after();
            const int k0 = rg.begin + j * TC_KEYS;
            const uint32_t* bits = s_in[j % TC_MASKS];
            const uint4 b4 = *reinterpret_cast<const uint4*>(bits);
            const bool whole = k0 + TC_KEYS - 1 <= p_min && k0 >= l_max && (b4.x & b4.y & b4.z & b4.w) == 0xffffffffu;
            const int hi_c = pos - k0, lo_c = lo_pos - k0;
            // A key that some rows (of either half: the tile is both's) see and others
            // do not must not reach the latter through 0 * v where v is not finite:
            // such a tile (rare) leaves the products to the row's thread, masked keys
            // left out.  Keys without a page are zeros.
            const bool equal = min(k0 + TC_KEYS, rg.end) - 1 <= p_min && max(k0, rg.seen) >= l_max;  // this half's rows see them all
            bool skip = false;
            uint32_t vt = 0;
            // keys of the tile that no row sees: what their memory holds is nobody's
            const bool strangers = TMA && (k0 < rg.seen || k0 + TC_KEYS > rg.end);
            if (!equal || strangers) {
                const int n = 2 * (j - rg.ja) + 1, slot = n % NS;
                ok = mbar_wait(&B.full[slot], (uint32_t)(n / NS) & 1u, &abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                vt = ring + slot * Sh::TILE;
            }
            if (strangers) {
                // their values become zeros (by both halves, before either's products)
                if (k0 + r < rg.seen || k0 + r >= rg.end)
#pragma unroll 1
                    for (int c = g; c < HD / 64; c += 2)
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(vt + (uint32_t)(c * (TC_KEYS * 128) + r * 128 + i * 16)), "r"(0) : "memory");
                fence_async_shared();
            }
            if (!equal) {
                // (the other half may still be writing its zeros: a stranger is not looked at)
                uint32_t bad = 0;
                for (int i = r + g * TC_HALF; i < Sh::TILE / 16; i += 2 * TC_HALF) {
                    const int key = k0 + (i >> 3) % TC_KEYS;
                    if (key < rg.seen || key >= rg.end || (key <= p_min && key >= l_max)) continue;  // nobody's, or everybody's
                    uint32_t w[4];
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                                 : "r"(vt + 16 * i));
#pragma unroll
                    for (int y = 0; y < 4; y++) bad |= (w[y] & 0x7C007C00u) + 0x04000400u;
                }
                if (bad & 0x80008000u) s_bad[h] = j + 1;
                mbar_arrive(&B.vote[h]);
                ok = mbar_wait(&B.vote[h], votes++ & 1u, &abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                skip = *(volatile int*)&s_bad[h] == j + 1;
            }
            if (r == 0 && g == 0) s_skip[h] = skip;

            uint32_t vis[2] = {0u, 0u};  // the visible ones of this thread's keys, as bits
            if (!whole) {
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const int up = min(hi_c - 64 * g - 32 * c, 31), dn = max(lo_c - 64 * g - 32 * c, 0);
                    if (up >= dn) vis[c] = bits[2 * g + c] & (0xffffffffu >> (31 - up)) & (0xffffffffu << dn);
                }
            }
            float sum0 = 0.0f, sum1 = 0.0f;
            // the row's maximum: this thread's 64 keys and the other's
            auto row_max = [&](float x) -> float {
                s_pair[h * TC_HALF + r][g] = x;
                pair_sync();
                return max3(x, s_pair[h * TC_HALF + r][g ^ 1], x) * cf;
            };
            if constexpr (HILO) {
                if (tile_out) add_tile();
                tile_out = true;
                float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint32_t v[16];
                    tmem_ld_x16(s_col + 16u * c, v);
                    tmem_wait_ld16(v);
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            if (!((vis[c >> 1] >> (16 * (c & 1) + i)) & 1u)) v[i] = 0xff800000u;
                        tmem_st_x16(s_col + 16u * c, v);  // they are read again
                    }
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        x0 = max3(x0, __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
                        x1 = max3(x1, __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
                    }
                }
                if (!whole) tmem_wait_st();
                const float nm = row_max(max3(x0, x1, x1));
                const bool raise = !(nm <= m);
                if (__any_sync(0xffffffffu, raise)) {
                    const float f = move_max(nm, raise);
                    const f2 ff = two(f, f);
#pragma unroll
                    for (int i = 0; i < HO; i += 2) untwo(mul2(two(acc[i], acc[i + 1]), ff), acc[i], acc[i + 1]);
                }
                const float nb = m == -INFINITY ? 0.0f : BIAS_EXACT - m;
                if (skip) careful(nb, false, vt, hi_c, lo_c, bits);
                const f2 cf2 = two(cf, cf), nb2 = two(nb, nb), minus = two(-1.0f, -1.0f);
                f2 sum = 0;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint32_t v[16], hi[8], lo[8];
                    tmem_ld_x16(s_col + 16u * c, v);
                    tmem_wait_ld16(v);
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        float a, b;
                        untwo(fma2(two(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), cf2, nb2), a, b);
                        const f2 w = two(ex2(a), ex2(b));
                        sum = add2(sum, w);
                        untwo(w, a, b);
                        hi[i / 2] = pack(a, b);
                        const float2 q = __half22float2(*reinterpret_cast<const __half2*>(&hi[i / 2]));
                        untwo(fma2(two(q.x, q.y), minus, w), a, b);
                        lo[i / 2] = pack(a, b);
                    }
                    // weights over the scores just read: hi in 8 columns, lo in the next 8
                    tmem_st_x8(s_col + 16u * c, hi);
                    tmem_st_x8(s_col + 16u * c + 8u, lo);
                    if (c == 1) {
                        tmem_wait_st();
                        tmem_fence_before();
                        mbar_arrive(&B.p_ready[h][0]);
                    }
                }
                untwo(sum, sum0, sum1);
            } else {
                uint32_t sr[64];
                tmem_ld_x32(s_col, sr);
                tmem_ld_x32(s_col + 32u, sr + 32);
                tmem_wait_ld();
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 64; i++)
                        if (!((vis[i >> 5] >> (i & 31)) & 1u)) sr[i] = 0xff800000u;
                }
                float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 64; c += 2) x[(c >> 1) & 3] = max3(x[(c >> 1) & 3], __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
                const float nm = row_max(max3(max3(x[0], x[1], x[2]), x[3], x[3]));
                const bool raise = !(nm <= m + TAU);
                if (__any_sync(0xffffffffu, raise)) {
                    const float f = move_max(nm, raise);
                    if (done > 0) {
                        // the products of the tile before are complete: this tile's
                        // scores were committed after them
#pragma unroll 1
                        for (int c = 0; c < HO / 16; c++) {
                            uint32_t o[16];
                            tmem_ld_x16(o_col + 16u * c, o);
                            tmem_wait_ld16(o);
#pragma unroll
                            for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tmem_st_x16(o_col + 16u * c, o);
                        }
                    }
                }
                const float nb = m == -INFINITY ? 0.0f : BIAS - m;
                if (skip) careful(nb, done > 0, vt, hi_c, lo_c, bits);
                const f2 cf2 = two(cf, cf), nb2 = two(nb, nb);
                f2 sum[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int k = 32 * c + 2 * i;
                        const f2 e = fma2(two(__uint_as_float(sr[k]), __uint_as_float(sr[k + 1])), cf2, nb2);
                        float a, b;
                        if ((i & 7) < POLY_OF_8) {
                            ex2_poly(e, a, b);
                        } else {
                            untwo(e, a, b);
                            a = ex2(a);
                            b = ex2(b);
                        }
                        sum[i & 1] = add2(sum[i & 1], two(a, b));
                        w[i] = pack(a, b);
                    }
                    // weights over this thread's own scores: 64 in 32 columns
                    tmem_st_x16(s_col + 16u * c, w);
                    if (c == 0) {
                        tmem_wait_st();
                        tmem_fence_before();
                        mbar_arrive(&B.p_ready[h][0]);
                    }
                }
                untwo(add2(sum[0], sum[1]), sum0, sum1);
            }
            l += m == -INFINITY ? 0.0f : sum0 + sum1;
            tmem_wait_st();
            tmem_fence_before();
            mbar_arrive(&B.p_ready[h][1]);
        }
        // ---- outputs
        const bool any = rg.hb[h] > rg.ha[h];
        if (any && ok) {
            ok = mbar_wait(&B.o_full[h], 0, &abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            tmem_fence_after();
            if (ok && tile_out) add_tile();
        }
        if (!ok) named_arrive(pair_id, 64);
        auto fin_sync = [&](uint32_t parity) -> bool {  // bounded: the other warp may have given up
            mbar_arrive(&B.fin[pair_id - 1]);
            return mbar_wait(&B.fin[pair_id - 1], parity, &abort_flag);
        };
        // the row's sum: this thread's keys and the other's
        if (rows > 0) {
            s_pair[h * TC_HALF + r][g] = l;
            ok = __all_sync(0xffffffffu, fin_sync(0) && ok && !*(volatile int*)&abort_flag);
            l += s_pair[h * TC_HALF + r][g ^ 1];
        }
        if (!ok) l = __int_as_float(0x7fffffff);  // a wait ran out: the row is NaN, not a wrong number
        const int64_t pr = (((int64_t)(at_tile / X.nsplit) * P.nkv + kvh) * X.nsplit + run) * TC_ROWS + h * TC_HALF + r;
        if (in && g == 0) {
            if (X.nsplit > 1) {
                X.pml[pr] = make_float2(m == -INFINITY ? m : m - (HILO ? BIAS_EXACT : BIAS), l);
            } else if (A.lse) {
                const int t = token_of(A, mh + r);
                A.lse[(int64_t)(r0 + t) * A.nh + kvh * A.G + (mh + r) - t * A.G] =
                    l == 0.0f ? -INFINITY : (m - (HILO ? BIAS_EXACT : BIAS) + log2f(l)) / LOG2E;
            }
        }
        __syncwarp();  // (the loads below are the warp's)
        const float inv = X.nsplit > 1 ? 1.0f : (l == 0.0f ? 0.0f : 1.0f / l);
        // 16 columns at a time: partial results straight to the workspace; results
        // through the half's query memory (its products are done), so that a
        // warp's stores are whole rows
        const uint32_t stage = qs + (uint32_t)((warp & 3) * 32 * HD * (int)sizeof(QT));
#pragma unroll(HILO ? HO / 16 : 1)
        for (int c = 0; c < HO / 16; c++) {
            const int cc = g * (HO / 16) + c;
            uint32_t o[16];
            if constexpr (HILO) {
#pragma unroll
                for (int i = 0; i < 16; i++) o[i] = __float_as_uint(acc[16 * c + i]);
            } else if (any && ok) {
                tmem_ld_x16(o_col + 16u * c, o);
                tmem_wait_ld();
            } else {
#pragma unroll
                for (int i = 0; i < 16; i++) o[i] = 0u;
            }
#pragma unroll
            for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * inv);
            if (X.nsplit > 1) {
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    if (in && 16 * cc + i < P.hd)
                        *reinterpret_cast<uint4*>(X.po + pr * P.hd + 16 * cc + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            } else {
                const uint32_t row_at = stage + (uint32_t)(lane * HD * (int)sizeof(QT));
                if constexpr (HILO) {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row_at + (((4 * cc + i) ^ (lane & 7)) << 4)),
                                     "r"(o[4 * i]), "r"(o[4 * i + 1]), "r"(o[4 * i + 2]), "r"(o[4 * i + 3])
                                     : "memory");
                } else {
                    uint32_t w[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) w[i] = pack(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1]));
#pragma unroll
                    for (int i = 0; i < 2; i++)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row_at + (((2 * cc + i) ^ (lane & 7)) << 4)),
                                     "r"(w[4 * i]), "r"(w[4 * i + 1]), "r"(w[4 * i + 2]), "r"(w[4 * i + 3])
                                     : "memory");
                }
            }
        }
        if (X.nsplit == 1 && rows > 0) {
            const int64_t at = in ? row_offset(A.o_rs, A.o_hs) : 0;
            fin_sync(1);
            constexpr int EPL = 16 / (int)sizeof(QT), LPR = HD / EPL, RPI = 32 / LPR;
            const int d = (lane % LPR) * EPL;
#pragma unroll 4
            for (int i = 0; i < 16 / RPI; i++) {
                const int rr = g * 16 + i * RPI + lane / LPR, row = (warp & 3) * 32 + rr;
                const int64_t off = __shfl_sync(0xffffffffu, at, rr);
                if (row >= rows || d >= P.hd) continue;
                uint32_t w[4];
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                             : "r"(stage + (uint32_t)(rr * HD * (int)sizeof(QT)) + (((lane % LPR) ^ (rr & 7)) << 4)));
                QT* out = (QT*)A.out + off + d;
                if (A.ovec) {
                    *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
#pragma unroll
                    for (int y = 0; y < EPL; y++) {
                        if constexpr (HILO) out[y] = __uint_as_float(w[y]);
                        else reinterpret_cast<unsigned short*>(out)[y] = (unsigned short)(w[y / 2] >> (16 * (y & 1)));
                    }
                }
            }
        }
        tmem_fence_before();
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REG_CTRL));
      if (warp == 16) {
        // ================ the products.  What addresses them is the same in all
        // lanes and said to be so: issued from ordinary registers a product took 90
        // to 110 cycles of the issuing warp, where the tensor core takes 64.
        constexpr uint32_t idesc_s = make_idesc_mn(128, 128);
        constexpr uint32_t idesc_o = make_idesc_mn(128, HD) | (1u << 16);  // V is MN-major
        const int ja = __shfl_sync(0xffffffffu, rg.ja, 0), jb = __shfl_sync(0xffffffffu, rg.jb, 0);
        const int ha0 = __shfl_sync(0xffffffffu, rg.ha[0], 0), hb0 = __shfl_sync(0xffffffffu, rg.hb[0], 0);
        const int ha1 = __shfl_sync(0xffffffffu, rg.ha[1], 0), hb1 = __shfl_sync(0xffffffffu, rg.hb[1], 0);
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        // eight rows of queries are QG apart
        const uint64_t q_d = (sw128_desc(q_s) & ~((uint64_t)0x3FFF << 32)) | (uint64_t)(Sh::QG >> 4) << 32;
        const uint64_t k_d0 = sw128_desc(ring), v_d0 = sw128_mn_desc(ring);
        bool ok = true;
        uint32_t pdone[2] = {0, 0};
        int ks = 0, vs = NS - 1;          // ring slots of K_j and V_(j-1), with their phases
        uint32_t kph = 0, vph = 1;
        if (NS > 3 && ja < jb) ok = quick_wait(&B.full[0], 0, &abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        for (int j = ja; j <= jb && ok; j++) {
            const uint64_t k_d = k_d0 + (uint64_t)(ks * (Sh::TILE >> 4)), v_d = v_d0 + (uint64_t)(vs * (Sh::TILE >> 4));
            int vs2 = vs + 2, ks2 = ks + 2;  // V_j, K_(j+1)
            uint32_t vph2 = vph, kph2 = kph;
            if (vs2 >= NS) vs2 -= NS, vph2 ^= 1u;
            if (ks2 >= NS) ks2 -= NS, kph2 ^= 1u;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t s_t = tm + (uint32_t)(h * 128), o_t = tm + 256u + (uint32_t)(h * 128);
                const int ha = h ? ha1 : ha0, hb = h ? hb1 : hb0;
                const bool pv = j - 1 >= ha && j - 1 < hb, sc = j >= ha && j < hb;
                bool mul = false;  // O_h += P_h V_(j-1), half of the keys as soon as their weights are there
                auto add_pv = [&](int part) {
#pragma unroll
                    for (int p = PL - 1; p >= 0; p--)
#pragma unroll
                        for (int k4 = 0; k4 < 4; k4++) {
                            const int kk = (k4 >> 1) * 4 + part * 2 + (k4 & 1);  // of the eight steps of 16 keys
                            mma_f16_ts(o_t, s_t + (uint32_t)(HILO ? kk * 16 + p * 8 : (kk >> 2) * 64 + (kk & 3) * 8), v_d + (uint64_t)(kk * (2048 >> 4)),
                                       idesc_o, (!HILO && pdone[h] > 0) || part > 0 || k4 > 0 || p < PL - 1);
                        }
                };
                bool both = false;
                if (pv) {
                    ok = ok && quick_wait(&B.p_ready[h][0], pdone[h] & 1u, &abort_flag);
                    __syncwarp();
                    both = __all_sync(0xffffffffu, mbar_try_wait(&B.p_ready[h][1], pdone[h] & 1u));
                    tmem_fence_after();
                    mul = !*(volatile int*)&s_skip[h];
                    ok = __all_sync(0xffffffffu, ok);
                    if (!both) {
                        if (mul && ok && elect_one()) add_pv(0);
                        __syncwarp();
                        ok = ok && quick_wait(&B.p_ready[h][1], pdone[h] & 1u, &abort_flag);
                    }
                }
                if (NS == 3 && h == 0 && j < jb) ok = ok && quick_wait(&B.full[ks], kph, &abort_flag);  // (its slot was V_(j-2)'s)
                if (sc && j == ha) ok = ok && quick_wait(&B.q_ready[h], 0, &abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tmem_fence_after();
                if (elect_one()) {
                    if (mul) {
                        if (both) add_pv(0);
                        add_pv(1);
                    }
                    if (h == 1 && j > ja) mma_commit(&B.empty[vs]);
                    if (sc) {  // S_h = Q_h K_j^T
#pragma unroll
                        for (int p = PL - 1; p >= 0; p--)
#pragma unroll
                            for (int kk = 0; kk < HD / 16; kk++) {
                                const uint32_t qo = (uint32_t)((p * (HD / 64) + (kk >> 2)) * 1024 + (kk & 3) * 32);
                                const uint32_t ko = (uint32_t)((kk >> 2) * (TC_KEYS * 128) + (kk & 3) * 32);
                                mma_f16_ss(s_t, q_d + (uint64_t)((h * Sh::QH + qo) >> 4), k_d + (uint64_t)(ko >> 4), idesc_s, kk > 0 || p < PL - 1);
                            }
                        mma_commit(&B.s_full[h]);
                    }
                    if (h == 1 && j < jb) mma_commit(&B.empty[ks]);
                    if (j == hb && hb > ha) mma_commit(&B.o_full[h]);
                }
                __syncwarp();
                if (pv) pdone[h]++;
                // the copies that the next products need, while the tensor core is busy with these
                if (h == 0 && j < jb) ok = ok && quick_wait(&B.full[vs2], vph2, &abort_flag);
                if (NS > 3 && h == 1 && j + 1 < jb) ok = ok && quick_wait(&B.full[ks2], kph2, &abort_flag);
            }
            ks = ks2;
            kph = kph2;
            vs = vs2;
            vph = vph2;
        }
        if (!ok) {  // let what is in flight end before tensor memory is given back
            if (elect_one()) mma_commit(&B.drain);
            __syncwarp();
            int none = 0;
            mbar_wait(&B.drain, 0, &none);
        }
        tmem_fence_before();
      } else if (TMA && warp == 17) {
        // ================ the copies: lane l takes the tile's l-th box
        bool ok = true;
        int copied = 0;
        const int box = X.box, nbox = TC_KEYS / box;
        int page, slot;
        auto look = [&](int j) {
            const int p = rg.begin + j * TC_KEYS + lane * box;
            page = -1;
            slot = 0;
            if (lane < nbox && j < rg.jb && p < rg.end) page = lookup(P, seq, p, slot);
        };
        look(rg.ja);
        for (int j = rg.ja; j < rg.jb && ok; j++) {
            const int pg = page >= 0 ? page : P.n_pages, sl = slot;  // no page: outside the pool, read as zeros
            const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
            look(j + 1);
            if (lane < 4) {  // the mask of keys 32 lane ..: bit by bit of the boxes
                uint32_t w = 0;
                if (box >= 32) w = (there >> (32 * lane / box)) & 1u ? 0xffffffffu : 0u;
                else
                    for (int i = 0; i < 32 / box; i++)
                        if ((there >> (32 / box * lane + i)) & 1u) w |= ((1u << box) - 1u) << (i * box);
                s_in[j % TC_MASKS][lane] = w;
            }
            __syncwarp();
#pragma unroll
            for (int kv = 0; kv < 2; kv++) {
                const int n = 2 * (j - rg.ja) + kv;
                if (n >= NS) ok = warp_wait(&B.empty[n % NS], (uint32_t)(n / NS - 1) & 1u, &abort_flag);
                if (!ok) break;
                if (lane == 0) mbar_expect_tx(&B.full[n % NS], (uint32_t)Sh::TILE);
                __syncwarp();
                if (lane < nbox) {
#pragma unroll
                    for (int c = 0; c < HD / 64; c++)
                        tma_box(ring + (n % NS) * Sh::TILE + (uint32_t)(c * (TC_KEYS * 128) + lane * box * 128), kv ? &X.vmap : &X.kmap,
                                &B.full[n % NS], c * 64, sl, kvh, pg);
                }
                copied = n + 1;
            }
        }
        if (!ok) {  // let the copies in flight land
            int none = 0;
            for (int n = max(0, copied - NS); n < copied; n++) mbar_wait(&B.full[n % NS], (uint32_t)(n / NS) & 1u, &none);
        }
      } else if constexpr (!TMA) {
        // ================ the copies: groups lw, lw + 3, ... of eight keys, four lanes a key
        const int lw = warp - 17;
        constexpr int CPL = HD / 32;     // 16-byte chunks of a row per lane
        constexpr int NG = 6;            // groups of a warp: 6, 5 and 5 of the 16
        bool ok = true;
        int next = 0;                    // first tile not yet announced
        auto announce = [&](int upto) {  // tiles below `upto` have landed
            if (next >= upto) return;
            fence_async_shared();
            __syncwarp();
            for (; next < upto; next++)
                if (lane == 0) mbar_arrive(&B.full[next % NS]);
        };
        int page[NG], slot[NG];          // of key 8 (lw + 3 g) + lane / 4
        auto look = [&](int j) {
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const int p = rg.begin + j * TC_KEYS + (lw + 3 * g) * 8 + (lane >> 2);
                page[g] = -1;
                slot[g] = 0;
                if (lw + 3 * g < 16 && j < rg.jb && p < rg.end) page[g] = lookup(P, seq, p, slot[g]);
            }
        };
        look(rg.ja);
        for (int j = rg.ja; j < rg.jb && ok; j++) {
            int64_t ko[NG], vo[NG];      // element offsets of the keys, -1 for none
#pragma unroll
            for (int g = 0; g < NG; g++) {
                ko[g] = page[g] >= 0 ? page[g] * P.kps + kvh * P.khs + slot[g] * P.kss + (lane & 3) * 8 : -1;
                vo[g] = page[g] >= 0 ? page[g] * P.vps + kvh * P.vhs + slot[g] * P.vss + (lane & 3) * 8 : -1;
            }
            look(j + 1);
#pragma unroll
            for (int kv = 0; kv < 2; kv++) {
                const int n = 2 * (j - rg.ja) + kv;
                if (n >= NS) {
                    const uint32_t par = (uint32_t)(n / NS - 1) & 1u;
                    if (!__all_sync(0xffffffffu, mbar_test_wait(&B.empty[n % NS], par))) {
                        cp_wait<0>();  // no room for a copy yet: announce what has landed
                        announce(n);
                        ok = warp_wait(&B.empty[n % NS], par, &abort_flag);
                    }
                    if (!ok) break;
                }
                const uint32_t dst = ring + (n % NS) * Sh::TILE + (uint32_t)(lw * 1024 + (lane >> 2) * 128 + (((lane & 3) ^ (lane >> 2)) << 4));
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    if (lw + 3 * g >= 16) break;
                    const int64_t off = kv ? vo[g] : ko[g];
                    const __half* src = (const __half*)(kv ? P.v : P.k) + off;
                    if (kv == 0) {
                        const uint32_t in = __ballot_sync(0xffffffffu, off >= 0);  // the lanes of a key agree
                        uint32_t byte = 0;
#pragma unroll
                        for (int i = 0; i < 8; i++) byte |= ((in >> (4 * i)) & 1u) << i;
                        if (lane == 0) reinterpret_cast<volatile uint8_t*>(s_in[j % TC_MASKS])[lw + 3 * g] = (uint8_t)byte;
                    }
#pragma unroll
                    for (int x = 0; x < CPL; x++) {
                        const bool in = off >= 0 && (lane & 3) * 8 + 32 * x < P.hd;
                        // chunk (lane % 4) + 4 x of the row: block x / 2, place ^ (row % 8)
                        cp16((dst ^ (uint32_t)((x & 1) << 6)) + (uint32_t)((x >> 1) * (TC_KEYS * 128) + g * 3072), in ? src + 32 * x : (const __half*)P.k, in);
                    }
                }
                cp_commit();
                cp_wait<1>();
                announce(n);
            }
        }
        cp_wait<0>();
        if (ok) announce(2 * (rg.jb - rg.ja));
      }
    }
    __syncthreads();
    if (warp == 16) {
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Joins the runs of a row tile, in their order.
template <typename QT>
__global__ void __launch_bounds__(256) k_paged_tc_join(const __grid_constant__ TcArgs X) {
    const PagedAttnArgs& A = X.a;
    const PagedArgs& P = A.p;
    int seq = 0, tile = 0;
    const bool any = tile_at(X, (int)blockIdx.x, seq, tile);  // (reads the batch before the wait, as k_paged_join does)
    pdl_wait();  // (every CTA waits: the next kernel on the stream begins when this grid has ended)
    if (!any) return;
    const int kvh = blockIdx.y, m0 = tile * TC_ROWS;
    int r0, r1;
    seq_rows(P, seq, r0, r1);
    const int mrows = (int)min((int64_t)TC_ROWS, (int64_t)(r1 - r0) * A.G - m0);
    const int hq = P.hd >> 2;
    const int64_t slot = ((int64_t)blockIdx.x * P.nkv + kvh) * X.nsplit;
    for (int x = blockIdx.z * 256 + threadIdx.x; x < mrows * hq; x += 256 * gridDim.z) {
        const int m = x / hq, d = (x - m * hq) * 4;
        float mx, l;
        float4 v;
        join_runs(X.nsplit, [&](int s) { return (slot + s) * TC_ROWS + m; }, X.po, X.pml, P.hd, d, mx, l, v);
        const int t = token_of(A, m0 + m), row = r0 + t, head = kvh * A.G + (m0 + m) - t * A.G;
        store_row4<QT>(A, row, head, d, l, v);
        if (A.lse && d == 0)
            A.lse[(int64_t)row * A.nh + head] = l == 0.0f ? -INFINITY : (mx + log2f(l)) / LOG2E;
    }
}

int64_t tc_tiles(const PagedAttnArgs& A) { return (int64_t)A.p.n_rows * A.G / TC_ROWS + A.p.n_seqs; }

// Runs per row tile: cut where the row tiles alone leave SMs idle, into runs of
// four key tiles at least and no more runs than SMs (128 rows of 32 heads over
// 16,384 keys: 64 us in nine runs, 286 in one; 8 sequences of 16 tokens over
// 4,096: 47 in two runs, 74 in one).
int tc_nsplit(const PagedAttnArgs& A, int max_q_len, int max_kv_len) {
    const int64_t pairs = paged_tiles(A, max_q_len, TC_ROWS) * A.p.nkv;
    const int64_t len = A.window > 0 ? std::min<int64_t>(max_kv_len, (int64_t)A.window + TC_ROWS) : max_kv_len;
    const int64_t units = (len + TC_KEYS - 1) / TC_KEYS;
    if (pairs * 2 > 148) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>(148 / pairs, units / 4));
}

template <typename QT, int HD, bool TMA>
int launch_tc_t(const TcArgs& X, cudaStream_t s) {
    using Sh = TcShape<HD, sizeof(QT) == 4>;
    HC_CUDA(cudaFuncSetAttribute(k_paged_tc<QT, HD, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM));
    const PagedArgs& P = X.a.p;
    const int64_t tiles = tc_tiles(X.a);
    HC_CHECK(tiles * X.nsplit * P.nkv <= 0x7fffffff, HC_ERR_INVALID, "paged attention: %d rows of %d heads", P.n_rows, X.a.nh);
    k_paged_tc<QT, HD, TMA><<<(unsigned)(tiles * X.nsplit * P.nkv), TC_THREADS, Sh::SMEM, s>>>(X);
    HC_LAUNCH_CHECK();
    if (X.nsplit > 1) {
        HC_TRY(launch_pdl(k_paged_tc_join<QT>, dim3((unsigned)tiles, P.nkv, 8), dim3(256), 0, s, X));
        HC_LAUNCH_CHECK();
    }
    return HC_OK;
}

// A pool's tensor map; a dimension of one entry may have any stride.
int pool_map(CUtensorMap* map, const PagedArgs& P, void* base, int64_t ps, int64_t hs, int64_t ss, int box) {
    const uint64_t dims[4] = {(uint64_t)P.hd, (uint64_t)P.page_size, (uint64_t)P.nkv, (uint64_t)P.n_pages};
    const uint64_t row = (uint64_t)((P.hd + 7) / 8 * 16);
    const uint64_t strides[3] = {P.page_size > 1 ? (uint64_t)ss * 2 : row, P.nkv > 1 ? (uint64_t)hs * 2 : row,
                                 P.n_pages > 1 ? (uint64_t)ps * 2 : row};
    return encode_4d(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, base, dims, strides, 64, (uint32_t)box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename QT, int HD>
int launch_tc_copy(TcArgs& X, cudaStream_t s) {
    const PagedArgs& P = X.a.p;
    X.box = 0;
    for (int b = 8; b <= TC_KEYS && P.page_size % b == 0; b *= 2) X.box = b;
    const int64_t widest = std::max({P.kps, P.khs, P.kss, P.vps, P.vhs, P.vss});
    if (X.box == 0 || widest >= (1ll << 38)) return launch_tc_t<QT, HD, false>(X, s);
    HC_TRY(pool_map(&X.kmap, P, P.k, P.kps, P.khs, P.kss, X.box));
    HC_TRY(pool_map(&X.vmap, P, P.v, P.vps, P.vhs, P.vss, X.box));
    return launch_tc_t<QT, HD, true>(X, s);
}

}  // namespace

// FP16 cache with 16-byte rows, head sizes the padded tiles hold, a positive
// scale (the maximum is taken before it is applied), row indexes of 31 bits.
bool paged_tc_ok(const PagedAttnArgs& A, int c16) {
    const PagedArgs& P = A.p;
    return c16 && P.hd <= 128 && P.hd % 8 == 0 && ((uintptr_t)P.k | (uintptr_t)P.v) % 16 == 0 &&
           (P.kps | P.khs | P.kss | P.vps | P.vhs | P.vss) % 8 == 0 && (int64_t)P.n_rows * A.G < (1 << 30);
}

size_t paged_tc_bytes(const PagedAttnArgs& A, int max_q_len, int max_kv_len) {
    const int n = tc_nsplit(A, max_q_len, max_kv_len);
    return n == 1 ? 0 : (size_t)tc_tiles(A) * A.p.nkv * n * TC_ROWS * ((size_t)A.p.hd * 4 + 8);
}

int launch_paged_tc(const PagedAttnArgs& A, int q16, int max_q_len, int max_kv_len, void* ws, cudaStream_t s) {
    TcArgs X;
    X.a = A;
    X.nsplit = tc_nsplit(A, max_q_len, max_kv_len);
    X.longest = paged_tiles(A, max_q_len, TC_ROWS) * A.p.nkv * X.nsplit <= 148 ? 0 : std::max(max_kv_len, 1);
    X.po = (float*)ws;
    X.pml = (float2*)((float*)ws + (size_t)tc_tiles(A) * A.p.nkv * X.nsplit * TC_ROWS * A.p.hd);
    if (q16) return A.p.hd <= 64 ? launch_tc_copy<__half, 64>(X, s) : launch_tc_copy<__half, 128>(X, s);
    return A.p.hd <= 64 ? launch_tc_copy<float, 64>(X, s) : launch_tc_copy<float, 128>(X, s);
}

}  // namespace hc
