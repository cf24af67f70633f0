// Attention over a paged FP16 cache for sequences with many rows (prompts,
// chunks): tcgen05 products, softmax in registers, accumulators in tensor
// memory.
//
// A CTA takes 256 packed (token, query head of the group) rows of one
// (sequence, KV head) as two halves of 128, and walks key tiles of 128:
//   S_h = Q_h K^T          tcgen05.mma, Q and K in shared memory (128 x 128 f32)
//   P_h = 2^(c S_h - m)    one thread per row, S read from tensor memory
//   O_h += P_h V           tcgen05.mma, P in tensor memory over S, V in shared memory
// While one half's threads work on their weights the tensor core works on
// the other half's products; S, P and O of both halves fill the 512 columns.
// The running maximum m moves only when a row's maximum passes it by more
// than 2^TAU (the weights are held times 2^BIAS and stay below 2^15, so that
// one of 2^-25 of the largest still has 11 bits): O is rescaled in tensor
// memory in the first tiles and rarely after them.
//
// f32 queries enter as q = 2^e (hi + lo), fp16 each, e the row's own, and their
// weights as hi + lo: twice the products, results to f32's precision.
//
// Warps: 0-3 and 4-7 the halves' rows (load Q, softmax, output; a row of S stays
// in registers, so these take most of the register file), 8 issues the
// products, 9 and 10 copy (11 is idle) K and V tiles by cp.async through the block table
// (any page size; 16-byte pieces, whose issue the tensor work hides, instead
// of tiled copies, which a page that ends inside a tile would cut).
#include "hc_paged.h"
#include "hc_tc.cuh"

namespace hc {

namespace {

constexpr int TC_HALF = 128, TC_ROWS = 256, TC_KEYS = 128;
constexpr int TC_THREADS = 384;
constexpr int REG_ROW = 208, REG_CTRL = 88;  // 256 x 208 + 128 x 88 = 384 x 168, what the launch holds
constexpr int TC_MASKS = 8;      // ring of the tiles' key bits
constexpr float TAU = 4.0f, BIAS = 11.0f;

struct TcArgs {
    PagedAttnArgs a;
    int nsplit;   // runs of key tiles per row tile
    float* po;    // [(tile * nkv + kvh) * nsplit + run][256][hd]
    float2* pml;  // [..][256] (maximum in log2 units, sum)
};

template <int HD, bool HILO>
struct TcShape {
    static constexpr int QH = TC_HALF * HD * 2 * (HILO ? 2 : 1);   // bytes of a half's queries: hi, lo
    static constexpr int TILE = TC_KEYS * HD * 2;
    static constexpr int NS = HD == 64 ? 6 : (HILO ? 3 : 5);       // key / value tiles in flight
    static constexpr int SMEM = 2 * QH + NS * TILE + 1024;
};

struct TcBarriers {
    uint64_t full[6], empty[6];
    uint64_t q_ready[2], s_full[2], p_ready[2], o_full[2], vote[2];
    uint64_t drain;
};

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

__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// The key tiles of a CTA: positions begin + 128 j for j in [ja, jb), of which
// half h is active in [ha[h], hb[h]).
struct TcRange {
    int begin, end;
    int ja, jb;
    int ha[2], hb[2];
};
__device__ __forceinline__ TcRange tc_range(const PagedAttnArgs& A, int first, int m0, int mtot, int run, int nsplit) {
    TcRange r;
    visible(A, first, m0, min(TC_ROWS, mtot - m0), r.begin, r.end);
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

template <typename QT, int HD>
__global__ void __launch_bounds__(TC_THREADS, 1) k_paged_tc(const __grid_constant__ TcArgs X) {
    constexpr bool HILO = sizeof(QT) == 4;
    using Sh = TcShape<HD, HILO>;
    constexpr int NS = Sh::NS, PL = HILO ? 2 : 1;
    constexpr int QPLANE = TC_HALF * HD * 2;
    const PagedAttnArgs& A = X.a;
    const PagedArgs& P = A.p;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ TcBarriers B;
    __shared__ uint32_t s_tmem;
    __shared__ int abort_flag, s_skip[2], s_bad[2];
    __shared__ int s_tile[3];
    __shared__ float s_cf[TC_ROWS];               // score factor of each row
    __shared__ uint32_t s_in[TC_MASKS][4];        // which keys of a tile exist
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t q_s = base, ring = base + 2 * Sh::QH;

    if (warp == 0) {
        int seq = 0, tile = 0;
        const int bound = gridDim.x / X.nsplit;
        // later tiles of a prompt see more keys: they go first
        const bool ok = find_tile(P, A.G, TC_ROWS, bound - 1 - (int)(blockIdx.x / X.nsplit), seq, tile);
        if (lane == 0) {
            s_tile[0] = ok;
            s_tile[1] = seq;
            s_tile[2] = tile;
        }
    }
    if (threadIdx.x == 32) {
        abort_flag = 0;
        s_bad[0] = s_bad[1] = 0;
        for (int i = 0; i < NS; i++) {
            mbar_init(&B.full[i], 64);
            mbar_init(&B.empty[i], 1);
        }
        for (int h = 0; h < 2; h++) {
            mbar_init(&B.q_ready[h], 128);
            mbar_init(&B.s_full[h], 1);
            mbar_init(&B.p_ready[h], 128);
            mbar_init(&B.o_full[h], 1);
            mbar_init(&B.vote[h], 128);
        }
        mbar_init(&B.drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (!s_tile[0]) return;  // the grid is an upper bound
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = s_tmem;
    const int run = blockIdx.x % X.nsplit, kvh = blockIdx.y;
    const int seq = s_tile[1], m0 = s_tile[2] * TC_ROWS;
    int r0, r1;
    seq_rows(P, seq, r0, r1);
    const int first = __ldg(P.kv_len + seq) - (r1 - r0);
    const int mtot = (int)min((int64_t)(r1 - r0) * A.G, (int64_t)m0 + TC_ROWS);  // rows up to this tile's end
    const TcRange rg = tc_range(A, first, m0, mtot, run, X.nsplit);

    if (warp < 8) {
        // ================ the halves: queries, weights, outputs
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REG_ROW));
        const int h = warp >> 2, r = (warp & 3) * 32 + lane;
        const int mh = m0 + h * TC_HALF, rows = min(max(mtot - mh, 0), TC_HALF);
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_col = tmem + lane_off + (uint32_t)(h * 128), o_col = tmem + lane_off + 256u + (uint32_t)(h * 128);
        const uint32_t qs = q_s + h * Sh::QH;
        bool ok = true;
        // ---- queries: whole rows per warp instruction, 16 bytes a lane
        if (rg.hb[h] > rg.ha[h]) {
            constexpr int EPL = HILO ? 4 : 8, LPR = HD / EPL, RPI = 32 / LPR, BATCH = 8;
            const int d = (lane % LPR) * EPL;
#pragma unroll 1
            for (int i0 = 0; i0 < 32 / RPI; i0 += BATCH) {
                uint4 v[BATCH];
#pragma unroll
                for (int i = 0; i < BATCH; i++) {
                    const int row = (warp & 3) * 32 + (i0 + i) * RPI + lane / LPR, m = mh + row;
                    v[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (row < rows && d < P.hd) {
                        const int t = m / A.G;
                        const QT* q = (const QT*)A.q + (int64_t)(r0 + t) * A.q_rs + (kvh * A.G + m - t * A.G) * A.q_hs + d;
                        if (A.qvec) {
                            v[i] = *reinterpret_cast<const uint4*>(q);
                        } else if constexpr (HILO) {
                            v[i] = make_uint4(__float_as_uint(q[0]), __float_as_uint(q[1]), __float_as_uint(q[2]), __float_as_uint(q[3]));
                        } else {
                            const unsigned short* u = reinterpret_cast<const unsigned short*>(q);
                            v[i] = make_uint4(u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16, u[4] | (uint32_t)u[5] << 16,
                                              u[6] | (uint32_t)u[7] << 16);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < BATCH; i++) {
                    const int row = (warp & 3) * 32 + (i0 + i) * RPI + lane / LPR;
                    const uint32_t dst = qs + (uint32_t)((d >> 6) * (TC_HALF * 128) + row * 128 + ((((d & 63) >> 3) ^ (row & 7)) << 4) + (d & 7) * 2);
                    float c = A.scale * LOG2E;
                    if constexpr (HILO) {
                        const float f[4] = {__uint_as_float(v[i].x), __uint_as_float(v[i].y), __uint_as_float(v[i].z), __uint_as_float(v[i].w)};
                        float mx = fmaxf(fmaxf(fabsf(f[0]), fabsf(f[1])), fmaxf(fabsf(f[2]), fabsf(f[3])));
#pragma unroll
                        for (int o = 1; o < LPR; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                        const int e = min(max((int)(__float_as_uint(mx) >> 23), 2), 252);
                        const float down = __uint_as_float((uint32_t)(254 - e) << 23);
                        c *= __uint_as_float((uint32_t)e << 23);
                        uint32_t hi[2], lo[2];
                        split2(f[0] * down, f[1] * down, hi[0], lo[0]);
                        split2(f[2] * down, f[3] * down, hi[1], lo[1]);
                        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(dst), "r"(hi[0]), "r"(hi[1]) : "memory");
                        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(dst + QPLANE), "r"(lo[0]), "r"(lo[1]) : "memory");
                    } else {
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v[i].x), "r"(v[i].y), "r"(v[i].z), "r"(v[i].w) : "memory");
                    }
                    if (lane % LPR == 0) s_cf[h * TC_HALF + row] = c;
                }
            }
            __syncwarp();
            fence_async_shared();
            mbar_arrive(&B.q_ready[h]);
        }
        const bool in = r < rows;
        const int pos = in ? first + (mh + r) / A.G : -1;
        const int lo_pos = A.window > 0 ? pos - A.window + 1 : 0;
        const int p_min = first + mh / A.G, l_max = A.window > 0 ? first + (mh + rows - 1) / A.G - A.window + 1 : 0;
        const bool one_token = rows > 0 && mh / A.G == (mh + rows - 1) / A.G;
        const float cf = in ? s_cf[h * TC_HALF + r] : 1.0f;
        float m = -INFINITY, l = 0.0f;  // running maximum (log2 units), sum of weights
        uint32_t done = 0, votes = 0;
        for (int j = rg.ha[h]; j < rg.hb[h] && ok; j++, done++) {
            ok = mbar_wait(&B.s_full[h], done & 1u, &abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tmem_fence_after();
            uint32_t sr[128];
#pragma unroll
            for (int c = 0; c < 4; c++) tmem_ld_x32(s_col + 32u * c, sr + 32 * c);
            tmem_wait_ld();
            const int k0 = rg.begin + j * TC_KEYS;
            const uint32_t* bits = s_in[j % TC_MASKS];
            const bool whole = k0 + TC_KEYS - 1 <= p_min && k0 >= l_max && (bits[0] & bits[1] & bits[2] & bits[3]) == 0xffffffffu;
            if (!whole) {
                const int hi_c = pos - k0, lo_c = lo_pos - k0;
#pragma unroll
                for (int c = 0; c < 128; c++)
                    if (c > hi_c || c < lo_c || !((bits[c >> 5] >> (c & 31)) & 1u)) sr[c] = 0xff800000u;
            }
            float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 128; c++) x[c & 3] = fmaxf(x[c & 3], __uint_as_float(sr[c]));
            const float nm = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * cf;
            const bool raise = nm > m + TAU || (m == -INFINITY && nm > m);
            if (__any_sync(0xffffffffu, raise)) {
                const float to = raise ? nm : m;
                const float f = to == m ? 1.0f : ex2(m - to);
                m = to;
                l *= f;
                if (done > 0) {
                    // the products of the tile before are complete: this tile's
                    // scores were committed after them
#pragma unroll
                    for (int c = 0; c < HD / 16; c++) {
                        uint32_t o[16];
                        tmem_ld_x16(o_col + 16u * c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_st_x16(o_col + 16u * c, o);
                    }
                }
            }
            const float nb = m == -INFINITY ? 0.0f : BIAS - m;
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < 128; c++) {
                const float p = ex2(fmaf(__uint_as_float(sr[c]), cf, nb));
                sum[c & 3] += p;
                sr[c] = __float_as_uint(p);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            // A key that some rows of the half see and others do not must not
            // reach the latter through 0 * v where v is not finite: such a tile
            // (rare) leaves the products to the row's thread, masked keys left out.
            bool skip = false;
            if (!whole && !one_token) {
                const int n = 2 * j + 1 - 2 * rg.ja, slot = n % NS;
                ok = mbar_wait(&B.full[slot], (uint32_t)(n / NS) & 1u, &abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const uint32_t vt = ring + slot * Sh::TILE;
                uint32_t bad = 0;
                for (int i = r; i < Sh::TILE / 16; i += TC_HALF) {
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
                if (skip) {
                    const int hi_c = pos - k0, lo_c = lo_pos - k0;
#pragma unroll 1
                    for (int c0 = 0; c0 < HD; c0 += 16) {
                        float o[16];
                        uint32_t u[16];
                        if (done > 0) {
                            tmem_ld_x16(o_col + c0, u);
                            tmem_wait_ld();
                        }
#pragma unroll
                        for (int i = 0; i < 16; i++) o[i] = done > 0 ? __uint_as_float(u[i]) : 0.0f;
#pragma unroll
                        for (int c = 0; c < 128; c++) {
                            if (c > hi_c || c < lo_c || !((bits[c >> 5] >> (c & 31)) & 1u)) continue;
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                const int d = c0 + i;
                                const float v = __half2float(lds_f16(vt + (d >> 6) * (TC_KEYS * 128) + c * 128 + ((((d & 63) >> 3) ^ (c & 7)) << 4) + (d & 7) * 2));
                                o[i] = fmaf(__uint_as_float(sr[c]), v, o[i]);
                            }
                        }
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 16; i++) u[i] = __float_as_uint(o[i]);
                        tmem_st_x16(o_col + c0, u);
                    }
                }
                if (r == 0) s_skip[h] = skip;
            } else if (r == 0) {
                s_skip[h] = 0;
            }
            // weights over the scores: hi in columns 0-63, lo in 64-127
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint32_t hi[16], lo[HILO ? 16 : 1];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float a = __uint_as_float(sr[32 * c + 2 * i]), b = __uint_as_float(sr[32 * c + 2 * i + 1]);
                    if constexpr (HILO) split2(a, b, hi[i], lo[i]);
                    else hi[i] = pack(a, b);
                }
                tmem_st_x16(s_col + 16u * c, hi);
                if constexpr (HILO) tmem_st_x16(s_col + 64u + 16u * c, lo);
            }
            tmem_wait_st();
            tmem_fence_before();
            mbar_arrive(&B.p_ready[h]);
        }
        // ---- outputs
        const bool any = rg.hb[h] > rg.ha[h];
        if (any && ok) {
            ok = mbar_wait(&B.o_full[h], 0, &abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            tmem_fence_after();
        }
        if (rows > 0) {
            const int t = (mh + r) / A.G, row = r0 + t, head = kvh * A.G + (mh + r) - t * A.G;
            if (!ok) l = __int_as_float(0x7fffffff);  // a wait ran out: the row is NaN, not a wrong number
            const int64_t slot = ((int64_t)(blockIdx.x / X.nsplit) * P.nkv + kvh) * X.nsplit + run;
            const int64_t pr = slot * TC_ROWS + h * TC_HALF + r;
#pragma unroll 1
            for (int c = 0; c < HD / 16; c++) {
                uint32_t o[16];
                if (any && ok) {
                    tmem_ld_x16(o_col + 16u * c, o);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i++) o[i] = 0u;
                }
                if (in && 16 * c < P.hd) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const int d = 16 * c + i;
                        const float4 v = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
                        if (d >= P.hd) break;
                        if (X.nsplit == 1) store_row4<QT>(A, row, head, d, l, v);
                        else *reinterpret_cast<float4*>(X.po + pr * P.hd + d) = v;
                    }
                }
            }
            if (in) {
                if (X.nsplit > 1) X.pml[pr] = make_float2(m == -INFINITY ? m : m - BIAS, l);
                else if (A.lse) A.lse[(int64_t)row * A.nh + head] = l == 0.0f ? -INFINITY : (m - BIAS + log2f(l)) / LOG2E;
            }
        }
        tmem_fence_before();
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REG_CTRL));
      if (warp == 8) {
        // ================ the products
        constexpr uint32_t idesc_s = make_idesc_mn(128, 128);
        constexpr uint32_t idesc_o = make_idesc_mn(128, HD) | (1u << 16);  // V is MN-major
        bool ok = true;
        uint32_t pdone[2] = {0, 0};
        for (int j = rg.ja; j <= rg.jb && ok; j++) {
            const int nk = 2 * (j - rg.ja), nv = nk - 1;  // ring places of K_j and V_(j-1)
            for (int h = 0; h < 2 && ok; h++) {
                const uint32_t s_t = tmem + (uint32_t)(h * 128), o_t = tmem + 256u + (uint32_t)(h * 128);
                if (j - 1 >= rg.ha[h] && j - 1 < rg.hb[h]) {  // O_h += P_h V_(j-1)
                    ok = warp_wait(&B.p_ready[h], pdone[h] & 1u, &abort_flag) &&
                         warp_wait(&B.full[nv % NS], (uint32_t)(nv / NS) & 1u, &abort_flag);
                    if (!ok) break;
                    tmem_fence_after();
                    const int skip = *(volatile int*)&s_skip[h];
                    const uint32_t vs = ring + (nv % NS) * Sh::TILE;
                    if (!skip && elect_one()) {
#pragma unroll
                        for (int p = PL - 1; p >= 0; p--)
#pragma unroll
                            for (int kk = 0; kk < TC_KEYS / 16; kk++)
                                mma_f16_ts(o_t, s_t + (uint32_t)(p * 64 + kk * 8), sw128_mn_desc(vs + kk * 2048), idesc_o,
                                           pdone[h] > 0 || kk > 0 || p < PL - 1);
                    }
                    __syncwarp();
                    pdone[h]++;
                }
                if (j >= rg.ha[h] && j < rg.hb[h]) {  // S_h = Q_h K_j^T
                    if (j == rg.ha[h]) ok = warp_wait(&B.q_ready[h], 0, &abort_flag);
                    ok = ok && warp_wait(&B.full[nk % NS], (uint32_t)(nk / NS) & 1u, &abort_flag);
                    if (!ok) break;
                    tmem_fence_after();
                    const uint32_t ks = ring + (nk % NS) * Sh::TILE, qs = q_s + h * Sh::QH;
                    if (elect_one()) {
#pragma unroll
                        for (int p = PL - 1; p >= 0; p--)
#pragma unroll
                            for (int kk = 0; kk < HD / 16; kk++) {
                                const uint32_t off = (uint32_t)((kk >> 2) * (128 * 128) + (kk & 3) * 32);
                                mma_f16_ss(s_t, sw128_desc(qs + p * QPLANE + off), sw128_desc(ks + off), idesc_s, kk > 0 || p < PL - 1);
                            }
                        mma_commit(&B.s_full[h]);
                    }
                    __syncwarp();
                }
                if (j == rg.hb[h] && rg.hb[h] > rg.ha[h]) {
                    if (elect_one()) mma_commit(&B.o_full[h]);
                    __syncwarp();
                }
            }
            if (!ok) break;
            if (elect_one()) {
                if (j > rg.ja) mma_commit(&B.empty[nv % NS]);
                if (j < rg.jb) mma_commit(&B.empty[nk % NS]);
            }
            __syncwarp();
        }
        if (!ok) {  // let what is in flight end before tensor memory is given back
            if (elect_one()) mma_commit(&B.drain);
            __syncwarp();
            int none = 0;
            mbar_wait(&B.drain, 0, &none);
        }
        tmem_fence_before();
      } else if (warp < 11) {
        // ================ the copies: warp lw takes keys 64 lw .. 64 lw + 63 of each tile
        const int lw = warp - 9;
        constexpr int CPL = HD / 32;  // 16-byte chunks of a row per lane (four lanes copy a row)
        bool ok = true;
        int waiting = -1;             // tile copied but not yet announced
        auto announce = [&]() {
            if (waiting >= 0) {
                fence_async_shared();
                mbar_arrive(&B.full[waiting % NS]);
            }
            waiting = -1;
        };
        int page[2], slot[2];
        auto look = [&](int j) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int p = rg.begin + j * TC_KEYS + lw * 64 + i * 32 + lane;
                page[i] = -1;
                slot[i] = 0;
                if (j < rg.jb && p < rg.end) page[i] = lookup(P, seq, p, slot[i]);
            }
        };
        look(rg.ja);
        for (int j = rg.ja; j < rg.jb && ok; j++) {
            int64_t ko[2], vo[2];
            uint32_t in[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                in[i] = __ballot_sync(0xffffffffu, page[i] >= 0);
                ko[i] = page[i] >= 0 ? page[i] * P.kps + kvh * P.khs + slot[i] * P.kss : 0;
                vo[i] = page[i] >= 0 ? page[i] * P.vps + kvh * P.vhs + slot[i] * P.vss : 0;
            }
            look(j + 1);
            for (int kv = 0; kv < 2 && ok; kv++) {
                const int n = 2 * (j - rg.ja) + kv;
                if (n >= NS) {
                    const uint32_t par = (uint32_t)(n / NS - 1) & 1u;
                    if (!mbar_test_wait(&B.empty[n % NS], par)) {
                        cp_wait<0>();  // nothing to copy yet: announce what has landed
                        announce();
                        ok = mbar_wait(&B.empty[n % NS], par, &abort_flag);
                    }
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                }
                if (kv == 0 && lane < 2) s_in[j % TC_MASKS][lw * 2 + lane] = lane ? in[1] : in[0];
                const __half* src = (const __half*)(kv ? P.v : P.k) + (lane & 3) * 8;
                const uint32_t dst = ring + (n % NS) * Sh::TILE + (uint32_t)((lw * 64 + (lane >> 2)) * 128);
#pragma unroll
                for (int g = 0; g < 8; g++) {  // rows 8 g + lane / 4
                    const int row = (g * 8 + (lane >> 2)) & 31;
                    const int64_t off = __shfl_sync(0xffffffffu, kv ? vo[g >> 2] : ko[g >> 2], row);
                    const bool row_in = (in[g >> 2] >> row) & 1u;
#pragma unroll
                    for (int x = 0; x < CPL; x++) {
                        const int c = (lane & 3) + 4 * x;
                        const bool ok_c = row_in && c * 8 < P.hd;
                        cp16(dst + (uint32_t)((c >> 3) * (TC_KEYS * 128) + g * 1024 + (((c & 7) ^ (lane >> 2)) << 4)),
                             ok_c ? src + off + 32 * x : (const __half*)P.k, ok_c);
                    }
                }
                cp_commit();
                if (waiting >= 0) {
                    cp_wait<1>();
                    announce();
                }
                waiting = n;
            }
        }
        cp_wait<0>();
        if (ok) announce();
      }
    }
    __syncthreads();
    if (warp == 8) {
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Joins the runs of a row tile, in their order.
template <typename QT>
__global__ void __launch_bounds__(256) k_paged_tc_join(const __grid_constant__ TcArgs X) {
    const PagedAttnArgs& A = X.a;
    const PagedArgs& P = A.p;
    pdl_wait();
    int seq = 0, tile = 0;
    if (!find_tile(P, A.G, TC_ROWS, gridDim.x - 1 - blockIdx.x, seq, tile)) return;
    const int kvh = blockIdx.y, m0 = tile * TC_ROWS;
    int r0, r1;
    seq_rows(P, seq, r0, r1);
    const int mrows = (int)min((int64_t)TC_ROWS, (int64_t)(r1 - r0) * A.G - m0);
    const int hq = P.hd >> 2;
    const int64_t slot = ((int64_t)blockIdx.x * P.nkv + kvh) * X.nsplit;
    for (int x = blockIdx.z * 256 + threadIdx.x; x < mrows * hq; x += 256 * gridDim.z) {
        const int m = x / hq, d = (x - m * hq) * 4;
        float mx = -INFINITY;
        for (int s = 0; s < X.nsplit; s++) mx = fmaxf(mx, X.pml[(slot + s) * TC_ROWS + m].x);
        float l = 0.0f;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int s = 0; s < X.nsplit; s++) {
            const float2 ml = X.pml[(slot + s) * TC_ROWS + m];
            const float4 y = *reinterpret_cast<const float4*>(X.po + ((slot + s) * TC_ROWS + m) * P.hd + d);
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

int64_t tc_tiles(const PagedAttnArgs& A) { return (int64_t)A.p.n_rows * A.G / TC_ROWS + A.p.n_seqs; }

// Runs per row tile: cut where the row tiles alone leave SMs idle, into runs
// of four key tiles at least.
int tc_nsplit(const PagedAttnArgs& A, int max_kv_len) {
    const int64_t pairs = ((int64_t)A.p.n_rows * A.G + TC_ROWS - 1) / TC_ROWS * A.p.nkv;
    const int64_t len = A.window > 0 ? std::min<int64_t>(max_kv_len, (int64_t)A.window + TC_ROWS) : max_kv_len;
    const int64_t units = (len + TC_KEYS - 1) / TC_KEYS;
    if (pairs * 2 > 148) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>(148 / pairs, units / 4));
}

template <typename QT, int HD>
int launch_tc_t(const TcArgs& X, cudaStream_t s) {
    using Sh = TcShape<HD, sizeof(QT) == 4>;
    HC_CUDA(cudaFuncSetAttribute(k_paged_tc<QT, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM));
    const PagedArgs& P = X.a.p;
    const int64_t tiles = tc_tiles(X.a);
    HC_CHECK(tiles * X.nsplit <= 0x7fffffff, HC_ERR_INVALID, "paged attention: %d rows of %d heads", P.n_rows, X.a.nh);
    k_paged_tc<QT, HD><<<dim3((unsigned)(tiles * X.nsplit), P.nkv), TC_THREADS, Sh::SMEM, s>>>(X);
    HC_LAUNCH_CHECK();
    if (X.nsplit > 1) {
        k_paged_tc_join<QT><<<dim3((unsigned)tiles, P.nkv, 8), 256, 0, s>>>(X);
        HC_LAUNCH_CHECK();
    }
    return HC_OK;
}

}  // namespace

// FP16 cache with 16-byte rows, head sizes the padded tiles hold, a positive
// scale (the maximum is taken before it is applied), rows that fit 32 bits.
bool paged_tc_ok(const PagedAttnArgs& A, int c16) {
    const PagedArgs& P = A.p;
    return c16 && P.hd <= 128 && P.hd % 8 == 0 && ((uintptr_t)P.k | (uintptr_t)P.v) % 16 == 0 &&
           (P.kps | P.khs | P.kss | P.vps | P.vhs | P.vss) % 8 == 0 && (int64_t)P.n_rows * A.G < (1 << 30);
}

size_t paged_tc_bytes(const PagedAttnArgs& A, int max_kv_len) {
    const int n = tc_nsplit(A, max_kv_len);
    return n == 1 ? 0 : (size_t)tc_tiles(A) * A.p.nkv * n * TC_ROWS * ((size_t)A.p.hd * 4 + 8);
}

int launch_paged_tc(const PagedAttnArgs& A, int q16, int max_kv_len, void* ws, cudaStream_t s) {
    TcArgs X;
    X.a = A;
    X.nsplit = tc_nsplit(A, max_kv_len);
    X.po = (float*)ws;
    X.pml = (float2*)((float*)ws + (size_t)tc_tiles(A) * A.p.nkv * X.nsplit * TC_ROWS * A.p.hd);
    if (q16) return A.p.hd <= 64 ? launch_tc_t<__half, 64>(X, s) : launch_tc_t<__half, 128>(X, s);
    return A.p.hd <= 64 ? launch_tc_t<float, 64>(X, s) : launch_tc_t<float, 128>(X, s);
}

}  // namespace hc
