// Bounds of the keys of a paged cache's pages, and the pages that a row's queries
// are to read by them.
#include "hc_paged.h"

#include <type_traits>

namespace hc {

namespace {

struct Bounds {
    int8_t* lo;
    int8_t* hi;
    float* scale;
};

// Biased exponent of the least power of two, from 2^-120 on, of which the
// magnitude with these bits (finite) is at most 127: 127 = 1.984375 x 64.
__device__ __forceinline__ int unit_exponent(uint32_t top) {
    return max((int)(top >> 23) - 6 + ((top & 0x7FFFFFu) > 0x7E0000u), 7);
}
__device__ __forceinline__ float power(int biased) { return __uint_as_float((uint32_t)biased << 23); }

// Four elements of a key as floats.
template <typename CT, bool VEC>
__device__ __forceinline__ void key4(const PagedArgs& P, const PagedScales& C, int page, int head, int slot, int d, float* x) {
    const int64_t at = page * P.kps + head * P.khs + slot * P.kss;
    if constexpr (std::is_same<CT, q4x>::value) {
        const uint32_t w = __ldg(reinterpret_cast<const unsigned short*>((const uint8_t*)P.k + at + (d >> 1)));
        const float s = __half2float(C.k[page * C.kps + head * C.khs + slot * C.kss + (d >> 5)]);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = (float)((int)(w >> (4 * i) & 15) - 8) * s;
    } else {
        const CT* p = (const CT*)P.k + at + d;
        if constexpr (VEC && sizeof(CT) == 4) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(p));
            x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
        } else if constexpr (VEC) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
            x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = to_f32(p[i]);
        }
    }
}

// Bounds.  Read from the keys that are stored, so that they hold whatever the cache
// rounds.  Bound by latency (places, page, keys, one after another): 4 prompts of
// 2,048 positions, 8 heads of 128, pages of 16, FP16: 12 us, 1.8 TB/s (17 us with a CTA
// and shared memory a page).
// A warp takes one page and KV head at a time, four elements of a key a lane: heads
// of up to 64 elements two or more keys at once, of more than 128 in two rounds.  Its
// loads do not depend on one another, so a page's keys are requested together.
constexpr int BD_WARPS = 4;

template <typename CT, bool VEC>
__global__ void __launch_bounds__(32 * BD_WARPS) k_page_bounds(PagedArgs P, PagedScales C, Bounds B) {
    const int b = blockIdx.z, lane = threadIdx.x & 31;
    int r0, r1;
    seq_rows(P, b, r0, r1);
    const int n = min(seq_len(P, b), P.reach);
    const int begin = max(seq_len(P, b) - (r1 - r0), 0);
    if (r1 == r0 || begin >= n) return;
    const int i0 = page_of(P, begin), i1 = page_of(P, n - 1);
    const int hq = P.hd >> 2, across = min(hq, 32), rows = 32 / across, q = lane % across, r = lane / across;
    const int head = blockIdx.y;
    for (int i = i0 + blockIdx.x * BD_WARPS + (threadIdx.x >> 5); i <= i1; i += gridDim.x * BD_WARPS) {
        int slot;
        const int page = lookup(P, b, i * P.page_size, slot);
        if (page < 0) continue;
        const int filled = min(P.page_size, n - i * P.page_size);
        float lo[2][4], hi[2][4];
        uint32_t top = 0;
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int k = 0; k < 4; k++) lo[h][k] = INFINITY, hi[h][k] = -INFINITY;
            if (q + 32 * h >= hq || (h && across < 32)) continue;
            if (r < rows) {
#pragma unroll 8
                for (int s = r; s < filled; s += rows) {
                    float x[4];
                    key4<CT, VEC>(P, C, page, head, s, 4 * (q + 32 * h), x);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        lo[h][k] = fminf(lo[h][k], x[k]);
                        hi[h][k] = fmaxf(hi[h][k], x[k]);
                        top = max(top, __float_as_uint(x[k]) & 0x7FFFFFFFu);
                    }
                }
            }
        }
        __syncwarp();
        for (int x = 1; x < rows; x++) {  // the other lanes of the same elements
            const int from = (lane % across) + x * across;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float l = __shfl_sync(0xffffffffu, lo[0][k], from), h = __shfl_sync(0xffffffffu, hi[0][k], from);
                if (r == 0) lo[0][k] = fminf(lo[0][k], l), hi[0][k] = fmaxf(hi[0][k], h);
            }
        }
        top = __reduce_max_sync(0xffffffffu, top);
        const bool fine = top < 0x7F800000u;
        const int e = fine ? unit_exponent(top) : 255;
        const float inv = fine ? power(254 - e) : 0.0f;
        const int64_t at = (int64_t)page * P.nkv + head;
        if (lane == 0) B.scale[at] = power(e);  // 255: infinity
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if (r != 0 || q + 32 * h >= hq || (h && across < 32)) continue;
            uint32_t lw = 0, hw = 0;
            if (fine) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    lw |= (uint32_t)((int)floorf(lo[h][k] * inv) & 255) << (8 * k);
                    hw |= (uint32_t)((int)ceilf(hi[h][k] * inv) & 255) << (8 * k);
                }
            }
            reinterpret_cast<uint32_t*>(B.lo + at * P.hd)[q + 32 * h] = lw;
            reinterpret_cast<uint32_t*>(B.hi + at * P.hd)[q + 32 * h] = hw;
        }
    }
}

__global__ void __launch_bounds__(256) k_bounds_values(Bounds B, int hd, int64_t quads, float* lo, float* hi) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= quads) return;
    const float s = B.scale[i * 4 / hd];
    const uint32_t l = reinterpret_cast<const uint32_t*>(B.lo)[i], h = reinterpret_cast<const uint32_t*>(B.hi)[i];
    float4 a, b;
    a.x = (float)(int8_t)l * s, a.y = (float)(int8_t)(l >> 8) * s, a.z = (float)(int8_t)(l >> 16) * s, a.w = (float)(int8_t)(l >> 24) * s;
    b.x = (float)(int8_t)h * s, b.y = (float)(int8_t)(h >> 8) * s, b.z = (float)(int8_t)(h >> 16) * s, b.w = (float)(int8_t)(h >> 24) * s;
    reinterpret_cast<float4*>(lo)[i] = a;
    reinterpret_cast<float4*>(hi)[i] = b;
}

// ============================================================ selection

struct SelectArgs {
    PagedArgs p;  // the batch, page size and heads; no pool
    Bounds b;
    const void* q;
    int64_t q_rs, q_hs;
    int G, qvec;  // query heads a KV head; four elements of a query lie on 16 (f16: 8) bytes
    int budget, first, recent;
    int32_t* out;
    uint32_t* keys;  // [row][KV head][max_pages], score_key()
};

// Position of packed row `row` and its sequence (false: it belongs to none).
__device__ __forceinline__ bool place_of(const PagedArgs& P, int row, int& seq, int& pos) {
    int lo = 0, hi = P.n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (__ldg(P.q_start + mid) <= row) lo = mid;
        else hi = mid - 1;
    }
    int r0, r1;
    seq_rows(P, lo, r0, r1);
    seq = lo;
    pos = seq_len(P, lo) - (r1 - r0) + (row - r0);
    return row >= r0 && row < r1;
}

// Scores: four lanes a page, 16 bytes of its bounds each in turn; eight query heads
// at a time, their codes in shared memory as two vectors, what is above zero (it
// meets hi) and what is below (it meets lo).  A sum of products of bytes is
// exact (below 2^22), and is held with the two powers of two as a whole number of
// the scores' order: 9 bits of exponent, 21 below the leading one, so that no score
// overflows, underflows or is rounded.
constexpr uint32_t KEY_ZERO = 0x80000000u, KEY_HOLE = 1u, KEY_INF = 0xfffffffeu, KEY_KEPT = 0xffffffffu;

// sum 2^(et - 127) 2^(es - 127), et and es from 7 to 249, et = 0: zero.
__device__ __forceinline__ uint32_t score_key(int sum, int et, int es) {
    if (sum == 0 || et == 0) return KEY_ZERO;
    const uint32_t b = __float_as_uint((float)abs(sum));
    const uint32_t m = ((b >> 23) - 127 + et + es - 13) << 21 | (b & 0x7FFFFFu) >> 2;
    return sum < 0 ? KEY_ZERO - m : KEY_ZERO + m;
}

constexpr int SC_THREADS = 128, SC_PAGES = SC_THREADS / 4, SC_HEADS = 8;

template <typename T>
__global__ void __launch_bounds__(SC_THREADS) k_page_scores(const __grid_constant__ SelectArgs A) {
    const PagedArgs& P = A.p;
    extern __shared__ __align__(16) uint8_t sm[];
    const int hd = P.hd, G = A.G, stride = (hd + 15) / 16 * 16;
    uint8_t* qp = sm;                       // [G][stride]
    uint8_t* qn = sm + (size_t)G * stride;  // [G][stride]
    int* unit = reinterpret_cast<int*>(sm + 2 * (size_t)G * stride);  // exponents of t, 0: not finite
    const int kvh = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_trigger();
    for (int row = blockIdx.z; row < P.n_rows; row += gridDim.z) {
        int seq, pos;
        if (!place_of(P, row, seq, pos)) continue;
        const int n = pages_seen(P, pos);
        if (n <= A.budget || blockIdx.x * SC_PAGES >= n) continue;  // all of them, or none here
        __syncthreads();
        for (int g = warp; g < G; g += SC_THREADS / 32) {
            const T* q = (const T*)A.q + row * A.q_rs + (kvh * G + g) * A.q_hs;
            uint32_t top = 0;
            for (int d = lane; d < hd; d += 32) top = max(top, __float_as_uint(to_f32(q[d])) & 0x7FFFFFFFu);
            top = __reduce_max_sync(0xffffffffu, top);
            const bool fine = top < 0x7F800000u;
            const int e = fine ? unit_exponent(top) : 0;
            const float inv = fine ? power(254 - e) : 0.0f;
            for (int d = lane; d < stride; d += 32) {
                const int c = fine && d < hd ? __float2int_rn(to_f32(q[d]) * inv) : 0;
                qp[g * stride + d] = (uint8_t)max(c, 0);
                qn[g * stride + d] = (uint8_t)min(c, 0);
            }
            if (lane == 0) unit[g] = e;
        }
        __syncthreads();
        uint32_t* keys = A.keys + ((int64_t)row * P.nkv + kvh) * P.max_pages;
        const int sub = threadIdx.x & 3;
        for (int i0 = blockIdx.x * SC_PAGES; i0 < n; i0 += gridDim.x * SC_PAGES) {
            const int i = i0 + (threadIdx.x >> 2);
            int slot, page = -1;
            if (i < n) page = lookup(P, seq, i * P.page_size, slot);
            const int64_t at = ((int64_t)max(page, 0) * P.nkv + kvh) * hd;
            uint32_t best = 0;
            const uint32_t scale = page < 0 ? 0 : __float_as_uint(__ldg(A.b.scale + (int64_t)page * P.nkv + kvh)) >> 23;
            const int es = min(max((int)scale, 7), 249);
            for (int g0 = 0; g0 < G; g0 += SC_HEADS) {
                int acc[SC_HEADS];
#pragma unroll
                for (int g = 0; g < SC_HEADS; g++) acc[g] = 0;
                if (page >= 0) {
                    if (hd % 16 == 0) {
                        for (int x = sub; x < hd / 16; x += 4) {
                            const int4 h = __ldg(reinterpret_cast<const int4*>(A.b.hi + at) + x), l = __ldg(reinterpret_cast<const int4*>(A.b.lo + at) + x);
#pragma unroll
                            for (int g = 0; g < SC_HEADS; g++) {
                                if (g0 + g >= G) break;
                                const int4 p = reinterpret_cast<const int4*>(qp + (g0 + g) * stride)[x], m = reinterpret_cast<const int4*>(qn + (g0 + g) * stride)[x];
                                acc[g] = __dp4a(h.x, p.x, __dp4a(h.y, p.y, __dp4a(h.z, p.z, __dp4a(h.w, p.w, acc[g]))));
                                acc[g] = __dp4a(l.x, m.x, __dp4a(l.y, m.y, __dp4a(l.z, m.z, __dp4a(l.w, m.w, acc[g]))));
                            }
                        }
                    } else {
                        for (int x = sub; x < hd / 4; x += 4) {
                            const int h = __ldg(reinterpret_cast<const int*>(A.b.hi + at) + x), l = __ldg(reinterpret_cast<const int*>(A.b.lo + at) + x);
#pragma unroll
                            for (int g = 0; g < SC_HEADS; g++) {
                                if (g0 + g >= G) break;
                                acc[g] = __dp4a(h, reinterpret_cast<const int*>(qp + (g0 + g) * stride)[x], acc[g]);
                                acc[g] = __dp4a(l, reinterpret_cast<const int*>(qn + (g0 + g) * stride)[x], acc[g]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int g = 0; g < SC_HEADS; g++) {
                    acc[g] += __shfl_xor_sync(0xffffffffu, acc[g], 1);
                    acc[g] += __shfl_xor_sync(0xffffffffu, acc[g], 2);
                    if (g0 + g < G) best = max(best, score_key(acc[g], unit[g0 + g], es));
                }
            }
            if (sub == 0 && i < n) {
                uint32_t key = KEY_KEPT;  // whatever it scores
                if (i >= A.first && i < n - A.recent) key = page < 0 ? KEY_HOLE : scale == 255 ? KEY_INF : best;
                keys[i] = key;
            }
        }
    }
}

// The pages of one row and KV head from their keys: the least key that is taken, by
// histograms of 2,048 equal steps of the range that still holds it (so that the
// keys of a row, which lie close together, spread over them: the shared counters
// of equal digits would be added to one by one), then what is above it and, of what
// equals it, the first by index.  A thread's keys are a run, so that one scan over
// the threads places them all.
constexpr int PK_THREADS = 256, PK_BINS = 2048;

struct PickShared {
    int hist[PK_BINS], sum[2][PK_THREADS / 32];
    uint32_t least[PK_THREADS / 32], most[PK_THREADS / 32];
    int bin, left, held;
};

__device__ __forceinline__ void pick_pages(const uint32_t* keys, int n, int budget, int first, int recent, int32_t* out, PickShared& S) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int begin = first, end = n - recent;  // the ones whose score counts (n > budget >= first + recent)
    int left = budget - first - recent;         // and how many of them are taken
    uint32_t least = 0xffffffffu, most = 0;
    for (int i = begin + tid; i < end; i += PK_THREADS) {
        const uint32_t k = keys[i];
        least = min(least, k);
        most = max(most, k);
    }
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) S.least[warp] = least, S.most[warp] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PK_THREADS / 32; w++) least = min(least, S.least[w]), most = max(most, S.most[w]);
    uint32_t lo = least, hi = most, above = 0xffffffffu;  // the range; taken: keys above `above`, and the first `left` that equal it
    int shift = max(32 - __clz(most - least) - 11, 0);
    while (left > 0) {
        for (int i = tid; i < PK_BINS; i += PK_THREADS) S.hist[i] = 0;
        __syncthreads();
        for (int i = begin + tid; i < end; i += PK_THREADS) {
            const uint32_t k = keys[i];
            if (k >= lo && k <= hi) atomicAdd(&S.hist[(k - lo) >> shift], 1);
        }
        __syncthreads();
        // eight bins a thread, from the top
        int c[PK_BINS / PK_THREADS], own = 0;
#pragma unroll
        for (int i = 0; i < PK_BINS / PK_THREADS; i++) own += c[i] = S.hist[PK_BINS - 1 - (tid * (PK_BINS / PK_THREADS) + i)];
        int incl = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        if (lane == 31) S.sum[0][warp] = incl;
        __syncthreads();
        for (int w = 0; w < warp; w++) incl += S.sum[0][w];
        int before = incl - own;
        if (before < left && incl >= left) {
#pragma unroll
            for (int i = 0; i < PK_BINS / PK_THREADS; i++) {
                if (before < left && before + c[i] >= left) {
                    S.bin = PK_BINS - 1 - (tid * (PK_BINS / PK_THREADS) + i);
                    S.left = left - before;
                    S.held = c[i];
                }
                before += c[i];
            }
        }
        __syncthreads();
        lo += (uint32_t)S.bin << shift;
        hi = lo + min(hi - lo, (1u << shift) - 1);  // (lo + a step may pass 32 bits: KEY_INF lies there)
        left = S.left;
        const int held = S.held;
        __syncthreads();
        if (shift == 0 || held == left) {  // one key's step, or all of the step is taken (a key is above 0)
            above = held == left ? lo - 1 : lo;
            if (held == left) left = 0;
            break;
        }
        shift = max(shift - 11, 0);
    }
    // (the last step's upper end needs no mark: what lies above it is above `above`)
    const int run = ((n + PK_THREADS - 1) / PK_THREADS) | 1, i0 = min(tid * run, n), i1 = min(i0 + run, n);
    int more = 0, equal = 0;
    for (int i = i0; i < i1; i++) {
        const uint32_t k = keys[i];
        const bool kept = i < begin || i >= end;
        more += kept || k > above;
        equal += !kept && k == above;
    }
    int a = more, e = equal;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, e, o);
        if (lane >= o) a += x, e += y;
    }
    if (lane == 31) S.sum[0][warp] = a, S.sum[1][warp] = e;
    __syncthreads();
    for (int w = 0; w < warp; w++) a += S.sum[0][w], e += S.sum[1][w];
    a -= more;
    e -= equal;
    int at = a + min(e, left);
    for (int i = i0; i < i1; i++) {
        const uint32_t k = keys[i];
        const bool kept = i < begin || i >= end;
        if ((kept || k > above || (k == above && e++ < left)) && at < budget) out[at++] = i;
    }
}

__global__ void __launch_bounds__(PK_THREADS) k_page_pick(const __grid_constant__ SelectArgs A) {
    const PagedArgs& P = A.p;
    __shared__ PickShared S;
    const int row = blockIdx.x, kvh = blockIdx.y;
    int seq, pos;
    const bool any = place_of(P, row, seq, pos);
    const int n = any ? pages_seen(P, pos) : 0;
    pdl_wait();
    if (!any) return;
    int32_t* out = A.out + ((int64_t)row * P.nkv + kvh) * A.budget;
    if (n <= A.budget) {
        for (int i = threadIdx.x; i < A.budget; i += PK_THREADS) out[i] = i < n ? i : -1;
        return;
    }
    pick_pages(A.keys + ((int64_t)row * P.nkv + kvh) * P.max_pages, n, A.budget, A.first, A.recent, out, S);
}

// ---- both in one: a cluster of CTAs scores a row and KV head's pages, each a share
// of them, into the first one's shared memory, which picks.  One launch and no
// workspace.  Bound by steps that follow one another: a cluster's start, the row's place, the
// queries, the bounds, and the pick, which the first CTA does alone.  Scores by mma.sync on bytes, 16 pages a warp
// against eight heads (the order of a head's elements is free, so a lane's operands
// are its 16-byte pieces of a page's bounds): by dp4a, 8 rows of 64 heads over 2,048
// pages took 17,000 to 27,000 cycles for the scores of a CTA's 256 pages, now 9,000.
// That call: 19.5 us with the host's part (two kernels 28.7), of a cluster's 22,000
// cycles some 3,000 for the queries and 8,000 for the pick.
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}

// Products of bytes, exact: 16 pages x 32 elements by 32 x 8 query heads.
__device__ __forceinline__ void mma_s8(int* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four elements of a query row from d on.
template <typename T>
__device__ __forceinline__ void query4(const T* q, int vec, float* x) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(q));
            x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
        } else {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(q));
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
            x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = to_f32(q[i]);
    }
}

// NX: 16-byte pieces of a head's bounds a lane (heads of 64 NX elements at most).
template <typename T, int NX>
__global__ void __launch_bounds__(PK_THREADS) k_page_select(const __grid_constant__ SelectArgs A) {
    const PagedArgs& P = A.p;
    extern __shared__ __align__(16) uint8_t sm[];
    __shared__ PickShared S;
    constexpr int STRIDE = 64 * NX;
    const int hd = P.hd, G = A.G;
    uint8_t* qp = sm;                       // [G][STRIDE]: codes above zero
    uint8_t* qn = sm + (size_t)G * STRIDE;  // and below
    int* unit = reinterpret_cast<int*>(sm + 2 * (size_t)G * STRIDE);
    uint32_t* keys = reinterpret_cast<uint32_t*>(unit + (G + 3) / 4 * 4);
    uint32_t rank, ctas, first_keys;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ctas));
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(first_keys) : "r"(smem_u32(keys)));
    const int row = blockIdx.z, kvh = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int seq = 0, pos = -1;
    const bool any = place_of(P, row, seq, pos);
    const int n = any ? pages_seen(P, pos) : 0;
    const bool score = any && n > A.budget;
    const int share = ((n + (int)ctas - 1) / (int)ctas + 63) / 64 * 64, p0 = min((int)rank * share, n), p1 = min(p0 + share, n);
    const int c = lane & 3;
    if (score && p0 < p1) {
        for (int g = warp; g < G; g += PK_THREADS / 32) {
            const T* q = (const T*)A.q + row * A.q_rs + (kvh * G + g) * A.q_hs;
            float x[(NX + 1) / 2][4];
            uint32_t top = 0;
#pragma unroll
            for (int h = 0; h < (NX + 1) / 2; h++) {
                const int d = 4 * lane + 128 * h;
#pragma unroll
                for (int i = 0; i < 4; i++) x[h][i] = 0.0f;
                if (d < hd) query4(q + d, A.qvec, x[h]);
#pragma unroll
                for (int i = 0; i < 4; i++) top = max(top, __float_as_uint(x[h][i]) & 0x7FFFFFFFu);
            }
            top = __reduce_max_sync(0xffffffffu, top);
            const bool fine = top < 0x7F800000u;
            const int e = fine ? unit_exponent(top) : 0;
            const float inv = fine ? power(254 - e) : 0.0f;
#pragma unroll
            for (int h = 0; h < (NX + 1) / 2; h++) {
                const int d = 4 * lane + 128 * h;
                uint32_t up = 0, down = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int c = fine ? __float2int_rn(x[h][i] * inv) : 0;
                    up |= (uint32_t)max(c, 0) << (8 * i);
                    down |= (uint32_t)(min(c, 0) & 255) << (8 * i);
                }
                if (d < STRIDE) {
                    *reinterpret_cast<uint32_t*>(qp + g * STRIDE + d) = up;
                    *reinterpret_cast<uint32_t*>(qn + g * STRIDE + d) = down;
                }
            }
            if (lane == 0) unit[g] = e;
        }
    }
    cluster_sync();  // (the codes are there, and the first CTA has begun)
    for (int i0 = p0 + 16 * warp; i0 < p1 && score; i0 += 16 * (PK_THREADS / 32)) {
        // pages i0 + lane / 4 and + 8: this lane's pieces c, c + 4, ... of their bounds
        uint32_t h[2][NX][4], l[2][NX][4];
        int es[2], kind[2];  // exponent of the scale; 0: a hole, 1: infinite, 2: others
#pragma unroll
        for (int y = 0; y < 2; y++) {
            const int i = i0 + (lane >> 2) + 8 * y;
            int slot, page = -1;
            if (i < p1) page = lookup(P, seq, i * P.page_size, slot);
            const int64_t at = (int64_t)max(page, 0) * P.nkv + kvh;
#pragma unroll
            for (int x = 0; x < NX; x++) {
                int4 u = make_int4(0, 0, 0, 0), v = u;
                if (page >= 0 && 16 * (c + 4 * x) < hd) {
                    u = __ldg(reinterpret_cast<const int4*>(A.b.hi + at * hd) + c + 4 * x);
                    v = __ldg(reinterpret_cast<const int4*>(A.b.lo + at * hd) + c + 4 * x);
                }
                h[y][x][0] = u.x, h[y][x][1] = u.y, h[y][x][2] = u.z, h[y][x][3] = u.w;
                l[y][x][0] = v.x, l[y][x][1] = v.y, l[y][x][2] = v.z, l[y][x][3] = v.w;
            }
            const uint32_t scale = page < 0 ? 0 : __float_as_uint(__ldg(A.b.scale + at)) >> 23;
            es[y] = min(max((int)scale, 7), 249);
            kind[y] = page < 0 ? 0 : scale == 255 ? 1 : 2;
        }
        uint32_t best[2] = {0, 0};
        for (int g0 = 0; g0 < G; g0 += 8) {
            int acc[4] = {0, 0, 0, 0};  // heads 2 c and 2 c + 1 of the first page, of the second
            const int g = min(g0 + (lane >> 2), G - 1);  // (columns past the last head are not used)
#pragma unroll
            for (int x = 0; x < NX; x++) {
                const uint4 p = *reinterpret_cast<const uint4*>(qp + g * STRIDE + 16 * (c + 4 * x));
                const uint4 m = *reinterpret_cast<const uint4*>(qn + g * STRIDE + 16 * (c + 4 * x));
                const uint32_t h0[4] = {h[0][x][0], h[1][x][0], h[0][x][1], h[1][x][1]}, h1[4] = {h[0][x][2], h[1][x][2], h[0][x][3], h[1][x][3]};
                const uint32_t l0[4] = {l[0][x][0], l[1][x][0], l[0][x][1], l[1][x][1]}, l1[4] = {l[0][x][2], l[1][x][2], l[0][x][3], l[1][x][3]};
                mma_s8(acc, h0, p.x, p.y);
                mma_s8(acc, h1, p.z, p.w);
                mma_s8(acc, l0, m.x, m.y);
                mma_s8(acc, l1, m.z, m.w);
            }
#pragma unroll
            for (int z = 0; z < 4; z++)
                if (g0 + 2 * c + (z & 1) < G) best[z >> 1] = max(best[z >> 1], score_key(acc[z], unit[g0 + 2 * c + (z & 1)], es[z >> 1]));
        }
#pragma unroll
        for (int y = 0; y < 2; y++) {
            best[y] = max(best[y], __shfl_xor_sync(0xffffffffu, best[y], 1));
            best[y] = max(best[y], __shfl_xor_sync(0xffffffffu, best[y], 2));
            const int i = i0 + (lane >> 2) + 8 * y;
            const uint32_t key = kind[y] == 0 ? KEY_HOLE : kind[y] == 1 ? KEY_INF : best[y];
            if (c == 0 && i < p1) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(first_keys + 4 * i), "r"(key) : "memory");
        }
    }
    cluster_sync();
    if (rank != 0 || !any) return;
    int32_t* out = A.out + ((int64_t)row * P.nkv + kvh) * A.budget;
    if (!score) {
        for (int i = tid; i < A.budget; i += PK_THREADS) out[i] = i < n ? i : -1;
        return;
    }
    pick_pages(keys, n, A.budget, A.first, A.recent, out, S);
}

constexpr int SELECT_SMEM = 200 * 1024;

template <typename T, int NX>
int launch_select_t(const SelectArgs& A, int ctas, size_t smem, cudaStream_t s) {
    static std::atomic<uint64_t> asked{0};
    HC_TRY(ask_smem((const void*)k_page_select<T, NX>, SELECT_SMEM, asked));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas, (unsigned)A.p.nkv, (unsigned)A.p.n_rows);
    cfg.blockDim = dim3(PK_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    HC_CUDA(cudaLaunchKernelEx(&cfg, k_page_select<T, NX>, A));
    HC_LAUNCH_CHECK();
    return HC_OK;
}

// Shared memory of the form in one kernel; 0: two kernels, where a head's bounds are no
// whole 16-byte pieces, a table's keys do not fit, or there are more rows than a
// grid has places.
size_t select_smem(int hd, int G, int max_pages, int n_rows) {
    const size_t stride = hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
    const size_t bytes = 2 * (size_t)G * stride + 4 * (size_t)((G + 3) / 4 * 4) + 4 * (size_t)max_pages;
    return hd % 16 == 0 && n_rows <= 65535 && bytes <= SELECT_SMEM ? bytes : 0;
}

template <typename CT>
int launch_bounds_t(const PagedArgs& P, const PagedScales& C, const Bounds& B, bool vec, int touched, cudaStream_t s) {
    const dim3 grid((unsigned)((touched + BD_WARPS - 1) / BD_WARPS), (unsigned)P.nkv, (unsigned)P.n_seqs);
    if (vec) k_page_bounds<CT, true><<<grid, 32 * BD_WARPS, 0, s>>>(P, C, B);
    else k_page_bounds<CT, false><<<grid, 32 * BD_WARPS, 0, s>>>(P, C, B);
    HC_LAUNCH_CHECK();
    return HC_OK;
}

int bounds_ok(const char* who, const hc_page_bounds* b) {
    HC_CHECK(b, HC_ERR_INVALID, "%s: NULL bounds", who);
    HC_CHECK(b->n_pages >= 1 && b->page_size >= 1 && b->n_kv_heads >= 1 && b->n_kv_heads <= 65535, HC_ERR_INVALID,
             "%s: bounds of %d pages of %d positions, %d heads", who, b->n_pages, b->page_size, b->n_kv_heads);
    HC_CHECK(b->head_dim >= 4 && b->head_dim % 4 == 0 && b->head_dim <= 256, HC_ERR_UNSUPPORTED,
             "%s: head_dim %d (a multiple of 4, at most 256)", who, b->head_dim);
    HC_CHECK(b->lo && b->hi && b->scale && ((uintptr_t)b->lo | (uintptr_t)b->hi) % 16 == 0 && (uintptr_t)b->scale % 4 == 0, HC_ERR_INVALID,
             "%s: NULL or misaligned bounds", who);
    return HC_OK;
}

size_t key_bytes(const hc_page_bounds* b, const hc_paged_batch* batch, int n_heads) {
    if (select_smem(b->head_dim, n_heads / b->n_kv_heads, batch->max_pages, batch->n_rows)) return 0;
    return (size_t)std::max(batch->n_rows, 0) * b->n_kv_heads * std::max(batch->max_pages, 0) * 4;
}

}  // namespace

}  // namespace hc

HC_EXPORT int hc_page_bounds_update_dev(const hc_page_bounds* b, const hc_paged_kv* kv, const hc_paged_batch* batch, void* stream) {
    const char* who = "hc_page_bounds_update_dev";
    hc::PagedArgs P;
    hc::PagedScales C;
    HC_TRY(hc::bounds_ok(who, b));
    HC_TRY(hc::page_args(who, kv, batch, P, C));
    HC_CHECK(b->n_pages == P.n_pages && b->page_size == P.page_size && b->n_kv_heads == P.nkv && b->head_dim == P.hd, HC_ERR_INVALID,
             "%s: bounds of %d pages of %d positions, %d heads of %d, for a cache of %d, %d, %d, %d", who, b->n_pages, b->page_size,
             b->n_kv_heads, b->head_dim, P.n_pages, P.page_size, P.nkv, P.hd);
    HC_CHECK(P.n_seqs <= 65535, HC_ERR_INVALID, "%s: %d sequences", who, P.n_seqs);
    if (P.n_rows == 0 || P.max_pages == 0) return HC_OK;
    const hc::Bounds B = {b->lo, b->hi, b->scale};
    cudaStream_t s = (cudaStream_t)stream;
    // (more pages than the host's bound of the rows are walked by the same CTAs)
    const int64_t rows = std::max(std::min(batch->max_q_len, P.n_rows), 1);
    const int touched = (int)std::min<int64_t>((rows + P.page_size - 2) / P.page_size + 1, P.max_pages);
    const bool vec = kv->kv_dtype == HC_KV_Q4 || ((uintptr_t)P.k % 16 == 0 && (P.kps | P.khs | P.kss) % 4 == 0);
    if (kv->kv_dtype == HC_KV_Q4) return hc::launch_bounds_t<hc::q4x>(P, C, B, true, touched, s);
    if (kv->kv_dtype == HC_KV_FP16) return hc::launch_bounds_t<__half>(P, C, B, vec, touched, s);
    return hc::launch_bounds_t<float>(P, C, B, vec, touched, s);
}

HC_EXPORT int hc_page_bounds_values_dev(const hc_page_bounds* b, float* lo_out, float* hi_out, void* stream) {
    const char* who = "hc_page_bounds_values_dev";
    HC_TRY(hc::bounds_ok(who, b));
    HC_CHECK(lo_out && hi_out && ((uintptr_t)lo_out | (uintptr_t)hi_out) % 16 == 0, HC_ERR_INVALID, "%s: NULL or misaligned output", who);
    const int64_t quads = (int64_t)b->n_pages * b->n_kv_heads * b->head_dim / 4, blocks = (quads + 255) / 256;
    HC_CHECK(blocks <= 0x7fffffff, HC_ERR_INVALID, "%s: %d pages", who, b->n_pages);
    const hc::Bounds B = {b->lo, b->hi, b->scale};
    hc::k_bounds_values<<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(B, b->head_dim, quads, lo_out, hi_out);
    HC_LAUNCH_CHECK();
    return HC_OK;
}

HC_EXPORT int hc_page_select_workspace(const hc_page_bounds* b, const hc_paged_batch* batch, int n_heads, size_t* bytes) {
    const char* who = "hc_page_select_workspace";
    HC_TRY(hc::bounds_ok(who, b));
    HC_CHECK(batch && bytes, HC_ERR_INVALID, "%s: NULL batch or bytes", who);
    HC_CHECK(n_heads >= 1 && n_heads % b->n_kv_heads == 0, HC_ERR_INVALID, "%s: %d query heads over %d KV heads", who, n_heads, b->n_kv_heads);
    *bytes = hc::key_bytes(b, batch, n_heads);
    return HC_OK;
}

HC_EXPORT int hc_page_select_dev(const hc_page_bounds* b, const hc_paged_batch* batch, const hc_rows* q, int n_heads, uint32_t dtype,
                                 int budget, int first, int recent, int32_t* out, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "hc_page_select_dev";
    hc::SelectArgs A;
    hc::PagedScales C;
    HC_TRY(hc::bounds_ok(who, b));
    // (a pool that stands for its sizes: no key is read)
    const hc_paged_kv kv = {b->lo, b->hi, 0, 0, 0, 0, 0, 0, HC_KV_FP16, b->n_pages, b->page_size, b->n_kv_heads, b->head_dim, 0};
    HC_TRY(hc::page_args(who, &kv, batch, A.p, C));
    HC_CHECK(dtype == HC_DTYPE_FP32 || dtype == HC_DTYPE_FP16, HC_ERR_UNSUPPORTED, "%s: dtype %u", who, dtype);
    HC_CHECK(n_heads >= 1 && n_heads % A.p.nkv == 0, HC_ERR_INVALID, "%s: %d query heads over %d KV heads", who, n_heads, A.p.nkv);
    HC_CHECK(first >= 0 && recent >= 0 && budget >= 1 && (int64_t)first + recent <= budget, HC_ERR_INVALID,
             "%s: a budget of %d pages with the first %d and the last %d", who, budget, first, recent);
    A.G = n_heads / A.p.nkv;
    const size_t smem = 2 * (size_t)A.G * ((A.p.hd + 15) / 16 * 16) + 4 * (size_t)A.G;
    HC_CHECK(smem <= 48 * 1024 || hc::select_smem(A.p.hd, A.G, A.p.max_pages, A.p.n_rows), HC_ERR_UNSUPPORTED,
             "%s: %d query heads of %d a KV head", who, A.G, A.p.hd);
    if (batch->n_rows == 0) return HC_OK;
    HC_TRY(hc::page_rows_ok(who, "q", q, dtype));
    HC_CHECK(out && (uintptr_t)out % 4 == 0, HC_ERR_INVALID, "%s: NULL or misaligned out", who);
    const size_t need = hc::key_bytes(b, batch, n_heads);
    HC_CHECK(workspace_bytes >= need && (need == 0 || (workspace && (uintptr_t)workspace % 16 == 0)), HC_ERR_INVALID,
             "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", who, need, workspace_bytes);
    A.b = {b->lo, b->hi, b->scale};
    A.q = q->data;
    A.q_rs = q->row_stride;
    A.q_hs = q->head_stride;
    A.budget = budget;
    A.first = first;
    A.recent = recent;
    A.out = out;
    A.keys = (uint32_t*)workspace;
    cudaStream_t s = (cudaStream_t)stream;
    const bool f16 = dtype == HC_DTYPE_FP16;
    A.qvec = (uintptr_t)q->data % (f16 ? 8 : 16) == 0 && (q->row_stride | q->head_stride) % 4 == 0;
    const size_t one = hc::select_smem(A.p.hd, A.G, A.p.max_pages, A.p.n_rows);
    if (one) {
        // as many CTAs a row and KV head as fill the SMs, 64 pages each at least
        const int64_t pairs = (int64_t)A.p.n_rows * A.p.nkv;
        int ctas = 1;
        while (ctas < 8 && ctas * pairs < 148 * 2 && ctas * 64 < A.p.max_pages) ctas *= 2;
        if (A.p.hd <= 64) return f16 ? hc::launch_select_t<__half, 1>(A, ctas, one, s) : hc::launch_select_t<float, 1>(A, ctas, one, s);
        if (A.p.hd <= 128) return f16 ? hc::launch_select_t<__half, 2>(A, ctas, one, s) : hc::launch_select_t<float, 2>(A, ctas, one, s);
        return f16 ? hc::launch_select_t<__half, 4>(A, ctas, one, s) : hc::launch_select_t<float, 4>(A, ctas, one, s);
    }
    if (A.p.max_pages > budget) {
        const int64_t pairs = (int64_t)A.p.n_rows * A.p.nkv, chunks = (A.p.max_pages + hc::SC_PAGES - 1) / hc::SC_PAGES;
        const dim3 grid((unsigned)std::max<int64_t>(1, std::min(chunks, (148 * 16 + pairs - 1) / pairs)), (unsigned)A.p.nkv,
                        (unsigned)std::min(A.p.n_rows, 65535));
        if (f16) hc::k_page_scores<__half><<<grid, hc::SC_THREADS, smem, s>>>(A);
        else hc::k_page_scores<float><<<grid, hc::SC_THREADS, smem, s>>>(A);
        HC_LAUNCH_CHECK();
        HC_TRY(hc::launch_pdl(hc::k_page_pick, dim3((unsigned)A.p.n_rows, (unsigned)A.p.nkv), dim3(hc::PK_THREADS), 0, s, A));
        HC_LAUNCH_CHECK();
    } else {
        hc::k_page_pick<<<dim3((unsigned)A.p.n_rows, (unsigned)A.p.nkv), hc::PK_THREADS, 0, s>>>(A);
        HC_LAUNCH_CHECK();
    }
    return HC_OK;
}
