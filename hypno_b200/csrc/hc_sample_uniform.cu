// The next token from the caller's uniform numbers: temperature, top-k, top-p
// and min-p over B rows of logits.
//
// Weights w_i = exp((l_i - max) * (1 / T)) are held as whole multiples of
// 2^-40 (64-bit integers; the largest is 2^40): integer sums do not depend on
// their order, so histograms may add by atomics and every thread layout gives
// the same token.  A weight below 2^-40 of the largest is 0 and can never be
// drawn.  The kept set is a head of the order (logit descending, index
// ascending), so one (key, index) pair cuts it off.
//
// k_sample_cluster: a cluster of up to 16 CTAs takes a row, each CTA a slice that
// it reads once into shared memory.  Passes over the slice: the maximum; for
// top-k a histogram (counts) of the tokens within HEAD of the maximum in units
// of T, or beyond it where that has fewer than k; the tokens of the bucket in
// which the order ends, gathered by the first CTA and sorted there; for top-p
// the same by mass, over what top-k kept; the kept mass of each warp's run, in
// which the draw is then found.  A bucket too full to sort (flat rows) is left
// to the first CTA and the kernel's slow path: a radix search over the logits'
// keys.  Bound by the latency of the cluster barriers for few rows, by the
// instructions of the passes (not by the one read of the logits) for many: a
// weight is some 30 of them.
#include "hc_internal.h"
#include "hc_common.cuh"

#include <cfloat>

namespace hc {

namespace {

constexpr int UT = 512;    // threads
constexpr int UB = 2048;   // buckets of a radix pass
constexpr int UW = UT / 32;
typedef unsigned long long u64;

// Larger logit -> larger key; 0 for NaN and -inf (never kept), -0 like +0.
__device__ __forceinline__ uint32_t ukey(float f) {
    if (!(f > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(f + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float ukey_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// floor(2^40 w) for w in [0, 1].  (Moving the mantissa to its place by shifts
// took a fifth longer than the conversion.)
__device__ __forceinline__ u64 mass_of(float w) { return __float2ull_rz(__fmul_rn(w, 1099511627776.0f)); }

struct URow {
    const float* l;
    int V;
    float mx, inv;
    __device__ __forceinline__ float weight(float f) const {
        return f == mx ? 1.0f : expf(__fmul_rn(__fsub_rn(f, mx), inv));
    }
    __device__ __forceinline__ u64 mass(float f) const {
        return f > -INFINITY ? mass_of(weight(f)) : 0ull;
    }
};

struct UShared {
    uint32_t cnt[UB];
    u64 sum[UB];
    u64 red[32];
    uint32_t redu[32];
    u64 before;        // mass above the chosen bucket
    uint32_t nbefore;  // tokens above it
    int sel;
    uint32_t cut;
    u64 seg;
};

__device__ __forceinline__ u64 block_sum_u64(u64 v, UShared& S) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) S.red[threadIdx.x >> 5] = v;
    __syncthreads();
    u64 t = (threadIdx.x & 31) < UW ? S.red[threadIdx.x & 31] : 0ull;
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    return t;
}

// Finds, among tokens with key >= floor_key (all above it, `floor_ties` at
// it), the key at which the head of the order ends: `by_count`: the head of
// `need` tokens; else the head of the tokens whose mass before them is below
// `goal`.  Returns the key and how many of its ties belong to the head.
__device__ void head_end(const URow& R, uint32_t floor_key, uint32_t floor_ties, bool by_count, uint32_t need,
                         double goal, UShared& S, uint32_t* key_out, uint32_t* ties_out) {
    uint32_t prefix = 0, mask = 0, nbefore = 0;
    u64 before = 0;
    const int shifts[3] = {21, 10, 0}, widths[3] = {11, 11, 10};
    for (int pass = 0; pass < 3; pass++) {
        const int nb = 1 << widths[pass];
        for (int b = threadIdx.x; b < nb; b += UT) {
            S.cnt[b] = 0;
            S.sum[b] = 0;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < R.V; i += UT) {
            const float f = R.l[i];
            const uint32_t k = ukey(f);
            if (k == 0 || k < floor_key || (k & mask) != prefix) continue;
            const int b = (k >> shifts[pass]) & (nb - 1);
            atomicAdd(&S.cnt[b], 1u);
            if (!by_count) atomicAdd(&S.sum[b], R.mass(f));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            // the last bucket, from the top, that holds a token of the head
            int sel = -1;
            uint32_t nb_sel = 0;
            u64 be_sel = 0, be = before;
            uint32_t n = nbefore;
            for (int b = nb - 1; b >= 0; b--) {
                if (S.cnt[b] == 0) continue;
                if (by_count ? n >= need : !((double)be < goal)) break;
                sel = b;
                nb_sel = n;
                be_sel = be;
                n += S.cnt[b];
                be += S.sum[b];
            }
            S.sel = sel;
            S.nbefore = nb_sel;
            S.before = be_sel;
        }
        __syncthreads();
        prefix |= (uint32_t)S.sel << shifts[pass];
        mask |= (uint32_t)(nb - 1) << shifts[pass];
        nbefore = S.nbefore;
        before = S.before;
        __syncthreads();
    }
    uint32_t ties = S.cnt[prefix & 1023u];
    if (prefix == floor_key && ties > floor_ties) ties = floor_ties;
    if (by_count) {
        ties = min(ties, need - nbefore);
    } else {
        const u64 w = R.mass(ukey_value(prefix));
        uint32_t lo = 1, hi = ties;  // the last tie whose mass before it is below the goal
        while (lo < hi) {
            const uint32_t mid = (lo + hi + 1) >> 1;
            if ((double)(before + (u64)(mid - 1) * w) < goal) lo = mid;
            else hi = mid - 1;
        }
        ties = lo;
    }
    __syncthreads();
    *key_out = prefix;
    *ties_out = ties;
}

// floor(u total), below total.
__device__ __forceinline__ u64 draw_goal(float u, u64 total) {
    const double g = (u >= 0.0f ? (double)u : 0.0) * (double)total;
    const u64 goal = (u64)floor(fmin(g, 9.0e18));
    return goal < total ? goal : total - 1;
}

struct URowArgs {
    float u, tp, mp;
    int tk;
};

// One CTA's way through a row of any kind, reading the logits pass by pass.
__device__ __noinline__ void sample_row(URow R, URowArgs P, UShared& S, int32_t* out, float* logprob) {
    const int V = R.V, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float tp = P.tp, mp = P.mp;
    const int tk = P.tk;
    uint32_t key = 1, ties = 0xffffffffu;  // every token
    if (tk > 0 && tk < V) head_end(R, key, ties, true, (uint32_t)tk, 0.0, S, &key, &ties);
    if (tp < 1.0f && tk != 1) {
        // mass of the tokens top-k kept
        u64 m = 0;
        for (int i = threadIdx.x; i < V; i += UT) {
            const float f = R.l[i];
            if (ukey(f) > key) m += R.mass(f);
        }
        u64 held = block_sum_u64(m, S);
        uint32_t n = 0;
        for (int i = threadIdx.x; i < V; i += UT) n += ukey(R.l[i]) == key;
        n = (uint32_t)block_sum_u64(n, S);
        held += (u64)min(n, ties) * R.mass(ukey_value(key));
        head_end(R, key, ties, false, 0, (double)tp * (double)held, S, &key, &ties);
    }
    const bool minp = mp <= 1.0f;

    // index of the last tie kept
    if (threadIdx.x == 0) S.cut = 0xffffffffu;
    __syncthreads();
    if (ties != 0xffffffffu && warp == 0) {
        uint32_t n = 0;
        for (int i0 = 0; i0 < V; i0 += 32) {
            const bool hit = i0 + lane < V && ukey(R.l[i0 + lane]) == key;
            const unsigned b = __ballot_sync(0xffffffffu, hit);
            if (n + __popc(b) >= ties) {
                if (hit && n + __popc(b & ((2u << lane) - 1u)) == ties) S.cut = (uint32_t)(i0 + lane);
                break;
            }
            n += __popc(b);
        }
    }
    __syncthreads();
    const uint32_t cut = S.cut;
    auto kept = [&](int i) -> u64 {
        const float f = R.l[i];
        const uint32_t k = ukey(f);
        if (k < key || (k == key && (uint32_t)i > cut)) return 0ull;
        if (minp && mp > 0.0f && !(R.weight(f) >= mp)) return 0ull;
        return R.mass(f);
    };

    // mass of each thread's segment of consecutive tokens, then the one that holds the goal
    const int per = (V + UT - 1) / UT;
    u64 mine = 0;
    const int i0 = min((int)threadIdx.x * per, V), i1 = min(i0 + per, V);
    for (int i = i0; i < i1; i++) mine += kept(i);
    u64 incl = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
    }
    if (lane == 31) S.red[warp] = incl;
    __syncthreads();
    u64 base = 0, total = 0;
    for (int w = 0; w < UW; w++) {
        if (w < warp) base += S.red[w];
        total += S.red[w];
    }
    incl += base;
    const u64 goal = draw_goal(P.u, total);
    if (goal < incl && goal >= incl - mine) {
        u64 run = incl - mine;
        for (int i = i0; i < i1; i++) {
            const u64 m = kept(i);
            run += m;
            if (run > goal) {
                *out = i;
                if (logprob) *logprob = logf((float)((double)m / (double)total));
                break;
            }
        }
    }
}

// ============================================================ the cluster kernel

constexpr int UC_MAX = 16;         // CTAs of a cluster (above 8 for few long rows only)
constexpr int HB2 = 1024;          // buckets of a histogram
// Distances (max - l) / T that the two histograms cover: weights from 1 to 6e-6,
// where most orders end and few tokens are, and from there to below 2^-40.
constexpr float HEAD = 12.0f, TAIL = 28.0f;
constexpr int CAP = 1024;          // tokens of a bucket that are sorted
constexpr int GO_ON = -2, ALL = -1, SLOW = HB2;  // instead of a bucket

struct __align__(16) CShared {
    union {
        UShared slow;
        struct {
            u64 sum[HB2];
            uint32_t cnt[HB2];
            u64 list[CAP];         // gathered tokens, key above ~index (first CTA)
        } h;
    };
    u64 red[32];
    uint32_t redu[32];
    // what the CTAs of the cluster tell one another, one word for each (all have the same copy)
    uint32_t c_max[UC_MAX], c_at[UC_MAX];
    u64 c_mass[UC_MAX];            // mass (pass 2), kept mass (pass 4)
    // what the first CTA tells all
    int n_list;
    int bucket;
    u64 cut;                       // the last token kept: key above ~index
    // the first CTA's own
    u64 sel_mass, head_mass;       // mass before the bucket; of the first histogram
    uint32_t sel_cnt, head_cnt;    // likewise tokens
    u64 w_mass[UW];                // of the warps' buckets
    uint32_t w_cnt[UW];
    u64 sorted[256];
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote(const void* p, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ void remote_st32(const void* p, uint32_t rank, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote(p, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void remote_st64(const void* p, uint32_t rank, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote(p, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t remote_ld32(const void* p, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ u64 remote_ld64(const void* p, uint32_t rank) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(remote(p, rank)) : "memory");
    return v;
}

// Descending sort of the first CTA's list: places by counting for short lists,
// bitonic for long ones.  Returns where the sorted list is.
__device__ u64* sort_list(CShared& S, int n) {
    if (n <= 256) {
        if ((int)threadIdx.x < n) {
            const u64 e = S.h.list[threadIdx.x];
            int at = 0;
            for (int j = 0; j < n; j++) at += S.h.list[j] > e;
            S.sorted[at] = e;
        }
        __syncthreads();
        return S.sorted;
    }
    int m = 512;
    while (m < n) m <<= 1;
    for (int j = n + (int)threadIdx.x; j < m; j += UT) S.h.list[j] = 0ull;
    __syncthreads();
    for (int k = 2; k <= m; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int i = threadIdx.x; i < m; i += UT) {
                const int o = i ^ j;
                if (o > i) {
                    const u64 a = S.h.list[i], b = S.h.list[o];
                    if ((i & k) == 0 ? a < b : a > b) {
                        S.h.list[i] = b;
                        S.h.list[o] = a;
                    }
                }
            }
            __syncthreads();
        }
    return S.h.list;
}

__global__ void __launch_bounds__(UT, 2) k_sample_cluster(const float* __restrict__ logits, size_t ld, int V, int slice,
                                                       const float* __restrict__ u, const float* __restrict__ temp,
                                                       const int* __restrict__ top_k, const float* __restrict__ top_p,
                                                       const float* __restrict__ min_p, int32_t* __restrict__ out,
                                                       float* __restrict__ logprob, int CS) {
    extern __shared__ __align__(16) uint8_t smem[];
    CShared& S = *reinterpret_cast<CShared*>(smem);
    const int rank = CS > 1 ? (int)cluster_rank() : 0, row = blockIdx.x / CS;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int base = rank * slice, n = max(0, min(slice, V - base));
    auto sync_all = [&]() {
        if (CS > 1) cluster_barrier();
        else __syncthreads();
    };
    const float T = temp[row];
    URowArgs P;
    P.u = u[row];
    P.tp = top_p[row];
    P.mp = min_p[row];
    P.tk = top_k[row];
    if (!(T > 0.0f) || !(P.tp > 0.0f) || !(P.mp <= 1.0f)) P.tk = 1;  // only the first token can be kept
    URow R;
    R.l = logits + (size_t)row * ld;
    R.V = V;
    R.inv = T > 0.0f ? __fdiv_rn(1.0f, T) : 1.0f;

    // ---- 1: the slice and the maximum
    float top = -INFINITY;  // (NaN never wins)
    const float* src = R.l + base;
    const int head = min(n, (int)((16 - ((uintptr_t)src & 15)) & 15) / 4), n4 = (n - head) >> 2;  // 16-byte loads in between
    float* L = reinterpret_cast<float*>(smem + sizeof(CShared)) + ((4 - head) & 3);  // and 16-byte stores
#pragma unroll 4
    for (int i = threadIdx.x; i < n4; i += UT) {
        const float4 v = __ldcs(reinterpret_cast<const float4*>(src + head) + i);
        *reinterpret_cast<float4*>(L + head + 4 * i) = v;
        top = fmaxf(fmaxf(fmaxf(top, v.x), fmaxf(v.y, v.z)), v.w);
    }
    for (int i = threadIdx.x; i < head; i += UT) top = fmaxf(top, L[i] = src[i]);
    for (int i = head + 4 * n4 + threadIdx.x; i < n; i += UT) top = fmaxf(top, L[i] = src[i]);
    uint32_t kmax = __reduce_max_sync(0xffffffffu, ukey(top));
    if (lane == 0) S.redu[warp] = kmax;
    if (threadIdx.x == 0) S.cut = 1ull << 32;  // keys from 1 on: every token
    __syncthreads();
    kmax = __reduce_max_sync(0xffffffffu, lane < UW ? S.redu[lane] : 0u);
    if (threadIdx.x < CS) remote_st32(&S.c_max[rank], threadIdx.x, kmax);
    sync_all();
    for (int c = 0; c < CS; c++) kmax = max(kmax, S.c_max[c]);
    if (kmax == 0) {  // nothing above -inf
        if (rank == 0 && threadIdx.x == 0) {
            out[row] = -1;
            if (logprob) logprob[row] = -INFINITY;
        }
        return;
    }
    R.mx = ukey_value(kmax);

    if (P.tk == 1) {  // the first of the maxima
        uint32_t at = 0xffffffffu;
        for (int i = threadIdx.x; i < n; i += UT)
            if (L[i] == R.mx) at = min(at, (uint32_t)(base + i));
        at = __reduce_min_sync(0xffffffffu, at);
        __syncthreads();  // (S.redu has been read)
        if (lane == 0) S.redu[warp] = at;
        __syncthreads();
        at = __reduce_min_sync(0xffffffffu, lane < UW ? S.redu[lane] : 0xffffffffu);
        if (threadIdx.x == 0) remote_st32(&S.c_at[rank], 0, at);
        sync_all();
        if (rank == 0 && threadIdx.x == 0) {
            for (int c = 0; c < CS; c++) at = min(at, S.c_at[c]);
            out[row] = (int)at;
            if (logprob) logprob[row] = 0.0f;
        }
        return;
    }

    auto block_sum = [&](u64 v) -> u64 {
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        __syncthreads();
        if (lane == 0) S.red[warp] = v;
        __syncthreads();
        u64 t = lane < UW ? S.red[lane] : 0ull;
        for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        return t;
    };
    // bucket of a logit in histogram 0 or 1, monotone in l; -1 outside it
    auto bucket_of = [&](float f, int level) -> int {
        const float d = f == R.mx ? 0.0f : __fmul_rn(__fsub_rn(R.mx, f), R.inv);
        if (level == 0) return d < HEAD ? (int)(d * (HB2 / HEAD)) : -1;
        return d >= HEAD && d < TAIL ? min((int)((d - HEAD) * (HB2 / (TAIL - HEAD))), HB2 - 1) : -1;
    };

    const bool by_k = P.tk > 0 && P.tk < V, by_p = P.tp < 1.0f && P.tk != 1;
    u64 cut = 1ull << 32;
    if (by_k || by_p) {
        u64 held = 0;      // (first CTA) the mass of which top_p is a share
        float kf = -FLT_MAX;               // top-k's end: logits above it, and equal ones up to index ki
        uint32_t ki = 0xffffffffu;
        // Two ends may have to be found: top-k's by count, then top-p's by mass.
        for (int pass = by_k ? 0 : 1; pass < (by_p ? 2 : 1); pass++) {
            int level = 0;
            for (;; level++) {
                // ---- 2: the histogram: counts, and for top-p masses
                for (int b = threadIdx.x; b < HB2; b += UT) {
                    S.h.sum[b] = 0ull;
                    S.h.cnt[b] = 0u;
                }
                __syncthreads();
                u64 mass = 0;
                if (pass == 0) {
                    for (int i = threadIdx.x; i < n; i += UT) {
                        const int b = bucket_of(L[i], level);
                        if (b >= 0) atomicAdd(&S.h.cnt[b], 1u);
                    }
                } else {
                    for (int i = threadIdx.x; i < n; i += UT) {
                        const float f = L[i];
                        if (!(f >= kf) || (f == kf && (uint32_t)(base + i) > ki)) continue;
                        const int b = bucket_of(f, level);
                        if (b < 0 && level == 1) continue;
                        const u64 m = mass_of(R.weight(f));
                        mass += m;
                        if (b >= 0) {
                            atomicAdd(&S.h.cnt[b], 1u);
                            atomicAdd(&S.h.sum[b], m);
                        }
                    }
                    if (level == 0) {
                        mass = block_sum(mass);
                        if (threadIdx.x == 0) remote_st64(&S.c_mass[rank], 0, mass);
                    }
                }
                sync_all();
                if (rank == 0) {  // the first CTA adds the histograms up
                    if (pass == 1 && level == 0)
                        for (int c = 0; c < CS; c++) held += S.c_mass[c];
                    for (int b = threadIdx.x; b < HB2; b += UT) {
                        uint32_t nc[UC_MAX];
                        u64 ms[UC_MAX];
#pragma unroll
                        for (int c = 1; c < UC_MAX; c++) {  // all on their way before the first is added
                            nc[c] = c < CS ? remote_ld32(&S.h.cnt[b], c) : 0u;
                            ms[c] = c < CS && pass == 1 ? remote_ld64(&S.h.sum[b], c) : 0ull;
                        }
#pragma unroll
                        for (int c = 1; c < UC_MAX; c++) {
                            S.h.cnt[b] += nc[c];
                            S.h.sum[b] += ms[c];
                        }
                    }
                    __syncthreads();
                }
                if (rank == 0) {
                    // the last bucket that holds a token of the order's head: two buckets a thread
                    const double goal = (double)P.tp * (double)held;
                    const int b0 = 2 * threadIdx.x;
                    const uint32_t c0 = S.h.cnt[b0], c1 = S.h.cnt[b0 + 1];
                    const u64 m0 = S.h.sum[b0], m1 = S.h.sum[b0 + 1];
                    uint32_t ci = c0 + c1;
                    u64 mi = m0 + m1;
                    for (int o = 1; o < 32; o <<= 1) {
                        const uint32_t tc = __shfl_up_sync(0xffffffffu, ci, o);
                        const u64 tm = __shfl_up_sync(0xffffffffu, mi, o);
                        if (lane >= o) {
                            ci += tc;
                            mi += tm;
                        }
                    }
                    if (lane == 31) {
                        S.w_cnt[warp] = ci;
                        S.w_mass[warp] = mi;
                    }
                    if (threadIdx.x == 0) {
                        S.bucket = -1;
                        S.n_list = 0;
                    }
                    __syncthreads();
                    uint32_t nb = level ? S.head_cnt : 0u, all_n = nb;
                    u64 be = level ? S.head_mass : 0ull, all_m = be;
                    for (int w = 0; w < UW; w++) {
                        if (w < warp) {
                            nb += S.w_cnt[w];
                            be += S.w_mass[w];
                        }
                        all_n += S.w_cnt[w];
                        all_m += S.w_mass[w];
                    }
                    nb += ci - c0 - c1;
                    be += mi - m0 - m1;
                    const bool over = pass == 0 ? all_n >= (uint32_t)P.tk : !((double)all_m < goal);
                    const bool in0 = c0 > 0 && (pass == 0 ? nb < (uint32_t)P.tk : (double)be < goal);
                    const bool in1 = c1 > 0 && (pass == 0 ? nb + c0 < (uint32_t)P.tk : (double)(be + m0) < goal);
                    const int mine = in1 ? b0 + 1 : in0 ? b0 : -1;
                    const int top = __reduce_max_sync(0xffffffffu, mine);
                    if (lane == 0 && top >= 0) atomicMax(&S.bucket, top);
                    __syncthreads();
                    const int sel = S.bucket;
                    __syncthreads();
                    if (over && sel >= 0 ? mine == sel : threadIdx.x == 0) {
                        // not over: the order ends further on, or (top-k) it keeps every token with a mass
                        const int b = over && sel >= 0 ? ((in1 ? c1 : c0) <= (uint32_t)CAP ? sel : SLOW) : level == 0 ? GO_ON : pass == 0 ? ALL : SLOW;
                        S.bucket = b;
                        S.sel_mass = in1 ? be + m0 : be;
                        S.sel_cnt = in1 ? nb + c0 : nb;
                        if (b == GO_ON) {
                            S.head_mass = all_m;
                            S.head_cnt = all_n;
                        }
                        for (int c = 1; c < CS; c++) remote_st32(&S.bucket, c, (uint32_t)b);
                    }
                }
                sync_all();
                if (S.bucket != GO_ON) break;
                sync_all();  // (all have read it)
            }
            const int sel = S.bucket;
            if (sel == SLOW) {  // by the first CTA
                if (rank == 0) sample_row(R, P, S.slow, out + row, logprob ? logprob + row : nullptr);
                return;
            }
            if (sel == ALL) {
                sync_all();
                continue;
            }
            // ---- 3: the bucket's tokens, to the first CTA
            for (int i = threadIdx.x; i < n; i += UT) {
                const float f = L[i];
                if (!(f >= kf) || bucket_of(f, level) != sel || (f == kf && (uint32_t)(base + i) > ki)) continue;
                uint32_t at;
                asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(CS > 1 ? remote(&S.n_list, 0) : smem_u32(&S.n_list)) : "memory");
                if (at >= (uint32_t)CAP) continue;
                const u64 e = (u64)ukey(f) << 32 | (uint32_t)~(base + i);
                if (CS > 1) remote_st64(&S.h.list[at], 0, e);
                else S.h.list[at] = e;
            }
            sync_all();
            if (rank == 0) {
                const int ln = S.n_list;
                const u64* list = sort_list(S, ln);
                if (warp == 0) {
                    // 32 tokens at a time: the masses before them, and the last one kept
                    u64 before = S.sel_mass, c = 0;
                    const double goal = (double)P.tp * (double)held;
                    for (int i0 = 0; i0 < ln; i0 += 32) {
                        const u64 e = i0 + lane < ln ? list[i0 + lane] : 0ull;
                        const u64 m = e ? R.mass(ukey_value((uint32_t)(e >> 32))) : 0ull;
                        u64 incl = m;
                        for (int o = 1; o < 32; o <<= 1) {
                            const u64 t = __shfl_up_sync(0xffffffffu, incl, o);
                            if (lane >= o) incl += t;
                        }
                        const bool in = e && (pass == 0 ? S.sel_cnt + i0 + lane < (uint32_t)P.tk : (double)(before + incl - m) < goal);
                        const unsigned b = __ballot_sync(0xffffffffu, in);  // a run of low lanes
                        if (b) {
                            const int l = 31 - __clz(b);
                            c = __shfl_sync(0xffffffffu, e, l);
                            before += __shfl_sync(0xffffffffu, incl, l);
                        }
                        if (b != 0xffffffffu) break;
                    }
                    if (lane == 0) {
                        S.cut = c;
                        for (int q = 1; q < CS; q++) remote_st64(&S.cut, q, c);
                    }
                }
            }
            sync_all();
            cut = S.cut;
            kf = ukey_value((uint32_t)(cut >> 32));
            ki = ~(uint32_t)cut;
        }
    }

    // ---- 4: the kept mass of each warp's run of tokens, and the draw
    const float cf = cut == 1ull << 32 ? -FLT_MAX : ukey_value((uint32_t)(cut >> 32));
    const uint32_t ci = ~(uint32_t)cut;
    const float least = P.mp <= 1.0f ? P.mp : 0.0f;
    auto kept = [&](int i) -> u64 {
        const float f = L[i];
        if (!(f >= cf) || (f == cf && (uint32_t)(base + i) > ci)) return 0ull;
        const float w = R.weight(f);
        return w >= least ? mass_of(w) : 0ull;
    };
    const int per = ((n + UW - 1) / UW + 31) & ~31, w0 = min(warp * per, n), w1 = min(w0 + per, n);
    u64 mine = 0;
    for (int i = w0 + lane; i < w1; i += 32) mine += kept(i);
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    __syncthreads();
    if (lane == 0) S.red[warp] = mine;
    __syncthreads();
    u64 cta = 0, below = 0;
    for (int w = 0; w < UW; w++) {
        if (w == warp) below = cta;
        cta += S.red[w];
    }
    if (threadIdx.x < CS) remote_st64(&S.c_mass[rank], threadIdx.x, cta);
    sync_all();  // (also the last access of another CTA's shared memory)
    u64 total = 0;
    for (int c = 0; c < CS; c++) {
        if (c == rank) below += total;
        total += S.c_mass[c];
    }
    const u64 goal = draw_goal(P.u, total);
    if (goal < below || goal >= below + mine) return;
    for (int i0 = w0; i0 < w1; i0 += 32) {
        const u64 m = i0 + lane < w1 ? kept(i0 + lane) : 0ull;
        u64 incl = m;
        for (int o = 1; o < 32; o <<= 1) {
            const u64 t = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += t;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, below + incl > goal);
        if (hit) {
            if (lane == __ffs(hit) - 1) {
                out[row] = base + i0 + lane;
                if (logprob) logprob[row] = logf((float)((double)m / (double)total));
            }
            return;
        }
        below += __shfl_sync(0xffffffffu, incl, 31);
    }
}

// Rows too long for the shared memory of a cluster.
__global__ void __launch_bounds__(UT) k_sample_uniform(const float* __restrict__ logits, size_t ld, int V,
                                                       const float* __restrict__ u, const float* __restrict__ temp,
                                                       const int* __restrict__ top_k, const float* __restrict__ top_p,
                                                       const float* __restrict__ min_p, int32_t* __restrict__ out,
                                                       float* __restrict__ logprob) {
    __shared__ UShared S;
    const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float T = temp[row];
    URowArgs P;
    P.u = u[row];
    P.tp = top_p[row];
    P.mp = min_p[row];
    P.tk = top_k[row];
    if (!(T > 0.0f) || !(P.tp > 0.0f) || !(P.mp <= 1.0f)) P.tk = 1;  // only the first token can be kept
    URow R;
    R.l = logits + (size_t)row * ld;
    R.V = V;
    R.inv = T > 0.0f ? __fdiv_rn(1.0f, T) : 1.0f;
    uint32_t kmax = 0;
    for (int i = threadIdx.x; i < V; i += UT) kmax = max(kmax, ukey(R.l[i]));
    kmax = __reduce_max_sync(0xffffffffu, kmax);
    if (lane == 0) S.redu[warp] = kmax;
    __syncthreads();
    kmax = __reduce_max_sync(0xffffffffu, lane < UW ? S.redu[lane] : 0u);
    if (kmax == 0) {  // nothing above -inf
        if (threadIdx.x == 0) {
            out[row] = -1;
            if (logprob) logprob[row] = -INFINITY;
        }
        return;
    }
    R.mx = ukey_value(kmax);
    sample_row(R, P, S, out + row, logprob ? logprob + row : nullptr);
}

}  // namespace

}  // namespace hc

HC_EXPORT int hc_sample_uniform_dev(const float* logits_dev, size_t ld, int B, int V, const float* u_dev,
                                    const float* temperature_dev, const int* top_k_dev, const float* top_p_dev,
                                    const float* min_p_dev, int32_t* out_dev, float* logprob_dev, void* stream) {
    HC_CHECK(B >= 0 && V > 0 && V <= (1 << 22) && ld >= (size_t)V, HC_ERR_INVALID,
             "hc_sample_uniform_dev: bad shape (B %d, V %d, ld %zu)", B, V, ld);
    HC_CHECK(B == 0 || (logits_dev && u_dev && temperature_dev && top_k_dev && top_p_dev && min_p_dev && out_dev),
             HC_ERR_INVALID, "hc_sample_uniform_dev: NULL argument");
    if (B == 0) return HC_OK;
    cudaStream_t s = (cudaStream_t)stream;
    // CTAs a row: slices of 4,096 logits or more, up to eight CTAs; a slice fits shared memory
    int cs = 1;
    while (cs < 8 && V > cs * 4096) cs *= 2;
    if ((int64_t)B * 16 <= 148 && V >= 16 * 4096) cs = 16;  // few long rows: shorter passes
    const int slice = (V + cs - 1) / cs;
    const size_t smem = sizeof(hc::CShared) + ((size_t)slice + 8) * sizeof(float);
    if (smem > 227 * 1024) {
        hc::k_sample_uniform<<<(unsigned)B, hc::UT, 0, s>>>(logits_dev, ld, V, u_dev, temperature_dev, top_k_dev, top_p_dev,
                                                           min_p_dev, out_dev, logprob_dev);
        HC_LAUNCH_CHECK();
        return HC_OK;
    }
    HC_CHECK((int64_t)B * cs <= 0x7fffffff, HC_ERR_INVALID, "hc_sample_uniform_dev: %d rows", B);
    HC_CUDA(cudaFuncSetAttribute(hc::k_sample_cluster, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    if (cs > 8) HC_CUDA(cudaFuncSetAttribute(hc::k_sample_cluster, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(B * cs));
    cfg.blockDim = dim3(hc::UT);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cs;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    HC_CUDA(cudaLaunchKernelEx(&cfg, hc::k_sample_cluster, logits_dev, ld, V, slice, u_dev, temperature_dev, top_k_dev,
                               top_p_dev, min_p_dev, out_dev, logprob_dev, cs));
    HC_LAUNCH_CHECK();
    return HC_OK;
}
