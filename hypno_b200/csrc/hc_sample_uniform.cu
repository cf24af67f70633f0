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
// k_sample_cluster: a cluster of up to 8 CTAs takes a row, each CTA a slice that
// it reads once into shared memory.  Passes over the slice: the maximum; the
// mass, with a histogram (count and mass) of the tokens within HEAD of the
// maximum in units of T; the tokens of the bucket in which the head of the
// order ends, gathered by the first CTA and sorted there; the kept mass of each
// warp's run, in which the draw is then found.  A row whose order ends beyond
// the histogram, or in a bucket too full to sort (flat rows), is left to the
// first CTA and the kernel's slow path: a radix search over the logits' keys.
// Bound by the latency of the cluster barriers for few rows, by the passes
// over shared memory (not by the one read of the logits) for many.
#include "hc_internal.h"
#include "hc_common.cuh"

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

struct URow {
    const float* l;
    int V;
    float mx, inv;
    __device__ __forceinline__ float weight(float f) const {
        return f == mx ? 1.0f : expf(__fmul_rn(__fsub_rn(f, mx), inv));
    }
    __device__ __forceinline__ u64 mass(float f) const {
        return f > -INFINITY ? __float2ull_rz(__fmul_rn(weight(f), 1099511627776.0f)) : 0ull;
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

constexpr int UC_MAX = 8;          // CTAs of a cluster
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
    uint32_t c_max[UC_MAX];
    u64 c_mass[UC_MAX];            // mass (pass 2), kept mass (pass 4)
    // what the first CTA tells all
    int n_list;
    int bucket;
    u64 cut;                       // the last token kept: key above ~index
    // the first CTA's own
    u64 sel_mass, head_mass;       // mass before the bucket; of the first histogram
    uint32_t sel_cnt, head_cnt;    // likewise tokens
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

// Descending bitonic sort of the first CTA's list.
__device__ void sort_list(CShared& S, int n) {
    int m = 1;
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
}

__global__ void __launch_bounds__(UT) k_sample_cluster(const float* __restrict__ logits, size_t ld, int V, int slice,
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
    uint32_t kmax = 0;
    const float* src = R.l + base;
    const int head = min(n, (int)((16 - ((uintptr_t)src & 15)) & 15) / 4), n4 = (n - head) >> 2;  // 16-byte loads in between
    float* L = reinterpret_cast<float*>(smem + sizeof(CShared)) + ((4 - head) & 3);  // and 16-byte stores
#pragma unroll 4
    for (int i = threadIdx.x; i < n4; i += UT) {
        const float4 v = __ldcs(reinterpret_cast<const float4*>(src + head) + i);
        *reinterpret_cast<float4*>(L + head + 4 * i) = v;
        kmax = max(max(max(kmax, ukey(v.x)), max(ukey(v.y), ukey(v.z))), ukey(v.w));
    }
    for (int i = threadIdx.x; i < n; i += UT)
        if (i < head || i >= head + 4 * n4) {
            const float v = src[i];
            L[i] = v;
            kmax = max(kmax, ukey(v));
        }
    kmax = __reduce_max_sync(0xffffffffu, kmax);
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
        int have = -1;     // the histogram at hand
        // Two ends may have to be found: top-k's by count, then top-p's by mass.
        for (int pass = by_k ? 0 : 1; pass < (by_p ? 2 : 1); pass++) {
            int level = 0;
            for (;; level++) {
                if (have != level) {
                    // ---- 2: the histogram, and (once) the mass
                    for (int b = threadIdx.x; b < HB2; b += UT) {
                        S.h.sum[b] = 0ull;
                        S.h.cnt[b] = 0u;
                    }
                    __syncthreads();
                    u64 mass = 0;
                    for (int i = threadIdx.x; i < n; i += UT) {
                        const float f = L[i];
                        if (!(f > -INFINITY)) continue;
                        const int b = bucket_of(f, level);
                        if (b < 0 && have >= 0) continue;
                        const u64 m = R.mass(f);
                        mass += m;
                        if (b >= 0) {
                            atomicAdd(&S.h.cnt[b], 1u);
                            atomicAdd(&S.h.sum[b], m);
                        }
                    }
                    if (have < 0) {
                        mass = block_sum(mass);
                        if (threadIdx.x < CS) remote_st64(&S.c_mass[rank], threadIdx.x, mass);
                    }
                    sync_all();
                    if (rank == 0) {  // the first CTA adds the histograms up
                        if (have < 0)
                            for (int c = 0; c < CS; c++) held += S.c_mass[c];
                        for (int b = threadIdx.x; b < HB2; b += UT) {
                            uint32_t nc = S.h.cnt[b];
                            u64 ms = S.h.sum[b];
                            for (int c = 1; c < CS; c++) {
                                nc += remote_ld32(&S.h.cnt[b], c);
                                ms += remote_ld64(&S.h.sum[b], c);
                            }
                            S.h.cnt[b] = nc;
                            S.h.sum[b] = ms;
                        }
                        __syncthreads();
                    }
                    have = level;
                }
                if (rank == 0 && warp == 0) {
                    // warp 0: the last bucket that holds a token of the order's head
                    const double goal = (double)P.tp * (double)held;
                    u64 be = level ? S.head_mass : 0ull, sel_be = 0;
                    uint32_t nb = level ? S.head_cnt : 0u, sel_nb = 0;
                    int sel = -1;
                    bool over = false;
                    for (int b0 = 0; b0 < HB2 && !over; b0 += 32) {
                        const uint32_t c = S.h.cnt[b0 + lane];
                        const u64 m = S.h.sum[b0 + lane];
                        uint32_t ci = c;
                        u64 mi = m;
                        for (int o = 1; o < 32; o <<= 1) {
                            const uint32_t tc = __shfl_up_sync(0xffffffffu, ci, o);
                            const u64 tm = __shfl_up_sync(0xffffffffu, mi, o);
                            if (lane >= o) {
                                ci += tc;
                                mi += tm;
                            }
                        }
                        const uint32_t nb_l = nb + ci - c;
                        const u64 be_l = be + mi - m;
                        const bool in = c > 0 && (pass == 0 ? nb_l < (uint32_t)P.tk : (double)be_l < goal);
                        const bool end = pass == 0 ? nb + ci >= (uint32_t)P.tk : !((double)(be + mi) < goal);
                        const unsigned has = __ballot_sync(0xffffffffu, in);
                        if (has) {
                            const int l = 31 - __clz(has);
                            sel = b0 + l;
                            sel_nb = __shfl_sync(0xffffffffu, nb_l, l);
                            sel_be = __shfl_sync(0xffffffffu, be_l, l);
                        }
                        over = __any_sync(0xffffffffu, end);
                        nb += __shfl_sync(0xffffffffu, ci, 31);
                        be += __shfl_sync(0xffffffffu, mi, 31);
                    }
                    if (lane == 0) {
                        // not over: the order ends further on, or (top-k) it keeps every token with a mass
                        int b = over && sel >= 0 ? (S.h.cnt[sel] <= (uint32_t)CAP ? sel : SLOW) : level == 0 ? GO_ON : pass == 0 ? ALL : SLOW;
                        S.bucket = b;
                        S.sel_mass = sel_be;
                        S.sel_cnt = sel_nb;
                        S.n_list = 0;
                        if (b == GO_ON) {
                            S.head_mass = be;
                            S.head_cnt = nb;
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
                if (!(f > -INFINITY) || bucket_of(f, level) != sel) continue;
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
                sort_list(S, ln);
                if (threadIdx.x == 0) {
                    u64 before = S.sel_mass;
                    const double goal = (double)P.tp * (double)held;
                    u64 c = 0;
                    for (int i = 0; i < ln; i++) {
                        const u64 e = S.h.list[i];
                        if (pass == 0 ? S.sel_cnt + i >= (uint32_t)P.tk : (!((double)before < goal) || e < cut)) break;
                        c = e;
                        before += R.mass(ukey_value((uint32_t)(e >> 32)));
                    }
                    if (c < cut) c = cut;  // (no token: the end that top-k gave)
                    S.cut = c;
                    S.sel_mass = before;
                    for (int q = 1; q < CS; q++) remote_st64(&S.cut, q, c);
                }
                __syncthreads();
                if (pass == 0) held = S.sel_mass;  // the mass of what top-k kept
                cut = S.cut;
                __syncthreads();
            }
        }
        sync_all();
        cut = S.cut;
    }

    // ---- 4: the kept mass of each warp's run of tokens, and the draw
    const uint32_t ck = (uint32_t)(cut >> 32), ci = ~(uint32_t)cut;
    const bool minp = P.mp > 0.0f && P.mp <= 1.0f;
    auto kept = [&](int i) -> u64 {
        const float f = L[i];
        const uint32_t k = ukey(f);
        if (k < ck || (k == ck && (uint32_t)(base + i) > ci)) return 0ull;
        const float w = R.weight(f);
        return minp && !(w >= P.mp) ? 0ull : __float2ull_rz(__fmul_rn(w, 1099511627776.0f));
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
    // CTAs a row: slices of 4,096 logits or more, up to eight; a slice fits shared memory
    int cs = 1;
    while (cs < hc::UC_MAX && V > cs * 4096) cs *= 2;
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
