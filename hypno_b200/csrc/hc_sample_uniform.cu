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
// k_sample_cluster: a cluster of up to 16 CTAs takes a row, each CTA a slice,
// each warp a run of it.  Passes over the logits (the first from memory, the
// others from L2): the maximum; the tokens near it (the head),
// where most orders end and few tokens are, into a list of each warp, by index
// (for top-p alone also the mass of all).  Then, from the lists: a histogram (for
// top-k by count, for top-p by mass over what top-k kept), the tokens of the
// bucket in which the order ends, gathered by the first CTA and sorted there,
// the kept mass of each warp, and the draw.  Where an order ends beyond the head, or
// keeps every token, the passes go over the logits instead of the lists; a
// bucket too full to sort (flat rows) is left to the first CTA and the kernel's
// slow path, a radix search over the logits' keys.  Nothing of a row stays in
// shared memory but the lists, so that several rows share an SM and one's
// serial parts (barriers, the first CTA's work) hide behind another's passes.
// Bound by latency: a row is a chain of 6 to 10 cluster barriers with the first
// CTA's work between them, and nothing is full even with 256 rows (43% of the issue
// slots, 12% of DRAM).  A row of 49,152 logits: 18 us; 32 rows of 128,256: 35 to
// 48 us; 256 rows: 120 to 146 us, 0.9 to 1.1 TB/s of logits.
#include "hc_internal.h"
#include "hc_common.cuh"

#include <cfloat>

namespace hc {

namespace {

constexpr int UT = 256;    // threads
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
constexpr int HB2 = 256;           // buckets of a histogram (the first CTA reads everyone's)
static_assert(HB2 == UT, "a bucket a thread");
// Distances (max - l) / T that the two histograms cover: up to the head's end and
// from there to TAIL, where weights are below 2^-40.  The head ends NEAR below the
// maximum in logits (a language model has some thousands of tokens there), and
// between weights of 3e-4 and 2e-12.
constexpr float NEAR = 12.0f, HEAD_MIN = 8.0f, HEAD_MAX = 27.0f, TAIL = 28.0f;
constexpr int CAP = 1024;          // tokens of a bucket that are sorted
constexpr int WCAP = 512;          // tokens of a warp's list
constexpr int FINER = -3, GO_ON = -2, ALL = -1, SLOW = HB2;  // instead of a bucket

struct __align__(16) CShared {
    union {
        UShared slow;
        struct {
            u64 sum[HB2];
            uint32_t cnt[HB2];
            u64 list[CAP];         // gathered tokens, key above ~index (first CTA)
            u64 sorted[UT];
            float near_l[UW][WCAP];  // the warps' lists: logits, indices
            uint32_t near_i[UW][WCAP];
        } h;
    };
    u64 red[32];
    uint32_t redu[32];
    // what the CTAs of the cluster tell one another, one word for each
    uint32_t c_max[UC_MAX], c_at[UC_MAX];
    u64 c_mass[UC_MAX];
    // what the first CTA tells all
    int n_list;
    int bucket, within;            // what the histogram gave; the bucket that a finer one divides
    u64 cut;                       // the last token kept: key above ~index
    // the first CTA's own
    u64 sel_mass, base_mass;       // mass before the bucket; before the histogram
    uint32_t sel_cnt, base_cnt;    // likewise tokens
    u64 w_mass[UW];                // of the warps' buckets
    uint32_t w_cnt[UW];
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
// (Not the .aligned forms: they are undefined for a warp whose lanes have not met
// again after a branch, which the compiler does not promise at inline assembly.)
__device__ __forceinline__ void cluster_barrier() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// The two halves apart: the first access of another CTA's shared memory comes
// after that CTA has begun, which nothing else promises.
__device__ __forceinline__ void cluster_begun() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
}
__device__ __forceinline__ void cluster_all_begun() {
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
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
    if (n <= UT) {
        if ((int)threadIdx.x < n) {
            const u64 e = S.h.list[threadIdx.x];
            int at = 0;
            for (int j = 0; j < n; j++) at += S.h.list[j] > e;
            S.h.sorted[at] = e;
        }
        __syncthreads();
        return S.h.sorted;
    }
    int m = 2 * UT;
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

static_assert(4 * (sizeof(CShared) + 1024) <= 228 * 1024, "four CTAs an SM");

__global__ void __launch_bounds__(UT, 4) k_sample_cluster(const float* __restrict__ logits, size_t ld, int V, int slice,
                                                          const float* __restrict__ u, const float* __restrict__ temp,
                                                          const int* __restrict__ top_k, const float* __restrict__ top_p,
                                                          const float* __restrict__ min_p, int32_t* __restrict__ out,
                                                          float* __restrict__ logprob, int CS) {
    extern __shared__ __align__(16) uint8_t smem[];
    CShared& S = *reinterpret_cast<CShared*>(smem);
    const int rank = CS > 1 ? (int)cluster_rank() : 0, row = blockIdx.x / CS;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto sync_all = [&]() {
        if (CS > 1) cluster_barrier();
        else __syncthreads();
    };
    if (CS > 1) cluster_begun();
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
    // Finite for every T: 1 / T overflows below 2^-128, and the maximum's exponent would be 0 * inf.
    R.inv = T > 0.0f ? fminf(__fdiv_rn(1.0f, T), FLT_MAX) : 1.0f;

    // Places are counted from the 16-byte boundary at or before the row's first
    // logit: place = index + off.  A warp has the run [w0, w1) of places, 128 at
    // a time, four a lane.
    const int off = (int)(((uintptr_t)R.l & 15) >> 2), places = V + off;
    const int per = slice / UW;  // (a multiple of 128)
    const int w0 = min(rank * slice + warp * per, places), w1 = min(w0 + per, places);
    const float* P0 = R.l - off;  // (never read below off)
    auto get4 = [&](int j, float* v) {
        if (j >= off && j + 4 <= places) {
            const float4 x = *reinterpret_cast<const float4*>(P0 + j);
            v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
        } else {
#pragma unroll
            for (int y = 0; y < 4; y++) v[y] = j + y >= off && j + y < places ? P0[j + y] : -INFINITY;
        }
    };

    // A later cluster's slice on its way to L2 while this one is worked on: the
    // one that will follow when four CTAs an SM have gone by.
    {
        const int64_t later = (int64_t)blockIdx.x / CS + 148 * 4 / CS;
        if (later < (int64_t)(gridDim.x / CS)) {
            const float* q = logits + (size_t)later * ld - off;
            for (int j = w0 + lane * 32; j < w1; j += 32 * 32)
                if (j >= off) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + j));
        }
    }

    // ---- 1: the maximum
    float top = -INFINITY;  // (NaN never wins)
    {
        int j = w0 + lane * 4;
        for (; j + 3 * 128 < w1; j += 4 * 128) {
            float v[4][4];
#pragma unroll
            for (int x = 0; x < 4; x++) get4(j + x * 128, v[x]);
#pragma unroll
            for (int x = 0; x < 4; x++) top = fmaxf(fmaxf(fmaxf(top, v[x][0]), fmaxf(v[x][1], v[x][2])), v[x][3]);
        }
        for (; j < w1; j += 128) {
            float v[4];
            get4(j, v);
            top = fmaxf(fmaxf(fmaxf(top, v[0]), fmaxf(v[1], v[2])), v[3]);
        }
    }
    uint32_t kmax = __reduce_max_sync(0xffffffffu, ukey(top));
    if (lane == 0) S.redu[warp] = kmax;
    if (threadIdx.x == 0) S.cut = 1ull << 32;  // keys from 1 on: every token
    __syncthreads();
    kmax = __reduce_max_sync(0xffffffffu, lane < UW ? S.redu[lane] : 0u);
    if (CS > 1) cluster_all_begun();
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
        if (__any_sync(0xffffffffu, top == R.mx)) {
            for (int j = w0 + lane * 4; j < w1; j += 128) {
                float v[4];
                get4(j, v);
#pragma unroll
                for (int y = 3; y >= 0; y--)
                    if (v[y] == R.mx) at = min(at, (uint32_t)(j + y - off));
            }
        }
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
    if (R.mx == INFINITY) {  // differences of infinities are left to the slow path
        if (rank == 0) sample_row(R, P, S.slow, out + row, logprob ? logprob + row : nullptr);
        return;
    }
    const float headd = fminf(fmaxf(NEAR * R.inv, HEAD_MIN), HEAD_MAX), step0 = HB2 / headd, step1 = HB2 / (TAIL - headd);
    // -(max - l) / T, the exponent of a weight; its bucket in histogram 0 or 1,
    // monotone in l, -1 outside it
    auto expo = [&](float f) -> float { return __fmul_rn(__fsub_rn(f, R.mx), R.inv); };
    auto bucket_at = [&](float x, int level) -> int {
        if (level == 0) return -x < headd ? min((int)(-x * step0), HB2 - 1) : -1;
        return -x >= headd && -x < TAIL ? min((int)((-x - headd) * step1), HB2 - 1) : -1;
    };
    // within >= 0: the places in a finer histogram of that bucket, -1 outside it
    auto place = [&](float x, int level, int within) -> int {
        const int b = bucket_at(x, level);
        if (within < 0) return b;
        if (b != within) return -1;
        const float step = level ? step1 : step0, lo = (level ? headd : 0.0f) + (float)within / step;
        return min(max((int)((-x - lo) * step * HB2), 0), HB2 - 1);
    };

    const bool by_k = P.tk > 0 && P.tk < V, by_p = P.tp < 1.0f && P.tk != 1;
    u64 cut = 1ull << 32;
    // What is kept so far: logits above kf, and equal ones up to index ki.
    float kf = -FLT_MAX;
    uint32_t ki = 0xffffffffu;
    auto in_head = [&](float f, uint32_t i) -> bool { return f >= kf && !(f == kf && i > ki); };
    // fn(logit, index) for this warp's tokens, by index over a lane's own; from the
    // list where all that matter are in it.
    int listed = 0;       // tokens in the warp's list, WCAP + 1 for more than it holds
    bool near = false;    // only tokens of the head matter
    auto each = [&](auto fn) {
        if (near && listed <= WCAP) {
            for (int e = lane; e < listed; e += 32) fn(S.h.near_l[warp][e], S.h.near_i[warp][e]);
        } else {
            for (int j = w0 + lane * 4; j < w1; j += 128) {
                float v[4];
                get4(j, v);
#pragma unroll
                for (int y = 0; y < 4; y++) fn(v[y], (uint32_t)(j + y - off));
            }
        }
    };
    if (by_k || by_p) {
        // ---- 2: the lists, and for top-p alone the mass
        u64 mass = 0;
        for (int j0 = w0; j0 < w1; j0 += 128) {
            float v[4];
            get4(j0 + lane * 4, v);
            unsigned b[4];
            bool any = false;
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const float x = expo(v[y]);
                b[y] = __ballot_sync(0xffffffffu, -x < headd);
                any = any || b[y];
                if (!by_k) mass += v[y] >= -FLT_MAX ? mass_of(expf(x)) : 0ull;
            }
            if (any) {
                const unsigned lt = (1u << lane) - 1u;
                int at = listed + __popc(b[0] & lt) + __popc(b[1] & lt) + __popc(b[2] & lt) + __popc(b[3] & lt);
#pragma unroll
                for (int y = 0; y < 4; y++)
                    if ((b[y] >> lane) & 1u) {
                        if (at < WCAP) {
                            S.h.near_l[warp][at] = v[y];
                            S.h.near_i[warp][at] = (uint32_t)(j0 + lane * 4 + y - off);
                        }
                        at++;
                    }
                listed = min(listed + __popc(b[0]) + __popc(b[1]) + __popc(b[2]) + __popc(b[3]), WCAP + 1);
                if (listed > WCAP && by_k) break;
            }
        }
        __syncwarp();
        if (!by_k) {
            mass = block_sum(mass);
            if (threadIdx.x == 0) remote_st64(&S.c_mass[rank], 0, mass);
        }
        u64 held = 0;          // (first CTA) the mass of which top_p is a share
        bool cut_near = false; // the end found last is within the head
        // Two ends may have to be found: top-k's by count, then top-p's by mass.
        for (int pass = by_k ? 0 : 1; pass < (by_p ? 2 : 1); pass++) {
            int level = 0, within = -1;
            if (rank == 0 && threadIdx.x == 0) {
                S.base_mass = 0ull;
                S.base_cnt = 0u;
            }
            for (int round = 0; round < 3; round++) {  // the head, the rest, a finer one
                // ---- 3: the histogram: counts, and for top-p masses
                for (int b = threadIdx.x; b < HB2; b += UT) {
                    S.h.sum[b] = 0ull;
                    S.h.cnt[b] = 0u;
                }
                __syncthreads();
                // (what top-k kept has its mass taken here, near or not)
                const bool first = level == 0 && within < 0;
                near = level == 0 && (pass == 0 || !by_k || cut_near || !first);
                u64 m2 = 0;
                each([&](float f, uint32_t i) {
                    if (!in_head(f, i)) return;
                    const float x = expo(f);
                    const int b = place(x, level, within);
                    if (pass == 0) {
                        if (b >= 0) atomicAdd(&S.h.cnt[b], 1u);
                        return;
                    }
                    if (b < 0 && (!first || !by_k)) return;
                    const u64 m = mass_of(expf(x));
                    m2 += m;
                    if (b >= 0) {
                        atomicAdd(&S.h.cnt[b], 1u);
                        atomicAdd(&S.h.sum[b], m);
                    }
                });
                if (pass == 1 && first && by_k) {
                    m2 = block_sum(m2);
                    if (threadIdx.x == 0) remote_st64(&S.c_mass[rank], 0, m2);
                }
                sync_all();
                if (rank == 0) {  // the first CTA adds the histograms up
                    if (pass == 1 && first)
                        for (int c = 0; c < CS; c++) held += S.c_mass[c];
                    {
                        const int b = threadIdx.x;
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
                    // the last bucket that holds a token of the order's head: a bucket a thread
                    const double goal = (double)P.tp * (double)held;
                    const uint32_t c = S.h.cnt[threadIdx.x];
                    const u64 m = S.h.sum[threadIdx.x];
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
                    if (lane == 31) {
                        S.w_cnt[warp] = ci;
                        S.w_mass[warp] = mi;
                    }
                    if (threadIdx.x == 0) {
                        S.bucket = -1;
                        S.n_list = 0;
                    }
                    __syncthreads();
                    uint32_t nb = S.base_cnt, all_n = nb;
                    u64 be = S.base_mass, all_m = be;
                    for (int w = 0; w < UW; w++) {
                        if (w < warp) {
                            nb += S.w_cnt[w];
                            be += S.w_mass[w];
                        }
                        all_n += S.w_cnt[w];
                        all_m += S.w_mass[w];
                    }
                    nb += ci - c;
                    be += mi - m;
                    const bool over = pass == 0 ? all_n >= (uint32_t)P.tk : !((double)all_m < goal);
                    const int mine = c > 0 && (pass == 0 ? nb < (uint32_t)P.tk : (double)be < goal) ? (int)threadIdx.x : -1;
                    const int best = __reduce_max_sync(0xffffffffu, mine);
                    if (lane == 0 && best >= 0) atomicMax(&S.bucket, best);
                    __syncthreads();
                    const int sel = S.bucket;
                    __syncthreads();
                    if (over && sel >= 0 ? mine == sel : threadIdx.x == 0) {
                        // not over: the order ends further on, or (top-k) it keeps every token with a mass
                        int b;
                        if (over && sel >= 0) {
                            b = c <= (uint32_t)CAP ? sel : within < 0 ? FINER : SLOW;
                            S.sel_mass = be;
                            S.sel_cnt = nb;
                            if (b == FINER) {
                                S.base_mass = be;
                                S.base_cnt = nb;
                            }
                        } else {
                            b = level == 0 && within < 0 ? GO_ON : pass == 0 && within < 0 ? ALL : SLOW;
                            if (b == GO_ON) {
                                S.base_mass = all_m;
                                S.base_cnt = all_n;
                            }
                        }
                        S.bucket = b;
                        S.within = sel;
                        for (int q = 1; q < CS; q++) remote_st32(&S.within, q, (uint32_t)sel);
                        for (int q = 1; q < CS; q++) remote_st32(&S.bucket, q, (uint32_t)b);
                    }
                }
                sync_all();
                const int got = S.bucket;
                if (got != GO_ON && got != FINER) break;
                if (got == GO_ON) level = 1;
                else within = S.within;
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
            // ---- 4: the bucket's tokens, to the first CTA
            near = level == 0;
            each([&](float f, uint32_t i) {
                if (!in_head(f, i) || place(expo(f), level, within) != sel) return;
                uint32_t at;
                asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(CS > 1 ? remote(&S.n_list, 0) : smem_u32(&S.n_list)) : "memory");
                if (at >= (uint32_t)CAP) return;
                const u64 e = (u64)ukey(f) << 32 | (uint32_t)~i;
                if (CS > 1) remote_st64(&S.h.list[at], 0, e);
                else S.h.list[at] = e;
            });
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
            cut_near = level == 0;
        }
        near = cut_near;
    }

    // ---- 5: the kept mass of each warp, and the draw
    const float least = P.mp <= 1.0f ? P.mp : 0.0f;
    auto kept = [&](float f, uint32_t i) -> u64 {
        if (!in_head(f, i)) return 0ull;
        const float w = expf(expo(f));
        return w >= least ? mass_of(w) : 0ull;
    };
    u64 mine = 0;
    each([&](float f, uint32_t i) { mine += kept(f, i); });
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
    // this warp's: its tokens in order, one a lane from the list, four a lane from the logits
    const bool list = near && listed <= WCAP;
    const int end = list ? listed : w1, stride = list ? 32 : 128;
    float v[4], next[4];
    if (!list) get4(w0 + lane * 4, next);
    for (int j0 = list ? 0 : w0; j0 < end; j0 += stride) {
        u64 m[4] = {0, 0, 0, 0};
        uint32_t i = 0;
        if (list) {
            if (j0 + lane < listed) m[0] = kept(S.h.near_l[warp][j0 + lane], i = S.h.near_i[warp][j0 + lane]);
        } else {
            const int j = j0 + lane * 4;
            i = (uint32_t)(j - off);
#pragma unroll
            for (int y = 0; y < 4; y++) v[y] = next[y];
            if (j0 + stride < end) get4(j + 128, next);
#pragma unroll
            for (int y = 0; y < 4; y++) m[y] = j + y < w1 ? kept(v[y], i + y) : 0ull;
        }
        const u64 sum = (m[0] + m[1]) + (m[2] + m[3]);
        u64 incl = sum;
        for (int o = 1; o < 32; o <<= 1) {
            const u64 t = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += t;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, below + incl > goal);
        if (hit) {
            if (lane == __ffs(hit) - 1) {
                u64 run = below + incl - sum;
                int y = 0;
                while (y < 3 && run + m[y] <= goal) run += m[y++];
                out[row] = (int)(i + y);
                if (logprob) logprob[row] = logf((float)((double)m[y] / (double)total));
            }
            return;
        }
        below += __shfl_sync(0xffffffffu, incl, 31);
    }
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
    HC_CHECK((uintptr_t)logits_dev % 4 == 0, HC_ERR_INVALID, "hc_sample_uniform_dev: misaligned logits");
    cudaStream_t s = (cudaStream_t)stream;
    // CTAs a row, of slices of 4,096 logits or more: eight, sixteen where each has
    // an SM of its own.  128,256 logits, top-k 50 and top-p, us, 4 / 8 / 16 CTAs:
    // 8 rows 99 / 61 / 43, 32 rows 102 / 64 / 86, 64 rows 108 / 76, 256 rows
    // 257 / 291 / 435; 256 rows of different settings (greedy, top-k, top-p, min-p,
    // none) 182 / 128: more CTAs a row even out rows that take unlike times.
    int cs = 1;
    while (cs < 8 && V > cs * 4096) cs *= 2;
    if ((int64_t)B * 16 <= 148 && V > 8 * 4096) cs = 16;
    const int runs = cs * hc::UW * 128;                       // a warp's run is a multiple of 128 places
    const int slice = (int)(((int64_t)V + 3 + runs - 1) / runs) * hc::UW * 128;
    const size_t smem = sizeof(hc::CShared);
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
