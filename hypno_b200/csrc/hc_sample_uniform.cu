// The next token from the caller's uniform numbers: temperature, top-k, top-p
// and min-p over B rows of logits, one CTA per row.
//
// Weights w_i = exp((l_i - max) * (1 / T)) are held as whole multiples of
// 2^-40 (64-bit integers; the largest is 2^40): integer sums do not depend on
// their order, so histograms may add by atomics and every thread layout gives
// the same token.  A weight below 2^-40 of the largest is 0 and can never be
// drawn.  The kept set is a head of the order (logit descending, index
// ascending), so it is described by a key and a number of ties: every token
// above the key, and the first `ties` tokens at the key, by index.
#include "hc_internal.h"
#include "hc_common.cuh"

namespace hc {

namespace {

constexpr int UT = 1024;   // threads
constexpr int UB = 2048;   // buckets of a radix pass
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
    u64 t = S.red[threadIdx.x & 31];
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

__global__ void __launch_bounds__(UT) k_sample_uniform(const float* __restrict__ logits, size_t ld, int V,
                                                       const float* __restrict__ u, const float* __restrict__ temp,
                                                       const int* __restrict__ top_k, const float* __restrict__ top_p,
                                                       const float* __restrict__ min_p, int32_t* __restrict__ out,
                                                       float* __restrict__ logprob) {
    __shared__ UShared S;
    const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    URow R;
    R.l = logits + (size_t)row * ld;
    R.V = V;
    const float T = temp[row], tp = top_p[row], mp = min_p[row];
    int tk = top_k[row];
    R.inv = T > 0.0f ? __fdiv_rn(1.0f, T) : 1.0f;
    if (!(T > 0.0f) || !(tp > 0.0f) || !(mp <= 1.0f)) tk = 1;  // only the first token can be kept

    uint32_t kmax = 0;
    for (int i = threadIdx.x; i < V; i += UT) kmax = max(kmax, ukey(R.l[i]));
    kmax = __reduce_max_sync(0xffffffffu, kmax);
    if (lane == 0) S.redu[warp] = kmax;
    __syncthreads();
    kmax = __reduce_max_sync(0xffffffffu, S.redu[lane]);
    if (kmax == 0) {  // nothing above -inf
        if (threadIdx.x == 0) {
            out[row] = -1;
            if (logprob) logprob[row] = -INFINITY;
        }
        return;
    }
    R.mx = ukey_value(kmax);

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
    for (int w = 0; w < 32; w++) {
        if (w < warp) base += S.red[w];
        total += S.red[w];
    }
    incl += base;
    const float uf = u[row];
    const double g = (uf >= 0.0f ? (double)uf : 0.0) * (double)total;
    u64 goal = (u64)floor(fmin(g, 9.0e18));
    if (goal >= total) goal = total - 1;
    if (goal < incl && goal >= incl - mine) {
        u64 run = incl - mine;
        for (int i = i0; i < i1; i++) {
            const u64 m = kept(i);
            run += m;
            if (run > goal) {
                out[row] = i;
                if (logprob) logprob[row] = logf((float)((double)m / (double)total));
                break;
            }
        }
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
    hc::k_sample_uniform<<<(unsigned)B, hc::UT, 0, (cudaStream_t)stream>>>(logits_dev, ld, V, u_dev, temperature_dev,
                                                                          top_k_dev, top_p_dev, min_p_dev, out_dev,
                                                                          logprob_dev);
    HC_LAUNCH_CHECK();
    return HC_OK;
}
