// Paged KV cache: the append kernel (rotation of keys and queries on the way
// into the pages), the attention kernel that takes every shape, and the C
// entry points with their checks of arguments.
#include "hc_paged.h"

#include <climits>

namespace hc {

namespace {

// ============================================================ append

__device__ __forceinline__ int seq_of_row(const PagedArgs& P, int r) {
    int lo = 0, hi = P.n_seqs - 1;  // the last sequence whose first row is <= r
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (__ldg(P.q_start + mid) <= r) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// 16-byte groups.  A unit is eight elements of a head: four pairs, which lie
// side by side (adjacent) or in two runs of four (halves), or eight elements
// past rot or of v, which pass through.  A thread takes one unit, a row's units
// are dealt over blocks; a thread's loads are in flight before the row's place
// in the cache (three dependent loads: row start, length, page) is known.
// Bound by its bytes: q is read and written, k and v are read and stored.
// (Three units a thread, with as many loads in flight, took 63 us where one
// takes 60: 8,192 rows of 32 + 8 + 8 heads of 128, f32 into FP16, 369 MB at
// 6.2 TB/s; 32 rows: 3.9 against 3.3.)
template <typename T>
__device__ __forceinline__ void load4(const T* p, float* v) {
    if constexpr (sizeof(T) == 4) {
        const float4 x = __ldcs(reinterpret_cast<const float4*>(p));
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
        const uint2 x = __ldcs(reinterpret_cast<const uint2*>(p));
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&x.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&x.y));
        v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
    }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float* v) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
        *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
}

constexpr int AP_THREADS = 256;

template <typename T, typename C>
__global__ void __launch_bounds__(AP_THREADS) k_paged_append_vec(AppendArgs A) {
    const PagedArgs& P = A.p;
    const int row = blockIdx.x, hu = P.hd >> 3, half = A.rot >> 1;
    const int unit = blockIdx.y * AP_THREADS + threadIdx.x;
    if (unit >= (A.nh + 2 * P.nkv) * hu) return;
    int head = unit / hu;
    const int u = unit - head * hu;
    const bool is_q = head < A.nh, is_v = head >= A.nh + P.nkv;
    if (!is_q) head -= is_v ? A.nh + P.nkv : A.nh;
    const bool rotated = 8 * u < A.rot && !is_v;
    int i0 = 8 * u, i1 = i0 + 4;  // first elements of the two runs of four
    if (A.halves && i0 < A.rot) {
        i0 = 4 * u;
        i1 = i0 + half;
    }
    const T* src = is_q   ? (const T*)A.q + row * A.q_rs + head * A.q_hs
                   : is_v ? (const T*)A.v + row * A.v_rs + head * A.v_hs
                          : (const T*)A.k + row * A.k_rs + head * A.k_hs;
    float x[8];
    load4(src + i0, x);
    load4(src + i1, x + 4);
    const int seq = seq_of_row(P, row);
    int r0, r1;
    seq_rows(P, seq, r0, r1);
    if (row < r0 || row >= r1) return;
    const int pos = seq_len(P, seq) - (r1 - r0) + (row - r0);
    if (rotated) {
        const float2* cs = A.rope + (int64_t)min(max(pos, 0), A.rope_rows - 1) * half + (A.halves ? i0 : i0 >> 1);
        const float4 c01 = __ldg(reinterpret_cast<const float4*>(cs)), c23 = __ldg(reinterpret_cast<const float4*>(cs + 2));
        const float c[4] = {c01.x, c01.z, c23.x, c23.z}, s[4] = {c01.y, c01.w, c23.y, c23.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            // static places: a pair is (i, i + 4) or (2 i, 2 i + 1)
            const float a = A.halves ? x[i] : x[2 * i], b = A.halves ? x[i + 4] : x[2 * i + 1];
            const float ra = a * c[i] - b * s[i], rb = a * s[i] + b * c[i];
            if (A.halves) x[i] = ra, x[i + 4] = rb;
            else x[2 * i] = ra, x[2 * i + 1] = rb;
        }
    }
    if (is_q) {
        T* dst = (T*)A.qo + row * A.o_rs + head * A.o_hs;
        store4(dst + i0, x);
        store4(dst + i1, x + 4);
        return;
    }
    if (pos < 0) return;
    int slot;
    const int page = lookup(P, seq, pos, slot);
    if (page < 0) return;
    C* dst = is_v ? (C*)P.v + page * P.vps + head * P.vhs + slot * P.vss : (C*)P.k + page * P.kps + head * P.khs + slot * P.kss;
    store4(dst + i0, x);
    store4(dst + i1, x + 4);
}

// Any head size and alignment (8,192 rows of 32 + 8 + 8 heads of 66: 85 us): one thread per pair of a head,
// (x0, x1) -> (x0 c - x1 s, x0 s + x1 c) for the pairs of the first rot
// elements, copies for the others and for v.
template <typename T, typename C>
__global__ void __launch_bounds__(256) k_paged_append(AppendArgs A) {
    const PagedArgs& P = A.p;
    const int row = blockIdx.x;
    const int hp = (P.hd + 1) >> 1;  // pairs of a head (an odd head ends with a lone element)
    const int unit = blockIdx.y * blockDim.x + threadIdx.x;
    if (unit >= (A.nh + 2 * P.nkv) * hp) return;
    int head = unit / hp;
    const int j = unit - head * hp;
    const int seq = seq_of_row(P, row);
    int r0, r1;
    seq_rows(P, seq, r0, r1);
    if (row < r0 || row >= r1) return;
    const int pos = seq_len(P, seq) - (r1 - r0) + (row - r0);
    int i0 = 2 * j, i1 = 2 * j + 1;
    const int half = A.rot >> 1;
    const bool rotated = j < half;
    if (rotated && A.halves) {
        i0 = j;
        i1 = j + half;
    }
    const bool two = i1 < P.hd;
    const T* src;
    const bool is_q = head < A.nh, is_v = !is_q && head >= A.nh + P.nkv;
    if (is_q) src = (const T*)A.q + row * A.q_rs + head * A.q_hs;
    else if (!is_v) src = (const T*)A.k + row * A.k_rs + (head -= A.nh) * A.k_hs;
    else src = (const T*)A.v + row * A.v_rs + (head -= A.nh + P.nkv) * A.v_hs;
    float a = to_f32(src[i0]), b = two ? to_f32(src[i1]) : 0.0f;
    if (rotated && !is_v) {
        const float2 cs = __ldg(A.rope + (int64_t)min(max(pos, 0), A.rope_rows - 1) * half + j);
        const float x = a * cs.x - b * cs.y;
        b = a * cs.y + b * cs.x;
        a = x;
    }
    if (is_q) {
        T* dst = (T*)A.qo + row * A.o_rs + head * A.o_hs;
        dst[i0] = from_f32<T>(a);
        if (two) dst[i1] = from_f32<T>(b);
        return;
    }
    if (pos < 0) return;
    int slot;
    const int page = lookup(P, seq, pos, slot);
    if (page < 0) return;
    C* dst = is_v ? (C*)P.v + page * P.vps + head * P.vhs + slot * P.vss
                  : (C*)P.k + page * P.kps + head * P.khs + slot * P.kss;
    dst[i0] = from_f32<C>(a);
    if (two) dst[i1] = from_f32<C>(b);
}

// ============================================================ attention, any shape

// One CTA per (32 packed rows of a sequence, KV head): key tiles of 32 in
// shared memory as f32, running maximum m and sum l of each row, and
//   m' = max(m, s), l' = l e^(m - m') + sum e^(s - m'), o' = o e^(m - m') + sum e^(s - m') v.
// Masked keys take no part (they are skipped, not multiplied by 0, so that
// whatever lies behind the mask cannot reach a row).  Eight threads share a
// row: keys t, t + 8, ... of a tile and columns t, t + 8, ... of the output.
// Bound by shared-memory reads (five for four multiply-adds); the shapes the
// tensor-core kernels take do not come here (8 single tokens over 4,096 FP16
// positions, 16 heads over 8 of 256, took 6.7 ms here and take 72 us there).
constexpr int GM = 32, GN = 32, GT = 256;

// LIST: a tile holds query heads of one token, whose keys are the positions of
// its listed pages one after another.
template <typename T, typename C, int HDMAX, bool LIST>
__global__ void __launch_bounds__(GT) k_paged_generic(PagedAttnArgs A, PagedList L) {
    const PagedArgs& P = A.p;
    extern __shared__ float sm[];
    const int hd = P.hd, ldk = hd + 1;
    float* Q = sm;                 // [GM][ldk]
    float* K = Q + GM * ldk;       // [GN][ldk]
    float* V = K + GN * ldk;       // [GN][ldk]
    float* S = V + GN * ldk;       // [GM][GN + 1]
    __shared__ int s_seq, s_tile, s_ok;
    __shared__ int64_t s_ko[GN], s_vo[GN];  // element offsets of the tile's positions, -1 for none
    const int kvh = blockIdx.y;
    if (threadIdx.x < 32) {
        int a = 0, b = 0;
        bool ok;
        if constexpr (LIST) {
            const int tg = (A.G + GM - 1) / GM;
            ok = find_tile(P, tg, 1, blockIdx.x, a, b);
        } else {
            ok = find_tile(P, A.G, GM, blockIdx.x, a, b);
        }
        if (threadIdx.x == 0) {
            s_ok = ok;
            s_seq = a;
            s_tile = b;
        }
    }
    __syncthreads();
    if (!s_ok) return;
    const int seq = s_seq;
    int r0, r1;
    seq_rows(P, seq, r0, r1);
    const int T_b = r1 - r0;
    int m0 = s_tile * GM, mrows = min(GM, T_b * A.G - m0);
    if constexpr (LIST) {
        const int tg = (A.G + GM - 1) / GM, g0 = (s_tile % tg) * GM;
        m0 = s_tile / tg * A.G + g0;
        mrows = min(GM, A.G - g0);
    }
    const int first = seq_len(P, seq) - T_b;  // position of the sequence's first row
    for (int i = threadIdx.x; i < mrows * hd; i += GT) {
        const int m = i / hd, d = i - m * hd, row = token_of(A, m0 + m), g = (m0 + m) - row * A.G;
        Q[m * ldk + d] = to_f32(((const T*)A.q)[(r0 + row) * A.q_rs + (kvh * A.G + g) * A.q_hs + d]) * A.scale;
    }
    const int m = threadIdx.x >> 3, t = threadIdx.x & 7;
    const int pos = m < mrows ? first + token_of(A, m0 + m) : -1;
    const int lo = A.window > 0 ? max(0, pos - A.window + 1) : 0;
    int begin, end;  // positions seen by the tile
    const int p_own = first + token_of(A, m0);
    const int32_t* list = nullptr;
    if constexpr (LIST) {
        const int lrow = r0 + token_of(A, m0);
        list = L.pages + lrow * L.row_stride + kvh * L.head_stride;
        begin = 0;
        end = (int)min((int64_t)min(list_count(L, lrow, kvh), pages_seen(P, p_own)) * P.page_size, (int64_t)0x7fffff00);
    } else {
        visible(A, first, m0, mrows, begin, end);
        begin = begin / GN * GN;
    }
    float o[HDMAX / 8];
#pragma unroll
    for (int i = 0; i < HDMAX / 8; i++) o[i] = 0.0f;
    float mx = -INFINITY, l = 0.0f;
    for (int j0 = begin; j0 < end; j0 += GN) {
        __syncthreads();
        if (threadIdx.x < GN) {
            const int j = j0 + threadIdx.x;
            int slot = 0;
            int page = -1;
            if (j < end) {
                if constexpr (LIST) page = lookup_listed(A, list, seq, j, p_own, slot);
                else page = lookup(P, seq, j, slot);
            }
            s_ko[threadIdx.x] = page < 0 ? -1 : page * P.kps + kvh * P.khs + slot * P.kss;
            s_vo[threadIdx.x] = page < 0 ? -1 : page * P.vps + kvh * P.vhs + slot * P.vss;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < GN * hd; i += GT) {
            const int n = i / hd, d = i - n * hd;
            const bool in = s_ko[n] >= 0;
            K[n * ldk + d] = in ? to_f32(((const C*)P.k)[s_ko[n] + d]) : 0.0f;
            V[n * ldk + d] = in ? to_f32(((const C*)P.v)[s_vo[n] + d]) : 0.0f;
        }
        __syncthreads();
        float s[GN / 8];
#pragma unroll
        for (int i = 0; i < GN / 8; i++) s[i] = 0.0f;
        for (int d = 0; d < hd; d++) {
            const float qv = Q[m * ldk + d];
#pragma unroll
            for (int i = 0; i < GN / 8; i++) s[i] = fmaf(qv, K[(t + 8 * i) * ldk + d], s[i]);
        }
        float tm = mx;
#pragma unroll
        for (int i = 0; i < GN / 8; i++) {
            const int j = j0 + t + 8 * i;
            if ((!LIST && (j > pos || j < lo)) || s_ko[t + 8 * i] < 0) s[i] = -INFINITY;
            tm = fmaxf(tm, s[i]);
        }
#pragma unroll
        for (int d = 4; d > 0; d >>= 1) tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, d));
        const float base = tm == -INFINITY ? 0.0f : tm;  // nothing seen yet: every weight is e^-inf = 0
        const float f = expf(mx - base);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < GN / 8; i++) {
            const float p = expf(s[i] - base);
            S[m * (GN + 1) + t + 8 * i] = s[i] == -INFINITY ? -1.0f : p;  // -1: masked
            sum += p;
        }
#pragma unroll
        for (int d = 4; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        l = l * f + sum;
        mx = tm;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < HDMAX / 8; i++) o[i] *= f;
        for (int n = 0; n < GN; n++) {
            const float p = S[m * (GN + 1) + n];
            if (p < 0.0f) continue;
#pragma unroll
            for (int i = 0; i < HDMAX / 8; i++)
                if (t + 8 * i < hd) o[i] = fmaf(p, V[n * ldk + t + 8 * i], o[i]);
        }
        __syncwarp();
    }
    if (m >= mrows) return;
    const int row = r0 + token_of(A, m0 + m), head = kvh * A.G + (m0 + m) % A.G;
    const float inv = 1.0f / l;
    T* out = (T*)A.out + row * A.o_rs + head * A.o_hs;
#pragma unroll
    for (int i = 0; i < HDMAX / 8; i++)
        if (t + 8 * i < hd) out[t + 8 * i] = from_f32<T>(l == 0.0f ? 0.0f : o[i] * inv);
    if (A.lse && t == 0) A.lse[(int64_t)row * A.nh + head] = l == 0.0f ? -INFINITY : mx + logf(l);
}

template <typename T, typename C, bool LIST>
int launch_generic_t(const PagedAttnArgs& A, const PagedList& L, cudaStream_t s) {
    const int64_t tiles = LIST ? (int64_t)A.p.n_rows * ((A.G + GM - 1) / GM) : ((int64_t)A.p.n_rows * A.G) / GM + A.p.n_seqs;
    HC_CHECK(tiles <= 0x7fffffff, HC_ERR_INVALID, "paged attention: too many rows");
    const size_t smem = (size_t)((GM + 2 * GN) * (A.p.hd + 1) + GM * (GN + 1)) * sizeof(float);
    auto kfn = A.p.hd <= 128 ? k_paged_generic<T, C, 128, LIST> : k_paged_generic<T, C, 256, LIST>;
    HC_CUDA(cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    kfn<<<dim3((unsigned)tiles, (unsigned)A.p.nkv), GT, smem, s>>>(A, L);
    HC_LAUNCH_CHECK();
    return HC_OK;
}

template <bool LIST>
int launch_generic_list(const PagedAttnArgs& A, const PagedList& L, int q16, int c16, cudaStream_t s) {
    if (q16) return c16 ? launch_generic_t<__half, __half, LIST>(A, L, s) : launch_generic_t<__half, float, LIST>(A, L, s);
    return c16 ? launch_generic_t<float, __half, LIST>(A, L, s) : launch_generic_t<float, float, LIST>(A, L, s);
}

}  // namespace

int launch_paged_generic(const PagedAttnArgs& A, const PagedList& L, int q16, int c16, cudaStream_t s) {
    return L.width ? launch_generic_list<true>(A, L, q16, c16, s) : launch_generic_list<false>(A, L, q16, c16, s);
}

}  // namespace hc

// ============================================================ C entry points

namespace {

// A pool's own part of the arguments.
int pool_args(const char* who, const hc_paged_kv* kv, hc::PagedArgs& P, hc::PagedScales& C) {
    C = {};
    HC_CHECK(kv, HC_ERR_INVALID, "%s: NULL cache or batch", who);
    HC_CHECK(kv->kv_dtype == HC_KV_FP32 || kv->kv_dtype == HC_KV_FP16 || kv->kv_dtype == HC_KV_Q4, HC_ERR_UNSUPPORTED,
             "%s: kv_dtype %d", who, kv->kv_dtype);
    HC_CHECK(kv->n_pages >= 1 && kv->page_size >= 1 && kv->n_kv_heads >= 1 && kv->head_dim >= 1, HC_ERR_INVALID,
             "%s: empty cache (%d pages of %d positions, %d heads of %d)", who, kv->n_pages, kv->page_size,
             kv->n_kv_heads, kv->head_dim);
    HC_CHECK(kv->n_kv_heads <= 65535, HC_ERR_INVALID, "%s: %d KV heads", who, kv->n_kv_heads);
    HC_CHECK(kv->k && kv->v, HC_ERR_INVALID, "%s: NULL pool", who);
    HC_CHECK(kv->k_page_stride >= 0 && kv->k_head_stride >= 0 && kv->k_pos_stride >= 0 && kv->v_page_stride >= 0 &&
                 kv->v_head_stride >= 0 && kv->v_pos_stride >= 0,
             HC_ERR_INVALID, "%s: negative pool stride", who);
    const uintptr_t es = kv->kv_dtype == HC_KV_FP16 ? 2 : kv->kv_dtype == HC_KV_Q4 ? 16 : 4;
    HC_CHECK(((uintptr_t)kv->k | (uintptr_t)kv->v) % es == 0, HC_ERR_INVALID, "%s: misaligned pool", who);
    if (kv->kv_dtype == HC_KV_Q4) {
        const hc_paged_kv_q4* q = (const hc_paged_kv_q4*)kv;
        HC_CHECK(kv->head_dim % 32 == 0 && kv->head_dim <= 256, HC_ERR_UNSUPPORTED,
                 "%s: head_dim %d of a cache in 4 bits (a multiple of 32, at most 256)", who, kv->head_dim);
        HC_CHECK((kv->k_page_stride | kv->k_head_stride | kv->k_pos_stride | kv->v_page_stride | kv->v_head_stride | kv->v_pos_stride) % 16 == 0,
                 HC_ERR_INVALID, "%s: strides of codes in 4 bits that are not multiples of 16 bytes", who);
        const int64_t sl = hc::q4_slots(kv->head_dim);
        HC_CHECK(q->k_scale && q->v_scale && ((uintptr_t)q->k_scale | (uintptr_t)q->v_scale) % (2 * sl) == 0, HC_ERR_INVALID,
                 "%s: NULL or misaligned scales", who);
        const int64_t st[6] = {q->ks_page_stride, q->ks_head_stride, q->ks_pos_stride, q->vs_page_stride, q->vs_head_stride, q->vs_pos_stride};
        for (int64_t x : st)
            HC_CHECK(x >= 0 && x % sl == 0, HC_ERR_INVALID, "%s: a stride of %lld scales (a multiple of %lld)", who, (long long)x, (long long)sl);
        C = {(__half*)q->k_scale, (__half*)q->v_scale, st[0], st[1], st[2], st[3], st[4], st[5]};
    }
    P.k = kv->k;
    P.v = kv->v;
    P.kps = kv->k_page_stride;
    P.khs = kv->k_head_stride;
    P.kss = kv->k_pos_stride;
    P.vps = kv->v_page_stride;
    P.vhs = kv->v_head_stride;
    P.vss = kv->v_pos_stride;
    P.n_pages = kv->n_pages;
    P.page_size = kv->page_size;
    P.page_shift = -1;
    for (int i = 0; i < 31; i++)
        if (kv->page_size == (1 << i)) P.page_shift = i;
    P.nkv = kv->n_kv_heads;
    P.hd = kv->head_dim;
    return HC_OK;
}

int paged_args(const char* who, const hc_paged_kv* kv, const hc_paged_batch* b, hc::PagedArgs& P, hc::PagedScales& C) {
    HC_CHECK(kv && b, HC_ERR_INVALID, "%s: NULL cache or batch", who);
    HC_TRY(pool_args(who, kv, P, C));
    HC_CHECK(b->n_seqs >= 0 && b->n_rows >= 0 && b->max_pages >= 0 && b->max_q_len >= 0 && b->max_kv_len >= 0,
             HC_ERR_INVALID, "%s: negative size in the batch", who);
    HC_CHECK(b->n_seqs > 0 || b->n_rows == 0, HC_ERR_INVALID, "%s: %d rows of no sequence", who, b->n_rows);
    HC_CHECK(b->n_seqs == 0 || (b->q_start && b->kv_len && (b->block_table || b->max_pages == 0)), HC_ERR_INVALID,
             "%s: NULL batch array", who);
    HC_CHECK(b->table_stride >= b->max_pages || b->n_seqs <= 1, HC_ERR_INVALID,
             "%s: table rows of %d pages at stride %lld", who, b->max_pages, (long long)b->table_stride);
    P.table = b->block_table;
    P.q_start = b->q_start;
    P.kv_len = b->kv_len;
    P.table_stride = b->table_stride;
    P.n_seqs = b->n_seqs;
    P.max_pages = b->max_pages;
    P.n_rows = b->n_rows;
    P.reach = (int)std::min<int64_t>((int64_t)b->max_pages * kv->page_size, INT_MAX - 1024);  // (tiles are counted past it)
    return HC_OK;
}

int rows_ok(const char* who, const char* what, const hc_rows* r, uint32_t dtype) {
    HC_CHECK(r && r->data, HC_ERR_INVALID, "%s: NULL %s", who, what);
    HC_CHECK((uintptr_t)r->data % (dtype == HC_DTYPE_FP16 ? 2 : 4) == 0, HC_ERR_INVALID, "%s: misaligned %s", who, what);
    return HC_OK;
}

template <typename T, typename C>
int launch_append(const hc::AppendArgs& A, cudaStream_t s) {
    const hc::PagedArgs& P = A.p;
    // 16-byte groups: whole eights of elements and pairs, rows and pools aligned
    const int64_t et = 16 / (int64_t)sizeof(T), ec = 16 / (int64_t)sizeof(C);
    const bool vec = P.hd % 8 == 0 && A.rot % 8 == 0 &&
                     ((uintptr_t)A.k | (uintptr_t)A.v | (uintptr_t)A.q | (uintptr_t)A.qo | (uintptr_t)A.rope | (uintptr_t)P.k | (uintptr_t)P.v) % 16 == 0 &&
                     (A.k_rs | A.k_hs | A.v_rs | A.v_hs | (A.nh ? A.q_rs | A.q_hs | A.o_rs | A.o_hs : 0)) % et == 0 &&
                     (P.kps | P.khs | P.kss | P.vps | P.vhs | P.vss) % ec == 0;
    const int64_t units = vec ? (int64_t)(A.nh + 2 * P.nkv) * (P.hd / 8) : (int64_t)(A.nh + 2 * P.nkv) * ((P.hd + 1) / 2);
    HC_CHECK(units <= 65535 * 256ll, HC_ERR_INVALID, "hc_paged_append_dev: %d + %d heads of %d", A.nh, P.nkv, P.hd);
    if (vec) {
        hc::k_paged_append_vec<T, C><<<dim3((unsigned)P.n_rows, (unsigned)((units + 255) / 256)), 256, 0, s>>>(A);
    } else {
        hc::k_paged_append<T, C><<<dim3((unsigned)P.n_rows, (unsigned)((units + 255) / 256)), 256, 0, s>>>(A);
    }
    HC_LAUNCH_CHECK();
    return HC_OK;
}

}  // namespace

HC_EXPORT int hc_paged_append_dev(const hc_paged_kv* kv, const hc_paged_batch* batch, const hc_rows* k, const hc_rows* v,
                                  const hc_rows* q, const hc_rows* q_out, int n_heads, uint32_t dtype, const float* rope, int rope_rows,
                                  int rot_dim, int half_pairs, void* stream) {
    const char* who = "hc_paged_append_dev";
    hc::AppendArgs A;
    hc::PagedScales C;
    HC_TRY(paged_args(who, kv, batch, A.p, C));
    HC_CHECK(dtype == HC_DTYPE_FP32 || dtype == HC_DTYPE_FP16, HC_ERR_UNSUPPORTED, "%s: dtype %u", who, dtype);
    HC_CHECK(n_heads >= 0, HC_ERR_INVALID, "%s: n_heads %d", who, n_heads);
    HC_CHECK(half_pairs == 0 || half_pairs == 1, HC_ERR_INVALID, "%s: half_pairs %d", who, half_pairs);
    if (rope) {
        HC_CHECK(rot_dim >= 0 && rot_dim % 2 == 0 && rot_dim <= A.p.hd, HC_ERR_INVALID, "%s: rot_dim %d of head_dim %d",
                 who, rot_dim, A.p.hd);
        HC_CHECK(rope_rows >= 1 && batch->max_kv_len <= rope_rows, HC_ERR_INVALID,
                 "%s: the rotation table has %d positions, the batch up to %d", who, rope_rows, batch->max_kv_len);
        HC_CHECK((uintptr_t)rope % 8 == 0, HC_ERR_INVALID, "%s: misaligned rotation table", who);
    }
    if (batch->n_rows == 0) return HC_OK;
    HC_TRY(rows_ok(who, "k", k, dtype));
    HC_TRY(rows_ok(who, "v", v, dtype));
    if (q) {
        HC_CHECK(n_heads > 0, HC_ERR_INVALID, "%s: q without heads", who);
        HC_TRY(rows_ok(who, "q", q, dtype));
        HC_TRY(rows_ok(who, "q_out", q_out, dtype));
    }
    const hc_rows none = {nullptr, 0, 0};
    if (!q) q = q_out = &none;
    A.k = k->data;
    A.k_rs = k->row_stride;
    A.k_hs = k->head_stride;
    A.v = v->data;
    A.v_rs = v->row_stride;
    A.v_hs = v->head_stride;
    A.q = q->data;
    A.q_rs = q->row_stride;
    A.q_hs = q->head_stride;
    A.qo = q_out->data;
    A.o_rs = q_out->row_stride;
    A.o_hs = q_out->head_stride;
    A.rope = (const float2*)rope;
    A.rope_rows = rope_rows;
    A.rot = rope ? rot_dim : 0;
    A.halves = half_pairs;
    A.nh = q->data ? n_heads : 0;
    cudaStream_t s = (cudaStream_t)stream;
    if (kv->kv_dtype == HC_KV_Q4) return hc::launch_append_q4(A, C, dtype == HC_DTYPE_FP16, s);
    if (dtype == HC_DTYPE_FP16)
        return kv->kv_dtype == HC_KV_FP16 ? launch_append<__half, __half>(A, s) : launch_append<__half, float>(A, s);
    return kv->kv_dtype == HC_KV_FP16 ? launch_append<float, __half>(A, s) : launch_append<float, float>(A, s);
}

namespace {

struct AttnCall {
    hc::PagedAttnArgs a;
    hc::PagedScales c;
    hc::PagedList l;
};

int attn_checks(const char* who, const hc_paged_kv* kv, const hc_paged_batch* batch, const hc_page_lists* lists, int n_heads,
                uint32_t dtype, int window, AttnCall& X) {
    hc::PagedAttnArgs& A = X.a;
    HC_TRY(paged_args(who, kv, batch, A.p, X.c));
    HC_CHECK(dtype == HC_DTYPE_FP32 || dtype == HC_DTYPE_FP16, HC_ERR_UNSUPPORTED, "%s: dtype %u", who, dtype);
    HC_CHECK(A.p.hd <= 256, HC_ERR_UNSUPPORTED, "%s: head_dim %d (at most 256)", who, A.p.hd);
    HC_CHECK(n_heads >= 1 && n_heads % A.p.nkv == 0, HC_ERR_INVALID, "%s: %d query heads over %d KV heads", who, n_heads,
             A.p.nkv);
    HC_CHECK(window >= 0, HC_ERR_INVALID, "%s: window %d", who, window);
    A.nh = n_heads;
    A.G = n_heads / A.p.nkv;
    A.g_shift = -1;
    for (int i = 0; i < 31; i++)
        if (A.G == (1 << i)) A.g_shift = i;
    A.window = window;
    X.l = {};
    if (lists) {
        HC_CHECK(lists->width >= 1 && (lists->pages || batch->n_rows == 0), HC_ERR_INVALID, "%s: NULL or empty lists of pages", who);
        HC_CHECK(lists->row_stride >= 0 && lists->head_stride >= 0 && (uintptr_t)lists->pages % 4 == 0, HC_ERR_INVALID,
                 "%s: negative stride of, or misaligned lists of pages", who);
        X.l = {lists->pages, lists->row_stride, lists->head_stride, lists->width};
    }
    return HC_OK;
}

// Which kernel takes a call, by its row tiles at most.  Few (single tokens; up to
// 16 packed rows of one sequence), or rows with lists of pages: the split kernel,
// which reads the keys once for 8 or 16 rows.  More, over an FP16 cache: the
// 256-row tiles of the tcgen05 kernel; over an FP32 one: the split kernel still;
// over one in 4 bits: the pages' values as float16 (exactly) in the workspace, and
// the tcgen05 kernel over those.  Unaligned or odd heads take the kernel for
// any shape.
enum AttnKernel { ATTN_ANY, ATTN_SPLIT, ATTN_TC };
struct AttnPlan {
    AttnKernel kernel;
    size_t bytes;      // of the workspace
    int at_once;       // 4 bits, ATTN_TC: sequences whose values the workspace holds
    size_t values, of_k;  // bytes of their values and page numbers, of the keys'
};

// The batch of up to n of its sequences from b on, over the values of their pages.
hc::PagedAttnArgs over_values(const hc::PagedAttnArgs& A, int b, int n, void* ws, const AttnPlan& plan) {
    hc::PagedAttnArgs B = A;
    hc::PagedArgs& P = B.p;
    P.n_seqs = std::min(n, A.p.n_seqs - b);
    P.q_start = A.p.q_start ? A.p.q_start + b : nullptr;
    P.kv_len = A.p.kv_len ? A.p.kv_len + b : nullptr;
    P.k = ws;
    P.v = (uint8_t*)ws + plan.of_k;
    P.n_pages = P.n_seqs * P.max_pages;
    P.kss = P.vss = P.hd;
    P.khs = P.vhs = (int64_t)P.hd * P.page_size;
    P.kps = P.vps = P.khs * P.nkv;
    P.table = (const int32_t*)((uint8_t*)ws + 2 * plan.of_k);
    P.table_stride = P.max_pages;
    return B;
}
constexpr size_t VALUES_AT_ONCE = (size_t)1 << 30;

size_t aligned(size_t n) { return (n + 255) / 256 * 256; }

AttnPlan attn_plan(const AttnCall& X, const hc_paged_batch* b, int kv) {
    const hc::PagedAttnArgs& A = X.a;
    AttnPlan plan = {ATTN_ANY, 0, 0, 0, 0};
    if (!hc::paged_split_ok(A.p, kv)) return plan;
    // Few rows: the split kernel, a sequence's rows in tiles of 16.  Many: tcgen05, in
    // tiles of 256, which take up to twice as long each, so from about twice as
    // many small tiles on.  (32 sequences of 4,096 keys, 32 heads over 8 of 128, us,
    // 16-row tiles / 256-row tiles: 4 tokens each, f16 119 / 147, f32 126 / 224; 6
    // tokens 207 / 147, 227 / 226; 32 tokens 702 / 148, 817 / 234.  One sequence
    // of 6 tokens: 26 / 19, 25 / 25.)
    const int64_t few = hc::paged_tiles(A, b->max_q_len, 16), many = hc::paged_tiles(A, b->max_q_len, 256);
    // Over 4 bits the values' way through memory comes on top (32 sequences as above: 230 us
    // of it), so from more than five small tiles a large one on.  (Small tiles / large ones,
    // us, those: 8 tokens, f16 129 / 307, f32 184 / 384; 16 tokens 235 / 308, 341 / 389; 32
    // tokens 439 / 309, 644 / 393.  One sequence of 16,384 keys: 16 tokens 54 / 58, 68 /
    // 72; 32 tokens 74 / 65, 100 / 78.  8 sequences of 1,024, 32 heads over 4 of 64: 16 tokens
    // 25 / 27, 27 / 29; 32 tokens 36 / 32, 40 / 36.)
    if (!X.l.width && (kv == HC_KV_Q4 ? few > 5 * many : 2 * few > 3 * many)) {
        if (kv == HC_KV_Q4 && A.p.max_pages > 0) {
            // (sized by the table, not by the host's bound of the lengths, which chooses no results)
            const size_t page = (size_t)A.p.page_size * A.p.nkv * A.p.hd * 2, each = page * A.p.max_pages;
            plan.at_once = (int)std::min<size_t>(std::min(A.p.n_seqs, 65535), std::max<size_t>(1, VALUES_AT_ONCE / (2 * each)));
            plan.of_k = aligned(each * plan.at_once);
            plan.values = 2 * plan.of_k + aligned((size_t)4 * plan.at_once * A.p.max_pages);
            const hc::PagedAttnArgs B = over_values(A, 0, plan.at_once, nullptr, plan);
            if ((int64_t)plan.at_once * A.p.max_pages <= INT_MAX && hc::paged_tc_ok(B, 1)) {
                plan.kernel = ATTN_TC;
                // (the last round may have fewer sequences, and so more runs of keys)
                const int rest = A.p.n_seqs % plan.at_once;
                size_t runs = hc::paged_tc_bytes(B, b->max_q_len, b->max_kv_len);
                if (rest) runs = std::max(runs, hc::paged_tc_bytes(over_values(A, 0, rest, nullptr, plan), b->max_q_len, b->max_kv_len));
                plan.bytes = plan.values + runs;
                return plan;
            }
        } else if (hc::paged_tc_ok(A, kv == HC_KV_FP16)) {
            plan.kernel = ATTN_TC;
            plan.bytes = hc::paged_tc_bytes(A, b->max_q_len, b->max_kv_len);
            return plan;
        }
    }
    plan.kernel = ATTN_SPLIT;
    plan.bytes = hc::paged_split_bytes(A, X.l, b->max_q_len, b->max_kv_len);
    return plan;
}

int attention(const char* who, const hc_paged_kv* kv, const hc_paged_batch* batch, const hc_page_lists* lists, const hc_rows* q,
              const hc_rows* out, float* lse, int n_heads, uint32_t dtype, float scale, int window, void* workspace,
              size_t workspace_bytes, cudaStream_t stream) {
    AttnCall X;
    hc::PagedAttnArgs& A = X.a;
    HC_TRY(attn_checks(who, kv, batch, lists, n_heads, dtype, window, X));
    if (batch->n_rows == 0) return HC_OK;
    HC_TRY(rows_ok(who, "q", q, dtype));
    HC_TRY(rows_ok(who, "out", out, dtype));
    A.q = q->data;
    A.q_rs = q->row_stride;
    A.q_hs = q->head_stride;
    A.out = out->data;
    A.o_rs = out->row_stride;
    A.o_hs = out->head_stride;
    A.lse = lse;
    A.scale = scale;
    const int q16 = dtype == HC_DTYPE_FP16, type = kv->kv_dtype;
    const int64_t e = q16 ? 8 : 4;
    A.qvec = (uintptr_t)q->data % 16 == 0 && (q->row_stride | q->head_stride) % e == 0;
    A.ovec = (uintptr_t)out->data % 16 == 0 && (out->row_stride | out->head_stride) % e == 0;
    AttnPlan plan = attn_plan(X, batch, type);
    HC_CHECK(workspace_bytes >= plan.bytes && (plan.bytes == 0 || (workspace && (uintptr_t)workspace % 16 == 0)),
             HC_ERR_INVALID, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", who, plan.bytes,
             workspace_bytes);
    // the tcgen05 kernel takes row maxima before it applies the scale; the
    // workspace does not know the scale, so another one goes to a kernel without one
    // (over 4 bits: one CTA of the split kernel per pair, which needs none)
    if (plan.kernel == ATTN_TC && !(scale > 0.0f)) {
        if (type == HC_KV_Q4) return hc::launch_paged_split(A, X.c, X.l, q16, type, batch->max_q_len, 0, nullptr, stream);
        plan.kernel = ATTN_ANY;
    }
    if (plan.kernel == ATTN_TC && type == HC_KV_Q4) {
        for (int b = 0; b < A.p.n_seqs; b += plan.at_once) {
            const hc::PagedAttnArgs B = over_values(A, b, plan.at_once, workspace, plan);
            hc::PagedArgs from = A.p;
            from.n_seqs = B.p.n_seqs;
            from.kv_len = B.p.kv_len;
            from.table = A.p.table + b * A.p.table_stride;
            HC_TRY(hc::launch_q4_values(from, X.c, true, (__half*)B.p.k, (__half*)B.p.v, (int32_t*)B.p.table, stream));
            HC_TRY(hc::launch_paged_tc(B, q16, batch->max_q_len, batch->max_kv_len, (uint8_t*)workspace + plan.values, stream));
        }
        return HC_OK;
    }
    if (plan.kernel == ATTN_TC) return hc::launch_paged_tc(A, q16, batch->max_q_len, batch->max_kv_len, workspace, stream);
    if (plan.kernel == ATTN_SPLIT)
        return hc::launch_paged_split(A, X.c, X.l, q16, type, batch->max_q_len, batch->max_kv_len, workspace, stream);
    return hc::launch_paged_generic(A, X.l, q16, type == HC_KV_FP16, stream);
}

int attention_workspace(const char* who, const hc_paged_kv* kv, const hc_paged_batch* batch, const hc_page_lists* lists, int n_heads,
                        uint32_t dtype, int window, size_t* bytes) {
    AttnCall X;
    HC_CHECK(bytes, HC_ERR_INVALID, "%s: NULL bytes", who);
    HC_TRY(attn_checks(who, kv, batch, lists, n_heads, dtype, window, X));
    *bytes = batch->n_rows == 0 ? 0 : attn_plan(X, batch, kv->kv_dtype).bytes;
    return HC_OK;
}

}  // namespace

HC_EXPORT int hc_paged_attention_workspace(const hc_paged_kv* kv, const hc_paged_batch* batch, int n_heads,
                                           uint32_t dtype, int window, size_t* bytes) {
    return attention_workspace("hc_paged_attention_workspace", kv, batch, nullptr, n_heads, dtype, window, bytes);
}

HC_EXPORT int hc_paged_attention_dev(const hc_paged_kv* kv, const hc_paged_batch* batch, const hc_rows* q,
                                     const hc_rows* out, float* lse, int n_heads, uint32_t dtype, float scale, int window, void* workspace,
                                     size_t workspace_bytes, void* stream) {
    return attention("hc_paged_attention_dev", kv, batch, nullptr, q, out, lse, n_heads, dtype, scale, window, workspace, workspace_bytes,
                     (cudaStream_t)stream);
}

HC_EXPORT int hc_paged_list_attention_workspace(const hc_paged_kv* kv, const hc_paged_batch* batch, const hc_page_lists* lists,
                                                int n_heads, uint32_t dtype, int window, size_t* bytes) {
    const char* who = "hc_paged_list_attention_workspace";
    HC_CHECK(lists, HC_ERR_INVALID, "%s: NULL or empty lists of pages", who);
    return attention_workspace(who, kv, batch, lists, n_heads, dtype, window, bytes);
}

HC_EXPORT int hc_paged_list_attention_dev(const hc_paged_kv* kv, const hc_paged_batch* batch, const hc_page_lists* lists,
                                          const hc_rows* q, const hc_rows* out, float* lse, int n_heads, uint32_t dtype, float scale,
                                          int window, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "hc_paged_list_attention_dev";
    HC_CHECK(lists, HC_ERR_INVALID, "%s: NULL or empty lists of pages", who);
    return attention(who, kv, batch, lists, q, out, lse, n_heads, dtype, scale, window, workspace, workspace_bytes, (cudaStream_t)stream);
}

HC_EXPORT int hc_paged_values_dev(const hc_paged_kv* kv, void* k_out, void* v_out, void* stream) {
    const char* who = "hc_paged_values_dev";
    hc::PagedArgs P = {};
    hc::PagedScales C;
    HC_TRY(pool_args(who, kv, P, C));
    HC_CHECK(kv->kv_dtype == HC_KV_Q4, HC_ERR_UNSUPPORTED, "%s: kv_dtype %d", who, kv->kv_dtype);
    HC_CHECK(k_out && v_out && ((uintptr_t)k_out | (uintptr_t)v_out) % 16 == 0, HC_ERR_INVALID, "%s: NULL or misaligned output", who);
    return hc::launch_q4_values(P, C, false, (__half*)k_out, (__half*)v_out, nullptr, (cudaStream_t)stream);
}

// What hc_page_select.cu's entry points take of these checks.
int hc::page_args(const char* who, const hc_paged_kv* kv, const hc_paged_batch* batch, hc::PagedArgs& P, hc::PagedScales& C) {
    return paged_args(who, kv, batch, P, C);
}
int hc::page_rows_ok(const char* who, const char* what, const hc_rows* r, uint32_t dtype) { return rows_ok(who, what, r, dtype); }

HC_EXPORT int hc_rope_table_host(size_t rows, size_t head_dim, float theta, float* out) {
    HC_CHECK(out || rows == 0 || head_dim == 0, HC_ERR_INVALID, "hc_rope_table_host: NULL out");
    HC_CHECK(head_dim % 2 == 0, HC_ERR_INVALID, "hc_rope_table_host: head_dim must be even");
    HC_CHECK(head_dim <= 65536 && rows <= (1u << 28), HC_ERR_INVALID, "hc_rope_table_host: %zu x %zu", rows, head_dim);
    const size_t half = head_dim / 2;
    if (rows == 0 || half == 0) return HC_OK;
    for (size_t j = 0; j < half; j++) {
        const float freq = 1.0f / powf(theta, (float)(2 * j) / (float)head_dim);
        for (size_t p = 0; p < rows; p++) {
            const float a = (float)p * freq;
            out[(p * half + j) * 2] = cosf(a);
            out[(p * half + j) * 2 + 1] = sinf(a);
        }
    }
    return HC_OK;
}
