// Paged KV cache: arguments and device helpers shared by the append kernel
// and the attention kernels (hc_paged.cu, hc_paged_split.cu, hc_paged_tc.cu).
#pragma once

#include "hc_common.cuh"
#include "hc_internal.h"

#include <algorithm>
#include <atomic>

namespace hc {

// The pool of one layer and the step's batch, as the kernels take them.
struct PagedArgs {
    void* k;
    void* v;
    int64_t kps, khs, kss;  // page / head / position strides of k, in elements
    int64_t vps, vhs, vss;
    const int32_t* table;
    const int32_t* q_start;
    const int32_t* kv_len;
    int64_t table_stride;
    int n_pages, page_size, page_shift;  // page_shift >= 0: page_size = 1 << page_shift
    int nkv, hd;
    int n_seqs, max_pages, n_rows;
    int reach;  // positions that a row of the table can name: what lies past them are holes, and not visited
};

// The scales of a pool in 4 bits (its k and v are bytes of two codes, their
// strides too); strides in scales.
struct PagedScales {
    __half* k;
    __half* v;
    int64_t kps, khs, kss;
    int64_t vps, vhs, vss;
};

// The pages that each row reads, per KV head: indexes into its sequence's row of
// the block table, in ascending order.  A list ends before the first entry that
// is not above the one in front of it (so -1 ends it).
struct PagedList {
    const int32_t* pages;
    int64_t row_stride, head_stride;
    int width;  // entries of a list, at most; 0: no lists, a row reads all that it sees
};

struct PagedAttnArgs {
    PagedArgs p;
    const void* q;
    void* out;
    int64_t q_rs, q_hs, o_rs, o_hs;  // row / head strides, in elements
    float* lse;                      // [n_rows][nh], may be null
    int nh, G;                       // query heads, query heads per KV head
    int g_shift;                     // >= 0: G = 1 << g_shift
    int window;                      // > 0: only the last `window` positions
    float scale;
    int qvec, ovec;                  // 16-byte aligned rows of q / out
};

__device__ __forceinline__ int page_of(const PagedArgs& P, int pos) {
    return P.page_shift >= 0 ? (pos >> P.page_shift) : pos / P.page_size;
}

// Token of packed row m (within its sequence).
__device__ __forceinline__ int token_of(const PagedAttnArgs& A, int m) { return A.g_shift >= 0 ? m >> A.g_shift : m / A.G; }

// Page of position pos (>= 0) of sequence seq, -1 for a hole; slot = the
// position's place in it.
__device__ __forceinline__ int lookup(const PagedArgs& P, int seq, int pos, int& slot) {
    const int i = page_of(P, pos);
    slot = pos - i * P.page_size;
    if (i >= P.max_pages) return -1;
    const int g = __ldg(P.table + (int64_t)seq * P.table_stride + i);
    return (unsigned)g < (unsigned)P.n_pages ? g : -1;
}

// Rows [r0, r1) of sequence b, held to the packed rows that exist.
__device__ __forceinline__ void seq_rows(const PagedArgs& P, int b, int& r0, int& r1) {
    r0 = min(max(__ldg(P.q_start + b), 0), P.n_rows);
    r1 = min(max(__ldg(P.q_start + b + 1), r0), P.n_rows);
}

// Positions of sequence b (a negative length counts as none).
__device__ __forceinline__ int seq_len(const PagedArgs& P, int b) { return max(__ldg(P.kv_len + b), 0); }

// Entries of the list of (row, KV head); a whole warp.
__device__ __forceinline__ int list_count(const PagedList& L, int row, int kvh) {
    const int lane = threadIdx.x & 31;
    const int32_t* e = L.pages + row * L.row_stride + kvh * L.head_stride;
    constexpr int N = 4;  // so many times 32 entries are requested at once
    int last = -1;
    for (int i0 = 0; i0 < L.width; i0 += 32 * N) {
        int here[N];
#pragma unroll
        for (int k = 0; k < N; k++) here[k] = i0 + 32 * k + lane < L.width ? __ldg(e + i0 + 32 * k + lane) : -1;
#pragma unroll
        for (int k = 0; k < N; k++) {
            int before = __shfl_up_sync(0xffffffffu, here[k], 1);
            if (lane == 0) before = last;
            const unsigned end = __ballot_sync(0xffffffffu, here[k] <= before);
            if (end) return i0 + 32 * k + __ffs(end) - 1;
            last = __shfl_sync(0xffffffffu, here[k], 31);
        }
    }
    return L.width;
}

// Pages of its block table that a row at position p sees.
__device__ __forceinline__ int pages_seen(const PagedArgs& P, int p) {
    return p < 0 ? 0 : min(page_of(P, p) + 1, P.max_pages);
}

// Page and slot of place v of a list, -1 where the row does not see it.
__device__ __forceinline__ int lookup_listed(const PagedAttnArgs& A, const int32_t* list, int seq, int v, int p, int& slot) {
    const PagedArgs& P = A.p;
    const int i = page_of(P, v);
    slot = v - i * P.page_size;
    const int e = __ldg(list + i);
    if (e >= P.max_pages) return -1;
    const int64_t pos = (int64_t)e * P.page_size + slot;
    if (pos > p || (A.window > 0 && pos <= (int64_t)p - A.window)) return -1;
    const int g = __ldg(P.table + (int64_t)seq * P.table_stride + e);
    return (unsigned)g < (unsigned)P.n_pages ? g : -1;
}

// ---- 4 bits: 32 elements of a head share a scale s, a float16 of seven
// significant bits at most (so that c s, |c| <= 8, and 72 s are float16 values
// too), an element is the nibble c + 8, element 2 i in the low half of byte i.
constexpr float Q4_TOP = 896.0f;  // the largest scale: 72 s stays below 65,504

// The scale of 32 elements from the bits of their largest magnitude.
__device__ __forceinline__ float q4_scale(uint32_t top) {
    if (top >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
    const float t = __fdiv_rn(__uint_as_float(top), 7.0f);
    const float s = __uint_as_float((__float_as_uint(t) + 0x1FFFFu) & ~0x1FFFFu);
    return fminf(ceilf(s * 16777216.0f) * 0x1p-24f, Q4_TOP);
}
__device__ __forceinline__ uint32_t q4_code(float x, float s) {
    if (!(s > 0.0f)) return 8;  // zeros, and a block that holds a value that is not finite
    return (uint32_t)((int)fminf(fmaxf(rintf(__fdiv_rn(x, s)), -7.0f), 7.0f) + 8);
}
// A scale's slots of a position: a power of two, so that they are copied at once.
__host__ __device__ constexpr int q4_slots(int hd) { return hd <= 64 ? 2 : hd <= 128 ? 4 : 8; }

// Nibbles j = 0..3 of each half of x as pairs of float16 values, exactly, s72 = -72 s:
// 0x5400 | nibble << 4 is 64 + c + 8, and (64 + c + 8) s - 72 s is c s; 0x6400 | nibble
// is 1024 + c + 8.  The first takes the nibbles that lie there after no shift, or one
// of the whole word by 8, the second the others: shifts and logic run at half the
// rate of the multiply-add units (one shift a word in place of three).
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {  // one instruction (written with & and |, two)
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
    return y;
}
__device__ __forceinline__ void q4_pairs(uint32_t x, __half2 s, __half2 s72, uint32_t* out) {
    const __half2 back = __half2half2(__ushort_as_half(0xE408));  // -1032
    auto odd = [&](uint32_t y) {
        const uint32_t b = and_or(y, 0x00F000F0u, 0x54005400u);
        const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&b), s, s72);
        return *reinterpret_cast<const uint32_t*>(&v);
    };
    auto even = [&](uint32_t y) {
        const uint32_t b = and_or(y, 0x000F000Fu, 0x64006400u);
        const __half2 v = __hmul2(__hadd2(*reinterpret_cast<const __half2*>(&b), back), s);
        return *reinterpret_cast<const uint32_t*>(&v);
    };
    const uint32_t y = x >> 8;
    out[0] = even(x);
    out[1] = odd(x);
    out[2] = even(y);
    out[3] = odd(y);
}

struct q4x {};  // the element type of a pool in 4 bits, for the kernels' templates

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// The tile-th tile of BM packed (token, query head of the group) rows, over
// the sequences in order; executed by a whole warp.  Returns false past the
// last tile.
__device__ __forceinline__ bool find_tile(const PagedArgs& P, int G, int BM, int tile, int& seq, int& in_seq) {
    const int lane = threadIdx.x & 31;
    int base = 0;
    for (int b0 = 0; b0 < P.n_seqs; b0 += 32) {
        int n = 0;
        if (b0 + lane < P.n_seqs) {
            int r0, r1;
            seq_rows(P, b0 + lane, r0, r1);
            n = (int)(((int64_t)(r1 - r0) * G + BM - 1) / BM);
        }
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += t;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, base + incl > tile);
        if (hit) {
            const int l = __ffs(hit) - 1;
            seq = b0 + l;
            in_seq = tile - base - (__shfl_sync(0xffffffffu, incl, l) - __shfl_sync(0xffffffffu, n, l));
            return true;
        }
        base += __shfl_sync(0xffffffffu, incl, 31);
    }
    return false;
}

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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
// Visible positions of packed rows [m0, m0 + n) of a sequence: [begin, end).
__device__ __forceinline__ void visible(const PagedAttnArgs& A, int first, int m0, int n, int& begin, int& end) {
    end = min(max(0, first + token_of(A, m0 + n - 1) + 1), A.p.reach);
    begin = A.window > 0 ? max(0, max(0, first + token_of(A, m0) + 1) - A.window) : 0;
    begin = min(begin, end);
}

// Four columns of a finished row: v / l, zeros for a row that saw nothing (l = 0).
template <typename T>
__device__ __forceinline__ void store_row4(const PagedAttnArgs& A, int row, int head, int d, float l, float4 v) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = (T*)A.out + row * A.o_rs + head * A.o_hs + d;
    if constexpr (sizeof(T) == 4) {
        if (A.ovec) {
            *reinterpret_cast<float4*>(out) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
            return;
        }
    } else {
        if (A.ovec) {
            const __half2 a = __floats2half2_rn(v.x * inv, v.y * inv), b = __floats2half2_rn(v.z * inv, v.w * inv);
            *reinterpret_cast<uint2*>(out) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
            return;
        }
    }
    out[0] = from_f32<T>(v.x * inv);
    out[1] = from_f32<T>(v.y * inv);
    out[2] = from_f32<T>(v.z * inv);
    out[3] = from_f32<T>(v.w * inv);
}

// Many rows per sequence (hc_paged_tc.cu): tcgen05 products over 256-row tiles.
bool paged_tc_ok(const PagedAttnArgs& A, int c16);
size_t paged_tc_bytes(const PagedAttnArgs& A, int max_q_len, int max_kv_len);  // workspace
int launch_paged_tc(const PagedAttnArgs& A, int q16, int max_q_len, int max_kv_len, void* ws, cudaStream_t s);

// Few rows per sequence, or rows with lists of pages (hc_paged_split.cuh): the keys
// split over CTAs.  kv: HC_KV_FP32, HC_KV_FP16 or HC_KV_Q4 (with its scales).
bool paged_split_ok(const PagedArgs& P, int kv);
bool paged_split_whole(const PagedAttnArgs& A, const PagedList& L, int max_q_len, int max_kv_len);
size_t paged_split_bytes(const PagedAttnArgs& A, const PagedList& L, int max_q_len, int max_kv_len);  // workspace
int launch_paged_split(const PagedAttnArgs& A, const PagedScales& C, const PagedList& L, int q16, int kv, int max_q_len,
                       int max_kv_len, void* ws, cudaStream_t s);

// Any shape (hc_paged.cu).
int launch_paged_generic(const PagedAttnArgs& A, const PagedList& L, int q16, int c16, cudaStream_t s);

// A pool in 4 bits (hc_paged_q4.cu): append, and the float16 values of pages.
struct AppendArgs {
    PagedArgs p;
    const void *k, *v, *q;
    void* qo;
    int64_t k_rs, k_hs, v_rs, v_hs, q_rs, q_hs, o_rs, o_hs;
    const float2* rope;
    int rope_rows, rot, halves;
    int nh;  // 0: no queries
};
int launch_append_q4(const AppendArgs& A, const PagedScales& C, int x16, cudaStream_t s);

// The C entry points' checks of a pool and a batch, and of rows.
int page_args(const char* who, const hc_paged_kv* kv, const hc_paged_batch* batch, PagedArgs& P, PagedScales& C);
int page_rows_ok(const char* who, const char* what, const hc_rows* r, uint32_t dtype);
// Every page of the pool, or (a table) page i of the batch's sequence b to page
// b max_pages + i, its number to `numbers`.
int launch_q4_values(const PagedArgs& P, const PagedScales& C, bool of_batch, __half* k, __half* v, int32_t* numbers,
                     cudaStream_t s);

// The results of a row's n runs of keys as one: with M = max m_s,
// l = sum 2^(m_s - M) l_s, o = sum 2^(m_s - M) o_s, four columns from d on, in the
// runs' order.  Eight runs' results are requested at once (a chain of loads, one
// after another, took 2 to 4 us longer).
template <typename RowOf>
__device__ __forceinline__ void join_runs(int n, RowOf row_of, const float* po, const float2* pml, int hd, int d, float& mx,
                                          float& l, float4& v) {
    constexpr int N = 8;
    mx = -INFINITY;
    l = 0.0f;
    v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s = 0; s < n; s += N) {
        float2 ml[N];
        float4 y[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int64_t r = row_of(min(s + i, n - 1));
            ml[i] = pml[r];
            y[i] = *reinterpret_cast<const float4*>(po + r * hd + d);
            if (s + i >= n) ml[i] = make_float2(-INFINITY, 0.0f);
        }
        float top = mx;
#pragma unroll
        for (int i = 0; i < N; i++) top = fmaxf(top, ml[i].x);
        if (l != 0.0f) {
            const float f = exp2f(mx - top);
            l *= f;
            v.x *= f;
            v.y *= f;
            v.z *= f;
            v.w *= f;
        }
        mx = top;
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (ml[i].y == 0.0f) continue;  // saw nothing
            const float f = exp2f(ml[i].x - mx);
            l = fmaf(f, ml[i].y, l);
            v.x = fmaf(f, y[i].x, v.x);
            v.y = fmaf(f, y[i].y, v.y);
            v.z = fmaf(f, y[i].z, v.z);
            v.w = fmaf(f, y[i].w, v.w);
        }
    }
}

// Shared memory beyond 48 KB has to be asked for, once a kernel and device (asking takes
// some 4 us of a call's 10 to 14); `asked` is the kernel's own.
inline int ask_smem(const void* kernel, int bytes, std::atomic<uint64_t>& asked) {
    int dev = 0;
    HC_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (asked.load(std::memory_order_acquire) & bit) return HC_OK;
    HC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    asked.fetch_or(bit, std::memory_order_release);
    return HC_OK;
}

// Row tiles of all sequences, at most, from what the host knows.
inline int64_t paged_tiles(const PagedAttnArgs& A, int max_q_len, int rows) {
    const int64_t each = ((int64_t)max_q_len * A.G + rows - 1) / rows;
    return std::max<int64_t>(1, std::min(A.p.n_seqs * each, (int64_t)A.p.n_rows * A.G / rows + A.p.n_seqs));
}

}  // namespace hc
