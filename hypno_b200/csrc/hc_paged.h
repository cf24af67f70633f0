// Paged KV cache: arguments and device helpers shared by the append kernel
// and the attention kernels (hc_paged.cu, hc_paged_split.cu, hc_paged_tc.cu).
#pragma once

#include "hc_common.cuh"
#include "hc_internal.h"

#include <algorithm>

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

// Few rows per sequence (hc_paged_split.cu): the keys split over CTAs.
bool paged_split_ok(const PagedArgs& P, int c16);
bool paged_split_whole(const PagedAttnArgs& A, int max_q_len, int max_kv_len);
size_t paged_split_bytes(const PagedAttnArgs& A, int max_q_len, int max_kv_len);  // workspace
int launch_paged_split(const PagedAttnArgs& A, int q16, int c16, int max_q_len, int max_kv_len, void* ws,
                       cudaStream_t s);

// Any shape (hc_paged.cu).
int launch_paged_generic(const PagedAttnArgs& A, int q16, int c16, cudaStream_t s);

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

// Row tiles of all sequences, at most, from what the host knows.
inline int64_t paged_tiles(const PagedAttnArgs& A, int max_q_len, int rows) {
    const int64_t each = ((int64_t)max_q_len * A.G + rows - 1) / rows;
    return std::max<int64_t>(1, std::min(A.p.n_seqs * each, (int64_t)A.p.n_rows * A.G / rows + A.p.n_seqs));
}

}  // namespace hc
