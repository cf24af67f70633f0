// A paged cache in 4 bits: append with rotation, and the values of its pages.
#include "hc_paged.h"

namespace hc {

namespace {

constexpr int Q4_THREADS = 256;

__device__ __forceinline__ int seq_of_row(const PagedArgs& P, int r) {
    int lo = 0, hi = P.n_seqs - 1;  // the last sequence whose first row is <= r
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (__ldg(P.q_start + mid) <= r) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float* x) {
    if (!vec) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = to_f32(p[i]);
        return;
    }
    if constexpr (sizeof(T) == 4) {
        const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p));
        const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, const float* x) {
    if (!vec) {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = from_f32<T>(x[i]);
        return;
    }
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack(x[0], x[1]), pack(x[2], x[3]), pack(x[4], x[5]), pack(x[6], x[7]));
    }
}

// Eight elements of a head a thread; the four threads of 32 elements find their
// largest magnitude together.  The turned pairs are separately rounded products
// (a c - b s, not contracted), so that a value at the border of two codes falls
// the same way whatever computes it.  A thread's loads are in flight before the
// row's place in the cache (three dependent loads) is known.
//
// Half pairs (HALVES): a thread reads its elements' partners too; of q, which may be
// turned in place, the thread of the first elements turns both, and the one of the
// second ones has nothing to do.
// 8,192 rows of 32 + 8 + 8 heads of 128, f32: 67 us, 5.2 TB/s; 32 rows: 5.4.
//
// Codes: with i = 1 / s rounded, x i is within 7 2^-24 < 2^-21 of x / s, which is 7 at most,
// and the difference to its nearest whole number rounds by less than 2^-24, so that number is
// the division's unless it lies within 2^-19 of the middle of two; such a block divides.  (Divisions alone, and angles pair by pair, took a third of the kernel's
// instructions: 8,192 rows 80 us.)
__device__ __forceinline__ uint32_t q4_codes(const float* x, float s) {
    uint32_t code = 0;
    const float inv = __frcp_rn(s);
    constexpr float MID = 12582912.0f + 8.0f;  // 1.5 2^23: the sum's low bits are the whole number + 8
    float off = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float y = __fmaf_rn(x[i], inv, MID);
        off = fmaxf(off, fabsf(__fmaf_rn(x[i], inv, MID - y)));
        code |= (__float_as_uint(y) & 15u) << (4 * i);
    }
    // (no scale, the largest one, where codes are held to 7, and what is not finite: by the division too)
    if (!(s > 0.0f && s < Q4_TOP && off < 0.5f - 0x1p-19f)) {
        code = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) code |= q4_code(x[i], s) << (4 * i);
    }
    return code;
}

template <typename T, bool HALVES>
__global__ void __launch_bounds__(Q4_THREADS) k_q4_append(AppendArgs A, PagedScales C, int vec, int hu_shift) {
    const PagedArgs& P = A.p;
    const int row = blockIdx.x, hu = P.hd >> 3, half = A.rot >> 1;
    const int unit = blockIdx.y * Q4_THREADS + threadIdx.x;
    if (unit >= (A.nh + 2 * P.nkv) * hu) return;  // (the four threads of a block of 32 leave together)
    int head = hu_shift >= 0 ? unit >> hu_shift : unit / hu;
    const int i0 = 8 * (unit - head * hu);
    const bool is_q = head < A.nh, is_v = head >= A.nh + P.nkv;
    if (!is_q) head -= is_v ? A.nh + P.nkv : A.nh;
    if (HALVES && is_q && i0 >= half && i0 + 8 <= A.rot) return;
    const T* src = is_q   ? (const T*)A.q + row * A.q_rs + head * A.q_hs
                   : is_v ? (const T*)A.v + row * A.v_rs + head * A.v_hs
                          : (const T*)A.k + row * A.k_rs + head * A.k_hs;
    const bool turns = !is_v && i0 < A.rot;
    float x[8], y[8];  // the elements; HALVES: their partners
    load8(src + i0, vec, x);
    if (HALVES && turns) {
        if (half % 8 == 0) {
            load8(src + (i0 < half ? i0 + half : i0 - half), vec, y);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int d = i0 + i;
                y[i] = d < A.rot ? to_f32(src[d < half ? d + half : d - half]) : 0.0f;
            }
        }
    }
    const int seq = seq_of_row(P, row);
    int r0, r1;
    seq_rows(P, seq, r0, r1);
    if (row < r0 || row >= r1) return;
    const int pos = seq_len(P, seq) - (r1 - r0) + (row - r0);
    if (!HALVES && turns && vec && i0 + 8 <= A.rot && half % 2 == 0) {
        // four whole pairs, their angles in 16-byte pieces
        const float4* cs = reinterpret_cast<const float4*>(A.rope + (int64_t)min(max(pos, 0), A.rope_rows - 1) * half + (i0 >> 1));
        const float4 t[2] = {__ldg(cs), __ldg(cs + 1)};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float c = i & 1 ? t[i >> 1].z : t[i >> 1].x, s = i & 1 ? t[i >> 1].w : t[i >> 1].y;
            const float a = x[2 * i], b = x[2 * i + 1];
            x[2 * i] = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
            x[2 * i + 1] = __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c));
        }
    } else if (turns) {
        const float2* cs = A.rope + (int64_t)min(max(pos, 0), A.rope_rows - 1) * half;
#pragma unroll
        for (int i = 0; i < 8; i += HALVES ? 1 : 2) {
            const int d = i0 + i;
            if (d >= A.rot) break;
            if constexpr (HALVES) {
                const bool one = d < half;  // the pair's first element
                const float2 t = __ldg(cs + (one ? d : d - half));
                const float a = one ? x[i] : y[i], b = one ? y[i] : x[i];
                const float u = __fsub_rn(__fmul_rn(a, t.x), __fmul_rn(b, t.y)), v = __fadd_rn(__fmul_rn(a, t.y), __fmul_rn(b, t.x));
                x[i] = one ? u : v;
                y[i] = one ? v : u;
            } else {
                const float2 t = __ldg(cs + (d >> 1));
                const float a = x[i], b = x[i + 1];
                x[i] = __fsub_rn(__fmul_rn(a, t.x), __fmul_rn(b, t.y));
                x[i + 1] = __fadd_rn(__fmul_rn(a, t.y), __fmul_rn(b, t.x));
            }
        }
    }
    if (is_q) {
        T* dst = (T*)A.qo + row * A.o_rs + head * A.o_hs;
        if (!HALVES || !turns) {
            store8(dst + i0, vec, x);
        } else if (half % 8 == 0) {
            store8(dst + i0, vec, x);
            store8(dst + i0 + half, vec, y);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int d = i0 + i;
                if (d < half) {
                    dst[d] = from_f32<T>(x[i]);
                    dst[d + half] = from_f32<T>(y[i]);
                } else if (d >= A.rot) {
                    dst[d] = from_f32<T>(x[i]);  // (a run of eight may end past the pairs)
                }
            }
        }
        return;
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    const uint32_t four = 0xFu << (threadIdx.x & 28);
    top = max(top, __shfl_xor_sync(four, top, 1));
    top = max(top, __shfl_xor_sync(four, top, 2));
    if (pos < 0) return;
    int slot;
    const int page = lookup(P, seq, pos, slot);
    if (page < 0) return;
    const float s = q4_scale(top);
    const uint32_t code = q4_codes(x, s);
    uint8_t* dst = is_v ? (uint8_t*)P.v + page * P.vps + head * P.vhs + slot * P.vss : (uint8_t*)P.k + page * P.kps + head * P.khs + slot * P.kss;
    *reinterpret_cast<uint32_t*>(dst + (i0 >> 1)) = code;
    if ((i0 & 31) == 0) {
        __half* sc = is_v ? C.v + page * C.vps + head * C.vhs + slot * C.vss : C.k + page * C.kps + head * C.khs + slot * C.kss;
        sc[i0 >> 5] = __float2half_rn(s);  // exact
    }
}

// Values as float16, exactly: a CTA takes one page of one KV head, a thread eight
// elements of K and of V of every (threads / eights)-th position.  Bound by its writes
// (with a thread's place worked out from one index for all of a pool it was bound by
// the divisions: 16,384 positions of 8 heads of 128, 25 us).
__global__ void __launch_bounds__(Q4_THREADS) k_q4_values(PagedArgs P, PagedScales C, int of_batch, __half* k, __half* v,
                                                          int32_t* numbers) {
    const int hu = P.hd >> 3, head = blockIdx.y;
    int64_t page = blockIdx.x, src = blockIdx.x;
    if (of_batch) {
        const int b = blockIdx.z;
        page += (int64_t)b * P.max_pages;
        src = __ldg(P.table + (int64_t)b * P.table_stride + blockIdx.x);
        const int64_t begin = (int64_t)blockIdx.x * P.page_size;
        if ((uint64_t)src >= (uint64_t)P.n_pages || begin >= seq_len(P, b)) src = -1;
        if (head == 0 && threadIdx.x == 0) numbers[page] = src < 0 ? -1 : (int32_t)page;
        if (src < 0) return;
    }
    const int u = threadIdx.x % hu, rows = Q4_THREADS / hu, r = threadIdx.x / hu;
    if (r >= rows) return;
    const uint8_t* kp = (const uint8_t*)P.k + src * P.kps + head * P.khs + 4 * u;
    const uint8_t* vp = (const uint8_t*)P.v + src * P.vps + head * P.vhs + 4 * u;
    const __half *ks = C.k + src * C.kps + head * C.khs + (u >> 2), *vs = C.v + src * C.vps + head * C.vhs + (u >> 2);
    const int64_t to = (page * P.nkv + head) * P.page_size * P.hd + 8 * u;
#pragma unroll 2
    for (int slot = r; slot < P.page_size; slot += rows) {
        const uint32_t w[2] = {__ldg(reinterpret_cast<const uint32_t*>(kp + slot * P.kss)), __ldg(reinterpret_cast<const uint32_t*>(vp + slot * P.vss))};
        const __half sc[2] = {ks[slot * C.kss], vs[slot * C.vss]};
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const __half2 s = __half2half2(sc[x]), z = __hmul2(s, __half2half2(__float2half_rn(-72.0f)));
            uint32_t e[4];
            q4_pairs(w[x], s, z, e);  // (0, 4), (1, 5), (2, 6), (3, 7)
            *reinterpret_cast<uint4*>((x ? v : k) + to + (int64_t)slot * P.hd) =
                make_uint4(__byte_perm(e[0], e[1], 0x5410), __byte_perm(e[2], e[3], 0x5410), __byte_perm(e[0], e[1], 0x7632), __byte_perm(e[2], e[3], 0x7632));
        }
    }
}

template <typename T>
int launch_append_t(const AppendArgs& A, const PagedScales& C, cudaStream_t s) {
    const PagedArgs& P = A.p;
    const int64_t et = 16 / (int64_t)sizeof(T);
    const int vec = ((uintptr_t)A.k | (uintptr_t)A.v | (uintptr_t)A.q | (uintptr_t)A.qo | (uintptr_t)A.rope) % 16 == 0 &&
                    (A.k_rs | A.k_hs | A.v_rs | A.v_hs | (A.nh ? A.q_rs | A.q_hs | A.o_rs | A.o_hs : 0)) % et == 0;
    const int64_t units = (int64_t)(A.nh + 2 * P.nkv) * (P.hd / 8);
    HC_CHECK(units <= 65535ll * Q4_THREADS, HC_ERR_INVALID, "hc_paged_append_dev: %d + %d heads of %d", A.nh, P.nkv, P.hd);
    const dim3 grid((unsigned)P.n_rows, (unsigned)((units + Q4_THREADS - 1) / Q4_THREADS));
    int shift = -1;
    for (int i = 0; i < 6; i++)
        if (P.hd / 8 == 1 << i) shift = i;
    if (A.halves) k_q4_append<T, true><<<grid, Q4_THREADS, 0, s>>>(A, C, vec, shift);
    else k_q4_append<T, false><<<grid, Q4_THREADS, 0, s>>>(A, C, vec, shift);
    HC_LAUNCH_CHECK();
    return HC_OK;
}

}  // namespace

int launch_append_q4(const AppendArgs& A, const PagedScales& C, int x16, cudaStream_t s) {
    return x16 ? launch_append_t<__half>(A, C, s) : launch_append_t<float>(A, C, s);
}

int launch_q4_values(const PagedArgs& P, const PagedScales& C, bool of_batch, __half* k, __half* v, int32_t* numbers, cudaStream_t s) {
    const dim3 grid((unsigned)(of_batch ? P.max_pages : P.n_pages), (unsigned)P.nkv, of_batch ? (unsigned)P.n_seqs : 1u);
    if (grid.x == 0) return HC_OK;
    k_q4_values<<<grid, Q4_THREADS, 0, s>>>(P, C, of_batch, k, v, numbers);
    HC_LAUNCH_CHECK();
    return HC_OK;
}

}  // namespace hc
