// Split attention over FP32 and FP16 pages, and which form a call takes
// (hc_paged_split.cuh has the kernels).
#include "hc_paged_split.cuh"

namespace hc {

int launch_split_dense(SplitArgs& X, int q16, int kv, cudaStream_t s) {
    const bool c16 = kv == HC_KV_FP16;
    if (q16) return c16 ? launch_split_hd<__half, __half, false>(X, s) : launch_split_hd<__half, float, false>(X, s);
    return c16 ? launch_split_hd<float, __half, false>(X, s) : launch_split_hd<float, float, false>(X, s);
}

// (a pool in 4 bits has its alignment checked at the C entry)
bool paged_split_ok(const PagedArgs& P, int kv) {
    if (kv == HC_KV_Q4) return true;
    const int64_t e = kv == HC_KV_FP16 ? 8 : 4;
    return P.hd <= (kv == HC_KV_FP16 ? 256 : 128) && P.hd % e == 0 && ((uintptr_t)P.k | (uintptr_t)P.v) % 16 == 0 &&
           (P.kps | P.khs | P.kss | P.vps | P.vhs | P.vss) % e == 0;
}

size_t paged_split_bytes(const PagedAttnArgs& A, const PagedList& L, int max_q_len, int max_kv_len) {
    return paged_split_whole(A, L, max_q_len, max_kv_len) ? 0 : (size_t)2 * SP_CTAS * 16 * ((size_t)A.p.hd * 4 + 8);
}

// 16 rows of more than 128 elements do not fit the registers
static int tile_height(const PagedAttnArgs& A, const PagedList& L, int max_q_len) {
    return (L.width ? 1 : (int64_t)max_q_len) * A.G <= 8 || A.p.hd > 128 ? 8 : 16;
}

// One CTA per pair where no pair is long enough to be worth cutting (64 sequences
// of 256 keys, 8 KV heads: 31 us cut, 21 whole; of 512 keys: 34 cut, 38 whole), and for
// chunks with many pairs: a chunk's early row tiles see fewer keys than the
// line counts for them, and a CTA's pairs cost a start each (7 chunks of 264
// tokens, 9 heads of 64, FP32 cache: 69 us cut, 51 whole).
bool paged_split_whole(const PagedAttnArgs& A, const PagedList& L, int max_q_len, int max_kv_len) {
    if (L.width) {
        const int R = tile_height(A, L, max_q_len);
        // lists are about as long as one another, so whole pairs are cut no worse than equal runs
        // from four fifths of the last round of SMs on (256 pairs of 2,048 keys in 4 bits: 41.0 us
        // cut, 40.4 whole)
        const int64_t pairs = (int64_t)A.p.n_rows * ((A.G + R - 1) / R) * A.p.nkv, rounds = (pairs + 147) / 148;
        if (5 * pairs >= 4 * 148 * rounds) return true;
        return (int64_t)L.width * A.p.page_size <= MIN_UNITS * UNIT;
    }
    if ((int64_t)max_q_len * A.G > 64 && (int64_t)A.p.n_rows * A.G / 16 * A.p.nkv >= 2 * SP_CTAS) return true;
    const int64_t len = A.window > 0 ? std::min<int64_t>(max_kv_len, (int64_t)A.window + 16) : max_kv_len;
    return len <= MIN_UNITS * UNIT;
}

int launch_paged_split(const PagedAttnArgs& A, const PagedScales& C, const PagedList& L, int q16, int kv, int max_q_len,
                       int max_kv_len, void* ws, cudaStream_t s) {
    SplitArgs X;
    X.a = A;
    X.c = C;
    X.l = L;
    X.whole = paged_split_whole(A, L, max_q_len, max_kv_len);
    X.rows = tile_height(A, L, max_q_len);
    X.tg = (A.G + X.rows - 1) / X.rows;
    // one page a tile: pages of whole tiles, at most what 16 bits count
    X.uni = (kv == HC_KV_Q4 || L.width) && A.p.page_size % SP_TK == 0 && A.p.page_size <= 65536;
    X.po = (float*)ws;
    X.pml = (float2*)((float*)ws + (size_t)2 * SP_CTAS * 16 * A.p.hd);
    if (kv == HC_KV_Q4 && X.uni && (A.p.hd == 64 || A.p.hd == 128)) return launch_q4_stream(X, q16, s);
    if (L.width) return launch_split_list(X, q16, kv, s);
    return kv == HC_KV_Q4 ? launch_split_q4(X, q16, s) : launch_split_dense(X, q16, kv, s);
}

}  // namespace hc
