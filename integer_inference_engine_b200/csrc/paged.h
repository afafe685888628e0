// Paged key/value cache: arguments of its kernels (paged.cu, paged_api.cu).
//
// kpages / vpages int32 [n_pages][Hkv][P][hd]: P rows per page, the rows of the contiguous caches (2^fa, keys rotated); table [B][table_ld]:
// physical page of a sequence's logical page; a sequence's position t is row t % P of logical page t / P.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace iie {

constexpr int PAGED_MAX_HEAD = 1024;               // head dimension: eight query heads of it as int64 are 64 KB of shared memory

struct PagedAppendArgs {
    const void *k, *v;             // new rows [T][Hkv * hd], int64 or (narrow) int32, keys before rotation
    bool narrow;
    long long k_ld, v_ld;          // distance of rows
    int32_t *kpages, *vpages;
    int n_pages, P;
    const int *table;
    long long table_ld;
    const int *start;              // [B] position of a sequence's first new row; negative: none
    const int *rows;               // [B + 1] sequence b's rows are rows[b] .. rows[b + 1] - 1; null: row b, one each
    long long T;
    int B;
    const int64_t *cos, *sin;      // [rope_rows][hd / 2]
    long long rope_rows;
    int rope, Hkv, hd, fa;
    int32_t *bounds;               // nullable [n_pages][Hkv][2][hd]: largest, smallest value of every dimension over a page's written rows
    int *flags;                    // bit 2 a value beyond int32, bit 4 a position or page outside the cache
};
cudaError_t launch_paged_append(const PagedAppendArgs &a, cudaStream_t s);

struct PagedAttnArgs {
    const int64_t *q;              // [B][H * hd] before rotation
    long long q_ld;
    const int32_t *kpages, *vpages;
    int n_pages, P;
    const int *table;
    long long table_ld;
    const int *lengths;            // [B] keys of a sequence, the new token's own among them
    long long max_len;             // their bound
    const int *sel;                // nullable [B][Hkv][n_sel]: logical pages that count (negative entries: none)
    int n_sel;
    long long window;              // > 0: the last `window` keys only
    const int64_t *cos, *sin;
    long long rope_rows;
    int rope, H, Hkv, hd, fa, B;
    long long inv_sqrt, log2e, clip;
    long long max_slots;           // keys of a sequence at most: visible ones, or rows of the selected pages
    void *work;                    // paged_attn_bytes, 16-byte aligned
    int64_t *out;                  // [B][H * hd]
    int *flags;
};
size_t paged_attn_bytes(const PagedAttnArgs &a);
cudaError_t launch_paged_attn(const PagedAttnArgs &a, cudaStream_t s);
// the form on tcgen05 (paged_tc.cu): whether a shape is its own, its scratch, its launches
bool paged_tc_ok(const PagedAttnArgs &a);
size_t paged_tc_bytes(const PagedAttnArgs &a);
cudaError_t launch_paged_tc(const PagedAttnArgs &a, cudaStream_t s);
int paged_sms();                   // SMs of the current device (0: no device)

struct PagedSelectArgs {
    const int64_t *q;
    long long q_ld;
    const int32_t *bounds;
    int n_pages, P;
    const int *table;
    long long table_ld;
    const int *lengths;
    long long max_len, window;
    const int64_t *cos, *sin;
    long long rope_rows;
    int rope, H, Hkv, hd, fa, B;
    int n_sel, keep_first, keep_last;
    long long *score;              // scratch [B][Hkv][table_ld]
    int *out;                      // [B][Hkv][n_sel]
    int *flags;
};
cudaError_t launch_paged_select(const PagedSelectArgs &a, cudaStream_t s);

#ifdef __CUDACC__
// A sequence's keys: positions lo .. len - 1.  False (and none) where the length lies outside its bound or the rotation table.
struct PagedSpan { int lo, len; };
template <typename A>
__device__ __forceinline__ bool paged_span(const A &a, int b, PagedSpan &s) {
    const long long len = a.lengths[b];
    s.lo = s.len = 0;
    if (len < 0 || len > a.max_len || (a.rope && len > a.rope_rows)) return false;
    s.len = (int)len;
    s.lo = a.window > 0 && len > a.window ? (int)(len - a.window) : 0;
    return true;
}
// rotation of a pair (x0, x1) = dimensions (2i, 2i + 1) or (i, i + hd / 2) at position pos
__device__ __forceinline__ void paged_rotate(const int64_t *cos, const int64_t *sin, int rope, int hd, int fa, long long pos, int i, int64_t &x0, int64_t &x1) {
    if (!rope) return;
    const int64_t c = cos[pos * (hd / 2) + i], s = sin[pos * (hd / 2) + i];
    const int64_t y0 = (x0 * c - x1 * s) >> fa, y1 = (x0 * s + x1 * c) >> fa;
    x0 = y0; x1 = y1;
}
#endif

}  // namespace iie
