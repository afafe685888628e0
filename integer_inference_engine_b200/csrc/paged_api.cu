// C-ABI of the paged key/value cache (include/iie_qk.h): argument checks, scratch layout, launches.  The scratch is the caller's, so calls on
// different streams, or in different captured graphs, share nothing.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/iie_qk.h"
#include "common.cuh"
#include "kernels.h"
#include "paged.h"

using namespace iie;

namespace {

constexpr long long PAGED_SLAB = 2LL << 30;        // scratch of a call: sequences beyond it go one part behind the other

bool shape_ok(int n_heads, int n_kv, int hd, int fa, int rope, const void *cos, const void *sin, long long rope_rows) {
    return n_heads > 0 && n_kv > 0 && n_heads % n_kv == 0 && n_heads <= 65535 && hd >= 2 && hd <= PAGED_MAX_HEAD && (hd & 1) == 0 && fa >= 1 && fa <= 29 &&
           rope >= 0 && rope <= 2 && (rope == 0 || (cos && sin && rope_rows > 0));
}
// (rows of a table, and of a pool and its KV heads, are numbered in 31 bits)
bool pool_ok(long long n_pages, long long P, long long n_seqs, long long table_ld) {
    return n_pages > 0 && n_pages <= INT32_MAX && P > 0 && P <= INT32_MAX && n_seqs >= 0 && n_seqs <= 65535 && table_ld > 0 && table_ld <= INT32_MAX / P;
}
// keys of a sequence at most
long long slots_of(long long max_length, long long window, long long n_sel, long long P) {
    if (n_sel > 0) return n_sel * P;
    return window > 0 ? std::min(window, max_length) : max_length;
}
PagedAttnArgs attn_shape(long long n_seqs, long long max_length, long long window, int n_sel, long long P, int n_heads, int n_kv, int hd, int fa) {
    PagedAttnArgs a = {};
    a.fa = fa;
    a.B = (int)n_seqs; a.H = n_heads; a.Hkv = n_kv; a.hd = hd; a.P = (int)P; a.n_sel = n_sel; a.window = window;
    a.max_len = max_length; a.max_slots = slots_of(max_length, window, n_sel, P);
    return a;
}
// sequences of a part whose scratch stays within the slab
long long slab_of(PagedAttnArgs a) {
    const long long n = a.B;
    a.B = 1;
    const size_t one = std::max<size_t>(1, paged_attn_bytes(a));
    return std::max<long long>(1, std::min<long long>(n, PAGED_SLAB / (long long)one));
}

}  // namespace

extern "C" int iie_paged_append_dev(const void *k_dev, const void *v_dev, int narrow, long long k_ld, long long v_ld, long long tokens, int32_t *kpages_dev,
                                    int32_t *vpages_dev, long long n_pages, long long page_rows, const int *table_dev, long long table_ld, const int *start_dev,
                                    const int *rows_dev, long long n_seqs, const int64_t *cos_dev, const int64_t *sin_dev, long long rope_rows, int rope, int n_kv,
                                    int head_dim, int fa, int32_t *bounds_dev, void *stream) {
    if (!pool_ok(n_pages, page_rows, n_seqs, table_ld) || !shape_ok(n_kv, n_kv, head_dim, fa, rope, cos_dev, sin_dev, rope_rows) || tokens < 0 || tokens > INT32_MAX ||
        k_ld < (long long)n_kv * head_dim || v_ld < (long long)n_kv * head_dim || (!rows_dev && tokens < n_seqs)) return 1;
    if (n_seqs == 0 || tokens == 0) return 0;
    int *flags = shared_flag_word();
    if (!flags || !library_is_here() || !k_dev || !v_dev || !kpages_dev || !vpages_dev || !table_dev || !start_dev) return 1;
    PagedAppendArgs a = {};
    a.k = k_dev; a.v = v_dev; a.narrow = narrow != 0; a.k_ld = k_ld; a.v_ld = v_ld; a.kpages = kpages_dev; a.vpages = vpages_dev;
    a.n_pages = (int)n_pages; a.P = (int)page_rows; a.table = table_dev; a.table_ld = table_ld; a.start = start_dev; a.rows = rows_dev; a.T = tokens; a.B = (int)n_seqs;
    a.cos = cos_dev; a.sin = sin_dev; a.rope_rows = rope_rows; a.rope = rope; a.Hkv = n_kv; a.hd = head_dim; a.fa = fa; a.bounds = bounds_dev; a.flags = flags;
    if (launch_paged_append(a, (cudaStream_t)stream) != cudaSuccess) { cudaGetLastError(); return 1; }
    return 0;
}

extern "C" long long iie_paged_attn_bytes(long long n_seqs, long long max_length, long long window, int n_selected, long long page_rows, int n_heads, int n_kv, int head_dim, int fa) {
    if (!pool_ok(1, page_rows, n_seqs, 1) || !shape_ok(n_heads, n_kv, head_dim, fa, 0, nullptr, nullptr, 0) || n_selected < 0 || max_length < 0 || max_length > INT32_MAX ||
        (long long)n_selected * page_rows > INT32_MAX) return -1;
    PagedAttnArgs a = attn_shape(n_seqs, max_length, window, n_selected, page_rows, n_heads, n_kv, head_dim, fa);
    a.B = (int)slab_of(a);
    return (long long)paged_attn_bytes(a);
}

extern "C" int iie_paged_attn_dev(const int64_t *q_dev, long long q_ld, const int32_t *kpages_dev, const int32_t *vpages_dev, long long n_pages, long long page_rows,
                                  const int *table_dev, long long table_ld, const int *lengths_dev, long long n_seqs, long long max_length, const int *selected_dev,
                                  int n_selected, long long window, const int64_t *cos_dev, const int64_t *sin_dev, long long rope_rows, int rope, int n_heads, int n_kv,
                                  int head_dim, int fa, long long inv_sqrt, void *work_dev, long long work_bytes, int64_t *out_dev, void *stream) {
    if (!pool_ok(n_pages, page_rows, n_seqs, table_ld) || !shape_ok(n_heads, n_kv, head_dim, fa, rope, cos_dev, sin_dev, rope_rows) ||
        q_ld < (long long)n_heads * head_dim || max_length < 0 || max_length > table_ld * page_rows || (selected_dev ? n_selected <= 0 : n_selected != 0) ||
        (long long)n_selected * page_rows > INT32_MAX || n_pages > INT32_MAX / page_rows / n_kv ||
        ((reinterpret_cast<uintptr_t>(kpages_dev) | reinterpret_cast<uintptr_t>(vpages_dev) | reinterpret_cast<uintptr_t>(work_dev)) & 15)) return 1;
    if (n_seqs == 0) return 0;
    int *flags = shared_flag_word();
    const long long need = iie_paged_attn_bytes(n_seqs, max_length, window, n_selected, page_rows, n_heads, n_kv, head_dim, fa);
    if (!flags || !library_is_here() || !q_dev || !kpages_dev || !vpages_dev || !table_dev || !lengths_dev || !out_dev || need < 0 || work_bytes < need || (need > 0 && !work_dev)) return 1;
    PagedAttnArgs a = attn_shape(n_seqs, max_length, window, n_selected, page_rows, n_heads, n_kv, head_dim, fa);
    a.q_ld = q_ld; a.kpages = kpages_dev; a.vpages = vpages_dev; a.n_pages = (int)n_pages; a.table_ld = table_ld;
    a.cos = cos_dev; a.sin = sin_dev; a.rope_rows = rope_rows; a.rope = rope; a.inv_sqrt = inv_sqrt; a.log2e = sigmoid_log2e(fa);
    a.clip = std::min(((long long)(fa + 2) << (2 * fa)) / a.log2e, (1LL << 62) / a.log2e);
    a.work = work_dev; a.flags = flags;
    const long long slab = slab_of(a);
    for (long long b = 0; b < n_seqs; b += slab) {
        a.B = (int)std::min(slab, n_seqs - b);
        a.q = q_dev + b * q_ld; a.table = table_dev + b * table_ld; a.lengths = lengths_dev + b; a.out = out_dev + b * n_heads * head_dim;
        a.sel = selected_dev ? selected_dev + b * n_kv * n_selected : nullptr;
        if (launch_paged_attn(a, (cudaStream_t)stream) != cudaSuccess) { cudaGetLastError(); return 1; }
    }
    return 0;
}

extern "C" int iie_paged_select_dev(const int64_t *q_dev, long long q_ld, const int32_t *bounds_dev, long long n_pages, long long page_rows, const int *table_dev,
                                    long long table_ld, const int *lengths_dev, long long n_seqs, int n_select, int keep_first, int keep_last, long long window,
                                    const int64_t *cos_dev, const int64_t *sin_dev, long long rope_rows, int rope, int n_heads, int n_kv, int head_dim, int fa,
                                    int64_t *score_dev, int *selected_dev, void *stream) {
    if (!pool_ok(n_pages, page_rows, n_seqs, table_ld) || !shape_ok(n_heads, n_kv, head_dim, fa, rope, cos_dev, sin_dev, rope_rows) ||
        q_ld < (long long)n_heads * head_dim || n_select <= 0 || keep_first < 0 || keep_last < 0 || (long long)keep_first + keep_last > n_select ||
        (long long)(n_heads / n_kv) * head_dim * 8 > 200 * 1024) return 1;
    if (n_seqs == 0) return 0;
    int *flags = shared_flag_word();
    if (!flags || !library_is_here() || !q_dev || !bounds_dev || !table_dev || !lengths_dev || !score_dev || !selected_dev) return 1;
    PagedSelectArgs a = {};
    a.q = q_dev; a.q_ld = q_ld; a.bounds = bounds_dev; a.n_pages = (int)n_pages; a.P = (int)page_rows; a.table = table_dev; a.table_ld = table_ld; a.lengths = lengths_dev;
    a.max_len = table_ld * page_rows; a.window = window; a.cos = cos_dev; a.sin = sin_dev; a.rope_rows = rope_rows; a.rope = rope; a.H = n_heads; a.Hkv = n_kv; a.hd = head_dim; a.fa = fa; a.B = (int)n_seqs;
    a.n_sel = n_select; a.keep_first = keep_first; a.keep_last = keep_last; a.score = reinterpret_cast<long long *>(score_dev); a.out = selected_dev; a.flags = flags;
    if (launch_paged_select(a, (cudaStream_t)stream) != cudaSuccess) { cudaGetLastError(); return 1; }
    return 0;
}
