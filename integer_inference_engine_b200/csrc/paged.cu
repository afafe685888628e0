// Paged key/value cache: append with rotation, ranking of pages by a bound of their scores, and the attention of one new token per
// sequence in its general form (any head dimension, page size and number of query heads).  Arithmetic of the attention: attn.cu.
//
// The general form keeps scores and exponentials in memory and takes five launches (three where no key has room): it carries the shapes that have no other.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "kernels.h"
#include "paged.h"
#include "tile_ops.cuh"

namespace cg = cooperative_groups;

namespace iie {

namespace {

// ---- append -------------------------------------------------------------------------------------------------------------------
// A CTA takes the new rows of one (page, KV head): a thread keeps a pair of dimensions and walks the rows, so that the page's bounds
// need no atomics.  They are formed again from the page's rows, old ones read back: a function of what the cache holds, whatever was
// appended and given up before.
//
// What bounds it: memory for long prompts (2350 rows of 8 KV heads of 128, 58 MB, 11.2 us: 5.2 TB/s), for a token each the launch and four dependent loads
// (a token's row, the table's entry, the row, the page's older rows; 3.2 us for 64 sequences).  A thread has the loads of PA_ROWS rows on their way
// at once; CTAs of 128 are all resident from the start (of 256, 16.3 us with four rows, 13.2 with two; 128: 14.3 with one, 12.2 with four).
constexpr int PA_THREADS = 128, PA_ROWS = 2;

template <typename T>
__global__ void __launch_bounds__(PA_THREADS) paged_append_kernel(const PagedAppendArgs a) {
    pdl_enter();
    __shared__ int s_seq, s_first, s_count;
    __shared__ long long s_page, s_row;
    __shared__ unsigned s_scan[PA_THREADS / 32];
    __shared__ int s_lim[4][PA_THREADS];
    const int tid = threadIdx.x, kv = blockIdx.y, P = a.P;
    if (tid == 0) s_seq = -1;
    __syncthreads();
    // the unit-th page that new rows reach: its sequence, first new row and count
    if (!a.rows) {
        if (tid == 0) {
            const int b = blockIdx.x, at = a.start[b];
            if (a.rope && at >= a.rope_rows) atomicOr(a.flags, 16);
            else if (at >= 0) { s_seq = b; s_page = at / P; s_first = at % P; s_count = 1; s_row = b; }
        }
    } else {
        // (Entries that descend may name so many rows that the count wraps and two sequences claim the unit: one of them gets it, within its own rows.  Counted in 64 bits,
        // 1000 sequences of four rows took 59 us instead of 50.)
        unsigned before = 0;                                       // units of the sequences in front
        for (int b0 = 0; b0 < a.B; b0 += PA_THREADS) {
            const int b = b0 + tid;
            long long at = -1, from = 0, n = 0;
            if (b < a.B) {
                at = a.start[b]; from = a.rows[b]; n = (long long)a.rows[b + 1] - from;
                if (at < 0 || n < 0 || from < 0 || from + n > a.T) n = 0;
            }
            const unsigned units = n > 0 ? (unsigned)((at + n - 1) / P - at / P + 1) : 0;
            unsigned upto = units;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) { const unsigned o = __shfl_up_sync(0xffffffffu, upto, d); if ((tid & 31) >= d) upto += o; }
            if ((tid & 31) == 31) s_scan[tid >> 5] = upto;
            __syncthreads();
            unsigned base = before, all = 0;
            for (int w = 0; w < PA_THREADS / 32; w++) { if (w < (tid >> 5)) base += s_scan[w]; all += s_scan[w]; }
            const unsigned mine = blockIdx.x - (base + upto - units);
            if (mine < units) {
                const long long p0 = (at / P + mine) * P, lo = max(at, p0), end = min(at + n, p0 + P), hi = a.rope ? min(end, a.rope_rows) : end;
                if (hi < end) atomicOr(a.flags, 16);               // positions behind the rotation table's end are left out
                if (hi > lo && atomicCAS(&s_seq, -1, b) == -1) { s_page = p0 / P; s_first = (int)(lo - p0); s_count = (int)(hi - lo); s_row = from + (lo - at); }
            }
            before += all;
            __syncthreads();
            if (s_seq >= 0 || before > blockIdx.x) break;
        }
        if (blockIdx.x == gridDim.x - 1 && kv == 0)                // who looks at every sequence's entries
            for (int b = tid; b < a.B; b += PA_THREADS)
                if (a.rows[b] < 0 || a.rows[b + 1] < a.rows[b] || a.rows[b + 1] > a.T) atomicOr(a.flags, 16);
    }
    __syncthreads();
    if (s_seq < 0) return;
    const long long logical = s_page;
    const int page = logical < a.table_ld ? a.table[(long long)s_seq * a.table_ld + logical] : -1;
    if (page < 0 || page >= a.n_pages) { if (tid == 0) atomicOr(a.flags, 16); return; }
    const int half = a.hd / 2, first = s_first, count = s_count;
    const long long cell = ((long long)page * a.Hkv + kv) * P * a.hd;
    int32_t *kp = a.kpages + cell, *vp = a.vpages + cell;
    const T *k = static_cast<const T *>(a.k) + s_row * a.k_ld + (long long)kv * a.hd, *v = static_cast<const T *>(a.v) + s_row * a.v_ld + (long long)kv * a.hd;
    bool bad = false;
    const int width = min(half, PA_THREADS), groups = PA_THREADS / width, i_own = tid % width, g = tid / width;
    for (int i0 = 0; i0 < half; i0 += width) {
        const int i = i0 + i_own, d0 = a.rope == 2 ? i : 2 * i, d1 = a.rope == 2 ? i + half : 2 * i + 1;
        int mx0 = INT32_MIN, mn0 = INT32_MAX, mx1 = INT32_MIN, mn1 = INT32_MAX;
        if (g < groups && i < half) {
            if (a.bounds)
                for (int r = g; r < first; r += groups) {
                    const int x0 = kp[(long long)r * a.hd + d0], x1 = kp[(long long)r * a.hd + d1];
                    mx0 = max(mx0, x0); mn0 = min(mn0, x0); mx1 = max(mx1, x1); mn1 = min(mn1, x1);
                }
            for (int r0 = g; r0 < count; r0 += PA_ROWS * groups) {
                int64_t x[PA_ROWS][2], y[PA_ROWS][2], c[PA_ROWS], n[PA_ROWS];
#pragma unroll
                for (int u = 0; u < PA_ROWS; u++) {
                    const int r = min(r0 + u * groups, count - 1);
                    const T *kr = k + r * a.k_ld, *vr = v + r * a.v_ld;
                    x[u][0] = kr[d0]; x[u][1] = kr[d1]; y[u][0] = vr[d0]; y[u][1] = vr[d1];
                    const long long turn = (logical * P + first + r) * half + i;
                    c[u] = a.rope ? a.cos[turn] : 0; n[u] = a.rope ? a.sin[turn] : 0;
                }
#pragma unroll
                for (int u = 0; u < PA_ROWS; u++) {
                    const int r = r0 + u * groups;
                    if (r >= count) break;
                    int64_t x0 = x[u][0], x1 = x[u][1];
                    const int64_t y0 = y[u][0], y1 = y[u][1];
                    if (a.rope) { x0 = (x[u][0] * c[u] - x[u][1] * n[u]) >> a.fa; x1 = (x[u][0] * n[u] + x[u][1] * c[u]) >> a.fa; }
                    bad = bad || x0 != (int32_t)x0 || x1 != (int32_t)x1 || y0 != (int32_t)y0 || y1 != (int32_t)y1;
                    const long long to = (long long)(first + r) * a.hd;
                    kp[to + d0] = (int32_t)x0; kp[to + d1] = (int32_t)x1; vp[to + d0] = (int32_t)y0; vp[to + d1] = (int32_t)y1;
                    mx0 = max(mx0, (int32_t)x0); mn0 = min(mn0, (int32_t)x0); mx1 = max(mx1, (int32_t)x1); mn1 = min(mn1, (int32_t)x1);
                }
            }
        }
        if (a.bounds) {
            __syncthreads();
            s_lim[0][tid] = mx0; s_lim[1][tid] = mn0; s_lim[2][tid] = mx1; s_lim[3][tid] = mn1;
            __syncthreads();
            if (g == 0 && i < half) {
                for (int o = 1; o < groups; o++) {
                    const int t = o * width + tid;
                    mx0 = max(mx0, s_lim[0][t]); mn0 = min(mn0, s_lim[1][t]); mx1 = max(mx1, s_lim[2][t]); mn1 = min(mn1, s_lim[3][t]);
                }
                int32_t *to = a.bounds + ((long long)page * a.Hkv + kv) * 2 * a.hd;
                to[d0] = mx0; to[d1] = mx1; to[a.hd + d0] = mn0; to[a.hd + d1] = mn1;
            }
        }
    }
    if (bad) atomicOr(a.flags, 4);
}

// ---- attention, general form ------------------------------------------------------------------------------------------------------
// Any head dimension, page and scale, in five launches: a start, scores with their maxima by 64 keys a CTA, exponentials with their sums, probabilities times values, the last shift;
// what lies between them is in memory as 64 bits.  Bound by its 64-bit multiply-adds: 8 sequences of 2000 keys, 2 KV heads of 256, 116 us, 0.56 TB/s (of 128, through the
// tensor cores, 22); 64 of 4096 keys, 4 KV heads of 128 in pages of 12 rows, 2.12 ms.
constexpr int PG_HEADS = 8, PG_KEYS = 64;

struct GeneralWork {
    long long *score;              // [B][H][slots]: scores, then exponentials
    long long *top;                // [B][H]
    unsigned long long *z;         // [B][H]
    long long *acc;                // [B][H][hd]
};
__host__ __device__ inline GeneralWork general_work(const PagedAttnArgs &a) {
    GeneralWork w;
    const long long rows = (long long)a.B * a.H;
    w.score = static_cast<long long *>(a.work);
    w.top = w.score + rows * a.max_slots;
    w.z = reinterpret_cast<unsigned long long *>(w.top + rows);
    w.acc = reinterpret_cast<long long *>(w.z + rows);
    return w;
}
// Row of slot j: key j of the visible ones, or row j of the selected pages; false where there is none.
__device__ __forceinline__ bool general_row(const PagedAttnArgs &a, const PagedSpan &s, int b, int kv, long long j, long long &row, bool &bad) {
    long long logical, r;
    if (a.sel) {
        if (j >= (long long)a.n_sel * a.P) return false;
        logical = a.sel[((long long)b * a.Hkv + kv) * a.n_sel + j / a.P];
        r = j % a.P;
        if (logical < 0) return false;
        if (logical >= a.table_ld) { bad = true; return false; }
        const long long pos = logical * a.P + r;
        if (pos < s.lo || pos >= s.len) return false;
    } else {
        const long long pos = s.lo + j;
        if (pos >= s.len) return false;
        logical = pos / a.P; r = pos % a.P;
    }
    const int page = a.table[(long long)b * a.table_ld + logical];
    if (page < 0 || page >= a.n_pages) { bad = true; return false; }
    row = ((long long)page * a.Hkv + kv) * a.P + r;
    return true;
}

__global__ void paged_general_init_kernel(const PagedAttnArgs a) {
    pdl_enter();
    const GeneralWork w = general_work(a);
    const long long rows = (long long)a.B * a.H, n = rows * a.hd;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        w.acc[i] = 0;
        if (i < rows) { w.top[i] = INT64_MIN; w.z[i] = 0; }
    }
}

// scores of 64 slots for up to eight query heads of a KV head: a warp per key, lanes over the dimensions
__global__ void __launch_bounds__(256) paged_general_scores_kernel(const PagedAttnArgs a) {
    pdl_enter();
    extern __shared__ __align__(16) int64_t pg_q[];                // [8][hd]
    const GeneralWork w = general_work(a);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rep = a.H / a.Hkv, groups = (rep + PG_HEADS - 1) / PG_HEADS;
    const int b = blockIdx.z, kv = blockIdx.y / groups, h0 = (blockIdx.y % groups) * PG_HEADS, heads = min(PG_HEADS, rep - h0), half = a.hd / 2;
    PagedSpan s;
    if (!paged_span(a, b, s)) { if (tid == 0 && blockIdx.x == 0 && blockIdx.y == 0) atomicOr(a.flags, 16); return; }
    const long long j0 = (long long)blockIdx.x * PG_KEYS;
    if (s.len == 0 || (!a.sel && s.lo + j0 >= s.len)) return;
    for (int idx = tid; idx < heads * half; idx += blockDim.x) {
        const int h = idx / half, i = idx % half, d0 = a.rope == 2 ? i : 2 * i, d1 = a.rope == 2 ? i + half : 2 * i + 1;
        const int64_t *src = a.q + b * a.q_ld + (long long)(kv * rep + h0 + h) * a.hd;
        int64_t x0 = src[d0], x1 = src[d1];
        paged_rotate(a.cos, a.sin, a.rope, a.hd, a.fa, s.len - 1, i, x0, x1);
        pg_q[h * a.hd + d0] = x0; pg_q[h * a.hd + d1] = x1;
    }
    __syncthreads();
    long long best[PG_HEADS];
#pragma unroll
    for (int h = 0; h < PG_HEADS; h++) best[h] = INT64_MIN;
    bool bad = false;
    for (long long j = j0 + warp; j < min(j0 + PG_KEYS, a.max_slots); j += 8) {
        long long row = 0;
        const bool seen = general_row(a, s, b, kv, j, row, bad);
#pragma unroll
        for (int h = 0; h < PG_HEADS; h++) {
            if (h >= heads) break;
            uint64_t dot = 0;
            if (seen) for (int d = lane; d < a.hd; d += 32) dot += (uint64_t)pg_q[h * a.hd + d] * (uint64_t)(int64_t)a.kpages[row * a.hd + d];
#pragma unroll
            for (int m = 16; m > 0; m >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, m);
            const long long sc = (long long)((uint64_t)((int64_t)dot >> a.fa) * (uint64_t)a.inv_sqrt) >> a.fa;
            if (lane == 0) w.score[((long long)b * a.H + kv * rep + h0 + h) * a.max_slots + j] = seen ? sc : INT64_MIN;
            if (seen) best[h] = max(best[h], sc);
        }
    }
    if (lane == 0)
#pragma unroll
        for (int h = 0; h < PG_HEADS; h++)
            if (h < heads && best[h] != INT64_MIN) atomicMax(w.top + (long long)b * a.H + kv * rep + h0 + h, best[h]);
    if (bad && lane == 0) atomicOr(a.flags, 16);
}

__global__ void __launch_bounds__(256) paged_general_exp_kernel(const PagedAttnArgs a) {
    pdl_enter();
    const GeneralWork w = general_work(a);
    const long long row = (long long)blockIdx.z * a.H + blockIdx.y, top = w.top[row];
    if (top == INT64_MIN) return;                                   // no key
    PagedSpan s;
    paged_span(a, blockIdx.z, s);
    const long long n = a.sel ? a.max_slots : min(a.max_slots, (long long)(s.len - s.lo));
    unsigned long long z = 0;
    for (long long j = (long long)blockIdx.x * 1024 + threadIdx.x; j < min(n, (long long)(blockIdx.x + 1) * 1024); j += 256) {
        const long long sc = w.score[row * a.max_slots + j];
        long long e = 0;
        if (sc != INT64_MIN) {
            const uint64_t below = min((uint64_t)top - (uint64_t)sc, (uint64_t)a.clip);
            e = exp2_neg_fixed((int64_t)(below * (uint64_t)a.log2e) >> a.fa, a.fa);
        }
        w.score[row * a.max_slots + j] = e;
        z += (unsigned long long)e;
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) z += __shfl_xor_sync(0xffffffffu, z, m);
    if ((threadIdx.x & 31) == 0 && z) atomicAdd(w.z + row, z);
}

// sum of p v over 128 slots: 32 dimensions x 8 groups of slots per CTA and turn
__global__ void __launch_bounds__(256) paged_general_values_kernel(const PagedAttnArgs a) {
    pdl_enter();
    __shared__ long long s_p[PG_HEADS][128];
    __shared__ long long s_row[128];
    const GeneralWork w = general_work(a);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rep = a.H / a.Hkv, groups = (rep + PG_HEADS - 1) / PG_HEADS;
    const int b = blockIdx.z, kv = blockIdx.y / groups, h0 = (blockIdx.y % groups) * PG_HEADS, heads = min(PG_HEADS, rep - h0);
    PagedSpan s;
    if (!paged_span(a, b, s)) return;
    const long long j0 = (long long)blockIdx.x * 128;
    if (s.len == 0 || (!a.sel && s.lo + j0 >= s.len)) return;
    bool bad = false;
    for (int i = tid; i < 128; i += 256) {
        long long row = -1;
        if (j0 + i >= a.max_slots || !general_row(a, s, b, kv, j0 + i, row, bad)) row = -1;
        s_row[i] = row;
    }
    __syncthreads();
    for (int i = tid; i < heads * 128; i += 256) {
        const int h = i >> 7, j = i & 127;
        const long long head = (long long)b * a.H + kv * rep + h0 + h;
        const unsigned long long z = w.z[head];
        s_p[h][j] = s_row[j] >= 0 && z ? (long long)(((unsigned long long)w.score[head * a.max_slots + j0 + j] << a.fa) / z) : 0;
    }
    __syncthreads();
    for (int d = lane; d < a.hd; d += 32) {
        long long sum[PG_HEADS];
#pragma unroll
        for (int h = 0; h < PG_HEADS; h++) sum[h] = 0;
        for (int j = warp * 16; j < warp * 16 + 16; j++) {
            if (s_row[j] < 0) continue;
            const long long v = a.vpages[s_row[j] * a.hd + d];
#pragma unroll
            for (int h = 0; h < PG_HEADS; h++) if (h < heads) sum[h] += s_p[h][j] * v;
        }
#pragma unroll
        for (int h = 0; h < PG_HEADS; h++)
            if (h < heads && sum[h]) atomicAdd(reinterpret_cast<unsigned long long *>(w.acc + ((long long)b * a.H + kv * rep + h0 + h) * a.hd + d), (unsigned long long)sum[h]);
    }
}

__global__ void paged_general_out_kernel(const PagedAttnArgs a) {
    pdl_enter();
    const GeneralWork w = general_work(a);
    const long long n = (long long)a.B * a.H * a.hd;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) a.out[i] = w.acc[i] >> a.fa;
}

// ---- ranking of pages -----------------------------------------------------------------------------------------------------------
// score(page) = max over the heads of a KV head of sum_i max(q_i mx_i, q_i mn_i), an upper bound of q . k over the page's keys.  The general form, a warp per page with its
// lanes over the dimensions (8 sequences of 500 pages, 2 KV heads of 24: 20 us; of 32, by the forms below, 11).
__global__ void __launch_bounds__(256) paged_rank_kernel(const PagedSelectArgs a) {
    pdl_enter();
    extern __shared__ __align__(16) int64_t pg_q[];                // [rep][hd]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rep = a.H / a.Hkv, b = blockIdx.z, kv = blockIdx.y, half = a.hd / 2;
    PagedSpan s;
    if (!paged_span(a, b, s)) { if (tid == 0 && blockIdx.x == 0 && kv == 0) atomicOr(a.flags, 16); return; }
    const int first = s.lo / a.P, last = (s.len + a.P - 1) / a.P;      // pages first .. last - 1
    const int page0 = first + blockIdx.x * 32;
    if (page0 >= last) return;
    for (int idx = tid; idx < rep * half; idx += blockDim.x) {
        const int h = idx / half, i = idx % half, d0 = a.rope == 2 ? i : 2 * i, d1 = a.rope == 2 ? i + half : 2 * i + 1;
        const int64_t *src = a.q + b * a.q_ld + (long long)(kv * rep + h) * a.hd;
        int64_t x0 = src[d0], x1 = src[d1];
        paged_rotate(a.cos, a.sin, a.rope, a.hd, a.fa, s.len - 1, i, x0, x1);
        pg_q[h * a.hd + d0] = x0; pg_q[h * a.hd + d1] = x1;
    }
    __syncthreads();
    bool bad = false;
    for (int at = page0 + warp; at < min(page0 + 32, last); at += 8) {
        const int page = a.table[(long long)b * a.table_ld + at];
        long long best = INT64_MIN;
        if (page < 0 || page >= a.n_pages) bad = true;
        else {
            const int32_t *mx = a.bounds + ((long long)page * a.Hkv + kv) * 2 * a.hd, *mn = mx + a.hd;
            for (int h = 0; h < rep; h++) {
                uint64_t sum = 0;
                for (int d = lane; d < a.hd; d += 32) {
                    const int64_t q = pg_q[h * a.hd + d];
                    sum += (uint64_t)q * (uint64_t)(int64_t)(q > 0 ? mx[d] : mn[d]);
                }
#pragma unroll
                for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
                best = max(best, (long long)sum);
            }
        }
        if (lane == 0) a.score[((long long)b * a.Hkv + kv) * a.table_ld + at - first] = best;
    }
    if (bad && lane == 0) atomicOr(a.flags, 16);
}

// ---- the best pages of one (sequence, KV head), by one CTA -------------------------------------------------------------------------
// Pages that always count apart, the rest by radix selection from the highest bit in which scores differ: eight bits a pass, until a bin ends
// where the selection does (two passes as a rule; from the top byte, which nearly all share, every count would hit one bin).  Equal scores: the
// lowest pages.  Then the pages in order.
constexpr int PS_THREADS = 256, PK_HELD = 8192;    // scores that shared memory has room for
struct PickScratch {
    int hist[256], scan[2][PS_THREADS / 32], digit, left, count;
    unsigned long long ends[2][PS_THREADS / 32];
};
template <typename Score>                          // score of the i-th visible page
__device__ void pick_pages(const PagedSelectArgs &a, PickScratch &s, int first, int n, int *out, Score score) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, from = min(a.keep_first, n), to = max(from, n - a.keep_last);      // ranked: from .. to - 1
    int left = min(n, a.n_sel) - (n - (to - from));                // of the ranked pages
    auto key = [&](int i) -> uint64_t { return (uint64_t)score(i) ^ (1ULL << 63); };
    uint64_t lo = ~0ULL, hi = 0;
    for (int i = from + tid; i < to; i += PS_THREADS) { const uint64_t u = key(i); lo = u < lo ? u : lo; hi = u > hi ? u : hi; }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) {
        const uint64_t l2 = __shfl_xor_sync(0xffffffffu, lo, m), h2 = __shfl_xor_sync(0xffffffffu, hi, m);
        lo = l2 < lo ? l2 : lo; hi = h2 > hi ? h2 : hi;
    }
    if (lane == 0) { s.ends[0][warp] = lo; s.ends[1][warp] = hi; }
    __syncthreads();
    for (int w = 0; w < PS_THREADS / 32; w++) { lo = s.ends[0][w] < lo ? s.ends[0][w] : lo; hi = s.ends[1][w] > hi ? s.ends[1][w] : hi; }
    int shift = 64 - __clzll((long long)(lo ^ hi));                // bits from `shift` on are everyone's
    uint64_t limit = shift < 64 ? hi >> shift : 0;                 // of the digits found so far
    while (shift > 0 && left > 0) {                                // (uniform)
        const int bits = min(8, shift);
        shift -= bits;
        s.hist[tid] = 0;
        __syncthreads();
        for (int i = from + tid; i < to; i += PS_THREADS) {
            const uint64_t u = key(i);
            if (shift + bits == 64 || (u >> (shift + bits)) == limit) atomicAdd(&s.hist[(u >> shift) & ((1u << bits) - 1)], 1);
        }
        __syncthreads();
        if (warp == 0) {                                           // the digit where the left-th largest lies: lane l has digits 255 - 8l ..
            int mine = 0;
            for (int d = 0; d < 8; d++) mine += s.hist[255 - 8 * lane - d];
            int upto = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) { const int o = __shfl_up_sync(0xffffffffu, upto, d); if (lane >= d) upto += o; }
            int above = upto - mine;
            if (above < left && upto >= left)
                for (int d = 0; d < 8; d++) {
                    const int c = s.hist[255 - 8 * lane - d];
                    if (above + c >= left) { s.digit = 255 - 8 * lane - d; s.left = left - above; s.count = c; break; }
                    above += c;
                }
        }
        __syncthreads();
        limit = (shift + bits == 64 ? 0 : limit << bits) | (uint64_t)s.digit;
        left = s.left;
        const bool all = s.count == left;
        __syncthreads();
        if (all) break;
    }
    if (shift == 64) shift = 0;                                    // (nothing ranked: lo ^ hi has its top bit)
    // a warp has a run of pages: what it takes is counted, then written behind what the warps before it take
    const int strips = (n + PS_THREADS - 1) / PS_THREADS, i0 = warp * strips * 32;
    auto look = [&](int i, bool &sure, bool &eq) {
        const bool ranked = i >= from && i < to;
        const uint64_t u = ranked ? key(i) >> shift : 0;
        sure = i < n && (!ranked || (left > 0 && u > limit));
        eq = ranked && left > 0 && u == limit;
    };
    int sures = 0, eqs = 0;
    for (int k = 0; k < strips; k++) {
        bool sure, eq;
        look(i0 + 32 * k + lane, sure, eq);
        sures += __popc(__ballot_sync(0xffffffffu, sure)); eqs += __popc(__ballot_sync(0xffffffffu, eq));
    }
    if (lane == 0) { s.scan[0][warp] = sures; s.scan[1][warp] = eqs; }
    __syncthreads();
    int at = 0, eq_before = 0;
    for (int w = 0; w < warp; w++) { at += s.scan[0][w] + max(0, min(s.scan[1][w], left - eq_before)); eq_before += s.scan[1][w]; }
    for (int k = 0; k < strips; k++) {
        const int i = i0 + 32 * k + lane;
        const unsigned below = (1u << lane) - 1;
        bool sure, eq;
        look(i, sure, eq);
        const unsigned eq_all = __ballot_sync(0xffffffffu, eq);
        const bool in = sure || (eq && eq_before + __popc(eq_all & below) < left);
        const unsigned in_all = __ballot_sync(0xffffffffu, in);
        if (in) out[at + __popc(in_all & below)] = first + i;
        at += __popc(in_all); eq_before += __popc(eq_all);
    }
}
// Visible pages first .. first + n - 1; what is not ranked is written: the whole list where they all fit, -1 behind its end.
__device__ __forceinline__ bool pick_begin(const PagedSelectArgs &a, int b, int kv, int &first, int &n, int *&out) {
    PagedSpan s;
    const bool ok = paged_span(a, b, s);
    out = a.out + ((long long)b * a.Hkv + kv) * a.n_sel;
    first = s.lo / a.P;
    n = ok && s.len > 0 ? (s.len - 1) / a.P - first + 1 : 0;
    return n > a.n_sel;
}
__device__ __forceinline__ void pick_rest(const PagedSelectArgs &a, int first, int n, int *out) {
    for (int i = threadIdx.x; i < a.n_sel; i += blockDim.x)
        if (i >= n) out[i] = -1;
        else if (n <= a.n_sel) out[i] = first + i;
}

__global__ void __launch_bounds__(PS_THREADS) paged_pick_kernel(const PagedSelectArgs a, const bool held) {
    pdl_enter();
    __shared__ PickScratch s;
    const int kv = blockIdx.x, b = blockIdx.y;
    int first, n, *out;
    const bool rank = pick_begin(a, b, kv, first, n, out);
    pick_rest(a, first, n, out);
    if (!rank) return;
    extern __shared__ long long pk_score[];
    const long long *score = a.score + ((long long)b * a.Hkv + kv) * a.table_ld;
    if (held) {                                    // (a pass over them in memory costs a microsecond)
        for (int i = threadIdx.x; i < n; i += 8 * PS_THREADS) {
            long long x[8];
#pragma unroll
            for (int u = 0; u < 8; u++) x[u] = score[min(i + u * PS_THREADS, n - 1)];
#pragma unroll
            for (int u = 0; u < 8; u++)
                if (i + u * PS_THREADS < n) pk_score[i + u * PS_THREADS] = x[u];
        }
        __syncthreads();
        score = pk_score;
    }
    pick_pages(a, s, first, n, out, [&](int i) { return score[i]; });
}

// Both in one launch where head dimension and page count allow (up to 1024: two turns of a cluster): a cluster of CTAs per (sequence, KV head) ranks the pages, 64 at a time each,
// into the first CTA's shared memory, and that one picks.  A warp has the bounds of eight pages copied into shared memory (a page's 8 hd bytes lie
// side by side; a gap behind each keeps the banks apart); four lanes share a page, a lane takes every fourth group of four dimensions of eight
// heads: 32 x 32 -> 64-bit multiply-adds (four clocks a warp) of a query value with the bound that its sign selects (four clocks on the
// other pipe).  What bounds it: those, 4 us a turn of 64 pages for two CTAs of an SM (3 of them multiply-adds), the query's 2 and picking's 3 to 7: 8.8 us for a sequence
// of 500 pages (4 KV heads of two bounds of 128, 8 query heads each).  (A page's bounds copied as halves, the next ones' while the others are multiplied: a third
// slower, four times as many copies.  Loads into registers instead, two pages a lane: four round trips a page, twice the time.)  A query beyond int32 takes
// 64-bit products.
constexpr int PR_PAGES = 8;                        // pages of a warp at a time
constexpr int PR_GAP = 64;
constexpr size_t PR_SHARED = 220 * 1024;           // of a CTA at most: queries and the warps' pages, beside them (in the one-launch form) the scores
constexpr int PR_CLUSTER = 8, PR_TURN = PR_PAGES * (PS_THREADS / 32), PR_MOST = 2 * PR_CLUSTER * PR_TURN;     // CTAs of a cluster; pages of one at a time; of a list for this form
__host__ __device__ inline int rank_heads(int rep) { return rep <= 4 ? 4 : (rep + 7) / 8 * 8; }
__host__ __device__ inline size_t rank_stage(int hd) { return (size_t)PR_PAGES * (8 * hd + PR_GAP); }       // of a warp
template <bool WIDE, int HEADS>                   // HEADS at a time: the queries are padded with zeros to a multiple
__device__ __forceinline__ bool rank_pages(const PagedSelectArgs &a, const int *q32, const int64_t *q64, unsigned char *stage, uint64_t *bar, int rep, int b, int kv, int first, int n, long long *to, int turn, int block,
                                           int blocks, uint32_t &pass, bool &bad, volatile int *abort_flag) {
    const int lane = threadIdx.x & 31, t = lane & 3, g = lane >> 2, ld = 8 * a.hd + PR_GAP;
    const uint32_t bar_at = tl_u32(bar), to_at = tl_u32(stage);
    const int step = blocks * (PS_THREADS / 32) * PR_PAGES;
    for (int p0 = (block * (PS_THREADS / 32) + turn) * PR_PAGES; p0 < n; p0 += step, pass ^= 1) {
        // the warp's pages; one outside the pool counts as lowest
        int page = -1;
        if (lane < PR_PAGES && p0 + lane < n) {
            page = a.table[(long long)b * a.table_ld + first + p0 + lane];
            if (page < 0 || page >= a.n_pages) { bad = true; page = -1; }
        }
        const unsigned there = __ballot_sync(0xffffffffu, page >= 0);
        if (lane == 0) tl_expect(bar_at, (uint32_t)__popc(there) * 8 * a.hd);
        __syncwarp();
        if (page >= 0)
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                         ::"r"(to_at + lane * ld), "l"(a.bounds + ((long long)page * a.Hkv + kv) * 2 * a.hd), "r"(8 * a.hd), "r"(bar_at) : "memory");
        if (!tl_wait(bar_at, pass, abort_flag)) {
            volatile int patient = 0;              // copies under way end first
            tl_wait_slow(bar_at, pass, &patient);
            return false;
        }
        const int4 *row = reinterpret_cast<const int4 *>(stage + g * ld) + t;
        long long best = INT64_MIN;
        for (int h0 = 0; h0 < rep; h0 += HEADS) {
            long long sum[HEADS];
#pragma unroll
            for (int h = 0; h < HEADS; h++) sum[h] = 0;
            const int4 *q4 = reinterpret_cast<const int4 *>(q32 + h0 * a.hd) + t;
#pragma unroll 1
            for (int d = 0; d < a.hd; d += 16) {
                const int4 mx = row[d / 4], mn = row[(a.hd + d) / 4];
                if (!WIDE) {
                    int4 q[HEADS];
#pragma unroll
                    for (int h = 0; h < HEADS; h++) q[h] = q4[(h * a.hd + d) / 4];
#pragma unroll
                    for (int h = 0; h < HEADS; h++) sum[h] += (long long)q[h].x * (q[h].x < 0 ? mn.x : mx.x);
#pragma unroll
                    for (int h = 0; h < HEADS; h++) sum[h] += (long long)q[h].y * (q[h].y < 0 ? mn.y : mx.y);
#pragma unroll
                    for (int h = 0; h < HEADS; h++) sum[h] += (long long)q[h].z * (q[h].z < 0 ? mn.z : mx.z);
#pragma unroll
                    for (int h = 0; h < HEADS; h++) sum[h] += (long long)q[h].w * (q[h].w < 0 ? mn.w : mx.w);
                } else {
#pragma unroll
                    for (int h = 0; h < HEADS; h++)
#pragma unroll 1
                        for (int e = 0; e < 4; e++) {
                            const int64_t q = q64[(h0 + h) * a.hd + d + 4 * t + e];
                            const int4 v = q < 0 ? mn : mx;
                            sum[h] = (long long)((uint64_t)sum[h] + (uint64_t)q * (uint64_t)(int64_t)(e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w));
                        }
                }
            }
#pragma unroll
            for (int h = 0; h < HEADS; h++) {
                sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
                sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
                if (h0 + h < rep) best = max(best, sum[h]);
            }
        }
        if (t == 0 && p0 + g < n) to[p0 + g] = (there >> g) & 1 ? best : INT64_MIN;
        __syncwarp();                                              // the stage may be filled again
    }
    return true;
}
// The queries of a KV head, rotated, as int64 and as int32: whether one of the thread's is beyond that.
__device__ __forceinline__ bool rank_queries(const PagedSelectArgs &a, int b, int kv, int rep, int padded, int64_t *q64, int *q32) {
    const int half = a.hd / 2;
    bool wide = false;
    const long long pos = a.lengths[b] - 1;
    for (int idx = threadIdx.x; idx < padded * half; idx += PS_THREADS) {
        const int h = idx / half, i = idx - h * half, d0 = a.rope == 2 ? i : 2 * i, d1 = a.rope == 2 ? i + half : 2 * i + 1;
        int64_t x0 = 0, x1 = 0;
        if (h < rep) {
            const int64_t *src = a.q + b * a.q_ld + (long long)(kv * rep + h) * a.hd;
            x0 = src[d0]; x1 = src[d1];
            paged_rotate(a.cos, a.sin, a.rope, a.hd, a.fa, pos, i, x0, x1);
        }
        q64[h * a.hd + d0] = x0; q64[h * a.hd + d1] = x1;
        q32[h * a.hd + d0] = (int)x0; q32[h * a.hd + d1] = (int)x1;
        wide = wide || x0 != (int)x0 || x1 != (int)x1;
    }
    return wide;
}
__global__ void __launch_bounds__(PS_THREADS, 2) paged_select_kernel(const PagedSelectArgs a) {
    pdl_enter();
    extern __shared__ __align__(16) int64_t pr_q[];                // queries [rep][hd] as int64, then as int32; the warps' pages; scores
    __shared__ PickScratch s;
    __shared__ __align__(8) uint64_t s_bar[PS_THREADS / 32];
    __shared__ int s_wide, s_abort;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, rep = a.H / a.Hkv, block = blockIdx.x, blocks = gridDim.x, kv = blockIdx.y, b = blockIdx.z;
    const int padded = rank_heads(rep);
    int *q32 = reinterpret_cast<int *>(pr_q + padded * a.hd);
    unsigned char *stage = reinterpret_cast<unsigned char *>(q32 + padded * a.hd);
    long long *score = reinterpret_cast<long long *>(stage + PS_THREADS / 32 * rank_stage(a.hd));
    int first, n, *out;
    const bool rank = pick_begin(a, b, kv, first, n, out);
    if (block == 0) pick_rest(a, first, n, out);
    if (!rank) {                                                   // the whole cluster
        PagedSpan span;
        if (tid == 0 && block == 0 && kv == 0 && !paged_span(a, b, span)) atomicOr(a.flags, 16);
        return;
    }
    if (tid == 0) {
        s_wide = 0; s_abort = 0;
        for (int w = 0; w < PS_THREADS / 32; w++) tl_init(tl_u32(&s_bar[w]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    bool bad = false;
    uint32_t pass = 0;
    const bool wide = rank_queries(a, b, kv, rep, padded, pr_q, q32);
    if (wide) s_wide = 1;
    if (blocks > 1) cluster.sync();                                // (the first CTA has started)
    else __syncthreads();
    long long *to = blocks > 1 ? cluster.map_shared_rank(score, 0) : score;
    unsigned char *mine = stage + (tid >> 5) * rank_stage(a.hd);
    const bool ok = s_wide ? rank_pages<true, 4>(a, q32, pr_q, mine, &s_bar[tid >> 5], rep, b, kv, first, n, to, tid >> 5, block, blocks, pass, bad, &s_abort)
                  : rep <= 4 ? rank_pages<false, 4>(a, q32, pr_q, mine, &s_bar[tid >> 5], rep, b, kv, first, n, to, tid >> 5, block, blocks, pass, bad, &s_abort)
                             : rank_pages<false, 8>(a, q32, pr_q, mine, &s_bar[tid >> 5], rep, b, kv, first, n, to, tid >> 5, block, blocks, pass, bad, &s_abort);
    if (!ok) atomicOr(a.flags, FLAG_GAVE_UP);
    if (bad) atomicOr(a.flags, 16);
    if (blocks > 1) cluster.sync();
    else __syncthreads();
    if (block == 0) pick_pages(a, s, first, n, out, [&](int i) { return score[i]; });
}

// Longer lists, in a launch of their own: the pages of all sequences and KV heads shared evenly, each pair of them by CTAs in proportion to its pages
// (whole groups of eight), two CTAs an SM.  For tables of more than 1024 pages, or of more than 128 where the clusters would not all be resident at once, whatever the lengths
// (a table of 2048 pages: 32 x 62 pages 17.9 in place of 11.2, 1 x 500 14.3 of 11.6, 8 x 500 23.2 of 18.1).  Both forms, a call alone,
// us (clusters first): 1 x 1000 pages 12.5 and 13.5, 1 x 2000 19.6 and 15.9, 1 x 8000 60.6 and 33.5; 8 x 500 13.9 and 19.4, 16 x 500 24.0 and 21.6, 32 x 1000 70.5 and 64.4; 64 x 200 38.6 and
// 32.2, 150 x 120 45.1 and 53.1, 300 x 60 41.7 and 65.4; 8 x up to 2000 29.7 and 27.1: plan 2, the part's place and query 2, ranking 11 to 15 (multiply-adds 8 of them), the launch
// between 1, picking 5.
__global__ void __launch_bounds__(PS_THREADS, 2) paged_rank_even_kernel(const PagedSelectArgs a) {
    pdl_enter();
    extern __shared__ __align__(16) int64_t pr_q[];                // queries as int64, then as int32; the warps' pages
    __shared__ __align__(8) uint64_t s_bar[PS_THREADS / 32];
    __shared__ int s_wide, s_abort, s_b, s_kv, s_from, s_count, s_first;
    __shared__ long long s_units;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rep = a.H / a.Hkv, padded = rank_heads(rep), ctas = gridDim.x;
    int *q32 = reinterpret_cast<int *>(pr_q + padded * a.hd);
    unsigned char *mine = reinterpret_cast<unsigned char *>(q32 + padded * a.hd) + warp * rank_stage(a.hd);
    if (tid == 0) {
        s_abort = 0;
        for (int w = 0; w < PS_THREADS / 32; w++) tl_init(tl_u32(&s_bar[w]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // pages of a sequence that are ranked; the first visible one
    auto pages = [&](int b, int &first) {
        PagedSpan s;
        first = 0;
        if (b >= a.B) return 0;
        if (!paged_span(a, b, s)) { if (blockIdx.x == 0) atomicOr(a.flags, 16); return 0; }
        first = s.lo / a.P;
        const int n = s.len > 0 ? (s.len - 1) / a.P - first + 1 : 0;
        return n > a.n_sel ? n : 0;
    };
    auto added = [&](long long x) {
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
        return x;
    };
    int quota = 1, first0 = 0, n0 = 0, first;                      // of warp 0: pages of a CTA on average; those of the first 32 sequences
    // pages of a part, parts
    auto parts_most = [&](int n) { return max(1, n / quota); };
    auto size = [&](int n) { const int p = parts_most(n); return ((n + p - 1) / p + PR_PAGES - 1) / PR_PAGES * PR_PAGES; };
    auto parts = [&](int n) { return n == 0 ? 0 : (n + size(n) - 1) / size(n); };
    if (warp == 0) {
        n0 = pages(lane, first0);
        long long total = n0, units = 0;
        for (int b = lane + 32; b - lane < a.B; b += 32) total += pages(b, first);
        total = added(total) * a.Hkv;
        quota = (int)max(1LL, min((total + ctas - 1) / ctas, (long long)INT32_MAX));
        units = parts(n0);
        for (int b = lane + 32; b - lane < a.B; b += 32) units += parts(pages(b, first));
        units = added(units) * a.Hkv;
        if (lane == 0) s_units = units;
    }
    __syncthreads();
    const long long units = s_units;
    const int turn = (warp + 2 * ((blockIdx.x & 1) ^ (blockIdx.x >= ctas / 2))) & 7;      // (warps with a group more of an SM's two CTAs issue from different places)
    uint32_t pass = 0;
    bool bad = false, ok = true;
    int b0 = 0;                                                    // of warp 0: sequences searched so far, their parts
    long long before = 0;
    for (long long unit = blockIdx.x; unit < units; unit += ctas) {
        if (warp == 0)                                             // its sequence, KV head, pages; the search goes on where the last one ended
            for (; b0 < a.B; b0 += 32) {
                first = first0;
                const int n = b0 ? pages(b0 + lane, first) : n0, each = parts(n), own = each * a.Hkv;
                long long upto = own;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) { const long long o = __shfl_up_sync(0xffffffffu, upto, d); if (lane >= d) upto += o; }
                const long long in = unit - (before + upto - own);
                if (in >= 0 && in < own) {
                    const int kv = (int)in / each, at = ((int)in - kv * each) * size(n);
                    s_b = b0 + lane; s_kv = kv; s_from = at; s_count = min(size(n), n - at); s_first = first;
                }
                const long long behind = before + __shfl_sync(0xffffffffu, upto, 31);
                if (behind > unit) break;
                before = behind;
            }
        if (tid == 0) s_wide = 0;
        __syncthreads();
        const int b = s_b, kv = s_kv, from = s_first + s_from, n = s_count;
        if (rank_queries(a, b, kv, rep, padded, pr_q, q32)) s_wide = 1;
        long long *to = a.score + ((long long)b * a.Hkv + kv) * a.table_ld + s_from;
        __syncthreads();
        ok = ok && (s_wide ? rank_pages<true, 4>(a, q32, pr_q, mine, &s_bar[warp], rep, b, kv, from, n, to, turn, 0, 1, pass, bad, &s_abort)
                    : rep <= 4 ? rank_pages<false, 4>(a, q32, pr_q, mine, &s_bar[warp], rep, b, kv, from, n, to, turn, 0, 1, pass, bad, &s_abort)
                               : rank_pages<false, 8>(a, q32, pr_q, mine, &s_bar[warp], rep, b, kv, from, n, to, turn, 0, 1, pass, bad, &s_abort));
        __syncthreads();
    }
    if (!ok) atomicOr(a.flags, FLAG_GAVE_UP);
    if (bad) atomicOr(a.flags, 16);
}

// a device's first launch of a kernel sets its attributes
template <typename F>
cudaError_t paged_once(std::atomic<unsigned long long> &devices, F set) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = device < 64 ? 1ULL << device : 0;
    if (devices & bit) return cudaSuccess;
    e = set();
    if (e == cudaSuccess) devices |= bit;
    return e;
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendArgs &a, cudaStream_t s) {
    if (a.B == 0 || a.T == 0) return cudaSuccess;
    // pages that T rows of B sequences reach: a sequence's first and last page beside those its rows fill
    const long long units = a.rows ? std::min(a.T, a.T / a.P + 2 * (long long)a.B) : a.B;
    if (units > INT32_MAX) return cudaErrorInvalidValue;
    const dim3 grid((unsigned)units, (unsigned)a.Hkv);
    // all of an SM's memory as shared memory, as the attention behind has it: an SM changes only while it is idle
    static std::atomic<unsigned long long> configured;
    const cudaError_t c = paged_once(configured, [] {
        const cudaError_t e = cudaFuncSetAttribute(paged_append_kernel<int64_t>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        return e != cudaSuccess ? e : cudaFuncSetAttribute(paged_append_kernel<int32_t>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    });
    if (c != cudaSuccess) return c;
    const cudaError_t e = a.narrow ? launch_behind(paged_append_kernel<int32_t>, grid, PA_THREADS, 0, s, a) : launch_behind(paged_append_kernel<int64_t>, grid, PA_THREADS, 0, s, a);
    note_launch();
    return e != cudaSuccess ? e : cudaGetLastError();
}

size_t paged_attn_bytes(const PagedAttnArgs &a) {
    if (paged_tc_ok(a)) return paged_tc_bytes(a);
    return (size_t)a.B * a.H * ((size_t)a.max_slots + 2 + a.hd) * 8;
}

cudaError_t launch_paged_attn(const PagedAttnArgs &a, cudaStream_t s) {
    if (paged_tc_ok(a)) return launch_paged_tc(a, s);
    const int rep = a.H / a.Hkv, pairs = a.Hkv * ((rep + PG_HEADS - 1) / PG_HEADS);
    const unsigned flat = (unsigned)std::min<long long>(1184, ((long long)a.B * a.H * a.hd + 255) / 256);
    const long long slots = a.max_slots;
    static std::atomic<unsigned long long> configured;
    cudaError_t e = paged_once(configured, [] {
        return cudaFuncSetAttribute(paged_general_scores_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PG_HEADS * PAGED_MAX_HEAD * 8);
    });
    if (e != cudaSuccess) return e;
    int launches = 0;
    auto behind = [&](auto kernel, dim3 grid, size_t smem) {       // (none behind one that failed)
        if (e != cudaSuccess) return;
        e = launch_behind(kernel, grid, 256, smem, s, a);
        launches += e == cudaSuccess;
    };
    behind(paged_general_init_kernel, flat, 0);
    // (with room for no key, too: it is the scores' kernel that flags lengths beyond their bound)
    behind(paged_general_scores_kernel, dim3((unsigned)std::max(1LL, (slots + PG_KEYS - 1) / PG_KEYS), pairs, a.B), (size_t)PG_HEADS * a.hd * 8);
    if (slots > 0) {
        behind(paged_general_exp_kernel, dim3((unsigned)((slots + 1023) / 1024), a.H, a.B), 0);
        behind(paged_general_values_kernel, dim3((unsigned)((slots + 127) / 128), pairs, a.B), 0);
    }
    behind(paged_general_out_kernel, flat, 0);
    note_launch(launches);
    return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t launch_paged_select(const PagedSelectArgs &a, cudaStream_t s) {
    const int rep = a.H / a.Hkv;
    const size_t rank = (size_t)rank_heads(rep) * a.hd * 12 + PS_THREADS / 32 * rank_stage(a.hd), fused = rank + (size_t)a.table_ld * 8;
    const bool staged = a.hd % 16 == 0 && (reinterpret_cast<uintptr_t>(a.bounds) & 15) == 0 && rank <= PR_SHARED;
    const int sms = paged_sms();
    if (sms <= 0) return cudaErrorInvalidDevice;
    const unsigned blocks = (unsigned)std::min<long long>(PR_CLUSTER, (a.table_ld + PR_TURN - 1) / PR_TURN);
    if (staged && fused <= PR_SHARED && a.table_ld <= PR_MOST && (a.table_ld <= 2 * PR_TURN || (long long)blocks * a.Hkv * a.B <= 2 * sms)) {
        static std::atomic<unsigned long long> configured;
        cudaError_t e = paged_once(configured, [] {
            const cudaError_t e = cudaFuncSetAttribute(paged_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PR_SHARED);
            return e != cudaSuccess ? e : cudaFuncSetAttribute(paged_select_kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        });
        if (e != cudaSuccess) return e;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(blocks, (unsigned)a.Hkv, (unsigned)a.B); cfg.blockDim = dim3(PS_THREADS); cfg.dynamicSmemBytes = fused; cfg.stream = s;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = blocks; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr; cfg.numAttrs = 2;
        e = cudaLaunchKernelEx(&cfg, paged_select_kernel, a);
        note_launch();
        return e != cudaSuccess ? e : cudaGetLastError();
    }
    static std::atomic<unsigned long long> configured;
    cudaError_t e = paged_once(configured, [] {
        cudaError_t e = cudaFuncSetAttribute(paged_rank_even_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PR_SHARED);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_rank_even_kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_rank_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_pick_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PK_HELD * 8);
        return e != cudaSuccess ? e : cudaFuncSetAttribute(paged_pick_kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    });
    if (e != cudaSuccess) return e;
    if (staged) {
        e = launch_behind(paged_rank_even_kernel, dim3(2 * sms), PS_THREADS, rank, s, a);
    } else e = launch_behind(paged_rank_kernel, dim3((unsigned)((a.table_ld + 31) / 32), a.Hkv, a.B), 256, (size_t)rep * a.hd * 8, s, a);
    if (e != cudaSuccess) return e;
    const bool held = a.table_ld <= PK_HELD;
    e = launch_behind(paged_pick_kernel, dim3(a.Hkv, a.B), PS_THREADS, held ? (size_t)a.table_ld * 8 : 0, s, a, held);
    note_launch(2);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace iie
