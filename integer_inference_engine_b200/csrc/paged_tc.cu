// Attention of one new token per sequence over a paged cache, both products on tcgen05 with the cache rows as they lie in memory.
//
// An int32 is its four bytes, so a row of keys is a row of 4 hd bytes, and with the query's balanced base-256 digits d_a (modulo 2^64)
//     q . k = sum_s 2^(8 s) sum_i sum_{b <= s} k_i,b d_{s-b}(q_i)          s = 0 .. 7, modulo 2^64:
// eight products of the raw bytes with eight columns per head that hold digit s - b beside byte b.  No key is unpacked: TMA puts rows into
// shared memory, 128 keys x 64 columns (8 heads) x 4 hd bytes is one MMA shape, and a query of any 64 bits needs nothing else.  The top byte
// of an int32 is signed and the others are not; an MMA takes its operand as one or the other, so that the tile is multiplied twice, by the
// columns of bytes 0 .. 2 and by those of byte 3.  Values likewise: bytes of the value rows, transposed by the operand descriptor (the sum runs
// over keys), times the three bytes of the probabilities floor(e 2^fa / Z) <= 2^fa; byte 3 of a value is read from the signed product,
// the others from the unsigned one.  Every sum stays below 2^31: 4 hd 255 128 for a score, 255^2 per key for an output (segments
// of at most 256 tiles of 128 keys).
//
// The softmax floors e and p, which takes the maximum and the normaliser of all keys in front of the values: three launches with the scores between
// them in memory, as 32-bit distances below the maximum of 32 keys and eight heads (a distance beyond `clip` has no weight, so nothing
// is lost).  Tiles of all sequences and KV heads form one list that the CTAs share evenly, whatever the lengths: a tile is sixteen
// groups of eight rows, a group lies in one page.  A pair whose tiles fall to several CTAs adds its output sums up in memory (integers: in any order).
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "paged.h"
#include "softmax.cuh"
#include "tile_ops.cuh"

namespace iie {

namespace {

constexpr int PT_KEYS = 128, PT_GROUPS = 16;       // keys of a tile, groups of eight
constexpr int PT_HEADS = 8;                        // query heads of a pair: a (sequence, KV head, up to eight heads)
constexpr int PT_WORKERS = 8;                      // warps that read TMEM out and write operands
constexpr int PT_THREADS = 64 + 32 * PT_WORKERS;
constexpr int PT_META = 8;                         // tiles whose group masks are kept
constexpr int PT_MAX_STAGES = 6;
constexpr int PT_MAX_SEGMENT = 256;                // tiles that one accumulation takes: 256 * 128 * 255^2 < 2^31

struct TcWork {
    uint32_t *dist;                // [tiles][128][8] distances below the base
    long long *base;               // [tiles][4][8] largest score of 32 keys
    long long *top;                // [pairs][8]
    unsigned long long *z;         // [pairs][8]
    unsigned long long *acc;       // [pairs][8][hd]
    unsigned *done;                // [pairs] tiles whose sums are in acc, counted by every warp
};
__host__ __device__ inline int tc_head_groups(const PagedAttnArgs &a) { return (a.H / a.Hkv + PT_HEADS - 1) / PT_HEADS; }
__host__ __device__ inline int tc_group_heads(const PagedAttnArgs &a) { const int g = tc_head_groups(a); return (a.H / a.Hkv + g - 1) / g; }
// tiles of a pair at most
__host__ __device__ inline long long tc_tiles_most(const PagedAttnArgs &a) {
    if (a.n_sel > 0) return ((long long)a.n_sel * a.P + PT_KEYS - 1) / PT_KEYS;
    return (a.max_slots / 8 + 2 + PT_GROUPS - 1) / PT_GROUPS;
}
__host__ __device__ inline TcWork tc_work(const PagedAttnArgs &a, size_t *bytes = nullptr) {
    const long long pairs = (long long)a.B * a.Hkv * tc_head_groups(a), tiles = pairs * tc_tiles_most(a);
    TcWork w;
    w.dist = static_cast<uint32_t *>(a.work);
    w.base = reinterpret_cast<long long *>(w.dist + tiles * PT_KEYS * PT_HEADS);
    w.top = w.base + tiles * 4 * PT_HEADS;
    w.z = reinterpret_cast<unsigned long long *>(w.top + pairs * PT_HEADS);
    w.acc = w.z + pairs * PT_HEADS;
    w.done = reinterpret_cast<unsigned *>(w.acc + pairs * PT_HEADS * a.hd);
    if (bytes) *bytes = (size_t)tiles * (PT_KEYS * PT_HEADS * 4 + 4 * PT_HEADS * 8) + (size_t)pairs * (PT_HEADS * 16 + (size_t)PT_HEADS * a.hd * 8 + 4);
    return w;
}

__device__ __forceinline__ int tc_tiles(const PagedAttnArgs &a, const PagedSpan &s) {
    if (s.len == 0) return 0;
    if (a.sel) return (int)tc_tiles_most(a);
    return (((s.len + 7) >> 3) - (s.lo >> 3) + PT_GROUPS - 1) / PT_GROUPS;
}

// One role's walk over the CTA's share of the list: tiles of sequence b, pair by pair.
struct TcWalk {
    int b, pair_of, t, nt, left, tile, seg;        // pair of the sequence, tile of the pair, its tiles, tiles left, number in the list, tiles of the segment so far
    PagedSpan s;
    __device__ __forceinline__ void load(const PagedAttnArgs &a) { paged_span(a, b, s); nt = tc_tiles(a, s); }
    __device__ __forceinline__ void next(const PagedAttnArgs &a, int per_seq) {
        seg = ends_segment() ? 0 : seg + 1;
        left--; tile++;
        if (++t < nt || left == 0) return;
        t = 0;
        if (++pair_of < per_seq) return;
        pair_of = 0;
        do {                                       // (tiles are left: there is a sequence that has some)
            if (++b >= a.B) { left = 0; return; }
            load(a);
        } while (nt == 0);
    }
    __device__ __forceinline__ bool ends_segment() const { return t + 1 == nt || left == 1 || seg + 1 == PT_MAX_SEGMENT; }
};

// The whole CTA: its share [first, first + left) of the list and the place where it begins.  scan: 33 ints of shared memory.
__device__ __forceinline__ void tc_share(const PagedAttnArgs &a, int *scan, TcWalk &w, bool flag) {
    const int tid = threadIdx.x, n = blockDim.x, lane = tid & 31, warp = tid >> 5, per_seq = a.Hkv * tc_head_groups(a), warps = n >> 5;
    auto count = [&](int b) {
        PagedSpan s;
        if (b >= a.B) return 0;
        if (!paged_span(a, b, s) && flag) atomicOr(a.flags, 16);
        return tc_tiles(a, s);
    };
    const int own = count(tid);
    int mine = own;
    for (int b = tid + n; b < a.B; b += n) mine += count(b);
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) scan[warp] = mine;
    __syncthreads();
    int all = 0;
    for (int i = 0; i < warps; i++) all += scan[i];
    __syncthreads();
    const long long total = (long long)all * per_seq;
    const int from = (int)(total * blockIdx.x / gridDim.x);
    w.left = (int)(total * (blockIdx.x + 1) / gridDim.x) - from;
    w.tile = from; w.seg = 0;
    if (tid == 0) scan[32] = -1;
    int before = 0;                                // tiles per pair of the sequences in front
    for (int b0 = 0; b0 < a.B; b0 += n) {
        const int c = b0 == 0 ? own : count(b0 + tid);
        int upto = c;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const int o = __shfl_up_sync(0xffffffffu, upto, d); if (lane >= d) upto += o; }
        if (lane == 31) scan[warp] = upto;
        __syncthreads();
        int sum = 0;
        for (int i = 0; i < warps; i++) { if (i < warp) upto += scan[i]; sum += scan[i]; }
        const long long lo = (long long)(before + upto - c) * per_seq;
        if (c > 0 && from >= lo && from < lo + (long long)c * per_seq) { scan[32] = b0 + tid; scan[31] = (int)(from - lo); }
        before += sum;
        __syncthreads();
        if (scan[32] >= 0) break;
        __syncthreads();
    }
    w.b = scan[32] < 0 ? 0 : scan[32];
    w.load(a);
    const int at = scan[31];
    w.pair_of = w.nt > 0 ? at / w.nt : 0;
    w.t = w.nt > 0 ? at - w.pair_of * w.nt : 0;
    if (scan[32] < 0) w.left = 0;
}

// Producer's lane l < 16: rows of group l of the walk's tile that count, as a byte; the row of the pool where it lies.
__device__ __forceinline__ uint32_t tc_group(const PagedAttnArgs &a, const TcWalk &w, int kv, int l, int &row) {
    int logical, r, pos;
    if (a.sel) {
        const unsigned slot = ((unsigned)w.t * PT_GROUPS + l) * 8, i = slot / (unsigned)a.P;
        if (i >= (unsigned)a.n_sel) return 0;
        r = (int)(slot - i * a.P);
        logical = a.sel[((long long)w.b * a.Hkv + kv) * a.n_sel + i];
        if (logical < 0) return 0;
        if (logical >= a.table_ld) { atomicOr(a.flags, 16); return 0; }
        pos = logical * a.P + r;                   // (a table's rows are numbered in 31 bits)
    } else {
        pos = ((w.s.lo >> 3) + w.t * PT_GROUPS + l) * 8;
        logical = (int)((unsigned)pos / (unsigned)a.P);
        r = pos - logical * a.P;
    }
    const int from = max(w.s.lo - pos, 0), to = min(w.s.len - pos, 8);
    if (from >= to) return 0;
    const int page = a.table[(long long)w.b * a.table_ld + logical];
    if (page < 0 || page >= a.n_pages) { atomicOr(a.flags, 16); return 0; }
    row = (page * a.Hkv + kv) * a.P + r;
    return ((1u << to) - 1) & ~((1u << from) - 1);
}

__device__ __forceinline__ uint64_t tc_desc(uint32_t addr, uint32_t stride, uint32_t swizzle) {      // stride between groups of eight rows
    return (uint64_t)((addr >> 4) & 0x3FFF) | (1ULL << 16) | ((uint64_t)(stride >> 4) << 32) | (1ULL << 46) | ((uint64_t)swizzle << 61);
}
constexpr uint32_t SW128 = 2, SW32 = 6;
template <int N>
__device__ __forceinline__ void tc_ld(uint32_t addr, int (&r)[N]) {
    static_assert(N == 8 || N == 32, "");
    if constexpr (N == 8)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(addr));
    else
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                       "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
                       "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                     : "r"(addr));
}
__device__ __forceinline__ void tc_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

struct TcShape { int chunks, stages, columns; };   // 128-byte chunks of a row, tiles in flight, TMEM columns

// what both product kernels keep in shared memory beside tiles and operands
struct TcBars {
    uint64_t full[PT_MAX_STAGES], empty[PT_MAX_STAGES], meta[PT_META];
    uint64_t acc_full[2], acc_free[2], op_full[2], op_free[2], drain;
    uint32_t tmem;
    int abort, scan[33];
    unsigned char mask[PT_META][PT_GROUPS];
};

// The producer warp: tiles of the list into the ring, sixteen boxes of eight rows each.
__device__ __forceinline__ void tc_produce(const PagedAttnArgs &a, TcWalk w, const CUtensorMap *map, TcBars &s, uint32_t ring, TcShape sh, volatile int *abort_flag) {
    const int lane = threadIdx.x & 31, per_seq = a.Hkv * tc_head_groups(a), groups = tc_head_groups(a);
    const uint32_t group_bytes = (uint32_t)sh.chunks * 1024, tile_bytes = group_bytes * PT_GROUPS;
    int slot = 0, issued = 0;
    uint32_t pass = 0;
    for (; w.left > 0; issued++) {
        int row = 0;
        const uint32_t rows = lane < PT_GROUPS ? tc_group(a, w, w.pair_of / groups, lane, row) : 0;
        if (issued >= sh.stages && !tl_wait(tl_u32(&s.empty[slot]), pass ^ 1, abort_flag)) break;
        if (lane < PT_GROUPS) s.mask[issued % PT_META][lane] = (unsigned char)rows;
        const uint32_t some = __ballot_sync(0xffffffffu, rows != 0);
        if (lane == 0) { tl_arrive(tl_u32(&s.meta[issued % PT_META])); tl_expect(tl_u32(&s.full[slot]), (uint32_t)__popc(some) * group_bytes); }
        __syncwarp();
        if (rows) tl_tma(ring + slot * tile_bytes + lane * group_bytes, map, 0, row, 0, tl_u32(&s.full[slot]));
        w.next(a, per_seq);
        if (++slot == sh.stages) { slot = 0; pass ^= 1; }
    }
    if (*abort_flag) {                             // copies under way end before the CTA does
        __syncwarp();
        for (int k = max(0, issued - sh.stages); k < issued; k++) {
            volatile int patient = 0;
            tl_wait(tl_u32(&s.full[k % sh.stages]), (uint32_t)(k / sh.stages) & 1, &patient);
        }
    }
}

__device__ __forceinline__ void tc_begin(TcBars &s, int columns, int writers) {      // writers: warps that write an operand
    const int tid = threadIdx.x;
    if (tid == 0) {
        s.abort = 0;
        for (int i = 0; i < PT_MAX_STAGES; i++) { tl_init(tl_u32(&s.full[i]), 1); tl_init(tl_u32(&s.empty[i]), 1); }
        for (int i = 0; i < PT_META; i++) tl_init(tl_u32(&s.meta[i]), 1);
        for (int i = 0; i < 2; i++) {
            tl_init(tl_u32(&s.acc_full[i]), 1); tl_init(tl_u32(&s.acc_free[i]), PT_WORKERS);
            tl_init(tl_u32(&s.op_full[i]), writers); tl_init(tl_u32(&s.op_free[i]), 1);
        }
        tl_init(tl_u32(&s.drain), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid >> 5 == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tl_u32(&s.tmem)), "r"(columns));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_before();
    __syncthreads();
    tc_after();
}
// The issuing warp, where a wait gave up: products under way end before their TMEM is given back.
__device__ __forceinline__ void tc_drain(TcBars &s) {
    if (!*(volatile int *)&s.abort) return;
    if (tl_elect()) tl_commit(tl_u32(&s.drain));
    __syncwarp();
    volatile int patient = 0;
    tl_wait(tl_u32(&s.drain), 0, &patient);
}
__device__ __forceinline__ void tc_end(TcBars &s, int columns, int *flags) {
    tc_before();
    __syncthreads();
    if (threadIdx.x >> 5 == 1) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s.tmem), "r"(columns));
    }
    if (threadIdx.x == 0 && s.abort) atomicOr(flags, FLAG_GAVE_UP);
}

// Query columns of one pair: column 8 h + s holds digit s - b of q_i at byte 4 i + b, bytes 0 .. 2 in one operand and byte 3 in the other.
// A thread takes four dimensions of a head.
__device__ __forceinline__ void tc_queries(const PagedAttnArgs &a, const TcWalk &w, int heads, int padded, unsigned char *lower, unsigned char *upper, int worker) {
    const int groups = tc_head_groups(a), kv = w.pair_of / groups, h0 = kv * (a.H / a.Hkv) + (w.pair_of % groups) * tc_group_heads(a), quads = a.hd / 4, half = a.hd / 2;
    const long long pos = w.s.len - 1;
    for (int task = worker; task < padded * quads; task += 32 * PT_WORKERS) {
        const int h = task / quads, j = task - h * quads, d = 4 * j;
        int64_t y[4] = {0, 0, 0, 0};
        if (h < heads) {
            const int64_t *q = a.q + (long long)w.b * a.q_ld + (long long)(h0 + h) * a.hd;
            if (a.rope == 2) {
                const bool second = d >= half;
                const int i = second ? d - half : d;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    int64_t x0 = q[i + e], x1 = q[i + e + half];
                    paged_rotate(a.cos, a.sin, 2, a.hd, a.fa, pos, i + e, x0, x1);
                    y[e] = second ? x1 : x0;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = q[d + e];
                paged_rotate(a.cos, a.sin, a.rope, a.hd, a.fa, pos, 2 * j, y[0], y[1]);
                paged_rotate(a.cos, a.sin, a.rope, a.hd, a.fa, pos, 2 * j + 1, y[2], y[3]);
            }
        }
        uint32_t hi[4], lo[4];                     // digits, first one on top
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint64_t digits = ((uint64_t)y[e] + 0x8080808080808080ULL) ^ 0x8080808080808080ULL;
            hi[e] = __byte_perm((uint32_t)digits, 0, 0x0123); lo[e] = __byte_perm((uint32_t)(digits >> 32), 0, 0x0123);
        }
        const uint32_t at = (uint32_t)(j >> 3) * (uint32_t)padded * 1024;
#pragma unroll
        for (int s = 0; s < 8; s++) {
            uint32_t x[4];
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = s < 4 ? hi[e] >> (24 - 8 * s) : (s == 7 ? lo[e] : __funnelshift_r(lo[e], hi[e], 56 - 8 * s));
            const uint32_t to = at + (uint32_t)(8 * h + s) * 128 + (uint32_t)(((j & 7) ^ s) * 16);
            *reinterpret_cast<uint4 *>(lower + to) = make_uint4(x[0] & 0xFFFFFFu, x[1] & 0xFFFFFFu, x[2] & 0xFFFFFFu, x[3] & 0xFFFFFFu);
            *reinterpret_cast<uint4 *>(upper + to) = make_uint4(x[0] & 0xFF000000u, x[1] & 0xFF000000u, x[2] & 0xFF000000u, x[3] & 0xFF000000u);
        }
    }
}

// ---- scores ---------------------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(PT_THREADS, 1) paged_scores_kernel(const PagedAttnArgs a, const __grid_constant__ CUtensorMap map, const TcShape sh) {
    extern __shared__ unsigned char pt_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(pt_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) TcBars s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, per_seq = a.Hkv * tc_head_groups(a);
    const int heads_most = tc_group_heads(a), padded = (heads_most + 1) & ~1;
    const uint32_t operand = (uint32_t)sh.chunks * padded * 1024, tile_bytes = (uint32_t)sh.chunks * 1024 * PT_GROUPS;
    unsigned char *lower = smem, *upper = smem + operand;
    const uint32_t ring = tl_u32(smem) + 2 * operand;
    volatile int *abort_flag = &s.abort;
    tc_begin(s, sh.columns, PT_WORKERS);
    pdl_enter();
    const TcWork work = tc_work(a);
    {                                              // what the kernels behind add to
        const long long pairs = (long long)a.B * per_seq, n = pairs * PT_HEADS * a.hd;
        for (long long i = (long long)blockIdx.x * PT_THREADS + tid; i < n; i += (long long)gridDim.x * PT_THREADS) {
            work.acc[i] = 0;
            if (i < pairs) work.done[i] = 0;
            if (i < pairs * PT_HEADS) work.z[i] = 0;
        }
    }
    TcWalk w;
    tc_share(a, s.scan, w, blockIdx.x == 0);
    const uint32_t tmem = s.tmem;
    if (warp == 0) tc_produce(a, w, &map, s, ring, sh, abort_flag);
    else if (warp == 1) {
        const uint32_t n = (uint32_t)padded * 8;
        int slot = 0, queries = 0;
        uint32_t pass = 0;
        bool fresh = true;
        for (int i = 0; w.left > 0; i++) {
            bool ok = tl_wait(tl_u32(&s.full[slot]), pass, abort_flag);
            if (ok && i >= 2) ok = tl_wait(tl_u32(&s.acc_free[i & 1]), ((i >> 1) & 1) ^ 1, abort_flag);
            if (ok && fresh) { ok = tl_wait(tl_u32(&s.op_full[0]), queries & 1, abort_flag); queries++; }
            if (!ok) break;
            tc_after();
            if (tl_elect()) {
                const uint32_t tile = ring + slot * tile_bytes;
#pragma unroll 1
                for (int side = 0; side < 2; side++) {
                    const uint32_t b = tl_u32(side ? upper : lower);
#pragma unroll 1
                    for (int c = 0; c < sh.chunks; c++)
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            tl_mma(tmem + (i & 1) * 64, tc_desc(tile + c * 1024 + k * 32, (uint32_t)sh.chunks * 1024, SW128),
                                   tc_desc(b + (uint32_t)c * padded * 1024 + k * 32, 1024, SW128), tl_idesc((int)n, side == 1), (side | c | k) != 0);
                }
                tl_commit(tl_u32(&s.empty[slot]));
                tl_commit(tl_u32(&s.acc_full[i & 1]));
            }
            __syncwarp();
            fresh = w.t + 1 == w.nt;
            w.next(a, per_seq);
            if (++slot == sh.stages) { slot = 0; pass ^= 1; }
        }
        tc_drain(s);
    } else {
        const int worker = tid - 64, half = (warp - 2) >> 2, quarter = warp & 3, key = quarter * 32 + lane;      // a warp reads TMEM lanes 32 (warp % 4) ..
        const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + half * 32;
        const bool serves = 4 * half < heads_most;
        bool fresh = true;
        for (int i = 0; w.left > 0; i++) {
            if (fresh) {                           // (the last tile of the pair in front has been multiplied: its sums were waited for)
                const int g = w.pair_of % tc_head_groups(a);
                tc_queries(a, w, min(heads_most, a.H / a.Hkv - g * heads_most), padded, lower, upper, worker);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) tl_arrive(tl_u32(&s.op_full[0]));
            }
            if (!tl_wait(tl_u32(&s.meta[i % PT_META]), (uint32_t)(i / PT_META) & 1, abort_flag)) break;
            const bool seen = (s.mask[i % PT_META][key >> 3] >> (key & 7)) & 1;
            if (!tl_wait(tl_u32(&s.acc_full[i & 1]), (i >> 1) & 1, abort_flag)) break;
            tc_after();
            int r[32];
            if (serves) { tc_ld(from + (i & 1) * 64, r); tc_ld_wait(); }
            tc_before();
            __syncwarp();
            if (lane == 0) tl_arrive(tl_u32(&s.acc_free[i & 1]));
            if (serves) {
                uint32_t d[4];
                long long base = INT64_MIN;
#pragma unroll
                for (int h = 0; h < 4; h++) {
                    const int *c = r + 8 * h;
                    const uint64_t low = (uint64_t)((long long)c[0] + (long long)c[1] * 256 + (long long)c[2] * 65536 + (long long)c[3] * 16777216);
                    const uint32_t high = (uint32_t)c[4] + ((uint32_t)c[5] << 8) + ((uint32_t)c[6] << 16) + ((uint32_t)c[7] << 24);
                    const long long dot = (long long)(low + ((uint64_t)high << 32));
                    const long long score = (long long)((uint64_t)(dot >> a.fa) * (uint64_t)a.inv_sqrt) >> a.fa;
                    // the largest of the warp's 32 keys: by the upper words, then by the lower ones where those are equal
                    const int up = seen ? (int)(score >> 32) : INT32_MIN;
                    const int up_most = __reduce_max_sync(0xffffffffu, up);
                    const uint32_t low_most = __reduce_max_sync(0xffffffffu, seen && up == up_most ? (uint32_t)score : 0u);
                    const long long most = (long long)(((uint64_t)(uint32_t)up_most << 32) | low_most);
                    d[h] = seen ? (uint32_t)min((uint64_t)most - (uint64_t)score, (uint64_t)0xFFFFFFFEu) : 0xFFFFFFFFu;
                    if (lane == h) base = most;
                }
                *reinterpret_cast<uint4 *>(work.dist + ((long long)w.tile * PT_KEYS + key) * PT_HEADS + 4 * half) = make_uint4(d[0], d[1], d[2], d[3]);
                const bool any = __any_sync(0xffffffffu, seen);
                if (lane < 4) work.base[((long long)w.tile * 4 + quarter) * PT_HEADS + 4 * half + lane] = any ? base : INT64_MIN;
            }
            fresh = w.t + 1 == w.nt;
            w.next(a, per_seq);
        }
    }
    tc_end(s, sh.columns, a.flags);
}

// ---- normalisers: the largest score of a pair, the sum of its exponentials -------------------------------------------------------------
constexpr int PN_THREADS = 256;

template <bool SHORT>
__global__ void __launch_bounds__(PN_THREADS) paged_norm_kernel(const PagedAttnArgs a) {
    using Exp = std::conditional_t<SHORT, SoftmaxExp16, SoftmaxExp>;
    __shared__ int scan[33];
    __shared__ long long s_most[PN_THREADS / 32][PT_HEADS];
    __shared__ unsigned long long s_z[PT_HEADS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, per_seq = a.Hkv * tc_head_groups(a);
    pdl_enter();
    TcWalk w;
    tc_share(a, scan, w, false);
    const TcWork work = tc_work(a);
    const Exp exp2(a.fa, a.log2e, a.clip);
    const int half = tid & 1, key = tid >> 1, quarter = key >> 5, heads = tc_group_heads(a);
    while (w.left > 0) {
        const long long pair = (long long)w.b * per_seq + w.pair_of;
        const int count = min(w.nt - w.t, w.left), first = w.tile - w.t;       // tiles of the pair here; its first one
        long long most = INT64_MIN;
        for (int i = tid >> 3; i < w.nt * 4; i += PN_THREADS / 8) most = max(most, work.base[((long long)first * 4 + i) * PT_HEADS + (tid & 7)]);
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 8));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 16));
        if (lane < 8) s_most[warp][lane] = most;
        if (tid < PT_HEADS) s_z[tid] = 0;
        __syncthreads();
        long long top[4];
#pragma unroll
        for (int h = 0; h < 4; h++) {
            top[h] = INT64_MIN;
            for (int v = 0; v < PN_THREADS / 32; v++) top[h] = max(top[h], s_most[v][4 * half + h]);
        }
        if (w.t == 0 && tid < 2)
            for (int h = 0; h < 4; h++) work.top[pair * PT_HEADS + 4 * half + h] = top[h];
        unsigned long long z[4] = {0, 0, 0, 0};
        if (4 * half < heads)
            for (int i = 0; i < count; i++) {
                const uint4 d4 = *reinterpret_cast<const uint4 *>(work.dist + ((long long)(w.tile + i) * PT_KEYS + key) * PT_HEADS + 4 * half);
                const uint32_t d[4] = {d4.x, d4.y, d4.z, d4.w};
                const long long *base = work.base + ((long long)(w.tile + i) * 4 + quarter) * PT_HEADS + 4 * half;
#pragma unroll
                for (int h = 0; h < 4; h++) {
                    if (d[h] == 0xFFFFFFFFu) continue;                     // no key
                    const uint64_t below = min((uint64_t)top[h] - (uint64_t)base[h], (uint64_t)a.clip) + d[h];
                    z[h] += (unsigned)exp2((uint32_t)min(below, (uint64_t)a.clip));
                }
            }
#pragma unroll
        for (int h = 0; h < 4; h++) {
#pragma unroll
            for (int m = 2; m < 32; m <<= 1) z[h] += __shfl_xor_sync(0xffffffffu, z[h], m);
            if (lane < 2 && z[h]) atomicAdd(&s_z[4 * half + h], z[h]);
        }
        __syncthreads();
        if (tid < heads && s_z[tid]) atomicAdd(work.z + pair * PT_HEADS + tid, s_z[tid]);
        w.left -= count; w.tile += count; w.t += count;
        if (w.left > 0) {                          // (the pair is through)
            w.t = 0;
            if (++w.pair_of == per_seq) {
                w.pair_of = 0;
                do {
                    if (++w.b >= a.B) { w.left = 0; break; }
                    w.load(a);
                } while (w.nt == 0);
            }
        }
        __syncthreads();
    }
}

// ---- probabilities and values --------------------------------------------------------------------------------------------------------
template <bool SHORT, bool SMALL>                  // SHORT: fa <= 16; SMALL: beside that every sum of exponentials at most 2^31
__global__ void __launch_bounds__(PT_THREADS, 1) paged_values_kernel(const PagedAttnArgs a, const __grid_constant__ CUtensorMap map, const TcShape sh) {
    using Exp = std::conditional_t<SHORT, SoftmaxExp16, SoftmaxExp>;
    using Quotient = std::conditional_t<SMALL, SoftmaxQuotient16, SoftmaxQuotient>;
    extern __shared__ unsigned char pt_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(pt_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) TcBars s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, groups = tc_head_groups(a), per_seq = a.Hkv * groups;
    const int heads_most = tc_group_heads(a);
    const uint32_t tile_bytes = (uint32_t)sh.chunks * 1024 * PT_GROUPS;
    unsigned char *probs = smem;                   // two tiles of probability bytes [128][32], 32-byte swizzle: byte a of head h at 8 a + h
    const uint32_t ring = tl_u32(smem) + 2 * PT_KEYS * 32;
    volatile int *abort_flag = &s.abort;
    tc_begin(s, sh.columns, PT_WORKERS / 2);
    TcWalk w;
    tc_share(a, s.scan, w, false);                 // (lengths, tables and pages are older than the kernel in front, which waited for what wrote them)
    const uint32_t tmem = s.tmem, buffer = (uint32_t)sh.chunks * 64;
    if (warp == 0) {
        tc_produce(a, w, &map, s, ring, sh, abort_flag);
    } else if (warp == 1) {
        const uint32_t idesc = (2u << 4) | (1u << 15) | (1u << 16) | ((32u >> 3) << 17) | ((128u >> 4) << 24);      // both operands transposed, unsigned
        int slot = 0, seg = 0;
        uint32_t pass = 0;
        for (int i = 0; w.left > 0; i++) {
            bool ok = tl_wait(tl_u32(&s.full[slot]), pass, abort_flag);
            if (ok) ok = tl_wait(tl_u32(&s.op_full[i & 1]), (i >> 1) & 1, abort_flag);
            if (ok && w.seg == 0 && seg >= 2) ok = tl_wait(tl_u32(&s.acc_free[seg & 1]), ((seg >> 1) & 1) ^ 1, abort_flag);
            if (!ok) break;
            tc_after();
            const bool last = w.ends_segment();
            if (tl_elect()) {
                const uint32_t tile = ring + slot * tile_bytes, p = tl_u32(probs) + (i & 1) * (PT_KEYS * 32);
#pragma unroll 1
                for (int c = 0; c < sh.chunks; c++)
#pragma unroll
                    for (int side = 0; side < 2; side++)
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            tl_mma(tmem + (seg & 1) * buffer + (2 * c + side) * 32, tc_desc(tile + c * 1024 + k * 4 * sh.chunks * 1024, (uint32_t)sh.chunks * 1024, SW128),
                                   tc_desc(p + k * 1024, 256, SW32), idesc | (side ? 1u << 7 : 0u), (w.seg | k) != 0);
                tl_commit(tl_u32(&s.empty[slot]));
                tl_commit(tl_u32(&s.op_free[i & 1]));
                if (last) tl_commit(tl_u32(&s.acc_full[seg & 1]));
            }
            __syncwarp();
            if (last) seg++;
            w.next(a, per_seq);
            if (++slot == sh.stages) { slot = 0; pass ^= 1; }
        }
        tc_drain(s);
    } else {
        pdl_enter();
        const TcWork work = tc_work(a);
        const int worker = tid - 64, set = (warp - 2) >> 2, quarter = warp & 3, key = quarter * 32 + lane;
        for (int b = blockIdx.x; b < a.B; b += gridDim.x) {                // sequences without keys
            PagedSpan none;
            paged_span(a, b, none);
            if (tc_tiles(a, none) == 0)
                for (long long i = worker; i < (long long)a.H * a.hd; i += 32 * PT_WORKERS) a.out[(long long)b * a.H * a.hd + i] = 0;
        }
        const Exp exp2(a.fa, a.log2e, a.clip);
        Quotient quotient[PT_HEADS] = {Quotient(0, a.fa), Quotient(0, a.fa), Quotient(0, a.fa), Quotient(0, a.fa), Quotient(0, a.fa), Quotient(0, a.fa), Quotient(0, a.fa), Quotient(0, a.fa)};
        long long top = 0;                         // of head lane & 7
        int seg = 0;
        bool fresh = true;
        for (int i = 0; w.left > 0; i++) {
            const long long pair = (long long)w.b * per_seq + w.pair_of;
            if (fresh) {
                top = work.top[pair * PT_HEADS + (lane & 7)];
                const Quotient mine((lane & 7) < heads_most ? work.z[pair * PT_HEADS + (lane & 7)] : 0, a.fa);
#pragma unroll
                for (int h = 0; h < PT_HEADS; h++) {
                    quotient[h] = mine;
                    if constexpr (SMALL) quotient[h].m = __shfl_sync(0xffffffffu, mine.m, h);
                    else { quotient[h].mh = __shfl_sync(0xffffffffu, mine.mh, h); quotient[h].ml = __shfl_sync(0xffffffffu, mine.ml, h); }
                    quotient[h].post = __shfl_sync(0xffffffffu, mine.post, h);
                }
            }
            if ((i & 1) == set) {
                const uint4 *d4 = reinterpret_cast<const uint4 *>(work.dist + ((long long)w.tile * PT_KEYS + key) * PT_HEADS);
                const uint4 da = d4[0], db = heads_most > 4 ? d4[1] : make_uint4(0, 0, 0, 0);
                const uint32_t d[PT_HEADS] = {da.x, da.y, da.z, da.w, db.x, db.y, db.z, db.w};
                const long long base = work.base[((long long)w.tile * 4 + quarter) * PT_HEADS + (lane & 7)];
                const uint32_t above = (uint32_t)min((uint64_t)top - (uint64_t)base, (uint64_t)a.clip);
                uint32_t p[PT_HEADS];
#pragma unroll
                for (int h = 0; h < PT_HEADS; h++) {
                    const uint64_t below = (uint64_t)__shfl_sync(0xffffffffu, above, h) + d[h];
                    const uint32_t e = h < heads_most && d[h] != 0xFFFFFFFFu ? (uint32_t)exp2((uint32_t)min(below, (uint64_t)a.clip)) : 0u;
                    p[h] = quotient[h](e);
                }
                if (i >= 2 && !tl_wait(tl_u32(&s.op_free[set]), ((i >> 1) & 1) ^ 1, abort_flag)) break;
                uint32_t out[8];                                           // bytes 8 a + h
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    const uint32_t x = p[4 * q], y = p[4 * q + 1], z = p[4 * q + 2], v = p[4 * q + 3];
                    const uint32_t t0 = __byte_perm(x, y, 0x5140), t1 = __byte_perm(x, y, 0x7362), t2 = __byte_perm(z, v, 0x5140), t3 = __byte_perm(z, v, 0x7362);
                    out[q] = __byte_perm(t0, t2, 0x5410); out[2 + q] = __byte_perm(t0, t2, 0x7632); out[4 + q] = __byte_perm(t1, t3, 0x5410);
                }
                unsigned char *to = probs + set * (PT_KEYS * 32) + key * 32;
                const int flip = ((key >> 2) & 1) * 16;
                *reinterpret_cast<uint4 *>(to + flip) = make_uint4(out[0], out[1], out[2], out[3]);
                *reinterpret_cast<uint4 *>(to + (16 ^ flip)) = make_uint4(out[4], out[5], 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) tl_arrive(tl_u32(&s.op_full[set]));
            }
            if (w.ends_segment()) {
                if (!tl_wait(tl_u32(&s.acc_full[seg & 1]), (seg >> 1) & 1, abort_flag)) break;
                tc_after();
                const bool whole = w.seg + 1 == w.nt;                      // the pair's only segment
                const int g = w.pair_of % groups, kv = w.pair_of / groups, heads = min(heads_most, a.H / a.Hkv - g * heads_most), byte = lane & 3;
                int64_t *out = a.out + ((long long)w.b * a.H + kv * (a.H / a.Hkv) + g * heads_most) * a.hd;
                unsigned long long *acc = work.acc + pair * PT_HEADS * a.hd;
                for (int c = set; c < sh.chunks; c += 2) {
                    const uint32_t from = tmem + (seg & 1) * buffer + ((uint32_t)(quarter * 32) << 16) + 2 * c * 32;
                    uint64_t sum[PT_HEADS];
#pragma unroll
                    for (int h = 0; h < PT_HEADS; h++) sum[h] = 0;
#pragma unroll
                    for (int part = 0; part < 3; part++) {
                        int u[8], v[8];
                        tc_ld(from + 8 * part, u); tc_ld(from + 32 + 8 * part, v);
                        tc_ld_wait();
#pragma unroll
                        for (int h = 0; h < PT_HEADS; h++) sum[h] += (uint64_t)(int64_t)(byte == 3 ? v[h] : u[h]) << (8 * part);
                    }
                    // four lanes hold a dimension's four bytes: two exchanges leave lane `byte` with heads 2 byte', 2 byte' + 1
#pragma unroll
                    for (int h = 0; h < PT_HEADS; h++) sum[h] <<= 8 * byte;
                    const bool upper = byte & 2, odd = byte & 1;
#pragma unroll
                    for (int h = 0; h < 4; h++) {
                        const uint64_t give = upper ? sum[h] : sum[h + 4];
                        sum[h] = (upper ? sum[h + 4] : sum[h]) + __shfl_xor_sync(0xffffffffu, give, 2);
                    }
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint64_t give = odd ? sum[h] : sum[h + 2];
                        sum[h] = (odd ? sum[h + 2] : sum[h]) + __shfl_xor_sync(0xffffffffu, give, 1);
                    }
                    const int d = 32 * c + 8 * quarter + (lane >> 2), h0 = 4 * (byte >> 1) + 2 * (byte & 1);
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        if (h0 + h < heads) {
                            if (whole) out[(long long)(h0 + h) * a.hd + d] = (int64_t)sum[h] >> a.fa;
                            else atomicAdd(acc + (h0 + h) * a.hd + d, (unsigned long long)sum[h]);
                        }
                }
                tc_before();
                __syncwarp();
                if (lane == 0) tl_arrive(tl_u32(&s.acc_free[seg & 1]));
                if (!whole) {                      // the warp that adds the pair's last sums writes it out
                    __threadfence();
                    __syncwarp();
                    const unsigned n = (unsigned)w.seg + 1;
                    unsigned before = 0;
                    if (lane == 0) before = atomicAdd(work.done + pair, n);
                    before = __shfl_sync(0xffffffffu, before, 0);
                    if (before + n == (unsigned)w.nt * PT_WORKERS) {
                        __threadfence();
                        for (int at = lane; at < heads * a.hd; at += 32) out[at] = (int64_t)__ldcg(acc + at) >> a.fa;
                    }
                }
                seg++;
            }
            fresh = w.t + 1 == w.nt;
            w.next(a, per_seq);
        }
    }
    tc_end(s, sh.columns, a.flags);
}

bool tc_map(CUtensorMap *map, const int32_t *pool, const PagedAttnArgs &a) {
    const cuuint64_t dims[3] = {32, (cuuint64_t)a.n_pages * a.Hkv * a.P, (cuuint64_t)a.hd / 32}, strides[2] = {(cuuint64_t)a.hd * 4, 128};
    const cuuint32_t box[3] = {32, 8, (cuuint32_t)a.hd / 32}, step[3] = {1, 1, 1};
    return tl_encode()(map, CU_TENSOR_MAP_DATA_TYPE_INT32, 3, const_cast<int32_t *>(pool), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename K>
cudaError_t tc_configure(K kernel, size_t smem) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
}

template <bool SHORT, bool SMALL>
cudaError_t launch_tc(const PagedAttnArgs &a, cudaStream_t s) {
    CUtensorMap kmap, vmap;
    if (!tl_encode() || !tc_map(&kmap, a.kpages, a) || !tc_map(&vmap, a.vpages, a)) return cudaErrorInvalidValue;
    constexpr size_t room = 226 * 1024 - 2048;     // beside the static part
    const int chunks = a.hd / 32, padded = (tc_group_heads(a) + 1) & ~1;
    const size_t tile = (size_t)chunks * 1024 * PT_GROUPS, queries = 2 * (size_t)chunks * padded * 1024, probs = 2 * PT_KEYS * 32;
    const TcShape ks = {chunks, (int)std::min<size_t>(PT_MAX_STAGES, (room - 1024 - queries) / tile), 128};
    const TcShape vs = {chunks, (int)std::min<size_t>(PT_MAX_STAGES, (room - 1024 - probs) / tile), chunks == 1 ? 128 : chunks == 2 ? 256 : 512};
    const size_t ksm = 1024 + queries + ks.stages * tile, vsm = 1024 + probs + vs.stages * tile;
    cudaError_t e = tc_configure(paged_scores_kernel, ksm);
    if (e == cudaSuccess) e = tc_configure(paged_values_kernel<SHORT, SMALL>, vsm);
    if (e != cudaSuccess) return e;
    const long long most = (long long)a.B * a.Hkv * tc_head_groups(a) * tc_tiles_most(a);
    const unsigned ctas = (unsigned)std::min<long long>(148, std::max<long long>(1, most));
    e = launch_behind(paged_scores_kernel, ctas, PT_THREADS, ksm, s, a, kmap, ks);
    if (e == cudaSuccess) e = launch_behind(paged_norm_kernel<SHORT>, (unsigned)std::min<long long>(296, std::max<long long>(1, most)), PN_THREADS, 0, s, a);
    if (e == cudaSuccess) e = launch_behind(paged_values_kernel<SHORT, SMALL>, ctas, PT_THREADS, vsm, s, a, vmap, vs);
    note_launch(3);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

// Rows that are whole 128-byte chunks (up to four), pages of whole groups of eight rows, probabilities of three bytes.
bool paged_tc_ok(const PagedAttnArgs &a) {
    return a.hd % 32 == 0 && a.hd <= 128 && a.P % 8 == 0 && a.fa <= 23;
}
size_t paged_tc_bytes(const PagedAttnArgs &a) {
    size_t n;
    tc_work(a, &n);
    return n;
}
cudaError_t launch_paged_tc(const PagedAttnArgs &a, cudaStream_t s) {
    if (a.fa > 16) return launch_tc<false, false>(a, s);
    return a.max_slots <= 1LL << (31 - a.fa) ? launch_tc<true, true>(a, s) : launch_tc<true, false>(a, s);
}

}  // namespace iie
