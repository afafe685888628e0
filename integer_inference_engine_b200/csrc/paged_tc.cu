// Attention of one new token per sequence over a paged cache, both products on tcgen05 with the cache rows as they lie in memory.
//
// An int32 is its four bytes, so a row of keys is a row of 4 hd bytes, and with the query's balanced base-256 digits d_a (modulo 2^64)
//     q . k = sum_s 2^(8 s) sum_i sum_{b <= s} k_i,b d_{s-b}(q_i)          s = 0 .. 7, modulo 2^64:
// products of the raw bytes with eight columns per head that hold digit s - b beside byte b.  No key is unpacked: TMA puts rows into
// shared memory, 128 keys x 64 columns (8 heads) x 4 hd bytes is one MMA shape, and a query of any 64 bits needs nothing else.  The top byte
// of an int32 is signed and the others are not; an MMA takes its operand as one or the other, so that the tile is multiplied twice, by the
// columns of bytes 0 .. 2 and by those of byte 3.  Values likewise: bytes of the value rows, transposed by the operand descriptor (the sum runs
// over keys), times the three bytes of the probabilities floor(e 2^fa / Z) <= 2^fa; byte 3 of a value is read from the signed product,
// the others from the unsigned one.  Every sum stays below 2^31: 4 hd 255 128 for a score, 255^2 per key for an output (at most 256 tiles
// of 128 keys before the sums are read out).
//
// Tiles of 128 keys of all sequences and KV heads form one list that one CTA per SM share (pair: a sequence's KV head with up to eight query heads): by whole pairs,
// by CTAs of a pair's own or by an even cut (tc_share).  The softmax floors e and p, which takes the maximum and then the normaliser of all of a pair's keys in
// front of its values: a CTA takes the scores of all its tiles (in memory, as 32-bit distances below the maximum of 32 keys; one beyond
// `clip` has no weight, so nothing is lost), the normalisers, then the values.  Pairs that lie in one CTA need nobody else.  Of those cut between CTAs
// (at most one begins in each) every CTA tells the others its maximum and its normaliser, and the output sums are added up in memory with a count of their
// parts: that launch is cooperative, every wait is bounded, integers are added in any order, and a small kernel in front clears what is told.  Where few tiles leave
// every pair whole whatever the lengths (launch_tc: `alone`) there is one launch, and it is not cooperative.
//
// What bounds it, replayed: memory where there is much of it, 118 us for 64 sequences of up to 4096 keys (4 KV heads of 128, 8 query heads each; 640 MB: 5.4 TB/s over the
// launch), 185 with 4096 keys each (1.07 GB: 5.8), 62 for 278 MB of three of up to 30000.  Beside that a call pays 3 us until the share is planned, 3 us until the first query
// columns are written, 6 to 9 us between keys and values (a microsecond or two for an exchange, twice, and the exponentials: 24 clocks for a warp's 32, 0.13 us for a tile of
// eight heads), 2 us for the outputs: 18 us for one sequence of 300 keys, 23 for one of 4096 (the contiguous caches' kernels, whose CTAs of a head are a cluster or
// know their place without a plan, 11 and 16 with the append in them).  A KV head with more than eight query heads is as many pairs as it has groups of eight, and
// its rows are read for each: 64 sequences of 4096 keys over one KV head 60 us with 8 heads, 99 with 16, 178 with 32.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "paged.h"
#include "softmax.cuh"
#include "tile_ops.cuh"

namespace iie {

namespace {

constexpr int PT_KEYS = 128, PT_GROUPS = 16;       // keys of a tile, groups of eight
constexpr int PT_HEADS = 8;                        // query heads of a pair at most
constexpr int PT_WORKERS = 16;                     // warps that read TMEM out and write operands: sets of four, one for each quarter of the keys; tile i is set i % 4's
constexpr int PT_SETS = PT_WORKERS / 4;
constexpr int PT_FIRST = 4;                         // warps in front of them: two that request copies, one that issues products
constexpr int PT_THREADS = 32 * (PT_FIRST + PT_WORKERS);
constexpr int PT_MAX_SLOTS = 13;                   // of the ring, 16 KB each: 128 bytes of 128 rows
constexpr int PT_META = 16;                        // tiles whose row masks are kept: those in the ring and two on their way out of TMEM
constexpr uint32_t PT_SLOT = PT_KEYS * 128, PT_PROBS = PT_KEYS * 32;
constexpr int PT_MAX_SEGMENT = 256;                // tiles that one accumulation takes: 256 * 128 * 255^2 < 2^31
constexpr unsigned PT_POLLS = 1u << 20;            // of another CTA's count, half a microsecond and more each
constexpr unsigned long long PT_BIAS = 1ULL << 63; // maxima are kept as unsigned: zero is below every score

constexpr int PT_COUNT = 56;                       // bit of an output sum where its parts are counted: the sum stays within 2^31 2^fa <= 2^54, as the probabilities' does within 2^fa

// What a CTA tells the others of a pair cut between them, one value per head: two words, each half a value and a bit that says that it is there.
struct TcNote { ulonglong2 head[PT_HEADS]; };
struct TcNotes { TcNote begins, goes_on; };        // of the pair that begins in a CTA, of the one that began in front of it
struct TcWork {
    uint32_t *dist;                // [tiles][N heads, 4 or 8][4 quarters][32] distances below the base (shifted, at most the limit): key k of a quarter at k % (32 / N) N + k / (32 / N), so
                                   // that the N keys of a lane lie side by side
    long long *base;               // [tiles][4 quarters][N] largest score of 32 keys
    unsigned long long *top, *z;   // [pairs][8], [pairs][16 warps][8] of pairs that lie in one CTA
    TcNotes *notes;                // [2: maxima, normalisers][CTAs]
    unsigned long long *acc;       // [CTAs][8][hd] output sums of the pair that begins in a CTA, and in bits 56 .. how many parts are in
};
__host__ __device__ inline int tc_head_groups(const PagedAttnArgs &a) { return (a.H / a.Hkv + PT_HEADS - 1) / PT_HEADS; }
__host__ __device__ inline int tc_group_heads(const PagedAttnArgs &a) { const int g = tc_head_groups(a); return (a.H / a.Hkv + g - 1) / g; }
// rows that a box of TMA brings, within a page (larger ones are slower: chunk after chunk of one SM alone 5.5 TB/s in all with 16 rows, 4.6 with 32 to 128)
__host__ __device__ inline int tc_box(const PagedAttnArgs &a) { return a.P % 16 == 0 ? 16 : 8; }
// tiles of a pair at most
__host__ __device__ inline long long tc_tiles_most(const PagedAttnArgs &a) {
    if (a.n_sel > 0) return ((long long)a.n_sel * a.P + PT_KEYS - 1) / PT_KEYS;
    return (a.max_slots + 2 * tc_box(a) + PT_KEYS - 1) / PT_KEYS;
}
// heads that warps are laid out for
__host__ __device__ inline int tc_room(const PagedAttnArgs &a) { return tc_group_heads(a) <= 4 ? 4 : 8; }
__host__ __device__ inline TcWork tc_work(const PagedAttnArgs &a, int ctas, size_t *bytes = nullptr) {
    const long long pairs = (long long)a.B * a.Hkv * tc_head_groups(a), tiles = pairs * tc_tiles_most(a);
    const int room = tc_room(a);
    TcWork w;
    w.dist = static_cast<uint32_t *>(a.work);
    w.base = reinterpret_cast<long long *>(w.dist + tiles * PT_KEYS * room);
    w.top = reinterpret_cast<unsigned long long *>(w.base + tiles * 4 * room);
    w.z = w.top + pairs * PT_HEADS;
    w.notes = reinterpret_cast<TcNotes *>(w.z + pairs * PT_WORKERS * PT_HEADS);
    w.acc = reinterpret_cast<unsigned long long *>(w.notes + 2 * ctas);
    if (bytes)
        *bytes = (size_t)tiles * room * (PT_KEYS * 4 + 4 * 8) + (size_t)pairs * (PT_WORKERS + 1) * PT_HEADS * 8 + (size_t)ctas * (2 * sizeof(TcNotes) + (size_t)PT_HEADS * a.hd * 8);
    return w;
}

__device__ __forceinline__ int tc_tiles(const PagedAttnArgs &a, const PagedSpan &s) {
    if (s.len == 0) return 0;
    if (a.sel) return (int)tc_tiles_most(a);
    return (s.len - (s.lo & ~(tc_box(a) - 1)) + PT_KEYS - 1) / PT_KEYS;
}

// A walk over a run of the list, tile by tile.
struct TcWalk {
    int owner, parts;                              // of a cut pair: the CTA where it begins, those that have a part
    int b, pair_of, t, nt, left, tile, part, seg;  // sequence; its pair; tile of the pair, its tiles; tiles left; number in the list; tiles of the pair and of the accumulation before this one
    PagedSpan s;
    __device__ __forceinline__ void load(const PagedAttnArgs &a) { paged_span(a, b, s); nt = tc_tiles(a, s); }
    __device__ __forceinline__ bool ends_part() const { return t + 1 == nt || left == 1; }             // of the pair, in this CTA
    __device__ __forceinline__ bool ends_segment() const { return ends_part() || seg + 1 == PT_MAX_SEGMENT; }
    __device__ __forceinline__ int rest() const { return min(nt - t, left); }                        // tiles of the pair from here on, in this CTA
    __device__ __forceinline__ void next(const PagedAttnArgs &a, int per_seq) {
        seg = ends_segment() ? 0 : seg + 1;
        part = ends_part() ? 0 : part + 1;
        skip(a, per_seq, 1);
    }
    __device__ __forceinline__ void skip(const PagedAttnArgs &a, int per_seq, int n) {               // n <= rest()
        left -= n; tile += n; t += n;
        if (t < nt || left == 0) return;
        t = 0;
        if (++pair_of < per_seq) return;
        pair_of = 0;
        do {                                       // (tiles are left: there is a sequence that has some)
            if (++b >= a.B) { left = 0; return; }
            load(a);
        } while (nt == 0);
    }
};

// One warp: the CTA's share of the list, as up to three runs: two pairs that it has in common with other CTAs, and whole pairs.  A pair that is cut costs its
// CTAs an exchange, some five microseconds; a second pair costs other query columns.
//  * Whole pairs, dealt out in order, where the launch says so (`alone`) or the longest pairs so dealt make a CTA no more than one tile above the average: a
//    tile is keys and values, one behind the other, some 2.6 us (1 x 600 keys, five tiles a pair: 25.0 us whole, 18.2 cut; 12 x 900 33.8 and 31.5; 16 x 600 25.8 either way).
//  * Else each pair has CTAs of its own in proportion to its tiles, where there are enough CTAs and no part is more than two tiles above it.
//  * Else the list is cut evenly: a CTA has the end of a pair, whole ones, the beginning of another.  (Cut pairs in an order that has two neighbours at
//    the same one first, normalised between tiles as soon as the maxima are in, were no faster: the registers and the code that this takes cost the
//    tiles what it hides.)
enum { RUN_WHOLE = 2, RUNS };
constexpr int PT_PAIR = 1;                         // what a pair costs beside its tiles, in tiles (64 x 4096 keys: 121 us with none, 118.3, 119.0 with two, 120.5 with three)
__device__ __noinline__ int tc_count(const PagedAttnArgs &a, int b) {
    PagedSpan s;
    if (b >= a.B) return 0;
    if (!paged_span(a, b, s) && blockIdx.x == 0) atomicOr(a.flags, 16);
    return tc_tiles(a, s);
}
__device__ __forceinline__ void tc_share(const PagedAttnArgs &a, bool alone, TcWalk (&run)[RUNS]) {
    const int lane = threadIdx.x & 31, per_seq = a.Hkv * tc_head_groups(a), ctas = gridDim.x, me = blockIdx.x;
    const int own = tc_count(a, lane);             // (32 sequences at a time; the first ones kept)
    auto count = [&](int b) { return b < 32 ? own : tc_count(a, b); };
    int sum = 0, some = 0, longest = 0;
#pragma unroll 1
    for (int b = lane; b - lane < a.B; b += 32) { const int c = count(b); sum += c; some += c > 0; longest = max(longest, c); }
    const int total = __reduce_add_sync(0xffffffffu, sum) * per_seq, pairs = __reduce_add_sync(0xffffffffu, some) * per_seq;       // (total * 256 fits 32 bits: paged_tc_ok)
    const int most = __reduce_max_sync(0xffffffffu, longest);
    const int average = total / ctas;
    // CTAs of a pair of c tiles that has its own, and the tiles of one
    auto parts = [&](int c) { return c == 0 ? 0 : max(1, min(c, (int)((uint32_t)c * ctas / total))); };
    auto part = [&](int c) { return c == 0 ? 0 : (c + parts(c) - 1) / parts(c); };
    enum { WHOLE_PAIRS, OWN_CTAS, EVEN } way = EVEN;
    if (alone || (pairs + ctas - 1) / ctas * most <= average + 1) way = WHOLE_PAIRS;
    else if (pairs <= ctas) {
        int ps = 0, pl = 0;
#pragma unroll 1
        for (int b = lane; b - lane < a.B; b += 32) { const int c = count(b); ps += parts(c); pl = max(pl, part(c)); }
        if ((int)__reduce_add_sync(0xffffffffu, ps) * per_seq <= ctas && (int)__reduce_max_sync(0xffffffffu, pl) <= average + 2) way = OWN_CTAS;
    }
    // the share in units of the way, and where in the list its first and last unit are
    const int all = way == EVEN ? total + PT_PAIR * pairs : pairs;
    const int from = way == OWN_CTAS ? me : (int)((uint32_t)all * me / ctas), to = way == OWN_CTAS ? me + 1 : (int)((uint32_t)all * (me + 1) / ctas);
    int at[2] = {-1, -1}, in[2] = {0, 0}, first[2] = {0, 0};       // sequence, unit in it, its first tile
    int before = 0, tiles_before = 0;              // units and tiles per pair of the sequences in front
#pragma unroll 1
    for (int b0 = 0; b0 < a.B && from < to && (at[0] < 0 || at[1] < 0); b0 += 32) {
        const int c = count(b0 + lane), mine = way == EVEN ? (c > 0) * (c + PT_PAIR) : way == OWN_CTAS ? parts(c) : (int)(c > 0);
        int upto = mine, tiles = c;
#pragma unroll 1
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, upto, d), p = __shfl_up_sync(0xffffffffu, tiles, d);
            if (lane >= d) { upto += o; tiles += p; }
        }
        const int lo = (before + upto - mine) * per_seq, hi = lo + mine * per_seq;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int unit = e ? to - 1 : from;
            const uint32_t here = __ballot_sync(0xffffffffu, unit >= lo && unit < hi);
            if (here && at[e] < 0) {
                const int l = __ffs(here) - 1;
                at[e] = b0 + l;
                in[e] = __shfl_sync(0xffffffffu, unit - lo, l);
                first[e] = __shfl_sync(0xffffffffu, (tiles_before + tiles - c) * per_seq, l);
            }
        }
        before += __shfl_sync(0xffffffffu, upto, 31); tiles_before += __shfl_sync(0xffffffffu, tiles, 31);
    }
    if (lane != 0) return;
    TcWalk w = {}, none = {};
    run[0] = run[1] = run[RUN_WHOLE] = none;
    if (from >= to || at[0] < 0 || at[1] < 0) return;
    w.b = at[0];
    w.load(a);
    TcWalk e = none;
    e.b = at[1];
    e.load(a);
    if (way == OWN_CTAS) {
        const int ps = parts(w.nt), size = part(w.nt), piece = in[0] % ps;
        w.pair_of = in[0] / ps;
        w.t = piece * size;
        w.left = max(0, min(size, w.nt - w.t));
        w.tile = first[0] + w.pair_of * w.nt + w.t;
        w.owner = me - piece; w.parts = (w.nt + size - 1) / size;
        if (w.left > 0) run[w.left == w.nt ? RUN_WHOLE : 0] = w;
    } else if (way == WHOLE_PAIRS) {
        w.pair_of = in[0];
        w.tile = first[0] + w.pair_of * w.nt;
        w.left = first[1] + (in[1] + 1) * e.nt - w.tile;
        run[RUN_WHOLE] = w;
    } else {
        // a pair's units: PT_PAIR without a tile, then one a tile; a CTA has the tiles whose units it has
        auto owner = [&](int unit) { return (int)((((uint32_t)unit + 1) * ctas - 1) / all); };
        const int units = w.nt + PT_PAIR, units_e = e.nt + PT_PAIR;
        w.pair_of = in[0] / units;
        const int begins = from - (in[0] - w.pair_of * units) + PT_PAIR;       // unit of its first tile
        w.t = max(0, from - begins);
        w.tile = first[0] + w.pair_of * w.nt + w.t;
        w.owner = owner(begins); w.parts = owner(begins + w.nt - 1) - w.owner + 1;
        e.pair_of = in[1] / units_e;
        const int begins_e = to - 1 - (in[1] - e.pair_of * units_e) + PT_PAIR;
        e.left = max(0, to - begins_e);            // (none where the share ends in front of its first tile)
        e.tile = first[1] + e.pair_of * e.nt;
        e.owner = owner(begins_e); e.parts = owner(begins_e + e.nt - 1) - e.owner + 1;
        w.left = e.tile + e.left - w.tile;
        if (w.left > 0 && w.rest() < w.nt) {
            run[0] = w;
            run[0].left = w.rest();
            w.skip(a, per_seq, w.rest());
        }
        if (w.left > 0) {
            if (e.left > 0 && e.left < e.nt) { run[1] = e; w.left -= e.left; }
            run[RUN_WHOLE] = w;
        }
    }
}

// Scores: the cut pairs first, which other CTAs wait for.  Values: whole pairs first, while normalisers of the others are on their way.
__device__ __forceinline__ int tc_value_run(int u) { return u == 0 ? RUN_WHOLE : u - 1; }

// Operand descriptors: the lower word has the address (in 16 bytes), the upper one the distance of groups of eight rows and the swizzle.  An
// MMA's descriptors are a constant away from those of its chunk: with both words computed for each, a product takes 250 clocks to issue, so 48
// (128 x 64 x 32) and 40 (128 x 32 x 32), what reading the operands from shared memory takes.
__device__ __forceinline__ uint32_t tc_desc(uint32_t addr) { return (addr >> 4) | (1u << 16); }
__host__ __device__ constexpr uint32_t tc_desc_upper(uint32_t stride, uint32_t swizzle) { return (stride >> 4) | (1u << 14) | (swizzle << 29); }
// (The collector cannot keep A for the second product: it holds what the first one made of the bytes' signs.)
template <uint32_t UPPER_A, uint32_t UPPER_B>
__device__ __forceinline__ void tc_mma(uint32_t d, uint32_t da, uint32_t db, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n .reg .b64 x, y;\n mov.b64 x, {%1, %5};\n mov.b64 y, {%2, %6};\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::i8 [%0], x, y, %3, p;\n}"
                 ::"r"(d), "r"(da), "r"(db), "r"(idesc), "r"(accumulate), "n"(UPPER_A), "n"(UPPER_B) : "memory");
}
constexpr uint32_t SW128 = 2, SW32 = 6;
__device__ __forceinline__ uint64_t tc_min(uint64_t x, long long most) { return x < (uint64_t)most ? x : (uint64_t)most; }
__device__ __forceinline__ void tc_ld8(uint32_t addr, int (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(addr));
}
__device__ __forceinline__ void tc_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Rows are read once: the second-level cache gives their lines up first, and keeps the distances that are written between them and read again
// (64 x 4096 keys 144 -> 129 us, from a flushed cache 158 -> 149).
__device__ __forceinline__ uint64_t tc_once() {
    uint64_t policy;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}
__device__ __forceinline__ void tc_tma(uint32_t dst, const CUtensorMap *map, int x, int row, uint32_t bar, uint64_t policy) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3}], [%4], %5;"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(row), "r"(bar), "l"(policy) : "memory");
}

// 128-byte chunks of a row, ring slots, TMEM columns, those of the scores (behind the outputs, or over their second buffer); whether no pair can be cut, so
// that no launch stands in front
struct TcShape { int chunks, slots, columns, score_at; bool alone; };

struct TcBars {
    uint64_t full[PT_MAX_SLOTS], empty[PT_MAX_SLOTS], meta[PT_META];
    uint64_t score_full[PT_SETS], score_free[2], query_full, prob_full[PT_SETS], prob_free[PT_SETS], out_full[2], out_free[2], pair_done, drain;
    uint64_t part_in[2], known[2];                 // of a cut pair: every warp's maxima, then normalisers; those of all CTAs
    uint32_t tmem;
    int abort;
    TcWalk run[RUNS];
    unsigned long long part[2][PT_WORKERS][PT_HEADS], top[2][PT_HEADS], z[2][PT_HEADS];     // of the cut pairs
    unsigned long long pair_top[2][PT_WORKERS][PT_HEADS];      // maxima of a whole pair and of the next
    unsigned char mask[PT_META][PT_GROUPS];
};

struct TcRing {
    int slot = 0;
    uint32_t pass = 0;
    __device__ __forceinline__ void step(int n) { if (++slot == n) { slot = 0; pass ^= 1; } }
};

// One thread's wait (tl_wait: a whole warp's, at twice the price).
__device__ __forceinline__ bool tc_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
    return tl_try(bar, parity) || tl_wait_slow(bar, parity, abort_flag);
}

// The two producer warps: the share's tiles into the ring, chunk by chunk in turn, a box per page (or part of one).  A chunk costs a thread 500
// clocks (a wait, the bytes to expect, up to sixteen boxes), and the memory's rate is one in 700 for each SM: one warp alone, which looked every
// box's page up in a lane of its own, took 1200.  The next tile's pages are looked up while this one's boxes are requested.
struct TcBoxes {
    uint32_t rows, sends, bytes;                   // this lane's rows that count; groups where a box begins; bytes of a chunk
    int row;                                       // of the box in the pool, in the lane where it begins
};
// a lane's group of the tile: where its page number stands in memory (asked for a tile ahead), and what else decides its rows
struct TcLook { uint32_t rows; int r, page; };
// Lane l < 16: rows of group l of the walk's tile that count by their positions, as a byte; the page's number on its way.
__device__ __forceinline__ TcLook tc_look(const PagedAttnArgs &a, const TcWalk &w, int kv, int box) {
    const int l = threadIdx.x & 31;
    TcLook x = {0, 0, 0};
    int logical, pos;
    if (w.left <= 0 || l >= PT_GROUPS) return x;
    if (a.sel) {
        const unsigned slot = ((unsigned)w.t * PT_GROUPS + l) * 8, i = slot / (unsigned)a.P;
        if (i >= (unsigned)a.n_sel) return x;
        x.r = (int)(slot - i * a.P);
        logical = a.sel[((long long)w.b * a.Hkv + kv) * a.n_sel + i];
        if (logical < 0) return x;
        if (logical >= a.table_ld) { atomicOr(a.flags, 16); return x; }
        pos = logical * a.P + x.r;                 // (a table's rows are numbered in 31 bits)
    } else {
        pos = (w.s.lo & ~(box - 1)) + (w.t * PT_GROUPS + l) * 8;
        logical = (int)((unsigned)pos / (unsigned)a.P);
        x.r = pos - logical * a.P;
    }
    const int from = max(w.s.lo - pos, 0), to = min(w.s.len - pos, 8);
    if (from >= to) return x;
    x.rows = ((1u << to) - 1) & ~((1u << from) - 1);
    x.page = a.table[(long long)w.b * a.table_ld + logical];
    return x;
}
__device__ __forceinline__ TcBoxes tc_boxes(const PagedAttnArgs &a, const TcLook &look, int kv, int box) {
    const int lane = threadIdx.x & 31, in_box = box / 8, first = lane & ~(in_box - 1);
    TcBoxes x;
    x.rows = look.rows;
    if (x.rows && (look.page < 0 || look.page >= a.n_pages)) { atomicOr(a.flags, 16); x.rows = 0; }
    const int row = (look.page * a.Hkv + kv) * a.P + look.r;
    const uint32_t some = __ballot_sync(0xffffffffu, x.rows != 0), mine = (some >> first) & ((1u << in_box) - 1);      // a box goes where one of its groups counts
    const int known = first + (mine ? __ffs(mine) - 1 : 0);
    x.row = __shfl_sync(0xffffffffu, row, known) - 8 * (known - first);
    x.sends = __ballot_sync(0xffffffffu, lane < PT_GROUPS && lane == first && mine != 0);
    x.bytes = (uint32_t)__popc(x.sends) * box * 128;
    return x;
}
// IN_BOX: groups of eight rows that a box brings.  `turn`: chunks requested so far, by both warps; `tile`: tiles.  (Asking the values into L2 ahead
// of the ring, too, while the normalisers are exchanged, was slower by a fifth: every other access waits behind them.)
template <int IN_BOX, bool KEYS>
__device__ __forceinline__ bool tc_produce(const PagedAttnArgs &a, TcWalk w, const CUtensorMap *map, TcBars &s, uint32_t ring, const TcShape &sh, int me, TcRing &at, int &turn,
                                           int &tile, volatile int *abort_flag) {
    const int lane = threadIdx.x & 31, groups = tc_head_groups(a), per_seq = a.Hkv * groups;
    constexpr uint32_t ALL = IN_BOX == 1 ? 0xFFFFu : 0x5555u;
    if (w.left == 0) return true;
    const uint64_t once = tc_once();
    int kv = w.pair_of / groups;
    TcLook look = tc_look(a, w, kv, 8 * IN_BOX);
    while (w.left > 0) {
        const TcBoxes x = tc_boxes(a, look, kv, 8 * IN_BOX);
        w.next(a, per_seq);
        kv = w.pair_of / groups;
        look = tc_look(a, w, kv, 8 * IN_BOX);      // of the next tile: used after this one's copies
        int row[PT_GROUPS / IN_BOX];
#pragma unroll
        for (int j = 0; j < PT_GROUPS / IN_BOX; j++) row[j] = __shfl_sync(0xffffffffu, x.row, j * IN_BOX);
        for (int c = 0; c < sh.chunks; c++, turn++, at.step(sh.slots)) {
            if ((turn & 1) != me) continue;
            if (turn >= sh.slots && !tl_wait(tl_u32(&s.empty[at.slot]), at.pass ^ 1, abort_flag)) return false;
            const bool marks = KEYS && c == 0;
            if (marks) {
                if (lane < PT_GROUPS) s.mask[tile % PT_META][lane] = (unsigned char)x.rows;
                __syncwarp();
            }
            if (tl_elect()) {
                const uint32_t bar = tl_u32(&s.full[at.slot]), to = ring + at.slot * PT_SLOT;
                if (marks) tl_arrive(tl_u32(&s.meta[tile % PT_META]));
                tl_expect(bar, x.bytes);
                if (x.sends == ALL) {
#pragma unroll
                    for (int j = 0; j < PT_GROUPS / IN_BOX; j++) tc_tma(to + j * IN_BOX * 1024, map, 32 * c, row[j], bar, once);
                } else {
#pragma unroll
                    for (int j = 0; j < PT_GROUPS / IN_BOX; j++)
                        if ((x.sends >> (j * IN_BOX)) & 1) tc_tma(to + j * IN_BOX * 1024, map, 32 * c, row[j], bar, once);
                }
            }
            __syncwarp();
        }
        tile++;
    }
    return true;
}
template <int IN_BOX>
__device__ __forceinline__ void tc_producer(const PagedAttnArgs &a, const CUtensorMap *kmap, const CUtensorMap *vmap, TcBars &s, uint32_t ring, const TcShape &sh, int me,
                                            volatile int *abort_flag) {
    TcRing at;
    int turn = 0, tile = 0;
    bool ok = true;
#pragma unroll 1
    for (int u = 0; ok && u < RUNS; u++) ok = tc_produce<IN_BOX, true>(a, s.run[u], kmap, s, ring, sh, me, at, turn, tile, abort_flag);
#pragma unroll 1
    for (int u = 0; ok && u < RUNS; u++) ok = tc_produce<IN_BOX, false>(a, s.run[tc_value_run(u)], vmap, s, ring, sh, me, at, turn, tile, abort_flag);
    if (!*abort_flag) return;
    __syncwarp();                                  // copies under way end before the CTA does
    for (int k = max(0, turn - sh.slots); k < turn; k++) {
        volatile int patient = 0;
        if ((k & 1) == me) tl_wait(tl_u32(&s.full[k % sh.slots]), (uint32_t)(k / sh.slots) & 1, &patient);
    }
}

// Query columns of one pair: column 8 h + s holds digit s - b of q_i at byte 4 i + b, bytes 0 .. 2 in one operand and byte 3 in the other.
// A thread rotates one value and writes its word of the eight columns; 3 us from the share to the last word, a round trip for queries and tables and code that is
// fetched once and run once (a thread with four values and columns, 16 bytes at a time, took no less).
__device__ __forceinline__ void tc_queries(const PagedAttnArgs &a, const TcWalk &w, int heads, int padded, unsigned char *lower, unsigned char *upper, int worker) {
    const int groups = tc_head_groups(a), kv = w.pair_of / groups, h0 = kv * (a.H / a.Hkv) + (w.pair_of % groups) * tc_group_heads(a), half = a.hd / 2;
    const int at_once = 32 * PT_WORKERS / a.hd, d = worker % a.hd;
    int h = worker / a.hd;
    if (h >= at_once) return;
    // the pair (x0, x1) that holds dimension d
    const bool pairs = a.rope == 1, second = pairs ? d & 1 : d >= half;
    const int i = pairs ? d >> 1 : second ? d - half : d, d0 = pairs ? d & ~1 : i, d1 = pairs ? d | 1 : i + half;
    const int64_t *q = a.q + (long long)w.b * a.q_ld + (long long)h0 * a.hd;
    uint64_t c = 0, n = 0, x0 = 0, x1 = 0;
    auto load = [&](int h) {
        x0 = x1 = 0;
        if (h >= heads) return;
        x0 = (uint64_t)q[h * a.hd + (a.rope ? d0 : d)];
        if (a.rope) x1 = (uint64_t)q[h * a.hd + d1];
    };
    load(h);
    if (a.rope) { c = (uint64_t)a.cos[(long long)(w.s.len - 1) * half + i]; n = (uint64_t)a.sin[(long long)(w.s.len - 1) * half + i]; }
#pragma unroll 1
    for (; h < padded; h += at_once) {
        const uint64_t y = a.rope ? (uint64_t)((int64_t)(second ? x0 * n + x1 * c : x0 * c - x1 * n) >> a.fa) : x0;
        load(h + at_once);
        const uint64_t v = (y + 0x8080808080808080ULL) ^ 0x8080808080808080ULL;
        const uint32_t first = __byte_perm((uint32_t)v, 0, 0x0123), last = __byte_perm((uint32_t)(v >> 32), 0, 0x0123);       // first digit on top
        uint32_t to = (uint32_t)(d >> 5) * (uint32_t)padded * 1024 + (uint32_t)h * 1024 + (uint32_t)(d & 3) * 4;
        const uint32_t j = (uint32_t)(d >> 2) & 7;
#pragma unroll
        for (uint32_t s = 0; s < 8; s++, to += 128) {
            const uint32_t x = s < 4 ? first >> (24 - 8 * s) : __funnelshift_r(last, first, 56 - 8 * s);
            *reinterpret_cast<uint32_t *>(lower + to + (j ^ s) * 16) = x & 0xFFFFFFu;
            *reinterpret_cast<uint32_t *>(upper + to + (j ^ s) * 16) = x & 0xFF000000u;
        }
    }
}

// One warp: a value per head of a cut pair (in the lanes 0 .. 7) told to the other CTAs, and the largest, or the sum, of what all of them tell.  A value comes with
// its own word that it is there: nothing waits for a fence, and nobody looks twice.
__device__ __forceinline__ TcNote *tc_note(TcNotes *notes, int cta, bool begins) { return begins ? &notes[cta].begins : &notes[cta].goes_on; }
__device__ __forceinline__ void tc_tell(TcNotes *notes, const TcWalk &w, unsigned long long x) {
    const int lane = threadIdx.x & 31;
    if (lane < PT_HEADS)
        asm volatile("st.relaxed.gpu.global.v2.u64 [%0], {%1, %2};" ::"l"(tc_note(notes, blockIdx.x, w.t == 0)->head + lane), "l"(x | 0xFFFFFFFFULL), "l"(x << 32 | 0xFFFFFFFFULL) : "memory");
}
template <bool LARGEST>
__device__ __forceinline__ bool tc_gather(TcNotes *notes, const TcWalk &w, unsigned long long *result, volatile int *abort_flag) {
    constexpr int DEEP = 8;                        // notes a lane asks for at once
    const int lane = threadIdx.x & 31, head = lane & 7;
    unsigned long long sum = 0;
    for (int c0 = lane >> 3; c0 - (lane >> 3) < w.parts; c0 += 4 * DEEP) {
        unsigned long long x;
        bool there = false;
        for (unsigned i = 0; i < PT_POLLS && !there && !*abort_flag; i++) {
            there = true;
            x = 0;
#pragma unroll
            for (int u = 0; u < DEEP; u++) {
                const int c = c0 + 4 * u;
                if (c >= w.parts) continue;
                unsigned long long high, low;
                asm volatile("ld.relaxed.gpu.global.v2.u64 {%0, %1}, [%2];" : "=l"(high), "=l"(low) : "l"(tc_note(notes, w.owner + c, c == 0)->head + head) : "memory");
                there = there && (uint32_t)high && (uint32_t)low;
                const unsigned long long y = (high & 0xFFFFFFFF00000000ULL) | low >> 32;
                x = LARGEST ? max(x, y) : x + y;
            }
        }
        if (!__all_sync(0xffffffffu, there)) { *abort_flag = 1; return false; }
        sum = LARGEST ? max(sum, x) : sum + x;
    }
#pragma unroll
    for (int d = 8; d < 32; d <<= 1) {
        const unsigned long long o = __shfl_xor_sync(0xffffffffu, sum, d);
        sum = LARGEST ? max(sum, o) : sum + o;
    }
    if (lane < PT_HEADS) result[lane] = sum;
    __syncwarp();
    return true;
}
// The warp that planned the share, afterwards: what the CTA's warps found about the cut pairs, exchanged.
__device__ __forceinline__ void tc_exchange(TcBars &s, const TcWork &work, volatile int *abort_flag) {
    const int lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");      // the notes are clear
#pragma unroll 1
    for (int round = 0; round < 2; round++) {      // maxima, normalisers
        TcNotes *notes = work.notes + round * gridDim.x;
#pragma unroll 1
        for (int x = 0; x < RUN_WHOLE; x++) {
            if (s.run[x].left == 0) continue;
            if (!tl_wait(tl_u32(&s.part_in[x]), round, abort_flag)) return;
            unsigned long long v = 0;
#pragma unroll 4
            for (int w = lane >> 3; w < PT_WORKERS; w += 4) {
                const unsigned long long y = s.part[x][w][lane & 7];
                v = round ? v + y : max(v, y);
            }
#pragma unroll
            for (int d = 8; d < 32; d <<= 1) {
                const unsigned long long o = __shfl_xor_sync(0xffffffffu, v, d);
                v = round ? v + o : max(v, o);
            }
            tc_tell(notes, s.run[x], v);
        }
#pragma unroll 1
        for (int x = 0; x < RUN_WHOLE; x++) {
            if (s.run[x].left == 0) continue;
            if (!(round ? tc_gather<false>(notes, s.run[x], s.z[x], abort_flag) : tc_gather<true>(notes, s.run[x], s.top[x], abort_flag))) return;
            if (lane == 0) tl_arrive(tl_u32(&s.known[x]));
        }
    }
}

// What a CTA's cut pairs need, cleared.  The attention's launch overlaps it: what lies in front of this kernel on the stream has ended when the
// attention's CTAs start, so that only this is waited for.
__global__ void paged_clear_kernel(TcNotes *notes, unsigned long long *acc, int per_cta) {
    pdl_enter();
    const int tid = threadIdx.x;
    constexpr int WORDS = 2 * sizeof(TcNotes) / 16;
    for (int i = tid; i < WORDS; i += blockDim.x) reinterpret_cast<ulonglong2 *>(notes)[(long long)blockIdx.x * WORDS + i] = make_ulonglong2(0, 0);
    for (int i = tid; i < per_cta / 2; i += blockDim.x) reinterpret_cast<ulonglong2 *>(acc)[(long long)blockIdx.x * (per_cta / 2) + i] = make_ulonglong2(0, 0);
}

// Exponential of a distance from the row's maximum, at most `limit`, where it is zero (a key that does not count stands there): of the general
// scale, and of fa = 16, where distances are kept shifted so that every product's shift is that of its upper word: 24 clocks a warp
// (six products of four, eight other instructions of two on another pipe) against 75.  The polynomial stays above 2^14 there.
struct TcExp {
    SoftmaxExp exp2;
    static constexpr int SHIFT = 0;
    uint32_t limit;
    __device__ __forceinline__ TcExp(const PagedAttnArgs &a) : exp2(a.fa, a.log2e, a.clip), limit((uint32_t)a.clip) {}
    __device__ __forceinline__ uint32_t operator()(uint32_t below) const { return (uint32_t)exp2((long long)below); }
};
struct TcExp16 {
    static constexpr int SHIFT = 11;
    uint32_t limit;                                // 18 2^32 / 94548 2^11 < 2^31
    __device__ __forceinline__ TcExp16(const PagedAttnArgs &a) : limit((uint32_t)a.clip << SHIFT) {}
    __device__ __forceinline__ uint32_t operator()(uint32_t below) const {
        const uint32_t u = __umulhi(below, 94548u << 5), f = u << 16, f1 = u & 0xFFFFu, f2 = __umulhi(f, f1), f3 = __umulhi(f, f2);
        return (65536u - __umulhi(f, 45426u) + __umulhi(f2, 15743u << 16) - __umulhi(f3, 3638u << 16)) >> (u >> 16);
    }
};

// Distances of a lane's N keys in one tile and the base they lie below; dist, base: of the lane in tile 0.
template <int N>
__device__ __forceinline__ void tc_distances(const uint32_t *dist, const long long *base, int tile, uint32_t (&d)[N], unsigned long long &biased) {
    const uint4 *from = reinterpret_cast<const uint4 *>(dist + (long long)tile * (N * PT_KEYS));
#pragma unroll
    for (int i = 0; i < N / 4; i++) {              // (the CTA's own: its SM's cache may hold them)
        const uint4 x = from[i];
        d[4 * i] = x.x; d[4 * i + 1] = x.y; d[4 * i + 2] = x.z; d[4 * i + 3] = x.w;
    }
    biased = (uint64_t)base[(long long)tile * 4 * N] ^ PT_BIAS;
}
// exponential of a key `d` below a base that lies `above` below the pair's largest score, both at most the limit
template <class Exp>
__device__ __forceinline__ uint32_t tc_weight(const Exp &exp2, uint32_t above, uint32_t d) { return exp2(min(above + d, exp2.limit)); }
// Sum of a head's exponentials over every fourth tile from `first` to `end`, the keys of a quarter.  A function of its own: inlined at each
// call its code, fetched once for every use, took longer than its work.
template <class Exp, int N>
__device__ __noinline__ unsigned long long tc_normalise(const PagedAttnArgs &a, const uint32_t *dist, const long long *base, int first, int end, unsigned long long top) {
    const Exp exp2(a);
    unsigned long long z = 0;
#pragma unroll 1
    for (int i = first; i < end; i += PT_SETS) {   // (two or four tiles' loads at once: registers that the rest of the kernel lacks, 64 x 4096 keys 128 instead of 122 us)
        uint32_t d[N], sum = 0;
        unsigned long long b;
        tc_distances<N>(dist, base, i, d, b);
        const uint32_t above = (uint32_t)tc_min(top - b, a.clip) << Exp::SHIFT;
#pragma unroll
        for (int e = 0; e < N; e++) sum += tc_weight(exp2, above, d[e]);
        z += sum;
    }
    __syncwarp();
#pragma unroll
    for (int d = 1; d < 32 / N; d <<= 1) z += __shfl_xor_sync(0xffffffffu, z, d);
    return z;                                      // the same in all lanes of the head
}

// AT16: fa = 16; SMALL: beside that every sum of exponentials at most 2^31; N: heads that a warp's lanes are dealt to, and keys of a lane (of four heads in a layout
// for eight, half of the lanes' exponentials would be for nothing)
template <bool AT16, bool SMALL, int N>
__global__ void __launch_bounds__(PT_THREADS, 1) paged_attn_kernel(const __grid_constant__ PagedAttnArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                                                                  const __grid_constant__ TcShape sh) {
    using Exp = std::conditional_t<AT16, TcExp16, TcExp>;
    using Quotient = std::conditional_t<SMALL, SoftmaxQuotient16, SoftmaxQuotient>;
    extern __shared__ unsigned char pt_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(pt_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) TcBars s;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), groups = tc_head_groups(a), per_seq = a.Hkv * groups;
    const int heads_most = tc_group_heads(a), padded = (heads_most + 1) & ~1;
    const uint32_t operand = (uint32_t)sh.chunks * padded * 1024;
    unsigned char *lower = smem, *upper = smem + operand, *probs = smem + 2 * operand;       // query columns; four tiles of probability bytes [128][32], byte a of head h at 8 a + h
    const uint32_t ring = tl_u32(smem) + 2 * operand + PT_SETS * PT_PROBS;
    volatile int *abort_flag = &s.abort;
    if (tid == 0) {
        s.abort = 0;
        for (int i = 0; i < sh.slots; i++) { tl_init(tl_u32(&s.full[i]), 1); tl_init(tl_u32(&s.empty[i]), 1); }
        for (int i = 0; i < PT_META; i++) tl_init(tl_u32(&s.meta[i]), 1);
        for (int i = 0; i < 2; i++) {
            tl_init(tl_u32(&s.score_free[i]), 4);
            tl_init(tl_u32(&s.out_full[i]), 1); tl_init(tl_u32(&s.out_free[i]), PT_WORKERS);
        }
        for (int i = 0; i < PT_SETS; i++) { tl_init(tl_u32(&s.score_full[i]), 1); tl_init(tl_u32(&s.prob_full[i]), 4); tl_init(tl_u32(&s.prob_free[i]), 1); }
        tl_init(tl_u32(&s.query_full), PT_WORKERS); tl_init(tl_u32(&s.pair_done), PT_WORKERS); tl_init(tl_u32(&s.drain), 1);
        for (int i = 0; i < 2; i++) { tl_init(tl_u32(&s.part_in[i]), PT_WORKERS); tl_init(tl_u32(&s.known[i]), 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tl_u32(&s.tmem)), "r"(sh.columns));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (warp == 3) {
        if (sh.alone) asm volatile("griddepcontrol.wait;" ::: "memory");       // (else what lies in front has ended: the clearing kernel waited for it)
        tc_share(a, sh.alone, s.run);
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s.tmem, 0), score_at = tmem + sh.score_at, buffer = (uint32_t)sh.chunks * 64;
    if (warp < 2) {
        if (tc_box(a) == 16) tc_producer<2>(a, &kmap, &vmap, s, ring, sh, warp, abort_flag);
        else tc_producer<1>(a, &kmap, &vmap, s, ring, sh, warp, abort_flag);
    } else if (warp == 2) {
        if (tl_elect()) {                          // one thread
            constexpr uint32_t up = tc_desc_upper(1024, SW128), pp = tc_desc_upper(256, SW32);
            constexpr uint32_t plain = (2u << 4) | (1u << 15) | (1u << 16) | ((32u >> 3) << 17) | ((128u >> 4) << 24), last_byte = plain | (1u << 7);      // both operands transposed; unsigned, values signed
            const uint32_t lower_i = tl_idesc(8 * padded, false), upper_i = tl_idesc(8 * padded, true);
            TcRing at;
            bool ok = true, fresh = true;
            int queries = 0, i = 0;
            for (int u = 0; u < RUNS; u++) {       // scores
                TcWalk v = s.run[u];
                for (fresh = true; ok && v.left > 0; i++) {
                    if (i >= 2) ok = tc_wait(tl_u32(&s.score_free[i & 1]), ((i >> 1) & 1) ^ 1, abort_flag);
                    if (ok && fresh) { ok = tc_wait(tl_u32(&s.query_full), queries & 1, abort_flag); queries++; }
                    const uint32_t d = score_at + (i & 1) * 64;
                    uint32_t q = tc_desc(tl_u32(smem));
                    for (int c = 0; ok && c < sh.chunks; c++, q += (uint32_t)padded * 64) {
                        ok = tc_wait(tl_u32(&s.full[at.slot]), at.pass, abort_flag);
                        if (!ok) break;
                        tc_after();
                        const uint32_t keys = tc_desc(ring + at.slot * PT_SLOT), q3 = q + (operand >> 4);
#pragma unroll
                        for (int k = 0; k < 8; k += 2) {       // 32 bytes of the rows
                            tc_mma<up, up>(d, keys + k, q + k, lower_i, (c | k) != 0);
                            tc_mma<up, up>(d, keys + k, q3 + k, upper_i, 1);
                        }
                        tl_commit(tl_u32(&s.empty[at.slot]));
                        at.step(sh.slots);
                    }
                    if (ok) tl_commit(tl_u32(&s.score_full[i % PT_SETS]));
                    fresh = v.t + 1 == v.nt;
                    v.next(a, per_seq);
                }
            }
            for (int k = max(0, i - 2); ok && k < i; k++) ok = tc_wait(tl_u32(&s.score_free[k & 1]), (k >> 1) & 1, abort_flag);      // (outputs take the scores' columns)
            int seg = 0;
            i = 0;
            for (int u = 0; u < RUNS; u++) {       // values
                TcWalk v = s.run[tc_value_run(u)];
                for (; ok && v.left > 0; i++) {
                    ok = tc_wait(tl_u32(&s.prob_full[i % PT_SETS]), (i / PT_SETS) & 1, abort_flag);
                    if (ok && v.seg == 0 && seg >= 2) ok = tc_wait(tl_u32(&s.out_free[seg & 1]), ((seg >> 1) & 1) ^ 1, abort_flag);
                    const uint32_t p = tc_desc(tl_u32(probs) + (i % PT_SETS) * PT_PROBS);
                    uint32_t d = tmem + (seg & 1) * buffer;
                    for (int c = 0; ok && c < sh.chunks; c++, d += 64) {
                        ok = tc_wait(tl_u32(&s.full[at.slot]), at.pass, abort_flag);
                        if (!ok) break;
                        tc_after();
                        const uint32_t values = tc_desc(ring + at.slot * PT_SLOT);
#pragma unroll
                        for (int k = 0; k < 4; k++) {          // 32 keys
                            tc_mma<up, pp>(d, values + 256 * k, p + 64 * k, plain, (v.seg | k) != 0);
                            tc_mma<up, pp>(d + 32, values + 256 * k, p + 64 * k, last_byte, (v.seg | k) != 0);
                        }
                        tl_commit(tl_u32(&s.empty[at.slot]));
                        at.step(sh.slots);
                    }
                    const bool last = v.ends_segment();
                    if (ok) {
                        tl_commit(tl_u32(&s.prob_free[i % PT_SETS]));
                        if (last) tl_commit(tl_u32(&s.out_full[seg & 1]));
                    }
                    if (last) seg++;
                    v.next(a, per_seq);
                }
            }
            if (*abort_flag) {                     // products under way end before their TMEM is given back
                tl_commit(tl_u32(&s.drain));
                volatile int patient = 0;
                tc_wait(tl_u32(&s.drain), 0, &patient);
            }
        }
        __syncwarp();
    } else if (warp == 3) {
        tc_exchange(s, tc_work(a, gridDim.x), abort_flag);
    } else {
        const int worker = tid - 32 * PT_FIRST, set = (warp - PT_FIRST) >> 2, quarter = warp & 3, key = quarter * 32 + lane;      // a warp reads TMEM lanes 32 (warp % 4) ..
        constexpr int LANES = 32 / N;              // of a head
        const int g = lane / LANES, t = lane % LANES;        // beyond the scores a lane has head g, keys t, t + LANES, .. of the quarter
        const TcWork work = tc_work(a, gridDim.x);
        const Exp exp2(a);
        bool ok = true;
        // sum of the exponentials of head g over those of n tiles from `first` on that this warp has read out: the first of them is `skip` on
        auto normalise = [&](int first, int n, int skip, unsigned long long top) {
            return tc_normalise<Exp, N>(a, work.dist + g * PT_KEYS + quarter * 32 + N * t, work.base + quarter * N + g, first + skip, g < heads_most ? first + n : first, top);
        };
        // what is left to do with the maxima of a pair (or of its part here) once the next pair's query columns are written, so that the
        // products go on meanwhile: exchange them; a whole pair's normaliser
        struct { int n = 0, nt, first, index, run; long long pair; } behind;       // tiles, the pair's; number of the first in the list, and among this CTA's scores
        long long largest = INT64_MIN;             // lane h: of head h, over this warp's tiles of the pair
        int whole_pairs = 0;
        auto settle = [&](long long most) {
            if (behind.n == 0) return true;
            const unsigned long long biased = (uint64_t)most ^ PT_BIAS;
            if (behind.n == behind.nt) {
                unsigned long long (&tops)[PT_WORKERS][PT_HEADS] = s.pair_top[whole_pairs & 1];
                if (lane < PT_HEADS) tops[4 * set + quarter][lane] = biased;
                __syncwarp();
                if (lane == 0) tl_arrive(tl_u32(&s.pair_done));
                __syncwarp();
                if (!tl_wait(tl_u32(&s.pair_done), whole_pairs & 1, abort_flag)) return false;
                whole_pairs++;
                unsigned long long m = 0;          // over the warps: some for each of a head's lanes
#pragma unroll
                for (int w = 0; w < PT_WORKERS / LANES; w++) m = max(m, tops[LANES * w + t][g]);
#pragma unroll
                for (int d = 1; d < LANES; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
                const unsigned long long sum = normalise(behind.first, behind.n, (set - behind.index) & 3, m);
                if (t == 0) work.z[(behind.pair * PT_WORKERS + 4 * set + quarter) * PT_HEADS + g] = sum;
                if (t == 0 && set + quarter == 0) work.top[behind.pair * PT_HEADS + g] = m;
            } else {
                if (lane < PT_HEADS) s.part[behind.run][4 * set + quarter][lane] = biased;
                __syncwarp();
                if (lane == 0) tl_arrive(tl_u32(&s.part_in[behind.run]));
            }
            behind.n = 0;
            return true;
        };
        for (int x = worker; x < (int)(PT_SETS * PT_PROBS / 16); x += 32 * PT_WORKERS) reinterpret_cast<uint4 *>(probs)[x] = make_uint4(0, 0, 0, 0);      // (the columns beyond 24 stay so)
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        for (int b = blockIdx.x; b < a.B; b += gridDim.x) {                // sequences without keys
            PagedSpan none;
            paged_span(a, b, none);
            if (tc_tiles(a, none) == 0)
                for (long long x = worker; x < (long long)a.H * a.hd; x += 32 * PT_WORKERS) a.out[(long long)b * a.H * a.hd + x] = 0;
        }
        // ---- scores ------------------------------------------------------------------------------------------------------------------
        int i = 0;
        for (int u = 0; u < RUNS; u++) {
            TcWalk v = s.run[u];
            for (bool fresh = true; ok && v.left > 0; i++) {
                if (fresh) {                       // the columns are free once the tile in front has been multiplied (a set has waited for one of the last four: no phase is mistaken)
                    if (i > 0 && !tl_wait(tl_u32(&s.score_full[(i - 1) % PT_SETS]), ((i - 1) / PT_SETS) & 1, abort_flag)) { ok = false; break; }
                    const long long most = largest;
                    largest = INT64_MIN;
                    tc_queries(a, v, min(heads_most, a.H / a.Hkv - v.pair_of % groups * heads_most), padded, lower, upper, worker);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) tl_arrive(tl_u32(&s.query_full));
                    if (!settle(most)) { ok = false; break; }
                }
                if (i % PT_SETS == set) {
                    if (!tl_wait(tl_u32(&s.meta[i % PT_META]), (uint32_t)(i / PT_META) & 1, abort_flag)) { ok = false; break; }
                    const bool seen = (s.mask[i % PT_META][key >> 3] >> (key & 7)) & 1, any = __any_sync(0xffffffffu, seen);
                    if (!tl_wait(tl_u32(&s.score_full[set]), (i / PT_SETS) & 1, abort_flag)) { ok = false; break; }
                    tc_after();
                    const uint32_t from = score_at + ((uint32_t)(quarter * 32) << 16) + (i & 1) * 64;
                    uint32_t *to = work.dist + (long long)v.tile * N * PT_KEYS + quarter * 32 + lane % LANES * N + lane / LANES;
                    long long base = INT64_MIN;
#pragma unroll 2
                    for (int h = 0; h < heads_most; h++) {
                        int c[8];
                        tc_ld8(from + 8 * h, c);
                        tc_ld_wait();
                        const uint64_t low = (uint64_t)((long long)c[0] + (long long)c[1] * 256 + (long long)c[2] * 65536 + (long long)c[3] * 16777216);
                        const uint32_t high = (uint32_t)c[4] + ((uint32_t)c[5] << 8) + ((uint32_t)c[6] << 16) + ((uint32_t)c[7] << 24);
                        const long long dot = (long long)(low + ((uint64_t)high << 32));
                        const long long score = (long long)((uint64_t)(dot >> a.fa) * (uint64_t)a.inv_sqrt) >> a.fa;
                        // the largest of the warp's 32 keys: by the upper words, then by the lower ones where those are equal
                        const int up = seen ? (int)(score >> 32) : INT32_MIN;
                        const int up_most = __reduce_max_sync(0xffffffffu, up);
                        const uint32_t low_most = __reduce_max_sync(0xffffffffu, seen && up == up_most ? (uint32_t)score : 0u);
                        const long long most = any ? (long long)(((uint64_t)(uint32_t)up_most << 32) | low_most) : INT64_MIN;
                        to[h * PT_KEYS] = seen ? (uint32_t)tc_min((uint64_t)most - (uint64_t)score, a.clip) << Exp::SHIFT : exp2.limit;
                        if (lane == h) base = most;
                    }
                    tc_before();
                    __syncwarp();
                    if (lane == 0) tl_arrive(tl_u32(&s.score_free[i & 1]));
                    if (lane < N) work.base[((long long)v.tile * 4 + quarter) * N + lane] = base;
                    largest = max(largest, base);
                }
                if (v.ends_part()) {
                    behind.n = v.part + 1; behind.nt = v.nt; behind.first = v.tile - v.t; behind.index = i - v.part; behind.run = u;
                    behind.pair = (long long)v.b * per_seq + v.pair_of;
                }
                fresh = v.t + 1 == v.nt;
                v.next(a, per_seq);
            }
        }
        __syncwarp();
        ok = ok && settle(largest);
        // ---- normalisers of the pairs that go on in other CTAs, once everybody's maxima are in ---------------------------------------
        for (int x = 0, index = 0; ok && x < RUN_WHOLE; x++) {
            const int n = s.run[x].left;
            if (n == 0) continue;
            ok = tl_wait(tl_u32(&s.known[x]), 0, abort_flag);
            if (!ok) break;
            const unsigned long long z = normalise(s.run[x].tile, n, (set - index) & 3, s.top[x][g]);
            if (t == 0) s.part[x][4 * set + quarter][g] = z;
            __syncwarp();
            if (lane == 0) tl_arrive(tl_u32(&s.part_in[x]));
            index += n;
        }
        asm volatile("griddepcontrol.wait;" ::: "memory");      // (whatever the share: what is launched behind counts on it)
        // ---- probabilities and values ---------------------------------------------------------------------------------------------
        if (ok) {                                  // what the CTA's warps left in memory
            if (lane == 0) tl_arrive(tl_u32(&s.pair_done));
            __syncwarp();
            ok = tl_wait(tl_u32(&s.pair_done), whole_pairs & 1, abort_flag);
        }
        Quotient quotient(0, a.fa);                // of head g
        constexpr int HELD = N / 4;                // heads of a lane in the sums
        unsigned long long top = 0, carry[HELD] = {};                     // of head g; output sums of earlier accumulations
        int seg = 0;
        struct { int tiles = 0, nt, owner, parts, heads; bool ends; int64_t *out; } pending;      // sums to read out: tiles of the pair in them (and in `carry`)
        auto read_out = [&]() {
            if (!tl_wait(tl_u32(&s.out_full[seg & 1]), (seg >> 1) & 1, abort_flag)) return false;
            tc_after();
            const int byte = lane & 3, d = 32 * set + 8 * quarter + (lane >> 2), h0 = HELD * byte;
            const bool whole = pending.tiles == pending.nt;
            unsigned long long *acc = work.acc + (long long)pending.owner * PT_HEADS * a.hd;
            if (set < sh.chunks) {                 // dimensions 32 set ..
                const uint32_t from = tmem + (seg & 1) * buffer + ((uint32_t)(quarter * 32) << 16) + 2 * set * 32;
                uint64_t sum[N];
#pragma unroll
                for (int h = 0; h < N; h++) sum[h] = 0;
#pragma unroll
                for (int part = 0; part < 3; part++) {
                    int x[8], y[8];
                    tc_ld8(from + 8 * part, x); tc_ld8(from + 32 + 8 * part, y);
                    tc_ld_wait();
#pragma unroll
                    for (int h = 0; h < N; h++) sum[h] += (uint64_t)(int64_t)(byte == 3 ? y[h] : x[h]) << (8 * part);
                }
                // four lanes hold a dimension's four bytes: two exchanges leave a lane with a quarter of the heads
                const bool high = byte & 2, odd = byte & 1;
#pragma unroll
                for (int h = 0; h < N; h++) sum[h] <<= 8 * byte;
#pragma unroll
                for (int h = 0; h < 2 * HELD; h++) {
                    const uint64_t give = high ? sum[h] : sum[h + 2 * HELD];
                    sum[h] = (high ? sum[h + 2 * HELD] : sum[h]) + __shfl_xor_sync(0xffffffffu, give, 2);
                }
#pragma unroll
                for (int h = 0; h < HELD; h++) {
                    const uint64_t give = odd ? sum[h] : sum[h + HELD];
                    carry[h] += (odd ? sum[h + HELD] : sum[h]) + __shfl_xor_sync(0xffffffffu, give, 1);
                }
#pragma unroll
                for (int h = 0; h < HELD; h++) {
                    if (!pending.ends || h0 + h >= pending.heads) continue;
                    if (!whole) {                  // added up in memory: who adds the last part finds the sum
                        const unsigned long long part = carry[h] + (1ULL << PT_COUNT), all = atomicAdd(acc + (h0 + h) * a.hd + d, part) + part;
                        const unsigned long long parts = (all + (1ULL << (PT_COUNT - 1))) >> PT_COUNT;
                        if (((parts ^ pending.parts) & 0xFF) != 0) continue;
                        carry[h] = all - (parts << PT_COUNT);
                    }
                    pending.out[(long long)(h0 + h) * a.hd + d] = (int64_t)carry[h] >> a.fa;
                }
            }
            tc_before();
            __syncwarp();
            if (lane == 0) tl_arrive(tl_u32(&s.out_free[seg & 1]));
            if (pending.ends)
                for (int h = 0; h < HELD; h++) carry[h] = 0;
            pending.tiles = 0;
            seg++;
            return true;
        };
        i = 0;
        for (int u = 0; u < RUNS; u++) {
            const int run = tc_value_run(u);
            TcWalk v = s.run[run];
            for (bool fresh = true; ok && v.left > 0; i++) {
                if (fresh) {
                    unsigned long long z = 0;
                    top = 0;
                    if (v.t == 0 && v.rest() == v.nt) {
                        const long long pair = (long long)v.b * per_seq + v.pair_of;
                        top = __ldcg(work.top + pair * PT_HEADS + g);
#pragma unroll
                        for (int w = 0; w < PT_WORKERS / LANES; w++) z += __ldcg(work.z + (pair * PT_WORKERS + LANES * w + t) * PT_HEADS + g);
#pragma unroll
                        for (int d = 1; d < LANES; d <<= 1) z += __shfl_xor_sync(0xffffffffu, z, d);
                    } else {
                        if (!tl_wait(tl_u32(&s.known[run]), 1, abort_flag)) { ok = false; break; }
                        top = s.top[run][g]; z = s.z[run][g];
                    }
                    quotient = Quotient(g < heads_most ? z : 0, a.fa);
                }
                if (i % PT_SETS == set) {
                    uint32_t p[N];
                    unsigned long long base;
                    tc_distances<N>(work.dist + g * PT_KEYS + quarter * 32 + N * t, work.base + quarter * N + g, v.tile, p, base);
                    const uint32_t above = (uint32_t)tc_min(top - base, a.clip) << Exp::SHIFT;
#pragma unroll
                    for (int e = 0; e < N; e++) p[e] = g < heads_most ? (uint32_t)quotient(tc_weight(exp2, above, p[e])) : 0u;
                    if (i >= PT_SETS && !tl_wait(tl_u32(&s.prob_free[set]), ((i / PT_SETS) & 1) ^ 1, abort_flag)) { ok = false; break; }
                    unsigned char *to = probs + set * PT_PROBS + (quarter * 32 + t) * 32 + g;
#pragma unroll
                    for (int e = 0; e < N; e++) {      // key t + LANES e: byte b at 8 b + g, the halves of 32 bytes swapped in every second group of four rows
                        const int at = LANES * 32 * e, swap = (((t + LANES * e) >> 2) & 1) * 16;
                        to[at + swap] = (unsigned char)p[e];
                        to[at + 8 + swap] = (unsigned char)(p[e] >> 8);
                        to[at + 16 - swap] = (unsigned char)(p[e] >> 16);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) tl_arrive(tl_u32(&s.prob_full[set]));
                }
                // (sums are read out behind the next tile's probabilities, so that the products go on meanwhile)
                if (pending.tiles && (i % PT_SETS == set) && !read_out()) { ok = false; break; }
                if (v.ends_segment()) {
                    if (pending.tiles && !read_out()) { ok = false; break; }
                    const int group = v.pair_of % groups, kv = v.pair_of / groups;
                    pending.tiles = v.part + 1; pending.nt = v.nt; pending.ends = v.ends_part(); pending.owner = v.owner; pending.parts = v.parts;
                    pending.heads = min(heads_most, a.H / a.Hkv - group * heads_most);
                    pending.out = a.out + ((long long)v.b * a.H + kv * (a.H / a.Hkv) + group * heads_most) * a.hd;
                }
                fresh = v.t + 1 == v.nt;
                v.next(a, per_seq);
            }
        }
        if (ok && pending.tiles) read_out();
    }
    tc_before();
    __syncthreads();
    if (warp == 2) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(sh.columns));
    }
    if (tid == 0 && s.abort) atomicOr(a.flags, FLAG_GAVE_UP);
}

bool tc_map(CUtensorMap *map, const int32_t *pool, const PagedAttnArgs &a) {
    const cuuint64_t dims[2] = {(cuuint64_t)a.hd, (cuuint64_t)a.n_pages * a.Hkv * a.P}, strides[1] = {(cuuint64_t)a.hd * 4};
    const cuuint32_t box[2] = {32, (cuuint32_t)tc_box(a)}, step[2] = {1, 1};
    return tl_encode()(map, CU_TENSOR_MAP_DATA_TYPE_INT32, 2, const_cast<int32_t *>(pool), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int PT_MOST_CTAS = 256;                  // that the scratch has room for

template <bool AT16, bool SMALL, int N>
cudaError_t launch_tc(const PagedAttnArgs &a, cudaStream_t s) {
    CUtensorMap kmap, vmap;
    if (!tl_encode() || !tc_map(&kmap, a.kpages, a) || !tc_map(&vmap, a.vpages, a)) return cudaErrorInvalidValue;
    const int chunks = a.hd / 32, padded = (tc_group_heads(a) + 1) & ~1;
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const int sms = paged_sms();                   // one CTA is resident on each, as a cooperative launch needs
    if (sms <= 0) return cudaErrorInvalidDevice;
    const size_t fixed = 1024 + 2 * (size_t)chunks * padded * 1024 + PT_SETS * PT_PROBS, room = 227 * 1024 - sizeof(TcBars) - 64;
    const int slots = (int)std::min<size_t>(PT_MAX_SLOTS, (room - fixed) / PT_SLOT);
    const size_t smem = fixed + (size_t)slots * PT_SLOT;
    static std::atomic<unsigned long long> configured;             // devices, a bit each
    const unsigned long long bit = device < 64 ? 1ULL << device : 0;
    if (!(configured & bit)) {
        e = cudaFuncSetAttribute(paged_attn_kernel<AT16, SMALL, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(room));
        if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_clear_kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);      // else the attention waits for idle SMs
        if (e != cudaSuccess) return e;
        configured |= bit;
    }
    const long long most = (long long)a.B * a.Hkv * tc_head_groups(a) * tc_tiles_most(a);
    const unsigned ctas = (unsigned)std::min<long long>(std::min(sms, PT_MOST_CTAS), std::max<long long>(1, most));
    // Whole pairs whatever the lengths, where that is at most eight tiles a CTA and two above an even share of the longest lists: nothing to exchange or to clear, one launch that is
    // not cooperative (1 x 300 keys 18.8 us replayed; with the launch in front 19.8; 32 sequences over 416 selected keys each 44.8 in place of 46.8 replayed, 45.6 of 51.5 called; 16 x 600
    // 24.2 of 25.8 and 24.6 of 28.9).
    const long long pairs = (long long)a.B * a.Hkv * tc_head_groups(a);
    const long long longest = (pairs + ctas - 1) / ctas * tc_tiles_most(a);
    const bool alone = longest <= 8 && longest * ctas <= pairs * tc_tiles_most(a) + 2 * (long long)ctas;
    // outputs: two buffers of 64 columns a chunk; scores: two of 64, behind them or, at four chunks, over the end of the second
    const TcShape sh = {chunks, slots, chunks == 1 ? 256 : 512, chunks == 4 ? 384 : 128 * chunks, alone};
    if (!alone) {
        const TcWork w = tc_work(a, (int)ctas);
        e = launch_behind(paged_clear_kernel, ctas, 128, 0, s, w.notes, w.acc, PT_HEADS * a.hd);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas); cfg.blockDim = dim3(PT_THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeCooperative; attr[1].val.cooperative = 1;
    cfg.attrs = attr; cfg.numAttrs = alone ? 1 : 2;
    e = cudaLaunchKernelEx(&cfg, paged_attn_kernel<AT16, SMALL, N>, a, kmap, vmap, sh);
    note_launch(alone ? 1 : 2);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

int paged_sms() {
    static std::atomic<int> known[64];
    int device = 0, n = 0;
    if (cudaGetDevice(&device) != cudaSuccess) { cudaGetLastError(); return 0; }
    if (device < 64 && known[device] > 0) return known[device];
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) { cudaGetLastError(); return 0; }
    if (device < 64) known[device] = n;
    return n;
}

// Rows that are whole 128-byte chunks (up to four), pages of whole groups of eight rows, probabilities of three bytes, a list whose place times the
// CTAs fits 32 bits.
bool paged_tc_ok(const PagedAttnArgs &a) {
    return a.hd % 32 == 0 && a.hd <= 128 && a.P % 8 == 0 && a.fa <= 23 && tc_tiles_most(a) * a.Hkv * tc_head_groups(a) <= 1 << 23;
}
size_t paged_tc_bytes(const PagedAttnArgs &a) {
    size_t n;
    tc_work(a, PT_MOST_CTAS, &n);
    return n;
}
cudaError_t launch_paged_tc(const PagedAttnArgs &a, cudaStream_t s) {
    const bool at16 = a.fa == 16, small = a.max_slots <= 1LL << 15;
    if (tc_room(a) == 4) return !at16 ? launch_tc<false, false, 4>(a, s) : small ? launch_tc<true, true, 4>(a, s) : launch_tc<true, false, 4>(a, s);
    return !at16 ? launch_tc<false, false, 8>(a, s) : small ? launch_tc<true, true, 8>(a, s) : launch_tc<true, false, 8>(a, s);
}

}  // namespace iie
