// Attention of trees of drafted tokens on the 5th-generation tensor cores: the same sums as csrc/tree_attention.cu (which says what a row
// sees), bfloat16 heads of 64 and 128, no window.  Per unit, which is up to 256 (row, query head) pairs of one request and key/value head, and
// tile of 64 keys
//
//     S = Q K^T      tcgen05.mma, M = 128 pairs (TMEM lanes), N = 64 keys, both operands in shared memory
//     P = exp2(..)   a pair a thread, from TMEM and back into it over its scores, two bfloat16 a column
//     O += P V       tcgen05.mma, A in TMEM, V as it lies ([key][column], MN-major), N = the head's columns
//
// Eight softmax warps are two turns with scores, O, reference and sum of their own, and a warp each that issues their products: while one tile
// is in the softmax, the other's P is multiplied and its buffer gets the scores after next.  A unit of more than 128 pairs has a turn for
// each half of its pairs, and each tile of keys serves both; a smaller one has its tiles by turns, and the two O are joined at its end.
//
// A tile's keys and its values take a slot each of two rings, laid out in the 128-byte swizzle that the products read.  Tiles of cached keys alone
// come by TMA, page by page; a unit's last ones, which end inside a page or hold the drafted rows, by cp.async (rows at any 16-byte stride,
// zeros for keys that are not there).  Nothing is waited for there but a free slot: copies arrive at their barrier by themselves.
//
// The work is the list of all units' tiles, cut into equal shares for as many blocks as there are SMs: a block's share may begin and end
// inside a unit, whose parts then go to memory and are joined by a second kernel.  (Requests of a batch differ in length by a factor of
// twenty and more; with a block or a cluster a unit the longest decides.)
//
// What bounds it, 8 trees of 24-64 rows of 32 heads over 8, heads of 128, behind 4000-30000 positions: 143 us, of which the launches, the list, the
// first loads and the join some 25; without the softmax 119, without it and most of the products 85.  A tile that serves both turns reads 48 KB of operands for each of
// them, 1300 cycles of shared memory's 128 bytes a cycle, against 1024 cycles of exponentials.  With heads of 64 (32 trees of 4-24
// rows behind 300-6000 positions, 63 us) it is the softmax's chain: 64 exponentials a thread and tile are 512 of its 2000 cycles.
#include "attention_tc_helpers.cuh"
#include "mma_helpers.cuh"

#define TT_KEYS 64                      // keys of a tile
#define TT_TILE 128                     // lanes of a product
#define TT_UNIT 256                     // pairs of a unit
#define TT_ROWS 128                     // rows of a tree: two tiles of keys
#define TT_SOFTMAX 8
#define TT_LOADERS 2                    // (twelve warps leave a thread 168 registers; with four loaders, 128)
#define TT_THREADS (32 * (TT_SOFTMAX + TT_LOADERS + 2))
#define TT_LEAST 4                      // cost of a share: fewer blocks take part when there is less than this for each (16: 20 instead of 15 us for one tree
                                        // of 32 rows of 32 heads behind 2000 positions)
// Cost of a unit beside its tiles: its first scores and its end.  (Blocks with shares of nine short units were the last by a third: none
// counted 86 us, this 69, when the 32 trees above were measured so.)
#define TT_EXTRA 6
#define TT_LOG2E 1.4426950408889634f

struct TtArgs {
    bf16* out;
    const bf16 *q, *k, *v, *pages;
    long long q_stride, k_stride, v_stride;
    const int *table, *cu, *ctx;
    const unsigned* mask;
    int table_width, words, S, N, page_size, page_shift, num_pages, H, G;
    int group, dual_cost, unit_extra;   // query heads of a key/value head; what a tile that both turns work on costs, and a unit beside its tiles
    int reach;                          // positions that a block table's row holds
    float scale;
    float* parts;                       // [2 blocks][D / 4][TT_UNIT][4]: O, then [2 blocks][TT_UNIT][2]: reference and sum, then [blocks] Cut
    int* status;
};

// ---- the list of tiles.  A request with n rows has units of 256 pairs by key/value head, the last ones of what is left; each unit has a
// tile for every 64 cached keys and one or two for the drafted rows.  What a tile that both turns work on costs beside one of a turn alone: with
// heads of 64 twice as much (the softmax's chain is the limit; counted the same, 32 trees of 4-24 rows take as long, 70 us with L2 flushed, and 8 of
// 33-64 rows 92 instead of 94); with heads of 128 the same (8 trees of 24-64 rows behind 4000-30000 positions 156 us, counted double 168; one of 64
// behind 30 000 63.5 and 65.7).
struct Request { int first, n, ctx, cached, tiles, row_units, last_cost; };
__device__ __forceinline__ int unit_cost(const TtArgs& a, int pairs) { return pairs > TT_TILE ? a.dual_cost : 1; }
__device__ __forceinline__ Request request_of(const TtArgs& a, int s, bool say) {
    Request r = {0, 0, 0, 0, 0, 0, 0};
    r.first = a.cu[s];
    const int end = a.cu[s + 1];
    r.n = end - r.first;
    r.ctx = max(a.ctx[s], 0);
    const bool outside = r.first < 0 || end < r.first || end > a.N;     // (the span is passed over; rows before the first span or behind the last: nobody's)
    if (say && (outside || (s == 0 && r.first != 0) || (s == a.S - 1 && end != a.N))) zai_raise(a.status, ZAI_ST_ROWS);
    if (outside || r.n == 0) {
        r.n = 0;
        return r;
    }
    if (r.n > TT_ROWS) {
        if (say) zai_raise(a.status, ZAI_ST_TREE);
        r.n = TT_ROWS;
    }
    if (r.ctx > a.reach) {                                      // (what is beyond has no page)
        if (say) zai_raise(a.status, ZAI_ST_POSITION);
        r.ctx = a.reach;
    }
    r.cached = (r.ctx + TT_KEYS - 1) / TT_KEYS;
    r.tiles = r.cached + (r.n + TT_KEYS - 1) / TT_KEYS;
    const int pairs = r.n * a.group;
    r.row_units = (pairs + TT_UNIT - 1) / TT_UNIT;
    r.last_cost = unit_cost(a, pairs - (r.row_units - 1) * TT_UNIT);
    return r;
}
__device__ __forceinline__ long long cost_of(const TtArgs& a, const Request& r) {
    return r.n ? a.G * (r.tiles * ((long long)a.dual_cost * (r.row_units - 1) + r.last_cost) + (long long)a.unit_extra * r.row_units) : 0;
}
__device__ __forceinline__ int divided(long long x, long long by) {      // (32-bit where both fit, which is nearly always)
    return (x | by) >> 31 ? (int)(x / by) : (int)((unsigned)x / (unsigned)by);
}
// The blocks' shares: equal ones, the first of them one larger where it does not come out even.
struct Shares {
    long long each, more;
    int blocks;
    __device__ __forceinline__ Shares(long long total, int most) {
        blocks = (int)max(min((total + TT_LEAST - 1) / TT_LEAST, (long long)most), 1LL);
        each = total / blocks;
        more = total - each * blocks;
    }
    __device__ __forceinline__ long long start(int b) const { return b * each + min((long long)b, more); }
    __device__ __forceinline__ int owner(long long cost) const {         // the block whose share holds it
        const long long larger = more * (each + 1);
        return cost < larger ? divided(cost, each + 1) : (int)more + divided(cost - larger, each);
    }
};
// What a block whose share begins inside a unit says of it for the joining kernel: the unit's pairs, and the blocks that have parts of it
// (the first one's is in its second place, the others' in their first).  b1 < b0: nothing to join here.
struct Cut { int first, pair0, pairs, head, b0, b1, spare[2]; };
// Where a cost lies: the unit (its row of units and head), its first cost, its tiles' cost.
struct Place { int row, head, w; long long unit, per; };
__device__ __forceinline__ Place place_of(const TtArgs& a, const Request& r, long long base, long long pos) {
    const int w = a.dual_cost;
    const long long full = a.G * ((long long)w * r.tiles + a.unit_extra);      // a row of full units
    Place p;
    p.row = min(divided(pos - base, full), r.row_units - 1);
    p.w = p.row + 1 < r.row_units ? w : r.last_cost;
    p.per = (long long)p.w * r.tiles + a.unit_extra;
    const long long row_base = base + p.row * full;
    p.head = divided(pos - row_base, p.per);
    p.unit = row_base + p.head * p.per;
    return p;
}
// (a unit's extra cost comes before its tiles')
__device__ __forceinline__ int tiles_before(const TtArgs& a, const Place& p, long long cost) {
    return (int)(max(cost - p.unit - a.unit_extra + p.w - 1, 0LL) >> (p.w - 1));
}

struct Segment {
    int s, first, n, ctx, pair0, pairs, head, cached, tiles, from, upto;       // key tiles [from, upto) of the unit's `tiles`, the first of them `cached` ones
    __device__ __forceinline__ bool dual() const { return pairs > TT_TILE; }
    __device__ __forceinline__ bool whole() const { return from == 0 && upto == tiles; }
};
// A walk over the segments of the costs [pos, end); `s` and `base`: the request that holds pos and its first cost.  From unit to unit of a request
// it goes without a look at memory or a division.
struct Walk {
    long long pos, end, base;
    int s;
    bool begun;
    Request r;
    Place p;
    __device__ __forceinline__ bool next(const TtArgs& a, Segment& g) {
        while (pos < end) {
            if (!begun) {
                begun = true;
                r = request_of(a, s, false);
                p = place_of(a, r, base, pos);
            } else if (++p.head < a.G) p.unit += p.per;
            else if (++p.row < r.row_units) {
                p.unit += p.per;
                p.head = 0;
                if (p.row + 1 == r.row_units) p.w = r.last_cost;
                p.per = (long long)p.w * r.tiles + a.unit_extra;
            } else {
                p.unit += p.per;
                do {                                            // (there is one: pos lies before the end)
                    r = request_of(a, ++s, false);
                } while (r.n == 0 && s < a.S - 1);
                p.row = p.head = 0;
                p.w = r.row_units > 1 ? a.dual_cost : r.last_cost;
                p.per = (long long)p.w * r.tiles + a.unit_extra;
            }
            const long long stop = min(end, p.unit + p.per);
            g.from = tiles_before(a, p, pos);
            g.upto = tiles_before(a, p, stop);
            pos = stop;
            if (g.from == g.upto) continue;
            g.s = s;
            g.first = r.first;
            g.n = r.n;
            g.ctx = r.ctx;
            g.head = p.head;
            g.pair0 = p.row * TT_UNIT;
            g.pairs = min(r.n * a.group - g.pair0, TT_UNIT);
            g.cached = r.cached;
            g.tiles = r.tiles;
            return true;
        }
        return false;
    }
};
// By one warp: the cost of all, and the request that holds `at` with its first cost (at < 0: the total alone).
__device__ __forceinline__ long long scan_costs(const TtArgs& a, long long at, int& s_out, long long& base_out, bool say) {
    const int lane = threadIdx.x & 31;
    long long total = 0;
    for (int s0 = 0; s0 < a.S; s0 += 32) {
        const int s = s0 + lane;
        const long long c = s < a.S ? cost_of(a, request_of(a, s, say)) : 0;
        long long x = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        const unsigned here = __ballot_sync(0xffffffffu, at >= total + x - c && at < total + x);
        if (here) {
            const int w = __ffs(here) - 1;
            s_out = s0 + w;
            base_out = total + __shfl_sync(0xffffffffu, x - c, w);
        }
        total += __shfl_sync(0xffffffffu, x, 31);
    }
    return total;
}
__device__ __forceinline__ Cut* cuts_of(const TtArgs& a, int blocks, int D) {
    return reinterpret_cast<Cut*>(a.parts + (size_t)2 * blocks * TT_UNIT * (D + 2));
}
// By one warp: a block's walk over its share, and what it says for the joining kernel.
__device__ __forceinline__ void begin_walk(const TtArgs& a, int D, long long* share, int* s_first) {
    int s = 0;
    long long base = 0;
    const long long total = scan_costs(a, -1, s, base, blockIdx.x == 0);
    const Shares shares(total, gridDim.x);
    const bool part = (int)blockIdx.x < shares.blocks;
    const long long pos = part ? shares.start(blockIdx.x) : 0, end = part ? shares.start(blockIdx.x + 1) : 0;
    if (pos < end) scan_costs(a, pos, s, base, false);
    if ((threadIdx.x & 31) == 0) {
        share[0] = pos;
        share[1] = end;
        share[2] = base;
        *s_first = s;
        Cut cut = {0, 0, 0, 0, 0, -1, {0, 0}};
        if (pos < end) {
            const Request r = request_of(a, s, false);
            const Place p = place_of(a, r, base, pos);
            const int b0 = shares.owner(p.unit + a.unit_extra), b1 = shares.owner(p.unit + p.per - p.w);     // the first tile's block and the last one's
            if (b0 < (int)blockIdx.x && (int)blockIdx.x <= b1) {
                cut.first = r.first;
                cut.pair0 = p.row * TT_UNIT;
                cut.pairs = min(r.n * a.group - cut.pair0, TT_UNIT);
                cut.head = p.head;
                cut.b0 = b0;
                cut.b1 = b1;
            }
        }
        cuts_of(a, gridDim.x, D)[blockIdx.x] = cut;
    }
}

// The two turns' warps of a quarter of the multiprocessor do their exponentials one after the other (64 x 8 cycles of its special-function unit
// each), while the other waits, loads and compares: 67 instead of 71 us for the 32 trees above, 58 instead of 61 for 8 of 33-64 rows.
#define TT_SYNC(i) asm volatile("bar.sync %0, 64;" ::"r"(2 + (i)) : "memory")
#define TT_ARRIVE(i) asm volatile("bar.arrive %0, 64;" ::"r"(2 + (i)) : "memory")
__device__ __forceinline__ void tt_ld16_nowait(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
}
__device__ __forceinline__ void tt_wait_ld16(uint32_t (&r)[16]) {        // (tied to its registers, as at_tmem_wait_ld)
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :: "memory");
}
__device__ __forceinline__ void tt_arrive(uint64_t* bar, int count) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(at_smem(bar)), "r"(count) : "memory");
}
// An arrival of this thread's at a barrier when its copies so far have landed
__device__ __forceinline__ void tt_arrive_landed(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(at_smem(bar)) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Where a segment's queries lie: `use` counts the halves (of 128 pairs) taken so far, one by a segment of one turn's pairs, two by another;
// both turns' product warps wait for all of them, and say of the other's half at once that they are done with it.
template <int QS> struct Queries {
    static __device__ __forceinline__ int slot(int use) { return use % QS; }
    static __device__ __forceinline__ uint32_t round(int use) { return (use / QS) & 1; }
};
// What the loaders and the other warps share.
struct Pipe {
    unsigned char *q, *ring;
    uint64_t *full, *empty, *q_full, *q_empty;
    volatile int *odd, *failed;         // odd [16] by segment: its number (8 bits) + 1 if a drafted value is not finite
};

// Where a tile's keys and values lie in the ring, `t` counting all tiles of the block's share, and the round of their slots' barriers.  A barrier's
// parity cannot tell "two phases behind" from "done", so whoever waits for one of a barrier's phases waits for all of them, in their order, and none
// ends before all have seen the one before: a turn's product warp waits for the other turn's tiles too, and says so to their slots' barriers.
template <int SIZE> struct Turning {
    int at = 0, slot = 0;               // tiles passed; the next one's slot
    uint32_t round = 0;                 // ... and the round of its barriers, 0 and 1 by turns
    __device__ __forceinline__ void step() {
        ++at;
        if (++slot == SIZE) {
            slot = 0;
            round ^= 1;
        }
    }
};

// 32 rows of D values, the 32 rows-th of their block (64 columns every `block` bytes), by a warp with a row's start in each lane; zeros for none
template <int D> __device__ __forceinline__ void copy_rows(const TtArgs& a, unsigned char* dst, const bf16* mine, int rows, int block) {
    constexpr int CHUNKS = D / 8;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int e = 0; e < CHUNKS; ++e) {
        const int f = e * 32 + lane, r = f / CHUNKS, c = f % CHUNKS, row = rows * 32 + r;
        const bf16* p = (const bf16*)__shfl_sync(0xffffffffu, (unsigned long long)mine, r);
        cp_async16(dst + (c >> 3) * block + row * 128 + (((c & 7) ^ (row & 7)) << 4), p ? p + c * 8 : a.pages, p != nullptr);
    }
}

// The two loading warps: one brings keys, the other queries and values (a tile's values are used two tiles of its turn after its keys: when one
// warp brought both, values held their slots for that long beforehand and keys came late, 112 instead of 89 us for 32 trees of 4-24 rows
// behind 300-6000 positions with heads of 128).  A warp's chain of instructions for a tile is some 700 cycles, so each does its own walk and nothing else.
template <int D, typename Shape, bool VALUES>
__device__ __forceinline__ void load_tiles(const TtArgs& a, const CUtensorMap* pages_map, Walk walk, const Pipe& pipe) {
    using Q = Queries<Shape::QS>;
    constexpr int BLOCK = Shape::BLOCK, SLOT = Shape::SLOT, SIZE = VALUES ? Shape::VS : Shape::KS, CHUNKS = D / 8;
    const int lane = threadIdx.x & 31, group = a.group;
    unsigned char* ring = pipe.ring + (VALUES ? Shape::KS * SLOT : 0);
    uint64_t *full = pipe.full + (VALUES ? Shape::KS : 0), *empty = pipe.empty + (VALUES ? Shape::KS : 0);
    volatile int* failed = pipe.failed;
    const int box = min(a.page_size, TT_KEYS), boxes = TT_KEYS / box;
    Segment g;
    int count = 0, seg = 0, use = 0;                        // tiles begun, segments, halves of queries
    bool ok = true;
    while (ok && walk.next(a, g)) {
        // the queries, as many segments ahead as there is room for, so that a unit's first scores need not wait for them
        for (int h = 0; VALUES && h < (g.dual() ? 2 : 1) && ok; ++h, ++use) {
            const int slot = Q::slot(use);
            ok = at_mbar_wait_warp(&pipe.q_empty[slot], Q::round(use) ^ 1, failed);
            if (!ok) break;
#pragma unroll
            for (int rows = 0; rows < TT_TILE / 32; ++rows) {
                const int r = h * TT_TILE + rows * 32 + lane, p = g.pair0 + r;
                copy_rows<D>(a, pipe.q + slot * Shape::QSLOT,
                             r < g.pairs ? a.q + (long long)(g.first + p / group) * a.q_stride + (g.head * group + p % group) * D : nullptr, rows, Shape::QBLOCK);
            }
            tt_arrive_landed(&pipe.q_full[slot]);
        }
        const int* table = a.table + (size_t)g.s * a.table_width;
        const int whole = g.ctx / TT_KEYS, used = (g.ctx + a.page_size - 1) >> a.page_shift;
        // entries of the block table, 32 at a time, one a lane; the next 32 are asked for when these come to use
        auto ask = [&](int first) { return first + lane < used && first + lane < a.table_width ? table[first + lane] : -1; };
        int entries0 = ((g.from * TT_KEYS) >> a.page_shift) & ~31, entries = ask(entries0), next = ask(entries0 + 32);
        auto entry = [&](int idx, bool needed) {            // the page at a lane's own idx of these
            const int page = __shfl_sync(0xffffffffu, entries, idx & 31);
            if ((unsigned)page < (unsigned)a.num_pages) return page;
            if (needed) zai_raise(a.status, ZAI_ST_PAGE);
            return 0;
        };
        for (int tile = g.from; tile < g.upto; ++tile, ++count) {
            const int slot = count % SIZE;
            unsigned char* dst = ring + (size_t)slot * SLOT;
            if ((tile * TT_KEYS) >> a.page_shift >= entries0 + 32) {
                entries0 += 32;
                entries = next;
                next = ask(entries0 + 32);
            }
            if (tile < whole) {                             // a lane a page
                const int at = tile * TT_KEYS + lane * box, page = entry(at >> a.page_shift, lane < boxes);
                ok = at_mbar_wait_warp(&empty[slot], (count / SIZE & 1) ^ 1, failed);
                if (!ok) break;
                if (lane == 0) {                            // (all of the barrier's 32 arrivals)
                    at_mbar_expect_tx(&full[slot], SLOT);
                    tt_arrive(&full[slot], 31);
                }
                __syncwarp();
                if (lane < boxes) {
                    const int row = ((page * 2 + (VALUES ? 1 : 0)) * a.G + g.head) * a.page_size + (at & (a.page_size - 1));
#pragma unroll
                    for (int c = 0; c < D / 64; ++c) at_tma_load_2d(dst + c * BLOCK + lane * box * 128, pages_map, c * 64, row, &full[slot]);
                }
                continue;
            }
            // a tile that ends inside a page, or of drafted rows: by cp.async, a row's start in each lane, zeros for what is not there
            const bool drafted = tile >= g.cached;
            const bf16* from[2];
            bool bad = false;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int at = u * 32 + lane;
                from[u] = nullptr;
                if (drafted) {
                    const int node = (tile - g.cached) * TT_KEYS + at;
                    if (node < g.n) from[u] = (VALUES ? a.v + (long long)(g.first + node) * a.v_stride : a.k + (long long)(g.first + node) * a.k_stride) + g.head * D;
                } else {
                    const int key = tile * TT_KEYS + at, page = entry(min(key, g.ctx - 1) >> a.page_shift, key < g.ctx);
                    if (key < g.ctx) from[u] = a.pages + ((((long long)page * 2 + (VALUES ? 1 : 0)) * a.G + g.head) * a.page_size + (key & (a.page_size - 1))) * D;
                }
            }
            ok = at_mbar_wait_warp(&empty[slot], (count / SIZE & 1) ^ 1, failed);
            if (!ok) break;
#pragma unroll
            for (int u = 0; u < 2; ++u) copy_rows<D>(a, dst, from[u], u, BLOCK);
            if (VALUES && drafted)                          // is one of the drafted values not finite?  (A look of its own at memory: to wait for the copies
#pragma unroll
                for (int u = 0; u < 2; ++u) {               // would hold up the next unit's)
                    if (!from[u]) continue;
                    uint4 x[CHUNKS];
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c) x[c] = *reinterpret_cast<const uint4*>(from[u] + c * 8);
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c) bad |= at_not_finite(x[c]);
                }
            if (VALUES && __any_sync(0xffffffffu, bad)) {   // zeros in their place (what a row sees is put right at its end)
                cp_async_wait_all();
                for (int e = 0; e < 2 * CHUNKS; ++e) {
                    const int f = e * 32 + lane, key = f / CHUNKS, c = f % CHUNKS;
                    unsigned char* at = dst + (c >> 3) * BLOCK + key * 128 + (((c & 7) ^ (key & 7)) << 4);
                    if (at_not_finite(*reinterpret_cast<const uint4*>(at))) {
                        pipe.odd[seg & 15] = (seg & 0xff) + 1;
                        unsigned short* v = reinterpret_cast<unsigned short*>(at);
                        for (int u = 0; u < 8; ++u)
                            if ((v[u] & 0x7f80) == 0x7f80) v[u] = 0;
                    }
                }
                at_proxy_fence();
                at_mbar_arrive(&full[slot]);
            } else tt_arrive_landed(&full[slot]);
        }
        ++seg;
    }
    cp_async_wait_all();
    if (!ok && lane < SIZE)                                 // a wait ran out: the copies still on their way are waited for, with a limit, before the block ends
        for (int t = max(count - SIZE, 0); t < count; ++t)
            if (t % SIZE == lane)
                for (int spin = 0; spin < AT_SPIN_LIMIT && !at_mbar_test(&full[lane], (t / SIZE) & 1); ++spin) {}
}

template <int D> struct TtShape {
    static constexpr int BLOCK = TT_KEYS * 128;                 // 64 columns of a tile's keys or values, a swizzled row of 128 bytes each
    static constexpr int SLOT = D / 64 * BLOCK;
    static constexpr int QBLOCK = TT_TILE * 128, QSLOT = D / 64 * QBLOCK;     // ... of 128 pairs' queries
    static constexpr int KS = 20 / (D / 64) / 2, VS = KS, SLOTS = KS + VS, QS = D == 128 ? 2 : 4;
    static_assert(KS >= 4 && VS >= 4, "two tiles are brought at once, and scores run two of a turn's tiles ahead of their products");
    static constexpr int ALLOC = 512;                           // TMEM: 256 columns for four score buffers, two O
    static constexpr size_t TILES = (size_t)QS * QSLOT + (size_t)SLOTS * SLOT;
    static constexpr size_t SMEM = TILES + sizeof(float) * 4 * TT_TILE + 8 * (2 * SLOTS + 10 + 2 * QS + 2 + 3) + 4 * 20;
};

template <int D>
__global__ void __launch_bounds__(TT_THREADS, 1) tree_attention_tc_kernel(const __grid_constant__ CUtensorMap pages_map, const TtArgs a) {
    using Shape = TtShape<D>;
    using Q = Queries<Shape::QS>;
    constexpr int SLOT = Shape::SLOT, SLOTS = Shape::SLOTS, QS = Shape::QS;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* sQ = smem_raw;                               // [QS][QSLOT]
    unsigned char* ring = smem_raw + QS * Shape::QSLOT;                 // [SLOTS][SLOT]
    float* exch = reinterpret_cast<float*>(smem_raw + Shape::TILES);   // [2][2][128]: maxima, then sums, by turn
    uint64_t* full = reinterpret_cast<uint64_t*>(exch + 4 * TT_TILE);  // [SLOTS]
    uint64_t* empty = full + SLOTS;                             // [SLOTS]
    uint64_t* s_ready = empty + SLOTS;                          // [2][2] a turn's scores, of its even and odd tiles
    uint64_t* p_ready = s_ready + 4;                            // [2][2] ... P
    uint64_t* o_done = p_ready + 4;                             // [2] a turn's last product is in O
    uint64_t* q_full = o_done + 2;                              // [QS] queries of 128 pairs
    uint64_t* q_empty = q_full + QS;                            // [QS] ... their last scores are made
    uint64_t* o_full = q_empty + QS;                            // a segment's last products are in O
    uint64_t* o_empty = o_full + 1;                             // ... and have been read
    long long* share = reinterpret_cast<long long*>(o_empty + 1);      // the block's walk: pos, end, base
    int* words = reinterpret_cast<int*>(share + 3);
    uint32_t& tmem_holder = reinterpret_cast<uint32_t*>(words)[0];
    int& failed_flag = words[1];
    int& s_first = words[2];
    volatile int* odd = words + 4;                              // [16] by segment: its number (8 bits) + 1 if a drafted value is not finite
    volatile int* failed = &failed_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = a.group;

    if (tid == 0) {
        failed_flag = (at_smem(sQ) & 1023u) ? 1 : 0;            // the swizzled tiles need 1024-byte alignment
        for (int i = 0; i < SLOTS; ++i) {
            at_mbar_init(&full[i], 32);
            at_mbar_init(&empty[i], 2);
        }
        for (int i = 0; i < 4; ++i) {
            at_mbar_init(&s_ready[i], 1);
            at_mbar_init(&p_ready[i], 4);
            if (i < 2) at_mbar_init(&o_done[i], 1);
        }
        for (int i = 0; i < QS; ++i) {
            at_mbar_init(&q_full[i], 32);
            at_mbar_init(&q_empty[i], 2);
        }
        at_mbar_init(o_full, 2);
        at_mbar_init(o_empty, TT_SOFTMAX);
        for (int i = 0; i < 16; ++i) odd[i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == TT_SOFTMAX + TT_LOADERS) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(at_smem(&tmem_holder)), "r"(Shape::ALLOC) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_trigger();
    pdl_wait();
    if (warp == 0) begin_walk(a, D, share, &s_first);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_holder;
    Walk walk = {share[0], share[1], share[2], s_first, false, {}, {}};
    Segment g;

    if (failed_flag) {
        // (nothing to wait for)
    } else if (warp >= TT_SOFTMAX && warp < TT_SOFTMAX + TT_LOADERS) {
        const Pipe pipe = {sQ, ring, full, empty, q_full, q_empty, odd, failed};
        if (warp == TT_SOFTMAX) load_tiles<D, Shape, false>(a, &pages_map, walk, pipe);
        else load_tiles<D, Shape, true>(a, &pages_map, walk, pipe);
    } else if (warp >= TT_SOFTMAX + TT_LOADERS) {
        if (zai_elect()) {
            // ---- products, a warp a turn: while one tile is in the softmax, the other's P is multiplied and its buffer gets the scores after next.
            // Instruction descriptors: D 32-bit, A and B bfloat16, M = 128; the scores have both operands K-major, O has P in TMEM and V MN-major,
            // blocks of 64 columns.
            constexpr uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(TT_KEYS >> 3) << 17) | ((uint32_t)(TT_TILE >> 4) << 24);
            constexpr uint32_t idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(TT_TILE >> 4) << 24);
            constexpr uint64_t V_BLOCKS = (uint64_t)(Shape::BLOCK / 16 - 1) << 16;     // from 64 columns of V to the next (at_desc's field holds 1)
            const int turn = warp - TT_SOFTMAX - TT_LOADERS;
            const uint32_t tS = tmem + turn * 128, tO = tmem + 256 + turn * D;
            const uint64_t dQ = at_desc(at_smem(sQ)), dR = at_desc(at_smem(ring));     // (an address is a field of 14 bits, in 16 bytes: offsets are added)
            int count = 0, seg = 0, made = 0, use = 0;          // tiles before the segment; the turn's tiles before it; halves of queries
            Turning<Shape::KS> keys;                            // tiles whose keys, and whose values, have been waited for
            Turning<Shape::VS> values;
            bool ok = true;
            while (ok && walk.next(a, g)) {
                const bool dual = g.dual();
                const int tiles = g.upto - g.from, t0 = dual ? 0 : turn, step = dual ? 1 : 2, jobs = t0 < tiles ? (tiles - t0 + step - 1) / step : 0;
                const int q_slot = Q::slot(use + (dual ? turn : 0));
                const uint64_t q0 = dQ + q_slot * (Shape::QSLOT / 16);
                // waits for the tiles up to t (or takes note of those that are there); a slot is free when both turns are done with it
                auto see = [&](auto& ring_at, int base, int t, bool wait) {
                    while (ring_at.at <= t && ok) {
                        const int slot = base + ring_at.slot;
                        if (wait) ok = at_mbar_wait(&full[slot], ring_at.round, failed);
                        else if (!at_mbar_test(&full[slot], ring_at.round)) return;
                        if (!dual && ((ring_at.at - count) & 1) != turn) at_mbar_arrive(&empty[slot]);
                        ring_at.step();
                    }
                };
                // (the last tile seen is the one that was asked for)
                auto slot_seen = [](const auto& ring_at, int size) { return ring_at.slot ? ring_at.slot - 1 : size - 1; };
                auto scores = [&](int j, int slot) {
                    const int buffer = (made + j) & 1;
                    const uint64_t k0 = dR + slot * (SLOT / 16);
#pragma unroll
                    for (int c = 0; c < D / 16; ++c)
                        at_umma(tS + buffer * 64, q0 + ((c >> 2) * Shape::QBLOCK + (c & 3) * 32) / 16, k0 + ((c >> 2) * Shape::BLOCK + (c & 3) * 32) / 16, idesc_s,
                                c > 0 ? 1u : 0u);
                    at_commit(&s_ready[turn * 2 + buffer]);
                    at_commit(&empty[slot]);
                    if (j == jobs - 1) at_commit(&q_empty[q_slot]);
                };
                for (int h = 0; h < (dual ? 2 : 1) && ok; ++h) {
                    ok = at_mbar_wait(&q_full[Q::slot(use + h)], Q::round(use + h), failed);
                    if (dual && h != turn) at_mbar_arrive(&q_empty[Q::slot(use + h)]);
                }
                if (jobs == 0) at_mbar_arrive(&q_empty[q_slot]);
                else {
                    for (int j = 0; j < min(jobs, 2) && ok; ++j) {
                        see(keys, 0, count + t0 + j * step, true);
                        if (!ok) break;
                        at_proxy_fence();                       // (copies by cp.async are generic writes, which the products read)
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        scores(j, slot_seen(keys, Shape::KS));
                    }
                }
                if (ok && seg > 0) ok = at_mbar_wait(o_empty, (seg - 1) & 1, failed);
                for (int j = 0; j < jobs && ok; ++j) {
                    // (P last: what follows it is the softmax's wait for its next scores)
                    const int buffer = (made + j) & 1, after = count + t0 + (j + 2) * step;
                    see(values, Shape::KS, count + t0 + j * step, true);
                    const int slot = Shape::KS + slot_seen(values, Shape::VS);
                    if (j + 2 < jobs) see(keys, 0, after, false);
                    at_proxy_fence();
                    if (ok) ok = at_mbar_wait(&p_ready[turn * 2 + buffer], ((made + j) >> 1) & 1, failed);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t v0 = dR + V_BLOCKS + slot * (SLOT / 16);
#pragma unroll
                    for (int kk = 0; kk < TT_KEYS / 16; ++kk)   // 16 keys a step: eight columns of P, two groups of 8 keys of V
                        at_umma_ts(tO, tS + buffer * 64 + kk * 8, v0 + kk * (2048 / 16), idesc_o, (j > 0 || kk > 0) ? 1u : 0u);
                    at_commit(&o_done[turn]);
                    at_commit(&empty[slot]);
                    if (j + 2 < jobs) {
                        if (keys.at <= after) {
                            see(keys, 0, after, true);
                            if (!ok) break;
                            at_proxy_fence();
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        }
                        scores(j + 2, slot_seen(keys, Shape::KS));
                    }
                }
                if (ok) at_commit(o_full);
                see(keys, 0, count + tiles - 1, true);
                see(values, Shape::KS, count + tiles - 1, true);
                made += jobs;
                count += tiles;
                use += dual ? 2 : 1;
                ++seg;
            }
            if (!ok) *failed = 1;
        }
        __syncwarp();
    } else if (warp < TT_SOFTMAX) {
        // ---- softmax: a pair a thread
        const int turn = warp >> 2, qd = warp & 3, row = qd * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(qd * 32) << 16), tS = lanes + turn * 128, tO = lanes + 256 + turn * D;
        const float c = a.scale * TT_LOG2E;
        int seg = 0, taken = 0;                                 // segments, the turn's tiles so far
        bool ok = true;                                         // (a warp that gives up still meets the others at their barriers)
        while (walk.next(a, g)) {
            const bool dual = g.dual();
            const int pair = dual ? turn * TT_TILE + row : row, p = g.pair0 + pair, node = p / group;
            const bool valid = pair < g.pairs, idle = __all_sync(0xffffffffu, !valid);
            float m = -INFINITY, l = 0.f;
            bool begun = false;
            // how many tiles the two warps take turns at: as many for one as for the other
            const bool paired = !idle && (!dual || TT_TILE + qd * 32 < g.pairs);
            int left = paired ? (dual ? g.upto - g.from : (g.upto - g.from + 1) >> 1) : 0;
            if (paired && turn == 1) TT_ARRIVE(qd);
            for (int tile = g.from + (dual ? 0 : turn); tile < g.upto && ok; tile += dual ? 1 : 2, ++taken) {
                const int buffer = taken & 1;
                const uint32_t tB = tS + buffer * 64;
                ok = at_mbar_wait_warp(&s_ready[turn * 2 + buffer], (taken >> 1) & 1, failed);
                if (!ok) break;
                if (idle) {                                     // (its lanes of P and O are nobody's)
                    if (lane == 0) at_mbar_arrive(&p_ready[turn * 2 + buffer]);
                    continue;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t x[2][32];
                at_tmem_ld32_nowait(tB, x[0]);
                at_tmem_ld32_nowait(tB + 32, x[1]);
                at_tmem_wait_ld(x[0]);
                at_tmem_wait_ld(x[1]);
                const bool nodes = tile >= g.cached;
                if (nodes || (tile + 1) * TT_KEYS > g.ctx)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {               // which of keys 32 i .. of the tile this pair sees
                        const int word = (tile - g.cached) * 2 + i, there = nodes ? g.n - 32 * word : g.ctx - tile * TT_KEYS - 32 * i;
                        uint32_t bits = there >= 32 ? 0xffffffffu : there <= 0 ? 0u : (1u << there) - 1;
                        if (nodes) bits &= valid && word < a.words ? a.mask[(size_t)(g.first + node) * a.words + word] : 0u;
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (!(bits >> j & 1)) x[i][j] = __float_as_uint(-INFINITY);
                    }
                float mx[8] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY};         // eight chains, not one of 64 links
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 32; j += 2)
                        mx[(j >> 1) & 7] = zai_max3(mx[(j >> 1) & 7], __uint_as_float(x[i][j]), __uint_as_float(x[i][j + 1]));
                // The reference is the first tile's maximum, and moves when a later one exceeds it by 2^8: a weight keeps its 8 bits whatever the
                // reference is.  They are rounded for the product, their sum is taken before, in 32 bits.  (The rounded ones' sum: 2.17e-3 instead
                // of 2.27e-3 from 64 bits for 32 trees, root mean square, and 2 to 6 us more; the rest is the rounding of the weights themselves and
                // of the result, 1.66e-3 together where the products are made in 32 bits.)
                const float most = zai_max3(zai_max3(mx[0], mx[1], mx[2]), zai_max3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7])) * c;
                const float top = !begun || m == -INFINITY ? most : most > m + 8.f ? most : m;
                if (begun && __any_sync(0xffffffffu, top != m)) {
                    // O with the turn's last product in it (those before it came ahead of these scores)
                    const float keep = m == -INFINITY ? 0.f : at_exp2(m - top);
                    l *= keep;
                    ok = at_mbar_wait_warp(&o_done[turn], (taken + 1) & 1, failed);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                    for (int d = 0; d < D; d += 16) {
                        uint32_t y[16];
                        tt_ld16_nowait(tO + d, y);
                        tt_wait_ld16(y);
#pragma unroll
                        for (int j = 0; j < 16; ++j) y[j] = __float_as_uint(__uint_as_float(y[j]) * keep);
                        at_tmem_st16(tO + d, y);
                    }
                }
                m = top;
                begun = true;
                if (paired) TT_SYNC(turn * 4 + qd);
                const float2 c2 = make_float2(c, c), minus = make_float2(m == -INFINITY ? 0.f : -m, m == -INFINITY ? 0.f : -m);
                float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                // P over its scores (they are in registers), two keys a column
                uint32_t pk[32];
#pragma unroll
                for (int j = 0; j < 64; j += 2) {
                    const float2 e = zai_fma2(make_float2(__uint_as_float(x[j >> 5][j & 31]), __uint_as_float(x[j >> 5][(j & 31) + 1])), c2, minus);
                    const float2 w2 = make_float2(at_exp2(e.x), at_exp2(e.y));
                    sums[(j >> 1) & 1] = zai_add2(sums[(j >> 1) & 1], w2);
                    pk[j >> 1] = pack_bf16(w2.x, w2.y);
                }
                at_tmem_st32(tB, pk);
                if (paired) {
                    --left;
                    if (turn == 0 || left > 0) TT_ARRIVE((turn ^ 1) * 4 + qd);
                }
                const float2 sum = zai_add2(sums[0], sums[1]);
                l += sum.x + sum.y;
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) at_mbar_arrive(&p_ready[turn * 2 + buffer]);
            }
            while (left > 0) {                                  // (a tile fewer, or given up)
                TT_SYNC(turn * 4 + qd);
                --left;
                if (turn == 0 || left > 0) TT_ARRIVE((turn ^ 1) * 4 + qd);
            }
            // ---- the unit's end, or the share's
            float f0 = 1.f, f1 = 0.f;
            if (!dual) {                                        // both turns' parts: each thread has half of the pair's columns
                exch[turn * TT_TILE + row] = m;
                exch[(2 + turn) * TT_TILE + row] = l;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                const float m0 = exch[row], m1 = exch[TT_TILE + row], l0 = exch[2 * TT_TILE + row], l1 = exch[3 * TT_TILE + row];
                asm volatile("bar.sync 1, 256;" ::: "memory");  // (read, before the next segment's are written)
                m = fmaxf(m0, m1);
                f0 = l0 == 0.f ? 0.f : at_exp2(m0 - m);
                f1 = l1 == 0.f ? 0.f : at_exp2(m1 - m);
                l = l0 * f0 + l1 * f1;
            }
            if (ok) ok = at_mbar_wait_warp(o_full, seg & 1, failed);
            if (!ok) {
                ++seg;
                continue;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const bool two = !dual && g.upto - g.from > 1, bad = odd[seg & 15] == (seg & 0xff) + 1;
            const int col0 = dual ? 0 : turn * (D / 2), cols = dual ? D : D / 2;
            const float inv = l == 0.f ? 0.f : 1.f / l;
            float* po = a.parts + (size_t)(2 * blockIdx.x + (g.from == 0 ? 1 : 0)) * (D * TT_UNIT);
            if (!g.whole() && (dual || turn == 0)) {
                float* ml = a.parts + (size_t)2 * gridDim.x * (D * TT_UNIT) + (size_t)(2 * blockIdx.x + (g.from == 0 ? 1 : 0)) * (2 * TT_UNIT);
                *reinterpret_cast<float2*>(ml + 2 * pair) = make_float2(m, l);
            }
            for (int d = col0; d < col0 + cols && !idle; d += 32) {
                uint32_t x[32], y[32];
                const uint32_t at = dual ? tO : lanes + 256;
                at_tmem_ld32_nowait(at + d, x);
                if (two) at_tmem_ld32_nowait(at + D + d, y);
                at_tmem_wait_ld(x);
                at_tmem_wait_ld(y);
                float (&o)[32] = reinterpret_cast<float(&)[32]>(x);
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    o[j] = f0 == 0.f ? 0.f : o[j] * f0;
                    if (two && f1 != 0.f) o[j] = fmaf(__uint_as_float(y[j]), f1, o[j]);
                }
                if (bad && valid)                               // drafted values that are not finite: NaN where the row sees one
                    for (int r = 0; r < g.n; ++r) {
                        if ((r >> 5) >= a.words || !(a.mask[(size_t)(g.first + node) * a.words + (r >> 5)] >> (r & 31) & 1u)) continue;
                        const bf16* v = a.v + (long long)(g.first + r) * a.v_stride + g.head * D + d;
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (!(fabsf(__bfloat162float(v[j])) < INFINITY)) o[j] = NAN;
                    }
                if (!valid) continue;
                if (g.whole()) {
                    bf16* dst = a.out + ((long long)(g.first + node) * a.H + g.head * group + p % group) * D + d;
#pragma unroll
                    for (int j = 0; j < 32; j += 8)
                        *reinterpret_cast<uint4*>(dst + j) = make_uint4(pack_bf16(o[j] * inv, o[j + 1] * inv), pack_bf16(o[j + 2] * inv, o[j + 3] * inv),
                                                                        pack_bf16(o[j + 4] * inv, o[j + 5] * inv), pack_bf16(o[j + 6] * inv, o[j + 7] * inv));
                } else {
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        *reinterpret_cast<float4*>(po + ((d + j) / 4 * TT_UNIT + pair) * 4) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) at_mbar_arrive(o_empty);
            ++seg;
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == TT_SOFTMAX + TT_LOADERS)                        // (the warp that has it allocated)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Shape::ALLOC) : "memory");
    if (tid == 0 && failed_flag) zai_raise(a.status, ZAI_ST_WAIT);
}


// ---- units that several blocks have parts of: a block (times the grid's y) for every border between two shares.  The blocks of the borders
// inside a unit share out its pairs and columns.
#define JOIN_THREADS 256
#define JOIN_AHEAD 8
template <int D>
__global__ void __launch_bounds__(JOIN_THREADS) tree_attention_join_kernel(const TtArgs a, int blocks) {
    pdl_trigger();
    pdl_wait();
    const int border = blockIdx.x + 1, group = a.group;
    const Cut cut = cuts_of(a, blocks, D)[border];
    if (cut.b1 < cut.b0) return;
    const size_t size = (size_t)TT_UNIT * D;
    const float* ml = a.parts + 2 * (size_t)blocks * size;
    const int parts = cut.b1 - cut.b0 + 1, quads = D / 4, elements = quads * cut.pairs;
    const int mine = (border - 1 - cut.b0) * gridDim.y + blockIdx.y, all = (cut.b1 - cut.b0) * gridDim.y;
    const int from = (int)((long long)elements * mine / all), upto = (int)((long long)elements * (mine + 1) / all);
    for (int e = from + (int)threadIdx.x; e < upto; e += JOIN_THREADS) {
        const int quad = e / cut.pairs, pair = e - quad * cut.pairs;
        float top = -INFINITY, sum = 0.f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = 0; i0 < parts; i0 += JOIN_AHEAD) {        // (asked for together: a trip to memory for each part was most of this kernel's time)
            float2 its[JOIN_AHEAD];
            float4 v[JOIN_AHEAD];
#pragma unroll
            for (int i = 0; i < JOIN_AHEAD; ++i) {
                its[i] = make_float2(0.f, 0.f);
                if (i0 + i < parts) {
                    const size_t slot = 2 * (size_t)(cut.b0 + i0 + i) + (i0 + i == 0 ? 1 : 0);
                    its[i] = *reinterpret_cast<const float2*>(ml + (slot * TT_UNIT + pair) * 2);
                    v[i] = *reinterpret_cast<const float4*>(a.parts + slot * size + (quad * TT_UNIT + pair) * 4);
                }
            }
#pragma unroll
            for (int i = 0; i < JOIN_AHEAD; ++i) {
                if (its[i].y == 0.f) continue;
                const float now = fmaxf(top, its[i].x), f = at_exp2(its[i].x - now), keep = sum == 0.f ? 0.f : at_exp2(top - now);
                sum = sum * keep + its[i].y * f;
                x = make_float4(x.x * keep + v[i].x * f, x.y * keep + v[i].y * f, x.z * keep + v[i].z * f, x.w * keep + v[i].w * f);
                top = now;
            }
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const int at = cut.pair0 + pair;
        uint2 y;
        y.x = pack_bf16(x.x * inv, x.y * inv);
        y.y = pack_bf16(x.z * inv, x.w * inv);
        *reinterpret_cast<uint2*>(a.out + ((long long)(cut.first + at / group) * a.H + cut.head * group + at % group) * D + quad * 4) = y;
    }
}

// ---------------------------------------------------------------------------------------------------- launching
template <int D> static int launch_tree_tc(TtArgs a, int blocks, cudaStream_t stream) {
    using Shape = TtShape<D>;
    static_assert(Shape::SMEM <= 227 * 1024, "the ring does not fit");
    CUtensorMap map;
    if (at_make_map(&map, a.pages, D, (cuuint64_t)a.num_pages * 2 * a.G * a.page_size, a.page_size < TT_KEYS ? a.page_size : TT_KEYS)) return ZAI_BAD_SIZE;
    a.dual_cost = D == 128 ? 1 : 2;
    a.unit_extra = TT_EXTRA;
    static unsigned long long done = 0;
    if (zai_first_on_device(&done)) cudaFuncSetAttribute(tree_attention_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape::SMEM);
    const int code = launch_pdl(tree_attention_tc_kernel<D>, dim3(blocks), dim3(TT_THREADS), Shape::SMEM, stream, map, a);
    if (code || blocks == 1) return code;
    return launch_pdl(tree_attention_join_kernel<D>, dim3(blocks - 1, D / 32), dim3(JOIN_THREADS), 0, stream, a, blocks);
}

// 1 if this kernel takes heads of D, and pages of this size and number: a power of two from 8 positions on, rows that 32 bits number.
ZAI_API int zai_tree_attention_tc_supports(int D, int page_size, int num_pages, int G) {
    if ((D != 64 && D != 128) || page_size < 8 || (page_size & (page_size - 1)) || num_pages < 1 || G < 1) return 0;
    return (long long)num_pages * 2 * G * page_size <= 0x7fffffffll && at_encode_tiled() != nullptr;
}
ZAI_API int zai_tree_attention_tc_rows() { return TT_ROWS; }
// Floats that a block leaves room for in `parts`.
ZAI_API int zai_tree_attention_tc_part(int D) { return 2 * TT_UNIT * (D + 2) + (int)(sizeof(Cut) / sizeof(float)); }

// bfloat16; everything starts on 16 bytes, spans have at most zai_tree_attention_tc_rows() rows (a longer one raises the status word);
// `blocks`: blocks of the grid, at most one an SM, each with zai_tree_attention_tc_part(D) floats of `parts`.
ZAI_API int zai_tree_attention_tc(void* out, const void* q, long long q_stride, const void* k, long long k_stride, const void* v, long long v_stride,
                                  const void* pages, const int* table, int table_width, const int* cu, const int* ctx, const int* mask, int words, int S,
                                  int N, int blocks, int page_size, int num_pages, int H, int G, int D, float scale, float* parts, int* status,
                                  cudaStream_t stream) {
    if (S < 1 || N < 1 || blocks < 1 || blocks > 65535 || !zai_tree_attention_tc_supports(D, page_size, num_pages, G) || H % G || words < 1 ||
        table_width < 1 || H / G > 0xffff)
        return ZAI_BAD_SIZE;
    if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)pages | (uintptr_t)out | (uintptr_t)parts) & 15) || ((q_stride | k_stride | v_stride) & 7))
        return ZAI_BAD_SIZE;
    int shift = 0;
    while ((1 << shift) < page_size) ++shift;
    const long long reach = (long long)table_width * page_size;
    const TtArgs a = {(bf16*)out, (const bf16*)q, (const bf16*)k, (const bf16*)v, (const bf16*)pages, q_stride, k_stride, v_stride, table, cu, ctx,
                      (const unsigned*)mask, table_width, words, S, N, page_size, shift, num_pages, H, G, H / G, 1, 0, reach > 0x3fffffffll ? 0x3fffffff : (int)reach, scale, parts, status};
    return D == 64 ? launch_tree_tc<64>(a, blocks, stream) : launch_tree_tc<128>(a, blocks, stream);
}
