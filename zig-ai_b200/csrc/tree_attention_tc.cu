// Attention of trees of drafted tokens on the 5th-generation tensor cores: the same sums as csrc/tree_attention.cu (which says what a row
// sees), bfloat16 heads of 64 and 128, no window.  Per unit, which is up to 256 (row, query head) pairs of one request and key/value head, and
// half a tile of 128 keys
//
//     S = Q K^T      tcgen05.mma, M = 128 pairs (TMEM lanes), N = 64 keys, both operands in shared memory
//     P = exp2(..)   a pair a thread, from TMEM and back into it over its scores, two bfloat16 a column
//     O += P V       tcgen05.mma, A in TMEM, V as it lies ([key][column], MN-major), N = the head's columns
//
// Eight softmax warps are two turns with scores, O, reference and sum of their own, and a warp each that issues their products: while one half
// is in the softmax, the other's P is multiplied and its buffer gets the scores after next.  A unit of more than 128 pairs has a turn for
// each half of its pairs, and each tile of keys serves both; a smaller one has its tiles by turns, and the two O are joined at its end.
//
// A tile's keys and its values take a slot each of a ring, laid out in the 128-byte swizzle that the products read.  Tiles of cached keys alone
// come by TMA, page by page; a unit's last two, which end inside a page or hold the drafted rows, by cp.async from four warps (rows at
// any 16-byte stride, zeros for keys that are not there).  Nothing is waited for there but a free slot: copies arrive at their barrier by
// themselves.
//
// The work is the list of all units' tiles, cut into equal shares for as many blocks as there are SMs: a block's share may begin and end
// inside a unit, whose parts then go to memory and are joined by a second kernel.  (Requests of a batch differ in length by a factor of
// twenty and more; with a block or a cluster a unit the longest decides.)
#include "attention_tc_helpers.cuh"
#include "mma_helpers.cuh"

#define TT_KEYS 128
#define TT_TILE 128                     // lanes of a product
#define TT_UNIT 256                     // pairs of a unit
#define TT_ROWS 128                     // rows of a tree: one tile of keys
#define TT_SOFTMAX 8
#define TT_LOADERS 2                    // (twelve warps leave a thread 168 registers; with four loaders, 128)
#define TT_SUB (TT_TILE / 32 / TT_LOADERS)      // groups of 32 rows of a tile that a loading warp copies
#define TT_THREADS (32 * (TT_SOFTMAX + TT_LOADERS + 2))
#define TT_LEAST 4                      // cost of a share: fewer blocks take part when there is less than this for each
#define TT_EXTRA 3                      // cost of a unit beside its tiles (its queries, first scores and end)
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
// tile for every 128 cached keys and one for the drafted rows.  With heads of 64 a tile that both turns work on costs twice what one of
// a turn alone does; with heads of 128, where the ring holds two tiles and a turn alone waits for the next, they cost the same.
struct Request { int first, n, ctx, tiles, row_units, last_cost; };
__device__ __forceinline__ int unit_cost(const TtArgs& a, int pairs) { return pairs > TT_TILE ? a.dual_cost : 1; }
__device__ __forceinline__ Request request_of(const TtArgs& a, int s, bool say) {
    Request r = {0, 0, 0, 0, 0, 0};
    r.first = a.cu[s];
    r.n = a.cu[s + 1] - r.first;
    r.ctx = max(a.ctx[s], 0);
    if (r.n <= 0) {
        r.n = 0;
        return r;
    }
    if (r.first < 0 || r.first + r.n > a.N) {
        if (say) zai_raise(a.status, ZAI_ST_ROWS);
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
    r.tiles = (r.ctx + TT_KEYS - 1) / TT_KEYS + 1;
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
    int s, first, n, ctx, pair0, pairs, head, tiles, from, upto;       // key tiles [from, upto) of the unit's `tiles`
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

// two 32-bit numbers in one instruction
__device__ __forceinline__ float2 tt_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(c)));
    return d;
}
__device__ __forceinline__ float2 tt_add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ float tt_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
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
// An arrival of this thread's at a barrier when its copies so far have landed
__device__ __forceinline__ void tt_arrive_landed(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(at_smem(bar)) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// (a loader's waits are long ones: it naps between its tries, whose instructions the softmax warps would miss)
__device__ __forceinline__ bool tt_wait_warp(uint64_t* bar, uint32_t parity, volatile int* failed) {
    return __all_sync(0xffffffffu, at_mbar_wait<AT_NAP_NS>(bar, parity, failed));
}
// What the loaders and the other warps share.
struct Pipe {
    unsigned char *q, *ring;
    uint64_t *full, *empty, *q_full, *q_empty;
    volatile int *odd, *failed;         // odd [4] by segment: its number (8 bits) + 1 if a drafted value is not finite
};

// Where a tile's keys and values lie in the ring, `t` counting all tiles of the block's share, and the round of their slots' barriers.  Keys and
// values have slots of their own, so that a slot's last tenant was waited for by the same warp that waits for the next: a barrier's parity
// cannot tell "two phases behind" from "done".  (With two turns' warps that wait for their own tiles alone, KS and VS are even.)
template <int KS, int VS> struct Ring {
    static constexpr int SLOTS = KS + VS;
    static __device__ __forceinline__ int k_slot(int t) { return t % KS; }
    static __device__ __forceinline__ int v_slot(int t) { return KS + t % VS; }
    static __device__ __forceinline__ uint32_t k_round(int t) { return (t / KS) & 1; }
    static __device__ __forceinline__ uint32_t v_round(int t) { return (t / VS) & 1; }
};

// The loading warps.  D: a head's columns; KS, VS: slots of the ring.
template <int D, int KS, int VS>
__device__ __forceinline__ void load_units(const TtArgs& a, const CUtensorMap* pages_map, Walk walk, const Pipe& pipe, int lw) {
    constexpr int BLOCK = TT_TILE * 128, SLOT = D / 64 * BLOCK, CHUNKS = D / 8;
    const int lane = threadIdx.x & 31, group = a.group;
    unsigned char *sQ = pipe.q, *ring = pipe.ring;
    uint64_t *full = pipe.full, *empty = pipe.empty, *q_full = pipe.q_full, *q_empty = pipe.q_empty;
    volatile int *odd = pipe.odd, *failed = pipe.failed;
    Segment g;
    using R = Ring<KS, VS>;
    int count = 0, seg = 0;                                 // tiles begun
    bool ok = true;
    auto copy_rows = [&](unsigned char* dst, const bf16* mine, int rows) {        // 32 rows of D values, the 32 rows-th of the tile, a row's start in each lane
#pragma unroll
        for (int e = 0; e < CHUNKS; ++e) {
            const int f = e * 32 + lane, r = f / CHUNKS, c = f % CHUNKS, row = rows * 32 + r;
            const bf16* p = (const bf16*)__shfl_sync(0xffffffffu, (unsigned long long)mine, r);
            cp_async16(dst + (c >> 3) * BLOCK + row * 128 + (((c & 7) ^ (row & 7)) << 4), p ? p + c * 8 : a.pages, p != nullptr);
        }
    };
    while (ok && walk.next(a, g)) {
        const int* table = a.table + (size_t)g.s * a.table_width;
        // The tiles that hold 128 cached keys: a lane's page of the tile is asked for a tile ahead.  The others: where this lane's key lies.
        const int whole = g.ctx / TT_KEYS, box = min(a.page_size, TT_KEYS), boxes = TT_KEYS / box;
        auto checked = [&](int page, int idx) {
            if ((unsigned)page < (unsigned)a.num_pages) return page;
            zai_raise(a.status, idx < a.table_width ? ZAI_ST_PAGE : ZAI_ST_POSITION);
            return 0;
        };
        auto ask = [&](int tile) {
            const int idx = (tile * TT_KEYS + lane * box) >> a.page_shift;
            return tile < whole && tile < g.upto && lane < boxes && idx < a.table_width ? table[idx] : -1;
        };
        auto find = [&](int tile, int rows, const bf16*& kp, const bf16*& vp) {
            const int node = rows * 32 + lane, key = tile * TT_KEYS + node;
            kp = vp = nullptr;
            if (tile == g.tiles - 1) {
                if (node < g.n) {
                    kp = a.k + (long long)(g.first + node) * a.k_stride + g.head * D;
                    vp = a.v + (long long)(g.first + node) * a.v_stride + g.head * D;
                }
            } else if (key < g.ctx) {
                const int idx = key >> a.page_shift, page = checked(idx < a.table_width ? table[idx] : -1, idx);
                kp = a.pages + (((long long)page * 2 * a.G + g.head) * a.page_size + (key & (a.page_size - 1))) * D;
                vp = kp + (long long)a.G * a.page_size * D;
            }
        };
        // the queries go to where the last unit's lie: its last scores come first, and keys and values need not wait for that
        bool have_q = false;
        auto queries = [&](bool wait) {
            const uint32_t parity = (seg & 1) ^ 1;
            if (wait) ok = tt_wait_warp(q_empty, parity, failed);
            else if (!__all_sync(0xffffffffu, at_mbar_test(q_empty, parity))) return;
            if (!ok) return;
            for (int h = 0; h < (g.dual() ? 2 : 1); ++h)
#pragma unroll
                for (int u = 0; u < TT_SUB; ++u) {
                    const int r = h * TT_TILE + (lw * TT_SUB + u) * 32 + lane, p = g.pair0 + r;
                    copy_rows(sQ + h * SLOT, r < g.pairs ? a.q + (long long)(g.first + p / group) * a.q_stride + (g.head * group + p % group) * D : nullptr, lw * TT_SUB + u);
                }
            tt_arrive_landed(q_full);
            have_q = true;
        };
        int page = ask(g.from), next = -1;
        const bf16 *kp[TT_SUB] = {}, *vp[TT_SUB] = {};
        for (int i = 0; i < 2 * (g.upto - g.from) && ok; count += i & 1, ++i) {
            const int slot = i & 1 ? R::v_slot(count) : R::k_slot(count), tile = g.from + (i >> 1);
            const uint32_t parity = (i & 1 ? R::v_round(count) : R::k_round(count)) ^ 1;
            if (!have_q) queries(i >= 2 * (KS < VS ? KS : VS) - 1);
            // (a slot that is in use may be one of this unit's own, which its queries free)
            if (ok && !have_q && !__all_sync(0xffffffffu, at_mbar_test(&empty[slot], parity))) queries(true);
            if (ok) ok = tt_wait_warp(&empty[slot], parity, failed);
            if (!ok) break;
            unsigned char* dst = ring + (size_t)slot * SLOT;
            if (tile < whole) {
                if (!(i & 1)) {
                    page = lane < boxes ? checked(page, (tile * TT_KEYS + lane * box) >> a.page_shift) : 0;
                    next = ask(tile + 1);
                }
                if (lw == 0) {                              // (the others' arrivals make up the barrier's count)
                    if (lane == 0) at_mbar_expect_tx(&full[slot], SLOT);
                    else at_mbar_arrive(&full[slot]);
                    __syncwarp();
                    if (lane < boxes) {                     // a lane a page
                        const int row = ((page * 2 + (i & 1)) * a.G + g.head) * a.page_size + ((tile * TT_KEYS + lane * box) & (a.page_size - 1));
#pragma unroll
                        for (int c = 0; c < D / 64; ++c)
                            at_tma_load_2d(dst + c * BLOCK + lane * box * 128, pages_map, c * 64, row, &full[slot]);
                    }
                } else at_mbar_arrive(&full[slot]);
                if (i & 1) page = next;
                continue;
            }
            if (!(i & 1)) {
#pragma unroll
                for (int u = 0; u < TT_SUB; ++u) {
                    find(tile, lw * TT_SUB + u, kp[u], vp[u]);
                    copy_rows(dst, kp[u], lw * TT_SUB + u);
                }
            } else {
                bool bad = false;                           // is one of this lane's values, drafted ones, not finite?  (A look at memory: to wait for the
#pragma unroll
                for (int u = 0; u < TT_SUB; ++u) {          // copies would hold up the next unit's)
                    copy_rows(dst, vp[u], lw * TT_SUB + u);
                    if (tile != g.tiles - 1 || !vp[u]) continue;
                    uint4 x[CHUNKS];
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c) x[c] = *reinterpret_cast<const uint4*>(vp[u] + c * 8);
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c) bad |= at_not_finite(x[c]);
                }
                if (__any_sync(0xffffffffu, bad)) {         // zeros in their place (what a row sees is put right at its end)
                    cp_async_wait_all();
                    bool mine = false;
                    __syncwarp();
                    for (int e = 0; e < CHUNKS * TT_SUB; ++e) {
                        const int f = e * 32 + lane, key = lw * TT_SUB * 32 + f / CHUNKS, c = f % CHUNKS;
                        unsigned char* at = dst + (c >> 3) * BLOCK + key * 128 + (((c & 7) ^ (key & 7)) << 4);
                        if (at_not_finite(*reinterpret_cast<const uint4*>(at))) {
                            mine = true;
                            unsigned short* v = reinterpret_cast<unsigned short*>(at);
                            for (int x = 0; x < 8; ++x)
                                if ((v[x] & 0x7f80) == 0x7f80) v[x] = 0;
                        }
                    }
                    if (mine) odd[seg & 3] = (seg & 0xff) + 1;
                    at_proxy_fence();
                    at_mbar_arrive(&full[slot]);
                    continue;
                }
            }
            tt_arrive_landed(&full[slot]);
        }
        if (ok && !have_q) queries(true);
        ++seg;
    }
    cp_async_wait_all();
    if (!ok && lw == 0)                                     // a wait ran out: the tiles still on their way are waited for, with a limit, before the block ends
        for (int t = max(count - (KS > VS ? KS : VS), 0); t <= count; ++t)
            for (int spin = 0; spin < AT_SPIN_LIMIT && !(at_mbar_test(&full[R::k_slot(t)], R::k_round(t)) && at_mbar_test(&full[R::v_slot(t)], R::v_round(t))); ++spin) {}
}

template <int D> struct TtShape {
    static constexpr int BLOCK = TT_TILE * 128;                 // 64 columns of 128 rows, a swizzled row of 128 bytes each
    static constexpr int SLOT = D / 64 * BLOCK;                 // a tile's keys or values, or 128 pairs of Q
    static constexpr int KS = D == 128 ? 2 : 6, VS = KS, SLOTS = KS + VS;
    static constexpr int COLS = 256 + 2 * D;                    // TMEM: two score buffers, two O
    static constexpr int ALLOC = 512;
    static constexpr size_t TILES = (size_t)(2 + SLOTS) * SLOT;
    static constexpr size_t SMEM = TILES + sizeof(float) * 4 * TT_TILE + 8 * (2 * SLOTS + 14 + 3) + 32;
};

template <int D>
__global__ void __launch_bounds__(TT_THREADS, 1) tree_attention_tc_kernel(const __grid_constant__ CUtensorMap pages_map, const TtArgs a) {
    using Shape = TtShape<D>;
    using R = Ring<Shape::KS, Shape::VS>;
    constexpr int SLOT = Shape::SLOT, SLOTS = Shape::SLOTS;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* sQ = smem_raw;                               // [2][SLOT]
    unsigned char* ring = smem_raw + 2 * SLOT;                  // [SLOTS][SLOT]
    float* exch = reinterpret_cast<float*>(smem_raw + Shape::TILES);   // [2][2][128]: maxima, then sums, by turn
    uint64_t* full = reinterpret_cast<uint64_t*>(exch + 4 * TT_TILE);  // [SLOTS]
    uint64_t* empty = full + SLOTS;                             // [SLOTS]
    uint64_t* s_ready = empty + SLOTS;                          // [2][2] a turn's scores, of the first and second half of a tile's keys
    uint64_t* p_ready = s_ready + 4;                            // [2][2] ... P
    uint64_t* o_done = p_ready + 4;                             // [2] a turn's last product is in O
    uint64_t* q_full = o_done + 2;                              // a segment's queries
    uint64_t* q_empty = q_full + 1;                             // ... its last scores are made
    uint64_t* o_full = q_empty + 1;                             // a segment's last products are in O
    uint64_t* o_empty = o_full + 1;                             // ... and have been read
    long long* share = reinterpret_cast<long long*>(o_empty + 1);      // the block's walk: pos, end, base
    int* words = reinterpret_cast<int*>(share + 3);
    uint32_t& tmem_holder = reinterpret_cast<uint32_t*>(words)[0];
    int& failed_flag = words[1];
    int& s_first = words[2];
    volatile int* odd = words + 4;                              // [4] by segment: its number (8 bits) + 1 if a drafted value is not finite
    volatile int* failed = &failed_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = a.group;

    if (tid == 0) {
        failed_flag = (at_smem(sQ) & 1023u) ? 1 : 0;            // the swizzled tiles need 1024-byte alignment
        for (int i = 0; i < SLOTS; ++i) {
            at_mbar_init(&full[i], 32 * TT_LOADERS);
            at_mbar_init(&empty[i], 2);
        }
        for (int i = 0; i < 4; ++i) {
            at_mbar_init(&s_ready[i], 1);
            at_mbar_init(&p_ready[i], 4);
            if (i < 2) at_mbar_init(&o_done[i], 1);
        }
        at_mbar_init(q_full, 32 * TT_LOADERS);
        at_mbar_init(q_empty, 2);
        at_mbar_init(o_full, 2);
        at_mbar_init(o_empty, TT_SOFTMAX);
        for (int i = 0; i < 4; ++i) odd[i] = 0;
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
        load_units<D, Shape::KS, Shape::VS>(a, &pages_map, walk, Pipe{sQ, ring, full, empty, q_full, q_empty, odd, failed}, warp - TT_SOFTMAX);
    } else if (warp >= TT_SOFTMAX + TT_LOADERS) {
        if (zai_elect()) {
            // ---- products, a warp a turn, half a tile's keys at a time: while one half is in the softmax, the other's P is multiplied and its buffer
            // gets the scores after next.  Instruction descriptors: D 32-bit, A and B bfloat16, M = 128; the scores have both operands K-major, O
            // has P in TMEM and V MN-major, blocks of 64 columns.
            constexpr uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(TT_KEYS / 2 >> 3) << 17) | ((uint32_t)(TT_TILE >> 4) << 24);
            constexpr uint32_t idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(TT_TILE >> 4) << 24);
            constexpr uint64_t V_BLOCKS = (uint64_t)(Shape::BLOCK / 16 - 1) << 16;     // from 64 columns of V to the next (at_desc's field holds 1)
            const int turn = warp - TT_SOFTMAX - TT_LOADERS;
            const uint32_t tS = tmem + turn * 128, tO = tmem + 256 + turn * D;
            int count = 0, seg = 0, made = 0;                   // tiles before the segment; the turn's tiles so far
            bool ok = true;
            while (ok && walk.next(a, g)) {
                const bool dual = g.dual();
                const int tiles = g.upto - g.from, t0 = dual ? 0 : turn, step = dual ? 1 : 2, jobs = t0 < tiles ? 2 * ((tiles - t0 + step - 1) / step) : 0;
                const uint32_t aQ = at_smem(sQ) + (dual ? turn * SLOT : 0);
                // what both turns have to say before a slot, the queries or O count as done, a turn that has no part in it says at once
                auto scores = [&](int j) {
                    const int t = t0 + (j >> 1) * step, half = j & 1, slot = R::k_slot(count + t);
                    if (!half) {
                        ok = at_mbar_wait(&full[slot], R::k_round(count + t), failed);
                        if (!ok) return;
                        at_proxy_fence();                       // (the copies are generic writes, which the products read)
                    }
                    const uint32_t aK = at_smem(ring + (size_t)slot * SLOT) + half * (TT_KEYS / 2 * 128);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                    for (int c = 0; c < D / 16; ++c)
                        at_umma(tS + half * 64, at_desc(aQ + (c >> 2) * Shape::BLOCK + (c & 3) * 32), at_desc(aK + (c >> 2) * Shape::BLOCK + (c & 3) * 32), idesc_s,
                                c > 0 ? 1u : 0u);
                    at_commit(&s_ready[turn * 2 + half]);
                    if (half) {
                        at_commit(&empty[slot]);
                        if (!dual) at_mbar_arrive(&empty[slot]);
                    }
                    if (j == jobs - 1) at_commit(q_empty);
                };
                auto product = [&](int j) {
                    const int t = t0 + (j >> 1) * step, half = j & 1, slot = R::v_slot(count + t);
                    if (!half) ok = at_mbar_wait(&full[slot], R::v_round(count + t), failed);
                    if (ok) ok = at_mbar_wait(&p_ready[turn * 2 + half], made & 1, failed);
                    if (!ok) return;
                    if (!half) at_proxy_fence();
                    const uint32_t aV = at_smem(ring + (size_t)slot * SLOT) + half * (TT_KEYS / 2 * 128);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                    for (int kk = 0; kk < TT_KEYS / 32; ++kk)   // 16 keys a step: eight columns of P, two groups of 8 keys of V
                        at_umma_ts(tO, tS + half * 64 + kk * 8, at_desc(aV + kk * 2048) + V_BLOCKS, idesc_o, (j > 0 || kk > 0) ? 1u : 0u);
                    at_commit(&o_done[turn]);
                    if (half) {
                        ++made;
                        at_commit(&empty[slot]);
                        if (!dual) at_mbar_arrive(&empty[slot]);
                    }
                };
                ok = at_mbar_wait(q_full, seg & 1, failed);
                if (jobs == 0) at_mbar_arrive(q_empty);
                else {
                    if (ok) scores(0);
                    if (ok) scores(1);
                }
                if (ok && seg > 0) ok = at_mbar_wait(o_empty, (seg - 1) & 1, failed);
                for (int j = 0; j < jobs && ok; ++j) {
                    product(j);
                    if (ok && j + 2 < jobs) scores(j + 2);
                }
                if (ok) at_commit(o_full);
                count += tiles;
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
        int seg = 0, taken = 0, jobs = 0;                       // the turn's tiles so far, and their halves
        bool ok = true;                                         // (a warp that gives up still meets the others at their barriers)
        while (walk.next(a, g)) {
            const bool dual = g.dual();
            const int pair = dual ? turn * TT_TILE + row : row, p = g.pair0 + pair, node = p / group;
            const bool valid = pair < g.pairs, idle = __all_sync(0xffffffffu, !valid);
            float m = -INFINITY, l = 0.f;
            int done = 0;
            for (int tile = g.from + (dual ? 0 : turn); tile < g.upto && ok; tile += dual ? 1 : 2, ++taken)
                for (int half = 0; half < 2; ++half, ++done) {
                    ok = at_mbar_wait_warp(&s_ready[turn * 2 + half], taken & 1, failed);
                    if (!ok) break;
                    if (idle) {                                 // (its lanes of P and O are nobody's)
                        ++jobs;
                        if (lane == 0) at_mbar_arrive(&p_ready[turn * 2 + half]);
                        continue;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    uint32_t x[2][32];
                    at_tmem_ld32_nowait(tS + half * 64, x[0]);
                    at_tmem_ld32_nowait(tS + half * 64 + 32, x[1]);
                    at_tmem_wait_ld(x[0]);
                    at_tmem_wait_ld(x[1]);
                    const bool nodes = tile == g.tiles - 1;
                    if (nodes || (tile + 1) * TT_KEYS > g.ctx)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {           // which of keys 32 i .. of the half this pair sees
                            const int word = half * 2 + i, left = (nodes ? g.n : g.ctx - tile * TT_KEYS) - 32 * word;
                            uint32_t bits = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1;
                            if (nodes) bits &= valid && word < a.words ? a.mask[(size_t)(g.first + node) * a.words + word] : 0u;
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (!(bits >> j & 1)) x[i][j] = __float_as_uint(-INFINITY);
                        }
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};         // four chains, not one of 64 links
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int j = 0; j < 32; j += 2)
                                                        mx[(j >> 1) & 3] = tt_max3(mx[(j >> 1) & 3], __uint_as_float(x[i][j]), __uint_as_float(x[i][j + 1]));
                    // The reference is the first half's maximum, and moves when a later one exceeds it by 2^8: a weight keeps its 8 bits whatever the
                    // reference is, and the sum is that of the rounded weights, so what one key dominates stays exact.
                    const float most = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
                    const float top = done == 0 || m == -INFINITY ? most : most > m + 8.f ? most : m;
                    if (done > 0 && __any_sync(0xffffffffu, top != m)) {
                        // O with the turn's last product in it (those before it came ahead of these scores)
                        const float keep = m == -INFINITY ? 0.f : at_exp2(m - top);
                        l *= keep;
                        ok = at_mbar_wait_warp(&o_done[turn], (jobs + 1) & 1, failed);
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
                    ++jobs;
                    const float2 c2 = make_float2(c, c), minus = make_float2(m == -INFINITY ? 0.f : -m, m == -INFINITY ? 0.f : -m);
                    float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                    // P over its scores (they are in registers), two keys a column
                    uint32_t pk[32];
#pragma unroll
                    for (int j = 0; j < 64; j += 2) {
                        const float2 e = tt_fma2(make_float2(__uint_as_float(x[j >> 5][j & 31]), __uint_as_float(x[j >> 5][(j & 31) + 1])), c2, minus);
                        const uint32_t w = pack_bf16(at_exp2(e.x), at_exp2(e.y));
                        sums[(j >> 1) & 1] = tt_add2(sums[(j >> 1) & 1], make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)));
                        pk[j >> 1] = w;
                    }
                    at_tmem_st32(tS + half * 64, pk);
                    const float2 sum = tt_add2(sums[0], sums[1]);
                    l += sum.x + sum.y;
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) at_mbar_arrive(&p_ready[turn * 2 + half]);
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
            const bool two = !dual && g.upto - g.from > 1, bad = odd[seg & 3] == (seg & 0xff) + 1 && g.upto == g.tiles;
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
