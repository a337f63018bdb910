// Attention of trees of drafted tokens.  Row i of a request's span sees the request's cached positions 0..ctx-1 and those rows j of
// the span whose bit stands in its mask (its ancestors and itself, as a rule); with a window w > 0, of all these the ones whose position
// is above the row's minus w:
//
//     o[i, h] = sum_j p_j v_j,  p = softmax over what i sees of scale q[i, h] . k_j         (nothing seen: zeros)
//
// Cached keys and values lie in the request's pages; the span's own are rows of k and v and enter no page before they are accepted.
// A row's position is ctx plus its depth in the tree, so between ctx and ctx plus the span's rows.
//
// What bounds it: the cached keys and values, read once for all rows and query heads that share a key/value head.  So a tile of rows is
// (row, query head) pairs of one key/value head, up to 128 of them, and the keys of a request are split over a cluster of up to 16
// blocks whose parts are joined through distributed shared memory: no scratch in global memory, no counters, one launch, and an
// order of the sums that depends on the sizes alone.
//
// Two kernels: bfloat16 heads of 32, 64, 96 and 128 on mma.sync, and a general one in 32-bit arithmetic for everything else.  (Many pairs or long
// contexts in bfloat16 go to csrc/tree_attention_tc.cu.)  Measured: 12 rows of 16 heads over 8 of 64 behind 1000 positions 11.8 us in bfloat16,
// four trees of up to 21 rows with a window of 256 in 32 bits 18 us; both wait for a chain of launch, tables, pages, tiles and join.
#include <cooperative_groups.h>
#include "mma_helpers.cuh"
namespace cg = cooperative_groups;

#define MAX_SPLITS 16
#define LOG2E 1.4426950408889634f

struct TreeArgs {
    void* out;
    const void *q, *k, *v, *pages;
    long long q_stride, k_stride, v_stride;                    // in elements
    const int *table, *cu, *ctx, *positions;
    const unsigned* mask;
    int table_width, words, S, N, page_size, page_shift, num_pages, H, G, D, window;     // page_shift: of a page size that is a power of two, else -1
    int reach;                                                 // positions that a block table's row holds
    float scale;
    int* status;
};

// The rows of one tile: span `s` of the step from row `first` on, `n` rows, `ctx` cached positions; the tile's pairs start at `pair0` of
// the span's n * H / G.
struct Tile { int s, first, n, ctx, pair0; };

// The tile with this number when every span is cut into tiles of M pairs; all lanes of a warp.  s < 0: there is none.  `last`: no later number
// is asked for, so a tile behind this one is a row that nobody computes (a span longer than the launch was told).
__device__ __forceinline__ Tile find_tile(const TreeArgs& a, int number, int M, bool last) {
    const int lane = threadIdx.x & 31, group = a.H / a.G;
    Tile t = {-1, 0, 0, 0, 0};
    for (int at = 0; at < a.S; at += 32) {
        const int s = at + lane;
        int first = 0, n = 0;
        if (s < a.S) {
            first = a.cu[s];
            const int end = a.cu[s + 1];
            n = end - first;
            // (rows outside the step, or fewer than none: the span is passed over; rows before the first span or behind the last one, which
            // the last tile's block gets to see in any case: nobody computes them)
            if (first < 0 || end < first || end > a.N) n = 0;
            if (first < 0 || end < first || end > a.N || (s == 0 && first != 0) || (s == a.S - 1 && end != a.N)) zai_raise(a.status, ZAI_ST_ROWS);
        }
        const int tiles = n > 0 ? (n * group + M - 1) / M : 0;
        int upto = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        const unsigned here = __ballot_sync(0xffffffffu, number < upto);
        if (here) {
            if (t.s >= 0) {                                    // (only the last number gets here: there is a tile behind it)
                zai_raise(a.status, ZAI_ST_TREE);
                return t;
            }
            const int w = __ffs(here) - 1;
            t.s = at + w;
            t.first = __shfl_sync(0xffffffffu, first, w);
            t.n = __shfl_sync(0xffffffffu, n, w);
            t.pair0 = (number - __shfl_sync(0xffffffffu, upto - tiles, w)) * M;
            t.ctx = max(a.ctx[t.s], 0);
            if (t.ctx > a.reach) {                             // (what is beyond has no page)
                zai_raise(a.status, ZAI_ST_POSITION);
                t.ctx = a.reach;
            }
            if (!last) return t;
            if (__shfl_sync(0xffffffffu, upto, 31) > number + 1) {
                zai_raise(a.status, ZAI_ST_TREE);
                return t;
            }
            number = 0;                                        // the first tile of a later span would be this one
            continue;
        }
        number -= t.s >= 0 ? 0 : __shfl_sync(0xffffffffu, upto, 31);
    }
    return t;
}

// Does row `node` of the tile's span see row `other`?
__device__ __forceinline__ bool sees_node(const TreeArgs& a, const Tile& t, int node, int pos, int other) {
    if (other >= t.n || (other >> 5) >= a.words) return false;
    if (!(a.mask[(size_t)(t.first + node) * a.words + (other >> 5)] >> (other & 31) & 1u)) return false;
    return a.window <= 0 || a.positions[t.first + other] > pos - a.window;
}

// The page that position `key` lies in.
__device__ __forceinline__ int page_index(const TreeArgs& a, int key) { return a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size; }

// ---------------------------------------------------------------------------------------------------- the general kernel
// A block owns 16 pairs, a warp four of them; per tile of 32 keys a lane computes its key's scores with the warp's pairs, the weights go
// through shared memory, and the lanes share out the columns.  Keys and values are 32-bit numbers in shared memory.  What are 32-bit numbers
// in memory too, with rows on 16-byte boundaries, comes by cp.async up to two tiles ahead (ASYNC); the rest is converted on its way, eight
// loads in flight a thread.  A key's place is looked up by one thread, a tile before its copies are issued.  What bounds it at a few
// hundred keys: the chain of a tile, some 3.5 us (copies' arrival 1000 cycles, scores 2700, softmax 1300, sums 1250), so the keys are
// split over many blocks, 3 us of prologue and 2 of join each (the window above with one block a tile's keys 42 us, with four 18).
#define GEN_PAIRS 16
#define GEN_KEYS 32
#define GEN_THREADS 128

// The sum p * v of a tile's keys; GUARD: a key that has no weight stays out whatever its value is.
template <int COLS, bool GUARD>
__device__ __forceinline__ void add_values(float (&o)[4][COLS], const float* p, const float* v, int D, int D4, int lane) {
    for (int j = 0; j < GEN_KEYS; ++j) {
        const float4 w = *reinterpret_cast<const float4*>(p + 4 * j);
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
            const int d = lane + 32 * c;
            const float x = d < D ? v[j * D4 + d] : 0.f;
            if (!GUARD || w.x != 0.f) o[0][c] = fmaf(w.x, x, o[0][c]);
            if (!GUARD || w.y != 0.f) o[1][c] = fmaf(w.y, x, o[1][c]);
            if (!GUARD || w.z != 0.f) o[2][c] = fmaf(w.z, x, o[2][c]);
            if (!GUARD || w.w != 0.f) o[3][c] = fmaf(w.w, x, o[3][c]);
        }
    }
}

template <typename T, int COLS, bool ASYNC>
__global__ void __launch_bounds__(GEN_THREADS) tree_attention_general_kernel(const TreeArgs a, int splits, int stages) {
    extern __shared__ __align__(16) float sm[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, D = a.D, group = a.H / a.G, head = blockIdx.y, rank = blockIdx.x % splits;
    const int D4 = (D + 3) & ~3, KS = D4 + 4;                  // a key's row: four floats further than its length, so that lanes meet no bank twice
    const int stage = GEN_KEYS * (KS + D4);                    // a tile: keys [32][KS], values [32][D4]
    float* qs = sm;                                            // [16][D4]
    float* ring = qs + GEN_PAIRS * D4;                         // [stages][stage]
    float* ps = ring + stages * stage;                         // [4 warps][32 keys][4 pairs]
    float* ml = ps + GEN_PAIRS * GEN_KEYS;                     // [16][2]
    const T** where = reinterpret_cast<const T**>(ml + 2 * GEN_PAIRS);     // [4][32][key, value]
    pdl_trigger();
    pdl_wait();
    const Tile t = find_tile(a, blockIdx.x / splits, GEN_PAIRS, blockIdx.x / splits == gridDim.x / splits - 1);
    if (t.s < 0) return;                                       // (the whole cluster's)
    const int pairs = min(t.n * group - t.pair0, GEN_PAIRS);
    const int first_key = a.window > 0 ? max(t.ctx - a.window + 1, 0) : 0;
    const int tile0 = first_key / GEN_KEYS, cached = max((t.ctx + GEN_KEYS - 1) / GEN_KEYS - tile0, 0), total = cached + (t.n + GEN_KEYS - 1) / GEN_KEYS;
    const int from = (int)((long long)total * rank / splits), upto = (int)((long long)total * (rank + 1) / splits);
    const ZaiTableRow table = {a.table + (size_t)t.s * a.table_width, a.table_width, a.num_pages, a.status};

    auto look_up = [&](int it, int by) {                       // where tile `it`'s keys lie, by one warp
        if (warp != by || it >= upto) return;
        const T *kp = nullptr, *vp = nullptr;
        if (it >= cached) {
            const int key = (it - cached) * GEN_KEYS + lane;
            if (key < t.n) {
                kp = (const T*)a.k + (long long)(t.first + key) * a.k_stride + head * D;
                vp = (const T*)a.v + (long long)(t.first + key) * a.v_stride + head * D;
            }
        } else {
            const int key = (tile0 + it) * GEN_KEYS + lane;
            if (key < t.ctx && key >= first_key) {
                const int idx = page_index(a, key);
                kp = (const T*)a.pages + (((long long)table.page(idx) * 2 * a.G + head) * a.page_size + (key - idx * a.page_size)) * D;
                vp = kp + (long long)a.G * a.page_size * D;
            }
        }
        const T** w = where + ((it & 3) * GEN_KEYS + lane) * 2;
        w[0] = kp;
        w[1] = vp;
    };
    // (a thread's pieces of 16 bytes of a tile, 128 apart: one division for all)
    const int quads = D4 >> 2, key_at = threadIdx.x / quads, quad_at = threadIdx.x - key_at * quads, key_step = GEN_THREADS / quads;
    const int quad_step = GEN_THREADS - key_step * quads;
    // tile `it` into its stage; keys that are not there become zeros.  Returns whether a value is not finite (ASYNC: not known here).
    auto bring = [&](int it) {
        bool odd = false;
        if (it < upto) {
            float *ks = ring + (it % stages) * stage, *vs = ks + GEN_KEYS * KS;
            const T* const* w = where + (it & 3) * GEN_KEYS * 2;
            if (ASYNC) {
                for (int j = key_at, q = quad_at; j < GEN_KEYS;) {
                    const int c = q * 4;
                    const T *kp = w[2 * j], *vp = w[2 * j + 1];
                    cp_async16(ks + j * KS + c, kp ? (const void*)(kp + c) : a.pages, kp != nullptr);
                    cp_async16(vs + j * D4 + c, vp ? (const void*)(vp + c) : a.pages, vp != nullptr);
                    j += key_step;
                    q += quad_step;
                    if (q >= quads) {
                        q -= quads;
                        ++j;
                    }
                }
            } else {
                for (int e0 = threadIdx.x; e0 < GEN_KEYS * D; e0 += 4 * GEN_THREADS) {
                    float kx[4], vx[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int e = e0 + u * GEN_THREADS, j = e / D, c = e - j * D;
                        kx[u] = vx[u] = 0.f;
                        if (e < GEN_KEYS * D && w[2 * j]) {
                            kx[u] = to_float(w[2 * j][c]);
                            vx[u] = to_float(w[2 * j + 1][c]);
                        }
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int e = e0 + u * GEN_THREADS, j = e / D, c = e - j * D;
                        if (e >= GEN_KEYS * D) break;
                        ks[j * KS + c] = kx[u];
                        vs[j * D4 + c] = vx[u];
                        odd |= !(fabsf(vx[u]) < INFINITY);
                    }
                }
            }
        }
        if (ASYNC) cp_async_commit();
        return odd;
    };
    if (D4 != D)                                               // the columns behind a key's own: zeros in every stage (never ASYNC)
        for (int e = threadIdx.x; e < stages * GEN_KEYS * (D4 - D); e += GEN_THREADS) {
            const int j = e / (D4 - D), c = D + e - j * (D4 - D);
            ring[(j / GEN_KEYS) * stage + (j % GEN_KEYS) * KS + c] = 0.f;
        }
    float o[4][COLS], m[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < COLS; ++c) o[i][c] = 0.f;
    }
    const int ahead = ASYNC ? stages - 1 : 0;                  // tiles whose copies are on their way
    // (the first tiles at once, each by a warp, and the queries while their copies are on their way)
    for (int i = 0; i <= ahead; ++i) look_up(from + i, i);
    __syncthreads();
    for (int i = 0; i < ahead; ++i) bring(from + i);
    int node[4], pos[4];                                       // this warp's pairs; their queries
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = warp * 4 + i, p = t.pair0 + r, at = p / group;
        node[i] = r < pairs ? at : -1;
        pos[i] = r < pairs && a.window > 0 ? a.positions[t.first + at] : 0;
        const T* row = (const T*)a.q + (long long)(t.first + at) * a.q_stride + (head * group + p - at * group) * D;
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
            const int d = lane + 32 * c;
            if (d < D4) qs[r * D4 + d] = r < pairs && d < D ? to_float(row[d]) : 0.f;
        }
    }
    for (int it = from; it < upto; ++it) {
        const bool nodes = it >= cached;
        const int key0 = nodes ? (it - cached) * GEN_KEYS : (tile0 + it) * GEN_KEYS;
        const float *ks = ring + (it % stages) * stage, *vs = ks + GEN_KEYS * KS;
        bool odd = false;
        if (ASYNC) {
            if (stages == 3) cp_async_wait<1>();
            else cp_async_wait<0>();                           // (two stages: the only tile on its way)
            __syncthreads();                                   // (arrived, and the tile before has been used)
            bring(it + ahead);
            look_up(it + ahead + 1, GEN_THREADS / 32 - 1);
            if (nodes || (a.window > 0 && key0 <= t.ctx + t.n - 1 - a.window)) {        // tiles that some pair sees in part
                for (int e = lane; e < GEN_KEYS * D4; e += 32) odd |= !(fabsf(vs[e]) < INFINITY);
                odd = __any_sync(0xffffffffu, odd);
            }
        } else {
            __syncthreads();                                   // (looked up, and the tile before has been used)
            odd = bring(it);
            odd = __syncthreads_or(odd);
            look_up(it + 1, GEN_THREADS / 32 - 1);
        }
        // scores: this lane's key with the warp's pairs
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        const float* kr = ks + lane * KS;   // (its columns behind D are zeros)
        const float* qr = qs + warp * 4 * D4;
        for (int d = 0; d < D4; d += 4) {
            const float4 k4 = *reinterpret_cast<const float4*>(kr + d);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 q4 = *reinterpret_cast<const float4*>(qr + i * D4 + d);
                s[i] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[i]))));
            }
        }
        float4 w;
        float* wp = &w.x;
        const int key = key0 + lane;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool seen = node[i] >= 0 && (nodes ? sees_node(a, t, node[i], pos[i], key)
                                                     : key < t.ctx && (a.window <= 0 || key > pos[i] - a.window));
            const float x = seen ? s[i] * a.scale : -INFINITY;
            const float top = fmaxf(m[i], warp_max(x));
            const float keep = top == -INFINITY ? 1.f : fast_exp2((m[i] - top) * LOG2E);
            const float p = seen ? fast_exp2((x - top) * LOG2E) : 0.f;
            l[i] = l[i] * keep + p;                            // (a lane's own keys; added up at the end)
            m[i] = top;
            wp[i] = p;
#pragma unroll
            for (int c = 0; c < COLS; ++c) o[i][c] *= keep;
        }
        float* mine = ps + warp * GEN_KEYS * 4;
        __syncwarp();
        *reinterpret_cast<float4*>(mine + 4 * lane) = w;
        __syncwarp();
        if (odd) add_values<COLS, true>(o, mine, vs, D, D4, lane);
        else add_values<COLS, false>(o, mine, vs, D, D4, lane);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) l[i] = warp_sum(l[i]);
    T* out = (T*)a.out;
    if (splits == 1) {
        if (ASYNC) cp_async_wait<0>();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (node[i] < 0) continue;
            const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
            T* row = out + ((long long)(t.first + node[i]) * a.H + head * group + (t.pair0 + warp * 4 + i) % group) * D;
#pragma unroll
            for (int c = 0; c < COLS; ++c)
                if (lane + 32 * c < D) row[lane + 32 * c] = from_float<T>(l[i] == 0.f ? 0.f : o[i][c] * inv);
        }
        return;
    }
    // the blocks' parts: O in shared memory (over the tiles), references and sums behind it; every block joins some of the pairs
    if (ASYNC) cp_async_wait<0>();
    __syncthreads();
    float* po = ring;                                            // [16][D]
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = warp * 4 + i;
#pragma unroll
        for (int c = 0; c < COLS; ++c)
            if (lane + 32 * c < D) po[r * D + lane + 32 * c] = o[i][c];
        if (lane == 0) {
            ml[2 * r] = m[i];
            ml[2 * r + 1] = l[i];
        }
    }
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int r = rank + warp * splits; r < pairs; r += splits * (GEN_THREADS / 32)) {
        // (a lane a part: one after the other these trips to the other blocks' memory were most of the join)
        float2 its = make_float2(-INFINITY, 0.f);
        if (lane < splits) its = *reinterpret_cast<const float2*>(cluster.map_shared_rank(ml, lane) + 2 * r);
        const float top = warp_max(its.y == 0.f ? -INFINITY : its.x), mine = its.y == 0.f ? 0.f : fast_exp2((its.x - top) * LOG2E), sum = warp_sum(mine * its.y);
        float x[COLS];
#pragma unroll
        for (int c = 0; c < COLS; ++c) x[c] = 0.f;
        for (int i0 = 0; i0 < splits; i0 += 4) {
            float f[4], vals[4][COLS];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                f[u] = i0 + u < splits ? __shfl_sync(0xffffffffu, mine, i0 + u) : 0.f;
                const float* from_part = cluster.map_shared_rank(po, min(i0 + u, splits - 1)) + r * D;
#pragma unroll
                for (int c = 0; c < COLS; ++c) vals[u][c] = f[u] != 0.f && lane + 32 * c < D ? from_part[lane + 32 * c] : 0.f;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)                        // (a block that saw nothing of this pair adds 0 times 0)
#pragma unroll
                for (int c = 0; c < COLS; ++c) x[c] = fmaf(f[u], vals[u][c], x[c]);
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const int p = t.pair0 + r;
        T* row = out + ((long long)(t.first + p / group) * a.H + head * group + p % group) * D;
#pragma unroll
        for (int c = 0; c < COLS; ++c)
            if (lane + 32 * c < D) row[lane + 32 * c] = from_float<T>(sum == 0.f ? 0.f : x[c] * inv);
    }
    cluster.sync();                                            // (the parts have been read)
}

// ---------------------------------------------------------------------------------------------------- bfloat16 on mma.sync
// A block owns 16 WM pairs; its warps are WM rows of 16 pairs times WN shares of every tile of KEYS keys, each share with a maximum,
// a sum and an O of its own (joined with those of the cluster's other blocks at the end).  Keys and values come by cp.async, STAGES tiles
// in a ring; where a tile's keys (64, or 128 where a block has up to 32 pairs of heads of up to 64) lie is looked up a turn before its copies
// are issued, by one thread a key.  Q stays in registers, scores go from the accumulators into the second product's operand without leaving
// them.  Weights are rounded to bfloat16 there, as the values are; their sum is taken before the rounding, in 32 bits.  Shared memory decides
// how many blocks an SM holds: a tile's places take two entries, not four, because with four the second block did not fit (22 instead of
// 12 us for the tree above).

template <int D, int WM, int WN, int KEYS, int STAGES> struct MmaShape {
    static_assert(KEYS <= 32 * WM * WN && KEYS / WN % 16 == 0, "a thread a key looks up where it lies");
    static constexpr int THREADS = 32 * WM * WN, PAIRS = 16 * WM, ROW = D + 8, STAGE = 2 * KEYS * ROW, KW = KEYS / WN, O_ROW = D + 8;
    static constexpr size_t RING = sizeof(bf16) * STAGES * STAGE;
    static constexpr size_t JOIN = sizeof(float) * WN * PAIRS * O_ROW;
    static constexpr size_t SMEM = (RING > JOIN ? RING : JOIN) + sizeof(void*) * 4 * KEYS + sizeof(float) * 2 * WN * PAIRS;
};

template <int D, int WM, int WN, int KEYS, int STAGES>
__global__ void __launch_bounds__(32 * WM * WN) tree_attention_mma_kernel(const TreeArgs a, int splits) {
    using Shape = MmaShape<D, WM, WN, KEYS, STAGES>;
    constexpr int THREADS = Shape::THREADS, PAIRS = Shape::PAIRS, ROW = Shape::ROW, KW = Shape::KW, NT = KW / 8, O_ROW = Shape::O_ROW;
    constexpr int CHUNKS = D / 8;                              // pieces of 16 bytes a key
    extern __shared__ __align__(16) char smem[];
    bf16* ring = reinterpret_cast<bf16*>(smem);
    const bf16** where = reinterpret_cast<const bf16**>(smem + (Shape::RING > Shape::JOIN ? Shape::RING : Shape::JOIN));     // [2][KEYS][key, value]
    float* ml = reinterpret_cast<float*>(where + 4 * KEYS);    // [WN][PAIRS][2]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wm = warp % WM, wn = warp / WM, head = blockIdx.y, rank = blockIdx.x % splits;
    const int group = a.H / a.G, g = lane >> 2, q4 = lane & 3;
    pdl_trigger();
    pdl_wait();
    const Tile t = find_tile(a, blockIdx.x / splits, PAIRS, blockIdx.x / splits == gridDim.x / splits - 1);
    if (t.s < 0) return;                                       // (the whole cluster's)
    const int pairs = min(t.n * group - t.pair0, PAIRS);
    const int first_key = a.window > 0 ? max(t.ctx - a.window + 1, 0) : 0;
    const int tile0 = first_key / KEYS, cached = max((t.ctx + KEYS - 1) / KEYS - tile0, 0), total = cached + (t.n + KEYS - 1) / KEYS;
    const int from = (int)((long long)total * rank / splits), upto = (int)((long long)total * (rank + 1) / splits);
    const ZaiTableRow table = {a.table + (size_t)t.s * a.table_width, a.table_width, a.num_pages, a.status};

    auto look_up = [&](int it) {                               // where tile `it`'s keys lie, by the first KEYS threads
        const int j = threadIdx.x;                             // (there are at least as many threads)
        if (j >= KEYS || it >= upto) return;
        const bf16 *kp = nullptr, *vp = nullptr;
        if (it >= cached) {
            const int key = (it - cached) * KEYS + j;
            if (key < t.n) {
                kp = (const bf16*)a.k + (long long)(t.first + key) * a.k_stride + head * D;
                vp = (const bf16*)a.v + (long long)(t.first + key) * a.v_stride + head * D;
            }
        } else {
            const int key = (tile0 + it) * KEYS + j;
            if (key < t.ctx && key >= first_key) {
                const int idx = page_index(a, key);
                kp = (const bf16*)a.pages + (((long long)table.page(idx) * 2 * a.G + head) * a.page_size + (key - idx * a.page_size)) * D;
                vp = kp + (long long)a.G * a.page_size * D;
            }
        }
        const bf16** w = where + ((it & 1) * KEYS + j) * 2;
        w[0] = kp;
        w[1] = vp;
    };
    auto issue = [&](int it) {                                 // tile `it`'s copies; keys that are not there become zeros
        if (it < upto) {
            bf16* ks = ring + (it % STAGES) * Shape::STAGE;
#pragma unroll
            for (int e = threadIdx.x; e < KEYS * CHUNKS; e += THREADS) {
                const int j = e / CHUNKS, c = e - j * CHUNKS;
                const bf16* const* w = where + ((it & 1) * KEYS + j) * 2;
                const bf16 *kp = w[0], *vp = w[1];
                cp_async16(ks + j * ROW + c * 8, kp ? kp + c * 8 : (const bf16*)a.pages, kp != nullptr);
                cp_async16(ks + (KEYS + j) * ROW + c * 8, vp ? vp + c * 8 : (const bf16*)a.pages, vp != nullptr);
            }
        }
        cp_async_commit();
    };

    static_assert(STAGES == 3, "two tiles on their way, a place for each");
    // (the first tiles' places at once, and the queries while their copies are on their way)
    look_up(from);
    look_up(from + 1);
    __syncthreads();
    issue(from);
    issue(from + 1);
    // this lane's two pairs: g and g + 8 of the warp's 16
    int node[2], pos[2];
    uint32_t qf[D / 16][4];
    {
        const bf16* qr[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = wm * 16 + g + 8 * i, p = t.pair0 + r;
            node[i] = r < pairs ? p / group : -1;
            pos[i] = node[i] >= 0 && a.window > 0 ? a.positions[t.first + node[i]] : 0;
            qr[i] = node[i] >= 0 ? (const bf16*)a.q + (long long)(t.first + node[i]) * a.q_stride + (head * group + p % group) * D + 2 * q4 : nullptr;
        }
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                qf[kk][i] = qr[i & 1] ? *reinterpret_cast<const uint32_t*>(qr[i & 1] + kk * 16 + (i >> 1) * 8) : 0u;
    }
    const bool idle = wm * 16 >= pairs;                        // a warp without pairs brings keys in and computes nothing
    __syncthreads();                                           // (the first two have been read)
    look_up(from + 2);
    float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int d = 0; d < D / 8; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][e] = 0.f;
    const float scale = a.scale * LOG2E;
    for (int it = from; it < upto; ++it) {
        cp_async_wait<STAGES - 2>();
        __syncthreads();
        issue(it + STAGES - 1);
        look_up(it + STAGES);
        if (idle) continue;
        const bf16* ks = ring + (it % STAGES) * Shape::STAGE + wn * KW * ROW;
        const bf16* vs = ks + KEYS * ROW;
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
                uint32_t b[4];
                ldmatrix_x4(b, ks + (n * 8 + (lane & 7) + ((lane & 16) >> 1)) * ROW + kk * 16 + (lane & 8));
                mma_bf16(s[n], qf[kk], b[0], b[1]);
                mma_bf16(s[n + 1], qf[kk], b[2], b[3]);
            }
        const bool nodes = it >= cached;
        const int key0 = (nodes ? it - cached : tile0 + it) * KEYS;
        // every pair sees all keys of the tile?  (positions lie between ctx and ctx + n)
        const bool whole = !nodes && key0 + KEYS <= t.ctx && (a.window <= 0 || key0 > t.ctx + t.n - 1 - a.window);
        bool odd = false;
        if (!whole) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = e >> 1, key = key0 + wn * KW + n * 8 + 2 * q4 + (e & 1);
                    const bool seen = node[i] >= 0 && (nodes ? sees_node(a, t, node[i], pos[i], key)
                                                             : key < t.ctx && (a.window <= 0 || key > pos[i] - a.window));
                    if (!seen) s[n][e] = -INFINITY;
                }
            // values that are not finite: they must not reach the pairs that do not see them as 0 times NaN
            uint32_t bad = 0;
            for (int e = lane; e < KW * CHUNKS; e += 32) {
                const int j = e / CHUNKS;
                const uint4 x = *reinterpret_cast<const uint4*>(vs + j * ROW + (e - j * CHUNKS) * 8);
                bad |= not_finite_pair(x.x) | not_finite_pair(x.y) | not_finite_pair(x.z) | not_finite_pair(x.w);
            }
            odd = __any_sync(0xffffffffu, bad != 0);
        }
        // the running maximum, in units of the exponent
        float top[2] = {m[0], m[1]};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            top[0] = fmaxf(top[0], fmaxf(s[n][0], s[n][1]) * scale);
            top[1] = fmaxf(top[1], fmaxf(s[n][2], s[n][3]) * scale);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
        }
        if (__any_sync(0xffffffffu, top[0] != m[0] || top[1] != m[1])) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float keep = top[i] == -INFINITY ? 1.f : fast_exp2(m[i] - top[i]);
                m[i] = top[i];
                l[i] *= keep;
#pragma unroll
                for (int d = 0; d < D / 8; ++d) {
                    o[d][2 * i] *= keep;
                    o[d][2 * i + 1] *= keep;
                }
            }
        }
        // weights; a pair that has seen nothing yet takes 0 as its reference, so that masked scores weigh 0
        const float ref[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
        uint32_t pf[NT / 2][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                p[e] = fast_exp2(fmaf(s[n][e], scale, -ref[e >> 1]));
                l[e >> 1] += p[e];
            }
            pf[n / 2][(n & 1) * 2] = pack_bf16(p[0], p[1]);
            pf[n / 2][(n & 1) * 2 + 1] = pack_bf16(p[2], p[3]);
        }
        if (!odd) {
#pragma unroll
            for (int kk = 0; kk < NT / 2; ++kk)
#pragma unroll
                for (int d = 0; d < D / 8; d += 2) {
                    uint32_t b[4];
                    ldmatrix_x4_trans(b, vs + (kk * 16 + (lane & 15)) * ROW + d * 8 + ((lane & 16) >> 1));
                    mma_bf16(o[d], pf[kk], b[0], b[1]);
                    mma_bf16(o[d + 1], pf[kk], b[2], b[3]);
                }
        } else {
            // the product without what is not finite, and a count of how many such values a pair gives weight to: those columns become NaN
#pragma unroll
            for (int d = 0; d < D / 8; d += 2) {
                float hit[2][4] = {};
#pragma unroll
                for (int kk = 0; kk < NT / 2; ++kk) {
                    uint32_t b[4], f[4], w[4];
                    ldmatrix_x4_trans(b, vs + (kk * 16 + (lane & 15)) * ROW + d * 8 + ((lane & 16) >> 1));
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t mark = not_finite_pair(b[i]) >> 15;             // 1 in the low bit of each half
                        f[i] = mark * 0x3f80u;                                         // one
                        b[i] &= ~(mark * 0xffffu);
                        w[i] = ((pf[kk][i] & 0x7fffu) ? 0x3f80u : 0u) | ((pf[kk][i] & 0x7fff0000u) ? 0x3f800000u : 0u);
                    }
                    mma_bf16(o[d], pf[kk], b[0], b[1]);
                    mma_bf16(o[d + 1], pf[kk], b[2], b[3]);
                    mma_bf16(hit[0], w, f[0], f[1]);
                    mma_bf16(hit[1], w, f[2], f[3]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (hit[0][e] > 0.f) o[d][e] = NAN;
                    if (hit[1][e] > 0.f) o[d + 1][e] = NAN;
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    bf16* out = (bf16*)a.out;
    if (WN == 1 && splits == 1) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (node[i] < 0) continue;
            const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
            bf16* row = out + ((long long)(t.first + node[i]) * a.H + head * group + (t.pair0 + wm * 16 + g + 8 * i) % group) * D + 2 * q4;
#pragma unroll
            for (int d = 0; d < D / 8; ++d)
                *reinterpret_cast<uint32_t*>(row + d * 8) = pack_bf16(o[d][2 * i] * inv, o[d][2 * i + 1] * inv);
        }
        cp_async_wait<0>();
        return;
    }
    // the parts: WN of each block of the cluster, in shared memory over the ring; every block joins some of the pairs
    cp_async_wait<0>();
    __syncthreads();
    float* po = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = wn * PAIRS + wm * 16 + g + 8 * i;
#pragma unroll
        for (int d = 0; d < D / 8; ++d) *reinterpret_cast<float2*>(po + r * O_ROW + d * 8 + 2 * q4) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
        if (q4 == 0) {
            ml[2 * r] = m[i];
            ml[2 * r + 1] = l[i];
        }
    }
    cg::cluster_group cluster = cg::this_cluster();
    if (splits > 1) cluster.sync();
    else __syncthreads();
    constexpr int QUADS = D / 4;
    const int mine = (pairs - rank + splits - 1) / splits;     // pairs rank, rank + splits, ...
    for (int e = threadIdx.x; e < mine * QUADS; e += THREADS) {
        const int r = rank + (e / QUADS) * splits, c = (e % QUADS) * 4;
        float top = -INFINITY;
#pragma unroll 4
        for (int i = 0; i < splits * WN; ++i) {
            const float* theirs = splits > 1 ? cluster.map_shared_rank(ml, i / WN) : ml;
            top = fmaxf(top, theirs[2 * ((i % WN) * PAIRS + r)]);
        }
        float sum = 0.f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int i = 0; i < splits * WN; ++i) {
            const float* theirs = splits > 1 ? cluster.map_shared_rank(ml, i / WN) : ml;
            const float* vals = splits > 1 ? cluster.map_shared_rank(po, i / WN) : po;
            const int at = (i % WN) * PAIRS + r;
            const float2 its = *reinterpret_cast<const float2*>(theirs + 2 * at);
            const float4 v = *reinterpret_cast<const float4*>(vals + at * O_ROW + c);
            if (its.y == 0.f) continue;                        // (a part that saw nothing of this pair)
            const float f = fast_exp2(its.x - top);
            sum = fmaf(f, its.y, sum);
            x.x = fmaf(f, v.x, x.x);
            x.y = fmaf(f, v.y, x.y);
            x.z = fmaf(f, v.z, x.z);
            x.w = fmaf(f, v.w, x.w);
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const int p = t.pair0 + r;
        bf16* row = out + ((long long)(t.first + p / group) * a.H + head * group + p % group) * D + c;
        uint2 w;
        w.x = pack_bf16(x.x * inv, x.y * inv);
        w.y = pack_bf16(x.z * inv, x.w * inv);
        *reinterpret_cast<uint2*>(row) = w;
    }
    if (splits > 1) cluster.sync();                            // (the parts have been read)
}

// ---------------------------------------------------------------------------------------------------- launching
// Positions that a row of `table_width` pages holds; 2^30 at most, so that sums of positions and rows stay within 32 bits.
static int reach_of(int table_width, int page_size) {
    const long long n = (long long)table_width * page_size;
    return n > 0x3fffffffll ? 0x3fffffff : (int)n;
}
static int page_shift_of(int page_size) {
    int shift = 0;
    while ((1 << shift) < page_size) ++shift;
    return 1 << shift == page_size ? shift : -1;
}
template <typename... K, typename... Args>
static int launch_cluster(void (*kernel)(K...), unsigned long long* done, dim3 grid, int threads, size_t smem, int splits, cudaStream_t stream, Args... args) {
    if (zai_first_on_device(done)) {
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, kernel, K(args)...);
}

template <typename T, int COLS, bool ASYNC>
static int launch_general(const TreeArgs& a, int tiles, int splits, cudaStream_t stream) {
    static unsigned long long done = 0;
    const size_t D4 = (a.D + 3) & ~3, stage = sizeof(float) * GEN_KEYS * (2 * D4 + 4);
    const size_t rest = sizeof(float) * (GEN_PAIRS * D4 + GEN_PAIRS * GEN_KEYS + 2 * GEN_PAIRS) + sizeof(void*) * 8 * GEN_KEYS;
    const int stages = !ASYNC ? 1 : 3 * stage + rest <= 76 * 1024 ? 3 : 2;      // (three of heads of up to 64, or two of 128: two blocks an SM and more)
    if (stages * stage + rest > 227 * 1024) return ZAI_BAD_SIZE;
    return launch_cluster(tree_attention_general_kernel<T, COLS, ASYNC>, &done, dim3((unsigned)splits * tiles, a.G), GEN_THREADS, stages * stage + rest,
                          splits, stream, a, splits, stages);
}
template <typename T, bool ASYNC> static int launch_general_cols(const TreeArgs& a, int tiles, int splits, cudaStream_t stream) {
    if (a.D <= 32) return launch_general<T, 1, ASYNC>(a, tiles, splits, stream);
    if (a.D <= 64) return launch_general<T, 2, ASYNC>(a, tiles, splits, stream);
    if (a.D <= 128) return launch_general<T, 4, ASYNC>(a, tiles, splits, stream);
    if (a.D <= 256) return launch_general<T, 8, ASYNC>(a, tiles, splits, stream);
    return launch_general<T, 16, false>(a, tiles, splits, stream);
}

// Pairs of (row, query head) a block of the general kernel owns.
ZAI_API int zai_tree_attention_general_pairs() { return GEN_PAIRS; }

ZAI_API int zai_tree_attention_general(void* out, const void* q, long long q_stride, const void* k, long long k_stride, const void* v, long long v_stride,
                                       const void* pages, int dtype, const int* table, int table_width, const int* cu, const int* ctx, const int* positions,
                                       const int* mask, int words, int S, int N, int tiles, int splits, int page_size, int num_pages, int H, int G, int D,
                                       float scale, int window, int* status, cudaStream_t stream) {
    if (S < 1 || N < 1 || tiles < 1 || tiles > 0x7ffffff || splits < 1 || splits > MAX_SPLITS || page_size < 1 || num_pages < 1 || G < 1 || H % G || G > 65535 ||
        D < 1 || D > 512 || words < 1 || table_width < 1 || (long long)N * (H / G) > 0x3fffffff)
        return ZAI_BAD_SIZE;
    const TreeArgs a = {out, q, k, v, pages, q_stride, k_stride, v_stride, table, cu, ctx, positions, (const unsigned*)mask, table_width, words, S, N,
                        page_size, page_shift_of(page_size), num_pages, H, G, D, window, reach_of(table_width, page_size), scale, status};
    if (dtype == ZAI_BF16) return launch_general_cols<bf16, false>(a, tiles, splits, stream);
    if (dtype != ZAI_F32) return ZAI_BAD_DTYPE;
    const bool wide = !(((uintptr_t)k | (uintptr_t)v | (uintptr_t)pages) & 15) && !((k_stride | v_stride | D) & 3);
    return wide ? launch_general_cols<float, true>(a, tiles, splits, stream) : launch_general_cols<float, false>(a, tiles, splits, stream);
}

template <int D, int WM, int WN, int KEYS, int STAGES> static int launch_mma(const TreeArgs& a, int tiles, int splits, cudaStream_t stream) {
    using Shape = MmaShape<D, WM, WN, KEYS, STAGES>;
    static_assert(Shape::SMEM <= 227 * 1024, "the ring does not fit");
    static unsigned long long done = 0;
    return launch_cluster(tree_attention_mma_kernel<D, WM, WN, KEYS, STAGES>, &done, dim3((unsigned)splits * tiles, a.G), Shape::THREADS, Shape::SMEM, splits,
                          stream, a, splits);
}
template <int D> static int launch_mma_pairs(const TreeArgs& a, int pairs, int tiles, int splits, cudaStream_t stream) {
    constexpr int KEYS = D <= 64 ? 128 : 64;                   // of a tile where a block has few pairs: 16 KB of keys, two blocks an SM
    if (pairs == 16) return launch_mma<D, 1, 4, KEYS, 3>(a, tiles, splits, stream);
    if (pairs == 32) return launch_mma<D, 2, 2, KEYS, 3>(a, tiles, splits, stream);
    if (pairs == 64) return launch_mma<D, 4, 1, 64, 3>(a, tiles, splits, stream);
    if (pairs == 128) return launch_mma<D, 8, 1, 64, 3>(a, tiles, splits, stream);
    return ZAI_BAD_SIZE;
}

ZAI_API int zai_tree_attention_mma_supports(int D) { return D == 32 || D == 64 || D == 96 || D == 128; }

// bfloat16; `pairs` (16, 32, 64 or 128): pairs of (row, query head) a block owns.  q starts on 4 bytes and has even row strides; keys and values,
// of the pages and of the rows, start on 16 bytes.
ZAI_API int zai_tree_attention_mma(void* out, const void* q, long long q_stride, const void* k, long long k_stride, const void* v, long long v_stride,
                                   const void* pages, const int* table, int table_width, const int* cu, const int* ctx, const int* positions,
                                   const int* mask, int words, int S, int N, int pairs, int tiles, int splits, int page_size, int num_pages, int H, int G,
                                   int D, float scale, int window, int* status, cudaStream_t stream) {
    if (S < 1 || N < 1 || tiles < 1 || tiles > 0x7ffffff || splits < 1 || splits > MAX_SPLITS || page_size < 1 || num_pages < 1 || G < 1 || H % G ||
        G > 65535 || words < 1 || table_width < 1 || (long long)N * (H / G) > 0x3fffffff)
        return ZAI_BAD_SIZE;
    if ((((uintptr_t)k | (uintptr_t)v | (uintptr_t)pages) & 15) || ((k_stride | v_stride) & 7) || ((uintptr_t)q & 3) || (q_stride & 1) || ((uintptr_t)out & 7))
        return ZAI_BAD_SIZE;
    const TreeArgs a = {out, q, k, v, pages, q_stride, k_stride, v_stride, table, cu, ctx, positions, (const unsigned*)mask, table_width, words, S, N,
                        page_size, page_shift_of(page_size), num_pages, H, G, D, window, reach_of(table_width, page_size), scale, status};
    switch (D) {
        case 32: return launch_mma_pairs<32>(a, pairs, tiles, splits, stream);
        case 64: return launch_mma_pairs<64>(a, pairs, tiles, splits, stream);
        case 96: return launch_mma_pairs<96>(a, pairs, tiles, splits, stream);
        case 128: return launch_mma_pairs<128>(a, pairs, tiles, splits, stream);
    }
    return ZAI_BAD_SIZE;
}
