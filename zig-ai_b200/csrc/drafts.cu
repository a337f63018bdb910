// Steps that check drafted tokens.  A request brings a span of rows: its last known token (row 0) and tokens drafted behind it,
// each hanging on an earlier row of the span (its parent; -1: on none).  Four things go with such a step:
//
//   zai_step_layout     the step's tables from the requests' lengths alone, on the device: with n[s] rows, c[s] cached positions
//                       and slot[s] of request s
//                           cu[s]     = n[0] + ... + n[s-1]
//                           row r of request s (i = r - cu[s]):  seq[r] = s;  pos[r] = c[s] + i, in a tree c[s] + depth(r)
//                           kv_slot[r] = page(s, c[s] + i) * page_size + (c[s] + i) mod page_size       (where the request's i-th new
//                                        token is cached; a tree's accepted tokens go there one after the other)
//                           table[s]  = the first `width` entries of the slot's row
//                           mask[r]   = bits of r's ancestors and of r among the span's rows
//                       and one more span, of no request, for the rows behind the last one
//   zai_accept_drafts   cur = 0; while some child c of cur has token[c] == choice[cur]: cur = the first such c
//   zai_commit_drafts   keys and values of the accepted rows into the pages, of one layer (as ModelRunner.verify calls it) or of several at once
//
// All three are a few kilobytes of whole numbers (the last a few megabytes): what bounds them is a launch and two or three trips to
// memory that depend on one another, so each is one kernel, blocks need nothing of one another, and what a block would need from
// another one (the spans' starts) it computes again.  Measured in a captured graph: tables of 32 trees of 4-24 rows 3.5 us, of 256 prompt portions
// 2.6; accepted paths of 256 trees of 8-64 rows 2.6; 640 accepted rows of six layers 9.2 us, 31 MB read and written.
#include "common.cuh"

#define LAYOUT_THREADS 256
#define MAX_SPANS 8192

struct LayoutArgs {
    int *cu, *ctx_out, *positions, *seq_idx, *kv_slots, *tables, *mask;
    const int *lens, *ctx, *slots, *page_rows, *parents;
    int S, N, width, row_width, n_slots, page_size, tree_rows, words, row_blocks;
    int* status;
};

// Exclusive sums of the spans' lengths in shared memory (cu[0..S]), by all threads; negative lengths count as none, and rows
// beyond the step's room are cut off.
__device__ __forceinline__ void span_starts(const int* __restrict__ lens, int S, int N, int* cu, int* warp_sums, int* status) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    int base = 0;
    bool bad = false;
    for (int at = 0; at < S; at += LAYOUT_THREADS) {
        const int s = at + t;
        int n = s < S ? lens[s] : 0;
        if (n < 0 || n > N) {
            bad = true;
            n = n < 0 ? 0 : N;                                 // (no sum of at most 256 of them wraps: N < 2^22)
        }
        int x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) warp_sums[warp] = x;
        __syncthreads();
        int before = 0, total = 0;
#pragma unroll
        for (int w = 0; w < LAYOUT_THREADS / 32; ++w) {
            const int v = warp_sums[w];
            before += w < warp ? v : 0;
            total += v;
        }
        if (s < S) {
            const int start = base + before + x - n;
            if (start + n > N) bad = true;
            cu[s] = min(start, N);
        }
        base = min(base + total, N);
        __syncthreads();
    }
    if (t == 0) cu[S] = base;
    if (bad) zai_raise(status, ZAI_ST_ROWS);
    __syncthreads();
}

__global__ void __launch_bounds__(LAYOUT_THREADS) step_layout_kernel(const LayoutArgs a) {
    extern __shared__ int sm[];
    const int t = threadIdx.x;
    pdl_trigger();
    pdl_wait();
    if ((int)blockIdx.x >= a.row_blocks) {                     // block tables: rows of the requests' slots, a row of the null page behind them
        const int e = ((int)blockIdx.x - a.row_blocks) * LAYOUT_THREADS + t;
        if (e < (a.S + 1) * a.width) {
            const int s = e / a.width, j = e - s * a.width;
            int page = 0;
            if (s < a.S && j < a.row_width) {
                const int slot = zai_checked_slot(a.slots[s], a.n_slots, j == 0 ? a.status : nullptr);
                page = a.page_rows[(size_t)slot * a.row_width + j];
            }
            a.tables[e] = page;
        }
        return;
    }
    int* cu = sm;                                              // [S + 1]
    int* warp_sums = cu + a.S + 1;                             // [8]
    int* par = warp_sums + LAYOUT_THREADS / 32;                // [tree_rows - 1 + threads]: the parents of the block's rows and of those before
    unsigned* bits = (unsigned*)(par + a.tree_rows + LAYOUT_THREADS);   // [threads][words]
    const int r0 = (int)blockIdx.x * LAYOUT_THREADS, par0 = r0 - (a.tree_rows - 1);
    if (a.tree_rows)                                           // (asked for before the sums, which they do not need)
        for (int i = t; i < a.tree_rows - 1 + LAYOUT_THREADS; i += LAYOUT_THREADS)
            par[i] = par0 + i >= 0 && par0 + i < a.N ? a.parents[par0 + i] : -1;
    span_starts(a.lens, a.S, a.N, cu, warp_sums, blockIdx.x == 0 ? a.status : nullptr);
    const int total = cu[a.S];
    if (blockIdx.x == 0) {
        for (int s = t; s < a.S; s += LAYOUT_THREADS) {
            a.cu[s] = cu[s];
            const int c = a.ctx[s];
            if (c < 0) zai_raise(a.status, ZAI_ST_POSITION);
            a.ctx_out[s] = max(c, 0);
        }
        if (t == 0) {
            a.cu[a.S] = total;
            a.cu[a.S + 1] = a.N;
            a.ctx_out[a.S] = 0;
        }
    }
    const int r = r0 + t;
    if (a.tree_rows)
        for (int w = 0; w < a.words; ++w) bits[t * a.words + w] = 0;
    if (r < a.N) {
        int s = a.S, pos = 0, slot = -1;
        if (r < total) {
            int lo = 0, hi = a.S;                              // the last span that starts at or before r (empty ones before it end there too)
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (cu[mid] <= r) lo = mid;
                else hi = mid;
            }
            s = lo;
            const int first = cu[s], i = r - first, c = max(a.ctx[s], 0);
            const int place = zai_checked_slot(a.slots[s], a.n_slots, a.status);
            const unsigned at_most = (unsigned)c + i, page_index = at_most / a.page_size;     // (unsigned: a length near the type's end must not wrap)
            const int j = (int)min(page_index, 0x7fffffffu);
            pos = (int)at_most;
            if (j >= a.width || j >= a.row_width || at_most > 0x7fffffffu) zai_raise(a.status, ZAI_ST_POSITION);
            else {
                const int page = a.page_rows[(size_t)place * a.row_width + j];
                const long long at = (long long)page * a.page_size + (pos - j * a.page_size);
                if (page < 0 || at > 0x7fffffffll) zai_raise(a.status, ZAI_ST_PAGE);
                else slot = (int)at;
            }
            if (a.tree_rows) {
                if (i >= a.tree_rows) zai_raise(a.status, ZAI_ST_TREE);     // a span of more rows than its tree may have: seen by none, in a row
                else {
                    const int* p = par + first - par0;         // p[i]: the parent of the span's row i (i < tree_rows: inside the window)
                    int cur = i, depth = 0;
                    unsigned* mine = bits + t * a.words;
                    mine[i >> 5] = 1u << (i & 31);
                    while (true) {
                        const int up = p[cur];
                        if (up < 0 || up >= cur) {
                            if (up != -1) zai_raise(a.status, ZAI_ST_TREE);
                            break;
                        }
                        mine[up >> 5] |= 1u << (up & 31);
                        cur = up;
                        ++depth;
                    }
                    pos = (int)((unsigned)c + depth);
                }
            }
        } else {
            pos = (r - total) % (a.width * a.page_size);
        }
        a.positions[r] = pos;
        a.seq_idx[r] = s;
        a.kv_slots[r] = slot;
    }
    if (a.tree_rows) {
        __syncthreads();
        const int n = min(a.N - r0, LAYOUT_THREADS) * a.words;
        for (int e = t; e < n; e += LAYOUT_THREADS) a.mask[(size_t)r0 * a.words + e] = (int)bits[e];
    }
}

ZAI_API int zai_step_layout(int* cu, int* ctx_out, int* positions, int* seq_idx, int* kv_slots, int* tables, int* mask,
                            const int* lens, const int* ctx, const int* slots, const int* page_rows, const int* parents, int S, int N,
                            int width, int row_width, int n_slots, int page_size, int tree_rows, int words, int* status, cudaStream_t stream) {
    if (S < 0 || S > MAX_SPANS || N < 0 || N >= (1 << 22) || width < 1 || row_width < 1 || n_slots < 1 || page_size < 1 || tree_rows < 0 ||
        tree_rows > 1024 || words * 32 < tree_rows || words > 32 || (long long)width * page_size > 0x7fffffffll ||
        (long long)(S + 1) * width > 0x7fffffffll - LAYOUT_THREADS)
        return ZAI_BAD_SIZE;
    const int row_blocks = N > 0 ? (N + LAYOUT_THREADS - 1) / LAYOUT_THREADS : 1;
    const int table_blocks = ((S + 1) * width + LAYOUT_THREADS - 1) / LAYOUT_THREADS;
    const size_t smem = sizeof(int) * ((size_t)S + 1 + LAYOUT_THREADS / 32 + tree_rows + LAYOUT_THREADS + (tree_rows ? LAYOUT_THREADS * words : 0));
    static unsigned long long done = 0;
    if (zai_first_on_device(&done)) cudaFuncSetAttribute(step_layout_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024);
    const LayoutArgs a = {cu, ctx_out, positions, seq_idx, kv_slots, tables, mask, lens, ctx, slots, page_rows, parents,
                          S, N, width, row_width, n_slots, page_size, tree_rows, words, row_blocks, status};
    return launch_pdl(step_layout_kernel, dim3(row_blocks + table_blocks), dim3(LAYOUT_THREADS), smem, stream, a);
}

// ---- the accepted path: a warp a request.  Every row whose token is its parent's choice offers itself as the parent's next row, the
// smallest index wins (an order of the atomics that does not show); then one lane follows the rows.
#define ACCEPT_WARPS 4
__global__ void __launch_bounds__(ACCEPT_WARPS * 32) accept_drafts_kernel(int* counts, int* path, int* tokens_out, int* ctx_out,
        const int* __restrict__ choices, const int* __restrict__ tokens, const int* __restrict__ parents, const int* __restrict__ cu,
        const int* __restrict__ ctx, int S, int N, int most, int* status) {
    extern __shared__ int sm[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, s = (int)blockIdx.x * ACCEPT_WARPS + warp;
    int* next = sm + warp * 2 * most;                          // [most], and behind it the path [most]
    int* taken = next + most;
    pdl_trigger();
    pdl_wait();
    if (s >= S) return;
    const int a = cu[s], end = cu[s + 1], cached = ctx[s];
    const bool inside = a >= 0 && end >= a && end <= N;
    int n = inside ? end - a : 0;
    if (!inside && lane == 0) zai_raise(status, ZAI_ST_ROWS);
    if (n > most) {                                            // a span of more rows than a tree may have: what is behind them is not looked at
        if (lane == 0) zai_raise(status, ZAI_ST_TREE);
        n = most;
    }
    for (int i = lane; i < n; i += 32) next[i] = n;
    __syncwarp();
    for (int i = lane + 1; i < n; i += 32) {
        const int p = parents[a + i];
        if (p < -1 || p >= i) zai_raise(status, ZAI_ST_TREE);
        else if (p >= 0 && tokens[a + i] == choices[a + p]) atomicMin(&next[p], i);
    }
    __syncwarp();
    int count = 0;
    if (lane == 0) {
        for (int cur = 0; cur < n; cur = next[cur]) taken[count++] = cur;
        counts[s] = count;
        ctx_out[s] = cached + count;
    }
    count = __shfl_sync(0xffffffffu, count, 0);                // (orders lane 0's writes before the reads below)
    __syncwarp();
    for (int i = lane; i < most; i += 32) {
        const int r = i < count ? a + taken[i] : -1;
        path[(size_t)s * most + i] = r;
        tokens_out[(size_t)s * most + i] = r >= 0 ? choices[r] : -1;
    }
}

ZAI_API int zai_accept_drafts(int* counts, int* path, int* tokens_out, int* ctx_out, const int* choices, const int* tokens, const int* parents,
                              const int* cu, const int* ctx, int S, int N, int most, int* status, cudaStream_t stream) {
    if (S < 1 || N < 0 || most < 1 || most > 1024) return ZAI_BAD_SIZE;
    return launch_pdl(accept_drafts_kernel, dim3((S + ACCEPT_WARPS - 1) / ACCEPT_WARPS), dim3(ACCEPT_WARPS * 32),
                      sizeof(int) * 2 * most * ACCEPT_WARPS, stream, counts, path, tokens_out, ctx_out, choices, tokens, parents, cu, ctx, S, N,
                      most, status);
}

// ---- accepted rows into the pages.  An item is one piece of C bytes of one accepted row's key or value; a block takes a request, a
// layer and COMMIT_ITEMS pieces a thread, asked for before the first is written: what bounds it is the chain path, slot, piece.
#define COMMIT_THREADS 256
#define COMMIT_ITEMS 4
struct CommitArgs {
    char* pages;
    const char *k, *v;
    long long k_plane, v_plane, k_row, v_row, plane;           // in bytes
    const int *path, *counts, *cu, *kv_slots;
    int S, N, most, kv_heads, head_bytes, page_size, num_pages;
    int* status;
};
template <typename C> __global__ void __launch_bounds__(COMMIT_THREADS) commit_drafts_kernel(const CommitArgs a) {
    pdl_trigger();
    pdl_wait();
    // (pieces are numbered in 32 bits: 64-bit divisions cost 1.3 of 10.5 us for 640 rows of six layers, 4 KB each)
    const int s = blockIdx.x;
    const unsigned per_head = a.head_bytes / (unsigned)sizeof(C), per_row = a.kv_heads * per_head;
    int count = a.counts[s];
    if (count > a.most) {
        if (threadIdx.x == 0) zai_raise(a.status, ZAI_ST_ROWS);
        count = a.most;
    }
    const int first = a.cu[s];
    const unsigned total = (unsigned)max(count, 0) * 2 * per_row;
    const unsigned at0 = blockIdx.z * (COMMIT_THREADS * COMMIT_ITEMS) + threadIdx.x;
    if (at0 >= total) return;
    C piece[COMMIT_ITEMS];
    char* to[COMMIT_ITEMS];
#pragma unroll
    for (int u = 0; u < COMMIT_ITEMS; ++u) {
        const unsigned e = at0 + u * COMMIT_THREADS;
        to[u] = nullptr;
        if (e >= total) continue;
        const unsigned i = e / (2 * per_row), in_row = e - i * 2 * per_row, which = in_row >= per_row, x = in_row - which * per_row;
        const unsigned head = x / per_head, part = x - head * per_head;
        const int row = a.path[(size_t)s * a.most + i];
        if ((unsigned)row >= (unsigned)a.N || first < 0 || (unsigned)first + i >= (unsigned)a.N) {
            zai_raise(a.status, ZAI_ST_ROWS);
            continue;
        }
        const int slot = a.kv_slots[first + i];
        if (slot < 0) continue;
        const int page = slot / a.page_size, off = slot - page * a.page_size;
        if (page >= a.num_pages) {
            zai_raise(a.status, ZAI_ST_PAGE);
            continue;
        }
        const char* from = which ? a.v + blockIdx.y * a.v_plane + row * a.v_row : a.k + blockIdx.y * a.k_plane + row * a.k_row;
        piece[u] = *reinterpret_cast<const C*>(from + (size_t)x * sizeof(C));
        to[u] = a.pages + blockIdx.y * a.plane + ((((long long)page * 2 + which) * a.kv_heads + head) * a.page_size + off) * a.head_bytes +
                (size_t)part * sizeof(C);
    }
#pragma unroll
    for (int u = 0; u < COMMIT_ITEMS; ++u)
        if (to[u]) *reinterpret_cast<C*>(to[u]) = piece[u];
}

ZAI_API int zai_commit_drafts(void* pages, const void* k, const void* v, long long k_plane, long long v_plane, long long k_row, long long v_row,
                              const int* path, const int* counts, const int* cu, const int* kv_slots, int dtype, int S, int N, int most,
                              int planes, int kv_heads, int head_dim, int page_size, int num_pages, int* status, cudaStream_t stream) {
    if (S < 1 || N < 0 || most < 1 || planes < 1 || planes > 65535 || kv_heads < 1 || head_dim < 1 || page_size < 1 || num_pages < 1)
        return ZAI_BAD_SIZE;
    if (dtype != ZAI_F32 && dtype != ZAI_BF16) return ZAI_BAD_DTYPE;
    const int es = dtype == ZAI_F32 ? 4 : 2, head_bytes = head_dim * es;
    const long long plane = (long long)num_pages * 2 * kv_heads * page_size * head_bytes;
    const CommitArgs a = {(char*)pages, (const char*)k, (const char*)v, k_plane * es, v_plane * es, k_row * es, v_row * es, plane,
                          path, counts, cu, kv_slots, S, N, most, kv_heads, head_bytes, page_size, num_pages, status};
    // pieces of 16 bytes where every row and head starts on one, else element by element
    const bool wide = !(((uintptr_t)pages | (uintptr_t)k | (uintptr_t)v) & 15) && !((a.k_plane | a.v_plane | a.k_row | a.v_row | head_bytes) & 15);
    const int size = wide ? 16 : es;
    if ((long long)most * 2 * kv_heads * (head_bytes / size) > 0x3fffffffll) return ZAI_BAD_SIZE;
    const long long items = (long long)most * 2 * kv_heads * (head_bytes / size), per_block = COMMIT_THREADS * COMMIT_ITEMS;
    const long long z = (items + per_block - 1) / per_block;
    if (z > 65535) return ZAI_BAD_SIZE;
    const dim3 grid(S, planes, (unsigned)z), block(COMMIT_THREADS);
    if (wide) return launch_pdl(commit_drafts_kernel<uint4>, grid, block, 0, stream, a);
    if (es == 4) return launch_pdl(commit_drafts_kernel<uint32_t>, grid, block, 0, stream, a);
    return launch_pdl(commit_drafts_kernel<uint16_t>, grid, block, 0, stream, a);
}
