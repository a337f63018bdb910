// Log probabilities of given tokens, with a row's entropy, the tokens' ranks and the best alternatives, in one walk over the logits.
//
// For a row x[0..V) and a token t, with m = max x, z = sum exp(x - m), u = sum (x - m) exp(x - m):
//     logprob(j) = x[j] - m - ln z          entropy = ln z - u / z
//     rank(t)    = how many j stand before t in the order by value, equal values by the lower index
//     top        = the first `top` of that order
// A thread keeps m, z, u of what it has seen (rescaled when its maximum grows) and the count for the rank; they are joined at the end.
//
// The best tokens.  An entry's key is its value's bits in an order that compares as a whole number, and behind them the complement
// of its index: keys are all different, and the order of keys is the order wanted.  The first round of the walk is split into 64 groups by
// lane and half of the block; the top-th largest of the groups' largest keys bounds the row's top-th key from below (`top` <= 32), so only keys at or above it are noted in
// shared memory: some twenty of each 4096 entries.  After 2, 4, 8, 16, .. rounds the list is cut down to the `top` largest, the last of which is the new bound,
// so that as many rounds again note as many again.  A key's place is the number of noted keys above it.  A row that
// notes more than there is room for (one that ascends) is walked again in steps that cut the list down as they go.
//
// What bounds it: instructions and the wait for memory together.  An entry takes 13 instructions of a thread without alternatives, 16 with five
// and 22 with 32, in either type (counted over 2048 rows of 64 401 and 65 536); they fill 56 to 60 % of the issue slots.  What a warp waits for
// between two of them is its next round's loads (half of the wait without alternatives; with five a fifth, and as much for the barriers of
// the list's cuts).  bfloat16 rows are half the bytes and the same instructions, and take as long.  So a thread looks for keys to note only where its
// round's maximum reaches the bound, the sums take two numbers an instruction, and 0 times -inf, which only masked tokens bring, is put right afterwards.
//
// A row is split over a cluster of up to 16 blocks when there are few rows; the first block joins the parts through distributed shared memory.
// Measured: 2048 rows of 64 401 in 32 bits 87 us without alternatives (6.1 TB/s), 103 with 5, 121 with 20, 139 with 32; in
// bfloat16 86, 115 and 133 (2048 of 65 536).  8 rows of 65 536 with 20 alternatives 10 us: two rounds a block, the candidates' counts, the join.
#include <cooperative_groups.h>
#include "common.cuh"
namespace cg = cooperative_groups;

#define LP_THREADS 256
#define LP_WARPS (LP_THREADS / 32)
#define LP_ROUND 16                 // entries of a row a thread looks at in one round
#define LP_ROOM 1024                // noted keys a block has room for
typedef unsigned long long u64;

__device__ __forceinline__ u64 key_of(float x, int j) {
    const int b = __float_as_int(x + 0.f);                     // (-0 counts as 0; what is not a number comes last)
    const unsigned order = x != x ? 0u : (unsigned)(b ^ (b >> 31 & 0x7fffffff)) ^ 0x80000000u;
    return ((u64)order << 32) | (unsigned)~j;
}
__device__ __forceinline__ float value_of(u64 key) {
    const int o = (int)((unsigned)(key >> 32) ^ 0x80000000u);
    return __int_as_float(o ^ (o >> 31 & 0x7fffffff));
}
// e^x, 2 ulp of 2^(x log2 e) beside the rounding of the product (x <= 0 here; large -x, where that shows, weigh nothing)
__device__ __forceinline__ float exp_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}

struct Sums { float m, z, u; };
// a's sums with b's: each relative to its own maximum
__device__ __forceinline__ Sums joined(const Sums& a, const Sums& b) {
    const float m = fmaxf(a.m, b.m);
    Sums r = {m, 0.f, 0.f};
    if (a.m != -INFINITY) {
        const float d = fmaxf(a.m - m, -150.f), f = exp_of(d);     // (0 beyond that, which a difference near the type's end must not turn into NaN)
        r.z += f * a.z;
        r.u += f * (a.u + d * a.z);
    }
    if (b.m != -INFINITY) {
        const float d = fmaxf(b.m - m, -150.f), f = exp_of(d);
        r.z += f * b.z;
        r.u += f * (b.u + d * b.z);
    }
    return r;
}

__device__ __forceinline__ float pow2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct Part { Sums sums; int before, noted; u64 bound; };      // what a block of a row's cluster hands to the first one

// Entries j0 .. j0 + VEC of a row, of which those in [lo, hi) count; others come back as -inf.
template <typename T> struct Piece;
template <> struct Piece<float> {
    static constexpr int VEC = 4;
    static __device__ __forceinline__ void load(const float* row, int j, float (&x)[4]) {
        const float4 v = *reinterpret_cast<const float4*>(row + j);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    }
};
template <> struct Piece<bf16> {
    static constexpr int VEC = 8;
    static __device__ __forceinline__ void load(const bf16* row, int j, float (&x)[8]) {
        const uint4 v = *reinterpret_cast<const uint4*>(row + j);
        const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};

// A round: the thread's LP_ROUND / VEC vectors, LP_THREADS vectors apart.  `row` starts on 16 bytes when `lead` entries before the row's first
// are counted in (they lie outside [lo, hi)).
template <typename T>
__device__ __forceinline__ void load_round(const T* __restrict__ row, int at, int lo, int hi, float (&x)[LP_ROUND]) {
    constexpr int VEC = Piece<T>::VEC;
    if (at >= lo && at + LP_THREADS * LP_ROUND <= hi) {        // (all of it counts: nearly every round)
        const T* from = row + at + (int)threadIdx.x * VEC;
#pragma unroll
        for (int u = 0; u < LP_ROUND / VEC; ++u) {
            float v[VEC];
            Piece<T>::load(from, u * LP_THREADS * VEC, v);
#pragma unroll
            for (int c = 0; c < VEC; ++c) x[u * VEC + c] = v[c];
        }
        return;
    }
#pragma unroll
    for (int u = 0; u < LP_ROUND / VEC; ++u) {
        const int j = at + (u * LP_THREADS + (int)threadIdx.x) * VEC;
        float v[VEC];
        if (j >= lo && j + VEC <= hi) Piece<T>::load(row, j, v);
        else {
#pragma unroll
            for (int c = 0; c < VEC; ++c) v[c] = j + c >= lo && j + c < hi ? to_float(row[j + c]) : -INFINITY;
        }
#pragma unroll
        for (int c = 0; c < VEC; ++c) x[u * VEC + c] = v[c];
    }
}
template <typename T> __device__ __forceinline__ int index_in_round(int at, int e) {
    constexpr int VEC = Piece<T>::VEC;
    return at + ((e / VEC) * LP_THREADS + (int)threadIdx.x) * VEC + e % VEC;
}

// The keys in list[0..n) cut down to the `keep` largest, in order; all threads; `out` holds `keep` keys.
__device__ __forceinline__ void select_largest(const u64* list, int n, int keep, u64* out) {
    for (int i = threadIdx.x; i < n; i += LP_THREADS) {
        const u64 mine = list[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += list[j] > mine;
        if (above < keep) out[above] = mine;
    }
    __syncthreads();
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_THREADS, 4) token_logprobs_kernel(float* __restrict__ logprobs, float* __restrict__ entropy,
        int* __restrict__ ranks, int* __restrict__ top_ids, float* __restrict__ top_logprobs, const T* __restrict__ logits, long long stride,
        const int* __restrict__ targets, int V, int top, int blocks, int* status) {
    constexpr int VEC = Piece<T>::VEC;
    __shared__ u64 list[TOP ? LP_ROOM : 1];
    __shared__ u64 best[32], groups[TOP ? 64 : 1];
    __shared__ u64 warp_best[TOP ? LP_THREADS : 1];
    __shared__ u64 bound_s;
    __shared__ int noted;
    __shared__ Part part;
    __shared__ Sums warp_sums[LP_WARPS];
    __shared__ int warp_before[LP_WARPS];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int r = (int)blockIdx.x / blocks, b = (int)blockIdx.x - r * blocks;
    if (t == 0) {
        noted = 0;
        bound_s = 0;
    }
    pdl_trigger();
    pdl_wait();
    const T* row = logits + (long long)r * stride;
    // indices from here on count from a 16-byte boundary at or before the row
    const int lead = (int)(((uintptr_t)row & 15) / sizeof(T));
    const T* base = row - lead;
    const int target = targets[r];
    const bool asked = (unsigned)target < (unsigned)V;
    const float xt = asked ? to_float(row[target]) + 0.f : 0.f;
    if (t == 0 && b == 0 && !asked && target != -1) zai_raise(status, ZAI_ST_TOKEN);
    // this block's share: whole rounds' vectors, [lo, hi)
    const int vectors = (V + lead + VEC - 1) / VEC, share = (vectors + blocks - 1) / blocks;
    const int first = b * share * VEC;
    const int lo = max(first, lead), hi = min(first + share * VEC, V + lead);
    const int jt = asked ? target + lead : -1;                 // entries before it count when they are equal
    // the next value above xt: x >= that is x > xt
    const float above_xt = xt == INFINITY ? NAN : xt == 0.f ? __int_as_float(1) : __int_as_float(__float_as_int(xt) + (xt > 0.f ? 1 : -1));

    Sums mine = {-INFINITY, 0.f, 0.f};
    int before = 0;
    u64 bound = 0;
    float bound_x = -INFINITY;
    const int step = LP_THREADS * LP_ROUND;
    auto round = [&](const float (&x)[LP_ROUND], int at) {
        float top4[LP_ROUND / 4], top_x;
#pragma unroll
        for (int e = 0; e < LP_ROUND; e += 4) top4[e / 4] = fmaxf(zai_max3(x[e], x[e + 1], x[e + 2]), x[e + 3]);
        top_x = fmaxf(zai_max3(top4[0], top4[1], top4[2]), top4[3]);
        if (TOP) {
            // (the entries of the lanes that have such a key are looked at once more, in memory, by few instructions: with the registers' sixteen
            // copies of this code it was a third of the kernel, most of it their own arrival)
            auto note = [&](int j) {
                if (j < lo || j >= hi) return;
                const u64 k = key_of(to_float(base[j]), j - lead);
                if (k < bound) return;
                const int p = atomicAdd(&noted, 1);
                if (p < LP_ROOM) list[p] = k;
            };
            unsigned hits = __ballot_sync(0xffffffffu, top_x >= bound_x || top_x != top_x);
            if (__popc(hits) > 8)
#pragma unroll 1
                for (int e = 0; e < LP_ROUND; ++e) note(index_in_round<T>(at, e));
            else
#pragma unroll 1
                while (hits) {                                 // two lanes' sixteen entries at a time
                    const int one = __ffs(hits) - 1;
                    hits &= hits - 1;
                    const int two = __ffs(hits) - 1, of = lane < LP_ROUND ? one : two, e = lane & (LP_ROUND - 1);
                    hits &= hits - 1;
                    if (of >= 0) note(at + ((e / VEC) * LP_THREADS + warp * 32 + of) * VEC + e % VEC);
                    __syncwarp();
                }
        }
        if (top_x > mine.m) {
            const Sums none = {top_x, 0.f, 0.f};
            mine = joined(mine, none);
        }
        if (mine.m != -INFINITY) {
            float2 z = make_float2(0.f, 0.f), u = z;
            const float2 m2 = make_float2(-mine.m, -mine.m), l2 = make_float2(1.4426950408889634f, 1.4426950408889634f);
#pragma unroll
            for (int e = 0; e < LP_ROUND; e += 2) {
                const float2 d = zai_add2(make_float2(x[e], x[e + 1]), m2), p = zai_mul2(d, l2), w = make_float2(pow2_of(p.x), pow2_of(p.y));
                z = zai_add2(z, w);
                u = zai_fma2(w, d, u);
            }
            if (u.x != u.x || u.y != u.y) {                    // 0 times -inf, which is 0 here
                u = make_float2(0.f, 0.f);
#pragma unroll
                for (int e = 0; e < LP_ROUND; ++e) {
                    const float d = x[e] - mine.m;
                    u.x += exp_of(d) * fmaxf(d, -150.f);
                }
            }
            mine.z += z.x + z.y;
            mine.u += u.x + u.y;
        } else {
#pragma unroll
            for (int e = 0; e < LP_ROUND; ++e)
                if (x[e] != x[e]) mine = {0.f, NAN, NAN};      // (nothing else than -inf so far)
        }
        if (jt < at || jt >= at + step) {                      // (the token is not in this round: one bound for all)
            const float need = at < jt ? xt : above_xt;
            int n0 = 0, n1 = 0;
#pragma unroll
            for (int e = 0; e < LP_ROUND; e += 2) {
                n0 += x[e] >= need;
                n1 += x[e + 1] >= need;
            }
            before += n0 + n1;
        } else {
#pragma unroll
            for (int e = 0; e < LP_ROUND; ++e) before += x[e] >= (index_in_round<T>(at, e) < jt ? xt : above_xt);
        }
    };
    // two rounds at a time, each asked for while the other is looked at
    float x[LP_ROUND], y[LP_ROUND];
    load_round<T>(base, first, lo, hi, x);
    if (first + step < hi) load_round<T>(base, first + step, lo, hi, y);
    if (TOP && first < hi) {
        // the first bound: the top-th largest of the groups' largest keys
        u64 k = 0;
        float top_x = x[0];
#pragma unroll
        for (int e = 1; e < LP_ROUND; ++e) top_x = fmaxf(top_x, x[e]);
        if (top_x > -INFINITY) {
            int e0 = 0;                                        // the first of the largest
#pragma unroll
            for (int e = LP_ROUND - 1; e >= 0; --e) e0 = x[e] == top_x ? e : e0;
            k = key_of(top_x, index_in_round<T>(first, e0) - lead);
        } else                                                 // nothing but -inf, or what is not a number: which of them are the share's is looked at
#pragma unroll 1
            for (int e = 0; e < LP_ROUND; ++e) {
                const int j = index_in_round<T>(first, e);
                if (j >= lo && j < hi) k = max(k, key_of(to_float(base[j]), j - lead));
            }
        warp_best[t] = k;
        __syncthreads();
        if (warp < 2) {                                        // (64 groups: a lane of either half of the warps)
            k = 0;
#pragma unroll
            for (int w = 0; w < LP_WARPS / 2; ++w) k = max(k, warp_best[(warp * (LP_WARPS / 2) + w) * 32 + lane]);
            groups[t] = k;
        }
        __syncthreads();
        if (warp < 2) {
            int above = 0;
#pragma unroll 8
            for (int i = 0; i < 64; ++i) above += groups[i] > k || (groups[i] == k && i < t);      // (groups without entries are equal)
            if (above == top - 1) bound_s = k;
        }
        __syncthreads();
        bound = bound_s;
        bound_x = fmaxf(value_of(bound), -INFINITY);           // (no bound, or one that is not a number: everything)
    }
    for (int at = first, number = 2; at < hi; at += 2 * step, number += 2) {
        round(x, at);
        if (at + 2 * step < hi) load_round<T>(base, at + 2 * step, lo, hi, x);
        if (at + step < hi) {
            round(y, at + step);
            if (at + 3 * step < hi) load_round<T>(base, at + 3 * step, lo, hi, y);
        }
        if (TOP && (number & (number - 1)) == 0 && at + 2 * step < hi) {
            // after 2, 4, 8, 16, .. rounds: the list cut down to the largest so far, and the bound raised
            __syncthreads();
            const int n = noted;
            __syncthreads();
            if (n > top && n <= LP_ROOM) {
                select_largest(list, n, top, best);
                if (t < top) list[t] = best[t];
                if (t == 0) noted = top;
                bound = best[top - 1];
                bound_x = fmaxf(value_of(bound), -INFINITY);
                if (t == 0) bound_s = bound;
                __syncthreads();
            }
        }
    }
    if (xt == -INFINITY && asked) {
        // entries outside [lo, hi) came as -inf and were counted as equal ones before the token: counted again, by index
        before = 0;
        for (int j = lo + t; j < hi; j += LP_THREADS) {
            const float v = to_float(base[j]);
            before += v > xt || (v == xt && j < jt);
        }
    }
    // the block's sums
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Sums other = {__shfl_xor_sync(0xffffffffu, mine.m, o), __shfl_xor_sync(0xffffffffu, mine.z, o), __shfl_xor_sync(0xffffffffu, mine.u, o)};
        mine = joined(mine, other);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    if (lane == 0) {
        warp_sums[warp] = mine;
        warp_before[warp] = before;
    }
    __syncthreads();
    if (TOP) {
        if (noted > LP_ROOM) {
            // more keys than there is room for: once more, a slice of at most LP_THREADS entries at a time, the list cut down when the next slice may not fit
            __syncthreads();
            if (t == 0) noted = 0;
            __syncthreads();
            for (int at = lo; at < hi; at += LP_THREADS) {
                const int j = at + t;
                if (j < hi) {
                    const u64 k = key_of(to_float(base[j]), j - lead);
                    if (k >= bound) list[atomicAdd(&noted, 1)] = k;
                }
                __syncthreads();
                const int now = noted;
                __syncthreads();
                if (now > LP_ROOM - LP_THREADS) {
                    select_largest(list, now, top, best);
                    if (t < top) list[t] = best[t];
                    if (t == 0) noted = top;
                    bound = best[top - 1];
                    __syncthreads();
                }
            }
            if (t == 0) bound_s = bound;
            __syncthreads();
        }
        if (blocks > 1 && noted > top) {                       // (the row's bound is then the highest of the blocks' own: few keys are handed on)
            select_largest(list, noted, top, best);
            if (t < top) list[t] = best[t];
            if (t == 0) {
                noted = top;
                bound_s = best[top - 1];
            }
            __syncthreads();
        }
    }
    if (warp == 0) {
        Sums s = lane < LP_WARPS ? warp_sums[lane] : Sums{-INFINITY, 0.f, 0.f};
        int n = lane < LP_WARPS ? warp_before[lane] : 0;
#pragma unroll
        for (int o = LP_WARPS / 2; o > 0; o >>= 1) {
            const Sums other = {__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.z, o), __shfl_xor_sync(0xffffffffu, s.u, o)};
            s = joined(s, other);
            n += __shfl_xor_sync(0xffffffffu, n, o);
        }
        if (lane == 0) part = {s, n, TOP ? noted : 0, bound_s};
    }
    __syncthreads();
    Sums all = part.sums;
    int rank = part.before, n = part.noted;
    if (blocks > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        if (b == 0) {
            all = {-INFINITY, 0.f, 0.f};
            rank = 0;
            u64 low = 0;
            for (int i = 0; i < blocks; ++i) {                 // (in the blocks' order: the sums do not depend on who comes first)
                const Part p = *cluster.map_shared_rank(&part, i);
                all = joined(all, p.sums);
                rank += p.before;
                low = max(low, p.bound);                       // every block's bound is one of the row's
            }
            if (TOP) {
                // the other blocks' keys at or above the highest bound, behind this block's own (at most LP_ROOM in all)
                for (int other = warp ? warp : LP_WARPS; other < blocks; other += LP_WARPS) {        // (a warp a block, or two)
                    const int count = cluster.map_shared_rank(&part, other)->noted;
                    const u64* theirs = cluster.map_shared_rank(list, other);
                    for (int i = lane; i < count; i += 32) {
                        const u64 k = theirs[i];
                        if (k >= low) list[atomicAdd(&noted, 1)] = k;
                    }
                }
                __syncthreads();
                n = noted;
            }
        }
        cluster.sync();                                        // the other blocks' shared memory has been read
        if (b != 0) return;
    }
    const float log_z = logf(all.z);
    if (t == 0) {
        logprobs[r] = asked ? xt - all.m - log_z : 0.f;
        entropy[r] = log_z - all.u / all.z;
        ranks[r] = asked ? rank : -1;
    }
    if (TOP) {
        select_largest(list, n, top, best);
        if (t < top) {
            const u64 k = best[t];
            top_ids[(size_t)r * top + t] = (int)~(unsigned)k;
            top_logprobs[(size_t)r * top + t] = value_of(k) - all.m - log_z;
        }
    }
}

template <typename T>
static int launch_logprobs(float* logprobs, float* entropy, int* ranks, int* top_ids, float* top_logprobs, const void* logits, long long stride,
                           const int* targets, int R, int V, int top, int blocks, int* status, cudaStream_t stream) {
    const auto kernel = top ? token_logprobs_kernel<T, true> : token_logprobs_kernel<T, false>;
    static unsigned long long done[2] = {0, 0};
    if (zai_first_on_device(&done[top > 0])) cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)R * blocks);
    cfg.blockDim = dim3(LP_THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = blocks;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&cfg, kernel, logprobs, entropy, ranks, top_ids, top_logprobs, (const T*)logits, stride, targets, V, top, blocks,
                                   status);
}

// `blocks` (a power of two up to 16): blocks that share a row; 0: as many as leave every block half a round of the walk at least and fit on the chip at
// once, four an SM less what clusters leave free (us at 1, 2, 4, 8 and 16 blocks, rows of 65 536: one row, 20 alternatives, 21, 16, 12, 9.8, 12; 64 rows,
// none, 10, 9.2, 7.8, 6.9, 14; 128 rows, five, 20, 17, 14, 19, 38; 148 rows 17, 14, 20, 25, 44; 256 rows 25, 19, 26, 36, 71).
ZAI_API int zai_token_logprobs(float* logprobs, float* entropy, int* ranks, int* top_ids, float* top_logprobs, const void* logits, int dtype,
                               long long stride, const int* targets, int R, int V, int top, int blocks, int sms, int* status,
                               cudaStream_t stream) {
    if (R < 1 || V < 1 || V > 0x7fffffff - 8 * LP_THREADS * LP_ROUND || R > 0x7fffffff / 16 || top < 0 || top > 32 || top > V || blocks < 0 || blocks > 16 ||
        (blocks & (blocks - 1)))
        return ZAI_BAD_SIZE;
    if (blocks == 0)
        for (blocks = 1; blocks < 8 && (long long)R * blocks * 2 * 2 <= 7 * sms && V / (blocks * 2) >= LP_THREADS * LP_ROUND / 2;) blocks *= 2;
    ZAI_DISPATCH(dtype, return launch_logprobs<T>(logprobs, entropy, ranks, top_ids, top_logprobs, logits, stride, targets, R, V, top, blocks, status, stream));
}
