// cuddle_rows_select.hpp — the selection of cuddle_rows.hpp's exhaustive search: the k smallest of rows of distances.
// Included by cuddle_rows.hpp behind cuddle_kernels.hpp, whose wave helpers it uses and nothing else, so that a host
// build with stand-ins for those can run these kernels thread by thread.
#pragma once

#include <cstdint>

namespace cuddle {

constexpr uint32_t kCountPitch = 32; // counters of candidates stand 128 bytes apart: atomics on one line wait for each other

// ---------------------------------------------------------------------------------------------
// top-k of rows of distances
// ---------------------------------------------------------------------------------------------
// An item is (key << 32 | row); keys are f32_key (NaN after everything), equal keys go by row. A level cuts a query's
// items into chunks and keeps each chunk's k smallest, in any order; a chunk short of k is filled up with ~0, which
// stands behind every row.
// Many rows and queries: the distances are not written at all. The k-th smallest key of a sample of the rows bounds the
// k-th smallest of all, a pass over the rows collects those within the bound (a few thousand), and the k smallest of the
// collection are the answer. Where the collection overflows, the levels answer instead.
constexpr uint32_t kTopChunk = 8192;
constexpr uint32_t kTopMaxK = 1024;
constexpr uint32_t kTopThreads = 1024;

// Items per block of a selection level: fewer where that fills the chip sooner (50 000 items, one query, k = 100: 16 us in 7
// blocks, 6 in 25), as long as one more level answers and a chunk is several times what it keeps.
inline uint32_t top_chunk(uint64_t items, uint32_t nq, uint32_t k) {
    const uint64_t fits = 3072 / k; // parts that the last level takes without becoming the longer one
    for (uint32_t chunk : {1024u, 2048u, 4096u}) {
        const uint64_t parts = (items + chunk - 1) / chunk;
        if (chunk >= 8 * k && parts <= fits && parts * nq <= 1024) return chunk;
    }
    return kTopChunk;
}

struct TopkLds {
    uint32_t hist[256];
    uint32_t lo[kTopThreads / 64], hi[kTopThreads / 64];
    uint32_t bin, rest, full, n;
};

// T and budget such that the k smallest (1 <= k <= C) of the keys key(0) .. key(C - 1) are those below T and `budget` of
// those equal to T: T is the k-th smallest or, where nothing lies between, larger. 8 bits at a time from the highest bit in
// which the keys differ: distances share their leading bits, and a histogram of those would be one counter that every
// thread adds to. All threads of a block of kTopThreads.
template <class KeyFn>
__device__ __forceinline__ void block_kth_key(uint32_t C, uint32_t k, KeyFn key, TopkLds &s, uint32_t &T, uint32_t &budget) {
    const uint32_t tid = threadIdx.x;
    uint32_t lo = 0xFFFFFFFFu, hi = 0;
    for (uint32_t i = tid; i < C; i += kTopThreads) {
        const uint32_t v = key(i);
        lo = min(lo, v);
        hi = max(hi, v);
    }
    lo = wave_min_u32(lo);
    hi = ~wave_min_u32(~hi);
    __syncthreads();
    if ((tid & 63) == 0) {
        s.lo[tid >> 6] = lo;
        s.hi[tid >> 6] = hi;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kTopThreads / 64; ++w) {
        lo = min(lo, s.lo[w]);
        hi = max(hi, s.hi[w]);
    }
    // the bits all keys share; one 64-bit shift, no case for lo == hi: a select on it came out of the compiler wrong
    uint32_t mask = ~(uint32_t)(0xFFFFFFFFull >> __clz((int)(lo ^ hi)));
    uint32_t prefix = lo & mask;
    budget = k;
    while (mask != 0xFFFFFFFFu) {
        const uint32_t low = 32 - __popc(mask), shift = low > 8 ? low - 8 : 0, bins = 1u << (low - shift);
        for (uint32_t i = tid; i < 256; i += kTopThreads) s.hist[i] = 0;
        __syncthreads();
        for (uint32_t i = tid; i < C; i += kTopThreads) {
            const uint32_t v = key(i);
            if ((v & mask) == prefix) atomicAdd(&s.hist[(v >> shift) & (bins - 1)], 1u);
        }
        __syncthreads();
        if (tid < 64) { // four bins per lane: the bin in which the running count reaches what is looked for
            const uint32_t b = tid * 4;
            const uint32_t c0 = s.hist[b], c1 = s.hist[b + 1], c2 = s.hist[b + 2], c3 = s.hist[b + 3];
            const uint32_t incl = wave_inclusive_sum(c0 + c1 + c2 + c3);
            uint32_t run = incl - (c0 + c1 + c2 + c3);
            if (run < budget && budget <= incl) {
                uint32_t bin = b, c = c0;
                if (run + c0 < budget) { run += c0; ++bin; c = c1;
                    if (run + c1 < budget) { run += c1; ++bin; c = c2;
                        if (run + c2 < budget) { run += c2; ++bin; c = c3; } } }
                s.bin = bin;
                s.rest = budget - run;
                s.full = c == budget - run ? 1u : 0u;
            }
        }
        __syncthreads();
        prefix |= s.bin << shift;
        mask |= (bins - 1) << shift;
        budget = s.rest;
        const bool full = s.full != 0;
        __syncthreads();
        if (full) { // everything that starts with these digits is wanted: no need to know how it goes on
            prefix |= ~mask;
            budget = C;
            break;
        }
    }
    T = prefix;
}

// The k smallest of C items with keys keys[i] (LDS) and item(i) = key << 32 | row: emit(place, item) in any order, places
// from 0 on. Of the items equal to the last key the lowest rows. Fill (~0) is never handed on: it has one row number for
// all, so among the k smallest - where fewer than k real items are left - no row would tell apart how many of it are
// wanted. s.n is zero on entry and counts what was emitted, at most k. All threads of the block.
template <class ItemFn, class EmitFn>
__device__ __forceinline__ void block_smallest(const uint32_t *keys, uint32_t C, uint32_t k, ItemFn item, EmitFn emit, TopkLds &s) {
    const uint32_t tid = threadIdx.x;
    uint32_t T = 0xFFFFFFFFu, budget = C, R = 0xFFFFFFFFu, rest;
    if (C > k) {
        block_kth_key(C, k, [&](uint32_t i) { return keys[i]; }, s, T, budget);
        if (budget < C) { // T is a key of its own: are there more items with it than wanted?
            uint32_t ties = 0;
            for (uint32_t i = tid; i < C; i += kTopThreads) ties += keys[i] == T ? 1u : 0u;
            if (ties) atomicAdd(&s.n, ties);
            __syncthreads();
            ties = s.n;
            __syncthreads();
            if (tid == 0) s.n = 0;
            if (ties > budget) block_kth_key(C, budget, [&](uint32_t i) { return keys[i] == T ? (uint32_t)item(i) : 0xFFFFFFFFu; }, s, R, rest);
            __syncthreads();
        }
    }
    for (uint32_t i = tid; i < C; i += kTopThreads) {
        if (keys[i] > T) continue;
        const uint64_t v = item(i);
        if (v != ~0ull && (keys[i] < T || (uint32_t)v <= R)) emit(atomicAdd(&s.n, 1u), v);
    }
}

// Level: from f32 distances (FIRST) or from the previous level's lists. in: [nq][in_stride]; out: [nq][parts][k].
// chunk <= kTopChunk items at a time. redo: nullptr, or only queries that count more than `cap` (few blocks then, since
// hardly ever one has work). grid (at most parts, nq), block kTopThreads.
template <bool FIRST>
__global__ void __launch_bounds__(kTopThreads)
int4_topk_level_kernel(const void *in, uint64_t in_stride, uint64_t items, uint32_t k, uint32_t chunk, uint32_t parts, uint64_t *out, const uint32_t *redo,
                       uint32_t cap) {
    __shared__ uint32_t keys[kTopChunk];
    __shared__ TopkLds s;
    if (redo && redo[blockIdx.y * kCountPitch] <= cap) return;
    const uint32_t tid = threadIdx.x;
    for (uint32_t part = blockIdx.x; part < parts; part += gridDim.x) {
        const uint64_t base = (uint64_t)part * chunk;
        const uint32_t C = (uint32_t)min((uint64_t)chunk, items - base);
        const float *df = static_cast<const float *>(in) + (uint64_t)blockIdx.y * in_stride + base;
        const uint64_t *dl = static_cast<const uint64_t *>(in) + (uint64_t)blockIdx.y * in_stride + base;
        __syncthreads(); // the part before has been read
#pragma unroll 8
        for (uint32_t i = tid; i < C; i += kTopThreads) keys[i] = FIRST ? f32_key(df[i]) : (uint32_t)(dl[i] >> 32);
        if (tid == 0) s.n = 0;
        __syncthreads();
        uint64_t *o = out + ((uint64_t)blockIdx.y * parts + part) * k;
        block_smallest(
            keys, C, k, [&](uint32_t i) -> uint64_t { return FIRST ? (uint64_t)keys[i] << 32 | (uint32_t)(base + i) : dl[i]; },
            [&](uint32_t at, uint64_t v) { o[at] = v; }, s);
        __syncthreads();
        for (uint32_t i = s.n + tid; i < k; i += kTopThreads) o[i] = ~0ull;
    }
}

// The bound of a query: the k-th smallest key of its sample, and its candidate count set to zero. One block per query;
// the keys in LDS where they fit (items words of dynamic LDS, or none).
__global__ void __launch_bounds__(kTopThreads)
int4_topk_bound_kernel(const float *dist, uint64_t dstride, uint32_t items, uint32_t k, uint32_t in_lds, uint32_t *tau, uint32_t *cnt) {
    extern __shared__ uint32_t s_keys[];
    __shared__ TopkLds s;
    const float *df = dist + (uint64_t)blockIdx.x * dstride;
    uint32_t T, budget;
    if (in_lds) {
#pragma unroll 8
        for (uint32_t i = threadIdx.x; i < items; i += kTopThreads) s_keys[i] = f32_key(df[i]);
        __syncthreads();
        block_kth_key(items, k, [&](uint32_t i) { return s_keys[i]; }, s, T, budget);
    } else
        block_kth_key(items, k, [&](uint32_t i) { return f32_key(df[i]); }, s, T, budget);
    if (threadIdx.x == 0) {
        tau[blockIdx.x] = T;
        cnt[blockIdx.x * kCountPitch] = 0;
    }
}

__device__ __forceinline__ float f32_of_key(uint32_t k) { // NaN for the NaN's key; the two zeros are one
    if (k == 0xFFFFFFFFu) return __builtin_nanf("");
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// Sort of n (a power of two, at most kTopThreads) distinct items, padded at the end with ~0: every item's place is the
// number of items below it, counted by kTopThreads / n neighbouring lanes (64 at most), a part of the items each.
__device__ __forceinline__ void block_sort_small(uint64_t *s, uint32_t n) {
    const uint32_t per = min(64u, kTopThreads / n), i = threadIdx.x / per, part = threadIdx.x % per, m = max(1u, n / per);
    const uint64_t v = i < n ? s[i] : ~0ull;
    uint32_t place = 0;
    if (i < n && part * m < n)
#pragma unroll 8
        for (uint32_t j = part * m; j < part * m + m; ++j) place += s[j] < v ? 1u : 0u;
    for (uint32_t d = 1; d < per; d <<= 1) place += (uint32_t)__shfl_xor((int)place, (int)d, 64);
    __syncthreads(); // every item has been read
    if (part == 0 && i < n && v != ~0ull) s[place] = v;
    __syncthreads();
}

// Last level: at most kTopChunk items; the k smallest, in order, as ids and distances. KIND 0: distances in row order,
// 1: a level's list, 2: a collection in any order, count[q] of them (left alone where they overflowed).
template <int KIND>
__global__ void __launch_bounds__(kTopThreads)
int4_topk_final_kernel(const void *in, uint64_t in_stride, uint32_t items, uint32_t k, uint32_t found, const uint32_t *cnt, uint32_t cap, uint64_t *ids, float *out,
                       uint32_t *count) {
    __shared__ uint32_t keys[kTopChunk];
    __shared__ uint64_t sel[kTopMaxK];
    __shared__ TopkLds s;
    const uint32_t tid = threadIdx.x, q = blockIdx.x;
    if (KIND == 2) {
        items = cnt[q * kCountPitch];
        if (items > cap) return;
    } else if (cnt && cnt[q * kCountPitch] <= cap)
        return;
    const float *df = static_cast<const float *>(in) + (uint64_t)q * in_stride;
    const uint64_t *dl = static_cast<const uint64_t *>(in) + (uint64_t)q * in_stride;
#pragma unroll 8
    for (uint32_t i = tid; i < items; i += kTopThreads) keys[i] = KIND == 0 ? f32_key(df[i]) : (uint32_t)(dl[i] >> 32);
    const uint32_t width = next_pow2(min(k, items));
    for (uint32_t i = tid; i < width; i += kTopThreads) sel[i] = ~0ull;
    if (tid == 0) s.n = 0;
    __syncthreads();
    block_smallest(
        keys, items, k, [&](uint32_t i) -> uint64_t { return KIND == 0 ? (uint64_t)keys[i] << 32 | i : dl[i]; },
        [&](uint32_t at, uint64_t v) { sel[at] = v; }, s);
    __syncthreads();
    block_sort_small(sel, width);
    for (uint32_t i = tid; i < k; i += kTopThreads) {
        const bool have = i < found;
        ids[(uint64_t)q * k + i] = have ? (uint64_t)(uint32_t)sel[i] : ~0ull;
        out[(uint64_t)q * k + i] = have ? f32_of_key((uint32_t)(sel[i] >> 32)) : __builtin_huge_valf();
    }
    if (count && tid == 0) count[q] = found;
}

// An empty table's answer.
__global__ void __launch_bounds__(256)
int4_topk_none_kernel(uint64_t *ids, float *out, uint32_t *count, uint64_t total, uint32_t nq) {
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
        ids[i] = ~0ull;
        out[i] = __builtin_huge_valf();
        if (count && i < nq) count[i] = 0;
    }
}

} // namespace cuddle
