// Runs the selection kernels of vectordb_amd/csrc/cuddle_rows_select.hpp on the CPU, thread by thread: a block is 1024
// fibers that switch at barriers and wave operations. Every buffer a kernel writes is followed by guard words.
// usage: select_on_host n k n_queries kind   (kind: random, ties, nan, collection); exit status 0 if all is as it should be.
#include <ucontext.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <random>
#include <vector>

#define __device__
#define __forceinline__ inline
#define __global__
#define __launch_bounds__(...)
#define __shared__ thread_local // static storage in a function, and "extern thread_local" is a declaration; there is one host thread

struct Index3 {
    uint32_t x, y;
};
static Index3 threadIdx, blockIdx, gridDim, blockDim;

namespace cuddle {
static void block_sync(), wave_sync_all();
static uint32_t g_lane[1024]; // what each thread put up for its wave
static inline uint32_t min(uint32_t a, uint32_t b) { return a < b ? a : b; }
static inline uint64_t min(uint64_t a, uint64_t b) { return a < b ? a : b; }
static inline uint32_t max(uint32_t a, uint32_t b) { return a > b ? a : b; }
static inline int __clz(int v) { return v ? __builtin_clz((unsigned)v) : 32; }
static inline int __popc(uint32_t v) { return __builtin_popcount(v); }
static inline uint32_t atomicAdd(uint32_t *p, uint32_t v) {
    const uint32_t o = *p;
    *p += v;
    return o;
}
static inline float __uint_as_float(uint32_t u) {
    float f;
    std::memcpy(&f, &u, 4);
    return f;
}
template <class F> static uint32_t wave_op(uint32_t v, F f) {
    const uint32_t t = threadIdx.x, b = t & ~63u;
    g_lane[t] = v;
    wave_sync_all();
    const uint32_t r = f(g_lane + b, t & 63);
    wave_sync_all();
    return r;
}
static inline int __shfl_xor(int v, int m, int) {
    return (int)wave_op((uint32_t)v, [&](const uint32_t *l, uint32_t i) { return l[i ^ (uint32_t)m]; });
}
static inline uint32_t wave_min_u32(uint32_t v) {
    return wave_op(v, [](const uint32_t *l, uint32_t) { return *std::min_element(l, l + 64); });
}
static inline uint32_t wave_inclusive_sum(uint32_t v) {
    return wave_op(v, [](const uint32_t *l, uint32_t i) {
        uint32_t s = 0;
        for (uint32_t j = 0; j <= i; ++j) s += l[j];
        return s;
    });
}
static inline void __syncthreads() { block_sync(); }
static inline uint32_t f32_key(float d) { // order of distances: the two zeros are one, NaN after everything
    if (d != d) return 0xFFFFFFFFu;
    uint32_t b;
    std::memcpy(&b, &d, 4);
    if ((b << 1) == 0u) b = 0u;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
static inline uint32_t next_pow2(uint32_t v) {
    uint32_t p = 1;
    while (p < v) p <<= 1;
    return p;
}
} // namespace cuddle

#include "cuddle_rows_select.hpp"

namespace cuddle {
thread_local uint32_t s_keys[36u << 10];

// ---- fibers --------------------------------------------------------------------------------------
enum class State { run, block, wave, done };
struct Fiber {
    ucontext_t ctx;
    State state;
    std::vector<char> stack;
};
static std::vector<Fiber> g_fibers(kTopThreads);
static ucontext_t g_main;
static uint32_t g_now;
static std::function<void()> g_body;

static void entry() {
    g_body();
    g_fibers[g_now].state = State::done;
    swapcontext(&g_fibers[g_now].ctx, &g_main);
}
static void wait_in(State s) {
    g_fibers[g_now].state = s;
    swapcontext(&g_fibers[g_now].ctx, &g_main);
}
static void block_sync() { wait_in(State::block); }
static void wave_sync_all() { wait_in(State::wave); }

static void run_block() {
    for (uint32_t i = 0; i < kTopThreads; ++i) {
        Fiber &f = g_fibers[i];
        if (f.stack.empty()) f.stack.resize(64 << 10);
        getcontext(&f.ctx);
        f.ctx.uc_stack.ss_sp = f.stack.data();
        f.ctx.uc_stack.ss_size = f.stack.size();
        f.ctx.uc_link = nullptr;
        makecontext(&f.ctx, entry, 0);
        f.state = State::run;
    }
    for (;;) {
        for (uint32_t i = 0; i < kTopThreads; ++i)
            if (g_fibers[i].state == State::run) {
                g_now = threadIdx.x = i;
                swapcontext(&g_main, &g_fibers[i].ctx);
            }
        bool any = false, all_block = true;
        for (uint32_t w = 0; w < kTopThreads; w += 64) { // waves whose threads have all come to a wave operation go on
            bool all = true;
            for (uint32_t i = w; i < w + 64; ++i) {
                all &= g_fibers[i].state == State::wave;
                all_block &= g_fibers[i].state == State::block;
            }
            if (!all) continue;
            any = true;
            for (uint32_t i = w; i < w + 64; ++i) g_fibers[i].state = State::run;
        }
        if (any) continue;
        if (all_block) {
            for (Fiber &f : g_fibers) f.state = State::run;
            continue;
        }
        for (Fiber &f : g_fibers)
            if (f.state != State::done) {
                std::printf("threads wait at different barriers\n");
                std::exit(2);
            }
        return;
    }
}
template <class F> static void launch(uint32_t gx, uint32_t gy, F f) {
    gridDim = {gx, gy};
    blockDim = {kTopThreads, 1};
    g_body = f;
    for (uint32_t y = 0; y < gy; ++y)
        for (uint32_t x = 0; x < gx; ++x) {
            blockIdx = {x, y};
            run_block();
        }
}

// ---- buffers with guards ---------------------------------------------------------------------------
template <class T> struct Guarded {
    static constexpr size_t kGuard = 4096;
    std::vector<T> v;
    size_t n;
    T mark;
    explicit Guarded(size_t n_) : v(n_ + kGuard), n(n_) {
        std::memset(&mark, 0xA5, sizeof(T));
        std::fill(v.begin(), v.end(), mark);
    }
    T *get() { return v.data(); }
    void check(const char *what) const {
        for (size_t i = n; i < v.size(); ++i)
            if (std::memcmp(&v[i], &mark, sizeof(T))) {
                std::printf("%s: written %zu places behind its end\n", what, i - n);
                std::exit(1);
            }
    }
};
} // namespace cuddle
using namespace cuddle;

int main(int argc, char **argv) {
    if (argc != 5) return 3;
    const uint64_t n = std::strtoull(argv[1], nullptr, 10);
    const uint32_t k = (uint32_t)std::atoi(argv[2]), nq = (uint32_t)std::atoi(argv[3]);
    const std::string kind = argv[4];
    std::mt19937 rng((uint32_t)(n * 31 + k));
    std::vector<float> dist((size_t)nq * n);
    for (float &d : dist) {
        d = kind == "ties" ? (float)(rng() % 3) : (float)(rng() % 1000003) * 1e-3f - 200.f;
        if (kind == "nan" && rng() % 10) d = std::nanf("");
    }
    Guarded<uint64_t> ids((size_t)nq * k);
    Guarded<float> out((size_t)nq * k);
    Guarded<uint32_t> count(nq);
    const uint32_t found = (uint32_t)std::min<uint64_t>(k, n);
    if (kind == "collection") { // all rows, in any order
        std::vector<uint64_t> list((size_t)nq * kTopChunk);
        std::vector<uint32_t> cnt(nq * kCountPitch);
        for (uint32_t q = 0; q < nq; ++q) {
            for (uint64_t i = 0; i < n; ++i) list[(size_t)q * kTopChunk + i] = (uint64_t)f32_key(dist[q * n + i]) << 32 | i;
            std::shuffle(list.begin() + (size_t)q * kTopChunk, list.begin() + (size_t)q * kTopChunk + n, rng);
            cnt[q * kCountPitch] = (uint32_t)n;
        }
        launch(nq, 1, [&] { int4_topk_final_kernel<2>(list.data(), kTopChunk, 0u, k, found, cnt.data(), kTopChunk, ids.get(), out.get(), count.get()); });
    } else { // the levels, as cuddle_int4_search_device enqueues them, each list buffer of the size it asks for
        std::vector<Guarded<uint64_t>> lists;
        const void *in = dist.data();
        uint64_t stride = n, items = n;
        int level = 0;
        for (; items > kTopChunk; ++level) {
            const uint32_t chunk = level == 0 ? top_chunk(items, nq, k) : kTopChunk;
            const uint32_t parts = (uint32_t)((items + chunk - 1) / chunk);
            lists.emplace_back((size_t)nq * parts * k);
            uint64_t *o = lists.back().get();
            launch(parts, nq, [&] {
                if (level == 0) int4_topk_level_kernel<true>(in, stride, items, k, chunk, parts, o, nullptr, kTopChunk);
                else int4_topk_level_kernel<false>(in, stride, items, k, chunk, parts, o, nullptr, kTopChunk);
            });
            lists.back().check("a level's lists");
            in = o;
            stride = items = (uint64_t)parts * k;
        }
        launch(nq, 1, [&] {
            if (level == 0) int4_topk_final_kernel<0>(in, stride, (uint32_t)items, k, found, nullptr, kTopChunk, ids.get(), out.get(), count.get());
            else int4_topk_final_kernel<1>(in, stride, (uint32_t)items, k, found, nullptr, kTopChunk, ids.get(), out.get(), count.get());
        });
    }
    ids.check("ids");
    out.check("distances");
    count.check("counts");
    for (uint32_t q = 0; q < nq; ++q) {
        std::vector<uint64_t> want(n);
        for (uint64_t i = 0; i < n; ++i) want[i] = (uint64_t)f32_key(dist[q * n + i]) << 32 | i;
        std::partial_sort(want.begin(), want.begin() + found, want.end());
        for (uint32_t i = 0; i < k; ++i) {
            const uint64_t id = ids.get()[(size_t)q * k + i];
            const float d = out.get()[(size_t)q * k + i];
            const bool ok = i < found ? id == (uint32_t)want[i] && f32_key(d) == (uint32_t)(want[i] >> 32) : id == ~0ull && d == INFINITY;
            if (!ok) {
                std::printf("query %u place %u: row %llu, distance %g\n", q, i, (unsigned long long)id, (double)d);
                return 1;
            }
        }
        if (count.get()[q] != found) return 1;
    }
    return 0;
}
