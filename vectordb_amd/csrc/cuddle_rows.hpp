// cuddle_rows.hpp — an embedding table on the device: 4-bit rows with group scales (encoding, decoding, distances of
// a few queries to every row, exhaustive top-k), row lookup by id, and the gradient of that lookup.
// No counterpart in the reference, whose codes are 1-bit (src/quantization/binary.rs, rabitq.rs) and whose rows are
// fetched one at a time (MmapVectorStore::get, src/storage/mmap.rs:106-115).
//
// 4-bit rows. A row's components are cut into groups of G (32, 64 or 128); group g has the scale
//   s = bf16(max|x| / 7)   and the codes   c = rint(x / s) (halves to even, clamped to -7..7),   and stands for s * c.
// A group whose scale rounds to zero has codes 0; a group that holds a NaN or an infinity gets s = NaN and codes 0,
// so it decodes to NaN and every distance of the row is NaN.
//
// Layout. What a wave wants to load is what matrix instructions eat: 16 rows x 64 components of int8 each, lane
// (r = lane & 15, h = lane >> 4) holding 16 components of row r. So codes are stored by tiles of 16 rows and units of 64
// components, 8 bytes of a unit per lane: byte i = component 8h + i in the low nibble, 32 + 8h + i in the high nibble
// (i < 8), two's complement. Units come in pairs of 1024 bytes,
//   byte r * 64 + h * 16 + (unit & 1) * 8 + i,
// so that a wave reads 16 bytes per lane, 1 KB in a run, and a row has 64 bytes in a run (fetching a row by id: half the
// lines that single units of 32 bytes a row would touch). An odd last unit has 512 bytes, byte r * 32 + h * 8 + i. The
// operand is made with a shift and two masks; the code stays in the high nibble of its byte, so the products come out 16 times too large
// (an exact factor, taken out at the end). Scales are row-major: [rows][gstride] bf16; gstride is the number of groups
// rounded up to 2, 4 or 8, so that the scales of neighbouring units come in one aligned load.
#pragma once

#include "cuddle_kernels.hpp"
#include "cuddle_rows_plan.hpp"
#include "cuddle_rows_select.hpp"

namespace cuddle {

typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));

constexpr uint32_t kTypeF32 = 0, kTypeF16 = 1, kTypeBF16 = 2;
// Offset in a tile of byte b = 8h + i of row r's unit u.
__device__ __forceinline__ uint32_t int4_code_at(uint32_t units, uint32_t u, uint32_t r, uint32_t b) {
    if (u == units - 1 && !(u & 1)) return u * kInt4UnitBytes + r * 32 + b;
    return (u >> 1) * (2 * kInt4UnitBytes) + r * 64 + (b >> 3) * 16 + (u & 1) * 8 + (b & 7);
}

// ---- element types ---------------------------------------------------------------------------
struct Bf16 { uint16_t b; };
__device__ __forceinline__ float bf16_to_f32(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
__device__ __forceinline__ uint16_t f32_to_bf16(float f) { // to nearest, halves to even; NaN stays NaN
    const uint32_t u = __float_as_uint(f);
    if (f != f) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(Bf16 v) { return bf16_to_f32(v.b); }
template <class T> __device__ __forceinline__ T from_f32(float f);
template <> __device__ __forceinline__ float from_f32<float>(float f) { return f; }
// The value as it stands, then rounded: without the barrier the compiler folds a product before it and this rounding
// into one mixed-precision instruction, whose single rounding is not the product's f32 rounding followed by this one.
template <> __device__ __forceinline__ _Float16 from_f32<_Float16>(float f) {
    asm("" : "+v"(f));
    return (_Float16)f;
}
template <> __device__ __forceinline__ Bf16 from_f32<Bf16>(float f) { return Bf16{f32_to_bf16(f)}; }

// N consecutive elements moved as one piece (the caller has checked the alignment).
template <class T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };

// Eight consecutive components of a row as f32, zeros from `dim` on.
template <class T, bool VEC>
__device__ __forceinline__ void load8(const T *row, uint32_t e0, uint32_t dim, float (&x)[8]) {
    if (VEC && e0 + 8 <= dim) {
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int p = 0; p < 8 / N; ++p) {
            const Pack<T, N> v = *reinterpret_cast<const Pack<T, N> *>(row + e0 + p * N);
#pragma unroll
            for (int i = 0; i < N; ++i) x[p * N + i] = to_f32(v.v[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = e0 + i < dim ? to_f32(row[e0 + i]) : 0.f;
    }
}

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------------------------
// encoding
// ---------------------------------------------------------------------------------------------
// The code of x under scale s > 0 (inv = 1 / s, or 0 where that overflows): rint(x / s), exactly. s has 8 significant
// bits and |n| <= 8, so n * s is exact; x - n * s is a multiple of the last place of x and no larger than x (or s),
// so the fma returns it exactly and comparing it with s / 2 decides the rounding, whatever the estimate n was off by.
__device__ __forceinline__ float int4_code(float x, float s, float inv) {
    float n = rintf(inv != 0.f ? x * inv : x / s);
    n = fminf(fmaxf(n, -8.f), 8.f);
    const float r = __builtin_fmaf(-n, s, x), h = 0.5f * s;
    if (fabsf(r) > h || (fabsf(r) == h && ((int32_t)n & 1))) n += r > 0.f ? 1.f : -1.f;
    return fminf(fmaxf(n, -7.f), 7.f);
}
constexpr float kInt4Magic = 12582912.f; // 1.5 * 2^23: x + this is rint(x) in the low bits of the sum

// LPR lanes per row (16: one tile of 16 rows per block, 64: four rows); a lane has 8 consecutive components, so the lanes
// of a row LPR / 8 units per step. The group's largest magnitude is a reduction over G / 8 neighbouring lanes; the low
// and the high nibbles of a byte come from lanes 4 apart. Rows outside [first, first + count) are left alone.
// sqnorm[r] = sum over groups of s^2 * sum c^2 in f64 (the integer sums are exact).
// Bound by the read of the rows. grid = blocks of 256 / LPR rows (x stride), block 256.
template <class T, bool VEC, int LPR>
__global__ void __launch_bounds__(256)
int4_encode_kernel(const T *x, uint64_t stride, uint64_t first, uint64_t count, uint32_t dim, uint32_t group, uint8_t *codes,
                   uint16_t *scales, double *sqnorm, uint64_t blocks) {
    constexpr uint32_t RPB = 256 / LPR, UPS = LPR / 8; // rows per block, units per step
    const uint32_t units = int4_units(dim), gs = int4_gstride(dim, group), lr = threadIdx.x & (LPR - 1);
    const uint32_t jj = lr & 7;
    for (uint64_t bl = first / RPB + blockIdx.x; bl < first / RPB + blocks; bl += gridDim.x) {
        const uint64_t row = bl * RPB + threadIdx.x / LPR, t = row >> 4;
        const uint32_t r = (uint32_t)row & 15;
        const bool act = row >= first && row < first + count;
        const T *src = x + (act ? row - first : 0) * stride;
        double sq = 0.0;
        float next[8]; // the next step's components are on their way while these are worked on
        if (act) load8<T, VEC>(src, (lr >> 3) * kInt4Unit + jj * 8, dim, next);
        for (uint32_t u0 = 0; u0 < units; u0 += UPS) {
            const uint32_t u = u0 + (lr >> 3), e0 = u * kInt4Unit + jj * 8;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = act ? next[i] : 0.f;
            if (act && u0 + UPS < units) load8<T, VEC>(src, e0 + UPS * kInt4Unit, dim, next);
            uint32_t ab = 0; // largest magnitude by its bits: infinities and NaN are above every number
#pragma unroll
            for (int i = 0; i < 8; ++i) ab = max(ab, __float_as_uint(v[i]) & 0x7FFFFFFFu);
            ab = max(ab, (uint32_t)__shfl_xor((int)ab, 1, 64));
            ab = max(ab, (uint32_t)__shfl_xor((int)ab, 2, 64));
            if (group >= 64) ab = max(ab, (uint32_t)__shfl_xor((int)ab, 4, 64));
            if (group >= 128) ab = max(ab, (uint32_t)__shfl_xor((int)ab, 8, 64));
            const bool bad = ab >= 0x7F800000u;
            const uint16_t sb = bad ? (uint16_t)0x7FC0u : f32_to_bf16(__uint_as_float(ab) / 7.0f);
            const float s = bf16_to_f32(sb);
            // s of a normal size: |x| / s <= 7 (1 + 2^-8), so rint gives at most 7 and only remainders of half a step or
            // more need the exact decision
            const float inv = s >= 1e-30f ? 1.0f / s : 0.f;
            float mg[8], worst = 0.f, c2 = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                mg[i] = __builtin_fmaf(v[i], inv, kInt4Magic);
                const float n = mg[i] - kInt4Magic;
                worst = fmaxf(worst, fabsf(__builtin_fmaf(-n, s, v[i])));
                c2 = __builtin_fmaf(n, n, c2);
            }
            if (bad || inv == 0.f || worst >= 0.5f * s) {
                c2 = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float n = (bad || s == 0.f) ? 0.f : int4_code(v[i], s, inv);
                    mg[i] = n + kInt4Magic;
                    c2 = __builtin_fmaf(n, n, c2);
                }
            }
            sq = __builtin_fma((double)s * (double)s, (double)c2, sq);
            // the low nibbles of the sums are the codes: bytes 0 of four of them side by side
            auto pack = [&](int i) {
                const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(mg[i + 1]), __float_as_uint(mg[i]), 0x0C0C0400u);
                const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(mg[i + 3]), __float_as_uint(mg[i + 2]), 0x04000C0Cu);
                return (lo | hi) & 0x0F0F0F0Fu;
            };
            const uint32_t p0 = pack(0), p1 = pack(4);
            const uint32_t q0 = (uint32_t)__shfl_xor((int)p0, 4, 64), q1 = (uint32_t)__shfl_xor((int)p1, 4, 64);
            if (act && u < units) {
                if (jj < 4)
                    *reinterpret_cast<uint2 *>(codes + t * units * kInt4UnitBytes + int4_code_at(units, u, r, jj * 8)) = make_uint2(p0 | q0 << 4, p1 | q1 << 4);
                const uint32_t g = e0 / group;
                if (e0 % group == 0 && g < gs) scales[row * gs + g] = sb;
            }
        }
        // padding groups of the scales' row that no lane above stands for
        if (act && lr < 8) {
            const uint32_t g = (units * kInt4Unit + group - 1) / group + lr;
            if (g < gs) scales[row * gs + g] = 0;
        }
#pragma unroll
        for (int m = 1; m < LPR; m <<= 1) sq += __shfl_xor(sq, m, 64);
        if (act && lr == 0) sqnorm[row] = sq;
    }
}

// ---------------------------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------------------------
// ids: 32- or 64-bit, signed; anything outside [0, n) gives `none`.
constexpr uint64_t kNoRow = ~0ull;
template <class I>
__device__ __forceinline__ uint64_t row_of_id(const I *ids, uint64_t t, uint64_t n) {
    const int64_t i = (int64_t)ids[t];
    return i >= 0 && (uint64_t)i < n ? (uint64_t)i : kNoRow;
}

// out[t] = scale * table[ids[t]]. A thread has one piece of N elements (column blockIdx.y * w + ...) of every rpi-th of
// the block's rpb outputs, four of them in flight: ids, then rows, then the stores. Bound by the writes (and by the reads
// where the rows are not found in a cache).
template <class T, class I, int N>
__global__ void __launch_bounds__(256)
rows_lookup_kernel(const T *table, uint64_t stride, uint64_t n, uint32_t dim, const I *ids, uint64_t n_ids, float scale, T *out, uint32_t w, uint32_t rpi,
                   uint32_t rpb) {
    const uint32_t rr = threadIdx.x / w, col = (blockIdx.y * w + threadIdx.x - rr * w) * N;
    if (rr >= rpi || col >= dim) return;
    constexpr int U = 4;
    for (uint64_t t0 = (uint64_t)blockIdx.x * rpb; t0 < n_ids; t0 += (uint64_t)gridDim.x * rpb) {
        const uint64_t te = min(t0 + rpb, n_ids);
        for (uint64_t t1 = t0 + rr; t1 < te; t1 += U * rpi) {
            uint64_t row[U];
            Pack<T, N> v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) row[u] = t1 + u * rpi < te ? row_of_id(ids, t1 + u * rpi, n) : kNoRow;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (row[u] != kNoRow)
                    v[u] = *reinterpret_cast<const Pack<T, N> *>(table + row[u] * stride + col);
                else
#pragma unroll
                    for (int i = 0; i < N; ++i) v[u].v[i] = from_f32<T>(0.f);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (t1 + u * rpi >= te) continue;
                if (row[u] != kNoRow)
#pragma unroll
                    for (int i = 0; i < N; ++i) v[u].v[i] = from_f32<T>(to_f32(v[u].v[i]) * scale);
                *reinterpret_cast<Pack<T, N> *>(out + (t1 + u * rpi) * dim + col) = v[u];
            }
        }
    }
}

// The same from 4-bit rows: a piece is what 16 bytes of output hold, one nibble of each of N bytes (threads 32 components
// apart share the bytes). s * c has 12 significant bits, so only the product with `scale` and the rounding to the output's
// type round. ids == nullptr: rows 0 .. n_ids - 1 in order, one at a time (U = 1), written without a claim to a cache.
template <class T, class I, bool VEC, int U>
__global__ void __launch_bounds__(256)
int4_lookup_kernel(const uint8_t *codes, const uint16_t *scales, uint64_t n, uint32_t dim, uint32_t group, const I *ids, uint64_t n_ids, float scale,
                   T *out, uint32_t w, uint32_t rpi, uint32_t rpb) {
    constexpr int N = 16 / sizeof(T), W = N / 4; // components, words of codes
    const uint32_t units = int4_units(dim), gs = int4_gstride(dim, group), rr = threadIdx.x / w, e0 = (blockIdx.y * w + threadIdx.x - rr * w) * N;
    if (rr >= rpi || e0 >= dim) return;
    const uint32_t e6 = e0 & 63, g = e0 / group, up = e6 < 32 ? 4 : 0;
    const uint32_t code_at = int4_code_at(units, e0 >> 6, 0, e6 & 31), pitch = int4_code_at(units, e0 >> 6, 1, e6 & 31) - code_at; // bytes between rows
    for (uint64_t t0 = (uint64_t)blockIdx.x * rpb; t0 < n_ids; t0 += (uint64_t)gridDim.x * rpb) {
        const uint64_t te = min(t0 + rpb, n_ids);
        for (uint64_t t1 = t0 + rr; t1 < te; t1 += U * rpi) {
            uint64_t row[U];
            Pack<uint32_t, W> c[U];
            uint16_t sb[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint64_t t = t1 + u * rpi;
                row[u] = t >= te ? kNoRow : ids ? row_of_id(ids, t, n) : t;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int i = 0; i < W; ++i) c[u].v[i] = 0;
                sb[u] = 0;
                if (row[u] != kNoRow) {
                    c[u] = *reinterpret_cast<const Pack<uint32_t, W> *>(codes + (row[u] >> 4) * units * kInt4UnitBytes + (uint32_t)(row[u] & 15) * pitch + code_at);
                    sb[u] = scales[row[u] * gs + g];
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (t1 + u * rpi >= te) continue;
                const float s = bf16_to_f32(sb[u]);
                Pack<T, N> o;
#pragma unroll
                for (int i = 0; i < N; ++i) o.v[i] = from_f32<T>(s * (float)((int32_t)((c[u].v[i / 4] << up) << (24 - 8 * (i & 3))) >> 28) * scale);
                T *dst = out + (t1 + u * rpi) * dim + e0;
                if (VEC && U == 1) {
                    u32x4_t b;
                    __builtin_memcpy(&b, &o, 16);
                    __builtin_nontemporal_store(b, reinterpret_cast<u32x4_t *>(dst));
                } else if (VEC)
                    *reinterpret_cast<Pack<T, N> *>(dst) = o;
                else
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (e0 + i < dim) dst[i] = o.v[i];
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------
// distances of queries to 4-bit rows
// ---------------------------------------------------------------------------------------------
// The query side of the products. A query is written in fixed point, q_i = Q_i * 2^(e - 30) with |Q_i| <= 2^30, e from
// its largest magnitude, and Q_i as four signed base-256 digits: with the codes as they are, every product and every
// sum over a group is then an exact integer product of int8 on the matrix cores. What is rounded is q_i itself, by at
// most 2^-31 of the largest |q| - f16 and bf16 queries, and whole numbers, not at all in practice.
// Operand order: [query quartet][unit][lane][16 bytes], lane = (h << 4) | (query & 3) << 2 | digit, byte b = component
// 8h + b (b < 8) or 32 + 8h + b - 8 of the unit.
struct Int4Query {
    double scale; // value of one unit of the products' last place, 2^(e - 34); NaN for a query with a non-finite value
    double sq;    // |q|^2
};

template <class T>
__global__ void __launch_bounds__(256)
int4_query_kernel(const T *queries, uint32_t nq, uint32_t dim, uint32_t units, uint8_t *dig, Int4Query *info) {
    __shared__ float s_max[4];
    __shared__ double s_sq[4];
    const uint32_t q = blockIdx.x, tid = threadIdx.x;
    const bool real = q < nq; // the last quartet is filled up with zero queries
    const T *src = queries + (uint64_t)(real ? q : 0) * dim;
    float m = 0.f;
    double sq = 0.0;
    if (real)
        for (uint32_t i = tid; i < dim; i += 256) {
            const float v = to_f32(src[i]), a = fabsf(v);
            m = fmaxf(m, a <= 3.4028234663852886e38f ? a : __builtin_huge_valf());
            sq = __builtin_fma((double)v, (double)v, sq);
        }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        m = fmaxf(m, __shfl_xor(m, d, 64));
        sq += __shfl_xor(sq, d, 64);
    }
    if ((tid & 63) == 0) {
        s_max[tid >> 6] = m;
        s_sq[tid >> 6] = sq;
    }
    __syncthreads();
    m = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    const bool bad = m > 3.4028234663852886e38f;
    int e = 0;
    if (!bad && m > 0.f) (void)frexp((double)m, &e);
    const double up = ldexp(1.0, 30 - e);
    if (tid == 0 && real) info[q] = Int4Query{bad ? __builtin_nan("") : ldexp(1.0, e - 34), (s_sq[0] + s_sq[1]) + (s_sq[2] + s_sq[3])};
    uint8_t *dst = dig + (uint64_t)(q >> 2) * units * 1024;
    for (uint32_t i = tid; i < units * kInt4Unit; i += 256) {
        const float v = real && i < dim && !bad ? to_f32(src[i]) : 0.f;
        int32_t f = (int32_t)rint((double)v * up);
        const uint32_t u = i >> 6, e6 = i & 63, h = (e6 & 31) >> 3, b = ((e6 >> 5) << 3) | (e6 & 7);
#pragma unroll
        for (uint32_t d = 0; d < 4; ++d) {
            const int32_t lo = (int32_t)(int8_t)(f & 255);
            f = (f - lo) >> 8;
            dst[(uint64_t)u * 1024 + ((h << 4) | ((q & 3) << 2) | d) * 16 + b] = (uint8_t)lo;
        }
    }
}

// 1 / sqrt(z) in f64: the hardware's estimate, refined twice (each step squares its error and trebles a half of it).
__device__ __forceinline__ double inv_sqrt(double z) {
    double y = __builtin_amdgcn_rsq(z);
    y = __builtin_fma(y * 0.5, __builtin_fma(-z * y, y, 1.0), y);
    return __builtin_fma(y * 0.5, __builtin_fma(-z * y, y, 1.0), y);
}

// distance from the product p = scale * sum: l2 |x|^2 + |q|^2 - 2p, cosine 1 - p / (|x||q|), dot -p; in f64, rounded once.
__device__ __forceinline__ float int4_finish(uint32_t metric, double sum, double scale, double xsq, double qsq) {
    if (metric == kMetricDot) return (float)(-scale * sum);
    if (metric == kMetricCosine) return (float)__builtin_fma(-scale * sum, inv_sqrt(xsq * qsq), 1.0); // the squares of f32 norms multiply within f64's range
    const float d = (float)__builtin_fma(-2.0 * scale, sum, xsq + qsq);
    return d < 0.f ? 0.f : d; // the three terms of a row next to the query round apart
}

// The digits of one quartet of queries, made by a block of 256 threads straight into LDS: what int4_query_kernel writes,
// for blocks that need a single quartet and hold all of it. Every wave has a quarter of the units of every query, so that
// a lone query is read in one trip. Units from ceil(dim / 64) to `pad` and queries from nq on are zero.
template <class TQ>
__device__ __forceinline__ void int4_block_digits(const TQ *queries, uint32_t nq, uint32_t dim, uint32_t pad, uint8_t *dig, Int4Query *info) {
    __shared__ float s_max[4][4];
    __shared__ double s_sq[4][4];
    const uint32_t w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    constexpr int U = 8; // units read at a time
    auto read8 = [&](const TQ *src, uint32_t u0, float (&v)[U]) {
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const uint32_t i = (u0 + 4 * j) * 64 + lane;
            v[j] = i < dim ? to_f32(src[i]) : 0.f;
        }
    };
    for (uint32_t q = 0; q < nq; ++q) {
        float m = 0.f;
        double sq = 0.0;
        for (uint32_t u0 = w; u0 * 64 < dim; u0 += 4 * U) {
            float v[U];
            read8(queries + (uint64_t)q * dim, u0, v);
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const float a = fabsf(v[j]);
                m = fmaxf(m, a <= 3.4028234663852886e38f ? a : __builtin_huge_valf());
                sq = __builtin_fma((double)v[j], (double)v[j], sq);
            }
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            m = fmaxf(m, __shfl_xor(m, d, 64));
            sq += __shfl_xor(sq, d, 64);
        }
        if (lane == 0) {
            s_max[q][w] = m;
            s_sq[q][w] = sq;
        }
    }
    __syncthreads();
    const uint32_t h = (lane & 31) >> 3, b = ((lane >> 5) << 3) | (lane & 7); // the lane's component of every unit
    for (uint32_t q = 0; q < 4; ++q) {
        const bool real = q < nq;
        const float m = real ? fmaxf(fmaxf(s_max[q][0], s_max[q][1]), fmaxf(s_max[q][2], s_max[q][3])) : 0.f;
        const bool bad = m > 3.4028234663852886e38f;
        int e = 0;
        if (!bad && m > 0.f) (void)frexp((double)m, &e);
        const double up = ldexp(1.0, 30 - e);
        if (threadIdx.x == 0)
            info[q] = Int4Query{bad ? __builtin_nan("") : ldexp(1.0, e - 34), real ? (s_sq[q][0] + s_sq[q][1]) + (s_sq[q][2] + s_sq[q][3]) : 0.0};
        for (uint32_t u0 = w; u0 < pad; u0 += 4 * U) {
            float v[U];
            if (real)
                read8(queries + (uint64_t)q * dim, u0, v);
            else
#pragma unroll
                for (int j = 0; j < U; ++j) v[j] = 0.f;
#pragma unroll
            for (int j = 0; j < U; ++j) {
                if (u0 + 4 * j >= pad) break;
                int32_t f = (int32_t)rint((double)(bad ? 0.f : v[j]) * up);
#pragma unroll
                for (uint32_t d = 0; d < 4; ++d) {
                    const int32_t lo = (int32_t)(int8_t)(f & 255);
                    f = (f - lo) >> 8;
                    dig[(u0 + 4 * j) * 1024 + ((h << 4) | (q << 2) | d) * 16 + b] = (uint8_t)lo;
                }
            }
        }
    }
}

// The running sum of one (row, query) pair gains one group: c = the integer products of the four digits, put together
// exactly (42 bits), times the group's scale. In f64 throughout: an f32 part for the lower digits would overflow where rows
// are large, and measured no faster.
__device__ __forceinline__ double int4_add(double acc, i32x4_t c, double s) {
    return __builtin_fma(s, __builtin_fma((double)(c[2] + (c[3] << 8)), 65536.0, (double)(c[0] + (c[1] << 8))), acc);
}

struct Int4DistArgs {
    const uint8_t *codes;
    const uint16_t *scales;
    const double *sqnorm;
    uint64_t n;
    uint32_t dim, units, gs;
    const void *queries;     // FUSED: the queries themselves
    const uint8_t *dig;      // otherwise their digits and scalars (int4_query_kernel)
    const Int4Query *info;
    uint32_t nq, metric;
    float *dist;
    uint64_t dstride;
    uint32_t ku;             // units of digits in LDS at a time, a multiple of P
    uint32_t xs, ys;         // blocks along the rows (a multiple of 8 if ys > 1) and along the queries
    // search: either a sample of the tiles (dist[q][16 i + r] = row r of the i-th sampled tile, NaN past the last row) ...
    uint64_t stiles;         // tiles to visit: all, or the sample
    uint32_t stride;         // 0, or a sampled tile out of every `stride`
    // ... or the candidates: rows whose key does not exceed tau[q] go to list[q][cap] in any order, cnt[q * kCountPitch] counts them
    const uint32_t *tau;
    uint32_t *cnt;
    uint64_t *list;
    uint32_t cap;
    const uint32_t *redo;    // nullptr, or the counts: only queries that have more than `cap` are wanted
};

struct Int4Held { uint32_t key, row, q; };

// The candidates' pass asks of nearly every (row, query) pair only whether its distance is beyond the bound, and f32
// answers that where it is not close. With S = the sum rounded to f32 a distance is t = A * S * R + B plus a constant of
// the query: l2 A = -2 scale, B = |x|^2; dot A = -scale; cosine A = -scale / |q|, R = 1 / |x|. |S| scale <= |x||q|, at most
// (|x|^2 + |q|^2) / 2, and each of fewer than eight roundings is at most 2^-24 of one of the terms: for l2 they stay below
// 2^-20 (|x|^2 + |q|^2), for cosine below 2^-20, taken off B and added to C = bound - constant beforehand, twice over.
// dot has no such measure at hand: S is moved by 2^-20 of itself. t > C: surely beyond. What is not a number, or too
// large or small for f32, is not "beyond" and goes on to the exact evaluation.
struct Int4Test {
    float A, C;
};
__device__ __forceinline__ Int4Test int4_test(uint32_t metric, uint32_t tau, const Int4Query &q) {
    constexpr double up = 1.0 / (1 << 19);
    const Int4Test all{0.f, __builtin_huge_valf()}; // every pair goes on
    if (tau >= 0xFF800000u) return all; // bound +inf or NaN
    const double t = (double)__uint_as_float(tau & 0x80000000u ? tau & 0x7FFFFFFFu : ~tau);
    const double A = metric == kMetricDot ? -q.scale : metric == kMetricCosine ? -q.scale / sqrt(q.sq) : -2.0 * q.scale;
    const double c = metric == kMetricDot ? 0.0 : metric == kMetricCosine ? 1.0 : q.sq, mag = fabs(t) + c;
    if (!(fabs(A) > 1e-30 && fabs(A) < 1e30 && mag < 1e30)) return all;
    return Int4Test{(float)A, (float)(t - c + up * mag)};
}
// Row side: B lowered, R; NaN beyond f32's range.
__device__ __forceinline__ float int4_test_row(uint32_t metric, double xsq) {
    if (metric == kMetricDot) return 0.f;
    if (!(xsq < 1e30 && xsq > 1e-30)) return __builtin_nanf("");
    return metric == kMetricCosine ? (float)inv_sqrt(xsq) : (float)(xsq * (1.0 - 1.0 / (1 << 19)));
}
template <uint32_t METRIC>
__device__ __forceinline__ bool int4_beyond(double sum, const Int4Test &q, float row) {
    float S = (float)sum;
    if (METRIC == kMetricL2) return __builtin_fmaf(q.A, S, row) > q.C;
    if (METRIC == kMetricCosine) return q.A * (S * row) > q.C;
    S = __builtin_fmaf(fabsf(S), 0x1p-20f, S); // A < 0: a larger S is a smaller t
    const float t = q.A * S;
    return t > q.C && t < 3.0e38f;
}

// The i-th sampled tile: one of every `stride`, at a place that varies from one to the next (no period of the rows'
// order can hide from it).
__device__ __forceinline__ uint64_t int4_sampled(uint64_t i, uint32_t stride) {
    uint32_t x = (uint32_t)i * 2654435761u;
    x ^= x >> 15;
    x *= 2246822519u;
    x ^= x >> 13;
    return i * stride + (uint32_t)(((uint64_t)x * stride) >> 32);
}

// Distances. A wave takes T tiles of 16 rows against QT quartets of queries; codes are the B operand (a lane has one
// row), digits the A operand, so a lane receives the four digits of one (row, query) pair and puts them together itself.
// The digits sit in LDS, all of them where they fit (loaded, or with FUSED made, once per block: few queries then take
// one launch), else `ku` units at a time. Codes and scales of P units and T tiles are requested together; units past
// the end repeat the last one against zero digits.
// Few queries: bound by the codes' read. Many: by the six vector instructions that a group's products cost per pair
// (two integer, two conversions, two f64 fma): about 21 cycles, and 16 of the matrix instruction, that overlap little.
// NT: codes that no cache holds until the next call are read without a claim to one (4 GiB: 6.3 -> 7.2 TB/s).
// Blocks of the same rows and different queries are neighbours on one XCD, so that the rows' codes come from its L2.
template <int G, int QT, int T, int P, bool FUSED, bool NT, class TQ>
__global__ void __launch_bounds__(int4_block(QT, T), QT >= 3 ? 4 : 2) // at most 256 registers: products land in vector registers, not accumulators
int4_distance_kernel(Int4DistArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t s_dig[];
    Int4Query *s_info = reinterpret_cast<Int4Query *>(s_dig + (size_t)a.ku * QT * 1024);
    constexpr uint32_t NW = int4_block(QT, T) / 64;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tid = threadIdx.x, lane = tid & 63, r = lane & 15, h = lane >> 4;
    uint32_t x = blockIdx.x, y = 0;
    if (a.ys > 1) {
        const uint32_t j = blockIdx.x >> 3;
        y = j % a.ys;
        x = (j / a.ys) * 8 + (blockIdx.x & 7);
    }
    const uint64_t tiles = (a.n + 15) / 16, groups = (a.stiles + NW * T - 1) / (NW * T);
    uint32_t *s_tau = reinterpret_cast<uint32_t *>(s_info + QT * 4);
    Int4Test *s_test = reinterpret_cast<Int4Test *>(s_tau + QT * 4);
    if (a.redo) { // uniform over the block
        bool any = false;
        for (uint32_t q = y * QT * 4; q < min((y + 1) * QT * 4, a.nq); ++q) any |= a.redo[q * kCountPitch] > a.cap;
        if (!any) return;
    }
    if (a.tau && tid < QT * 4) s_tau[tid] = a.tau[min(y * QT * 4 + tid, a.nq - 1)];
    // Candidates wait in LDS, the wave's own 128 places, and go out 64 at a time: one trip to the counters for 64 of them
    // instead of one for each.
    Int4Held *s_held = reinterpret_cast<Int4Held *>(s_test + QT * 4) + wave * 128;
    uint32_t held = 0;
    auto wave_sync = []() {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    auto flush = [&](uint32_t count) { // the first `count` <= 64
        if (lane < count) {
            const Int4Held c = s_held[lane];
            const uint32_t at = atomicAdd(&a.cnt[c.q * kCountPitch], 1u);
            if (at < a.cap) a.list[(uint64_t)c.q * a.cap + at] = (uint64_t)c.key << 32 | c.row;
        }
    };
    auto keep = [&](bool take, uint32_t key, uint32_t row, uint32_t q) { // all lanes of the wave call
        const uint64_t m = __ballot(take);
        if (!m) return;
        if (take) s_held[held + (uint32_t)__popcll(m & lanemask_lt())] = Int4Held{key, row, q};
        held += (uint32_t)__popcll(m);
        wave_sync();
        if (held >= 64) {
            flush(64);
            wave_sync();
            held -= 64;
            if (lane < held) s_held[lane] = s_held[64 + lane];
            wave_sync();
        }
    };
    const uint64_t out_at = h * a.dstride + r;
    auto load_digits = [&](uint32_t u0) { // digits of units [u0, u0 + ku): [unit][quartet][1 KB]
        const uint32_t cnt = min(a.ku, a.units - u0), quads = (a.nq + 3) / 4;
        for (uint32_t i = tid; i < a.ku * QT * 64; i += NW * 64) {
            const uint32_t u = i / (QT * 64), q = i / 64 % QT, qq = y * QT + q;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (u < cnt && qq < quads) v = reinterpret_cast<const uint4 *>(a.dig)[((uint64_t)qq * a.units + u0 + u) * 64 + (i & 63)];
            reinterpret_cast<uint4 *>(s_dig)[i] = v;
        }
    };
    if (FUSED)
        int4_block_digits(static_cast<const TQ *>(a.queries), a.nq, a.dim, a.ku, s_dig, s_info);
    else {
        if (tid < QT * 4) s_info[tid] = y * QT * 4 + tid < a.nq ? a.info[y * QT * 4 + tid] : Int4Query{0.0, 0.0};
        if (a.units <= a.ku) load_digits(0);
    }
    __syncthreads();
    if (a.tau) {
        if (tid < QT * 4) // places past the last query: nothing passes
            s_test[tid] = y * QT * 4 + tid < a.nq ? int4_test(a.metric, s_tau[tid], s_info[tid]) : Int4Test{0.f, -__builtin_huge_valf()};
        __syncthreads();
    }
    constexpr int SC = int4_scales(P, G);
    struct Piece {
        uint2 w[T][P];
        Pack<uint16_t, SC> sc[T];
    };
    const uint32_t pair_at = r * 64 + h * 16, single_at = r * 32 + h * 8;
    auto request = [&](uint64_t g, uint32_t ub, Piece &v) {
#pragma unroll
        for (int t = 0; t < T; ++t) { // tile and pointers are the wave's, only the offsets are the lane's
            const uint64_t i = (g * NW + wave) * T + t, tile = min(a.stride ? int4_sampled(i, a.stride) : i, tiles - 1);
            const uint8_t *wp = a.codes + tile * a.units * kInt4UnitBytes;
            const uint8_t *sp = reinterpret_cast<const uint8_t *>(a.scales + tile * 16 * a.gs);
            const uint32_t so = min(r, (uint32_t)min(a.n - 1 - tile * 16, (uint64_t)15)) * a.gs * 2; // rows past the last: the last
#pragma unroll
            for (int p = 0; p < P; p += 2) { // a pair of units; of an odd last one the second half is not its own and meets zero digits
                const uint32_t u = min(ub + p, (a.units - 1) & ~1u);
                const uint8_t *at = wp + (uint64_t)u * kInt4UnitBytes + (u == a.units - 1 ? single_at : pair_at);
                typedef uint32_t u32x4_8 __attribute__((ext_vector_type(4), aligned(8)));
                const u32x4_8 b = NT ? __builtin_nontemporal_load(reinterpret_cast<const u32x4_8 *>(at)) : *reinterpret_cast<const u32x4_8 *>(at);
                v.w[t][p] = make_uint2(b[0], b[1]);
                v.w[t][p + 1] = make_uint2(b[2], b[3]);
            }
            v.sc[t] = *reinterpret_cast<const Pack<uint16_t, SC> *>(sp + 2 * (ub * 64 / G) + so); // gs is a multiple of SC (checked at the launch): these are the row's own
        }
    };
    // The next piece is on its way while this one is worked on. Few queries from a cache: the waves cover for each other
    // (50K x 1536: 13.7 us without, 14.5 with; from memory, 5M x 768: 339 and 333).
    constexpr bool AHEAD = QT >= 3 || NT;
    Piece next;
    if (AHEAD) request(min((uint64_t)x, groups - 1), 0, next);
    for (uint64_t g = x; g < groups; g += a.xs) {
        uint64_t row[T];
        double xsq[T]; // on its way from here, needed after the last piece
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const uint64_t i = (g * NW + wave) * T + t;
            row[t] = (a.stride ? int4_sampled(i, a.stride) : i) * 16 + r;
            xsq[t] = a.metric == kMetricDot ? 0.0 : a.sqnorm[min(row[t], a.n - 1)];
        }
        double acc[T][QT];
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int q = 0; q < QT; ++q) acc[t][q] = 0.0;
        for (uint32_t u0 = 0; u0 < a.units; u0 += a.ku) {
            if (!FUSED && a.units > a.ku) {
                __syncthreads();
                load_digits(u0);
                __syncthreads();
            }
            const uint32_t ue = min(u0 + a.ku, a.units);
            for (uint32_t ub = u0; ub < ue; ub += P) {
                Piece now;
                if (AHEAD) {
                    now = next;
                    const bool more = ub + P < a.units; // else the first piece of the wave's next tiles
                    request(more ? g : min(g + a.xs, groups - 1), more ? ub + P : 0, next);
                    __builtin_amdgcn_sched_barrier(0); // all of it now, not next to its use
                } else
                    request(g, ub, now);
                auto &w = now.w;
                auto &sc = now.sc;
                const i32x4_t zero = {0, 0, 0, 0};
                constexpr uint32_t M = 0xF0F0F0F0u;
                constexpr int PP = G == 128 ? 2 : 1; // units per group sum
#pragma unroll
                for (int p0 = 0; p0 < P; p0 += PP) {
                    if (QT >= 3 && ub + p0 >= a.units) break; // uniform; with few queries the zero digits do
                    i32x4_t dg[PP][QT];
#pragma unroll
                    for (int p = 0; p < PP; ++p)
#pragma unroll
                        for (int q = 0; q < QT; ++q) dg[p][q] = *reinterpret_cast<const i32x4_t *>(s_dig + ((ub - u0 + p0 + p) * QT + q) * 1024 + lane * 16);
#pragma unroll
                    for (int t = 0; t < T; ++t) {
                        i32x4_t b[PP];
#pragma unroll
                        for (int p = 0; p < PP; ++p) {
                            const uint2 v = w[t][p0 + p];
                            b[p] = i32x4_t{(int)((v.x << 4) & M), (int)((v.y << 4) & M), (int)(v.x & M), (int)(v.y & M)};
                        }
                        auto scale = [&](int i) { return (double)bf16_to_f32(sc[t].v[i]); };
                        if (G == 32) {
                            auto half = [](i32x4_t v, int i) { return (long)(uint32_t)v[2 * i] | (long)((uint64_t)(uint32_t)v[2 * i + 1] << 32); };
#pragma unroll
                            for (int i = 0; i < 2; ++i)
#pragma unroll
                                for (int q = 0; q < QT; ++q)
                                    acc[t][q] = int4_add(acc[t][q], __builtin_amdgcn_mfma_i32_16x16x32_i8(half(dg[0][q], i), half(b[0], i), zero, 0, 0, 0), scale(2 * p0 + i));
                        } else {
                            i32x4_t c[QT];
#pragma unroll
                            for (int q = 0; q < QT; ++q) c[q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(dg[0][q], b[0], zero, 0, 0, 0);
                            if (PP == 2) {
#pragma unroll
                                for (int q = 0; q < QT; ++q) c[q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(dg[PP - 1][q], b[PP - 1], c[q], 0, 0, 0);
                            }
#pragma unroll
                            for (int q = 0; q < QT; ++q) acc[t][q] = int4_add(acc[t][q], c[q], scale(p0 / PP));
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const uint64_t i = (g * NW + wave) * T + t;
            if (a.tau) {
                const float rt = int4_test_row(a.metric, xsq[t]);
                const bool real = i < a.stiles && row[t] < a.n;
                auto pass = [&](auto metric) {
                    constexpr uint32_t M = decltype(metric)::value;
                    uint64_t any = 0;
#pragma unroll
                    for (int q = 0; q < QT; ++q) any |= __ballot(!int4_beyond<M>(acc[t][q], s_test[q * 4 + h], rt));
                    if (!any) return;
#pragma unroll
                    for (int q = 0; q < QT; ++q) {
                        const bool take = real && !int4_beyond<M>(acc[t][q], s_test[q * 4 + h], rt);
                        if (!__ballot(take)) continue;
                        const uint32_t qi = (y * QT + q) * 4 + h;
                        const Int4Query qv = s_info[q * 4 + h];
                        const uint32_t key = f32_key(int4_finish(M, acc[t][q], qv.scale, xsq[t], qv.sq));
                        keep(take && qi < a.nq && key <= s_tau[q * 4 + h], key, (uint32_t)row[t], qi);
                    }
                };
                if (a.metric == kMetricL2) pass(std::integral_constant<uint32_t, kMetricL2>{});
                else if (a.metric == kMetricCosine) pass(std::integral_constant<uint32_t, kMetricCosine>{});
                else pass(std::integral_constant<uint32_t, kMetricDot>{});
                continue;
            }
            if (i >= a.stiles || (row[t] >= a.n && !a.stride)) continue;
#pragma unroll
            for (int q = 0; q < QT; ++q) {
                const uint32_t q0 = (y * QT + q) * 4;
                const Int4Query qv = s_info[q * 4 + h];
                float *o = a.dist + q0 * a.dstride + i * 16;
                const float d = int4_finish(a.metric, acc[t][q], qv.scale, xsq[t], qv.sq);
                if (q0 + h < a.nq) o[out_at] = row[t] < a.n ? d : __builtin_nanf(""); // NaN sorts last: never makes the bound smaller
            }
        }
    }
    if (a.tau) flush(held);
}

// ---------------------------------------------------------------------------------------------
// gradient of the lookup
// ---------------------------------------------------------------------------------------------
// The places (positions in the list of ids) are sorted by row, stably, so that a row's places are neighbours in the
// order they came in; then each row's run of places is added up. Ids outside the table get the key n_rows, which sorts
// behind everything and is left out. All of it is integer work until the sums, and the sums' order depends on the
// sizes alone.

// Key of place i: its row, or n_rows.
template <class I>
__device__ __forceinline__ uint32_t grad_key(const I *ids, uint64_t i, uint64_t n_rows) {
    const uint64_t r = row_of_id(ids, i, n_rows);
    return r == kNoRow ? (uint32_t)n_rows : (uint32_t)r;
}

// A block's share of zeroing `bytes` at p, 16 bytes per store where the address allows.
__device__ __forceinline__ void zero_share(void *p, uint64_t bytes, uint64_t part, uint64_t parts) {
    uint8_t *b = static_cast<uint8_t *>(p);
    const uint64_t head = min(bytes, (uint64_t)(-(intptr_t)b & 15)), vecs = (bytes - head) / 16;
    uint4 *v = reinterpret_cast<uint4 *>(b + head);
    for (uint64_t i = part * blockDim.x + threadIdx.x; i < vecs; i += parts * blockDim.x) v[i] = make_uint4(0, 0, 0, 0);
    if (part == 0) {
        for (uint64_t i = threadIdx.x; i < head; i += blockDim.x) b[i] = 0;
        for (uint64_t i = head + vecs * 16 + threadIdx.x; i < bytes; i += blockDim.x) b[i] = 0;
    }
}

__global__ void __launch_bounds__(256)
rows_zero_kernel(void *p, uint64_t bytes) { zero_share(p, bytes, blockIdx.x, gridDim.x); }

// Where 64 neighbouring keys of one wave go: off[digit] (LDS, this wave's own) holds the next place of each digit;
// lanes with the same digit find each other by one ballot per digit bit, their order is the lane order.
template <class C>
__device__ __forceinline__ uint32_t wave_rank(uint32_t d, bool in, uint32_t bits, C *off) {
    uint64_t same = __ballot(in);
    for (uint32_t b = 0; b < bits; ++b) {
        const uint64_t m = __ballot((d >> b) & 1);
        same &= (d >> b) & 1 ? m : ~m;
    }
    const uint64_t below = same & lanemask_lt();
    const uint32_t at = in ? off[d] + (uint32_t)__popcll(below) : 0u;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront"); // the reads above, before the update below
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (in && below == 0) off[d] = (C)(off[d] + (uint32_t)__popcll(same));
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    return at;
}

// Few places: block 0 sorts them all in LDS, 8 bits per pass, 16 waves with an equal share each; the other blocks zero
// the gradient meanwhile (zero == nullptr: it is added to). The keys stay where they are, 2-byte places move. block 1024,
// dynamic LDS sort_small_lds(t).
constexpr uint32_t kSortSmall = 8192; // beyond, the launches of the passes cost less (8000 places among 50 000 rows 28 us, 16 000 44 against 34)
__host__ __device__ __forceinline__ uint32_t sort_small_lds(uint32_t t) { return (t + 1) / 2 * 16 + (16 * 256 + 257) * 4; }
template <class I>
__global__ void __launch_bounds__(1024)
rows_sort_small_kernel(const I *ids, uint32_t t, uint64_t n_rows, uint32_t passes, uint2 *out, void *zero, uint64_t zero_bytes) {
    if (blockIdx.x) {
        zero_share(zero, zero_bytes, blockIdx.x - 1, gridDim.x - 1);
        return;
    }
    extern __shared__ uint32_t smem_sort[];
    uint32_t *off = smem_sort, *tot = off + 16 * 256, *key = tot + 257;
    uint16_t *pos[2] = {reinterpret_cast<uint16_t *>(key + (t + 1) / 2 * 2), nullptr};
    pos[1] = pos[0] + (t + 1) / 2 * 2;
    const uint32_t tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    const uint32_t per = (((t + 15) / 16) + 63) & ~63u, b = w * per; // places of a wave
    uint32_t *mine = off + w * 256;
    for (uint32_t i = tid; i < t; i += 1024) {
        key[i] = grad_key(ids, i, n_rows);
        pos[0][i] = (uint16_t)i;
    }
    for (uint32_t p = 0; p < passes; ++p) {
        const uint32_t shift = 8 * p;
        const uint16_t *from = pos[p & 1];
        uint16_t *to = pos[(p & 1) ^ 1];
        for (uint32_t i = tid; i < 16 * 256; i += 1024) off[i] = 0;
        __syncthreads();
        for (uint32_t i = b + lane; i < min(b + per, t); i += 64) atomicAdd(&mine[(key[from[i]] >> shift) & 255], 1u);
        __syncthreads();
        if (tid < 256) {
            uint32_t run = 0;
            for (int v = 0; v < 16; ++v) run += off[v * 256 + tid];
            tot[tid] = run;
        }
        __syncthreads();
        wave0_exclusive_scan_lds(tot, 256);
        __syncthreads();
        if (tid < 256) {
            uint32_t run = tot[tid];
            for (int v = 0; v < 16; ++v) {
                const uint32_t c = off[v * 256 + tid];
                off[v * 256 + tid] = run;
                run += c;
            }
        }
        __syncthreads();
        for (uint32_t i0 = b; i0 < min(b + per, t); i0 += 64) {
            const uint32_t i = i0 + lane;
            const bool in = i < t;
            const uint16_t f = in ? from[i] : (uint16_t)0;
            const uint32_t at = wave_rank(((in ? key[f] : 0u) >> shift) & 255, in, 8, mine);
            if (in) to[at] = f;
        }
        __syncthreads();
    }
    const uint16_t *sorted = pos[passes & 1];
    for (uint32_t i = tid; i < t; i += 1024) out[i] = make_uint2(key[sorted[i]], sorted[i]);
}

// More places: passes of up to 10 bits over tiles of J * 256 places, a count of the digits per tile (the first also clears
// the map of rows that ids name, one byte each), then the scatter. Up to kSortSumTiles tiles a scatter's block adds the
// counts up itself, beyond that a scan between the two does it. (Counting the next pass's digits in the scatter, by atomic
// adds where the places land, measured slower: 64K skewed places 17 us for scatter and count, against 6.5 + 3.5.) J = 4 up to
// 256 K places (more blocks, shorter chains of ranks), 16 beyond (the counts grow with the tiles).
constexpr uint32_t kSortMaxBits = 10, kSortSumTiles = 64;

template <int J, bool FIRST, class I>
__global__ void __launch_bounds__(256)
rows_sort_hist_kernel(const void *src, uint32_t t, uint64_t n_rows, uint32_t shift, uint32_t bits, uint32_t tiles, uint32_t *hist, uint8_t *named) {
    if (blockIdx.x >= tiles) {
        zero_share(named, n_rows, blockIdx.x - tiles, gridDim.x - tiles);
        return;
    }
    __shared__ uint32_t h[1u << kSortMaxBits];
    const uint32_t bins = 1u << bits;
    for (uint32_t i = threadIdx.x; i < bins; i += 256) h[i] = 0;
    __syncthreads();
    const uint32_t b = blockIdx.x * (J * 256);
#pragma unroll
    for (uint32_t j = 0; j < J; ++j) {
        const uint32_t i = b + j * 256 + threadIdx.x;
        if (i < t) {
            const uint32_t k = FIRST ? grad_key(static_cast<const I *>(src), i, n_rows) : static_cast<const uint2 *>(src)[i].x;
            atomicAdd(&h[(k >> shift) & (bins - 1)], 1u);
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < bins; i += 256) hist[(uint64_t)blockIdx.x * bins + i] = h[i];
}

// hist[tile][digit] -> places of that digit in the tiles before; total[digit]. A block has 64 digits, its 16 waves a
// sixteenth of the tiles each. grid ceil(bins / 64), block 1024.
__global__ void __launch_bounds__(1024)
rows_sort_scan_kernel(uint32_t *hist, uint32_t tiles, uint32_t bins, uint32_t *total) {
    __shared__ uint32_t part[16][64];
    const uint32_t lane = threadIdx.x & 63, w = threadIdx.x >> 6, d = blockIdx.x * 64 + lane;
    const uint32_t per = (tiles + 15) / 16, b = min(w * per, tiles), e = min(b + per, tiles);
    uint32_t sum = 0;
    if (d < bins)
#pragma unroll 8
        for (uint32_t i = b; i < e; ++i) sum += hist[(uint64_t)i * bins + d];
    part[w][lane] = sum;
    __syncthreads();
    uint32_t run = 0;
    for (uint32_t v = 0; v < w; ++v) run += part[v][lane];
    if (d >= bins) return;
    if (w == 15) total[d] = run + sum;
    for (uint32_t i0 = b; i0 < e; i0 += 8) { // eight reads in flight
        uint32_t v[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) v[j] = i0 + j < e ? hist[(uint64_t)(i0 + j) * bins + d] : 0u;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
            if (i0 + j < e) {
                hist[(uint64_t)(i0 + j) * bins + d] = run;
                run += v[j];
            }
    }
}

// total == nullptr: hist holds plain counts, to be added up here. Sixteen waves: the ranking is a chain per wave, and a
// block's start waits for the counts (64K places: 6.5 us, 8.2 with four waves; 1M: 15 to 20, and 20 to 24). Block 1024, a
// wave has J / 4 times 64 neighbouring places.
template <int J, bool FIRST, class I>
__global__ void __launch_bounds__(1024)
rows_sort_scatter_kernel(const void *src, uint32_t t, uint64_t n_rows, uint32_t shift, uint32_t bits, uint32_t tiles, const uint32_t *hist, const uint32_t *total,
                         uint2 *out, uint8_t *named) {
    constexpr int W = 16, K = J * 4 / W;
    __shared__ __attribute__((aligned(4))) uint16_t off[W][1u << kSortMaxBits]; // a wave's next place of the digit, from the tile's first
    __shared__ uint32_t tot[(1u << kSortMaxBits) + 1];
    __shared__ uint32_t before[1u << kSortMaxBits]; // places of the digit in the tiles before
    const uint32_t tid = threadIdx.x, w = tid >> 6, lane = tid & 63, bins = 1u << bits;
    uint32_t k[K], ps[K];
    const uint32_t b = blockIdx.x * (J * 256) + w * (K * 64);
#pragma unroll
    for (int j = 0; j < K; ++j) { // on their way while the counts are added up
        const uint32_t i = b + j * 64 + lane;
        k[j] = ps[j] = 0u;
        if (i < t && FIRST) {
            k[j] = grad_key(static_cast<const I *>(src), i, n_rows);
            ps[j] = i;
        } else if (i < t) {
            const uint2 e = static_cast<const uint2 *>(src)[i];
            k[j] = e.x;
            ps[j] = e.y;
        }
    }
    for (uint32_t i = tid; i < bins; i += 1024) {
        tot[i] = total ? total[i] : 0u;
        before[i] = total ? hist[(uint64_t)blockIdx.x * bins + i] : 0u;
    }
    for (uint32_t i = tid; i < W << bits; i += 1024) off[i >> bits][i & (bins - 1)] = 0;
    __syncthreads();
    if (!total) { // 1024 / bins threads per digit, a share of the tiles each
        const uint32_t i = tid & (bins - 1), step = 1024u >> bits;
        uint32_t all = 0, bef = 0;
        for (uint32_t u0 = tid >> bits; u0 < tiles; u0 += 16 * step) { // sixteen reads in flight
            uint32_t v[16];
#pragma unroll
            for (uint32_t j = 0; j < 16; ++j) v[j] = u0 + j * step < tiles ? hist[(uint64_t)(u0 + j * step) * bins + i] : 0u;
#pragma unroll
            for (uint32_t j = 0; j < 16; ++j) {
                all += v[j];
                bef += u0 + j * step < blockIdx.x ? v[j] : 0u;
            }
        }
        if (all) atomicAdd(&tot[i], all);
        if (bef) atomicAdd(&before[i], bef);
    }
#pragma unroll
    for (int j = 0; j < K; ++j) { // the wave's own counts
        const bool in = b + j * 64 + lane < t;
        const uint32_t d = (k[j] >> shift) & (bins - 1);
        if (in) atomicAdd(reinterpret_cast<uint32_t *>(off[w]) + (d >> 1), 1u << (16 * (d & 1))); // a half: 64 K counts at most
        if (FIRST && named && in && k[j] < n_rows) named[k[j]] = 1;
    }
    __syncthreads();
    wave0_exclusive_scan_lds(tot, bins);
    for (uint32_t i = tid; i < bins; i += 1024) {
        uint32_t run = 0;
#pragma unroll
        for (int v = 0; v < W; ++v) {
            const uint32_t c = off[v][i];
            off[v][i] = (uint16_t)run;
            run += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const uint32_t d = (k[j] >> shift) & (bins - 1);
        const bool in = b + j * 64 + lane < t;
        const uint32_t at = wave_rank(d, in, bits, off[w]);
        if (in) out[tot[d] + before[d] + at] = make_uint2(k[j], ps[j]);
    }
}

template <class O, int V>
__device__ __forceinline__ void grad_store(O *o, const float (&sum)[V], float scale, uint32_t accumulate) {
    Pack<O, V> v;
    if (accumulate) {
        v = *reinterpret_cast<const Pack<O, V> *>(o);
#pragma unroll
        for (int i = 0; i < V; ++i) v.v[i] = from_f32<O>(__builtin_fmaf(scale, sum[i], to_f32(v.v[i])));
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v.v[i] = from_f32<O>(scale * sum[i]);
    }
    *reinterpret_cast<Pack<O, V> *>(o) = v;
}

// The sums. The sorted places are cut into chunks of R; L = 1 << lg lanes take one chunk and L * V columns, V columns a
// lane, and walk the chunk with the rows of U places in flight. A run that lies inside the chunk goes to the gradient;
// of a run that the chunk's borders cut, the part that opens the run goes to part[2c + 1], a part that continues one to
// part[2c] (f32, dim columns), and rows_grad_join_kernel adds them up. So no run, however long, is summed by one wave; its parts are joined by
// one block per 64 * V columns.
// Blocks from `blocks` on zero the rows that no id names. Bound by the read of the gradients, a row at a time, and the
// write of the table's gradient.
struct GradArgs {
    const uint2 *place; // (row, position in the list of ids), sorted
    uint32_t t, chunks, R, lg, cbs, blocks; // cbs: column blocks of L * V
    uint64_t n_rows;
    uint32_t dim;
    float scale;
    uint32_t accumulate;
    float *part;
    const uint8_t *named; // nullptr: nothing to zero here
};

template <class T, class O, int V>
__global__ void __launch_bounds__(256)
rows_grad_kernel(const T *g, uint64_t stride, GradArgs a, O *grad) {
    if (blockIdx.x >= a.blocks) {
        const uint32_t ppr = a.dim / V, rpb = max(1u, 1024u / ppr); // V divides dim
        const uint64_t step = (uint64_t)(gridDim.x - a.blocks) * rpb;
        Pack<O, V> z;
#pragma unroll
        for (int i = 0; i < V; ++i) z.v[i] = from_f32<O>(0.f);
        for (uint64_t r0 = (uint64_t)(blockIdx.x - a.blocks) * rpb; r0 < a.n_rows; r0 += step) {
            const uint32_t items = (uint32_t)min((uint64_t)rpb, a.n_rows - r0) * ppr;
            for (uint32_t it = threadIdx.x; it < items; it += 256) {
                const uint32_t rr = it / ppr, p = it - rr * ppr;
                if (!a.named[r0 + rr]) *reinterpret_cast<Pack<O, V> *>(grad + (r0 + rr) * a.dim + (uint64_t)p * V) = z;
            }
        }
        return;
    }
    const uint32_t L = 1u << a.lg, sub = threadIdx.x & (L - 1);
    const uint64_t item = ((uint64_t)blockIdx.x << (8 - a.lg)) + (threadIdx.x >> a.lg);
    const uint32_t c = (uint32_t)(item / a.cbs), cb = (uint32_t)(item % a.cbs);
    const uint32_t col = (cb * L + sub) * V;
    if (c >= a.chunks || col >= a.dim) return;
    const uint32_t begin = c * a.R, end = min(begin + a.R, a.t);
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.f;
    uint32_t cur = a.place[begin].x;
    bool cont = begin > 0 && a.place[begin - 1].x == cur;
    auto flush = [&](bool open) {
        if (cur >= a.n_rows) return;
        if (!cont && !open) {
            grad_store<O, V>(grad + (uint64_t)cur * a.dim + col, sum, a.scale, a.accumulate);
        } else {
            Pack<float, V> v;
#pragma unroll
            for (int i = 0; i < V; ++i) v.v[i] = sum[i];
            *reinterpret_cast<Pack<float, V> *>(a.part + ((uint64_t)c * 2 + (cont ? 0 : 1)) * a.dim + col) = v;
        }
    };
    constexpr int U = 8;
    for (uint32_t j0 = begin; j0 < end; j0 += U) {
        uint32_t k[U];
        Pack<T, V> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t j = min(j0 + u, end - 1);
            const uint2 e = a.place[j];
            k[u] = e.x;
            v[u] = *reinterpret_cast<const Pack<T, V> *>(g + (uint64_t)e.y * stride + col);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (j0 + u >= end) break;
            if (k[u] != cur) {
                flush(false);
                cur = k[u];
                cont = false;
#pragma unroll
                for (int i = 0; i < V; ++i) sum[i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < V; ++i) sum[i] += to_f32(v[u].v[i]);
        }
    }
    flush(end < a.t && a.place[end].x == cur);
}

// The cut runs. A block looks at 8 chunks; where a run opens in one and goes on beyond it, its four waves add the run's
// parts up, a quarter of them each in order, 64 * V columns at a time (grid.y), and the quarters in order. The last chunk
// of the run is found by bisection (keys are sorted).
template <class O, int V>
__global__ void __launch_bounds__(256)
rows_grad_join_kernel(GradArgs a, O *grad) {
    __shared__ float s_part[4][64 * V];
    const uint32_t lane = threadIdx.x & 63, w = threadIdx.x >> 6, col = (blockIdx.y * 64 + lane) * V;
    const bool have = col < a.dim; // V divides dim
    for (uint32_t c0 = blockIdx.x * 8; c0 + 1 < a.chunks; c0 += gridDim.x * 8) {
        // lane j: the run that opens in chunk c0 + j and goes on, its row and last chunk
        uint32_t row = 0xFFFFFFFFu, last = 0;
        const uint32_t c = c0 + (lane & 7);
        if (c + 1 < a.chunks) {
            const uint32_t begin = c * a.R, end = begin + a.R; // not the last chunk: it is full
            row = a.place[end - 1].x;
            const bool opens = !(a.place[begin].x == row && begin > 0 && a.place[begin - 1].x == row);
            if (row >= a.n_rows || a.place[end].x != row || !opens) row = 0xFFFFFFFFu;
            if (row != 0xFFFFFFFFu) {
                uint32_t lo = c + 1, hi = a.chunks - 1; // the last chunk whose first key is the row
                for (uint32_t step = 1; lo + step <= hi; step *= 2) { // most runs end in the next chunk
                    if (a.place[(lo + step) * a.R].x != row) {
                        hi = lo + step - 1;
                        break;
                    }
                    lo += step;
                }
                while (lo < hi) {
                    const uint32_t m = (lo + hi + 1) / 2;
                    if (a.place[m * a.R].x == row) lo = m;
                    else hi = m - 1;
                }
                last = lo;
            }
        }
        uint64_t todo = __ballot(row != 0xFFFFFFFFu && lane < 8); // the same in every wave
        while (todo) {
            const uint32_t j = (uint32_t)__ffsll((unsigned long long)todo) - 1;
            todo &= todo - 1;
            const uint32_t rr = (uint32_t)__builtin_amdgcn_readlane((int)row, (int)j), cl = (uint32_t)__builtin_amdgcn_readlane((int)last, (int)j);
            const uint32_t cc = c0 + j, parts = cl - cc, per = (parts + 3) / 4, p0 = min(w * per, parts), p1 = min(p0 + per, parts);
            float sum[V];
#pragma unroll
            for (int i = 0; i < V; ++i) sum[i] = 0.f;
            if (have) {
                if (w == 0) {
                    const Pack<float, V> v = *reinterpret_cast<const Pack<float, V> *>(a.part + ((uint64_t)cc * 2 + 1) * a.dim + col);
#pragma unroll
                    for (int i = 0; i < V; ++i) sum[i] = v.v[i];
                }
#pragma unroll 8
                for (uint32_t p = p0; p < p1; ++p) {
                    const Pack<float, V> v = *reinterpret_cast<const Pack<float, V> *>(a.part + (uint64_t)(cc + 1 + p) * 2 * a.dim + col);
#pragma unroll
                    for (int i = 0; i < V; ++i) sum[i] += v.v[i];
                }
            }
            if (parts > 1) { // not the first wave's work alone
                __syncthreads(); // the sums before have been read
#pragma unroll
                for (int i = 0; i < V; ++i) s_part[w][lane * V + i] = sum[i];
                __syncthreads();
#pragma unroll
                for (int i = 0; i < V; ++i)
                    sum[i] = ((s_part[0][lane * V + i] + s_part[1][lane * V + i]) + s_part[2][lane * V + i]) + s_part[3][lane * V + i];
            }
            if (w == 0 && have) grad_store<O, V>(grad + (uint64_t)rr * a.dim + col, sum, a.scale, a.accumulate);
        }
    }
}

} // namespace cuddle
