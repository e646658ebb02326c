// muon_b200.cu -- orthogonalisation of matrices by Newton-Schulz products and the Muon step that uses it, behind the C ABI
// of include/framewise_b200.h.
//
// With U (m,n), m <= n (the others lie transposed), X = U / max(|U|, eps) and per step, for coefficients a, b, c:
//     A = X X^T;   B = b A + c A A;   X = a X + B X
// which makes of each singular value s the value s (a + b s^2 + c s^4): after some steps they are all near one.
// Per step 2 m n m + 2 m m m + 2 m m n operations, of which half of the first two are not needed, for A and B are symmetric.
//
// X is held in 32 bits; the products' operands are rounded from it to fp16: one part (11 bits) for bf16 matrices, but two of A
// where it has up to 128 rows (see gram_parts), two parts (22 bits, three products) for f32 ones.  a X is added in 32 bits, outside of
// the products: small singular values are those that grow, by a factor of a step, and an error that a product made of X would
// grow with them.  What B's and A's roundings do is a change of the factor B, small for small singular values, and does not grow.  fp16
// rather than bf16: as fast, eight times finer, and all operands are bounded, so that powers of two (from the coefficients, for any
// matrix) keep them in its range.
// Once singular values are near one, B is near (b + c) times the identity and undoes most of a X.  So a multiple t of the
// identity is taken from B and added to a, where it costs no rounding: t = b s^2 + c s^4 for the singular value s that all
// would have if they were equal (1 / sqrt(m) at first; a matrix below eps, which stays small, has small t).  Errors of bf16
// results besides their own rounding, as a part of their norm: 64 x 256 0.93e-3 (1.9e-3 without t), 512 x 2048 0.6e-3
// (1.3e-3); the rounding alone is 1.66e-3.
//
// Matrices of up to 128 x 256: k_muon_small, a CTA each, all in one launch.  Others go through a chain of launches together: two
// passes over the gradients (k_muon_collect: momentum and norm; k_muon_begin: X), then a launch of k_muon_tiles for each product,
// of which the last updates the parameters.
#include "framewise_b200.h"
#include "framewise_host.h"
#include "tensor_core.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>
#include <vector>

namespace {

using namespace framewise_host;
using namespace tensor_core;

constexpr int kMostMatrices = 256;   // of a chain of launches
constexpr int kSlots        = 24;    // matrices in a launch's arguments
constexpr int kChunk        = 8192;  // values per CTA of the pass over gradients
constexpr int kRowsPerCta   = 128;   // of a tile: the lanes of tensor memory
constexpr int kMostWide     = 256;   // columns of a tile at most
constexpr int kColumns      = 512;   // of tensor memory: a ring of accumulators
constexpr int kMostAccs     = 8;
constexpr int kDepth        = 64;    // K per stage: one part of both operands
// f32: steps of 64 of K after which an accumulator is added up in registers, for tensor cores cut off what they add, at 2^-24 of the
// sum a step, and never round it up.  What A A is off by shows most (b A and c A A undo each other where singular values are near
// one), and it is the smallest product: there it is done after each step, and so in short sums, whose tiles wait for other things.
// Off by, as a part of their norm (plain 32 bits): 500 x 2001 2.6e-6 (2.8e-6; four steps in A A as well 5.1e-6, two throughout
// 3.4e-6, in 531 us for six instead of 480).
// Matrices of at most 128 rows, which fill a tile a step, have all their sums cut: 1 x 2869 was off by 1.3e-6 (plain 3.3e-7).
__host__ __device__ constexpr int segment_of(bool always, int depth) { return always || depth <= 4 ? 1 : 4; }
// Parts of A.  bf16 matrices of few rows have two of them: b A and c A A undo each other, and where B has few values their errors do not
// average out (with one part, worst of 40 matrices, bf16 result: 2 x 257 off by 4.1e-3 of its norm, with two by 2.5e-3; 3 x 1024 3.3e-3 and
// 2.2e-3; 128 x 300 1.86e-3 and 1.75e-3, of which the result's own rounding 1.67e-3; more rows gain as little and would pay three times
// the product).
__host__ __device__ constexpr int gram_parts(int parts, int m) { return m <= 128 ? 2 : parts; }
constexpr int kMostStages   = 12;
constexpr int kEpilogue     = 8;     // warps that finish tiles
constexpr int kThreads      = 64 + 32 * kEpilogue;
constexpr int kShared       = 232448 - 2048;  // dynamic; the rest: the static arrays
constexpr uint64_t kPatience = 4000000000ull;  // nanoseconds after which a wait gives up; they end within microseconds

// A matrix of a chain.  Operands lie in units of 128 rows by 64 columns of fp16, 16 KB, a row of units after the other: one
// tensor copy brings 128 rows of 64 columns, or 64 rows of 128.  (With panels of 64 columns, and copies of 64 by 64, the thread that
// asks for them held up the products.)  X itself is met by warps whose lanes have a row each: squares of 32 x 32 values, in which four
// columns of 32 rows, 512 bytes, follow each other (see place).
struct Entry {
    const void* grad;
    float*      momentum;   // or null: grad is what is made orthogonal
    void*       param;      // or the result
    float*      master;     // or null
    double*     partial;    // sums of squares of the chunks
    float*      shift;      // per step: the multiple of the identity that B does without
    float*      x;          // X
    int         operand[2]; // its fp16 parts, as units of the workspace
    int         gram, factor; // A and B, likewise
    int         rows, cols; // of the parameter
    int         m, n, mp, panels;  // m <= n; rows (a multiple of 128) and units of a row of X
    int         chunks, first_chunk, first_block, first_sym, first_apply;  // where its work begins in each launch
    float       rate;
};

constexpr int kMostSteps = 100;
struct Steps {
    int   count;
    float abc[3 * kMostSteps];
};

struct Slots {
    int   count, base;
    Entry* table;
    Entry entry[kSlots];
};

// Which matrix a unit of work belongs to: the last whose first is not past it.
template <typename F>
__device__ __forceinline__ int find(int count, int unit, F&& first) {
    int lo = 0, hi = count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (first(mid) <= unit) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ float value(float x) { return x; }
__device__ __forceinline__ float value(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* to, float v) { *to = v; }
__device__ __forceinline__ void put(__nv_bfloat16* to, float v) { *to = __float2bfloat16_rn(v); }

// Where a value of X lies.
__device__ __forceinline__ int64_t place(int mp, int row, int col) {
    return ((int64_t)(col / 32) * (mp / 32) + row / 32) * 1024 + col % 32 / 4 * 128 + row % 32 * 4 + col % 4;
}

// Where an operand's value lies in its units, `panels` of them a row.
constexpr int kUnit = 128 * 64;
__device__ __forceinline__ int64_t in_units(int panels, int row, int col) {
    return ((int64_t)(row / 128) * panels + col / 64) * kUnit + row % 128 * 64 + col % 64;
}

struct Rates {
    double eps;
    float  keep, beta, nesterov;  // 1 - beta; nesterov: 0 or 1
    float  decay;                 // 1 - lr weight_decay
    int    follow;
};

// The nearest fp16 numbers of two values, which keep what is left of them.
__device__ __forceinline__ uint32_t part_of(float2& v) {
    const __half2 h = __floats2half2_rn(v.x, v.y);
    const float2  back = __half22float2(h);
    v.x -= back.x, v.y -= back.y;
    return reinterpret_cast<const uint32_t&>(h);
}

// Launches of a chain follow each other without a gap: the next one's CTAs come when this one's leave, and wait for
// all of it to be done before they read or write memory.
__device__ __forceinline__ void next_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void former_is_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// what is made orthogonal, from the gradient and the new momentum
__device__ __forceinline__ float direction(float g, float v, const Rates& r) { return r.nesterov != 0.f ? g + (v - g) * r.beta : v; }

// 1 / max(|U|, eps), from the sum of squares.  |U| may be past the range of 32 bits, or below, and its reciprocal where 32 bits hold few
// digits: two factors, of which the second is a power of two, and one but for those.
struct Reciprocal {
    float  first, second;
    double both;
    __device__ __forceinline__ Reciprocal(double sum, double eps) {
        both = sum == 0.0 ? 0.0 : 1.0 / fmax(sqrt(sum), eps);  // zeros stay zeros, however small eps is
        second = both > 1e30 ? 0x1p100f : both < 1e-30 ? 0x1p-100f : 1.f;
        first  = (float)(both > 1e30 ? both * 0x1p-100 : both < 1e-30 ? both * 0x1p100 : both);
    }
    __device__ __forceinline__ float times(float u) const { return u * first * second; }
};

// four values in a row; `wide`: aligned for one access, else as many as there are (`left`)
__device__ __forceinline__ void load4(const float* x, bool wide, int left, float (&v)[4]) {
    if (wide) {
        const float4 a = *reinterpret_cast<const float4*>(x);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = i < left ? x[i] : 0.f;
    }
}
__device__ __forceinline__ void load4(const __nv_bfloat16* x, bool wide, int left, float (&v)[4]) {
    if (wide) {
        const uint2 a = *reinterpret_cast<const uint2*>(x);
        v[0] = __uint_as_float(a.x << 16), v[1] = __uint_as_float(a.x & 0xffff0000u), v[2] = __uint_as_float(a.y << 16), v[3] = __uint_as_float(a.y & 0xffff0000u);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = i < left ? value(x[i]) : 0.f;
    }
}
template <typename X>
__device__ __forceinline__ bool aligned4(const X* g, const float* v) {
    return reinterpret_cast<uintptr_t>(g) % (4 * sizeof(X)) == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0;
}

// Momentum, and the sum of squares of each chunk in 64 bits (so that no square leaves the range); writes the table down.
template <typename X>
__global__ void __launch_bounds__(256) k_muon_collect(const __grid_constant__ Slots s, const Rates r) {
    const int  e = find(s.count, blockIdx.x + s.entry[0].first_chunk, [&](int i) { return s.entry[i].first_chunk; });
    const Entry& m = s.entry[e];
    const int  chunk = blockIdx.x + s.entry[0].first_chunk - m.first_chunk;
    if (chunk == 0) {
        const int* from = reinterpret_cast<const int*>(&m);
        int*       to   = reinterpret_cast<int*>(s.table + s.base + e);
        for (int i = threadIdx.x; i < (int)(sizeof(Entry) / 4); i += 256) to[i] = from[i];
    }
    next_may_start();
    const int64_t begin = (int64_t)chunk * kChunk;
    const int     left = (int)min((int64_t)m.rows * m.cols - begin, (int64_t)kChunk);
    const X* const g = static_cast<const X*>(m.grad) + begin;
    float* const   v = m.momentum ? m.momentum + begin : nullptr;
    const bool wide = aligned4(g, v);
    double sum = 0.0;
    constexpr int kAhead = 4;
    for (int i0 = threadIdx.x * 4; i0 < left; i0 += 1024 * kAhead) {
        float u[kAhead][4], old[kAhead][4];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int i = i0 + a * 1024;
            if (i >= left) continue;
            load4(g + i, wide && i + 4 <= left, left - i, u[a]);
            if (v) load4(v + i, wide && i + 4 <= left, left - i, old[a]);
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int i = i0 + a * 1024;
            if (i >= left) continue;
            if (v) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    old[a][j] += (u[a][j] - old[a][j]) * r.keep;
                    u[a][j] = direction(u[a][j], old[a][j], r);
                }
                if (wide && i + 4 <= left) {
                    *reinterpret_cast<float4*>(v + i) = make_float4(old[a][0], old[a][1], old[a][2], old[a][3]);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (i + j < left) v[i + j] = old[a][j];
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j < left) sum += (double)u[a][j] * (double)u[a][j];
        }
    }
#pragma unroll
    for (int j = 16; j > 0; j >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, j);
    __shared__ double part[8];
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 8; ++i) sum += part[i];
        m.partial[chunk] = sum;
    }
}

// X = U / max(|U|, eps) in 32 bits and as operands, zeros where there are none: a CTA takes kBlocks squares of 64 columns and rows, the
// next of which is loaded while one is written.  (A square each: 204 us for 4 x 2048 x 8192 bf16, 184 with four, its bytes at the
// copy's rate 123.  Smaller calls end sooner with more CTAs: all five steps of 6 x 500 x 2001 f32 487 us with four and chunks of 16384,
// 472 with two and 8192; 16 x 512 x 2048 bf16 502 and 494; 8 x 2048 x 8192 bf16 5390 and 5430.)  The loads ahead are kept across the
// norm's division: 120 to 160 bytes a thread spill there, at five CTAs an SM.
constexpr int kBlocks = 2;
template <typename X, int PARTS>
__global__ void __launch_bounds__(256, 5) k_muon_begin(const Entry* __restrict__ table, int count, const Rates r, float scale, __half* work, const __grid_constant__ Steps steps) {
    __shared__ double part[8];
    __shared__ float  tile[64][65];
    next_may_start();
    former_is_done();
    const int   e = find(count, blockIdx.x, [&](int i) { return table[i].first_block; });
    const Entry& m = table[e];
    const int first = (blockIdx.x - m.first_block) * kBlocks, high = m.mp / 64, blocks = min(kBlocks, m.panels * high - first);
    const X* const     g = static_cast<const X*>(m.grad);
    const float* const v = m.momentum;
    const bool tall = m.rows > m.cols, wide = aligned4(g, v) && m.cols % 4 == 0;
    const int  lines = tall ? m.n : m.m, at = threadIdx.x % 16 * 4, l0 = threadIdx.x / 16;
    // neighbours in memory first: lines of U as it lies, four values from `at` on
    float u[4][4], mom[4][4];
    auto load = [&](int block) {
        const int panel = block / high, row0 = block % high * 64;
        const int line0 = tall ? panel * 64 : row0, col0 = tall ? row0 : panel * 64, left = m.cols - col0 - at;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int line = line0 + l0 + i * 16;
            const bool some = line < lines && left > 0;
            const int64_t from = some ? (int64_t)line * m.cols + col0 + at : 0;
            load4(g + from, some && wide, some ? left : 0, u[i]);
            if (v) load4(v + from, some && wide, some ? left : 0, mom[i]);
        }
    };
    load(first);
    double sum = 0.0;
    for (int i = threadIdx.x; i < m.chunks; i += 256) sum += m.partial[i];
#pragma unroll
    for (int j = 16; j > 0; j >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, j);
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = sum;
    __syncthreads();
    sum = part[0];
    for (int i = 1; i < 8; ++i) sum += part[i];
    const Reciprocal by(sum, r.eps);
    if (first == 0 && threadIdx.x == 0) {
        float one = (float)(fmin(1.0, sqrt(sum) * by.both) * rsqrt((double)m.m));  // all singular values, if they are equal
        for (int i = 0; i < steps.count; ++i) {
            const float square = one * one, t = square * (steps.abc[3 * i + 1] + steps.abc[3 * i + 2] * square);
            m.shift[i] = t;
            one *= steps.abc[3 * i] + t;
        }
    }
    for (int b = 0; b < blocks; ++b) {
        if (b > 0) __syncthreads();  // the square before has been read
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float d = v ? direction(u[i][j], mom[i][j], r) : u[i][j], x = by.times(d);
                if (tall) tile[at + j][l0 + i * 16] = x;
                else tile[l0 + i * 16][at + j] = x;
            }
        __syncthreads();
        if (b + 1 < blocks) load(first + b + 1);
        const int panel = (first + b) / high, row0 = (first + b) % high * 64;
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // a warp: 32 rows of four columns, 512 bytes of X
            const int row = (threadIdx.x / 32 & 1) * 32 + threadIdx.x % 32, col = (threadIdx.x / 64 + i * 4) * 4;
            *reinterpret_cast<float4*>(m.x + place(m.mp, row0 + row, panel * 64 + col)) = make_float4(tile[row][col], tile[row][col + 1], tile[row][col + 2], tile[row][col + 3]);
        }
        __half* const op = work + (int64_t)m.operand[0] * kUnit + in_units(m.panels, row0, panel * 64);
        const int64_t plane = (int64_t)m.panels * m.mp * 64;
#pragma unroll
        for (int i = 0; i < 2; ++i) {  // a row's 128 bytes by eight lanes
            const int row = threadIdx.x / 8 + i * 32, col = threadIdx.x % 8 * 8;
            uint32_t w[PARTS][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float2 x = make_float2(tile[row][col + 2 * j] * scale, tile[row][col + 2 * j + 1] * scale);
#pragma unroll
                for (int q = 0; q < PARTS; ++q) w[q][j] = part_of(x);
            }
#pragma unroll
            for (int q = 0; q < PARTS; ++q) *reinterpret_cast<uint4*>(op + q * plane + row * 64 + col) = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
        }
    }
}

// ------------------------------------------------------------------------------------------ products

enum Kind { kGram = 0, kSquare = 1, kApply = 2, kLast = 3 };

struct Params {
    const Entry* table;
    int     count, tiles, wide, stages;
    int     span;        // columns of the second operand that a copy brings
    int     from, step;  // from: which operands of X are read
    __half* work;
    int*    failed;      // a wait ran out
    float   product;     // factor of the finished sums
    float   old;         // kSquare: of A; kApply: a
    float   scale;       // kSquare: of the identity; kApply: of the next operands
    Rates   rates;       // kLast
};

// fp16 operands, f32 sums
__host__ __device__ constexpr uint32_t half_kind(int m, int n, bool b_mn) {
    return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void load_sector(const __half* x, uint32_t* w) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(x)
                 : "memory");
}
__device__ __forceinline__ void store_sector(__half* x, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(x), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]),
                 "r"(w[7])
                 : "memory");
}

constexpr int kTurn = 32 * 32 * 4;  // shared memory of a warp that updates parameters: to turn 32 x 32 values

// Parameters of 32 x 32 values of X, by lines of the parameter: line 0 of them, how many there are, and how many values of each.
struct Lines {
    int64_t first;
    int     count, width;
    __device__ __forceinline__ Lines(const Entry& m, int row0, int col0) {  // of X
        const bool tall = m.rows > m.cols;
        const int  line = tall ? col0 : row0, at = tall ? row0 : col0;
        first = (int64_t)line * m.cols + at, count = max(0, min(32, m.rows - line)), width = max(0, min(32, m.cols - at));
    }
};

// 16 bytes of parameters at a time
template <typename X>
struct Grain {
    static constexpr int kValues = 16 / sizeof(X), kLanes = 32 / kValues, kLines = 32 / kLanes;  // lanes a line, lines at once
    uint4 w;
    __device__ __forceinline__ float get(int i) const {
        const uint32_t* const u = reinterpret_cast<const uint32_t*>(&w);
        return sizeof(X) == 4 ? __uint_as_float(u[i]) : __uint_as_float(i % 2 ? u[i / 2] & 0xffff0000u : u[i / 2] << 16);
    }
    __device__ __forceinline__ void set(const float (&v)[kValues]) {
        uint32_t* const u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(X) == 4) u[i] = __float_as_uint(v[i]);
            else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
        }
    }
};
template <typename X>
__device__ __forceinline__ bool by_grains(const Entry& m) {
    return m.cols * sizeof(X) % 16 == 0 && (reinterpret_cast<uintptr_t>(m.param) | reinterpret_cast<uintptr_t>(m.master)) % 16 == 0;
}

// The new value of a parameter; `held`: its copy, if there is one.
template <typename X>
__device__ __forceinline__ float updated(float old, float held, bool copied, float x, const Rates& r, float rate) {
    if (copied) {
        X rounded;
        put(&rounded, held);
        // a copy of which the parameter is not the rounded value has been left behind by the program
        if (!r.follow || value(rounded) == old || (old != old && held != held)) old = held;
    }
    return old * r.decay - rate * x;
}

// FIRST to LAST: of the lane's grains
template <typename X, int FIRST, int LAST, int N>
__device__ __forceinline__ void load_parameters(const Entry& m, const Lines& at, int lane, Grain<X> (&was)[N]) {
    using G = Grain<X>;
    const X* p = static_cast<const X*>(m.param) + at.first + (int64_t)(FIRST * G::kLines + lane / G::kLanes) * m.cols + lane % G::kLanes * G::kValues;
#pragma unroll
    for (int i = FIRST; i < LAST; ++i, p += (int64_t)G::kLines * m.cols)
        if (i * G::kLines + lane / G::kLanes < at.count && lane % G::kLanes * G::kValues < at.width) was[i - FIRST].w = *reinterpret_cast<const uint4*>(p);
}

// p = p decay - rate X, or the result X itself, for 32 x 32 values of X, a row a lane.  They go through shared memory, so that
// neighbouring lanes have neighbouring values in memory whichever way the parameter lies: 16 bytes a lane, where lines of the
// parameter begin at multiples of that (EARLY: `was` has been loaded before), else a value a lane.  (A value a lane throughout:
// 71 us for the last product of 16 x 512 x 2048 bf16, 54 this way.)
template <typename X, bool EARLY, int N>
__device__ __forceinline__ void update(const Entry& m, const Rates& r, const float* v, const Lines& at, bool grains, char* turn, int lane, Grain<X> (&was)[N]) {
    using G = Grain<X>;
    const bool tall = m.rows > m.cols;
    float* const t = reinterpret_cast<float*>(turn);
    __syncwarp();
    if (tall) {
#pragma unroll
        for (int j = 0; j < 32; ++j) t[j * 32 + (lane ^ (j & 7) << 2)] = v[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) *reinterpret_cast<float4*>(t + lane * 32 + (j * 4 ^ (lane & 7) << 2)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    }
    __syncwarp();
    X* const p = static_cast<X*>(m.param) + at.first;
    const int l0 = lane / G::kLanes, c0 = lane % G::kLanes * G::kValues;
    auto store_grain = [&](int i, const G& old) {
        const int line = i * G::kLines + l0;
        if (line >= at.count || c0 >= at.width) return;
        float x[G::kValues];
#pragma unroll
        for (int j = 0; j < G::kValues; j += 4) {
            const float4 f = *reinterpret_cast<const float4*>(t + line * 32 + (c0 + j ^ (line & 7) << 2));
            x[j] = f.x, x[j + 1] = f.y, x[j + 2] = f.z, x[j + 3] = f.w;
        }
        const int64_t to = (int64_t)line * m.cols + c0;
        if (m.momentum) {
            float* const copy = m.master ? m.master + at.first + to : nullptr;
#pragma unroll
            for (int j = 0; j < G::kValues; j += 4) {
                float4 held = copy ? *reinterpret_cast<const float4*>(copy + j) : make_float4(0.f, 0.f, 0.f, 0.f);
                float* const h = reinterpret_cast<float*>(&held);
#pragma unroll
                for (int k = 0; k < 4; ++k) h[k] = x[j + k] = updated<X>(old.get(j + k), h[k], copy != nullptr, x[j + k], r, m.rate);
                if (copy) *reinterpret_cast<float4*>(copy + j) = held;
            }
        }
        G now;
        now.set(x);
        *reinterpret_cast<uint4*>(p + to) = now.w;
    };
    if (grains) {
        constexpr int kAll = 32 / G::kLines;
        if constexpr (EARLY) {
#pragma unroll
            for (int i = 0; i < kAll; ++i) store_grain(i, was[i]);
        } else {
#pragma unroll
            for (int i0 = 0; i0 < kAll; i0 += N) {
                if (m.momentum) i0 == 0 ? load_parameters<X, 0, N>(m, at, lane, was) : load_parameters<X, N, 2 * N>(m, at, lane, was);
                static_assert(EARLY || kAll == 2 * N, "");
#pragma unroll
                for (int i = 0; i < N; ++i) store_grain(i0 + i, was[i]);
            }
        }
    } else if (lane < at.width) {
#pragma unroll 4
        for (int j = 0; j < 32; ++j) {
            if (j >= at.count) continue;
            const int64_t to = (int64_t)j * m.cols + lane;
            float x = t[j * 32 + (lane ^ (j & 7) << 2)];
            if (m.momentum) {
                float* const copy = m.master ? m.master + at.first + to : nullptr;
                x = updated<X>(value(p[to]), copy ? *copy : 0.f, copy != nullptr, x, r, m.rate);
                if (copy) *copy = x;
            }
            put(p + to, x);
        }
    }
    __syncwarp();
}

// After a wait ran out the results are NaN.
template <typename X>
__global__ void __launch_bounds__(256) k_muon_check(const Entry* __restrict__ table, int count, const int* failed) {
    former_is_done();
    if (*failed == 0) return;
    for (int e = 0; e < count; ++e) {
        const Entry& m = table[e];
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)m.rows * m.cols; i += (int64_t)gridDim.x * 256) {
            put(static_cast<X*>(m.param) + i, __uint_as_float(0x7fffffffu));
            if (m.master) m.master[i] = __uint_as_float(0x7fffffffu);
        }
    }
}

// A product of all matrices of a chain, as tiles of 128 rows (CG 2: of 256, on a pair of CTAs, each with 128 of them and half of the
// second operand) by up to 256 columns, dealt out in turn to CTAs that stay.
//   kGram    A = X X^T       of both the tiles on and above the diagonal; what lies above it is written to both places
//   kSquare  b A + c A A - t
//   kApply   (a + t) X + B X; kLast: likewise, and the parameters' update
// One warp asks for copies, one for products, eight finish tiles, a row a lane, while the next is multiplied.  What bounds it: products
// and their feeding where m is 2048 (4 x 2048 x 8192 bf16, in us of which products at 1.69 PFLOP/s: A 124 of 85, B 43 of 21, X 232 of
// 163; power lowers the clock in long runs), X in 32 bits and its latency where m is 512 (16 x 512 x 2048 bf16: A 25, B 17, X 44 of
// 31 at the copy's rate).  Tried and not kept: all products in one cooperative launch in which a tile waits for its matrix's tiles
// alone (3.9 us for a product of the smallest either way; 4 x 2048 x 8192 10 % slower: two stages of the ring went to the update),
// X and results by the copy engine (its queue holds them up; the ring lost three stages: X 249), X brought to the second cache ahead.
// f32: the 128 sums a thread leave the last product no registers for parameters: it spills 336 to 344 bytes a thread and takes 91 us for
// 12 x 500 x 2000, where a X + B X alone takes 54 (the other products spill 52 to 96; bf16 none).
template <int KIND, int PARTS, int CG>
__global__ void __launch_bounds__(kThreads, 1) k_muon_tiles(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Params p) {
    constexpr bool kApplies = KIND == kApply || KIND == kLast;
    constexpr bool kBMn = kApplies;             // the second operand's rows lie along K
    constexpr bool kSegments = PARTS == 2;
    constexpr int  kTile = kRowsPerCta * CG;
    extern __shared__ char shared_raw[];
    __shared__ int firsts[kMostMatrices];
    __shared__ uint64_t bars_at[2 * kMostStages + 2 * kMostAccs + 1];
    __shared__ uint32_t slot_at;
    __shared__ volatile int give_up;
    const uint32_t full = smem_addr(bars_at), empty = full + 8 * kMostStages, done = empty + 8 * kMostStages, freed = done + 8 * kMostAccs,
                   drained = freed + 8 * kMostAccs;
    const int rank = CG == 2 ? (int)cluster_rank() : 0, worker = blockIdx.x / CG, workers = gridDim.x / CG, accs = min(kMostAccs, kColumns / p.wide);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kTurns = KIND == kLast ? kEpilogue * kTurn : 0;
    const uint32_t base = (smem_addr(shared_raw) + kTurns + 1023u) & ~1023u;
    const int part_b = p.wide / CG * kDepth * 2, part_a = kRowsPerCta * kDepth * 2, stage_bytes = part_a + part_b;

    next_may_start();
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) bar_init(full + 8 * s, 1), bar_init(empty + 8 * s, 1);
        for (int i = 0; i < accs; ++i) bar_init(done + 8 * i, 1), bar_init(freed + 8 * i, kEpilogue * CG);
        bar_init(drained, 1);
        give_up = 0;
        bar_init_fence();
        prefetch_map(&map_a);
        prefetch_map(&map_b);
    }
    if (warp == 1) tmem_alloc<CG>(smem_addr(&slot_at), kColumns);
    former_is_done();
    for (int i = threadIdx.x; i < p.count; i += kThreads) firsts[i] = kApplies ? p.table[i].first_apply : p.table[i].first_sym;
    fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync();
    fence_after();
    const uint32_t tmem = *const_cast<volatile uint32_t*>(&slot_at);

    auto bounded = [&](uint32_t bar, uint32_t parity, bool heed) -> bool {
        uint64_t since = 0;
        for (int i = 1;; ++i) {
            if (bar_try(bar, parity)) return true;
            if (i % 64) continue;
            uint64_t now;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
            if (since == 0) since = now;
            if (now - since > kPatience || (heed && give_up)) return false;
        }
    };
    auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
        if (bounded(bar, parity, true)) return true;
        give_up = 1;
        atomicExch(p.failed, 1);
        return false;
    };

    // Tile u: its matrix, and the first row and column.  Symmetric results: rows of tiles from the diagonal on.
    struct Tile {
        int e, row, col, depth, segment;
    };
    auto tile_at = [&](int u) -> Tile {
        Tile t;
        t.e = find(p.count, u, [&](int i) { return firsts[i]; });
        const Entry& m = p.table[t.e];
        int at = u - firsts[t.e];
        if (kApplies) {
            // a column after the other: its part of X is met by all rows at once, B stays near
            const int mt = m.mp / kTile;
            t.row = at % mt * kTile, t.col = at / mt * p.wide;
        } else {
            const int nt = (m.mp + p.wide - 1) / p.wide;
            int row = 0;
            for (;; ++row) {
                const int first = row * kTile / p.wide, tiles = nt - first;
                if (at < tiles) {
                    t.col = (first + at) * p.wide;
                    break;
                }
                at -= tiles;
            }
            t.row = row * kTile;
        }
        t.depth = KIND == kGram ? m.panels : (m.m + 63) / 64;
        t.segment = kSegments ? segment_of(KIND == kSquare || m.m <= 128, t.depth) : t.depth;
        return t;
    };

    if (warp == 0 && lane == 0) {  // ---- copies
        int      stage = 0, issued = 0;
        uint32_t phase = 0;
        bool     ok = true;
        for (int u = worker; u < p.tiles && ok; u += workers) {
            const Tile t = tile_at(u);
            const Entry m = p.table[t.e];
            // units: where the operands begin, and those of their second parts
            const int x0 = p.from ? m.operand[1] : m.operand[0], x_part = m.mp / 128 * m.panels, s_row = m.mp / 64, s_part = m.mp / 128 * s_row;
            const int a0 = KIND == kGram ? x0 : KIND == kSquare ? m.gram : m.factor, b0 = KIND == kSquare ? m.gram : x0;
            const int a_part = KIND == kGram ? x_part : s_part, b_part = KIND == kSquare ? s_part : x_part, b_row = KIND == kSquare ? s_row : m.panels;
            const int a_first = a0 + (t.row / 128 + rank) * (KIND == kGram ? m.panels : s_row);
            // columns of the tile that there are and are this CTA's
            const int limit = kApplies ? m.panels * 64 : m.mp, have = min(p.wide, limit - t.col) / CG, from = t.col + rank * have;
            const int copies = (have + p.span - 1) / p.span, span_bytes = p.span * kDepth * 2, parts = KIND == kSquare ? gram_parts(PARTS, m.m) : PARTS;
            for (int k = 0; k < t.depth && ok; ++k) {
                for (int q = parts - 1; q >= 0; --q) {  // the small part is met, and its stage free again, first
                    ok = wait(empty + 8 * stage, phase ^ 1);
                    if (!ok) break;
                    const uint32_t a = base + stage * stage_bytes, b = a + part_a, bar = CG == 2 ? in_cta(full + 8 * stage, 0) : full + 8 * stage;
                    if (rank == 0) bar_expect(full + 8 * stage, CG * (part_a + copies * span_bytes));
                    load_box<CG>(a, &map_a, bar, 0, 0, a_first + q * a_part + k);
                    for (int j = 0; j < copies; ++j) {
                        const int col = from + j * p.span;
                        if (kBMn) load_box<CG>(b + j * span_bytes, &map_b, bar, 0, k % 2 * 64, b0 + q * b_part + k / 2 * b_row + col / 64);
                        else load_box<CG>(b + j * span_bytes, &map_b, bar, 0, col % 128, b0 + q * b_part + col / 128 * b_row + k);
                    }
                    ++issued;
                    if (++stage == p.stages) stage = 0, phase ^= 1;
                }
            }
        }
        // the last stages are handed back before the CTA ends; where a wait ran out, copies in flight end first
        for (int i = 0; ok && i < p.stages && i < issued; ++i) {
            ok = wait(empty + 8 * stage, phase ^ 1);
            if (ok && ++stage == p.stages) stage = 0, phase ^= 1;
        }
        if (give_up && rank == 0) {
            for (int i = 0; i < p.stages && i < issued; ++i) {
                if (--stage < 0) stage = p.stages - 1, phase ^= 1;
                bounded(full + 8 * stage, phase, false);
            }
        }
    } else if (warp == 1 && lane == 0 && rank == 0) {  // ---- products
        int      stage = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool     ok = true;
        for (int u = worker; u < p.tiles && ok; u += workers) {
            const Tile t = tile_at(u);
            const Entry m = p.table[t.e];
            const int limit = kApplies ? m.panels * 64 : m.mp;
            const uint32_t kind = half_kind(kTile, min(p.wide, limit - t.col), kBMn);
            for (int k0 = 0; k0 < t.depth && ok; k0 += t.segment) {
                ok = wait(freed + 8 * acc, acc_phase ^ 1);
                if (!ok) break;
                fence_after();
                const uint32_t d = tmem + acc * p.wide;
                auto next = [&](int& at, uint32_t& at_phase) {
                    if (++at == p.stages) at = 0, at_phase ^= 1;
                };
                auto multiply = [&](int stage_a, int stage_b, bool add) {
                    const uint32_t a = base + stage_a * stage_bytes, b = base + stage_b * stage_bytes + part_a;
#pragma unroll
                    for (int i = 0; i < kDepth / 16; ++i)
                        product<CG>(d, operand(a + i * 32, 8192), operand(b + i * (kBMn ? 2048 : 32), 8192), kind, add || i > 0);
                };
                auto arrived = [&](int at, uint32_t at_phase) {
                    ok = ok && wait(full + 8 * at, at_phase);
                    if (ok) fence_after();
                    return ok;
                };
                const int  k1 = kSegments ? min(t.depth, k0 + t.segment) : t.depth;
                const bool two = kSegments || (KIND == kSquare && gram_parts(PARTS, m.m) == 2);
                for (int k = k0; k < k1; ++k) {
                    if (!arrived(stage, phase)) break;
                    if (two) {  // the small products first
                        const int low = stage;
                        next(stage, phase);
                        if (!arrived(stage, phase)) break;
                        multiply(low, stage, k > k0);
                        multiply(stage, low, true);
                        products_commit<CG>(empty + 8 * low);
                    }
                    multiply(stage, stage, two || k > k0);
                    products_commit<CG>(empty + 8 * stage);
                    next(stage, phase);
                }
                if (!ok) break;
                products_commit<CG>(done + 8 * acc);
                if (++acc == accs) acc = 0, acc_phase ^= 1;
            }
        }
        if (!ok) {  // products under way still read shared memory
            products_commit<CG>(drained);
            bounded(drained, 0, false);
        }
    } else if (warp >= 2) {  // ---- finished tiles: a row a lane
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const int half_wide = p.wide / 2;
        const uint32_t freed0 = CG == 2 ? in_cta(freed, 0) : freed;
        int      acc = 0;
        uint32_t acc_phase = 0;
        bool     ok = true;
        for (int u = worker; u < p.tiles && ok; u += workers) {
            const Tile t = tile_at(u);
            const Entry m = p.table[t.e];
            const int row = t.row + rank * kRowsPerCta + quarter * 32 + lane, col0 = t.col + half * half_wide;
            const int limit = kApplies ? m.panels * 64 : m.mp;
            const int64_t s_plane = (int64_t)m.mp * m.mp, x_plane = (int64_t)m.panels * m.mp * 64;
            const float shift = KIND == kGram ? 0.f : m.shift[p.step], old = kApplies ? p.old + shift : p.old;
            const int64_t at0 = kApplies ? place(m.mp, row, col0) : 0;
            const int          target = KIND == kGram ? m.gram : KIND == kSquare ? m.factor : p.from ? m.operand[0] : m.operand[1];
            using X = std::conditional_t<PARTS == 2, float, __nv_bfloat16>;
            // (f32: the sums need the registers; half of the parameters at a time)
            constexpr int kGrains = 32 / Grain<X>::kLines / (kSegments ? 2 : 1);
            Grain<X> was[kGrains];
            const bool grains = KIND == kLast && by_grains<X>(m), early = grains && m.momentum && !kSegments;
            auto load_x = [&](int c, float4 (&x)[8]) {  // 32 columns of X
                if (col0 + c >= limit) return;
                const float4* const from = reinterpret_cast<const float4*>(m.x + at0 + (int64_t)(c / 32) * m.mp * 32);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = from[j * 32];
            };
            auto finish = [&](float* v, int c, const float4 (&x)[8]) {  // 32 columns
                const int col = col0 + c;
                if (col >= limit) return;
                if (kApplies) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        v[4 * j] = fmaf(old, x[j].x, v[4 * j] * p.product), v[4 * j + 1] = fmaf(old, x[j].y, v[4 * j + 1] * p.product);
                        v[4 * j + 2] = fmaf(old, x[j].z, v[4 * j + 2] * p.product), v[4 * j + 3] = fmaf(old, x[j].w, v[4 * j + 3] * p.product);
                    }
                }
                if constexpr (KIND == kLast) {
                    update<X, !kSegments>(m, p.rates, v, Lines(m, row - lane, col), grains, shared_raw + (warp - 2) * kTurn, lane, was);
                    if (early && c + 32 < half_wide && col + 32 < limit) load_parameters<X, 0, kGrains>(m, Lines(m, row - lane, col + 32), lane, was);
                    return;
                }
                if (KIND == kApply) {
                    float4* const to = reinterpret_cast<float4*>(m.x + at0 + (int64_t)(c / 32) * m.mp * 32);
#pragma unroll
                    for (int j = 0; j < 8; ++j) to[j * 32] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                } else if (row / 128 > col / 128) {
                    return;  // below the diagonal
                }
                const int64_t at = in_units(kApplies ? m.panels : m.mp / 64, row, col);
                __half* const to = p.work + (int64_t)target * kUnit;
                const int64_t plane = KIND == kApply ? x_plane : s_plane;
                const int of_gram = gram_parts(PARTS, m.m), parts = KIND == kGram ? of_gram : PARTS;
                if (KIND == kSquare) {
#pragma unroll
                    for (int q = 1; q >= 0; --q) {
                        if (q >= of_gram) continue;
                        uint32_t w[16];
                        load_sector(p.work + (int64_t)m.gram * kUnit + q * plane + at, w), load_sector(p.work + (int64_t)m.gram * kUnit + q * plane + at + 16, w + 8);
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const float2 a = __half22float2(reinterpret_cast<const __half2&>(w[j]));
                            v[2 * j] = fmaf(old, a.x, q == of_gram - 1 ? v[2 * j] * p.product : v[2 * j]);
                            v[2 * j + 1] = fmaf(old, a.y, q == of_gram - 1 ? v[2 * j + 1] * p.product : v[2 * j + 1]);
                        }
                    }
                    const int hit = row - col;  // the diagonal's place among these columns
                    if (hit >= 0 && hit < 32) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] -= j == hit ? shift * p.scale : 0.f;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] *= KIND == kApply ? p.scale : p.product;
                }
                const bool mirror = KIND != kApply && col / 128 > row / 128;
#pragma unroll
                for (int q = 0; q < (KIND == kGram ? 2 : PARTS); ++q) {
                    if (q >= parts) continue;
                    uint32_t w[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        float2 two = make_float2(v[2 * j], v[2 * j + 1]);
                        w[j] = part_of(two);
                        v[2 * j] = two.x, v[2 * j + 1] = two.y;
                    }
                    store_sector(to + q * plane + at, w), store_sector(to + q * plane + at + 16, w + 8);
                    if (mirror) {
                        __half* const under = to + q * plane + in_units(m.mp / 64, col, row);
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const __half2 h = reinterpret_cast<const __half2&>(w[j]);
                            under[(2 * j) * 64] = h.x, under[(2 * j + 1) * 64] = h.y;
                        }
                    }
                }
            };
            constexpr int kBuffers = KIND == kApply && !kSegments ? 2 : 1;
            float4 x_of[kBuffers][8];
            if (KIND == kApply && !kSegments) load_x(0, x_of[0]);  // ahead of the sums
            if (KIND == kLast && early && col0 < limit) load_parameters<X, 0, kGrains>(m, Lines(m, row - lane, col0), lane, was);
            float total[kSegments ? kMostWide / 2 : 1];
            if constexpr (kSegments) {
#pragma unroll
                for (int j = 0; j < kMostWide / 2; ++j) total[j] = 0.f;
            }
            for (int k0 = 0; k0 < t.depth; k0 += t.segment) {
                ok = __all_sync(0xffffffffu, wait(done + 8 * acc, acc_phase));
                if (!ok) break;
                fence_after();
                const uint32_t acc_at = tmem + ((uint32_t)(quarter * 32) << 16) + acc * p.wide + half * half_wide;
                auto columns = [&](int c, auto buffer) {
                    constexpr int kBuffer = decltype(buffer)::value;
                    float2 pairs[16];
                    float* const v = reinterpret_cast<float*>(pairs);
                    if constexpr (KIND == kLast && !kSegments) load_x(c, x_of[0]);
                    tmem_load32(acc_at + c, pairs);
                    tmem_loaded(pairs);
                    if constexpr (kBuffers == 2)
                        if (c + 32 < half_wide) load_x(c + 32, x_of[kBuffer ^ 1]);
                    finish(v, c, x_of[kBuffer]);
                    __syncwarp();
                };
                if constexpr (kSegments) {
#pragma unroll
                    for (int c = 0; c < kMostWide / 2; c += 32) {
                        if (c >= half_wide || col0 + c >= limit) continue;
                        float2 pairs[16];
                        const float* const v = reinterpret_cast<const float*>(pairs);
                        tmem_load32(acc_at + c, pairs);
                        tmem_loaded(pairs);
#pragma unroll
                        for (int j = 0; j < 32; ++j) total[c + j] += v[j];
                    }
                } else if constexpr (kBuffers == 2) {
                    for (int c = 0; c < half_wide && col0 + c < limit; c += 64) {
                        columns(c, std::integral_constant<int, 0>());
                        if (c + 32 < half_wide && col0 + c + 32 < limit) columns(c + 32, std::integral_constant<int, 1>());
                    }
                } else {
#pragma unroll 1
                    for (int c = 0; c < half_wide && col0 + c < limit; c += 32) columns(c, std::integral_constant<int, 0>());
                }
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(freed0 + 8 * acc);
                if (++acc == accs) acc = 0, acc_phase ^= 1;
            }
            if (!ok) break;
            if constexpr (kSegments) {
#pragma unroll
                for (int c = 0; c < kMostWide / 2; c += 32) {
                    if (c >= half_wide) continue;
                    if (kApplies) load_x(c, x_of[0]);
                    finish(total + c, c, x_of[0]);
                    __syncwarp();
                }
            }
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync();
    fence_after();
    if (warp == 1) tmem_free<CG>(tmem, kColumns);
}

// ------------------------------------------------------------------------------------------ small matrices

constexpr int kSmallM = 128, kSmallN = 256;  // a matrix that one CTA holds: X in registers, its operands, A and B in shared memory
constexpr int kSmallThreads = 512;
constexpr int kSmallPitch = kSmallN + 1;     // of the values on their way in and out
__host__ __device__ constexpr int small_bytes(int parts) {
    const int operands = (parts * (kSmallN / 64) + 2 * 2) * kUnit * 2, values = kSmallM * kSmallPitch * 4;
    return 1024 + (operands > values ? operands : values);
}

struct SmallSlot {  // `count` matrices of one shape, `stride` values apart
    const void* grad;
    float*      momentum;
    void*       param;
    float*      master;
    int64_t     stride;
    int         rows, cols, count;
    float       rate;
};
struct SmallSlots {
    int       count;
    SmallSlot slot[kSlots];
};

// A step's factors, of what they are in Params.
struct SmallStep {
    float gram, square, of_gram, of_one, apply, a, operand, b, c;
};
struct SmallSteps {
    int       count;
    SmallStep step[kMostSteps];
};

// All steps of a matrix of at most 128 x 256 in one CTA, and its update: nothing but the gradient, the momentum and the parameter
// crosses memory.  A row of X by four threads, 64 columns each (one unit's row), 32 columns of A and B.  What bounds it is latency:
// three products a step, each behind a barrier, and what turns its sums into the next operands: 64 x 256 bf16 14 us and 4.6 a step, f32 14 and
// 9.2 (a chain of launches: 80 and 136 for five steps, and 17 launches of the host's time).  Descriptors counted up instead of formed for
// each product, and waits that ask without a pause, changed nothing.
// (f32 spills 368 bytes a thread, bf16 108.)
// A has two parts for bf16 as well: with one, results of few rows are off by up to 1.9 times their own rounding (2 x 27; 1.2 times with two).
template <typename X>
__global__ void __launch_bounds__(kSmallThreads, 1) k_muon_small(const __grid_constant__ SmallSlots s, const Rates r, const __grid_constant__ SmallSteps steps) {
    constexpr int PARTS = sizeof(X) == 4 ? 2 : 1;
    extern __shared__ char shared_raw[];
    __shared__ double   part[kSmallThreads / 32];
    __shared__ uint64_t bar_at;
    __shared__ uint32_t slot_at;
    const uint32_t base = (smem_addr(shared_raw) + 1023u) & ~1023u, bar = smem_addr(&bar_at);
    char* const    mem  = shared_raw + (base - smem_addr(shared_raw));
    float* const   values = reinterpret_cast<float*>(mem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = warp % 4 * 32 + lane, group = warp / 4;
    int at = 0, index = blockIdx.x;
    while (index >= s.slot[at].count) index -= s.slot[at++].count;
    const SmallSlot& m = s.slot[at];
    const int  rows = m.rows, cols = m.cols, all = rows * cols;
    const bool tall = rows > cols;
    const int  small = min(rows, cols), wide = max(rows, cols), units = (wide + 63) / 64;
    const X* const g = static_cast<const X*>(m.grad) + index * m.stride;
    X* const       p = static_cast<X*>(m.param) + index * m.stride;
    float* const   v = m.momentum ? m.momentum + index * m.stride : nullptr;
    float* const   master = m.master ? m.master + index * m.stride : nullptr;

    if (threadIdx.x == 0) {
        bar_init(bar, 1);
        bar_init_fence();
    }
    if (warp == 0) tmem_alloc<1>(smem_addr(&slot_at), kColumns);
    double sum = 0.0;
    // four values at a time, of which a line's lie side by side
    constexpr int kAhead = 4;
    const bool wide4 = aligned4(g, v) && aligned4(p, master) && cols % 4 == 0;
    auto place_of = [&](int i) {
        const int line = i / cols, place = i - line * cols;
        return tall ? place * kSmallPitch + line : line * kSmallPitch + place;
    };
    const int hop = tall ? kSmallPitch : 1;
    for (int i0 = threadIdx.x * 4; i0 < all; i0 += kSmallThreads * 4 * kAhead) {
        float u[kAhead][4], old[kAhead][4];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = i0 + k * kSmallThreads * 4;
            if (i >= all) continue;
            load4(g + i, wide4, all - i, u[k]);
            if (v) load4(v + i, wide4, all - i, old[k]);
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = i0 + k * kSmallThreads * 4;
            if (i >= all) continue;
            const int at = place_of(i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!wide4 && i + j >= all) continue;
                if (v) {
                    old[k][j] += (u[k][j] - old[k][j]) * r.keep;
                    if (!wide4) v[i + j] = old[k][j];
                    u[k][j] = direction(u[k][j], old[k][j], r);
                }
                values[wide4 ? at + j * hop : place_of(i + j)] = u[k][j];
                sum += (double)u[k][j] * (double)u[k][j];
            }
            if (v && wide4) *reinterpret_cast<float4*>(v + i) = make_float4(old[k][0], old[k][1], old[k][2], old[k][3]);
        }
    }
#pragma unroll
    for (int j = 16; j > 0; j >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, j);
    if (lane == 0) part[warp] = sum;
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *const_cast<volatile uint32_t*>(&slot_at);
    sum = 0.0;
    for (int i = 0; i < kSmallThreads / 32; ++i) sum += part[i];
    const Reciprocal by(sum, r.eps);
    float x[64];
    const bool mine = row < small;
#pragma unroll
    for (int j = 0; j < 64; ++j) {
        const int col = group * 64 + j;
        const float u = mine && col < wide ? values[row * kSmallPitch + col] : 0.f;
        x[j] = by.times(u);
    }
    __syncthreads();  // the operands take the values' place
    float one = (float)(fmin(1.0, sqrt(sum) * by.both) * rsqrt((double)small));
    const uint32_t x_at = base, s_at = base + PARTS * (kSmallN / 64) * (kUnit * 2);
    constexpr int kXPart = kSmallN / 64 * kUnit * 2, kSPart = 2 * kUnit * 2;
    // 8 values as an operand's 16 bytes: piece `piece` of this row in a unit
    auto put8 = [&](auto parts, uint32_t unit, int part_bytes, int piece, float* v8, float scale, bool round = false) {
        float2 two[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) two[j] = make_float2(v8[2 * j] * scale, v8[2 * j + 1] * scale);
#pragma unroll
        for (int q = 0; q < decltype(parts)::value; ++q) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = part_of(two[j]);
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(unit + q * part_bytes + row * 128 + ((piece ^ (row & 7)) << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                         : "memory");
        }
        if (round) {  // the values become what the parts hold
#pragma unroll
            for (int j = 0; j < 4; ++j) v8[2 * j] -= two[j].x, v8[2 * j + 1] -= two[j].y;
        }
    };
    constexpr std::integral_constant<int, PARTS> of_type{};
    constexpr std::integral_constant<int, 2>     both{};
    auto put_x = [&](float scale) {
#pragma unroll
        for (int j = 0; j < 8; ++j) put8(of_type, x_at + group * kUnit * 2, kXPart, j, x + 8 * j, scale);
    };
    uint32_t phase = 0;
    bool     ok = true;
    // a product of the operands that all threads have written, by one of them; the others wait for it
    // each: accumulators for 64 of K, `apart` columns apart (0: one for all)
    auto multiply = [&](auto parts, int each, int apart, uint32_t a, int a_part, uint32_t b, int b_part, uint32_t kind, int depth, bool b_mn) {
        fence_before();
        async_fence();
        __syncthreads();
        fence_after();
        if (threadIdx.x == 0) {
            for (int k = 0; k < depth; ++k)
#pragma unroll
                for (int q = decltype(parts)::value == 2 ? 0 : 2; q < 3; ++q)  // of two parts: the small products first
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        product<1>(tmem + (k * each + i * each / 4) * apart, operand(a + (q == 0 ? a_part : 0) + k * kUnit * 2 + i * 32, 8192),
                                   operand(b + (q == 1 ? b_part : 0) + (b_mn ? (k * 4 + i) * 2048 : k * kUnit * 2 + i * 32), kUnit * 2), kind,
                                   q > (decltype(parts)::value == 2 ? 0 : 2) || (each > 0 ? i * each % 4 != 0 : k > 0 || i > 0));
            products_commit<1>(bar);
        }
        uint64_t since = 0;
        for (int i = 1; ok; ++i) {
            if (bar_try(bar, phase)) break;
            if (i % 64) continue;
            uint64_t now;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
            if (since == 0) since = now;
            if (now - since > 4000000000ull) ok = false;
        }
        phase ^= 1;
        fence_after();
    };
    const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16;
    // f32: an accumulator for 64 of K, and for A A, whose errors show most (see segment_of), as many as there is room for: 64 x 256 is off
    // by 1.1e-6 of its norm, with one accumulator each by 2.4e-6 (plain 32 bits: 1.4e-6)
    const int depth_x = units, depth_s = (small + 63) / 64, each = PARTS == 2 ? 4 / depth_s : 0;
    const bool square_too = group < 2 * depth_s;  // A and B have columns for this warp
    if (group < units) put_x(steps.step[0].operand);
    for (int i = 0; i < steps.count; ++i) {
        const SmallStep& f = steps.step[i];
        const float square = one * one, shift = square * (f.b + f.c * square);
        one *= f.a + shift;
        float2 pairs[16];
        float* const sums = reinterpret_cast<float*>(pairs);
        float a[32];
        auto add_up = [&](int count, int apart, int col) {  // 32 columns
            tmem_load32(tmem + lanes + col, pairs);
            tmem_loaded(pairs);
            for (int k = 1; k < count; ++k) {
                float2 more[16];
                tmem_load32(tmem + lanes + k * apart + col, more);
                tmem_loaded(more);
#pragma unroll
                for (int j = 0; j < 16; ++j) pairs[j] = add2(pairs[j], more[j]);
            }
        };
        multiply(of_type, PARTS - 1, 128, x_at, kXPart, x_at, kXPart, half_kind(128, depth_s * 64, false), depth_x, false);  // A = X X^T
        if (square_too) {
            add_up(PARTS == 2 ? depth_x : 1, 128, group * 32);
#pragma unroll
            for (int j = 0; j < 32; ++j) a[j] = sums[j] * f.gram;
#pragma unroll
            for (int j = 0; j < 4; ++j) put8(both, s_at + group / 2 * kUnit * 2, kSPart, group % 2 * 4 + j, a + 8 * j, 1.f, true);  // b A and c A A agree about A
        }
        multiply(both, each, 128, s_at, kSPart, s_at, kSPart, half_kind(128, depth_s * 64, false), depth_s, false);  // B = b A + c A A - t
        if (square_too) {
            add_up(max(1, each * depth_s), 128, group * 32);
            const int hit = row - group * 32;
#pragma unroll
            for (int j = 0; j < 32; ++j) a[j] = fmaf(f.of_gram, a[j], sums[j] * f.square) - (j == hit ? shift * f.of_one : 0.f);
#pragma unroll
            for (int j = 0; j < 4; ++j) put8(of_type, s_at + group / 2 * kUnit * 2, kSPart, group % 2 * 4 + j, a + 8 * j, 1.f);
        }
        multiply(of_type, PARTS - 1, 256, s_at, kSPart, x_at, kXPart, half_kind(128, units * 64, true), depth_s, true);  // (a + t) X + B X
        if (group < units) {
#pragma unroll
            for (int c = 0; c < 64; c += 32) {
                add_up(PARTS == 2 ? depth_s : 1, 256, group * 64 + c);
#pragma unroll
                for (int j = 0; j < 32; ++j) x[c + j] = fmaf(f.a + shift, x[c + j], sums[j] * f.apply);
            }
            if (i + 1 < steps.count) put_x(steps.step[i + 1].operand);
        }
    }
    ok = __syncthreads_and(ok);  // and all products have been read: the values take the operands' place again
#pragma unroll
    for (int j = 0; j < 64; ++j)
        if (mine && group * 64 + j < wide) values[row * kSmallPitch + group * 64 + j] = ok ? x[j] : __uint_as_float(0x7fffffffu);
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 0) tmem_free<1>(tmem, kColumns);
    for (int i0 = threadIdx.x * 4; i0 < all; i0 += kSmallThreads * 4 * kAhead) {
        float was[kAhead][4], held[kAhead][4];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = i0 + k * kSmallThreads * 4;
            if (i >= all || !v) continue;
            load4(p + i, wide4, all - i, was[k]);
            if (master) load4(master + i, wide4, all - i, held[k]);
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = i0 + k * kSmallThreads * 4;
            if (i >= all) continue;
            const int at = place_of(i);
            float o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!wide4 && i + j >= all) continue;
                o[j] = values[wide4 ? at + j * hop : place_of(i + j)];
                if (v) o[j] = updated<X>(was[k][j], master ? held[k][j] : 0.f, master != nullptr, o[j], r, m.rate);
                if (!wide4) {
                    if (master) master[i + j] = o[j];
                    put(p + i + j, o[j]);
                }
            }
            if (wide4) {
                if (master) *reinterpret_cast<float4*>(master + i) = make_float4(o[0], o[1], o[2], o[3]);
                if constexpr (sizeof(X) == 4) {
                    *reinterpret_cast<float4*>(p + i) = make_float4(o[0], o[1], o[2], o[3]);
                } else {
                    uint2 w;
                    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w.x) : "f"(o[1]), "f"(o[0]));
                    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w.y) : "f"(o[3]), "f"(o[2]));
                    *reinterpret_cast<uint2*>(p + i) = w;
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------ host side

struct Matrix {  // `count` of them, one after another
    void*       param;
    const void* grad;
    float*      momentum;
    float*      master;
    int64_t     rows, cols;
    double      rate;
    bool        small() const { return std::min(rows, cols) <= kSmallM && std::max(rows, cols) <= kSmallN; }
};

// Powers of two that bring the operands of each step into the range of fp16, for singular values of at most one before.
struct Step {
    float a, b, c;
    int   x, gram, factor;  // exponents
};

bool steps_of(const double* abc, int count, std::vector<Step>* steps) {
    double most = 1.0 + 1.0 / 1024;  // of the singular values; the first are at most one but for roundings
    auto exponent = [](double bound) { return bound > 0 ? 15 - std::max(-60, (int)std::ceil(std::log2(bound))) : 15; };
    for (int i = 0; i < count; ++i) {
        const double a = abc[3 * i], b = abc[3 * i + 1], c = abc[3 * i + 2];
        if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
        // B, less any of its own values, and the next singular values: largest at the range's end or where a derivative is zero
        double low = 0, high = 0, next = 0;
        auto meet = [&](double square) {
            if (!(square >= 0)) return;
            const double q = std::min(square, most * most), f = q * (b + c * q);
            low = std::min(low, f), high = std::max(high, f), next = std::max(next, std::sqrt(q) * std::fabs(a + f));
        };
        meet(most * most);
        meet(-b / (2 * c));
        const double root = std::sqrt(9 * b * b - 20 * a * c);
        meet((-3 * b + root) / (10 * c)), meet((-3 * b - root) / (10 * c));
        if (c == 0) meet(-a / (3 * b));
        const double factor = 1.01 * (high - low);
        next *= 1.01;
        steps->push_back({(float)a, (float)b, (float)c, exponent(most), exponent(most * most), exponent(factor)});
        if (!(next < 1e6)) return false;
        most = std::max(next, 1e-6);
    }
    return true;
}

struct Chain {  // matrices of a chain of launches, and what its workspace holds
    std::vector<Entry> entry;
    Entry*   table;
    int32_t* failed;
    int64_t  chunks, blocks;
    bool     pairs;  // tiles of pairs of CTAs are possible
    size_t   bytes;
};

Chain chain_of(const Matrix* matrices, int64_t count, int parts, int steps, void* work) {
    Chain c;
    Parts w(work);
    c.failed = w.take<int32_t>(64);
    c.table  = w.take<Entry>(count);
    c.chunks = c.blocks = 0;
    c.entry.resize(count);
    // pairs of CTAs take 256 rows: where that pads little
    double padded = 0, least = 0;
    for (int64_t i = 0; i < count; ++i) {
        const int64_t m = std::min(matrices[i].rows, matrices[i].cols), n = std::max(matrices[i].rows, matrices[i].cols);
        least += (double)up(m, 128) * up(n, 64) * m, padded += (double)up(m, 256) * up(n, 128) * m;
    }
    c.pairs = padded <= 1.1 * least;
    for (int64_t i = 0; i < count; ++i) {
        Entry& e = c.entry[i];
        const Matrix& m = matrices[i];
        e = {};
        e.grad = m.grad, e.momentum = m.momentum, e.param = m.param, e.master = m.master, e.rate = (float)m.rate;
        e.rows = (int)m.rows, e.cols = (int)m.cols;
        e.m = std::min(e.rows, e.cols), e.n = std::max(e.rows, e.cols);
        e.mp = (int)up(e.m, c.pairs ? 256 : 128), e.panels = (int)(up(e.n, c.pairs ? 128 : 64) / 64);
        e.chunks = (int)((m.rows * m.cols + kChunk - 1) / kChunk);
        e.first_chunk = (int)c.chunks, e.first_block = (int)c.blocks;
        c.chunks += e.chunks, c.blocks += ((int64_t)e.panels * (e.mp / 64) + kBlocks - 1) / kBlocks;
        e.partial = w.take<double>(e.chunks);
        e.shift   = w.take<float>(steps);
        const int64_t values = (int64_t)e.panels * e.mp * 64;
        e.x = w.take<float>(values);
        auto units = [&](int* at, int64_t halves) {
            w.used = (size_t)up((int64_t)w.used, kUnit * 2);
            *at = (int)(w.used / (kUnit * 2));
            w.take<__half>(halves);
        };
        for (int& at : e.operand) units(&at, parts * values);
        units(&e.gram, (int64_t)gram_parts(parts, e.m) * e.mp * e.mp), units(&e.factor, (int64_t)parts * e.mp * e.mp);
    }
    c.bytes = (size_t)up((int64_t)w.used, kUnit * 2);
    return c;
}

// How many of the matrices, from the first on, go together: as many as two gigabytes hold.
constexpr size_t kChainBytes = (size_t)2 << 30;
int64_t together(const Matrix* matrices, int64_t count, int parts) {
    size_t bytes = 0;
    int64_t i = 0;
    for (; i < count && i < kMostMatrices; ++i) {
        const int64_t m = std::min(matrices[i].rows, matrices[i].cols), n = std::max(matrices[i].rows, matrices[i].cols);
        const size_t more = (size_t)up(m, 256) * ((size_t)up(n, 128) * (4 + 4 * parts) + (size_t)up(m, 256) * 2 * (parts + gram_parts(parts, (int)std::min<int64_t>(m, 256))));
        if (i > 0 && bytes + more > kChainBytes) break;
        bytes += more;
    }
    return i;
}

bool matrices_ok(const Matrix* m, int64_t count) {
    for (int64_t i = 0; i < count; ++i) {
        const int64_t rows = m[i].rows, cols = m[i].cols;
        // rows of the workspace are counted in 32 bits
        if (rows < 1 || cols < 1 || rows >= ((int64_t)1 << 30) || cols >= ((int64_t)1 << 30) || up(std::min(rows, cols), 256) > ((int64_t)1 << 20) ||
            (double)up(std::min(rows, cols), 256) * up(std::max(rows, cols), 128) >= 1e10)
            return false;
    }
    return true;
}

// A launch of the chain, which may begin before the former has ended (see former_is_done), with CTAs in clusters of `cluster`.
template <typename... P, typename... A>
int follow(void (*kernel)(P...), int64_t grid, int threads, int shared, int cluster, cudaStream_t stream, A&&... args) {
    cudaLaunchConfig_t c = {};
    c.gridDim          = dim3((unsigned)grid);
    c.blockDim         = dim3(threads);
    c.dynamicSmemBytes = shared;
    c.stream           = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster, at[1].val.clusterDim.y = 1, at[1].val.clusterDim.z = 1;
    c.attrs    = at;
    c.numAttrs = cluster > 1 ? 2 : 1;
    FW_TRY(cudaLaunchKernelEx(&c, kernel, std::forward<A>(args)...));
    FW_LAUNCHED();
    return FRAMEWISE_B200_OK;
}

template <int KIND, int PARTS, int CG>
int launch(const CUtensorMap& a, const CUtensorMap& b, const Params& p, int sms, cudaStream_t stream) {
    auto kernel = k_muon_tiles<KIND, PARTS, CG>;
    static std::atomic<uint64_t> allowed{0};
    FW_DO(allow_shared(kernel, kShared, allowed));
    return follow(kernel, std::min(p.tiles, sms / CG) * CG, kThreads, kShared, CG, stream, a, b, p);
}

template <typename X>
int run_chain(Chain& c, const Rates& rates, const std::vector<Step>& steps, char* work, cudaStream_t stream) {
    constexpr int PARTS = sizeof(X) == 4 ? 2 : 1;
    const int sms = sm_count(), count = (int)c.entry.size();
    if (sms < 2) return FRAMEWISE_B200_CUDA_ERROR;
    struct Shape {
        int     pair, wide;
        int64_t tiles;
    };
    auto lay = [&](int pair, int wide, bool apply, bool write) {
        int64_t tiles = 0;
        const int rows = kRowsPerCta * pair;
        for (Entry& e : c.entry) {
            if (write) (apply ? e.first_apply : e.first_sym) = (int)tiles;
            const int mt = e.mp / rows, nt = ((apply ? e.panels * 64 : e.mp) + wide - 1) / wide;
            if (apply) tiles += (int64_t)mt * nt;
            else for (int r = 0; r < mt; ++r) tiles += nt - r * rows / wide;
        }
        return tiles;
    };
    // The shape of the tiles whose time is the shortest by this count: clocks of a stage of 64 of K by what the products take or what
    // a CTA can be fed (48 bytes a clock, measured), some thousand clocks a tile for what does not overlap, and whole rounds.
    auto shape = [&](bool apply) {
        Shape  best = {1, 64, 0};
        double least = 1e300;
        for (int pair = 1; pair <= (c.pairs ? 2 : 1); ++pair)
            for (int wide = 64 * pair; wide <= kMostWide; wide *= 2) {
                const double products = wide * 2.0 * (PARTS == 2 ? 3 : 1), fed = PARTS * (kRowsPerCta + wide / pair) * kDepth * 2 / 48.0;
                const int64_t tiles = lay(pair, wide, apply, false), workers = sms / pair;
                double stages = 0;
                for (const Entry& e : c.entry) stages = std::max(stages, (double)(apply ? (e.m + 63) / 64 : e.panels));
                const double time = (double)((tiles + workers - 1) / workers) * (stages * std::max(products, fed) + 3000);
                if (time < least) least = time, best = {pair, wide, tiles};
            }
        lay(best.pair, best.wide, apply, true);
        return best;
    };
    const Shape sym = shape(false), apply = shape(true);
    if (sym.tiles >= INT32_MAX || apply.tiles >= INT32_MAX || c.chunks >= INT32_MAX || c.blocks >= INT32_MAX || c.bytes / (kUnit * 2) >= INT32_MAX)
        return FRAMEWISE_B200_BAD_ARGUMENT;
    FW_DO(bind_device());
    // 128 rows of a unit; 64 of them; 64 rows of two units
    CUtensorMap tall, square, two;
    const int64_t units = (int64_t)(c.bytes / (kUnit * 2));
    if (!map_of(&tall, work, false, 64, 128, units, 64, kUnit, 64, 128) || !map_of(&square, work, false, 64, 128, units, 64, kUnit, 64, 64) ||
        !map_of(&two, work, false, 64, 128, units, 64, kUnit, 64, 64, 2))
        return FRAMEWISE_B200_TENSOR_MAP;
    FW_TRY(cudaMemsetAsync(c.failed, 0, 4, stream));
    Steps abc;
    abc.count = (int)steps.size();
    for (size_t i = 0; i < steps.size(); ++i) abc.abc[3 * i] = steps[i].a, abc.abc[3 * i + 1] = steps[i].b, abc.abc[3 * i + 2] = steps[i].c;
    for (int i = 0; i < count; i += kSlots) {
        Slots s;
        s.count = std::min(kSlots, count - i), s.base = i, s.table = c.table;
        int64_t chunks = 0;
        for (int j = 0; j < s.count; ++j) s.entry[j] = c.entry[i + j], chunks += s.entry[j].chunks;
        k_muon_collect<X><<<(unsigned)chunks, 256, 0, stream>>>(s, rates);
        FW_LAUNCHED();
    }
    __half* const halves = reinterpret_cast<__half*>(work);
    FW_DO(follow(k_muon_begin<X, PARTS>, c.blocks, 256, 0, 1, stream, (const Entry*)c.table, count, rates, std::ldexp(1.f, steps[0].x), halves, abc));
    auto go = [&](auto kind, const Shape& sh, Params& p) {
        constexpr int KIND = decltype(kind)::value;
        const int other = KIND == kLast ? kEpilogue * kTurn : 0;
        p.tiles = (int)sh.tiles, p.wide = sh.wide;
        p.stages = std::min(kMostStages, (kShared - 1024 - other) / ((kRowsPerCta + sh.wide / sh.pair) * kDepth * 2));
        p.span = std::min(128, sh.wide / sh.pair);
        const CUtensorMap& b = p.span == 64 ? square : KIND == kApply || KIND == kLast ? two : tall;
        return sh.pair == 2 ? launch<KIND, PARTS, 2>(tall, b, p, sms, stream) : launch<KIND, PARTS, 1>(tall, b, p, sms, stream);
    };
    Params p = {};
    p.table = c.table, p.count = count, p.work = halves, p.failed = c.failed, p.rates = rates;
    for (size_t i = 0; i < steps.size(); ++i) {
        const Step& s = steps[i];
        p.step = (int)i, p.from = (int)(i & 1);
        p.product = std::ldexp(1.f, s.gram - 2 * s.x);
        FW_DO(go(std::integral_constant<int, kGram>(), sym, p));
        p.product = std::ldexp(s.c, s.factor - 2 * s.gram), p.old = std::ldexp(s.b, s.factor - s.gram), p.scale = std::ldexp(1.f, s.factor);
        FW_DO(go(std::integral_constant<int, kSquare>(), sym, p));
        const bool last = i + 1 == steps.size();
        p.product = std::ldexp(1.f, -s.factor - s.x), p.old = s.a, p.scale = last ? 0.f : std::ldexp(1.f, steps[i + 1].x);
        if (last) FW_DO(go(std::integral_constant<int, kLast>(), apply, p));
        else FW_DO(go(std::integral_constant<int, kApply>(), apply, p));
    }
    return follow(k_muon_check<X>, sms, 256, 0, 1, stream, (const Entry*)c.table, count, (const int*)c.failed);
}

size_t bytes_for(const std::vector<Matrix>& list, int parts) {
    // (room for the most steps, so that it does not depend on them)
    size_t most = 256;
    for (size_t i = 0; i < list.size();) {
        const int64_t n = together(list.data() + i, (int64_t)(list.size() - i), parts);
        most = std::max(most, chain_of(list.data() + i, n, parts, kMostSteps, nullptr).bytes);
        i += n;
    }
    return most;
}

template <typename X>
int run_small(const std::vector<SmallSlot>& slots, const Rates& rates, const std::vector<Step>& steps, cudaStream_t stream) {
    constexpr int PARTS = sizeof(X) == 4 ? 2 : 1;
    static std::atomic<uint64_t> allowed{0};
    FW_DO(allow_shared(k_muon_small<X>, small_bytes(PARTS), allowed));
    SmallSteps f;
    f.count = (int)steps.size();
    for (size_t i = 0; i < steps.size(); ++i) {
        const Step& t = steps[i];
        f.step[i] = {std::ldexp(1.f, t.gram - 2 * t.x), std::ldexp(t.c, t.factor - 2 * t.gram), std::ldexp(t.b, t.factor - t.gram), std::ldexp(1.f, t.factor),
                     std::ldexp(1.f, -t.factor - t.x), t.a, std::ldexp(1.f, t.x), t.b, t.c};
    }
    for (size_t i = 0; i < slots.size(); i += kSlots) {
        SmallSlots s;
        s.count = (int)std::min<size_t>(kSlots, slots.size() - i);
        int64_t grid = 0;
        for (int j = 0; j < s.count; ++j) s.slot[j] = slots[i + j], grid += s.slot[j].count;
        k_muon_small<X><<<(unsigned)grid, kSmallThreads, small_bytes(PARTS), stream>>>(s, rates, f);
        FW_LAUNCHED();
    }
    return FRAMEWISE_B200_OK;
}

// the matrices that a CTA holds, and the others
int run(const std::vector<SmallSlot>& small, const std::vector<Matrix>& list, int dtype, const Rates& rates, const double* coefficients, int steps, void* work,
        size_t work_bytes, cudaStream_t stream) {
    if (list.empty() && small.empty()) return FRAMEWISE_B200_OK;
    const int parts = dtype == FRAMEWISE_B200_F32 ? 2 : 1;
    std::vector<Step> plan;
    if (!work || misaligned(work) || !coefficients || steps < 1 || steps > kMostSteps || !steps_of(coefficients, steps, &plan)) return FRAMEWISE_B200_BAD_ARGUMENT;
    if (work_bytes < bytes_for(list, parts)) return FRAMEWISE_B200_WORKSPACE;
    FW_DO(dtype == FRAMEWISE_B200_F32 ? run_small<float>(small, rates, plan, stream) : run_small<__nv_bfloat16>(small, rates, plan, stream));
    for (size_t i = 0; i < list.size();) {
        const int64_t n = together(list.data() + i, (int64_t)(list.size() - i), parts);
        Chain c = chain_of(list.data() + i, n, parts, kMostSteps, work);
        FW_DO(dtype == FRAMEWISE_B200_F32 ? run_chain<float>(c, rates, plan, static_cast<char*>(work), stream)
                                          : run_chain<__nv_bfloat16>(c, rates, plan, static_cast<char*>(work), stream));
        i += n;
    }
    return FRAMEWISE_B200_OK;
}

bool dtype_ok(int dtype) { return dtype == FRAMEWISE_B200_F32 || dtype == FRAMEWISE_B200_BF16; }

// the matrices of a Muon step; those without values are passed over
int muon_list(const framewise_b200_matrix* matrices, int64_t count, double lr, int adjust, std::vector<SmallSlot>* small, std::vector<Matrix>* list) {
    if (count < 0 || (count > 0 && !matrices)) return FRAMEWISE_B200_BAD_ARGUMENT;
    for (int64_t i = 0; i < count; ++i) {
        const framewise_b200_matrix& m = matrices[i];
        if (m.rows < 0 || m.cols < 0) return FRAMEWISE_B200_BAD_ARGUMENT;
        if (m.rows == 0 || m.cols == 0) continue;
        const double by = adjust ? 0.2 * std::sqrt((double)std::max(m.rows, m.cols)) : std::sqrt(std::max(1.0, (double)m.rows / m.cols));
        const Matrix one = {m.param, m.grad, m.momentum, m.master, m.rows, m.cols, lr * by};
        if (one.small()) small->push_back({m.grad, m.momentum, m.param, m.master, 0, (int)m.rows, (int)m.cols, 1, (float)one.rate});
        else list->push_back(one);
    }
    return matrices_ok(list->data(), (int64_t)list->size()) ? FRAMEWISE_B200_OK : FRAMEWISE_B200_BAD_ARGUMENT;
}

// Whether something that a step writes overlaps something else that it writes or reads.  (The momentum is written before the gradient
// is read again, and matrices are not done in order.)
bool overlaps(const framewise_b200_matrix* matrices, int64_t count, int64_t size) {
    struct Range {
        uintptr_t begin, end;
        bool      written;
    };
    std::vector<Range> ranges;
    ranges.reserve(4 * count);
    for (int64_t i = 0; i < count; ++i) {
        const framewise_b200_matrix& m = matrices[i];
        if (m.rows == 0 || m.cols == 0) continue;
        auto add = [&](const void* at, int64_t each, bool written) {
            const uintptr_t begin = reinterpret_cast<uintptr_t>(at);
            ranges.push_back({begin, begin + (uintptr_t)(m.rows * m.cols * each), written});
        };
        add(m.param, size, true), add(m.grad, size, false), add(m.momentum, 4, true);
        if (m.master) add(m.master, 4, true);
    }
    std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
    uintptr_t written = 0, any = 0;  // where the ranges so far end
    for (const Range& r : ranges) {
        if (r.begin < (r.written ? any : written)) return true;
        any = std::max(any, r.end);
        if (r.written) written = std::max(written, r.end);
    }
    return false;
}

// `count` matrices of one shape, one after another
int batch_list(int64_t count, int64_t rows, int64_t cols, int dtype, const void* x, void* out, std::vector<SmallSlot>* small, std::vector<Matrix>* list) {
    const int64_t values = rows * cols, bytes = values * (dtype == FRAMEWISE_B200_F32 ? 4 : 2);
    const Matrix  one = {out, x, nullptr, nullptr, rows, cols, 0.0};
    if (one.small()) {
        constexpr int64_t kMost = 1 << 26;  // of a slot: the CTAs of a launch's slots stay below 2^31
        for (int64_t i = 0; i < count; i += kMost)
            small->push_back({x ? static_cast<const char*>(x) + i * bytes : nullptr, nullptr, out ? static_cast<char*>(out) + i * bytes : nullptr, nullptr, values, (int)rows,
                              (int)cols, (int)std::min<int64_t>(count - i, kMost), 0.f});
        return FRAMEWISE_B200_OK;
    }
    if (!matrices_ok(&one, 1)) return FRAMEWISE_B200_BAD_ARGUMENT;
    for (int64_t i = 0; i < count; ++i)
        list->push_back({out ? static_cast<char*>(out) + i * bytes : nullptr, x ? static_cast<const char*>(x) + i * bytes : nullptr, nullptr, nullptr, rows, cols, 0.0});
    return FRAMEWISE_B200_OK;
}

}  // namespace

extern "C" {

size_t framewise_b200_muon_bytes(const framewise_b200_matrix* matrices, int64_t count, int32_t dtype) try {
    std::vector<SmallSlot> small;
    std::vector<Matrix>    list;
    if (!dtype_ok(dtype) || muon_list(matrices, count, 0.0, 0, &small, &list) != FRAMEWISE_B200_OK) return 0;
    return bytes_for(list, dtype == FRAMEWISE_B200_F32 ? 2 : 1);
} catch (...) {  // no memory for the lists
    return 0;
}

int framewise_b200_muon(const framewise_b200_matrix* matrices, int64_t count, int32_t dtype, double lr, double beta, int32_t nesterov,
                        double weight_decay, int32_t match_rms, const double* coefficients, int32_t steps, double eps, int32_t follow,
                        void* work, size_t work_bytes, framewise_b200_stream_t stream) try {
    std::vector<SmallSlot> small;
    std::vector<Matrix>    list;
    if (!dtype_ok(dtype) || !(eps > 0)) return FRAMEWISE_B200_BAD_ARGUMENT;
    FW_DO(muon_list(matrices, count, lr, match_rms, &small, &list));
    auto bad = [&](const auto& m) { return !m.param || !m.grad || !m.momentum || (m.master && dtype == FRAMEWISE_B200_F32); };
    if (std::any_of(list.begin(), list.end(), bad) || std::any_of(small.begin(), small.end(), bad)) return FRAMEWISE_B200_BAD_ARGUMENT;
    if (overlaps(matrices, count, dtype == FRAMEWISE_B200_F32 ? 4 : 2)) return FRAMEWISE_B200_OVERLAP;
    const Rates rates = {eps, (float)(1 - beta), (float)beta, nesterov ? 1.f : 0.f, (float)(1 - lr * weight_decay), follow};
    return run(small, list, dtype, rates, coefficients, steps, work, work_bytes, stream);
} catch (...) {
    return FRAMEWISE_B200_BAD_ARGUMENT;
}

size_t framewise_b200_orthogonalize_bytes(int64_t count, int64_t rows, int64_t cols, int32_t dtype) try {
    if (!dtype_ok(dtype) || count < 0 || rows < 0 || cols < 0) return 0;
    if (count == 0 || rows == 0 || cols == 0) return 256;
    std::vector<SmallSlot> small;
    std::vector<Matrix>    list;
    // more than a chain's go through the same scratch
    if (batch_list(std::min<int64_t>(count, kMostMatrices), rows, cols, dtype, nullptr, nullptr, &small, &list) != FRAMEWISE_B200_OK) return 0;
    return bytes_for(list, dtype == FRAMEWISE_B200_F32 ? 2 : 1);
} catch (...) {
    return 0;
}

int framewise_b200_orthogonalize(int64_t count, int64_t rows, int64_t cols, int32_t dtype, const void* x, void* out, const double* coefficients,
                                 int32_t steps, double eps, void* work, size_t work_bytes, framewise_b200_stream_t stream) try {
    if (!dtype_ok(dtype) || count < 0 || rows < 0 || cols < 0 || !(eps > 0)) return FRAMEWISE_B200_BAD_ARGUMENT;
    if (count == 0 || rows == 0 || cols == 0) return FRAMEWISE_B200_OK;
    if (!x || !out) return FRAMEWISE_B200_BAD_ARGUMENT;
    std::vector<SmallSlot> small;
    std::vector<Matrix>    list;
    FW_DO(batch_list(count, rows, cols, dtype, x, out, &small, &list));
    const Rates rates = {eps, 0.f, 0.f, 0.f, 1.f, 0};
    return run(small, list, dtype, rates, coefficients, steps, work, work_bytes, stream);
} catch (...) {
    return FRAMEWISE_B200_BAD_ARGUMENT;
}

}  // extern "C"
