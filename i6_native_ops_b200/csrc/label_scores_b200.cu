// label_scores_b200.cu -- what a program reads off distributions over the classes that are in memory, behind the C ABI of
// include/framewise_b200.h: log probabilities of given labels, entropies, the best alternatives, and their gradient.
//
// With z a row of V logits, t its label, m = max z, s = sum 2^d, d = (z - m) log2 e:
//     log p = ln 2 (d - log2 s);  entropy = ln 2 (log2 s - (sum 2^d d) / s)
//     alternatives: the `top` largest of z, equal ones by their index
//     dz = g (onehot(t) - p) - g_H p (log p + entropy) + sum_j g_j (onehot(top_j) - p)
// The forward pass meets each logit once and keeps of a row its maximum, log2 s and entropy; the backward pass meets it once
// more and writes the gradient.  (The maximum is kept apart from log2 s: their sum would round off what lies near one.)
#include "framewise_b200.h"
#include "framewise_host.h"
#include "tensor_core.h"

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>

namespace {

using namespace framewise_host;
using namespace tensor_core;

constexpr int   kMostTop  = 32;      // alternatives: one per lane
constexpr int   kWarps    = 8;       // per CTA
constexpr int   kMostTeam = 64;      // warps that share a row: up to 8 CTAs
constexpr int   kCell     = 4;       // vectors of 8 logits that a lane has in a cell (see Best)
constexpr int   kCells    = 16;      // cells of a lane between looks for the best
constexpr int   kFew      = 8;       // alternatives that the lanes' largest cells alone single out well
constexpr float kLog2e    = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNever    = -200.f;  // of an exponent of 2: zero in 32 bits

struct Rows {  // where the rows are and which count
    int64_t        N;
    int            T, V, top, team;  // team: warps per row, a power of two
    int64_t        stride_b, stride_t;
    const void*    labels;
    const int32_t* lens;
    int64_t        ignore;
};

template <typename L>
__device__ __forceinline__ bool counted(const Rows& r, int64_t n, int64_t& label) {
    label = static_cast<const L*>(r.labels)[n];
    return (r.lens == nullptr || (int)((uint32_t)n % (uint32_t)r.T) < r.lens[(uint32_t)n / (uint32_t)r.T]) && label != r.ignore;
}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if one is
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
    return d;
}

// 8 logits in a row, as they are in memory (aligned: 32 bytes for f32, 16 for bf16)
template <typename X>
struct Raw;
template <>
struct Raw<float> {
    float w[8];
    __device__ __forceinline__ void load(const float* x) {
        asm volatile("ld.global.L1::no_allocate.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=f"(w[0]), "=f"(w[1]), "=f"(w[2]), "=f"(w[3]), "=f"(w[4]), "=f"(w[5]), "=f"(w[6]), "=f"(w[7])
                     : "l"(x));
    }
    __device__ __forceinline__ void set(int i, const float* x) { w[i] = x ? *x : -INFINITY; }
    __device__ __forceinline__ void none() {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = -INFINITY;
    }
    __device__ __forceinline__ float get(int i) const { return w[i]; }
};
template <>
struct Raw<__nv_bfloat16> {
    uint32_t w[4];
    __device__ __forceinline__ void load(const __nv_bfloat16* x) {
        asm volatile("ld.global.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(x));
    }
    __device__ __forceinline__ void set(int i, const __nv_bfloat16* x) {
        const uint32_t v = x ? *reinterpret_cast<const uint16_t*>(x) : 0xff80u;  // -inf
        w[i / 2] = i % 2 ? (w[i / 2] & 0xffffu) | v << 16 : v;
    }
    __device__ __forceinline__ void none() {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = 0xff80ff80u;
    }
    __device__ __forceinline__ float get(int i) const { return __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16); }
};
// The largest of kCell vectors' values.
__device__ __forceinline__ float largest(const Raw<float>* v) {
    float a = max_nan(v[0].get(0), v[0].get(1), v[0].get(2)), b = max_nan(v[0].get(3), v[0].get(4), v[0].get(5));
    a = max_nan(a, v[0].get(6), v[0].get(7));
#pragma unroll
    for (int i = 1; i < kCell; ++i) {
        a = max_nan(max_nan(a, v[i].get(0), v[i].get(1)), v[i].get(2), v[i].get(3));
        b = max_nan(max_nan(b, v[i].get(4), v[i].get(5)), v[i].get(6), v[i].get(7));
    }
    return max_nan(a, b);
}
// (Of the unpacked values the compiler would keep 64 until the sums are formed, some of them in local memory.)
__device__ __forceinline__ float largest(const Raw<__nv_bfloat16>* v) {
    uint32_t a = v[0].w[0];
#pragma unroll
    for (int i = 0; i < kCell; ++i)
#pragma unroll
        for (int j = i == 0 ? 1 : 0; j < 4; ++j) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(v[i].w[j]));
    return max_nan(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u));
}
__device__ __forceinline__ float value(float x) { return x; }
__device__ __forceinline__ float value(__nv_bfloat16 x) { return __bfloat162float(x); }

// A lane has 128 bytes under way: a block of so many vectors.  (bf16, 20000 x 12001: 89 us, and the gradient 170; half of them with
// the next half loaded before they are worked on took 4 and 14 us more.)
template <typename X>
constexpr int kAhead = 128 / (8 * (int)sizeof(X));

// A row in vectors of 8, 32 of them a step.  The vectors' addresses are aligned: the first begins `ahead` places before the row.
// Those from `low` to `high` are inside of it.
template <typename X>
struct Row {
    const X* x;
    int      V, ahead, low, high;
    __device__ Row(const X* x, int V) : x(x), V(V) {
        ahead = (int)(reinterpret_cast<uintptr_t>(x) / sizeof(X) % 8);
        low = ahead > 0, high = (V + ahead) / 8;
    }
    __device__ __forceinline__ int first(int step, int lane) const { return (step * 32 + lane) * 8 - ahead; }
    // A block: kAhead<X> steps, `team` apart.
    __device__ __forceinline__ bool inside(int step, int team) const {
        return step * 32 >= low && (step + (kAhead<X> - 1) * team + 1) * 32 <= high;
    }
    __device__ __forceinline__ void load_inside(int step, int team, int lane, Raw<X> (&v)[kAhead<X>]) const {
        const X* const from = x + first(step, lane);
#pragma unroll
        for (int i = 0; i < kAhead<X>; ++i) v[i].load(from + (int64_t)i * team * 256);
    }
    // The vectors inside of the row; -inf, which changes no sum, in place of others.
    __device__ __forceinline__ void load_whole(int step, int team, int lane, Raw<X> (&v)[kAhead<X>]) const {
        if (inside(step, team)) return load_inside(step, team, lane, v);
#pragma unroll
        for (int i = 0; i < kAhead<X>; ++i) {
            const int q = (step + i * team) * 32 + lane;
            if (q >= low && q < high) v[i].load(x + q * 8 - ahead);
            else v[i].none();
        }
    }
    // Where in the row the value is that a lane takes of the two vectors that lie partly outside; -1: none.
    __device__ __forceinline__ int edge(int lane) const {
        if (lane < 8) return low && lane >= ahead && lane - ahead < V ? lane - ahead : -1;
        return lane < 16 && !(low && high == 0) && high * 8 - ahead + lane - 8 < V ? high * 8 - ahead + lane - 8 : -1;
    }
    // All values inside of the row, one by one where they are not `aligned` or a vector is not whole.
    __device__ __forceinline__ void load(int step, int team, int lane, Raw<X> (&v)[kAhead<X>], bool aligned) const {
        if (aligned && inside(step, team)) return load_inside(step, team, lane, v);
#pragma unroll
        for (int i = 0; i < kAhead<X>; ++i) {
            const int at = first(step + i * team, lane);
            if (aligned && at >= 0 && at + 8 <= V) {
                v[i].load(x + at);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i].set(j, at + j >= 0 && at + j < V ? x + at + j : nullptr);
            }
        }
    }
};

// Larger values have larger keys, equal ones those of the lower index; NaN is the largest value.  0: no value.
__device__ __forceinline__ uint64_t key_of(float v, int index) {
    const uint32_t u = __float_as_uint(v + 0.f);  // one zero
    const uint32_t o = v != v ? 0xffffffffu : (u >> 31) ? ~u : u | 0x80000000u;
    return (uint64_t)o << 32 | (uint32_t)~index;
}
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return o == 0xffffffffu ? __uint_as_float(0x7fffffffu) : __uint_as_float((o >> 31) ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int index_of(uint64_t key) { return (int)~(uint32_t)key; }

__device__ __forceinline__ uint64_t keep(uint64_t a, uint64_t b, bool larger) { return (a > b) == larger ? a : b; }

// Networks of Batcher's over the lanes: `key` in falling order; a falling `list` and the 32 largest of it and `more` (falling).
__device__ __forceinline__ uint64_t sorted(uint64_t key, int lane) {
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1)
            key = keep(key, __shfl_xor_sync(0xffffffffu, key, j), ((lane & j) == 0) == ((lane & k) == 0));
    return key;
}
__device__ __forceinline__ uint64_t joined(uint64_t list, uint64_t more, int lane) {
    list = max(list, __shfl_sync(0xffffffffu, more, 31 - lane));
#pragma unroll
    for (int j = 16; j > 0; j >>= 1) list = keep(list, __shfl_xor_sync(0xffffffffu, list, j), (lane & j) == 0);
    return list;
}

// One copy of the networks, and six cells at a time in Best::look, so that the instructions stay in their cache (20000 x 12001 f32
// with 8 alternatives: a dozen copies 225 us, one 213, six cells instead of a dozen 198).
__device__ __noinline__ uint64_t merged(uint64_t list, uint64_t key, int lane) { return joined(list, sorted(key, lane), lane); }

struct Sums {  // of a part of a row: maximum, sum of 2^d, sum of 2^d d
    float m, s, t;
};
__device__ __forceinline__ void rescale(Sums& a, float m) {
    const float d = max_nan((a.m - m) * kLog2e, kNever), c = exp2_approx(d);
    a.t = c * (a.t + a.s * d);
    a.s = c * a.s;
    a.m = m;
}
__device__ __forceinline__ Sums joined(Sums a, Sums b) {
    const float m = max_nan(a.m, b.m);
    rescale(a, m), rescale(b, m);
    return {m, a.s + b.s, a.t + b.t};
}

// The lanes' values in falling order.
__device__ __forceinline__ float falling(float v, int lane) {
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) {
            const float o = __shfl_xor_sync(0xffffffffu, v, j);
            v = ((lane & j) == 0) == ((lane & k) == 0) ? fmaxf(v, o) : fminf(v, o);
        }
    return v;
}

// What a warp needs to find a row's best.
struct Room {
    float    cell[kCells][32];
    uint16_t near[kCells * 32];
    uint64_t wait[64];
};

// The best that a warp has met.  While the sums are formed only the maximum of each cell, 32 values of a lane in kCell steps
// that the team takes in turn, is written down.  After kCells of them, or at the row's end, those cells are read again whose maximum is no smaller
// than the `top`-th largest of the lanes' maxima: some more than `top` of them.  (Looking at each value while the sums are formed,
// against the list so far: 26 instructions a value for the whole kernel, 20000 x 12001 f32 with 8 alternatives 664 us; 199 this way,
// and 148 without alternatives.)
struct Best {
    uint64_t list;    // the 32 largest so far, a lane each, in falling order
    Room&    room;
    int      count, top;
    float    least;   // the last of the list that counts
    bool     full;
    __device__ Best(Room& room, int top) : list(0), room(room), count(0), top(top), least(-INFINITY), full(false) {}
    // those that wait; more than 32 never do, so that a row in rising order costs a network per 32 of its values
    __device__ void sort_in(int lane) {
        __syncwarp();
        const uint64_t key = lane < min(count, 32) ? room.wait[lane] : 0, rest = lane + 32 < count ? room.wait[lane + 32] : 0;
        __syncwarp();
        list  = merged(list, key, lane);
        count = max(0, count - 32);
        if (lane < count) room.wait[lane] = rest;
        const uint64_t last = __shfl_sync(0xffffffffu, list, top - 1);
        full  = last != 0;
        least = full ? value_of(last) : -INFINITY;
        __syncwarp();
    }
    template <typename X>
    __device__ void look(const Row<X>& row, int step, int team, int blocks, int lane) {  // blocks: of cells, from `step` on
        __syncwarp();
        float most = -INFINITY, second = -INFINITY;
        for (int b = 0; b < blocks; ++b) {
            float c = room.cell[b][lane];
            c = c != c ? INFINITY : c;
            second = fmaxf(second, fminf(most, c)), most = fmaxf(most, c);
        }
        // The `top`-th largest of the lanes' maxima, or of their two largest cells: as many cells' are no smaller.
        float order = falling(most, lane);
        if (top > kFew) {
            order = fmaxf(order, __shfl_sync(0xffffffffu, falling(second, lane), 31 - lane));
#pragma unroll
            for (int j = 16; j > 0; j >>= 1) {
                const float o = __shfl_xor_sync(0xffffffffu, order, j);
                order = (lane & j) == 0 ? fmaxf(order, o) : fminf(order, o);
            }
        }
        const float from = __shfl_sync(0xffffffffu, order, top - 1);
        int cells = 0;
        for (int b = 0; b < blocks; ++b) {
            const float    c = room.cell[b][lane];
            const bool     in = !(c < from) && !(full && c <= least);
            const uint32_t lanes = __ballot_sync(0xffffffffu, in);
            if (in) room.near[cells + __popc(lanes & ((1u << lane) - 1))] = (uint16_t)(b * 32 + lane);
            cells += __popc(lanes);
        }
        __syncwarp();
        // What the list holds when a block begins has lower indices than the block's values: equal ones stay out.  Within a block
        // they come in any order, and equal ones come in.  (NaN: nothing is larger, and `least` is as large.)
        int   block = -1;
        bool  before = false;
        float floor = -INFINITY;
        const int begin = row.low * 8 - row.ahead;  // the vectors inside of the row
        const uint32_t span = max(0, row.high - row.low) * 8;
        constexpr int kLoads = 6;  // cells
        for (int i = 0; i < cells; i += kLoads) {
            float v[kLoads];
            int   at[kLoads];
#pragma unroll
            for (int q = 0; q < kLoads; ++q) {
                v[q] = -INFINITY, at[q] = begin - 1;
                if (i + q >= cells) continue;
                const int cell = room.near[i + q];
                const float c = room.cell[cell / 32][cell % 32];
                if (cell / 32 != block && full && (c <= least || least != least)) continue;  // has been overtaken
                at[q] = row.first(step + (cell / 32 * kCell + lane / 8) * team, cell % 32) + lane % 8;
                if ((uint32_t)(at[q] - begin) < span) v[q] = value(row.x[at[q]]);
            }
#pragma unroll
            for (int q = 0; q < kLoads; ++q) {
                if (i + q >= cells) break;
                const int cell = room.near[i + q];
                if (cell / 32 != block) block = cell / 32, before = full, floor = least;
                const bool in = (uint32_t)(at[q] - begin) < span && !(v[q] < from) && !(before && (v[q] <= floor || floor != floor)) && !(v[q] < least);
                const uint32_t lanes = __ballot_sync(0xffffffffu, in);
                if (in) room.wait[count + __popc(lanes & ((1u << lane) - 1))] = key_of(v[q], at[q]);
                count += __popc(lanes);
                if (count >= 32) sort_in(lane);
            }
        }
        while (count > 0) sort_in(lane);
    }
    // one more value a lane; index < 0: none
    __device__ __forceinline__ void take(float v, int index, int lane) {
        const bool in = index >= 0 && !(v < least);
        if (__any_sync(0xffffffffu, in)) list = merged(list, in ? key_of(v, index) : 0, lane);
    }
};

struct Scored {
    float*  log_prob;
    float*  entropy;
    float*  top_log_prob;
    void*   top_label;
    float4* kept;  // or null: maximum, log2 s, entropy
};

// A row per team of r.team warps (1 to 8 of a CTA; 16 to 64: all of 2 to 8 CTAs of a cluster), which take its steps of 256
// logits in turn.  f32 without alternatives is bound by memory (20000 x 12001 6.5 TB/s), bf16 by exponentials and the instructions
// around them (5.3 TB/s).  Three CTAs an SM where the registers of four do not do (f32 with 8 alternatives 221 us for 199).
template <typename X, typename L, bool TOP>
__global__ void __launch_bounds__(kWarps * 32, sizeof(X) == 4 && !TOP ? 4 : 3) k_label_scores(const X* __restrict__ z, const Rows r, const Scored out) {
    __shared__ Sums     part[kWarps];
    __shared__ uint64_t best[TOP ? kWarps : 1][32];
    __shared__ Room     room[TOP ? kWarps : 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ctas = r.team > kWarps ? r.team / kWarps : 1, in_cta_team = min(r.team, kWarps);
    const int rank = ctas > 1 ? (int)(blockIdx.x % ctas) : 0;
    const int64_t n = ctas > 1 ? (int64_t)(blockIdx.x / ctas) : (int64_t)blockIdx.x * (kWarps / r.team) + warp / r.team;
    const int member = rank * kWarps + warp % in_cta_team;
    int64_t label = 0;
    const bool inside = n < r.N, counts = inside && counted<L>(r, n, label);
    const X* const x = counts ? z + (int64_t)((uint32_t)n / (uint32_t)r.T) * r.stride_b + (int64_t)((uint32_t)n % (uint32_t)r.T) * r.stride_t : z;

    float at_label = __uint_as_float(0x7fffffffu);  // NaN outside of the vocabulary
    if (counts && member == 0 && lane == 0 && label >= 0 && label < r.V) at_label = value(x[label]);
    Sums a = {-FLT_MAX, 0.f, 0.f};
    Best b(room[TOP ? warp : 0], r.top);
    if (counts) {
        const Row<X> row(x, r.V);
        constexpr int A = kAhead<X>;
        Raw<X> v[A];
        const int hop = r.team * A, steps = (row.high + 31) / 32, edge = member == 0 ? row.edge(lane) : -1;
        int cells = 0, looked = member;
        if (member < steps) row.load_whole(member, r.team, lane, v);
        const float at_edge = edge >= 0 ? value(x[edge]) : 0.f;
        if (edge >= 0) {
            a.m = max_nan(a.m, at_edge);
            a.s = exp2_approx(max_nan((at_edge - a.m) * kLog2e, kNever));
        }
        for (int step = member; step < steps; step += hop) {
            const bool more = step + hop < steps;
            float all = -FLT_MAX;
#pragma unroll
            for (int c = 0; c < A; c += kCell) {
                const float of = largest(v + c);
                all = max_nan(all, of);
                if (TOP) room[warp].cell[cells++][lane] = of;
            }
            const float m = max_nan(a.m, all);
            rescale(a, m);
            const float2 off = make_float2(-m, -m), scale = make_float2(kLog2e, kLog2e);
            float2 s = make_float2(0.f, 0.f), t = s;
#pragma unroll
            for (int i = 0; i < A; ++i)
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    float2 d = mul2(add2(make_float2(v[i].get(j), v[i].get(j + 1)), off), scale);
                    d = make_float2(max_nan(d.x, kNever), max_nan(d.y, kNever));
                    const float2 e = make_float2(exp2_approx(d.x), exp2_approx(d.y));
                    s = add2(s, e);
                    t = fma2(e, d, t);
                }
            a.s += s.x + s.y;
            a.t += t.x + t.y;
            if (TOP && (cells == kCells || !more)) {
                b.look(row, looked, r.team, cells, lane);
                cells = 0, looked = step + hop;
            }
            if (more) row.load_whole(step + hop, r.team, lane, v);
        }
        if (TOP) b.take(at_edge, edge, lane);
#pragma unroll
        for (int j = 16; j > 0; j >>= 1) a = joined(a, {__shfl_xor_sync(0xffffffffu, a.m, j), __shfl_xor_sync(0xffffffffu, a.s, j), __shfl_xor_sync(0xffffffffu, a.t, j)});
        // the lanes' sums may differ in their last bit: all go by the first's, so that equal logits have equal results
        a = {__shfl_sync(0xffffffffu, a.m, 0), __shfl_sync(0xffffffffu, a.s, 0), __shfl_sync(0xffffffffu, a.t, 0)};
    }
    // the team's parts, pairs of warps at a time
    if (r.team > 1) {
        if (lane == 0) part[warp] = a;
        if (TOP) best[warp][lane] = b.list;
        for (int j = 1; j < in_cta_team; j <<= 1) {
            __syncthreads();
            if ((warp & (2 * j - 1)) == 0) {
                a = joined(a, part[warp + j]);
                if (lane == 0) part[warp] = a;
                if constexpr (TOP) {
                    b.list = joined(b.list, best[warp + j][lane], lane);
                    best[warp][lane] = b.list;
                }
            }
        }
        if (ctas > 1) {
            cluster_sync();
            if (rank == 0 && warp == 0) {
                for (int j = 1; j < ctas; ++j) {
                    const uint32_t from = in_cta(smem_addr(&part[0]), j);
                    Sums o;
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.m) : "r"(from) : "memory");
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.s) : "r"(from + 4) : "memory");
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.t) : "r"(from + 8) : "memory");
                    a = joined(a, o);
                    if constexpr (TOP) {
                        uint64_t key;
                        asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(key) : "r"(in_cta(smem_addr(&best[0][lane]), j)) : "memory");
                        b.list = joined(b.list, key, lane);
                    }
                }
            }
            cluster_sync();  // what is read from a CTA is there until it has been
        }
    }
    if (member != 0 || !inside) return;
    // a row without a class that is possible has log probabilities of -inf and no entropy
    const float log2_s = log2f(a.s), entropy = a.s == 0.f ? 0.f : kLn2 * (log2_s - a.t / a.s);
    // each operation rounded by itself, so that the label's and its alternative's are equal to the last bit
    const float log_s = logf(a.s);
    auto log_prob = [&](float v) { return a.s == 0.f ? -INFINITY : __fsub_rn(__fsub_rn(v, a.m), log_s); };
    if (lane == 0) {
        out.log_prob[n] = !counts ? 0.f : at_label != at_label ? at_label : log_prob(at_label);
        out.entropy[n]  = counts ? entropy : 0.f;
        if (out.kept) out.kept[n] = make_float4(a.m, log2_s, entropy, 0.f);
    }
    if constexpr (TOP) {
        // In the order of the logits, which no rounding touches: what is left of two of them after the maximum and the logarithm are
        // taken off may be equal, and the last bit of the sum, which hangs on how many warps share the row, then decided.
        if (lane < r.top) {
            out.top_log_prob[n * r.top + lane] = counts ? log_prob(value_of(b.list)) : 0.f;
            static_cast<L*>(out.top_label)[n * r.top + lane] = counts ? (L)index_of(b.list) : (L)r.ignore;
        }
    }
}

struct Incoming {  // strides in elements; null: none
    const float *log_prob, *entropy, *top;
    int64_t log_prob_b, log_prob_t, entropy_b, entropy_t, top_b, top_t, top_k;
    const void*   top_label;
    const float4* kept;
};

__device__ __forceinline__ void store8(float* to, const float (&v)[8]) {
    asm volatile("st.global.L1::no_allocate.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
                 "f"(v[5]), "f"(v[6]), "f"(v[7])
                 : "memory");
}
__device__ __forceinline__ void store8(__nv_bfloat16* to, const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
    asm volatile("st.global.L1::no_allocate.v4.b32 [%0], {%1,%2,%3,%4};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}
__device__ __forceinline__ void put(float* to, float v) { *to = v; }
__device__ __forceinline__ void put(__nv_bfloat16* to, float v) { *to = __float2bfloat16_rn(v); }

// The gradient: a row per team as above, in steps that are aligned where it is written (`even`: and where it is read).
template <typename X, typename L>
__global__ void __launch_bounds__(kWarps * 32, sizeof(X) == 4 ? 4 : 3) k_label_scores_back(const X* __restrict__ z, const Rows r, const Incoming in, X* __restrict__ dz) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t all = (int64_t)blockIdx.x * kWarps + warp, n = all / r.team;
    const int member = (int)(all % r.team);
    if (n >= r.N) return;
    const int64_t seq = (uint32_t)n / (uint32_t)r.T, at_t = (uint32_t)n % (uint32_t)r.T;
    X* const to = dz + n * r.V;
    const Row<X> row(to, r.V);
    const int steps = (row.high + ((r.V + row.ahead) % 8 > 0) + 31) / 32;
    int64_t label = 0;
    const bool   counts = counted<L>(r, n, label);
    const float4 kept   = counts ? in.kept[n] : make_float4(0.f, -INFINITY, 0.f, 0.f);
    float g_top = 0.f;  // of this lane's alternative
    int   alternative = -1;
    if (counts && in.top && lane < r.top) {
        g_top = in.top[seq * in.top_b + at_t * in.top_t + lane * in.top_k];
        alternative = (int)static_cast<const L*>(in.top_label)[n * r.top + lane];
    }
    const float g = counts && in.log_prob ? in.log_prob[seq * in.log_prob_b + at_t * in.log_prob_t] : 0.f;
    const float h = counts && in.entropy ? in.entropy[seq * in.entropy_b + at_t * in.entropy_t] : 0.f;
    float total = g_top;
#pragma unroll
    for (int j = 16; j > 0; j >>= 1) total += __shfl_xor_sync(0xffffffffu, total, j);
    total += g;
    // a value's gradient is p (c0 + c1 log2 p)
    float c0 = -total - h * kept.z;
    const float c1 = -h * kLn2;
    if (counts && in.log_prob && (label < 0 || label >= r.V)) c0 = __uint_as_float(0x7fffffffu);
    if (kept.y == -INFINITY) {  // does not count, or no class is possible
        const float none = c0 != c0 ? c0 : 0.f;
        const float v[8] = {none, none, none, none, none, none, none, none};
        for (int step = member; step < steps; step += r.team) {
            const int at = row.first(step, lane);
            if (at >= 0 && at + 8 <= r.V) {
                store8(to + at, v);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (at + i >= 0 && at + i < r.V) put(to + at + i, none);
            }
        }
        return;
    }
    const X* const x = z + seq * r.stride_b + at_t * r.stride_t;
    // read by vectors where they are aligned in the logits as in the gradient
    const bool even = (reinterpret_cast<uintptr_t>(x) / sizeof(X)) % 8 == row.ahead;
    Row<X> from(x, r.V);
    from.ahead = row.ahead, from.low = row.low, from.high = row.high;
    const float2 off = make_float2(-kept.x, -kept.x), scale = make_float2(kLog2e, kLog2e), log2_s = make_float2(-kept.y, -kept.y);
    const float2 c0s = make_float2(c0, c0), c1s = make_float2(c1, c1);
    auto gradients = [&](float2 v) {
        float2 l = fma2(add2(v, off), scale, log2_s);  // log2 p
        l = make_float2(max_nan(l.x, kNever), max_nan(l.y, kNever));
        return mul2(make_float2(exp2_approx(l.x), exp2_approx(l.y)), fma2(c1s, l, c0s));
    };
    auto gradient = [&](float v) { return gradients(make_float2(v, v)).x; };
    constexpr int A = kAhead<X>;
    Raw<X> v[A];
    const int hop = r.team * A;
    if (member < steps) from.load(member, r.team, lane, v, even);
    for (int step = member; step < steps; step += hop) {
        const bool inside = row.inside(step, r.team);
#pragma unroll
        for (int i = 0; i < A; ++i) {
            float out[8];
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float2 g2 = gradients(make_float2(v[i].get(j), v[i].get(j + 1)));
                out[j] = g2.x, out[j + 1] = g2.y;
            }
            const int at = row.first(step + i * r.team, lane);
            if (inside || (at >= 0 && at + 8 <= r.V)) {
                store8(to + at, out);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (at + j >= 0 && at + j < r.V) put(to + at + j, out[j]);
            }
        }
        if (step + hop < steps) from.load(step + hop, r.team, lane, v, even);
    }
    // The label and the alternatives: by the warp that wrote their places.
    __syncwarp();
    auto mine = [&](int index) { return (index + row.ahead) / 256 % r.team == member; };
    const bool listed = __any_sync(0xffffffffu, alternative >= 0 && alternative == label);
    if (alternative >= 0 && mine(alternative)) put(to + alternative, gradient(value(x[alternative])) + g_top + (alternative == label ? g : 0.f));
    if (lane == 0 && !listed && label >= 0 && label < r.V && mine((int)label)) put(to + label, gradient(value(x[label])) + g);
}

// Warps per row: enough for `busy` on each SM, a step each at least.  Forward 8 of them, and more than a CTA's only where each has
// 1024 logits: what is joined costs more than further warps bring.  (us without and with 8 alternatives, f32: 256 x 10025 5.0 and
// 10.7, with 16 busy warps 6.2 and 18; 8 x 10025 3.8 and 8.5, with a team of 64 4.2 and 15; 16 x 100000 with a team of 8 11.4 and
// 16.5, of 64 5.5 and 12.9.)  The gradient, where nothing is joined: 16.
int team_of(int64_t N, int64_t V, int most, int busy) {
    const int64_t want = (int64_t)sm_count() * busy;
    int team = 1;
    while (2 * team <= most && N * team < want && team * 256 < V) team *= 2;
    return team;
}

bool sizes_ok(const framewise_b200_scores_shape* s) {
    const int64_t kMost = (int64_t)1 << 31;
    return s && s->B >= 0 && s->T >= 0 && s->V >= 1 && s->B < kMost && s->T < kMost && s->B * s->T < kMost && s->V < kMost / 16 && s->top >= 0 &&
           s->top <= kMostTop && s->top <= s->V && (s->dtype == FRAMEWISE_B200_F32 || s->dtype == FRAMEWISE_B200_BF16);
}

Rows rows_of(const framewise_b200_scores_shape& s, const void* labels, const int32_t* lens, int most_team, int busy) {
    Rows r = {};
    r.N = s.B * s.T, r.T = (int)s.T, r.V = (int)s.V, r.top = s.top, r.team = team_of(r.N, s.V, most_team, busy);
    r.stride_b = s.logits_stride_b, r.stride_t = s.logits_stride_t;
    r.labels = labels, r.lens = lens, r.ignore = s.ignore_index;
    return r;
}

template <typename X, typename L, bool TOP>
int forward(const Rows& r, const X* z, const Scored& out, cudaStream_t stream) {
    const int ctas = r.team > kWarps ? r.team / kWarps : 1;
    const int64_t grid = ctas > 1 ? r.N * ctas : (r.N + kWarps / r.team - 1) / (kWarps / r.team);
    cudaLaunchConfig_t c = {};
    c.gridDim  = dim3((unsigned)grid);
    c.blockDim = dim3(kWarps * 32);
    c.stream   = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ctas, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    c.attrs    = at;
    c.numAttrs = ctas > 1 ? 1 : 0;
    FW_TRY(cudaLaunchKernelEx(&c, k_label_scores<X, L, TOP>, z, r, out));
    FW_LAUNCHED();
    return FRAMEWISE_B200_OK;
}

}  // namespace

extern "C" {

int framewise_b200_scores_forward(const framewise_b200_scores_shape* shape, const void* logits, const void* labels, const int32_t* seq_lens,
                                  float* log_probs, float* entropy, float* top_log_probs, void* top_labels, void* kept,
                                  framewise_b200_stream_t stream) {
    if (!sizes_ok(shape)) return FRAMEWISE_B200_BAD_ARGUMENT;
    if (shape->B * shape->T == 0) return FRAMEWISE_B200_OK;
    if (!logits || !labels || !log_probs || !entropy || (shape->top > 0 && (!top_log_probs || !top_labels)) || reinterpret_cast<uintptr_t>(kept) % 16 != 0)
        return FRAMEWISE_B200_BAD_ARGUMENT;
    const Rows   r   = rows_of(*shape, labels, seq_lens, (int)std::clamp<int64_t>(shape->V / 1024, kWarps, kMostTeam), 8);
    const Scored out = {log_probs, entropy, top_log_probs, top_labels, static_cast<float4*>(kept)};
    auto go = [&](auto x, auto l) {
        using X = decltype(x);
        using L = decltype(l);
        return shape->top > 0 ? forward<X, L, true>(r, (const X*)logits, out, stream) : forward<X, L, false>(r, (const X*)logits, out, stream);
    };
    if (shape->dtype == FRAMEWISE_B200_F32) return shape->labels64 ? go(float(), int64_t()) : go(float(), int32_t());
    return shape->labels64 ? go(__nv_bfloat16(), int64_t()) : go(__nv_bfloat16(), int32_t());
}

int framewise_b200_scores_backward(const framewise_b200_scores_shape* shape, const void* logits, const void* labels, const int32_t* seq_lens,
                                   const void* top_labels, const void* kept, const framewise_b200_scores_grads* grads, void* grad_logits,
                                   framewise_b200_stream_t stream) {
    if (!sizes_ok(shape)) return FRAMEWISE_B200_BAD_ARGUMENT;
    if (shape->B * shape->T == 0) return FRAMEWISE_B200_OK;
    if (!logits || !labels || !kept || !grads || !grad_logits || reinterpret_cast<uintptr_t>(kept) % 16 != 0 ||
        (grads->top_log_probs && shape->top > 0 && !top_labels))
        return FRAMEWISE_B200_BAD_ARGUMENT;
    const Rows r = rows_of(*shape, labels, seq_lens, 1 << 16, 16);
    Incoming   in = {};
    in.log_prob = grads->log_probs, in.log_prob_b = grads->log_probs_stride_b, in.log_prob_t = grads->log_probs_stride_t;
    in.entropy = grads->entropy, in.entropy_b = grads->entropy_stride_b, in.entropy_t = grads->entropy_stride_t;
    in.top = shape->top > 0 ? grads->top_log_probs : nullptr, in.top_b = grads->top_stride_b, in.top_t = grads->top_stride_t, in.top_k = grads->top_stride_k;
    in.top_label = top_labels, in.kept = static_cast<const float4*>(kept);
    const unsigned grid = (unsigned)((r.N * r.team + kWarps - 1) / kWarps);
    auto go = [&](auto x, auto l) -> int {
        using X = decltype(x);
        using L = decltype(l);
        k_label_scores_back<X, L><<<grid, kWarps * 32, 0, stream>>>((const X*)logits, r, in, (X*)grad_logits);
        FW_LAUNCHED();
        return FRAMEWISE_B200_OK;
    };
    if (shape->dtype == FRAMEWISE_B200_F32) return shape->labels64 ? go(float(), int64_t()) : go(float(), int32_t());
    return shape->labels64 ? go(__nv_bfloat16(), int64_t()) : go(__nv_bfloat16(), int32_t());
}

}  // extern "C"
