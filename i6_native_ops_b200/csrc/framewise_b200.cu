// framewise_b200.cu -- the operators of framewise training behind the C ABI of include/framewise_b200.h: output layer
// with softmax cross entropy (linear_ce_b200.inc), label embedding (embedding_b200.inc), AdamW (adamw_b200.inc).
// This file holds their host side: sizes, launch shapes, tensor maps.
#include "framewise_b200.h"
#include "framewise_host.h"
#include "tensor_core.h"

#include <cuda_runtime.h>
#include <math_constants.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <type_traits>

namespace {

using namespace framewise_host;

#include "embedding_b200.inc"
#include "adamw_b200.inc"
#include "linear_ce_b200.inc"

// ------------------------------------------------------------------------------------------ cross entropy

// What a call keeps and uses, from its sizes alone.
struct CePlan {
    int64_t N, V, D;
    int     pair;                    // CTAs per tile
    int     parts, q_parts;          // planes of X and the weight, of q
    int     pitch, chunks, chunk;
    bool    copy_weight;
    int     wide_v, wide_d;          // columns of the tiles over V and over D
    int     row_chunks;                  // chunks of rows
    int     q_blocks;                // columns of q in blocks of 64
    int64_t out_pitch;
    // saved
    int32_t*       head;
    int*           chunk_count;
    int*           row_label;
    int*           row_position;
    uint8_t*       counted;  // per position
    float*         bias;
    float2*        stats;
    __nv_bfloat16* rows;
    __nv_bfloat16* weight;
    size_t         saved_bytes;
    // forward
    float2* part;
    float*  target;
    size_t  forward_bytes;
    // backward
    __nv_bfloat16* q;
    float*         pieces;        // of the two products' shared tiles
    int64_t        piece_values;  // of each
    float*         acc;       // the weight's gradient in 32 bits, where it takes several chunks
    float*         col_part;
    float*         bias_acc;  // the bias's, likewise
    size_t         backward_bytes;
};

// q of a chunk takes this much at most: some hundred rows of the largest vocabularies, all rows of small batches.
constexpr int64_t kChunkBytes = (int64_t)768 << 20;
// Up to this many rows a tile is one CTA's, a pair's above.  Device time of loss and gradients, one CTA / pairs:
// 200 x 10025 x 512 79 / 82 us, 600 x 5000 x 512 85 / 88, 1000 x 12001 x 512 117 / 118, 2000 x 5000 x 512 (f32) 285 / 267,
// 4000 x 12001 x 512 246 / 235.
constexpr int64_t kOneCta = 1024;

// Up to this many positions each CTA of k_prepare counts those before its own by itself; above, a launch before does (us
// by itself / with that launch: 4000 positions 7.4 / 11.5, 8000 11.7 / 12.5, 16000 16.8 / 12.5).
constexpr int64_t kCountHere = 4096;
// bf16: up to this many rows q is held in two parts, 16 bits: with few rows the gradients' error would be up to 1.8 times
// that of their own rounding (1.4 times with many), and a product more each costs little beside launches (200 x 10025 x
// 512: 69 us, 62 with one part).  With many rows it would be most of a step: 20700 x 12001 x 500 1689 us instead of 1053.
constexpr int64_t kTwoParts = 256;

int ce_plan(const framewise_b200_ce_shape* sh, void* saved, void* forward, void* backward, CePlan* p) {
    if (!sh) return FRAMEWISE_B200_BAD_ARGUMENT;
    const int64_t kMost = (int64_t)1 << 31;
    if (sh->B < 0 || sh->T < 0 || sh->V < 1 || sh->D < 1 || sh->B >= kMost || sh->T >= kMost || sh->V >= kMost - 256 ||
        sh->D >= kMost - 256 || sh->B * sh->T >= kMost - 256)
        return FRAMEWISE_B200_BAD_ARGUMENT;
    if (sh->dtype != FRAMEWISE_B200_F32 && sh->dtype != FRAMEWISE_B200_BF16) return FRAMEWISE_B200_BAD_ARGUMENT;
    p->N = sh->B * sh->T, p->V = sh->V, p->D = sh->D;
    p->pair = p->N > kOneCta ? 2 : 1;
    const int kPair = p->pair, workers = sm_count() / kPair;
    if (workers < 1) return FRAMEWISE_B200_CUDA_ERROR;
    p->parts       = sh->dtype == FRAMEWISE_B200_F32 ? 3 : 1;
    p->q_parts     = p->parts == 1 && p->N <= kTwoParts ? 2 : p->parts;
    p->copy_weight = p->parts == 3 || sh->copy_weight != 0;
    p->pitch       = (int)up(sh->D, 64);  // rows of whole lines of 128 bytes: copies of 128 would touch two lines each
    p->chunks      = (int)((p->N + ce::kCountChunk - 1) / ce::kCountChunk);
    const int     tile   = ce::kRowsPerCta * kPair;
    const int64_t rows   = up(std::max<int64_t>(p->N, 1), 256);
    const int64_t mt     = rows / tile;
    // narrower tiles where wide ones would leave SMs idle
    p->wide_v = 256;
    while (p->wide_v > 64 * kPair && (p->wide_v / 2 >= p->V || mt * ((p->V + p->wide_v - 1) / p->wide_v) < workers)) p->wide_v /= 2;
    p->wide_d  = (int)std::min<int64_t>(256, up(p->D, 64 * kPair));
    p->q_blocks = (int)((p->V + 63) / 64);
    p->chunk   = (int)std::min(rows, std::max<int64_t>(256, kChunkBytes / (128 * (int64_t)p->q_parts * p->q_blocks) / 256 * 256));
    p->out_pitch = up(p->D, 4);
    // tiles, and stages of the tiles that are shared out, are counted in 32 bits
    const int64_t depth = std::max(p->V, (int64_t)p->chunk) / ce::kDepth + 1;
    if (mt * ((p->V + p->wide_v - 1) / p->wide_v) >= kMost / 2 || depth * workers >= kMost / 2 ||
        (std::max(p->V, rows) / tile + 1) * ((p->D + p->wide_d - 1) / p->wide_d) >= kMost / 2)
        return FRAMEWISE_B200_BAD_ARGUMENT;
    p->row_chunks = (int)((rows + p->chunk - 1) / p->chunk);

    Parts s(saved);
    p->head         = s.take<int32_t>(64);
    p->chunk_count  = s.take<int>(p->chunks);
    p->row_label    = s.take<int>(rows);
    p->row_position = s.take<int>(rows);
    p->counted      = s.take<uint8_t>(sh->train ? p->N : 0);
    p->bias         = s.take<float>(up(p->V, 256));
    p->stats        = s.take<float2>(sh->train ? rows : 0);
    p->rows         = s.take<__nv_bfloat16>(p->parts * rows * p->pitch);
    p->weight       = s.take<__nv_bfloat16>(p->copy_weight ? p->parts * p->V * p->pitch : 0);
    p->saved_bytes  = s.used;
    Parts f(forward);
    p->part   = f.take<float2>((workers + mt) * ce::Layout<ce::kLogits, 1, 1, false>::kGroups * tile);
    p->target = f.take<float>(rows);
    p->forward_bytes = f.used;
    Parts b(backward);
    p->q           = b.take<__nv_bfloat16>((int64_t)p->q_parts * p->q_blocks * 64 * p->chunk);
    p->piece_values = (int64_t)2 * workers * tile * ce::kWide;
    p->pieces   = b.take<float>(2 * p->piece_values);
    p->acc      = b.take<float>(p->row_chunks > 1 ? p->V * p->out_pitch : 0);
    p->col_part = b.take<float>(sh->has_bias ? (int64_t)p->chunk / 32 * up(p->V, 64) : 0);
    p->bias_acc = b.take<float>(sh->has_bias ? p->V : 0);
    p->backward_bytes = b.used;
    return FRAMEWISE_B200_OK;
}

template <int KIND, int kPair, int PARTS, bool LONG = false>
int launch_tiles(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& out, const ce::Params& p, int workers, cudaStream_t stream) {
    using L = ce::Layout<KIND, kPair, PARTS, LONG>;
    auto kernel = ce::k_ce_tiles<KIND, kPair, PARTS, LONG>;
    static std::atomic<uint64_t> allowed{0};
    FW_DO(allow_shared(kernel, L::kBytes, allowed));
    cudaLaunchConfig_t c = {};
    c.gridDim          = dim3(workers * kPair);
    c.blockDim         = dim3(L::kThreads);
    c.dynamicSmemBytes = L::kBytes;
    c.stream           = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = kPair, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    c.attrs    = at;
    c.numAttrs = kPair > 1 ? 1 : 0;
    FW_TRY(cudaLaunchKernelEx(&c, kernel, a, b, out, p));
    FW_LAUNCHED();
    return FRAMEWISE_B200_OK;
}

template <int kPair, typename X, typename L>
int ce_forward(const framewise_b200_ce_shape& sh, const CePlan& p, const X* hidden, const X* weight, const X* bias, const L* targets,
               const int32_t* lens, float* loss, cudaStream_t stream) {
    constexpr int PARTS = sizeof(X) == 4 ? 3 : 1;
    const int workers = sm_count() / kPair, tile = ce::kRowsPerCta * kPair;
    const int64_t rows = up(p.N, 256);
    FW_DO(bind_device());
    const bool count = p.N > kCountHere;
    if (count) {
        ce::k_count_rows<L><<<p.chunks, 256, 0, stream>>>(p.N, (int)sh.T, targets, lens, sh.ignore_index, p.chunk_count);
        FW_LAUNCHED();
    }
    const int     per_cta = p.N > 64 * 128 ? ce::kGatherRows : ce::kGatherFew;
    const int64_t gather = (p.N + per_cta - 1) / per_cta, biases = up(p.V, 256) / 256, splits = p.copy_weight ? (p.V + 7) / 8 : 0;
    ce::k_prepare<X, L, PARTS><<<(unsigned)(gather + biases + splits), 256, 0, stream>>>(
        p.N, (int)sh.T, hidden, sh.hidden_stride_b, sh.hidden_stride_t, targets, lens, sh.ignore_index, count ? p.chunk_count : nullptr, p.head, (int)p.V,
        (int)p.D, p.pitch, p.rows, rows * p.pitch, p.row_label, p.row_position, sh.train ? p.counted : nullptr, loss, bias, p.bias, weight,
        p.weight, per_cta, (int)gather, (int)biases);
    FW_LAUNCHED();
    const void*   w       = p.copy_weight ? (const void*)p.weight : (const void*)weight;
    const int64_t w_pitch = p.copy_weight ? p.pitch : p.D;
    CUtensorMap a, b;
    if (!map_of(&a, p.rows, false, p.D, rows, PARTS, p.pitch, rows * p.pitch, 64, ce::kRowsPerCta) ||
        !map_of(&b, w, false, p.D, p.V, PARTS, w_pitch, p.V * w_pitch, 64, p.wide_v / kPair))
        return FRAMEWISE_B200_TENSOR_MAP;
    ce::Params q = {};
    q.head = p.head, q.V = (int)p.V, q.D = (int)p.D, q.wide = p.wide_v;
    q.bias = p.bias, q.label = p.row_label, q.part = p.part, q.target = p.target;
    FW_DO((p.D > ce::kLong ? launch_tiles<ce::kLogits, kPair, PARTS, true> : launch_tiles<ce::kLogits, kPair, PARTS>)(a, b, a, q, workers, stream));
    const int nt = (int)((p.V + p.wide_v - 1) / p.wide_v);
    auto join = [&](auto* kernel, int64_t lanes) {
        kernel<<<(unsigned)((p.N * lanes + 255) / 256), 256, 0, stream>>>(p.head, nt, tile, workers, p.part, p.target, p.row_label, p.row_position,
                                                                       loss, sh.train ? p.stats : nullptr);
    };
    constexpr int kGroups = ce::Layout<ce::kLogits, kPair, PARTS, false>::kGroups, kLongGroups = ce::Layout<ce::kLogits, kPair, PARTS, true>::kGroups;
    if (p.N > 4096) p.D > ce::kLong ? join(ce::k_join_rows<4, kLongGroups>, 4) : join(ce::k_join_rows<4, kGroups>, 4);
    else p.D > ce::kLong ? join(ce::k_join_rows<32, kLongGroups>, 32) : join(ce::k_join_rows<32, kGroups>, 32);
    FW_LAUNCHED();
    return FRAMEWISE_B200_OK;
}

template <int kPair, int Q_PARTS, typename X>
int ce_backward(const framewise_b200_ce_shape& sh, const CePlan& p, const X* weight, const float* grad, int64_t grad_b, int64_t grad_t,
                X* grad_hidden, X* grad_weight, X* grad_bias, cudaStream_t stream) {
    constexpr int PARTS = sizeof(X) == 4 ? 3 : 1;
    const int workers = sm_count() / kPair;
    const int64_t rows = up(p.N, 256);
    const void*   w       = p.copy_weight ? (const void*)p.weight : (const void*)weight;
    const int64_t w_pitch = p.copy_weight ? p.pitch : p.D, V = p.V, D = p.D;
    FW_DO(bind_device());
    const bool several = p.row_chunks > 1;
    CUtensorMap x_k, w_k, q_out, q_k, w_mn, q_mn, x_mn, w_out;
    if (!map_of(&x_k, p.rows, false, D, rows, PARTS, p.pitch, rows * p.pitch, 64, ce::kRowsPerCta) ||
        !map_of(&w_k, w, false, D, V, PARTS, w_pitch, V * w_pitch, 64, p.wide_v / kPair) ||
        !map_of(&q_out, p.q, false, 64, p.chunk, Q_PARTS * p.q_blocks, 64, (int64_t)p.chunk * 64, 32, 32) ||
        !map_of(&q_k, p.q, false, 64, p.chunk, Q_PARTS * p.q_blocks, 64, (int64_t)p.chunk * 64, 64, ce::kRowsPerCta) ||
        !map_of(&q_mn, p.q, false, 64, p.chunk, Q_PARTS * p.q_blocks, 64, (int64_t)p.chunk * 64, 64, 64) ||
        !map_of(&w_mn, w, false, D, V, PARTS, w_pitch, V * w_pitch, 64, 64) ||
        !map_of(&x_mn, p.rows, false, D, rows, PARTS, p.pitch, rows * p.pitch, 64, 64) ||
        (several && !map_of(&w_out, p.acc, true, D, V, 1, p.out_pitch, V * p.out_pitch, 32, 32)))
        return FRAMEWISE_B200_TENSOR_MAP;
    if (!several) w_out = x_mn;  // not used
    ce::Params g = {};
    g.head = p.head, g.V = (int)V, g.D = (int)D, g.chunk = p.chunk;
    g.bias = p.bias, g.label = p.row_label, g.position = p.row_position, g.stats = p.stats;
    g.grad = grad, g.grad_b = grad_b, g.grad_t = grad_t, g.T = (int)sh.T;
    g.q = p.q, g.q_blocks = p.q_blocks, g.col_part = grad_bias ? p.col_part : nullptr, g.col_pitch = (int)up(V, 64);
    auto grain = [&](const X* out) {  // at least a value's size
        const uintptr_t odd = (uintptr_t)(D * sizeof(X)) | reinterpret_cast<uintptr_t>(out) | 16;
        return (int)(odd & (~odd + 1));
    };
    for (int c = 0; c < p.row_chunks; ++c) {
        ce::After after = {};
        g.row0 = c * p.chunk, g.add = c > 0;
        g.wide = p.wide_v;
        FW_DO((D > ce::kLong ? launch_tiles<ce::kGradients, kPair, Q_PARTS, true> : launch_tiles<ce::kGradients, kPair, Q_PARTS>)(x_k, w_k, q_out, g,
                                                                                                                           workers, stream));
        g.wide = p.wide_d;
        if (grad_hidden) {
            g.out = grad_hidden, g.out_grain = grain(grad_hidden), g.pieces = p.pieces;
            FW_DO(launch_tiles<ce::kToHidden, kPair, Q_PARTS>(q_k, w_mn, w_mn, g, workers, stream));
            after.with_hidden = true;
        }
        after.hidden = g;
        if (grad_weight) {
            g.out = several ? nullptr : grad_weight, g.out_grain = grain(grad_weight), g.pieces = p.pieces + p.piece_values;
            FW_DO(launch_tiles<ce::kToWeight, kPair, Q_PARTS>(q_mn, x_mn, w_out, g, workers, stream));
            after.with_weight = true;
        }
        after.weight = g;
        after.last = c + 1 == p.row_chunks, after.with_bias = grad_bias != nullptr;
        after.workers = workers, after.acc = several ? p.acc : nullptr, after.acc_pitch = (int)p.out_pitch, after.bias_acc = p.bias_acc;
        after.N = p.N, after.counted = p.counted;
        ce::k_after<kPair, X><<<sm_count() * 8, 256, 0, stream>>>(after, grad_hidden, grad_weight, grad_bias);
        FW_LAUNCHED();
    }
    if (grad_weight && several) {
        ce::k_weight_out<X><<<(unsigned)((V * p.out_pitch / 4 + 255) / 256), 256, 0, stream>>>(p.head, p.acc, (int)V, (int)D, (int)p.out_pitch, grad_weight);
        FW_LAUNCHED();
    }
    return FRAMEWISE_B200_OK;
}

// ------------------------------------------------------------------------------------------ embedding

struct EmbedPlan {
    int64_t   N;
    int       chunks, passes, shift, digits[2];
    uint32_t *keys[2], *places[2];
    int32_t * counts, *before, *total, *all;
    float*    edge;
    size_t    bytes;
};

bool embed_sizes_ok(int64_t B, int64_t T, int64_t V, int64_t D) {
    const int64_t kMost = (int64_t)1 << 31;
    return B >= 0 && T >= 0 && B < kMost && T < kMost && B * T < kMost - 1024 && V >= 1 && V < ((int64_t)1 << 28) && D >= 1 && D < kMost - 256;
}

EmbedPlan embed_plan(int64_t B, int64_t T, int64_t V, int64_t D, void* work) {
    EmbedPlan p;
    p.N         = B * T;
    p.chunks    = (int)((p.N + embed::kChunk - 1) / embed::kChunk);
    // Keys up to V (labels outside the vocabulary).  One pass where a chunk's counters fit shared memory and all chunks'
    // take some ten megabytes at most; else two of half the bits.
    int bits = 1;
    while (V >> bits) ++bits;
    p.passes    = V + 1 > embed::kDigits || p.chunks > embed::kOnePassChunks ? 2 : 1;
    p.shift     = p.passes == 1 ? bits : (bits + 1) / 2;
    p.digits[0] = p.passes == 1 ? (int)(V + 1) : 1 << p.shift;
    p.digits[1] = (int)(V >> p.shift) + 1;
    const int digits = std::max(p.digits[0], p.passes == 2 ? p.digits[1] : 0);
    Parts b(work);
    for (int i = 0; i < 2; ++i) {
        p.keys[i]   = b.take<uint32_t>(i < p.passes ? p.N : 0);
        p.places[i] = b.take<uint32_t>(i < p.passes ? p.N : 0);
    }
    p.counts = b.take<int32_t>((int64_t)p.chunks * digits);
    p.before = b.take<int32_t>(digits);
    p.total  = b.take<int32_t>(digits / embed::kScanRow + 1);
    p.all    = b.take<int32_t>(1);
    p.edge   = b.take<float>((p.N + embed::kPiece - 1) / embed::kPiece * 2 * D);
    p.bytes  = b.used;
    return p;
}

template <typename S>
int sort_pass(const S& src, const EmbedPlan& p, int pass, void* zero, int64_t zero_bytes, cudaStream_t stream) {
    const int digits = p.digits[pass], shift = p.shift * pass, scans = (digits + embed::kScanRow - 1) / embed::kScanRow;
    const uint32_t mask = p.passes == 2 && pass == 0 ? (1u << p.shift) - 1 : 0xffffffffu;
    const size_t bytes = (size_t)digits * 4;
    if (bytes > 24 * 1024) {  // with the static arrays, more than a kernel gets without asking
        static std::atomic<uint64_t> count{0}, place{0};
        FW_DO(allow_shared(embed::k_sort_count<S>, embed::kDigits * 4, count));
        FW_DO(allow_shared(embed::k_sort_place<S>, embed::kDigits * 4, place));
    }
    const int grid = (int)std::max<int64_t>(p.chunks, std::min<int64_t>(zero ? zero_bytes / 16384 : 0, 1024));
    embed::k_sort_count<S><<<grid, 256, bytes, stream>>>(src, shift, mask, digits, p.chunks, p.counts, static_cast<char*>(zero), zero_bytes);
    FW_LAUNCHED();
    embed::k_sort_scan<<<scans, 256, 0, stream>>>(p.counts, p.chunks, digits, p.before, p.total);
    FW_LAUNCHED();
    embed::k_sort_place<S><<<p.chunks, 256, bytes, stream>>>(src, shift, mask, digits, p.counts, p.before, p.total, scans, p.keys[pass], p.places[pass], p.all);
    FW_LAUNCHED();
    return FRAMEWISE_B200_OK;
}

template <typename X, typename L>
int embed_forward(int64_t N, int64_t T, int64_t V, int64_t D, int64_t ignore, float scale, const X* table, const L* labels,
                  const int32_t* lens, X* out, cudaStream_t stream) {
    const bool wide = D % 8 == 0 && (reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(out)) % (8 * sizeof(X)) == 0;
    const unsigned grid = (unsigned)((N + 8 * embed::kRows - 1) / (8 * embed::kRows));
    if (wide)
        embed::k_embed<X, L, true><<<grid, 256, 0, stream>>>(N, (int)T, V, (int)D, table, labels, lens, ignore, scale, out);
    else
        embed::k_embed<X, L, false><<<grid, 256, 0, stream>>>(N, (int)T, V, (int)D, table, labels, lens, ignore, scale, out);
    FW_LAUNCHED();
    return FRAMEWISE_B200_OK;
}

template <typename X, typename L>
int embed_backward(const EmbedPlan& p, int64_t T, int64_t V, int64_t D, int64_t ignore, float scale, const X* grad, int64_t grad_b,
                   int64_t grad_t, const L* labels, const int32_t* lens, X* out, cudaStream_t stream) {
    if (reinterpret_cast<uintptr_t>(out) % 16 != 0) return FRAMEWISE_B200_BAD_ARGUMENT;
    FW_DO(sort_pass(embed::FromLabels<L>{labels, lens, p.N, ignore, V, (int)T}, p, 0, out, V * D * (int64_t)sizeof(X), stream));
    if (p.passes == 2) FW_DO(sort_pass(embed::FromKeys{p.keys[0], p.places[0], p.all}, p, 1, nullptr, 0, stream));
    const uint32_t *keys = p.keys[p.passes - 1], *places = p.places[p.passes - 1];
    const int     slices = (int)((D + embed::kSlice - 1) / embed::kSlice);
    const int64_t jobs   = (p.N + embed::kPiece - 1) / embed::kPiece * slices;
    const int64_t lanes  = 16 / (int64_t)sizeof(X);
    const bool wide = D % 8 == 0 && grad_b % lanes == 0 && grad_t % lanes == 0 && (reinterpret_cast<uintptr_t>(grad) & 15) == 0;
    if ((jobs + 7) / 8 >= (int64_t)1 << 31) return FRAMEWISE_B200_BAD_ARGUMENT;
    if (wide)
        embed::k_embed_pieces<X, true><<<(unsigned)((jobs + 7) / 8), 256, 0, stream>>>(p.all, V, (int)D, slices, (int)T, grad, grad_b, grad_t, keys, places, scale, p.edge, out);
    else
        embed::k_embed_pieces<X, false><<<(unsigned)((jobs + 7) / 8), 256, 0, stream>>>(p.all, V, (int)D, slices, (int)T, grad, grad_b, grad_t, keys, places, scale, p.edge, out);
    FW_LAUNCHED();
    const int64_t pieces = (p.N + embed::kPiece - 1) / embed::kPiece;
    embed::k_embed_runs<X><<<(unsigned)((pieces + 7) / 8), 256, 0, stream>>>(p.all, V, (int)D, keys, scale, p.edge, out);
    FW_LAUNCHED();
    return FRAMEWISE_B200_OK;
}

// ------------------------------------------------------------------------------------------ AdamW

// Calls `launch` for groups of up to kSlots tensors.
template <typename F>
int for_slots(const framewise_b200_tensor* tensors, int64_t count, bool codes, F&& launch) {
    int64_t i = 0;
    while (i < count) {
        adamw::Slots s;
        s.count = 0, s.blocks = 0;
        for (; i < count && s.count < adamw::kSlots; ++i) {
            const framewise_b200_tensor& t = tensors[i];
            if (t.n == 0) continue;
            adamw::Slot& o = s.slot[s.count++];
            o.param = t.param, o.grad = t.grad, o.master = t.master, o.m = t.exp_avg, o.v = t.exp_avg_sq;
            o.m_steps = t.exp_avg_steps, o.v_steps = t.exp_avg_sq_steps, o.n = t.n, o.first = s.blocks;
            const uintptr_t all = reinterpret_cast<uintptr_t>(t.param) | reinterpret_cast<uintptr_t>(t.grad) | reinterpret_cast<uintptr_t>(t.master);
            const uintptr_t held = reinterpret_cast<uintptr_t>(t.exp_avg) | reinterpret_cast<uintptr_t>(t.exp_avg_sq);
            o.wide = all % 32 == 0 && held % (codes ? 8 : 32) == 0 ? 2 : all % 16 == 0 && held % (codes ? 8 : 16) == 0 ? 1 : 0;
            s.blocks += (t.n + adamw::kBlock - 1) / adamw::kBlock;
        }
        if (s.count) FW_DO(launch(s));
    }
    return FRAMEWISE_B200_OK;
}

unsigned adamw_grid(int64_t blocks) { return (unsigned)std::min<int64_t>((blocks + 7) / 8, (int64_t)sm_count() * 64); }

int adamw_step(const framewise_b200_tensor* tensors, int64_t count, int32_t dtype, int32_t state_bits, double lr, double beta1,
                         double beta2, double eps, double weight_decay, int64_t step, bool follow, cudaStream_t stream) {
    if ((count > 0 && !tensors) || count < 0 || step < 1 || (state_bits != 8 && state_bits != 32) ||
        (dtype != FRAMEWISE_B200_F32 && dtype != FRAMEWISE_B200_BF16))
        return FRAMEWISE_B200_BAD_ARGUMENT;
    for (int64_t i = 0; i < count; ++i) {
        const framewise_b200_tensor& t = tensors[i];
        if (t.n < 0 || (t.n > 0 && (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq ||
                                    (state_bits == 8 && (!t.exp_avg_steps || !t.exp_avg_sq_steps)))))
            return FRAMEWISE_B200_BAD_ARGUMENT;
    }
    const adamw::Rates r = {(float)beta1, (float)(1 - beta1), (float)beta2, (float)(1 - beta2), (float)(1 - lr * weight_decay),
                            (float)(lr / (1 - std::pow(beta1, (double)step))), (float)(1 / std::sqrt(1 - std::pow(beta2, (double)step))), (float)eps,
                            (uint32_t)step * adamw::kTurn1, (uint32_t)step * adamw::kTurn2};
    const bool dither = state_bits == 8 && std::max(beta1, beta2) > adamw::kNearest;
    return for_slots(tensors, count, state_bits == 8, [&](const adamw::Slots& s) -> int {
        const unsigned grid = adamw_grid(s.blocks);
        auto go = [&](auto x, auto f) {
            using X = decltype(x);
            constexpr bool kFollow = decltype(f)::value;
            if (state_bits == 32) adamw::k_adamw<X, 32, false, kFollow><<<grid, 256, 0, stream>>>(s, r);
            else if (dither) adamw::k_adamw<X, 8, true, kFollow><<<grid, 256, 0, stream>>>(s, r);
            else adamw::k_adamw<X, 8, false, kFollow><<<grid, 256, 0, stream>>>(s, r);
        };
        if (dtype == FRAMEWISE_B200_F32) go(float(), std::false_type());  // a copy of one would be the same
        else if (follow) go(__nv_bfloat16(), std::true_type());
        else go(__nv_bfloat16(), std::false_type());
        FW_LAUNCHED();
        return FRAMEWISE_B200_OK;
    });
}

}  // namespace

extern "C" {

int64_t framewise_b200_launch_count(void) { return g_launches.load(); }

const char* framewise_b200_status_string(int status) {
    switch (status) {
        case FRAMEWISE_B200_OK: return "ok";
        case FRAMEWISE_B200_BAD_ARGUMENT: return "bad argument";
        case FRAMEWISE_B200_WORKSPACE: return "buffer too small";
        case FRAMEWISE_B200_CUDA_ERROR: return "CUDA error";
        case FRAMEWISE_B200_TENSOR_MAP: return "a tensor map could not be made";
        case FRAMEWISE_B200_OVERLAP: return "a tensor that is written is given twice, or overlaps another one or a gradient";
        default: return "unknown status";
    }
}

int framewise_b200_ce_bytes(const framewise_b200_ce_shape* shape, size_t* saved_bytes, size_t* forward_work_bytes,
                            size_t* backward_work_bytes) {
    CePlan p;
    if (!saved_bytes || !forward_work_bytes || !backward_work_bytes) return FRAMEWISE_B200_BAD_ARGUMENT;
    FW_DO(ce_plan(shape, nullptr, nullptr, nullptr, &p));
    *saved_bytes = p.saved_bytes, *forward_work_bytes = p.forward_bytes, *backward_work_bytes = p.backward_bytes;
    return FRAMEWISE_B200_OK;
}

int framewise_b200_ce_forward(const framewise_b200_ce_shape* shape, const void* hidden, const void* weight, const void* bias,
                              const void* targets, const int32_t* seq_lens, float* loss, void* saved, size_t saved_bytes, void* work,
                              size_t work_bytes, framewise_b200_stream_t stream) {
    CePlan p;
    FW_DO(ce_plan(shape, saved, work, nullptr, &p));
    if (p.N == 0) return FRAMEWISE_B200_OK;
    if (!hidden || !weight || !targets || !loss || !saved || !work || misaligned(saved) || misaligned(work) || (shape->has_bias && !bias))
        return FRAMEWISE_B200_BAD_ARGUMENT;
    if (!p.copy_weight && (reinterpret_cast<uintptr_t>(weight) % 16 != 0 || p.D % 8 != 0)) return FRAMEWISE_B200_BAD_ARGUMENT;
    if (saved_bytes < p.saved_bytes || work_bytes < p.forward_bytes) return FRAMEWISE_B200_WORKSPACE;
    if (!shape->has_bias) bias = nullptr;
    auto go = [&](auto x, auto l) {
        using X = decltype(x);
        using L = decltype(l);
        return (p.pair == 2 ? ce_forward<2, X, L> : ce_forward<1, X, L>)(*shape, p, (const X*)hidden, (const X*)weight, (const X*)bias,
                                                                       (const L*)targets, seq_lens, loss, stream);
    };
    if (shape->dtype == FRAMEWISE_B200_F32) return shape->labels64 ? go(float(), int64_t()) : go(float(), int32_t());
    return shape->labels64 ? go(__nv_bfloat16(), int64_t()) : go(__nv_bfloat16(), int32_t());
}

int framewise_b200_ce_backward(const framewise_b200_ce_shape* shape, const void* weight, const float* grad_loss, int64_t grad_stride_b,
                               int64_t grad_stride_t, void* grad_hidden, void* grad_weight, void* grad_bias, const void* saved,
                               size_t saved_bytes, void* work, size_t work_bytes, framewise_b200_stream_t stream) {
    CePlan p;
    FW_DO(ce_plan(shape, const_cast<void*>(saved), nullptr, work, &p));
    const size_t size = shape->dtype == FRAMEWISE_B200_F32 ? 4 : 2;
    if (p.N == 0) {
        if (grad_weight) FW_TRY(cudaMemsetAsync(grad_weight, 0, (size_t)p.V * p.D * size, stream));
        if (grad_bias) FW_TRY(cudaMemsetAsync(grad_bias, 0, (size_t)p.V * size, stream));
        return FRAMEWISE_B200_OK;
    }
    if (!shape->train || !weight || !grad_loss || !saved || !work || misaligned(saved) || misaligned(work) || (grad_bias && !shape->has_bias))
        return FRAMEWISE_B200_BAD_ARGUMENT;
    if (!p.copy_weight && (reinterpret_cast<uintptr_t>(weight) % 16 != 0 || p.D % 8 != 0)) return FRAMEWISE_B200_BAD_ARGUMENT;
    if (saved_bytes < p.saved_bytes || work_bytes < p.backward_bytes) return FRAMEWISE_B200_WORKSPACE;
    auto go = [&](auto x) {
        using X = decltype(x);
        constexpr int P = sizeof(X) == 4 ? 3 : 1, FEW = sizeof(X) == 4 ? 3 : 2;
        static_assert(kTwoParts <= kOneCta, "");
        auto run = p.pair == 2 ? ce_backward<2, P, X> : p.q_parts == FEW ? ce_backward<1, FEW, X> : ce_backward<1, P, X>;
        return run(*shape, p, (const X*)weight, grad_loss, grad_stride_b, grad_stride_t, (X*)grad_hidden, (X*)grad_weight, (X*)grad_bias, stream);
    };
    return shape->dtype == FRAMEWISE_B200_F32 ? go(float()) : go(__nv_bfloat16());
}

int framewise_b200_embed_forward(int64_t B, int64_t T, int64_t V, int64_t D, int32_t dtype, int32_t labels64, int64_t ignore_index,
                                 float scale, const void* table, const void* labels, const int32_t* seq_lens, void* out,
                                 framewise_b200_stream_t stream) {
    if (!embed_sizes_ok(B, T, V, D) || (dtype != FRAMEWISE_B200_F32 && dtype != FRAMEWISE_B200_BF16)) return FRAMEWISE_B200_BAD_ARGUMENT;
    if (B * T == 0) return FRAMEWISE_B200_OK;
    if (!table || !labels || !out) return FRAMEWISE_B200_BAD_ARGUMENT;
    auto go = [&](auto x, auto l) {
        using X = decltype(x);
        using L = decltype(l);
        return embed_forward<X, L>(B * T, T, V, D, ignore_index, scale, (const X*)table, (const L*)labels, seq_lens, (X*)out, stream);
    };
    if (dtype == FRAMEWISE_B200_F32) return labels64 ? go(float(), int64_t()) : go(float(), int32_t());
    return labels64 ? go(__nv_bfloat16(), int64_t()) : go(__nv_bfloat16(), int32_t());
}

size_t framewise_b200_embed_bytes(int64_t B, int64_t T, int64_t V, int64_t D) {
    return embed_sizes_ok(B, T, V, D) ? embed_plan(B, T, V, D, nullptr).bytes : 0;
}

int framewise_b200_embed_backward(int64_t B, int64_t T, int64_t V, int64_t D, int32_t dtype, int32_t labels64, int64_t ignore_index,
                                  float scale, const void* grad_out, int64_t grad_stride_b, int64_t grad_stride_t, const void* labels,
                                  const int32_t* seq_lens, void* grad_table, void* work, size_t work_bytes, framewise_b200_stream_t stream) {
    if (!embed_sizes_ok(B, T, V, D) || (dtype != FRAMEWISE_B200_F32 && dtype != FRAMEWISE_B200_BF16) || !grad_table)
        return FRAMEWISE_B200_BAD_ARGUMENT;
    if (B * T == 0) {
        FW_TRY(cudaMemsetAsync(grad_table, 0, (size_t)V * D * (dtype == FRAMEWISE_B200_F32 ? 4 : 2), stream));
        return FRAMEWISE_B200_OK;
    }
    if (!grad_out || !labels || !work || misaligned(work)) return FRAMEWISE_B200_BAD_ARGUMENT;
    const EmbedPlan p = embed_plan(B, T, V, D, work);
    if (work_bytes < p.bytes) return FRAMEWISE_B200_WORKSPACE;
    auto go = [&](auto x, auto l) {
        using X = decltype(x);
        using L = decltype(l);
        return embed_backward<X, L>(p, T, V, D, ignore_index, scale, (const X*)grad_out, grad_stride_b, grad_stride_t, (const L*)labels, seq_lens,
                                    (X*)grad_table, stream);
    };
    if (dtype == FRAMEWISE_B200_F32) return labels64 ? go(float(), int64_t()) : go(float(), int32_t());
    return labels64 ? go(__nv_bfloat16(), int64_t()) : go(__nv_bfloat16(), int32_t());
}

int framewise_b200_adamw(const framewise_b200_tensor* tensors, int64_t count, int32_t dtype, int32_t state_bits, double lr, double beta1,
                         double beta2, double eps, double weight_decay, int64_t step, framewise_b200_stream_t stream) {
    return adamw_step(tensors, count, dtype, state_bits, lr, beta1, beta2, eps, weight_decay, step, false, stream);
}

int framewise_b200_adamw_follow(const framewise_b200_tensor* tensors, int64_t count, int32_t dtype, int32_t state_bits, double lr,
                                double beta1, double beta2, double eps, double weight_decay, int64_t step,
                                framewise_b200_stream_t stream) {
    return adamw_step(tensors, count, dtype, state_bits, lr, beta1, beta2, eps, weight_decay, step, true, stream);
}

int framewise_b200_adamw_decode(const framewise_b200_tensor* tensors, int64_t count, framewise_b200_stream_t stream) {
    if ((count > 0 && !tensors) || count < 0) return FRAMEWISE_B200_BAD_ARGUMENT;
    for (int64_t i = 0; i < count; ++i) {
        const framewise_b200_tensor& t = tensors[i];
        if (t.n < 0 || (t.n > 0 && (!t.param || !t.master || !t.exp_avg || !t.exp_avg_sq || !t.exp_avg_steps || !t.exp_avg_sq_steps)))
            return FRAMEWISE_B200_BAD_ARGUMENT;
    }
    return for_slots(tensors, count, true, [&](const adamw::Slots& s) -> int {
        adamw::k_adamw_decode<<<adamw_grid(s.blocks), 256, 0, stream>>>(s);
        FW_LAUNCHED();
        return FRAMEWISE_B200_OK;
    });
}

}  // extern "C"
