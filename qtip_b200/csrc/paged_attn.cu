// Single-query attention over the key/value cache in 8 bits (paged.cuh): out = softmax(q K^T / sqrt(hd)) V for each sequence and head.
// Stands where the decode loop has the scaled_dot_product_attention of LlamaSdpaAttention.forward (model/llama.py:884-891 upstream).
//
// Bound by the bytes of the cache: 2 per token, key/value head and dim, read once for all query heads that share them.
// A pair is a sequence and a key/value head (of at most 16 query heads; more are further pairs).  Its tokens are cut into tiles of 32, and the
// tiles of all pairs, in order, are dealt to the CTAs in equal contiguous ranges, computed by every CTA from the lengths: a long sequence is
// spread over the chip, and a CTA goes through several short ones.  A cut that would leave less than kSnap + 1 tiles on one side is moved
// to the pair's border.  A pair inside one range is finished there; the parts of others go to the workspace, and a second kernel joins
// them in the order of the tokens.
// A warp takes every fourth tile of a range.  One of its lanes keeps kStages copies of tiles in flight (a tile of a block of 32 tokens or
// more is one piece of memory: K and V of 32 tokens); the lanes read the bytes in the order of the operands of the matrix instruction
// (16 rows: query heads; 16 in depth: dims, then tokens) and widen them to fp16, which holds every code.
#include <cuda_fp8.h>

#include "paged.cuh"

namespace qtip {
namespace {

constexpr int kAttnWarps = 4, kAttnThreads = 32 * kAttnWarps, kStages = 3, kTile = 32, kSnap = 4, kRowsMax = 16;
constexpr float kLift = 15.f;        // weights are 2^15 times exp(score - maximum): fp16 then reaches down to 2^-39 of the largest
constexpr unsigned kPolls = 1u << 20;
constexpr int kStatusWait = 64;

struct AttnArgs {
    __half *out;
    const __half *q;
    long out_stride, q_stride;
    const uint8_t *data;
    const float4 *scales;
    const __half *tail_k, *tail_v;
    long tail_k_stride, tail_v_stride;
    const int *tables, *lengths;
    int n_seqs, n_heads, n_kv, max_blocks, n_blocks, shift;      // block = 1 << shift
    float scale;                     // log2(e) / sqrt(hd)
    float *part_o;                   // (slot, row, hd): sums of a part, not divided
    float2 *part_ml;                 // (slot, row): maximum (in bits of the exponent), sum of weights
    int2 *meta;                      // pair: slot of its first part, number of parts (0: nothing to join)
    int groups, rows;                // groups of query heads per key/value head, the most heads in one
    unsigned *status;
};

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
    for (unsigned i = 0; i < kPolls; i++) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
    }
    return false;
}

__device__ __forceinline__ void bulk_copy(uint32_t to, const void *from, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from), "r"(bytes), "r"(bar) : "memory");
}

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four codes -> two pairs of fp16.  int8: 0x64xx is 1024 + xx, exact, so is the difference.
template <int KIND>
__device__ __forceinline__ void widen(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if constexpr (KIND == kKvInt8) {
        const uint32_t l = __byte_perm(w, 0x64646464u, 0x4140), h = __byte_perm(w, 0x64646464u, 0x4342), bias = 0x64806480u;
        const __half2 a = __hsub2(*reinterpret_cast<const __half2 *>(&l), *reinterpret_cast<const __half2 *>(&bias));
        const __half2 b = __hsub2(*reinterpret_cast<const __half2 *>(&h), *reinterpret_cast<const __half2 *>(&bias));
        lo = *reinterpret_cast<const uint32_t *>(&a);
        hi = *reinterpret_cast<const uint32_t *>(&b);
    } else {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
    }
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

struct Sequence {
    int full, tail;       // tokens in blocks, in the tail
    int coded, tiles;     // tiles of 8-bit tokens, all tiles
};
__device__ __forceinline__ Sequence sequence(const AttnArgs &a, int s, bool *bad = nullptr) {
    int len = a.lengths[s];
    if (len < 0 || len >> a.shift > a.max_blocks) {
        if (bad) *bad = true;
        len = 0;
    }
    Sequence q;
    q.full = len >> a.shift << a.shift;
    q.tail = len - q.full;
    q.coded = (q.full + kTile - 1) / kTile;
    q.tiles = q.coded + (q.tail + kTile - 1) / kTile;
    return q;
}

// A place in the list of all tiles.
struct Place {
    long long at;         // tiles before it
    int s, i, x;          // sequence, pair of it, tile of the pair
    int tiles;            // of the pair
};

// Walks over the pairs of a range.
struct Walk {
    int s, i, t, t_end, t_coded;      // current tile of this warp, end of the pair's part in the range, and of its 8-bit tiles
    long long left;                   // tiles of the range from the start of this pair's part
    Sequence q;
};

template <int HD, int KIND, bool R16>
__global__ void __launch_bounds__(kAttnThreads, 2) attn_paged_kernel(const AttnArgs a) {
    constexpr int kUnit = 32 * HD, kTileBytes = 2 * kUnit, NT = HD / 8, HALVES = HD / 64;
    constexpr int UP = R16 ? 2 : 1, E = 2 * UP, kJoin = 2 * NT + 4;              // rows of a lane; values of a lane in a tile of 8 columns
    extern __shared__ __align__(128) uint8_t attn_smem[];
    uint8_t *ring = attn_smem;                                                            // [warp][stage][kTileBytes]
    float4 *ring_scale = reinterpret_cast<float4 *>(attn_smem + kAttnWarps * kStages * kTileBytes);      // [warp][stage][2]
    float *join = reinterpret_cast<float *>(ring_scale + kAttnWarps * kStages * 2);       // [2][kJoin][32]
    __shared__ uint64_t bars[kAttnWarps][kStages];
    __shared__ long long s_tiles[kAttnWarps], s_seqs[kAttnWarps];
    __shared__ Place s_place[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3, sh = a.shift, b = 1 << sh;
    const int pairs = a.n_kv * a.groups;                                                  // of a sequence
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid < kAttnWarps * kStages) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&bars[0][0] + tid)));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // ---- this CTA's range of tiles
    const int per = (a.n_seqs + kAttnThreads - 1) / kAttnThreads, s_lo = min(tid * per, a.n_seqs), s_hi = min(s_lo + per, a.n_seqs);
    long long mine = 0, filled = 0;
    bool bad = false;
    for (int s = s_lo; s < s_hi; s++) {
        const int tiles = sequence(a, s, &bad).tiles;
        mine += tiles;
        filled += tiles > 0;
    }
    if (bad && a.status && blockIdx.x == 0) atomicOr(a.status, 1u);
    long long upto = mine, seqs = filled;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(kFullMask, upto, o), v = __shfl_up_sync(kFullMask, seqs, o);
        if (lane >= o) { upto += u; seqs += v; }
    }
    if (lane == 31) { s_tiles[warp] = upto; s_seqs[warp] = seqs; }
    __syncthreads();
    long long total = 0;
    seqs = 0;
#pragma unroll
    for (int w = 0; w < kAttnWarps; w++) {
        if (w < warp) upto += s_tiles[w];
        total += s_tiles[w];
        seqs += s_seqs[w];
    }
    total *= pairs;
    // at least four tiles each, one per warp, or one pair
    const long long want = max(total / kAttnWarps, seqs * pairs), ctas = max(min((long long)gridDim.x, min(want, total)), 1ll);
    const bool works = blockIdx.x < ctas && total > 0;
    if (works) {
        for (int k = 0; k < 2; k++) {
            long long at = (blockIdx.x + k) * total / ctas;
            if (at >= total) {
                if (tid == 0) s_place[k] = {total, a.n_seqs, 0, 0, 0};
            } else if ((upto - mine) * pairs <= at && at < upto * pairs) {
                long long before = (upto - mine) * pairs;
                for (int s = s_lo; s < s_hi; s++) {
                    const int tiles = sequence(a, s).tiles;
                    if (at < before + (long long)tiles * pairs) {
                        int i = (int)((at - before) / tiles), x = (int)((at - before) % tiles);
                        if (x <= kSnap) { at -= x; x = 0; }
                        else if (tiles - x <= kSnap) { at += tiles - x; x = 0; i++; }
                        s_place[k] = {at, s, i, x, tiles};
                        break;
                    }
                    before += (long long)tiles * pairs;
                }
            }
        }
    }
    __syncthreads();
    // sequences without tokens: zeros
    for (int s = blockIdx.x; s < a.n_seqs; s += gridDim.x)
        if (sequence(a, s).tiles == 0) {
            for (int i = tid; i < a.n_heads * HD / 8; i += kAttnThreads) reinterpret_cast<uint4 *>(a.out + (size_t)s * a.out_stride)[i] = make_uint4(0, 0, 0, 0);
            for (int i = tid; i < pairs; i += kAttnThreads) a.meta[s * pairs + i] = make_int2(0, 0);
        }
    if (!works) return;
    const Place from = s_place[0], upto_place = s_place[1];
    const long long length = upto_place.at - from.at;
    if (length <= 0) return;

    auto open = [&](Walk &w) {           // the part of pair (s, i) from tile w.t on, `left` tiles of the range being left; then this warp's first tile
        w.t_end = (int)min((long long)w.q.tiles, w.t + w.left);
        w.t_coded = min(w.t_end, w.q.coded);
    };
    auto next_pair = [&](Walk &w) {
        if (++w.i >= pairs || w.q.tiles == 0) {
            w.i = 0;
            do {
                w.s++;
                w.q = sequence(a, w.s);
            } while (w.q.tiles == 0);
        }
    };
    auto begin = [&](Walk &w) {
        w.s = from.s;
        w.i = from.i;
        w.t = from.x;
        w.left = length;
        w.q = sequence(a, w.s);
        if (w.i >= pairs) { w.i = pairs - 1; next_pair(w); }
        open(w);
    };

    // ---- copies of 8-bit tiles, kStages ahead
    Walk ahead;
    begin(ahead);
    long long ahead_left = length;       // tiles of the range from this pair's part on
    int ahead_from = ahead.t;
    ahead.t += warp;
    bool more = true;
    int id0 = 0, id1 = 0, ahead_h = ahead.i / a.groups;
    auto settle = [&]() {                // to this warp's next 8-bit tile, and its blocks' numbers
        while (more && ahead.t >= ahead.t_coded) {
            ahead_left -= ahead.t_end - ahead_from;
            if (ahead_left <= 0) { more = false; break; }
            next_pair(ahead);
            ahead_h = ahead.i / a.groups;
            ahead.t = ahead_from = 0;
            ahead.left = ahead_left;
            open(ahead);
            ahead.t = warp;
        }
        if (more) {
            const int *row = a.tables + (size_t)ahead.s * a.max_blocks;
            const int tok = ahead.t * kTile;
            id0 = row[tok >> sh];
            if (b < kTile) id1 = tok + 16 < ahead.q.full ? row[(tok >> sh) + 1] : id0;
        }
    };
    unsigned bad_stages = 0;
    uint8_t *my_ring = ring + warp * kStages * kTileBytes;
    float4 *my_scale = ring_scale + warp * kStages * 2;
    auto issue = [&](int stage) {        // copies the tile that settle() found
        const int tok = ahead.t * kTile, h = ahead_h;
        const bool two = b < kTile, second = two && tok + 16 < ahead.q.full;
        const bool ok = (unsigned)id0 < (unsigned)a.n_blocks && (unsigned)(two ? id1 : id0) < (unsigned)a.n_blocks;
        bad_stages = (bad_stages & ~(1u << stage)) | (ok ? 0u : 1u << stage);
        if (lane == 0) {
            const uint32_t bar = smem_u32(&bars[warp][stage]), to = smem_u32(my_ring + stage * kTileBytes), to_scale = smem_u32(my_scale + stage * 2);
            const uint32_t bytes = !ok ? 0u : two ? (kUnit + 16u) * (second ? 2u : 1u) : kTileBytes + 16u;
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
            if (!ok) {
                if (a.status) atomicOr(a.status, 16u);
            } else {
                const size_t at = (size_t)id0 * a.n_kv + h;
                bulk_copy(to, a.data + ((at << (sh - 4)) + ((tok & (b - 1)) >> 4)) * kUnit, two ? kUnit : kTileBytes, bar);
                bulk_copy(to_scale, a.scales + at, 16, bar);
                if (second) {
                    const size_t at1 = (size_t)id1 * a.n_kv + h;
                    bulk_copy(to + kUnit, a.data + at1 * kUnit, kUnit, bar);
                    bulk_copy(to_scale + 16, a.scales + at1, 16, bar);
                }
            }
        }
    };
    auto feed = [&](int stage) {
        if (!more) return;
        issue(stage);
        ahead.t += kAttnWarps;
        settle();
    };
    settle();
#pragma unroll
    for (int k = 0; k < kStages; k++) feed(k);

    // ---- the range, a pair's part at a time
    Walk w;
    begin(w);
    int w_from = w.t, stage = 0;
    uint32_t parity = 0;
    bool waited = true, first = true;
    for (;;) {
        const int s = w.s, h = w.i / a.groups, grp = w.i % a.groups, rep = a.n_heads / a.n_kv, head0 = h * rep + grp * kRowsMax, rows = min(kRowsMax, rep - grp * kRowsMax);
        // q as the first operand: rows g and g + 8, dims 16c + 4k + (0, 1), (2, 3) of step k
        uint32_t qa[HALVES * 4][4];
#pragma unroll
        for (int half = 0; half < HALVES; half++)
#pragma unroll
            for (int up = 0; up < 2; up++) {
                uint4 v[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
                if (up < UP && g + 8 * up < rows) {
                    const uint4 *p = reinterpret_cast<const uint4 *>(a.q + (size_t)s * a.q_stride + (head0 + g + 8 * up) * HD + half * 64 + c * 16);
                    v[0] = p[0];
                    v[1] = p[1];
                }
                const uint32_t r[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
                for (int k = 0; k < 4; k++) { qa[half * 4 + k][up] = r[2 * k]; qa[half * 4 + k][2 + up] = r[2 * k + 1]; }
            }
        float o[NT][4], m[UP], l[UP], ref = 0.f;      // sums in units of ref
#pragma unroll
        for (int up = 0; up < UP; up++) { m[up] = -INFINITY; l[up] = 0.f; }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[n][e] = 0.f;

        // products of a tile -> weights, with sc: bits of the exponent per unit of a product, and the sums so far brought to the new maximum
        auto weigh = [&](float (&x)[4][4], float sc0, float sc1) {
            float shift[UP], fix[UP];
            bool moved = false;
#pragma unroll
            for (int up = 0; up < UP; up++) {
                float mx = fmaxf(fmaxf(fmaxf(x[0][2 * up], x[0][2 * up + 1]), fmaxf(x[1][2 * up], x[1][2 * up + 1])) * sc0,
                                 fmaxf(fmaxf(x[2][2 * up], x[2][2 * up + 1]), fmaxf(x[3][2 * up], x[3][2 * up + 1])) * sc1);
                mx = fmaxf(mx, __shfl_xor_sync(kFullMask, mx, 1));
                mx = fmaxf(m[up], fmaxf(mx, __shfl_xor_sync(kFullMask, mx, 2)));
                const float at = mx == -INFINITY ? 0.f : mx;
                fix[up] = ex2(m[up] - at);
                moved |= mx != m[up];
                m[up] = mx;
                shift[up] = kLift - at;
                l[up] *= fix[up];
            }
            if (__any_sync(kFullMask, moved)) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[n][e] *= fix[R16 ? e >> 1 : 0];
            }
#pragma unroll
            for (int n = 0; n < 4; n++)
#pragma unroll
                for (int e = 0; e < E; e++) {
                    x[n][e] = ex2(fmaf(x[n][e], n < 2 ? sc0 : sc1, shift[e >> 1]));
                    l[e >> 1] += x[n][e];
                }
        };
        // weights of 16 tokens, times f, as the first operand.  Up to 8 query heads leave the rows 8 to 15 free: they take what the rounding
        // of the weights to fp16 leaves over, and their sums are added in the end.
        auto operand = [&](uint32_t (&p)[4], const float (&x)[4][4], int u, float f) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const float y0 = x[2 * u + k][0] * f, y1 = x[2 * u + k][1] * f;
                p[2 * k] = pack(y0, y1);
                if constexpr (R16) p[2 * k + 1] = pack(x[2 * u + k][2] * f, x[2 * u + k][3] * f);
                else {
                    const float2 r = __half22float2(*reinterpret_cast<const __half2 *>(&p[2 * k]));
                    p[2 * k + 1] = pack(y0 - r.x, y1 - r.y);
                }
            }
        };
        // brings the sums to a unit that is not below sv; the factor of weights whose values have the scale sv
        auto unit_factor = [&](float sv) {
            if (sv > ref) {
                const float f = ref / sv;
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[n][e] *= f;
                ref = sv;
            }
            return ref > 0.f ? sv / ref : sv;
        };

        for (int t = w.t + warp; t < w.t_end; t += kAttnWarps) {
            float x[4][4] = {};
            if (t < w.t_coded) {
                waited &= bar_wait(smem_u32(&bars[warp][stage]), parity);
                const uint8_t *tile = my_ring + stage * kTileBytes;
                const bool lone = b < kTile && t * kTile + 16 >= w.q.full;             // 16 tokens only
                float2 sc[2];
                sc[0] = *reinterpret_cast<const float2 *>(my_scale + stage * 2);
                sc[1] = b < kTile ? *reinterpret_cast<const float2 *>(my_scale + stage * 2 + 1) : sc[0];
                if (bad_stages >> stage & 1) sc[0] = sc[1] = make_float2(NAN, NAN);
#pragma unroll
                for (int half = 0; half < HALVES; half++) {
                    uint4 v[4];
#pragma unroll
                    for (int n = 0; n < 4; n++)
                        v[n] = *reinterpret_cast<const uint4 *>(tile + (n >> 1) * kUnit + ((n & 1) * HALVES + half) * 512 + lane * 16);
#pragma unroll
                    for (int k = 0; k < 4; k++)
#pragma unroll
                        for (int n = 0; n < 4; n++) {
                            uint32_t b0, b1;
                            widen<KIND>(k == 0 ? v[n].x : k == 1 ? v[n].y : k == 2 ? v[n].z : v[n].w, b0, b1);
                            mma(x[n], qa[half * 4 + k], b0, b1);
                        }
                }
                if (lone) {
#pragma unroll
                    for (int e = 0; e < E; e++) x[2][e] = x[3][e] = -INFINITY;
                }
                weigh(x, a.scale * sc[0].x, lone ? 1.f : a.scale * sc[1].x);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    if (u == 1 && lone) continue;
                    const float f = unit_factor(sc[u].y);
                    uint32_t p[4];
                    operand(p, x, u, f);
#pragma unroll
                    for (int n = 0; n < NT / 4; n++) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(tile + u * kUnit + 16 * HD + n * 512 + lane * 16);
                        const uint32_t r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            uint32_t b0, b1;
                            widen<KIND>(r[j], b0, b1);
                            mma(o[4 * n + j], p, b0, b1);
                        }
                    }
                }
                __syncwarp();
                feed(stage);
                if (++stage == kStages) { stage = 0; parity ^= 1; }
            } else {
                // tokens in 16 bits, from the tail
                const int t0 = (t - w.q.coded) * kTile, n_tok = min(kTile, w.q.tail - t0);
                const __half *tk = a.tail_k + (size_t)s * a.tail_k_stride + ((size_t)h * b + t0) * HD;
                const __half *tv = a.tail_v + (size_t)s * a.tail_v_stride + ((size_t)h * b + t0) * HD;
#pragma unroll
                for (int n = 0; n < 4; n++)
#pragma unroll
                    for (int half = 0; half < HALVES; half++) {
                        uint4 v[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
                        if (n * 8 + g < n_tok) {
                            const uint4 *p = reinterpret_cast<const uint4 *>(tk + (n * 8 + g) * HD + half * 64 + c * 16);
                            v[0] = p[0];
                            v[1] = p[1];
                        }
                        const uint32_t r[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
                        for (int k = 0; k < 4; k++) mma(x[n], qa[half * 4 + k], r[2 * k], r[2 * k + 1]);
                    }
#pragma unroll
                for (int n = 0; n < 4; n++)
#pragma unroll
                    for (int e = 0; e < E; e++)
                        if (n * 8 + 2 * c + (e & 1) >= n_tok) x[n][e] = -INFINITY;
                weigh(x, a.scale, a.scale);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    if (16 * u >= n_tok) continue;
                    uint4 v[2][NT / 4];
                    uint32_t top = 0;
#pragma unroll
                    for (int hh = 0; hh < 2; hh++) {
                        const int tok = 16 * u + 8 * hh + 2 * c;          // and the next one
#pragma unroll
                        for (int n = 0; n < NT / 4; n++) {
                            v[hh][n] = make_uint4(0, 0, 0, 0);
                            if (tok < n_tok) v[hh][n] = *reinterpret_cast<const uint4 *>(tv + (size_t)tok * HD + (g * NT + 4 * n) * 2);
                            if (tok + 1 >= n_tok) { v[hh][n].x &= 0xFFFFu; v[hh][n].y &= 0xFFFFu; v[hh][n].z &= 0xFFFFu; v[hh][n].w &= 0xFFFFu; }
                            top = __vmaxu2(top, __vmaxu2(__vmaxu2(v[hh][n].x & 0x7FFF7FFFu, v[hh][n].y & 0x7FFF7FFFu),
                                                         __vmaxu2(v[hh][n].z & 0x7FFF7FFFu, v[hh][n].w & 0x7FFF7FFFu)));
                        }
                    }
                    // a power of two for the scale, so that small values keep their weights' digits: the exponent that covers all of them
                    top = __reduce_max_sync(kFullMask, max(top & 0xFFFFu, top >> 16));
                    const int e2 = top >= 0x7C00u ? 0 : max((int)(top >> 10), 1) - 15 - 6;
                    const float up_by = exp2f((float)-e2);
                    const float f = unit_factor(exp2f((float)e2));
                    uint32_t p[4];
                    operand(p, x, u, f);
                    auto scaled = [&](uint32_t r) {
                        const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&r));
                        return pack(y.x * up_by, y.y * up_by);
                    };
#pragma unroll
                    for (int n = 0; n < NT / 4; n++) {
                        mma(o[4 * n], p, scaled(v[0][n].x), scaled(v[1][n].x));
                        mma(o[4 * n + 1], p, scaled(v[0][n].y), scaled(v[1][n].y));
                        mma(o[4 * n + 2], p, scaled(v[0][n].z), scaled(v[1][n].z));
                        mma(o[4 * n + 3], p, scaled(v[0][n].w), scaled(v[1][n].w));
                    }
                }
            }
        }

        // ---- the four warps' sums, half of the columns at a time
#pragma unroll
        for (int up = 0; up < UP; up++) {
            l[up] += __shfl_xor_sync(kFullMask, l[up], 1);
            l[up] += __shfl_xor_sync(kFullMask, l[up], 2);
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < E; e++) o[n][e] = (R16 ? o[n][e] : o[n][e] + o[n][2 + e]) * ref;
#pragma unroll
        for (int step = 2; step >= 1; step >>= 1) {
            float *at = join + (warp & (step - 1)) * (kJoin * 32) + lane;
            float fa[UP], fb[UP];
#pragma unroll
            for (int half = 0; half < 2; half++) {
                if (warp >= step && warp < 2 * step) {
#pragma unroll
                    for (int n = 0; n < NT / 2; n++)
#pragma unroll
                        for (int e = 0; e < E; e++) at[(E * n + e) * 32] = o[half * (NT / 2) + n][e];
                    if (half == 0) {
#pragma unroll
                        for (int up = 0; up < UP; up++) { at[(kJoin - 1 - up) * 32] = m[up]; at[(kJoin - 3 - up) * 32] = l[up]; }
                    }
                }
                __syncthreads();
                if (warp < step) {
                    if (half == 0) {
#pragma unroll
                        for (int up = 0; up < UP; up++) {
                            const float mb = at[(kJoin - 1 - up) * 32], mx = fmaxf(m[up], mb), ref_m = mx == -INFINITY ? 0.f : mx;
                            fa[up] = ex2(m[up] - ref_m);
                            fb[up] = ex2(mb - ref_m);
                            l[up] = l[up] * fa[up] + at[(kJoin - 3 - up) * 32] * fb[up];
                            m[up] = mx;
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT / 2; n++)
#pragma unroll
                        for (int e = 0; e < E; e++)
                            o[half * (NT / 2) + n][e] = o[half * (NT / 2) + n][e] * fa[e >> 1] + at[(E * n + e) * 32] * fb[e >> 1];
                }
                __syncthreads();
            }
        }
        if (warp == 0) {
            const bool starts = w.t == 0, whole = starts && w.t_end == w.q.tiles;
            const int slot = 2 * blockIdx.x + (first ? 0 : 1);
            if (lane == 0 && starts) {
                // the CTAs from this one to the one that ends the pair
                int parts = 1;
                if (!whole) {
                    const long long end = from.at + (length - w.left) + w.q.tiles;
                    long long last = (end - 1) * ctas / total;
                    last = min(last + 1, ctas - 1);
                    while (last > blockIdx.x) {
                        // where that CTA's range begins, as above; inside this pair it is at x of its tiles
                        const long long at = last * total / ctas, x = at - (end - w.q.tiles);
                        if (at < end && x > kSnap && w.q.tiles - x > kSnap) break;
                        last--;
                    }
                    parts = (int)(last - blockIdx.x) + 1;
                }
                a.meta[s * pairs + w.i] = make_int2(slot, whole ? 0 : parts);
            }
#pragma unroll
            for (int up = 0; up < UP; up++) {
                const int row = g + 8 * up;
                if (row >= rows) continue;
                if (whole) {
                    const float inv = 1.f / l[up];
                    __half *to = a.out + (size_t)s * a.out_stride + (head0 + row) * HD;
#pragma unroll
                    for (int e = 0; e < 2; e++)
#pragma unroll
                        for (int n = 0; n < NT; n += 8) {
                            uint4 v;
                            v.x = pack(o[n][2 * up + e] * inv, o[n + 1][2 * up + e] * inv);
                            v.y = pack(o[n + 2][2 * up + e] * inv, o[n + 3][2 * up + e] * inv);
                            v.z = pack(o[n + 4][2 * up + e] * inv, o[n + 5][2 * up + e] * inv);
                            v.w = pack(o[n + 6][2 * up + e] * inv, o[n + 7][2 * up + e] * inv);
                            *reinterpret_cast<uint4 *>(to + (2 * c + e) * NT + n) = v;
                        }
                } else {
                    float *to = a.part_o + ((size_t)slot * a.rows + row) * HD;
#pragma unroll
                    for (int e = 0; e < 2; e++)
#pragma unroll
                        for (int n = 0; n < NT; n += 4)
                            *reinterpret_cast<float4 *>(to + (2 * c + e) * NT + n) =
                                make_float4(o[n][2 * up + e], o[n + 1][2 * up + e], o[n + 2][2 * up + e], o[n + 3][2 * up + e]);
                    if (c == 0) a.part_ml[slot * a.rows + row] = make_float2(m[up], l[up]);
                }
            }
        }
        first = false;
        w.left -= w.t_end - w_from;
        if (w.left <= 0) break;
        next_pair(w);
        w.t = w_from = 0;
        open(w);
    }
    if (!waited) {                       // a copy did not arrive in time: report, and leave only when none is in flight
        if (a.status && lane == 0) atomicOr(a.status, (unsigned)kStatusWait);
        for (int k = 0; k < kStages; k++) {
            bar_wait(smem_u32(&bars[warp][k]), 0);
            bar_wait(smem_u32(&bars[warp][k]), 1);
        }
    }
}

// One CTA per query head and sequence: the parts of its pair, a warp every fourth, then the four sums.
template <int HD>
__global__ void __launch_bounds__(128) attn_join_kernel(const AttnArgs a) {
    __shared__ float s_o[4][HD], s_m[4], s_l[4];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int rep = a.n_heads / a.n_kv, head = blockIdx.x, in = head % rep, pair = (head / rep) * a.groups + in / kRowsMax, row = in % kRowsMax;
    const int2 meta = a.meta[blockIdx.y * a.n_kv * a.groups + pair];
    if (meta.y == 0) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, E = HD / 32;
    float m = -INFINITY, l = 0.f, o[E] = {};
    for (int k = warp; k < meta.y; k += 4) {
        const int slot = k == 0 ? meta.x : 2 * (meta.x / 2 + k);
        const float2 ml = a.part_ml[slot * a.rows + row];
        const float *from = a.part_o + ((size_t)slot * a.rows + row) * HD + lane * E;
        const float mx = fmaxf(m, ml.x), at = mx == -INFINITY ? 0.f : mx, fa = ex2(m - at), fb = ex2(ml.x - at);
        m = mx;
        l = l * fa + ml.y * fb;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = o[e] * fa + from[e] * fb;
    }
#pragma unroll
    for (int e = 0; e < E; e++) s_o[warp][lane * E + e] = o[e];
    if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
    __syncthreads();
    const float mx = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3])), at = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, v = 0.f;
    if (threadIdx.x < HD) {
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float f = ex2(s_m[w] - at);
            sum += s_l[w] * f;
            v += s_o[w][threadIdx.x] * f;
        }
        a.out[(size_t)blockIdx.y * a.out_stride + head * HD + threadIdx.x] = __float2half_rn(v / sum);
    }
}

struct Workspace {
    size_t o, ml, meta, bytes;
    int ctas, groups, rows;
};
Workspace workspace_of(int n_seqs, int n_heads, int n_kv, int hd) {
    Workspace w;
    const int rep = n_heads / n_kv;
    w.groups = (rep + kRowsMax - 1) / kRowsMax;
    w.rows = rep < kRowsMax ? rep : kRowsMax;
    w.ctas = 2 * sm_count();
    w.o = 0;
    w.ml = w.o + (size_t)2 * w.ctas * w.rows * hd * sizeof(float);
    w.meta = w.ml + (size_t)2 * w.ctas * w.rows * sizeof(float2);
    w.bytes = w.meta + (size_t)n_seqs * n_kv * w.groups * sizeof(int2);
    return w;
}

}  // namespace
}  // namespace qtip

using namespace qtip;

extern "C" size_t qtip_attn_paged_workspace_bytes(int n_seqs, int n_heads, int n_kv_heads, int head_dim) {
    if (n_seqs < 1 || n_heads < 1 || n_kv_heads < 1 || n_heads % n_kv_heads || head_dim < 1) return 0;
    return workspace_of(n_seqs, n_heads, n_kv_heads, head_dim).bytes;
}

extern "C" int qtip_attn_decode_paged(void *out, long out_stride, const void *q, long q_stride, const void *data, const float *scales, const void *tail_k,
                                      long tail_k_stride, const void *tail_v, long tail_v_stride, const int *tables, const int *lengths, int n_seqs,
                                      int n_heads, int n_kv_heads, int head_dim, int max_blocks, int n_blocks, int block, int kind, void *workspace,
                                      size_t workspace_bytes, unsigned *status, void *stream) {
    if (!out || !q || !data || !scales || !tail_k || !tail_v || !tables || !lengths) return QTIP_ERR_BAD_ARG;
    if (!paged_shape_ok(n_heads, n_kv_heads, head_dim, block, kind) || n_seqs < 1 || n_seqs > 65535 || max_blocks < 1 || n_blocks < 1 || n_heads > 65535)
        return QTIP_ERR_BAD_SHAPE;
    if (((long)max_blocks + 1) * block > 0x7FFFFFFFl) return QTIP_ERR_BAD_SHAPE;
    const Workspace ws = workspace_of(n_seqs, n_heads, n_kv_heads, head_dim);
    if (!workspace || workspace_bytes < ws.bytes) return QTIP_ERR_WORKSPACE;
    const void *ptrs[] = {out, q, data, scales, tail_k, tail_v, workspace};
    for (const void *p : ptrs)
        if (!aligned(p, 16)) return QTIP_ERR_ALIGNMENT;
    if ((out_stride | q_stride | tail_k_stride | tail_v_stride) & 7) return QTIP_ERR_ALIGNMENT;
    uint8_t *w = static_cast<uint8_t *>(workspace);
    const AttnArgs a = {static_cast<__half *>(out), static_cast<const __half *>(q), out_stride, q_stride, static_cast<const uint8_t *>(data),
                        reinterpret_cast<const float4 *>(scales), static_cast<const __half *>(tail_k), static_cast<const __half *>(tail_v), tail_k_stride,
                        tail_v_stride, tables, lengths, n_seqs, n_heads, n_kv_heads, max_blocks, n_blocks, block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7,
                        1.4426950408889634f / sqrtf((float)head_dim), reinterpret_cast<float *>(w + ws.o), reinterpret_cast<float2 *>(w + ws.ml),
                        reinterpret_cast<int2 *>(w + ws.meta), ws.groups, ws.rows, status};
    const bool r16 = ws.rows > 8;
    auto kernel = head_dim == 128 ? (kind == kKvInt8 ? (r16 ? attn_paged_kernel<128, kKvInt8, true> : attn_paged_kernel<128, kKvInt8, false>)
                                                     : (r16 ? attn_paged_kernel<128, kKvE4m3, true> : attn_paged_kernel<128, kKvE4m3, false>))
                                  : (kind == kKvInt8 ? (r16 ? attn_paged_kernel<64, kKvInt8, true> : attn_paged_kernel<64, kKvInt8, false>)
                                                     : (r16 ? attn_paged_kernel<64, kKvE4m3, true> : attn_paged_kernel<64, kKvE4m3, false>));
    const size_t smem = (size_t)kAttnWarps * kStages * (64 * head_dim + 32) + (size_t)2 * (head_dim / 4 + 4) * 32 * sizeof(float);
    QTIP_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ws.ctas);
    cfg.blockDim = dim3(kAttnThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    QTIP_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a));
    // a pair of at most 2 * kSnap tiles is never cut
    if (((long)max_blocks * block + kTile - 1) / kTile + (block - 1 + kTile - 1) / kTile > 2 * kSnap) {
        cfg.gridDim = dim3(n_heads, n_seqs);
        cfg.blockDim = dim3(128);
        cfg.dynamicSmemBytes = 0;
        QTIP_CUDA_TRY(cudaLaunchKernelEx(&cfg, head_dim == 128 ? attn_join_kernel<128> : attn_join_kernel<64>, a));
    }
    return check_launch();
}
