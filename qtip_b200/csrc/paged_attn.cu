// Single-query attention over the key/value cache in 8 bits (paged.cuh): out = softmax(q K^T / sqrt(hd)) V for each sequence and head.
// Stands where the decode loop has the scaled_dot_product_attention of LlamaSdpaAttention.forward (model/llama.py:884-891 upstream).
//
// Bound by the bytes of the cache: 2 per token, key/value head and dim, read once for up to 16 query heads that share them (their scores and sums fill a
// warp's registers), twice for 17 to 32, and so on.
// A pair is a sequence and a key/value head (of at most 16 query heads; more are further pairs).  Its tokens are cut into tiles of 32, and the
// tiles of all pairs, in order, are dealt to the CTAs in equal contiguous ranges, computed by every CTA from the lengths: a long sequence is
// spread over the chip, and a CTA goes through several short ones.  The start of a pair counts as kStart tiles (its queries, and the join of the
// four warps' sums).  A cut that would leave less than kSnap + 1 tiles on one side is moved to the pair's border.  A pair inside one range is finished there; the parts of others go to the workspace, and a second kernel joins
// them in the order of the tokens.
// A warp takes every fourth tile of a range.  One of its lanes keeps kStages copies of tiles in flight (a tile of a block of 32 tokens or
// more is one piece of memory: K and V of 32 tokens); the lanes read the bytes in the order of the operands of the matrix instruction
// (K q^T: 16 tokens by 8 query heads, 16 dims deep; V^T p^T: 16 dims by 8 heads, 16 tokens deep) and widen them to fp16, which holds every code.
#include <type_traits>
#include <utility>

#include "paged.cuh"

namespace qtip {
namespace {

// kStart, kSnap: 2, 4, 8 tiles as the start of a pair take 51.1 / 51.1 / 50.0 us for 64 sequences of 8000 to 16000, 16 heads on one, and 202 / 200 / 202 for 32 of
// 1025 to 8191, 32 heads; as the least part of a pair 9.6 / 9.7 / 12.4 for one of 500, 32 heads, 14.9 / 15.7 / 14.9 for eight of them, 202 / 200 / 199 for the 32.
constexpr int kAttnWarps = 4, kAttnThreads = 32 * kAttnWarps, kTile = 32, kSnap = 4, kStart = 4, kRowsMax = 16;
// Waves of CTAs for much work, the share of the first in %, and how much is much: bytes of a CTA's tiles, if there were one wave.  The 32 sequences above: 289 us in
// one wave, 211 / 200 / 242 with 40 / 60 / 80 %.  Their tiles are 340 * 8192 bytes to a CTA; with 101 * 8192 (64 sequences of 2000 to 9000, 32 heads on 8 of 64 dims) one
// wave takes 78 us and three 89.
constexpr int kWaves = 3, kFirst = 60, kMuch = 160 * 8192;
constexpr float kLift = 32768.f;     // weights are multiplied by 2^15 before they are rounded: fp16 then reaches down to 2^-39 of the largest
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

// An 8 x 8 matrix of fp16, a row in four lanes, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

constexpr int kTailTile = 16;      // tokens of a tile of the tail: as many bytes as 32 in 8 bits

// A sequence's tokens in blocks, all of them, and tiles of either; what one of its pairs counts.
struct Sequence {
    int full, len, coded, tiles;
    __device__ __forceinline__ int cost() const { return tiles ? tiles + kStart : 0; }
};
__device__ __forceinline__ Sequence sequence(const AttnArgs &a, int len) {
    Sequence q;
    q.full = len >> a.shift << a.shift;
    q.len = len;
    q.coded = (q.full + kTile - 1) / kTile;
    q.tiles = q.coded + (len - q.full + kTailTile - 1) / kTailTile;
    return q;
}
__device__ __forceinline__ int length_of(const AttnArgs &a, int s) {
    const int len = a.lengths[s];
    return len < 0 || len >> a.shift > a.max_blocks ? 0 : len;
}

// A walk over the parts of pairs in a range: sequence, pair of it, the part's tiles t0 .. t1, and what the range counts from t0 on.
struct Walk {
    int s, i, t0, t1, left;
    Sequence q;
};

// NB: groups of 8 query heads.
template <int HD, int NB>
struct AttnShape {
    static constexpr int kUnit = 32 * HD, kTileBytes = 2 * kUnit, MT = HD / 16, HALVES = HD / 64;
    static constexpr int kCtas = NB == 1 ? 3 : 2, kStages = NB == 1 && HD == 128 ? 2 : 3;      // per SM; copies in flight per warp
    static constexpr int kJoin = NB * 2 * MT;                                                 // half of a lane's sums
    static constexpr size_t kSmem = (size_t)kAttnWarps * (kStages * (kTileBytes + 32) + (kJoin * 32 + NB * 16) * sizeof(float));
};

template <int HD, int KIND, int NB>
__global__ void __launch_bounds__(kAttnThreads, AttnShape<HD, NB>::kCtas) attn_paged_kernel(const AttnArgs a) {
    using Shape = AttnShape<HD, NB>;
    constexpr int kUnit = Shape::kUnit, kTileBytes = Shape::kTileBytes, MT = Shape::MT, HALVES = Shape::HALVES, kStages = Shape::kStages, kJoin = Shape::kJoin;
    extern __shared__ __align__(128) uint8_t attn_smem[];
    uint8_t *ring = attn_smem;                                                            // [warp][stage][kTileBytes]
    float4 *ring_scale = reinterpret_cast<float4 *>(attn_smem + kAttnWarps * kStages * kTileBytes);      // [warp][stage][2]
    float *join = reinterpret_cast<float *>(ring_scale + kAttnWarps * kStages * 2);       // [warp][kJoin][32]
    float2 *join_ml = reinterpret_cast<float2 *>(join + kAttnWarps * kJoin * 32);         // [warp][head of 8 NB]
    __shared__ uint64_t bars[kAttnWarps][kStages];
    // The ranges are cut for kCtas per SM.  Registers are held to that by the launch bounds, shared memory (228 KB per SM, in steps of 128 bytes, 1 KB of it
    // the system's for each CTA; for 128 dims and 16 query heads it is used to the last byte) by this.
    static_assert(Shape::kCtas * ((Shape::kSmem + sizeof(bars) + 127) / 128 * 128 + 1024) <= 228 * 1024, "an SM does not hold kCtas of these CTAs");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3, sh = a.shift, b = 1 << sh;
    const int pairs = a.n_kv * a.groups;                                                  // of a sequence
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (lane < kStages) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&bars[warp][lane])));      // a warp's own
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // ---- this CTA's range of tiles; every warp computes it, from a piece of the lengths in each lane
    const int per = (a.n_seqs + 31) >> 5, s_lo = min(lane * per, a.n_seqs), s_hi = min(s_lo + per, a.n_seqs);
    int mine = 0, seqs = 0;
    for (int s = s_lo; s < s_hi; s++) {
        const int cost = sequence(a, length_of(a, s)).cost();
        mine += cost;
        seqs += cost > 0;
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(kFullMask, upto, o);
        if (lane >= o) upto += u;
    }
    seqs = __reduce_add_sync(kFullMask, seqs);
    const int total = __shfl_sync(kFullMask, upto, 31) * pairs;
    // A range is at least four tiles, one per warp, or a pair.  With more work the chip's first CTAs take equal ranges of kFirst % of it, and as many
    // CTAs per further wave equal ranges of the rest, as the first ones end: some SMs get at the memory faster than others.
    const int least = max(total / kAttnWarps, seqs * pairs), room = gridDim.x / kWaves;
    int ctas = max(min(min(total, least), room), 1), share2 = 0, rest2 = 0, early = ctas, early_tiles = total;
    if (kWaves > 1 && total >= room * (kMuch / kTileBytes)) {
        ctas = gridDim.x;
        early = room;
        early_tiles = total / 100 * kFirst;
        share2 = (total - early_tiles) / (ctas - early);
        rest2 = total - early_tiles - share2 * (ctas - early);
    }
    const int share = early_tiles / early, rest = early_tiles - share * early;
    auto border = [&](int cta) {                       // where a CTA's range begins, before it is moved to a pair's border
        return cta <= early ? cta * share + min(cta, rest) : early_tiles + (cta - early) * share2 + min(cta - early, rest2);
    };
    auto owner = [&](int tile) {                       // the last CTA whose border is not behind this
        const int base = tile < early_tiles ? 0 : early, n = tile < early_tiles ? share : share2, r = tile < early_tiles ? rest : rest2;
        if (tile >= early_tiles) tile -= early_tiles;
        return base + (tile < r * (n + 1) ? tile / (n + 1) : (tile - r) / n);
    };
    // sequences without tokens: zeros
    for (int s = blockIdx.x; s < a.n_seqs; s += gridDim.x) {
        if (length_of(a, s) > 0) continue;
        if (a.lengths[s] != 0 && a.status && tid == 0) atomicOr(a.status, 1u);
        for (int i = tid; i < a.n_heads * HD / 8; i += kAttnThreads) reinterpret_cast<uint4 *>(a.out + (size_t)s * a.out_stride)[i] = make_uint4(0, 0, 0, 0);
        for (int i = tid; i < pairs; i += kAttnThreads) a.meta[s * pairs + i] = make_int2(0, 0);
    }
    if (blockIdx.x >= ctas || total == 0) return;
    int from = 0, length = 0;
    Walk w;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        int at = border(blockIdx.x + k), ps = 0, pi = 0, px = 0, plen = 0;
        const bool here = (upto - mine) * pairs <= at && at < upto * pairs;
        if (here) {
            int before = (upto - mine) * pairs;
            for (int s = s_lo; s < s_hi; s++) {
                const int len = length_of(a, s), cost = sequence(a, len).cost();
                if (at < before + cost * pairs) {
                    ps = s;
                    plen = len;
                    pi = (at - before) / cost;
                    px = at - before - pi * cost;
                    if (px <= kStart + kSnap) { at -= px; px = 0; }
                    else if (cost - px <= kSnap) { at += cost - px; px = 0; pi++; }
                    else px -= kStart;
                    break;
                }
                before += cost * pairs;
            }
        }
        const unsigned who = __ballot_sync(kFullMask, here);      // none for the end of all tiles
        const int src = who ? __ffs(who) - 1 : 0;
        at = __shfl_sync(kFullMask, at, src);
        if (k == 1) { length = at - from; break; }
        from = at;
        w.s = __shfl_sync(kFullMask, ps, src);
        w.i = __shfl_sync(kFullMask, pi, src);
        w.t0 = __shfl_sync(kFullMask, px, src);
        w.q = sequence(a, __shfl_sync(kFullMask, plen, src));
    }
    if (length <= 0) return;

    auto next_pair = [&](Walk &y) {
        y.t0 = 0;
        if (++y.i >= pairs) {
            y.i = 0;
            do y.q = sequence(a, length_of(a, ++y.s));
            while (y.q.tiles == 0);
        }
    };
    if (w.i >= pairs) next_pair(w);
    w.left = length;
    auto bound = [&](Walk &y) { y.t1 = min(y.q.tiles, y.t0 ? y.t0 + y.left : y.left - kStart); };
    auto count = [](const Walk &y) { return y.t1 - y.t0 + (y.t0 ? 0 : kStart); };          // of the part
    bound(w);

    // ---- copies of this warp's tiles, kStages ahead
    Walk ahead = w;
    int ahead_t = w.t0 + warp, ahead_h = w.i / a.groups, id0 = 0, id1 = 0;
    bool more = true;
    auto settle = [&]() {                // to this warp's next tile, and its blocks' numbers
        while (more && ahead_t >= ahead.t1) {
            ahead.left -= count(ahead);
            if (ahead.left <= 0) { more = false; break; }
            next_pair(ahead);
            bound(ahead);
            ahead_t = warp;
            ahead_h = ahead.i / a.groups;
        }
        if (more && ahead_t < ahead.q.coded) {
            const int *row = a.tables + (size_t)ahead.s * a.max_blocks;
            const int tok = ahead_t * kTile;
            id0 = id1 = row[tok >> sh];
            if (b < kTile && tok + 16 < ahead.q.full) id1 = row[(tok >> sh) + 1];
        }
    };
    unsigned bad_stages = 0;
    uint8_t *my_ring = ring + warp * kStages * kTileBytes;
    float4 *my_scale = ring_scale + warp * kStages * 2;
    auto feed = [&](int stage) {         // copies the tile that settle() found, and goes to the next
        if (!more) return;
        const uint32_t bar = smem_u32(&bars[warp][stage]), to = smem_u32(my_ring + stage * kTileBytes), to_scale = smem_u32(my_scale + stage * 2);
        bad_stages &= ~(1u << stage);
        if (ahead_t >= ahead.q.coded) {
            const int t0 = (ahead_t - ahead.q.coded) * kTailTile, n = min(kTailTile, ahead.q.len - ahead.q.full - t0);
            if (lane == 0) {
                const size_t at = ((size_t)ahead_h * b + t0) * HD;
                const uint32_t bytes_k = n * HD * 2, bytes_v = (n + 1) / 2 * HD * 4;
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes_k + bytes_v) : "memory");
                bulk_copy(to, a.tail_k + (size_t)ahead.s * a.tail_k_stride + at, bytes_k, bar);
                bulk_copy(to + kTileBytes / 2, a.tail_v + (size_t)ahead.s * a.tail_v_stride + at, bytes_v, bar);
            }
        } else {
            const int tok = ahead_t * kTile;
            const bool two = b < kTile, second = two && tok + 16 < ahead.q.full;
            const bool ok = (unsigned)id0 < (unsigned)a.n_blocks && (unsigned)id1 < (unsigned)a.n_blocks;
            if (!ok) bad_stages |= 1u << stage;
            if (lane == 0) {
                const uint32_t bytes = !ok ? 0u : two ? (kUnit + 16u) * (second ? 2u : 1u) : kTileBytes + 16u;
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
                if (!ok) {
                    if (a.status) atomicOr(a.status, 16u);
                } else {
                    const size_t at = (size_t)id0 * a.n_kv + ahead_h;
                    bulk_copy(to, a.data + ((at << (sh - 4)) + ((tok & (b - 1)) >> 4)) * kUnit, two ? kUnit : kTileBytes, bar);
                    bulk_copy(to_scale, a.scales + at, 16, bar);
                    if (second) {
                        const size_t at1 = (size_t)id1 * a.n_kv + ahead_h;
                        bulk_copy(to + kUnit, a.data + at1 * kUnit, kUnit, bar);
                        bulk_copy(to_scale + 16, a.scales + at1, 16, bar);
                    }
                }
            }
        }
        ahead_t += kAttnWarps;
        settle();
    };
    settle();
#pragma unroll
    for (int k = 0; k < kStages; k++) feed(k);

    // ---- the range, a pair's part at a time
    int stage = 0;
    uint32_t parity = 0;
    bool waited = true, first = true;
    for (;;) {
        const int s = w.s, h = w.i / a.groups, grp = w.i % a.groups, rep = a.n_heads / a.n_kv, head0 = h * rep + grp * kRowsMax, rows = min(kRowsMax, rep - grp * kRowsMax);
        // q as the second operand: head 8 nb + g, dims 16c + 4k + (0, 1), (2, 3) of step k
        uint32_t qb[NB][HALVES * 4][2];
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int half = 0; half < HALVES; half++) {
                uint4 v[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
                if (8 * nb + g < rows) {
                    const uint4 *p = reinterpret_cast<const uint4 *>(a.q + (size_t)s * a.q_stride + (head0 + 8 * nb + g) * HD + half * 64 + c * 16);
                    v[0] = p[0];
                    v[1] = p[1];
                }
                const uint32_t r[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
                for (int k = 0; k < 4; k++) { qb[nb][half * 4 + k][0] = r[2 * k]; qb[nb][half * 4 + k][1] = r[2 * k + 1]; }
            }
        // sums in units of ref / kLift: [i][0], [1]: dim g * HD/8 + 2i of heads 2c, 2c + 1; [2], [3]: the next dim.  m, l: of heads 2c, 2c + 1
        float o[NB][MT][4], m[NB][2], l[NB][2], ref = 0.f;
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            m[nb][0] = m[nb][1] = -INFINITY;
            l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[nb][i][e] = 0.f;
        }

        // products of a tile (x[u]: tokens 16u + g, + 8) -> weights, with sc: bits of the exponent per unit of a product, and the sums so far
        // brought to the new maximum.  Scores are rounded before the maximum is taken and subtracted, so that the largest weight is 1 whatever
        // their size (rounded once after the difference, it would be up to 2^64 or down to 2^-64 with scores of 2^30).
        auto weigh = [&](float (&x)[NB][2][4], float sc0, float sc1) {
            float at[NB][2], fix[NB][2];
            bool moved = false;
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        x[nb][u][e] = __fmul_rn(x[nb][u][e], u ? sc1 : sc0);
                        x[nb][u][2 + e] = __fmul_rn(x[nb][u][2 + e], u ? sc1 : sc0);
                    }
                    float mx = fmaxf(fmaxf(x[nb][0][e], x[nb][0][2 + e]), fmaxf(x[nb][1][e], x[nb][1][2 + e]));
                    mx = fmaxf(mx, __shfl_xor_sync(kFullMask, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(kFullMask, mx, 8));
                    mx = fmaxf(m[nb][e], fmaxf(mx, __shfl_xor_sync(kFullMask, mx, 16)));
                    at[nb][e] = mx == -INFINITY ? 0.f : mx;
                    fix[nb][e] = ex2(m[nb][e] - at[nb][e]);
                    moved |= mx != m[nb][e];
                    m[nb][e] = mx;
                }
            if (__any_sync(kFullMask, moved)) {
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
                    l[nb][0] *= fix[nb][0];
                    l[nb][1] *= fix[nb][1];
#pragma unroll
                    for (int i = 0; i < MT; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[nb][i][e] *= fix[nb][e & 1];
                }
            }
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        x[nb][u][e] = ex2(x[nb][u][e] - at[nb][e & 1]);
                        l[nb][e & 1] += x[nb][u][e];
                    }
        };
        // brings the sums to a unit that is not below sv; the factor of weights whose values have the scale sv, kLift in it
        auto unit_factor = [&](float sv) {
            if (sv > ref) {
                const float f = ref / sv;
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int i = 0; i < MT; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[nb][i][e] *= f;
                ref = sv;
            }
            return (ref > 0.f ? __fdividef(sv, ref) : sv) * kLift;
        };
        // weights of 16 tokens, times f, as the second operand, in two parts of fp16: the second takes what the rounding of the first leaves.
        // (With one part the error of the result is 1.4 times that of its own rounding to fp16.)
        auto operand = [&](uint32_t (&p)[2][2], const float (&x)[4], float f) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const float y0 = x[2 * k] * f, y1 = x[2 * k + 1] * f;
                const uint32_t hi = pack(y0, y1);
                const float2 r = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
                p[0][k] = transposed(hi);
                p[1][k] = transposed(pack(y0 - r.x, y1 - r.y));
            }
        };

        for (int t = w.t0 + warp; t < w.t1; t += kAttnWarps) {
            float x[NB][2][4] = {};
            uint32_t p[NB][2][2];
            waited &= bar_wait(smem_u32(&bars[warp][stage]), parity);
            const uint8_t *tile = my_ring + stage * kTileBytes;
            if (t < w.q.coded) {
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
                        for (int u = 0; u < 2; u++) {
                            uint32_t ka[4];
#pragma unroll
                            for (int n = 0; n < 2; n++) {
                                const uint4 &y = v[2 * u + n];
                                widen<KIND>(k == 0 ? y.x : k == 1 ? y.y : k == 2 ? y.z : y.w, ka[n], ka[2 + n]);
                            }
#pragma unroll
                            for (int nb = 0; nb < NB; nb++) mma(x[nb][u], ka, qb[nb][half * 4 + k][0], qb[nb][half * 4 + k][1]);
                        }
                }
                if (lone) {
#pragma unroll
                    for (int nb = 0; nb < NB; nb++)
#pragma unroll
                        for (int e = 0; e < 4; e++) x[nb][1][e] = -INFINITY;
                }
                weigh(x, a.scale * sc[0].x, lone ? 1.f : a.scale * sc[1].x);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    if (u == 1 && lone) continue;
                    const float f = unit_factor(sc[u].y);
#pragma unroll
                    for (int nb = 0; nb < NB; nb++) operand(p[nb], x[nb][u], f);
#pragma unroll
                    for (int n = 0; n < MT / 2; n++) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(tile + u * kUnit + 16 * HD + n * 512 + lane * 16);
                        uint32_t va[2][4];
                        widen<KIND>(v.x, va[0][0], va[0][2]);
                        widen<KIND>(v.y, va[0][1], va[0][3]);
                        widen<KIND>(v.z, va[1][0], va[1][2]);
                        widen<KIND>(v.w, va[1][1], va[1][3]);
#pragma unroll
                        for (int part = 0; part < 2; part++)
#pragma unroll
                            for (int j = 0; j < 2; j++)
#pragma unroll
                                for (int nb = 0; nb < NB; nb++) mma(o[nb][2 * n + j], va[j], p[nb][part][0], p[nb][part][1]);
                    }
                }
            } else {
                // up to 16 tokens in 16 bits, from the tail
                const int n_tok = min(kTailTile, w.q.len - w.q.full - (t - w.q.coded) * kTailTile);
#pragma unroll
                for (int half = 0; half < HALVES; half++) {
                    uint4 v[2][2];
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int j = 0; j < 2; j++) v[n][j] = *reinterpret_cast<const uint4 *>(tile + (8 * n + g) * (2 * HD) + half * 128 + c * 32 + j * 16);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint4 &y0 = v[0][k >> 1], &y1 = v[1][k >> 1];
                        const uint32_t ka[4] = {k & 1 ? y0.z : y0.x, k & 1 ? y1.z : y1.x, k & 1 ? y0.w : y0.y, k & 1 ? y1.w : y1.y};
#pragma unroll
                        for (int nb = 0; nb < NB; nb++) mma(x[nb][0], ka, qb[nb][half * 4 + k][0], qb[nb][half * 4 + k][1]);
                    }
                }
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if (8 * (e >> 1) + g >= n_tok) x[nb][0][e] = -INFINITY;          // (what lies there is no token)
                        x[nb][1][e] = -INFINITY;
                    }
                weigh(x, a.scale, 1.f);
                uint4 v[2][MT / 2];
                uint32_t top = 0;
#pragma unroll
                for (int hh = 0; hh < 2; hh++)
#pragma unroll
                    for (int n = 0; n < MT / 2; n++) {
                        // tokens 8hh + 2c and the next one, dims g * HD/8 + 4n ..; zeros where there is no token
                        const int tok = 8 * hh + 2 * c;
                        const uint32_t keep = tok + 1 < n_tok ? 0xFFFFFFFFu : tok < n_tok ? 0xFFFFu : 0u;
                        uint4 y = *reinterpret_cast<const uint4 *>(tile + kTileBytes / 2 + (4 * hh + c) * (4 * HD) + (g * (HD / 8) + 4 * n) * 4);
                        y.x &= keep; y.y &= keep; y.z &= keep; y.w &= keep;
                        v[hh][n] = y;
                        top = __vmaxu2(top, __vmaxu2(__vmaxu2(y.x & 0x7FFF7FFFu, y.y & 0x7FFF7FFFu), __vmaxu2(y.z & 0x7FFF7FFFu, y.w & 0x7FFF7FFFu)));
                    }
                // a power of two for the scale, so that small values keep their weights' digits: the exponent that covers all of them
                top = __reduce_max_sync(kFullMask, max(top & 0xFFFFu, top >> 16));
                const int e2 = top >= 0x7C00u ? 0 : max((int)(top >> 10), 1) - 15 - 6;
                const float up_by = exp2f((float)-e2);
                const float f = unit_factor(exp2f((float)e2));
#pragma unroll
                for (int nb = 0; nb < NB; nb++) operand(p[nb], x[nb][0], f);
                auto scaled = [&](uint32_t r) {
                    const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&r));
                    return pack(y.x * up_by, y.y * up_by);
                };
#pragma unroll
                for (int n = 0; n < MT / 2; n++) {
                    const uint32_t va[2][4] = {{scaled(v[0][n].x), scaled(v[0][n].y), scaled(v[1][n].x), scaled(v[1][n].y)},
                                               {scaled(v[0][n].z), scaled(v[0][n].w), scaled(v[1][n].z), scaled(v[1][n].w)}};
#pragma unroll
                    for (int part = 0; part < 2; part++)
#pragma unroll
                        for (int j = 0; j < 2; j++)
#pragma unroll
                            for (int nb = 0; nb < NB; nb++) mma(o[nb][2 * n + j], va[j], p[nb][part][0], p[nb][part][1]);
                }
            }
            __syncwarp();
            feed(stage);
            if (++stage == kStages) { stage = 0; parity ^= 1; }
        }

        // ---- the four warps' sums, half of the dims at a time
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                l[nb][e] += __shfl_xor_sync(kFullMask, l[nb][e], 4);
                l[nb][e] += __shfl_xor_sync(kFullMask, l[nb][e], 8);
                l[nb][e] += __shfl_xor_sync(kFullMask, l[nb][e], 16);
            }
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[nb][i][e] *= ref * (1.f / kLift);
        }
        const bool starts = w.t0 == 0, whole = starts && w.t1 == w.q.tiles;
        const int slot = 2 * blockIdx.x + (first ? 0 : 1);
        float fw[NB][2][kAttnWarps], inv[NB][2];
#pragma unroll
        for (int half = 0; half < 2; half++) {
            // all warps' values to shared memory, then each warp adds every fourth tile of dims
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
#pragma unroll
                for (int i = 0; i < MT / 2; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) join[(warp * kJoin + (nb * (MT / 2) + i) * 4 + e) * 32 + lane] = o[nb][half * (MT / 2) + i][e];
                if (half == 0 && g == 0) {
#pragma unroll
                    for (int e = 0; e < 2; e++) join_ml[warp * 8 * NB + 8 * nb + 2 * c + e] = make_float2(m[nb][e], l[nb][e]);
                }
            }
            __syncthreads();
            if (half == 0) {
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float2 y[kAttnWarps];
                        float mx = -INFINITY, sum = 0.f;
#pragma unroll
                        for (int v = 0; v < kAttnWarps; v++) { y[v] = join_ml[v * 8 * NB + 8 * nb + 2 * c + e]; mx = fmaxf(mx, y[v].x); }
                        const float at = mx == -INFINITY ? 0.f : mx;
#pragma unroll
                        for (int v = 0; v < kAttnWarps; v++) { fw[nb][e][v] = ex2(y[v].x - at); sum += y[v].y * fw[nb][e][v]; }
                        inv[nb][e] = whole ? 1.f / sum : 1.f;
                        if (!whole && warp == 0 && g == 0 && 8 * nb + 2 * c + e < rows) a.part_ml[slot * a.rows + 8 * nb + 2 * c + e] = make_float2(mx, sum);
                    }
            }
            for (int i = warp; i < MT / 2; i += kAttnWarps) {
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
                    float y[4] = {};
#pragma unroll
                    for (int v = 0; v < kAttnWarps; v++)
#pragma unroll
                        for (int e = 0; e < 4; e++) y[e] = fmaf(join[(v * kJoin + (nb * (MT / 2) + i) * 4 + e) * 32 + lane], fw[nb][e & 1][v], y[e]);
                    const int d = g * (HD / 8) + 2 * (half * (MT / 2) + i);
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int row = 8 * nb + 2 * c + e;
                        if (row >= rows) continue;
                        if (whole) *reinterpret_cast<uint32_t *>(a.out + (size_t)s * a.out_stride + (head0 + row) * HD + d) = pack(y[e] * inv[nb][e], y[2 + e] * inv[nb][e]);
                        else *reinterpret_cast<float2 *>(a.part_o + ((size_t)slot * a.rows + row) * HD + d) = make_float2(y[e], y[2 + e]);
                    }
                }
            }
            __syncthreads();
        }
        if (tid == 0 && starts) {
            // the CTAs from this one to the one that ends the pair
            int parts = 0;
            if (!whole) {
                const int begins = from + (length - w.left), end = begins + w.q.cost();
                int last = owner(end - 1);
                for (; last > (int)blockIdx.x; last--) {
                    const int x = border(last) - begins - kStart;      // its range begins inside this pair
                    if (x > kSnap && w.q.tiles - x > kSnap) break;
                }
                parts = last - (int)blockIdx.x + 1;
            }
            a.meta[s * pairs + w.i] = make_int2(slot, parts);
        }
        first = false;
        w.left -= count(w);
        if (w.left <= 0) break;
        next_pair(w);
        bound(w);
    }
    if (!waited) {                       // a copy did not arrive in time: report, and leave only when none is in flight
        if (a.status && lane == 0) atomicOr(a.status, (unsigned)kStatusWait);
        for (int k = 0; k < kStages; k++) {
            bar_wait(smem_u32(&bars[warp][k]), 0);
            bar_wait(smem_u32(&bars[warp][k]), 1);
        }
    }
}

// One CTA per query head and sequence: joins the parts of its pair, a warp every eighth part.  The weights of the parts come first, so that
// the loads of their sums do not wait for one another.
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32;

template <int HD>
__global__ void __launch_bounds__(kJoinThreads) attn_join_kernel(const AttnArgs a) {
    constexpr int E = HD / 32;
    __shared__ float s_o[kJoinWarps][HD], s_w[kJoinThreads], s_red[2][kJoinWarps];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int rep = a.n_heads / a.n_kv, head = blockIdx.x, in = head % rep, pair = (head / rep) * a.groups + in / kRowsMax, row = in % kRowsMax;
    const int2 meta = a.meta[blockIdx.y * a.n_kv * a.groups + pair];
    if (meta.y == 0) return;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    auto slot = [&](int k) { return (size_t)(k == 0 ? meta.x : 2 * (meta.x / 2 + k)) * a.rows + row; };
    float m = -INFINITY, l = 0.f, o[E] = {};
    for (int k0 = 0; k0 < meta.y; k0 += kJoinThreads) {
        const float2 ml = k0 + tid < meta.y ? a.part_ml[slot(k0 + tid)] : make_float2(-INFINITY, 0.f);
        float mx = ml.x;
#pragma unroll
        for (int o2 = 16; o2 > 0; o2 >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kFullMask, mx, o2));
        __syncthreads();
        if (lane == 0) s_red[0][warp] = mx;
        __syncthreads();
        mx = m;
#pragma unroll
        for (int w = 0; w < kJoinWarps; w++) mx = fmaxf(mx, s_red[0][w]);
        const float at = mx == -INFINITY ? 0.f : mx, fix = ex2(m - at), weight = ex2(ml.x - at);
        m = mx;
        s_w[tid] = weight;
        float sum = ml.y * weight;
#pragma unroll
        for (int o2 = 16; o2 > 0; o2 >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o2);
        if (lane == 0) s_red[1][warp] = sum;
        __syncthreads();
        l *= fix;
#pragma unroll
        for (int w = 0; w < kJoinWarps; w++) l += s_red[1][w];
#pragma unroll
        for (int e = 0; e < E; e++) o[e] *= fix;
#pragma unroll 8
        for (int k = warp; k < min(kJoinThreads, meta.y - k0); k += kJoinWarps) {
            const float *from = a.part_o + slot(k0 + k) * HD + lane * E;
            float v[E];
            if constexpr (E == 4) *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(from);
            else *reinterpret_cast<float2 *>(v) = *reinterpret_cast<const float2 *>(from);
#pragma unroll
            for (int e = 0; e < E; e++) o[e] = fmaf(v[e], s_w[k], o[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < E; e++) s_o[warp][lane * E + e] = o[e];
    __syncthreads();
    if (tid < HD) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; w++) v += s_o[w][tid];
        a.out[(size_t)blockIdx.y * a.out_stride + head * HD + tid] = __float2half_rn(v / l);
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
    w.ctas = kWaves * sm_count() * (w.rows > 8 ? AttnShape<128, 2>::kCtas : AttnShape<128, 1>::kCtas);
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
    const int most = (int)(((long)max_blocks * block + kTile - 1) / kTile) + block / kTailTile;                // tiles of a pair
    if ((long)(most + kStart) * n_seqs * n_kv_heads * ws.groups > 0x3FFFFFFFl) return QTIP_ERR_TOO_LARGE;          // tiles are counted in 32 bits
    if (!workspace || workspace_bytes < ws.bytes) return QTIP_ERR_WORKSPACE;
    const void *ptrs[] = {out, q, data, scales, tail_k, tail_v, workspace};
    for (const void *p : ptrs)
        if (!aligned(p, 16)) return QTIP_ERR_ALIGNMENT;
    if (!aligned(tables, 4) || !aligned(lengths, 4) || !aligned(status, 4)) return QTIP_ERR_ALIGNMENT;
    if ((out_stride | q_stride | tail_k_stride | tail_v_stride) & 7) return QTIP_ERR_ALIGNMENT;
    if (n_seqs > 1 && out_stride < (long)n_heads * head_dim) return QTIP_ERR_BAD_SHAPE;               // rows that are written share no memory
    uint8_t *w = static_cast<uint8_t *>(workspace);
    const AttnArgs a = {static_cast<__half *>(out), static_cast<const __half *>(q), out_stride, q_stride, static_cast<const uint8_t *>(data),
                        reinterpret_cast<const float4 *>(scales), static_cast<const __half *>(tail_k), static_cast<const __half *>(tail_v), tail_k_stride,
                        tail_v_stride, tables, lengths, n_seqs, n_heads, n_kv_heads, max_blocks, n_blocks, block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7,
                        1.4426950408889634f / sqrtf((float)head_dim), reinterpret_cast<float *>(w + ws.o), reinterpret_cast<float2 *>(w + ws.ml),
                        reinterpret_cast<int2 *>(w + ws.meta), ws.groups, ws.rows, status};
    auto pick = [&](auto hd, auto nb) {
        constexpr int HD = decltype(hd)::value, NB = decltype(nb)::value;
        return std::make_pair(kind == kKvInt8 ? attn_paged_kernel<HD, kKvInt8, NB> : attn_paged_kernel<HD, kKvE4m3, NB>, AttnShape<HD, NB>::kSmem);
    };
    using std::integral_constant;
    const auto [kernel, smem] = head_dim == 128 ? (ws.rows > 8 ? pick(integral_constant<int, 128>(), integral_constant<int, 2>()) : pick(integral_constant<int, 128>(), integral_constant<int, 1>()))
                                                : (ws.rows > 8 ? pick(integral_constant<int, 64>(), integral_constant<int, 2>()) : pick(integral_constant<int, 64>(), integral_constant<int, 1>()));
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
    if (most > 2 * kSnap) {
        cfg.gridDim = dim3(n_heads, n_seqs);
        cfg.blockDim = dim3(kJoinThreads);
        cfg.dynamicSmemBytes = 0;
        QTIP_CUDA_TRY(cudaLaunchKernelEx(&cfg, head_dim == 128 ? attn_join_kernel<128> : attn_join_kernel<64>, a));
    }
    return check_launch();
}
