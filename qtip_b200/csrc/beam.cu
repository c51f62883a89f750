// Beam search: the selection of each group's best continuations, and the reordering of what belongs to a beam (caches, block tables,
// token logs).  They stand where the decode loop samples (eval/interactive_gen.py:15-40 upstream).
#include <atomic>

#include "common.cuh"

namespace qtip {
namespace {

constexpr int kMaxBeams = 16, kMaxStates = 8;

// ---- selection -------------------------------------------------------------------------------------------------------------------
// A group's beams w < W with scores c_w and logits x_w: the W largest of c_w + (x_wv - lse_w), lse_w = log sum_v exp x_wv.
// One cluster per group; its warps share the rows.  A warp reads its slice once, in batches of 24 logits per lane that are copied to shared memory
// one batch ahead: the sum of exponentials with a running maximum in each lane, and the W largest logits, sorted in its lanes.  A batch without
// a logit above the last of these costs one comparison; in the first batch the W-th largest of the lanes' largest is the bound.  CTA 0
// merges the lists of a row, one warp per row, adds scores in 64 bits and takes the W largest of the W * W continuations that are left.
constexpr int kSelectThreads = 256, kSelectCluster = 16, kSelectWarps = kSelectThreads / 32 * kSelectCluster, kSelectHeld = 24, kSelectStages = 2;

struct SelectArgs {
    long long *tokens;
    int *parents;
    float *scores;
    const void *logits;
    long stride;
    const float *prev_scores;
    const long long *prev_tokens;
    int width, vocab;
    long long eos;
    unsigned *status;
};

struct SelectSmem {
    unsigned long long keys[kSelectWarps * kMaxBeams];       // (row, warp of the row, rank)
    float2 sums[kSelectWarps];                               // (row, warp of the row): unit, sum of exponentials
    unsigned long long total[kMaxBeams * kMaxBeams];         // ordered bits of the continuations' scores; 0: none
    int token[kMaxBeams * kMaxBeams];
};

// Order of floats (doubles) as unsigned integers; 0 is below every number.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);             // -0 and 0 are equal
    return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u ^ ((u >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }
__device__ __forceinline__ unsigned long long ordered(double x) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(x + 0.0);
    return u ^ ((u >> 63) ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double unordered(unsigned long long u) { return __longlong_as_double((long long)(u ^ ((u >> 63) ? 1ull << 63 : ~0ull))); }

__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
    const uint32_t hi = __reduce_max_sync(kFullMask, (uint32_t)(v >> 32));
    const uint32_t lo = __reduce_max_sync(kFullMask, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
    return (unsigned long long)hi << 32 | lo;
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }

// exp(x - unit): the difference first (exact for what matters), so that logits of any size keep their distances.
constexpr float kLog2e = 1.44269502162933349609375f, kSumTop = 4294967296.f;

// A warp's batch in shared memory: vector j of lane l holds logits base + (j * 32 + l) * N + k; -inf behind the end of the slice.  A lane reads what
// it copied itself.
template <typename T>
struct Batch {
    static constexpr int N = 16 / sizeof(T), V = kSelectHeld / N, kSize = 32 * kSelectHeld;
    uint4 v[V][32];
    __device__ __forceinline__ void load(const T *row, int base, int end, int lane, bool vectors) {
        if (vectors && base + kSize <= end) copy<true>(row, base, end, lane, true);
        else copy<false>(row, base, end, lane, vectors);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    template <bool whole>
    __device__ __forceinline__ void copy(const T *row, int base, int end, int lane, bool vectors) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int at = base + (j * 32 + lane) * N;
            if (vectors && (whole || at + N <= end)) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(&v[j][lane])), "l"(row + at) : "memory");
            } else {
                T *e = reinterpret_cast<T *>(&v[j][lane]);
#pragma unroll
                for (int k = 0; k < N; k++) e[k] = at + k < end ? row[at + k] : T(-INFINITY);
            }
        }
    }
    __device__ __forceinline__ void values(float (&x)[N], int j, int lane) const {
        const uint4 raw = v[j][lane];
#pragma unroll
        for (int k = 0; k < N; k++) x[k] = to_f(reinterpret_cast<const T *>(&raw)[k]);
    }
    __device__ __forceinline__ float value(int i, int lane) const { return to_f(reinterpret_cast<const T *>(&v[i / N][lane])[i % N]); }
    __device__ __forceinline__ float largest(int lane) const {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < V; j++) {
            float x[N];
            values(x, j, lane);
#pragma unroll
            for (int k = 0; k < N; k++) top = fmaxf(top, x[k]);
        }
        return top;
    }
    // Sum of exp(x - unit), and the largest.
    __device__ __forceinline__ float sum(float unit, float &top, int lane) const {
        float s[4] = {}, t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < V; j++) {
            float x[N];
            values(x, j, lane);
#pragma unroll
            for (int k = 0; k < N; k++) {
                float e;
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((x[k] - unit) * kLog2e));
                s[k & 3] += e;
                t[k & 3] = fmaxf(t[k & 3], x[k]);
            }
        }
        top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
        return (s[0] + s[1]) + (s[2] + s[3]);
    }
    __device__ __forceinline__ void only_finite(int lane) {
        for (int j = 0; j < V; j++)
            for (int k = 0; k < N; k++) {
                T *e = reinterpret_cast<T *>(&v[j][lane]) + k;
                if (!isfinite(to_f(*e))) *e = T(-INFINITY);
            }
    }
};

template <typename T>
__global__ void __launch_bounds__(kSelectThreads, 4) beam_select_kernel(const SelectArgs a) {
    extern __shared__ __align__(16) uint8_t select_smem[];
    SelectSmem &S = *reinterpret_cast<SelectSmem *>(select_smem);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = a.width, g = blockIdx.y;
    Batch<T> *ring = reinterpret_cast<Batch<T> *>(select_smem) + warp * kSelectStages;
    uint32_t rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int per = (int)gridDim.x * (kSelectThreads / 32) / W, id = (int)rank * (kSelectThreads / 32) + warp, w = id / per, part = id % per;
    unsigned long long list = 0;                             // lane i < W: the i-th largest (logit, ~index)
    float unit = -INFINITY, sum = 0.f;
    if (w < W) {
        const size_t beam = (size_t)g * W + w;
        const T *row = static_cast<const T *>(a.logits) + beam * (size_t)a.stride;
        const bool dead = !isfinite(a.prev_scores[beam]) || (a.eos >= 0 && a.prev_tokens && a.prev_tokens[beam] == a.eos);
        const bool vectors = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
        const int slice = ((a.vocab + per - 1) / per + 7) & ~7;
        const long long lo = (long long)part * slice;
        const int end = (int)min((long long)a.vocab, lo + slice);
        int stage = 0;
        if (lo < end && !dead) ring[0].load(row, (int)lo, end, lane, vectors);
        for (long long at = lo; at < end && !dead; at += Batch<T>::kSize) {
            Batch<T> &x = ring[stage];
            stage ^= 1;
            if (at + Batch<T>::kSize < end) {                          // in flight during this one
                ring[stage].load(row, (int)at + Batch<T>::kSize, end, lane, vectors);
                asm volatile("cp.async.wait_group 1;" ::: "memory");
            } else {
                asm volatile("cp.async.wait_group 0;" ::: "memory");
            }
            // A lane's unit is the largest logit of its first batch, until a batch's sum in that unit is above kSumTop (a logit some 20 above it), which
            // raises it.  So a lane adds at most 2^21 batches of at most 2^32, 32 lanes 2^58: no sum leaves fp32.
            float top;
            if (__any_sync(kFullMask, unit == -INFINITY)) {
                top = x.largest(lane);
                if (unit == -INFINITY && fabsf(top) < INFINITY) unit = top;
            }
            float more = x.sum(unit == -INFINITY ? 0.f : unit, top, lane);
            if (__any_sync(kFullMask, !(more <= kSumTop))) {           // a change of the unit, or an infinity or NaN, which do not count
                x.only_finite(lane);
                top = x.largest(lane);
                const float old = unit;
                unit = fmaxf(unit, top);
                if (old > -INFINITY) sum *= exp2f((old - unit) * kLog2e);
                more = x.sum(unit == -INFINITY ? 0.f : unit, top, lane);
            }
            sum += more;
            // what can enter the list: not below its last entry; in the first batch not below the W-th largest of the lanes' largest
            uint32_t bound = (uint32_t)(__shfl_sync(kFullMask, list, W - 1) >> 32);
            if (bound == 0u) {
                uint32_t mine = top > -INFINITY ? ordered(top) : 0u;
                for (int r = 0; r < W; r++) {
                    bound = __reduce_max_sync(kFullMask, mine);
                    const unsigned who = __ballot_sync(kFullMask, mine == bound);
                    if (lane == __ffs(who) - 1) mine = 0u;
                }
            }
            const float least = bound ? unordered(bound) : -INFINITY;
            if (!__any_sync(kFullMask, top >= least && top > -INFINITY)) continue;
            unsigned open = 0;
            if (top >= least) {
#pragma unroll
                for (int j = 0; j < Batch<T>::V; j++) {
                    float y[Batch<T>::N];
                    x.values(y, j, lane);
#pragma unroll
                    for (int k = 0; k < Batch<T>::N; k++) open |= y[k] >= least && y[k] > -INFINITY ? 1u << (j * Batch<T>::N + k) : 0u;
                }
            }
            __syncwarp();
            while (__any_sync(kFullMask, open != 0u)) {
                // every lane's next one, then one lane after the other
                const int j = open ? __ffs(open) - 1 : 0;
                const uint32_t idx = (uint32_t)((int)at + ((j / Batch<T>::N) * 32 + lane) * Batch<T>::N + j % Batch<T>::N);
                const unsigned long long key = open ? (unsigned long long)ordered(x.value(j, lane)) << 32 | (0xFFFFFFFFu - idx) : 0ull;
                open &= open - 1;
                unsigned long long last = __shfl_sync(kFullMask, list, W - 1);
                unsigned who = __ballot_sync(kFullMask, key > last);
                while (who) {
                    const int src = __ffs(who) - 1;
                    const unsigned long long k = __shfl_sync(kFullMask, key, src), before = __shfl_up_sync(kFullMask, list, 1);
                    if (k > list) list = lane == 0 || before > k ? k : before;
                    last = __shfl_sync(kFullMask, list, W - 1);
                    who = __ballot_sync(kFullMask, key > last) & who & (who - 1);
                }
            }
        }
        // the lanes' sums
        float all = unit;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor_sync(kFullMask, all, o));
        sum = unit > -INFINITY ? sum * exp2f((unit - all) * kLog2e) : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
        unit = all;
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");      // the lists take the place of the batches
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (w < W) {
        uint32_t to;
        if (lane < W) {
            asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"((uint32_t)__cvta_generic_to_shared(&S.keys[id * W + lane])));
            asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(list) : "memory");
        }
        if (lane == 0) {
            asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"((uint32_t)__cvta_generic_to_shared(&S.sums[id])));
            asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(unit), "f"(sum) : "memory");
        }
    }
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
    if (rank != 0) return;
    for (int row = warp; row < W; row += kSelectThreads / 32) {
        const size_t beam = (size_t)g * W + row;
        const float score = a.prev_scores[beam];
        const bool active = isfinite(score), ended = a.eos >= 0 && a.prev_tokens && a.prev_tokens[beam] == a.eos;
        // log of the row's sum: terms of 32 bits, added in 64
        float mx = -INFINITY;
        for (int i = lane; i < per; i += 32) mx = fmaxf(mx, S.sums[row * per + i].x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kFullMask, mx, o));
        double s = 0.0;
        for (int i = lane; i < per; i += 32) {
            const float2 v = S.sums[row * per + i];
            if (v.y > 0.f) s += (double)v.y * (double)exp2f((v.x - mx) * kLog2e);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFullMask, s, o);
        const double lse = (double)(float)((double)mx + log(s));
        unsigned long long k[kSelectWarps / 32];
#pragma unroll
        for (int e = 0; e < kSelectWarps / 32; e++) {
            const int i = lane + 32 * e;
            k[e] = i < per * W ? S.keys[row * per * W + i] : 0ull;
        }
        for (int r = 0; r < W; r++) {
            unsigned long long best = k[0];
#pragma unroll
            for (int e = 1; e < kSelectWarps / 32; e++) best = max(best, k[e]);
            best = warp_max(best);
#pragma unroll
            for (int e = 0; e < kSelectWarps / 32; e++)
                if (k[e] == best) k[e] = 0ull;
            if (lane == 0) {
                unsigned long long total = 0ull;
                int token = (int)(0xFFFFFFFFu - (uint32_t)best);
                if (active && ended) {
                    if (r == 0) total = ordered((double)score);
                    token = -1;
                } else if (active && best != 0ull) {
                    total = ordered((double)score + ((double)unordered((uint32_t)(best >> 32)) - lse));
                }
                S.total[row * W + r] = total;
                S.token[row * W + r] = token;
            }
        }
    }
    __syncthreads();
    if (warp != 0) return;
    // the W largest; equal ones in the order of beams, then of ranks
    unsigned long long t[kMaxBeams * kMaxBeams / 32], mine = 0ull;
    int at = -1;
#pragma unroll
    for (int e = 0; e < kMaxBeams * kMaxBeams / 32; e++) t[e] = lane + 32 * e < W * W ? S.total[lane + 32 * e] : 0ull;
    for (int r = 0; r < W; r++) {
        unsigned long long best = t[0];
#pragma unroll
        for (int e = 1; e < kMaxBeams * kMaxBeams / 32; e++) best = max(best, t[e]);
        best = warp_max(best);
        if (best == 0ull) break;
        uint32_t where = 0xFFFFFFFFu;
#pragma unroll
        for (int e = kMaxBeams * kMaxBeams / 32 - 1; e >= 0; e--)
            if (t[e] == best) where = lane + 32 * e;
        where = __reduce_min_sync(kFullMask, where);
#pragma unroll
        for (int e = 0; e < kMaxBeams * kMaxBeams / 32; e++)
            if (lane + 32 * e == (int)where) t[e] = 0ull;
        if (lane == r) { at = (int)where; mine = best; }
    }
    // the best continuation of a parent stays in its row, the others fill the rows left, in order
    const int parent = at >= 0 ? at / W : -1 - lane;
    const unsigned same = __match_any_sync(kFullMask, parent);
    const bool stays = at >= 0 && __ffs(same) - 1 == lane, moves = lane < W && !stays;
    const unsigned taken = __reduce_or_sync(kFullMask, stays ? 1u << parent : 0u), moving = __ballot_sync(kFullMask, moves);
    if (lane < W) {
        const int to = stays ? parent : (int)__fns(~taken, 0, __popc(moving & ((1u << lane) - 1)) + 1);
        const size_t out = (size_t)g * W + to;
        const int token = at >= 0 ? S.token[at] : -1;
        a.tokens[out] = token >= 0 ? token : max(a.eos, 0ll);
        a.parents[out] = at >= 0 ? parent : to;
        a.scores[out] = at >= 0 ? (float)unordered(mine) : -INFINITY;
    }
    if (lane == 0 && at < 0 && a.status) atomicOr(a.status, 2u);
}

// ---- reordering ------------------------------------------------------------------------------------------------------------------
// Row b of a group becomes a copy of row parents[b].  Rows that stay are not touched.  Bound by the bytes of the rows that are copied.
// A thread owns columns of the group's rows and makes all copies of them in an order in which no row is read after it was written: where no
// row that is copied from is itself replaced (beam_select's parents), any order, with several loads in flight; else rows that nobody
// needs any more first, and then what is left, cycles, through a register.
struct ReorderState {
    uint8_t *base;
    long seq_stride, outer_stride;       // bytes
    int outer, row_bytes, rows, per_row, mod;
    int first;                           // first CTA of this state
    int wide;                            // columns of 16 bytes, else of 4
};
struct ReorderArgs {
    ReorderState state[kMaxStates];
    const int *parents, *lengths;
    int n_states, width;
    unsigned *status;
};

constexpr int kReorderThreads = 256, kReorderColumns = 4;

struct Moves {
    int n;                               // steps
    int ordered;                         // they have to be made one after another
    int to[2 * kMaxBeams], from[2 * kMaxBeams];      // rows; to -1: into the register, from -1: out of it
    int bytes[2 * kMaxBeams];            // of a piece, from its start
};

// One thread; rarely needed.
__device__ __noinline__ void order_moves(Moves &m, const int *parent, const int *bytes, int width) {
    unsigned left = 0;
    for (int b = 0; b < width; b++)
        if (parent[b] != b) left |= 1u << b;
    int n = 0;
    while (left) {
        int pick = -1;
        for (int b = 0; b < width && pick < 0; b++) {
            if (!(left >> b & 1)) continue;
            bool needed = false;
            for (int o = 0; o < width; o++) needed |= (left >> o & 1) && parent[o] == b;
            if (!needed) pick = b;
        }
        if (pick >= 0) {
            m.to[n] = pick; m.from[n] = parent[pick]; m.bytes[n++] = bytes[pick];
            left &= ~(1u << pick);
            continue;
        }
        // a cycle: its first row is kept, each row takes its parent's, the last the kept one
        const int start = __ffs(left) - 1;
        m.to[n] = -1; m.from[n] = start; m.bytes[n++] = 0x7FFFFFFF;
        for (int b = start;;) {
            const int p = parent[b];
            m.to[n] = b; m.from[n] = p == start ? -1 : p; m.bytes[n++] = bytes[b];
            left &= ~(1u << b);
            if (p == start) break;
            b = p;
        }
    }
    m.n = n;
}

template <typename V>
__device__ __forceinline__ void copy_columns(const ReorderState &s, const Moves &m, uint8_t *base, int per_outer, int total, int cta, int ctas) {
    constexpr int kBytes = sizeof(V), U = kReorderColumns;
    const int stride = ctas * kReorderThreads;
    for (int i0 = cta * kReorderThreads + threadIdx.x; i0 < total; i0 += U * stride) {
        uint8_t *col[U];
        int at[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const unsigned i = (unsigned)i0 + (unsigned)u * stride, o = i / (unsigned)per_outer;
            at[u] = i < (unsigned)total ? (int)((i - o * per_outer) * kBytes) : 0x7FFFFFFF - 16;      // behind every row
            col[u] = base + (long)o * s.outer_stride + (i - o * per_outer) * kBytes;
        }
        if (!m.ordered) {
            for (int k = 0; k < m.n; k++) {
                const long to = m.to[k] * s.seq_stride, from = m.from[k] * s.seq_stride;
                const int bytes = m.bytes[k];
                V v[U];
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (at[u] + kBytes <= bytes) v[u] = __ldcs(reinterpret_cast<const V *>(col[u] + from));
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (at[u] + kBytes <= bytes) *reinterpret_cast<V *>(col[u] + to) = v[u];
                if constexpr (kBytes > 4) {          // a row that ends inside the column
#pragma unroll
                    for (int u = 0; u < U; u++)
                        for (int j = 0; at[u] < bytes && at[u] + kBytes > bytes && at[u] + j < bytes; j += 4)
                            *reinterpret_cast<uint32_t *>(col[u] + to + j) = *reinterpret_cast<const uint32_t *>(col[u] + from + j);
                }
            }
        } else {
            for (int u = 0; u < U; u++) {
                if (i0 + (long)u * stride >= total) break;
                for (int j = 0; j < kBytes; j += 4) {
                    uint32_t kept = 0;
                    for (int k = 0; k < m.n; k++) {
                        if (at[u] + j >= m.bytes[k] || at[u] + j >= s.rows * s.row_bytes) continue;
                        volatile uint32_t *to = reinterpret_cast<uint32_t *>(col[u] + j + max(m.to[k], 0) * s.seq_stride);
                        const volatile uint32_t *from = reinterpret_cast<const uint32_t *>(col[u] + j + max(m.from[k], 0) * s.seq_stride);
                        if (m.to[k] < 0) kept = *from;
                        else *to = m.from[k] < 0 ? kept : *from;
                    }
                }
            }
        }
    }
}

__global__ void __launch_bounds__(kReorderThreads) beam_reorder_kernel(const ReorderArgs a) {
    __shared__ Moves m;
    __shared__ int s_parent[kMaxBeams], s_bytes[kMaxBeams], s_most;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int g = blockIdx.y, lane = threadIdx.x & 31;
    int k = 0;
    while (k + 1 < a.n_states && (int)blockIdx.x >= a.state[k + 1].first) k++;
    const ReorderState s = a.state[k];
    if (threadIdx.x < 32) {
        int parent = lane, bytes = 0;
        bool bad = false;
        if (lane < a.width) {
            const int p = a.parents[g * a.width + lane];
            bad = (unsigned)p >= (unsigned)a.width;
            if (!bad) parent = p;
            int n = s.rows;
            if (parent != lane && a.lengths) {
                n = max(a.lengths[g * a.width + parent], 0);
                if (s.mod) n %= s.mod;
                n = min(n / s.per_row + (n % s.per_row != 0), s.rows);
            }
            if (parent == lane) n = 0;
            bytes = n * s.row_bytes;
            s_parent[lane] = parent;
            s_bytes[lane] = bytes;
        }
        if (__any_sync(kFullMask, bad) && a.status && lane == 0) atomicOr(a.status, 32u);
        const bool moves = parent != lane && bytes > 0;
        const unsigned moving = __ballot_sync(kFullMask, moves), sources = __reduce_or_sync(kFullMask, parent != lane ? 1u << parent : 0u);
        const bool hazard = __any_sync(kFullMask, parent != lane && (sources >> lane & 1));
        if (moves) {
            const int at = __popc(moving & ((1u << lane) - 1));
            m.to[at] = lane; m.from[at] = parent; m.bytes[at] = bytes;
        }
        const int most = __reduce_max_sync(kFullMask, bytes);
        __syncwarp();
        if (lane == 0) {
            m.n = __popc(moving);
            m.ordered = hazard;
            s_most = most;
            if (hazard) order_moves(m, s_parent, s_bytes, a.width);
        }
    }
    __syncthreads();
    const int ctas = (k + 1 < a.n_states ? a.state[k + 1].first : (int)gridDim.x) - s.first, cta = blockIdx.x - s.first;
    const int vec = s.wide ? 16 : 4, per_outer = (s_most + vec - 1) / vec;
    if (per_outer == 0) return;
    uint8_t *base = s.base + (long)g * a.width * s.seq_stride;
    if (s.wide) copy_columns<uint4>(s, m, base, per_outer, per_outer * s.outer, cta, ctas);
    else copy_columns<uint32_t>(s, m, base, per_outer, per_outer * s.outer, cta, ctas);
}

template <typename T>
constexpr size_t select_smem_bytes() {
    constexpr size_t ring = (size_t)kSelectThreads / 32 * kSelectStages * sizeof(Batch<T>);
    return ring > sizeof(SelectSmem) ? ring : sizeof(SelectSmem);
}

// CTAs of a group: as many as the chip holds at once for all groups; more would be a second round.  64 groups of 8 beams over 128256 tokens take
// 74 us with 4 and 60 with 8; one group 28 us with 8 and 21 with 16 (where the GPU has room for clusters of 16).
template <typename T>
int launch_select(const SelectArgs &a, int groups, cudaStream_t stream) {
    // clusters of 1, 2, 4, 8, 16 CTAs at once, plus one; filled by whichever thread comes first, after it has set what a launch of that size needs
    static std::atomic<int> cached[64][5] = {};
    int dev = 0, cluster = 0;
    QTIP_CUDA_TRY(cudaGetDevice(&dev));
    QTIP_CUDA_TRY(cudaFuncSetAttribute(beam_select_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)select_smem_bytes<T>()));
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kSelectThreads);
    cfg.dynamicSmemBytes = select_smem_bytes<T>();
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    double best = 0;
    for (int k = 0; k < 5; k++) {
        const int c = 1 << k, per = c * (kSelectThreads / 32) / a.width;                   // warps of a row
        if (per == 0) continue;
        int n = dev < 64 ? cached[dev][k].load(std::memory_order_acquire) - 1 : -1;
        if (n < 0) {
            cfg.gridDim = dim3(c);
            cfg.numAttrs = 1;
            attr[0].val.clusterDim.x = c;
            if ((c == 16 && cudaFuncSetAttribute(beam_select_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) ||
                cudaOccupancyMaxActiveClusters(&n, beam_select_kernel<T>, &cfg) != cudaSuccess) {
                (void)cudaGetLastError();
                n = 0;
            }
            if (dev < 64) cached[dev][k].store(n + 1, std::memory_order_release);
        }
        if (c == 16 && n < groups) continue;
        const double time = n ? (double)((groups + n - 1) / n) / per : 1e30;               // rounds, each as long as a warp's part of a row
        if (!cluster || time < best) { cluster = c; best = time; }
    }
    cfg.gridDim = dim3(cluster, groups);
    cfg.numAttrs = 2;
    attr[0].val.clusterDim.x = cluster;
    QTIP_CUDA_TRY(cudaLaunchKernelEx(&cfg, beam_select_kernel<T>, a));
    return check_launch();
}

}  // namespace
}  // namespace qtip

using namespace qtip;

extern "C" int qtip_beam_select(long long *tokens, int *parents, float *scores, const void *logits, int logits_dtype, long logits_stride,
                                const float *prev_scores, const long long *prev_tokens, int groups, int width, int vocab, long long eos, unsigned *status,
                                void *stream) {
    if (!tokens || !parents || !scores || !logits || !prev_scores || (logits_dtype != QTIP_F16 && logits_dtype != QTIP_F32) || (eos >= 0 && !prev_tokens))
        return QTIP_ERR_BAD_ARG;
    if (groups < 1 || groups > 65535 || width < 1 || width > kMaxBeams || vocab < 1 || vocab > (1 << 30) || logits_stride < vocab) return QTIP_ERR_BAD_SHAPE;
    if (!aligned(tokens, 8) || (prev_tokens && !aligned(prev_tokens, 8)) || !aligned(parents, 4) || !aligned(scores, 4) || !aligned(prev_scores, 4) ||
        !aligned(status, 4) || !aligned(logits, logits_dtype == QTIP_F32 ? 4 : 2))
        return QTIP_ERR_ALIGNMENT;
    const SelectArgs a = {tokens, parents, scores, logits, logits_stride, prev_scores, prev_tokens, width, vocab, eos, status};
    return logits_dtype == QTIP_F32 ? launch_select<float>(a, groups, static_cast<cudaStream_t>(stream))
                                    : launch_select<__half>(a, groups, static_cast<cudaStream_t>(stream));
}

extern "C" int qtip_beam_reorder(const qtip_beam_state *states, int n_states, const int *parents, const int *lengths, int groups, int width,
                                 unsigned *status, void *stream) {
    if (!states || !parents || n_states < 1 || n_states > kMaxStates) return QTIP_ERR_BAD_ARG;
    if (groups < 1 || groups > 65535 || width < 1 || width > kMaxBeams) return QTIP_ERR_BAD_SHAPE;
    if (!aligned(parents, 4) || (lengths && !aligned(lengths, 4)) || !aligned(status, 4)) return QTIP_ERR_ALIGNMENT;
    ReorderArgs a = {};
    a.parents = parents;
    a.lengths = lengths;
    a.n_states = n_states;
    a.width = width;
    a.status = status;
    int ctas = 0;
    for (int k = 0; k < n_states; k++) {
        const qtip_beam_state &s = states[k];
        if (!s.base) return QTIP_ERR_BAD_ARG;
        for (int j = 0; j < k; j++)
            if (states[j].base == s.base) return QTIP_ERR_BAD_ARG;              // it would be reordered twice
        if (s.outer < 1 || s.rows < 1 || s.row_bytes < 4 || s.per_row < 1 || s.mod < 0 || (s.row_bytes & 3) || (s.seq_stride & 3) || (s.outer_stride & 3) ||
            (long)s.rows * s.row_bytes > s.seq_stride || (s.outer > 1 && ((long)s.rows * s.row_bytes > s.outer_stride || (s.outer - 1) * s.outer_stride + (long)s.rows * s.row_bytes > s.seq_stride)))
            return QTIP_ERR_BAD_SHAPE;
        if (!aligned(s.base, 4)) return QTIP_ERR_ALIGNMENT;
        const bool wide = aligned(s.base, 16) && !(s.seq_stride & 15) && (s.outer == 1 || !(s.outer_stride & 15));
        const long piece = (long)s.rows * s.row_bytes, units = (piece + (wide ? 15 : 3)) / (wide ? 16 : 4) * s.outer;
        if (piece > 0x3FFFFFFF || units > 0x3FFFFFFF) return QTIP_ERR_TOO_LARGE;        // columns and bytes of a piece are counted in 32 bits
        a.state[k] = {static_cast<uint8_t *>(s.base), s.seq_stride, s.outer_stride, s.outer, s.row_bytes, s.rows, s.per_row, s.mod, ctas, wide};
        const long want = (units + kReorderThreads * kReorderColumns - 1) / (kReorderThreads * kReorderColumns), most = (long)sm_count() * 8;
        ctas += (int)(want < most ? want : most);
    }
    if (width == 1) return QTIP_OK;
    // every CTA reads these while others copy
    const uintptr_t ints = 4u * (uintptr_t)groups * width;
    for (int k = 0; k < n_states; k++) {
        const qtip_beam_state &s = states[k];
        const uintptr_t lo = reinterpret_cast<uintptr_t>(s.base),
                        hi = lo + ((uintptr_t)groups * width - 1) * s.seq_stride + (uintptr_t)(s.outer - 1) * s.outer_stride + (uintptr_t)s.rows * s.row_bytes;
        for (const int *p : {parents, lengths})
            if (p && reinterpret_cast<uintptr_t>(p) < hi && lo < reinterpret_cast<uintptr_t>(p) + ints) return QTIP_ERR_BAD_ARG;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, groups);
    cfg.blockDim = dim3(kReorderThreads);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    QTIP_CUDA_TRY(cudaLaunchKernelEx(&cfg, beam_reorder_kernel, a));
    return check_launch();
}
