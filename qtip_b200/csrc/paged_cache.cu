// Writers of the key/value cache in 8 bits (paged.cuh): block tables and runs of new tokens from the sequences' lengths, and the rotary
// embedding with the append of new tokens.  They stand where the decode loop has StaticCache.update (model/cache_utils.py:1147-1193
// upstream) and apply_rotary_pos_emb (model/llama.py:797-898).
#include <cuda_fp8.h>

#include "paged.cuh"

namespace qtip {
namespace {

// ---- block tables and runs -------------------------------------------------------------------------------------------------------
// A block is free when no sequence's table names it among its complete blocks (a bitmap in shared memory): there is no free
// list to keep, a sequence whose length is set to zero has released its blocks, and tables that name the same block (beams of one
// search, a common prompt) share it.  The new blocks are the lowest free ones, in the order of the sequences.
// One CTA; for many table entries a cluster of eight, each of which marks every eighth share of 32 sequences in a bitmap of its own, which the first
// then takes over: marking is bound by the shared-memory atomics of an SM.  With one CTA and with eight, tables of n entries, all but a few in
// use: 1024 entries 4.6 and 5.5 us, 8192 6.0 and 6.6, 16384 7.2 and 7.0, 32768 9.4 and 7.5, 65536 13.7 and 8.7, 262144 34 and 16.
constexpr int kPlanThreads = 1024, kPlanLoads = 8, kPlanCluster = 8, kPlanEntries = 32768, kPlanMaxBlocks = 1600000, kPlanMaxTokens = 1 << 20;

struct PlanArgs {
    int *tables;
    const int *lengths, *fresh;
    int *lengths_out, *runs, *n_runs;
    int n_seqs, max_blocks, n_blocks, block, n_tokens;
    unsigned *status;
};

// Inclusive sum over the CTA; `total` gets the sum.  sums: 33 values.
__device__ __forceinline__ int block_scan(int v, int *sums, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(kFullMask, v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = v;
    __syncthreads();
    if (warp == 0) {
        int s = sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(kFullMask, s, o);
            if (lane >= o) s += u;
        }
        sums[lane] = s;
    }
    __syncthreads();
    total = sums[31];
    return v + (warp ? sums[warp - 1] : 0);
}

__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(const PlanArgs a) {
    extern __shared__ uint32_t held[];                       // a bit per block of the pool
    __shared__ int sums[33], s_len[kPlanThreads], s_new[kPlanThreads], s_base[kPlanThreads], s_run[kPlanThreads], s_tok[kPlanThreads], s_free[kPlanThreads];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = a.block;
    const int words = (a.n_blocks + 31) >> 5, per = (words + kPlanThreads - 1) / kPlanThreads;
    unsigned bad = 0;
    const int ctas = gridDim.x, rank = blockIdx.x;           // one cluster
    for (int w = tid; w < words; w += kPlanThreads) {
        const int left = a.n_blocks - w * 32;
        held[w] = left >= 32 ? 0u : ~0u << left;             // places behind the pool's last block are never free
    }
    __syncthreads();
    for (int s = warp * ctas + rank; s < a.n_seqs; s += ctas * (kPlanThreads / 32)) {
        const int live = min(max(a.lengths[s], 0) / b, a.max_blocks);
        const int *row = a.tables + (size_t)s * a.max_blocks;
        for (int j0 = lane; j0 < live; j0 += 32 * kPlanLoads) {      // the loads of a step are in flight together
            int id[kPlanLoads];
#pragma unroll
            for (int u = 0; u < kPlanLoads; u++) id[u] = j0 + 32 * u < live ? row[j0 + 32 * u] : 0;
#pragma unroll
            for (int u = 0; u < kPlanLoads; u++) {
                if (j0 + 32 * u >= live) break;
                if ((unsigned)id[u] < (unsigned)a.n_blocks) atomicOr(&held[id[u] >> 5], 1u << (id[u] & 31));
                else bad |= 16u;
            }
        }
    }
    if (ctas > 1) {
        asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
        if (rank == 0)
            for (int w = tid; w < words; w += kPlanThreads) {
                const uint32_t at = (uint32_t)__cvta_generic_to_shared(held + w);
                uint32_t v[kPlanCluster];
#pragma unroll
                for (int r = 1; r < kPlanCluster; r++) {
                    uint32_t from;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(at), "r"(r));
                    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v[r]) : "r"(from) : "memory");
                }
                uint32_t all = held[w];
#pragma unroll
                for (int r = 1; r < kPlanCluster; r++) all |= v[r];
                held[w] = all;
            }
        asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");      // the bitmaps are read
        if (rank != 0) {
            if (bad && a.status) atomicOr(a.status, bad);
            return;
        }
    }
    __syncthreads();
    int mine = 0, n_free;
    for (int w = tid * per; w < min((tid + 1) * per, words); w++) mine += 32 - __popc(held[w]);
    s_free[tid] = block_scan(mine, sums, n_free);            // free blocks up to and with this thread's words

    long long tok_at = 0;
    long long base_at = 0;
    int run_at = 0;
    for (int s0 = 0; s0 < a.n_seqs; s0 += kPlanThreads) {
        const int s = s0 + tid, count = min(kPlanThreads, a.n_seqs - s0);
        int len = 0, fresh = 0, total;
        const bool in = s < a.n_seqs;
        if (in) { len = a.lengths[s]; fresh = a.fresh[s]; }
        const int rows = max(fresh, 0);
        const long long tok = tok_at + block_scan(min(rows, a.n_tokens + 1), sums, total) - min(rows, a.n_tokens + 1);
        tok_at = min(tok_at + total, (long long)a.n_tokens + 1);
        // a sequence that cannot be served keeps its length; its token rows are left out
        if (in && (len < 0 || fresh < 0 || (len / b) > a.max_blocks || ((long long)len + rows) / b > a.max_blocks || tok + rows > a.n_tokens)) {
            bad |= 1u;
            fresh = 0;
            len = max(len, 0);
        }
        const int need = in ? (len + fresh) / b - len / b : 0;
        const int upto = block_scan(need, sums, total);
        long long base = base_at + upto - need;
        if (base_at + total <= n_free) base_at += total;
        else {
            // The pool is exhausted: one sequence after the other, and one that does not fit takes nothing from those behind it.  (One thread; rare.)
            s_base[tid] = need;
            __syncthreads();
            if (tid == 0) {
                for (int i = 0; i < count; i++) {
                    const int n = s_base[i];
                    const bool fits = base_at + n <= n_free;
                    s_base[i] = fits ? (int)base_at : -1;
                    if (fits) base_at += n;
                }
                s_run[0] = (int)base_at;
            }
            __syncthreads();
            base = s_base[tid];
            base_at = s_run[0];
            if (base < 0) {
                bad |= 8u;
                fresh = 0;
            }
        }
        const int runs = fresh > 0 ? (len + fresh - 1) / b - len / b + 1 : 0;
        const int run = run_at + block_scan(runs, sums, total) - runs;
        run_at += total;
        s_len[tid] = len;
        s_new[tid] = fresh;
        s_base[tid] = (int)base;
        s_run[tid] = run;
        s_tok[tid] = (int)tok;
        if (in) a.lengths_out[s] = len + fresh;
        __syncthreads();
        // a run each thread: its sequence is the last that begins not behind it
        for (int r = run_at - total + tid; r < run_at; r += kPlanThreads) {
            int q = 0, beyond = count;
            while (beyond - q > 1) {
                const int mid = (q + beyond) >> 1;
                if (s_run[mid] <= r) q = mid;
                else beyond = mid;
            }
            const int L = s_len[q], n = s_new[q], i = r - s_run[q], first = L / b, end = L + n, nr = (end - 1) / b - first + 1;
            const bool shared = L % b != 0 && nr > 1 && end % b != 0;
            const int pos0 = i == 0 ? L : (first + i) * b, stop = min((first + i + 1) * b, end);
            int id = -1;
            if (stop % b == 0) {
                // the free block of rank s_base + i: the thread whose words hold it, then the word, then the bit
                const int rank = s_base[q] + i;
                int lo = 0, hi = kPlanThreads - 1;
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (s_free[mid] > rank) hi = mid;
                    else lo = mid + 1;
                }
                int left = rank - (lo ? s_free[lo - 1] : 0), w = lo * per;
                for (; w < words; w++) {
                    const int c = 32 - __popc(held[w]);
                    if (left < c) break;
                    left -= c;
                }
                uint32_t open = ~held[min(w, words - 1)];
                for (; left > 0; left--) open &= open - 1;
                id = w * 32 + __ffs(open) - 1;
                a.tables[(size_t)(s0 + q) * a.max_blocks + first + i] = id;
            } else if (shared && i == nr - 1) id = -2;
            int4 *out = reinterpret_cast<int4 *>(a.runs + (size_t)r * kRunInts);
            out[0] = make_int4(s0 + q, s_tok[q] + pos0 - L, pos0, stop - pos0);
            out[1] = make_int4(id, shared && i == 0 ? s_run[q] + nr - 1 : -1, 0, 0);
        }
        __syncthreads();
    }
    if (tid == 0) *a.n_runs = run_at;
    if (bad && a.status) atomicOr(a.status, bad);
}

// ---- rotary embedding and append -------------------------------------------------------------------------------------------------
struct AppendArgs {
    __half *q_out;
    const __half *q, *k, *v;
    long q_out_stride, q_stride, k_stride, v_stride;
    uint8_t *data;
    float4 *scales;
    __half *tail_k, *tail_v;
    long tail_k_stride, tail_v_stride;
    const int *runs, *n_runs;
    const double *inv_freq;
    int n_tokens, n_seqs, n_heads, n_kv, n_blocks, block;
    unsigned *status;
};

// One CTA per run and share of the heads: all its copies are 16 bytes wide.  Bound by the bytes of q, k and v.  The angle is in 64 bits: at position
// 10^6 its rounding to 32 would turn a key by 0.03.  The products and sums of the rotation are rounded one by one, as in torch.
constexpr int kAppendThreads = 256, kAppendUnroll = 4;

struct Turn {
    float cs[8], sn[8];
    __device__ __forceinline__ void load(const float2 *t) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float4 v = reinterpret_cast<const float4 *>(t)[j];
            cs[2 * j] = v.x; sn[2 * j] = v.y; cs[2 * j + 1] = v.z; sn[2 * j + 1] = v.w;
        }
    }
    // dims i .. i + 7 and i + HD/2 .. of one head
    __device__ __forceinline__ void apply(uint4 &lo, uint4 &hi) const {
        __half2 *a = reinterpret_cast<__half2 *>(&lo), *b = reinterpret_cast<__half2 *>(&hi);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float2 x = __half22float2(a[j]), y = __half22float2(b[j]);
            const float c0 = cs[2 * j], s0 = sn[2 * j], c1 = cs[2 * j + 1], s1 = sn[2 * j + 1];
            a[j] = __floats2half2_rn(__fsub_rn(__fmul_rn(x.x, c0), __fmul_rn(y.x, s0)), __fsub_rn(__fmul_rn(x.y, c1), __fmul_rn(y.y, s1)));
            b[j] = __floats2half2_rn(__fadd_rn(__fmul_rn(y.x, c0), __fmul_rn(x.x, s0)), __fadd_rn(__fmul_rn(y.y, c1), __fmul_rn(x.y, s1)));
        }
    }
};

template <int KIND>
__device__ __forceinline__ uint32_t code_of(float x, bool finite) {
    if constexpr (KIND == kKvInt8) return finite ? (uint32_t)((int)rintf(x) + 128) : 128u;
    else return finite ? (uint32_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3) : 0u;
}

template <int HD, int KIND>
__global__ void __launch_bounds__(kAppendThreads, 4) append_kernel(const AppendArgs a) {
    constexpr int kChunks = HD / 16;                         // pairs of 8 dims of a head
    extern __shared__ __align__(16) uint8_t append_smem[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int b = a.block, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float2 *turn = reinterpret_cast<float2 *>(append_smem);                   // [block][HD/2] cos, sin
    __half *tile = reinterpret_cast<__half *>(turn + b * (HD / 2));           // [block][HD] one head's rows of K or V
    __shared__ unsigned s_amax[2];
    const int n_runs = min(*a.n_runs, (int)gridDim.x);
    if ((int)blockIdx.x >= n_runs) return;
    int run = blockIdx.x, extra = -1;
    const int kv_per = (a.n_kv + gridDim.y - 1) / gridDim.y, kv0 = blockIdx.y * kv_per, kv1 = min(kv0 + kv_per, a.n_kv);
    const int rep = a.n_heads / a.n_kv, q0 = kv0 * rep, nq = max(kv1 - kv0, 0) * rep;
    for (int part = 0; part < 2; part++) {
        const int4 r0 = reinterpret_cast<const int4 *>(a.runs)[2 * run], r1 = reinterpret_cast<const int4 *>(a.runs)[2 * run + 1];
        const int seq = r0.x, tok0 = r0.y, pos0 = r0.z, count = r0.w, id = r1.x, o = pos0 & (b - 1);
        if ((unsigned)seq >= (unsigned)a.n_seqs || tok0 < 0 || count < 0 || count > b || pos0 < 0 || o + count > b || tok0 > a.n_tokens - count ||
            id >= a.n_blocks || (id >= 0 && o + count != b)) {
            if (a.status && tid == 0) atomicOr(a.status, 1u);
            return;
        }
        if (part == 0) {
            if (id == -2) return;                            // the CTA of the sequence's first run does this one
            extra = r1.y;
        }
        __syncthreads();
        for (int i = tid; i < count * (HD / 2); i += kAppendThreads) {
            double sn, cs;
            sincos((double)(pos0 + i / (HD / 2)) * a.inv_freq[i % (HD / 2)], &sn, &cs);
            turn[i] = make_float2((float)cs, (float)sn);
        }
        __syncthreads();
        // q: a warp takes a token; its lanes keep their dims and go through the heads
        for (int t = warp; t < count; t += kAppendThreads / 32) {
            constexpr int kHeads = 32 / kChunks;             // heads of a step
            Turn w;
            w.load(turn + t * (HD / 2) + lane % kChunks * 8);
            const size_t at = (size_t)(q0 + lane / kChunks) * HD + lane % kChunks * 8;
            const __half *x = a.q + (size_t)(tok0 + t) * a.q_stride + at;
            __half *y = a.q_out + (size_t)(tok0 + t) * a.q_out_stride + at;
            for (int h = lane / kChunks; h < nq; h += kHeads * kAppendUnroll) {
                uint4 lo[kAppendUnroll], hi[kAppendUnroll];
#pragma unroll
                for (int u = 0; u < kAppendUnroll; u++)
                    if (h + u * kHeads < nq) {
                        const uint4 *p = reinterpret_cast<const uint4 *>(x + (h - lane / kChunks + u * kHeads) * HD);
                        lo[u] = p[0];
                        hi[u] = p[kChunks];
                    }
#pragma unroll
                for (int u = 0; u < kAppendUnroll; u++)
                    if (h + u * kHeads < nq) {
                        w.apply(lo[u], hi[u]);
                        uint4 *p = reinterpret_cast<uint4 *>(y + (h - lane / kChunks + u * kHeads) * HD);
                        p[0] = lo[u];
                        p[kChunks] = hi[u];
                    }
            }
        }
        for (int h = kv0; h < kv1; h++)
            for (int which = 0; which < 2; which++) {
                __half *tail = (which == 0 ? a.tail_k + (size_t)seq * a.tail_k_stride : a.tail_v + (size_t)seq * a.tail_v_stride) + (size_t)h * b * HD;
                __syncthreads();
                if (tid == 0) s_amax[which] = 0;
                unsigned top = 0;                            // the largest magnitude as bits: an infinity or NaN is above every number
                auto see = [&](const uint4 &v) {
                    top = __vmaxu2(top, __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu)));
                };
                if (which == 0) {
                    for (int i = tid; i < count * kChunks; i += kAppendThreads) {
                        const int t = i / kChunks, d = i % kChunks * 8;
                        const uint4 *p = reinterpret_cast<const uint4 *>(a.k + (size_t)(tok0 + t) * a.k_stride + h * HD + d);
                        uint4 lo = p[0], hi = p[kChunks];
                        Turn w;
                        w.load(turn + t * (HD / 2) + d);
                        w.apply(lo, hi);
                        see(lo);
                        see(hi);
                        uint4 *to = reinterpret_cast<uint4 *>(id < 0 ? tail + (o + t) * HD + d : tile + (o + t) * HD + d);
                        to[0] = lo;
                        to[kChunks] = hi;
                    }
                } else {
                    for (int i = tid; i < count * (HD / 8); i += kAppendThreads) {
                        const int t = i / (HD / 8), d = i % (HD / 8) * 8;
                        const uint4 v = *reinterpret_cast<const uint4 *>(a.v + (size_t)(tok0 + t) * a.v_stride + h * HD + d);
                        see(v);
                        if (id >= 0) *reinterpret_cast<uint4 *>(tile + (o + t) * HD + d) = v;
                        else {
                            const __half *e = reinterpret_cast<const __half *>(&v);
#pragma unroll
                            for (int j = 0; j < 8; j++) tail[((o + t) >> 1) * (2 * HD) + (d + j) * 2 + ((o + t) & 1)] = e[j];
                        }
                    }
                }
                if (id < 0) continue;
                for (int i = tid; i < o * (HD / 8); i += kAppendThreads) {
                    const int t = i / (HD / 8), d = i % (HD / 8) * 8;
                    uint4 v;
                    if (which == 0) v = *reinterpret_cast<const uint4 *>(tail + t * HD + d);
                    else {
                        __half *e = reinterpret_cast<__half *>(&v);
#pragma unroll
                        for (int j = 0; j < 8; j++) e[j] = tail[(t >> 1) * (2 * HD) + (d + j) * 2 + (t & 1)];
                    }
                    see(v);
                    *reinterpret_cast<uint4 *>(tile + t * HD + d) = v;
                }
                __syncthreads();
                top = __reduce_max_sync(kFullMask, max(top & 0xFFFFu, top >> 16));
                if (lane == 0) atomicMax(&s_amax[which], top);
                __syncthreads();
                const unsigned bits = s_amax[which];
                const bool finite = bits < 0x7C00;
                const float amax = fmaxf(__half2float(__ushort_as_half((unsigned short)bits)), kTinyAmax), full = KIND == kKvInt8 ? 127.f : 448.f;
                const float inv = __fdiv_rn(full, amax);
                uint8_t *out = a.data + ((size_t)id * a.n_kv + h) * (size_t)(2 * b * HD) + which * (16 * HD);
                for (int i = tid; i < b * HD / 16; i += kAppendThreads) {
                    // 16 bytes of a unit
                    const int u = i / HD, at = i % HD * 16;
                    uint32_t word[4];
                    if (which == 0) {                        // (group of 8 tokens, half of 64 dims, token, dim)
                        const int t = (at >> 9) / (HD >> 6) * 8 + ((at >> 6) & 7), d = (at >> 9) % (HD >> 6) * 64 + (at & 63);
                        const __half2 *src = reinterpret_cast<const __half2 *>(tile + (16 * u + t) * HD + d);
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const float2 x = __half22float2(src[2 * k]), y = __half22float2(src[2 * k + 1]);
                            word[k] = code_of<KIND>(__fmul_rn(x.x, inv), finite) | code_of<KIND>(__fmul_rn(x.y, inv), finite) << 8 |
                                      code_of<KIND>(__fmul_rn(y.x, inv), finite) << 16 | code_of<KIND>(__fmul_rn(y.y, inv), finite) << 24;
                        }
                    } else {                                 // token 8h + 2c + e, dim g * HD/8 + 4n + j, order (n, g, c, j, h, e)
                        const int c = (at >> 4) & 3, g = (at >> 6) & 7, n = at >> 9;
                        const __half *src = tile + (16 * u + 2 * c) * HD + g * (HD / 8) + 4 * n;
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            word[j] = 0;
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                word[j] |= code_of<KIND>(__fmul_rn(__half2float(src[((k >> 1) * 8 + (k & 1)) * HD + j]), inv), finite) << (8 * k);
                        }
                    }
                    *reinterpret_cast<uint4 *>(out + (size_t)u * (32 * HD) + at) = make_uint4(word[0], word[1], word[2], word[3]);
                }
                // a block that holds something not finite stands for NaN everywhere
                if (tid == 0) reinterpret_cast<float *>(a.scales + (size_t)id * a.n_kv + h)[which] = finite ? __fmul_rn(amax, 1.f / full) : NAN;
            }
        if (part == 1 || extra < 0 || extra >= n_runs) return;
        run = extra;
    }
}

template <typename... Args>
int launch_dependent(void (*kernel)(Args...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    QTIP_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));
    return check_launch();
}

}  // namespace
}  // namespace qtip

using namespace qtip;

extern "C" int qtip_kv_plan(int *tables, const int *lengths, const int *new_tokens, int *lengths_out, int *runs, int *n_runs, int n_seqs, int max_blocks,
                            int n_blocks, int block, int n_tokens, int max_runs, unsigned *status, void *stream) {
    if (!tables || !lengths || !new_tokens || !lengths_out || !runs || !n_runs || lengths_out == lengths || lengths_out == new_tokens) return QTIP_ERR_BAD_ARG;
    if (n_seqs < 1 || n_seqs > 65535 || max_blocks < 1 || n_blocks < 1 || n_blocks > kPlanMaxBlocks || n_tokens < 0) return QTIP_ERR_BAD_SHAPE;
    // token rows of 1024 sequences and positions are added in 32 bits
    if (n_tokens > kPlanMaxTokens || ((long)max_blocks + 1) * block + n_tokens > 0x7FFFFFFFl) return QTIP_ERR_BAD_SHAPE;
    if (block != 16 && block != 32 && block != 64 && block != 128) return QTIP_ERR_BAD_SHAPE;
    if (max_runs < n_tokens / block + 2 * n_seqs) return QTIP_ERR_WORKSPACE;
    const void *words[] = {tables, lengths, new_tokens, lengths_out, n_runs, status};
    for (const void *p : words)
        if (!aligned(p, 4)) return QTIP_ERR_ALIGNMENT;
    if (!aligned(runs, 16)) return QTIP_ERR_ALIGNMENT;
    const PlanArgs a = {tables, lengths, new_tokens, lengths_out, runs, n_runs, n_seqs, max_blocks, n_blocks, block, n_tokens, status};
    const size_t smem = (size_t)((n_blocks + 31) / 32) * 4;
    if (smem > 16384) QTIP_CUDA_TRY(cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kPlanMaxBlocks + 31) / 32 * 4));
    const int ctas = (long)n_seqs * max_blocks < kPlanEntries ? 1 : kPlanCluster;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kPlanThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctas > 1 ? 2 : 1;
    QTIP_CUDA_TRY(cudaLaunchKernelEx(&cfg, kv_plan_kernel, a));
    return check_launch();
}

extern "C" int qtip_rope_kv_append_paged(void *q_out, long q_out_stride, const void *q, long q_stride, const void *k, long k_stride, const void *v,
                                         long v_stride, void *data, float *scales, void *tail_k, long tail_k_stride, void *tail_v, long tail_v_stride,
                                         const int *runs, const int *n_runs, int max_runs, const double *inv_freq, int n_tokens, int n_seqs, int n_heads,
                                         int n_kv_heads, int head_dim, int n_blocks, int block, int kind, unsigned *status, void *stream) {
    if (!q_out || !q || !k || !v || !data || !scales || !tail_k || !tail_v || !runs || !n_runs || !inv_freq) return QTIP_ERR_BAD_ARG;
    if (!paged_shape_ok(n_heads, n_kv_heads, head_dim, block, kind) || n_tokens < 0 || n_seqs < 1 || n_blocks < 1 || max_runs < 0) return QTIP_ERR_BAD_SHAPE;
    if (n_tokens == 0 || max_runs == 0) return QTIP_OK;
    const void *ptrs[] = {q_out, q, k, v, data, scales, tail_k, tail_v, runs};
    for (const void *p : ptrs)
        if (!aligned(p, 16)) return QTIP_ERR_ALIGNMENT;
    if (!aligned(inv_freq, 8) || !aligned(n_runs, 4) || !aligned(status, 4)) return QTIP_ERR_ALIGNMENT;
    if ((q_out_stride | q_stride | k_stride | v_stride | tail_k_stride | tail_v_stride) & 7) return QTIP_ERR_ALIGNMENT;
    // rows that are written share no memory
    const long tail = (long)n_kv_heads * block * head_dim;
    if ((n_tokens > 1 && q_out_stride < (long)n_heads * head_dim) || (n_seqs > 1 && (tail_k_stride < tail || tail_v_stride < tail))) return QTIP_ERR_BAD_SHAPE;
    const AppendArgs a = {static_cast<__half *>(q_out), static_cast<const __half *>(q), static_cast<const __half *>(k), static_cast<const __half *>(v),
                          q_out_stride, q_stride, k_stride, v_stride, static_cast<uint8_t *>(data), reinterpret_cast<float4 *>(scales),
                          static_cast<__half *>(tail_k), static_cast<__half *>(tail_v), tail_k_stride, tail_v_stride, runs, n_runs, inv_freq, n_tokens,
                          n_seqs, n_heads, n_kv_heads, n_blocks, block, status};
    const size_t smem = (size_t)block * head_dim * (sizeof(float) + sizeof(__half));
    auto kernel = head_dim == 128 ? (kind == kKvInt8 ? append_kernel<128, kKvInt8> : append_kernel<128, kKvE4m3>)
                                  : (kind == kKvInt8 ? append_kernel<64, kKvInt8> : append_kernel<64, kKvE4m3>);
    if (smem > 48 * 1024 - 64) QTIP_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * 128 * 6));
    // shares of the heads: eight CTAs per SM, where there are as many heads (16 prompts of 512 tokens, 32 heads: 98 us, with four 121)
    const int wanted = (8 * sm_count() + max_runs - 1) / max_runs, shares = wanted < 1 ? 1 : wanted < n_kv_heads ? wanted : n_kv_heads;
    const int per = (n_kv_heads + shares - 1) / shares;
    return launch_dependent(kernel, dim3(max_runs, (n_kv_heads + per - 1) / per), dim3(kAppendThreads), smem, static_cast<cudaStream_t>(stream), a);
}
