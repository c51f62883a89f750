// Writers of the key/value cache in 8 bits (paged.cuh): block tables and runs of new tokens from the sequences' lengths, and the rotary
// embedding with the append of new tokens.  They stand where the decode loop has StaticCache.update (model/cache_utils.py:1147-1193
// upstream) and apply_rotary_pos_emb (model/llama.py:797-898).
#include <cuda_fp8.h>

#include "paged.cuh"

namespace qtip {
namespace {

// ---- block tables and runs -------------------------------------------------------------------------------------------------------
// One CTA.  A block is free when no sequence's table names it among its complete blocks (a bitmap in shared memory): there is no free
// list to keep, a sequence whose length is set to zero has released its blocks, and tables that name the same block (beams of one
// search, a common prompt) share it.  The new blocks are the lowest free ones, in the order of the sequences.
constexpr int kPlanThreads = 1024, kPlanMaxBlocks = 1600000, kPlanMaxTokens = 1 << 20;

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
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = a.block;
    const int words = (a.n_blocks + 31) >> 5, per = (words + kPlanThreads - 1) / kPlanThreads;
    unsigned bad = 0;
    for (int w = tid; w < words; w += kPlanThreads) {
        const int left = a.n_blocks - w * 32;
        held[w] = left >= 32 ? 0u : ~0u << left;             // places behind the pool's last block are never free
    }
    __syncthreads();
    for (int s = warp; s < a.n_seqs; s += kPlanThreads / 32) {
        const int live = min(max(a.lengths[s], 0) / b, a.max_blocks);
        for (int j = lane; j < live; j += 32) {
            const int id = a.tables[(size_t)s * a.max_blocks + j];
            if ((unsigned)id < (unsigned)a.n_blocks) atomicOr(&held[id >> 5], 1u << (id & 31));
            else bad |= 16u;
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
        int need = in ? (len + fresh) / b - len / b : 0;
        const int upto = block_scan(need, sums, total);
        const long long base = base_at + upto - need;
        base_at += total;
        if (need > 0 && base + need > n_free) {              // the pool is exhausted
            bad |= 8u;
            fresh = need = 0;
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
        for (int q = warp; q < count; q += kPlanThreads / 32) {
            const int L = s_len[q], n = s_new[q];
            if (n == 0) continue;
            const int first = L / b, end = L + n, nr = (end - 1) / b - first + 1;
            const bool shared = L % b != 0 && nr > 1 && end % b != 0;
            for (int i = lane; i < nr; i += 32) {
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
                    id = w * 32 + (int)__fns(~held[min(w, words - 1)], 0, left + 1);
                    a.tables[(size_t)(s0 + q) * a.max_blocks + first + i] = id;
                } else if (shared && i == nr - 1) id = -2;
                int4 *out = reinterpret_cast<int4 *>(a.runs + (size_t)(s_run[q] + i) * kRunInts);
                out[0] = make_int4(s0 + q, s_tok[q] + pos0 - L, pos0, stop - pos0);
                out[1] = make_int4(id, shared && i == 0 ? s_run[q] + nr - 1 : -1, 0, 0);
            }
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

constexpr int kAppendThreads = 256;

template <int HD, int KIND>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendArgs a) {
    extern __shared__ __align__(16) uint8_t append_smem[];
    const int b = a.block, tid = threadIdx.x;
    float2 *turn = reinterpret_cast<float2 *>(append_smem);                   // [block][HD/2] cos, sin
    __half *tile = reinterpret_cast<__half *>(turn + b * (HD / 2));           // [block][HD] one head's rows
    __shared__ unsigned s_amax;
    if ((int)blockIdx.x >= *a.n_runs) return;
    int run = blockIdx.x, extra = -1;
    const int kv_per = (a.n_kv + gridDim.y - 1) / gridDim.y, kv0 = blockIdx.y * kv_per, kv1 = min(kv0 + kv_per, a.n_kv);
    const int q_per = (a.n_heads + gridDim.y - 1) / gridDim.y, q0 = blockIdx.y * q_per, q1 = min(q0 + q_per, a.n_heads);
    for (int part = 0; part < 2; part++) {
        const int4 r0 = reinterpret_cast<const int4 *>(a.runs)[2 * run], r1 = reinterpret_cast<const int4 *>(a.runs)[2 * run + 1];
        const int seq = r0.x, tok0 = r0.y, pos0 = r0.z, count = r0.w, id = r1.x, o = pos0 % b;
        if ((unsigned)seq >= (unsigned)a.n_seqs || tok0 < 0 || count < 0 || pos0 < 0 || o + count > b || tok0 + count > a.n_tokens || id >= a.n_blocks ||
            (id >= 0 && o + count != b)) {
            if (a.status && tid == 0) atomicOr(a.status, 1u);
            return;
        }
        if (part == 0) {
            if (id == -2) return;                            // the CTA of the sequence's first run does this one
            extra = r1.y;
        }
        __syncthreads();
        // the angle in 64 bits: at position 10^6 its rounding to 32 would turn a key by 0.03
        for (int i = tid; i < count * (HD / 2); i += kAppendThreads) {
            double sn, cs;
            sincos((double)(pos0 + i / (HD / 2)) * a.inv_freq[i % (HD / 2)], &sn, &cs);
            turn[i] = make_float2((float)cs, (float)sn);
        }
        __syncthreads();
        for (int i = tid; i < count * (q1 - q0) * (HD / 2); i += kAppendThreads) {
            const int d = i % (HD / 2), h = q0 + i / (HD / 2) % (q1 - q0), t = i / (HD / 2) / (q1 - q0);
            const float2 w = turn[t * (HD / 2) + d];
            const __half *x = a.q + (size_t)(tok0 + t) * a.q_stride + h * HD + d;
            __half *y = a.q_out + (size_t)(tok0 + t) * a.q_out_stride + h * HD + d;
            const float x0 = __half2float(x[0]), x1 = __half2float(x[HD / 2]);
            y[0] = __float2half_rn(__fsub_rn(__fmul_rn(x0, w.x), __fmul_rn(x1, w.y)));
            y[HD / 2] = __float2half_rn(__fadd_rn(__fmul_rn(x1, w.x), __fmul_rn(x0, w.y)));
        }
        for (int h = kv0; h < kv1; h++)
            for (int which = 0; which < 2; which++) {
                __half *tk = a.tail_k + (size_t)seq * a.tail_k_stride + (size_t)h * b * HD;
                __half *tv = a.tail_v + (size_t)seq * a.tail_v_stride + (size_t)h * b * HD;
                __syncthreads();
                if (tid == 0) s_amax = 0;
                if (which == 0) {
                    for (int i = tid; i < count * (HD / 2); i += kAppendThreads) {
                        const int d = i % (HD / 2), t = i / (HD / 2);
                        const float2 w = turn[i];
                        const __half *x = a.k + (size_t)(tok0 + t) * a.k_stride + h * HD + d;
                        const float x0 = __half2float(x[0]), x1 = __half2float(x[HD / 2]);
                        tile[(o + t) * HD + d] = __float2half_rn(__fsub_rn(__fmul_rn(x0, w.x), __fmul_rn(x1, w.y)));
                        tile[(o + t) * HD + d + HD / 2] = __float2half_rn(__fadd_rn(__fmul_rn(x1, w.x), __fmul_rn(x0, w.y)));
                    }
                } else {
                    for (int i = tid; i < count * HD; i += kAppendThreads)
                        tile[(o + i / HD) * HD + i % HD] = a.v[(size_t)(tok0 + i / HD) * a.v_stride + h * HD + i % HD];
                }
                if (id < 0) {
                    __syncthreads();
                    for (int i = tid; i < count * HD; i += kAppendThreads) {
                        const int t = o + i / HD, d = i % HD;
                        if (which == 0) tk[t * HD + d] = tile[t * HD + d];
                        else tv[((t >> 1) * HD + d) * 2 + (t & 1)] = tile[t * HD + d];
                    }
                    continue;
                }
                for (int i = tid; i < o * HD; i += kAppendThreads) {
                    const int t = i / HD, d = i % HD;
                    tile[i] = which == 0 ? tk[i] : tv[((t >> 1) * HD + d) * 2 + (t & 1)];
                }
                __syncthreads();
                // the largest magnitude as bits: an infinity or NaN is larger than every number
                unsigned m = 0;
                for (int i = tid; i < b * HD; i += kAppendThreads) m = max(m, (unsigned)(__half_as_ushort(tile[i]) & 0x7FFF));
                m = __reduce_max_sync(kFullMask, m);
                if ((tid & 31) == 0) atomicMax(&s_amax, m);
                __syncthreads();
                const bool finite = s_amax < 0x7C00;
                const float amax = fmaxf(__half2float(__ushort_as_half((unsigned short)s_amax)), kTinyAmax), top = KIND == kKvInt8 ? 127.f : 448.f;
                const float inv = __fdiv_rn(top, amax);
                uint8_t *out = a.data + ((size_t)id * a.n_kv + h) * (size_t)(2 * b * HD);
                for (int i = tid; i < b * HD; i += kAppendThreads) {
                    const int t = i / HD, d = i % HD;
                    const float x = __fmul_rn(__half2float(tile[i]), inv);
                    uint8_t c;
                    if constexpr (KIND == kKvInt8) c = (uint8_t)(finite ? (int)rintf(x) + 128 : 128);
                    else c = finite ? (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3) : 0;
                    out[((t >> 4) * 2 + which) * (16 * HD) + (which == 0 ? k_byte(t & 15, d, HD) : v_byte(t & 15, d, HD))] = c;
                }
                // a block that holds something not finite stands for NaN everywhere
                if (tid == 0) reinterpret_cast<float *>(a.scales + (size_t)id * a.n_kv + h)[which] = finite ? __fmul_rn(amax, 1.f / top) : NAN;
            }
        if (part == 1 || extra < 0 || extra >= *a.n_runs) return;
        run = extra;
    }
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
    if (!aligned(runs, 16)) return QTIP_ERR_ALIGNMENT;
    const PlanArgs a = {tables, lengths, new_tokens, lengths_out, runs, n_runs, n_seqs, max_blocks, n_blocks, block, n_tokens, status};
    const size_t smem = (size_t)((n_blocks + 31) / 32) * 4;
    QTIP_CUDA_TRY(cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kPlanMaxBlocks + 31) / 32 * 4));
    kv_plan_kernel<<<1, kPlanThreads, smem, static_cast<cudaStream_t>(stream)>>>(a);
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
    if ((q_out_stride | q_stride | k_stride | v_stride | tail_k_stride | tail_v_stride) & 7) return QTIP_ERR_ALIGNMENT;
    const AppendArgs a = {static_cast<__half *>(q_out), static_cast<const __half *>(q), static_cast<const __half *>(k), static_cast<const __half *>(v),
                          q_out_stride, q_stride, k_stride, v_stride, static_cast<uint8_t *>(data), reinterpret_cast<float4 *>(scales),
                          static_cast<__half *>(tail_k), static_cast<__half *>(tail_v), tail_k_stride, tail_v_stride, runs, n_runs, inv_freq, n_tokens,
                          n_seqs, n_heads, n_kv_heads, n_blocks, block, status};
    const size_t smem = (size_t)block * head_dim * (sizeof(float) + sizeof(__half));
    auto kernel = head_dim == 128 ? (kind == kKvInt8 ? append_kernel<128, kKvInt8> : append_kernel<128, kKvE4m3>)
                                  : (kind == kKvInt8 ? append_kernel<64, kKvInt8> : append_kernel<64, kKvE4m3>);
    QTIP_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * 128 * 6));
    kernel<<<dim3(max_runs, min(n_kv_heads, 8)), kAppendThreads, smem, static_cast<cudaStream_t>(stream)>>>(a);
    return check_launch();
}
