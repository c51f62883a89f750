// Single-query attention over the key/value cache in 8 bits (paged.cuh): out = softmax(q K^T / sqrt(hd)) V for each sequence and head.
// Stands where the decode loop has the scaled_dot_product_attention of LlamaSdpaAttention.forward (model/llama.py:884-891 upstream).
#include <cuda_fp8.h>

#include "paged.cuh"

namespace qtip {
namespace {

struct AttnArgs {
    __half *out;
    const __half *q;
    long out_stride, q_stride;
    const uint8_t *data;
    const float4 *scales;
    const __half *tail_k, *tail_v;
    long tail_k_stride, tail_v_stride;
    const int *tables, *lengths;
    int n_heads, n_kv, max_blocks, n_blocks, block;
    float scale;
    unsigned *status;
};

template <int KIND>
__device__ __forceinline__ float value_of(uint8_t c) {
    if constexpr (KIND == kKvInt8) return (float)((int)c - 128);
    else return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
}

// One CTA per sequence and head: the scores of 128 tokens, one each thread, then their weights times V, one dim each thread, with the
// running maximum and sum of the softmax.
template <int HD, int KIND>
__global__ void __launch_bounds__(128) attn_paged_kernel(const AttnArgs a) {
    __shared__ float qs[HD], ps[128], red[4];
    const int tid = threadIdx.x, b = a.block, seq = blockIdx.y, head = blockIdx.x, h = head / (a.n_heads / a.n_kv);
    int len = a.lengths[seq];
    __half *out = a.out + (size_t)seq * a.out_stride + head * HD;
    if (len < 0 || len / b > a.max_blocks) {
        if (a.status && tid == 0) atomicOr(a.status, 1u);
        len = 0;
    }
    const int full = len / b;
    if (tid < HD) qs[tid] = __half2float(a.q[(size_t)seq * a.q_stride + head * HD + tid]) * a.scale;
    float m = -INFINITY, l = 0.f, acc = 0.f;
    for (int t0 = 0; t0 < len; t0 += 128) {
        __syncthreads();
        const int t = t0 + tid;
        float s = -INFINITY;
        if (t < len) {
            s = 0.f;
            if (t / b < full) {
                const int id = a.tables[(size_t)seq * a.max_blocks + t / b];
                if ((unsigned)id < (unsigned)a.n_blocks) {
                    const uint8_t *k = a.data + ((size_t)id * a.n_kv + h) * (2 * b * HD) + (t % b / 16) * (32 * HD);
                    for (int d = 0; d < HD; d++) s = fmaf(qs[d], value_of<KIND>(k[k_byte(t & 15, d, HD)]), s);
                    s *= a.scales[(size_t)id * a.n_kv + h].x;
                } else {
                    s = -INFINITY;
                    if (a.status) atomicOr(a.status, 16u);
                }
            } else {
                const __half *k = a.tail_k + (size_t)seq * a.tail_k_stride + ((size_t)h * b + t % b) * HD;
                for (int d = 0; d < HD; d++) s = fmaf(qs[d], __half2float(k[d]), s);
            }
        }
        float mx = s;
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kFullMask, mx, o));
        if ((tid & 31) == 0) red[tid >> 5] = mx;
        __syncthreads();
        const float m_new = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]))), ref = m_new == -INFINITY ? 0.f : m_new;
        const float corr = __expf(m - ref);
        ps[tid] = t < len ? __expf(s - ref) : 0.f;
        __syncthreads();
        l *= corr;
        acc *= corr;
        m = m_new;
        for (int i = 0; i < min(128, len - t0); i++) {
            const float p = ps[i];
            l += p;
            const int u = t0 + i;
            if (tid >= HD || p == 0.f) continue;
            if (u / b < full) {
                const int id = a.tables[(size_t)seq * a.max_blocks + u / b];
                if ((unsigned)id >= (unsigned)a.n_blocks) continue;
                const uint8_t *v = a.data + ((size_t)id * a.n_kv + h) * (2 * b * HD) + (u % b / 16) * (32 * HD) + 16 * HD;
                acc = fmaf(p * a.scales[(size_t)id * a.n_kv + h].y, value_of<KIND>(v[v_byte(u & 15, tid, HD)]), acc);
            } else {
                const __half *v = a.tail_v + (size_t)seq * a.tail_v_stride + (size_t)h * b * HD;
                acc = fmaf(p, __half2float(v[((u % b >> 1) * HD + tid) * 2 + (u & 1)]), acc);
            }
        }
    }
    if (tid < HD) out[tid] = __float2half_rn(len > 0 ? acc / l : 0.f);
}

}  // namespace
}  // namespace qtip

using namespace qtip;

extern "C" size_t qtip_attn_paged_workspace_bytes(int n_seqs, int n_heads, int n_kv_heads, int head_dim) {
    (void)n_seqs; (void)n_heads; (void)n_kv_heads; (void)head_dim;
    return 16;
}

extern "C" int qtip_attn_decode_paged(void *out, long out_stride, const void *q, long q_stride, const void *data, const float *scales, const void *tail_k,
                                      long tail_k_stride, const void *tail_v, long tail_v_stride, const int *tables, const int *lengths, int n_seqs,
                                      int n_heads, int n_kv_heads, int head_dim, int max_blocks, int n_blocks, int block, int kind, void *workspace,
                                      size_t workspace_bytes, unsigned *status, void *stream) {
    if (!out || !q || !data || !scales || !tail_k || !tail_v || !tables || !lengths) return QTIP_ERR_BAD_ARG;
    if (!paged_shape_ok(n_heads, n_kv_heads, head_dim, block, kind) || n_seqs < 1 || n_seqs > 65535 || max_blocks < 1 || n_blocks < 1) return QTIP_ERR_BAD_SHAPE;
    if (!workspace || workspace_bytes < qtip_attn_paged_workspace_bytes(n_seqs, n_heads, n_kv_heads, head_dim)) return QTIP_ERR_WORKSPACE;
    const void *ptrs[] = {out, q, data, scales, tail_k, tail_v, workspace};
    for (const void *p : ptrs)
        if (!aligned(p, 16)) return QTIP_ERR_ALIGNMENT;
    if ((out_stride | q_stride | tail_k_stride | tail_v_stride) & 7) return QTIP_ERR_ALIGNMENT;
    const AttnArgs a = {static_cast<__half *>(out), static_cast<const __half *>(q), out_stride, q_stride, static_cast<const uint8_t *>(data),
                        reinterpret_cast<const float4 *>(scales), static_cast<const __half *>(tail_k), static_cast<const __half *>(tail_v), tail_k_stride,
                        tail_v_stride, tables, lengths, n_heads, n_kv_heads, max_blocks, n_blocks, block, 1.f / sqrtf((float)head_dim), status};
    auto kernel = head_dim == 128 ? (kind == kKvInt8 ? attn_paged_kernel<128, kKvInt8> : attn_paged_kernel<128, kKvE4m3>)
                                  : (kind == kKvInt8 ? attn_paged_kernel<64, kKvInt8> : attn_paged_kernel<64, kKvE4m3>);
    kernel<<<dim3(n_heads, n_seqs), 128, 0, static_cast<cudaStream_t>(stream)>>>(a);
    return check_launch();
}
