// Layout of the key/value cache in 8 bits (paged_cache.cu writes it, paged_attn.cu reads it).
//
// A block holds `block` tokens (16, 32, 64 or 128) of one layer.  Per key/value head: units of 16 tokens, K then V of 16 * hd bytes each.
// A block is written once, when its last token arrives; until then its tokens are in the sequence's tail in fp16, so that every value is
// rounded to 8 bits once and with the block's own largest value, whatever the pieces in which the tokens came.
#pragma once
#include "common.cuh"

namespace qtip {

constexpr int kRunInts = 8;      // sequence, first token row, first position, tokens, pool block (-1 none, -2 left to the first run's CTA), run of the tail, 0, 0
constexpr float kTinyAmax = 5.9604644775390625e-8f;      // 2^-24, the smallest fp16: a block of zeros has a scale above zero

enum { kKvInt8 = QTIP_KV_INT8, kKvE4m3 = QTIP_KV_E4M3 };

inline bool paged_shape_ok(int n_heads, int n_kv, int hd, int block, int kind) {
    return n_heads > 0 && n_kv > 0 && n_heads % n_kv == 0 && (hd == 64 || hd == 128) && (block == 16 || block == 32 || block == 64 || block == 128) &&
           (kind == kKvInt8 || kind == kKvE4m3);
}

// Byte of (token t < 16, dim d) in a unit's K: (group of 8 tokens, half of 64 dims, token, dim); a lane of the product q K^T then finds 16
// dims of one token in 16 bytes, and a warp's 16-byte loads are consecutive.
__host__ __device__ __forceinline__ int k_byte(int t, int d, int hd) { return ((t >> 3) * (hd >> 6) + (d >> 6)) * 512 + (t & 7) * 64 + (d & 63); }
// Byte of (t, d) in a unit's V: token t = 8h + 2c + e, dim d = g * (hd/8) + 4n + j, order (n, g, c, j, h, e): the four tokens of a word are
// the ones a lane of the product p V multiplies.
__host__ __device__ __forceinline__ int v_byte(int t, int d, int hd) {
    const int g = d / (hd >> 3), n = (d % (hd >> 3)) >> 2, j = d & 3;
    return ((((n * 8 + g) * 4 + ((t & 7) >> 1)) * 4 + j) << 2) + ((t >> 3) << 1) + (t & 1);
}

}  // namespace qtip
