// What the kernels of the 8-bit cache share: its sequences as the device finds them, codes and scales, and the host's checks of the cache and its sequences.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "row_sequences.h"

namespace uzu {

// A number that is not below this makes its block and head not a number: code * scale stays finite for all others, and is a bf16 number, and so do sums over many tokens.
constexpr uint32_t kCacheHugeBits = 0x6f800000u;      // 2^96
constexpr int kCacheLeastExponent = -100;
constexpr uint32_t kNoIndex = 0xffffffffu;
// Attention's rows are the tokens that they are, of a sequence that has grown behind max_length as well (its keys there are left out, windows and kept first tokens stay); row numbers added, 32 bits hold them.
constexpr uint32_t kCacheAnyLength = 0x7fffffffu;
// A row of queries is brought to 2^14 .. 2^15 by a power of two, from 2^-113 for the largest numbers on up to this: 2^-126, its inverse, is still a normal number. Rows below 2^-112 stay below 2^14.
constexpr int kCacheMostPower = 126;
// Capped scores of 16-bit rows come of 1 - 2 / (1 + e^2x), which is off by 2^-22 of the cap whatever the score: up to this cap 2^-16, an eighth of what an f16 output's rounding moves. Above it tanhf, in the kernel for
// few rows. Caps are brought between the other two, where 1 / cap and its products stay normal numbers: below 2^-40 all weights are alike, and above 2^80 scores of up to 2^68 are left as they are, in f32.
constexpr float kCacheFastCap = 64.0f, kCacheLeastCap = 0x1p-40f, kCacheMostCap = 0x1p80f;
// What the kernel for few rows takes where the tcgen05 kernel takes the others: sequences of so many (row, head) pairs of a key head, or of so few rows. The latter has no split of the
// keys, so one CTA would read a long cache for a few rows of many heads. The border is where the other kernel needs a second tile of pairs; for one sequence alone the two cross later.
// One sequence, 32 heads of 128 on 8 (i8), us on tcgen05 / in the other kernel, behind 4096 tokens: 17 rows 78 / 30, 64 rows 94 / 66, 128 rows 95 / 125; behind 131072: 17 rows 2275 / 467, 64 rows 2676 / 1608, 128
// rows 2605 / 3655. 6144 rows of three sequences: 655 to 710 / 5083.
constexpr uint32_t kCacheFewPairs = 64, kCacheFewRows = 8;

// tokens that a sequence can have: what the host bounds and its table holds
inline uint32_t cache_capacity(const uzu_cache_sequences& s, uint32_t block_tokens) {
    const uint64_t table = (uint64_t)s.table_stride * block_tokens;
    return (uint32_t)(table < s.max_length ? table : s.max_length);
}

// null, or what is wrong
inline const char* check_cache(const uzu_quantized_cache& c) {
    if (c.code_type > UZU_CACHE_CODE_E4M3) return "code_type must be i8 or e4m3";
    if (c.block_tokens != 16 && c.block_tokens != 32 && c.block_tokens != 64) return "block_tokens must be 16, 32 or 64";
    if (c.head_dim == 0 || c.head_dim > 256 || c.head_dim % 16) return "head_dim must be a multiple of 16 up to 256";
    if (c.kv_heads == 0 || c.kv_heads > 65535) return "kv_heads must be in 1 .. 65535";
    if (!c.blocks) return "a cache without blocks";
    if (!c.key_codes || !c.value_codes || !c.key_scales || !c.value_scales) return "null cache";
    if ((c.key_codes | c.value_codes) % 16 || (c.key_scales | c.value_scales | c.key_weights) % 4) return "the cache is not aligned";
    return nullptr;
}
inline const char* check_cache_sequences(const uzu_cache_sequences& s, bool with_rows) {
    if (s.count > 65535) return "at most 65535 sequences";
    if (s.max_length >> 31 || s.rows >> 31) return "max_length and rows are below 2^31";
    if (!s.count) return nullptr;
    if (!s.tables || !s.lengths || (with_rows && !s.row_offsets)) return "null sequences";
    if ((s.tables | s.lengths | (with_rows ? s.row_offsets : 0)) % 4) return "the sequences are not aligned";
    if (!s.table_stride || !s.max_length) return "table_stride and max_length are at least 1";
    if ((uint64_t)s.table_stride * s.count >> 40) return "tables are too large";
    return nullptr;
}
struct CacheSpan {
    uint64_t at, bytes;
};
// whether [at, at + bytes) meets an array of the cache
inline bool meets_cache(const uzu_quantized_cache& c, uint64_t at, uint64_t bytes) {
    const uint64_t pairs = (uint64_t)c.blocks * c.kv_heads, codes = pairs * c.block_tokens * c.head_dim;
    const CacheSpan spans[5] = {{c.key_codes, codes}, {c.value_codes, codes}, {c.key_scales, pairs * 4}, {c.value_scales, pairs * 4}, {c.key_weights, pairs * c.block_tokens * 4}};
    for (const CacheSpan& s : spans)
        if (bytes_overlap(at, bytes, s.at, s.bytes)) return true;
    return false;
}
inline bool cache_meets_itself(const uzu_quantized_cache& c) {
    const uint64_t pairs = (uint64_t)c.blocks * c.kv_heads, codes = pairs * c.block_tokens * c.head_dim;
    const CacheSpan spans[5] = {{c.key_codes, codes}, {c.value_codes, codes}, {c.key_scales, pairs * 4}, {c.value_scales, pairs * 4}, {c.key_weights, pairs * c.block_tokens * 4}};
    for (int i = 0; i < 5; ++i)
        for (int j = 0; j < i; ++j)
            if (bytes_overlap(spans[i].at, spans[i].bytes, spans[j].at, spans[j].bytes)) return true;
    return false;
}
// whether a written array meets what says which sequences there are
inline bool meets_sequences(const uzu_cache_sequences& s, uint64_t at, uint64_t bytes) {
    return bytes_overlap(at, bytes, s.tables, (uint64_t)s.count * s.table_stride * 4) || bytes_overlap(at, bytes, s.lengths, (uint64_t)s.count * 4) ||
           bytes_overlap(at, bytes, s.row_offsets, ((uint64_t)s.count + 1) * 4);
}

// attention of a prompt's rows on tcgen05 (quantized_cache_umma.cu); maxima and sums (f32 [rows, heads, 2], optional) are of every row
bool quantized_cache_umma_applicable(const uzu_quantized_cache_attention_args& a);
void encode_quantized_cache_umma(uzu_command_buffer* cmd, const uzu_quantized_cache_attention_args& a, uint64_t row_stats);

#ifdef __CUDACC__
struct CacheSequence {
    uint32_t row, rows, length;      // first row, rows of the pass, tokens before it: whatever the device holds, inside the arrays
};
__device__ __forceinline__ CacheSequence cache_sequence(const uzu_cache_sequences& s, uint32_t capacity, uint32_t i) {
    CacheSequence q;
    q.length = min(reinterpret_cast<const uint32_t*>(s.lengths)[i], capacity);
    const uint32_t *offsets = reinterpret_cast<const uint32_t*>(s.row_offsets), begin = min(offsets[i], s.rows), end = min(offsets[i + 1], s.rows);
    q.row = begin;
    q.rows = end > begin ? min(end - begin, s.max_rows) : 0u;
    return q;
}
__device__ __forceinline__ uint32_t cache_block(const uzu_cache_sequences& s, uint32_t sequence, uint32_t nth) {      // (nth is below table_stride)
    return reinterpret_cast<const uint32_t*>(s.tables)[(size_t)sequence * s.table_stride + nth];
}

// the smallest scale that brings magnitudes of up to `most` into the codes' range; NaN for what has none
template <int CODE>
__device__ __forceinline__ float cache_scale(uint32_t most_bits) {
    if (most_bits >= kCacheHugeBits) return __uint_as_float(0x7fc00000u);
    if (most_bits == 0) return 0.0f;
    // 127 = 2^6 * (1 + 0x7e0000 / 2^23), 448 = 2^8 * (1 + 0x600000 / 2^23)
    constexpr uint32_t top = CODE == UZU_CACHE_CODE_I8 ? 0x7e0000u : 0x600000u;
    constexpr int power = CODE == UZU_CACHE_CODE_I8 ? 6 : 8;
    const int e = (int)(most_bits >> 23) - 127 - power + ((most_bits & 0x7fffffu) > top ? 1 : 0);
    return __uint_as_float((uint32_t)(max(e, kCacheLeastExponent) + 127) << 23);
}
// 1 / scale, exact; 0 for scales without codes (0, NaN)
__device__ __forceinline__ float cache_inverse(float scale) { return scale > 0.0f ? __uint_as_float((254u << 23) - __float_as_uint(scale)) : 0.0f; }

__device__ __forceinline__ uint32_t cache_pack_i8(float a, float b, float c, float d) {      // (already within +-127)
    return ((uint32_t)__float2int_rn(a) & 0xffu) | ((uint32_t)__float2int_rn(b) & 0xffu) << 8 | ((uint32_t)__float2int_rn(c) & 0xffu) << 16 | (uint32_t)__float2int_rn(d) << 24;
}
__device__ __forceinline__ uint32_t cache_pack_e4m3(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | (uint32_t)hi << 16;
}
template <int CODE>
__device__ __forceinline__ uint32_t cache_pack(float a, float b, float c, float d) {
    return CODE == UZU_CACHE_CODE_I8 ? cache_pack_i8(a, b, c, d) : cache_pack_e4m3(a, b, c, d);
}
// two codes (bytes of the low half) as f16 numbers, exact
__device__ __forceinline__ uint32_t cache_e4m3x2_f16x2(uint32_t w) {
    uint32_t r;
    asm("{ .reg .b16 lo, hi; mov.b32 {lo, hi}, %1; cvt.rn.f16x2.e4m3x2 %0, lo; }" : "=r"(r) : "r"(w));
    return r;
}
// four codes to numbers
template <int CODE>
__device__ __forceinline__ void cache_unpack(uint32_t w, float (&x)[4]) {
    if (CODE == UZU_CACHE_CODE_I8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
    } else {
        const uint32_t lo = cache_e4m3x2_f16x2(w), hi = cache_e4m3x2_f16x2(w >> 16);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
    }
}
#endif

}  // namespace uzu
