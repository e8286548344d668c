// Attention of a prompt's rows over the 8-bit cache on the 5th-generation tensor cores (bf16 rows, heads of up to 128 channels).
//
// A CTA has 256 (row, head) pairs of a key head as two tiles of 128, which take turns on the tensor cores: while one's scores become weights, the other's products run.
//   convert  four warps turn 128 keys' and values' codes into f16 numbers, which hold them exactly, in 128-byte swizzled rows of 64 channels, two stages each. Scales stay out: those
//            of keys multiply scores, those of values enter the weights and a tile's sum. What a tile of keys has (which of its groups of 16, their scales) goes along in shared memory.
//   issue    S = Q K^T into tensor memory (128 columns for each tile of rows), O = P V with P as operand A in S's place, both for one tile of rows at a time.
//   softmax  a thread a row: the largest score (scores are read twice, their registers are O's), the tile of keys before added to O by rounded additions, then weights as one f16
//            number each: 11 bits, which moves an output by an eighth of a bf16 rounding's half step or so. The row's maximum moves when it has grown by 2^8.
// A value scale more than 2^8 below the largest of its tile would lose its weights below f16's range: such groups of keys take a pass of their own, the others masked.
// Queries are brought to 2^14 .. 2^15 by a power of two for each row, as in the kernel for few rows.
// Every barrier wait is bounded (wait_errors.h).
#include "quantized_cache.cuh"
#include "umma.cuh"

namespace uzu {

namespace {

constexpr uint32_t QU_ROWS = 128, QU_KEYS = 128, QU_GROUPS = QU_KEYS / 16, QU_THREADS = 512, QU_STAGES = 2, QU_ITEMS = 4;
constexpr float QU_LIFT = 7.0f, QU_SLACK = 8.0f;      // weights: at most 2^(LIFT + SLACK)
constexpr uint32_t QU_BLOCK = 128 * 128;               // bytes of 128 rows of 64 channels
// registers of a thread: the launch's 128 shared out anew
constexpr uint32_t QU_SOFT_REGS = 200, QU_CONVERT_REGS = 72, QU_ISSUE_REGS = 40;

struct QuItem {
    uint32_t key0, groups, more;      // first key, which groups of 16 count, 0: no tile, the end
    float unit;                       // what the tile's products are multiplied by
    float key_scale[QU_GROUPS], lower[QU_GROUPS], gain[QU_GROUPS];      // lower: what a weight's exponent loses for its value scale, gain = 2^lower
};
struct QuParams {
    uzu_quantized_cache_attention_args a;
    uint32_t capacity, group;
    float* stats;
    unsigned int* error;
};

template <int D>
struct QuShape {
    static constexpr uint32_t BLOCKS = D / 64, Q = BLOCKS * QU_BLOCK, KV = BLOCKS * QU_BLOCK;
    static constexpr uint32_t O_COL = 256;      // tensor memory: scores of two tiles, 128 columns each, then their products
    static constexpr size_t SMEM = 2 * Q + 2 * QU_STAGES * KV + 1024;
};

__device__ __forceinline__ float qu_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float2 qu_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
    return d;
}
__device__ __forceinline__ float2 qu_add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return d;
}
__device__ __forceinline__ uint32_t qu_pack(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void qu_sts(uint32_t at, uint4 v) { asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory"); }
// four codes as f16 numbers
template <int CODE>
__device__ __forceinline__ uint2 qu_numbers(uint32_t w) {
    if (CODE == UZU_CACHE_CODE_E4M3) return make_uint2(cache_e4m3x2_f16x2(w), cache_e4m3x2_f16x2(w >> 16));
    const uint32_t off = 0x64806480u;
    w ^= 0x80808080u;
    const uint32_t lo = __byte_perm(w, 0x64646464u, 0x4140), hi = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), *reinterpret_cast<const __half2*>(&off)), b = __hsub2(*reinterpret_cast<const __half2*>(&hi), *reinterpret_cast<const __half2*>(&off));
    return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

template <int CODE, int D, bool CAP>
__global__ void __launch_bounds__(QU_THREADS, 1) quantized_cache_umma_kernel(const __grid_constant__ QuParams p) {
    using S = QuShape<D>;
    extern __shared__ uint8_t qu_raw[];
    __shared__ __align__(8) uint64_t bars[16];
    __shared__ QuItem items[QU_ITEMS];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile uint32_t gave_up;
    const uzu_quantized_cache_attention_args& a = p.a;
    const uzu_quantized_cache& c = a.cache;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t base = (um_smem(qu_raw) + 1023u) & ~1023u, q0 = base, k0 = q0 + 2 * S::Q, v0 = k0 + QU_STAGES * S::KV, bar0 = um_smem(bars);
    auto q_full = [&](uint32_t r) { return bar0 + 8u * r; };
    auto s_full = [&](uint32_t r) { return bar0 + 8u * (2 + r); };
    auto p_full = [&](uint32_t r) { return bar0 + 8u * (4 + r); };
    auto k_full = [&](uint32_t s) { return bar0 + 8u * (6 + s); };
    auto k_empty = [&](uint32_t s) { return bar0 + 8u * (8 + s); };
    auto v_full = [&](uint32_t s) { return bar0 + 8u * (10 + s); };
    auto v_empty = [&](uint32_t s) { return bar0 + 8u * (12 + s); };
    const uint32_t last_products = bar0 + 8u * 14;

    // (the sequence is looked up behind pdl_wait; tensor memory first, a dependent's CTA that took it would wait for this one)
    if (warp == 0) {
        if (lane == 0) {
            for (uint32_t r = 0; r < 2; ++r) {
                um_init(q_full(r), 4); um_init(s_full(r), 2); um_init(p_full(r), 4);
                um_init(k_full(r), 4); um_init(k_empty(r), 1); um_init(v_full(r), 4); um_init(v_empty(r), 1);
            }
            um_init(last_products, 1);
            gave_up = 0;
            um_fence_init();
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(um_smem(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    um_fence_before();
    __syncthreads();
    um_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_launch_dependents();
    pdl_wait();

    const uint32_t sequence = blockIdx.z, head = blockIdx.y, G = p.group, dim = c.head_dim, bt = c.block_tokens;
    const CacheSequence q = cache_sequence(a.sequences, p.capacity, sequence);
    const uint32_t pairs = q.rows * G, tiles = (pairs + 2 * QU_ROWS - 1) / (2 * QU_ROWS);
    const bool mine = pairs > kCacheFewPairs && blockIdx.x < tiles;
    const uint32_t pair0 = mine ? (tiles - 1u - blockIdx.x) * 2 * QU_ROWS : 0u;      // the rows with the most keys first
    const uint32_t row_tiles = pair0 + QU_ROWS < pairs ? 2u : 1u;
    const uint32_t token0 = q.length + pair0 / G, token1 = q.length + (min(pair0 + 2 * QU_ROWS, pairs) - 1u) / G;
    const uint32_t end = min(token1 + 1u, p.capacity), begin = a.window && token0 >= a.window ? (token0 - a.window + 1u) & ~(QU_KEYS - 1u) : 0u;
    const uint32_t kept = (min(min(a.keep_first, begin), end) + QU_KEYS - 1u) / QU_KEYS;      // tiles of first keys
    const uint32_t key_tiles = kept + (end > begin ? (end - begin + QU_KEYS - 1u) / QU_KEYS : 0u);
    bool ok = true;

    if (!mine) {
        // nothing of this sequence is this CTA's
    } else if (warp < 8) {
        // ================================ softmax ================================
        um_more_registers<QU_SOFT_REGS>();
        const uint32_t r = warp >> 2, lr = tid & (QU_ROWS - 1u), pair = pair0 + r * QU_ROWS + lr, token = pair / G, h = head * G + pair % G;
        const bool live = pair < pairs;
        if (r < row_tiles) {
            // the row to shared memory as f16 numbers, its largest magnitude brought to 2^14 .. 2^15
            const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(a.query) + (live ? (size_t)(q.row + token) * a.query_row_stride + (size_t)h * a.query_head_stride : 0);
            uint32_t most_bits = 0;
            for (uint32_t i = 0; i < dim / 8 && live; ++i) {
                const uint4 w = *reinterpret_cast<const uint4*>(src + i * 8);
                const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) most_bits = max(most_bits, max(ws[k] & 0x7fffu, ws[k] >> 16 & 0x7fffu));
            }
            most_bits <<= 16;
            const int e = most_bits ? max(-100, min(100, 14 + 127 - (int)(most_bits >> 23))) : 0;
            const float up = __uint_as_float((uint32_t)(e + 127) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);
            const uint32_t my_q = q0 + r * S::Q + lr * 128u;
            for (uint32_t i = 0; i < dim / 8; ++i) {
                const uint4 w = live ? *reinterpret_cast<const uint4*>(src + i * 8) : make_uint4(0, 0, 0, 0);
                const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
                uint32_t o[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] = qu_pack(um_lo(ws[k]) * up, um_hi(ws[k]) * up);
                qu_sts(my_q + (i >> 3) * QU_BLOCK + (((i & 7u) ^ (lr & 7u)) << 4), make_uint4(o[0], o[1], o[2], o[3]));
            }
            um_fence_proxy();
            um_arrive(q_full(r));
            // of a score in units of ln 2, or (capped) of a fraction of the cap, doubled and in units of ln 2 as the exponential takes it
            const float factor = most_bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : (CAP ? 2.0f * a.scale / a.softcap : a.scale) * 1.4426950408889634f * down;
            const float cap = a.softcap * 1.4426950408889634f;
            const uint32_t index = q.length + token, lowest = a.window && index >= a.window ? index - a.window + 1u : 0u, tm = tmem + ((warp & 3u) << 21);
            // bits of the keys [first, first + 32) that the row sees
            auto seen = [&](uint32_t first, uint32_t groups) {
                auto below = [&](uint32_t key) { return key <= first ? 0u : key - first >= 32u ? 0xffffffffu : (1u << (key - first)) - 1u; };
                const uint32_t group_bits = (groups & 1u ? 0xffffu : 0u) | (groups & 2u ? 0xffff0000u : 0u);
                return live ? below(min(index + 1u, end)) & (~below(lowest) | below(a.keep_first)) & group_bits : 0u;
            };
            float acc[D], top = -INFINITY, sum = 0.0f, unit = 0.0f;
#pragma unroll
            for (int j = 0; j < D; ++j) acc[j] = 0.0f;
            auto capped = [&](float x) { return cap - 2.0f * cap * __frcp_rn(1.0f + qu_exp2(x)); };      // cap * tanh: within 2^-22 of the cap
            for (uint32_t i = 0;; ++i) {
                ok = um_wait(s_full(r), i & 1u, &gave_up, 0x901u);
                if (!ok) break;
                um_fence_after();
                const QuItem& item = items[i % QU_ITEMS];
                const bool more = item.more != 0;
                const uint32_t key0 = item.key0, groups = item.groups;
                const bool whole = more && groups == (1u << QU_GROUPS) - 1u && key0 + QU_KEYS <= min(token0 + 1u, end) && (!a.window || token1 - key0 < a.window);
                float factor_now = 1.0f;
                if (more) {
                    float most = -INFINITY;
#pragma unroll
                    for (uint32_t cc = 0; cc < QU_KEYS / 32; ++cc) {
                        uint32_t s[2][16];
                        um_ld16x2(tm + r * 128u + cc * 32u, tm + r * 128u + cc * 32u + 16u, s[0], s[1]);
                        const uint32_t bits = whole ? 0xffffffffu : seen(key0 + cc * 32u, groups >> (2 * cc));
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            float m = -INFINITY;
#pragma unroll
                            for (int j = 0; j < 16; ++j) m = fmaxf(m, whole || (bits >> (16 * g + j) & 1u) ? __uint_as_float(s[g][j]) : -INFINITY);
                            if (m > -INFINITY) {
                                m *= factor * item.key_scale[2 * cc + g];
                                most = fmaxf(most, CAP ? capped(m) : m);
                            }
                        }
                    }
                    if (most > top + QU_SLACK || (top == -INFINITY && most > -INFINITY)) {
                        factor_now = top == -INFINITY ? 0.0f : qu_exp2(top - most);
                        top = most;
                    }
                }
                if (i) {      // the tile before is done: its products are there when this one's scores are
#pragma unroll
                    for (int n = 0; n < D; n += 32) {
                        uint32_t o[2][16];
                        um_ld16x2(tm + S::O_COL + r * 128u + n, tm + S::O_COL + r * 128u + n + 16u, o[0], o[1]);
                        const float2 times = make_float2(unit, unit);
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            const float2 x = qu_fma2(make_float2(__uint_as_float(o[j >> 4][j & 15]), __uint_as_float(o[j >> 4][(j & 15) + 1])), times, make_float2(acc[n + j], acc[n + j + 1]));
                            acc[n + j] = x.x;
                            acc[n + j + 1] = x.y;
                        }
                    }
                }
                if (!more) break;
                if (__any_sync(0xffffffffu, factor_now != 1.0f)) {
#pragma unroll
                    for (int j = 0; j < D; ++j) acc[j] *= factor_now;
                }
                unit = item.unit;
                sum *= factor_now;
                const float from = top == -INFINITY ? QU_LIFT : QU_LIFT - top;
#pragma unroll
                for (uint32_t cc = 0; cc < QU_KEYS / 32; ++cc) {
                    uint32_t s[2][16], w[2][8];
                    um_ld16x2(tm + r * 128u + cc * 32u, tm + r * 128u + cc * 32u + 16u, s[0], s[1]);
                    const uint32_t bits = whole ? 0xffffffffu : seen(key0 + cc * 32u, groups >> (2 * cc));
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const float by = factor * item.key_scale[2 * cc + g], add = from - item.lower[2 * cc + g];
                        const float2 by2 = make_float2(by, by), add2 = make_float2(add, add);
                        float2 all = make_float2(0.0f, 0.0f);
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            float2 x = make_float2(__uint_as_float(s[g][j]), __uint_as_float(s[g][j + 1]));
                            if (CAP) x = make_float2(capped(x.x * by) + add, capped(x.y * by) + add);
                            else x = qu_fma2(x, by2, add2);
                            x = make_float2(qu_exp2(x.x), qu_exp2(x.y));
                            if (!whole) {
                                if (!(bits >> (16 * g + j) & 1u)) x.x = 0.0f;
                                if (!(bits >> (16 * g + j + 1) & 1u)) x.y = 0.0f;
                            }
                            all = qu_add2(all, x);
                            w[g][j / 2] = qu_pack(x.x, x.y);
                        }
                        sum = fmaf(all.x + all.y, item.gain[2 * cc + g], sum);
                        um_st8(tm + r * 128u + cc * 16u + g * 8u, w[g]);
                    }
                }
                um_wait_st();
                um_fence_before();
                um_arrive(p_full(r));
            }
            if (ok && live) {
                float f = 1.0f, high = top;
                if (a.sinks && sum != 0.0f) {
                    const float sink = reinterpret_cast<const float*>(a.sinks)[h] * 1.4426950408889634f;
                    high = fmaxf(top, sink);
                    f = qu_exp2(top - high);
                    sum = sum * f + qu_exp2(sink - high + QU_LIFT);
                }
                const float inv = sum != 0.0f ? f * (float)(1 << (int)QU_LIFT) / sum : 0.0f;      // (the weights' sum is lifted, the units are not)
                if (p.stats) *reinterpret_cast<float2*>(p.stats + ((size_t)(q.row + token) * a.heads + h) * 2) = make_float2(high, sum != 0.0f ? (float)(1 << (int)QU_LIFT) / sum : 0.0f);
                __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out) + (size_t)(q.row + token) * a.out_stride + (size_t)h * dim;
#pragma unroll
                for (int j = 0; j < D; j += 8)
                    if ((uint32_t)j < dim)
                        *reinterpret_cast<uint4*>(out + j) = make_uint4(um_pack(acc[j] * inv, acc[j + 1] * inv), um_pack(acc[j + 2] * inv, acc[j + 3] * inv), um_pack(acc[j + 4] * inv, acc[j + 5] * inv),
                                                                        um_pack(acc[j + 6] * inv, acc[j + 7] * inv));
            }
        }
    } else if (warp < 12) {
        // ================================ codes to numbers ================================
        um_fewer_registers<QU_CONVERT_REGS>();
        const uint32_t w = warp - 8u;
        const uint32_t* table = reinterpret_cast<const uint32_t*>(a.sequences.tables) + (size_t)sequence * a.sequences.table_stride;
        uint32_t n = 0;      // items
        // the keys or values of an item into their stage: a warp has 8 rows of each 32
        auto convert = [&](const uint8_t* codes, uint32_t to, uint32_t empty, uint32_t full, uint32_t key0, uint32_t block_of_lane, uint32_t groups, uint32_t code) {
            uint4 x[4 * S::BLOCKS];
#pragma unroll
            for (uint32_t rr = 0; rr < 4; ++rr) {
                const uint32_t row = rr * 32 + w * 8 + (lane >> 2), group = rr * 2 + (w >> 1), block = __shfl_sync(0xffffffffu, block_of_lane, group);
                const bool there = (groups >> group & 1u) && key0 + row < end;
                const uint8_t* from = codes + (((size_t)block * c.kv_heads + head) * bt + (key0 + row) % bt) * dim;
#pragma unroll
                for (uint32_t b = 0; b < S::BLOCKS; ++b) {
                    const uint32_t ch = (b * 4 + (lane & 3u)) * 16;
                    x[rr * S::BLOCKS + b] = make_uint4(0, 0, 0, 0);
                    if (there && ch < dim) x[rr * S::BLOCKS + b] = *reinterpret_cast<const uint4*>(from + ch);
                    else if (CODE == UZU_CACHE_CODE_I8) x[rr * S::BLOCKS + b] = make_uint4(0, 0, 0, 0);
                }
            }
            ok = um_wait(empty, (n / QU_STAGES & 1u) ^ 1u, &gave_up, code);
            if (!ok) return;
#pragma unroll
            for (uint32_t rr = 0; rr < 4; ++rr)
#pragma unroll
                for (uint32_t b = 0; b < S::BLOCKS; ++b) {
                    const uint32_t row = rr * 32 + w * 8 + (lane >> 2), at = to + b * QU_BLOCK + row * 128u;
                    const uint4& v = x[rr * S::BLOCKS + b];
                    const uint2 y[4] = {qu_numbers<CODE>(v.x), qu_numbers<CODE>(v.y), qu_numbers<CODE>(v.z), qu_numbers<CODE>(v.w)};
                    qu_sts(at + (((2 * (lane & 3u)) ^ (row & 7u)) << 4), make_uint4(y[0].x, y[0].y, y[1].x, y[1].y));
                    qu_sts(at + (((2 * (lane & 3u) + 1u) ^ (row & 7u)) << 4), make_uint4(y[2].x, y[2].y, y[3].x, y[3].y));
                }
            um_fence_proxy();
            um_arrive(full);
        };
        for (uint32_t t = 0; t < key_tiles && ok; ++t) {
            const uint32_t key0 = t < kept ? t * QU_KEYS : begin + (t - kept) * QU_KEYS, key = key0 + lane * 16;
            uint32_t block = c.blocks;
            float ks = 0.0f, vs = 0.0f;
            if (lane < QU_GROUPS && key < end) block = table[key / bt];
            const bool present = block < c.blocks;
            if (present) {
                const size_t pair = (size_t)block * c.kv_heads + head;
                ks = reinterpret_cast<const float*>(c.key_scales)[pair];
                vs = reinterpret_cast<const float*>(c.value_scales)[pair];
            }
            uint32_t todo = __ballot_sync(0xffffffffu, present);
            while (todo && ok) {
                const bool number = (todo >> lane & 1u) && vs > 0.0f;      // (a scale of 0 or NaN goes with any others)
                const float largest = __uint_as_float(__reduce_max_sync(0xffffffffu, number ? __float_as_uint(vs) : 0u));
                const uint32_t take = __ballot_sync(0xffffffffu, (todo >> lane & 1u) && (!number || vs * 256.0f >= largest)), zeros = __ballot_sync(0xffffffffu, vs == 0.0f);
                if (w == 0) {
                    QuItem& item = items[n % QU_ITEMS];
                    if (lane < QU_GROUPS) {
                        // log2 of two powers of two
                        const float lower = vs != vs ? vs : number ? (float)((int)(__float_as_uint(largest) >> 23) - (int)(__float_as_uint(vs) >> 23)) : 0.0f;
                        item.key_scale[lane] = ks;
                        item.lower[lane] = take >> lane & 1u ? lower : 0.0f;
                        item.gain[lane] = number ? exp2f(lower) : 1.0f;      // (of a scale that is NaN the weights are)
                    }
                    if (lane == 0) {
                        item.key0 = key0;
                        item.groups = take;
                        item.more = 1;
                        item.unit = largest * (1.0f / (float)(1 << (int)QU_LIFT));
                    }
                }
                const uint32_t s = n % QU_STAGES;
                convert(reinterpret_cast<const uint8_t*>(c.key_codes), k0 + s * S::KV, k_empty(s), k_full(s), key0, block, take, 0x902u);
                if (ok) convert(reinterpret_cast<const uint8_t*>(c.value_codes), v0 + s * S::KV, v_empty(s), v_full(s), key0, block, take & ~zeros, 0x903u);
                ++n;
                todo &= ~take;
            }
        }
        if (ok) ok = um_wait(k_empty(n % QU_STAGES), (n / QU_STAGES & 1u) ^ 1u, &gave_up, 0x904u);
        if (ok) {
            if (w == 0 && lane == 0) items[n % QU_ITEMS].more = 0;
            um_arrive(k_full(n % QU_STAGES));
        }
    } else {
        // ================================ products ================================
        um_fewer_registers<QU_ISSUE_REGS>();
        if (warp == 12) {
            // shared-memory descriptors: 128-byte swizzle, 1024 bytes between groups of 8 rows; values N-major, QU_BLOCK between blocks of 64 channels; f16 operands, f32 sums
            constexpr uint64_t desc_hi = (uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29)) << 32;
            const uint32_t idesc_s = (1u << 4) | ((QU_KEYS >> 3) << 17) | ((QU_ROWS >> 4) << 24), idesc_o = (1u << 4) | (1u << 16) | ((dim >> 3) << 17) | ((QU_ROWS >> 4) << 24);
            const uint32_t steps = dim / 16;
            auto scores = [&](uint32_t i, uint32_t r, bool more) {
                if (um_elect()) {
                    if (more)
                        for (uint32_t kk = 0; kk < steps; ++kk) {
                            const uint32_t off = (kk >> 2) * QU_BLOCK + (kk & 3u) * 32u, qa = q0 + r * S::Q + off, ka = k0 + i % QU_STAGES * S::KV + off;
                            um_mma_ss(tmem + r * 128u, desc_hi | (1u << 16) | (qa >> 4), desc_hi | (1u << 16) | (ka >> 4), idesc_s, kk != 0);
                        }
                    um_commit(s_full(r));
                    if (more && r + 1 == row_tiles) um_commit(k_empty(i % QU_STAGES));
                }
                um_arrive(s_full(r));      // (what the converting warps say of the tile is handed on with it)
            };
            for (uint32_t r = 0; r < row_tiles && ok; ++r) ok = um_wait(q_full(r), 0, &gave_up, 0x905u);
            if (ok) ok = um_wait(k_full(0), 0, &gave_up, 0x906u);
            um_fence_after();
            bool more = false;
            if (ok) {
                more = items[0].more != 0;
                for (uint32_t r = 0; r < row_tiles; ++r) scores(0, r, more);
            }
            for (uint32_t i = 0; more && ok; ++i) {
                const uint32_t next = i + 1;
                bool next_more = false;
                for (uint32_t r = 0; r < row_tiles && ok; ++r) {
                    if (r == 0) ok = um_wait(v_full(i % QU_STAGES), i / QU_STAGES & 1u, &gave_up, 0x907u);
                    if (ok) ok = um_wait(p_full(r), i & 1u, &gave_up, 0x908u);
                    if (!ok) break;
                    um_fence_after();
                    if (um_elect()) {
                        for (uint32_t kk = 0; kk < QU_KEYS / 16; ++kk) {
                            const uint32_t va = v0 + i % QU_STAGES * S::KV + kk * 2048u;
                            um_mma_ts(tmem + S::O_COL + r * 128u, tmem + r * 128u + kk * 8u, desc_hi | ((uint64_t)(QU_BLOCK >> 4) << 16) | (va >> 4), idesc_o, kk != 0);
                        }
                        if (r + 1 == row_tiles) um_commit(v_empty(i % QU_STAGES));
                    }
                    __syncwarp();
                    if (r == 0) {
                        ok = um_wait(k_full(next % QU_STAGES), next / QU_STAGES & 1u, &gave_up, 0x909u);
                        if (!ok) break;
                        um_fence_after();
                        next_more = items[next % QU_ITEMS].more != 0;
                    }
                    scores(next, r, next_more);
                }
                more = next_more;
            }
            if (!ok) {
                if (um_elect()) um_commit(last_products);
                __syncwarp();
                um_settle(last_products, 0);      // none in flight when tensor memory is given back
            }
        }
    }
    um_fence_before();
    __syncthreads();
    if (warp == 0) {
        um_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
        if (lane == 0) um_report(&gave_up, p.error);
    }
}

template <int CODE, int D, bool CAP>
void qu_launch(uzu_command_buffer* cmd, const QuParams& p, dim3 grid) {
    static std::atomic<uint64_t> opted{0};
    opt_in_dynamic_smem(cmd, quantized_cache_umma_kernel<CODE, D, CAP>, (int)QuShape<D>::SMEM, opted);
    launch(cmd, "quantized_cache_umma_kernel", quantized_cache_umma_kernel<CODE, D, CAP>, grid, dim3(QU_THREADS), QuShape<D>::SMEM, p);
}

}  // namespace

bool quantized_cache_umma_applicable(const uzu_quantized_cache_attention_args& a) {
    return a.data_type == UZU_DT_BF16 && a.cache.head_dim <= 128 && a.scale > 0.0f && ((a.query | a.out) & 15u) == 0 && a.query_row_stride % 8 == 0 && a.query_head_stride % 8 == 0 && a.out_stride % 8 == 0 &&
           (uint64_t)std::min(a.sequences.max_rows, a.sequences.rows) * (a.heads / a.cache.kv_heads) > kCacheFewPairs;
}

// sequences with more than kCacheFewPairs pairs of a row and a head of a key head's group
void encode_quantized_cache_umma(uzu_command_buffer* cmd, const uzu_quantized_cache_attention_args& a, uint64_t row_stats) {
    QuParams p{};
    p.a = a;
    p.capacity = cache_capacity(a.sequences, a.cache.block_tokens);
    p.group = a.heads / a.cache.kv_heads;
    p.stats = reinterpret_cast<float*>(row_stats);
    p.error = cmd->ctx->wait_errors.device_word;
    const uint64_t pairs = (uint64_t)std::min(a.sequences.max_rows, a.sequences.rows) * p.group;
    const dim3 grid((uint32_t)((pairs + 2 * QU_ROWS - 1) / (2 * QU_ROWS)), a.cache.kv_heads, a.sequences.count);
    auto caps = [&](auto code, auto d) {
        if (a.softcap > 0.0f) qu_launch<decltype(code)::value, decltype(d)::value, true>(cmd, p, grid);
        else qu_launch<decltype(code)::value, decltype(d)::value, false>(cmd, p, grid);
    };
    auto dims = [&](auto code) {
        if (a.cache.head_dim <= 64) caps(code, std::integral_constant<int, 64>());
        else caps(code, std::integral_constant<int, 128>());
    };
    if (a.cache.code_type == UZU_CACHE_CODE_I8) dims(std::integral_constant<int, UZU_CACHE_CODE_I8>());
    else dims(std::integral_constant<int, UZU_CACHE_CODE_E4M3>());
}

}  // namespace uzu
