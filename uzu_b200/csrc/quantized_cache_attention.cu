// Attention of a few rows over the 8-bit cache, and the sums of attention weight for each of its tokens.
//
// A CTA has 16 (row, head) pairs of a key head and a part of the keys they see; its four warps take 16 keys at a time, in turns. Bytes go by cp.async into a ring that each lane
// keeps for itself (it reads what it copied, so a step needs no barrier) and become f16 numbers in registers, exactly; products run on mma.sync m16n8k16 with the pairs as rows:
//   scores  a lane copies 16 codes in a row of a key, which are its four channels of four products; the order of channels within a sum is free as long as the query has the same;
//   output  a lane copies a row of codes of four keys, the keys of its own weights, and pairs them by bytes: the column of a product is any channel.
// So no code is exchanged and nothing is converted twice. A step's products start from zero and are added to the f32 sums times the block's scale; scales of keys multiply scores.
// Queries are brought to 2^14 .. 2^15 by a power of two for each row, which is exact; f32 ones are two f16 parts. A weight, up to 2^15, is two f16 parts: with one, every
// eighth bf16 result or so would be the neighbour of the right one.
#include "quantized_cache.cuh"

namespace uzu {

namespace {

constexpr uint32_t QA_WARPS = 4, QA_THREADS = QA_WARPS * 32, QA_ROWS = 16, QA_STEP = 16;
constexpr uint32_t QA_TICKETS = 16384;      // words at the start of the scratch
constexpr float QA_LIFT = 15.0f;            // weights are relative to 2^-15 of the largest so far: 22 bits down to 2^-29 of it, and off by 2^-40 of it at most below that

struct QaParams {
    uzu_quantized_cache_attention_args a;
    uint32_t capacity, group, tiles, splits;
    uint32_t* tickets;
    float *partials, *stats;      // stats: of every row and head, the largest score (in units of ln 2) and what a weight is multiplied by; null: not asked for
};

template <int DP>
struct QaShape {
    static constexpr uint32_t STEP_BYTES = 32 * DP, STAGE = STEP_BYTES + 128, STAGES = DP == 256 ? 3 : 4, RING = QA_WARPS * STAGES * STAGE;
    static constexpr uint32_t K_LOADS = DP / 32, V_UNIT = DP == 64 ? 8 : 16, V_UNITS = DP == 64 ? 1 : DP / 128;
    static constexpr uint32_t QUERY = DP / 16 * 512;      // one part's fragments
};

__device__ __forceinline__ uint32_t qa_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void qa_copy16(uint32_t to, const void* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void qa_copy8(uint32_t to, const void* from, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(there ? 8u : 0u) : "memory");
}
__device__ __forceinline__ void qa_copy4(uint32_t to, const void* from) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void qa_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void qa_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 qa_lds16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint2 qa_lds8(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void qa_mma(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float qa_exp2(float x) {      // 2 ulp; weights below 2^-126 are zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t qa_pack(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 qa_unpack(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
// 1024 + (a byte ^ 0x80) as an f16 number, less 1152: the signed byte
__device__ __forceinline__ uint32_t qa_i8_f16x2(uint32_t biased) {
    const uint32_t off = 0x64806480u;
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&biased), *reinterpret_cast<const __half2*>(&off));
    return *reinterpret_cast<const uint32_t*>(&v);
}
// four codes of a word as two pairs
template <int CODE>
__device__ __forceinline__ void qa_pairs(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if (CODE == UZU_CACHE_CODE_I8) {
        w ^= 0x80808080u;
        lo = qa_i8_f16x2(__byte_perm(w, 0x64646464u, 0x4140));
        hi = qa_i8_f16x2(__byte_perm(w, 0x64646464u, 0x4342));
    } else {
        lo = cache_e4m3x2_f16x2(w);
        hi = cache_e4m3x2_f16x2(w >> 16);
    }
}

// Steps of 16 keys that rows of tokens [first, last] of a sequence can see: the first kept ones, then the window's.
struct QaSteps {
    uint32_t kept, begin, steps, end;      // steps of first keys, the window's first key (a multiple of 16), all steps, one behind the last key
    __device__ __forceinline__ QaSteps(uint32_t first, uint32_t last, uint32_t window, uint32_t keep_first, uint32_t capacity) {
        end = min(last + 1u, capacity);
        begin = window && first >= window ? (first - window + 1u) & ~(QA_STEP - 1u) : 0u;
        kept = (min(keep_first, begin) + QA_STEP - 1u) / QA_STEP;
        steps = kept + (end > begin ? (end - begin + QA_STEP - 1u) / QA_STEP : 0u);
        if (begin >= end) {      // (a capacity that ends before the window)
            kept = (min(min(keep_first, begin), end) + QA_STEP - 1u) / QA_STEP;
            steps = kept;
        }
    }
    __device__ __forceinline__ uint32_t key(uint32_t step) const { return step < kept ? step * QA_STEP : begin + (step - kept) * QA_STEP; }
};

// The queries of a tile of 16 pairs as fragments of operand A, in shared memory: part, product, lane. Pair r is row r / group, head r % group of the key head.
// factor[r]: what a sum of products is multiplied by (but for the block's scale) to become a score in units of ln 2, or a fraction of the cap.
template <typename T, int DP>
__device__ __forceinline__ void qa_query(const QaParams& p, const CacheSequence& q, uint32_t head0, uint32_t pair0, uint32_t pairs, uint32_t at, float* factor) {
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
    const uzu_quantized_cache_attention_args& a = p.a;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3u, dim = a.cache.head_dim;
    if (warp >= 2) return;      // warp 0: rows 0 .. 7, warp 1: rows 8 .. 15
    const uint32_t row = g + 8 * warp, r = pair0 + row;
    const T* from = reinterpret_cast<const T*>(a.query);
    const bool there = r < pairs;
    if (there) from += (size_t)(q.row + r / p.group) * a.query_row_stride + (size_t)(head0 + r % p.group) * a.query_head_stride;
    uint32_t most = 0;
    for (uint32_t s = 0; s < DP / 64; ++s) {
        const uint32_t d0 = s * 64 + c * 16;
        if (there && d0 < dim)
            for (uint32_t j = 0; j < 16; ++j) {
                const float v = sizeof(T) == 4 ? *reinterpret_cast<const float*>(from + d0 + j) : sizeof(T) == 2 && a.data_type == UZU_DT_F16 ? __half2float(reinterpret_cast<const __half*>(from)[d0 + j]) : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(from)[d0 + j]);
                most = max(most, __float_as_uint(v) & 0x7fffffffu);
            }
    }
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const int e = most ? max(-100, min(100, 14 + 127 - (int)(most >> 23))) : 0;
    const float up = __uint_as_float((uint32_t)(e + 127) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);
    if (c == 0) factor[row] = most >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : a.softcap > 0.0f ? a.scale / a.softcap * down : a.scale * 1.4426950408889634f * down;
    for (uint32_t s = 0; s < DP / 64; ++s) {
        const uint32_t d0 = s * 64 + c * 16;
        for (uint32_t k = 0; k < 4; ++k) {
            float x[4];
            for (uint32_t j = 0; j < 4; ++j) {
                x[j] = 0.0f;
                if (there && d0 < dim) {
                    const uint32_t i = d0 + 4 * k + j;
                    x[j] = up * (sizeof(T) == 4 ? *reinterpret_cast<const float*>(from + i) : sizeof(T) == 2 && a.data_type == UZU_DT_F16 ? __half2float(reinterpret_cast<const __half*>(from)[i]) : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(from)[i]));
                }
            }
            for (int part = 0; part < PARTS; ++part) {
                const uint32_t lo = qa_pack(x[0], x[1]), hi = qa_pack(x[2], x[3]);
                // fragment words: 0 row g first pair, 1 row g + 8 first pair, 2 row g second pair, 3 row g + 8 second pair
                const uint32_t to = at + part * QaShape<DP>::QUERY + (s * 4 + k) * 512 + lane * 16 + warp * 4;
                asm volatile("st.shared.u32 [%0], %1;" ::"r"(to), "r"(lo) : "memory");
                asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + 8), "r"(hi) : "memory");
                if (part + 1 < PARTS) {
                    const float2 l = qa_unpack(lo), h = qa_unpack(hi);
                    x[0] -= l.x; x[1] -= l.y; x[2] -= h.x; x[3] -= h.y;
                }
            }
        }
    }
}

// what a row of this lane sees
struct QaRow {
    uint32_t index;      // the row's token
    bool live;
    __device__ __forceinline__ bool sees(uint32_t key, uint32_t end, uint32_t window, uint32_t keep_first) const {
        return live && key <= index && key < end && (!window || index - key < window || key < keep_first);
    }
};

// A score from a sum of products
__device__ __forceinline__ float qa_score(float sum, float factor, float cap) {
    const float x = sum * factor;
    return cap > 0.0f ? cap * 1.4426950408889634f * tanhf(x) : x;
}

template <typename T, int CODE, int DP>
__global__ void __launch_bounds__(QA_THREADS) quantized_cache_attention_kernel(const __grid_constant__ QaParams p) {
    using S = QaShape<DP>;
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
    extern __shared__ __align__(128) uint8_t qa_raw[];
    __shared__ float factors[QA_ROWS], tops[QA_WARPS][QA_ROWS], sums[QA_WARPS][QA_ROWS];
    __shared__ uint32_t last_of_all;
    const uzu_quantized_cache_attention_args& a = p.a;
    const uzu_quantized_cache& c = a.cache;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, g = lane >> 2, quad = lane & 3u;
    const uint32_t ring = qa_smem(qa_raw) + warp * S::STAGES * S::STAGE, query = qa_smem(qa_raw) + S::RING;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t sequence = blockIdx.z, head = blockIdx.y, split = blockIdx.x % p.splits, tile = blockIdx.x / p.splits;
    const CacheSequence q = cache_sequence(a.sequences, p.capacity, sequence);
    const uint32_t pairs = q.rows * p.group, pair0 = tile * QA_ROWS;
    if (pair0 >= pairs) return;
    const uint32_t dim = c.head_dim, bt = c.block_tokens;
    const uint32_t token0 = q.length + pair0 / p.group, token1 = q.length + min(pair0 + QA_ROWS - 1u, pairs - 1u) / p.group;
    const QaSteps steps(token0, token1, a.window, a.keep_first, p.capacity);
    const uint32_t from = (uint32_t)((uint64_t)steps.steps * split / p.splits), to = (uint32_t)((uint64_t)steps.steps * (split + 1) / p.splits);

    const uint32_t* table = reinterpret_cast<const uint32_t*>(a.sequences.tables) + (size_t)sequence * a.sequences.table_stride;
    auto copy = [&](uint32_t step, uint32_t slot) {
        if (step < to) {
            const uint32_t key0 = steps.key(step), block = table[key0 / bt], at = ring + slot * S::STAGE;
            const bool there = block < c.blocks;
            const size_t pair = (size_t)(there ? block : 0u) * c.kv_heads + head;
            const uint32_t in_block = key0 % bt, left = steps.end - key0;      // keys of the step that are there
            const uint8_t *keys = reinterpret_cast<const uint8_t*>(c.key_codes) + (pair * bt + in_block) * dim, *values = reinterpret_cast<const uint8_t*>(c.value_codes) + (pair * bt + in_block) * dim;
#pragma unroll
            for (uint32_t n = 0; n < S::K_LOADS; ++n) {
                const uint32_t key = (n & 1u) * 8 + g, d = (n >> 1) * 64 + quad * 16;
                const bool ok = there && key < left && d < dim;
                qa_copy16(at + n * 512 + lane * 16, keys + (ok ? key * dim + d : 0u), ok);
            }
#pragma unroll
            for (uint32_t n = 0; n < 4 * S::V_UNITS; ++n) {
                const uint32_t k = n & 3u, key = (k >> 1) * 8 + quad * 2 + (k & 1u), d = (g + 8 * (n >> 2)) * S::V_UNIT;
                const bool ok = there && key < left && d < dim;
                const uint32_t to_v = at + 16 * DP + n * (32 * S::V_UNIT) + lane * S::V_UNIT;
                if (S::V_UNIT == 16) qa_copy16(to_v, values + (ok ? key * dim + d : 0u), ok);
                else qa_copy8(to_v, values + (ok ? key * dim + d : 0u), ok);
            }
            if (lane < 2) qa_copy4(at + S::STEP_BYTES + lane * 4, reinterpret_cast<const float*>(lane ? c.value_scales : c.key_scales) + pair);
            if (lane == 2) asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + S::STEP_BYTES + 8), "r"((uint32_t)there) : "memory");
        }
        qa_commit();
    };
#pragma unroll
    for (uint32_t s = 0; s < S::STAGES - 1; ++s) copy(from + warp + s * QA_WARPS, s);
    qa_query<T, DP>(p, q, head * p.group, pair0, pairs, query, factors);
    __syncthreads();

    QaRow row[2];
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f}, factor[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t r = pair0 + g + 8 * h;
        row[h].live = r < pairs;
        row[h].index = q.length + (r < pairs ? r : pairs - 1u) / p.group;
        factor[h] = factors[g + 8 * h];
    }
    float acc[DP / 8][4];
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;

    uint32_t slot = 0;
    for (uint32_t step = from + warp; step < to; step += QA_WARPS) {
        copy(step + (S::STAGES - 1) * QA_WARPS, slot ? slot - 1 : S::STAGES - 1);
        qa_wait<S::STAGES - 1>();
        __syncwarp();
        const uint32_t at = ring + slot * S::STAGE, key0 = steps.key(step);
        slot = slot + 1 == S::STAGES ? 0 : slot + 1;
        float key_scale, value_scale;
        uint32_t there;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(key_scale) : "r"(at + S::STEP_BYTES) : "memory");
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(value_scale) : "r"(at + S::STEP_BYTES + 4) : "memory");
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(there) : "r"(at + S::STEP_BYTES + 8) : "memory");
        if (!there) {
            __syncwarp();
            continue;
        }

        float s[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][i] = 0.0f;
#pragma unroll
        for (int b = 0; b < DP / 64; ++b) {
            const uint4 w[2] = {qa_lds16(at + (2 * b) * 512 + lane * 16), qa_lds16(at + (2 * b + 1) * 512 + lane * 16)};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
#pragma unroll
                for (int part = PARTS - 1; part >= 0; --part) {
                    const uint4 f = qa_lds16(query + part * S::QUERY + (b * 4 + k) * 512 + lane * 16);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        uint32_t lo, hi;
                        qa_pairs<CODE>(reinterpret_cast<const uint32_t*>(&w[t])[k], lo, hi);
                        qa_mma(s[t], f, lo, hi);
                    }
                }
            }
        }
        // keys 8 t + 2 quad, + 1 of rows g, g + 8
        const bool all = key0 + QA_STEP - 1 <= token0 && key0 + QA_STEP <= steps.end && (!a.window || token1 - key0 < a.window);
        float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = qa_score(s[t][i], factor[i >> 1] * key_scale, a.softcap);
                if (!all && !row[i >> 1].sees(key0 + 8 * t + 2 * quad + (i & 1), steps.end, a.window, a.keep_first)) x = -INFINITY;
                s[t][i] = x;
                most[i >> 1] = fmaxf(most[i >> 1], x);
            }
        float keep[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            most[h] = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], 1));
            most[h] = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], 2));
            const float next = fmaxf(top[h], most[h]);
            keep[h] = next == top[h] ? 1.0f : qa_exp2(top[h] - next);
            top[h] = next;
        }
        uint4 hi_part, lo_part;
        {
            float w[2][4], add[2] = {0.0f, 0.0f};
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float base = top[i >> 1] == -INFINITY ? 0.0f : top[i >> 1] - QA_LIFT;
                    w[t][i] = qa_exp2(s[t][i] - base);
                    add[i >> 1] += w[t][i];
                }
#pragma unroll
            for (int h = 0; h < 2; ++h) sum[h] = sum[h] * keep[h] + add[h];
            uint32_t hi[4], lo[4];      // fragment words: row g of tile 0, row g + 8 of tile 0, row g of tile 1, row g + 8 of tile 1
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const float x = w[n >> 1][(n & 1) * 2], y = w[n >> 1][(n & 1) * 2 + 1];
                hi[n] = qa_pack(x, y);
                const float2 r = qa_unpack(hi[n]);
                lo[n] = qa_pack(x - r.x, y - r.y);
            }
            hi_part = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            lo_part = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        // a block whose scale is NaN makes the rows NaN that see one of its keys here, and no others
        float times[2] = {value_scale, value_scale};
        if (value_scale != value_scale) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                bool any = all;
                for (uint32_t k = 0; k < QA_STEP; ++k) any |= row[h].sees(key0 + k, steps.end, a.window, a.keep_first);
                if (!any) times[h] = 0.0f;
            }
        }
        const bool moved = __any_sync(0xffffffffu, keep[0] != 1.0f || keep[1] != 1.0f);
#pragma unroll
        for (int u = 0; u < (int)S::V_UNITS; ++u) {
            uint32_t v[4][S::V_UNIT / 4];      // key, word
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t v_at = at + 16 * DP + (u * 4 + k) * (32 * S::V_UNIT) + lane * S::V_UNIT;
                if (S::V_UNIT == 16) {
                    const uint4 x = qa_lds16(v_at);
                    v[k][0] = x.x; v[k][1] = x.y;
                    v[k][S::V_UNIT / 4 - 2] = x.z; v[k][S::V_UNIT / 4 - 1] = x.w;
                } else {
                    const uint2 x = qa_lds8(v_at);
                    v[k][0] = x.x; v[k][1] = x.y;
                }
            }
#pragma unroll
            for (int w = 0; w < (int)S::V_UNIT / 4; ++w) {
                uint32_t b[4][2];      // channel, pair of keys
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    uint32_t x = v[2 * k][w], y = v[2 * k + 1][w];
                    if (CODE == UZU_CACHE_CODE_I8) { x ^= 0x80808080u; y ^= 0x80808080u; }
                    const uint32_t lo = __byte_perm(x, y, 0x5140), hi = __byte_perm(x, y, 0x7362);
                    if (CODE == UZU_CACHE_CODE_I8) {
                        b[0][k] = qa_i8_f16x2(__byte_perm(lo, 0x64646464u, 0x4140));
                        b[1][k] = qa_i8_f16x2(__byte_perm(lo, 0x64646464u, 0x4342));
                        b[2][k] = qa_i8_f16x2(__byte_perm(hi, 0x64646464u, 0x4140));
                        b[3][k] = qa_i8_f16x2(__byte_perm(hi, 0x64646464u, 0x4342));
                    } else {
                        b[0][k] = cache_e4m3x2_f16x2(lo);
                        b[1][k] = cache_e4m3x2_f16x2(lo >> 16);
                        b[2][k] = cache_e4m3x2_f16x2(hi);
                        b[3][k] = cache_e4m3x2_f16x2(hi >> 16);
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    qa_mma(d, lo_part, b[j][0], b[j][1]);
                    qa_mma(d, hi_part, b[j][0], b[j][1]);
                    float(&o)[4] = acc[u * 16 + w * 4 + j];
                    if (moved) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[i] *= keep[i >> 1];
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = fmaf(d[i], times[i >> 1], o[i]);
                }
            }
        }
        __syncwarp();      // (the scales are read before the slot is filled again)
    }
    qa_wait<0>();

    // ---- the warps' sums: [row][channel] each, in the place of the rings ----
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
        if (quad == 0) {
            tops[warp][g + 8 * h] = top[h];
            sums[warp][g + 8 * h] = sum[h];
        }
    }
    __syncthreads();
    float* const all_sums = reinterpret_cast<float*>(qa_raw);
    float whole[2];      // the largest score of the row over the warps
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        whole[h] = -INFINITY;
#pragma unroll
        for (int w = 0; w < (int)QA_WARPS; ++w) whole[h] = fmaxf(whole[h], tops[w][g + 8 * h]);
        const float f = top[h] == whole[h] ? 1.0f : qa_exp2(top[h] - whole[h]);
        float* out = all_sums + (size_t)warp * (QA_ROWS * DP) + (g + 8 * h) * DP;
#pragma unroll
        for (int u = 0; u < (int)S::V_UNITS; ++u)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int n = 0; n < (int)S::V_UNIT; n += 4) {
                    const int at = u * 16 + n;
                    *reinterpret_cast<float4*>(out + (2 * quad + j + 8 * u) * S::V_UNIT + n) =
                        make_float4(acc[at][2 * h + j] * f, acc[at + 1][2 * h + j] * f, acc[at + 2][2 * h + j] * f, acc[at + 3][2 * h + j] * f);
                }
    }
    __syncthreads();
    const uint32_t rows = min(QA_ROWS, pairs - pair0), quads = dim / 4;
    auto row_top = [&](uint32_t r) {
        float m = tops[0][r];
#pragma unroll
        for (int w = 1; w < (int)QA_WARPS; ++w) m = fmaxf(m, tops[w][r]);
        return m;
    };
    auto row_sum = [&](uint32_t r, float m) {
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < (int)QA_WARPS; ++w) l += sums[w][r] * (tops[w][r] == m ? 1.0f : qa_exp2(tops[w][r] - m));
        return l;
    };
    auto row_quad = [&](uint32_t r, uint32_t n) {
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < (int)QA_WARPS; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(all_sums + (size_t)w * (QA_ROWS * DP) + r * DP + n * 4);
            o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
        }
        return o;
    };
    // a row's numbers, with the sink in its sum
    auto finish = [&](uint32_t r, uint32_t n, float m, float l, float4 o) {
        const uint32_t pair = pair0 + r, t = q.row + pair / p.group, h = head * p.group + pair % p.group;
        float f = 1.0f, base = m;
        if (a.sinks && l != 0.0f) {
            const float sink = reinterpret_cast<const float*>(a.sinks)[h] * 1.4426950408889634f;
            base = fmaxf(m, sink);
            f = m == base ? 1.0f : qa_exp2(m - base);
            l = l * f + qa_exp2(sink - base + QA_LIFT);
        }
        const float inv = l != 0.0f ? f / l : 0.0f;
        if (p.stats && n == 0) *reinterpret_cast<float2*>(p.stats + ((size_t)t * a.heads + h) * 2) = make_float2(base, l != 0.0f ? exp2f(QA_LIFT) / l : 0.0f);
        T* out = reinterpret_cast<T*>(a.out) + (size_t)t * a.out_stride + (size_t)h * dim + n * 4;
        const float v[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) out[i] = v[i];
            else if (a.data_type == UZU_DT_F16) reinterpret_cast<__half*>(out)[i] = __float2half_rn(v[i]);
            else reinterpret_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v[i]);
        }
    };
    if (p.splits == 1) {
        for (uint32_t i = tid; i < rows * quads; i += QA_THREADS) {
            const uint32_t r = i / quads, n = i % quads;
            const float m = row_top(r);
            finish(r, n, m, row_sum(r, m), row_quad(r, n));
        }
        return;
    }
    // ---- several CTAs: the last to be ready adds up what each has left, in their order ----
    const size_t place = ((size_t)sequence * gridDim.y + head) * p.tiles + tile;
    float* const mine = p.partials + (place * p.splits + split) * (QA_ROWS * (dim + 2));
    for (uint32_t i = tid; i < rows * quads; i += QA_THREADS) {
        const uint32_t r = i / quads, n = i % quads;
        reinterpret_cast<float4*>(mine)[r * quads + n] = row_quad(r, n);
        if (n == 0) {
            const float m = row_top(r);
            *reinterpret_cast<float2*>(mine + QA_ROWS * dim + r * 2) = make_float2(m, row_sum(r, m));
        }
    }
    __threadfence();
    __syncthreads();
    if (tid == 0) {
        const uint32_t before = atomicAdd(p.tickets + place, 1u);
        last_of_all = before == p.splits - 1;
        if (last_of_all) p.tickets[place] = 0;
    }
    __syncthreads();
    if (!last_of_all) return;
    __threadfence();
    const float* const theirs = p.partials + place * p.splits * (QA_ROWS * (dim + 2));
    for (uint32_t i = tid; i < rows * quads; i += QA_THREADS) {
        const uint32_t r = i / quads, n = i % quads;
        float m = -INFINITY, l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
        for (uint32_t z = 0; z < p.splits; ++z) {
            const float* part = theirs + (size_t)z * (QA_ROWS * (dim + 2));
            const float2 ml = *reinterpret_cast<const float2*>(part + QA_ROWS * dim + r * 2);
            const float4 x = reinterpret_cast<const float4*>(part)[r * quads + n];
            const float next = fmaxf(m, ml.x), keep = m == next ? 1.0f : qa_exp2(m - next), f = ml.x == next ? 1.0f : qa_exp2(ml.x - next);
            l = l * keep + ml.y * f;
            o.x = o.x * keep + x.x * f; o.y = o.y * keep + x.y * f; o.z = o.z * keep + x.z * f; o.w = o.w * keep + x.w * f;
            m = next;
        }
        finish(r, n, m, l, o);
    }
}

// The weight of each key, summed over the last rows of its sequence and the heads of its key head, in the order of the pairs: scores once more, with the rows' maxima and sums.
template <typename T, int CODE, int DP>
__global__ void __launch_bounds__(QA_THREADS) quantized_cache_weights_kernel(const __grid_constant__ QaParams p) {
    using S = QaShape<DP>;
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
    extern __shared__ __align__(128) uint8_t qa_raw[];
    __shared__ float factors[QA_ROWS];
    const uzu_quantized_cache_attention_args& a = p.a;
    const uzu_quantized_cache& c = a.cache;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, g = lane >> 2, quad = lane & 3u, query = qa_smem(qa_raw);
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t sequence = blockIdx.z, head = blockIdx.y;
    const CacheSequence q = cache_sequence(a.sequences, p.capacity, sequence);
    const uint32_t pairs = q.rows * p.group, dim = c.head_dim, bt = c.block_tokens;
    const uint32_t* table = reinterpret_cast<const uint32_t*>(a.sequences.tables) + (size_t)sequence * a.sequences.table_stride;
    for (uint32_t pair0 = (q.rows - min(q.rows, a.weight_rows)) * p.group; pair0 < pairs; pair0 += QA_ROWS) {
        __syncthreads();
        qa_query<T, DP>(p, q, head * p.group, pair0, pairs, query, factors);
        __syncthreads();
        const uint32_t token0 = q.length + pair0 / p.group, token1 = q.length + min(pair0 + QA_ROWS - 1u, pairs - 1u) / p.group;
        const QaSteps steps(token0, token1, a.window, a.keep_first, p.capacity);
        QaRow row[2];
        float factor[2], base[2], times[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t r = pair0 + g + 8 * h, pair = r < pairs ? r : pairs - 1u;
            row[h].live = r < pairs;
            row[h].index = q.length + pair / p.group;
            factor[h] = factors[g + 8 * h];
            const float2 st = *reinterpret_cast<const float2*>(p.stats + ((size_t)(q.row + pair / p.group) * a.heads + head * p.group + pair % p.group) * 2);
            base[h] = st.x == -INFINITY ? 0.0f : st.x;
            times[h] = st.y;
        }
        // a key is always the same warp's, whatever the tile of rows: steps are named by their first key
        const uint32_t stride = gridDim.x * QA_WARPS, mine = blockIdx.x * QA_WARPS + warp;
        for (uint32_t step = 0; step < steps.steps; ++step) {
            const uint32_t key0 = steps.key(step);
            const uint32_t owner = key0 / QA_STEP % stride;
            if (owner != mine) {      // on to the next one of this warp
                const uint32_t ahead = (mine + stride - owner) % stride;
                const uint32_t run = step < steps.kept ? steps.kept - step : steps.steps - step;
                step += min(ahead, run) - 1u;
                continue;
            }
            const uint32_t block = table[key0 / bt];
            if (block >= c.blocks) continue;
            const size_t pair = (size_t)block * c.kv_heads + head;
            const uint32_t in_block = key0 % bt, left = steps.end - key0;
            const uint8_t* keys = reinterpret_cast<const uint8_t*>(c.key_codes) + (pair * bt + in_block) * dim;
            const float key_scale = reinterpret_cast<const float*>(c.key_scales)[pair];
            uint4 w[S::K_LOADS];
#pragma unroll
            for (uint32_t n = 0; n < S::K_LOADS; ++n) {
                const uint32_t key = (n & 1u) * 8 + g, d = (n >> 1) * 64 + quad * 16;
                w[n] = key < left && d < dim ? *reinterpret_cast<const uint4*>(keys + key * dim + d) : make_uint4(0, 0, 0, 0);
            }
            float s[2][4];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[t][i] = 0.0f;
#pragma unroll
            for (int b = 0; b < DP / 64; ++b)
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int part = PARTS - 1; part >= 0; --part) {
                        const uint4 f = qa_lds16(query + part * S::QUERY + (b * 4 + k) * 512 + lane * 16);
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            uint32_t lo, hi;
                            qa_pairs<CODE>(reinterpret_cast<const uint32_t*>(&w[2 * b + t])[k], lo, hi);
                            qa_mma(s[t], f, lo, hi);
                        }
                    }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t key = key0 + 8 * t + 2 * quad + j;
                    float x = 0.0f;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (row[h].sees(key, steps.end, a.window, a.keep_first)) x += qa_exp2(qa_score(s[t][2 * h + j], factor[h] * key_scale, a.softcap) - base[h]) * times[h];
                    x += __shfl_xor_sync(0xffffffffu, x, 4);
                    x += __shfl_xor_sync(0xffffffffu, x, 8);
                    x += __shfl_xor_sync(0xffffffffu, x, 16);
                    if (g == 0 && key < steps.end) reinterpret_cast<float*>(c.key_weights)[pair * bt + in_block + 8 * t + 2 * quad + j] += x;
                }
        }
    }
}

struct QaPlan {
    uint32_t group, tiles, splits, most_rows;
    uint64_t partial_bytes, stats_bytes;
};
QaPlan qa_plan(uint32_t sm_count, const uzu_quantized_cache_attention_args& a) {
    QaPlan p{};
    const uzu_cache_sequences& s = a.sequences;
    const uint32_t capacity = cache_capacity(s, a.cache.block_tokens);
    p.group = a.heads / a.cache.kv_heads;
    p.most_rows = std::min(s.max_rows, s.rows);
    p.tiles = (uint32_t)(((uint64_t)p.most_rows * p.group + QA_ROWS - 1) / QA_ROWS);
    const uint64_t ctas = (uint64_t)s.count * a.cache.kv_heads * p.tiles;
    const uint64_t keys = a.window ? std::min<uint64_t>(capacity, (uint64_t)a.window + p.most_rows + a.keep_first + 32) : capacity, steps = (keys + QA_STEP - 1) / QA_STEP;
    p.splits = 1;
    if (ctas && ctas <= QA_TICKETS) {
        const uint64_t wanted = ((uint64_t)sm_count * 3 + ctas - 1) / ctas;
        p.splits = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>({wanted, (steps + 2 * QA_WARPS - 1) / (2 * QA_WARPS), 64}));
    }
    if (p.splits > 1) p.partial_bytes = ctas * p.splits * QA_ROWS * (a.cache.head_dim + 2) * 4;
    if (a.weight_rows) p.stats_bytes = (uint64_t)s.rows * a.heads * 8;
    return p;
}
uint64_t qa_align(uint64_t v) { return (v + 255) & ~255ull; }
uint64_t qa_scratch(const QaPlan& p) { return QA_TICKETS * 4 + qa_align(p.partial_bytes) + qa_align(p.stats_bytes); }

const char* attention_check(const uzu_quantized_cache_attention_args* a) {
    if (!a) return "null arguments";
    if (a->data_type > UZU_DT_F16) return "data_type must be bf16, f32 or f16";
    if (const char* e = check_cache(a->cache)) return e;
    if (const char* e = check_cache_sequences(a->sequences, true)) return e;
    const uzu_cache_sequences& s = a->sequences;
    const uzu_quantized_cache& c = a->cache;
    if (!a->heads || a->heads > 65535 || a->heads % c.kv_heads) return "heads must be a multiple of kv_heads";
    if (!(a->scale == a->scale) || a->scale - a->scale != 0.0f) return "scale must be a number";
    if (!(a->softcap >= 0.0f) || a->softcap - a->softcap != 0.0f) return "softcap must be at least 0";
    const uint64_t width = (uint64_t)a->heads * c.head_dim, size = a->data_type == UZU_DT_F32 ? 4 : 2;
    if ((uint64_t)std::min(s.rows, s.max_rows) * (a->heads / c.kv_heads) >> 29) return "too many rows for one call";
    if (a->out_stride < width) return "a row is shorter than its heads";
    if (a->weight_rows && !c.key_weights) return "weight_rows without key_weights";
    if (!s.count || !s.rows) return nullptr;
    if (!a->query || !a->out || !a->scratch) return "null operand";
    if ((a->query | a->out) % size || a->sinks % 4) return "an operand is not aligned to its elements";
    if (a->scratch % 256) return "the scratch is not aligned";
    const uint64_t out_bytes = rows_extent(s.rows, a->out_stride, width, size), query_bytes = ((uint64_t)(s.rows - 1) * a->query_row_stride + (uint64_t)(a->heads - 1) * a->query_head_stride + c.head_dim) * size;
    if (cache_meets_itself(c)) return "the cache overlaps itself";
    if (meets_cache(c, a->out, out_bytes) || meets_cache(c, a->query, query_bytes) || meets_cache(c, a->scratch, a->scratch_bytes)) return "the cache overlaps another operand";
    const bool dense = a->query_head_stride == c.head_dim;      // (rows of heads side by side may be slices of the same wide rows)
    if (dense ? rows_overlap(a->query, a->query_row_stride, width, a->out, a->out_stride, width, s.rows, size) : bytes_overlap(a->query, query_bytes, a->out, out_bytes)) return "query and out overlap";
    if (meets_sequences(s, a->out, out_bytes) || meets_sequences(s, a->scratch, a->scratch_bytes)) return "an operand overlaps what says which sequences there are";
    if (bytes_overlap(a->scratch, a->scratch_bytes, a->out, out_bytes) || bytes_overlap(a->scratch, a->scratch_bytes, a->query, query_bytes)) return "the scratch overlaps rows";
    if (a->sinks && (bytes_overlap(a->sinks, a->heads * 4ull, a->out, out_bytes) || bytes_overlap(a->sinks, a->heads * 4ull, a->scratch, a->scratch_bytes) || meets_cache(c, a->sinks, a->heads * 4ull)))
        return "sinks overlap another operand";
    return nullptr;
}

template <typename F>
void qa_instance(const uzu_quantized_cache_attention_args& a, F f) {
    auto dims = [&](auto t, auto code) {
        if (a.cache.head_dim <= 64) f(t, code, std::integral_constant<int, 64>());
        else if (a.cache.head_dim <= 128) f(t, code, std::integral_constant<int, 128>());
        else f(t, code, std::integral_constant<int, 256>());
    };
    auto codes = [&](auto t) {
        if (a.cache.code_type == UZU_CACHE_CODE_I8) dims(t, std::integral_constant<int, UZU_CACHE_CODE_I8>());
        else dims(t, std::integral_constant<int, UZU_CACHE_CODE_E4M3>());
    };
    if (a.data_type == UZU_DT_F32) codes(float());
    else codes(uint16_t());
}

template <typename T, int CODE, int DP>
void qa_attend(uzu_command_buffer* cmd, const QaParams& p) {
    using S = QaShape<DP>;
    static std::atomic<uint64_t> opted{0};
    const uint32_t parts = sizeof(T) == 4 ? 2 : 1, sums = QA_WARPS * QA_ROWS * DP * 4, smem = std::max(S::RING + parts * S::QUERY, sums);
    opt_in_dynamic_smem(cmd, quantized_cache_attention_kernel<T, CODE, DP>, (int)smem, opted);
    launch(cmd, "quantized_cache_attention_kernel", quantized_cache_attention_kernel<T, CODE, DP>, dim3(p.tiles * p.splits, p.a.cache.kv_heads, p.a.sequences.count), dim3(QA_THREADS), smem, p);
}
template <typename T, int CODE, int DP>
void qa_weigh(uzu_command_buffer* cmd, const QaParams& p) {
    const uint32_t parts = sizeof(T) == 4 ? 2 : 1, ctas = p.a.sequences.count * p.a.cache.kv_heads, steps = (p.capacity + QA_STEP - 1) / QA_STEP;
    const uint32_t parts_of_keys = std::max(1u, std::min((steps + QA_WARPS - 1) / QA_WARPS, ((uint32_t)cmd->ctx->sm_count * 8 + ctas - 1) / ctas));
    launch(cmd, "quantized_cache_weights_kernel", quantized_cache_weights_kernel<T, CODE, DP>, dim3(parts_of_keys, p.a.cache.kv_heads, p.a.sequences.count), dim3(QA_THREADS), parts * QaShape<DP>::QUERY, p);
}

}  // namespace
}  // namespace uzu

using namespace uzu;

extern "C" {

size_t uzu_quantized_cache_attention_scratch_bytes(uzu_context* ctx, const uzu_quantized_cache_attention_args* a) {
    if (!ctx || !a || check_cache(a->cache) || check_cache_sequences(a->sequences, true) || !a->heads || a->heads % a->cache.kv_heads) return 0;
    return qa_scratch(qa_plan(ctx->sm_count, *a));
}

uzu_status uzu_quantized_cache_attention_validate(const uzu_quantized_cache_attention_args* a) {
    const char* e = attention_check(a);
    return e ? fail(UZU_ERROR_INVALID_ARGUMENT, std::string("quantized_cache_attention: ") + e) : UZU_OK;
}

void uzu_quantized_cache_attention_encode(uzu_command_buffer* cmd, const uzu_quantized_cache_attention_args* a) {
    if (!encodable(cmd, "quantized_cache_attention")) return;
    if (const char* e = attention_check(a)) {
        cmd->record_error(UZU_ERROR_INVALID_ARGUMENT, std::string("quantized_cache_attention: ") + e);
        return;
    }
    if (!a->sequences.count || !a->sequences.rows || !a->sequences.max_rows) return;
    const QaPlan plan = qa_plan(cmd->ctx->sm_count, *a);
    if (a->scratch_bytes < qa_scratch(plan)) {
        cmd->record_error(UZU_ERROR_INVALID_ARGUMENT, "quantized_cache_attention: the scratch is too small");
        return;
    }
    QaParams p{};
    p.a = *a;
    p.capacity = cache_capacity(a->sequences, a->cache.block_tokens);
    p.group = plan.group;
    p.tiles = plan.tiles;
    p.splits = plan.splits;
    p.tickets = reinterpret_cast<uint32_t*>(a->scratch);
    p.partials = reinterpret_cast<float*>(a->scratch + QA_TICKETS * 4);
    p.stats = a->weight_rows ? reinterpret_cast<float*>(a->scratch + QA_TICKETS * 4 + qa_align(plan.partial_bytes)) : nullptr;
    qa_instance(*a, [&](auto t, auto code, auto dim) {
        qa_attend<decltype(t), decltype(code)::value, decltype(dim)::value>(cmd, p);
        if (a->weight_rows) qa_weigh<decltype(t), decltype(code)::value, decltype(dim)::value>(cmd, p);
    });
}

}  // extern "C"
