// Attention of a few rows over the 8-bit cache, and the sums of attention weight for each of its tokens.
//
// A CTA has 8 or more (row, head) pairs of a key head and a part of the keys they see; each of its four warps takes a run of them, 32 keys at a time. Bytes go by cp.async into a
// ring that each lane keeps for itself (it reads what it copied, so a step needs no barrier) and become f16 numbers in registers, exactly. Products run on mma.sync m16n8k16 with the
// keys as rows, then the channels, and the pairs as columns, eight a product, so that few pairs waste little:
//   scores  a lane copies 16 codes in a row of a key, which are its four channels of four products; the order of channels within a sum is free as long as the query has the same;
//   output  a lane copies a row of codes of four keys, the keys of its own weights, and pairs them by bytes: the row of a product is any channel.
// So no code is exchanged and nothing is converted twice; weights are turned by movmatrix. Products of bf16 and f16 rows are added up by the tensor cores in units of the block's value
// scale, and rescaled where it changes; scales of keys multiply scores.
// Queries are brought to 2^14 .. 2^15 by a power of two for each row, which is exact; f32 ones are two f16 parts. A weight, up to 2^15, is two f16 parts: with one, every
// eighth bf16 result or so would be the neighbour of the right one.
// What bounds it: instructions and their latency, not memory: schedulers issue in 40 % of the cycles at 11 warps an SM, DRAM is busy for 43 % of the time, the tensor pipe for 15 % (capped drafted rows: 39 %, 10 warps,
// 13 % and 13 %). One row behind 131071 tokens of 8 heads of 128 (i8): 75 to 77 us, 3.6 TB/s. On the way there: 134 us first, 122 with wide loads of the queries, 82 with pairs as columns of a product, 75 with 32 keys a
// step. 64 sequences of 4096 tokens on average 170 us, the weights' sums from kept scores 34. With 16 keys a step four CTAs an SM took 100 us, five with a ring of two 106, three 113; the rings of 32 keys of heads of 128
// leave room for three, and of heads of 64 four are slower too (16 x 5 rows 65 against 55 us, registers of four spill). A grid of 448 CTAs where 444 fit at once doubled the time, so splits fill one wave.
#include "quantized_cache.cuh"

namespace uzu {

namespace {

constexpr uint32_t QA_WARPS = 4, QA_THREADS = QA_WARPS * 32, QA_STEP = 32, QA_HALF = 16;      // keys of a step, which is two halves with blocks and scales of their own
constexpr uint32_t QA_SUM = 256;
constexpr uint64_t QA_SCORES = 256u << 20;      // bytes of scores that are kept at most
constexpr uint32_t QA_TICKETS = 16384;      // words at the start of the scratch
constexpr float QA_LIFT = 15.0f;            // weights are relative to 2^-15 of the largest so far: 22 bits down to 2^-29 of it, and off by 2^-40 of it at most below that

struct QaParams {
    uzu_quantized_cache_attention_args a;
    uint32_t capacity, group, tiles, splits, shift, few;      // shift: log2 of a block's tokens; few: sequences of more pairs, and more than kCacheFewRows rows, are another kernel's
    uint32_t* tickets;
    float *partials, *stats;      // stats: of every row and head, the largest score (in units of ln 2) and what a weight is multiplied by; null: not asked for
    float* scores;                // of the sequences of few pairs: [sequence, key head, pair, score_stride]; null: not kept
    uint32_t score_stride, score_pairs, tile_rows;
};

// DP: channels a head has at most; NT: eights of pairs
template <int DP, int NT>
struct QaShape {
    static constexpr uint32_t HALF_BYTES = 32 * DP, STEP_BYTES = 2 * HALF_BYTES, STAGE = STEP_BYTES + 128, STAGES = DP == 64 ? 3 : 2, RING = QA_WARPS * STAGES * STAGE;
    static constexpr uint32_t K_LOADS = DP / 32, V_UNIT = DP == 64 ? 8 : 16, V_UNITS = DP == 64 ? 1 : DP / 128;
    static constexpr uint32_t ROWS = 8 * NT, QUERY = NT * DP / 16 * 256;      // one part's fragments
    static constexpr uint32_t CTAS = DP == 256 ? 1 : 3;                       // of an SM
    static constexpr bool KEPT = NT * DP <= 128;                              // the queries' fragments stay in registers (of one part)
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
extern __shared__ __align__(128) uint8_t qa_raw[];
__device__ __forceinline__ uint4 qa_lds16(uint32_t offset) { return *reinterpret_cast<const uint4*>(qa_raw + offset); }      // (of the dynamic shared memory)
__device__ __forceinline__ uint2 qa_lds8(uint32_t offset) { return *reinterpret_cast<const uint2*>(qa_raw + offset); }
__device__ __forceinline__ void qa_mma(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float qa_exp2(float x) {      // 2 ulp; weights below 2^-126 are zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t qa_turn(uint32_t v) {      // an 8 x 8 tile of f16 numbers
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
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

// Steps of 32 keys that rows of tokens [first, last] of a sequence can see: the first kept ones, then the window's.
struct QaSteps {
    uint32_t kept, begin, steps, end;      // steps of first keys, the window's first key (a multiple of 32), all steps, one behind the last key
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

template <typename T>
__device__ __forceinline__ float qa_number(T v, bool f16) {
    if constexpr (sizeof(T) == 4) return v;
    else return f16 ? __half2float(__ushort_as_half(v)) : __uint_as_float((uint32_t)v << 16);
}
// The queries of a tile of pairs as fragments of operand B, in shared memory: part, eight of pairs, product, lane. Pair r is row r / group, head r % group of the key head.
// factor[r]: what a sum of products is multiplied by (but for the block's scale) to become a score in units of ln 2, or a fraction of the cap. By all threads, with barriers.
template <typename T, int DP, int NT>
__device__ __forceinline__ void qa_query(const QaParams& p, const CacheSequence& q, uint32_t head0, uint32_t pair0, uint32_t pairs, uint32_t at, float* factor, uint32_t* most_of) {
    using S = QaShape<DP, NT>;
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
    constexpr uint32_t UNITS = NT * DP / 64, EACH = (UNITS + QA_WARPS - 1) / QA_WARPS;      // of 8 pairs and 64 channels, a warp's
    const uzu_quantized_cache_attention_args& a = p.a;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3u, dim = a.cache.head_dim;
    const bool f16 = a.data_type == UZU_DT_F16, wide = ((a.query | (uint64_t)a.query_row_stride * sizeof(T) | (uint64_t)a.query_head_stride * sizeof(T)) & 15u) == 0;
    if (threadIdx.x < S::ROWS) most_of[threadIdx.x] = 0;
    __syncthreads();
    alignas(16) T x[EACH][16];
#pragma unroll
    for (uint32_t e = 0; e < EACH; ++e) {
        const uint32_t u = warp + e * QA_WARPS, r = pair0 + u % NT * 8 + g, d0 = u / NT * 64 + c * 16;
#pragma unroll
        for (int j = 0; j < 16; ++j) x[e][j] = 0;
        if (u >= UNITS || r >= pairs || d0 >= dim) continue;
        const T* from = reinterpret_cast<const T*>(a.query) + (size_t)(q.row + r / p.group) * a.query_row_stride + (size_t)(head0 + r % p.group) * a.query_head_stride + d0;
        if (wide) {
#pragma unroll
            for (int j = 0; j < (int)sizeof(T); ++j) reinterpret_cast<uint4*>(x[e])[j] = reinterpret_cast<const uint4*>(from)[j];
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) x[e][j] = from[j];
        }
    }
#pragma unroll
    for (uint32_t e = 0; e < EACH; ++e) {
        const uint32_t u = warp + e * QA_WARPS;
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) most = max(most, __float_as_uint(qa_number(x[e][j], f16)) & 0x7fffffffu);
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        if (u < UNITS && c == 0) atomicMax(&most_of[u % NT * 8 + g], most);
    }
    __syncthreads();
#pragma unroll
    for (uint32_t e = 0; e < EACH; ++e) {
        const uint32_t u = warp + e * QA_WARPS, n = u % NT, s = u / NT;
        if (u >= UNITS) continue;
        const uint32_t most = most_of[n * 8 + g];
        const int power = most ? min(kCacheMostPower, 14 + 127 - (int)(most >> 23)) : 0;
        const float up = __uint_as_float((uint32_t)(power + 127) << 23), down = __uint_as_float((uint32_t)(127 - power) << 23);
        if (s == 0 && c == 0) factor[n * 8 + g] = most >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : a.softcap > 0.0f ? a.scale * down / a.softcap : a.scale * down * 1.4426950408889634f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = up * qa_number(x[e][4 * k + j], f16);
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                const uint32_t lo = qa_pack(y[0], y[1]), hi = qa_pack(y[2], y[3]);
                *reinterpret_cast<uint2*>(qa_raw + at + part * S::QUERY + ((n * (DP / 16) + s * 4 + k) * 32 + lane) * 8) = make_uint2(lo, hi);
                if (part + 1 < PARTS) {
                    const float2 l = qa_unpack(lo), h = qa_unpack(hi);
                    y[0] -= l.x; y[1] -= l.y; y[2] -= h.x; y[3] -= h.y;
                }
            }
        }
    }
    __syncthreads();
}

// what a row of this lane sees
struct QaRow {
    uint32_t index;      // the row's token
    bool live;
    __device__ __forceinline__ bool sees(uint32_t key, uint32_t end, uint32_t window, uint32_t keep_first) const {
        return live && key <= index && key < end && (!window || index - key < window || key < keep_first);
    }
};

// tanh(x) = 1 - 2 / (1 + e^2x), within 2^-22
__device__ __forceinline__ float qa_tanh(float x) { return 1.0f - 2.0f * __frcp_rn(1.0f + qa_exp2(2.8853900817779268f * x)); }

// the queries' fragments, from shared memory or, once read, from registers
template <int DP, int NT, int PARTS, bool KEPT>
struct QaQuery {
    using S = QaShape<DP, NT>;
    uint2 kept[KEPT ? NT * DP / 16 : 1];
    uint32_t at;
    __device__ __forceinline__ QaQuery(uint32_t query, uint32_t lane) : at(query + lane * 8) {
        if (KEPT) {
#pragma unroll
            for (int i = 0; i < NT * DP / 16; ++i) kept[i] = qa_lds8(at + i * 256);
        }
    }
    __device__ __forceinline__ uint2 get(int part, int i) const { return KEPT && part == 0 ? kept[i] : qa_lds8(at + part * S::QUERY + i * 256); }
};
// Scores of 16 keys (rows g, g + 8) and pairs 2 quad, + 1 of each eight, in units of ln 2 (or, with a cap, behind it); word(n): the lane's codes, of both keys by turns
template <int CODE, int DP, int NT, int PARTS, typename Query, typename Word>
__device__ __forceinline__ void qa_scores(const Query& query, Word word, const float (&factor)[NT][2], float key_scale, float softcap, float (&s)[NT][4]) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
#pragma unroll
    for (int b = 0; b < DP / 64; ++b) {
        const uint4 w[2] = {word(2 * b), word(2 * b + 1)};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint4 f;      // a key's channels: row g, row g + 8, then the second two channels of each
            qa_pairs<CODE>(reinterpret_cast<const uint32_t*>(&w[0])[k], f.x, f.z);
            qa_pairs<CODE>(reinterpret_cast<const uint32_t*>(&w[1])[k], f.y, f.w);
#pragma unroll
            for (int part = PARTS - 1; part >= 0; --part)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint2 x = query.get(part, n * (DP / 16) + b * 4 + k);
                    qa_mma(s[n], f, x.x, x.y);
                }
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const float times[2] = {factor[n][0] * key_scale, factor[n][1] * key_scale};
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] *= times[i & 1];
    }
    if (softcap > 0.0f) {
        const float cap = softcap * 1.4426950408889634f;
        if (PARTS == 1 && softcap <= kCacheFastCap) {      // (within 2^-22 of the cap, for a fifth of the instructions)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][i] = cap * qa_tanh(s[n][i]);
        } else {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][i] = cap * tanhf(s[n][i]);
        }
    }
}

template <typename T, int CODE, int DP, int NT>
__global__ void __launch_bounds__(QA_THREADS, QaShape<DP, NT>::CTAS) quantized_cache_attention_kernel(const __grid_constant__ QaParams p) {
    using S = QaShape<DP, NT>;
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
    constexpr uint32_t ROWS = S::ROWS;
    __shared__ float factors[ROWS], tops[QA_WARPS][ROWS], sums[QA_WARPS][ROWS];
    __shared__ uint32_t mosts[ROWS], last_of_all;
    const uzu_quantized_cache_attention_args& a = p.a;
    const uzu_quantized_cache& c = a.cache;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, g = lane >> 2, quad = lane & 3u;
    const uint32_t ring = warp * S::STAGES * S::STAGE, query = S::RING, raw = qa_smem(qa_raw);
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t sequence = blockIdx.z, head = blockIdx.y, split = blockIdx.x % p.splits, tile = blockIdx.x / p.splits;
    const CacheSequence q = cache_sequence(a.sequences, kCacheAnyLength, sequence);
    const uint32_t pairs = q.rows * p.group, pair0 = tile * ROWS;
    if (pair0 >= pairs || (pairs > p.few && q.rows > kCacheFewRows)) return;
    const uint32_t dim = c.head_dim, bt = c.block_tokens;
    const uint32_t token0 = q.length + pair0 / p.group, token1 = q.length + min(pair0 + ROWS - 1u, pairs - 1u) / p.group;
    const QaSteps steps(token0, token1, a.window, a.keep_first, p.capacity);
    // this warp's run of steps: neighbours share a block's scales
    const uint32_t part = split * QA_WARPS + warp, parts = p.splits * QA_WARPS;
    const uint32_t from = (uint32_t)((uint64_t)steps.steps * part / parts), to = (uint32_t)((uint64_t)steps.steps * (part + 1) / parts);

    const uint32_t* table = reinterpret_cast<const uint32_t*>(a.sequences.tables) + (size_t)sequence * a.sequences.table_stride;
    // (the blocks of the next step to be copied are asked for a step ahead: of halves 0 and 1, the same one where blocks have 32 tokens)
    uint32_t next_block[2];
    auto ask = [&](uint32_t step) {
        if (step >= to) return;
        const uint32_t key = steps.key(step);
        next_block[0] = table[key >> p.shift];
        next_block[1] = p.shift > 4 ? next_block[0] : key + QA_HALF < steps.end ? table[(key + QA_HALF) >> p.shift] : 0xffffffffu;
    };
    ask(from);
    const uint32_t k_lane = g * dim + quad * 16, v_lane = quad * 2 * dim + g * S::V_UNIT, k_to = lane * 16, v_to = 16 * DP + lane * S::V_UNIT;
    const uint8_t *const all_keys = reinterpret_cast<const uint8_t*>(c.key_codes), *const all_values = reinterpret_cast<const uint8_t*>(c.value_codes);
    const float* const all_scales = reinterpret_cast<const float*>(lane & 1u ? c.value_scales : c.key_scales);
    auto copy = [&](uint32_t step, uint32_t slot) {
        if (step < to) {
            const uint32_t key0 = steps.key(step), blocks[2] = {next_block[0], next_block[1]};
            ask(step + 1);
            const uint32_t at = raw + ring + slot * S::STAGE, left = steps.end - key0;      // keys of the step that are there
            if (blocks[0] < c.blocks && blocks[1] < c.blocks && left >= QA_STEP && dim == DP) {
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    const size_t first = ((((size_t)blocks[h] * c.kv_heads + head) << p.shift) + ((key0 + h * QA_HALF) & (bt - 1u))) * DP;
                    const uint8_t *keys = all_keys + first + k_lane, *values = all_values + first + v_lane;
#pragma unroll
                    for (uint32_t n = 0; n < S::K_LOADS; ++n) qa_copy16(at + h * S::HALF_BYTES + k_to + n * 512, keys + (n & 1u) * 8 * DP + (n >> 1) * 64, true);
#pragma unroll
                    for (uint32_t n = 0; n < 4 * S::V_UNITS; ++n) {
                        const uint8_t* v = values + ((n >> 1 & 1u) * 8 + (n & 1u)) * DP + (n >> 2) * 8 * S::V_UNIT;
                        if (S::V_UNIT == 16) qa_copy16(at + h * S::HALF_BYTES + v_to + n * (32 * S::V_UNIT), v, true);
                        else qa_copy8(at + h * S::HALF_BYTES + v_to + n * (32 * S::V_UNIT), v, true);
                    }
                }
            } else {      // a part of the step's keys, or of the channels: zeros for the rest
#pragma unroll 1
                for (uint32_t h = 0; h < 2; ++h) {
                    const bool there = blocks[h] < c.blocks;
                    const uint32_t mine = left > h * QA_HALF ? left - h * QA_HALF : 0u;
                    const size_t first = ((((size_t)(there ? blocks[h] : 0u) * c.kv_heads + head) << p.shift) + ((key0 + h * QA_HALF) & (bt - 1u))) * dim;
#pragma unroll 1
                    for (uint32_t n = 0; n < S::K_LOADS; ++n) {
                        const bool ok = there && (n & 1u) * 8 + g < mine && (n >> 1) * 64 + quad * 16 < dim;
                        qa_copy16(at + h * S::HALF_BYTES + k_to + n * 512, all_keys + (ok ? first + k_lane + (n & 1u) * 8 * dim + (n >> 1) * 64 : 0u), ok);
                    }
#pragma unroll 1
                    for (uint32_t n = 0; n < 4 * S::V_UNITS; ++n) {
                        const uint32_t key = (n >> 1 & 1u) * 8 + (n & 1u);
                        const bool ok = there && key + quad * 2 < mine && (g + 8 * (n >> 2)) * S::V_UNIT < dim;
                        const uint8_t* v = all_values + (ok ? first + v_lane + key * dim + (n >> 2) * 8 * S::V_UNIT : 0u);
                        if (S::V_UNIT == 16) qa_copy16(at + h * S::HALF_BYTES + v_to + n * (32 * S::V_UNIT), v, ok);
                        else qa_copy8(at + h * S::HALF_BYTES + v_to + n * (32 * S::V_UNIT), v, ok);
                    }
                }
            }
            // scales of keys and values of both halves, then which halves have a block
            if (lane < 4) {
                const uint32_t block = blocks[lane >> 1];
                qa_copy4(at + S::STEP_BYTES + lane * 4, all_scales + ((size_t)(block < c.blocks ? block : 0u) * c.kv_heads + head));
            }
            if (lane == 4) asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + S::STEP_BYTES + 16), "r"((blocks[0] < c.blocks ? 1u : 0u) | (blocks[1] < c.blocks ? 2u : 0u)) : "memory");
        }
        qa_commit();
    };
#pragma unroll
    for (uint32_t s = 0; s < S::STAGES - 1; ++s) copy(from + s, s);
    qa_query<T, DP, NT>(p, q, head * p.group, pair0, pairs, query, factors, mosts);

    QaRow row[NT][2];
    float top[NT][2], sum[NT][2], factor[NT][2], acc[NT][DP / 16][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t r = pair0 + n * 8 + 2 * quad + h;
            row[n][h].live = r < pairs;
            row[n][h].index = q.length + (r < pairs ? r : pairs - 1u) / p.group;
            factor[n][h] = factors[n * 8 + 2 * quad + h];
            top[n][h] = -INFINITY;
            sum[n][h] = 0.0f;
        }
#pragma unroll
        for (int m = 0; m < DP / 16; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][m][i] = 0.0f;
    }

    const QaQuery<DP, NT, PARTS, S::KEPT> fragments(query, lane);
    // what acc is counted in (0: nothing yet): a block's value scale, so that its products are added where they are made, or 1
    float unit = 0.0f;
    constexpr float LOWER = 1.0f / (1 << (int)QA_LIFT);
    uint32_t slot = 0;
    for (uint32_t step = from; step < to; ++step) {
        copy(step + S::STAGES - 1, slot ? slot - 1 : S::STAGES - 1);
        qa_wait<S::STAGES - 1>();
        __syncwarp();
        const uint32_t at = ring + slot * S::STAGE, key0 = steps.key(step);
        slot = slot + 1 == S::STAGES ? 0 : slot + 1;
        const float4 scales_at = *reinterpret_cast<const float4*>(qa_raw + at + S::STEP_BYTES);
        const float scales[4] = {scales_at.x, scales_at.y, scales_at.z, scales_at.w};      // of keys and values, of both halves
        const uint32_t there = *reinterpret_cast<const uint32_t*>(qa_raw + at + S::STEP_BYTES + 16);
        float s[2][NT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
            qa_scores<CODE, DP, NT, PARTS>(fragments, [&](int n) { return qa_lds16(at + h * S::HALF_BYTES + k_to + n * 512); }, factor, scales[2 * h], a.softcap, s[h]);
        // keys g, g + 8 of a half, pairs 2 quad, + 1 of each eight
        const bool all = there == 3 && key0 + QA_STEP - 1 <= token0 && key0 + QA_STEP <= steps.end && (!a.window || token1 - key0 < a.window);
        if (!all) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!(there >> h & 1u) || !row[n][i & 1].sees(key0 + h * QA_HALF + g + 8 * (i >> 1), steps.end, a.window, a.keep_first)) s[h][n][i] = -INFINITY;
        }
        if (p.scores && pairs <= p.score_pairs) {      // (for the weights' sums)
            float* const mine = p.scores + (((size_t)sequence * c.kv_heads + head) * p.score_pairs + pair0) * p.score_stride + key0;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (row[n][e].live) {
                        float* at_row = mine + (size_t)(n * 8 + 2 * quad + e) * p.score_stride + g;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            at_row[h * QA_HALF] = s[h][n][e];
                            at_row[h * QA_HALF + 8] = s[h][n][2 + e];
                        }
                    }
        }
        float keep[NT][2];
        bool moved = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float most = fmaxf(fmaxf(s[0][n][e], s[0][n][2 + e]), fmaxf(s[1][n][e], s[1][n][2 + e]));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
                const float next = fmaxf(top[n][e], most);
                keep[n][e] = next == top[n][e] ? 1.0f : qa_exp2(top[n][e] - next);
                moved |= next != top[n][e];
                top[n][e] = next;
                sum[n][e] *= keep[n][e];
            }
        float rescaled = 1.0f;      // of acc, behind what the rows' maxima say
        moved = __any_sync(0xffffffffu, moved);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint2 hi_part[NT], lo_part[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float w[4];
                const float base[2] = {top[n][0] == -INFINITY ? 0.0f : top[n][0] - QA_LIFT, top[n][1] == -INFINITY ? 0.0f : top[n][1] - QA_LIFT};
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = qa_exp2(s[h][n][i] - base[i & 1]);
#pragma unroll
                for (int e = 0; e < 2; ++e) sum[n][e] += w[e] + w[2 + e];
                const uint32_t a0 = qa_pack(w[0], w[1]), a1 = qa_pack(w[2], w[3]);
                const float2 r0 = qa_unpack(a0), r1 = qa_unpack(a1);
                hi_part[n] = make_uint2(qa_turn(a0), qa_turn(a1));
                lo_part[n] = make_uint2(qa_turn(qa_pack(w[0] - r0.x, w[1] - r0.y)), qa_turn(qa_pack(w[2] - r1.x, w[3] - r1.y)));
            }
            // Products of bf16 and f16 rows are added to acc by the tensor cores where its unit is, or can be made, the block's scale. Others, of f32 rows, of scales that are 0,
            // NaN or too far from the last one, are added in f32 with the unit 1.
            const float value_scale = scales[2 * h + 1], scale_now = value_scale * LOWER, ratio = unit * cache_inverse(scale_now);
            const bool direct = PARTS == 1 && scale_now > 0.0f && (unit == 0.0f || (ratio >= 0x1p-60f && ratio <= 0x1p40f));
            rescaled = direct ? ratio : unit;
            if ((h == 0 && moved) || rescaled != 1.0f) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float times[2] = {h ? rescaled : keep[n][0] * rescaled, h ? rescaled : keep[n][1] * rescaled};
#pragma unroll
                    for (int m = 0; m < DP / 16; ++m)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[n][m][i] *= times[i & 1];
                }
            }
            unit = direct ? scale_now : 1.0f;
            // the values' products: rows of operand A are channels, two of a lane's each time
            auto products = [&](auto add) {
#pragma unroll
                for (int u = 0; u < (int)S::V_UNITS; ++u) {
                    uint32_t v[4][S::V_UNIT / 4];      // key, word
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t v_at = at + h * S::HALF_BYTES + v_to + (u * 4 + k) * (32 * S::V_UNIT);
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
                        for (int j = 0; j < 2; ++j) add((u * (int)S::V_UNIT + w * 4) / 2 + j, make_uint4(b[2 * j][0], b[2 * j + 1][0], b[2 * j][1], b[2 * j + 1][1]));
                    }
                }
            };
            if (PARTS == 1 && direct)
                products([&](int m, const uint4& f) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        qa_mma(acc[n][m], f, lo_part[n].x, lo_part[n].y);
                        qa_mma(acc[n][m], f, hi_part[n].x, hi_part[n].y);
                    }
                });
            else {
                float times[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        times[n][e] = scale_now;
                        // a block whose scale is NaN makes the rows NaN that see one of its keys here, and no others
                        if (value_scale != value_scale) {
                            bool any = all;
                            for (uint32_t k = 0; k < QA_HALF; ++k) any |= (there >> h & 1u) && row[n][e].sees(key0 + h * QA_HALF + k, steps.end, a.window, a.keep_first);
                            if (!any) times[n][e] = 0.0f;
                        }
                    }
                products([&](int m, const uint4& f) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        qa_mma(d, f, lo_part[n].x, lo_part[n].y);
                        qa_mma(d, f, hi_part[n].x, hi_part[n].y);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[n][m][i] = fmaf(d[i], times[n][i & 1], acc[n][m][i]);
                    }
                });
            }
        }
        __syncwarp();      // (the scales are read before the slot is filled again)
    }
    qa_wait<0>();

    // ---- the warps' sums: [row][channel] each, in the place of the rings ----
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sum[n][h] += __shfl_xor_sync(0xffffffffu, sum[n][h], 4);
            sum[n][h] += __shfl_xor_sync(0xffffffffu, sum[n][h], 8);
            sum[n][h] += __shfl_xor_sync(0xffffffffu, sum[n][h], 16);
            if (g == 0) {
                tops[warp][n * 8 + 2 * quad + h] = top[n][h];
                sums[warp][n * 8 + 2 * quad + h] = sum[n][h];
            }
        }
    __syncthreads();
    float* const all_sums = reinterpret_cast<float*>(qa_raw);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t r = n * 8 + 2 * quad + h;
            float whole = -INFINITY;      // the largest score of the row over the warps
#pragma unroll
            for (int w = 0; w < (int)QA_WARPS; ++w) whole = fmaxf(whole, tops[w][r]);
            const float f = (top[n][h] == whole ? 1.0f : qa_exp2(top[n][h] - whole)) * unit;
            float* out = all_sums + (size_t)warp * (ROWS * DP) + r * DP;
            // (channels of a unit: 2 m and 2 m + 1 are rows g and g + 8 of product m)
#pragma unroll
            for (int u = 0; u < (int)S::V_UNITS; ++u)
#pragma unroll
                for (int k = 0; k < (int)S::V_UNIT; k += 4) {
                    const int m = (u * (int)S::V_UNIT + k) / 2;
                    *reinterpret_cast<float4*>(out + (g + 8 * u) * S::V_UNIT + k) = make_float4(acc[n][m][h] * f, acc[n][m][2 + h] * f, acc[n][m + 1][h] * f, acc[n][m + 1][2 + h] * f);
                }
        }
    __syncthreads();
    const uint32_t rows = min(ROWS, pairs - pair0), quads = dim / 4;
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
            const float4 x = *reinterpret_cast<const float4*>(all_sums + (size_t)w * (ROWS * DP) + r * DP + n * 4);
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
        const float inv = l != 0.0f ? f * (float)(1 << (int)QA_LIFT) / l : 0.0f;      // (the sum of the weights is lifted, the sums of values are not)
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
    float* const mine = p.partials + (place * p.splits + split) * (ROWS * (dim + 2));
    for (uint32_t i = tid; i < rows * quads; i += QA_THREADS) {
        const uint32_t r = i / quads, n = i % quads;
        reinterpret_cast<float4*>(mine)[r * quads + n] = row_quad(r, n);
        if (n == 0) {
            const float m = row_top(r);
            *reinterpret_cast<float2*>(mine + ROWS * dim + r * 2) = make_float2(m, row_sum(r, m));
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
    const float* const theirs = p.partials + place * p.splits * (ROWS * (dim + 2));
    for (uint32_t i = tid; i < rows * quads; i += QA_THREADS) {
        const uint32_t r = i / quads, n = i % quads;
        float m = -INFINITY, l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
        for (uint32_t z = 0; z < p.splits; ++z) {
            const float* part = theirs + (size_t)z * (ROWS * (dim + 2));
            const float2 ml = *reinterpret_cast<const float2*>(part + ROWS * dim + r * 2);
            const float4 x = reinterpret_cast<const float4*>(part)[r * quads + n];
            const float next = fmaxf(m, ml.x), keep = m == next ? 1.0f : qa_exp2(m - next), f = ml.x == next ? 1.0f : qa_exp2(ml.x - next);
            l = l * keep + ml.y * f;
            o.x = o.x * keep + x.x * f; o.y = o.y * keep + x.y * f; o.z = o.z * keep + x.z * f; o.w = o.w * keep + x.w * f;
            m = next;
        }
        finish(r, n, m, l, o);
    }
}

// The weight of each key, summed over the last rows of its sequence and the heads of its key head, in the order of the pairs, from the scores that the kernel above has kept (4 bytes
// a key and pair, where the keys' codes are head_dim a key): a thread a key.
__global__ void __launch_bounds__(QA_SUM) quantized_cache_sum_kernel(const __grid_constant__ QaParams p) {
    __shared__ float2 rows[64];
    __shared__ uint2 spans[64];      // keys that a row's tile has scores of: from .x (or the first kept ones) to .y
    pdl_launch_dependents();
    pdl_wait();
    const uzu_quantized_cache_attention_args& a = p.a;
    const uzu_quantized_cache& c = a.cache;
    const uint32_t sequence = blockIdx.z, head = blockIdx.y;
    const CacheSequence q = cache_sequence(a.sequences, kCacheAnyLength, sequence);
    const uint32_t pairs = q.rows * p.group, first = (q.rows - min(q.rows, a.weight_rows)) * p.group;
    if (pairs > p.score_pairs || !pairs) return;
    const QaSteps steps(q.length, q.length + q.rows - 1u, a.window, a.keep_first, p.capacity);      // (what some row sees)
    const float* const scores = p.scores + ((size_t)sequence * c.kv_heads + head) * p.score_pairs * p.score_stride;
    for (uint32_t r = threadIdx.x; r < pairs; r += QA_SUM) {
        const float2 st = *reinterpret_cast<const float2*>(p.stats + ((size_t)(q.row + r / p.group) * a.heads + head * p.group + r % p.group) * 2);
        rows[r] = make_float2(st.x == -INFINITY ? 0.0f : st.x, st.y);
        const uint32_t pair0 = r / p.tile_rows * p.tile_rows, token0 = q.length + pair0 / p.group, token1 = q.length + min(pair0 + p.tile_rows - 1u, pairs - 1u) / p.group;
        spans[r] = make_uint2(a.window && token0 >= a.window ? (token0 - a.window + 1u) & ~(QA_STEP - 1u) : 0u, token1);
    }
    __syncthreads();
    const uint32_t keys = steps.steps * QA_STEP;
    for (uint32_t i = blockIdx.x * QA_SUM + threadIdx.x; i < keys; i += gridDim.x * QA_SUM) {
        const uint32_t key = steps.key(i / QA_STEP) + i % QA_STEP;
        if (key >= steps.end) continue;
        const uint32_t block = reinterpret_cast<const uint32_t*>(a.sequences.tables)[(size_t)sequence * a.sequences.table_stride + (key >> p.shift)];
        if (block >= c.blocks) continue;
        float x = 0.0f;
        const bool kept = (key & ~(QA_STEP - 1u)) < a.keep_first;
#pragma unroll 4
        for (uint32_t r = first; r < pairs; ++r) {
            const uint2 span = spans[r];
            const float score = (key >= span.x || kept) && key <= span.y ? scores[(size_t)r * p.score_stride + key] : -INFINITY;
            if (score != -INFINITY) x += qa_exp2(score - rows[r].x) * rows[r].y;      // (a row that is NaN gives so to the keys that it sees)
        }
        float* at = reinterpret_cast<float*>(c.key_weights) + (((size_t)block * c.kv_heads + head) << p.shift) + (key & (c.block_tokens - 1u));
        *at += x;
    }
}

// The same with the scores once more, for the rows of prompts, or where they would take too much memory.
template <typename T, int CODE, int DP, int NT>
__global__ void __launch_bounds__(QA_THREADS) quantized_cache_weights_kernel(const __grid_constant__ QaParams p) {
    using S = QaShape<DP, NT>;
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
    __shared__ float factors[S::ROWS];
    __shared__ uint32_t mosts[S::ROWS];
    const uzu_quantized_cache_attention_args& a = p.a;
    const uzu_quantized_cache& c = a.cache;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, g = lane >> 2, quad = lane & 3u, query = 0;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t sequence = blockIdx.z, head = blockIdx.y;
    const CacheSequence q = cache_sequence(a.sequences, kCacheAnyLength, sequence);
    const uint32_t pairs = q.rows * p.group, dim = c.head_dim, bt = c.block_tokens;
    if (p.scores && pairs <= p.score_pairs) return;      // (the kernel above's)
    const uint32_t* table = reinterpret_cast<const uint32_t*>(a.sequences.tables) + (size_t)sequence * a.sequences.table_stride;
    for (uint32_t pair0 = (q.rows - min(q.rows, a.weight_rows)) * p.group; pair0 < pairs; pair0 += S::ROWS) {
        __syncthreads();
        qa_query<T, DP, NT>(p, q, head * p.group, pair0, pairs, query, factors, mosts);
        const uint32_t token0 = q.length + pair0 / p.group, token1 = q.length + min(pair0 + S::ROWS - 1u, pairs - 1u) / p.group;
        const QaSteps steps(token0, token1, a.window, a.keep_first, p.capacity);
        QaRow row[NT][2];
        float factor[NT][2], base[NT][2], times[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t r = pair0 + n * 8 + 2 * quad + h, pair = r < pairs ? r : pairs - 1u;
                row[n][h].live = r < pairs;
                row[n][h].index = q.length + pair / p.group;
                factor[n][h] = factors[n * 8 + 2 * quad + h];
                const float2 st = *reinterpret_cast<const float2*>(p.stats + ((size_t)(q.row + pair / p.group) * a.heads + head * p.group + pair % p.group) * 2);
                base[n][h] = st.x == -INFINITY ? 0.0f : st.x;
                times[n][h] = st.y;
            }
        const QaQuery<DP, NT, PARTS, S::KEPT> fragments(query, lane);
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
#pragma unroll 2
            for (uint32_t at = key0; at < min(key0 + QA_STEP, steps.end); at += QA_HALF) {
                const uint32_t block = table[at >> p.shift];
                if (block >= c.blocks) continue;
                const size_t pair = (size_t)block * c.kv_heads + head;
                const uint32_t in_block = at & (bt - 1u), left = steps.end - at;
                const uint8_t* keys = reinterpret_cast<const uint8_t*>(c.key_codes) + (pair * bt + in_block) * dim;
                const float key_scale = reinterpret_cast<const float*>(c.key_scales)[pair];
                uint4 w[S::K_LOADS];
#pragma unroll
                for (uint32_t n = 0; n < S::K_LOADS; ++n) {
                    const uint32_t key = (n & 1u) * 8 + g, d = (n >> 1) * 64 + quad * 16;
                    w[n] = key < left && d < dim ? *reinterpret_cast<const uint4*>(keys + key * dim + d) : make_uint4(0, 0, 0, 0);
                }
                float s[NT][4];
                qa_scores<CODE, DP, NT, PARTS>(fragments, [&](int n) { return w[n]; }, factor, key_scale, a.softcap, s);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const uint32_t key = at + g + 8 * t;
                    float x = 0.0f;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            if (row[n][h].sees(key, steps.end, a.window, a.keep_first)) x += qa_exp2(s[n][2 * t + h] - base[n][h]) * times[n][h];
                    x += __shfl_xor_sync(0xffffffffu, x, 1);
                    x += __shfl_xor_sync(0xffffffffu, x, 2);
                    if (quad == 0 && key < steps.end) reinterpret_cast<float*>(c.key_weights)[pair * bt + in_block + g + 8 * t] += x;
                }
            }
        }
    }
}

struct QaPlan {
    uint32_t group, tiles, splits, few, eights;      // eights: of pairs, a tile's
    uint32_t score_pairs, score_stride;      // 0: scores are not kept
    uint64_t partial_bytes, stats_bytes, score_bytes;
};
// how so many pairs of a key head of each sequence would be taken
struct QaWays {
    uint32_t eights, tiles;
    uint64_t ctas, slots, most_splits;
};
QaWays qa_ways(uint32_t sm_count, const uzu_quantized_cache_attention_args& a, uint64_t pairs) {
    QaWays w{};
    const uzu_cache_sequences& s = a.sequences;
    const uint32_t capacity = cache_capacity(s, a.cache.block_tokens);
    // tiles as wide as registers allow: a tile reads its keys once. (24 pairs: 55 us where 32 for the same 20 or 24 take 72, 16 sequences of 6000 tokens)
    w.eights = pairs <= 8 ? 1 : a.cache.head_dim <= 64 && pairs > 16 ? (pairs <= 24 ? 3 : 4) : 2;
    w.tiles = (uint32_t)((pairs + w.eights * 8 - 1) / (w.eights * 8));
    w.ctas = (uint64_t)s.count * a.cache.kv_heads * w.tiles;
    w.slots = (uint64_t)sm_count * (a.cache.head_dim > 128 ? 1 : 3);
    const uint64_t keys = a.window ? std::min<uint64_t>(capacity, (uint64_t)a.window + std::min(s.max_rows, s.rows) + a.keep_first + 32) : capacity, steps = (keys + QA_STEP - 1) / QA_STEP;
    w.most_splits = std::min<uint64_t>((steps + QA_WARPS - 1) / QA_WARPS, 128);
    return w;
}
uint64_t qa_partial_bytes(const uzu_quantized_cache_attention_args& a, uint64_t parts, uint32_t eights) { return parts * eights * 8 * (a.cache.head_dim + 2) * 4; }
uint64_t qa_stats_bytes(const uzu_quantized_cache_attention_args& a) { return (uint64_t)a.sequences.rows * a.heads * 8; }
uint64_t qa_score_pairs(const uzu_quantized_cache_attention_args& a) {
    return std::min<uint64_t>((uint64_t)std::min(a.sequences.max_rows, a.sequences.rows) * (a.heads / a.cache.kv_heads), kCacheFewPairs);
}
uint64_t qa_score_stride(const uzu_quantized_cache_attention_args& a) { return ((uint64_t)cache_capacity(a.sequences, a.cache.block_tokens) + 63) & ~63ull; }
// (more than QA_SCORES: any number above it, so that nothing overflows)
uint64_t qa_score_bytes(const uzu_quantized_cache_attention_args& a) {
    const uint64_t rows = (uint64_t)a.sequences.count * a.cache.kv_heads * qa_score_pairs(a), row = qa_score_stride(a) * 4;
    return rows && row > QA_SCORES / rows ? QA_SCORES + 1 : rows * row;
}

QaPlan qa_plan(uint32_t sm_count, const uzu_quantized_cache_attention_args& a) {
    QaPlan p{};
    const uzu_cache_sequences& s = a.sequences;
    p.group = a.heads / a.cache.kv_heads;
    const uint32_t most_rows = std::min(s.max_rows, s.rows);
    const uint64_t most_pairs = (uint64_t)most_rows * p.group;
    p.few = quantized_cache_umma_applicable(a) ? kCacheFewPairs : 0xffffffffu;
    const QaWays w = qa_ways(sm_count, a, std::min<uint64_t>(most_pairs, std::max<uint64_t>(p.few, (uint64_t)std::min(most_rows, kCacheFewRows) * p.group)));
    p.eights = w.eights;
    p.tiles = w.tiles;
    p.splits = 1;
    if (w.ctas && w.ctas <= QA_TICKETS) {
        // one wave where the tiles are few (a CTA too many would double the time), else parts short enough for lengths that differ
        const uint64_t wanted = w.ctas <= w.slots ? w.slots / w.ctas : (2 * w.slots + w.ctas - 1) / w.ctas;
        p.splits = (uint32_t)std::max<uint64_t>(1, std::min(wanted, w.most_splits));
    }
    if (p.splits > 1) p.partial_bytes = qa_partial_bytes(a, w.ctas * p.splits, p.eights);
    if (a.weight_rows) {
        p.stats_bytes = qa_stats_bytes(a);
        const uint64_t bytes = qa_score_bytes(a);
        if ((most_pairs <= kCacheFewPairs || p.few == kCacheFewPairs) && bytes <= QA_SCORES) {
            p.score_pairs = (uint32_t)qa_score_pairs(a);
            p.score_stride = (uint32_t)qa_score_stride(a);
            p.score_bytes = bytes;
        }
    }
    return p;
}
uint64_t qa_align(uint64_t v) { return (v + 255) & ~255ull; }
uint64_t qa_scratch(const QaPlan& p) { return QA_TICKETS * 4 + qa_align(p.partial_bytes) + qa_align(p.stats_bytes) + p.score_bytes; }
// Enough for the plans of all calls with at most these sequences, rows and lengths, wherever rows are and whatever the scale is. Which kernel has a sequence, and with it the pairs here, hangs on those; and fewer
// tiles have more splits: their product is at most one wave, or with more tiles than that two waves and the tiles, as long as there are splits at all.
uint64_t qa_scratch_of_all(uint32_t sm_count, const uzu_quantized_cache_attention_args& a) {
    const QaWays w = qa_ways(sm_count, a, (uint64_t)std::min(a.sequences.max_rows, a.sequences.rows) * (a.heads / a.cache.kv_heads));
    QaPlan p{};
    if (w.most_splits > 1) {
        const uint64_t ctas = std::min(w.ctas, 4 * w.slots), parts = std::min(ctas * w.most_splits, ctas <= w.slots ? w.slots : std::min(4 * w.slots, 2 * w.slots + ctas));
        p.partial_bytes = qa_partial_bytes(a, parts, w.eights);
    }
    if (a.weight_rows) {
        p.stats_bytes = qa_stats_bytes(a);
        p.score_bytes = std::min(qa_score_bytes(a), QA_SCORES);
    }
    return qa_scratch(p);
}

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
void qa_instance(const uzu_quantized_cache_attention_args& a, uint32_t eights, F f) {
    auto tiles = [&](auto t, auto code, auto dp) {
        if (eights == 1) f(t, code, dp, std::integral_constant<int, 1>());
        else if constexpr (decltype(dp)::value == 64) {
            if (eights == 2) f(t, code, dp, std::integral_constant<int, 2>());
            else if (eights == 3) f(t, code, dp, std::integral_constant<int, 3>());
            else f(t, code, dp, std::integral_constant<int, 4>());
        } else f(t, code, dp, std::integral_constant<int, 2>());
    };
    auto dims = [&](auto t, auto code) {
        if (a.cache.head_dim <= 64) tiles(t, code, std::integral_constant<int, 64>());
        else if (a.cache.head_dim <= 128) tiles(t, code, std::integral_constant<int, 128>());
        else tiles(t, code, std::integral_constant<int, 256>());
    };
    auto codes = [&](auto t) {
        if (a.cache.code_type == UZU_CACHE_CODE_I8) dims(t, std::integral_constant<int, UZU_CACHE_CODE_I8>());
        else dims(t, std::integral_constant<int, UZU_CACHE_CODE_E4M3>());
    };
    if (a.data_type == UZU_DT_F32) codes(float());
    else codes(uint16_t());
}

template <typename T, int CODE, int DP, int NT>
void qa_attend(uzu_command_buffer* cmd, const QaParams& p) {
    using S = QaShape<DP, NT>;
    static std::atomic<uint64_t> opted{0};
    const uint32_t parts = sizeof(T) == 4 ? 2 : 1, sums = QA_WARPS * S::ROWS * DP * 4, smem = std::max(S::RING + parts * S::QUERY, sums);
    opt_in_dynamic_smem(cmd, quantized_cache_attention_kernel<T, CODE, DP, NT>, (int)smem, opted);
    launch(cmd, "quantized_cache_attention_kernel", quantized_cache_attention_kernel<T, CODE, DP, NT>, dim3(p.tiles * p.splits, p.a.cache.kv_heads, p.a.sequences.count), dim3(QA_THREADS), smem, p);
}
template <typename T, int CODE, int DP, int NT>
void qa_weigh(uzu_command_buffer* cmd, const QaParams& p) {
    const uint32_t parts = sizeof(T) == 4 ? 2 : 1, ctas = p.a.sequences.count * p.a.cache.kv_heads, steps = (p.capacity + QA_STEP - 1) / QA_STEP;
    const uint32_t parts_of_keys = std::max(1u, std::min((steps + QA_WARPS - 1) / QA_WARPS, ((uint32_t)cmd->ctx->sm_count * 8 + ctas - 1) / ctas));
    launch(cmd, "quantized_cache_weights_kernel", quantized_cache_weights_kernel<T, CODE, DP, NT>, dim3(parts_of_keys, p.a.cache.kv_heads, p.a.sequences.count), dim3(QA_THREADS), parts * QaShape<DP, NT>::QUERY, p);
}

}  // namespace
}  // namespace uzu

using namespace uzu;

extern "C" {

size_t uzu_quantized_cache_attention_scratch_bytes(uzu_context* ctx, const uzu_quantized_cache_attention_args* a) {
    if (!ctx || !a || check_cache(a->cache) || check_cache_sequences(a->sequences, true) || !a->heads || a->heads % a->cache.kv_heads) return 0;
    return qa_scratch_of_all(ctx->sm_count, *a);
}

uzu_status uzu_quantized_cache_attention_validate(const uzu_quantized_cache_attention_args* a) {
    const char* e = attention_check(a);
    return e ? fail(UZU_ERROR_INVALID_ARGUMENT, std::string("quantized_cache_attention: ") + e) : UZU_OK;
}

void uzu_quantized_cache_attention_encode(uzu_command_buffer* cmd, const uzu_quantized_cache_attention_args* args) {
    if (!encodable(cmd, "quantized_cache_attention")) return;
    if (const char* e = attention_check(args)) {
        cmd->record_error(UZU_ERROR_INVALID_ARGUMENT, std::string("quantized_cache_attention: ") + e);
        return;
    }
    uzu_quantized_cache_attention_args within = *args;
    if (within.softcap > 0.0f) within.softcap = std::min(std::max(within.softcap, kCacheLeastCap), kCacheMostCap);
    const uzu_quantized_cache_attention_args* const a = &within;
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
    p.few = plan.few;
    p.shift = a->cache.block_tokens == 16 ? 4 : a->cache.block_tokens == 32 ? 5 : 6;
    p.tickets = reinterpret_cast<uint32_t*>(a->scratch);
    p.partials = reinterpret_cast<float*>(a->scratch + QA_TICKETS * 4);
    p.stats = a->weight_rows ? reinterpret_cast<float*>(a->scratch + QA_TICKETS * 4 + qa_align(plan.partial_bytes)) : nullptr;
    if (plan.score_pairs) p.scores = reinterpret_cast<float*>(a->scratch + QA_TICKETS * 4 + qa_align(plan.partial_bytes) + qa_align(plan.stats_bytes));
    p.score_pairs = plan.score_pairs;
    p.score_stride = plan.score_stride;
    p.tile_rows = plan.eights * 8;
    // prompts, then sequences of few rows (a pass may have both), then the weights of both
    if (plan.few == kCacheFewPairs) encode_quantized_cache_umma(cmd, *a, reinterpret_cast<uint64_t>(p.stats));
    qa_instance(*a, plan.eights, [&](auto t, auto code, auto dim, auto eights) {
        qa_attend<decltype(t), decltype(code)::value, decltype(dim)::value, decltype(eights)::value>(cmd, p);
        if (a->weight_rows && (!p.scores || plan.few == kCacheFewPairs)) qa_weigh<decltype(t), decltype(code)::value, decltype(dim)::value, decltype(eights)::value>(cmd, p);
    });
    if (p.scores) {
        const uint32_t ctas = a->sequences.count * a->cache.kv_heads, most = (p.capacity + QA_SUM - 1) / QA_SUM;
        launch(cmd, "quantized_cache_sum_kernel", quantized_cache_sum_kernel, dim3(std::max(1u, std::min(most, ((uint32_t)cmd->ctx->sm_count * 16 + ctas - 1) / ctas)), a->cache.kv_heads, a->sequences.count), dim3(QA_SUM), 0, p);
    }
}

}  // extern "C"
