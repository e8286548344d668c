// Tokens of the 8-bit cache that had the least attention weight give way: which ones stay, and the ones that do move up in place.
//
// Choice (a CTA for each sequence and head): the weights' bits in an order of unsigned numbers, the least one that stays found digit by digit (8 bits a pass), then the tokens that
// stay counted off in their order; of those alike at the border the first ones.
// Move (a CTA for each block to be filled, keys or values): a block's new numbers come from blocks at or behind it, so it may be written once those who read it have. CTAs take their
// blocks from a counter in ascending order, load first, say so, and wait only for earlier ones' loads, which wait for nothing: no order of CTAs can stop it. Nothing goes
// through memory twice and no second copy of the cache is needed.
// What bounds it: latency, a CTA's way through counter, indices, table, scales and codes. 16 sequences of 16000 tokens cut to 8000, 8 heads of 128 (e4m3): choice 55 us, move 240 (524 MB of
// codes read and written, 2.2 TB/s; 408 with registers for blocks of 64 x 256), reading the kept tokens back 145 (786 MB, 5.4 TB/s). One sequence of 9001 to 4096: 26, 16 and 8 us.
#include "quantized_cache.cuh"

namespace uzu {

namespace {

constexpr uint32_t QE_CHOICE = 1024, QE_ITEMS = 4, QE_MOVE = 256;
constexpr uint32_t QE_CACHED = 40960;              // weights of a sequence that are kept in shared memory

struct QeParams {
    uzu_quantized_cache_evict_args a;
    uint32_t capacity, blocks, cached;             // blocks: that `budget` tokens take; cached: weights in shared memory
    uint32_t *counter, *loaded, *starts, *indices;      // [1], [count * kv_heads * 2, blocks], [count * kv_heads, blocks + 1], [count, kv_heads, budget]
    unsigned int* error;
};

// larger weights are larger numbers, NaN and tokens without a block the smallest
__device__ __forceinline__ uint32_t qe_order(float w) {
    const uint32_t b = __float_as_uint(w + 0.0f);      // (-0 is 0)
    return w != w ? 0u : b >> 31 ? ~b : b | 0x80000000u;
}

__global__ void __launch_bounds__(QE_CHOICE) quantized_cache_choice_kernel(const __grid_constant__ QeParams p) {
    extern __shared__ uint32_t qe_keys[];
    __shared__ uint32_t counts[256], warp_counts[2][32], found[2];
    pdl_launch_dependents();
    pdl_wait();
    const uzu_quantized_cache_evict_args& a = p.a;
    const uzu_quantized_cache& c = a.cache;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, head = blockIdx.x, sequence = blockIdx.y, bt = c.block_tokens;
    const uint32_t length = min(reinterpret_cast<const uint32_t*>(a.sequences.lengths)[sequence], p.capacity);
    const size_t chain = (size_t)sequence * c.kv_heads + head;
    uint32_t* indices = p.indices + chain * a.budget;
    if (head == 0 && tid == 0) reinterpret_cast<uint32_t*>(a.new_lengths)[sequence] = min(length, a.budget);
    if (head == 0 && sequence == 0 && tid == 0) *p.counter = 0;
    for (uint32_t i = tid; i < 2 * p.blocks; i += QE_CHOICE) p.loaded[chain * 2 * p.blocks + i] = 0;
    if (length <= a.budget) {
        if (a.indices)
            for (uint32_t i = tid; i < a.budget; i += QE_CHOICE) indices[i] = i < length ? i : kNoIndex;
        return;
    }
    const uint32_t* table = reinterpret_cast<const uint32_t*>(a.sequences.tables) + (size_t)sequence * a.sequences.table_stride;
    auto read = [&](uint32_t j) {
        const uint32_t block = table[j / bt];
        return block < c.blocks ? qe_order(reinterpret_cast<const float*>(c.key_weights)[((size_t)block * c.kv_heads + head) * bt + j % bt]) : 0u;
    };
    const bool cached = length <= p.cached;
    if (cached) {
        for (uint32_t j = tid; j < length; j += QE_CHOICE) qe_keys[j] = read(j);
        __syncthreads();
    }
    auto key = [&](uint32_t j) { return cached ? qe_keys[j] : read(j); };

    // the `want` largest of tokens [begin, end): all above `border`, and the first `equal` of those at it
    const uint32_t begin = a.keep_first, end = length - a.keep_last;
    uint32_t want = a.budget - a.keep_first - a.keep_last, border = 0, known = 0;
    for (int shift = 24; shift >= 0 && want; shift -= 8) {
        if (tid < 256) counts[tid] = 0;
        __syncthreads();
        for (uint32_t j0 = begin; j0 < end; j0 += QE_CHOICE) {
            const uint32_t j = j0 + tid, k = j < end ? key(j) : 0u;
            const bool mine = j < end && (k & known) == border;
            const uint32_t digit = mine ? k >> shift & 255u : 256u, same = __match_any_sync(0xffffffffu, digit);
            if (mine && lane == __ffs(same) - 1) atomicAdd(&counts[digit], __popc(same));
        }
        __syncthreads();
        if (warp == 0) {      // from the largest digit down: 8 digits a lane
            uint32_t mine = 0;
            for (uint32_t d = 0; d < 8; ++d) mine += counts[255 - lane * 8 - d];
            uint32_t sum = mine;
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t x = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += x;
            }
            if (sum - mine < want && want <= sum) {
                uint32_t above = sum - mine, d = lane * 8;
                while (above + counts[255 - d] < want) above += counts[255 - d++];
                found[0] = 255 - d;
                found[1] = want - above;
            }
        }
        __syncthreads();
        border |= found[0] << shift;
        want = found[1];
        known |= 255u << shift;
        __syncthreads();
    }
    const bool choose = known != 0;      // (otherwise only the first and the last stay)

    // the kept ones in order
    uint32_t* starts = p.starts + chain * (p.blocks + 1);
    uint32_t kept = 0, alike = 0;
    for (uint32_t j0 = 0; j0 < length; j0 += QE_CHOICE * QE_ITEMS) {
        uint32_t state[QE_ITEMS], equal = 0;      // 0: gives way, 1: stays, 2: alike
#pragma unroll
        for (uint32_t i = 0; i < QE_ITEMS; ++i) {
            const uint32_t j = j0 + tid * QE_ITEMS + i;
            state[i] = 0;
            if (j >= length) continue;
            if (j < begin || j >= end) state[i] = 1;
            else if (choose) {
                const uint32_t k = key(j);
                state[i] = k > border ? 1 : k == border ? 2 : 0;
            }
            equal += state[i] == 2;
        }
        auto scan = [&](uint32_t mine, uint32_t which, uint32_t& all) {      // sums of the threads before this one
            uint32_t sum = mine;
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t x = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += x;
            }
            if (lane == 31) warp_counts[which][warp] = sum;
            __syncthreads();
            uint32_t other = warp_counts[which][lane], before = lane < warp ? other : 0u;
            before = __reduce_add_sync(0xffffffffu, before);
            all = __reduce_add_sync(0xffffffffu, other);
            return before + sum - mine;
        };
        uint32_t all_equal, all_kept, at_equal = alike + scan(equal, 0, all_equal), stay = 0;
#pragma unroll
        for (uint32_t i = 0; i < QE_ITEMS; ++i) {
            if (state[i] == 2) state[i] = at_equal++ < want ? 1 : 0;
            stay += state[i];
        }
        uint32_t at = kept + scan(stay, 1, all_kept);
#pragma unroll
        for (uint32_t i = 0; i < QE_ITEMS; ++i) {
            const uint32_t j = j0 + tid * QE_ITEMS + i;
            if (j % bt == 0 && j / bt <= p.blocks) starts[j / bt] = at;      // (kept ones before the block)
            if (state[i]) indices[at++] = j;
        }
        kept += all_kept;
        alike += all_equal;
    }
}

__device__ __forceinline__ uint32_t qe_acquire(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

// UNITS: of 16 codes a thread
template <int CODE, int UNITS>
__global__ void __launch_bounds__(QE_MOVE, UNITS == 4 ? 2 : 5) quantized_cache_move_kernel(const __grid_constant__ QeParams p) {
    __shared__ uint32_t most_of[QE_MOVE / 32], item_at, late;
    pdl_launch_dependents();
    pdl_wait();
    const uzu_quantized_cache_evict_args& a = p.a;
    const uzu_quantized_cache& c = a.cache;
    const uint32_t tid = threadIdx.x, bt = c.block_tokens, dim = c.head_dim, chunks = dim / 16;
    if (tid == 0) {
        item_at = atomicAdd(p.counter, 1u);
        late = 0;
    }
    __syncthreads();
    const uint32_t chains = a.sequences.count * c.kv_heads * 2, item = item_at, b = item / chains, chain = item % chains;
    const bool values = chain & 1u;
    const uint32_t head = (chain >> 1) % c.kv_heads, sequence = (chain >> 1) / c.kv_heads;
    const uint32_t length = min(reinterpret_cast<const uint32_t*>(a.sequences.lengths)[sequence], p.capacity);
    if (length <= a.budget) return;
    const uint32_t* indices = p.indices + (size_t)(chain >> 1) * a.budget;
    const uint32_t* table = reinterpret_cast<const uint32_t*>(a.sequences.tables) + (size_t)sequence * a.sequences.table_stride;
    const uint32_t first = b * bt, tokens = min(bt, a.budget - first), units = tokens * chunks;
    uint8_t* codes = reinterpret_cast<uint8_t*>(values ? c.value_codes : c.key_codes);
    float* scales = reinterpret_cast<float*>(values ? c.value_scales : c.key_scales);

    // (asked for early: what says who reads this block, and where it is)
    const uint32_t* starts = p.starts + (size_t)(chain >> 1) * (p.blocks + 1);
    const uint32_t at[2] = {starts[b], (uint64_t)(b + 1) * bt < length ? starts[b + 1] : a.budget}, block = table[b];

    uint4 x[UNITS];
    float from[UNITS];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
        const uint32_t u = tid + i * QE_MOVE, token = u / chunks;
        x[i] = make_uint4(0, 0, 0, 0);
        from[i] = 0.0f;
        if (u >= units) continue;
        const uint32_t j = indices[first + token], its = table[j / bt];
        if (its >= c.blocks) continue;      // (a token without a block: zeros)
        const size_t pair = (size_t)its * c.kv_heads + head;
        from[i] = scales[pair];
        x[i] = *reinterpret_cast<const uint4*>(codes + (pair * bt + j % bt) * dim + (u - token * chunks) * 16);
    }
    float weight = 0.0f;
    if (!values && tid < tokens) {
        const uint32_t j = indices[first + tid], its = table[j / bt];
        if (its < c.blocks) weight = reinterpret_cast<const float*>(c.key_weights)[((size_t)its * c.kv_heads + head) * bt + j % bt];
    }
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
        const uint32_t* ws = reinterpret_cast<const uint32_t*>(&x[i]);
        if (from[i] != from[i]) most = 0x7fc00000u;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float y[4];
            cache_unpack<CODE>(ws[k], y);
#pragma unroll
            for (int n = 0; n < 4; ++n) most = max(most, __float_as_uint(y[n] * from[i]) & 0x7fffffffu);
        }
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if ((tid & 31u) == 0) most_of[tid >> 5] = most;
    __syncthreads_or(__float_as_uint(weight) == 0x7fc0deadu);      // (a barrier that waits for the weight as well: what this block takes has been read)
    uint32_t* loaded = p.loaded + (size_t)chain * p.blocks;
    if (tid == 0) asm volatile("st.release.gpu.global.u32 [%0], 1;" ::"l"(loaded + b) : "memory");
#pragma unroll
    for (int w = 0; w < (int)(QE_MOVE / 32); ++w) most = max(most, most_of[w]);

    // who reads block b: the blocks of the kept tokens [lo, hi) that are in it, all of them at or before b
    if (tid < 32) {
        if (at[1] > at[0]) {
            const uint32_t last = min((at[1] - 1) / bt, b);      // (b itself has)
            uint64_t t0, t1;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
            for (uint32_t other = at[0] / bt + tid; other <= last; other += 32) {
                if (other == b) continue;
                while (!qe_acquire(loaded + other)) {
                    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t1));
                    if (t1 - t0 > 1000000000ull) {
                        late = 1;
                        report_wait_error(p.error, 0xa01u);
                        break;
                    }
                }
            }
        }
    }
    __syncthreads();
    if (late) return;      // (nothing is written over what may still be read)
    if (block >= c.blocks) return;
    const size_t pair = (size_t)block * c.kv_heads + head;
    const float scale = cache_scale<CODE>(most), inverse = cache_inverse(scale);
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
        const uint32_t u = tid + i * QE_MOVE;
        if (u >= units) continue;
        uint32_t* ws = reinterpret_cast<uint32_t*>(&x[i]);
        if (!(scale > 0.0f)) x[i] = make_uint4(0, 0, 0, 0);
        else if (from[i] != scale) {
            const float times = from[i] * inverse;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float y[4];
                cache_unpack<CODE>(ws[k], y);
                ws[k] = cache_pack<CODE>(y[0] * times, y[1] * times, y[2] * times, y[3] * times);
            }
        }
        *reinterpret_cast<uint4*>(codes + pair * bt * dim + (size_t)u * 16) = x[i];
    }
    if (tid == 0) scales[pair] = scale;
    if (!values && tid < tokens) reinterpret_cast<float*>(c.key_weights)[pair * bt + tid] = weight;
}

struct QePlan {
    uint32_t blocks;
    uint64_t loaded_bytes, starts_bytes, index_bytes;
};
uint64_t qe_align(uint64_t v) { return (v + 255) & ~255ull; }
QePlan qe_plan(const uzu_quantized_cache_evict_args& a) {
    QePlan p{};
    p.blocks = (uint32_t)(((uint64_t)a.budget + a.cache.block_tokens - 1) / a.cache.block_tokens);
    const uint64_t chains = (uint64_t)a.sequences.count * a.cache.kv_heads;
    p.loaded_bytes = chains * 2 * p.blocks * 4;
    p.starts_bytes = chains * (p.blocks + 1) * 4;
    p.index_bytes = a.indices ? 0 : chains * a.budget * 4;
    return p;
}
constexpr uint64_t QE_HEAD = 256;
uint64_t qe_scratch(const QePlan& p) { return QE_HEAD + qe_align(p.loaded_bytes) + qe_align(p.starts_bytes) + qe_align(p.index_bytes); }

const char* evict_check(const uzu_quantized_cache_evict_args* a) {
    if (!a) return "null arguments";
    if (const char* e = check_cache(a->cache)) return e;
    if (const char* e = check_cache_sequences(a->sequences, false)) return e;
    const uzu_quantized_cache& c = a->cache;
    const uzu_cache_sequences& s = a->sequences;
    if (!c.key_weights) return "null key_weights";
    if (!a->budget || a->budget >> 31) return "budget must be in 1 .. 2^31 - 1";
    if ((uint64_t)a->keep_first + a->keep_last > a->budget) return "keep_first and keep_last are more than budget";
    if (!s.count) return nullptr;
    if (!a->new_lengths || !a->scratch) return "null operand";
    if ((a->new_lengths | a->indices) % 4) return "an operand is not aligned to its elements";
    if (a->scratch % 256) return "the scratch is not aligned";
    const uint64_t chains = (uint64_t)s.count * c.kv_heads, blocks = ((uint64_t)a->budget + c.block_tokens - 1) / c.block_tokens;
    if (chains * 2 * blocks >> 31) return "too many blocks for one call";
    if (cache_meets_itself(c)) return "the cache overlaps itself";
    const uint64_t at[3] = {a->new_lengths, a->indices, a->scratch}, bytes[3] = {s.count * 4ull, chains * a->budget * 4, a->scratch_bytes};
    for (int i = 0; i < 3; ++i) {
        if (!at[i]) continue;
        if (meets_cache(c, at[i], bytes[i]) || bytes_overlap(at[i], bytes[i], s.tables, (uint64_t)s.count * s.table_stride * 4) || bytes_overlap(at[i], bytes[i], s.lengths, s.count * 4ull))
            return "an operand overlaps the cache or what says which sequences there are";
        for (int j = 0; j < i; ++j)
            if (bytes_overlap(at[i], bytes[i], at[j], bytes[j])) return "operands overlap";
    }
    if (meets_cache(c, s.tables, (uint64_t)s.count * s.table_stride * 4) || meets_cache(c, s.lengths, s.count * 4ull)) return "the cache overlaps what says which sequences there are";
    return nullptr;
}

}  // namespace
}  // namespace uzu

using namespace uzu;

extern "C" {

size_t uzu_quantized_cache_evict_scratch_bytes(uzu_context* ctx, const uzu_quantized_cache_evict_args* a) {
    if (!ctx || !a || check_cache(a->cache) || check_cache_sequences(a->sequences, false) || !a->budget || a->budget >> 31) return 0;
    return qe_scratch(qe_plan(*a));
}

uzu_status uzu_quantized_cache_evict_validate(const uzu_quantized_cache_evict_args* a) {
    const char* e = evict_check(a);
    return e ? fail(UZU_ERROR_INVALID_ARGUMENT, std::string("quantized_cache_evict: ") + e) : UZU_OK;
}

void uzu_quantized_cache_evict_encode(uzu_command_buffer* cmd, const uzu_quantized_cache_evict_args* a) {
    if (!encodable(cmd, "quantized_cache_evict")) return;
    if (const char* e = evict_check(a)) {
        cmd->record_error(UZU_ERROR_INVALID_ARGUMENT, std::string("quantized_cache_evict: ") + e);
        return;
    }
    const uzu_cache_sequences& s = a->sequences;
    if (!s.count) return;
    const QePlan plan = qe_plan(*a);
    if (a->scratch_bytes < qe_scratch(plan)) {
        cmd->record_error(UZU_ERROR_INVALID_ARGUMENT, "quantized_cache_evict: the scratch is too small");
        return;
    }
    QeParams p{};
    p.a = *a;
    p.capacity = cache_capacity(s, a->cache.block_tokens);
    p.blocks = plan.blocks;
    p.cached = std::min(p.capacity, QE_CACHED);
    p.counter = reinterpret_cast<uint32_t*>(a->scratch);
    p.loaded = reinterpret_cast<uint32_t*>(a->scratch + QE_HEAD);
    p.starts = reinterpret_cast<uint32_t*>(a->scratch + QE_HEAD + qe_align(plan.loaded_bytes));
    p.indices = reinterpret_cast<uint32_t*>(a->indices ? a->indices : a->scratch + QE_HEAD + qe_align(plan.loaded_bytes) + qe_align(plan.starts_bytes));
    p.error = cmd->ctx->wait_errors.device_word;
    static std::atomic<uint64_t> opted{0};
    opt_in_dynamic_smem(cmd, quantized_cache_choice_kernel, (int)(QE_CACHED * 4), opted);
    launch(cmd, "quantized_cache_choice_kernel", quantized_cache_choice_kernel, dim3(a->cache.kv_heads, s.count), dim3(QE_CHOICE), p.cached * 4, p);
    if (p.capacity <= a->budget) return;      // (no sequence can be longer)
    const dim3 grid(plan.blocks * s.count * a->cache.kv_heads * 2);
    const uint32_t units = a->cache.block_tokens * a->cache.head_dim / 16;
    auto go = [&](auto kernel) { launch(cmd, "quantized_cache_move_kernel", kernel, grid, dim3(QE_MOVE), 0, p); };
    auto by_units = [&](auto code) {
        constexpr int CODE = decltype(code)::value;
        if (units <= QE_MOVE) go(quantized_cache_move_kernel<CODE, 1>);
        else if (units <= 2 * QE_MOVE) go(quantized_cache_move_kernel<CODE, 2>);
        else go(quantized_cache_move_kernel<CODE, 4>);
    };
    if (a->cache.code_type == UZU_CACHE_CODE_I8) by_units(std::integral_constant<int, UZU_CACHE_CODE_I8>());
    else by_units(std::integral_constant<int, UZU_CACHE_CODE_E4M3>());
}

}  // extern "C"
