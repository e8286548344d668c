// Rows into the 8-bit cache and back: code = round(x / 2^e), x' = code * 2^e, e of a block of tokens and a head.
//
// Bound by memory for prompts, by latency for single tokens. A CTA has one block, one head, keys or values: it holds the block's new numbers in registers (16 a thread and
// turn) while their largest magnitude goes around, so rows are read once. Scales are powers of two: 1 / scale is exact, and a code that is there already is rounded to a larger
// scale in the same CTA, which is the only one that touches the block and head.
// 16384 rows of 8 heads of 128 in and back out: 47 us, 4.3 TB/s (55 with registers for blocks of 64 x 256 in all kernels); one row of each of 64 sequences 12 us, two launches.
#include "quantized_cache.cuh"

namespace uzu {

namespace {

constexpr uint32_t QC_THREADS = 256;

template <typename T> __device__ __forceinline__ float qc_f(T v);
template <> __device__ __forceinline__ float qc_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float qc_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float qc_f(float v) { return v; }
template <typename T> __device__ __forceinline__ T qc_t(float v);
template <> __device__ __forceinline__ __nv_bfloat16 qc_t(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half qc_t(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float qc_t(float v) { return v; }

// 16 numbers of a row
template <typename T, bool WIDE>
struct QcUnit {
    alignas(16) T v[16];
    __device__ __forceinline__ void load(const T* p) {
        if (WIDE) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T); ++i) reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(p)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = p[i];
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if (WIDE) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T); ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(v)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] = v[i];
        }
    }
};

struct QcAppendParams {
    uzu_quantized_cache_append_args a;
    uint32_t capacity;
};

// UNITS: of 16 numbers a thread
template <typename T, int CODE, bool WIDE, int UNITS>
__global__ void __launch_bounds__(QC_THREADS) quantized_cache_append_kernel(const __grid_constant__ QcAppendParams p) {
    __shared__ uint32_t most_of[QC_THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    const uzu_quantized_cache& c = p.a.cache;
    const uint32_t tid = threadIdx.x, sequence = blockIdx.z, head = blockIdx.y, nth = blockIdx.x >> 1, bt = c.block_tokens;
    const bool values = blockIdx.x & 1u;
    const CacheSequence q = cache_sequence(p.a.sequences, p.capacity, sequence);
    const uint32_t begin = q.length, end = min(begin + q.rows, p.capacity);
    if (blockIdx.x == 0 && head == 0 && tid == 0 && p.a.new_lengths) reinterpret_cast<uint32_t*>(p.a.new_lengths)[sequence] = end;
    const uint64_t first = (uint64_t)(begin / bt + nth) * bt;      // the block's first token
    if (first >= end) return;
    const uint32_t block = cache_block(p.a.sequences, sequence, begin / bt + nth);
    if (block >= c.blocks) return;
    const uint32_t old = begin > first ? begin - (uint32_t)first : 0u, tokens = min(bt, end - (uint32_t)first);      // [old, tokens) of the block are new
    const size_t pair = (size_t)block * c.kv_heads + head;
    const uint32_t chunks = c.head_dim / 16, units = tokens * chunks, stride = values ? p.a.value_stride : p.a.key_stride;
    const T* rows = reinterpret_cast<const T*>(values ? p.a.values : p.a.keys) + (size_t)q.row * stride + head * c.head_dim;
    uint8_t* codes = reinterpret_cast<uint8_t*>(values ? c.value_codes : c.key_codes) + pair * bt * c.head_dim;
    float* scale_at = reinterpret_cast<float*>(values ? c.value_scales : c.key_scales) + pair;
    const float was = old ? *scale_at : 0.0f;

    QcUnit<T, WIDE> x[UNITS];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
        const uint32_t u = tid + i * QC_THREADS, token = u / chunks;
        if (u >= units || token < old) continue;
        x[i].load(rows + (size_t)((uint32_t)first + token - begin) * stride + (u - token * chunks) * 16);
    }
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
        const uint32_t u = tid + i * QC_THREADS;
        if (u >= units || u / chunks < old) continue;
#pragma unroll
        for (int j = 0; j < 16; ++j) most = max(most, __float_as_uint(qc_f(x[i].v[j])) & 0x7fffffffu);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if ((tid & 31u) == 0) most_of[tid >> 5] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < (int)(QC_THREADS / 32); ++w) most = max(most, most_of[w]);
    const float need = cache_scale<CODE>(most), scale = was != was ? was : need != need ? need : fmaxf(was, need), inverse = cache_inverse(scale);
    if (tid == 0) *scale_at = scale;
    const float again = was * inverse;      // (NaN is not asked for below)
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
        const uint32_t u = tid + i * QC_THREADS, token = u / chunks;
        if (u >= units) continue;
        uint4* at = reinterpret_cast<uint4*>(codes + (size_t)u * 16);
        uint4 w;
        uint32_t* ws = reinterpret_cast<uint32_t*>(&w);
        if (token >= old) {
            if (!(scale > 0.0f)) w = make_uint4(0, 0, 0, 0);
            else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    ws[k] = cache_pack<CODE>(qc_f(x[i].v[4 * k]) * inverse, qc_f(x[i].v[4 * k + 1]) * inverse, qc_f(x[i].v[4 * k + 2]) * inverse, qc_f(x[i].v[4 * k + 3]) * inverse);
            }
            *at = w;
        } else if (scale > was) {
            w = *at;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float y[4];
                cache_unpack<CODE>(ws[k], y);
                ws[k] = cache_pack<CODE>(y[0] * again, y[1] * again, y[2] * again, y[3] * again);
            }
            *at = w;
        }
    }
    if (!values && c.key_weights && tid < tokens && tid >= old) reinterpret_cast<float*>(c.key_weights)[pair * bt + tid] = 0.0f;
}

struct QcReadParams {
    uzu_quantized_cache_read_args a;
    uint32_t capacity;
};

// a thread has 16 numbers of a row's keys and the same of its values
template <typename T, int CODE, bool WIDE>
__global__ void __launch_bounds__(QC_THREADS) quantized_cache_read_kernel(const __grid_constant__ QcReadParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const uzu_quantized_cache& c = p.a.cache;
    const CacheSequence q = cache_sequence(p.a.sequences, p.capacity, blockIdx.y);
    const uint32_t chunks = c.head_dim / 16, width = chunks * c.kv_heads;
    const uint64_t at = (uint64_t)blockIdx.x * QC_THREADS + threadIdx.x;
    const uint32_t t = (uint32_t)(at / width), u = (uint32_t)(at - (uint64_t)t * width), token = q.length + t;
    if (t >= q.rows || token >= p.capacity) return;
    const uint32_t block = cache_block(p.a.sequences, blockIdx.y, token / c.block_tokens);
    if (block >= c.blocks) return;
    const uint32_t head = u / chunks;
    const size_t pair = (size_t)block * c.kv_heads + head, from = (pair * c.block_tokens + token % c.block_tokens) * c.head_dim + (u - head * chunks) * 16;
    uint4 w[2];
    float scale[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (!(k ? p.a.values : p.a.keys)) continue;
        w[k] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(k ? c.value_codes : c.key_codes) + from);
        scale[k] = reinterpret_cast<const float*>(k ? c.value_scales : c.key_scales)[pair];
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (!(k ? p.a.values : p.a.keys)) continue;
        QcUnit<T, WIDE> x;
        const uint32_t* ws = reinterpret_cast<const uint32_t*>(&w[k]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float y[4];
            cache_unpack<CODE>(ws[j], y);
#pragma unroll
            for (int i = 0; i < 4; ++i) x.v[4 * j + i] = qc_t<T>(y[i] * scale[k]);
        }
        x.store(reinterpret_cast<T*>(k ? p.a.values : p.a.keys) + (size_t)(q.row + t) * (k ? p.a.value_stride : p.a.key_stride) + u * 16);
    }
}

inline uint64_t qc_size(uint32_t data_type) { return data_type == UZU_DT_F32 ? 4 : 2; }

// keys and values rows of an append or a read
const char* check_rows(const uzu_quantized_cache& c, const uzu_cache_sequences& s, uint64_t keys, uint64_t values, uint32_t key_stride, uint32_t value_stride, uint32_t data_type, bool written) {
    const uint64_t width = (uint64_t)c.kv_heads * c.head_dim, size = qc_size(data_type);
    if ((keys && key_stride < width) || (values && value_stride < width)) return "a row is shorter than its heads";
    if ((keys | values) % size) return "a row is not aligned to its elements";
    const uint64_t kb = rows_extent(s.rows, key_stride, width, size), vb = rows_extent(s.rows, value_stride, width, size);
    if ((keys && meets_cache(c, keys, kb)) || (values && meets_cache(c, values, vb))) return "the cache overlaps rows";
    if (written) {
        if (keys && values && rows_overlap(keys, key_stride, width, values, value_stride, width, s.rows, size)) return "keys and values overlap";
        if ((keys && meets_sequences(s, keys, kb)) || (values && meets_sequences(s, values, vb))) return "rows overlap what says which sequences there are";
    }
    return nullptr;
}
bool cache_touches_sequences(const uzu_quantized_cache& c, const uzu_cache_sequences& s) {
    return meets_cache(c, s.tables, (uint64_t)s.count * s.table_stride * 4) || meets_cache(c, s.lengths, (uint64_t)s.count * 4) ||
           (s.row_offsets && meets_cache(c, s.row_offsets, ((uint64_t)s.count + 1) * 4));
}

const char* append_check(const uzu_quantized_cache_append_args* a) {
    if (!a) return "null arguments";
    if (a->data_type > UZU_DT_F16) return "data_type must be bf16, f32 or f16";
    if (const char* e = check_cache(a->cache)) return e;
    if (const char* e = check_cache_sequences(a->sequences, true)) return e;
    const uzu_cache_sequences& s = a->sequences;
    if (!s.count) return nullptr;
    if (s.rows && (!a->keys || !a->values)) return "null rows";
    if (cache_meets_itself(a->cache) || cache_touches_sequences(a->cache, s)) return "the cache overlaps itself or what says which sequences there are";
    if (const char* e = check_rows(a->cache, s, a->keys, a->values, a->key_stride, a->value_stride, a->data_type, false)) return e;
    const uint64_t bytes = (uint64_t)s.count * 4, width = (uint64_t)a->cache.kv_heads * a->cache.head_dim, size = qc_size(a->data_type);
    if (a->new_lengths % 4) return "new_lengths is not aligned";
    if (a->new_lengths && (meets_sequences(s, a->new_lengths, bytes) || meets_cache(a->cache, a->new_lengths, bytes) ||
                           bytes_overlap(a->new_lengths, bytes, a->keys, rows_extent(s.rows, a->key_stride, width, size)) ||
                           bytes_overlap(a->new_lengths, bytes, a->values, rows_extent(s.rows, a->value_stride, width, size))))
        return "new_lengths overlaps another operand";
    return nullptr;
}
const char* read_check(const uzu_quantized_cache_read_args* a) {
    if (!a) return "null arguments";
    if (a->data_type > UZU_DT_F16) return "data_type must be bf16, f32 or f16";
    if (const char* e = check_cache(a->cache)) return e;
    if (const char* e = check_cache_sequences(a->sequences, true)) return e;
    if (!a->sequences.count) return nullptr;
    return check_rows(a->cache, a->sequences, a->keys, a->values, a->key_stride, a->value_stride, a->data_type, true);
}

template <typename F>
void by_type(uint32_t data_type, F f) {
    if (data_type == UZU_DT_F32) f(float());
    else if (data_type == UZU_DT_F16) f(__half());
    else f(__nv_bfloat16());
}

}  // namespace
}  // namespace uzu

using namespace uzu;

extern "C" {

uzu_status uzu_quantized_cache_append_validate(const uzu_quantized_cache_append_args* a) {
    const char* e = append_check(a);
    return e ? fail(UZU_ERROR_INVALID_ARGUMENT, std::string("quantized_cache_append: ") + e) : UZU_OK;
}

void uzu_quantized_cache_append_encode(uzu_command_buffer* cmd, const uzu_quantized_cache_append_args* a) {
    if (!encodable(cmd, "quantized_cache_append")) return;
    if (const char* e = append_check(a)) {
        cmd->record_error(UZU_ERROR_INVALID_ARGUMENT, std::string("quantized_cache_append: ") + e);
        return;
    }
    const uzu_cache_sequences& s = a->sequences;
    if (!s.count) return;
    QcAppendParams p{};
    p.a = *a;
    p.capacity = cache_capacity(s, a->cache.block_tokens);
    // blocks that a sequence's rows can touch
    const uint32_t bt = a->cache.block_tokens, most = std::min(std::min(s.max_rows, s.rows), p.capacity), blocks = std::min((most + 2 * bt - 2) / bt, s.table_stride);
    const dim3 grid(std::max(blocks, 1u) * 2, a->cache.kv_heads, s.count);
    const uint32_t units = bt * (a->cache.head_dim / 16);      // of a whole block
    const uint64_t size = qc_size(a->data_type);
    const bool wide = ((a->keys | a->values) & 15u) == 0 && a->key_stride * size % 16 == 0 && a->value_stride * size % 16 == 0;
    by_type(a->data_type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto kernel) { launch(cmd, "quantized_cache_append_kernel", kernel, grid, dim3(QC_THREADS), 0, p); };
        auto by_units = [&](auto code) {
            constexpr int CODE = decltype(code)::value;
            if (units <= QC_THREADS) wide ? go(quantized_cache_append_kernel<T, CODE, true, 1>) : go(quantized_cache_append_kernel<T, CODE, false, 1>);
            else if (units <= 2 * QC_THREADS) wide ? go(quantized_cache_append_kernel<T, CODE, true, 2>) : go(quantized_cache_append_kernel<T, CODE, false, 2>);
            else wide ? go(quantized_cache_append_kernel<T, CODE, true, 4>) : go(quantized_cache_append_kernel<T, CODE, false, 4>);
        };
        if (a->cache.code_type == UZU_CACHE_CODE_I8) by_units(std::integral_constant<int, UZU_CACHE_CODE_I8>());
        else by_units(std::integral_constant<int, UZU_CACHE_CODE_E4M3>());
    });
}

uzu_status uzu_quantized_cache_read_validate(const uzu_quantized_cache_read_args* a) {
    const char* e = read_check(a);
    return e ? fail(UZU_ERROR_INVALID_ARGUMENT, std::string("quantized_cache_read: ") + e) : UZU_OK;
}

void uzu_quantized_cache_read_encode(uzu_command_buffer* cmd, const uzu_quantized_cache_read_args* a) {
    if (!encodable(cmd, "quantized_cache_read")) return;
    if (const char* e = read_check(a)) {
        cmd->record_error(UZU_ERROR_INVALID_ARGUMENT, std::string("quantized_cache_read: ") + e);
        return;
    }
    const uzu_cache_sequences& s = a->sequences;
    if (!s.count || (!a->keys && !a->values)) return;
    QcReadParams p{};
    p.a = *a;
    p.capacity = cache_capacity(s, a->cache.block_tokens);
    const uint64_t most = std::min(std::min(s.max_rows, s.rows), p.capacity), units = most * a->cache.kv_heads * (a->cache.head_dim / 16);
    if (!units) return;
    if (units > (uint64_t)0x7fffffff * QC_THREADS) {
        cmd->record_error(UZU_ERROR_INVALID_ARGUMENT, "quantized_cache_read: too many rows for one call");
        return;
    }
    const dim3 grid((uint32_t)((units + QC_THREADS - 1) / QC_THREADS), s.count);
    const uint64_t size = qc_size(a->data_type);
    const bool wide = ((a->keys | a->values) & 15u) == 0 && a->key_stride * size % 16 == 0 && a->value_stride * size % 16 == 0;
    by_type(a->data_type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto kernel) { launch(cmd, "quantized_cache_read_kernel", kernel, grid, dim3(QC_THREADS), 0, p); };
        if (a->cache.code_type == UZU_CACHE_CODE_I8) wide ? go(quantized_cache_read_kernel<T, UZU_CACHE_CODE_I8, true>) : go(quantized_cache_read_kernel<T, UZU_CACHE_CODE_I8, false>);
        else wide ? go(quantized_cache_read_kernel<T, UZU_CACHE_CODE_E4M3, true>) : go(quantized_cache_read_kernel<T, UZU_CACHE_CODE_E4M3, false>);
    });
}

}  // extern "C"
