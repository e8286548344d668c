// Short causal convolution over packed sequences: y[t, c] = act(bias[c] + sum_j w[c, j] u[t - taps + 1 + j, c]).
//
// Bound by memory: a value is read and written once, 2 taps flops each, an exponential and a reciprocal. A thread has 8 bytes of channels (four of 16 bits, two of 32) and walks a strip
// of a sequence's rows with the last taps - 1 of them in registers, eight rows of loads under way at a time; a strip reads taps - 1 rows of the one before it again (from L2). 16384 rows
// of 10240 bf16 channels, 4 taps, 16 sequences: 125 us, 5.4 TB/s of the 6.45 of a copy (one reciprocal for two gates, whose denominators had to be cut for it, 131; and with that 16
// bytes a thread 178: fewer warps; 4 bytes 223; batches of four rows 146; limits on the registers 170 to 284). Rows off whole groups of 8 bytes take
// one channel a thread: 153 us (f32: 233 against 213).
// The strip that starts a sequence reads the slot's inputs and, behind its rows, writes the new ones: nobody else touches these channels of the slot, so the order is its own.
#include "state_space.cuh"

namespace uzu {

namespace {

constexpr uint32_t CC_THREADS = 128;

struct ConvParams {
    uzu_causal_conv_args a;
    uint32_t strip, groups;      // rows of a strip, blocks beside one another: those of a row run together
    SequenceTable table;
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) ConvVec {
    T v[VEC];
};

// the last `kept` inputs of (slot, rows), by the strip that starts the sequence: nobody else touches these channels of the slot
template <typename T, int VEC, int TAPS>
__device__ __forceinline__ void conv_keep(const ConvParams& p, const PackedSequence& s) {
    using V = ConvVec<T, VEC>;
    const uzu_causal_conv_args& a = p.a;
    constexpr uint32_t kept = TAPS - 1;
    const uint32_t c = (blockIdx.x % p.groups * CC_THREADS + threadIdx.x) * VEC;
    const T* in = reinterpret_cast<const T*>(a.input) + (size_t)s.first * a.input_stride + c;
    T* state = reinterpret_cast<T*>(a.state) + (size_t)s.slot() * kept * a.channels + c;
    V v[TAPS > 1 ? TAPS - 1 : 1];      // (all read before one is written)
#pragma unroll
    for (uint32_t k = 0; k < kept; ++k) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[k].v[i] = ss_t<T>(0.0f);
        if (s.rows + k >= kept) v[k] = *reinterpret_cast<const V*>(in + (size_t)(s.rows + k - kept) * a.input_stride);
        else if (!s.fresh()) v[k] = *reinterpret_cast<const V*>(state + (size_t)(s.rows + k) * a.channels);
    }
#pragma unroll
    for (uint32_t k = 0; k < kept; ++k) *reinterpret_cast<V*>(state + (size_t)k * a.channels) = v[k];
}

template <typename T, int VEC, int TAPS>
__global__ void __launch_bounds__(CC_THREADS) causal_conv_kernel(const __grid_constant__ ConvParams p) {
    using V = ConvVec<T, VEC>;
    constexpr int BATCH = 8;
    pdl_launch_dependents();
    pdl_wait();
    const uzu_causal_conv_args& a = p.a;
    const uint32_t c = (blockIdx.x % p.groups * CC_THREADS + threadIdx.x) * VEC;
    if (c >= a.channels) return;
    const uint32_t tile = blockIdx.x / p.groups, q = ss_find(p.table, tile);
    const PackedSequence s = p.table.s[q];
    const uint32_t t0 = (tile - s.tile0) * p.strip, t1 = min(t0 + p.strip, s.rows);
    constexpr uint32_t kept = TAPS - 1;
    const T* in = reinterpret_cast<const T*>(a.input) + (size_t)s.first * a.input_stride + c;
    T* out = reinterpret_cast<T*>(a.output) + (size_t)s.first * a.output_stride + c;
    T* state = reinterpret_cast<T*>(a.state) + (size_t)s.slot() * kept * a.channels + c;

    constexpr int PAIRS = (VEC + 1) / 2;      // (one channel: a pair's second half is nobody's)
    float2 w[TAPS][PAIRS], bias[PAIRS];
#pragma unroll
    for (int i = 0; i < 2 * PAIRS; ++i) {
        const bool there = i < VEC;
        (i & 1 ? bias[i / 2].y : bias[i / 2].x) = there && a.bias ? reinterpret_cast<const float*>(a.bias)[c + i] : 0.0f;
#pragma unroll
        for (int j = 0; j < TAPS; ++j) (i & 1 ? w[j][i / 2].y : w[j][i / 2].x) = there ? reinterpret_cast<const float*>(a.weights)[(size_t)(c + i) * TAPS + j] : 0.0f;
    }
    // the inputs before the strip, oldest first
    V past[TAPS > 1 ? TAPS - 1 : 1];
#pragma unroll
    for (int j = 0; j < TAPS - 1; ++j) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) past[j].v[i] = ss_t<T>(0.0f);
        if (t0) past[j] = *reinterpret_cast<const V*>(in + (size_t)(t0 - kept + j) * a.input_stride);
        else if (!s.fresh()) past[j] = *reinterpret_cast<const V*>(state + (size_t)j * a.channels);
    }
    float2 u[TAPS][PAIRS];      // u[TAPS - 1]: the row at hand
    auto pairs = [](const V& v, float2 (&to)[PAIRS]) {
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) to[i] = make_float2(ss_f(v.v[2 * i]), VEC > 1 ? ss_f(v.v[VEC > 1 ? 2 * i + 1 : 0]) : 0.0f);
    };
#pragma unroll
    for (int j = 0; j < TAPS - 1; ++j) pairs(past[j], u[j]);

    auto step = [&](const V& row) {
        V o;
        pairs(row, u[TAPS - 1]);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            float2 y = bias[i];
#pragma unroll
            for (int j = 0; j < TAPS; ++j) y = ss_fma2(w[j][i], u[j][i], y);
            if (a.activation == UZU_ACT_SILU) y = ss_silu2(y);
            o.v[2 * i] = ss_t<T>(y.x);
            if (VEC > 1) o.v[VEC > 1 ? 2 * i + 1 : 0] = ss_t<T>(y.y);
#pragma unroll
            for (int j = 0; j < TAPS - 1; ++j) u[j][i] = u[j + 1][i];
        }
        return o;
    };
    const T* from = in + (size_t)t0 * a.input_stride;
    T* to = out + (size_t)t0 * a.output_stride;
    uint32_t left = t1 - t0;
    for (; left >= BATCH; left -= BATCH) {
        V rows[BATCH];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) rows[b] = *reinterpret_cast<const V*>(from + (size_t)b * a.input_stride);
#pragma unroll
        for (int b = 0; b < BATCH; ++b) *reinterpret_cast<V*>(to + (size_t)b * a.output_stride) = step(rows[b]);
        from += (size_t)BATCH * a.input_stride;
        to += (size_t)BATCH * a.output_stride;
    }
    for (; left; --left) {
        *reinterpret_cast<V*>(to) = step(*reinterpret_cast<const V*>(from));
        from += a.input_stride;
        to += a.output_stride;
    }
    if (t0 == 0) conv_keep<T, VEC, TAPS>(p, s);
}

const char* conv_check(const uzu_causal_conv_args* a) {
    if (!a) return "null arguments";
    if (!ss_data_type(a->data_type)) return "data_type must be bf16, f32 or f16";
    if (a->activation != UZU_ACT_SILU && a->activation != UZU_ACT_IDENTITY) return "the activation must be silu or identity";
    if (a->taps == 0 || a->taps > 8) return "taps must be in 1 .. 8";
    if (a->channels == 0 || a->channels > 65535 * CC_THREADS) return "channels must be in 1 .. 8388480";
    if (a->input_stride < a->channels || a->output_stride < a->channels) return "a row is shorter than its channels";
    if (const char* e = check_sequences(a->sequences, a->sequence_count, a->rows, a->slots)) return e;
    if (a->sequence_count == 0) return nullptr;
    if (!a->input || !a->output || !a->weights || (a->taps > 1 && !a->state)) return "null operand";
    const uint64_t size = ss_size(a->data_type);
    if ((a->input | a->output | (a->taps > 1 ? a->state : 0)) % size || (a->weights | a->bias) % 4) return "an operand is not aligned to its elements";
    if (rows_overlap(a->input, a->input_stride, a->channels, a->output, a->output_stride, a->channels, a->rows, size)) return "input and output overlap";
    const uint64_t state_bytes = (uint64_t)a->slots * (a->taps - 1) * a->channels * size;
    if (bytes_overlap(a->state, state_bytes, a->input, rows_extent(a->rows, a->input_stride, a->channels, size)) ||
        bytes_overlap(a->state, state_bytes, a->output, rows_extent(a->rows, a->output_stride, a->channels, size)))
        return "the state overlaps rows";
    return nullptr;
}

template <typename T, int VEC>
void conv_launch(uzu_command_buffer* cmd, ConvParams& p) {
    p.groups = (p.a.channels + CC_THREADS * VEC - 1) / (CC_THREADS * VEC);
    const dim3 grid(p.table.tiles * p.groups);
    auto go = [&](auto kernel) { launch(cmd, "causal_conv_kernel", kernel, grid, dim3(CC_THREADS), 0, p); };
    // (a kernel for each number of taps: one with more would multiply rows outside the window by zeros, which makes NaN of an infinity)
    switch (p.a.taps) {
        case 1: return go(causal_conv_kernel<T, VEC, 1>);
        case 2: return go(causal_conv_kernel<T, VEC, 2>);
        case 3: return go(causal_conv_kernel<T, VEC, 3>);
        case 4: return go(causal_conv_kernel<T, VEC, 4>);
        case 5: return go(causal_conv_kernel<T, VEC, 5>);
        case 6: return go(causal_conv_kernel<T, VEC, 6>);
        case 7: return go(causal_conv_kernel<T, VEC, 7>);
        default: return go(causal_conv_kernel<T, VEC, 8>);
    }
}
template <typename T>
void conv_by_alignment(uzu_command_buffer* cmd, ConvParams& p) {
    constexpr int VEC = 8 / sizeof(T);
    const uzu_causal_conv_args& a = p.a;
    const bool wide = a.channels % VEC == 0 && a.input_stride % VEC == 0 && a.output_stride % VEC == 0 && ((a.input | a.output | a.state) & 15u) == 0;
    if (wide) conv_launch<T, VEC>(cmd, p);
    else conv_launch<T, 1>(cmd, p);
}

}  // namespace
}  // namespace uzu

using namespace uzu;

extern "C" {

uzu_status uzu_causal_conv_validate(const uzu_causal_conv_args* a) {
    const char* e = conv_check(a);
    return e ? fail(UZU_ERROR_INVALID_ARGUMENT, std::string("causal_conv: ") + e) : UZU_OK;
}

void uzu_causal_conv_encode(uzu_command_buffer* cmd, const uzu_causal_conv_args* a) {
    if (!encodable(cmd, "causal_conv")) return;
    if (const char* e = conv_check(a)) {
        cmd->record_error(UZU_ERROR_INVALID_ARGUMENT, std::string("causal_conv: ") + e);
        return;
    }
    ConvParams p{};
    p.a = *a;
    // the longest strips that still give every SM a dozen warps: a strip reads taps - 1 rows again
    const uint64_t threads = (uint64_t)a->channels * ss_size(a->data_type) / 16 + 1;
    p.strip = 64;
    while (p.strip > 8 && threads * (a->rows / p.strip + 1) < (uint64_t)cmd->ctx->sm_count * 384) p.strip /= 2;
    for (uint32_t begin = 0; begin < a->sequence_count;) {
        auto tiles_of = [&](uint32_t rows) { return std::max(1u, (uint32_t)(((uint64_t)rows + p.strip - 1) / p.strip)); };
        begin = fill_sequences(p.table, a->sequences, a->sequence_count, begin, tiles_of);
        if (a->data_type == UZU_DT_F32) conv_by_alignment<float>(cmd, p);
        else if (a->data_type == UZU_DT_F16) conv_by_alignment<__half>(cmd, p);
        else conv_by_alignment<__nv_bfloat16>(cmd, p);
    }
}

}  // extern "C"
