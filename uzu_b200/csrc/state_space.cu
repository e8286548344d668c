// Selective state space scan token by token, for every type and shape (prompts in bf16 of the usual shapes take state_space_umma.cu), and one token of running
// sequences in one launch: S_t = exp(step a) S_(t-1) + step x_t b_t^T, y_t = S_t c_t + d x_t, out = y silu(z).
//
// Scan: a CTA has 32 rows p of a head's state, four threads a row with every fourth group of four columns in registers. Rows of 16 tokens are converted into shared
// memory while the batch before them is walked, four tokens side by side. Bound by the way through a batch (3 us of 16 tokens with one CTA an SM: its loads, two barriers,
// the walk): long sequences of few heads are cut into parts whose states are summed first, so that several CTAs share an SM. Two sequences of 1001 f32 tokens, 24 heads of 64 x 64:
// 70 us (whole 125 us); 1400 bf16 tokens of 80 heads of 64 x 40 280 us; 8192 tokens of 64 heads of 64 x 128 1370 us in f16 and 1210 in f32 (bf16 on the tensor cores 112). Up to a state
// size of 128 the kernels spill 4 to 36 bytes of a thread's registers.
//
// Step: bound by the state, read and written once. A CTA has up to 64 rows p of one head of one sequence. What the convolution takes is asked for first, then all of the state;
// the CTA convolves its x channels and its group's b and c while that comes. The conv slots of b and c are read by all CTAs of the group: each counts itself when it has
// them, the last one writes the new inputs and takes the count back to zero. 64 rows of 80 heads of 64 x 128: 74 us, 4.6 TB/s (as many bytes multiplied in place: 53 us); 256 rows of 128 heads 486 us
// (three CTAs an SM, by registers, do not cover all of a CTA's phases; 32 rows a CTA: 5 percent slower; one CTA an SM that streams the state through shared memory by bulk copies: slower too).
#include "state_space.cuh"

namespace uzu {

namespace {

constexpr uint32_t SS_THREADS = 128, SS_BATCH = 16, SS_ROWS = 32;

struct ScanParams {
    uzu_state_space_scan_args a;
    float* ends;       // of the parts: [tile][heads, head_dim, state_size]; the last part's place holds a copy of the start
    float* logs;       // [tile][heads]: the logarithm of all decays of a part
    SequenceTable table;
};

// GROUPS: of four columns a thread; columns past state_size are zeros. STATE: only the state at the end of every part but the last
template <typename T, int GROUPS, bool STATE>
__global__ void __launch_bounds__(SS_THREADS) state_space_scan_kernel(const __grid_constant__ ScanParams p) {
    constexpr uint32_t COLS = 16 * GROUPS, PER = SS_BATCH * COLS / SS_THREADS, XPER = SS_BATCH * SS_ROWS / SS_THREADS;
    __shared__ __align__(16) float bs[SS_BATCH][COLS], cs[SS_BATCH][COLS];
    __shared__ float xs[SS_BATCH][SS_ROWS], ys[SS_BATCH][SS_ROWS], zs[SS_BATCH][SS_ROWS], decay[SS_BATCH], step[SS_BATCH];
    pdl_launch_dependents();
    pdl_wait();
    const uzu_state_space_scan_args& a = p.a;
    const uint32_t tid = threadIdx.x, h = blockIdx.y, p0 = blockIdx.x * SS_ROWS, part = tid & 3u, pl = tid >> 2, N = a.state_size, P = a.head_dim;
    const uint32_t q = ss_find(p.table, blockIdx.z);
    PackedSequence s = p.table.s[q];
    const uint32_t parts = (q + 1 < p.table.count ? p.table.s[q + 1].tile0 : p.table.tiles) - s.tile0, part_of = blockIdx.z - s.tile0;
    if (STATE && part_of + 1 == parts) return;
    const uint32_t per = (s.rows + parts - 1) / parts, begin = min(s.rows, part_of * per);
    const bool nothing = s.rows == 0;
    s.first += begin;
    s.rows = min(s.rows - begin, per);
    const bool mine = p0 + pl < P;
    const T* x = reinterpret_cast<const T*>(a.x) + (size_t)s.first * a.x_stride + (size_t)h * P + p0;
    const T* z = reinterpret_cast<const T*>(a.z) + (size_t)s.first * a.z_stride + (size_t)h * P + p0;
    const T* dt = reinterpret_cast<const T*>(a.dt) + (size_t)s.first * a.dt_stride + h;
    const size_t group = (size_t)(h / (a.heads / a.groups)) * N;
    const T* b = reinterpret_cast<const T*>(a.b) + (size_t)s.first * a.b_stride + group;
    const T* c = reinterpret_cast<const T*>(a.c) + (size_t)s.first * a.c_stride + group;
    T* out = reinterpret_cast<T*>(a.out) + (size_t)s.first * a.out_stride + (size_t)h * P + p0;
    const size_t in_state = ((size_t)h * P + p0 + pl) * N, whole_state = (size_t)a.heads * P * N;
    float* state = reinterpret_cast<float*>(a.state) + s.slot() * whole_state + in_state;
    auto end_of = [&](uint32_t k) { return p.ends + (s.tile0 + k) * whole_state + in_state; };
    const float rate = reinterpret_cast<const float*>(a.a)[h], skip = a.d ? reinterpret_cast<const float*>(a.d)[h] : 0.0f;
    const float dt_bias = a.dt_bias ? reinterpret_cast<const float*>(a.dt_bias)[h] : 0.0f;

    float2 S[2 * GROUPS];
    auto each = [&](auto f) {      // of this thread's columns: index in S, column
#pragma unroll
        for (int i = 0; i < GROUPS; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float& v = j & 1 ? S[2 * i + j / 2].y : S[2 * i + j / 2].x;
                const uint32_t n = 16 * i + 4 * part + j;
                if (mine && n < N) f(v, n);
            }
    };
#pragma unroll
    for (int i = 0; i < 2 * GROUPS; ++i) S[i] = make_float2(0.0f, 0.0f);
    if (parts == 1 || (STATE && part_of == 0)) {
        if (!s.fresh()) each([&](float& v, uint32_t n) { v = state[n]; });
        if (STATE) each([&](float& v, uint32_t n) { end_of(parts - 1)[n] = v; });
    } else if (!STATE) {
        if (part_of == 0) each([&](float& v, uint32_t n) { v = end_of(parts - 1)[n]; });
        for (uint32_t k = 0; k < part_of; ++k) {      // the parts before, in order
            const float f = k ? expf(p.logs[(size_t)(s.tile0 + k) * a.heads + h]) : 0.0f;
            each([&](float& v, uint32_t n) { v = k ? fmaf(f, v, end_of(k)[n]) : end_of(k)[n]; });
        }
    }
    float log_sum = 0.0f;      // (thread 0 alone)
    T nb[PER], nc[PER], nx[XPER], nz[XPER];
    float nd = 0.0f;
    auto fetch = [&](uint32_t t) {
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) {
            const uint32_t e = tid + i * SS_THREADS, r = e / COLS, n = e % COLS;
            const bool there = t + r < s.rows && n < N;
            nb[i] = there ? b[(size_t)(t + r) * a.b_stride + n] : ss_t<T>(0.0f);
            if (!STATE) nc[i] = there ? c[(size_t)(t + r) * a.c_stride + n] : ss_t<T>(0.0f);
        }
#pragma unroll
        for (uint32_t i = 0; i < XPER; ++i) {
            const uint32_t e = tid + i * SS_THREADS, r = e / SS_ROWS, q = e % SS_ROWS;
            const bool there = t + r < s.rows && p0 + q < P;
            nx[i] = there ? x[(size_t)(t + r) * a.x_stride + q] : ss_t<T>(0.0f);
            if (!STATE) nz[i] = there && a.z ? z[(size_t)(t + r) * a.z_stride + q] : ss_t<T>(0.0f);
        }
        if (tid < SS_BATCH && t + tid < s.rows) nd = ss_f(dt[(size_t)(t + tid) * a.dt_stride]);
    };
    fetch(0);
    for (uint32_t t = 0; t < s.rows; t += SS_BATCH) {
        const uint32_t count = min(SS_BATCH, s.rows - t);
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) {
            const uint32_t e = tid + i * SS_THREADS;
            bs[e / COLS][e % COLS] = ss_f(nb[i]);
            if (!STATE) cs[e / COLS][e % COLS] = ss_f(nc[i]);
        }
#pragma unroll
        for (uint32_t i = 0; i < XPER; ++i) {
            const uint32_t e = tid + i * SS_THREADS;
            xs[e / SS_ROWS][e % SS_ROWS] = ss_f(nx[i]);
            if (!STATE) zs[e / SS_ROWS][e % SS_ROWS] = a.z ? ss_silu(ss_f(nz[i])) : 1.0f;
        }
        if (tid < SS_BATCH) {
            const float v = tid < count ? ss_step(nd, dt_bias, a.dt_softplus, a.dt_min, a.dt_max) : 0.0f;
            step[tid] = v;
            decay[tid] = tid < count ? expf(v * rate) : 1.0f;
            if (STATE) log_sum += v * rate;
        }
        __syncthreads();
        if (t + SS_BATCH < s.rows) fetch(t + SS_BATCH);
        // four tokens at a time: only a multiplication and an addition of the state depend on the token before, everything else of the four runs side by side (tokens behind the
        // last have a decay of 1 and a step of 0)
#pragma unroll 1
        for (uint32_t r0 = 0; r0 < count; r0 += 4) {
            float y[4];
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                const uint32_t r = r0 + k;
                const float sx = step[r] * xs[r][pl], f = decay[r];
                const float2 sx2 = make_float2(sx, sx), f2 = make_float2(f, f);
                float2 y0 = make_float2(0.0f, 0.0f), y1 = y0;
#pragma unroll
                for (int i = 0; i < GROUPS; ++i) {
                    const float4 bv = *reinterpret_cast<const float4*>(&bs[r][16 * i + 4 * part]);
                    S[2 * i] = ss_fma2(f2, S[2 * i], ss_mul2(sx2, make_float2(bv.x, bv.y)));
                    S[2 * i + 1] = ss_fma2(f2, S[2 * i + 1], ss_mul2(sx2, make_float2(bv.z, bv.w)));
                    if (STATE) continue;
                    const float4 cv = *reinterpret_cast<const float4*>(&cs[r][16 * i + 4 * part]);
                    y0 = ss_fma2(S[2 * i], make_float2(cv.x, cv.y), y0);
                    y1 = ss_fma2(S[2 * i + 1], make_float2(cv.z, cv.w), y1);
                }
                y[k] = (y0.x + y0.y) + (y1.x + y1.y);
            }
            if (STATE) continue;
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) y[k] += __shfl_xor_sync(0xffffffffu, y[k], 1);
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) y[k] += __shfl_xor_sync(0xffffffffu, y[k], 2);
            // thread `part` of a row writes its token
            const float mine_y = part == 0 ? y[0] : part == 1 ? y[1] : part == 2 ? y[2] : y[3];
            ys[r0 + part][pl] = fmaf(skip, xs[r0 + part][pl], mine_y);
        }
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < XPER; ++i) {
            const uint32_t e = tid + i * SS_THREADS, r = e / SS_ROWS, q = e % SS_ROWS;
            if (!STATE && r < count && p0 + q < P) out[(size_t)(t + r) * a.out_stride + q] = ss_t<T>(ys[r][q] * zs[r][q]);
        }
    }
    if (STATE) {
        each([&](float& v, uint32_t n) { end_of(part_of)[n] = v; });
        if (tid < SS_BATCH) {
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) log_sum += __shfl_xor_sync(0xffffu, log_sum, o);
            if (tid == 0 && p0 == 0) p.logs[(size_t)blockIdx.z * a.heads + h] = log_sum;
        }
    } else if (part_of + 1 == parts && (!nothing || s.fresh())) each([&](float& v, uint32_t n) { state[n] = v; });
}

// how many parts a sequence is cut into where `ctas` CTAs would run without cutting (four an SM run beside one another): the pass over the parts' states costs less than the one
// over the rows, so three parts pay
uint32_t scan_parts(uint32_t rows, uint64_t ctas, uint32_t sms) {
    const uint64_t room = 4ull * sms / std::max<uint64_t>(1, ctas);
    if (room < 3 || rows < 8 * SS_BATCH) return 1;
    const uint32_t want = (uint32_t)std::min<uint64_t>(room, rows / (2 * SS_BATCH)), per = (rows + want - 1) / want;
    return (rows + per - 1) / per;
}
uint64_t scan_ctas(const uzu_state_space_scan_args& a) { return (uint64_t)a.sequence_count * a.heads * ((a.head_dim + SS_ROWS - 1) / SS_ROWS); }
size_t scan_scratch_bytes(const uzu_state_space_scan_args& a, uint32_t sms) {
    uint64_t tiles = 0;
    for (uint32_t i = 0; i < a.sequence_count; ++i) tiles += scan_parts(a.sequences[i].rows, scan_ctas(a), sms);
    return tiles == a.sequence_count ? 0 : tiles * a.heads * ((uint64_t)a.head_dim * a.state_size + 1) * 4;
}

template <typename T>
void scan_launch(uzu_command_buffer* cmd, const ScanParams& p) {
    const dim3 grid((p.a.head_dim + SS_ROWS - 1) / SS_ROWS, p.a.heads, p.table.tiles);
    auto go = [&](auto state_only) {
        constexpr bool ST = decltype(state_only)::value;
        auto run = [&](auto kernel) { launch(cmd, "state_space_scan_kernel", kernel, grid, dim3(SS_THREADS), 0, p); };
        const uint32_t n = p.a.state_size;
        if (n <= 16) run(state_space_scan_kernel<T, 1, ST>);
        else if (n <= 64) run(state_space_scan_kernel<T, 4, ST>);
        else if (n <= 128) run(state_space_scan_kernel<T, 8, ST>);
        else run(state_space_scan_kernel<T, 16, ST>);
    };
    if (p.table.tiles > p.table.count) go(std::true_type{});
    go(std::false_type{});
}

const char* shape_check(uint32_t heads, uint32_t groups, uint32_t head_dim, uint32_t state_size, float dt_min, float dt_max, uint32_t data_type) {
    if (!ss_data_type(data_type)) return "data_type must be bf16, f32 or f16";
    if (heads == 0 || groups == 0 || heads % groups || heads > 65535) return "groups must divide heads, heads must be in 1 .. 65535";
    if (head_dim == 0 || head_dim > 256 || state_size == 0 || state_size > 256) return "head_dim and state_size must be in 1 .. 256";
    if (!(dt_min >= 0.0f) || !(dt_max >= dt_min)) return "0 <= dt_min <= dt_max is needed";
    return nullptr;
}

const char* scan_check(const uzu_state_space_scan_args* a) {
    if (!a) return "null arguments";
    if (const char* e = shape_check(a->heads, a->groups, a->head_dim, a->state_size, a->dt_min, a->dt_max, a->data_type)) return e;
    const uint64_t inner = (uint64_t)a->heads * a->head_dim, gn = (uint64_t)a->groups * a->state_size, size = ss_size(a->data_type);
    if (a->x_stride < inner || a->out_stride < inner || (a->z && a->z_stride < inner) || a->dt_stride < a->heads || a->b_stride < gn || a->c_stride < gn) return "a row is shorter than what it holds";
    if (const char* e = check_sequences(a->sequences, a->sequence_count, a->rows, a->slots)) return e;
    if (a->sequence_count == 0) return nullptr;
    if (!a->x || !a->dt || !a->b || !a->c || !a->a || !a->state || !a->out) return "null operand";
    if ((a->x | a->dt | a->b | a->c | a->z | a->out) % size || (a->a | a->d | a->dt_bias | a->state) % 4) return "an operand is not aligned to its elements";
    const struct { uint64_t at, stride, width; } in[5] = {{a->x, a->x_stride, inner}, {a->dt, a->dt_stride, a->heads}, {a->b, a->b_stride, gn}, {a->c, a->c_stride, gn}, {a->z, a->z_stride, inner}};
    const uint64_t state_bytes = (uint64_t)a->slots * inner * a->state_size * 4;
    for (const auto& r : in) {
        if (!r.at) continue;
        if (rows_overlap(r.at, r.stride, r.width, a->out, a->out_stride, inner, a->rows, size)) return "an input and the output overlap";
        if (bytes_overlap(r.at, rows_extent(a->rows, r.stride, r.width, size), a->state, state_bytes)) return "the state overlaps rows";
    }
    if (bytes_overlap(a->out, rows_extent(a->rows, a->out_stride, inner, size), a->state, state_bytes)) return "the state overlaps rows";
    if (a->scratch % 16) return "the scratch must be 16-byte aligned";
    return nullptr;
}

// ---- one token ------------------------------------------------------------------------------------------------------------------------------
// L threads a row of the state, NV groups of four columns each; PASSES rows p a thread
template <typename T, int L, int NV>
struct StepShape {
    static constexpr uint32_t ROWS = NV == 1 ? 64 : 32, AT_ONCE = SS_THREADS / L, PASSES = ROWS / AT_ONCE, COLS = 4 * L * NV;
};

template <typename T, int L, int NV>
__global__ void __launch_bounds__(SS_THREADS) state_space_step_kernel(const __grid_constant__ uzu_state_space_step_args a) {
    using Sh = StepShape<T, L, NV>;
    constexpr int PASSES = Sh::PASSES;
    constexpr uint32_t ROWS = Sh::ROWS, COLS = Sh::COLS;
    __shared__ __align__(16) float bs[COLS], cs[COLS];
    __shared__ float xs[ROWS], ys[ROWS];
    __shared__ uint32_t last;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t tid = threadIdx.x, lane = tid & 31u, part = tid % L, P = a.head_dim, N = a.state_size, slices = (P + ROWS - 1) / ROWS;
    const uint32_t row = blockIdx.y, h = blockIdx.x / slices, p0 = blockIdx.x % slices * ROWS, per_group = a.heads / a.groups, g = h / per_group;
    const uint32_t* slots = reinterpret_cast<const uint32_t*>(a.slots);
    const uint32_t slot = slots ? slots[row] : row;
    if (slot >= a.slot_count) return;
    // Asked for first: what the convolution takes, so that it is computed while the state is on its way. This CTA's channels: its rows of x, then b and c of the group.
    constexpr int PER = (ROWS + 2 * COLS + SS_THREADS - 1) / SS_THREADS;
    const uint32_t inner = a.heads * P, channels = inner + 2 * a.groups * N, kept = a.taps - 1, xrows = min(ROWS, P - p0);
    const T* now = reinterpret_cast<const T*>(a.xbc) + (size_t)row * a.xbc_stride;
    T* past = reinterpret_cast<T*>(a.conv_state) + (size_t)slot * kept * channels;
    const float *w = reinterpret_cast<const float*>(a.conv_weights), *bias = reinterpret_cast<const float*>(a.conv_bias);
    const bool four = kept == 3 && (a.conv_weights & 15u) == 0;
    auto channel = [&](uint32_t i) { return i < xrows ? h * P + p0 + i : i < xrows + N ? inner + g * N + (i - xrows) : inner + a.groups * N + g * N + (i - xrows - N); };
    T u[PER][8];      // the slot's inputs, oldest first, and (7) the row's own
    float4 w4[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const uint32_t i = tid + k * SS_THREADS;
        if (i >= xrows + 2 * N) break;
        const uint32_t c = channel(i);
#pragma unroll
        for (uint32_t j = 0; j < 7; ++j)
            if (j < kept) u[k][j] = past[(size_t)j * channels + c];
        u[k][7] = now[c];
        if (four) w4[k] = *reinterpret_cast<const float4*>(w + (size_t)c * 4);
    }
    float* state = reinterpret_cast<float*>(a.state) + (((size_t)slot * a.heads + h) * P + p0) * N;
    const bool vector = N % 4 == 0 && (a.state & 15u) == 0;
    float4 S[PASSES][NV];
#pragma unroll
    for (int i = 0; i < PASSES; ++i)
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const uint32_t pl = i * Sh::AT_ONCE + tid / L, n = 4 * (v * L + part);
            S[i][v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (p0 + pl >= P || n >= N) continue;
            const float* at = state + (size_t)pl * N + n;
            if (vector) S[i][v] = __ldcs(reinterpret_cast<const float4*>(at));      // (read once: not to push out what others share)
            else {
                S[i][v].x = at[0];
                if (n + 1 < N) S[i][v].y = at[1];
                if (n + 2 < N) S[i][v].z = at[2];
                if (n + 3 < N) S[i][v].w = at[3];
            }
        }
    // a slot that an earlier row names is that row's
    bool taken = false;
    if (slots)
        for (uint32_t r = tid; r < row; r += SS_THREADS) taken |= slots[r] == slot;
    if (__syncthreads_or(taken)) return;

#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const uint32_t i = tid + k * SS_THREADS;
        if (i >= xrows + 2 * N) break;
        const uint32_t c = channel(i);
        float y = bias ? bias[c] : 0.0f;
        if (four) y = fmaf(w4[k].w, ss_f(u[k][7]), fmaf(w4[k].z, ss_f(u[k][2]), fmaf(w4[k].y, ss_f(u[k][1]), fmaf(w4[k].x, ss_f(u[k][0]), y))));
        else {
#pragma unroll
            for (uint32_t j = 0; j < 7; ++j)
                if (j < kept) y = fmaf(w[(size_t)c * a.taps + j], ss_f(u[k][j]), y);
            y = fmaf(w[(size_t)c * a.taps + kept], ss_f(u[k][7]), y);
        }
        if (a.activation == UZU_ACT_SILU) y = ss_silu(y);
        if (i < xrows) {      // nobody else reads or writes these
            xs[i] = y;
#pragma unroll
            for (uint32_t j = 0; j < 7; ++j)
                if (j < kept) past[(size_t)j * channels + c] = j + 1 < kept ? u[k][j < 6 ? j + 1 : 6] : u[k][7];
        } else if (i < xrows + N) bs[i - xrows] = y;
        else cs[i - xrows - N] = y;
    }
    for (uint32_t n = N + tid; n < COLS; n += SS_THREADS) bs[n] = cs[n] = 0.0f;
    const float step = ss_step(ss_f(reinterpret_cast<const T*>(a.dt)[(size_t)row * a.dt_stride + h]), a.dt_bias ? reinterpret_cast<const float*>(a.dt_bias)[h] : 0.0f, a.dt_softplus, a.dt_min, a.dt_max);
    const float decay = expf(step * reinterpret_cast<const float*>(a.a)[h]);
    __syncthreads();      // (and every thread of the CTA has read b's and c's inputs)
    if (kept && tid == 0) {
        unsigned int* ticket = reinterpret_cast<unsigned int*>(a.tickets) + (size_t)row * a.groups + g;
        // (no fence: what was read is in registers, which no later write changes)
        last = atomicAdd(ticket, 1u) == per_group * slices - 1;
        if (last) *ticket = 0;
    }

    float y[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const uint32_t pl = i * Sh::AT_ONCE + tid / L;
        const float sx = pl < xrows ? step * xs[pl] : 0.0f;
        y[i] = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const uint32_t n = 4 * (v * L + part);
            const float4 bv = *reinterpret_cast<const float4*>(&bs[n]), cv = *reinterpret_cast<const float4*>(&cs[n]);
            float4& s = S[i][v];
            s.x = fmaf(decay, s.x, sx * bv.x);
            s.y = fmaf(decay, s.y, sx * bv.y);
            s.z = fmaf(decay, s.z, sx * bv.z);
            s.w = fmaf(decay, s.w, sx * bv.w);
            y[i] = fmaf(s.x, cv.x, fmaf(s.y, cv.y, fmaf(s.z, cv.z, fmaf(s.w, cv.w, y[i]))));
            if (p0 + pl >= P || n >= N) continue;
            float* at = state + (size_t)pl * N + n;
            if (vector) __stcs(reinterpret_cast<float4*>(at), s);
            else {
                at[0] = s.x;
                if (n + 1 < N) at[1] = s.y;
                if (n + 2 < N) at[2] = s.z;
                if (n + 3 < N) at[3] = s.w;
            }
        }
    }
    // sums over the L threads of a row: while a thread has several rows it gives half of them away
    uint32_t mine = 0;
    int have = PASSES;
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) {
        if (have > 1) {
            have /= 2;
            const bool upper = (lane & o) != 0;
            mine += upper ? have : 0;
#pragma unroll
            for (int i = 0; i < PASSES / 2; ++i) {
                if (i >= have) break;
                const float give = upper ? y[i] : y[i + have], keep = upper ? y[i + have] : y[i];
                y[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
            }
        } else y[0] += __shfl_xor_sync(0xffffffffu, y[0], o);
    }
    static_assert(PASSES <= L, "a thread ends with one row");
    if ((part & (L / PASSES - 1)) == 0) ys[mine * Sh::AT_ONCE + tid / L] = y[0];
    __syncthreads();
    for (uint32_t i = tid; i < xrows; i += SS_THREADS) {
        const uint32_t c = h * P + p0 + i;
        float v = a.d ? fmaf(reinterpret_cast<const float*>(a.d)[h], xs[i], ys[i]) : ys[i];
        if (a.z) v *= ss_silu(ss_f(reinterpret_cast<const T*>(a.z)[(size_t)row * a.z_stride + c]));
        reinterpret_cast<T*>(a.out)[(size_t)row * a.out_stride + c] = ss_t<T>(v);
    }
    if (kept && last) {      // b's and c's inputs, read by all: one back
        for (uint32_t i = xrows + tid; i < xrows + 2 * N; i += SS_THREADS) {
            const uint32_t c = channel(i);
            for (uint32_t j = 0; j < kept; ++j) past[(size_t)j * channels + c] = j + 1 < kept ? past[(size_t)(j + 1) * channels + c] : now[c];
        }
    }
}

const char* step_check(const uzu_state_space_step_args* a) {
    if (!a) return "null arguments";
    if (const char* e = shape_check(a->heads, a->groups, a->head_dim, a->state_size, a->dt_min, a->dt_max, a->data_type)) return e;
    if (a->activation != UZU_ACT_SILU && a->activation != UZU_ACT_IDENTITY) return "the activation must be silu or identity";
    if (a->taps == 0 || a->taps > 8) return "taps must be in 1 .. 8";
    if (a->rows > 65535) return "at most 65535 rows";
    const uint64_t inner = (uint64_t)a->heads * a->head_dim, channels = inner + 2ull * a->groups * a->state_size, size = ss_size(a->data_type);
    if (channels >> 31) return "too many channels";
    if (a->xbc_stride < channels || a->dt_stride < a->heads || a->out_stride < inner || (a->z && a->z_stride < inner)) return "a row is shorter than what it holds";
    if (!a->slots && a->rows > a->slot_count) return "more rows than slots, and no list of slots";
    if (a->rows == 0) return nullptr;
    if (!a->xbc || !a->dt || !a->conv_weights || !a->a || !a->state || !a->out || (a->taps > 1 && (!a->conv_state || !a->tickets))) return "null operand";
    if ((a->xbc | a->dt | a->z | a->out | a->conv_state) % size || (a->conv_weights | a->conv_bias | a->a | a->d | a->dt_bias | a->state | a->slots | a->tickets) % 4)
        return "an operand is not aligned to its elements";
    const struct { uint64_t at, stride, width; } in[3] = {{a->xbc, a->xbc_stride, channels}, {a->dt, a->dt_stride, a->heads}, {a->z, a->z_stride, inner}};
    const uint64_t state_bytes = (uint64_t)a->slot_count * inner * a->state_size * 4, conv_bytes = (uint64_t)a->slot_count * (a->taps - 1) * channels * size;
    const uint64_t out_bytes = rows_extent(a->rows, a->out_stride, inner, size);
    for (const auto& r : in) {
        if (!r.at) continue;
        if (rows_overlap(r.at, r.stride, r.width, a->out, a->out_stride, inner, a->rows, size)) return "an input and the output overlap";
        const uint64_t bytes = rows_extent(a->rows, r.stride, r.width, size);
        if (bytes_overlap(r.at, bytes, a->state, state_bytes) || bytes_overlap(r.at, bytes, a->conv_state, conv_bytes)) return "the state overlaps rows";
    }
    if (bytes_overlap(a->out, out_bytes, a->state, state_bytes) || bytes_overlap(a->out, out_bytes, a->conv_state, conv_bytes)) return "the state overlaps rows";
    if (bytes_overlap(a->state, state_bytes, a->conv_state, conv_bytes)) return "the states overlap";
    return nullptr;
}

template <typename T>
void step_launch(uzu_command_buffer* cmd, const uzu_state_space_step_args& a) {
    auto go = [&](auto kernel, uint32_t rows) { launch(cmd, "state_space_step_kernel", kernel, dim3(a.heads * ((a.head_dim + rows - 1) / rows), a.rows), dim3(SS_THREADS), 0, a); };
    const uint32_t n = a.state_size;
    if (n <= 16) go(state_space_step_kernel<T, 4, 1>, StepShape<T, 4, 1>::ROWS);
    else if (n <= 32) go(state_space_step_kernel<T, 8, 1>, StepShape<T, 8, 1>::ROWS);
    else if (n <= 64) go(state_space_step_kernel<T, 16, 1>, StepShape<T, 16, 1>::ROWS);
    else if (n <= 128) go(state_space_step_kernel<T, 32, 1>, StepShape<T, 32, 1>::ROWS);
    else go(state_space_step_kernel<T, 32, 2>, StepShape<T, 32, 2>::ROWS);
}

}  // namespace
}  // namespace uzu

using namespace uzu;

extern "C" {

uzu_status uzu_state_space_scan_validate(const uzu_state_space_scan_args* a) {
    const char* e = scan_check(a);
    return e ? fail(UZU_ERROR_INVALID_ARGUMENT, std::string("state_space_scan: ") + e) : UZU_OK;
}

size_t uzu_state_space_scan_scratch_bytes(uzu_context* ctx, const uzu_state_space_scan_args* a) {
    // (what the call's checks would refuse needs none)
    if (!ctx || !a || (a->sequence_count && !a->sequences) || shape_check(a->heads, a->groups, a->head_dim, a->state_size, a->dt_min, a->dt_max, a->data_type)) return 0;
    return scan_umma_applicable(*a) ? scan_umma_scratch_bytes(ctx, *a) : scan_scratch_bytes(*a, ctx->sm_count);
}

void uzu_state_space_scan_encode(uzu_command_buffer* cmd, const uzu_state_space_scan_args* a) {
    if (!encodable(cmd, "state_space_scan")) return;
    if (const char* e = scan_check(a)) {
        cmd->record_error(UZU_ERROR_INVALID_ARGUMENT, std::string("state_space_scan: ") + e);
        return;
    }
    if (a->sequence_count == 0) return;
    if (scan_umma_applicable(*a) && encode_scan_umma(cmd, *a)) return;
    ScanParams p{};
    p.a = *a;
    const uint32_t sms = cmd->ctx->sm_count;
    const size_t need = scan_scratch_bytes(*a, sms);
    const bool cut = need && a->scratch && a->scratch_bytes >= need;
    for (uint32_t begin = 0; begin < a->sequence_count;) {
        begin = fill_sequences(p.table, a->sequences, a->sequence_count, begin, [&](uint32_t rows) { return cut ? scan_parts(rows, scan_ctas(*a), sms) : 1u; });
        p.ends = reinterpret_cast<float*>(a->scratch);      // (one launch behind the other: the next may use the same)
        p.logs = p.ends + (uint64_t)p.table.tiles * a->heads * a->head_dim * a->state_size;
        if (a->data_type == UZU_DT_F32) scan_launch<float>(cmd, p);
        else if (a->data_type == UZU_DT_F16) scan_launch<__half>(cmd, p);
        else scan_launch<__nv_bfloat16>(cmd, p);
    }
}

uzu_status uzu_state_space_step_validate(const uzu_state_space_step_args* a) {
    const char* e = step_check(a);
    return e ? fail(UZU_ERROR_INVALID_ARGUMENT, std::string("state_space_step: ") + e) : UZU_OK;
}

void uzu_state_space_step_encode(uzu_command_buffer* cmd, const uzu_state_space_step_args* a) {
    if (!encodable(cmd, "state_space_step")) return;
    if (const char* e = step_check(a)) {
        cmd->record_error(UZU_ERROR_INVALID_ARGUMENT, std::string("state_space_step: ") + e);
        return;
    }
    if (a->rows == 0) return;
    if (a->data_type == UZU_DT_F32) step_launch<float>(cmd, *a);
    else if (a->data_type == UZU_DT_F16) step_launch<__half>(cmd, *a);
    else step_launch<__nv_bfloat16>(cmd, *a);
}

}  // extern "C"
