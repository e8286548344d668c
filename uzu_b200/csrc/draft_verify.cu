// Verification of drafted tokens against the target's probabilities, and the token behind the kept ones.
//
// A cluster of CTAs has a sequence; a warp has the same run of the vocabulary in every row, and asks for the next row's numbers before it sums up one's. One reading of all rows
// gives each row's maximum and sum (f32 in a warp, f64 from there on); the CTAs exchange them and all come to the same first refusal. Only the row that a token is drawn from is read
// again (it lies in L2), in f64, as is the draft's: where a sum of weights passes its aim must not depend on f32 roundings, nor must whether a draft is kept: one that the f32 sums leave open has its row read in
// f64 as well. One pass gives all its sums: which tokens have p > q is known from the f32 sums but for those where both are alike to 2^-22 or so; so the weights of the others are summed before their
// divisors are known, numerators and denominators by themselves, and once more, with the divisors, only where those few could matter. Then the warp's run where the sum passes the aim is looked through by its
// whole CTA.
// What bounds it: instructions (0.64 a cycle and scheduler) for exponentials of all rows and, at half rate, of two rows in f64; 74 million numbers and 16 million of them again. 64 sequences
// of four drafts, vocabulary of 128256 (148 MB): 95 to 97 us; 427 with a row after another and the library's exponential in f64 three times, 212 with rows ahead and the series here, 112 with one
// pass in f64 and sums by warps, 91 to 93 with registers for four CTAs an SM (one wave) and without the decisions in f64, which spill 44 bytes. One sequence: 85 -> 29 to 35 us.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "row_sequences.h"

namespace uzu {

namespace {

constexpr uint32_t DV_TILE = 256, DV_GROUP = 4, DV_DRAFTS = 16, DV_ROWS = 2 * DV_DRAFTS + 1;

constexpr float DV_COLDEST = 0x1p-60f;      // (1 / temperature stays a number)

struct DvParams {
    uzu_draft_verify_args a;
    uint32_t tiles;      // of 256 tokens, of a warp
};

template <typename T> __device__ __forceinline__ T dv_nothing();
template <> __device__ __forceinline__ __nv_bfloat16 dv_nothing() { return __ushort_as_bfloat16(0xff80u); }
template <> __device__ __forceinline__ __half dv_nothing() { return __ushort_as_half(0xfc00u); }
template <typename T> __device__ __forceinline__ float dv_f(T v);
template <> __device__ __forceinline__ float dv_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float dv_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float dv_f(float v) { return v; }

// a lane's eight tokens of a tile; -infinity behind the last
template <typename T, bool WIDE>
__device__ __forceinline__ void dv_load(const T* row, uint32_t at, uint32_t vocab, T (&v)[8]) {
    if (WIDE && at + 8 <= vocab) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(row + at)[i];
    } else {
        T none;
        if constexpr (sizeof(T) == 4) none = -INFINITY;
        else none = dv_nothing<T>();
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = at + i < vocab ? row[at + i] : none;
    }
}

__device__ __forceinline__ float dv_exp2(float x) {      // 2 ulp; what is below 2^-126 is zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^y for -1000 <= y <= 0, within 2^-37 of itself: the series of the exponential around the nearest power of two
__device__ __forceinline__ double dv_power(double y) {
    constexpr double magic = 6755399441055744.0;      // 1.5 * 2^52: a sum with it has the rounded integer in its low word
    const double t = y + magic, f = y - (t - magic);
    constexpr double l = 0.69314718055994530942;      // ln 2
    constexpr double c2 = l * l / 2, c3 = c2 * l / 3, c4 = c3 * l / 4, c5 = c4 * l / 5, c6 = c5 * l / 6, c7 = c6 * l / 7, c8 = c7 * l / 8, c9 = c8 * l / 9;
    double v = fma(c9, f, c8);
    v = fma(v, f, c7);
    v = fma(v, f, c6);
    v = fma(v, f, c5);
    v = fma(v, f, c4);
    v = fma(v, f, c3);
    v = fma(v, f, c2);
    v = fma(v, f, l);
    v = fma(v, f, 1.0);
    return __hiloint2double(__double2hiint(v) + (__double2loint(t) << 20), __double2loint(v));
}
// weights exp((x - most) / temperature) of a row whose largest number is `most`. The difference first: x * k - most * k, most * k rounded, would be off by what a cold row's or large
// numbers' k * most has of roundings, and the largest number's weight, 1, would be any other
struct DvHeat {
    double most, k;      // (x - most) k: the exponent of 2
    __device__ __forceinline__ DvHeat(float most, float temperature) : most((double)most), k(1.4426950408889634074 / (double)temperature) {}
    __device__ __forceinline__ double operator()(float x) const {
        const double y = ((double)x - most) * k;
        return y >= -1000.0 ? dv_power(y) : 0.0;
    }
};

struct DvRow {
    float most;          // NaN: no distribution
    uint32_t index;      // of the largest, the lowest of several
    double sum;          // of exp((x - most) / temperature)
};
__device__ __forceinline__ double dv_warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// parts of a row, one a lane (most = -infinity: nothing), to a whole one in all lanes; per: log2 e / temperature
__device__ __forceinline__ DvRow dv_merge(DvRow m, float per) {
    const float top = warp_max(m.most);
    DvRow all;
    all.most = top;
    all.index = __reduce_min_sync(0xffffffffu, m.most == top ? m.index : UZU_NO_TOKEN);
    // (a part of nothing but -infinity and NaN has a sum that is NaN; NaN stays NaN)
    all.sum = dv_warp_sum(m.most == -INFINITY ? m.sum : m.most == top ? (top < INFINITY ? m.sum : m.sum * __longlong_as_double(0x7ff8000000000000ll)) : m.sum * (double)exp2f((m.most - top) * per));
    return all;
}

template <uint32_t WARPS>
struct DvShared {
    DvRow part[DV_ROWS], row[DV_ROWS];      // this CTA's run; the whole vocabulary
    float row_most[DV_ROWS][WARPS], row_sum[DV_ROWS][WARPS];
    uint32_t row_index[DV_ROWS][WARPS];
    double sums[5][WARPS], cta[5];
    uint32_t accepted, close, token;
};

template <typename T, bool WIDE, uint32_t WARPS, uint32_t CLUSTER>
__global__ void __launch_bounds__(WARPS * 32, WARPS == 8 ? 4 : 1) draft_verify_kernel(const __grid_constant__ DvParams p) {
    namespace cg = cooperative_groups;
    static_assert(WARPS <= 32 && CLUSTER <= 32, "a lane for each");
    __shared__ DvShared<WARPS> s;
    cg::cluster_group cluster = cg::this_cluster();
    pdl_launch_dependents();
    pdl_wait();
    const uzu_draft_verify_args& a = p.a;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, rank = cluster.block_rank(), sequence = blockIdx.x / CLUSTER, k1 = a.drafts + 1, vocab = a.vocab;
    const bool greedy = a.temperature == 0.0f, with_draft = a.draft_logits && !greedy;
    const uint32_t count = a.draft_counts ? min(reinterpret_cast<const uint32_t*>(a.draft_counts)[sequence], a.drafts) : a.drafts;
    const uint32_t rows = count + 1 + (with_draft ? count : 0u);      // targets, then drafts
    const uint32_t* drafted = reinterpret_cast<const uint32_t*>(a.drafted) + (size_t)sequence * a.drafts;
    const float* uniforms = reinterpret_cast<const float*>(a.uniforms) + (size_t)sequence * k1;
    auto row_of = [&](uint32_t r) {
        return r <= count ? reinterpret_cast<const T*>(a.target_logits) + ((size_t)sequence * k1 + r) * a.target_stride
                          : reinterpret_cast<const T*>(a.draft_logits) + ((size_t)sequence * a.drafts + (r - count - 1)) * a.draft_stride;
    };
    const uint32_t first = (rank * WARPS + warp) * p.tiles * DV_TILE;      // this warp's run of tokens (behind the last one there is none)
    const float per_target = greedy ? 1.0f : 1.4426950408889634f / a.temperature, per_draft = with_draft ? 1.4426950408889634f / a.draft_temperature : 1.0f;

    // ---- maxima and sums of all rows, some tiles of a row at a time ----
    {
        const uint32_t groups = (p.tiles + DV_GROUP - 1) / DV_GROUP, all = rows * groups;
        alignas(16) T next[DV_GROUP][8];
        auto ask = [&](uint32_t r, uint32_t group) {
            const T* row = row_of(r);
#pragma unroll
            for (uint32_t t = 0; t < DV_GROUP; ++t) {
                const uint32_t tile = group * DV_GROUP + t;
                dv_load<T, WIDE>(row, tile < p.tiles ? first + tile * DV_TILE + lane * 8 : vocab, vocab, next[t]);
            }
        };
        ask(0, 0);
        float most = -INFINITY, sum = 0.0f;
        uint32_t index = UZU_NO_TOKEN, r = 0, group = 0;
        for (uint32_t n = 0; n < all; ++n) {
            alignas(16) T x[DV_GROUP][8];
#pragma unroll
            for (uint32_t t = 0; t < DV_GROUP; ++t)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[t][i] = next[t][i];
            const uint32_t now = r, at = first + group * (DV_GROUP * DV_TILE) + lane * 8;
            const bool last = ++group == groups;
            if (last) {
                group = 0;
                ++r;
            }
            if (n + 1 < all) ask(r, group);
            const float per = now <= count ? per_target : per_draft;
            float m = -INFINITY;
#pragma unroll
            for (uint32_t t = 0; t < DV_GROUP; ++t)
#pragma unroll
                for (int i = 0; i < 8; ++i) m = fmaxf(m, dv_f(x[t][i]));
            if (m > most) {
                if (greedy) {
#pragma unroll
                    for (int t = DV_GROUP - 1; t >= 0; --t)
#pragma unroll
                        for (int i = 7; i >= 0; --i)
                            if (dv_f(x[t][i]) == m) index = at + t * DV_TILE + i;
                }
                sum *= exp2f((most - m) * per);
                most = m;
            }
            const float base = most == -INFINITY ? 0.0f : most;
            float add[2] = {0.0f, 0.0f};
#pragma unroll
            for (uint32_t t = 0; t < DV_GROUP; ++t)
#pragma unroll
                for (int i = 0; i < 8; ++i) add[i & 1] += dv_exp2((dv_f(x[t][i]) - base) * per);
            sum += add[0] + add[1];
            if (!last) continue;
            const float top = warp_max(most);
            sum = warp_sum(most == -INFINITY || most == top ? sum : sum * dv_exp2((most - top) * per));      // (a NaN among nothing else stays one)
            if (greedy) index = __reduce_min_sync(0xffffffffu, most == top ? index : UZU_NO_TOKEN);
            if (lane == 0) {
                s.row_most[now][warp] = top;
                s.row_sum[now][warp] = sum;
                s.row_index[now][warp] = index;
            }
            most = -INFINITY;
            sum = 0.0f;
            index = UZU_NO_TOKEN;
        }
        __syncthreads();
        for (uint32_t q = warp; q < rows; q += WARPS) {
            DvRow m{-INFINITY, UZU_NO_TOKEN, 0.0};
            if (lane < WARPS) m = DvRow{s.row_most[q][lane], s.row_index[q][lane], (double)s.row_sum[q][lane]};
            m = dv_merge(m, q <= count ? per_target : per_draft);
            if (lane == 0) s.part[q] = m;
        }
    }
    cluster.sync();
    for (uint32_t q = warp; q < rows; q += WARPS) {
        DvRow m{-INFINITY, UZU_NO_TOKEN, 0.0};
        if (lane < CLUSTER) m = *cluster.map_shared_rank(&s.part[q], lane);
        m = dv_merge(m, q <= count ? per_target : per_draft);
        if (!(m.most > -INFINITY && m.most < INFINITY) || !(m.sum < INFINITY)) m.most = __uint_as_float(0x7fc00000u);
        if (lane == 0) s.row[q] = m;
    }
    __syncthreads();

    // ---- the first draft that is not kept, and one row in f64: sums of p's and q's weights, and of both where p is above q ----
    // The f32 sums say which drafts are kept, but for those whose u q is as near p as the sums may be off: by 2^-17 of themselves for exponents of 2^6 and their factor in 32 bits, and by what a group's additions
    // and a new maximum's factor round, below 2^-21 a group. (A factor below f32's normal numbers has fewer bits: all drafts with p above a half of u q, then.) For such a draft the f64 sums of its row, which the
    // token behind needs where it is refused, say whether it is kept.
    const double margin = fminf(per_target, per_draft) < 0x1p-120f ? 1.0 : 0x1p-15 + 0x1p-20 * (double)((p.tiles + DV_GROUP - 1) / DV_GROUP);
    uint32_t at_row = 0;
    double parts[5], all[5];              // of CTA `lane`, of the whole vocabulary: p's weights, q's, both again where p is above q, p's where the two are alike within the margin
    auto answer = [&](uint32_t token) {
        if (tid < k1) reinterpret_cast<uint32_t*>(a.tokens)[(size_t)sequence * k1 + tid] = tid < at_row ? drafted[tid] : tid == at_row ? token : UZU_NO_TOKEN;
        if (tid == 0) reinterpret_cast<uint32_t*>(a.accepted)[sequence] = at_row;
    };
#pragma unroll 1
    for (uint32_t from = 0;; from = at_row + 1) {      // (alike in all CTAs; from: drafts before it are kept)
        if (warp == 0) {
            bool kept = false, close = false;
            if (lane >= from && lane < count) {
                const uint32_t token = drafted[lane];
                const DvRow& t = s.row[lane];
                if (token < vocab && t.most == t.most) {
                    if (greedy) kept = token == t.index;
                    else {
                        const double pt = DvHeat(t.most, a.temperature)(dv_f(row_of(lane)[token])) / t.sum;
                        double qt = 1.0;
                        if (with_draft) {
                            const DvRow& d = s.row[count + 1 + lane];
                            qt = d.most == d.most ? DvHeat(d.most, a.draft_temperature)(dv_f(row_of(count + 1 + lane)[token])) / d.sum : INFINITY;
                        }
                        const double uq = (double)uniforms[lane] * qt;
                        kept = uq < pt;
                        close = pt > 0.0 && fabs(uq - pt) <= margin * pt;
                    }
                }
            }
            const uint32_t open = __ballot_sync(0xffffffffu, lane >= from && lane < count && (!kept || close)), closes = __ballot_sync(0xffffffffu, close);
            if (lane == 0) {
                s.accepted = open ? __ffs(open) - 1 : count;
                s.close = open & (0u - open) & closes;
            }
        }
        __syncthreads();
        at_row = s.accepted;
        const bool close = s.close != 0;
        const DvRow target = s.row[at_row];
        const bool residual = at_row < count, against = residual && with_draft;
        const DvRow other = against ? s.row[count + 1 + at_row] : target;
        const bool valid = target.most == target.most && other.most == other.most;
        if (!valid || greedy) {
            if (rank == 0) answer(valid ? target.index : UZU_NO_TOKEN);
            cluster.sync();      // (nobody leaves while its parts are read)
            return;
        }
        const T *row = row_of(at_row), *draft = against ? row_of(count + 1 + at_row) : row;
        const DvHeat heat(target.most, a.temperature), draft_heat(other.most, against ? a.draft_temperature : a.temperature);
        const uint32_t without = residual && !with_draft ? drafted[at_row] : UZU_NO_TOKEN;      // a certain draft has all of q
        bool kept = false;
        double per_w = other.sum, per_v = target.sum;      // p is above q where w / target.sum is above v / other.sum
#pragma unroll 1
        for (bool again = false;; again = true) {
            double sum[5] = {0.0, 0.0, 0.0, 0.0, 0.0};
            for (uint32_t t = 0; t < p.tiles; ++t) {
                const uint32_t at = first + t * DV_TILE + lane * 8;
                if (at >= vocab) break;
                alignas(16) T x[8], y[8];
                dv_load<T, WIDE>(row, at, vocab, x);
                if (against) dv_load<T, WIDE>(draft, at, vocab, y);
#pragma unroll 4
                for (int i = 0; i < 8; ++i) {
                    const double w = at + i == without ? 0.0 : heat(dv_f(x[i]));
                    sum[0] += w;
                    if (!against) continue;
                    const double v = draft_heat(dv_f(y[i])), much = w * per_w, more = fma(-v, per_v, much);
                    sum[1] += v;
                    if (more > 0.0) {
                        sum[2] += w;
                        sum[3] += v;
                    }
                    if (fabs(more) <= margin * much) sum[4] += w;
                }
            }
#pragma unroll
            for (int i = 0; i < 5; ++i) {
                if (i && !against) break;
                sum[i] = dv_warp_sum(sum[i]);
                if (lane == 0) s.sums[i][warp] = sum[i];
            }
            __syncthreads();
            if (warp < 5 && (warp == 0 || against)) {
                const double v = dv_warp_sum(lane < WARPS ? s.sums[warp][lane] : 0.0);
                if (lane == 0) s.cta[warp] = v;
            }
            cluster.sync();
#pragma unroll
            for (int i = 0; i < 5; ++i) {
                parts[i] = all[i] = 0.0;
                if (i && !against) continue;
                if (lane < CLUSTER) parts[i] = *cluster.map_shared_rank(&s.cta[i], lane);
                all[i] = dv_warp_sum(parts[i]);
            }
            cluster.sync();      // (from here on, or until it sums up again, nobody reads another CTA's shared memory)
            if (close && !again) {
                const double w = heat(dv_f(row[drafted[at_row]]));
                const double pt = w / (against ? all[0] : all[0] + w), qt = against ? draft_heat(dv_f(draft[drafted[at_row]])) / all[1] : 1.0;
                kept = (double)uniforms[at_row] * qt < pt;
                if (kept) break;
            }
            if (!against || again) break;
            // How far the f32 sums' quotient was off, times p's share that is as near q as that: what the border between p and q may have moved. More than 2^-32 of the difference, as with a draft
            // model that is nearly the target: once more with the sums of 64 bits.
            const double off = fabs(other.sum * all[0] - target.sum * all[1]) / (target.sum * all[1]);
            if (off <= margin && off * all[4] <= 0x1p-32 * (all[2] - all[3] * (all[0] / all[1]))) break;
            per_w = all[1];
            per_v = all[0];
        }
        if (!kept) break;
    }
    const bool residual = at_row < count, against = residual && with_draft;
    const T *row = row_of(at_row), *draft = against ? row_of(count + 1 + at_row) : row;
    const DvHeat heat(s.row[at_row].most, a.temperature), draft_heat(s.row[against ? count + 1 + at_row : at_row].most, against ? a.draft_temperature : a.temperature);
    const uint32_t without = residual && !with_draft ? drafted[at_row] : UZU_NO_TOKEN;
    const double inv = against ? 1.0 / all[0] : 1.0, draft_inv = against ? 1.0 / all[1] : 0.0;
    double whole = against ? all[2] * inv - all[3] * draft_inv : all[0];
    const bool plain = !against || !(whole > 0x1p-44);      // (nothing is left of the difference but roundings: the target's own weights)
    if (plain) whole = all[0];
    auto left = [&](double w, double w_over, double v_over) { return plain ? w : fmax(w_over * inv - v_over * draft_inv, 0.0); };
    // the first of the lanes' parts, in their order, where the sum from `before` on passes the aim, else the last with any weight; before: the sum up to it
    const double aim = (double)uniforms[a.drafts] * whole;
    bool hit = false;
    auto find = [&](double mine, double& before) {
        double upto = mine;
        for (int o = 1; o < 32; o <<= 1) {
            const double v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= (uint32_t)o) upto += v;
        }
        const uint32_t some = __ballot_sync(0xffffffffu, mine > 0.0), passed = __ballot_sync(0xffffffffu, mine > 0.0 && before + upto > aim);
        const uint32_t at = passed ? __ffs(passed) - 1 : some ? 31 - __clz(some) : 0;
        before += __shfl_sync(0xffffffffu, upto - mine, at);
        hit = passed != 0;
        return at;
    };
    double before = 0.0;
    const uint32_t owner = find(left(parts[0], parts[2], parts[3]), before);
    if (owner != rank) return;
    const uint32_t owner_warp = find(lane < WARPS ? left(s.sums[0][lane], against ? s.sums[2][lane] : 0.0, against ? s.sums[3][lane] : 0.0) : 0.0, before);
    // its run by the whole CTA, a token a thread
    const uint32_t run = (rank * WARPS + owner_warp) * p.tiles * DV_TILE, end = min(run + p.tiles * DV_TILE, vocab);
    uint32_t token = UZU_NO_TOKEN;
    for (uint32_t at0 = run; at0 < end; at0 += WARPS * 32) {
        const uint32_t at = at0 + tid;
        double w = 0.0;
        if (at < end && at != without) {
            w = heat(dv_f(row[at]));
            if (!plain) w = fmax(w * inv - draft_heat(dv_f(draft[at])) * draft_inv, 0.0);
        }
        const double mine = dv_warp_sum(w);
        __syncthreads();      // (the sums before are read)
        if (lane == 0) s.sums[0][warp] = mine;
        __syncthreads();
        const double sums = lane < WARPS ? s.sums[0][lane] : 0.0, chunk = dv_warp_sum(sums);
        if (!(chunk > 0.0)) continue;
        double from = before;
        const uint32_t in_warp = find(sums, from);
        const bool last = hit;
        if (warp == in_warp) {
            const uint32_t l = find(w, from);
            if (lane == 0) s.token = at0 + in_warp * 32 + l;
        }
        __syncthreads();
        token = s.token;
        if (last) break;
        before += chunk;
    }
    answer(token != UZU_NO_TOKEN ? token : without);      // (a certain draft that has all of p as well, but for a rounding)
}

const char* verify_check(const uzu_draft_verify_args* a) {
    if (!a) return "null arguments";
    if (a->data_type > UZU_DT_F16) return "data_type must be bf16, f32 or f16";
    if (a->drafts > DV_DRAFTS) return "at most 16 drafts";
    if (!a->vocab || a->vocab >> 31) return "vocab must be in 1 .. 2^31 - 1";
    if (a->sequences > (1u << 24)) return "at most 2^24 sequences";
    if (a->target_stride < a->vocab) return "a row is shorter than the vocabulary";
    auto number = [](float t) { return t >= DV_COLDEST && t - t == 0.0f; };
    if (a->temperature != 0.0f && !number(a->temperature)) return "temperature must be 0 or at least 2^-60";
    const bool with_draft = a->draft_logits && a->drafts && a->temperature != 0.0f;
    if (with_draft && !number(a->draft_temperature)) return "draft_temperature must be at least 2^-60";
    if (with_draft && a->draft_stride < a->vocab) return "a row is shorter than the vocabulary";
    if (!a->sequences) return nullptr;
    if (!a->target_logits || !a->tokens || !a->accepted || (a->drafts && !a->drafted) || (a->temperature != 0.0f && !a->uniforms)) return "null operand";
    const uint64_t size = a->data_type == UZU_DT_F32 ? 4 : 2;
    if ((a->target_logits | (with_draft ? a->draft_logits : 0)) % size || (a->drafted | a->draft_counts | a->uniforms | a->tokens | a->accepted) % 4) return "an operand is not aligned to its elements";
    const uint64_t n = a->sequences, k1 = a->drafts + 1;
    const uint64_t in[5] = {a->target_logits, with_draft ? a->draft_logits : 0, a->drafted, a->draft_counts, a->uniforms};
    const uint64_t in_bytes[5] = {rows_extent(n * k1, a->target_stride, a->vocab, size), rows_extent(n * a->drafts, a->draft_stride, a->vocab, size), n * a->drafts * 4, n * 4, n * k1 * 4};
    if (bytes_overlap(a->tokens, n * k1 * 4, a->accepted, n * 4)) return "tokens and accepted overlap";
    for (int i = 0; i < 5; ++i)
        if (bytes_overlap(in[i], in_bytes[i], a->tokens, n * k1 * 4) || bytes_overlap(in[i], in_bytes[i], a->accepted, n * 4)) return "a result overlaps an input";
    return nullptr;
}

template <typename F>
void by_type(uint32_t data_type, F f) {
    if (data_type == UZU_DT_F32) f(float());
    else if (data_type == UZU_DT_F16) f(__half());
    else f(__nv_bfloat16());
}

template <typename T, bool WIDE, uint32_t WARPS, uint32_t CLUSTER>
void dv_launch(uzu_command_buffer* cmd, const uzu_draft_verify_args& a) {
    DvParams p{};
    p.a = a;
    p.tiles = (a.vocab + CLUSTER * WARPS * DV_TILE - 1) / (CLUSTER * WARPS * DV_TILE);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.sequences * CLUSTER);
    cfg.blockDim = dim3(WARPS * 32);
    cfg.stream = cmd->ctx->stream;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CLUSTER;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
    if (cmd->dependent()) {
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 2;
    }
    const cudaError_t e = cudaLaunchKernelEx(&cfg, draft_verify_kernel<T, WIDE, WARPS, CLUSTER>, p);
    if (e != cudaSuccess) cmd->record_error(UZU_ERROR_CUDA, std::string("draft_verify_kernel: ") + cudaGetErrorString(e));
    cmd->launches++;
}

}  // namespace
}  // namespace uzu

using namespace uzu;

extern "C" {

uzu_status uzu_draft_verify_validate(const uzu_draft_verify_args* a) {
    const char* e = verify_check(a);
    return e ? fail(UZU_ERROR_INVALID_ARGUMENT, std::string("draft_verify: ") + e) : UZU_OK;
}

void uzu_draft_verify_encode(uzu_command_buffer* cmd, const uzu_draft_verify_args* a) {
    if (!encodable(cmd, "draft_verify")) return;
    if (const char* e = verify_check(a)) {
        cmd->record_error(UZU_ERROR_INVALID_ARGUMENT, std::string("draft_verify: ") + e);
        return;
    }
    if (!a->sequences) return;
    const uint64_t size = a->data_type == UZU_DT_F32 ? 4 : 2;
    const bool wide = ((a->target_logits | a->draft_logits) & 15u) == 0 && a->target_stride * size % 16 == 0 && (!a->draft_logits || a->draft_stride * size % 16 == 0);
    // Few sequences, an SM for each CTA: 16 warps a CTA. Four drafts, vocabulary of 128256, calls back to back: one sequence 22.5 us against 34.7 with 8 warps, eight 31 against 51, 14 32 against 53, 18 52 against 57, 24 60 alike, 32 81
    // against 60: what is left to take lies between the border and 18.
    const bool few = (uint64_t)a->sequences * 16 <= (uint64_t)cmd->ctx->sm_count;
    by_type(a->data_type, [&](auto t) {
        using T = decltype(t);
        if (few) wide ? dv_launch<T, true, 16, 8>(cmd, *a) : dv_launch<T, false, 16, 8>(cmd, *a);
        else wide ? dv_launch<T, true, 8, 8>(cmd, *a) : dv_launch<T, false, 8, 8>(cmd, *a);
    });
}

}  // extern "C"
