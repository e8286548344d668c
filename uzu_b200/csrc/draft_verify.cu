// Verification of drafted tokens against the target's probabilities, and the token behind the kept ones.
//
// A cluster of CTAs has a sequence; a warp has the same run of the vocabulary in every row. One reading of all rows gives each row's maximum and sum (f32, sums of exponentials by
// lane, in f64 from there on); the CTAs exchange them and all come to the same first refusal. Only the row that a token is drawn from is read again (it lies in L2), in f64, as is the
// draft's: where a sum of weights passes its aim must not depend on f32 roundings. The sum of each warp's run, then the warp where the aim lies looks for the token.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "row_sequences.h"

namespace uzu {

namespace {

constexpr uint32_t DV_THREADS = 512, DV_WARPS = DV_THREADS / 32, DV_CLUSTER = 8, DV_TILE = 256, DV_DRAFTS = 16, DV_ROWS = 2 * DV_DRAFTS + 1;

constexpr float DV_COLDEST = 0x1p-60f;      // (1 / temperature stays a number)

struct DvParams {
    uzu_draft_verify_args a;
    uint32_t tiles;      // of 256 tokens, of a warp
};

template <typename T> __device__ __forceinline__ float dv_f(T v);
template <> __device__ __forceinline__ float dv_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float dv_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float dv_f(float v) { return v; }

// a lane's eight tokens of a tile; -infinity behind the last
template <typename T, bool WIDE>
__device__ __forceinline__ void dv_load(const T* row, uint32_t at, uint32_t vocab, float (&x)[8]) {
    if (WIDE && at + 8 <= vocab) {
        alignas(16) T v[8];
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(v)[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(row + at) + 16 * i);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = dv_f(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = at + i < vocab ? dv_f(row[at + i]) : -INFINITY;
    }
}

struct DvRow {
    float most;          // NaN: no distribution
    uint32_t index;      // of the largest, the lowest of several
    double sum;          // of exp((x - most) / temperature)
};
struct DvShared {
    DvRow part[DV_ROWS], row[DV_ROWS];      // this CTA's run; the whole vocabulary
    float warp_most[DV_WARPS];
    double warp_sum[DV_WARPS], cta_sum;
    double sums[2];
    uint32_t warp_index[DV_WARPS], accepted, token;
};

__device__ __forceinline__ double dv_warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename T, bool WIDE>
__global__ void __cluster_dims__(DV_CLUSTER, 1, 1) __launch_bounds__(DV_THREADS) draft_verify_kernel(const __grid_constant__ DvParams p) {
    namespace cg = cooperative_groups;
    __shared__ DvShared s;
    cg::cluster_group cluster = cg::this_cluster();
    pdl_launch_dependents();
    pdl_wait();
    const uzu_draft_verify_args& a = p.a;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, rank = cluster.block_rank(), sequence = blockIdx.x / DV_CLUSTER, k1 = a.drafts + 1, vocab = a.vocab;
    const bool greedy = a.temperature == 0.0f, with_draft = a.draft_logits && !greedy;
    const uint32_t count = a.draft_counts ? min(reinterpret_cast<const uint32_t*>(a.draft_counts)[sequence], a.drafts) : a.drafts;
    const uint32_t rows = count + 1 + (with_draft ? count : 0u);      // targets, then drafts
    const uint32_t* drafted = reinterpret_cast<const uint32_t*>(a.drafted) + (size_t)sequence * a.drafts;
    const float* uniforms = reinterpret_cast<const float*>(a.uniforms) + (size_t)sequence * k1;
    auto row_of = [&](uint32_t r) {
        return r <= count ? reinterpret_cast<const T*>(a.target_logits) + ((size_t)sequence * k1 + r) * a.target_stride
                          : reinterpret_cast<const T*>(a.draft_logits) + ((size_t)sequence * a.drafts + (r - count - 1)) * a.draft_stride;
    };
    const uint32_t first = (rank * DV_WARPS + warp) * p.tiles * DV_TILE;      // this warp's run of tokens (behind the last one there is none)
    const float per_target = greedy ? 1.0f : 1.4426950408889634f / a.temperature, per_draft = with_draft ? 1.4426950408889634f / a.draft_temperature : 1.0f;

    // ---- maxima and sums of all rows ----
    for (uint32_t r = 0; r < rows; ++r) {
        const T* row = row_of(r);
        const float per = r <= count ? per_target : per_draft;
        float most = -INFINITY, sum = 0.0f;
        uint32_t index = UZU_NO_TOKEN;
        for (uint32_t t = 0; t < p.tiles; ++t) {
            const uint32_t at = first + t * DV_TILE + lane * 8;
            if (at >= vocab) break;
            float x[8], m = -INFINITY;
            dv_load<T, WIDE>(row, at, vocab, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, x[i]);
            if (m > most) {
                if (greedy) {
#pragma unroll
                    for (int i = 7; i >= 0; --i)
                        if (x[i] == m) index = at + i;
                }
                sum *= exp2f((most - m) * per);
                most = m;
            }
            const float base = most == -INFINITY ? 0.0f : most;
            float add = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) add += exp2f((x[i] - base) * per);
            sum += add;
        }
        float top = warp_max(most);
        double whole = dv_warp_sum(most == -INFINITY ? (double)sum : (double)sum * exp2f((most - top) * per));      // (a NaN among nothing else stays one)
        if (greedy) {
            uint32_t best = most == top ? index : UZU_NO_TOKEN;
            best = __reduce_min_sync(0xffffffffu, best);
            index = best;
        }
        if (lane == 0) {
            s.warp_most[warp] = top;
            s.warp_sum[warp] = whole;
            s.warp_index[warp] = index;
        }
        __syncthreads();
        if (tid == 0) {
            DvRow m{-INFINITY, UZU_NO_TOKEN, 0.0};
            for (uint32_t w = 0; w < DV_WARPS; ++w)
                if (s.warp_most[w] > m.most) {
                    m.most = s.warp_most[w];
                    m.index = s.warp_index[w];
                }
            for (uint32_t w = 0; w < DV_WARPS; ++w) m.sum += s.warp_most[w] == -INFINITY ? s.warp_sum[w] : s.warp_sum[w] * exp2((double)(s.warp_most[w] - m.most) * per);
            s.part[r] = m;
        }
        __syncthreads();
    }
    cluster.sync();
    if (tid < rows) {
        const float per = tid <= count ? per_target : per_draft;
        DvRow m{-INFINITY, UZU_NO_TOKEN, 0.0};
        for (uint32_t c = 0; c < DV_CLUSTER; ++c) {
            const DvRow& o = *cluster.map_shared_rank(&s.part[tid], c);
            if (o.most > m.most) {
                m.most = o.most;
                m.index = o.index;
            }
        }
        for (uint32_t c = 0; c < DV_CLUSTER; ++c) {
            const DvRow& o = *cluster.map_shared_rank(&s.part[tid], c);
            m.sum += o.most == -INFINITY ? o.sum : o.sum * exp2((double)(o.most - m.most) * per);
        }
        if (!(m.most > -INFINITY && m.most < INFINITY) || !(m.sum < INFINITY)) m.most = __uint_as_float(0x7fc00000u);
        s.row[tid] = m;
    }
    __syncthreads();

    // ---- the first draft that is not kept ----
    if (warp == 0) {
        bool kept = false;
        if (lane < count) {
            const uint32_t token = drafted[lane];
            const DvRow &t = s.row[lane];
            if (token < vocab && t.most == t.most) {
                if (greedy) kept = token == t.index;
                else {
                    const double pt = exp(((double)dv_f(row_of(lane)[token]) - t.most) / a.temperature) / t.sum;
                    double qt = 1.0;
                    if (with_draft) {
                        const DvRow& d = s.row[count + 1 + lane];
                        qt = d.most == d.most ? exp(((double)dv_f(row_of(count + 1 + lane)[token]) - d.most) / a.draft_temperature) / d.sum : INFINITY;
                    }
                    kept = (double)uniforms[lane] * qt < pt;
                }
            }
        }
        const uint32_t refused = __ballot_sync(0xffffffffu, lane < count && !kept);
        if (lane == 0) s.accepted = refused ? __ffs(refused) - 1 : count;
    }
    __syncthreads();
    const uint32_t at_row = s.accepted;
    const DvRow target = s.row[at_row];
    const bool residual = at_row < count, against = residual && with_draft;
    bool valid = target.most == target.most;
    if (against) valid = valid && s.row[count + 1 + at_row].most == s.row[count + 1 + at_row].most;
    uint32_t token = valid && greedy ? target.index : UZU_NO_TOKEN;

    if (valid && !greedy) {
        // ---- one row in f64 ----
        const T *row = row_of(at_row), *draft = against ? row_of(count + 1 + at_row) : row;
        const double top = target.most, draft_top = against ? s.row[count + 1 + at_row].most : 0.0, per = 1.0 / (double)a.temperature, draft_per = against ? 1.0 / (double)a.draft_temperature : 0.0;
        const uint32_t without = residual && !with_draft ? drafted[at_row] : UZU_NO_TOKEN;      // a certain draft has all of q
        // sums over the cluster, in the order of the vocabulary
        auto over_cluster = [&](double mine) {
            mine = dv_warp_sum(mine);
            __syncthreads();
            if (lane == 0) s.warp_sum[warp] = mine;
            __syncthreads();
            if (tid == 0) {
                double v = 0.0;
                for (uint32_t w = 0; w < DV_WARPS; ++w) v += s.warp_sum[w];
                s.cta_sum = v;
            }
            cluster.sync();
            double all = 0.0;
            for (uint32_t c = 0; c < DV_CLUSTER; ++c) all += *cluster.map_shared_rank(&s.cta_sum, c);
            return all;
        };
        double z = 1.0, draft_z = 1.0;
        if (against) {
            double sum = 0.0, draft_sum = 0.0;
            for (uint32_t t = 0; t < p.tiles; ++t) {
                const uint32_t at = first + t * DV_TILE + lane * 8;
                if (at >= vocab) break;
                float x[8], y[8];
                dv_load<T, WIDE>(row, at, vocab, x);
                dv_load<T, WIDE>(draft, at, vocab, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    sum += exp(((double)x[i] - top) * per);
                    draft_sum += exp(((double)y[i] - draft_top) * draft_per);
                }
            }
            z = over_cluster(sum);
            cluster.sync();
            draft_z = over_cluster(draft_sum);
            cluster.sync();
        }
        bool plain = !against;      // weights are the target's alone
        auto weight = [&](float x, float y, uint32_t i) {
            if (i == without) return 0.0;
            const double w = exp(((double)x - top) * per);
            return plain ? w : fmax(w / z - exp(((double)y - draft_top) * draft_per) / draft_z, 0.0);
        };
        auto run = [&]() {
            double sum = 0.0;
            for (uint32_t t = 0; t < p.tiles; ++t) {
                const uint32_t at = first + t * DV_TILE + lane * 8;
                if (at >= vocab) break;
                float x[8], y[8];
                dv_load<T, WIDE>(row, at, vocab, x);
                if (!plain) dv_load<T, WIDE>(draft, at, vocab, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += weight(x[i], plain ? 0.0f : y[i], at + i);
            }
            return sum;
        };
        double all = over_cluster(run());
        if (!(all > 0.0)) {      // nothing is left of the difference: the target's own weights
            cluster.sync();
            plain = true;
            all = over_cluster(run());
        }
        // the CTA, then the warp, where the sum passes the aim (or the last one with any weight)
        const double aim = (double)uniforms[a.drafts] * all;
        double before = 0.0, mine_before = 0.0;
        uint32_t owner = 0;
        bool passed = false;
        for (uint32_t c = 0; c < DV_CLUSTER && !passed; ++c) {
            const double v = *cluster.map_shared_rank(&s.cta_sum, c);
            if (v > 0.0) {
                owner = c;
                mine_before = before;
                passed = before + v > aim;
            }
            before += v;
        }
        if (owner == rank) {
            uint32_t owner_warp = 0;
            double at_warp = mine_before, sum = mine_before;
            passed = false;
            for (uint32_t w = 0; w < DV_WARPS && !passed; ++w) {
                const double v = s.warp_sum[w];
                if (v > 0.0) {
                    owner_warp = w;
                    at_warp = sum;
                    passed = sum + v > aim;
                }
                sum += v;
            }
            if (warp == owner_warp) {
                uint32_t last = UZU_NO_TOKEN, hit = UZU_NO_TOKEN;      // the last token with any weight, the one that passes
                double sum = at_warp;
                for (uint32_t t = 0; t < p.tiles && hit == UZU_NO_TOKEN; ++t) {
                    const uint32_t at = first + t * DV_TILE + lane * 8;
                    double w[8], mine = 0.0;
                    float x[8], y[8];
                    if (at < vocab) {
                        dv_load<T, WIDE>(row, at, vocab, x);
                        if (!plain) dv_load<T, WIDE>(draft, at, vocab, y);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        w[i] = at < vocab ? weight(x[i], plain ? 0.0f : y[i], at + i) : 0.0;
                        mine += w[i];
                    }
                    double upto = mine;
                    for (int o = 1; o < 32; o <<= 1) {
                        const double v = __shfl_up_sync(0xffffffffu, upto, o);
                        if (lane >= (uint32_t)o) upto += v;
                    }
                    double at_lane = sum + (upto - mine);
                    uint32_t found = UZU_NO_TOKEN, mine_last = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        at_lane += w[i];
                        if (w[i] > 0.0) {
                            mine_last = at + i + 1;
                            if (found == UZU_NO_TOKEN && at_lane > aim) found = at + i;
                        }
                    }
                    hit = __reduce_min_sync(0xffffffffu, found);
                    mine_last = __reduce_max_sync(0xffffffffu, mine_last);
                    if (mine_last) last = mine_last - 1;
                    sum += __shfl_sync(0xffffffffu, upto, 31);
                }
                if (lane == 0) s.token = hit != UZU_NO_TOKEN ? hit : last;
            }
            __syncthreads();
            token = s.token;
            if (tid < k1) reinterpret_cast<uint32_t*>(a.tokens)[(size_t)sequence * k1 + tid] = tid < at_row ? drafted[tid] : tid == at_row ? token : UZU_NO_TOKEN;
            if (tid == 0) reinterpret_cast<uint32_t*>(a.accepted)[sequence] = at_row;
        }
        cluster.sync();      // (nobody leaves while its sums are read)
        return;
    }
    if (rank == 0) {
        if (tid < k1) reinterpret_cast<uint32_t*>(a.tokens)[(size_t)sequence * k1 + tid] = tid < at_row ? drafted[tid] : tid == at_row ? token : UZU_NO_TOKEN;
        if (tid == 0) reinterpret_cast<uint32_t*>(a.accepted)[sequence] = at_row;
    }
    cluster.sync();
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
    DvParams p{};
    p.a = *a;
    p.tiles = (a->vocab + DV_CLUSTER * DV_WARPS * DV_TILE - 1) / (DV_CLUSTER * DV_WARPS * DV_TILE);
    const uint64_t size = a->data_type == UZU_DT_F32 ? 4 : 2;
    const bool wide = ((a->target_logits | a->draft_logits) & 15u) == 0 && a->target_stride * size % 16 == 0 && (!a->draft_logits || a->draft_stride * size % 16 == 0);
    const dim3 grid(a->sequences * DV_CLUSTER);
    auto go = [&](auto kernel) { launch(cmd, "draft_verify_kernel", kernel, grid, dim3(DV_THREADS), 0, p); };
    if (a->data_type == UZU_DT_F32) wide ? go(draft_verify_kernel<float, true>) : go(draft_verify_kernel<float, false>);
    else if (a->data_type == UZU_DT_F16) wide ? go(draft_verify_kernel<__half, true>) : go(draft_verify_kernel<__half, false>);
    else wide ? go(draft_verify_kernel<__nv_bfloat16, true>) : go(draft_verify_kernel<__nv_bfloat16, false>);
}

}  // extern "C"
