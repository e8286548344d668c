// A whole layer of routed experts for 1 .. 64 tokens in one cooperative launch, one CTA an SM: router, choice, the chosen experts' gated units, the weighted sum.
//
// Bound by the chosen experts' weights, each read once: a warp streams them by TMA into a ring of 32 KB stages (32 rows of 512 columns) and never waits for anything but
// room, over the units and over the phases, so that the wait of all CTAs for the hidden values is spent filling the ring with rows of `down`. Eight warps multiply:
// warp w has columns [64 w, 64 w + 64) of a stage, weights as operand A of m16n8k16, up to eight tokens as operand B from L2; which column of a chunk a thread has does
// not matter to a sum, so a thread reads 16-byte chunks (2 t + i of a row of eight: no two of a phase share banks). The warps' sums are added in order in shared memory.
//   1  logits: an (expert, four tokens) pair a warp, or a CTA where there are fewer pairs than CTAs; rows are copied as bf16 planes (f32 rows: three, 24 bits, and a stage's products summed by themselves: the results are 2.8e-7 off, in one
//      running sum of matrix instructions 1.8e-6, with two planes 4.5e-6; a plain product in f32 1.3e-6).
//   2  every CTA makes the choice for itself from the logits (waiting for one to do it would cost more), lists the chosen experts and their tokens.
//   3  up: a unit is 16 rows of an expert's up and the 16 of its gate; hidden values, times the routing weight, go to scratch as bf16 planes (of bf16 rows two, 16 bits: with one the
//      results were 0.0024 off where their own rounding is 0.0017, and took 2 percent less time).
//   4  down: all stages of all 32-row tiles over all chosen experts, cut evenly over the CTAs; a tile that several have is summed by the last of them, in their order.
// In both products an expert's tokens stand side by side, eight a tile; the rows of the next stage are asked for a stage ahead.
// Two waits for all CTAs, behind phases 1 and 3. They and the ring's barriers are bounded (wait_errors.h).
// One token of 8 experts of 4096 x 14336, two chosen: 125 us, 5.6 TB/s of the 6.45 of a copy (router, choice and the two waits take 12). Of 64 experts of 2048 x 1408, six chosen and
// two shared: 16 bf16 tokens 182 to 191 us of 142, 32 273, 64 336; f32 250, 311, 407. 48 f32 tokens of 128 experts of 2048 x 768: 349 us of 179, bound by the warps' way through a stage
// (three planes, 1400 cycles where the bytes take 1400) and the 39 units' ends of 1500 cycles each.
#include <algorithm>

#include "row_sequences.h"
#include "umma.cuh"

namespace uzu {

namespace {

constexpr uint32_t XL_WARPS = 8, XL_THREADS = 32 * XL_WARPS + 32, XL_STAGE = 32 * 1024, XL_COLS = 512, XL_BOX = 4096;
constexpr uint32_t XL_MAX_TOKENS = 64, XL_MAX_EXPERTS = 528, XL_MAX_LISTED = 656 /* every expert, and 128 of at most 2048 pairs with 16 more */, XL_MAX_TOP = 16, XL_MAX_PAIRS = 64 * 32, XL_CTAS = 148, XL_MAX_WIDTH = 65536;

// bf16 planes of hidden values, where rows have `planes`
constexpr uint32_t xl_hidden_planes(uint32_t planes) { return planes == 1 ? 2 : planes; }

// where what lies in the scratch; the counters and tickets are zero between calls
struct XlScratch {
    uint64_t logits, rows, hidden, partials, total;
    static constexpr uint64_t TICKETS = 256, FIXED = 16384;
};
inline XlScratch xl_scratch(const uzu_expert_layer_args& a) {
    auto up = [](uint64_t v) { return (v + 255) & ~255ull; };
    const uint64_t planes = a.data_type == UZU_DT_F32 ? 3 : 1;
    XlScratch s;
    s.logits = up(XlScratch::FIXED);
    s.rows = up(s.logits + (uint64_t)a.rows * a.experts * 4);
    s.hidden = up(s.rows + planes * a.rows * a.width * 2);
    s.partials = up(s.hidden + xl_hidden_planes(planes) * a.rows * (a.top + a.shared) * a.ff * 2);
    s.total = up(s.partials + (uint64_t)XL_CTAS * 2 * 32 * a.rows * 4);
    return s;
}

static_assert(XlScratch::TICKETS + XL_MAX_WIDTH / 32 * 4 <= XlScratch::FIXED, "a ticket for every tile");

struct XlParams {
    uzu_expert_layer_args a;
    XlScratch s;
    unsigned int* error;
};

// Token tiles of eight that one reading of an expert's weights serves, rows of the call at most, bf16 planes of a value. (An expert with more tokens than that is listed, and
// read, twice: with eight tiles the sums would not leave the registers that the products need. Of three planes two tiles: with four some registers are spilled, and 24, 40 and 64
// rows of four layers took 2 to 7 percent longer, also where most experts have more than 16 tokens: 1024 x 512, 8 of 32 experts, 64 rows 147 us, 145 with two.)
template <int NT, int ROWS, int PLANES>
struct XlShape {
    static constexpr uint32_t TOK = ROWS + 1, RED = XL_WARPS * 32 * TOK * 4;      // tokens of a row of sums, and one place to keep rows off one another's banks
    static constexpr uint32_t STAGES = ROWS <= 16 ? 6 : ROWS == 32 ? 5 : 4;
    static constexpr size_t SMEM = STAGES * XL_STAGE + RED + 1024;
};

__device__ __forceinline__ void xl_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void xl_tma3(uint32_t dst, const CUtensorMap* map, uint32_t x, uint32_t y, uint32_t z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
// A value as PLANES bf16 parts, each what the ones before leave (of what is no number or infinite: the first alone, the product shows it by that). Several parts are cut off, not
// rounded: three keep the 24 bits all the same, and a value above the largest bf16 number is not infinite.
template <int PLANES>
__device__ __forceinline__ void xl_planes(float v, __nv_bfloat16* to, size_t plane) {
#pragma unroll
    for (int pl = 0; pl < PLANES; ++pl) {
        const __nv_bfloat16 part = PLANES > 1 ? __float2bfloat16_rz(v) : __float2bfloat16_rn(v);
        to[pl * plane] = part;
        v = fabsf(v) < INFINITY ? v - __bfloat162float(part) : 0.0f;
    }
}
__device__ __forceinline__ float xl_x(const uzu_expert_layer_args& a, uint32_t t, uint32_t c) {
    return a.data_type == UZU_DT_F32 ? reinterpret_cast<const float*>(a.x)[(size_t)t * a.x_stride + c] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.x)[(size_t)t * a.x_stride + c]);
}

// all CTAs of the launch; false: not within about a second
__device__ __noinline__ bool xl_all(unsigned int* counter, volatile uint32_t* gave_up, uint32_t code) {
    __threadfence();
    atomicAdd(counter, 1u);
    const uint64_t until = um_now() + 1000000000ull;
    for (uint32_t n = 1;; ++n) {
        unsigned int v;
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(counter) : "memory");
        if (v >= gridDim.x) return true;
        if ((n & 63u) == 0) {
            if (*gave_up) return false;
            if (um_now() > until) {
                *gave_up = code;
                return false;
            }
        }
    }
}

// A CTA is done; the last one makes the scratch ready for the next call. Where a wait ran out some CTAs had no share of `down`, and tiles in parts still hold the tickets of the others.
__device__ __forceinline__ void xl_leave(const XlParams& p, uint32_t gave_up) {
    unsigned int* counters = reinterpret_cast<unsigned int*>(p.a.scratch);
    if (gave_up) {
        atomicExch(counters + 3, 1u);
        __threadfence();
    }
    if (atomicAdd(counters + 2, 1u) != gridDim.x - 1) return;      // (behind a fence of the thread's own since its last ticket)
    if (atomicExch(counters + 3, 0u)) {
        __threadfence();
        for (uint32_t i = 0; i < (p.a.width + 31) / 32; ++i) counters[XlScratch::TICKETS / 4 + i] = 0;
    }
    counters[0] = counters[1] = counters[2] = 0;
    __threadfence();
}

// Operand B: eight tokens' columns from `col` on, 16 of a thread, P bf16 planes `plane` elements behind one another (no row: zeros)
template <int P, int N>
__device__ __forceinline__ void xl_ask(const __nv_bfloat16* at, uint32_t col, uint32_t width, size_t plane, uint4 (&to)[N][2]) {
#pragma unroll
    for (int pl = 0; pl < P; ++pl)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t c = col + (2 * (threadIdx.x & 3u) + i) * 8;
            to[pl][i] = at && c < width ? __ldcg(reinterpret_cast<const uint4*>(at + pl * plane + c)) : make_uint4(0, 0, 0, 0);
        }
}

// eight values of a row
__device__ __forceinline__ void xl_x8(const uzu_expert_layer_args& a, uint32_t t, uint32_t c, bool wide, float (&v)[8]) {
    if (!wide) {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) v[j] = xl_x(a, t, c + j);
    } else if (a.data_type == UZU_DT_F32) {
        const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.x) + (size_t)t * a.x_stride + c);
        const float4 x = p[0], y = p[1];
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
    } else {
        const uint4 x = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.x) + (size_t)t * a.x_stride + c);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) { v[2 * j] = um_lo(w[j]); v[2 * j + 1] = um_hi(w[j]); }
    }
}

struct XlLists {
    uint32_t mask[XL_MAX_EXPERTS][2];      // tokens of an expert
    uint16_t expert[XL_MAX_LISTED];        // the chosen ones, ascending; one with many tokens several times
    uint16_t base[XL_MAX_LISTED + 1];      // their pairs, in that order
    uint16_t token[XL_MAX_PAIRS];          // a pair's token, and behind it (64 times) which of the token's choices the expert is (31: shared)
    uint16_t id[XL_MAX_TOKENS][XL_MAX_TOP];
    float weight[XL_MAX_TOKENS][XL_MAX_TOP];
    uint32_t chosen;
};

// the choice for one token by a warp, PER scores a lane
template <int PER>
__device__ void xl_choose(const uzu_expert_layer_args& a, const float* logits, uint32_t t, XlLists& l, bool write) {
    const uint32_t lane = threadIdx.x & 31u;
    float v[PER];
    bool scored = true;      // softmax over all: there is one
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const uint32_t e = lane + 32 * i;
        v[i] = e < a.experts ? __ldcg(logits + (size_t)t * a.experts + e) : -INFINITY;
    }
    if (a.score == UZU_EXPERT_SCORE_SIGMOID) {
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = 1.0f / (1.0f + expf(-v[i]));
    } else if (a.score == UZU_EXPERT_SCORE_ALL) {
        float most = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) most = fmaxf(most, v[i]);      // (passes over what is no number)
        most = warp_max(most);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            v[i] = expf(v[i] - most);      // (an infinite largest one: no number, as all others come to 0)
            if (v[i] == v[i]) sum += v[i];
        }
        sum = warp_sum(sum);
        scored = sum > 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = scored ? v[i] / sum : -INFINITY;      // (the lanes have to agree on an order)
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (v[i] != v[i]) v[i] = -INFINITY;      // behind scores that come to 0 too
    uint32_t taken = 0;
    float mine = 0.0f, first = 0.0f;      // lane k: the score of choice k
    uint32_t mine_id = 0;
    for (uint32_t k = 0; k < a.top; ++k) {
        float best = -INFINITY;
        uint32_t at = 0xffffffffu;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t e = lane + 32 * i;
            if (e < a.experts && !(taken >> i & 1u) && (at == 0xffffffffu || v[i] > best)) { best = v[i]; at = e; }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float ob = __shfl_xor_sync(0xffffffffu, best, o);
            const uint32_t oa = __shfl_xor_sync(0xffffffffu, at, o);
            if (oa != 0xffffffffu && (at == 0xffffffffu || ob > best || (ob == best && oa < at))) { best = ob; at = oa; }
        }
        if ((at & 31u) == lane) taken |= 1u << (at >> 5);
        if (k == 0) first = best;
        if (lane == k) { mine = best; mine_id = at; }
    }
    if (a.score != UZU_EXPERT_SCORE_CHOSEN && mine == -INFINITY) mine = scored ? 0.0f : __int_as_float(0x7fc00000);
    float w = lane < a.top ? mine : 0.0f;
    if (a.score == UZU_EXPERT_SCORE_CHOSEN) {
        w = lane < a.top ? expf(mine - first) : 0.0f;
        w /= warp_sum(w);
    }
    if (a.renormalise) w /= warp_sum(w);
    w *= a.weight_scale;
    if (lane < a.top) {
        l.id[t][lane] = (uint16_t)mine_id;
        l.weight[t][lane] = w;
        atomicOr(&l.mask[mine_id][t >> 5], 1u << (t & 31u));
        if (write && a.ids) reinterpret_cast<uint32_t*>(a.ids)[(size_t)t * a.top + lane] = mine_id;
        if (write && a.weights) reinterpret_cast<float*>(a.weights)[(size_t)t * a.top + lane] = w;
    }
}

}  // namespace

template <int NT, int ROWS, int PLANES>
__global__ void __launch_bounds__(XL_THREADS, 1) expert_layer_kernel(const __grid_constant__ CUtensorMap map_up, const __grid_constant__ CUtensorMap map_down, const __grid_constant__ XlParams p) {
    using S = XlShape<NT, ROWS, PLANES>;
    constexpr uint32_t TOK = S::TOK;
    constexpr int HIDDEN = xl_hidden_planes(PLANES);
    extern __shared__ uint8_t xl_raw[];
    __shared__ __align__(8) uint64_t bars[2 * S::STAGES];
    __shared__ volatile uint32_t gave_up;
    __shared__ uint32_t last;
    __shared__ XlLists l;
    const uzu_expert_layer_args& a = p.a;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), g = lane >> 2, t4 = lane & 3u;
    const uint32_t ring = (um_smem(xl_raw) + 1023u) & ~1023u, bar0 = um_smem(bars);
    float* red = reinterpret_cast<float*>(xl_raw + (ring - um_smem(xl_raw)) + S::STAGES * XL_STAGE);
    uint8_t* scratch = reinterpret_cast<uint8_t*>(a.scratch);
    unsigned int* counters = reinterpret_cast<unsigned int*>(scratch);
    unsigned int* tickets = reinterpret_cast<unsigned int*>(scratch + XlScratch::TICKETS);
    float* logits = reinterpret_cast<float*>(scratch + p.s.logits);
    __nv_bfloat16* rows = reinterpret_cast<__nv_bfloat16*>(scratch + p.s.rows);
    __nv_bfloat16* hidden = reinterpret_cast<__nv_bfloat16*>(scratch + p.s.hidden);
    float* partials = reinterpret_cast<float*>(scratch + p.s.partials);
    const uint32_t T = a.rows, D = a.width, F = a.ff, E = a.experts, all = E + a.shared, ctas = gridDim.x, cta = blockIdx.x;
    const size_t row_plane = (size_t)T * D, hidden_plane = (size_t)T * (a.top + a.shared) * F;
    auto full = [&](uint32_t s) { return bar0 + 8u * s; };
    auto empty = [&](uint32_t s) { return bar0 + 8u * (S::STAGES + s); };

    if (tid == 0) {
        for (uint32_t s = 0; s < S::STAGES; ++s) { um_init(full(s), 1); um_init(empty(s), XL_WARPS); }
        gave_up = 0;
        um_fence_init();
    }
    for (uint32_t e = tid; e < all; e += XL_THREADS) {      // shared experts have every token
        l.mask[e][0] = e < E ? 0u : T >= 32 ? 0xffffffffu : (1u << T) - 1u;
        l.mask[e][1] = e < E || T <= 32 ? 0u : T >= 64 ? 0xffffffffu : (1u << (T - 32)) - 1u;
    }
    pdl_wait();

    // ---- 1: rows as planes, logits ----
    for (uint32_t i = cta * XL_THREADS + tid; i < T * D; i += ctas * XL_THREADS) {
        const float v = xl_x(a, i / D, i % D);
        xl_planes<PLANES>(v, rows + i, row_plane);
    }
    {
        const uint32_t quads = (T + 3) / 4, pairs = E * quads;
        const bool split = pairs <= ctas;      // the CTA's warps share the columns
        const bool wide = (a.x & 15u) == 0 && a.x_stride % 8 == 0;
        const __nv_bfloat16* router = reinterpret_cast<const __nv_bfloat16*>(a.router);
        for (uint32_t i = split ? cta : cta * XL_WARPS + warp; i < pairs && (split || warp < XL_WARPS); i += split ? ctas : ctas * XL_WARPS) {
            const uint32_t e = i / quads, tk = i % quads * 4;
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (warp < XL_WARPS) {
                for (uint32_t c = (split ? warp * 256 : 0) + lane * 8; c < D; c += split ? XL_WARPS * 256 : 256) {
                    const uint4 w = ldg_stream_u4(router + (size_t)e * D + c);
                    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k)
                        if (tk + k < T) {
                            float v[8];
                            xl_x8(a, tk + k, c, wide, v);
#pragma unroll
                            for (uint32_t j = 0; j < 4; ++j) sum[k] = fmaf(um_hi(ws[j]), v[2 * j + 1], fmaf(um_lo(ws[j]), v[2 * j], sum[k]));
                        }
                }
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) sum[k] = warp_sum(sum[k]);
            }
            const float bias = a.router_bias ? reinterpret_cast<const float*>(a.router_bias)[e] : 0.0f;
            if (split) {
                if (warp < XL_WARPS && lane < 4) red[warp * 4 + lane] = lane == 0 ? sum[0] : lane == 1 ? sum[1] : lane == 2 ? sum[2] : sum[3];
                __syncthreads();
                if (tid < 4 && tk + tid < T) {
                    float v = bias;
                    for (uint32_t w = 0; w < XL_WARPS; ++w) v += red[w * 4 + tid];
                    logits[(size_t)(tk + tid) * E + e] = v;
                }
                __syncthreads();
            } else if (lane < 4 && tk + lane < T) logits[(size_t)(tk + lane) * E + e] = bias + (lane == 0 ? sum[0] : lane == 1 ? sum[1] : lane == 2 ? sum[2] : sum[3]);
        }
    }
    __syncthreads();
    if (tid == 0) xl_all(counters, &gave_up, 0x801u);
    __syncthreads();
    bool ok = !gave_up;

    // ---- 2: the choice ----
    if (ok) {
        for (uint32_t t = warp; t < T; t += XL_THREADS / 32) {
            if (E <= 128) xl_choose<4>(a, logits, t, l, cta == 0);
            else xl_choose<16>(a, logits, t, l, cta == 0);
        }
        __syncthreads();
        if (warp == 0) {
            uint32_t count = 0, pairs = 0;
            for (uint32_t e0 = 0; e0 < all; e0 += 32) {
                const uint32_t e = e0 + lane, n = e < all ? __popc(l.mask[e][0]) + __popc(l.mask[e][1]) : 0u, times = (n + 8 * NT - 1) / (8 * NT);
                uint32_t before = n | times << 16;      // pairs and entries of the experts below, this one's included
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t v = __shfl_up_sync(0xffffffffu, before, o);
                    if (lane >= o) before += v;
                }
                if (n) {
                    uint32_t pair = pairs + (before & 0xffffu) - n;
                    for (uint32_t k = 0; k < times; ++k) {
                        l.expert[count + (before >> 16) - times + k] = (uint16_t)e;
                        l.base[count + (before >> 16) - times + k] = (uint16_t)(pair + k * 8 * NT);
                    }
                    for (uint32_t half = 0; half < 2; ++half)
                        for (uint32_t m = l.mask[e][half]; m; m &= m - 1) {
                            const uint32_t t = half * 32 + __ffs(m) - 1;
                            uint32_t j = 31;
                            if (e < E)
                                for (j = 0; j + 1 < a.top && l.id[t][j] != e; ++j) {}
                            l.token[pair++] = (uint16_t)(j * 64 + t);
                        }
                }
                const uint32_t sums = __shfl_sync(0xffffffffu, before, 31);
                count += sums >> 16;
                pairs += sums & 0xffffu;
            }
            if (lane == 0) {
                l.base[count] = (uint16_t)pairs;
                l.chosen = count;
            }
        }
        __syncthreads();
    }
    const uint32_t chosen = ok ? l.chosen : 0, f_tiles = (F + 15) / 16, units = chosen * f_tiles, up_stages = (D + XL_COLS - 1) / XL_COLS;
    const uint32_t d_tiles = (D + 31) / 32, f_stages = (F + XL_COLS - 1) / XL_COLS, tile_stages = chosen * f_stages;
    const uint64_t work = (uint64_t)d_tiles * tile_stages, parts = min((uint64_t)ctas, work), begin = cta < parts ? work * cta / parts : work, end = cta < parts ? work * (cta + 1) / parts : work;
    uint32_t it = 0;      // stages so far

    if (warp == XL_WARPS) {
        // ---- weights by TMA ----
        auto stage = [&](bool up, uint32_t col, uint32_t width, uint32_t row, uint32_t which) {
            const uint32_t s = it % S::STAGES;
            if (ok) ok = um_wait(empty(s), (it / S::STAGES & 1u) ^ 1u, &gave_up, 0x802u);
            if (!ok) return;
            if (um_elect()) {
                const uint32_t boxes = min(XL_WARPS, (width - col + 63) / 64);
                um_expect(full(s), boxes * XL_BOX);
                for (uint32_t b = 0; b < boxes; ++b) {
                    if (up) xl_tma3(ring + s * XL_STAGE + b * XL_BOX, &map_up, col + b * 64, row, which, full(s));      // 16 up rows, 16 gate rows
                    else um_tma(ring + s * XL_STAGE + b * XL_BOX, &map_down, col + b * 64, row, full(s));
                }
            }
            __syncwarp();
            ++it;
        };
        for (uint32_t u = cta; u < units && ok; u += ctas) {
            const uint32_t row = u % f_tiles * 16, which = 2 * l.expert[u / f_tiles];
            for (uint32_t s = 0; s < up_stages && ok; ++s) stage(true, s * XL_COLS, D, row, which);
        }
        if (begin < end) {
            uint32_t tile = (uint32_t)(begin / tile_stages), at = (uint32_t)(begin % tile_stages) / f_stages, s = (uint32_t)(begin % tile_stages) % f_stages;
            for (uint64_t w = begin; w < end && ok; ++w) {
                stage(false, s * XL_COLS, F, l.expert[at] * D + tile * 32, 0);
                if (++s < f_stages) continue;
                s = 0;
                if (++at < chosen) continue;
                at = 0;
                ++tile;
            }
        }
        if (!ok)      // copies on their way end before the CTA does
            for (uint32_t n = 1; n <= S::STAGES && n <= it; ++n) um_settle(full((it - n) % S::STAGES), (it - n) / S::STAGES & 1u);
    } else {
        // ---- products ----
        float acc[2][NT][4];
        auto clear = [&]() {
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[m][n][j] = 0.0f;
        };
        // 16 rows times 32 columns of eight tokens
        auto pair = [&](float (&c)[4], const uint4& lo, const uint4& hi, const uint4& b) {
            xl_mma(c, lo.x, hi.x, lo.y, hi.y, b.x, b.y);
            xl_mma(c, lo.z, hi.z, lo.w, hi.w, b.z, b.w);
        };
        // A stage, for `count` tokens whose rows `src(k)` gives, eight at a time. The first eight of it were asked for a stage ago, into `first`; those of the next stage are asked for
        // (`next`) before this one's products, since they come from L2 no faster than a stage.
        uint4 first[HIDDEN][2];
        auto multiply = [&](auto planes, uint32_t col, uint32_t width, size_t plane, uint32_t count, auto src, auto next) {
            const uint32_t s = it % S::STAGES;
            const bool there = col + warp * 64 < width;
            if (ok) ok = um_wait(full(s), it / S::STAGES & 1u, &gave_up, 0x803u);
            if (!ok) return;
            uint32_t seen = 0;
            constexpr int P = decltype(planes)::value;
            uint4 b[HIDDEN][2];
#pragma unroll
            for (int pl = 0; pl < P; ++pl) { b[pl][0] = first[pl][0]; b[pl][1] = first[pl][1]; }
            next();
            if (there) {
                const uint32_t box = ring + s * XL_STAGE + warp * XL_BOX + g * 128;
                uint4 w[2][4];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        w[i][q] = um_lds(box + q * 1024 + (((2 * t4 + i) ^ g) << 4));
                        seen ^= w[i][q].x;
                    }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (n * 8 >= count) break;
                    uint4 v[HIDDEN][2];
#pragma unroll
                    for (int pl = 0; pl < P; ++pl) { v[pl][0] = b[pl][0]; v[pl][1] = b[pl][1]; }
                    if (n + 1 < NT && (n + 1) * 8 < count) xl_ask<P>((n + 1) * 8 + g < count ? src((n + 1) * 8 + g) : nullptr, col + warp * 64, width, plane, b);
                    if (PLANES == 1) {
#pragma unroll
                        for (int pl = P - 1; pl >= 0; --pl)
#pragma unroll
                            for (int i = 0; i < 2; ++i)
#pragma unroll
                                for (int m = 0; m < 2; ++m) pair(acc[m][n], w[i][2 * m], w[i][2 * m + 1], v[pl][i]);
                    } else {
                        // A matrix instruction cuts its sum off where an addition rounds it: a stage's products, smallest planes first, have sums of their own
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            float stage[4] = {};
#pragma unroll
                            for (int pl = P - 1; pl >= 0; --pl)
#pragma unroll
                                for (int i = 0; i < 2; ++i) pair(stage, w[i][2 * m], w[i][2 * m + 1], v[pl][i]);
#pragma unroll
                            for (int j = 0; j < 4; ++j) acc[m][n][j] += stage[j];
                        }
                    }
                }
            }
            um_arrive_after(empty(s), seen, a.reserved0);
            ++it;
        };
        auto meet = [&]() {
            __syncwarp();
            asm volatile("bar.sync 1, 256;" ::: "memory");
        };
        // the warps' sums side by side: red[warp][row][token]
        auto share = [&](uint32_t count) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (n * 8 >= count) break;
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int j = 0; j < 4; ++j) red[(warp * 32 + m * 16 + j / 2 * 8 + g) * TOK + n * 8 + 2 * t4 + j % 2] = acc[m][n][j];
            }
            meet();
        };
        auto total = [&](uint32_t row, uint32_t tok) {
            float v = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < XL_WARPS; ++w) v += red[(w * 32 + row) * TOK + tok];
            return v;
        };

        // ---- 3: up ----
        auto ask_up = [&](uint32_t at, uint32_t s) {
            if (at >= chosen) return;
            const uint32_t base = l.base[at], count = l.base[at + 1] - base;
            xl_ask<PLANES>(g < count ? rows + (size_t)(l.token[base + g] & 63u) * D : nullptr, s * XL_COLS + warp * 64, D, row_plane, first);
        };
        const uint32_t ahead = ctas / f_tiles, over = ctas % f_tiles;      // a CTA's next unit: experts and tiles on
        uint32_t at = cta / f_tiles, tile = cta % f_tiles;
        ask_up(at, 0);
        for (; at < chosen;) {
            const uint32_t next_tile = tile + over < f_tiles ? tile + over : tile + over - f_tiles, next_at = at + ahead + (tile + over < f_tiles ? 0 : 1);
            const uint32_t f0 = tile * 16, base = l.base[at], count = l.base[at + 1] - base;
            clear();
            for (uint32_t s = 0; s < up_stages && ok; ++s)
                multiply(std::integral_constant<int, PLANES>{}, s * XL_COLS, D, row_plane, count, [&](uint32_t k) { return rows + (size_t)(l.token[base + k] & 63u) * D; },
                         [&]() { s + 1 < up_stages ? ask_up(at, s + 1) : ask_up(next_at, 0); });
            share(count);      // (also where a wait ran out: nobody is left waiting)
            for (uint32_t i = tid; i < count * 16; i += 256) {
                const uint32_t f = i & 15u, k = i >> 4, pair = l.token[base + k], choice = pair >> 6;
                if (f0 + f >= F) continue;
                const float w = choice < XL_MAX_TOP ? l.weight[pair & 63u][choice] : 1.0f;
                const float v = act_f32(a.activation, total(16 + f, k)) * total(f, k) * w;
                xl_planes<HIDDEN>(v, hidden + (size_t)(base + k) * F + f0 + f, hidden_plane);
            }
            meet();
            at = next_at;
            tile = next_tile;
        }
        if (tid == 0) xl_all(counters + 1, &gave_up, 0x804u);
        meet();
        ok = ok && !gave_up;

        // ---- 4: down ----
        auto cta_of = [&](uint64_t w) { return (uint32_t)(((w + 1) * parts - 1) / work); };
        auto store = [&](uint32_t d, uint32_t tok, float v) {
            if (a.data_type == UZU_DT_F32) reinterpret_cast<float*>(a.out)[(size_t)tok * a.out_stride + d] = v;
            else reinterpret_cast<__nv_bfloat16*>(a.out)[(size_t)tok * a.out_stride + d] = __float2bfloat16_rn(v);
        };
        auto ask_down = [&](uint32_t expert, uint32_t s) {
            const uint32_t base = l.base[expert], count = l.base[expert + 1] - base;
            xl_ask<HIDDEN>(g < count ? hidden + (size_t)(base + g) * F : nullptr, s * XL_COLS + warp * 64, F, hidden_plane, first);
        };
        uint32_t expert = 0, stage_of = 0;      // of the stage at hand
        if (ok && begin < end) {
            expert = (uint32_t)(begin % tile_stages) / f_stages;
            stage_of = (uint32_t)(begin % tile_stages) % f_stages;
            ask_down(expert, stage_of);
        }
        for (uint64_t w = begin; w < end;) {
            const uint32_t tile = (uint32_t)(w / tile_stages);
            const uint64_t tile0 = (uint64_t)tile * tile_stages, tile1 = tile0 + tile_stages, stop = min(tile1, end);
            const bool whole = w == tile0 && stop == tile1;
            const uint32_t slot = begin > tile0 ? 0u : 1u;      // of this CTA's two tiles in parts
            // an expert's sums belong to its own tokens: they are added to the warp's sums of all tokens when its stages end
            for (uint32_t i = lane; i < 32 * TOK; i += 32) red[warp * 32 * TOK + i] = 0.0f;
            __syncwarp();
            clear();
            for (; w < stop && ok; ++w) {
                const uint32_t s = stage_of, base = l.base[expert], count = l.base[expert + 1] - base, after = expert + 1 < chosen ? expert + 1 : 0;
                const bool ends = s + 1 == f_stages;
                multiply(std::integral_constant<int, HIDDEN>{}, s * XL_COLS, F, hidden_plane, count, [&](uint32_t k) { return hidden + (size_t)(base + k) * F; },
                         [&]() { if (w + 1 < end) ask_down(ends ? after : expert, ends ? 0 : s + 1); });
                stage_of = ends ? 0 : s + 1;
                if (ends) expert = after;
                if (!ends && w + 1 < stop) continue;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (n * 8 >= count) break;
#pragma unroll
                    for (uint32_t j = 0; j < 2; ++j) {
                        const uint32_t k = n * 8 + 2 * t4 + j;
                        if (k >= count) continue;
                        float* to = &red[(warp * 32 + g) * TOK + (l.token[base + k] & 63u)];
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            to[(m * 16) * TOK] += acc[m][n][j];
                            to[(m * 16 + 8) * TOK] += acc[m][n][2 + j];
                        }
                    }
                }
                clear();
            }
            w = stop;
            meet();
            if (whole) {
                if (ok)
                    for (uint32_t i = tid; i < 32 * T; i += 256)
                        if (tile * 32 + (i & 31u) < D) store(tile * 32 + (i & 31u), i >> 5, total(i & 31u, i >> 5));
            } else {
                float* part = partials + ((size_t)cta * 2 + slot) * 32 * T;
                for (uint32_t i = tid; i < 32 * T; i += 256) part[i] = total(i & 31u, i >> 5);
                __threadfence();
                meet();
                const uint32_t from = cta_of(tile0), to = cta_of(tile1 - 1);
                if (tid == 0) {
                    last = atomicAdd(&tickets[tile], 1u) == to - from;
                    if (last) tickets[tile] = 0;
                    __threadfence();
                }
                meet();
                if (last && ok)
                    for (uint32_t i = tid; i < 32 * T; i += 256) {
                        if (tile * 32 + (i & 31u) >= D) continue;
                        float v = 0.0f;
                        for (uint32_t c = from; c <= to; ++c) v += __ldcg(partials + ((size_t)c * 2 + (work * c / parts > tile0 ? 0u : 1u)) * 32 * T + i);
                        store(tile * 32 + (i & 31u), i >> 5, v);
                    }
            }
            meet();
        }
    }
    __syncthreads();
    if (tid == 0) um_report(&gave_up, p.error);
    if (tid == 0) xl_leave(p, gave_up);
}

namespace {

const char* xl_check(const uzu_expert_layer_args* a, bool run) {
    if (!a) return "null arguments";
    if (a->data_type != UZU_DT_BF16 && a->data_type != UZU_DT_F32) return "data_type must be bf16 or f32";
    if (a->rows > XL_MAX_TOKENS) return "at most 64 rows";
    if (a->width == 0 || a->width > XL_MAX_WIDTH || a->ff == 0 || a->ff > XL_MAX_WIDTH || a->width % 8 || a->ff % 8) return "width and ff must be multiples of 8 up to 65536";
    if (a->experts == 0 || a->experts > 512 || a->shared > 16) return "experts must be in 1 .. 512, shared in 0 .. 16";
    if (a->top == 0 || a->top > XL_MAX_TOP || a->top > a->experts) return "top must be in 1 .. 16 and not above experts";
    if (a->score > UZU_EXPERT_SCORE_SIGMOID || a->activation > UZU_ACT_SOFTPLUS) return "unknown score or activation";
    if ((uint64_t)(a->experts + a->shared) * std::max(2ull * a->ff, (unsigned long long)a->width) >> 31) return "too many rows of weights";
    if (a->x_stride < a->width || a->out_stride < a->width) return "a row is shorter than width";
    if (!run || a->rows == 0) return nullptr;
    if (!a->x || !a->out || !a->router || !a->up_gate || !a->down || !a->scratch) return "null operand";
    const uint64_t size = a->data_type == UZU_DT_F32 ? 4 : 2;
    if ((a->x | a->out) % size || (a->router | a->up_gate | a->down) % 16 || (a->router_bias | a->ids | a->weights) % 4) return "an operand is not aligned";
    if (a->scratch % 256 || a->scratch_bytes < xl_scratch(*a).total) return "the scratch is too small or not 256-byte aligned";
    if (rows_overlap(a->x, a->x_stride, a->width, a->out, a->out_stride, a->width, a->rows, size)) return "x and out overlap";
    return nullptr;
}

template <int NT, int ROWS, int PLANES>
void xl_launch(uzu_command_buffer* cmd, const XlParams& p, const CUtensorMap& up, const CUtensorMap& down) {
    static std::atomic<uint64_t> opted{0};
    opt_in_dynamic_smem(cmd, expert_layer_kernel<NT, ROWS, PLANES>, (int)XlShape<NT, ROWS, PLANES>::SMEM, opted);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(std::min<uint32_t>(cmd->ctx->sm_count, XL_CTAS));
    cfg.blockDim = dim3(XL_THREADS);
    cfg.dynamicSmemBytes = XlShape<NT, ROWS, PLANES>::SMEM;
    cfg.stream = cmd->ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeCooperative;      // all CTAs run together, or the launch fails
    attr[0].val.cooperative = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, expert_layer_kernel<NT, ROWS, PLANES>, up, down, p);
    if (e != cudaSuccess) {
        cmd->record_error(UZU_ERROR_CUDA, std::string("expert_layer_kernel: ") + cudaGetErrorString(e));
        cudaGetLastError();
    }
    cmd->launches++;
}

}  // namespace
}  // namespace uzu

using namespace uzu;

extern "C" {

uzu_status uzu_expert_layer_validate(const uzu_expert_layer_args* a) {
    const char* e = xl_check(a, true);
    return e ? fail(UZU_ERROR_INVALID_ARGUMENT, std::string("expert_layer: ") + e) : UZU_OK;
}

size_t uzu_expert_layer_scratch_bytes(const uzu_expert_layer_args* a) { return xl_check(a, false) ? 0 : xl_scratch(*a).total; }

void uzu_expert_layer_encode(uzu_command_buffer* cmd, const uzu_expert_layer_args* a) {
    if (!encodable(cmd, "expert_layer")) return;
    if (const char* e = xl_check(a, true)) {
        cmd->record_error(UZU_ERROR_INVALID_ARGUMENT, std::string("expert_layer: ") + e);
        return;
    }
    if (a->rows == 0) return;
    XlParams p{};
    p.a = *a;
    p.a.reserved0 = 0;      // (um_arrive_after)
    p.s = xl_scratch(*a);
    p.error = cmd->ctx->wait_errors.device_word;
    CUtensorMap up, down;
    const uint64_t all = a->experts + a->shared;
    // up and gate rows of all experts in turn, in boxes of 16 of each
    const cuuint64_t dims[3] = {a->width, a->ff, 2 * all}, strides[2] = {(cuuint64_t)a->width * 2, (cuuint64_t)a->ff * a->width * 2};
    const cuuint32_t box[3] = {64, 16, 2}, steps[3] = {1, 1, 1};
    if (!um_encoder() || um_encoder()(&up, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, (void*)a->up_gate, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS ||
        !um_map(&down, a->down, a->ff, all * a->width, a->ff, 32)) {
        cmd->record_error(UZU_ERROR_CUDA, "expert_layer: cuTensorMapEncodeTiled failed");
        return;
    }
    // token tiles of eight: the smallest kernel that holds the rows (a larger one's ring is shorter)
    auto go = [&](auto planes) {
        constexpr int PL = decltype(planes)::value, most = PL == 1 ? 4 : 2;
        if (a->rows <= 8) xl_launch<1, 8, PL>(cmd, p, up, down);
        else if (a->rows <= 16) xl_launch<2, 16, PL>(cmd, p, up, down);
        else if (a->rows <= 32) xl_launch<most, 32, PL>(cmd, p, up, down);
        else xl_launch<most, 64, PL>(cmd, p, up, down);
    };
    if (a->data_type == UZU_DT_F32) go(std::integral_constant<int, 3>{});
    else go(std::integral_constant<int, 1>{});
}

}  // extern "C"
