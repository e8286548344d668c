// The selective state space scan of prompts on the 5th-generation tensor cores, in chunks of 128 tokens. With L_t the sum of step a up to token t of the chunk (log2):
//   y_i = sum_(j <= i) 2^(L_i - L_j) step_j (c_i . b_j) x_j  +  2^(L_i) S c_i  +  d x_i,      S' = 2^(L_end) S + sum_j 2^(L_end - L_j) step_j x_j b_j^T
// A CTA walks one sequence (or a part of it) for 64 rows of one head:
//   copy     x, b and c of a chunk by TMA, two stages
//   steps    one warp: step sizes, sums of logarithms of each block of 32 tokens from its front and from its end (accurate where their weights are not small)
//   scores   c b^T out of tensor memory, times 2^(L_i - L_j) step_j, back as bf16 operand A. Below the diagonal's 32 x 32 blocks the factor is a product of a row's and
//            a column's, both relative to the row block's start, so that neither overflows (decays are at most 1) and no exponential is taken per element. In the
//            diagonal's blocks the exponent is a difference of sums of at most 32 tokens of at most 150 each: off by a few 2^-12, where a score's rounding is 2^-8.
//   state    x times its weight as two bf16 parts (16 bits: the state keeps what f32 sums need) for the state's sum, the state in registers, f32, its bf16 copy as operand
//   output   the two sums, d x and the gate
//   issue    scores c b^T (128 x 128), their product with x (64), c S (64), b^T [x hi | x lo] (128 columns, both parts at one reading of b)
// Rows past the sequence's end are zeroed in shared memory (what another sequence or nobody left there may be no number).
// An input x that is not finite is taken out of the product with the scores, where its zero weights would make NaN of earlier tokens; rows from it on become NaN.
// Few heads: a sequence is cut into parts; a first pass leaves each part's state from zero (the first's from its start), a second one starts from the sums of those.
// Two warps share a block of 32 rows in each role; the roles' loops are short and stand once, since seven of them share the instruction caches (with unrolled loops and waits of forty
// instructions a chunk took 40 percent longer).
// What bounds it: the roles' way through a chunk and the handshakes between them, 5700 cycles where the products take 1500 and the bytes 2000 (16384 tokens of 128 heads of 64 x
// 128: 380 us against a floor of 137; nine sequences of 8192 tokens in all, 64 heads: 112 against 38, with 64 x 64 110; token by token, as f16 rows go, 1.4 ms). With state_size 64 some 400
// bytes of a thread's registers are spilled.
// Scores and the state that is read out are one bf16 part each: outputs are 0.0017 to 0.0025 off (norms, against 64 bits) where their own rounding is 0.0017. With two parts of both they
// are off by that alone, in 15 to 17 percent more time (129 and 450 us: longer ways of two roles, not the products); with two parts of the state alone 0.0017, in 9 to 12 percent more.
// Every barrier wait is bounded (wait_errors.h).
#include "state_space.cuh"
#include "umma.cuh"

namespace uzu {

namespace {

constexpr uint32_t SU_Q = 128, SU_P = 64, SU_THREADS = 28 * 32, SU_BLOCK = SU_Q * 128;      // tokens of a chunk, rows of the state, bytes of 64 columns of a chunk
// shared memory: x, z (whose place takes the chunk's results) and b of two chunks, c, the parts, the state's operand
constexpr uint32_t SU_Z = 2 * SU_BLOCK, SU_B = SU_Z + 2 * SU_BLOCK, SU_C = SU_B + 4 * SU_BLOCK, SU_WX = SU_C + 2 * SU_BLOCK, SU_S = SU_WX + 2 * SU_BLOCK;
constexpr size_t SU_SMEM = SU_S + SU_BLOCK + 1024;
// registers of a thread: of the scores' warps, the states' and outputs', the others'; together those of the launch (896 threads with 72)
constexpr uint32_t SU_SCORES_REGS = 56, SU_WORK_REGS = 88, SU_OTHER_REGS = 40;
static_assert(256 * SU_SCORES_REGS + 512 * SU_WORK_REGS + 128 * SU_OTHER_REGS <= SU_THREADS * 72, "a split above the launch's registers waits forever");
// tensor memory
constexpr uint32_t SU_G = 0, SU_SCORES = 128, SU_YI = 192, SU_YX = 256, SU_U = 320, SU_COLUMNS = 512;

struct ScanUmmaParams {
    uzu_state_space_scan_args a;
    unsigned int* error;
    float* ends;       // of the parts: [tile][head][64 rows][state_size]
    float* logs;       // [tile][head]
    SequenceTable table;
};

__device__ __forceinline__ void su_sts(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

}  // namespace

// N: state_size, 64 or 128. STATE: only the state at the end of every part but the last
template <int N, bool STATE>
__global__ void __launch_bounds__(SU_THREADS, 1) scan_umma_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_c,
                                                                  const __grid_constant__ CUtensorMap map_out, const __grid_constant__ CUtensorMap map_z, const __grid_constant__ ScanUmmaParams p) {
    extern __shared__ uint8_t su_raw[];
    __shared__ __align__(8) uint64_t bars[43];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile uint32_t gave_up;
    __shared__ __align__(16) float steps[4][SU_Q], front[4][SU_Q], back[4][SU_Q];      // [chunk & 3][token]: step, log2 of the decays of its block of 32 up to it, behind it
    __shared__ __align__(16) float4 blocks[4][4];                                      // [chunk & 3][block]: log2 of all decays of the block, of those before it, behind it, of the chunk
    __shared__ __align__(16) float column[4][96];                                      // of a row block of scores: step_j 2^(L_ref - L_j)
    __shared__ volatile uint32_t odd_rows[4][8];                                       // [chunk & 3][half, row block]: rows with an x that is not finite
    const uzu_state_space_scan_args& a = p.a;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t base = (um_smem(su_raw) + 1023u) & ~1023u, bar0 = um_smem(bars);
    // rings of two (x, z, b), one, and four (steps, odd_rows): a chunk's barrier, the parity of its use
    auto x_full = [&](uint32_t c) { return bar0 + 8u * (c & 1u); };
    auto x_empty = [&](uint32_t c) { return bar0 + 8u * (2 + (c & 1u)); };
    auto b_full = [&](uint32_t c) { return bar0 + 8u * (4 + (c & 1u)); };
    auto b_empty = [&](uint32_t c) { return bar0 + 8u * (6 + (c & 1u)); };
    auto z_full = [&](uint32_t c) { return bar0 + 8u * (8 + (c & 1u)); };
    auto z_empty = [&](uint32_t c) { return bar0 + 8u * (10 + (c & 1u)); };
    auto d_full = [&](uint32_t c) { return bar0 + 8u * (12 + (c & 3u)); };
    auto d_empty = [&](uint32_t c) { return bar0 + 8u * (16 + (c & 3u)); };
    auto o_full = [&](uint32_t c) { return bar0 + 8u * (20 + (c & 3u)); };             // odd_rows; x and the steps have been seen by who arrives
    auto out_full = [&](uint32_t c, uint32_t block) { return bar0 + 8u * (24 + (c & 1u) * 4 + block); };      // both halves of 32 rows of output
    const uint32_t c_full = bar0 + 8u * 32, c_empty = bar0 + 8u * 33, g_full = bar0 + 8u * 34, p_full = bar0 + 8u * 35, w_full = bar0 + 8u * 36, s_full = bar0 + 8u * 37, s_free = bar0 + 8u * 38,
                   y_full = bar0 + 8u * 39, y_empty = bar0 + 8u * 40, u_full = bar0 + 8u * 41, last_products = bar0 + 8u * 42;
    auto two = [](uint32_t c) { return c >> 1 & 1u; };
    auto four = [](uint32_t c) { return c >> 2 & 1u; };
    auto x_at = [&](uint32_t c) { return base + (c & 1u) * SU_BLOCK; };
    auto z_at = [&](uint32_t c) { return base + SU_Z + (c & 1u) * SU_BLOCK; };
    auto b_at = [&](uint32_t c) { return base + SU_B + (c & 1u) * 2 * SU_BLOCK; };

    const uint32_t slices = a.head_dim / SU_P, h = blockIdx.x / slices, slice = blockIdx.x % slices, group = h / (a.heads / a.groups);
    const uint32_t tile = blockIdx.y, q = ss_find(p.table, tile);
    const PackedSequence s_ = p.table.s[q];
    const uint32_t parts = (q + 1 < p.table.count ? p.table.s[q + 1].tile0 : p.table.tiles) - s_.tile0, part = tile - s_.tile0;
    const uint32_t all = (s_.rows + SU_Q - 1) / SU_Q, per = (all + parts - 1) / parts, chunk0 = min(all, part * per), chunks = min(all, chunk0 + per) - chunk0;
    if (STATE && part + 1 == parts) return;
    const uint32_t row0 = s_.first + chunk0 * SU_Q, rows = min(s_.rows - chunk0 * SU_Q, chunks * SU_Q), col0 = h * a.head_dim + slice * SU_P;      // of this CTA

    if (warp == 0) {
        if (lane == 0) {
            for (uint32_t s = 0; s < 2; ++s) {
                um_init(x_full(s), 1); um_init(x_empty(s), STATE ? 1 : 8); um_init(b_full(s), 1); um_init(b_empty(s), 1); um_init(z_full(s), 1); um_init(z_empty(s), 4);
                for (uint32_t k = 0; k < 4; ++k) um_init(out_full(s, k), 2);
            }
            for (uint32_t s = 0; s < 4; ++s) { um_init(d_full(s), 1); um_init(d_empty(s), STATE ? 8 : 24); um_init(o_full(s), 8); }
            um_init(c_full, 1); um_init(c_empty, 1); um_init(g_full, 1); um_init(p_full, 8); um_init(w_full, 8); um_init(s_full, 8); um_init(s_free, 1);
            um_init(y_full, 1); um_init(y_empty, 8); um_init(u_full, 1);
            um_init(last_products, 1);
            gave_up = 0;
            um_fence_init();
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(um_smem(&tmem_slot)), "r"(SU_COLUMNS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    um_fence_before();
    __syncthreads();
    um_fence_after();
    const uint32_t tmem = tmem_slot, w = warp & 3u, half = warp >> 2 & 1u, t = w * 32 + lane, lanes = w << 21;      // of the first 24 warps: block of 32 rows, which of its two warps
    auto chunk_of = [&](uint32_t row, uint32_t i) { return row * 128 + (((half * 4 + i) ^ (row & 7u)) << 4); };      // 16 bytes of a swizzled row, of this warp's half
    pdl_launch_dependents();
    pdl_wait();
    bool ok = true;

    if (warp < 8) {
        um_fewer_registers<SU_SCORES_REGS>();
        // ================================ scores ================================
        if (!STATE) {
            // Blocks of 32 tokens up to the row block's own, the diagonal one: one warp has that and, of four, the one before it; the other one the rest.
            const uint32_t own = w == 3 ? 2 : w, jb0 = half ? own : 0, jb1 = half ? w : own;      // off the diagonal
            if (!half) {
                const uint32_t zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                for (uint32_t k = 2 * (w + 1); k < 8; ++k) um_st8(tmem + lanes + SU_SCORES + k * 8, zero);      // tokens behind the row's: once for all chunks
                um_wait_st();
            }
            for (uint32_t c = 0; c < chunks; ++c) {
                const float *st = steps[c & 3u], *fr = front[c & 3u], *bk = back[c & 3u];
                ok = um_wait(d_full(c), four(c), &gave_up, 0x701u);
                if (!ok) break;
                const float mine = um_ldf(&fr[t]);
                float between = 0.0f;      // the blocks between a column's and the row's
#pragma unroll 1
                for (uint32_t jb = w; jb-- > jb0;) {
                    if (jb < jb1) column[w][jb * 32 + lane] = um_ldf(&st[jb * 32 + lane]) * ss_exp2(um_ldf(&bk[jb * 32 + lane]) + between);
                    between += um_ldf(&blocks[c & 3u][jb].x);
                }
                __syncwarp();
                const float r = ss_exp2(mine);
                const float2 r2 = make_float2(r, r);
                ok = um_wait(g_full, c & 1u, &gave_up, 0x702u);
                if (ok && c) ok = um_wait(y_full, (c - 1) & 1u, &gave_up, 0x703u);      // the scores before are read
                if (!ok) break;
                um_fence_after();
#pragma unroll 1
                for (uint32_t k = 2 * jb0; k < 2 * jb1; ++k) {
                    uint32_t v[16], o[8];
                    um_ld16(tmem + lanes + SU_G + k * 16, v);
#pragma unroll
                    for (uint32_t j = 0; j < 16; j += 4) {
                        const float4 f = *reinterpret_cast<const float4*>(&column[w][k * 16 + j]);
                        const float2 e0 = ss_mul2(ss_mul2(make_float2(f.x, f.y), r2), make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])));
                        const float2 e1 = ss_mul2(ss_mul2(make_float2(f.z, f.w), r2), make_float2(__uint_as_float(v[j + 2]), __uint_as_float(v[j + 3])));
                        o[j / 2] = um_pack(e0.x, e0.y);
                        o[j / 2 + 1] = um_pack(e1.x, e1.y);
                    }
                    um_st8(tmem + lanes + SU_SCORES + k * 8, o);
                }
                if (half) {
#pragma unroll 1
                    for (uint32_t k = 0; k < 2; ++k) {
                        uint32_t v[16], o[8];
                        um_ld16(tmem + lanes + SU_G + w * 32 + k * 16, v);
#pragma unroll
                        for (uint32_t j = 0; j < 16; j += 4) {
                            const float4 f = um_ldf4(&fr[w * 32 + k * 16 + j]), sj = um_ldf4(&st[w * 32 + k * 16 + j]);
                            const float e[4] = {sj.x * ss_exp2(mine - f.x), sj.y * ss_exp2(mine - f.y), sj.z * ss_exp2(mine - f.z), sj.w * ss_exp2(mine - f.w)};
                            float x[4];
#pragma unroll
                            for (uint32_t i = 0; i < 4; ++i) x[i] = k * 16 + j + i <= lane ? e[i] * __uint_as_float(v[j + i]) : 0.0f;
                            o[j / 2] = um_pack(x[0], x[1]);
                            o[j / 2 + 1] = um_pack(x[2], x[3]);
                        }
                        um_st8(tmem + lanes + SU_SCORES + w * 16 + k * 8, o);
                    }
                }
                um_wait_st();
                um_fence_before();
                um_arrive(p_full);
                um_arrive(d_empty(c));
            }
        }
    } else if (warp < 16) {
        um_more_registers<SU_WORK_REGS>();
        // ================================ state: column n = t, rows [32 half, 32 half + 32) ================================
        const uint32_t n = t, heads = a.heads * slices;
        const size_t at = (((size_t)s_.slot() * a.heads + h) * a.head_dim + slice * SU_P + half * 32) * N + n;
        float* slot = reinterpret_cast<float*>(a.state) + at;
        auto end_of = [&](uint32_t k) { return p.ends + (((size_t)(s_.tile0 + k) * heads + blockIdx.x) * SU_P + half * 32) * N + n; };      // (the last part's place: a copy of the start)
        float S[32];
#pragma unroll
        for (uint32_t i = 0; i < 32; ++i) S[i] = 0.0f;
        if (n < N) {
            if (STATE) {
                if (part == 0) {
                    float* copy = end_of(parts - 1);
#pragma unroll
                    for (uint32_t i = 0; i < 32; ++i) {
                        if (!s_.fresh()) S[i] = slot[i * N];
                        copy[i * N] = S[i];
                    }
                }
            } else if (parts == 1) {
                if (!s_.fresh()) {
#pragma unroll
                    for (uint32_t i = 0; i < 32; ++i) S[i] = slot[i * N];
                }
            } else if (part == 0) {
                const float* copy = end_of(parts - 1);
#pragma unroll
                for (uint32_t i = 0; i < 32; ++i) S[i] = copy[i * N];
            } else {
                for (uint32_t k = 0; k < part; ++k) {      // the parts before, in order
                    const float f = k ? ss_exp2(p.logs[(size_t)(s_.tile0 + k) * heads + blockIdx.x]) : 0.0f;
                    const float* end = end_of(k);
#pragma unroll
                    for (uint32_t i = 0; i < 32; ++i) S[i] = k ? fmaf(f, S[i], end[i * N]) : end[i * N];
                }
            }
        }
        auto store = [&]() {      // row n of the operand: its rows of the state
            if (!STATE) {
                if (n < N) {
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i)
                        su_sts(base + SU_S + chunk_of(n, i), um_pack(S[8 * i], S[8 * i + 1]), um_pack(S[8 * i + 2], S[8 * i + 3]), um_pack(S[8 * i + 4], S[8 * i + 5]), um_pack(S[8 * i + 6], S[8 * i + 7]));
                }
                um_fence_proxy();
                um_arrive(s_full);
            }
        };
        float total = 0.0f, end = 0.0f;      // log2 of all decays, of the chunk's whose parts were made last
        // x of chunk c times its weights, as two bf16 parts (the products that read the parts before are done)
        auto parts_of = [&](uint32_t c) {
            const uint32_t x0 = x_at(c), b0 = b_at(c), valid = min(SU_Q, rows - c * SU_Q);
            ok = um_wait(d_full(c), four(c), &gave_up, 0x704u);
            if (ok) ok = um_wait(x_full(c), two(c), &gave_up, 0x705u);
            if (ok && valid < SU_Q) ok = um_wait(b_full(c), two(c), &gave_up, 0x717u);      // (b's rows are there)
            if (!ok) return;
            // (the products that read the parts of chunk c - 1 are done: u_full was waited for)
            const float weight = um_ldf(&steps[c & 3u][t]) * ss_exp2(um_ldf(&back[c & 3u][t]) + um_ldf(&blocks[c & 3u][w].z));
            end = um_ldf(&blocks[c & 3u][w].w);
            const float2 w2 = make_float2(weight, weight);
            total += end;
            bool odd = false;
            float2 check = make_float2(0.0f, 0.0f);      // stays 0 while all are finite
            if (t < valid) {
                uint4 next = um_lds(x0 + chunk_of(t, 0));
#pragma unroll 1
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t v[4] = {next.x, next.y, next.z, next.w}, o = chunk_of(t, i);
                    next = um_lds(x0 + chunk_of(t, i < 3 ? i + 1 : i));
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) {
                        const float2 x = make_float2(um_lo(v[k]), um_hi(v[k])), y = ss_mul2(x, w2);
                        check = ss_fma2(x, make_float2(0.0f, 0.0f), check);
                        hi[k] = um_pack(y.x, y.y);
                        const float2 rest = ss_fma2(make_float2(um_lo(hi[k]), um_hi(hi[k])), make_float2(-1.0f, -1.0f), y);
                        lo[k] = um_pack(rest.x, rest.y);
                    }
                    su_sts(base + SU_WX + o, hi[0], hi[1], hi[2], hi[3]);
                    su_sts(base + SU_WX + SU_BLOCK + o, lo[0], lo[1], lo[2], lo[3]);
                }
                odd = !(check.x + check.y == 0.0f);
                if (odd) {      // not finite: not in the product with the scores
#pragma unroll 1
                    for (uint32_t i = 0; i < 4; ++i) {
                        const uint4 in = um_lds(x0 + chunk_of(t, i));
                        uint32_t v[4] = {in.x, in.y, in.z, in.w};
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k) {
                            if ((v[k] & 0x7f80u) == 0x7f80u) v[k] &= 0xffff0000u;
                            if ((v[k] & 0x7f800000u) == 0x7f800000u) v[k] &= 0xffffu;
                        }
                        su_sts(x0 + chunk_of(t, i), v[0], v[1], v[2], v[3]);
                    }
                }
            } else {            // behind the sequence
#pragma unroll 1
                for (uint32_t i = 0; i < 4; ++i) {
                    su_sts(x0 + chunk_of(t, i), 0, 0, 0, 0);
                    su_sts(b0 + chunk_of(t, i), 0, 0, 0, 0);
                    if (N == 128) su_sts(b0 + SU_BLOCK + chunk_of(t, i), 0, 0, 0, 0);
                    su_sts(base + SU_WX + chunk_of(t, i), 0, 0, 0, 0);
                    su_sts(base + SU_WX + SU_BLOCK + chunk_of(t, i), 0, 0, 0, 0);
                }
            }
            const uint32_t odds = __ballot_sync(0xffffffffu, odd);
            if (lane == 0) odd_rows[c & 3u][warp - 8] = odds;
            um_fence_proxy();
            um_arrive(w_full);
            um_arrive(o_full(c));
            um_arrive(d_empty(c));
        };
        for (uint32_t c = 0;; ++c) {
            if (c) {      // the sum over chunk c - 1
                const float f = ss_exp2(end);
                const float2 f2 = make_float2(f, f);
                ok = um_wait(u_full, (c - 1) & 1u, &gave_up, 0x706u);
                if (!ok) break;
                um_fence_after();
#pragma unroll
                for (uint32_t k = 0; k < 2; ++k) {
                    uint32_t hi[16], lo[16];
                    um_ld16x2(tmem + lanes + SU_U + half * 32 + k * 16, tmem + lanes + SU_U + 64 + half * 32 + k * 16, hi, lo);
#pragma unroll
                    for (uint32_t j = 0; j < 16; j += 2) {
                        const float2 old = ss_fma2(f2, make_float2(S[k * 16 + j], S[k * 16 + j + 1]), make_float2(__uint_as_float(hi[j]), __uint_as_float(hi[j + 1])));
                        const float2 now = ss_add2(old, make_float2(__uint_as_float(lo[j]), __uint_as_float(lo[j + 1])));
                        S[k * 16 + j] = now.x;
                        S[k * 16 + j + 1] = now.y;
                    }
                }
                um_fence_before();
            }
            if (c == chunks) break;
            parts_of(c);      // (first: the next sum waits for them)
            if (!STATE && ok && c) ok = um_wait(s_free, (c - 1) & 1u, &gave_up, 0x707u);      // the operand before is read
            if (!ok) break;
            store();
        }
        if (ok && n < N) {
            float* to = STATE ? end_of(part) : slot;
            if ((STATE || part + 1 == parts) && (chunks || s_.fresh())) {
#pragma unroll
                for (uint32_t i = 0; i < 32; ++i) to[i * N] = S[i];
            }
            if (STATE && n == 0 && half == 0) p.logs[(size_t)tile * heads + blockIdx.x] = total;
        }
    } else if (warp < 24) {
        um_more_registers<SU_WORK_REGS>();
        // ================================ output: row t, columns [32 half, 32 half + 32) ================================
        if (!STATE) {
            const float skip = a.d ? reinterpret_cast<const float*>(a.d)[h] : 0.0f;
            const bool gated = a.z != 0;
            __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out) + (size_t)row0 * a.out_stride + col0 + half * 32;
            const float2 skip2 = make_float2(skip, skip);
            for (uint32_t c = 0; c < chunks; ++c) {
                const uint32_t valid = min(SU_Q, rows - c * SU_Q), r = c * SU_Q + t;
                const bool whole = w * 32 + 32 <= valid;      // all rows of the block are the sequence's
                if (c && half == 0) {      // the results stored a chunk ago are read: z may come there
                    um_store_read();
                    um_arrive(z_empty(c - 1));
                }
                ok = um_wait(o_full(c), four(c), &gave_up, 0x70au);
                if (ok) ok = um_wait(y_full, c & 1u, &gave_up, 0x70bu);
                if (!ok) break;
                um_fence_after();
                const float f = ss_exp2(um_ldf(&front[c & 3u][t]) + um_ldf(&blocks[c & 3u][w].y));
                const float2 f2 = make_float2(f, f);
                float2 ys[16];
                uint32_t seen = 0;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    uint32_t vi[8], vx[8];
                    const uint4 xx = um_lds(x_at(c) + chunk_of(t, i));
                    um_ld8x2(tmem + lanes + SU_YI + half * 32 + i * 8, tmem + lanes + SU_YX + half * 32 + i * 8, vi, vx);
                    const uint32_t xs[4] = {xx.x, xx.y, xx.z, xx.w};
                    seen ^= xx.x;
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) {
                        const float2 y = ss_fma2(f2, make_float2(__uint_as_float(vx[2 * e]), __uint_as_float(vx[2 * e + 1])), make_float2(__uint_as_float(vi[2 * e]), __uint_as_float(vi[2 * e + 1])));
                        ys[4 * i + e] = ss_fma2(skip2, make_float2(um_lo(xs[e]), um_hi(xs[e])), y);
                    }
                }
                um_fence_before();
                um_arrive(y_empty);
                um_arrive_after(x_empty(c), seen, a.reserved0);
                uint32_t odd = 0, bad = 0;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) odd |= odd_rows[c & 3u][half * 4 + i];
                if (odd) {      // columns whose x was not finite at this token or before it in the chunk
                    const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(a.x) + (size_t)(row0 + c * SU_Q) * a.x_stride + col0 + half * 32;
#pragma unroll 1
                    for (uint32_t j = 0; j <= t; ++j)
                        if (odd_rows[c & 3u][half * 4 + (j >> 5)] >> (j & 31u) & 1u) {
#pragma unroll 1
                            for (uint32_t e = 0; e < 32; ++e)
                                if (!(fabsf(__bfloat162float(x[(size_t)j * a.x_stride + e])) < INFINITY)) bad |= 1u << e;
                        }
                }
                um_arrive(d_empty(c));
                ok = um_wait(z_full(c), two(c), &gave_up, 0x718u);
                if (!ok) break;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t chunk = z_at(c) + chunk_of(t, i);
                    float2* y = ys + 4 * i;
                    if (gated) {
                        const uint4 zz = um_lds(chunk);
                        const uint32_t zs[4] = {zz.x, zz.y, zz.z, zz.w};
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e) y[e] = ss_mul2(y[e], ss_silu2(make_float2(um_lo(zs[e]), um_hi(zs[e]))));
                    }
                    if (odd) {
#pragma unroll
                        for (uint32_t e = 0; e < 8; ++e)
                            if (bad >> (8 * i + e) & 1u) (e & 1u ? y[e / 2].y : y[e / 2].x) = __int_as_float(0x7fc00000);
                    }
                    const uint4 o = make_uint4(um_pack(y[0].x, y[0].y), um_pack(y[1].x, y[1].y), um_pack(y[2].x, y[2].y), um_pack(y[3].x, y[3].y));
                    if (whole) su_sts(chunk, o.x, o.y, o.z, o.w);      // over z
                    else if (t < valid) *reinterpret_cast<uint4*>(out + (size_t)r * a.out_stride + i * 8) = o;
                }
                if (whole) um_fence_proxy();
                um_arrive(out_full(c, w));
                if (half == 0) {
                    ok = um_wait(out_full(c, w), two(c), &gave_up, 0x70cu);
                    if (!ok) break;
                    if (whole && lane == 0) um_tma_store(&map_out, z_at(c) + w * 4096, col0, row0 + c * SU_Q + w * 32);
                    __syncwarp();
                }
            }
            um_store_done();
        }
    } else {
        um_fewer_registers<SU_OTHER_REGS>();
        if (warp == 24) {
            // ================================ b and c by TMA ================================
            uint32_t asked = 0, asked_c = 0;
            for (uint32_t c = 0; c < chunks; ++c) {
                const uint32_t row = row0 + c * SU_Q;
                ok = um_wait(b_empty(c), two(c) ^ 1u, &gave_up, 0x70du);
                if (!ok) break;
                if (um_elect()) {
                    um_expect(b_full(c), SU_BLOCK * (N / 64));
                    for (uint32_t i = 0; i < N / 64; ++i) um_tma(b_at(c) + SU_BLOCK * i, &map_b, group * N + i * 64, row, b_full(c));
                }
                __syncwarp();
                ++asked;
                if (STATE) continue;
                ok = um_wait(c_empty, (c & 1u) ^ 1u, &gave_up, 0x719u);
                if (!ok) break;
                if (um_elect()) {
                    um_expect(c_full, SU_BLOCK * (N / 64));
                    for (uint32_t i = 0; i < N / 64; ++i) um_tma(base + SU_C + SU_BLOCK * i, &map_c, group * N + i * 64, row, c_full);
                }
                __syncwarp();
                ++asked_c;
            }
            if (!ok) {      // copies that are on their way end before the CTA does
                for (uint32_t n = 1; n <= 2 && n <= asked; ++n) um_settle(b_full(asked - n), two(asked - n));
                if (asked_c) um_settle(c_full, (asked_c - 1) & 1u);
            }
        } else if (warp == 27) {
            // ================================ x and z by TMA ================================
            uint32_t asked_x = 0, asked_z = 0;
            for (uint32_t c = 0; c < chunks; ++c) {
                ok = um_wait(x_empty(c), two(c) ^ 1u, &gave_up, 0x70eu);
                if (!ok) break;
                if (um_elect()) {
                    um_expect(x_full(c), SU_BLOCK);
                    um_tma(x_at(c), &map_x, col0, row0 + c * SU_Q, x_full(c));
                }
                __syncwarp();
                ++asked_x;
                if (STATE) continue;
                ok = um_wait(z_empty(c), two(c) ^ 1u, &gave_up, 0x71au);
                if (!ok) break;
                if (a.z) {
                    if (um_elect()) {
                        um_expect(z_full(c), SU_BLOCK);
                        um_tma(z_at(c), &map_z, col0, row0 + c * SU_Q, z_full(c));
                    }
                    __syncwarp();
                    ++asked_z;
                } else um_arrive(z_full(c));      // the place is free
            }
            if (!ok)
                for (uint32_t n = 1; n <= 2; ++n) {
                    if (n <= asked_x) um_settle(x_full(asked_x - n), two(asked_x - n));
                    if (n <= asked_z) um_settle(z_full(asked_z - n), two(asked_z - n));
                }
        } else if (warp == 25) {
            // ================================ products ================================
            // shared-memory descriptors: 128-byte swizzle, 1024 bytes between groups of 8 rows, SU_BLOCK between blocks of 64 columns
            constexpr uint64_t desc = (uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29)) << 32, k_major = desc | (1u << 16), wide = desc | ((uint64_t)(SU_BLOCK >> 4) << 16);
            constexpr uint32_t common = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 4) << 24), a_wide = 1u << 15, b_wide = 1u << 16;
            constexpr uint32_t i_scores = common | ((128u >> 3) << 17), i_y = common | b_wide | ((64u >> 3) << 17), i_u = common | a_wide | b_wide | ((128u >> 3) << 17);
            // What needs no scores runs while they are made.
            for (uint32_t k = 0; k <= chunks; ++k) {
                if (k) {
                    const uint32_t c = k - 1, x0 = x_at(c), b0 = b_at(c), c0 = base + SU_C;
                    if (STATE) ok = um_wait(b_full(c), two(c), &gave_up, 0x714u);
                    if (ok) ok = um_wait(w_full, c & 1u, &gave_up, 0x715u);
                    if (!ok) break;
                    um_fence_after();
                    if (um_elect()) {
                        // (64 columns: operand A's second block is whatever lies behind; the sums' lanes 64 .. 127 are not read)
#pragma unroll 1
                        for (uint32_t kk = 0; kk < SU_Q / 16; ++kk) um_mma_ss(tmem + SU_U, wide | ((b0 + kk * 2048u) >> 4), wide | ((base + SU_WX + kk * 2048u) >> 4), i_u, kk != 0);
                        um_commit(u_full);
                        um_commit(b_empty(c));
                        if (STATE) um_commit(x_empty(c));
                    }
                    __syncwarp();
                    if (STATE) continue;
                    ok = um_wait(s_full, c & 1u, &gave_up, 0x712u);
                    if (ok && c) ok = um_wait(y_empty, (c - 1) & 1u, &gave_up, 0x713u);
                    if (!ok) break;
                    um_fence_after();
                    if (um_elect()) {
#pragma unroll 1
                        for (uint32_t kk = 0; kk < N / 16; ++kk)
                            um_mma_ss(tmem + SU_YX, k_major | ((c0 + (kk >> 2) * SU_BLOCK + (kk & 3u) * 32u) >> 4), wide | ((base + SU_S + kk * 2048u) >> 4), i_y, kk != 0);
                        um_commit(s_free);
                        um_commit(c_empty);
                    }
                    __syncwarp();
                    ok = um_wait(p_full, c & 1u, &gave_up, 0x711u);      // (the scores' sums are read, too)
                    if (!ok) break;
                    um_fence_after();
                    if (um_elect()) {
#pragma unroll 1
                        for (uint32_t kk = 0; kk < SU_Q / 16; ++kk) um_mma_ts(tmem + SU_YI, tmem + SU_SCORES + kk * 8u, wide | ((x0 + kk * 2048u) >> 4), i_y, kk != 0);
                        um_commit(y_full);
                    }
                    __syncwarp();
                }
                if (k < chunks && !STATE) {
                    const uint32_t b0 = b_at(k), c0 = base + SU_C;
                    ok = um_wait(b_full(k), two(k), &gave_up, 0x70fu);
                    if (ok) ok = um_wait(c_full, k & 1u, &gave_up, 0x71bu);
                    if (!ok) break;
                    um_fence_after();
                    if (um_elect()) {
#pragma unroll 1
                        for (uint32_t kk = 0; kk < N / 16; ++kk) {
                            const uint32_t o = (kk >> 2) * SU_BLOCK + (kk & 3u) * 32u;
                            um_mma_ss(tmem + SU_G, k_major | ((c0 + o) >> 4), k_major | ((b0 + o) >> 4), i_scores, kk != 0);
                        }
                        um_commit(g_full);
                    }
                    __syncwarp();
                }
            }
            if (!ok) {
                if (um_elect()) um_commit(last_products);
                __syncwarp();
                um_settle(last_products, 0);                                 // none in flight when tensor memory is given back
            }
        } else {
            // ================================ steps: four tokens a lane ================================
            const float rate = reinterpret_cast<const float*>(a.a)[h] * 1.4426950408889634f, bias = a.dt_bias ? reinterpret_cast<const float*>(a.dt_bias)[h] : 0.0f;
            const __nv_bfloat16* dt = reinterpret_cast<const __nv_bfloat16*>(a.dt) + (size_t)row0 * a.dt_stride + h;
            __nv_bfloat16 next[4];
            auto fetch = [&](uint32_t c) {
    #pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t r = c * SU_Q + 4 * lane + i;
                    next[i] = r < rows ? dt[(size_t)r * a.dt_stride] : __float2bfloat16_rn(0.0f);
                }
            };
            if (chunks) fetch(0);
            for (uint32_t c = 0; c < chunks; ++c) {
                float step[4], l[4];
    #pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const bool there = c * SU_Q + 4 * lane + i < rows;
                    step[i] = there ? ss_step(__bfloat162float(next[i]), bias, a.dt_softplus, a.dt_min, a.dt_max) : 0.0f;
                    l[i] = there ? step[i] * rate : 0.0f;
                    l[i] = l[i] < -150.0f ? -150.0f : l[i];      // (nothing is left of a state then; sums stay fine)
                }
                if (c + 1 < chunks) fetch(c + 1);
                const float f0 = l[0], f1 = f0 + l[1], f2 = f1 + l[2], f3 = f2 + l[3], b2 = l[3], b1 = b2 + l[2], b0 = b1 + l[1];
                // Sums of blocks of 32 tokens: a difference of sums from the chunk's start on would lose the digits of quiet tokens behind loud ones.
                const int of = lane & 7u;
                float up = f3, down = b0 + l[0];
    #pragma unroll
                for (int o = 1; o < 8; o <<= 1) {
                    const float u = __shfl_up_sync(0xffffffffu, up, o, 8), d = __shfl_down_sync(0xffffffffu, down, o, 8);
                    if (of >= o) up += u;
                    if (of + o < 8) down += d;
                }
                float before = __shfl_up_sync(0xffffffffu, up, 1, 8), behind = __shfl_down_sync(0xffffffffu, down, 1, 8);
                if (of == 0) before = 0.0f;
                if (of == 7) behind = 0.0f;
                float sum[4];
    #pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = __shfl_sync(0xffffffffu, up, 8 * i + 7);
                const uint32_t block = lane >> 3;
                const float front_of = (block > 0 ? sum[0] : 0.0f) + (block > 1 ? sum[1] : 0.0f) + (block > 2 ? sum[2] : 0.0f);
                const float back_of = (block < 1 ? sum[1] : 0.0f) + (block < 2 ? sum[2] : 0.0f) + (block < 3 ? sum[3] : 0.0f);
                ok = um_wait(d_empty(c), four(c) ^ 1u, &gave_up, 0x716u);
                if (!ok) break;
                *reinterpret_cast<float4*>(&steps[c & 3u][4 * lane]) = make_float4(step[0], step[1], step[2], step[3]);
                *reinterpret_cast<float4*>(&front[c & 3u][4 * lane]) = make_float4(before + f0, before + f1, before + f2, before + f3);
                *reinterpret_cast<float4*>(&back[c & 3u][4 * lane]) = make_float4(behind + b0, behind + b1, behind + b2, behind);
                if (of == 7) blocks[c & 3u][block] = make_float4(up, front_of, back_of, sum[0] + sum[1] + sum[2] + sum[3]);
                um_arrive(d_full(c));
            }
        }
    }

    __syncthreads();
    if (tid == 0) um_report(&gave_up, p.error);
    um_fence_before();
    __syncthreads();
    if (warp == 0) {
        um_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(SU_COLUMNS) : "memory");
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------------------------
// how many parts a sequence of `chunks` chunks is cut into, where `ctas` CTAs would run without cutting: two passes cost 1.6 times the one, so three parts pay and two do not
static uint32_t su_parts(uint32_t chunks, uint64_t ctas, uint32_t sms) {
    const uint64_t room = sms / std::max<uint64_t>(1, ctas);
    if (room < 3 || chunks < 8) return 1;
    const uint32_t want = (uint32_t)std::min<uint64_t>(room, chunks / 2), per = (chunks + want - 1) / want;
    return (chunks + per - 1) / per;
}
static uint64_t su_ctas(const uzu_state_space_scan_args& a) { return (uint64_t)a.sequence_count * a.heads * (a.head_dim / SU_P); }
static uint64_t su_tiles(const uzu_state_space_scan_args& a, uint32_t sms) {
    uint64_t n = 0;
    for (uint32_t i = 0; i < a.sequence_count; ++i) n += su_parts((uint32_t)(((uint64_t)a.sequences[i].rows + SU_Q - 1) / SU_Q), su_ctas(a), sms);
    return n;
}

// shapes, types and alignment (of arguments that scan_check takes)
bool scan_umma_applicable(const uzu_state_space_scan_args& a) {
    return a.data_type == UZU_DT_BF16 && a.head_dim % SU_P == 0 && (a.state_size == 64 || a.state_size == 128) && ((a.x | a.b | a.c | a.z | a.out) & 15u) == 0 && a.x_stride % 8 == 0 && a.b_stride % 8 == 0 &&
           a.c_stride % 8 == 0 && (a.z == 0 || a.z_stride % 8 == 0) && a.out_stride % 8 == 0 && um_encoder() != nullptr;
}

size_t scan_umma_scratch_bytes(const uzu_context* ctx, const uzu_state_space_scan_args& a) {
    const uint64_t tiles = su_tiles(a, ctx->sm_count), heads = (uint64_t)a.heads * (a.head_dim / SU_P);
    return tiles == a.sequence_count ? 0 : tiles * heads * (SU_P * a.state_size + 4) * 4;
}

template <int N, bool STATE>
static void su_launch(uzu_command_buffer* cmd, const CUtensorMap& mx, const CUtensorMap& mb, const CUtensorMap& mc, const CUtensorMap& mo, const CUtensorMap& mz, const ScanUmmaParams& p) {
    static std::atomic<uint64_t> opted{0};
    opt_in_dynamic_smem(cmd, scan_umma_kernel<N, STATE>, (int)SU_SMEM, opted);
    launch(cmd, "scan_umma_kernel", scan_umma_kernel<N, STATE>, dim3(p.a.heads * (p.a.head_dim / SU_P), p.table.tiles), dim3(SU_THREADS), SU_SMEM, mx, mb, mc, mo, mz, p);
}

bool encode_scan_umma(uzu_command_buffer* cmd, const uzu_state_space_scan_args& a) {
    CUtensorMap mx, mb, mc, mo, mz;
    if (!um_map(&mx, a.x, (uint64_t)a.heads * a.head_dim, a.rows, a.x_stride, SU_Q) || !um_map(&mb, a.b, (uint64_t)a.groups * a.state_size, a.rows, a.b_stride, SU_Q) ||
        !um_map(&mc, a.c, (uint64_t)a.groups * a.state_size, a.rows, a.c_stride, SU_Q) || !um_map(&mo, a.out, (uint64_t)a.heads * a.head_dim, a.rows, a.out_stride, 32))
        return false;
    mz = mo;
    if (a.z && !um_map(&mz, a.z, (uint64_t)a.heads * a.head_dim, a.rows, a.z_stride, SU_Q)) return false;
    // the longest first: the last CTAs to start are short ones
    std::vector<uzu_row_sequence> order;
    try {
        order.assign(a.sequences, a.sequences + a.sequence_count);
        std::sort(order.begin(), order.end(), [](const uzu_row_sequence& x, const uzu_row_sequence& y) { return x.rows != y.rows ? x.rows > y.rows : x.slot < y.slot; });
    } catch (const std::bad_alloc&) {
        cmd->record_error(UZU_ERROR_OUT_OF_MEMORY, "state_space_scan: out of host memory");
        return true;
    }
    const uint32_t sms = cmd->ctx->sm_count;
    const size_t need = scan_umma_scratch_bytes(cmd->ctx, a);
    const bool cut = need && a.scratch && a.scratch_bytes >= need;
    const uint64_t heads = (uint64_t)a.heads * (a.head_dim / SU_P);
    ScanUmmaParams p{};
    p.a = a;
    p.error = cmd->ctx->wait_errors.device_word;
    p.a.reserved0 = 0;      // (um_arrive_after)
    for (uint32_t begin = 0; begin < a.sequence_count;) {
        begin = fill_sequences(p.table, order.data(), a.sequence_count, begin, [&](uint32_t rows) { return cut ? su_parts((uint32_t)(((uint64_t)rows + SU_Q - 1) / SU_Q), su_ctas(a), sms) : 1u; });
        // (one launch behind the other: the next may use the same scratch)
        p.ends = reinterpret_cast<float*>(a.scratch);
        p.logs = p.ends + (uint64_t)p.table.tiles * heads * SU_P * a.state_size;
        if (a.state_size == 128) {
            if (p.table.tiles > p.table.count) su_launch<128, true>(cmd, mx, mb, mc, mo, mz, p);
            su_launch<128, false>(cmd, mx, mb, mc, mo, mz, p);
        } else {
            if (p.table.tiles > p.table.count) su_launch<64, true>(cmd, mx, mb, mc, mo, mz, p);
            su_launch<64, false>(cmd, mx, mb, mc, mo, mz, p);
        }
    }
    return true;
}

}  // namespace uzu
