// Attention of a prompt's rows over the 8-bit cache on the 5th-generation tensor cores (bf16 rows, heads of up to 128 channels).
//
// A CTA has 256 (row, head) pairs of a key head as two tiles of 128, which take turns on the tensor cores: while one's scores become weights, the other's products run.
//   convert  four warps for the keys and three for the values turn 128 tokens' codes into f16 numbers, which hold them exactly, in 128-byte swizzled rows of 64 channels, two stages each. Scales stay out: those
//            of keys multiply scores, those of values enter the weights and a tile's sum. What a tile of keys has (which of its groups of 16, their scales) goes along in shared memory.
//   issue    S = Q K^T into tensor memory (128 columns for each tile of rows), O += P V with P as operand A in S's place, both for one tile of rows at a time.
//   softmax  a thread a row: its 128 scores in registers, the largest, then weights as one f16 number each: 11 bits, which moves an output by an eighth of a bf16 rounding's half
//            step or so, and more than what the pipe cuts off as it adds to O. O is rescaled only where a row's maximum has grown by 2^12, or the unit changes.
// A row of O is counted in a unit, a power of two near the largest value scale of the keys that it sees, and weights carry their group's scale over the unit. A scale more than 2^2
// below the largest of its tile would bring its weights below f16's range: such groups of keys take a pass of their own, the others masked. The unit moves where the largest has left it
// by more than 2^2; it stays within 2^80 of the largest that the row has seen, so that O neither over- nor underflows.
// Queries are brought to 2^14 .. 2^15 by a power of two for each row, as in the kernel for few rows.
// What bounds it: a tile of 256 rows and 128 keys takes about 5000 cycles; the softmax of a half's rows takes 2700 of them, its scores and products follow one another (1450). The tensor
// pipe is busy for 35 % of the time, schedulers issue in 47 % of the cycles. 6144 rows of three sequences that hold 12000 tokens together, 32 heads of 128 (i8): 655 to 710 us, 712 to 772
// TFLOP/s. On the way there: O in registers, added tile by tile 1180 us; masks and maxima apart for whole tiles 819; codes asked for ahead 745; O in tensor memory 702. With a part left
// out for measuring: without the conversion of codes 649, without weights 551. Slower: weights made before the largest score is known 936, two threads a row 842, codes through registers 927.
// Every barrier wait is bounded (wait_errors.h).
#include <type_traits>

#include "quantized_cache.cuh"
#include "umma.cuh"

namespace uzu {

namespace {

constexpr uint32_t QU_ROWS = 128, QU_KEYS = 128, QU_GROUPS = QU_KEYS / 16, QU_THREADS = 512, QU_STAGES = 2, QU_ITEMS = 4;
constexpr float QU_LIFT = 1.0f, QU_SLACK = 12.0f;      // weights: at most 2^(LIFT + SLACK + 2)
constexpr uint32_t QU_BLOCK = 128 * 128;               // bytes of 128 rows of 64 channels
// registers of a thread: the launch's 128 shared out anew among the four warpgroups
constexpr uint32_t QU_SOFT_REGS = 184, QU_CONVERT_REGS = 72;
static_assert(2 * QU_SOFT_REGS + 2 * QU_CONVERT_REGS == 4 * 128, "a warpgroup that asks for more than there are waits for good");

constexpr float QU_NONE = 1000.0f;      // no unit yet; less than any (-): no largest scale, of groups among which one's is NaN
struct alignas(16) QuGroup {
    float key_scale, value_log, value_inverse, none;             // log2 of the value scale, and 1 / it (of a scale that is 0, whose numbers are zeros in any unit, or NaN: as if it were the largest); NaN or 0
};
struct alignas(16) QuItem {
    uint32_t key0, groups, more;                                 // first key, which groups of 16 count, 0: no tile, the end
    float largest;                                               // of value_log; -QU_NONE where a value scale is NaN
    QuGroup group[QU_GROUPS];
};
struct QuParams {
    uzu_quantized_cache_attention_args a;
    uint32_t capacity, group;
    float* stats;
    unsigned int* error;
};

template <int D>
struct QuShape {
    static constexpr uint32_t BLOCKS = D / 64, Q = BLOCKS * QU_BLOCK, KV = BLOCKS * QU_BLOCK;
    static constexpr uint32_t O_COL = 256;      // tensor memory: scores of two tiles, 128 columns each, then their products
    static constexpr uint32_t RAW = 64 * BLOCKS * 128;      // codes of a tile's keys or values, as the threads that convert them have them
    static constexpr size_t SMEM = 2 * Q + 2 * QU_STAGES * KV + 2 * RAW + 1024;
};

__device__ __forceinline__ float qu_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float2 qu_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
    return d;
}
__device__ __forceinline__ float2 qu_add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return d;
}
__device__ __forceinline__ uint32_t qu_pack(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void qu_sts(uint32_t at, uint4 v) { asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory"); }
// four codes as f16 numbers
template <int CODE>
__device__ __forceinline__ uint2 qu_numbers(uint32_t w) {
    if (CODE == UZU_CACHE_CODE_E4M3) return make_uint2(cache_e4m3x2_f16x2(w), cache_e4m3x2_f16x2(w >> 16));
    const uint32_t off = 0x64806480u;
    w ^= 0x80808080u;
    const uint32_t lo = __byte_perm(w, 0x64646464u, 0x4140), hi = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), *reinterpret_cast<const __half2*>(&off)), b = __hsub2(*reinterpret_cast<const __half2*>(&hi), *reinterpret_cast<const __half2*>(&off));
    return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// 128 columns of the warp's lanes, with their wait
__device__ __forceinline__ void qu_ld128(uint32_t at, uint32_t (&v)[128]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%128];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127}, [%129];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=&r"(v[0]), "=&r"(v[1]), "=&r"(v[2]), "=&r"(v[3]), "=&r"(v[4]), "=&r"(v[5]), "=&r"(v[6]), "=&r"(v[7]), "=&r"(v[8]), "=&r"(v[9]), "=&r"(v[10]), "=&r"(v[11]), "=&r"(v[12]), "=&r"(v[13]), "=&r"(v[14]), "=&r"(v[15]), "=&r"(v[16]), "=&r"(v[17]), "=&r"(v[18]), "=&r"(v[19]), "=&r"(v[20]), "=&r"(v[21]), "=&r"(v[22]), "=&r"(v[23]), "=&r"(v[24]), "=&r"(v[25]), "=&r"(v[26]), "=&r"(v[27]), "=&r"(v[28]), "=&r"(v[29]), "=&r"(v[30]), "=&r"(v[31]), "=&r"(v[32]), "=&r"(v[33]), "=&r"(v[34]), "=&r"(v[35]), "=&r"(v[36]), "=&r"(v[37]), "=&r"(v[38]), "=&r"(v[39]), "=&r"(v[40]), "=&r"(v[41]), "=&r"(v[42]), "=&r"(v[43]), "=&r"(v[44]), "=&r"(v[45]), "=&r"(v[46]), "=&r"(v[47]), "=&r"(v[48]), "=&r"(v[49]), "=&r"(v[50]), "=&r"(v[51]), "=&r"(v[52]), "=&r"(v[53]), "=&r"(v[54]), "=&r"(v[55]), "=&r"(v[56]), "=&r"(v[57]), "=&r"(v[58]), "=&r"(v[59]), "=&r"(v[60]), "=&r"(v[61]), "=&r"(v[62]), "=&r"(v[63]), "=&r"(v[64]), "=&r"(v[65]), "=&r"(v[66]), "=&r"(v[67]), "=&r"(v[68]), "=&r"(v[69]), "=&r"(v[70]), "=&r"(v[71]), "=&r"(v[72]), "=&r"(v[73]), "=&r"(v[74]), "=&r"(v[75]), "=&r"(v[76]), "=&r"(v[77]), "=&r"(v[78]), "=&r"(v[79]), "=&r"(v[80]), "=&r"(v[81]), "=&r"(v[82]), "=&r"(v[83]), "=&r"(v[84]), "=&r"(v[85]), "=&r"(v[86]), "=&r"(v[87]), "=&r"(v[88]), "=&r"(v[89]), "=&r"(v[90]), "=&r"(v[91]), "=&r"(v[92]), "=&r"(v[93]), "=&r"(v[94]), "=&r"(v[95]), "=&r"(v[96]), "=&r"(v[97]), "=&r"(v[98]), "=&r"(v[99]), "=&r"(v[100]), "=&r"(v[101]), "=&r"(v[102]), "=&r"(v[103]), "=&r"(v[104]), "=&r"(v[105]), "=&r"(v[106]), "=&r"(v[107]), "=&r"(v[108]), "=&r"(v[109]), "=&r"(v[110]), "=&r"(v[111]), "=&r"(v[112]), "=&r"(v[113]), "=&r"(v[114]), "=&r"(v[115]), "=&r"(v[116]), "=&r"(v[117]), "=&r"(v[118]), "=&r"(v[119]), "=&r"(v[120]), "=&r"(v[121]), "=&r"(v[122]), "=&r"(v[123]), "=&r"(v[124]), "=&r"(v[125]), "=&r"(v[126]), "=&r"(v[127])
        : "r"(at), "r"(at + 64u)
        : "memory");
}

template <int CODE, int D, bool CAP>
__global__ void __launch_bounds__(QU_THREADS, 1) quantized_cache_umma_kernel(const __grid_constant__ QuParams p) {
    using S = QuShape<D>;
    extern __shared__ uint8_t qu_raw[];
    __shared__ __align__(8) uint64_t bars[20];
    __shared__ QuItem items[QU_ITEMS];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile uint32_t gave_up;
    const uzu_quantized_cache_attention_args& a = p.a;
    const uzu_quantized_cache& c = a.cache;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t base = (um_smem(qu_raw) + 1023u) & ~1023u, q0 = base, k0 = q0 + 2 * S::Q, v0 = k0 + QU_STAGES * S::KV, bar0 = um_smem(bars);
    auto q_full = [&](uint32_t r) { return bar0 + 8u * r; };
    auto s_full = [&](uint32_t r) { return bar0 + 8u * (2 + r); };
    auto p_full = [&](uint32_t r) { return bar0 + 8u * (4 + r); };
    auto k_full = [&](uint32_t s) { return bar0 + 8u * (6 + s); };
    auto k_empty = [&](uint32_t s) { return bar0 + 8u * (8 + s); };
    auto v_full = [&](uint32_t s) { return bar0 + 8u * (10 + s); };
    auto v_empty = [&](uint32_t s) { return bar0 + 8u * (12 + s); };
    auto raw_full = [&](uint32_t v) { return bar0 + 8u * (14 + v); };      // codes of keys (0), of values (1)
    auto raw_empty = [&](uint32_t v) { return bar0 + 8u * (16 + v); };
    const uint32_t last_products = bar0 + 8u * 18;

    // (the sequence is looked up behind pdl_wait; tensor memory first, a dependent's CTA that took it would wait for this one)
    if (warp == 0) {
        if (lane == 0) {
            for (uint32_t r = 0; r < 2; ++r) {
                um_init(q_full(r), 4); um_init(s_full(r), 2); um_init(p_full(r), 4);
                um_init(k_full(r), 4); um_init(k_empty(r), 1); um_init(v_full(r), 3); um_init(v_empty(r), 1);
            }
            um_init(raw_full(0), 1); um_init(raw_full(1), 1); um_init(raw_empty(0), 4); um_init(raw_empty(1), 3);
            um_init(last_products, 1);
            gave_up = 0;
            um_fence_init();
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(um_smem(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    um_fence_before();
    __syncthreads();
    um_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_launch_dependents();
    pdl_wait();

    const uint32_t sequence = blockIdx.z, head = blockIdx.y, G = p.group, dim = c.head_dim, bt = c.block_tokens;
    const CacheSequence q = cache_sequence(a.sequences, kCacheAnyLength, sequence);
    const uint32_t pairs = q.rows * G, tiles = (pairs + 2 * QU_ROWS - 1) / (2 * QU_ROWS);
    const bool mine = pairs > kCacheFewPairs && q.rows > kCacheFewRows && blockIdx.x < tiles;
    const uint32_t pair0 = mine ? (tiles - 1u - blockIdx.x) * 2 * QU_ROWS : 0u;      // the rows with the most keys first
    const uint32_t row_tiles = pair0 + QU_ROWS < pairs ? 2u : 1u;
    const uint32_t token0 = q.length + pair0 / G, token1 = q.length + (min(pair0 + 2 * QU_ROWS, pairs) - 1u) / G;
    const uint32_t end = min(token1 + 1u, p.capacity), begin = a.window && token0 >= a.window ? (token0 - a.window + 1u) & ~(QU_KEYS - 1u) : 0u;
    const uint32_t kept = (min(min(a.keep_first, begin), end) + QU_KEYS - 1u) / QU_KEYS;      // tiles of first keys
    const uint32_t key_tiles = kept + (end > begin ? (end - begin + QU_KEYS - 1u) / QU_KEYS : 0u);
    bool ok = true;

    if (mine) {      // (a warpgroup's four warps at the same instruction)
        if (warp >= 8) um_fewer_registers<QU_CONVERT_REGS>();
        else um_more_registers<QU_SOFT_REGS>();
    }
    if (!mine) {
        // nothing of this sequence is this CTA's
    } else if (warp < 8) {
        // ================================ softmax ================================
        const uint32_t r = warp >> 2, lr = tid & (QU_ROWS - 1u), pair = pair0 + r * QU_ROWS + lr, token = pair / G, h = head * G + pair % G;
        const bool live = pair < pairs;
        if (r < row_tiles) {
            // the row to shared memory as f16 numbers, its largest magnitude brought to 2^14 .. 2^15
            const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(a.query) + (live ? (size_t)(q.row + token) * a.query_row_stride + (size_t)h * a.query_head_stride : 0);
            uint32_t most_bits = 0;
            for (uint32_t i = 0; i < dim / 8 && live; ++i) {
                const uint4 w = *reinterpret_cast<const uint4*>(src + i * 8);
                const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) most_bits = max(most_bits, max(ws[k] & 0x7fffu, ws[k] >> 16 & 0x7fffu));
            }
            most_bits <<= 16;
            const int e = most_bits ? min(kCacheMostPower, 14 + 127 - (int)(most_bits >> 23)) : 0;
            const float up = __uint_as_float((uint32_t)(e + 127) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);
            const uint32_t my_q = q0 + r * S::Q + lr * 128u;
            for (uint32_t i = 0; i < dim / 8; ++i) {
                const uint4 w = live ? *reinterpret_cast<const uint4*>(src + i * 8) : make_uint4(0, 0, 0, 0);
                const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
                uint32_t o[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] = qu_pack(um_lo(ws[k]) * up, um_hi(ws[k]) * up);
                qu_sts(my_q + (i >> 3) * QU_BLOCK + (((i & 7u) ^ (lr & 7u)) << 4), make_uint4(o[0], o[1], o[2], o[3]));
            }
            um_fence_proxy();
            um_arrive(q_full(r));
            // of a score in units of ln 2, or (capped) of a fraction of the cap, doubled and in units of ln 2 as the exponential takes it
            const float factor = most_bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : (CAP ? 2.0f * (a.scale * down) / a.softcap : a.scale * down) * 1.4426950408889634f;
            const float cap = a.softcap * 1.4426950408889634f;
            const uint32_t index = q.length + token, lowest = a.window && index >= a.window ? index - a.window + 1u : 0u, tm = tmem + ((warp & 3u) << 21);
            // bits of the keys [first, first + 32) that the row sees
            auto seen = [&](uint32_t first, uint32_t groups) {
                auto below = [&](uint32_t key) { return key <= first ? 0u : key - first >= 32u ? 0xffffffffu : (1u << (key - first)) - 1u; };
                const uint32_t group_bits = (groups & 1u ? 0xffffu : 0u) | (groups & 2u ? 0xffff0000u : 0u);
                return live ? below(min(index + 1u, end)) & (~below(lowest) | below(a.keep_first)) & group_bits : 0u;
            };
            float top = -INFINITY, sum = 0.0f, unit = QU_NONE, top_unit = -QU_NONE, unit_scale = 1.0f, none = 0.0f;      // (the unit's logarithm, and itself; NaN: a value that the row sees is)
            auto capped = [&](float x) { return cap - 2.0f * cap * __frcp_rn(1.0f + qu_exp2(x)); };      // cap * tanh: within 2^-22 of the cap
            const uint32_t my_s = tm + r * 128u, my_o = tm + S::O_COL + r * 128u;
            for (uint32_t i = 0;; ++i) {
                ok = um_wait(s_full(r), i & 1u, &gave_up, 0x901u);
                if (!ok) break;
                um_fence_after();
                const QuItem& item = items[i % QU_ITEMS];
                if (!item.more) break;      // (the products of the last tile are done)
                const uint32_t key0 = item.key0, groups = item.groups;
                const bool whole = groups == (1u << QU_GROUPS) - 1u && key0 + QU_KEYS <= min(token0 + 1u, end) && (!a.window || token1 - key0 < a.window);
                uint32_t s[QU_KEYS];
                qu_ld128(my_s, s);
                uint32_t bits[QU_KEYS / 32];
#pragma unroll
                for (uint32_t cc = 0; cc < QU_KEYS / 32; ++cc) bits[cc] = 0xffffffffu;
                if (!whole) {
#pragma unroll
                    for (uint32_t cc = 0; cc < QU_KEYS / 32; ++cc) {
                        bits[cc] = seen(key0 + cc * 32u, groups >> (2 * cc));
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (!(bits[cc] >> j & 1u)) s[cc * 32 + j] = 0xff800000u;
                    }
                }
                float most = -INFINITY;
#pragma unroll
                for (int g = 0; g < (int)QU_GROUPS; ++g) {
                    float m[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        m[0] = fmaxf(m[0], fmaxf(__uint_as_float(s[16 * g + j]), __uint_as_float(s[16 * g + j + 1])));
                        m[1] = fmaxf(m[1], fmaxf(__uint_as_float(s[16 * g + j + 2]), __uint_as_float(s[16 * g + j + 3])));
                    }
                    m[0] = fmaxf(m[0], m[1]);
                    // (nothing seen times a scale of 0 is NaN, which is no maximum)
                    m[0] *= factor * item.group[g].key_scale;
                    most = fmaxf(most, CAP ? capped(m[0]) : m[0]);
                }
                if (CAP && !whole && !(bits[0] | bits[1] | bits[2] | bits[3])) most = -INFINITY;      // (capped, nothing seen is -cap)
                float times = 1.0f;      // of O
                if (most > top + QU_SLACK || (top == -INFINITY && most > -INFINITY)) {
                    times = top == -INFINITY ? 0.0f : qu_exp2(top - most);
                    top = most;
                    sum *= times;
                }
                if (const float away = item.largest - unit; !whole || !(away <= 2.0f && away >= -2.0f)) {
                    if (item.largest == -QU_NONE) {      // (weights are of scores alone and stay numbers: the output is not)
#pragma unroll
                        for (int g = 0; g < (int)QU_GROUPS; ++g)
                            if (bits[g / 2] >> (16 * (g & 1)) & 0xffffu) none += item.group[g].none;
                    }
                    float largest = -QU_NONE;      // of the groups that the row sees
#pragma unroll
                    for (int g = 0; g < (int)QU_GROUPS; ++g)
                        if (bits[g / 2] >> (16 * (g & 1)) & 0xffffu) largest = fmaxf(largest, item.group[g].value_log);
                    if (largest > -QU_NONE && (unit == QU_NONE || largest > unit + 2.0f || largest < unit - 2.0f)) {
                        top_unit = fmaxf(top_unit, largest);
                        const float next = fmaxf(largest, top_unit - 80.0f);
                        const int power = unit == QU_NONE ? -127 : (int)(unit - next);
                        times *= power > -127 ? __uint_as_float((uint32_t)(power + 127) << 23) : 0.0f;
                        unit = next;
                        unit_scale = __uint_as_float((uint32_t)((int)next + 127) << 23);
                    }
                }
                if (i && __any_sync(0xffffffffu, times != 1.0f)) {
#pragma unroll 1
                    for (int n = 0; n < D; n += 32) {
                        uint32_t o[2][16];
                        um_ld16x2(my_o + n, my_o + n + 16u, o[0], o[1]);
#pragma unroll
                        for (int k = 0; k < 32; k += 8) {
                            uint32_t x[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) x[j] = __float_as_uint(__uint_as_float(o[k >> 4][(k & 15) + j]) * times);
                            um_st8(my_o + n + k, x);
                        }
                    }
                }
                // the weight of a group's key: 2^(score - top + lift) times the group's value scale over the unit, which their sum takes back
                const float from = (top == -INFINITY ? QU_LIFT : QU_LIFT - top) - (unit == QU_NONE ? 0.0f : unit);
                auto weigh = [&](auto masked) {
#pragma unroll
                    for (int g = 0; g < (int)QU_GROUPS; ++g) {
                        uint32_t w[8];
                        const float4 group = *reinterpret_cast<const float4*>(&item.group[g]);
                        const float by = factor * group.x, add = from + group.y;
                        const float2 by2 = make_float2(by, by), add2 = make_float2(add, add);
                        float2 all[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            float2 x = make_float2(__uint_as_float(s[16 * g + j]), __uint_as_float(s[16 * g + j + 1]));
                            if (CAP) x = make_float2(capped(x.x * by) + add, capped(x.y * by) + add);
                            else x = qu_fma2(x, by2, add2);
                            x = make_float2(qu_exp2(x.x), qu_exp2(x.y));
                            if (decltype(masked)::value) {
                                if (!(bits[g / 2] >> (16 * (g & 1) + j) & 1u)) x.x = 0.0f;
                                if (!(bits[g / 2] >> (16 * (g & 1) + j + 1) & 1u)) x.y = 0.0f;
                            }
                            all[j >> 1 & 1] = qu_add2(all[j >> 1 & 1], x);
                            w[j / 2] = qu_pack(x.x, x.y);
                        }
                        all[0] = qu_add2(all[0], all[1]);
                        sum = fmaf(all[0].x + all[0].y, group.z * unit_scale, sum);
                        um_st8(my_s + g * 8u, w);
                    }
                };
                if (whole) weigh(std::false_type());
                else weigh(std::true_type());
                um_wait_st();
                um_fence_before();
                um_arrive(p_full(r));
            }
            if (ok) {
                float scale = unit_scale, f = 1.0f, high = top;
                if (a.sinks && sum != 0.0f) {
                    const float sink = reinterpret_cast<const float*>(a.sinks)[h] * 1.4426950408889634f;
                    high = fmaxf(top, sink);
                    f = qu_exp2(top - high);
                    sum = sum * f + qu_exp2(sink - high + QU_LIFT);
                    scale *= f;
                }
                const float inv = none != 0.0f ? none : sum != 0.0f ? scale / sum : 0.0f;      // (both sums are lifted)
                if (p.stats && live) *reinterpret_cast<float2*>(p.stats + ((size_t)(q.row + token) * a.heads + h) * 2) = make_float2(high, sum != 0.0f ? (float)(1 << (int)QU_LIFT) / sum : 0.0f);
                __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out) + (live ? (size_t)(q.row + token) * a.out_stride + (size_t)h * dim : 0);
                for (uint32_t n = 0; n < dim; n += 16) {      // (by whole warps; a row without weights has no products to read, or none of its own)
                    uint32_t o[2][8];
                    um_ld8x2(my_o + n, my_o + n + 8u, o[0], o[1]);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        uint32_t v[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[j] = sum != 0.0f ? um_pack(__uint_as_float(o[e][2 * j]) * inv, __uint_as_float(o[e][2 * j + 1]) * inv) : 0u;
                        if (live) *reinterpret_cast<uint4*>(out + n + 8 * e) = make_uint4(v[0], v[1], v[2], v[3]);
                    }
                }
            }
        }
    } else if (warp != 12) {
        // ================================ codes to numbers ================================
        const bool values = warp > 12;
        const uint32_t w = values ? warp - 13u : warp - 8u, warps = values ? 3u : 4u;
        const uint32_t* table = reinterpret_cast<const uint32_t*>(a.sequences.tables) + (size_t)sequence * a.sequences.table_stride;
        auto empty = [&](uint32_t s) { return values ? v_empty(s) : k_empty(s); };
        auto full = [&](uint32_t s) { return values ? v_full(s) : k_full(s); };
        // The items: tiles of keys, or parts of one whose value scales are within 2^2 of one another. A lane of the first eight has a group's block and scales; those of the next
        // tile are asked for while this one is converted.
        uint32_t tile = 0, todo = 0, key0 = 0, block = 0, take = 0, zeros = 0, next_block = c.blocks;
        float ks = 0.0f, vs = 0.0f, next_ks = 0.0f, next_vs = 0.0f;
        auto first_key = [&](uint32_t t) { return t < kept ? t * QU_KEYS : begin + (t - kept) * QU_KEYS; };
        auto ask_block = [&]() {      // of tile `tile`
            next_block = c.blocks;
            const uint32_t key = first_key(tile) + lane * 16;
            if (tile < key_tiles && lane < QU_GROUPS && key < end) next_block = table[key / bt];
        };
        auto ask_scales = [&]() {
            next_ks = next_vs = 0.0f;
            if (next_block < c.blocks) {
                const size_t pair = (size_t)next_block * c.kv_heads + head;
                next_ks = reinterpret_cast<const float*>(c.key_scales)[pair];
                next_vs = reinterpret_cast<const float*>(c.value_scales)[pair];
            }
        };
        bool asked = false;      // the next tile's scales
        auto next_item = [&]() {
            while (!todo) {
                if (tile == key_tiles) return false;
                if (!asked) ask_scales();
                key0 = first_key(tile);
                block = next_block;
                ks = next_ks;
                vs = next_vs;
                todo = __ballot_sync(0xffffffffu, block < c.blocks);
                ++tile;
                ask_block();
                asked = false;
            }
            const bool number = (todo >> lane & 1u) && vs > 0.0f;      // (a scale of 0 or NaN goes with any others)
            const float largest = __uint_as_float(__reduce_max_sync(0xffffffffu, number ? __float_as_uint(vs) : 0u));
            take = __ballot_sync(0xffffffffu, (todo >> lane & 1u) && (!number || vs * 4.0f >= largest));
            zeros = __ballot_sync(0xffffffffu, vs == 0.0f);
            todo &= ~take;
            return true;
        };
        // A warp has units of 8 rows of 64 channels, a thread 16 codes of each. A block's codes are one run of memory, which one lane copies; what is no key of the item becomes zeros
        constexpr uint32_t UNITS = 16 * S::BLOCKS, MINE = (UNITS + 2) / 3;
        const uint32_t raw = v0 + QU_STAGES * S::KV + (values ? S::RAW : 0u), my_row = lane >> 2, my_channel = (lane & 3u) * 16;
        const uint8_t* const codes = reinterpret_cast<const uint8_t*>(values ? c.value_codes : c.key_codes);
        auto ask = [&]() {      // by the role's first warp
            const bool first = lane < QU_GROUPS && (take >> lane & 1u) && lane * 16 % bt == 0;
            const uint32_t copies = __popc(__ballot_sync(0xffffffffu, first));
            if (lane == 0) um_expect(raw_full(values), copies * bt * dim);
            __syncwarp();
            if (first)
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(raw + lane * 16 * dim),
                             "l"(codes + ((size_t)block * c.kv_heads + head) * bt * dim), "r"(bt * dim), "r"(raw_full(values))
                             : "memory");
            __syncwarp();
        };
        const uint32_t stage0 = values ? v0 : k0;
        uint32_t n = 0;      // items
        ask_block();
        bool more = next_item();
        if (more && w == 0) ask();
        while (more && ok) {
            if (warp == 8) {
                QuItem& item = items[n % QU_ITEMS];
                const uint32_t among = vs > 0.0f && (take >> lane & 1u) ? __float_as_uint(vs) : 0u, largest = __reduce_max_sync(0xffffffffu, among);
                const bool nan = __any_sync(0xffffffffu, (take >> lane & 1u) && vs != vs);
                // (a scale of 0 or NaN goes as the largest; so do groups that do not count)
                const uint32_t as = among ? among : largest ? largest : 0x3f800000u;
                const float log = (float)((int)(as >> 23) - 127);
                if (lane < QU_GROUPS) item.group[lane] = QuGroup{ks, log, cache_inverse(__uint_as_float(as)), vs != vs && (take >> lane & 1u) ? vs : 0.0f};
                if (lane == 0) {
                    item.key0 = key0;
                    item.groups = take;
                    item.more = 1;
                    item.largest = nan ? -QU_NONE : (float)((int)((largest ? largest : 0x3f800000u) >> 23) - 127);
                }
            }
            const uint32_t s = n % QU_STAGES, to = stage0 + s * S::KV;
            if (!asked) ask_scales();
            asked = true;
            ok = um_wait(empty(s), (n / QU_STAGES & 1u) ^ 1u, &gave_up, values ? 0x903u : 0x902u);
            if (ok) ok = um_wait(raw_full(values), n & 1u, &gave_up, values ? 0x90bu : 0x90au);
            if (!ok) break;
            const uint32_t groups = values ? take & ~zeros : take, keys = min(end - key0, QU_KEYS);
#pragma unroll
            for (uint32_t m = 0; m < MINE; ++m) {
                const uint32_t u = w + m * warps, b = u % S::BLOCKS, at = to + b * QU_BLOCK + (u / S::BLOCKS * 8 + my_row) * 128u;
                if (u >= UNITS) break;
                const uint32_t row = u / S::BLOCKS * 8 + my_row, channel = b * 64 + my_channel;
                const uint4 v = (groups >> (row / 16) & 1u) && row < keys && channel < dim ? um_lds(raw + row * dim + channel) : make_uint4(0, 0, 0, 0);
                const uint2 y[4] = {qu_numbers<CODE>(v.x), qu_numbers<CODE>(v.y), qu_numbers<CODE>(v.z), qu_numbers<CODE>(v.w)};
                qu_sts(at + (((2 * (lane & 3u)) ^ my_row) << 4), make_uint4(y[0].x, y[0].y, y[1].x, y[1].y));
                qu_sts(at + (((2 * (lane & 3u) + 1u) ^ my_row) << 4), make_uint4(y[2].x, y[2].y, y[3].x, y[3].y));
            }
            um_fence_proxy();
            um_arrive(full(s));
            um_arrive(raw_empty(values));
            more = next_item();
            if (more && w == 0) {
                ok = um_wait(raw_empty(values), n & 1u, &gave_up, values ? 0x90du : 0x90cu);
                if (ok) ask();
            }
            ++n;
        }
        if (!ok && w == 0) um_settle(raw_full(values), n & 1u);      // a copy that may be on its way ends before the CTA does
        if (ok && !values) {
            ok = um_wait(k_empty(n % QU_STAGES), (n / QU_STAGES & 1u) ^ 1u, &gave_up, 0x904u);
            if (ok) {
                if (warp == 8 && lane == 0) items[n % QU_ITEMS].more = 0;
                um_arrive(k_full(n % QU_STAGES));
            }
        }
    } else {
        // ================================ products ================================
        {
            // shared-memory descriptors: 128-byte swizzle, 1024 bytes between groups of 8 rows; values N-major, QU_BLOCK between blocks of 64 channels; f16 operands, f32 sums
            constexpr uint64_t desc_hi = (uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29)) << 32;
            const uint32_t idesc_s = (1u << 4) | ((QU_KEYS >> 3) << 17) | ((QU_ROWS >> 4) << 24), idesc_o = (1u << 4) | (1u << 16) | ((dim >> 3) << 17) | ((QU_ROWS >> 4) << 24);
            const uint32_t steps = dim / 16;
            auto scores = [&](uint32_t i, uint32_t r, bool more) {
                if (um_elect()) {
                    if (more)
                        for (uint32_t kk = 0; kk < steps; ++kk) {
                            const uint32_t off = (kk >> 2) * QU_BLOCK + (kk & 3u) * 32u, qa = q0 + r * S::Q + off, ka = k0 + i % QU_STAGES * S::KV + off;
                            um_mma_ss(tmem + r * 128u, desc_hi | (1u << 16) | (qa >> 4), desc_hi | (1u << 16) | (ka >> 4), idesc_s, kk != 0);
                        }
                    um_commit(s_full(r));
                    if (more && r + 1 == row_tiles) um_commit(k_empty(i % QU_STAGES));
                }
                um_arrive(s_full(r));      // (what the converting warps say of the tile is handed on with it)
            };
            for (uint32_t r = 0; r < row_tiles && ok; ++r) ok = um_wait(q_full(r), 0, &gave_up, 0x905u);
            if (ok) ok = um_wait(k_full(0), 0, &gave_up, 0x906u);
            um_fence_after();
            bool more = false;
            if (ok) {
                more = items[0].more != 0;
                for (uint32_t r = 0; r < row_tiles; ++r) scores(0, r, more);
            }
            for (uint32_t i = 0; more && ok; ++i) {
                const uint32_t next = i + 1;
                bool next_more = false;
                for (uint32_t r = 0; r < row_tiles && ok; ++r) {
                    if (r == 0) ok = um_wait(v_full(i % QU_STAGES), i / QU_STAGES & 1u, &gave_up, 0x907u);
                    if (ok) ok = um_wait(p_full(r), i & 1u, &gave_up, 0x908u);
                    if (!ok) break;
                    um_fence_after();
                    if (um_elect()) {
                        for (uint32_t kk = 0; kk < QU_KEYS / 16; ++kk) {
                            const uint32_t va = v0 + i % QU_STAGES * S::KV + kk * 2048u;
                            um_mma_ts(tmem + S::O_COL + r * 128u, tmem + r * 128u + kk * 8u, desc_hi | ((uint64_t)(QU_BLOCK >> 4) << 16) | (va >> 4), idesc_o, (i | kk) != 0);
                        }
                        if (r + 1 == row_tiles) um_commit(v_empty(i % QU_STAGES));
                    }
                    __syncwarp();
                    if (r == 0) {
                        ok = um_wait(k_full(next % QU_STAGES), next / QU_STAGES & 1u, &gave_up, 0x909u);
                        if (!ok) break;
                        um_fence_after();
                        next_more = items[next % QU_ITEMS].more != 0;
                    }
                    scores(next, r, next_more);
                }
                more = next_more;
            }
            if (!ok) {
                if (um_elect()) um_commit(last_products);
                __syncwarp();
                um_settle(last_products, 0);      // none in flight when tensor memory is given back
            }
        }
    }
    um_fence_before();
    __syncthreads();
    if (warp == 0) {
        um_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
        if (lane == 0) um_report(&gave_up, p.error);
    }
}

template <int CODE, int D, bool CAP>
void qu_launch(uzu_command_buffer* cmd, const QuParams& p, dim3 grid) {
    static std::atomic<uint64_t> opted{0};
    opt_in_dynamic_smem(cmd, quantized_cache_umma_kernel<CODE, D, CAP>, (int)QuShape<D>::SMEM, opted);
    // the warpgroups' shares are of 128 registers a thread: with fewer a warpgroup would wait for registers that never come free
    static const int registers = [] {
        cudaFuncAttributes f{};
        return cudaFuncGetAttributes(&f, quantized_cache_umma_kernel<CODE, D, CAP>) == cudaSuccess ? f.numRegs : 0;
    }();
    if (registers != 128) {
        cmd->record_error(UZU_ERROR_UNSUPPORTED, "quantized_cache_umma_kernel: built with other than 128 registers a thread");
        return;
    }
    launch(cmd, "quantized_cache_umma_kernel", quantized_cache_umma_kernel<CODE, D, CAP>, grid, dim3(QU_THREADS), QuShape<D>::SMEM, p);
}

}  // namespace

bool quantized_cache_umma_applicable(const uzu_quantized_cache_attention_args& a) {
    return a.data_type == UZU_DT_BF16 && a.cache.head_dim <= 128 && a.scale > 0.0f && a.softcap <= kCacheFastCap && ((a.query | a.out) & 15u) == 0 && a.query_row_stride % 8 == 0 && a.query_head_stride % 8 == 0 && a.out_stride % 8 == 0 &&
           std::min(a.sequences.max_rows, a.sequences.rows) > kCacheFewRows && (uint64_t)std::min(a.sequences.max_rows, a.sequences.rows) * (a.heads / a.cache.kv_heads) > kCacheFewPairs;
}

// sequences of more than kCacheFewRows rows and kCacheFewPairs pairs of a row and a head of a key head's group
void encode_quantized_cache_umma(uzu_command_buffer* cmd, const uzu_quantized_cache_attention_args& a, uint64_t row_stats) {
    QuParams p{};
    p.a = a;
    p.capacity = cache_capacity(a.sequences, a.cache.block_tokens);
    p.group = a.heads / a.cache.kv_heads;
    p.stats = reinterpret_cast<float*>(row_stats);
    p.error = cmd->ctx->wait_errors.device_word;
    const uint64_t pairs = (uint64_t)std::min(a.sequences.max_rows, a.sequences.rows) * p.group;
    const dim3 grid((uint32_t)((pairs + 2 * QU_ROWS - 1) / (2 * QU_ROWS)), a.cache.kv_heads, a.sequences.count);
    auto caps = [&](auto code, auto d) {
        if (a.softcap > 0.0f) qu_launch<decltype(code)::value, decltype(d)::value, true>(cmd, p, grid);
        else qu_launch<decltype(code)::value, decltype(d)::value, false>(cmd, p, grid);
    };
    auto dims = [&](auto code) {
        if (a.cache.head_dim <= 64) caps(code, std::integral_constant<int, 64>());
        else caps(code, std::integral_constant<int, 128>());
    };
    if (a.cache.code_type == UZU_CACHE_CODE_I8) dims(std::integral_constant<int, UZU_CACHE_CODE_I8>());
    else dims(std::integral_constant<int, UZU_CACHE_CODE_E4M3>());
}

}  // namespace uzu
