// Causal attention of prompts and chunks of prompts over the paged INT8 cache on the 5th-generation tensor cores
// (tcgen05.mma, scores, weights and sums in tensor memory), head_dim 64 / 96 / 128.
//
// Bound: the two products, 4 * head_dim FLOP per (row, position), and as much time of the exponentials: 16 a clock of an SM
// against 128 x 128 x head_dim x 2 FLOP in 2 * head_dim clocks of its tensor cores.  32/8 heads of 128: 12 000 tokens 1145 us
// (1030 TFLOP/s in bursts, 896 in long runs; the softmax warps issue half of the time, their waits are the rest), 11 packed prompts of 41-1900 tokens 218 us.
//
// An item is 256 rows (128 where there are few) of one (sequence, kv head): row = (new token, query head of the group), two tiles of 128 whose
// products and softmax take turns, and the positions in tiles of 128.  The grid has a CTA for each; one that runs takes over, one
// after the other, items of CTAs that have not begun (cluster launch control), so that the next item's keys are converted and
// its rows of q on their way while this one ends (11 packed prompts 245 -> 226 us, 12 000 tokens 1184 -> 1173).  What is done
// once an item is rolled up: the 32 rows of q of a warp in one piece of code cost 237 us for the former, in a loop of eights 226;
// rows that are not there read the last one instead of zeros: 216 -> 208.
//   warps 0-3, 4-7   softmax of row tile 0 / 1, a thread per row: scores from tensor memory, running maximum and sum,
//                    weights back to tensor memory as f16 in the place of the scores; the output at the end
//   warps 8-11       int8 codes from global memory to f16 in swizzled shared memory; the next tile's loads are in flight
//                    meanwhile
//   warp 14          looks for the next item
//   warps 12, 13     issue the MMAs of row tile 0 / 1, one thread each: S = Q K^T (both from shared memory), O += P V (P from
//                    tensor memory, V with the dims contiguous), 64 positions at a time: the next 64 scores are there
//                    when the softmax has done with these
// Numbers: all operands are f16 (11 significant bits; bf16 would round a weight and a value to 8).  q is multiplied by a
// power of two that takes its row's largest element to 2^14..2^15.  A K operand is code * scale over a power of two of its
// tile, rounded once (the scale goes in as two f16 numbers); multiplying the scores by the scales instead took a tenth of the
// softmax's time.  A weight is at most 2^15: 2^7 times its distance from the row's maximum, which follows the scores
// only when they exceed it by 2^8, since the sums have to be multiplied then.  A V operand is code * scale / 2^E with one E
// for all, after the largest scale so far; when that grows the sums are multiplied, too.  Sums are 32-bit.
// That holds while the scales of an item's values, and those of a tile's keys, lie in two neighbouring ranges of eight binary orders:
// a row must not lose what it sees to the scale of a position that it does not see, or whose weight is nothing.  From the first
// tile on that breaks it ("wide") an item's operands are the codes themselves, exact; the softmax multiplies the scores by the
// keys' scales and the weights by the values', and a row has a power of two of its own, after the largest such product that it
// sees (pr_wide_halves; an item takes about twice as long).  As a function: as a second loop in its place it cost the first
// one 3 % (three chunks 244 -> 253 us).
// A position that a row may not see gets weight 0, and its value must be finite for that: values behind the sequence's end
// are zeros, and one whose scale is not finite is zero with its K scale made NaN, which marks the rows that see it.
#include "paged.cuh"
#include <algorithm>
#include <atomic>

namespace s12 {

constexpr int kPrRows = 128;                        // rows of an MMA
constexpr int kPrTile = 128;                        // positions of a conversion step
constexpr int kPrHalf = 64;                         // positions of an MMA and softmax step
constexpr int kPrThreads = 512;
constexpr int kPrScaleStages = 4;                    // tiles whose powers of two are kept
constexpr unsigned int kPrSite = 0x200000u;         // a wait of this kernel gave up
constexpr float kPrLowest = -3e38f;                  // a maximum of no scores
constexpr float kPrLift = 7.f;                       // weights are multiplied by 2^7: 2^15 at most
constexpr int kPrCtaRows = 2 * kPrRows;             // rows of a CTA
constexpr float kPrSlack = 8.f;                     // a maximum may be exceeded by 2^8 before the sums are scaled

__host__ __device__ constexpr int pr_tile_bytes(int hd) { return (hd + 63) / 64 * kPrRows * 128; }   // blocks of 64 dims: [128 rows][128 bytes]
__host__ __device__ constexpr int pr_smem_bytes(int hd) { return 6 * pr_tile_bytes(hd) + 1024; }

constexpr int kPrItems = 4;                         // places for items
struct PrItem { int seq, lo, row0, rows, kvh, before, room, seen; };   // seq -1: no more
struct PrBars { uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2][2], p_full[2][2], sums_done[2], all_done[2], item_full[kPrItems], item_empty[kPrItems], more, next; };

__device__ __forceinline__ uint32_t pr_elect()
{
    uint32_t leader;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(leader));
    return leader;
}
__device__ __forceinline__ void pr_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pr_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pr_commit(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void pr_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void pr_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void pr_ld32(uint32_t at, float (&r)[32])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
                   "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
                   "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
                   "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
                 : "r"(at) : "memory");
}
// Waits for this warp's loads; r is what one of them brought.  The compiler takes a load's registers for ready before the wait, so
// the wait names them: no use of r can come before it.  Between the load and this no branch may define r either.
__device__ __forceinline__ void pr_ld_wait(float (&r)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
                   "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]),
                   "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]),
                   "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31]) :: "memory");
}
__device__ __forceinline__ void pr_st32(uint32_t at, const uint32_t (&u)[32])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(at), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]),
                   "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]),
                   "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]),
                   "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]), "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31])
                 : "memory");
}
__device__ __forceinline__ void pr_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float pr_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pr_max3(float a, float b, float c)
{
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ uint32_t pr_bf16x2(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pr_f16x2(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// four codes as f16, exactly: code + 128 in the low bits of 1024, minus 1152
__device__ __forceinline__ void pr_codes_f16(uint32_t w, uint32_t& lo, uint32_t& hi)
{
    const uint32_t u = w ^ 0x80808080u, a = prmt(u, 0x64646464u, 0x4140u), b = prmt(u, 0x64646464u, 0x4342u);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
}
// whether x is true in any of the four converter warps
__device__ __forceinline__ bool pr_any(bool x)
{
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(any) : "r"((uint32_t)x) : "memory");
    return any != 0;
}
// Binary orders of scales, eight to a bit: bit i stands for [2^(8 i - 127), 2^(8 i - 119)).  A unit that takes them below 2^8:
__device__ __forceinline__ int pr_unit(uint32_t orders) { return max(8 * (31 - __clz(orders)) - 127, -110); }
// whether there are more than the largest order's bit and the next, or any too small for that unit
__device__ __forceinline__ bool pr_wide(uint32_t orders)
{
    return (orders & (((0x40000000u >> __clz(orders | 1u)) - 1u) | 3u)) != 0;
}
__device__ __forceinline__ float pr_over_1(float power) { return __uint_as_float(0x7F000000u - __float_as_uint(power)); }   // of a power of two
struct PrUnits { float key, value, shift; bool wide; };
// What the scales of a tile's keys and of an item's values are multiplied by, from their orders; `before` and `old` are the values' orders and
// multiplier before this tile.  shift: 2^(E before - E), or, where the item becomes wide here, -zu for the unit that the sums are in
__device__ __forceinline__ PrUnits pr_units(uint32_t before, float old, uint32_t orders_k, uint32_t orders_v)
{
    PrUnits u = {1.f, 1.f, 1.f, (before & 1u) || pr_wide(orders_k) || pr_wide(orders_v)};
    if (u.wide) { if (!(before & 1u)) u.shift = before ? -65536.f * old : -1.f; return u; }
    u.key = __uint_as_float((uint32_t)(127 - pr_unit(orders_k)) << 23);
    u.value = __uint_as_float((uint32_t)(127 - pr_unit(orders_v)) << 23);
    u.shift = u.value * pr_over_1(old);
    return u;
}
// asks for the work of a CTA that has not begun; the answer's 16 bytes arrive at `at`, counted on `bar`
__device__ __forceinline__ void pr_take_cta(uint32_t at, uint32_t bar)
{
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(at), "r"(bar) : "memory");
}
// that CTA's number, or -1: none is left, and no further question is allowed
__device__ __forceinline__ int pr_taken_cta(uint32_t at)
{
    int cta;
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b128 x;\n\tld.shared.b128 x, [%1];\n\tmov.b32 %0, -1;\n\t"
                 "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, x;\n\t"
                 "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, x;\n\t}" : "=r"(cta) : "r"(at) : "memory");
    return cta;
}
// two at a time
typedef float2 Pair;
__device__ __forceinline__ Pair mul2(Pair a, Pair b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ Pair add2(Pair a, Pair b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) { return __ffma2_rn(a, b, c); }

// Operand tiles: blocks of 64 dims, each [128 rows][128 bytes] with the 128-byte swizzle (16-byte chunk c of row r sits at
// c ^ (r & 7)).  For Q and K the rows are the MMA's M and N and the dims its K (K-major); for V the rows are its K and the
// dims its N (MN-major: 8-row groups 1024 bytes apart, blocks of 64 dims 16384 apart).
__device__ __forceinline__ uint32_t pr_chunk(int row, int chunk) { return (uint32_t)((chunk >> 3) * (kPrRows * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)); }
__device__ __forceinline__ uint64_t pr_desc(uint32_t at, uint32_t lead)
{
    return (uint64_t)((at >> 4) & 0x3FFF) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// The halves of a wide item from h on, for a row of the softmax: the operands are codes, their scales come in here.  Seldom, so that they
// are read from the cache again, a lane those of two positions.  m, sum: the row's maximum and sum so far.  Returns the sum and zu:
// the row's unit is 2^16 / zu.
template <int kHD>
__device__ __noinline__ float2 pr_wide_halves(const PagedArgs& C, PrBars& bars, int* s_abort, const uint8_t (&absent_s)[kPrScaleStages][4], const float2 (&unit_s2)[kPrScaleStages], const PrItem w,
                                              int i, int h, int halves, int g0, int c0, int c1, int cs, uint32_t s_at, uint32_t o_at, int limit, float factor, float m, float sum)
{
    const int lane = threadIdx.x & 31;
    auto bar = [](const uint64_t& b) { return smem_addr(&b); };
    auto wait = [&](const uint64_t& b, int phase) { mbar_wait(smem_addr(&b), (uint32_t)phase & 1, C.status, kPrSite, s_abort); };
    float zu = 0.f, zt = 0.f;                                   // the row's unit is 2^16 / zu; its largest weighted value so far over 2^16
#pragma unroll 1
    for (; h < halves; h++) {
        const int j = (g0 + (h >> 1)) % kPrScaleStages, b = h & 1;
        float sk[2], sv[2];
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int t = h * kPrHalf + c * 32 + lane, page = t < w.seen ? paged_page(C, w.seq, t) : -1;
            const size_t at = ((size_t)max(page, 0) * C.n_head_kv + w.kvh) << C.page_shift | (size_t)(t & ((1 << C.page_shift) - 1));
            sk[c] = page < 0 ? 0.f : C.sk[at];
            sv[c] = page < 0 ? 0.f : C.sv[at] * (1.f / 65536.f);
            if (!(fabsf(sv[c]) < INFINITY)) { sk[c] = __uint_as_float(0x7FC00000u); sv[c] = 0.f; }
            if (!(fabsf(sk[c]) < INFINITY)) sk[c] = __uint_as_float(0x7FC00000u);   // an infinity, too
        }
        float x[2][32];
        wait(bars.s_full[i][b], (b ? c1 : c0) + (h >> 1));
        pr_fence_after();
        pr_ld32(s_at + b * kPrHalf, x[0]);
        pr_ld32(s_at + b * kPrHalf + 32, x[1]);
        pr_ld_wait(x[0]);
        pr_ld_wait(x[1]);
        const int left = limit - h * kPrHalf;
        const uint32_t absent = *reinterpret_cast<const uint16_t*>(&absent_s[j][2 * b]);
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < kPrHalf; c++) {
            float& y = x[c / 32][c % 32];
            y *= factor * __shfl_sync(0xFFFFFFFFu, sk[c / 32], c % 32);
            if (c >= left || (absent >> (c / 32 * 8 + c / 16 % 2) & 1)) y = -INFINITY;
            top = fmaxf(top, y);
        }
        const float mn = top - m > kPrSlack ? top : m, f = pr_exp2(m - mn);
        m = mn;
        sum *= f;
        if (zu == 0.f) {                                    // the sums so far are in this unit
            zu = -unit_s2[j].y;
            zt = sum > 0.f ? 8.f / zu : 0.f;                    // about: 2^-1 to 2^23 over zu
        }
        float z = 0.f;
#pragma unroll
        for (int c = 0; c < kPrHalf; c++) {
            float& y = x[c / 32][c % 32];
            y = pr_exp2(__fsub_rn(y, m) + kPrLift);
            sum += y;
            y *= __shfl_sync(0xFFFFFFFFu, sv[c / 32], c % 32);
            z = fmaxf(z, fabsf(y));
        }
        zt = fmaxf(zt * f, z);
        const bool turn = zt > 0.f && !(zt * zu >= 64.f && zt * zu <= 32768.f);
        const int e_old = (int)(__float_as_uint(zu) >> 23), e_new = turn ? min(max(264 - (int)(__float_as_uint(zt) >> 23), 1), 254) : e_old;
        if (__any_sync(0xFFFFFFFFu, f != 1.f || turn)) {
            if (h > 0) {
                const int by = e_new - e_old;               // in two steps: each is a float
                const float f0 = f * __uint_as_float((uint32_t)(127 + by / 2) << 23), f1 = __uint_as_float((uint32_t)(127 + by - by / 2) << 23);
                wait(bars.sums_done[i], cs + h - 1);
                pr_fence_after();
#pragma unroll 1
                for (int c = 0; c < kHD; c += 32) {
                    float o[32];
                    pr_ld32(o_at + c, o);
                    pr_ld_wait(o);
                    uint32_t u[32];
#pragma unroll
                    for (int d = 0; d < 32; d++) u[d] = __float_as_uint(o[d] * f0 * f1);
                    pr_st32(o_at + c, u);
                }
            }
            zu = __uint_as_float((uint32_t)e_new << 23);
        }
        uint32_t p[32];
#pragma unroll
        for (int c = 0; c < 32; c++) p[c] = pr_f16x2(x[c / 16][2 * c % 32] * zu, x[c / 16][2 * c % 32 + 1] * zu);
        pr_st32(s_at + b * kPrHalf, p);
        pr_st_wait();
        pr_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(bars.p_full[i][b]));
    }
    return make_float2(sum, zu);
}

struct PromptParams {
    PagedAttn a;
    int item_rows;              // of an item: 256, or 128
    uint32_t gqa_mul;           // ceil(2^32 / query heads of a kv head), 0 for one: divides what is below 2^32 / that number
};

template <int kHD>
__global__ void __launch_bounds__(kPrThreads, 1)
paged_prompt_kernel(const __grid_constant__ PromptParams P)
{
    constexpr int kTileBytes = pr_tile_bytes(kHD), kPieces = kHD / 16;
    extern __shared__ __align__(16) uint8_t pr_smem[];
    __shared__ PrBars bars;
    // of a tile: the power of two of its keys; 2^(E before - E) of its values, or, where the item becomes wide, less the first zu (pr_wide_halves)
    __shared__ __align__(8) float2 unit_s2[kPrScaleStages];
    __shared__ uint2 orders_s[2][4];                               // the converters' binary orders of a tile's scales: keys, values
    __shared__ float unit_s[2 * kPrItems];                         // of an item: 2^E at the end; four items may be read ahead of one
    __shared__ __align__(16) PrItem item_s[kPrItems];
    __shared__ __align__(16) uint4 taken_s;
    __shared__ __align__(4) uint8_t absent_s[kPrScaleStages][4];   // byte i, bit h: the 16 positions from 32 i + 16 h on have no page
    __shared__ float factor_s[kPrCtaRows];
    __shared__ uint32_t tmem_s;
    __shared__ int s_abort;
    uint8_t* smem = pr_smem + ((1024u - (smem_addr(pr_smem) & 1023u)) & 1023u);
    uint8_t* q_s = smem, *k_s = smem + 2 * kTileBytes, *v_s = smem + 4 * kTileBytes;
    const PagedArgs& C = P.a.c;
    // the same in all lanes, for the compiler to see: a warp's addresses are computed once (226 -> 215 us, 1180 -> 1157)
    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int gqa = P.a.n_head / C.n_head_kv;
    auto token_of = [&](int row) { return P.gqa_mul ? (int)__umulhi((uint32_t)row, P.gqa_mul) : row; };
    grid_launch_dependents();
    grid_dependency_wait();

    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int i = 0; i < kPrItems; i++) { mbar_init(smem_addr(&bars.item_full[i]), 1); mbar_init(smem_addr(&bars.item_empty[i]), 14); }
        mbar_init(smem_addr(&bars.more), 1); mbar_init(smem_addr(&bars.next), 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(smem_addr(&bars.q_full[i]), 4);
            mbar_init(smem_addr(&bars.k_full[i]), 4); mbar_init(smem_addr(&bars.v_full[i]), 4);
            mbar_init(smem_addr(&bars.k_empty[i]), 2); mbar_init(smem_addr(&bars.v_empty[i]), 2);
            for (int b = 0; b < 2; b++) { mbar_init(smem_addr(&bars.s_full[i][b]), 1); mbar_init(smem_addr(&bars.p_full[i][b]), 4); }
            mbar_init(smem_addr(&bars.sums_done[i]), 1); mbar_init(smem_addr(&bars.all_done[i]), 1);
        }
        mbar_fence_init();
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&tmem_s)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pr_fence_before();
    __syncthreads();
    pr_fence_after();
    const uint32_t tmem = tmem_s;
    auto bar = [](const uint64_t& b) { return smem_addr(&b); };
    auto wait = [&](const uint64_t& b, int phase) { mbar_wait(smem_addr(&b), (uint32_t)phase & 1, C.status, kPrSite, &s_abort); };

    // the k-th item of this CTA, for a whole warp
    auto item_at = [&](int k) {
        wait(bars.item_full[k % kPrItems], k / kPrItems);
        const PrItem w = item_s[k % kPrItems];
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(bars.item_empty[k % kPrItems]));
        if (*(volatile int*)&s_abort) return PrItem{-1};
        return w;
    };
    auto halves_of = [](const PrItem& w) { return max(1, (w.seen + kPrHalf - 1) / kPrHalf); };

    if (warp < 8) {
        // ------------------------------ softmax -------------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
        const int i = warp >> 2, r = warp * 32 + lane;               // row tile, row of the CTA
        const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t s_at = mine + i * 2 * kPrHalf, o_at = mine + 4 * kPrHalf + i * 128;
        uint8_t* const tile_q = q_s + i * kTileBytes;                // the warp's 32 rows in it are its own: q, then the output
        int g = 0, c0 = 0, c1 = 0, cs = 0, done = 0;                 // tiles; halves of this row tile in either buffer, all, and items, so far
        for (int item = 0; ; item++) {
            const PrItem w = item_at(item);
            if (w.seq < 0) break;
            const int halves = halves_of(w), rows = w.rows, row0 = w.row0, g0 = g;
            g += (halves + 1) / 2;
            if (i > 0 && rows <= kPrRows) continue;
            // ---- the warp's rows of q as f16, all of them in flight together, a lane four dims of each
            {
                const float to_log2 = fabsf(P.a.scale) * 1.4426950408889634f;
                const float* q0 = P.a.q + (size_t)w.lo * P.a.q_stride + (size_t)w.kvh * gqa * kHD + 4 * (lane % (kHD / 4));
                const bool in_row = 4 * lane < kHD;
                auto row_of = [&](int r) {
                    const int t = token_of(row0 + r);
                    return q0 + (size_t)t * P.a.q_stride + (row0 + r - t * gqa) * kHD;
                };
                auto top_of = [&](const float4& v) {
                    const uint32_t a = __float_as_uint(v.x) & 0x7FFFFFFFu, b = __float_as_uint(v.y) & 0x7FFFFFFFu;
                    const uint32_t c = __float_as_uint(v.z) & 0x7FFFFFFFu, d = __float_as_uint(v.w) & 0x7FFFFFFFu;
                    return __reduce_max_sync(0xFFFFFFFFu, max(max(a, b), max(c, d))) & 0x7F800000u;
                };
                auto put = [&](int n, const float4& v, uint32_t top) {   // row 32 warp + n
                    // 2^e of the largest, e >= -100, or nothing: rows of smaller ones count as zero, and a NaN or an infinity, the
                    // largest of all, becomes a NaN
                    const bool fine = top - (27u << 23) < (228u << 23);
                    const float up = fine ? __uint_as_float((268u << 23) - top ^ (P.a.scale < 0.f ? 0x80000000u : 0u)) : 0.f;   // 2^(14 - e)
                    const Pair xy = mul2({v.x, v.y}, {up, up}), zw = mul2({v.z, v.w}, {up, up});
                    if (in_row) *reinterpret_cast<uint2*>(tile_q + pr_chunk((warp & 3) * 32 + n, lane >> 1) + (lane & 1) * 8) = make_uint2(pr_f16x2(xy.x, xy.y), pr_f16x2(zw.x, zw.y));
                    if (lane == 0) factor_s[warp * 32 + n] = fine ? to_log2 * __uint_as_float(top - (14u << 23)) : 0.f;
                };
                if (((reinterpret_cast<uintptr_t>(P.a.q) & 15) | (P.a.q_stride & 3)) == 0) {
                    float4 v[8], next[8];
                    auto fetch = [&](float4 (&to)[8], int n) {
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            to[e] = *reinterpret_cast<const float4*>(row_of(min(warp * 32 + n + e, rows - 1)));
                        }
                    };
                    fetch(v, 0);
                    fetch(next, 8);
#pragma unroll 1
                    for (int n = 0; n < 32; n += 8) {                // no store is moved before a reduction: eight of them together
                        uint32_t top[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) top[e] = top_of(v[e]);
#pragma unroll
                        for (int e = 0; e < 8; e++) put(n + e, v[e], top[e]);
#pragma unroll
                        for (int e = 0; e < 8; e++) v[e] = next[e];
                        if (n < 16) fetch(next, n + 16);
                    }
                } else {
#pragma unroll 1
                    for (int n = 0; n < 32; n++) {
                        const float* q = row_of(min(warp * 32 + n, rows - 1));
                        const float4 v = make_float4(q[0], q[1], q[2], q[3]);
                        put(n, v, top_of(v));
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the MMAs read what ordinary stores wrote
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(bars.q_full[i]));
            }
            const int tok = token_of(row0 + r);
            const int limit = r < rows ? min(w.before + tok, w.room) : 0;   // positions that this row sees
            const int least = __reduce_min_sync(0xFFFFFFFFu, limit);
            const float factor = factor_s[r];
            float m = kPrLowest;
            Pair l = {0.f, 0.f};
            int h = 0;
#pragma unroll 1
            for (; h < halves; h++) {
                const int j = (g0 + (h >> 1)) % kPrScaleStages, b = h & 1;
                float x[2][32];
                wait(bars.s_full[i][b], (b ? c1 : c0) + (h >> 1));                    // then half h - 2 is in the sums
                pr_fence_after();
                pr_ld32(s_at + b * kPrHalf, x[0]);
                pr_ld32(s_at + b * kPrHalf + 32, x[1]);
                pr_ld_wait(x[0]);
                pr_ld_wait(x[1]);                                   // nothing is left to wait for: names the registers
                const float2 unit = unit_s2[j];
                const float fac = fmaxf(factor * unit.x, 1e-37f);   // above 0: a masked score stays -infinity
                const int left = limit - h * kPrHalf;               // positions of the half that the row sees
                const uint32_t absent = *reinterpret_cast<const uint16_t*>(&absent_s[j][2 * b]);
                if (least - h * kPrHalf < kPrHalf || absent) {
#pragma unroll
                    for (int c = 0; c < kPrHalf; c++) if (c >= left || (absent >> (c / 32 * 8 + c / 16 % 2) & 1)) x[c / 32][c % 32] = -INFINITY;
                }
                float t0 = x[0][0], t1 = x[0][1], t2 = x[0][2], t3 = x[0][3];
                auto at = [&](int e) { return x[e / 32][e % 32]; };
#pragma unroll
                for (int c = 4; c + 8 <= kPrHalf; c += 8) {
                    t0 = pr_max3(t0, at(c), at(c + 1)); t1 = pr_max3(t1, at(c + 2), at(c + 3));
                    t2 = pr_max3(t2, at(c + 4), at(c + 5)); t3 = pr_max3(t3, at(c + 6), at(c + 7));
                }
                const float top = pr_max3(fmaxf(t0, t1), pr_max3(t2, at(kPrHalf - 4), at(kPrHalf - 3)), pr_max3(t3, at(kPrHalf - 2), at(kPrHalf - 1))) * fac;
                const bool rise = top - m > kPrSlack;
                const float shift = b == 0 ? unit.y : 1.f;
                if (__any_sync(0xFFFFFFFFu, rise) || shift != 1.f) {
                    if (shift < 0.f) break;                         // from here on the item is wide
                    const float mn = rise ? top : m, f = pr_exp2(m - mn);
                    m = mn;
                    l = mul2(l, {f, f});
                    if (h > 0) {
                        wait(bars.sums_done[i], cs + h - 1);                 // the half before it, too
                        pr_fence_after();
#pragma unroll 1
                        for (int c = 0; c < kHD; c += 32) {
                            float o[32];
                            pr_ld32(o_at + c, o);
                            pr_ld_wait(o);
                            uint32_t u[32];
#pragma unroll
                            for (int d = 0; d < 32; d++) u[d] = __float_as_uint(o[d] * (f * shift));
                            pr_st32(o_at + c, u);
                        }
                    }
                }
                Pair fac2 = {fac, fac}, neg = {kPrLift - m, kPrLift - m};
                // Scores this large are their own roundings apart from x * fac, which is not rounded below: a weight could leave f16
                if (__any_sync(0xFFFFFFFFu, fabsf(m) > 1048576.f && m != kPrLowest)) {
#pragma unroll
                    for (int c = 0; c < kPrHalf; c++) x[c / 32][c % 32] = __fsub_rn(__fmul_rn(x[c / 32][c % 32], fac), m);
                    fac2 = {1.f, 1.f}; neg = {kPrLift, kPrLift};
                }
                uint32_t p[32];
#pragma unroll
                for (int c = 0; c < 32; c++) {
                    Pair y = fma2({x[c / 16][2 * c % 32], x[c / 16][2 * c % 32 + 1]}, fac2, neg);
                    y.x = pr_exp2(y.x); y.y = pr_exp2(y.y);
                    l = add2(l, y);
                    p[c] = pr_f16x2(y.x, y.y);
                }
                pr_st32(s_at + b * kPrHalf, p);
                pr_st_wait();
                pr_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(bars.p_full[i][b]));
            }
            float zu = 0.f;                                         // wide: the row's unit is 2^16 / zu
            if (h < halves) {
                const float2 rest = pr_wide_halves<kHD>(C, bars, &s_abort, absent_s, unit_s2, w, i, h, halves, g0, c0, c1, cs, s_at, o_at, limit, factor, m, l.x + l.y);
                l = {rest.x, 0.f};
                zu = rest.y;
            }
            // ---- the output
            wait(bars.all_done[i], done++);                          // a wait tells odd from even only: of sums_done's phases two may be ahead
            pr_fence_after();
            const float sum = l.x + l.y, rd = sum == 0.f ? 0.f : zu != 0.f ? 65536.f / sum / zu : unit_s[item % (2 * kPrItems)] / sum;   // no position at all: zeros
            // A row as one piece: by way of shared memory, in the place of the warp's rows of q, which have been read
            constexpr int kChunks = kHD / 8;
            auto chunk_at = [&](int row, int c) { return tile_q + pr_chunk((warp & 3) * 32 + row, c); };
#pragma unroll 1
            for (int c = 0; c < kHD; c += 32) {
                float o[32];
                pr_ld32(o_at + c, o);
                pr_ld_wait(o);
#pragma unroll
                for (int d = 0; d < 32; d += 8)
                    *reinterpret_cast<uint4*>(chunk_at(lane, (c + d) / 8)) =
                        make_uint4(pr_bf16x2(o[d] * rd, o[d + 1] * rd), pr_bf16x2(o[d + 2] * rd, o[d + 3] * rd),
                                   pr_bf16x2(o[d + 4] * rd, o[d + 5] * rd), pr_bf16x2(o[d + 6] * rd, o[d + 7] * rd));
            }
            __syncwarp();
            const bool aligned = ((reinterpret_cast<uintptr_t>(P.a.out) & 15) | (P.a.out_stride & 7)) == 0;
            const int first = warp * 32;                            // this warp's rows
            int16_t* out0 = P.a.out + (size_t)w.lo * P.a.out_stride + (size_t)w.kvh * gqa * kHD;
#pragma unroll 2
            for (int it = 0; it < kChunks; it++) {
                const int x = it * 32 + lane, row = x / kChunks, c = x - row * kChunks, t = token_of(row0 + first + row), hd = row0 + first + row - t * gqa;
                const uint4 y = *reinterpret_cast<const uint4*>(chunk_at(row, c));
                int16_t* out = out0 + (size_t)t * P.a.out_stride + hd * kHD + c * 8;
                if (first + row >= rows) continue;
                if (aligned) {
                    *reinterpret_cast<uint4*>(out) = y;
                } else {
                    const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int e = 0; e < 8; e++) out[e] = (int16_t)(w[e >> 1] >> (16 * (e & 1)));
                }
            }
            __syncwarp();                                           // the next item's q goes where the rows were
            c0 += (halves + 1) / 2; c1 += halves / 2; cs += halves;
        }
    } else if (warp < 12) {
        // ------------------------------ codes to operands ---------------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        // A warp has 32 rows of the tile, four (eight at head_dim 64) at a time: a lane 16 codes of one of them.  Lanes 0-7 of
        // a store have two neighbouring rows, whose chunks the swizzle puts on different banks.  Lane l has the scales of row l.
        const int cw = warp - 8;
        constexpr int kRowsAt = kHD == 64 ? 8 : 4, kIts = 32 / kRowsAt;
        const int row_of = kHD == 64 ? lane >> 2 : (lane >> 4) << 1 | (lane >> 2 & 1), piece = kHD == 64 ? lane & 3 : (lane >> 3 & 1) * 4 + (lane & 3);
        const bool live = piece < kPieces;
        const int ps = 1 << C.page_shift, mine = cw * 32 + lane;
        bool missing = false;
        int g = 0;                                                  // tiles so far
        for (int item = 0; ; item++) {
            const PrItem w = item_at(item);
            if (pr_any(w.seq < 0)) break;                           // all four together, also where a wait gave up: they share a barrier
            const int halves = halves_of(w), n = (halves + 1) / 2, seen = w.seen, kvh = w.kvh;
            const int* table = C.table + (size_t)w.seq * C.table_stride;
            if (paged_past_table(C, w.before + token_of(w.row0 + w.rows - 1))) missing = true;
            // the pools' row of position p, and whether there is one; -1 where the table has no page or no row sees p
            auto row_at = [&](int p) {
                if (p >= seen) return -1ll;
                const int page = table[p >> C.page_shift];
                if ((unsigned)page >= (unsigned)C.num_pages) { missing = true; return -1ll; }
                return (long long)((((uint32_t)page * C.n_head_kv + kvh) << C.page_shift) + (p & (ps - 1)));
            };
            const int8_t* k_at = C.k + row_of * kHD + 16 * piece, *v_at = C.v + row_of * kHD + 16 * piece;
            uint4 k[kIts], v[kIts];
            float sk = 0.f, sv = 0.f;
            // 16 rows lie together; absent ones read row 0 and are masked later
            auto fetch = [&](uint4 (&to)[kIts], const int8_t* at, long long row) {
                const uint32_t r = (uint32_t)max(row, 0ll);
                const int8_t* half[2] = {at + (size_t)__shfl_sync(0xFFFFFFFFu, r, 0) * kHD, at + (size_t)__shfl_sync(0xFFFFFFFFu, r, 16) * kHD};
#pragma unroll
                for (int it = 0; it < kIts; it++)
                    if (live) to[it] = *reinterpret_cast<const uint4*>(half[it / (kIts / 2)] + it % (kIts / 2) * kRowsAt * kHD);
            };
            auto fetch_scales = [&](long long row) { sk = row >= 0 ? C.sk[row] : 0.f; sv = row >= 0 ? C.sv[row] : 0.f; };
            // Where a lane's chunks go: row + 4 changes bit 2 of the chunk
            const uint32_t to0 = pr_chunk(cw * 32 + row_of, 2 * piece);
            auto store = [&](uint8_t* tile, int it, const uint32_t (&y)[8]) {
                const uint32_t to = (kRowsAt == 4 && (it & 1) ? to0 ^ 64u : to0) + it * kRowsAt * 128;
                *reinterpret_cast<uint4*>(tile + to) = make_uint4(y[0], y[1], y[2], y[3]);
                *reinterpret_cast<uint4*>(tile + (to ^ 16u)) = make_uint4(y[4], y[5], y[6], y[7]);
            };
            long long row = row_at(mine), row_next = n > 1 ? row_at(kPrTile + mine) : -1;
            fetch_scales(row);
            fetch(k, k_at, row);
            fetch(v, v_at, row);
            uint32_t orders_k = 0, orders_v = 0;                    // of the last tile's keys, and of the item's values so far
            float unit_k = 0.f, unit_v = 0.f;                       // what these scales are multiplied by
            // Binary orders of the tile's scales, eight to a bit: bit i for [2^(8 i - 127), 2^(8 i - 119)); zeros and what is not finite have none
            auto note_orders = [&](int st) {
                const uint32_t bits_k = __float_as_uint(sk) & 0x7FFFFFFFu, bits_v = __float_as_uint(sv) & 0x7FFFFFFFu;
                const uint32_t mine_k = __reduce_or_sync(0xFFFFFFFFu, bits_k - 1 < 0x7F7FFFFFu ? 1u << (bits_k >> 26) : 0u);
                const uint32_t mine_v = __reduce_or_sync(0xFFFFFFFFu, bits_v - 1 < 0x7F7FFFFFu ? 1u << (bits_v >> 26) : 0u);
                if (lane == 0) orders_s[st][cw] = make_uint2(mine_k, mine_v);
            };
            note_orders(g & 1);
            for (int j = 0; j < n; j++, g++) {
                const int st = g & 1;
                if (j == max(n - 2, 0) && mine == 0) mbar_arrive(bar(bars.more));   // the item after this one may be looked for
                const bool absent = row < 0;
                named_bar_sync(1, 128);
                const uint2 w0 = orders_s[st][0], w1 = orders_s[st][1], w2 = orders_s[st][2], w3 = orders_s[st][3];
                const uint32_t now_k = w0.x | w1.x | w2.x | w3.x, now_v = orders_v | w0.y | w1.y | w2.y | w3.y;
                float shift = 1.f;
                if (j == 0 || now_k != orders_k || now_v != orders_v) {   // seldom
                    const PrUnits u = pr_units(j == 0 ? 0u : orders_v, unit_v, now_k, now_v);
                    unit_k = u.key; unit_v = u.value; shift = j == 0 && u.shift > 0.f ? 1.f : u.shift;
                    orders_k = now_k; orders_v = u.wide ? now_v | 1u : now_v;
                }
                const bool fine = (__float_as_uint(sv) & 0x7FFFFFFFu) < 0x7F800000u;
                if (orders_v & 1u) sk = sv = 1.f;                   // wide: the codes themselves
                const float key_scale = (fine ? sk : __uint_as_float(0x7FC00000u)) * unit_k;
                const uint32_t key_hi = pr_f16x2(key_scale, 0.f) & 0xFFFFu;       // the scale as a sum of two f16
                float key_hi_f;
                asm("{\n\t.reg .b16 h, z;\n\tmov.b32 {h, z}, %1;\n\tcvt.f32.f16 %0, h;\n\t}" : "=f"(key_hi_f) : "r"(key_hi));
                const uint32_t key_parts = key_hi | pr_f16x2(0.f, key_scale - key_hi_f);
                // ---- K
                if (g >= 2) wait(bars.k_empty[st], (g >> 1) - 1);
                const uint32_t gone = __ballot_sync(0xFFFFFFFFu, absent);   // a whole half, or rows that nobody sees
                if (lane == 0) absent_s[g % kPrScaleStages][cw] = (uint8_t)((gone & 1u) | (gone >> 16 & 1u) << 1);
                if (mine == 0) {
                    unit_s2[g % kPrScaleStages] = make_float2(pr_over_1(unit_k), shift);
                    if (j == n - 1) unit_s[item % (2 * kPrItems)] = pr_over_1(unit_v);
                }
#pragma unroll
                for (int it = 0; it < kIts; it++) {
                    const uint32_t parts = __shfl_sync(0xFFFFFFFFu, key_parts, it * kRowsAt + row_of), f_hi = prmt(parts, parts, 0x1010u), f_lo = prmt(parts, parts, 0x3232u);
                    if (!live) continue;
                    const uint32_t w[4] = {k[it].x, k[it].y, k[it].z, k[it].w};
                    uint32_t y[8];
#pragma unroll
                    for (int d = 0; d < 4; d++) {
                        pr_codes_f16(w[d], y[2 * d], y[2 * d + 1]);
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            uint32_t low;
                            asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(low) : "r"(y[2 * d + h]), "r"(f_lo));
                            asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(y[2 * d + h]) : "r"(f_hi), "r"(low));
                        }
                    }
                    store(k_s + st * kTileBytes, it, y);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(bars.k_full[st]));
                const float scale = fine ? sv * unit_v : 0.f;
                const uint32_t scale2 = pr_f16x2(scale, scale);
                const long long row_next2 = j + 2 < n ? row_at((j + 2) * kPrTile + mine) : -1;
                if (j + 1 < n) { fetch_scales(row_next); fetch(k, k_at, row_next); }
                // ---- V
                if (g >= 2) wait(bars.v_empty[st], (g >> 1) - 1);
#pragma unroll
                for (int it = 0; it < kIts; it++) {
                    const uint32_t f2 = __shfl_sync(0xFFFFFFFFu, scale2, it * kRowsAt + row_of);
                    if (!live) continue;
                    const uint32_t w[4] = {v[it].x, v[it].y, v[it].z, v[it].w};
                    uint32_t y[8];
#pragma unroll
                    for (int d = 0; d < 4; d++) {
                        pr_codes_f16(w[d], y[2 * d], y[2 * d + 1]);
                        asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(y[2 * d]) : "r"(f2));
                        asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(y[2 * d + 1]) : "r"(f2));
                    }
                    store(v_s + st * kTileBytes, it, y);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(bars.v_full[st]));
                if (j + 1 < n) { fetch(v, v_at, row_next); note_orders(st ^ 1); }
                row = row_next; row_next = row_next2;
            }
        }
        if (missing) atomicOr(C.status, kStatusPage);
    } else {
        // ------------------------------ MMAs ----------------------------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        // the rows of CTA number cta: tiles of all sequences counted from the last, a kv head after the other
        auto find = [&](int cta) {
            const int kvh = cta % C.n_head_kv;
            int seq = -1, lo = 0, hi = 0, tile = cta / C.n_head_kv;
            for (int s1 = C.num_seqs; s1 > 0 && seq < 0; s1 -= 32) {   // sequence s1 - 1 - lane
                const int s = s1 - 1 - lane;
                int a = 0, b = 0, n = 0;
                if (s >= 0) { paged_rows(C, s, a, b); n = b > a ? (int)(((long long)(b - a) * gqa + P.item_rows - 1) / P.item_rows) : 0; }
                int upto = n;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) { const int o = __shfl_up_sync(0xFFFFFFFFu, upto, off); if (lane >= off) upto += o; }
                const unsigned over = __ballot_sync(0xFFFFFFFFu, upto > tile);
                if (over) {
                    const int l = __ffs(over) - 1;
                    seq = s1 - 1 - l; lo = __shfl_sync(0xFFFFFFFFu, a, l); hi = __shfl_sync(0xFFFFFFFFu, b, l);
                    tile = __shfl_sync(0xFFFFFFFFu, upto, l) - 1 - tile;   // the sequence's last tile, which sees most, comes first
                } else {
                    tile -= __shfl_sync(0xFFFFFFFFu, upto, 31);
                }
            }
            PrItem w = {-1};
            if (seq >= 0) {
                const int row0 = tile * P.item_rows, rows = min(P.item_rows, (hi - lo) * gqa - row0);
                const int room = paged_len(C, seq), before = C.kv_len[seq] - (hi - lo) + 1;   // token t sees min(before + t, room) positions
                w = {seq, lo, row0, rows, kvh, before, room, max(0, min(before + token_of(row0 + rows - 1), room))};
            }
            return w;
        };
        // the number of a CTA that has not begun, which then never does; -1: none
        int asked = 0;
        auto take = [&] {
            if (lane == 0) { mbar_arrive_expect_tx(bar(bars.next), 16); pr_take_cta(smem_addr(&taken_s), bar(bars.next)); }
            __syncwarp();
            wait(bars.next, asked++);
            const int cta = *(volatile int*)&s_abort ? -1 : pr_taken_cta(smem_addr(&taken_s));
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // read before the next answer comes
            __syncwarp();
            return cta;
        };
        // an item's rows of q on their way to L2 while the one before it is worked on
        auto ask = [&](const PrItem& w) {
            if (((reinterpret_cast<uintptr_t>(P.a.q) & 15) | (P.a.q_stride & 3)) != 0) return;
            const int first = token_of(w.row0), last = token_of(w.row0 + w.rows - 1);
            for (int t = first + lane; t <= last; t += 32)
                asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(P.a.q + (size_t)(w.lo + t) * P.a.q_stride + (size_t)w.kvh * gqa * kHD), "r"(gqa * kHD * 4) : "memory");
        };
        if (warp < 14) {                                           // a warp per row tile
            const int i = warp - 12;
            const uint32_t idesc_s = 1u << 4 | (uint32_t)(kPrHalf >> 3) << 17 | (uint32_t)(kPrRows >> 4) << 24;                        // f16 x f16
            const uint32_t idesc_o = 1u << 4 | 1u << 16 | (uint32_t)(kHD >> 3) << 17 | (uint32_t)(kPrRows >> 4) << 24;   // the same, B with N contiguous
            const uint64_t qd = pr_desc(smem_addr(q_s) + i * kTileBytes, 16), kd = pr_desc(smem_addr(k_s), 16), vd = pr_desc(smem_addr(v_s), kPrRows * 128);
            const uint32_t s_at = tmem + i * 2 * kPrHalf, o_at = tmem + 4 * kPrHalf + i * 128;
            int g = 0, c0 = 0, c1 = 0, cs = 0, nq = 0;              // tiles, halves in either buffer, halves, items of two row tiles so far
            for (int item = 0; ; item++) {
                const PrItem w = item_at(item);
                if (w.seq < 0) break;
                const int halves = halves_of(w), n = (halves + 1) / 2, g0 = g;
                g += n;
                if (i > 0 && w.rows <= kPrRows) {                       // nothing to do with the item's keys and values
                    for (int j = g0; j < g; j++) {
                        wait(bars.k_full[j & 1], j >> 1);
                        if (lane == 0) mbar_arrive(bar(bars.k_empty[j & 1]));
                        wait(bars.v_full[j & 1], j >> 1);
                        if (lane == 0) mbar_arrive(bar(bars.v_empty[j & 1]));
                    }
                    continue;
                }
                // scores of half h; the tile's keys have been used with its last half
                auto scores = [&](int h) {
                    const uint64_t k = kd + (uint32_t)((g0 + (h >> 1) & 1) * (kTileBytes >> 4) + (h & 1) * (kPrHalf * 128 >> 4));
                    const uint32_t d = s_at + (h & 1) * kPrHalf;
#pragma unroll
                    for (int s = 0; s < kHD / 16; s++) {
                        const uint32_t off = (uint32_t)((s >> 2) * (kPrRows * 128) + (s & 3) * 32) >> 4;
                        pr_mma_ss(d, qd + off, k + off, idesc_s, s > 0);
                    }
                    pr_commit(bar(bars.s_full[i][h & 1]));
                    if ((h & 1) || h + 1 == halves) pr_commit(bar(bars.k_empty[g0 + (h >> 1) & 1]));
                };
                wait(bars.q_full[i], nq++);
                wait(bars.k_full[g0 & 1], g0 >> 1);
                pr_fence_after();
                __syncwarp();
                if (pr_elect()) {
                    scores(0);
                    if (halves > 1) scores(1);
                }
                __syncwarp();
#pragma unroll 1
                for (int h = 0; h < halves; h++) {
                    const int b = h & 1, at = g0 + (h >> 1), st = at & 1;      // tile of all
                    if (b == 0) wait(bars.v_full[st], at >> 1);
                    wait(bars.p_full[i][b], (b ? c1 : c0) + (h >> 1));
                    const bool more = h + 2 < halves;
                    if (more && b == 0) wait(bars.k_full[st ^ 1], (at + 1) >> 1);
                    pr_fence_after();
                    __syncwarp();
                    if (pr_elect()) {
                        const uint64_t v = vd + (uint32_t)((st * kTileBytes + b * kPrHalf * 128) >> 4);
                        const uint32_t p = s_at + b * kPrHalf;
#pragma unroll
                        for (int s = 0; s < kPrHalf / 16; s++)          // 16 positions: 8 columns of weights, 16 rows of values
                            pr_mma_ts(o_at, p + 8 * s, v + (uint32_t)(s * 16 * 128 >> 4), idesc_o, h > 0 || s > 0);
                        if (b == 1 || h + 1 == halves) pr_commit(bar(bars.v_empty[st]));
                        pr_commit(bar(bars.sums_done[i]));
                        if (h + 1 == halves) pr_commit(bar(bars.all_done[i]));
                    }
                    __syncwarp();
                    if (more) {                                         // in the weights' place, when they have been read
                        wait(bars.sums_done[i], cs + h);
                        pr_fence_after();
                        __syncwarp();
                        if (pr_elect()) scores(h + 2);
                        __syncwarp();
                    }
                }
                c0 += (halves + 1) / 2; c1 += halves / 2; cs += halves;
            }
        } else if (warp == 14) {
            // ---- the items: this CTA's, then those of CTAs that have not begun
            int cta = (int)blockIdx.x;
            for (int k = 0; ; k++) {
                PrItem w = {-1};
                while (cta >= 0 && w.seq < 0) {
                    w = find(cta);
                    if (w.seq >= 0) break;
                    cta = take();                                   // more CTAs than items
                }
                if (k >= kPrItems) wait(bars.item_empty[k % kPrItems], k / kPrItems - 1);
                if (lane == 0) { item_s[k % kPrItems] = w; mbar_arrive(bar(bars.item_full[k % kPrItems])); }
                __syncwarp();
                if (w.seq < 0 || *(volatile int*)&s_abort) break;
                if (k > 0) ask(w);
                wait(bars.more, k);
                cta = take();
            }
        }
    }
    if (*(volatile int*)&s_abort)                                  // a wait gave up: MMAs in flight finish before tensor memory goes
        for (int i = 0; i < 256; i++) __nanosleep(1000);
    pr_fence_before();
    __syncthreads();
    if (warp == 12) {
        pr_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

template <int kHD>
static int prompt_launch(const PromptParams& P, long long grid, void* stream, const char* who)
{
    static std::atomic<bool> attr_set[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_set[dev].load(std::memory_order_relaxed)) {
        const int rc = check_cuda(cudaFuncSetAttribute(paged_prompt_kernel<kHD>, cudaFuncAttributeMaxDynamicSharedMemorySize, pr_smem_bytes(kHD)), who);
        if (rc) return rc;
        if (dev >= 0 && dev < 64) attr_set[dev].store(true, std::memory_order_relaxed);
    }
    return launch(paged_prompt_kernel<kHD>, dim3((unsigned)grid), dim3(kPrThreads), pr_smem_bytes(kHD), stream, who, P);
}

// 1: not a shape of this kernel
int paged_prompt_launch(const PagedAttn& A, void* stream, const char* who)
{
    const int hd = A.c.head_dim, gqa = A.n_head / A.c.n_head_kv;
    if (hd != 64 && hd != 96 && hd != 128) return 1;
    // rows as far as the division by multiplication holds
    if ((long long)A.c.num_tokens * gqa + kPrCtaRows >= (1ll << 32) / gqa) return 1;
    PromptParams P = {A, kPrCtaRows, gqa == 1 ? 0u : (uint32_t)(((1ull << 32) + gqa - 1) / gqa)};
    // items at most: every sequence's last one may be a part of one
    auto items = [&](int rows) {
        return std::min((long long)A.c.num_tokens * gqa / rows + std::min(A.c.num_seqs, A.c.num_tokens), A.c.num_seqs * (((long long)A.max_new * gqa + rows - 1) / rows)) * A.c.n_head_kv;
    };
    // So few that halves of them are all resident together: halves.  One prompt of 300 tokens (32/8 heads) 17.2 -> 15.0 us, of 512 20.7 ->
    // 18.2, two of 256 behind 8000 149 -> 138; halves in the last round alone: three chunks of 2.3 rounds 250 -> 244, but one prompt
    // of 4000 tokens 161 -> 170
    if (2 * items(kPrCtaRows) <= sm_count()) P.item_rows = kPrRows;
    const long long grid = items(P.item_rows);
    if (grid > 0x7FFFFFFF) return fail(S12_ERR_TOO_LARGE, "%s: %d tokens", who, A.c.num_tokens);
    return hd == 64 ? prompt_launch<64>(P, grid, stream, who) : hd == 96 ? prompt_launch<96>(P, grid, stream, who) : prompt_launch<128>(P, grid, stream, who);
}

}  // namespace s12
