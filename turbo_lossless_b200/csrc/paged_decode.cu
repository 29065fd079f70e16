// Attention of a few new tokens per sequence (one, as a rule) over the paged INT8 cache, head_dim 64 / 96 / 128.
//
// Bound: the cache, 2 * head_dim + 8 bytes a position and kv head.  Both products are mma.m16n8k32 of int8 with 32-bit
// integer sums, so that the codes go from memory to the tensor cores as they are (a conversion to bf16 costs 3 instructions
// per pair of codes, which bounds attention_mma_kernel at 2.9 TB/s).  The other operand is cut into two int8 digits,
// x = s * (256 hi + lo) with |256 hi + lo| <= 32512: q by its row's largest element, a weight times its value's scale by
// the largest such product of its 32 positions.  The integer sums are exact and 256 hi + lo is put together before it is a float.
//   rows      of one kv head: (new token, query head), eight to an MMA: row g holds the high digits, row g + 8 the low ones
//   chunk     32 positions of a warp, K and V straight from global memory into registers as the B operands; the next
//             chunk's loads are issued as soon as this one's registers are free
//   softmax   each chunk has a maximum of its own, its sums join the running ones by powers of two
//   positions column n of QK tile u is position 4 n + u, so that a lane's scores are of eight consecutive positions: they
//             are the A operand of the second product as they lie, against V's rows in order
//   dims      column n of PV tile j is dim n * head_dim / 8 + j: a lane reads consecutive bytes of each of eight rows
//             and turns them by byte permutes
// 24 sequences of 2-4 k positions (32/8 heads of 128) take 38.2 us (4.2 TB/s), 256 of 70-320 30.6 us (3.6 TB/s), two of 65 521
// with one kv head 20.4 us, one of 256 5.2 us.
// Work is cut by the device, which alone knows the lengths: the positions of a (sequence, kv head, rows) item go in equal
// parts to teams of warps, as many as are resident together (dec_part_units).  The parts of an item leave their results in
// the workspace; of 16 neighbouring parts the team that comes last adds them in order, and of these sums the last again, so
// that the result does not depend on who came when.
#include "paged.cuh"
#include <algorithm>
#include <atomic>

namespace s12 {

constexpr int kDecWarps = 4;
constexpr int kDecThreads = kDecWarps * 32;
constexpr int kDecChunk = 32;                       // positions of a warp's step
constexpr int kDecCtasPerSm = 3;                    // resident with 8 rows; 2 with 16
__host__ __device__ constexpr int dec_ctas_per_sm(int tiles) { return tiles == 1 ? kDecCtasPerSm : 2; }
constexpr int kDecMaxRows = 16, kDecMaxDim = 128;
constexpr int kDecMostRows = 1024;                  // of a sequence and kv head: in groups of 16
constexpr int kDecGroup = 16;                       // parts that are added up together
constexpr float kDigits = 32512.f;                  // 127 * 256: the high digit stays below 128
constexpr float kDecLowest = -3e38f;                // a maximum of no scores
// a partial result: [rows][head_dim], then [rows][max, sum], then the same of a group that begins with this part
__host__ __device__ constexpr int64_t dec_slot_floats(int rows) { return (int64_t)rows * (kDecMaxDim + 4); }

struct DecodeParams {
    PagedAttn a;
    float* slots;               // [parts of cut items] partial results
    unsigned int* groups_done;  // [parts of cut items] parts of a group that are there, zero between calls
    unsigned int* items_done;   // [items] groups of an item that are there, zero between calls
    int row_groups;             // groups of rows of a kv head
    int min_units;              // units of a part, at least
    int whole;                  // no item is cut, whatever its length: a team's item follows from its number
    int teams;                  // that are resident together
    uint32_t gqa_mul;           // ceil(2^20 / query heads of a kv head): x / that for x below 2^10
};

__host__ __device__ constexpr int dec_row_floats(int hd) { return hd + hd / 8; }   // padded: the lanes of a store meet different banks
__device__ __forceinline__ int dec_pad(int d) { return d + (d >> 5) * 4; }

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float dec_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// kDigits / top; both quartered, since __fdividef gives 0 for divisors above 2^126
__device__ __forceinline__ float dec_digits_over(float top) { return __fdividef(kDigits / 4, top * 0.25f); }

// kHD codes of a K row that a lane needs: kHD / 4 consecutive bytes of every 64 (or 32) go to its quad's lanes
template <int kHD> struct KRow { uint32_t w[kHD / 16]; };
template <int kHD>
__device__ __forceinline__ void load_k(KRow<kHD>& r, const int8_t* row, int t4)
{
    if (kHD % 64 == 0) {
#pragma unroll
        for (int j = 0; j < kHD / 64; j++) {
            const uint4 x = *reinterpret_cast<const uint4*>(row + 64 * j + 16 * t4);
            r.w[4 * j] = x.x; r.w[4 * j + 1] = x.y; r.w[4 * j + 2] = x.z; r.w[4 * j + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < kHD / 32; j++) {
            const uint2 x = *reinterpret_cast<const uint2*>(row + 32 * j + 8 * t4);
            r.w[2 * j] = x.x; r.w[2 * j + 1] = x.y;
        }
    }
}
// first dim of the eight that MMA step s takes from lane t4
template <int kHD> __device__ __forceinline__ int k_dim(int s, int t4) { return kHD % 64 == 0 ? 64 * (s >> 1) + 16 * t4 + 8 * (s & 1) : 32 * s + 8 * t4; }
template <int kHD> struct VRow { uint32_t w[kHD / 32]; };
template <int kHD>
__device__ __forceinline__ void load_v(VRow<kHD>& r, const int8_t* row, int g)
{
    if (kHD == 128) {
        const uint4 x = *reinterpret_cast<const uint4*>(row + 16 * g);
        r.w[0] = x.x; r.w[1] = x.y; r.w[kHD / 32 - 2] = x.z; r.w[kHD / 32 - 1] = x.w;
    } else if (kHD == 64) {
        const uint2 x = *reinterpret_cast<const uint2*>(row + 8 * g);
        r.w[0] = x.x; r.w[1] = x.y;
    } else {
#pragma unroll
        for (int j = 0; j < kHD / 32; j++) r.w[j] = *reinterpret_cast<const uint32_t*>(row + kHD / 8 * g + 4 * j);
    }
}


// floor(n / d): 64-bit divisions take long
__device__ __forceinline__ unsigned long long div_small(unsigned long long n, uint32_t d) { return n >> 32 ? n / d : (uint32_t)n / d; }
// f(the units of sequence s: its steps of `unit` positions, at least one) for s from first to end - 1, the lengths of many four at a time: each CTA looks at them all (1000
// sequences of 320 positions, 2 kv heads of 64, teams of four: 103 -> 52 us)
template <class F> __device__ __forceinline__ void dec_each(const PagedArgs& C, int first, int end, int unit, F f)
{
    const int room = (int)min((long long)C.table_pages << C.page_shift, (long long)C.max_len);
    auto one = [&](int n) { n = min(n, room); f(n <= 0 ? 1u : (uint32_t)(n + unit - 1) / (uint32_t)unit); };
    if (C.num_seqs <= 32) { if (first < end) one(C.kv_len[first]); return; }      // one to a lane
    const bool wide = ((reinterpret_cast<uintptr_t>(C.kv_len) | first * 4u) & 15) == 0;
    int s = first;
    if (wide)
#pragma unroll 2
        for (; s + 4 <= end; s += 4) { const int4 n = *reinterpret_cast<const int4*>(C.kv_len + s); one(n.x); one(n.y); one(n.z); one(n.w); }
    for (; s < end; s++) one(C.kv_len[s]);
}
// The most units of a part: the least that gives all items' parts to resident teams.  With so many items that this would
// cut nothing or nearly nothing, twice a team's share: only what is far longer than the others is cut (cutting all of 2400
// items so that they fill two rounds of teams measured the same).  At least min_units, and a 128th of the longest item:
// adding up more parts takes longer than they save.  For a whole warp; a lane looks at `per_lane` neighbouring sequences.
__device__ __forceinline__ uint32_t dec_part_units(const DecodeParams& P, int unit, int per_seq, int per_lane)
{
    const PagedArgs& C = P.a.c;
    const int first = (threadIdx.x & 31) * per_lane, end = min(first + per_lane, C.num_seqs);
    uint32_t n = 0, top = 0;
    dec_each(C, first, end, unit, [&](uint32_t u) { n += u; top = max(top, u); });
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    const unsigned long long total = (unsigned long long)__reduce_add_sync(0xFFFFFFFFu, n) * (unsigned long long)per_seq;
    const unsigned long long items = (unsigned long long)C.num_seqs * per_seq, share = div_small(total, P.teams) + 1;
    const uint32_t least = max((uint32_t)P.min_units, (top + 127) >> 7);
    if (2 * items > P.teams) return max((uint32_t)min(2 * share, 0x7FFFFFFFull), least);
    uint32_t lo = max((uint32_t)share, least), hi = max((uint32_t)div_small(total, P.teams - (uint32_t)items) + 1, lo);   // hi is enough: total / hi + items <= teams
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        uint32_t parts = 0;
        dec_each(C, first, end, unit, [&](uint32_t u) { parts += (u + mid - 1) / mid; });
        if ((unsigned long long)__reduce_add_sync(0xFFFFFFFFu, parts) * (unsigned long long)per_seq <= (unsigned long long)P.teams) hi = mid; else lo = mid + 1;
    }
    return lo;
}

// four values over their sum as bf16
__device__ __forceinline__ uint2 dec_bf16x4(const float4& n, float rd)
{
    uint32_t lo, hi;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(n.y * rd), "f"(n.x * rd));
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(n.w * rd), "f"(n.z * rd));
    return make_uint2(lo, hi);
}
__device__ __forceinline__ float dec_over(float den) { return den == 0.f ? 0.f : 1.f / den; }   // no position at all: zeros
__device__ __forceinline__ void dec_store4(int16_t* o, const float4& n, float rd, bool aligned)
{
    const uint2 y = dec_bf16x4(n, rd);
    if (aligned) *reinterpret_cast<uint2*>(o) = y;
    else { o[0] = (int16_t)y.x; o[1] = (int16_t)(y.x >> 16); o[2] = (int16_t)y.y; o[3] = (int16_t)(y.y >> 16); }
}

// A team is one warp (many short items: nothing waits for another warp; an item is one team's) or the CTA (long ones, cut).
template <int kHD, int kTiles, int kTeam>
__global__ void __launch_bounds__(kDecThreads, dec_ctas_per_sm(kTiles))
paged_decode_kernel(const __grid_constant__ DecodeParams P)
{
    constexpr int kRows = 8 * kTiles, kSteps = kHD / 32, kCols = kHD / 8, kUnit = kTeam * kDecChunk, kRow = dec_row_floats(kHD);
    constexpr int64_t kSlot = dec_slot_floats(kRows);
    constexpr int kTeamThreads = kTeam * 32;
    struct Digits { int8_t d[2][kRows][kHD + 16]; };               // padded: the lanes of a load meet different banks
    union WarpRoom { Digits q; float acc[kTeam > 1 ? kRows * kRow : 4]; };   // q as digits, then the warp's sums
    __shared__ __align__(16) WarpRoom room_s[kDecWarps];
    __shared__ float m_s[kTeam][kRows], l_s[kTeam][kRows];
    __shared__ int last_s;
    grid_launch_dependents();
    grid_dependency_wait();
    const PagedArgs& C = P.a.c;
    // warp: the same in all lanes, for the compiler to see (256 sequences of 70-320 positions 33.9 -> 30.6 us)
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), g = lane >> 2, t4 = lane & 3;
    const int team = blockIdx.x * (kDecWarps / kTeam) + warp / kTeam, tw = warp % kTeam, tt = threadIdx.x % kTeamThreads;
    const int gqa = P.a.n_head / C.n_head_kv, per_seq = C.n_head_kv * P.row_groups;

    // ---- this team's part: part `part` of `parts` of item `item` of sequence seq; slot0: the item's first slot
    int seq = -1, parts = 0, slot0 = 0;
    uint32_t units = 0, left = team;
    if (kTeam == 1 || P.whole) {
        if (team < C.num_seqs * per_seq) { seq = team / per_seq; left = team - seq * per_seq; parts = 1; }
    } else {
        const int per_lane = C.num_seqs > 32 ? (C.num_seqs + 127) >> 7 << 2 : 1;   // fours of lengths
        const uint32_t most = dec_part_units(P, kUnit, per_seq, per_lane);
        // left: teams of the sequences from here on that come before this one
        // the lane whose sequences hold the team, then the sequence: two scans, each of (teams, slots) of a lane's sequences
        for (int s0 = 0, per = per_lane, n_seqs = C.num_seqs; ; ) {
            uint32_t n = 0, cut = 0, u = 0, parts_of = 0;
            dec_each(C, s0 + lane * per, min(s0 + (lane + 1) * per, n_seqs), kUnit, [&](uint32_t units_of) {
                u = units_of;
                parts_of = (u + most - 1) / most;
                n += parts_of; cut += parts_of > 1 ? parts_of : 0;
            });
            unsigned long long mine = (unsigned long long)(n * per_seq) | (unsigned long long)(cut * per_seq) << 32, upto = mine;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const unsigned long long o = __shfl_up_sync(0xFFFFFFFFu, upto, off);
                if (lane >= off) upto += o;
            }
            const unsigned over = __ballot_sync(0xFFFFFFFFu, (uint32_t)upto > left);
            const int l = over ? __ffs(over) - 1 : 31;
            const unsigned long long before = __shfl_sync(0xFFFFFFFFu, over ? upto - mine : upto, l);
            if (over || per == 1) { left -= (uint32_t)before; slot0 += (int)(before >> 32); }
            if (per == 1) {
                if (over) { seq = s0 + l; units = __shfl_sync(0xFFFFFFFFu, u, l); parts = (int)__shfl_sync(0xFFFFFFFFu, parts_of, l); break; }
                s0 += 32;
                if (s0 >= n_seqs) break;
                continue;
            }
            if (!over) break;
            s0 += l * per;
            n_seqs = min(s0 + per, n_seqs);
            per = 1;
        }
    }
    if (seq < 0) return;                                           // more teams than parts
    const int item = (int)(left / (uint32_t)parts), part = (int)left - item * parts;
    if (parts > 1) slot0 += item * parts;
    auto token_of = [&](int row) { return (int)((uint32_t)row * P.gqa_mul >> 20); };
    const float to_log2 = P.a.scale * 1.4426950408889634f;
    const int ps = 1 << C.page_shift;
    const bool out_aligned = ((reinterpret_cast<uintptr_t>(P.a.out) & 7) | (P.a.out_stride & 3)) == 0;
    const bool q_aligned = ((reinterpret_cast<uintptr_t>(P.a.q) & 15) | (P.a.q_stride & 3)) == 0;
    {
        const int kvh = item / P.row_groups, row_base = (item - kvh * P.row_groups) * kRows;
        int lo, hi;
        paged_rows(C, seq, lo, hi);
        const int rows = min(kRows, (hi - lo) * gqa - row_base);   // rows of this item; 0 or less: none
        if (rows > 0) {
            const int t_lo = kTeam == 1 || P.whole ? 0 : (int)((unsigned long long)units * part / parts) * kUnit;
            // the first chunks' pages are asked for before the lengths are there
            const int kt = (g >> 2) * 16, vt = (t4 >> 1) * 16;
            const int* table = C.table + (size_t)seq * C.table_stride;
            auto entry_at = [&](int t) { return (t >> C.page_shift) < C.table_pages ? table[t >> C.page_shift] : -1; };
            int t0 = t_lo + tw * kDecChunk;
            const int entry[4] = {entry_at(t0 + kt), entry_at(t0 + vt), entry_at(t0 + kUnit + kt), entry_at(t0 + kUnit + vt)};
            const int room = paged_len(C, seq), before = C.kv_len[seq] - (hi - lo) + 1;   // row r sees min(before + token, room) positions
            const int least = min(before + token_of(row_base), room), most_seen = min(before + token_of(row_base + rows - 1), room);
            const int t_hi = kTeam == 1 || P.whole ? most_seen : (int)min((long long)((unsigned long long)units * (part + 1) / parts) * kUnit, (long long)most_seen);
            bool missing = paged_past_table(C, before + token_of(row_base + rows - 1));
            // the page of position t, whose table entry was read; -1: none, or t not below t_hi
            auto page_of = [&](int entry, int t) {
                if (t >= t_hi) return -1;
                if ((unsigned)entry < (unsigned)C.num_pages) return entry;
                missing = true;
                return -1;
            };
            auto entry_in = [&](int t) { return t < t_hi ? entry_at(t) : -1; };
            // row of the pools' arrays (2^32 rows are more than a GPU holds); absent pages read page 0, masked later
            auto row_at = [&](int page, int t) { return (((uint32_t)max(page, 0) * C.n_head_kv + kvh) << C.page_shift) + (t & (ps - 1)); };
            KRow<kHD> k[4];
            VRow<kHD> v[8];
            float4 sk[2], sv[2];
            auto fetch_k = [&](int t0, int page) {
                const int8_t* row = C.k + (size_t)row_at(page, t0 + 4 * g) * kHD;
#pragma unroll
                for (int u = 0; u < 4; u++) load_k<kHD>(k[u], row + u * kHD, t4);
            };
            auto fetch_v = [&](uint32_t at) {
                const int8_t* row = C.v + (size_t)at * kHD;
#pragma unroll
                for (int u = 0; u < 8; u++) load_v<kHD>(v[u], row + u * kHD, g);
            };
            auto fetch_s = [&](float4 (&s)[2], const float* scales, uint32_t at) {
                s[0] = *reinterpret_cast<const float4*>(scales + at); s[1] = *reinterpret_cast<const float4*>(scales + at + 4);
            };
            // a chunk has one page, or two of 16 positions: K rows 4 g + u lie in the half of g >> 2, V rows 8 t4 + u of t4 >> 1
            int pk = page_of(entry[0], t0 + kt), pv = page_of(entry[1], t0 + vt), pk_next = page_of(entry[2], t0 + kUnit + kt), pv_next = page_of(entry[3], t0 + kUnit + vt);
            int entry_k = entry_in(t0 + 2 * kUnit + kt), entry_v = entry_in(t0 + 2 * kUnit + vt);   // one chunk further
            float4 qv[kRows];                                      // lane: dims 4 lane .. + 3 of every row
#pragma unroll
            for (int r = 0; r < kRows; r++) {
                qv[r] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (r < rows && 4 * lane < kHD) {
                    const int tok = token_of(row_base + r), head = row_base + r - tok * gqa;
                    const float* q = P.a.q + (size_t)(lo + tok) * P.a.q_stride + (size_t)(kvh * gqa + head) * kHD + 4 * lane;
                    if (q_aligned) qv[r] = *reinterpret_cast<const float4*>(q);
                    else qv[r] = make_float4(q[0], q[1], q[2], q[3]);
                }
            }
            if (t0 < t_hi) {
                const uint32_t at = row_at(pv, t0 + 8 * t4);
                fetch_k(t0, pk); fetch_s(sk, C.sk, at); fetch_s(sv, C.sv, at); fetch_v(at);
            }
            // ---- q as digits, every warp for itself
            uint32_t qa[kTiles][kSteps][4];
            float factor[kTiles];
            int limit[kTiles];                                     // positions that the lane's row may see
#pragma unroll
            for (int i = 0; i < kTiles; i++) factor[i] = 0.f;
            auto& digits = room_s[warp].q.d;
#pragma unroll
            for (int r = 0; r < kRows; r++) {
                if (r >= rows) break;
                const float e[4] = {qv[r].x, qv[r].y, qv[r].z, qv[r].w};
                uint32_t bits = 0;                                 // of the largest magnitude; a NaN is the largest
#pragma unroll
                for (int j = 0; j < 4; j++) bits = max(bits, __float_as_uint(e[j]) & 0x7FFFFFFFu);
                bits = __reduce_max_sync(0xFFFFFFFFu, bits);
                const float top = __uint_as_float(bits);
                const bool fine = top >= 1e-30f && bits < 0x7F800000u;   // rows of smaller ones count as zero
                const float inv = fine ? dec_digits_over(top) : 0.f;
                uint32_t y[4];
#pragma unroll
                for (int j = 0; j < 4; j++) y[j] = __float_as_uint(fmaf(fine ? e[j] : 0.f, inv, 12582912.f + 128.f));   // 256 hi + lo + 128
                const uint32_t p01 = prmt(y[0], y[1], 0x5140u), p23 = prmt(y[2], y[3], 0x5140u);
                if (4 * lane < kHD) {
                    *reinterpret_cast<uint32_t*>(&digits[0][r][4 * lane]) = prmt(p01, p23, 0x7632u);
                    *reinterpret_cast<uint32_t*>(&digits[1][r][4 * lane]) = prmt(p01, p23, 0x5410u) ^ 0x80808080u;
                }
                if ((r & 7) == g) factor[r >> 3] = bits >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : top * (1.f / kDigits) * to_log2;
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kTiles; i++) {
                const int r = i * 8 + g;
                const bool there = r < rows;
#pragma unroll
                for (int s = 0; s < kSteps; s++) {
                    const uint2 h = *reinterpret_cast<const uint2*>(&digits[0][r][k_dim<kHD>(s, t4)]);
                    const uint2 l = *reinterpret_cast<const uint2*>(&digits[1][r][k_dim<kHD>(s, t4)]);
                    qa[i][s][0] = there ? h.x : 0u; qa[i][s][1] = there ? l.x : 0u; qa[i][s][2] = there ? h.y : 0u; qa[i][s][3] = there ? l.y : 0u;
                }
                limit[i] = there ? min(before + token_of(row_base + r), room) : 0;
            }
            float acc[kTiles][kCols][2], m[kTiles], l[kTiles];
#pragma unroll
            for (int i = 0; i < kTiles; i++) {
                m[i] = kDecLowest; l[i] = 0.f;
#pragma unroll
                for (int j = 0; j < kCols; j++) acc[i][j][0] = acc[i][j][1] = 0.f;
            }
#pragma unroll 1
            for (; t0 < t_hi; t0 += kUnit) {
                const bool more = t0 + kUnit < t_hi;
                // Long items: the codes of the chunk after the next, 2 KB that lie together from each of four lanes, on their way
                // to L2 (24 sequences of 2-4 k positions 40.1 -> 38.4 us; 256 short ones, where a warp has six chunks, 33.5 -> 35.8)
                if (kTeam > 1 && t0 + 2 * kUnit + 16 < t_hi) {
                    auto ask = [&](const int8_t* codes, int entry, int t) {
                        if ((unsigned)entry < (unsigned)C.num_pages)
                            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(codes + (size_t)row_at(entry, t) * kHD), "r"(16 * kHD) : "memory");
                    };
                    if ((lane & 15) == 0) ask(C.k, entry_k, t0 + 2 * kUnit + kt);
                    if ((lane & ~2) == 0) ask(C.v, entry_v, t0 + 2 * kUnit + vt);
                }
                const uint32_t at_next = row_at(pv_next, t0 + kUnit + 8 * t4);
                // ---- scores, in powers of two: s[p] of position t0 + 8 t4 + p
                float s[kTiles][8];
                {
                    int c[kTiles][4][4];
#pragma unroll
                    for (int i = 0; i < kTiles; i++)
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            c[i][u][0] = c[i][u][1] = c[i][u][2] = c[i][u][3] = 0;
#pragma unroll
                            for (int st = 0; st < kSteps; st++)
                                mma_s8(c[i][u], qa[i][st][0], qa[i][st][1], qa[i][st][2], qa[i][st][3], k[u].w[2 * st], k[u].w[2 * st + 1]);
                        }
                    if (more) fetch_k(t0 + kUnit, pk_next);
                    const float skv[8] = {sk[0].x, sk[0].y, sk[0].z, sk[0].w, sk[1].x, sk[1].y, sk[1].z, sk[1].w};
#pragma unroll
                    for (int i = 0; i < kTiles; i++)
#pragma unroll
                        for (int e = 0; e < 2; e++)
#pragma unroll
                            for (int u = 0; u < 4; u++) s[i][4 * e + u] = (float)(256 * c[i][u][e] + c[i][u][2 + e]) * (skv[4 * e + u] * factor[i]);
                }
                if (more) fetch_s(sk, C.sk, at_next);
                const float svv[8] = {sv[0].x, sv[0].y, sv[0].z, sv[0].w, sv[1].x, sv[1].y, sv[1].z, sv[1].w};
                float odd = 0.f;                                    // NaN where a value's scale is not finite
#pragma unroll
                for (int p = 0; p < 8; p++) odd = fmaf(svv[p], 0.f, odd);
                const bool plain = __all_sync(0xFFFFFFFFu, odd == 0.f && pv >= 0 && t0 + kDecChunk <= least);
                // ---- weights: of the chunk's own maximum, times the values' scales, as two digits of the largest such product
                uint32_t pa[kTiles][4];
                float gain[kTiles];
#pragma unroll
                for (int i = 0; i < kTiles; i++) {
                    if (!plain) {
#pragma unroll
                        for (int p = 0; p < 8; p++) if (pv < 0 || t0 + 8 * t4 + p >= limit[i]) s[i][p] = -INFINITY;
                    }
                    float mx = kDecLowest;
#pragma unroll
                    for (int p = 0; p < 8; p++) mx = fmaxf(mx, s[i][p]);
                    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
                    float sum = 0.f, top = 0.f, z[8];
                    if (plain) {
#pragma unroll
                        for (int p = 0; p < 8; p++) {
                            const float w = dec_exp2(s[i][p] - mx);
                            z[p] = w * svv[p];
                            sum += w;
                            top = fmaxf(top, fabsf(z[p]));
                        }
                    } else {
#pragma unroll
                        for (int p = 0; p < 8; p++) {
                            const float w = dec_exp2(s[i][p] - mx);
                            const bool masked = s[i][p] == -INFINITY;
                            z[p] = masked ? 0.f : w * svv[p];
                            sum += masked ? 0.f : fmaf(svv[p], 0.f, w);   // a scale that is not finite marks the rows that use it
                            if (!(fabsf(z[p]) < INFINITY)) z[p] = 0.f;
                            top = fmaxf(top, fabsf(z[p]));
                        }
                    }
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                    const float inv = top >= 1e-30f ? dec_digits_over(top) : 0.f;
                    uint32_t y[8];                                  // 256 hi + lo + 128 in the low half
#pragma unroll
                    for (int p = 0; p < 8; p++) y[p] = __float_as_uint(fmaf(z[p], inv, 12582912.f + 128.f));
                    const float mn = fmaxf(m[i], mx), f = dec_exp2(m[i] - mn), fc = dec_exp2(mx - mn);
                    gain[i] = fc * (top * (1.f / kDigits));
                    l[i] = l[i] * f + sum * fc;
                    if (__any_sync(0xFFFFFFFFu, f != 1.f)) {
#pragma unroll
                        for (int j = 0; j < kCols; j++) { acc[i][j][0] *= f; acc[i][j][1] *= f; }
                    }
                    m[i] = mn;
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const uint32_t p01 = prmt(y[4 * e], y[4 * e + 1], 0x5140u), p23 = prmt(y[4 * e + 2], y[4 * e + 3], 0x5140u);
                        pa[i][2 * e] = prmt(p01, p23, 0x7632u);
                        pa[i][2 * e + 1] = prmt(p01, p23, 0x5410u) ^ 0x80808080u;
                    }
                }
                if (more) fetch_s(sv, C.sv, at_next);
                // ---- weighted values
#pragma unroll
                for (int w = 0; w < kHD / 32; w++) {
                    uint32_t b[2][4];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const uint32_t x0 = prmt(v[4 * e].w[w], v[4 * e + 1].w[w], 0x5140u), x1 = prmt(v[4 * e + 2].w[w], v[4 * e + 3].w[w], 0x5140u);
                        const uint32_t x2 = prmt(v[4 * e].w[w], v[4 * e + 1].w[w], 0x7362u), x3 = prmt(v[4 * e + 2].w[w], v[4 * e + 3].w[w], 0x7362u);
                        b[e][0] = prmt(x0, x1, 0x5410u); b[e][1] = prmt(x0, x1, 0x7632u);
                        b[e][2] = prmt(x2, x3, 0x5410u); b[e][3] = prmt(x2, x3, 0x7632u);
                    }
#pragma unroll
                    for (int d = 0; d < 4; d++)
#pragma unroll
                        for (int i = 0; i < kTiles; i++) {
                            int o[4] = {0, 0, 0, 0};
                            mma_s8(o, pa[i][0], pa[i][1], pa[i][2], pa[i][3], b[0][d], b[1][d]);
#pragma unroll
                            for (int e = 0; e < 2; e++) acc[i][4 * w + d][e] = fmaf((float)(256 * o[e] + o[2 + e]), gain[i], acc[i][4 * w + d][e]);
                        }
                }
                if (more) fetch_v(at_next);
                pk = pk_next; pv = pv_next;
                pk_next = page_of(entry_k, t0 + 2 * kUnit + kt); pv_next = page_of(entry_v, t0 + 2 * kUnit + vt);
                entry_k = entry_in(t0 + 3 * kUnit + kt); entry_v = entry_in(t0 + 3 * kUnit + vt);
            }
            if (missing) atomicOr(C.status, kStatusPage);
            // ---- the team's sums: thread tt has elements 4 (tt + n * threads) of the rows.  A warp alone: its own.
#pragma unroll
            for (int i = 0; i < kTiles; i++) {
                l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 1);
                l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 2);
            }
            const bool alone = kTeam == 1 || parts == 1;
            auto out_at = [&](int r, int d) {
                const int tok = token_of(row_base + r), head = row_base + r - tok * gqa;
                return P.a.out + (size_t)(lo + tok) * P.a.out_stride + (size_t)(kvh * gqa + head) * kHD + d;
            };
            float* mine = P.slots + (size_t)(slot0 + part) * kSlot;
            if (kTeam == 1) {
#pragma unroll
                for (int i = 0; i < kTiles; i++) {
                    const int r = i * 8 + g;
                    if (r >= rows) continue;
                    const float rd = dec_over(l[i]);
                    int16_t* o = out_at(r, 0);
#pragma unroll
                    for (int e = 0; e < 2; e++)
#pragma unroll
                        for (int j = 0; j < kCols; j += 4) {
                            const float4 n = make_float4(acc[i][j][e], acc[i][j + 1][e], acc[i][j + 2][e], acc[i][j + 3][e]);
                            const int d = (2 * t4 + e) * kCols + j;
                            dec_store4(o + d, n, rd, out_aligned);
                        }
                }
            } else {
                __syncwarp();                                      // this warp's digits have been read
#pragma unroll
                for (int i = 0; i < kTiles; i++) {
                    const int r = i * 8 + g;
                    if (t4 == 0) { m_s[tw][r] = m[i]; l_s[tw][r] = l[i]; }
#pragma unroll
                    for (int e = 0; e < 2; e++)
#pragma unroll
                        for (int j = 0; j < kCols; j += 4)
                            *reinterpret_cast<float4*>(&room_s[tw].acc[r * kRow + dec_pad((2 * t4 + e) * kCols + j)]) =
                                make_float4(acc[i][j][e], acc[i][j + 1][e], acc[i][j + 2][e], acc[i][j + 3][e]);
                }
                __syncthreads();
                for (int i = tt; i < rows * (kHD / 4); i += kTeamThreads) {
                    const int r = i / (kHD / 4), d = (i - r * (kHD / 4)) * 4;
                    float mm = kDecLowest, den = 0.f;
                    float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < kTeam; w++) mm = fmaxf(mm, m_s[w][r]);
#pragma unroll
                    for (int w = 0; w < kTeam; w++) {
                        const float f = dec_exp2(m_s[w][r] - mm);
                        const float4 y = *reinterpret_cast<const float4*>(&room_s[w].acc[r * kRow + dec_pad(d)]);
                        num.x += f * y.x; num.y += f * y.y; num.z += f * y.z; num.w += f * y.w;
                        den += f * l_s[w][r];
                    }
                    if (alone) { dec_store4(out_at(r, d), num, dec_over(den), out_aligned); continue; }
                    *reinterpret_cast<float4*>(mine + r * kHD + d) = num;
                    if (d == 0) { mine[kRows * kHD + 2 * r] = mm; mine[kRows * kHD + 2 * r + 1] = den; }
                }
            }
            if (kTeam > 1 && !alone) {
                const int ngroups = (parts + kDecGroup - 1) / kDecGroup;
                // true in the team that is the last of `n` to come
                auto last_of = [&](unsigned int* counter, int n) {
                    __syncthreads();
                    if (tt == 0) {
                        __threadfence();                            // with the barrier before it: all the team's writes
                        last_s = atomicAdd(counter, 1u) == (unsigned)n - 1;
                        if (last_s) *counter = 0;
                    }
                    __syncthreads();
                    __threadfence();
                    return last_s != 0;
                };
                // adds n parts, or sums of groups (stats: where their statistics lie): to the output, or over the first one
                auto add_up = [&](int first, int step, int n, int stats, bool finish) {
                    for (int i = tt; i < rows * (kHD / 4); i += kTeamThreads) {
                        const int r = i / (kHD / 4), d = (i - r * (kHD / 4)) * 4;
                        float mm = kDecLowest, den = 0.f;
                        float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
                        for (int j = 0; j < n; j++) {
                            const float* p = P.slots + (size_t)(slot0 + first + j * step) * kSlot;
                            const float2 ml = __ldcg(reinterpret_cast<const float2*>(p + kRows * kHD + stats + 2 * r));
                            const float4 y = __ldcg(reinterpret_cast<const float4*>(p + r * kHD + d));
                            const float mn = fmaxf(mm, ml.x), f0 = dec_exp2(mm - mn), f = dec_exp2(ml.x - mn);
                            num.x = num.x * f0 + f * y.x; num.y = num.y * f0 + f * y.y; num.z = num.z * f0 + f * y.z; num.w = num.w * f0 + f * y.w;
                            den = den * f0 + f * ml.y;
                            mm = mn;
                        }
                        if (finish) { dec_store4(out_at(r, d), num, dec_over(den), out_aligned); continue; }
                        float* p = P.slots + (size_t)(slot0 + first) * kSlot;
                        *reinterpret_cast<float4*>(p + r * kHD + d) = num;      // read by this thread alone; the statistics by all of the row
                        if (d == 0) *reinterpret_cast<float2*>(p + kRows * kHD + 2 * kRows + 2 * r) = make_float2(mm, den);
                    }
                };
                const int group = part / kDecGroup, n_in = min(kDecGroup, parts - group * kDecGroup);
                if (last_of(P.groups_done + slot0 + group * kDecGroup, n_in)) {
                    add_up(group * kDecGroup, 1, n_in, 0, ngroups == 1);
                    if (ngroups > 1 && last_of(P.items_done + (size_t)seq * per_seq + item, ngroups)) add_up(0, kDecGroup, ngroups, 2 * kRows, true);
                }
            }
        }
    }
}

// The workspace: partial results, then the counters; the same places for every call on a device.  The parts of cut items
// are at most 2 * teams: an item of u units has at most 2 u / (units of a part).
static int64_t dec_teams() { return (int64_t)sm_count() * kDecCtasPerSm; }   // of four warps, resident together
static int64_t dec_slot_bytes() { return 2 * dec_teams() * dec_slot_floats(kDecMaxRows) * 4; }
static int64_t dec_group_bytes() { return 2 * dec_teams() * 4; }
int64_t paged_decode_workspace_bytes(int n_head, int n_head_kv, int num_seqs, int max_new)
{
    const long long rows = std::min((long long)(n_head / n_head_kv) * max_new, (long long)kDecMostRows);   // enough for fewer, too
    return dec_slot_bytes() + dec_group_bytes() + (int64_t)num_seqs * n_head_kv * ((rows + 7) / 8) * 4;
}

template <int kHD, int kTiles, int kTeam>
static int decode_launch(DecodeParams P, void* stream, const char* who)
{
    P.whole = kTeam == 1 || P.a.c.max_len <= kTeam * kDecChunk * P.min_units;
    // at most, by the caller's bounds: every item whole, and what cutting adds; a grid for less than all resident teams
    P.teams = (int)dec_teams() * dec_ctas_per_sm(kTiles) / kDecCtasPerSm;
    const long long items = (long long)P.a.c.num_seqs * P.a.c.n_head_kv * P.row_groups;
    const long long parts = (P.a.c.max_len + (long long)kTeam * kDecChunk * P.min_units - 1) / ((long long)kTeam * kDecChunk * P.min_units);
    const long long grid = ((P.whole ? items : std::min(items * parts, items + P.teams)) * kTeam + kDecWarps - 1) / kDecWarps;
    if (grid > 0x7FFFFFFF || items > 1 << 30) return fail(S12_ERR_TOO_LARGE, "%s: %lld sequences' heads", who, items);
    return launch(paged_decode_kernel<kHD, kTiles, kTeam>, dim3((unsigned)grid), dim3(kDecThreads), 0, stream, who, P);
}
template <int kHD>
static int decode_launch_hd(DecodeParams P, int tiles, void* stream, const char* who)
{
    const PagedAttn& A = P.a;
    const long long items = (long long)A.c.num_seqs * A.c.n_head_kv * P.row_groups;
    P.min_units = std::max(1, env_knob("S12_PAGED_MIN_UNITS", 2));
    if (tiles == 2) return decode_launch<kHD, 2, kDecWarps>(P, stream, who);
    // us with one / four warps, sequences of half of these lengths to all: 8 kv heads of 128, 64 sequences of 128 positions
    // 8.0 / 9.4, 320 15.8 / 15.6, 500 27.6 / 21.8; 256 of 500 57 / 60, 700 81 / 73; 800 of 900 237 / 255; 2 kv heads of 64, 100
    // sequences of 128 6.2 / 5.4, 256 of 500 13.6 / 17.1, 1000 of 900 59 / 76, 1500 95 / 102
    const int team = env_knob("S12_PAGED_TEAM", 0);                // 1, 4: whatever the rule says
    if (team == 1 || (team == 0 && (long long)kHD * A.c.max_len <= std::min(40 * items, 131072ll))) return decode_launch<kHD, 1, 1>(P, stream, who);
    return decode_launch<kHD, 1, kDecWarps>(P, stream, who);
}

// 1: not a shape of this kernel
int paged_decode_launch(const PagedAttn& A, void* stream, const char* who)
{
    const int hd = A.c.head_dim, gqa = A.n_head / A.c.n_head_kv;
    const long long rows = (long long)gqa * A.max_new;
    if ((hd != 64 && hd != 96 && hd != 128) || rows > kDecMostRows) return 1;
    // Groups of 16 rows read the cache anew, 256 rows of the other kernel share it, but without cutting the positions: this one
    // while all groups are resident together.  us here / there, 32/8 heads of 128: 128 tokens (256 groups) 9.1 / 11.5, 200 (400)
    // 17.7 / 13.0, 128 behind 8000 77.5 / 82.6, 256 (512) behind 8000 211 / 117, 4 x 32 (256) behind 6000 100 / 106, 16 x 16 (512)
    // behind 6000 189 / 123; and always with two groups to a sequence or one: 64 sequences of 8000, 32 rows, 552 / 589.
    const long long groups16 = (rows + 15) / 16 * A.c.num_seqs * A.c.n_head_kv;
    const int force = env_knob("S12_PAGED_FORCE", 0);              // 1: here, 2: there
    if (force == 2 || (force == 0 && rows > 32 && groups16 > (long long)dec_ctas_per_sm(2) * sm_count())) return 1;
    const int64_t need = paged_decode_workspace_bytes(A.n_head, A.c.n_head_kv, A.c.num_seqs, A.max_new);
    if (!A.workspace || A.workspace_bytes < need || (reinterpret_cast<uintptr_t>(A.workspace) & 15))
        return fail(S12_ERR_BAD_ARG, "%s: needs a 16-byte aligned workspace of %lld bytes", who, (long long)need);
    DecodeParams P = {};
    P.a = A;
    P.slots = (float*)A.workspace;
    P.groups_done = (unsigned int*)((char*)A.workspace + dec_slot_bytes());
    P.items_done = P.groups_done + dec_group_bytes() / 4;
    const int tiles = rows <= 8 ? 1 : 2;
    P.gqa_mul = (uint32_t)(((1 << 20) + gqa - 1) / gqa);
    P.row_groups = (int)((rows + 8 * tiles - 1) / (8 * tiles));
    if (hd == 64) return decode_launch_hd<64>(P, tiles, stream, who);
    if (hd == 96) return decode_launch_hd<96>(P, tiles, stream, who);
    return decode_launch_hd<128>(P, tiles, stream, who);
}

}  // namespace s12
