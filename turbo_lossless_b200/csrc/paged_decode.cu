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
// Work is cut by the device, which alone knows the lengths: the units of 128 positions of all (sequence, kv head, rows)
// items follow one another and every CTA takes an equal range; ends within an eighth of a range of an item's end move
// there.  An item of several CTAs leaves its partial results in the workspace, and the CTA that comes last adds them in
// order, so that the result does not depend on who came when.
#include "paged.cuh"
#include <algorithm>
#include <atomic>

namespace s12 {

constexpr int kDecWarps = 4;
constexpr int kDecThreads = kDecWarps * 32;
constexpr int kDecChunk = 32;                       // positions of a warp's step
constexpr int kDecUnit = kDecWarps * kDecChunk;     // positions of a unit
constexpr int kDecCtasPerSm = 3;
constexpr int kDecMaxRows = 16, kDecMaxDim = 128;
constexpr float kDigits = 32512.f;                  // 127 * 256: the high digit stays below 128
constexpr int64_t kDecSlotFloats = kDecMaxRows * (kDecMaxDim + 2);

struct DecodeParams {
    PagedAttn a;
    float* slots;               // [2 * CTAs][rows][head_dim + 2] partial results
    unsigned int* counters;     // [items] partial results written, zero between calls
    int groups;                 // groups of rows of a kv head
    int min_units;              // units of a CTA, at least
};

__host__ __device__ constexpr int dec_row_floats(int hd) { return hd + hd / 8; }   // padded: the lanes of a store meet different banks
__device__ __forceinline__ int dec_pad(int d) { return d + (d >> 5) * 4; }
template <int kHD, int kTiles>
__host__ __device__ constexpr int dec_smem_bytes() { return kDecWarps * kTiles * 8 * dec_row_floats(kHD) * 4; }

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

// units of an item of sequence s
__device__ __forceinline__ int dec_units(const PagedArgs& C, int s)
{
    const int n = paged_len(C, s);
    return n <= 0 ? 1 : (n + kDecUnit - 1) / kDecUnit;
}

template <int kHD, int kTiles>
__global__ void __launch_bounds__(kDecThreads, kTiles == 1 ? kDecCtasPerSm : 2)
paged_decode_kernel(const __grid_constant__ DecodeParams P)
{
    constexpr int kRows = 8 * kTiles, kSteps = kHD / 32, kCols = kHD / 8;
    extern __shared__ __align__(16) float dec_smem[];
    __shared__ __align__(16) int8_t digits[2][kRows][kHD + 16];    // padded: the lanes of a load meet different banks
    __shared__ float factor_s[kRows], m_s[kDecWarps][kRows], l_s[kDecWarps][kRows];
    __shared__ int last_s;
    grid_launch_dependents();
    grid_dependency_wait();
    const PagedArgs& C = P.a.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
    const int gqa = P.a.n_head / C.n_head_kv, per_seq = C.n_head_kv * P.groups;

    // ---- the units of all items, and this CTA's start: the sequence that holds it (every warp for itself)
    long long total = 0;
    for (int s0 = 0; s0 < C.num_seqs; s0 += 32) {
        long long u = s0 + lane < C.num_seqs ? dec_units(C, s0 + lane) : 0;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) u += __shfl_xor_sync(0xFFFFFFFFu, u, off);
        total += u * per_seq;
    }
    const long long most = (total + P.min_units - 1) / P.min_units;
    const int ctas = most < (long long)gridDim.x ? (int)most : (int)gridDim.x, cta = blockIdx.x;
    if (cta >= ctas) return;
    const long long tol = max(1ll, total / ctas / 8);
    auto cut = [&](int c) { return total * c / ctas; };            // a range's end before it moves to an item's
    auto snap = [&](long long x, long long a, long long b) { return x - a < tol ? a : b - x < tol ? b : x; };   // x in item [a, b)
    long long x = cut(cta), base = 0;                              // base: first unit of sequence seq
    int seq = 0;
    for (int s0 = 0; s0 < C.num_seqs; s0 += 32) {
        long long u = s0 + lane < C.num_seqs ? (long long)dec_units(C, s0 + lane) * per_seq : 0;
        long long upto = u;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long long o = __shfl_up_sync(0xFFFFFFFFu, upto, off);
            if (lane >= off) upto += o;
        }
        const unsigned over = __ballot_sync(0xFFFFFFFFu, base + upto > x);
        if (over) {
            const int l = __ffs(over) - 1;
            seq = s0 + l;
            base += __shfl_sync(0xFFFFFFFFu, upto - u, l);
            break;
        }
        base += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    int units = dec_units(C, seq), item = (int)((x - base) / units);   // item of the sequence
    long long a = base + (long long)item * units;                  // its first unit
    x = snap(x, a, a + units);
    const long long next = cut(cta + 1);                           // this CTA's end lies in or at the end of an item met below

    const float to_log2 = P.a.scale * 1.4426950408889634f;
    while (a < total) {
        if (x >= a + units) {                                      // the start moved to the item's end
            a += units;
            if (++item == per_seq) {
                if (++seq == C.num_seqs) break;
                item = 0; units = dec_units(C, seq);
            }
            if (x > a) x = a;
        }
        // the part [x, end) of item [a, a + units)
        long long end = a + units;
        if (next < end) end = snap(next, a, end);
        if (x >= end) break;
        const int kvh = item / P.groups, row_base = (item - kvh * P.groups) * kRows;
        int lo, hi;
        paged_rows(C, seq, lo, hi);
        const int rows = min(kRows, (hi - lo) * gqa - row_base);   // rows of this item; 0 or less: none
        if (rows > 0) {
            const int len = C.kv_len[seq], room = paged_len(C, seq);
            __syncthreads();                                       // the last item's shared memory has been read
            for (int r = warp; r < kRows; r += kDecWarps) {
                float v[kHD / 32], top = 0.f;
                const int tok = (row_base + r) / gqa, head = row_base + r - tok * gqa;
                const float* q = P.a.q + (size_t)(lo + tok) * P.a.q_stride + (size_t)(kvh * gqa + head) * kHD;
#pragma unroll
                for (int i = 0; i < kHD / 32; i++) v[i] = r < rows ? q[i * 32 + lane] : 0.f;
                uint32_t bits = 0;                                 // of magnitudes: a NaN is the largest
#pragma unroll
                for (int i = 0; i < kHD / 32; i++) bits = max(bits, __float_as_uint(v[i]) & 0x7FFFFFFFu);
                bits = __reduce_max_sync(0xFFFFFFFFu, bits);
                top = __uint_as_float(bits);
                const bool fine = top >= 1e-30f && bits < 0x7F800000u;   // smaller ones count as zero
                const float inv = fine ? kDigits / top : 0.f;
#pragma unroll
                for (int i = 0; i < kHD / 32; i++) {
                    const int X = fine ? __float2int_rn(v[i] * inv) : 0, h = (X + 128) >> 8;
                    digits[0][r][i * 32 + lane] = (int8_t)h; digits[1][r][i * 32 + lane] = (int8_t)(X - 256 * h);
                }
                if (lane == 0) factor_s[r] = bits >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : top / kDigits * to_log2;
            }
            __syncthreads();
            uint32_t qa[kTiles][kSteps][4];
            float factor[kTiles];
            int limit[kTiles];                                     // positions that the lane's row may see
#pragma unroll
            for (int i = 0; i < kTiles; i++) {
                const int r = i * 8 + g;
#pragma unroll
                for (int s = 0; s < kSteps; s++) {
                    const uint2 h = *reinterpret_cast<const uint2*>(&digits[0][r][k_dim<kHD>(s, t4)]);
                    const uint2 l = *reinterpret_cast<const uint2*>(&digits[1][r][k_dim<kHD>(s, t4)]);
                    qa[i][s][0] = h.x; qa[i][s][1] = l.x; qa[i][s][2] = h.y; qa[i][s][3] = l.y;
                }
                factor[i] = factor_s[r];
                limit[i] = r < rows ? min(len - (hi - lo) + (row_base + r) / gqa + 1, room) : 0;
            }
            const int least = min(len - (hi - lo) + row_base / gqa + 1, room);                    // of all rows
            const int most_seen = min(len - (hi - lo) + (row_base + rows - 1) / gqa + 1, room);
            const int t_lo = (int)(x - a) * kDecUnit, t_hi = min((int)(end - a) * kDecUnit, most_seen);
            float acc[kTiles][kCols][2], m[kTiles], l[kTiles];
#pragma unroll
            for (int i = 0; i < kTiles; i++) {
                m[i] = -1e30f; l[i] = 0.f;
#pragma unroll
                for (int j = 0; j < kCols; j++) acc[i][j][0] = acc[i][j][1] = 0.f;
            }
            const int ps = 1 << C.page_shift;
            const int* table = C.table + (size_t)seq * C.table_stride;
            bool missing = false;
            // page of position t, -1: none
            auto page_at = [&](int t) {
                if (t >= t_hi || (t >> C.page_shift) >= C.table_pages) return -1;
                const int p = table[t >> C.page_shift];
                if ((unsigned)p < (unsigned)C.num_pages) return p;
                missing = true;
                return -1;
            };
            KRow<kHD> k[4];
            VRow<kHD> v[8];
            float4 sk[2], sv[2];
            auto fetch_k = [&](int t0, int page) {
                const size_t at = ((size_t)page * C.n_head_kv + kvh) << C.page_shift;
                const int8_t* row = C.k + (at + ((t0 + 4 * g) & (ps - 1))) * kHD;
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    if (page >= 0) load_k<kHD>(k[u], row + u * kHD, t4);
                    else
#pragma unroll
                        for (int i = 0; i < kHD / 16; i++) k[u].w[i] = 0;
                }
            };
            auto fetch_v = [&](int t0, int page) {
                const size_t at = (((size_t)page * C.n_head_kv + kvh) << C.page_shift) + ((t0 + 8 * t4) & (ps - 1));
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    if (page >= 0) load_v<kHD>(v[u], C.v + (at + u) * kHD, g);
                    else
#pragma unroll
                        for (int i = 0; i < kHD / 32; i++) v[u].w[i] = 0;
                }
            };
            auto fetch_s = [&](float4 (&s)[2], const float* scales, int t0, int page) {
                const size_t at = (((size_t)page * C.n_head_kv + kvh) << C.page_shift) + ((t0 + 8 * t4) & (ps - 1));
#pragma unroll
                for (int u = 0; u < 2; u++) s[u] = page >= 0 ? reinterpret_cast<const float4*>(scales + at)[u] : make_float4(0.f, 0.f, 0.f, 0.f);
            };
            int t0 = t_lo + warp * kDecChunk;
            // a chunk has one page, or two of 16 positions: K rows 4 g + u lie in the half of g >> 2, V rows 8 t4 + u of t4 >> 1
            int pk = page_at(t0 + (g >> 2) * 16), pv = page_at(t0 + (t4 >> 1) * 16);
            int pk_next = page_at(t0 + kDecUnit + (g >> 2) * 16), pv_next = page_at(t0 + kDecUnit + (t4 >> 1) * 16);
            fetch_k(t0, pk);
            fetch_s(sk, C.sk, t0, pv);
            fetch_s(sv, C.sv, t0, pv);
            fetch_v(t0, pv);
#pragma unroll 1
            for (; t0 < t_hi; t0 += kDecUnit) {
                const int t_next = t0 + kDecUnit;
                // ---- scores
                int c[kTiles][4][4];
#pragma unroll
                for (int i = 0; i < kTiles; i++)
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        c[i][u][0] = c[i][u][1] = c[i][u][2] = c[i][u][3] = 0;
#pragma unroll
                        for (int s = 0; s < kSteps; s++)
                            mma_s8(c[i][u], qa[i][s][0], qa[i][s][1], qa[i][s][2], qa[i][s][3], k[u].w[2 * s], k[u].w[2 * s + 1]);
                    }
                fetch_k(t_next, pk_next);
                const float skv[8] = {sk[0].x, sk[0].y, sk[0].z, sk[0].w, sk[1].x, sk[1].y, sk[1].z, sk[1].w};
                const bool whole = __all_sync(0xFFFFFFFFu, pv >= 0 && t0 + kDecChunk <= least);
                float s[kTiles][8];                                 // score of position t0 + 8 t4 + i, in powers of two
#pragma unroll
                for (int i = 0; i < kTiles; i++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
#pragma unroll
                        for (int u = 0; u < 4; u++) s[i][4 * e + u] = (float)(256 * c[i][u][e] + c[i][u][2 + e]) * skv[4 * e + u] * factor[i];
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < kTiles; i++)
#pragma unroll
                        for (int p = 0; p < 8; p++) if (pv < 0 || t0 + 8 * t4 + p >= limit[i]) s[i][p] = -INFINITY;
                }
                fetch_s(sk, C.sk, t_next, pv_next);
                // ---- weights: of the chunk's own maximum, times the values' scales, as two digits of the largest such product
                const float svv[8] = {sv[0].x, sv[0].y, sv[0].z, sv[0].w, sv[1].x, sv[1].y, sv[1].z, sv[1].w};
                uint32_t pa[kTiles][4];
                float gain[kTiles];
#pragma unroll
                for (int i = 0; i < kTiles; i++) {
                    float mx = -1e30f;
#pragma unroll
                    for (int p = 0; p < 8; p++) mx = fmaxf(mx, s[i][p]);
                    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
                    float sum = 0.f, top = 0.f, z[8];
#pragma unroll
                    for (int p = 0; p < 8; p++) {
                        const float w = dec_exp2(s[i][p] - mx);
                        z[p] = w * svv[p];
                        float mark = fmaf(svv[p], 0.f, w);          // w, or NaN where the scale is not finite
                        if (!whole && s[i][p] == -INFINITY) z[p] = mark = 0.f;
                        sum += mark;
                        if (!(fabsf(z[p]) < INFINITY)) z[p] = 0.f;
                        top = fmaxf(top, fabsf(z[p]));
                    }
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                    const float inv = top >= 1e-30f ? __fdividef(kDigits, top) : 0.f;
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
                fetch_s(sv, C.sv, t_next, pv_next);
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
                fetch_v(t_next, pv_next);
                pk = pk_next; pv = pv_next;
                pk_next = page_at(t_next + kDecUnit + (g >> 2) * 16); pv_next = page_at(t_next + kDecUnit + (t4 >> 1) * 16);
            }
            if (missing) atomicOr(C.status, kStatusPage);
            // ---- the warps' results meet in shared memory
#pragma unroll
            for (int i = 0; i < kTiles; i++) {
                l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 1);
                l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 2);
                const int r = i * 8 + g;
                if (t4 == 0) { m_s[warp][r] = m[i]; l_s[warp][r] = l[i]; }
                float* row = dec_smem + (size_t)(warp * kRows + r) * dec_row_floats(kHD);
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int j = 0; j < kCols; j += 4)
                        *reinterpret_cast<float4*>(row + dec_pad((2 * t4 + e) * kCols + j)) = make_float4(acc[i][j][e], acc[i][j + 1][e], acc[i][j + 2][e], acc[i][j + 3][e]);
            }
            __syncthreads();
            const bool alone = x == a && end == a + units;
            const int slot = 2 * cta + (x == a ? 1 : 0);            // at most one part of an item that began before, one of one that goes on
            float* part = P.slots + (size_t)slot * kDecSlotFloats;
            for (int i = threadIdx.x; i < rows * (kHD / 4); i += kDecThreads) {
                const int r = i / (kHD / 4), d = (i - r * (kHD / 4)) * 4;
                float mm = -1e30f, den = 0.f;
                float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kDecWarps; w++) mm = fmaxf(mm, m_s[w][r]);
#pragma unroll
                for (int w = 0; w < kDecWarps; w++) {
                    const float f = dec_exp2(m_s[w][r] - mm);
                    const float4 y = *reinterpret_cast<const float4*>(dec_smem + (size_t)(w * kRows + r) * dec_row_floats(kHD) + dec_pad(d));
                    num.x += f * y.x; num.y += f * y.y; num.z += f * y.z; num.w += f * y.w;
                    den += f * l_s[w][r];
                }
                if (!alone) {
                    *reinterpret_cast<float4*>(part + r * kHD + d) = num;
                    if (d == 0) { part[kRows * kHD + 2 * r] = mm; part[kRows * kHD + 2 * r + 1] = den; }
                    continue;
                }
                const int tok = (row_base + r) / gqa, head = row_base + r - tok * gqa;
                int16_t* o = P.a.out + (size_t)(lo + tok) * P.a.out_stride + (size_t)(kvh * gqa + head) * kHD + d;
                const float rd = den == 0.f ? 0.f : 1.f / den;      // no position at all: zero
                o[0] = paged_bf16_rne(num.x * rd); o[1] = paged_bf16_rne(num.y * rd);
                o[2] = paged_bf16_rne(num.z * rd); o[3] = paged_bf16_rne(num.w * rd);
            }
            if (!alone) {
                // CTAs whose ends lie strictly inside this item
                const long long A = a + tol, B = a + units - tol;
                const int c_lo = (int)((A * ctas + total - 1) / total), c_hi = (int)(((B + 1) * ctas + total - 1) / total) - 1;
                const int parts = c_hi - c_lo + 2;
                unsigned int* counter = P.counters + (size_t)seq * per_seq + item;
                __threadfence();
                __syncthreads();
                if (threadIdx.x == 0) last_s = atomicAdd(counter, 1u) == (unsigned)parts - 1;
                __syncthreads();
                if (last_s) {
                    __threadfence();
                    if (threadIdx.x == 0) *counter = 0;
                    for (int i = threadIdx.x; i < rows * (kHD / 4); i += kDecThreads) {
                        const int r = i / (kHD / 4), d = (i - r * (kHD / 4)) * 4;
                        auto of = [&](int c) { return P.slots + (size_t)(2 * c + (c == c_lo - 1 ? 1 : 0)) * kDecSlotFloats; };
                        float mm = -1e30f, den = 0.f;
                        float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
                        for (int c = c_lo - 1; c <= c_hi; c++) mm = fmaxf(mm, __ldcg(of(c) + kRows * kHD + 2 * r));
                        for (int c = c_lo - 1; c <= c_hi; c++) {
                            const float* p = of(c);
                            const float f = dec_exp2(__ldcg(p + kRows * kHD + 2 * r) - mm);
                            const float4 y = __ldcg(reinterpret_cast<const float4*>(p + r * kHD + d));
                            num.x += f * y.x; num.y += f * y.y; num.z += f * y.z; num.w += f * y.w;
                            den += f * __ldcg(p + kRows * kHD + 2 * r + 1);
                        }
                        const int tok = (row_base + r) / gqa, head = row_base + r - tok * gqa;
                        int16_t* o = P.a.out + (size_t)(lo + tok) * P.a.out_stride + (size_t)(kvh * gqa + head) * kHD + d;
                        const float rd = den == 0.f ? 0.f : 1.f / den;
                        o[0] = paged_bf16_rne(num.x * rd); o[1] = paged_bf16_rne(num.y * rd);
                        o[2] = paged_bf16_rne(num.z * rd); o[3] = paged_bf16_rne(num.w * rd);
                    }
                }
            }
        }
        x = end;
        if (end < a + units) break;                                 // the range ends inside the item
    }
}

static int64_t dec_slot_bytes() { return 2ll * sm_count() * kDecCtasPerSm * kDecSlotFloats * 4; }
static int dec_groups(int n_head, int n_head_kv, int max_new)
{
    const long long rows = (long long)(n_head / n_head_kv) * max_new;
    return (int)((rows + kDecMaxRows - 1) / kDecMaxRows);
}
int64_t paged_decode_workspace_bytes(int n_head, int n_head_kv, int num_seqs, int max_new)
{
    return dec_slot_bytes() + (int64_t)num_seqs * n_head_kv * dec_groups(n_head, n_head_kv, max_new) * 4;
}

template <int kHD, int kTiles>
static int decode_launch(const DecodeParams& P, int ctas, void* stream, const char* who)
{
    constexpr int smem = dec_smem_bytes<kHD, kTiles>();
    static std::atomic<bool> attr_set[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (smem > 40 * 1024 && (dev < 0 || dev >= 64 || !attr_set[dev].load(std::memory_order_relaxed))) {
        const int rc = check_cuda(cudaFuncSetAttribute(paged_decode_kernel<kHD, kTiles>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), who);
        if (rc) return rc;
        if (dev >= 0 && dev < 64) attr_set[dev].store(true, std::memory_order_relaxed);
    }
    return launch(paged_decode_kernel<kHD, kTiles>, dim3(ctas), dim3(kDecThreads), smem, stream, who, P);
}

// 1: not a shape of this kernel
int paged_decode_launch(const PagedAttn& A, void* stream, const char* who)
{
    const int hd = A.c.head_dim, gqa = A.n_head / A.c.n_head_kv;
    const long long rows = (long long)gqa * A.max_new;
    if ((hd != 64 && hd != 96 && hd != 128) || rows > 64) return 1;
    const int64_t need = paged_decode_workspace_bytes(A.n_head, A.c.n_head_kv, A.c.num_seqs, A.max_new);
    if (!A.workspace || A.workspace_bytes < need || (reinterpret_cast<uintptr_t>(A.workspace) & 15))
        return fail(S12_ERR_BAD_ARG, "%s: needs a 16-byte aligned workspace of %lld bytes", who, (long long)need);
    DecodeParams P = {};
    P.a = A;
    P.slots = (float*)A.workspace;
    P.counters = (unsigned int*)((char*)A.workspace + dec_slot_bytes());
    const int tiles = rows <= 8 ? 1 : 2;
    P.groups = (int)((rows + 8 * tiles - 1) / (8 * tiles));
    P.min_units = 4;
    // units that the bounds allow: no more CTAs than that
    const long long units = (long long)A.c.num_seqs * A.c.n_head_kv * P.groups * ((std::max(A.max_len, 1) + kDecUnit - 1) / kDecUnit);
    const int ctas = (int)std::max(1ll, std::min((units + P.min_units - 1) / P.min_units, (long long)sm_count() * kDecCtasPerSm));
    if (hd == 64) return tiles == 1 ? decode_launch<64, 1>(P, ctas, stream, who) : decode_launch<64, 2>(P, ctas, stream, who);
    if (hd == 96) return tiles == 1 ? decode_launch<96, 1>(P, ctas, stream, who) : decode_launch<96, 2>(P, ctas, stream, who);
    return tiles == 1 ? decode_launch<128, 1>(P, ctas, stream, who) : decode_launch<128, 2>(P, ctas, stream, who);
}

}  // namespace s12
