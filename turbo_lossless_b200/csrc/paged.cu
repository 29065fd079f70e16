// The paged INT8 key-value cache: sequences of different lengths share one pool of pages, and prompts go through in one
// pass instead of token by token.  New entry points: the reference engine has one contiguous cache and runs a prompt
// as decode steps (engine/inference.cpp:198-366).
//
//   store      rotation of q and k, quantisation of k and v, store into the pages
//   attention  causal attention of packed new tokens (a prompt, a chunk behind a cached prefix, one token) over the pages
//   copy       pages copied over all layers: fork, compaction
//
// Pages are head-major, [page][kv head][position][head_dim]: what a CTA reads of a page is contiguous.
#include "paged.cuh"
#include <algorithm>
#include <cmath>
#include <mutex>

namespace s12 {

// ---------------------------------------------------------------------------
// Store.  angle = position * theta^(-2 d / head_dim); (x0, x1) = elements d, d + head_dim / 2 of a head become
// (x0 cos - x1 sin, x0 sin + x1 cos); scale = absmax / 127, code = rint(x * (127 * (1 / absmax))) of the rotated k and of v,
// each operation rounded to 64 bits: so are values on a border between two codes put to one side by all.
// The angles, k's rotation and the codes are computed in 64 bits (an angle of position 100 000 rounded to 32 bits is off
// by 4e-3): the cache's bytes are those of the exact values but for ties; q is rotated in 32 bits.
// ---------------------------------------------------------------------------
struct StoreParams {
    PagedArgs c;
    const float* q; const float* k; const float* v; float* q_out;
    int q_stride, kv_stride, q_out_stride, n_head;
    int group_shift;            // paged_store_rows_kernel: 2^this lanes have a head
};
struct HalfTurns { double f[128]; };                            // theta^(-2 d / head_dim) / pi

constexpr int kStoreWarps = 8;
constexpr int kStoreThreads = kStoreWarps * 32;

__device__ __forceinline__ unsigned long long abs_bits(double x) { return (unsigned long long)__double_as_longlong(x) & 0x7FFFFFFFFFFFFFFFull; }

// grid (tokens, head groups); a warp per head, lane owns elements d and d + half for d = lane, lane + 32, ...
__global__ void __launch_bounds__(kStoreThreads)
paged_store_kernel(const __grid_constant__ StoreParams P, const __grid_constant__ HalfTurns F)
{
    __shared__ double cos_s[128], sin_s[128];
    grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.x;
    const int hd = P.c.head_dim, half = hd >> 1;
    const int seq = paged_seq_of(P.c, row);
    if (seq < 0) return;                                          // a row behind the last sequence
    const int after = P.c.q_start ? P.c.q_start[seq + 1] - row : 1;
    const int pos = P.c.kv_len[seq] - after;
    for (int d = threadIdx.x; d < half; d += kStoreThreads) sincospi((double)pos * F.f[d], &sin_s[d], &cos_s[d]);
    const bool inside = pos >= 0 && (pos >> P.c.page_shift) < P.c.table_pages;
    const int page = inside ? paged_page(P.c, seq, pos) : -1;     // position below 0: a row of a sequence that is not there
    if (page < 0 && pos >= 0 && threadIdx.x == 0 && blockIdx.y == 0) atomicOr(P.c.status, kStatusPage);
    __syncthreads();
    const int hkv = P.c.n_head_kv, heads = P.n_head + 2 * hkv;
    const int h = blockIdx.y * kStoreWarps + warp;
    if (h >= heads) return;
    if (h < P.n_head) {
        const float* x = P.q + (size_t)row * P.q_stride + (size_t)h * hd;
        float* y = P.q_out + (size_t)row * P.q_out_stride + (size_t)h * hd;
        for (int d = lane; d < half; d += 32) {
            const float c = (float)cos_s[d], s = (float)sin_s[d], x0 = x[d], x1 = x[d + half];
            y[d] = x0 * c - x1 * s; y[d + half] = x0 * s + x1 * c;
        }
        return;
    }
    if (page < 0) return;
    const bool is_v = h >= P.n_head + hkv;
    const int kvh = h - P.n_head - (is_v ? hkv : 0);
    const float* x = (is_v ? P.v : P.k) + (size_t)row * P.kv_stride + (size_t)kvh * hd;
    double lo[4], hi[4];
    unsigned long long top = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int d = i * 32 + lane;
        if (d >= half) continue;
        lo[i] = x[d]; hi[i] = x[d + half];
        if (!is_v) {
            const double c = cos_s[d], s = sin_s[d], x0 = lo[i], x1 = hi[i];
            lo[i] = x0 * c - x1 * s; hi[i] = x0 * s + x1 * c;
        }
        top = max(top, max(abs_bits(lo[i]), abs_bits(hi[i])));
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, off));
    const double amax = __longlong_as_double((long long)top), inv = __dmul_rn(1.0 / amax, 127.0);   // a NaN counts as the largest
    const size_t at = ((size_t)page * hkv + kvh) << P.c.page_shift | (size_t)(pos & ((1 << P.c.page_shift) - 1));
    int8_t* dst = (is_v ? P.c.v : P.c.k) + at * hd;
    auto code = [&](double v) { const double r = rint(__dmul_rn(v, inv)); return (int8_t)(r == r ? (int)fmin(fmax(r, -127.0), 127.0) : 0); };
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int d = i * 32 + lane;
        if (d < half) { dst[d] = code(lo[i]); dst[d + half] = code(hi[i]); }
    }
    if (lane == 0) (is_v ? P.c.sv : P.c.sk)[at] = (float)(amax / 127.0);
}

// The same for rows on 16-byte boundaries and head_dim a multiple of 8.  Bound: HBM, 4 bytes an element in, 4 or 1 out.
// A group of lanes has a head, a lane four neighbouring elements of each half, so that a pair lies in one lane; a warp takes
// kPasses times as many heads as it has groups, all of their loads in flight while the angles are computed, once a CTA.
// 7 k tokens of 32/8 heads of 128: 61 us (4.7 TB/s), a warp a head 181, one / two / four / six passes 83 / 84 / 73 / 81; bound by a
// CTA's chain of length, page and angles.  Slower: CTAs that walk neighbouring rows with the next one's loads in flight and
// the angles turned on from position to position (67), four CTAs an SM in 64 registers (61), fewer 64-bit instructions (65).
template <int kPasses>
__global__ void __launch_bounds__(kStoreThreads)
paged_store_rows_kernel(const __grid_constant__ StoreParams P, const __grid_constant__ HalfTurns F)
{
    __shared__ __align__(16) double cos_s[128], sin_s[128];
    grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.x;
    const int hd = P.c.head_dim, half = hd >> 1, hkv = P.c.n_head_kv, heads = P.n_head + 2 * hkv;
    const int group = lane >> P.group_shift, d = (lane & ((1 << P.group_shift) - 1)) * 4;   // the lane's head of a pass, its elements
    const int per_pass = kStoreWarps * (32 >> P.group_shift);
    const int h0 = blockIdx.y * kPasses * per_pass + warp * (32 >> P.group_shift) + group;
    const int seq = paged_seq_of(P.c, row);
    if (seq < 0) return;                                          // a row behind the last sequence
    float4 lo[kPasses], hi[kPasses];
#pragma unroll
    for (int i = 0; i < kPasses; i++) {
        const int h = h0 + i * per_pass;
        if (h >= heads || d >= half) continue;
        const float* x = h < P.n_head ? P.q + (size_t)row * P.q_stride + (size_t)h * hd
                                      : (h < P.n_head + hkv ? P.k + (size_t)(h - P.n_head) * hd : P.v + (size_t)(h - P.n_head - hkv) * hd) + (size_t)row * P.kv_stride;
        lo[i] = *reinterpret_cast<const float4*>(x + d); hi[i] = *reinterpret_cast<const float4*>(x + d + half);
    }
    const int after = P.c.q_start ? P.c.q_start[seq + 1] - row : 1;
    const int pos = P.c.kv_len[seq] - after;
    const bool inside = pos >= 0 && (pos >> P.c.page_shift) < P.c.table_pages;
    const int page = inside ? paged_page(P.c, seq, pos) : -1;     // position below 0: a row of a sequence that is not there
    if (page < 0 && pos >= 0 && threadIdx.x == 0 && blockIdx.y == 0) atomicOr(P.c.status, kStatusPage);
    for (int i = threadIdx.x; i < half; i += kStoreThreads) sincospi((double)pos * F.f[i], &sin_s[i], &cos_s[i]);
    __syncthreads();
    double c[4], s[4];
#pragma unroll
    for (int e = 0; e < 4; e++) { c[e] = d < half ? cos_s[d + e] : 0.; s[e] = d < half ? sin_s[d + e] : 0.; }
#pragma unroll
    for (int i = 0; i < kPasses; i++) {
        const int h = h0 + i * per_pass;
        const bool live = h < heads && d < half;
        const float a[4] = {lo[i].x, lo[i].y, lo[i].z, lo[i].w}, b[4] = {hi[i].x, hi[i].y, hi[i].z, hi[i].w};
        if (live && h < P.n_head) {
            float x[4], y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float cf = (float)c[e], sf = (float)s[e];
                x[e] = a[e] * cf - b[e] * sf; y[e] = a[e] * sf + b[e] * cf;
            }
            float* to = P.q_out + (size_t)row * P.q_out_stride + (size_t)h * hd + d;
            *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(to + half) = make_float4(y[0], y[1], y[2], y[3]);
        }
        if (!__any_sync(0xFFFFFFFFu, live && h >= P.n_head) || page < 0) continue;
        const bool is_v = h >= P.n_head + hkv, keep = live && h >= P.n_head;
        double x[8];
        unsigned long long top = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const double x0 = a[e], x1 = b[e];
            x[e] = is_v ? x0 : x0 * c[e] - x1 * s[e]; x[4 + e] = is_v ? x1 : x0 * s[e] + x1 * c[e];
            if (keep) top = max(top, max(abs_bits(x[e]), abs_bits(x[4 + e])));
        }
        for (int off = 1 << P.group_shift >> 1; off > 0; off >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, off));
        if (!keep) continue;
        const double amax = __longlong_as_double((long long)top), inv = __dmul_rn(1.0 / amax, 127.0);   // a NaN counts as the largest
        const bool fine = top < 0x7FF0000000000000ull && top > 0;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; e++) {
            // rounded to nearest by 1.5 * 2^52: the low word holds the code; the product is rounded first, not fused
            const uint32_t r = fine ? (uint32_t)__double2loint(__dadd_rn(__dmul_rn(x[e], inv), 6755399441055744.0)) : 0u;
            w[e >> 2] |= (r & 0xFFu) << (8 * (e & 3));
        }
        const int kvh = h - P.n_head - (is_v ? hkv : 0);
        const size_t at = ((size_t)page * hkv + kvh) << P.c.page_shift | (size_t)(pos & ((1 << P.c.page_shift) - 1));
        int8_t* dst = (is_v ? P.c.v : P.c.k) + at * hd + d;
        *reinterpret_cast<uint32_t*>(dst) = w[0];
        *reinterpret_cast<uint32_t*>(dst + half) = w[1];
        if (d == 0) (is_v ? P.c.sv : P.c.sk)[at] = (float)(amax / 127.0);
    }
}

// ---------------------------------------------------------------------------
// Copy.  A CTA copies 16 KB of a page in one layer, four 16-byte loads a thread in flight.  Bound: HBM; 300 pages of 8 x 64 x 128
// in 16 layers 197.5 us (6.57 TB/s, a plain copy's rate), one page in 32 layers 2.8 us.
// ---------------------------------------------------------------------------
struct CopyParams {
    uint4* part[4];             // k, v, their scales
    uint32_t units[2];          // 16-byte units of a page's codes and of its scales
    uint32_t chunks;            // CTAs of a page
    const int* src; const int* dst;
    unsigned int* status;
    int num_pages;
};
constexpr int kCopyThreads = 256, kCopyUnits = 4;

__global__ void __launch_bounds__(kCopyThreads)
paged_copy_kernel(const __grid_constant__ CopyParams P)
{
    grid_launch_dependents();
    grid_dependency_wait();
    const uint32_t move = blockIdx.x / P.chunks, chunk = blockIdx.x - move * P.chunks;
    const int src = P.src[move], dst = P.dst[move];
    if ((unsigned)src >= (unsigned)P.num_pages || (unsigned)dst >= (unsigned)P.num_pages) {
        if (threadIdx.x == 0) atomicOr(P.status, kStatusPage);
        return;
    }
    const uint32_t all = 2 * (P.units[0] + P.units[1]);
    uint4 x[kCopyUnits];
    uint4* to[kCopyUnits];
#pragma unroll
    for (int i = 0; i < kCopyUnits; i++) {
        uint32_t u = (chunk * kCopyUnits + i) * kCopyThreads + threadIdx.x;
        to[i] = nullptr;
        if (u >= all) continue;
        const int kind = u >= 2 * P.units[0];                     // codes or scales
        if (kind) u -= 2 * P.units[0];
        const uint32_t n = P.units[kind];
        const int part = 2 * kind + (u >= n);
        if (u >= n) u -= n;
        uint4* base = P.part[part] + (size_t)blockIdx.y * P.num_pages * n + u;
        x[i] = base[(size_t)src * n];
        to[i] = base + (size_t)dst * n;
    }
#pragma unroll
    for (int i = 0; i < kCopyUnits; i++) if (to[i]) *to[i] = x[i];
}

// ---------------------------------------------------------------------------
// Attention, any other head_dim that is a multiple of 4 up to 256, for completeness: a CTA per (token, query head), a warp per position, running
// maximum and sum per warp, the warps' partial results merged in shared memory.  Sums in 32 bits.
// out[t] = sum_j p_j v_j / sum_j p_j, p_j = exp(scale * q . k_j - m) over the positions j <= position of t; 0 where there
// is none.
// ---------------------------------------------------------------------------
constexpr int kGenWarps = 8;

__global__ void __launch_bounds__(kGenWarps * 32)
paged_attention_general_kernel(const __grid_constant__ PagedAttn P)
{
    __shared__ float acc_s[kGenWarps][256], m_s[kGenWarps], l_s[kGenWarps];
    grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.x, head = blockIdx.y;
    const PagedArgs& C = P.c;
    const int hd = C.head_dim, kvh = head / (P.n_head / C.n_head_kv);
    const int seq = paged_seq_of(C, row);
    if (seq < 0) return;
    const int after = C.q_start ? C.q_start[seq + 1] - row : 1;   // the token's position counts from the sequence's end
    const int own = C.kv_len[seq] - after + 1, room = paged_len(C, seq), n = own < room ? own : room;
    const float* q = P.q + (size_t)row * P.q_stride + (size_t)head * hd;
    float qv[2][4], acc[2][4];
    bool live[2];
#pragma unroll
    for (int c = 0; c < 2; c++) {
        live[c] = c * 128 + lane * 4 < hd;
#pragma unroll
        for (int e = 0; e < 4; e++) { qv[c][e] = live[c] ? q[c * 128 + lane * 4 + e] * P.scale : 0.f; acc[c][e] = 0.f; }
    }
    float m = -INFINITY, l = 0.f;
    bool bad = paged_past_table(C, own);
    for (int t = warp; t < n; t += kGenWarps) {
        const int page = paged_page(C, seq, t);
        if (page < 0) { bad = true; continue; }
        const size_t at = ((size_t)page * C.n_head_kv + kvh) << C.page_shift | (size_t)(t & ((1 << C.page_shift) - 1));
        char4 kc[2] = {}, vc[2] = {};
        float dot = 0.f;
#pragma unroll
        for (int c = 0; c < 2; c++) {
            if (!live[c]) continue;
            kc[c] = *reinterpret_cast<const char4*>(C.k + at * hd + c * 128 + lane * 4);
            vc[c] = *reinterpret_cast<const char4*>(C.v + at * hd + c * 128 + lane * 4);
            dot += qv[c][0] * kc[c].x + qv[c][1] * kc[c].y + qv[c][2] * kc[c].z + qv[c][3] * kc[c].w;
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, off);
        const float s = dot * C.sk[at];
        if (s > m) {
            const float f = expf(m - s);
            m = s; l *= f;
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[c][e] *= f;
        }
        const float p = s == -INFINITY ? 0.f : expf(s - m), w = p * C.sv[at];
        l += p;
#pragma unroll
        for (int c = 0; c < 2; c++) {
            acc[c][0] += w * vc[c].x; acc[c][1] += w * vc[c].y; acc[c][2] += w * vc[c].z; acc[c][3] += w * vc[c].w;
        }
    }
    if (bad && lane == 0) atomicOr(C.status, kStatusPage);
#pragma unroll
    for (int c = 0; c < 2; c++)
#pragma unroll
        for (int e = 0; e < 4; e++) if (live[c]) acc_s[warp][c * 128 + lane * 4 + e] = acc[c][e];
    if (lane == 0) { m_s[warp] = m; l_s[warp] = l; }
    __syncthreads();
    float mm = -INFINITY;
    for (int w = 0; w < kGenWarps; w++) mm = fmaxf(mm, m_s[w]);
    for (int d = threadIdx.x; d < hd; d += kGenWarps * 32) {
        float num = 0.f, den = 0.f;
        for (int w = 0; w < kGenWarps; w++) {
            const float f = m_s[w] == -INFINITY ? 0.f : expf(m_s[w] - mm);   // a warp without positions
            num += f * acc_s[w][d]; den += f * l_s[w];
        }
        P.out[(size_t)row * P.out_stride + (size_t)head * hd + d] = paged_bf16_rne(den == 0.f ? 0.f : num / den);
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static int paged_cache_args(PagedArgs& C, const S12PagedKv* kv, const char* who)
{
    if (!kv || !kv->k || !kv->v || !kv->scale_k || !kv->scale_v) return fail(S12_ERR_BAD_ARG, "%s: null cache", who);
    const int ps = kv->page_size;
    if (ps < 16 || ps > 1024 || (ps & (ps - 1))) return fail(S12_ERR_UNSUPPORTED, "%s: page_size %d (a power of two from 16 to 1024)", who, ps);
    if (kv->num_pages < 1 || kv->n_head_kv < 1 || kv->head_dim < 4 || kv->head_dim > 256 || (kv->head_dim & 3))
        return fail(S12_ERR_UNSUPPORTED, "%s: needs num_pages >= 1, n_head_kv >= 1, head_dim a multiple of 4 up to 256", who);
    if ((reinterpret_cast<uintptr_t>(kv->k) | reinterpret_cast<uintptr_t>(kv->v) | reinterpret_cast<uintptr_t>(kv->scale_k) |
         reinterpret_cast<uintptr_t>(kv->scale_v)) & 15)
        return fail(S12_ERR_BAD_ARG, "%s: the cache's arrays must be 16-byte aligned", who);
    C.k = kv->k; C.v = kv->v; C.sk = kv->scale_k; C.sv = kv->scale_v;
    C.num_pages = kv->num_pages; C.n_head_kv = kv->n_head_kv; C.head_dim = kv->head_dim;
    C.page_shift = 0;
    while ((1 << C.page_shift) < ps) C.page_shift++;
    return S12_OK;
}
// the last table made, for the next call of the same shape
static void half_turns(int head_dim, float theta, HalfTurns& F)
{
    static std::mutex mu;
    static HalfTurns cached;
    static int c_dim = 0;
    static float c_theta = 0.f;
    std::lock_guard<std::mutex> lk(mu);
    if (c_dim != head_dim || c_theta != theta) {
        for (int d = 0; d < head_dim / 2; d++) cached.f[d] = std::pow((double)theta, -2.0 * d / head_dim) / 3.14159265358979323846;
        c_dim = head_dim; c_theta = theta;
    }
    F = cached;
}
static int paged_status(PagedArgs& C, const char* who)
{
    C.status = device_status_word();
    return C.status ? S12_OK : fail(S12_ERR_CUDA, "%s: status word allocation failed", who);
}
static int paged_batch_args(PagedArgs& C, const S12PagedBatch* b, int n_head, const char* who)
{
    if (!b || !b->block_table || !b->kv_len) return fail(S12_ERR_BAD_ARG, "%s: null batch", who);
    if (b->num_seqs < 1 || b->num_tokens < 1 || b->table_pages < 1 || b->table_stride < b->table_pages)
        return fail(S12_ERR_BAD_ARG, "%s: needs num_seqs, num_tokens, table_pages >= 1 and table_stride >= table_pages", who);
    if (!b->q_start && b->num_tokens != b->num_seqs)
        return fail(S12_ERR_BAD_ARG, "%s: without q_start every sequence has one token (%d tokens, %d sequences)", who, b->num_tokens, b->num_seqs);
    if (n_head < C.n_head_kv || n_head % C.n_head_kv != 0)
        return fail(S12_ERR_UNSUPPORTED, "%s: n_head %d is not a multiple of n_head_kv %d", who, n_head, C.n_head_kv);
    if (n_head > 65535) return fail(S12_ERR_UNSUPPORTED, "%s: %d heads", who, n_head);
    C.table = b->block_table; C.kv_len = b->kv_len; C.q_start = b->q_start;
    C.num_seqs = b->num_seqs; C.num_tokens = b->num_tokens; C.table_pages = b->table_pages; C.table_stride = b->table_stride;
    return S12_OK;
}

}  // namespace s12

using namespace s12;

extern "C" {

int s12_rope_store_kv_paged_async(const float* q, int q_stride, const float* k, const float* v, int kv_stride, float* q_out,
                                  int q_out_stride, const S12PagedKv* kv, const S12PagedBatch* batch, int n_head, float theta,
                                  void* stream)
{
    static const char* who = "s12_rope_store_kv_paged_async";
    StoreParams P = {};
    int rc = paged_cache_args(P.c, kv, who);
    if (!rc) rc = paged_batch_args(P.c, batch, n_head, who);
    if (rc) return rc;
    const int hd = kv->head_dim;
    if (!q || !k || !v || !q_out) return fail(S12_ERR_BAD_ARG, "%s: null argument", who);
    if (q_stride < n_head * hd || q_out_stride < n_head * hd || kv_stride < kv->n_head_kv * hd || !(theta > 0.f && std::isfinite(theta)))
        return fail(S12_ERR_BAD_ARG, "%s: a row stride shorter than the row, or theta not above 0", who);
    if ((rc = paged_status(P.c, who)) != S12_OK) return rc;
    HalfTurns F;
    half_turns(hd, theta, F);
    P.q = q; P.k = k; P.v = v; P.q_out = q_out;
    P.q_stride = q_stride; P.kv_stride = kv_stride; P.q_out_stride = q_out_stride; P.n_head = n_head;
    const bool rows16 = hd % 8 == 0 && ((q_stride | kv_stride | q_out_stride) & 3) == 0 &&
                        ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(q_out)) & 15) == 0;
    if (rows16) {
        while ((1 << P.group_shift) < hd / 8) P.group_shift++;
        const int all = n_head + 2 * kv->n_head_kv, per_pass = kStoreWarps * (32 >> P.group_shift);
        // Up to three passes a warp, so that the angles are computed once for 48 heads of 128; one where the tokens are few.
        const int needed = (all + per_pass - 1) / per_pass, parts = batch->num_tokens >= sm_count() ? (needed + 2) / 3 : needed, passes = (needed + parts - 1) / parts;
        return launch(passes == 1 ? paged_store_rows_kernel<1> : passes == 2 ? paged_store_rows_kernel<2> : paged_store_rows_kernel<3>,
                      dim3(batch->num_tokens, parts), dim3(kStoreThreads), 0, stream, who, P, F);
    }
    return launch(paged_store_kernel, dim3(batch->num_tokens, (n_head + 2 * kv->n_head_kv + kStoreWarps - 1) / kStoreWarps), dim3(kStoreThreads), 0, stream, who, P, F);
}

int s12_copy_pages_async(const S12PagedKv* kv, int layers, const int32_t* src, const int32_t* dst, int count, void* stream)
{
    static const char* who = "s12_copy_pages_async";
    PagedArgs C = {};
    int rc = paged_cache_args(C, kv, who);
    if (rc) return rc;
    if (layers < 1 || layers > 65535 || count < 0) return fail(S12_ERR_BAD_ARG, "%s: layers %d, count %d", who, layers, count);
    if (count == 0) return S12_OK;
    if (!src || !dst) return fail(S12_ERR_BAD_ARG, "%s: null argument", who);
    CopyParams P = {};
    P.part[0] = (uint4*)kv->k; P.part[1] = (uint4*)kv->v; P.part[2] = (uint4*)kv->scale_k; P.part[3] = (uint4*)kv->scale_v;
    const long long rows = (long long)kv->n_head_kv * kv->page_size, units = rows * kv->head_dim / 16 + rows / 4;
    P.units[0] = (uint32_t)(rows * kv->head_dim / 16); P.units[1] = (uint32_t)(rows / 4);
    const long long chunks = (2 * units + kCopyThreads * kCopyUnits - 1) / (kCopyThreads * kCopyUnits);
    if (units > (1 << 29) || chunks * count > 0x7FFFFFFF) return fail(S12_ERR_TOO_LARGE, "%s: %d pages of %lld bytes", who, count, 32 * units);
    if ((rc = paged_status(C, who)) != S12_OK) return rc;
    P.chunks = (uint32_t)chunks; P.src = src; P.dst = dst; P.status = C.status; P.num_pages = kv->num_pages;
    return launch(paged_copy_kernel, dim3((unsigned)(chunks * count), layers), dim3(kCopyThreads), 0, stream, who, P);
}

int64_t s12_attention_paged_workspace_bytes(int n_head, int n_head_kv, int head_dim, int num_seqs, int max_new)
{
    if (n_head < 1 || n_head_kv < 1 || head_dim < 1 || num_seqs < 1 || max_new < 1)
        return fail(S12_ERR_BAD_ARG, "s12_attention_paged_workspace_bytes: sizes must be positive");
    if (n_head % n_head_kv) return fail(S12_ERR_UNSUPPORTED, "s12_attention_paged_workspace_bytes: n_head is not a multiple of n_head_kv");
    return paged_decode_workspace_bytes(n_head, n_head_kv, num_seqs, max_new);
}

int s12_attention_paged_async(const float* q, int q_stride, const S12PagedKv* kv, const S12PagedBatch* batch, void* out_bf16,
                              int out_stride, int n_head, float scale, void* workspace, int64_t workspace_bytes, void* stream)
{
    static const char* who = "s12_attention_paged_async";
    PagedAttn P = {};
    int rc = paged_cache_args(P.c, kv, who);
    if (!rc) rc = paged_batch_args(P.c, batch, n_head, who);
    if (rc) return rc;
    if (!q || !out_bf16) return fail(S12_ERR_BAD_ARG, "%s: null argument", who);
    if (q_stride < n_head * kv->head_dim || out_stride < n_head * kv->head_dim || batch->max_new < 1 || batch->max_len < 1 || !std::isfinite(scale))
        return fail(S12_ERR_BAD_ARG, "%s: a row stride shorter than the row, max_new or max_len below 1, or a scale that is not finite", who);
    if ((rc = paged_status(P.c, who)) != S12_OK) return rc;
    P.q = q; P.out = (int16_t*)out_bf16; P.q_stride = q_stride; P.out_stride = out_stride; P.n_head = n_head; P.scale = scale;
    P.max_new = batch->max_new; P.c.max_len = std::min(batch->max_len, kPagedMostPositions); P.workspace = workspace; P.workspace_bytes = workspace_bytes;
    if ((rc = paged_decode_launch(P, stream, who)) <= 0 || (rc = paged_prompt_launch(P, stream, who)) <= 0) return rc;
    return launch(paged_attention_general_kernel, dim3(batch->num_tokens, n_head), dim3(kGenWarps * 32), 0, stream, who, P);
}

}  // extern "C"
