// What the kernels of the paged INT8 cache share: the cache and batch as they see them.
#pragma once
#include "common.cuh"

namespace s12 {

constexpr int kPagedMostPositions = 0x7FFFFFFF - 4096;     // of a sequence: positions of a step further stay below 2^31
constexpr unsigned int kStatusPage = 0x100000u;     // a block table entry outside the pool, or a position past the table

// A position t of sequence s lies in page table[s * table_stride + (t >> page_shift)], row t & (page_size - 1):
// codes at ((page * n_head_kv + kv head) * page_size + row) * head_dim, scales at the same index without head_dim.
struct PagedArgs {
    int8_t* k; int8_t* v; float* sk; float* sv;
    const int* table; const int* kv_len; const int* q_start;   // q_start null: token i belongs to sequence i
    unsigned int* status;
    int num_pages, page_shift, n_head_kv, head_dim;
    int num_seqs, table_stride, table_pages, num_tokens;
    int max_len;                // the caller's bound: positions from it on are masked
};

#ifdef __CUDACC__
__device__ __forceinline__ int16_t paged_bf16_rne(float v)
{
    uint16_t r;
    asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(v));
    return (int16_t)r;
}
// the page that holds position t of sequence s, -1 where the table has none (t inside the table)
__device__ __forceinline__ int paged_page(const PagedArgs& P, int s, int t)
{
    const int page = P.table[(size_t)s * P.table_stride + (t >> P.page_shift)];
    return (unsigned)page < (unsigned)P.num_pages ? page : -1;
}
// positions of sequence s inside the table and the caller's bound
__device__ __forceinline__ int paged_len(const PagedArgs& P, int s)
{
    const int n = P.kv_len[s];
    const long long room = min((long long)P.table_pages << P.page_shift, (long long)P.max_len);
    return n < 0 ? 0 : n < room ? n : (int)room;
}
// whether a row that sees n positions, by its place, needs pages past the table's end
__device__ __forceinline__ bool paged_past_table(const PagedArgs& P, int n) { return min(n, P.max_len) > (long long)P.table_pages << P.page_shift; }
// rows [lo, hi) of the packed tokens that belong to sequence s
__device__ __forceinline__ void paged_rows(const PagedArgs& P, int s, int& lo, int& hi)
{
    if (!P.q_start) { lo = s; hi = s + 1; return; }
    lo = P.q_start[s]; hi = P.q_start[s + 1];
    lo = lo < 0 ? 0 : lo; hi = hi < P.num_tokens ? hi : P.num_tokens;
}
// The sequence of packed token `row`, for a whole warp at once: the last s with q_start[s] <= row, or -1 where row lies
// outside [q_start[0], q_start[num_seqs]).  32 entries a round: two rounds up to 1023 sequences.
__device__ __forceinline__ int paged_seq_of(const PagedArgs& P, int row)
{
    if (!P.q_start) return row < P.num_seqs ? row : -1;
    const int lane = threadIdx.x & 31;
    int lo = 0, n = P.num_seqs + 1;                               // the entries looked at: [lo, lo + n)
    while (true) {
        const int step = (n + 31) >> 5, at = lane * step;
        const bool below = at < n && P.q_start[lo + at] <= row;
        const unsigned m = __ballot_sync(0xFFFFFFFFu, below);
        if (m == 0) return lo - 1;                                // only in the first round: before the first token
        const int last = 31 - __clz(m);
        lo += last * step;
        if (step == 1) break;
        n = n - last * step < step ? n - last * step : step;
    }
    return lo < P.num_seqs ? lo : -1;
}
#endif

// attention over the pages; each returns S12_OK, an error, or 1 where it does not take the shape
struct PagedAttn {
    PagedArgs c;
    const float* q; int16_t* out;
    int q_stride, out_stride, n_head;
    float scale;
    int max_new;                // the caller's bound on a sequence's new tokens
    void* workspace; int64_t workspace_bytes;
};
int64_t paged_decode_workspace_bytes(int n_head, int n_head_kv, int num_seqs, int max_new);
int paged_decode_launch(const PagedAttn& A, void* stream, const char* who);
int paged_prompt_launch(const PagedAttn& A, void* stream, const char* who);

}  // namespace s12
