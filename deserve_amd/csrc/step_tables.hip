// Block tables, slot map, positions and tree masks of a step, from lengths that live on the device.
//
// With len_b = kv_b + n_b (cached tokens and new rows of request b):
//   qo_indptr, kv_page_indptr   sums of n_b and of ceil(len_b / P);   last_b = (len_b - 1) mod P + 1
//   kv_page_indices             the first ceil(len_b / P) entries of the request's table row
//   slot(i)     = page((kv_b + i) / P) * P + (kv_b + i) mod P of new row i
//   mask(i)     = bit i, with the bits of the rows that i descends from
//   position(i) = kv_b + number of those rows; without a tree kv_b + i
//
// Bound by latency: lengths -> sums -> table row -> stores.  One workgroup per request, which takes the
// sums over all requests before it for itself (8 KB of lengths at 1024 requests, from L2): a launch in front that
// takes them once would cost more than that.  One request 3.8 us, 512 trees with half a million pages 7.7 (4.5 MB).  A tree's masks take six rounds of pointer doubling in one wave
// (after k rounds a row holds its 2^k nearest ancestors), since a row's parent has a smaller index.
#include "common.h"

namespace dskv {

constexpr int kTableThreads = 256;

struct Sums {
    long tokens, pages;
};

// What request b asks for; a request whose entries contradict each other or its table asks for nothing.
__device__ __forceinline__ void request_of(const dskv_step_tables_t &a, int b, long &kv, long &rows, long &pages,
                                           long &table_row)
{
    kv = a.kv_lens[b];
    rows = a.qo_lens[b];
    table_row = a.rows ? a.rows[b] : b;
    const bool fine = kv >= 0 && rows >= 0 && table_row >= 0 && table_row < a.table_rows &&
                      kv + rows <= (long)a.table_width * a.page_size && (!a.masks || rows <= DSKV_MAX_TREE_ROWS);
    if (!fine) kv = rows = 0;
    pages = (kv + rows + a.page_size - 1) / a.page_size;
}

// Sums up to and with this thread's entry over the workgroup, and the whole sum.
__device__ __forceinline__ Sums block_scan(Sums v, Sums &all, Sums *of_wave)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long t = __shfl_up(v.tokens, o), p = __shfl_up(v.pages, o);
        if (lane >= o) {
            v.tokens += t;
            v.pages += p;
        }
    }
    if (lane == 63) of_wave[wave] = v;
    __syncthreads();
    all = {0, 0};
#pragma unroll
    for (int w = 0; w < kTableThreads / 64; w++) {
        if (w == wave) {
            v.tokens += all.tokens;
            v.pages += all.pages;
        }
        all.tokens += of_wave[w].tokens;
        all.pages += of_wave[w].pages;
    }
    return v;
}

constexpr int kTableAhead = 8;          // table entries a thread requests before it knows where they go

__global__ __launch_bounds__(kTableThreads) void step_tables_kernel(dskv_step_tables_t a)
{
    __shared__ Sums of_wave[2][kTableThreads / 64], fit_of_wave[2][kTableThreads / 64];
    __shared__ int fits_in_wave[2][kTableThreads / 64];
    const int b = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    // the request's own entries first, and what of its table row they ask for: the sums below take as long
    long kv = 0, n = 0, pages = 0, table_row = 0;
    if (b < a.batch) request_of(a, b, kv, n, pages, table_row);
    const int32_t *table = a.page_tables + table_row * a.table_stride;
    int32_t held[kTableAhead], page_of_row = 0;
#pragma unroll
    for (int i = 0; i < kTableAhead; i++)
        if (t + i * kTableThreads < pages) held[i] = table[t + i * kTableThreads];
    if (t < n) page_of_row = table[(kv + t) / a.page_size];

    // Sums grow, so from the first request on that does not fit the arrays none does: it and all behind it get
    // nothing, and the entries stay at the sums of those that fit.
    Sums before = {0, 0}, fit = {0, 0};
    bool b_fits = false;
    for (int first = 0, turn = 0; first <= b && first < a.batch; first += kTableThreads, turn ^= 1) {
        const int r = first + t;
        const bool there = r <= b && r < a.batch;
        long r_kv, r_rows = 0, r_pages = 0, r_table;
        if (there) request_of(a, r, r_kv, r_rows, r_pages, r_table);
        Sums all;
        Sums upto = block_scan({r_rows, r_pages}, all, of_wave[turn]);
        upto.tokens += before.tokens;
        upto.pages += before.pages;
        const unsigned long long fits = __ballot(there && upto.tokens <= a.max_tokens && upto.pages <= a.max_pages);
        if (fits && lane == 63 - __builtin_clzll(fits)) fit_of_wave[turn][wave] = upto;
        if (lane == 0) fits_in_wave[turn][wave] = __popcll(fits);
        __syncthreads();
        int fitting = 0;
#pragma unroll
        for (int w = 0; w < kTableThreads / 64; w++)
            if (fits_in_wave[turn][w]) {
                fit = fit_of_wave[turn][w];
                fitting += fits_in_wave[turn][w];
            }
        b_fits = fitting > b - first;
        before.tokens += all.tokens;
        before.pages += all.pages;
    }
    if (!b_fits) kv = n = pages = 0;
    const long row0 = fit.tokens - n, page0 = fit.pages - pages;
    if (t == 0) {
        if (b == 0) a.qo_indptr[0] = a.kv_page_indptr[0] = 0;
        if (b < a.batch) {
            a.qo_indptr[b + 1] = (int32_t)fit.tokens;
            a.kv_page_indptr[b + 1] = (int32_t)fit.pages;
            a.kv_last_page_lens[b] = kv + n > 0 ? (int32_t)((kv + n - 1) % a.page_size) + 1 : 0;
        }
    }
    // a tree's parents lie by row, so they are requested last
    const bool tree = a.masks != nullptr;
    int up = -1;
    if (tree && t < n && row0 + t < a.n_parents) up = a.parents[row0 + t];
#pragma unroll
    for (int i = 0; i < kTableAhead; i++)
        if (t + i * kTableThreads < pages) a.kv_page_indices[page0 + t + i * kTableThreads] = held[i];
    for (long i = t + kTableAhead * kTableThreads; i < pages; i += kTableThreads) a.kv_page_indices[page0 + i] = table[i];
    for (long i = t; i < n; i += kTableThreads) {
        const long at = kv + i;
        const long page = i == t ? page_of_row : table[at / a.page_size];
        a.slots[row0 + i] = page < 0 ? -1 : page * a.page_size + at % a.page_size;
        if (!tree) a.positions[row0 + i] = (int32_t)at;
    }
    if (tree && wave == 0 && n > 0) {
        if (up >= t || up < 0) up = -1;            // a row without a parent among the rows before it
        unsigned long long mask = 1ull << t;
#pragma unroll
        for (int round = 0; round < 6; round++) {
            const unsigned long long theirs = __shfl(mask, max(up, 0));
            const int further = __shfl(up, max(up, 0));
            if (up >= 0) {
                mask |= theirs;
                up = further;
            }
        }
        if (t < n) {
            a.masks[row0 + t] = (int64_t)mask;
            a.positions[row0 + t] = (int32_t)(kv + __popcll(mask) - 1);
        }
    }
    // rows behind the last request have no slot
    if (b == (int)gridDim.x - 1)
        for (long i = fit.tokens + t; i < a.max_tokens; i += kTableThreads) {
            a.slots[i] = -1;
            a.positions[i] = 0;
            if (tree) a.masks[i] = 0;
        }
}

}  // namespace dskv

extern "C" int dskv_step_tables(const dskv_step_tables_t *a, void *stream)
{
    using namespace dskv;
    DSKV_REQUIRE(a, "step_tables: null arguments");
    DSKV_REQUIRE(a->batch >= 0 && a->max_tokens >= 0 && a->max_pages >= 0, "step_tables: negative batch or size");
    DSKV_REQUIRE(a->page_size > 0, "step_tables: page_size must be positive");
    DSKV_REQUIRE(a->table_rows >= 0 && a->table_width >= 0 && a->table_stride >= a->table_width,
                 "step_tables: bad table shape");
    DSKV_REQUIRE(a->qo_indptr && a->kv_page_indptr, "step_tables: null pointer argument");
    DSKV_REQUIRE(a->batch == 0 || (a->kv_lens && a->qo_lens && a->kv_last_page_lens), "step_tables: null pointer argument");
    DSKV_REQUIRE(a->table_rows == 0 || a->table_width == 0 || a->page_tables, "step_tables: null page tables");
    DSKV_REQUIRE(a->max_tokens == 0 || (a->slots && a->positions), "step_tables: null pointer argument");
    DSKV_REQUIRE(a->max_pages == 0 || a->kv_page_indices, "step_tables: null pointer argument");
    DSKV_REQUIRE(a->n_parents >= 0 && (a->n_parents == 0 || a->parents), "step_tables: null parents");
    hipLaunchKernelGGL(step_tables_kernel, dim3((unsigned)(a->batch > 0 ? a->batch : 1)), dim3(kTableThreads), 0,
                       (hipStream_t)stream, *a);
    DSKV_LAUNCH_CHECK("step_tables_kernel");
    return 0;
}
