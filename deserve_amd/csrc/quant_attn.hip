// Attention of a step's rows over pages of 8-bit K/V: what tree_attn.hip computes, with k_j = code * scale of its block and v_j alike.
// A token that an append took for no number has K codes that are none: its score is none either, which reaches the rows that see it and, chosen
// away by the mask, no others.  V codes are numbers.
#include "quant_wide_kernel.h"

#include <algorithm>

namespace dskv {

// Any type and head dim: one workgroup per (row, q head) whose waves take every kQuantWaves-th group of four keys.  Lane
// (g, c) holds dims 8 c .. 8 c + 7 (and 128 more ..) of key g of the group.  Bound by the latency of its loads: K and V are read once per row and q
// head, from the caches but for the first time (64 requests of one row over 256 - 4096 tokens, 32 heads over 8, 80 dims: 501 us, of five rows 1460).
constexpr int kQuantWaves = 8;

template <int DT, int kChunks>
__global__ __launch_bounds__(kQuantWaves * 64) void quant_generic_kernel(QuantArgs a)
{
    constexpr int E = DT == DSKV_F32 ? 4 : 2;                    // bytes of an element of q and out
    const int t = blockIdx.x, h = blockIdx.y;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
    const int b = request_of_row(a.qo_indptr, a.batch, t);
    if (b < 0) return;
    const int first = a.qo_indptr[b], i = t - first;
    if (i < 0 || i >= a.max_rows) return;
    const int page0 = a.kv_page_indptr[b];
    const TreeTokens tokens = tree_tokens(page0, a.kv_page_indptr[b + 1], a.kv_last_page_lens[b], a.page_size, a.n_page_indices);
    const long prior = tokens.len - ((long)a.qo_indptr[b + 1] - first);
    const unsigned long long mask = a.masks ? (unsigned long long)a.masks[t] : 0;
    const long seen = a.masks ? tokens.walk : min(tokens.walk, prior + i + 1);
    const int kv_head = h / (a.n_qo_heads / a.n_kv_heads);
    const char *const block = a.pages + kv_head * a.head_bytes, *const scales = a.pages + 2 * a.half_bytes + kv_head * 4;
    float q[kChunks][8], o[kChunks][8];
#pragma unroll
    for (int k = 0; k < kChunks; k++)
#pragma unroll
        for (int d = 0; d < 8; d++) q[k][d] = o[k][d] = 0;
#pragma unroll
    for (int k = 0; k < kChunks; k++)
        if (k * 128 + c * 8 < a.head_dim) {
            const char *p = a.q + t * a.q_stride + ((long)h * a.head_dim + k * 128 + c * 8) * E;
            Chunk<DT>::unpack(*reinterpret_cast<const u32x4 *>(p), q[k]);
            if constexpr (E == 4) Chunk<DT>::unpack(*reinterpret_cast<const u32x4 *>(p + 16), q[k] + 4);
        }
    float m = -INFINITY, l = 0;
    for (long j = wave * 4 + g; j - g < seen; j += kQuantWaves * 4) {
        bool there = j < seen;
        if (there && a.masks && j >= prior) there = j - prior < DSKV_MAX_TREE_ROWS && (mask >> (j - prior)) & 1;
        long page = -1;
        if (there) {
            const long entry = page0 + j / a.page_size;
            if (entry >= 0 && entry < a.n_page_indices) page = a.kv_page_indices[entry];
        }
        there = page >= 0 && page < a.num_pages;
        const long record = (there ? page : 0) * a.page_bytes;
        const char *key = block + record + (there ? j % a.page_size : 0) * a.head_dim;
        float s = 0, v[kChunks][8];
#pragma unroll
        for (int k = 0; k < kChunks; k++) {
#pragma unroll
            for (int d = 0; d < 8; d++) v[k][d] = 0;
            if (there && k * 128 + c * 8 < a.head_dim) {
                float x[8];
                decode8(*reinterpret_cast<const u32x2 *>(key + k * 128 + c * 8), x);
                decode8(*reinterpret_cast<const u32x2 *>(key + a.half_bytes + k * 128 + c * 8), v[k]);
#pragma unroll
                for (int d = 0; d < 8; d++) s = fmaf(q[k][d], x[d], s);
            }
        }
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) s += __shfl_xor(s, x);
        if (there) {
            const float *scale = reinterpret_cast<const float *>(scales + record);
            s *= scale[0] * a.scale;
            const float top = fmaxf(m, s);
            const float base = top == -INFINITY ? 0.f : top;
            const float keep = __builtin_amdgcn_exp2f(m - base), p = __builtin_amdgcn_exp2f(s - base), pv = p * scale[a.n_kv_heads];
            m = top;
            l = l * keep + p;
#pragma unroll
            for (int k = 0; k < kChunks; k++)
#pragma unroll
                for (int d = 0; d < 8; d++) o[k][d] = fmaf(o[k][d], keep, pv * v[k][d]);
        }
    }
    // the 4 * kQuantWaves running sums meet in LDS
    __shared__ float ms[kQuantWaves * 4], ls[kQuantWaves * 4];
    __shared__ float os[kQuantWaves * 4][kChunks * 128 + 4];
    const int part = wave * 4 + g;
    if (c == 0) {
        ms[part] = m;
        ls[part] = l;
    }
#pragma unroll
    for (int k = 0; k < kChunks; k++)
#pragma unroll
        for (int d = 0; d < 8; d++) os[part][k * 128 + c * 8 + d] = o[k][d];
    __syncthreads();
    float top = -INFINITY;
    for (int p = 0; p < kQuantWaves * 4; p++) top = fmaxf(top, ms[p]);
    const float base = top == -INFINITY ? 0.f : top;
    for (int d = threadIdx.x; d < a.head_dim; d += kQuantWaves * 64) {
        float sum = 0, acc = 0;
        for (int p = 0; p < kQuantWaves * 4; p++) {
            const float w = __builtin_amdgcn_exp2f(ms[p] - base);
            sum += ls[p] * w;
            acc += os[p][d] * w;
        }
        LoadElt<DT>::put(a.out, ((long)t * a.n_qo_heads + h) * a.head_dim + d, sum > 0 ? acc / sum : sum == 0 ? 0.f : NAN);
    }
}

// How rows of a step are computed.  wide_waves > 0: quant_wide_kernel.h with so many waves that have columns; else quant_kernel.h with tiles of
// `blocks` * 16 columns, few and each as narrow as it can be.
struct QuantForm {
    int wide_waves, blocks, cols, shares, sides;
    long col_tiles;                     // (of max_qo_len rows, which may be any number)
};
constexpr int kQuantUnits = 256;        // compute units
static bool quant_matrix_form(int head_dim) { return head_dim == 64 || head_dim == 128; }
static QuantForm quant_form(bool wide, int max_rows, int n_qo_heads, int n_kv_heads, int head_dim, int dtype)
{
    QuantForm f;
    const long cols = (long)std::max(max_rows, 1) * (n_qo_heads / n_kv_heads);
    f.wide_waves = !wide ? 0 : head_dim == 128 && cols <= 64 ? 2 : cols <= 128 ? 4 : 8;
    const int widest = wide ? f.wide_waves * 32 : quant_columns(dtype, head_dim);
    f.col_tiles = (cols + widest - 1) / widest;
    f.blocks = wide ? 0 : (int)((cols + 16 * f.col_tiles - 1) / (16 * f.col_tiles));
    f.cols = wide ? widest : f.blocks * 16;
    const int resident = kQuantUnits * (wide ? (f.wide_waves <= 4 ? 2 : 1) : quant_workgroups(dtype, head_dim, f.blocks));
    f.shares = resident >= n_kv_heads ? resident / n_kv_heads : 1;
    if (f.shares > 8) f.shares = f.shares / 8 * 8;         // (see share_and_head)
    f.sides = wide && f.col_tiles > 1 && f.shares % (8 * f.col_tiles) == 0 ? f.col_tiles : 1;
    return f;
}
// Requests of so many rows and fewer are the narrow form's, the others the wide one's, whose waves share what they read.  Single rows of more columns
// than its tiles hold are in several of them: 64 requests, 64 heads over one, 27.5 us; wide 34.0.  Where a step has both, the narrow
// form's are those for one block of 16 columns, which would be padded to more beside a chunk, or for as many blocks as one row has in a
// tile: 32 rows and a chunk of 300, 64 heads over one, all wide 57 us; else 66.
static int narrow_rows(int max_rows, int n_qo_heads, int n_kv_heads, int head_dim, int dtype)
{
    if (dtype == DSKV_F32) return INT32_MAX;
    const int group = n_qo_heads / n_kv_heads, fit = quant_columns(dtype, head_dim) / group;
    return max_rows <= std::max(fit, 1) ? std::max(fit, 1) : std::max(16 / group, std::min(fit, 1));
}
static int64_t units_bytes(int batch) { return ((int64_t)batch + 7) / 4 * 16; }
static int64_t slots_of(const QuantForm &f, int n_kv_heads) { return 2LL * f.shares * n_kv_heads * f.cols; }
static int64_t cuts_bytes(const QuantForm &f) { return (2LL * f.shares * (int64_t)sizeof(QuantCut) + 15) / 16 * 16; }
static int64_t form_bytes(const QuantForm &f, int batch, int n_kv_heads, int head_dim)
{
    return units_bytes(batch) + cuts_bytes(f) + slots_of(f, n_kv_heads) * (head_dim + 2) * (int64_t)sizeof(float);
}

template <int DT, int kD, int kBlocks> static int launch_quant(const QuantArgs &a, const QuantForm &f, hipStream_t stream)
{
    hipLaunchKernelGGL((quant_matrix_kernel<DT, kD, kBlocks>), dim3((unsigned)(f.shares * a.n_kv_heads)), dim3(kTreeThreads), 0, stream, a);
    DSKV_LAUNCH_CHECK("quant_matrix_kernel");
    return 0;
}
template <int DT, int kD, int kWaves, int kFetch> static int launch_quant_wide(const QuantArgs &a, const QuantForm &f, hipStream_t stream)
{
    hipLaunchKernelGGL((quant_wide_kernel<DT, kD, kWaves, kFetch>), dim3((unsigned)(f.shares * a.n_kv_heads)), dim3(kWaves * 64), 0, stream, a);
    DSKV_LAUNCH_CHECK("quant_wide_kernel");
    constexpr int kCols = QuantWide<kD, kWaves, kFetch>::kCols, kColumns = 256 / (kD / 4);
    auto merge = [&](auto kernel, int each) {
        const dim3 grid((unsigned)((kCols + kColumns * each - 1) / (kColumns * each)), (unsigned)a.n_kv_heads, (unsigned)(2 * f.shares));
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, a);
    };
    // Items of many parts: eight of them together and a column a thread.  One request of 12 rows over 4000 tokens 5.0 us, with four columns and two parts
    // 8.6; two over 16 K 9.4, 17.9; 8 of 64 rows over 4 - 8 K, four parts an item, 10.9, 9.7.
    if (f.shares > 4L * a.batch * f.col_tiles) merge(quant_merge_kernel<DT, kD, kCols, 1, 8>, 1);
    else merge(quant_merge_kernel<DT, kD, kCols, 4, 2>, 4);
    DSKV_LAUNCH_CHECK("quant_merge_kernel");
    return 0;
}
template <int DT, int kD> static int launch_quant_blocks(const QuantArgs &a, const QuantForm &f, hipStream_t stream)
{
    if constexpr (DT != DSKV_F32) {
        if constexpr (kD == 128)
            if (f.wide_waves == 2) return launch_quant_wide<DT, kD, 4, 2>(a, f, stream);
        if (f.wide_waves == 4) return launch_quant_wide<DT, kD, 4, 0>(a, f, stream);
        if (f.wide_waves == 8) return launch_quant_wide<DT, kD, 8, 0>(a, f, stream);
    }
    switch (f.blocks) {
    case 1: return launch_quant<DT, kD, 1>(a, f, stream);
    case 2: return launch_quant<DT, kD, 2>(a, f, stream);
    case 3:
        if constexpr (quant_columns(DT, kD) >= 48) return launch_quant<DT, kD, 3>(a, f, stream);
        break;
    case 4:
        if constexpr (quant_columns(DT, kD) >= 64) return launch_quant<DT, kD, 4>(a, f, stream);
        break;
    }
    set_error("quant_attn: no form for %d columns", f.cols);
    return DSKV_E_INVAL;
}
template <int DT> static int launch_quant_dim(const QuantArgs &a, const QuantForm &f, hipStream_t stream)
{
    return a.head_dim == 64 ? launch_quant_blocks<DT, 64>(a, f, stream) : launch_quant_blocks<DT, 128>(a, f, stream);
}
// The requests of rows_from .. rows_to rows, in form f.
static int launch_quant_form(QuantArgs a, const QuantForm &f, int dtype, int rows_from, int rows_to, void *workspace, hipStream_t stream)
{
    a.units_before = (int32_t *)workspace;
    a.cuts = (QuantCut *)((char *)workspace + units_bytes(a.batch));
    a.part_o = (float *)((char *)a.cuts + cuts_bytes(f));
    a.part_ml = a.part_o + slots_of(f, a.n_kv_heads) * a.head_dim;
    a.n_shares = f.shares;
    a.sides = f.sides;
    a.rows_from = rows_from;
    a.rows_to = rows_to;
    if (dtype == DSKV_F32) return launch_quant_dim<DSKV_F32>(a, f, stream);
    if (dtype == DSKV_F16) return launch_quant_dim<DSKV_F16>(a, f, stream);
    return launch_quant_dim<DSKV_BF16>(a, f, stream);
}

}  // namespace dskv

extern "C" int64_t dskv_quant_attn_workspace(int32_t batch, int32_t nnz, int32_t max_qo_len, int32_t n_qo_heads,
                                             int32_t n_kv_heads, int32_t head_dim, int32_t dtype)
{
    using namespace dskv;
    if (batch <= 0 || nnz <= 0 || max_qo_len <= 0 || n_kv_heads <= 0 || n_qo_heads < n_kv_heads || !quant_matrix_form(head_dim)) return 0;
    const int narrow_most = narrow_rows(max_qo_len, n_qo_heads, n_kv_heads, head_dim, dtype);
    const int64_t narrow = form_bytes(quant_form(false, max_qo_len < narrow_most ? max_qo_len : narrow_most, n_qo_heads, n_kv_heads, head_dim, dtype),
                                      batch, n_kv_heads, head_dim);
    if (max_qo_len <= narrow_most) return narrow;
    const int64_t wide = form_bytes(quant_form(true, max_qo_len, n_qo_heads, n_kv_heads, head_dim, dtype), batch, n_kv_heads, head_dim);
    return narrow > wide ? narrow : wide;
}

// two for each share and kv head: workgroups are two a compute unit at most, or one for each head
extern "C" int64_t dskv_quant_attn_counters(int32_t n_kv_heads)
{
    return n_kv_heads <= 0 ? 0 : 2 * (int64_t)std::max(2 * dskv::kQuantUnits, (int)n_kv_heads);
}

extern "C" int dskv_quant_attn(const dskv_quant_step_t *step, void *out, const void *q, int64_t q_stride,
                               const void *pages_layer, void *stream)
{
    using namespace dskv;
    DSKV_REQUIRE(step, "quant_attn: null arguments");
    const dskv_tree_step_t *s = &step->step;
    DSKV_REQUIRE(s->batch >= 0 && s->nnz >= 0 && s->max_qo_len >= 0 && step->min_qo_len >= 0, "quant_attn: negative batch, nnz or rows");
    DSKV_REQUIRE(s->dtype == DSKV_F32 || s->dtype == DSKV_F16 || s->dtype == DSKV_BF16, "quant_attn: unknown dtype %d", s->dtype);
    DSKV_REQUIRE(s->n_kv_heads > 0 && s->n_qo_heads > 0 && s->n_qo_heads % s->n_kv_heads == 0,
                 "quant_attn: n_qo_heads %d must be a multiple of n_kv_heads %d", s->n_qo_heads, s->n_kv_heads);
    DSKV_REQUIRE(s->head_dim > 0 && s->head_dim % 8 == 0 && s->head_dim <= 256,
                 "quant_attn: head_dim %d must be a multiple of 8 up to 256", s->head_dim);
    DSKV_REQUIRE(s->page_size > 0 && s->num_pages > 0 && s->n_page_indices >= 0, "quant_attn: bad page shape");
    DSKV_REQUIRE(s->sm_scale > 0, "quant_attn: sm_scale must be positive");
    DSKV_REQUIRE(!s->masks || s->max_qo_len <= DSKV_MAX_TREE_ROWS, "quant_attn: masks hold %d rows a request, max_qo_len is %d",
                 DSKV_MAX_TREE_ROWS, s->max_qo_len);
    if (s->batch == 0 || s->nnz == 0 || s->max_qo_len == 0) return 0;
    const int size = s->dtype == DSKV_F32 ? 4 : 2;
    DSKV_REQUIRE(out && q && pages_layer && s->qo_indptr && s->kv_page_indptr && s->kv_last_page_lens &&
                 (s->kv_page_indices || s->n_page_indices == 0), "quant_attn: null pointer argument");
    DSKV_REQUIRE(q_stride >= (int64_t)s->n_qo_heads * s->head_dim, "quant_attn: rows of q overlap");
    DSKV_REQUIRE(((uintptr_t)out | (uintptr_t)q | (uintptr_t)pages_layer) % 16 == 0 && q_stride * size % 16 == 0,
                 "quant_attn: tensors and their rows must be 16-byte aligned");
    const QuantShape shape = quant_shape(s->num_pages, s->page_size, s->n_kv_heads, s->head_dim);
    QuantArgs a = {};
    (TreeArgs &)a = {s->qo_indptr, s->kv_page_indptr, s->kv_page_indices, s->kv_last_page_lens, s->masks, (char *)out,
                     (const char *)q, (const char *)pages_layer, (long)q_stride * size, (long)s->n_page_indices, s->batch,
                     s->nnz, s->max_qo_len, s->n_qo_heads, s->n_kv_heads, s->head_dim, s->page_size, s->num_pages,
                     s->sm_scale * 1.4426950408889634f};
    a.head_bytes = shape.head_bytes;
    a.half_bytes = shape.half_bytes;
    a.page_bytes = shape.page_bytes;
    hipStream_t st = (hipStream_t)stream;
    // two launches where some requests have few rows and others many, one after the other over the same workspace
    const int narrow_most = narrow_rows(s->max_qo_len, s->n_qo_heads, s->n_kv_heads, s->head_dim, s->dtype);
    const bool some_narrow = narrow_most > 0 && step->min_qo_len <= narrow_most, some_wide = s->max_qo_len > narrow_most;
    const QuantForm narrow = quant_form(false, some_wide ? narrow_most : s->max_qo_len, s->n_qo_heads, s->n_kv_heads, s->head_dim, s->dtype);
    const QuantForm wide = quant_form(true, s->max_qo_len, s->n_qo_heads, s->n_kv_heads, s->head_dim, s->dtype);
    const int64_t col_tiles = some_wide && wide.col_tiles > narrow.col_tiles ? wide.col_tiles : narrow.col_tiles;
    // (places in the pool, tokens of a request and units are numbered in 32 bits there)
    if (quant_matrix_form(s->head_dim) && s->num_pages * (shape.page_bytes / 16) < UINT32_MAX &&
        s->n_page_indices < kMostTokens / s->page_size &&
        col_tiles <= (INT32_MAX - 1) / (s->n_page_indices * s->page_size / 32 + 2LL * s->batch)) {
        const int64_t need = dskv_quant_attn_workspace(s->batch, s->nnz, s->max_qo_len, s->n_qo_heads, s->n_kv_heads, s->head_dim, s->dtype);
        if (!s->workspace || s->workspace_bytes < need) {
            set_error("quant_attn: workspace of %lld bytes, %lld are needed", (long long)s->workspace_bytes, (long long)need);
            return DSKV_E_NOMEM;
        }
        DSKV_REQUIRE((uintptr_t)s->workspace % 16 == 0, "quant_attn: the workspace must be 16-byte aligned");
        DSKV_REQUIRE((int64_t)s->batch * col_tiles < INT32_MAX && s->n_kv_heads <= 65535, "quant_attn: too large a batch");
        if (!step->counters || step->n_counters < dskv_quant_attn_counters(s->n_kv_heads)) {
            set_error("quant_attn: %lld counters, %lld are needed", (long long)step->n_counters, (long long)dskv_quant_attn_counters(s->n_kv_heads));
            return DSKV_E_NOMEM;
        }
        DSKV_REQUIRE((uintptr_t)step->counters % 4 == 0, "quant_attn: the counters must be 4-byte aligned");
        a.counters = step->counters;
        a.group = s->n_qo_heads / s->n_kv_heads;
        a.page_shift = 31 + ilog2(s->page_size);
        a.page_magic = (uint32_t)(((1ull << a.page_shift) + s->page_size - 1) / s->page_size);
        a.page16 = (uint32_t)(shape.page_bytes / 16);
        a.row16 = (uint32_t)(s->head_dim / 16);
        if (some_narrow || !some_wide)
            if (int rc = launch_quant_form(a, narrow, s->dtype, 0, some_wide ? narrow_most : INT32_MAX, s->workspace, st)) return rc;
        return some_wide ? launch_quant_form(a, wide, s->dtype, some_narrow ? narrow_most + 1 : 0, INT32_MAX, s->workspace, st) : 0;
    }
    DSKV_REQUIRE(s->n_qo_heads <= 65535, "quant_attn: at most 65535 heads");
    const dim3 grid((unsigned)s->nnz, (unsigned)s->n_qo_heads), block(kQuantWaves * 64);
#define DSKV_QUANT_GENERIC(DT)                                                                                 \
    do {                                                                                                       \
        if (s->head_dim <= 128) hipLaunchKernelGGL((quant_generic_kernel<DT, 1>), grid, block, 0, st, a);      \
        else hipLaunchKernelGGL((quant_generic_kernel<DT, 2>), grid, block, 0, st, a);                         \
    } while (0)
    if (s->dtype == DSKV_F32) DSKV_QUANT_GENERIC(DSKV_F32);
    else if (s->dtype == DSKV_F16) DSKV_QUANT_GENERIC(DSKV_F16);
    else DSKV_QUANT_GENERIC(DSKV_BF16);
#undef DSKV_QUANT_GENERIC
    DSKV_LAUNCH_CHECK("quant_generic_kernel");
    return 0;
}
