// Attention of a step's rows over the paged context and over the rows that they descend from: one pass over the
// keys with a running maximum m and sum l,
//   m' = max(m, s_j),  l' = l 2^(m - m') + 2^(s_j - m'),  O' = O 2^(m - m') + 2^(s_j - m') v_j,   out = O / l,
// with scores in units of log 2.  A place that a row does not see has score -infinity and weight 0; a row that
// sees nothing keeps l = 0 and gets zeros.
#include "rope_math.h"
#include "tree_wide_kernel.h"

namespace dskv {

// Any type and head dim: one workgroup per (row, q head) whose waves take every kGenericWaves-th group of four
// keys.  Lane (g, c) holds dims 8 c .. 8 c + 7 (and 128 more ..) of key g of the group.  Bound by the
// latency of its loads: K and V are read once per row and q head, from the caches but for the first time (64 requests of 5 rows
// over 256 - 4096 tokens, 128 dims, 1625 us where the matrix form takes 117): for head dims and sizes that the others do not take.
constexpr int kGenericWaves = 8;
constexpr int kTreeUnits = 256;        // compute units

template <int DT> __device__ __forceinline__ void load8(const char *p, float *f)
{
    typedef Chunk<DT> C;
    C::unpack(*reinterpret_cast<const u32x4 *>(p), f);
    if (C::kElems == 4) C::unpack(*reinterpret_cast<const u32x4 *>(p + 16), f + 4);
}

template <int DT, int kChunks>
__global__ __launch_bounds__(kGenericWaves * 64) void tree_generic_kernel(TreeArgs a)
{
    constexpr int E = DT == DSKV_F32 ? 4 : 2;                    // bytes of an element
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
    const long head_bytes = (long)a.head_dim * E, row_bytes = a.n_kv_heads * head_bytes;
    float q[kChunks][8], o[kChunks][8];
#pragma unroll
    for (int k = 0; k < kChunks; k++)
#pragma unroll
        for (int d = 0; d < 8; d++) q[k][d] = o[k][d] = 0;
#pragma unroll
    for (int k = 0; k < kChunks; k++)
        if (k * 128 + c * 8 < a.head_dim)
            load8<DT>(a.q + t * a.q_stride + h * head_bytes + (k * 128 + c * 8) * E, q[k]);
    float m = -INFINITY, l = 0;
    for (long j = wave * 4 + g; j - g < seen; j += kGenericWaves * 4) {
        bool there = j < seen;
        if (there && a.masks && j >= prior) there = j - prior < DSKV_MAX_TREE_ROWS && (mask >> (j - prior)) & 1;
        long page = -1;
        if (there) {
            const long entry = page0 + j / a.page_size;
            if (entry >= 0 && entry < a.n_page_indices) page = a.kv_page_indices[entry];
        }
        there = page >= 0 && page < a.num_pages;
        const char *key = a.pages + ((there ? page : 0) * 2 * a.page_size + (there ? j % a.page_size : 0)) * row_bytes +
                          kv_head * head_bytes;
        float s = 0, v[kChunks][8];
#pragma unroll
        for (int k = 0; k < kChunks; k++) {
#pragma unroll
            for (int d = 0; d < 8; d++) v[k][d] = 0;
            if (there && k * 128 + c * 8 < a.head_dim) {
                float x[8];
                load8<DT>(key + (k * 128 + c * 8) * E, x);
                load8<DT>(key + a.page_size * row_bytes + (k * 128 + c * 8) * E, v[k]);
#pragma unroll
                for (int d = 0; d < 8; d++) s = fmaf(q[k][d], x[d], s);
            }
        }
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) s += __shfl_xor(s, x);
        if (there) {
            s *= a.scale;
            const float top = fmaxf(m, s);
            const float base = top == -INFINITY ? 0.f : top;
            const float keep = __builtin_amdgcn_exp2f(m - base), p = __builtin_amdgcn_exp2f(s - base);
            m = top;
            l = l * keep + p;
#pragma unroll
            for (int k = 0; k < kChunks; k++)
#pragma unroll
                for (int d = 0; d < 8; d++) o[k][d] = fmaf(o[k][d], keep, p * v[k][d]);
        }
    }
    // the 4 * kGenericWaves running sums meet in LDS
    __shared__ float ms[kGenericWaves * 4], ls[kGenericWaves * 4];
    __shared__ float os[kGenericWaves * 4][kChunks * 128 + 4];
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
    for (int p = 0; p < kGenericWaves * 4; p++) top = fmaxf(top, ms[p]);
    const float base = top == -INFINITY ? 0.f : top;
    for (int d = threadIdx.x; d < a.head_dim; d += kGenericWaves * 64) {
        float sum = 0, acc = 0;
        for (int p = 0; p < kGenericWaves * 4; p++) {
            const float w = __builtin_amdgcn_exp2f(ms[p] - base);
            sum += ls[p] * w;
            acc += os[p][d] * w;
        }
        LoadElt<DT>::put(a.out, ((long)t * a.n_qo_heads + h) * a.head_dim + d, sum > 0 ? acc / sum : sum == 0 ? 0.f : NAN);
    }
}

// How a step is computed.  wide_waves > 0: tree_wide_kernel.h with so many waves; else the matrix form of tree_kernel.h with
// tiles of `blocks` * 16 columns, up to tree_columns: few tiles, each as narrow as it can be.
struct TreeForm {
    int wide_waves, blocks, cols, shares, sides;
    long col_tiles;                     // (of max_qo_len rows, which may be any number)
};
static bool matrix_form(int head_dim) { return head_dim == 64 || head_dim == 128; }
static TreeForm tree_form(bool wide, int max_rows, int n_qo_heads, int n_kv_heads, int head_dim)
{
    TreeForm f;
    const long cols = (long)max_rows * (n_qo_heads / n_kv_heads);
    f.wide_waves = !wide ? 0 : cols <= 128 ? 4 : 8;
    const int widest = wide ? f.wide_waves * 32 : tree_columns(head_dim);
    f.col_tiles = (cols + widest - 1) / widest;
    f.blocks = wide ? 0 : (int)((cols + 16 * f.col_tiles - 1) / (16 * f.col_tiles));
    f.cols = wide ? widest : f.blocks * 16;
    // two workgroups a compute unit where their registers and LDS allow it
    const int resident = kTreeUnits * (wide ? (f.wide_waves == 4 ? 2 : 1) : tree_workgroups(head_dim, f.blocks));
    f.shares = resident >= n_kv_heads ? resident / n_kv_heads : 1;
    if (f.shares > 8) f.shares = f.shares / 8 * 8;         // (see share_and_head)
    f.sides = wide && f.col_tiles > 1 && f.shares % (8 * f.col_tiles) == 0 ? f.col_tiles : 1;
    return f;
}
// More columns than a wave of the narrow form holds go to the wide one, which reads K and V once for all of them: 64
// requests of 13 rows (52 columns) over 4 K tokens each 214 us, narrow 372; of 12 rows 199 narrow, 213 wide (bf16, 32 heads over 8).
// Up to 128 columns by four waves, two workgroups a unit: 64 requests of 16 rows 214 us, by eight waves 218; more by
// eight: 16 trees of 48 rows over 160 K tokens in all (64 heads) 324 us, by four waves 368.  With 64 dims 64 requests of 20 rows (80
// columns) over 4 K tokens 130 us, narrow 211; of 16 rows 115 narrow, 129 wide.
static bool wide_form(int max_rows, int n_qo_heads, int n_kv_heads, int head_dim, int dtype)
{
    return dtype != DSKV_F32 && (long)max_rows * (n_qo_heads / n_kv_heads) > tree_columns(head_dim);
}
static int64_t units_bytes(int batch) { return ((int64_t)batch + 7) / 4 * 16; }
static int64_t slots_of(const TreeForm &f, int n_kv_heads) { return 2LL * f.shares * n_kv_heads * f.cols; }
static int64_t form_bytes(const TreeForm &f, int batch, int n_kv_heads, int head_dim)
{
    return units_bytes(batch) + slots_of(f, n_kv_heads) * (head_dim + 2) * (int64_t)sizeof(float);
}

template <int DT, int kD, int kCols, int kSub> static int launch_tree_merge(const TreeArgs &a, const TreeForm &f, hipStream_t stream)
{
    // few items are cut into many parts each, many into few: one request over 4 K tokens 16.5 us with four groups of parts and 20.1 with
    // one, 64 requests 183 with one and 190 with four
    const bool many_parts = (long)a.batch * f.col_tiles * 4 < f.shares;
    constexpr int kEach = kCols >= 128 ? 4 : 1;
    const int columns = 256 / (kD / 4) * (many_parts ? 1 : kEach) / (many_parts ? 4 : 1);
    const dim3 grid((unsigned)(a.batch * f.col_tiles), (unsigned)a.n_kv_heads, (unsigned)((kCols + columns - 1) / columns));
    if (many_parts) hipLaunchKernelGGL((tree_merge_kernel<DT, kD, kCols, kSub, 4, 1>), grid, dim3(256), 0, stream, a, (int)f.col_tiles);
    else hipLaunchKernelGGL((tree_merge_kernel<DT, kD, kCols, kSub, 1, kEach>), grid, dim3(256), 0, stream, a, (int)f.col_tiles);
    DSKV_LAUNCH_CHECK("tree_merge_kernel");
    return 0;
}
template <int DT, int kD, int kBlocks> static int launch_tree(const TreeArgs &a, const TreeForm &f, hipStream_t stream)
{
    typedef TreeShape<DT, kD, kBlocks> S;
    hipLaunchKernelGGL((tree_matrix_kernel<DT, kD, kBlocks>), dim3((unsigned)(f.shares * a.n_kv_heads)),
                       dim3(kTreeThreads), 0, stream, a);
    DSKV_LAUNCH_CHECK("tree_matrix_kernel");
    return launch_tree_merge<DT, kD, S::kCols, S::kSub>(a, f, stream);
}
template <int DT, int kD, int kWaves> static int launch_tree_wide(const TreeArgs &a, const TreeForm &f, hipStream_t stream)
{
    hipLaunchKernelGGL((tree_wide_kernel<DT, kD, kWaves>), dim3((unsigned)(f.shares * a.n_kv_heads)), dim3(kWaves * 64), 0, stream, a);
    DSKV_LAUNCH_CHECK("tree_wide_kernel");
    return launch_tree_merge<DT, kD, kWaves * 32, kWideBlock>(a, f, stream);
}
template <int DT, int kD> static int launch_tree_blocks(const TreeArgs &a, const TreeForm &f, hipStream_t stream)
{
    if constexpr (DT != DSKV_F32) {
        if (f.wide_waves == 4) return launch_tree_wide<DT, kD, 4>(a, f, stream);
        if (f.wide_waves == 8) return launch_tree_wide<DT, kD, 8>(a, f, stream);
    }
    switch (f.blocks) {
    case 1: return launch_tree<DT, kD, 1>(a, f, stream);
    case 2: return launch_tree<DT, kD, 2>(a, f, stream);
    case 3: return launch_tree<DT, kD, 3>(a, f, stream);
    default:
        if constexpr (tree_columns(kD) >= 64) return launch_tree<DT, kD, 4>(a, f, stream);
        set_error("tree_attn: no form for %d columns", f.cols);
        return DSKV_E_INVAL;
    }
}
template <int DT> static int launch_tree_dim(const TreeArgs &a, const TreeForm &f, hipStream_t stream)
{
    return a.head_dim == 64 ? launch_tree_blocks<DT, 64>(a, f, stream) : launch_tree_blocks<DT, 128>(a, f, stream);
}

}  // namespace dskv

extern "C" int64_t dskv_tree_attn_workspace(int32_t batch, int32_t nnz, int32_t max_qo_len, int32_t n_qo_heads,
                                            int32_t n_kv_heads, int32_t head_dim, int32_t dtype)
{
    using namespace dskv;
    if (batch <= 0 || nnz <= 0 || max_qo_len <= 0 || n_kv_heads <= 0 || n_qo_heads < n_kv_heads || !matrix_form(head_dim)) return 0;
    const int64_t narrow = form_bytes(tree_form(false, max_qo_len, n_qo_heads, n_kv_heads, head_dim), batch, n_kv_heads, head_dim);
    if (!wide_form(max_qo_len, n_qo_heads, n_kv_heads, head_dim, dtype)) return narrow;
    const int64_t wide = form_bytes(tree_form(true, max_qo_len, n_qo_heads, n_kv_heads, head_dim), batch, n_kv_heads, head_dim);
    return narrow > wide ? narrow : wide;
}

extern "C" int dskv_tree_attn(const dskv_tree_step_t *s, void *out, const void *q, int64_t q_stride,
                              const void *pages_layer, void *stream)
{
    using namespace dskv;
    DSKV_REQUIRE(s, "tree_attn: null arguments");
    DSKV_REQUIRE(s->batch >= 0 && s->nnz >= 0 && s->max_qo_len >= 0, "tree_attn: negative batch, nnz or rows");
    DSKV_REQUIRE(s->dtype == DSKV_F32 || s->dtype == DSKV_F16 || s->dtype == DSKV_BF16, "tree_attn: unknown dtype %d", s->dtype);
    DSKV_REQUIRE(s->n_kv_heads > 0 && s->n_qo_heads > 0 && s->n_qo_heads % s->n_kv_heads == 0,
                 "tree_attn: n_qo_heads %d must be a multiple of n_kv_heads %d", s->n_qo_heads, s->n_kv_heads);
    DSKV_REQUIRE(s->head_dim > 0 && s->head_dim % 8 == 0 && s->head_dim <= 256,
                 "tree_attn: head_dim %d must be a multiple of 8 up to 256", s->head_dim);
    DSKV_REQUIRE(s->page_size > 0 && s->num_pages > 0 && s->n_page_indices >= 0, "tree_attn: bad page shape");
    DSKV_REQUIRE(!s->masks || s->max_qo_len <= DSKV_MAX_TREE_ROWS, "tree_attn: masks hold %d rows a request, max_qo_len is %d",
                 DSKV_MAX_TREE_ROWS, s->max_qo_len);
    if (s->batch == 0 || s->nnz == 0 || s->max_qo_len == 0) return 0;
    const int size = s->dtype == DSKV_F32 ? 4 : 2;
    DSKV_REQUIRE(out && q && pages_layer && s->qo_indptr && s->kv_page_indptr && s->kv_last_page_lens &&
                 (s->kv_page_indices || s->n_page_indices == 0), "tree_attn: null pointer argument");
    DSKV_REQUIRE(q_stride >= (int64_t)s->n_qo_heads * s->head_dim, "tree_attn: rows of q overlap");
    DSKV_REQUIRE(((uintptr_t)out | (uintptr_t)q | (uintptr_t)pages_layer) % 16 == 0 && q_stride * size % 16 == 0,
                 "tree_attn: tensors and their rows must be 16-byte aligned");
    TreeArgs a = {s->qo_indptr, s->kv_page_indptr, s->kv_page_indices, s->kv_last_page_lens, s->masks, (char *)out,
                  (const char *)q, (const char *)pages_layer, (long)q_stride * size, (long)s->n_page_indices, s->batch,
                  s->nnz, s->max_qo_len, s->n_qo_heads, s->n_kv_heads, s->head_dim, s->page_size, s->num_pages,
                  s->sm_scale * 1.4426950408889634f};
    hipStream_t st = (hipStream_t)stream;
    const TreeForm f = tree_form(s->sm_scale > 0 && wide_form(s->max_qo_len, s->n_qo_heads, s->n_kv_heads, s->head_dim, s->dtype),
                                 s->max_qo_len, s->n_qo_heads, s->n_kv_heads, s->head_dim);
    // (rows of the pool, tokens of a request and units are numbered in 32 bits there)
    if (matrix_form(s->head_dim) && (int64_t)s->num_pages * 2 * s->page_size < INT32_MAX &&
        s->n_page_indices < kMostTokens / s->page_size && s->max_qo_len <= kTreeMostRows &&
        (s->n_page_indices * s->page_size / 16 + 2LL * s->batch) * f.col_tiles < INT32_MAX) {
        const int64_t need = dskv_tree_attn_workspace(s->batch, s->nnz, s->max_qo_len, s->n_qo_heads, s->n_kv_heads, s->head_dim, s->dtype);
        if (!s->workspace || s->workspace_bytes < need) {
            set_error("tree_attn: workspace of %lld bytes, %lld are needed", (long long)s->workspace_bytes, (long long)need);
            return DSKV_E_NOMEM;
        }
        DSKV_REQUIRE((uintptr_t)s->workspace % 16 == 0, "tree_attn: the workspace must be 16-byte aligned");
        DSKV_REQUIRE((int64_t)s->batch * f.col_tiles < INT32_MAX && s->n_kv_heads <= 65535, "tree_attn: too large a batch");
        a.units_before = (int32_t *)s->workspace;
        a.part_o = (float *)((char *)s->workspace + units_bytes(s->batch));
        a.part_ml = a.part_o + slots_of(f, s->n_kv_heads) * s->head_dim;
        a.n_shares = f.shares;
        a.sides = f.sides;
        a.group = s->n_qo_heads / s->n_kv_heads;
        a.page_shift = 31 + ilog2(s->page_size);
        a.page_magic = (uint32_t)(((1ull << a.page_shift) + s->page_size - 1) / s->page_size);
        if (s->dtype == DSKV_F32) return launch_tree_dim<DSKV_F32>(a, f, st);
        if (s->dtype == DSKV_F16) return launch_tree_dim<DSKV_F16>(a, f, st);
        return launch_tree_dim<DSKV_BF16>(a, f, st);
    }
    DSKV_REQUIRE(s->n_qo_heads <= 65535, "tree_attn: at most 65535 heads");
    const dim3 grid((unsigned)s->nnz, (unsigned)s->n_qo_heads), block(kGenericWaves * 64);
#define DSKV_TREE_GENERIC(DT)                                                                                  \
    do {                                                                                                       \
        if (s->head_dim <= 128) hipLaunchKernelGGL((tree_generic_kernel<DT, 1>), grid, block, 0, st, a);       \
        else hipLaunchKernelGGL((tree_generic_kernel<DT, 2>), grid, block, 0, st, a);                          \
    } while (0)
    if (s->dtype == DSKV_F32) DSKV_TREE_GENERIC(DSKV_F32);
    else if (s->dtype == DSKV_F16) DSKV_TREE_GENERIC(DSKV_F16);
    else DSKV_TREE_GENERIC(DSKV_BF16);
#undef DSKV_TREE_GENERIC
    DSKV_LAUNCH_CHECK("tree_generic_kernel");
    return 0;
}
