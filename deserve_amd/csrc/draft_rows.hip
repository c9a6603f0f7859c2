// Rows of a step by their slots: the append of new rows, rotated on their way, and the move of accepted ones.
// A slot is page id * page size + place in the page.
#include "rope_math.h"

namespace dskv {

// q and k rotated by their rows' angles, k and v into their slots.  Elementwise and bound by HBM: every row is
// read and written once.  One workgroup per row; a thread owns a 16-byte column of the head dimension, whose
// cosines and sines (the table's, the same for every layer and so not evaluated here) it loads once, and
// walks the heads.  The addresses depend on nothing but the slot, which is requested beside the rows.  4096 rows of 64 heads
// over 8 (fp16, 170 MB) 32 us, 5.3 TB/s; 320 rows of 32 heads 4.4 us, launch and three trips.
constexpr int kSlotHeads = 6;      // heads a thread has in flight

struct SlotRows {
    char *q_out, *pages;
    const char *q, *k, *v;
    long q_stride, k_stride, v_stride;   // bytes
    const int64_t *slots;
    const float *table;
    long n_slots;
    int page_size, n_qo_heads, n_kv_heads, head_dim;
};

template <int DT>
__global__ __launch_bounds__(256, 6) void append_slots_kernel(SlotRows a)
{
    typedef Chunk<DT> C;
    constexpr int E = C::kElems;
    const long t = blockIdx.x;
    const int cols = a.head_dim / E;
    const int col = threadIdx.x % cols, head_lane = threadIdx.x / cols, head_lanes = 256 / cols;
    const bool works = head_lane < head_lanes;
    const long head_bytes = (long)a.head_dim * (16 / E);
    const long row_bytes = a.n_kv_heads * head_bytes;
    const int q_heads = a.table ? a.n_qo_heads : 0;          // without rotation q stays where it is
    const int heads = q_heads + a.n_kv_heads;
    auto source = [&](int h) {
        return h < q_heads ? a.q + t * a.q_stride + h * head_bytes + col * 16
                           : a.k + t * a.k_stride + (h - q_heads) * head_bytes + col * 16;
    };
    const long slot = a.slots[t];
    u32x4 raw[kSlotHeads], v_raw = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kSlotHeads; i++) {
        const int h = head_lane + i * head_lanes;
        if (works && h < heads) raw[i] = *reinterpret_cast<const u32x4 *>(source(h));
    }
    const char *v_row = a.v + t * a.v_stride;
    if (threadIdx.x * 16L < row_bytes) v_raw = *reinterpret_cast<const u32x4 *>(v_row + threadIdx.x * 16L);
    float cs[E / 2], sn[E / 2];
    if (a.table && works) {
        typedef float Half __attribute__((ext_vector_type(E / 2)));
        const float *cosines = a.table + t * a.head_dim + col * (E / 2);
        const Half c = *reinterpret_cast<const Half *>(cosines), s = *reinterpret_cast<const Half *>(cosines + a.head_dim / 2);
#pragma unroll
        for (int j = 0; j < E / 2; j++) {
            cs[j] = c[j];
            sn[j] = s[j];
        }
    }
    const bool there = slot >= 0 && slot < a.n_slots;
    const long page = there ? slot / a.page_size : 0;
    char *k_dst = a.pages + (page * a.page_size + slot) * row_bytes;      // page * 2 P + slot - page * P
    char *v_dst = k_dst + a.page_size * row_bytes;
    auto put = [&](int h, u32x4 chunk) {
        if (h >= q_heads && !there) return;
        if (a.table) {
            float f[E];
            C::unpack(chunk, f);
            rope_rotate<E / 2>(f, cs, sn);
            chunk = C::pack(f);
        }
        char *dst = h < q_heads ? a.q_out + (t * a.n_qo_heads + h) * head_bytes + col * 16
                                : k_dst + (h - q_heads) * head_bytes + col * 16;
        *reinterpret_cast<u32x4 *>(dst) = chunk;
    };
    if (works) {
#pragma unroll
        for (int i = 0; i < kSlotHeads; i++) {
            const int h = head_lane + i * head_lanes;
            if (h < heads) put(h, raw[i]);
        }
        for (int h = head_lane + kSlotHeads * head_lanes; h < heads; h += head_lanes)
            put(h, *reinterpret_cast<const u32x4 *>(source(h)));
    }
    if (there) {
        if (threadIdx.x * 16L < row_bytes) *reinterpret_cast<u32x4 *>(v_dst + threadIdx.x * 16L) = v_raw;
        for (long off = threadIdx.x * 16L + 256 * 16; off < row_bytes; off += 256 * 16)
            *reinterpret_cast<u32x4 *>(v_dst + off) = *reinterpret_cast<const u32x4 *>(v_row + off);
    }
}

// Moves of accepted rows, one workgroup per (request, layer).  Row j of the walk comes from row path[j] >= j, and a
// row is never the target of an earlier j and the source of a later one: path[j'] > path[j] >= j for j' > j.  A thread
// owns the same 16 bytes of every row, so that rows may be requested several at a time and written in order.
// 64 requests of 16 - 64 rows, 32 layers: 13 us for 49 MB; one request of 16 layers 3.6 us, a chain of trips.
constexpr int kMoveRows = 8;

struct MoveRows {
    char *pages;
    long layer_stride, row_bytes, n_slots;
    const int64_t *slots;
    const int32_t *qo_indptr, *path, *counts;
    int page_size, nnz;
};

__global__ __launch_bounds__(256) void move_rows_kernel(MoveRows a)
{
    const int b = blockIdx.x;
    const long first = a.qo_indptr[b], n = a.qo_indptr[b + 1] - first;
    const long count = min((long)a.counts[b], n);
    if (first < 0 || first + n > a.nnz || count < 2) return;
    __shared__ long from[256], to[256];
    char *layer = a.pages + blockIdx.y * a.layer_stride;
    for (long j0 = 1; j0 < count; j0 += 256) {
        const long j = j0 + threadIdx.x;
        long src = -1, dst = -1;
        if (j < count) {
            const long p = a.path[first + j];
            if (p > j && p < n && p > a.path[first + j - 1]) {
                src = a.slots[first + p];
                dst = a.slots[first + j];
            }
        }
        if (src < 0 || src >= a.n_slots || dst < 0 || dst >= a.n_slots) src = -1;
        __syncthreads();
        from[threadIdx.x] = src < 0 ? -1 : (src / a.page_size * a.page_size + src) * a.row_bytes;
        to[threadIdx.x] = src < 0 ? 0 : (dst / a.page_size * a.page_size + dst) * a.row_bytes;
        __syncthreads();
        const int held = (int)min(count - j0, 256L);
        const long half = a.page_size * a.row_bytes;
        for (long c = threadIdx.x * 16L; c < 2 * a.row_bytes; c += 256 * 16) {
            const long at = c < a.row_bytes ? c : c - a.row_bytes + half;
            for (int i0 = 0; i0 < held; i0 += kMoveRows) {
                u32x4 raw[kMoveRows];
#pragma unroll
                for (int i = 0; i < kMoveRows; i++)
                    if (i0 + i < held && from[i0 + i] >= 0)
                        raw[i] = *reinterpret_cast<const u32x4 *>(layer + from[i0 + i] + at);
#pragma unroll
                for (int i = 0; i < kMoveRows; i++)
                    if (i0 + i < held && from[i0 + i] >= 0) *reinterpret_cast<u32x4 *>(layer + to[i0 + i] + at) = raw[i];
            }
        }
    }
}

}  // namespace dskv

extern "C" int dskv_rope_append_slots(void *q_out, void *pages_layer, int32_t num_pages, const void *q,
                                      const void *k, const void *v, int64_t q_stride, int64_t k_stride,
                                      int64_t v_stride, const int64_t *slots, const float *rope_table, int32_t nnz,
                                      int32_t page_size, int32_t n_qo_heads, int32_t n_kv_heads, int32_t head_dim,
                                      int32_t dtype, void *stream)
{
    using namespace dskv;
    DSKV_REQUIRE(nnz >= 0, "rope_append_slots: negative nnz");
    if (nnz == 0) return 0;
    DSKV_REQUIRE(pages_layer && k && v && slots && (!rope_table || (q && q_out)), "rope_append_slots: null pointer argument");
    DSKV_REQUIRE(dtype == DSKV_F32 || dtype == DSKV_F16 || dtype == DSKV_BF16, "rope_append_slots: unknown dtype %d", dtype);
    const int elems = dtype == DSKV_F32 ? 4 : 8, size = dtype == DSKV_F32 ? 4 : 2;
    DSKV_REQUIRE(head_dim > 0 && head_dim % elems == 0 && head_dim / elems <= 256,
                 "rope_append_slots: head_dim %d must be a multiple of %d and at most %d", head_dim, elems, 256 * elems);
    DSKV_REQUIRE(n_qo_heads > 0 && n_kv_heads > 0 && page_size > 0 && num_pages > 0, "rope_append_slots: bad shape");
    DSKV_REQUIRE((!rope_table || q_stride >= (int64_t)n_qo_heads * head_dim) && k_stride >= (int64_t)n_kv_heads * head_dim &&
                 v_stride >= (int64_t)n_kv_heads * head_dim, "rope_append_slots: rows overlap");
    DSKV_REQUIRE((((uintptr_t)q_out | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)pages_layer | (uintptr_t)rope_table) % 16 == 0) &&
                 ((rope_table ? q_stride : 0) | k_stride | v_stride) * size % 16 == 0,
                 "rope_append_slots: tensors and their rows must be 16-byte aligned");
    SlotRows a = {(char *)q_out, (char *)pages_layer, (const char *)q, (const char *)k, (const char *)v,
                  (long)q_stride * size, (long)k_stride * size, (long)v_stride * size, slots, rope_table,
                  (long)num_pages * page_size, page_size, n_qo_heads, n_kv_heads, head_dim};
    hipStream_t s = (hipStream_t)stream;
    if (dtype == DSKV_F32) hipLaunchKernelGGL((append_slots_kernel<DSKV_F32>), dim3((unsigned)nnz), dim3(256), 0, s, a);
    else if (dtype == DSKV_F16) hipLaunchKernelGGL((append_slots_kernel<DSKV_F16>), dim3((unsigned)nnz), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((append_slots_kernel<DSKV_BF16>), dim3((unsigned)nnz), dim3(256), 0, s, a);
    DSKV_LAUNCH_CHECK("append_slots_kernel");
    return 0;
}

extern "C" int dskv_move_rows(void *pages, int64_t layer_stride_bytes, int32_t n_layers, int32_t num_pages,
                              int32_t page_size, int64_t row_bytes, const int64_t *slots, const int32_t *qo_indptr,
                              const int32_t *path, const int32_t *counts, int32_t batch, int32_t nnz, void *stream)
{
    using namespace dskv;
    DSKV_REQUIRE(batch >= 0 && nnz >= 0 && n_layers >= 0, "move_rows: negative batch, nnz or layers");
    if (batch == 0 || nnz == 0 || n_layers == 0) return 0;
    DSKV_REQUIRE(pages && slots && qo_indptr && path && counts, "move_rows: null pointer argument");
    DSKV_REQUIRE(num_pages > 0 && page_size > 0, "move_rows: bad page shape");
    DSKV_REQUIRE(row_bytes > 0 && row_bytes % 16 == 0, "move_rows: row_bytes must be a multiple of 16");
    DSKV_REQUIRE(n_layers <= 65535, "move_rows: at most 65535 layers a call");
    DSKV_REQUIRE((uintptr_t)pages % 16 == 0 && layer_stride_bytes % 16 == 0, "move_rows: pages must be 16-byte aligned");
    DSKV_REQUIRE(n_layers == 1 || layer_stride_bytes >= 2 * (int64_t)num_pages * page_size * row_bytes,
                 "move_rows: layers overlap");
    MoveRows a = {(char *)pages, (long)layer_stride_bytes, (long)row_bytes, (long)num_pages * page_size, slots,
                  qo_indptr, path, counts, page_size, nnz};
    hipLaunchKernelGGL(move_rows_kernel, dim3((unsigned)batch, (unsigned)n_layers), dim3(256), 0, (hipStream_t)stream, a);
    DSKV_LAUNCH_CHECK("move_rows_kernel");
    return 0;
}
