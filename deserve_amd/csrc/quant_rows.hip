// Rows of a step into pages of 8-bit K/V: the append of new rows, rotated on their way, and the move of accepted ones.
#include "quant.h"
#include "rope_math.h"

#include <algorithm>

namespace dskv {

// Requests of a step: their rows' places, from the index arrays and within the bounds of the tensors.
struct QuantRows {
    const int32_t *qo_indptr, *kv_page_indices, *kv_page_indptr, *kv_last_page_lens;
    long n_page_indices;
    int batch, nnz;
    QuantShape s;
};

// Request b: its rows and the tokens in front of them; n = 0 where the arrays contradict themselves.
struct QuantRequest {
    int first, n, prior, page0;
};
__device__ __forceinline__ QuantRequest quant_request(const QuantRows &a, int b)
{
    const long first = a.qo_indptr[b], n = (long)a.qo_indptr[b + 1] - first, page0 = a.kv_page_indptr[b];
    const long pages = (long)a.kv_page_indptr[b + 1] - page0;
    const int last = a.kv_last_page_lens[b];
    const long length = (pages - 1) * a.s.page_size + last;
    const bool fine = first >= 0 && n >= 0 && first + n <= a.nnz && pages >= 1 && last >= 1 && last <= a.s.page_size &&
                      length >= n && length <= INT32_MAX;
    return {(int)first, fine ? (int)n : 0, (int)(length - n), (int)page0};
}
// Page of the request's token t, -1 where there is none.
__device__ __forceinline__ int quant_page(const QuantRows &a, const QuantRequest &r, int t)
{
    const long entry = (long)r.page0 + (unsigned)t / (unsigned)a.s.page_size;
    if (entry < 0 || entry >= a.n_page_indices) return -1;
    const int page = a.kv_page_indices[entry];
    return page >= 0 && page < a.s.num_pages ? page : -1;
}

// ---- append

struct QuantAppend {
    QuantRows r;
    char *q_out, *pages;
    const char *q, *k, *v;
    long q_stride, k_stride, v_stride;   // bytes
    const float *table;
    int n_qo_heads, kv_blocks, rows_each;
    float most;                          // the largest value that code * scale may take in the type
};

// 8 elements of a row as floats, rotated by the row's angles (table null: not).
template <int DT> struct Eight {
    u32x4 raw[DT == DSKV_F32 ? 2 : 1];
    __device__ __forceinline__ void load(const char *p)
    {
        raw[0] = *reinterpret_cast<const u32x4 *>(p);
        if constexpr (DT == DSKV_F32) raw[1] = *reinterpret_cast<const u32x4 *>(p + 16);
    }
    __device__ __forceinline__ void unpack(float *f) const
    {
        Chunk<DT>::unpack(raw[0], f);
        if constexpr (DT == DSKV_F32) Chunk<DT>::unpack(raw[1], f + 4);
    }
    __device__ __forceinline__ void store(char *p, const float *f) const
    {
        *reinterpret_cast<u32x4 *>(p) = Chunk<DT>::pack(f);
        if constexpr (DT == DSKV_F32) *reinterpret_cast<u32x4 *>(p + 16) = Chunk<DT>::pack(f + 4);
    }
};
struct Angles {
    float cs[4], sn[4];
    __device__ __forceinline__ Angles(const float *table, long t, int col, int head_dim)
    {
        const f32x4 c = *reinterpret_cast<const f32x4 *>(table + t * head_dim + col * 4);
        const f32x4 s = *reinterpret_cast<const f32x4 *>(table + t * head_dim + head_dim / 2 + col * 4);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            cs[i] = c[i];
            sn[i] = s[i];
        }
    }
};
__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

// Workgroups of the first kv_blocks rows of the grid: one wave per (rows_each rows of the step, kv head).  Of these it takes every one that is the first of
// its request in a page, and all rows of the request there with it, and so the whole block: their largest values, the scale, what the
// block holds already rounded anew where that grows, and the codes.  Workgroups behind: q, rows_each rows each.
// kLanes: lanes of a row, 8 elements each, a power of two.
// Bound by HBM where there are many rows: what is read a second time comes from the caches.  (More rows held in registers: 180 of these instead of 89,
// 80 us for the 62 below.)
template <int DT, int kLanes>
__global__ __launch_bounds__(256, 4) void quant_append_kernel(QuantAppend a)
{
    constexpr int kElt = DT == DSKV_F32 ? 4 : 2, kRows = 64 / kLanes;
    const QuantShape &s = a.r.s;
    const int t0 = blockIdx.x * a.rows_each, t1 = min(t0 + a.rows_each, a.r.nnz);
    const int lane = threadIdx.x & 63, col = lane % kLanes, row = lane / kLanes;
    const bool works = col * 8 < s.head_dim;
    if ((int)blockIdx.y >= a.kv_blocks) {
        constexpr int kHeads = 256 / kLanes, kAtOnce = 4;
        for (int t = t0; t < t1; t++) {
            if (!works) continue;
            const Angles angles(a.table, t, col, s.head_dim);
            for (int h0 = threadIdx.x / kLanes; h0 < a.n_qo_heads; h0 += kAtOnce * kHeads) {
                Eight<DT> x[kAtOnce];
#pragma unroll
                for (int i = 0; i < kAtOnce; i++)
                    if (h0 + i * kHeads < a.n_qo_heads)
                        x[i].load(a.q + t * a.q_stride + ((long)(h0 + i * kHeads) * s.head_dim + col * 8) * kElt);
#pragma unroll
                for (int i = 0; i < kAtOnce; i++)
                    if (h0 + i * kHeads < a.n_qo_heads) {
                        float f[8];
                        x[i].unpack(f);
                        rope_rotate<4>(f, angles.cs, angles.sn);
                        x[i].store(a.q_out + (((long)t * a.n_qo_heads + h0 + i * kHeads) * s.head_dim + col * 8) * kElt, f);
                    }
            }
        }
        return;
    }
    const int head = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (head >= s.n_kv_heads) return;
    int b = request_of_row(a.r.qo_indptr, a.r.batch, t0);
    if (b < 0) {
        if (t0 >= a.r.qo_indptr[0]) return;                               // rows behind the last request
        b = 0;
    }
    for (int t = t0; t < t1;) {
        while (b < a.r.batch && a.r.qo_indptr[b + 1] <= t) b++;           // on to the request of row t
        if (b == a.r.batch) return;
        const QuantRequest r = quant_request(a.r, b);
        if (r.n > 0 && r.first > t) {                                     // rows in front of the first request
            t = r.first;
            continue;
        }
        if (r.n == 0) {                                                   // its arrays contradict themselves
            const int next = a.r.qo_indptr[b + 1];
            if (next <= t) return;
            t = next;
            continue;
        }
        const int i = t - r.first, at = r.prior + i;
        const int place = (int)((unsigned)at % (unsigned)s.page_size);
        const int count = min(s.page_size - place, r.n - i);              // rows of the request in this page from t on
        const int begin = t;
        t += count;
        if (i > 0 && place > 0) continue;                                 // another wave's
        const char *const k_rows = a.k + begin * a.k_stride + ((long)head * s.head_dim + col * 8) * kElt;
        const char *const v_rows = a.v + begin * a.v_stride + ((long)head * s.head_dim + col * 8) * kElt;
        struct Pass {
            float k[8], v[8];
            bool fine;
        };
        float k_most = 0, v_most = 0;
        // a token of which a value is no finite number: its K becomes no number, so that rows that see it get none and
        // the others, whose weight of it is 0, are not touched by its V, which becomes 0
        auto fetch = [&](int j, Pass &p) {
#pragma unroll
            for (int d = 0; d < 8; d++) p.k[d] = p.v[d] = 0;
            if (works && j < count) {
                Eight<DT> x, y;
                x.load(k_rows + j * a.k_stride);
                y.load(v_rows + j * a.v_stride);
                x.unpack(p.k);
                y.unpack(p.v);
                if (a.table) {
                    const Angles angles(a.table, begin + j, col, s.head_dim);
                    rope_rotate<4>(p.k, angles.cs, angles.sn);
                }
            }
        };
        auto measure = [&](Pass &p) {
            float k_top = 0, v_top = 0, zero = 0;
#pragma unroll
            for (int d = 0; d < 8; d++) {
                k_top = fmaxf(k_top, fabsf(p.k[d]));
                v_top = fmaxf(v_top, fabsf(p.v[d]));
                zero = fmaf(p.k[d], 0.f, fmaf(p.v[d], 0.f, zero));        // no number if one of them is infinite or none
            }
            const unsigned long long odd = __ballot(zero != 0.f) >> (row * kLanes);
            p.fine = (odd & ((1ull << kLanes) - 1)) == 0;
            k_most = fmaxf(k_most, p.fine ? k_top : 0.f);
            v_most = fmaxf(v_most, p.fine ? v_top : 0.f);
        };
        // rows of one pass stay in registers; of more, what the second reading needs is in the L2
        Pass first;
        fetch(row, first);
        const int page = quant_page(a.r, r, at);
        if (page < 0) continue;
        char *const record = a.pages + page * s.page_bytes;
        char *const k_block = record + head * s.head_bytes, *const v_block = k_block + s.half_bytes;
        uint32_t *const scales = reinterpret_cast<uint32_t *>(record + 2 * s.half_bytes) + head;
        uint32_t scale[2] = {0, 0};                                       // of the rows that stay
        if (place > 0) {
            scale[0] = stored_scale(scales[0]);
            scale[1] = stored_scale(scales[s.n_kv_heads]);
        }
        measure(first);
#pragma unroll 1
        for (int j = kRows; j < count; j += kRows) {
            Pass p;
            fetch(j + row, p);
            measure(p);
        }
        const float most[2] = {fminf(wave_max(k_most), a.most), fminf(wave_max(v_most), a.most)};
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const uint32_t old = scale[x];
            scale[x] = max(needed_scale(most[x]), old);
            if (old != 0 && scale[x] > old) {
                const float ratio = __builtin_bit_cast(float, old) * reciprocal_of(scale[x]);
                for (int j = lane; j < place * s.head_dim / 8; j += 64) {
                    u32x2 *const codes = reinterpret_cast<u32x2 *>(x ? v_block : k_block) + j;
                    float f[8];
                    decode8(*codes, f);
#pragma unroll
                    for (int d = 0; d < 8; d++) f[d] *= ratio;
                    *codes = encode8(f);
                }
            }
        }
        if (lane < 2) scales[lane * s.n_kv_heads] = lane ? scale[1] : scale[0];
        const float k_by = reciprocal_of(scale[0]), v_by = reciprocal_of(scale[1]);
        auto put = [&](int j, Pass &p) {
            if (!works || j >= count) return;
#pragma unroll
            for (int d = 0; d < 8; d++) {
                p.k[d] = fminf(fmaxf(p.k[d], -a.most), a.most) * k_by;
                p.v[d] = fminf(fmaxf(p.v[d], -a.most), a.most) * v_by;
            }
            const uint32_t none = kNoNumberCode * 0x01010101u;
            const long to = (long)(place + j) * s.head_dim + col * 8;
            *reinterpret_cast<u32x2 *>(k_block + to) = p.fine ? encode8(p.k) : u32x2{none, none};
            *reinterpret_cast<u32x2 *>(v_block + to) = p.fine ? encode8(p.v) : u32x2{0, 0};
        };
        put(row, first);
#pragma unroll 1
        for (int j = kRows; j < count; j += kRows) {
            Pass p;
            fetch(j + row, p);
            measure(p);                                                   // (for p.fine)
            put(j + row, p);
        }
    }
}

// ---- move

struct QuantMove {
    QuantRows r;
    char *pages;
    long layer_stride;
    const int32_t *path, *counts;
    int n_layers, layers_each;
};

// One wave per (request, half and head) and run of layers, for which the rows and their places are the same.  In a layer all rows that
// move are read first.  Where a page that they go to has too small a scale for one of them, the pages are taken one by one: the scale
// that the rows need there, and what else the block holds rounded anew.  Then the rows are written, by their new scales.
// A lane keeps one of the rows that move; kLanes: lanes of a row's codes, 4 * kWords each.
template <int kLanes, int kWords>
__global__ __launch_bounds__(256) void quant_move_kernel(QuantMove a)
{
    constexpr int kRows = 64 / kLanes, kPasses = DSKV_MAX_TREE_ROWS / kRows, kBytes = 4 * kWords;
    typedef uint32_t Codes __attribute__((ext_vector_type(kWords)));
    __shared__ long from_of[4][64], to_of[4][64];
    __shared__ float by_of[4][64];
    const QuantShape &s = a.r.s;
    const int b = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane % kLanes, row = lane / kLanes;
    const int block = blockIdx.y * 4 + wave;                               // half and head
    if (block >= 2 * s.n_kv_heads) return;
    const QuantRequest r = quant_request(a.r, b);
    const int walk = a.counts[b], count = min(walk, r.n);
    if (count < 2 || walk > DSKV_MAX_TREE_ROWS) return;
    const long block_at = block * s.head_bytes, scale_at = 2 * s.half_bytes + block * 4L;

    const int p = lane < count ? a.path[r.first + lane] : -1;
    const int before = __shfl_up(p, 1);
    int from = -1, to = -1, from_place = 0, to_place = 0;                  // pages and places in them
    if (lane > 0 && lane < count && p > lane && p < r.n && p > before) {
        from = quant_page(a.r, r, r.prior + p);
        to = quant_page(a.r, r, r.prior + lane);
        from_place = (int)((unsigned)(r.prior + p) % (unsigned)s.page_size);
        to_place = (int)((unsigned)(r.prior + lane) % (unsigned)s.page_size);
    }
    const bool moves = from >= 0 && to >= 0;
    const unsigned long long moving = __ballot(moves);
    if (moving == 0) return;
    const int rows = __popcll(moving);
    const int mine = __popcll(moving & ((1ull << lane) - 1));              // which of the moving rows the lane keeps
    if (moves) {
        from_of[wave][mine] = from * s.page_bytes + block_at + (long)from_place * s.head_dim;
        to_of[wave][mine] = to * s.page_bytes + block_at + (long)to_place * s.head_dim;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int layer_end = min((int)(blockIdx.z + 1) * a.layers_each, a.n_layers);
    const bool loads = col * kBytes < s.head_dim;
    struct Layer {
        Codes codes[kPasses];
        float from_scale;
        uint32_t held;
    };
    auto fetch = [&](int at, Layer &x) {
        const char *layer = a.pages + at * a.layer_stride;
        x.from_scale = moves ? *reinterpret_cast<const float *>(layer + from * s.page_bytes + scale_at) : 0.f;
        x.held = moves ? *reinterpret_cast<const uint32_t *>(layer + to * s.page_bytes + scale_at) : 0u;
#pragma unroll
        for (int i = 0; i < kPasses; i++)
            if (i * kRows < rows) {
#pragma unroll
                for (int w = 0; w < kWords; w++) x.codes[i][w] = 0;
                if (loads && i * kRows + row < rows)
                    x.codes[i] = *reinterpret_cast<const Codes *>(layer + from_of[wave][i * kRows + row] + col * kBytes);
            }
    };
    auto put = [&](int at, const Layer &x) {
        char *const layer = a.pages + at * a.layer_stride;
        uint32_t top = 0;                                                 // the largest code of the lane's row
#pragma unroll
        for (int i = 0; i < kPasses; i++)
            if (i * kRows < rows) {
                // (codes without their sign are ordered as their values; 0x7F is none)
                uint32_t most = 0;
#pragma unroll
                for (int w = 0; w < kWords; w++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint32_t c = x.codes[i][w] >> (8 * e) & 0x7F;
                        most = c == kNoNumberCode ? most : max(most, c);
                    }
#pragma unroll
                for (int o = kLanes / 2; o > 0; o >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o));
                const uint32_t theirs = (uint32_t)__shfl((int)most, mine % kRows * kLanes);      // of row i * kRows + mine % kRows
                if (mine / kRows == i) top = theirs;
            }
        const float value = __builtin_amdgcn_cvt_f32_fp8((int)top, 0) * x.from_scale;
        uint32_t scale = stored_scale(x.held);
        if (__ballot(moves && value > 0 && needed_scale(value) > scale) != 0) {
            for (int j = 1; j < count;) {                                 // page by page of those that rows go to
                const int begin = r.prior + j - (int)((unsigned)(r.prior + j) % (unsigned)s.page_size);     // its first token
                const int end = min(count, begin + s.page_size - r.prior);
                const bool here = lane >= j && lane < end && moves;
                const float most = wave_max(here ? value : 0.f);
                const unsigned long long some = __ballot(here);
                j = end;
                if (some == 0 || !(most > 0)) continue;
                const int first = __builtin_ctzll(some);
                char *const record = layer + __shfl(to, first) * s.page_bytes;
                const uint32_t old = (uint32_t)__shfl((int)scale, first), now = max(needed_scale(most), old);
                if (now == old) continue;
                if (old != 0) {
                    const float ratio = __builtin_bit_cast(float, old) * reciprocal_of(now);
                    const int tokens = min(s.page_size, r.prior + r.n - begin);
                    for (int x = lane; x < tokens * s.head_dim / 8; x += 64) {
                        u32x2 *const c = reinterpret_cast<u32x2 *>(record + block_at) + x;
                        float f[8];
                        decode8(*c, f);
#pragma unroll
                        for (int d = 0; d < 8; d++) f[d] *= ratio;
                        *c = encode8(f);
                    }
                }
                if (lane == 0) *reinterpret_cast<uint32_t *>(record + scale_at) = now;
                if (here) scale = now;
            }
            __builtin_amdgcn_s_waitcnt(0);                                // the blocks have been rounded anew
            asm volatile("" ::: "memory");
        }
        // A row of zeros asks for no scale, and its own may be so far above the one that is there that no 32 bits hold their ratio: by 0,
        // which keeps zeros and codes of no number what they are.
        if (moves) by_of[wave][mine] = value > 0 ? x.from_scale * reciprocal_of(scale) : 0.f;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < kPasses; i++) {
            const int at_row = i * kRows + row;
            if (i * kRows < rows && loads && at_row < rows) {
                const float ratio = by_of[wave][at_row];
                Codes now;
#pragma unroll
                for (int w = 0; w < kWords; w += 2) {
                    float f[8];
                    decode8(u32x2{x.codes[i][w], x.codes[i][w + 1]}, f);
#pragma unroll
                    for (int d = 0; d < 8; d++) f[d] *= ratio;
                    const u32x2 pair = encode8(f);
                    now[w] = pair.x;
                    now[w + 1] = pair.y;
                }
                *reinterpret_cast<Codes *>(layer + to_of[wave][at_row] + col * kBytes) = now;
            }
        }
        __builtin_amdgcn_wave_barrier();
    };
    Layer x;
    for (int at = blockIdx.z * a.layers_each; at < layer_end; at++) {
        fetch(at, x);
        put(at, x);
    }
}

// Rows of a wave of the append: one as long as that makes few waves, else as many as make about kAppendWaves.  8192 rows (16 chunks of 512, 64 heads
// over 8, f16, 323 MB) 62 us, 5.2 TB/s; with one row a wave, most of them for nothing, 76; 320 rows 6.4 us, with two each 7.9.
constexpr int kAppendMost = 8192, kAppendWaves = 2048;
static int rows_each(int64_t nnz, int64_t n_kv_heads)
{
    const int64_t waves = nnz * n_kv_heads;
    return waves <= kAppendMost ? 1 : (int)std::min<int64_t>((waves + kAppendWaves - 1) / kAppendWaves, 64);
}
// Waves that a move is cut into, about: 64 walks in 32 layers 21.8 us, with 4096 24.2, with 16384 23.4.
constexpr int kMoveWaves = 8192;

static int lanes_of(int head_dim)
{
    int lanes = 1;
    while (lanes * 8 < head_dim) lanes *= 2;
    return lanes;
}
static int check_rows(const dskv_quant_rows_t *r, const char *what)
{
    DSKV_REQUIRE(r, "%s: null arguments", what);
    DSKV_REQUIRE(r->batch >= 0 && r->nnz >= 0 && r->n_page_indices >= 0, "%s: negative batch, nnz or table", what);
    DSKV_REQUIRE(r->num_pages > 0 && r->page_size > 0 && r->n_kv_heads > 0, "%s: bad page shape", what);
    DSKV_REQUIRE(r->head_dim > 0 && r->head_dim % 8 == 0 && r->head_dim <= 256,
                 "%s: head_dim %d must be a multiple of 8 up to 256", what, r->head_dim);
    DSKV_REQUIRE((int64_t)r->page_size * r->head_dim < INT32_MAX && r->n_kv_heads <= 65535, "%s: too large a page", what);
    if (r->batch == 0 || r->nnz == 0) return 0;
    DSKV_REQUIRE(r->qo_indptr && r->kv_page_indptr && r->kv_last_page_lens && (r->kv_page_indices || r->n_page_indices == 0),
                 "%s: null pointer argument", what);
    return 0;
}
static QuantRows rows_of(const dskv_quant_rows_t *r)
{
    return {r->qo_indptr, r->kv_page_indices, r->kv_page_indptr, r->kv_last_page_lens, (long)r->n_page_indices, r->batch, r->nnz,
            quant_shape(r->num_pages, r->page_size, r->n_kv_heads, r->head_dim)};
}
template <int DT> static int launch_quant_append(const QuantAppend &a, hipStream_t stream)
{
    const dim3 grid((unsigned)((a.r.nnz + a.rows_each - 1) / a.rows_each), (unsigned)(a.kv_blocks + (a.table ? 1 : 0))), block(256);
    switch (lanes_of(a.r.s.head_dim)) {
    case 1: hipLaunchKernelGGL((quant_append_kernel<DT, 1>), grid, block, 0, stream, a); break;
    case 2: hipLaunchKernelGGL((quant_append_kernel<DT, 2>), grid, block, 0, stream, a); break;
    case 4: hipLaunchKernelGGL((quant_append_kernel<DT, 4>), grid, block, 0, stream, a); break;
    case 8: hipLaunchKernelGGL((quant_append_kernel<DT, 8>), grid, block, 0, stream, a); break;
    case 16: hipLaunchKernelGGL((quant_append_kernel<DT, 16>), grid, block, 0, stream, a); break;
    default: hipLaunchKernelGGL((quant_append_kernel<DT, 32>), grid, block, 0, stream, a); break;
    }
    DSKV_LAUNCH_CHECK("quant_append_kernel");
    return 0;
}

}  // namespace dskv

extern "C" int64_t dskv_quant_page_bytes(int32_t page_size, int32_t n_kv_heads, int32_t head_dim)
{
    return page_size > 0 && n_kv_heads > 0 && head_dim > 0 ? dskv::quant_page_bytes(page_size, n_kv_heads, head_dim) : 0;
}

extern "C" int dskv_rope_append_quant(const dskv_quant_rows_t *rows, void *q_out, void *pages_layer, const void *q, const void *k,
                                      const void *v, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                      const float *rope_table, int32_t n_qo_heads, int32_t dtype, void *stream)
{
    using namespace dskv;
    if (int rc = check_rows(rows, "rope_append_quant")) return rc;
    DSKV_REQUIRE(dtype == DSKV_F32 || dtype == DSKV_F16 || dtype == DSKV_BF16, "rope_append_quant: unknown dtype %d", dtype);
    if (rows->batch == 0 || rows->nnz == 0) return 0;
    DSKV_REQUIRE(pages_layer && k && v && (!rope_table || (q && q_out)), "rope_append_quant: null pointer argument");
    const int size = dtype == DSKV_F32 ? 4 : 2;
    const int64_t kv_row = (int64_t)rows->n_kv_heads * rows->head_dim;
    DSKV_REQUIRE(!rope_table || n_qo_heads > 0, "rope_append_quant: n_qo_heads %d", n_qo_heads);
    DSKV_REQUIRE((!rope_table || q_stride >= (int64_t)n_qo_heads * rows->head_dim) && k_stride >= kv_row && v_stride >= kv_row,
                 "rope_append_quant: rows overlap");
    DSKV_REQUIRE((((uintptr_t)q_out | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)pages_layer | (uintptr_t)rope_table) % 16 == 0) &&
                 ((rope_table ? q_stride : 0) | k_stride | v_stride) * size % 16 == 0,
                 "rope_append_quant: tensors and their rows must be 16-byte aligned");
    QuantAppend a = {rows_of(rows), (char *)q_out, (char *)pages_layer, (const char *)q, (const char *)k, (const char *)v,
                     (long)q_stride * size, (long)k_stride * size, (long)v_stride * size, rope_table, n_qo_heads,
                     (rows->n_kv_heads + 3) / 4,
                     rows_each(rows->nnz, rows->n_kv_heads),
                     // 240 * 2^8, 240 * 2^120: the code above, 256, would make an infinity of the type with that scale
                     dtype == DSKV_F16 ? 61440.f : 3.1901472e38f};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == DSKV_F32) return launch_quant_append<DSKV_F32>(a, st);
    if (dtype == DSKV_F16) return launch_quant_append<DSKV_F16>(a, st);
    return launch_quant_append<DSKV_BF16>(a, st);
}

extern "C" int dskv_move_quant_rows(const dskv_quant_rows_t *rows, void *pages, int64_t layer_stride_bytes, int32_t n_layers,
                                    const int32_t *path, const int32_t *counts, void *stream)
{
    using namespace dskv;
    if (int rc = check_rows(rows, "move_quant_rows")) return rc;
    DSKV_REQUIRE(n_layers >= 0 && n_layers <= 65535, "move_quant_rows: %d layers", n_layers);
    if (rows->batch == 0 || rows->nnz == 0 || n_layers == 0) return 0;
    DSKV_REQUIRE(pages && path && counts, "move_quant_rows: null pointer argument");
    DSKV_REQUIRE((uintptr_t)pages % 16 == 0 && layer_stride_bytes % 16 == 0, "move_quant_rows: pages must be 16-byte aligned");
    QuantMove a = {rows_of(rows), (char *)pages, (long)layer_stride_bytes, path, counts, n_layers, 1};
    DSKV_REQUIRE(n_layers == 1 || layer_stride_bytes >= rows->num_pages * a.r.s.page_bytes, "move_quant_rows: layers overlap");
    const int64_t waves = (int64_t)rows->batch * 2 * rows->n_kv_heads * n_layers;
    a.layers_each = waves <= kMoveWaves ? 1 : (int)std::min<int64_t>(n_layers, (waves + kMoveWaves - 1) / kMoveWaves);
    const dim3 grid((unsigned)rows->batch, (unsigned)((2 * rows->n_kv_heads + 3) / 4),
                    (unsigned)((n_layers + a.layers_each - 1) / a.layers_each)), block(256);
    hipStream_t st = (hipStream_t)stream;
    if (rows->head_dim % 16) {
        switch (lanes_of(rows->head_dim)) {
        case 1: hipLaunchKernelGGL((quant_move_kernel<1, 2>), grid, block, 0, st, a); break;
        case 4: hipLaunchKernelGGL((quant_move_kernel<4, 2>), grid, block, 0, st, a); break;
        case 8: hipLaunchKernelGGL((quant_move_kernel<8, 2>), grid, block, 0, st, a); break;
        case 16: hipLaunchKernelGGL((quant_move_kernel<16, 2>), grid, block, 0, st, a); break;
        default: hipLaunchKernelGGL((quant_move_kernel<32, 2>), grid, block, 0, st, a); break;
        }
    } else {
        switch (lanes_of(rows->head_dim) / 2) {
        case 1: hipLaunchKernelGGL((quant_move_kernel<1, 4>), grid, block, 0, st, a); break;
        case 2: hipLaunchKernelGGL((quant_move_kernel<2, 4>), grid, block, 0, st, a); break;
        case 4: hipLaunchKernelGGL((quant_move_kernel<4, 4>), grid, block, 0, st, a); break;
        case 8: hipLaunchKernelGGL((quant_move_kernel<8, 4>), grid, block, 0, st, a); break;
        default: hipLaunchKernelGGL((quant_move_kernel<16, 4>), grid, block, 0, st, a); break;
        }
    }
    DSKV_LAUNCH_CHECK("quant_move_kernel");
    return 0;
}
