// The attention over 8-bit pages for few columns (head_dim 64 and 128, all three types): one row per request, drafted tokens, short
// chunks.  Work is cut as in tree_kernel.h - columns of a kv head, subtiles of 32 tokens, equal shares, one workgroup per (share, kv head), a wave
// per subtile -, and what differs is what a wave does with a subtile:
// codes go by whole rows through registers and the wave's LDS as they are; the matrix instructions' operands are made of them behind LDS,
// two codes an instruction, exactly: every code is a number of bf16 and of f16.  K's scales multiply the scores and V's the weights, in 32 bits,
// token by token, so that pages may end anywhere in a subtile.
// Weights times V's scale span more than f16 holds: the second product is in bf16 for all types.  A weight is rounded to bf16 for bf16
// results (2^-9 of it, half of what the result's own rounding is), to two bf16 terms for f16 (2^-17) and to three, that is to 32
// bits, for fp32, whose q is three terms as well.  (A weight is up to most_weight, 2^8: times V, and summed, that has to fit fp32, which bounds
// the magnitudes of V: see dskv_quant_attn in dskv.h.)
// Bound by HBM: 64 requests of one row over 256 - 4096 tokens, 32 heads over 8, 128 dims, bf16, 279 MB, 52.3 us, 5.3 TB/s; its loads alone 51.  With 8
// rows each 68, where items end: 50 if all are as long.
#pragma once

#include "quant.h"
#include "tree_kernel.h"

namespace dskv {

struct QuantArgs : TreeArgs {
    long head_bytes, half_bytes, page_bytes;      // see quant.h
    uint32_t page16, row16;                       // bytes of a page and of a token's row, in sixteens
    uint32_t *counters;                           // narrow form: one for each partial and kv head; zero between launches
    struct QuantCut *cuts;                        // wide form: two for each share
    int rows_from, rows_to;                       // rows of a request that this launch computes, 0 of any other's
};
__device__ __forceinline__ int rows_taken(const QuantArgs &a, int n) { return n >= a.rows_from && n <= a.rows_to ? n : 0; }

// (beside a chunk there may be many requests that this launch has nothing of; one request in one tile is cut evenly)
__device__ __forceinline__ bool parts_apply(const QuantArgs &a, int spans, int busy)
{
    return busy <= spans && (busy > 1 || a.max_rows * a.group > 128);
}

constexpr uint32_t kNoQuantRow = 0xFFFFFFFFu;
// Where token t's K lies in the head's part of the pool, in sixteens of bytes.
__device__ __forceinline__ uint32_t quant_row(const QuantArgs &a, int t, int page)
{
    return page >= 0 && page < a.num_pages ? (uint32_t)page * a.page16 + (uint32_t)(t - page_number(a, t) * a.page_size) * a.row16
                                           : kNoQuantRow;
}

// ---- Items that share boundaries cut leave a partial (maximum, sum, O in fp32, for every column) for each part.
struct QuantParts {
    int first, n;        // shares (spans) that hold a part; n == 1: not cut
    bool second;         // in the first of them the item is the second
    uint32_t slot;       // of the first
};
__device__ __forceinline__ uint32_t part_slot(const QuantArgs &a, const TreePlace &place, const QuantParts &p, int ct, int i)
{
    const int span = p.first + i, share = place.beside ? share_of_span(span, ct, a.sides) : span;
    return 2u * (uint32_t)share + (i == 0 && p.second ? 1u : 0u);
}
// item: its first unit, of `units`.
__device__ __forceinline__ QuantParts parts_of(const QuantArgs &a, const TreePlace &place, int item, int units, int ct)
{
    QuantParts p = {place.first_part, place.n_parts, false, 0};
    if (p.n == 0) {
        Shares s = place.shares;
        s.each = __builtin_amdgcn_readfirstlane(s.each);
        s.longer = __builtin_amdgcn_readfirstlane(s.longer);
        p.first = share_with(s, item);
        p.n = share_with(s, item + units - 1) - p.first + 1;
        p.second = share_begin(s, p.first) < item;
    }
    p.slot = part_slot(a, place, p, ct, 0);
    return p;
}
// The narrow form's parts are merged in the launch: partials are stored with device scope, a part whose stores are acknowledged counts itself
// in, and the one that completes the count reads all of them, past its XCD's L2, and writes the rows.  The order of the sums does not depend on
// which that is.  (A launch of its own: one request over 1.8 K tokens 15.0 us, so 12.3.  With the wide form's 133 KB a part that is too much for one
// workgroup: 16 chunks 983 us, with a launch of its own 941.)
constexpr int kDeviceScope = 16;                                   // cache policy of the buffer instructions: sc1
template <int kCols, int kD> struct PartSlot {
    __amdgpu_buffer_rsrc_t o, ml;
    __device__ __forceinline__ PartSlot(const QuantArgs &a, int head, uint32_t slot)
    {
        const long part = ((long)slot * a.n_kv_heads + head) * kCols;
        o = __builtin_amdgcn_make_buffer_rsrc(a.part_o + part * kD, 0, kCols * kD * 4, kBufferFlags);
        ml = __builtin_amdgcn_make_buffer_rsrc(a.part_ml + part * 2, 0, kCols * 8, kBufferFlags);
    }
    __device__ __forceinline__ void put_o(int col, int dim, f32x4 v) const
    {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), o, (col * kD + dim) * 4, 0, kDeviceScope);
    }
    __device__ __forceinline__ void put_ml(int col, float m, float l) const
    {
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, f32x2{m, l}), ml, col * 8, 0, kDeviceScope);
    }
    __device__ __forceinline__ f32x4 get_o(int col, int dim) const
    {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(o, (col * kD + dim) * 4, 0, kDeviceScope));
    }
    __device__ __forceinline__ f32x2 get_ml(int col) const
    {
        return __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(ml, col * 8, 0, kDeviceScope));
    }
};
// Four dims of a column's row.
template <int DT, int kD>
__device__ __forceinline__ void put_result(const QuantArgs &a, long first, int head, int at, int dim, f32x4 acc, float sum)
{
    constexpr int kElt = DT == DSKV_F32 ? 4 : 2;
    const int i = (int)((unsigned)at / (unsigned)a.group), hq = head * a.group + at - i * a.group;
    const float inv = sum == 0 ? 0.f : 1.f / sum;
    char *dst = a.out + (((first + i) * a.n_qo_heads + hq) * kD + dim) * kElt;
    if constexpr (DT == DSKV_F32) *reinterpret_cast<f32x4 *>(dst) = acc * inv;
    else *reinterpret_cast<u32x2 *>(dst) = u32x2{Elt<DT>::pack2(acc.x * inv, acc.y * inv), Elt<DT>::pack2(acc.z * inv, acc.w * inv)};
}
// kEach quads of dims a thread, of x and every kThreads-th behind it, and kAtOnce parts requested together.
template <int DT, int kD, int kCols, int kThreads, int kEach, int kAtOnce>
__device__ __forceinline__ void merge_parts(const QuantArgs &a, const TreePlace &place, const TreeRequest &r, const QuantParts &p,
                                            int head, int ct, int cols, int x)
{
    constexpr int kQuads = kD / 4;
    float top[kEach], sum[kEach];
    f32x4 acc[kEach];
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        top[e] = -INFINITY;
        sum[e] = 0;
        acc[e] = f32x4{0, 0, 0, 0};
    }
    for (int i0 = 0; i0 < p.n; i0 += kAtOnce) {
        f32x4 o[kAtOnce][kEach];
        f32x2 ml[kAtOnce][kEach];
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) {
            const PartSlot<kCols, kD> part(a, head, part_slot(a, place, p, ct, min(i0 + i, p.n - 1)));
#pragma unroll
            for (int e = 0; e < kEach; e++) {
                const int col = min((x + e * kThreads) / kQuads, cols - 1);
                ml[i][e] = part.get_ml(col);
                o[i][e] = part.get_o(col, x % kQuads * 4);
            }
        }
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            float m = top[e];
#pragma unroll
            for (int i = 0; i < kAtOnce; i++) m = fmaxf(m, ml[i][e].x);
            const float from = m == -INFINITY ? 0.f : m, keep = __builtin_amdgcn_exp2f(top[e] - from);
            top[e] = m;
            sum[e] *= keep;
            acc[e] *= keep;
#pragma unroll
            for (int i = 0; i < kAtOnce; i++)
                if (i0 + i < p.n) {
                    const float w = __builtin_amdgcn_exp2f(ml[i][e].x - from);
                    sum[e] += ml[i][e].y * w;
                    acc[e] += o[i][e] * w;
                }
        }
    }
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        const int col = (x + e * kThreads) / kQuads;
        if (col < cols) put_result<DT, kD>(a, r.first, head, ct * kCols + col, x % kQuads * 4, acc[e], sum[e]);
    }
}
// By all threads of a workgroup, behind its stores of a part's partial.  last: a word of LDS.
template <int DT, int kD, int kCols, int kThreads>
__device__ __forceinline__ void join_parts(const QuantArgs &a, const TreePlace &place, const TreeRequest &r, const QuantParts &p,
                                           int head, int ct, int cols, int *last)
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");               // the partial is where other XCDs see it
    __syncthreads();
    if (threadIdx.x == 0) {
        uint32_t *const counter = a.counters + (long)p.slot * a.n_kv_heads + head;
        const uint32_t before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *last = before + 1 == (uint32_t)p.n;
        if (before + 1 == (uint32_t)p.n) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!*last) return;
    asm volatile("" ::: "memory");
    // All of a workgroup's columns together, and as many parts as leave the loads their registers: one request of 8 rows over 16 K tokens 35.0 us;
    // with eight parts of one column after the other 47.9.
    constexpr int kQuads = kD / 4, kEach = kCols * kQuads / kThreads;
    static_assert(kThreads % kQuads == 0 && kCols * kQuads % kThreads == 0, "a thread's quads lie at one place of their columns");
    const int x = threadIdx.x;
    if (cols * kQuads <= kThreads) {
        if (x < cols * kQuads) merge_parts<DT, kD, kCols, kThreads, 1, 8>(a, place, r, p, head, ct, cols, x);
    } else if (p.n <= 4) {
        merge_parts<DT, kD, kCols, kThreads, kEach, 2>(a, place, r, p, head, ct, cols, x);
    } else {
        merge_parts<DT, kD, kCols, kThreads, kEach, 4>(a, place, r, p, head, ct, cols, x);
    }
}

// 8 codes as a matrix operand of type T
template <int T> __device__ __forceinline__ u32x4 operand_of(u32x2 codes)
{
    u32x4 x;
#pragma unroll
    for (int w = 0; w < 2; w++) {
        if constexpr (T == DSKV_F16) {
            x[2 * w] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[w], 1.0f, false));
            x[2 * w + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[w], 1.0f, true));
        } else {
            x[2 * w] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[w], 1.0f, false));
            x[2 * w + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[w], 1.0f, true));
        }
    }
    return x;
}
// Eight floats as kTerms operands of bf16 that add up to them; what is left is rounded away.
template <int kTerms> __device__ __forceinline__ void split8(const float *f, u32x4 *terms)
{
#pragma unroll
    for (int w = 0; w < 4; w++) {
        float a = f[2 * w], b = f[2 * w + 1];
#pragma unroll
        for (int i = 0; i < kTerms; i++) {
            const uint32_t pair = Elt<DSKV_BF16>::pack2(a, b);
            terms[i][w] = pair;
            if (i + 1 < kTerms) {
                float x, y;
                Elt<DSKV_BF16>::unpack2(pair, x, y);
                a -= x;
                b -= y;
            }
        }
    }
}

// Units that a share has at least, two turns of its waves: shorter parts cost more to merge than they save.  8 requests of 5 rows over 300 - 1100 tokens
// 13.8 us, with one turn 15.8, with three 14.5; one row over 1.8 K 9.6, 10.1, 10.4, over 500 8.9, 8.0, 8.9.
constexpr int kQuantLeast = 2 * kTreeWaves;

// Columns of a tile at most; where q's operands lie, in registers or, where these would be too many beside O and the weights' terms, in
// LDS; and workgroups of a compute unit, with one subtile of a wave in flight.  64 requests over 256 - 4096 tokens, 128 dims:
//   bf16, one row    52.3 us; with two subtiles in flight 54.5, with those and one workgroup 62.5, with three workgroups 56.7
//   f16, 5 rows      64.0 (two blocks); with two subtiles in flight 85.6, with three workgroups 87.8
//   fp32, one row    55.6; with q in registers, one workgroup 69.7.  5 rows 108 (one workgroup); with q in LDS 111
// and 64 dims: bf16 of 12 rows 54 (three blocks; with one workgroup 78), of 16 rows 66 (four; as wide tiles 79); fp32, one row 38;
// 51.  5 rows 53.4; with one workgroup 74, with q in LDS 55.
// (Four blocks at 64 dims keep 4 or 5 registers, of the item, in scratch while its subtiles run.
// With 128 dims three blocks leave registers for one workgroup only, 113 us for 12 rows; see QuantWide.)
constexpr int quant_columns(int dtype, int dim) { return dtype == DSKV_F32 || dim == 128 ? 32 : 64; }
constexpr bool quant_q_in_lds(int dtype, int blocks) { return dtype == DSKV_F32 && blocks == 1; }
constexpr int quant_workgroups(int dtype, int dim, int blocks)
{
    return dim == 64 || blocks <= (dtype == DSKV_F32 ? 1 : 2) ? 2 : 1;
}

template <int DT, int kD, int kBlocks> struct QuantTile {
    static constexpr int kElt = DT == DSKV_F32 ? 4 : 2;
    static constexpr int kSub = 32;                                  // tokens of a subtile
    static constexpr int kTiles = 2;
    static constexpr int kChunks = kD / 16;                          // 16-byte chunks of a row
    static constexpr int kRowsPerLoad = 64 / kChunks;
    static constexpr int kLoads = kSub / kRowsPerLoad;
    static constexpr int kSteps = kD / 32;                           // matrix instructions of a tile's scores
    static constexpr int kDimTiles = kD / 16;
    static constexpr int kCols = kBlocks * 16;
    static constexpr int kQTerms = DT == DSKV_F32 ? 3 : 1, kPTerms = DT == DSKV_BF16 ? 1 : DT == DSKV_F16 ? 2 : 3;
    static constexpr int kKeyType = DT == DSKV_F16 ? DSKV_F16 : DSKV_BF16;
    static constexpr int kPitch = kD + 16;                           // bytes; 16 rows' chunks at one offset meet no bank twice
    static constexpr int kWaveLds = 2 * kSub * kPitch + 2 * kSub * 4;      // K, V, their scales
    static constexpr int kOPitch = kD + 4;                           // floats
    static constexpr bool kQInLds = quant_q_in_lds(DT, kBlocks);
    static constexpr int kQLds = kQInLds ? kBlocks * kSteps * kQTerms * 1024 : 0;
    static constexpr int kMergeLds = kTreeWaves * kCols * (kOPitch + 2) * 4;
    static constexpr int kLds = kTreeWaves * kWaveLds > kMergeLds ? kTreeWaves * kWaveLds : kMergeLds;
    static constexpr int kWorkgroups = quant_workgroups(DT, kD, kBlocks);
};

template <int DT, int kD, int kBlocks>
__global__ __launch_bounds__(kTreeThreads, (QuantTile<DT, kD, kBlocks>::kWorkgroups)) void quant_matrix_kernel(QuantArgs a)
{
    typedef QuantTile<DT, kD, kBlocks> S;
    __shared__ __align__(16) char lds[S::kLds + S::kQLds];
    __shared__ int last_part;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, c = lane & 15;
    int share, head;
    share_and_head(a, share, head);
    TreePlace place;
    tree_place<S::kCols, S::kSub, kTreeThreads, false, kQuantLeast, kTreeWaves>(a, share, place);
    make_uniform(place);
    const int begin = place.begin, end = place.end;
    if (begin >= end) return;

    char *const k_lds = lds + wave * S::kWaveLds, *const v_lds = k_lds + S::kSub * S::kPitch;
    float *const scale_lds = reinterpret_cast<float *>(v_lds + S::kSub * S::kPitch);
    const int load_row = lane / S::kChunks, load_chunk = lane % S::kChunks;
    const char *const pool = a.pages + head * a.head_bytes + load_chunk * 16;
    // lanes 0 .. 31 fetch the scales of K, the others those of V
    const char *const scales = a.pages + 2 * a.half_bytes + ((lane >> 5) * a.n_kv_heads + head) * 4;
    const char *const none = reinterpret_cast<const char *>(kNoRow) + load_chunk * 16;

    // ---- what is requested: the wave's subtiles through all items of the share, one in flight, its page ids one step
    // further ahead (see tree_kernel.h)
    TreeItem ahead;
    ahead.b = place.b;
    ahead.base = place.base;
    ahead.r = place.r;
    open_item<S::kCols, S::kSub>(a, begin, begin, end, ahead);
    int ahead_st = ahead.st0 + wave;
    bool more = true;
    auto settle = [&]() {                                       // on to a subtile that there is
        if (__builtin_expect(ahead_st < ahead.st1, 1)) return;
        while (more && ahead_st >= ahead.st1) {
            more = ahead.next < end;
            if (more) {
                open_item<S::kCols, S::kSub>(a, ahead.next, begin, end, ahead);
                ahead_st = ahead.st0 + wave;
            }
        }
    };
    struct Ids {
        int page, t;
    };
    auto next_ids = [&]() {                                     // of the lane's token of the next subtile; moves on
        settle();
        Ids x;
        x.t = ahead_st * S::kSub + (lane & (S::kSub - 1));
        x.page = more ? page_of(a, ahead.r, x.t) : -1;
        ahead_st += kTreeWaves;
        return x;
    };
    struct Held {
        u32x4 k[S::kLoads], v[S::kLoads];
        float scale;
        uint32_t there;                                         // bit per token: there is one
    };
    Held held;
    auto request = [&](const Ids &x, Held &to) {
        const uint32_t mine = quant_row(a, x.t, x.page);
        to.there = (uint32_t)__ballot(mine != kNoQuantRow);     // (lanes repeat)
        uint32_t row[S::kLoads];
#pragma unroll
        for (int i = 0; i < S::kLoads; i++) row[i] = (uint32_t)__shfl((int)mine, load_row + S::kRowsPerLoad * i);
        const char *s = mine != kNoQuantRow ? scales + x.page * a.page_bytes : reinterpret_cast<const char *>(kNoRow);
        to.scale = *(const __attribute__((address_space(1))) float *)s;
#pragma unroll
        for (int i = 0; i < S::kLoads; i++) {
            const char *k = pool + (uint64_t)row[i] * 16, *v = k + a.half_bytes;
            k = row[i] != kNoQuantRow ? k : none;
            v = row[i] != kNoQuantRow ? v : none;
            to.k[i] = __builtin_nontemporal_load((global_chunk_ptr)k);
            to.v[i] = __builtin_nontemporal_load((global_chunk_ptr)v);
        }
    };
    Ids ids = next_ids();

    // ---- what is computed: one item after the other
    TreeItem it;
    it.b = place.b;
    it.base = place.base;
    it.r = place.r;
    int cols, prior, st;
    u32x4 q[kBlocks][S::kSteps][S::kQTerms];                    // step 2 h + s: dims 64 h + 16 g + 8 s .. of the column
    u32x4 *const q_lds = reinterpret_cast<u32x4 *>(lds + S::kLds) + lane;
    unsigned long long mask[kBlocks];
    int limit[kBlocks];
    f32x4 o[kBlocks][S::kDimTiles];
    float m[kBlocks], l[kBlocks];
    auto start_item = [&](int unit) {
        open_item<S::kCols, S::kSub>(a, unit, begin, end, it);
        cols = min(it.r.n * a.group - it.ct * S::kCols, S::kCols);
        prior = it.r.prior;
        st = it.st0 + wave;
#pragma unroll
        for (int k = 0; k < kBlocks; k++) {
            const int col = it.ct * S::kCols + k * 16 + c;
            const int i = (int)((unsigned)col / (unsigned)a.group), hq = head * a.group + col - i * a.group;
            const bool there = k * 16 + c < cols;
            const char *row = there ? a.q + (it.r.first + i) * a.q_stride + hq * kD * S::kElt + g * 16 * S::kElt
                                    : reinterpret_cast<const char *>(kNoRow);
            const int apart = there ? 1 : 0;
#pragma unroll
            for (int e = 0; e < S::kSteps; e++) {
                if (S::kQInLds && (k * S::kSteps + e) % kTreeWaves != wave) continue;      // each wave a few
                const char *at = row + apart * ((e >> 1) * 64 + (e & 1) * 8) * S::kElt;
                q[k][e][0] = *(global_chunk_ptr)at;
                if constexpr (DT == DSKV_F32) q[k][e][1] = *(global_chunk_ptr)(at + 16);
            }
            mask[k] = !a.masks ? ~0ull : there ? (unsigned long long)a.masks[it.r.first + i] : 0;
            // tokens from `limit` on are not seen whatever the mask says
            const long lim = min(it.r.kv_len, (long)prior + (a.masks ? DSKV_MAX_TREE_ROWS : i + 1));
            limit[k] = there ? (int)max(lim, 0L) : 0;
            m[k] = -__FLT_MAX__;
            l[k] = 0;
#pragma unroll
            for (int d = 0; d < S::kDimTiles; d++) o[k][d] = f32x4{0, 0, 0, 0};
        }
    };
    // q and the masks are waited for in front of the loop
    auto settle_item = [&]() {
#pragma unroll
        for (int k = 0; k < kBlocks; k++) {
#pragma unroll
            for (int e = 0; e < S::kSteps; e++) {
                if (S::kQInLds && (k * S::kSteps + e) % kTreeWaves != wave) continue;
                if constexpr (DT == DSKV_F32) {
                    float f[8];
                    Chunk<DSKV_F32>::unpack(q[k][e][0], f);
                    Chunk<DSKV_F32>::unpack(q[k][e][1], f + 4);
                    split8<3>(f, q[k][e]);
                }
                asm volatile("" : "+v"(q[k][e][0]));
                if constexpr (S::kQInLds) {
#pragma unroll
                    for (int i = 0; i < S::kQTerms; i++) q_lds[((k * S::kSteps + e) * S::kQTerms + i) * 64] = q[k][e][i];
                }
            }
            asm volatile("" : "+v"(mask[k]));
        }
        if (S::kQInLds) __syncthreads();
    };
    auto subtile = [&]() {
        const uint32_t there_bits = held.there;
        const bool whole = there_bits == ~0u && (st + 1) * S::kSub <= prior + (a.masks ? 0 : 1);
        u32x4 key[S::kTiles][kD / 64];
        f32x4 k_scale[S::kTiles], v_scale[S::kTiles];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < S::kLoads; i++) {
            const int row = load_row + S::kRowsPerLoad * i;
            *reinterpret_cast<u32x4 *>(k_lds + row * S::kPitch + load_chunk * 16) = held.k[i];
            *reinterpret_cast<u32x4 *>(v_lds + row * S::kPitch + load_chunk * 16) = held.v[i];
        }
        scale_lds[lane] = lane < 32 ? held.scale * a.scale : held.scale;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        // LDS operands are read together and ahead
#pragma unroll
        for (int t = 0; t < S::kTiles; t++) {
#pragma unroll
            for (int h = 0; h < kD / 64; h++)
                key[t][h] = *reinterpret_cast<const u32x4 *>(k_lds + (t * 16 + c) * S::kPitch + h * 64 + g * 16);
            k_scale[t] = *reinterpret_cast<const f32x4 *>(scale_lds + t * 16 + 4 * g);
            v_scale[t] = *reinterpret_cast<const f32x4 *>(scale_lds + 32 + t * 16 + 4 * g);
        }
        __builtin_amdgcn_sched_barrier(0);
        const Ids ids_next = next_ids();
        request(ids, held);
        ids = ids_next;

        // ---- scores
        f32x4 s[kBlocks][S::kTiles];
#pragma unroll
        for (int t = 0; t < S::kTiles; t++) {
#pragma unroll
            for (int k = 0; k < kBlocks; k++) s[k][t] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < S::kSteps; e++) {
                const u32x4 chunk = key[t][e >> 1];
                const u32x4 x = operand_of<S::kKeyType>((e & 1) ? u32x2{chunk.z, chunk.w} : u32x2{chunk.x, chunk.y});
#pragma unroll
                for (int k = 0; k < kBlocks; k++)
#pragma unroll
                    for (int i = 0; i < S::kQTerms; i++)
                        s[k][t] = Elt<S::kKeyType>::mfma_k32(
                            x, S::kQInLds ? q_lds[((k * S::kSteps + e) * S::kQTerms + i) * 64] : q[k][e][i], s[k][t]);
            }
        }
        // V's codes: eight of a lane along the tokens for every 16 dims, in the order that the scores have them: 4 g .. 4 g + 3 and
        // 16 more.  Lane (g, x) supplies dims 8 (x % 2) .. of the x / 2-th of these.
        u32x2 value[S::kDimTiles];
        {
            typedef int lds_i32x2 __attribute__((ext_vector_type(2)));
            const int j = c >> 1, token = 4 * g + (j & 3) + (j >> 2) * 16;
            const char *at = v_lds + token * S::kPitch + (c & 1) * 8;
#pragma unroll
            for (int d = 0; d < S::kDimTiles; d++)
                value[d] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                                                         (__attribute__((address_space(3))) lds_i32x2 *)(at + d * 16)));
        }
        __builtin_amdgcn_sched_barrier(0);
        // ---- weights, under a maximum that is raised only where they ask for it
        u32x4 p[kBlocks][S::kPTerms];
#pragma unroll
        for (int k = 0; k < kBlocks; k++) {
            float x[8], w[8];
#pragma unroll
            for (int t = 0; t < S::kTiles; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) x[t * 4 + e] = s[k][t][e] * k_scale[t][e];
            if (!whole) {
                const uint32_t bits = (there_bits & seen_bits(st * S::kSub, prior, limit[k], mask[k], !a.masks)) >> (4 * g);
#pragma unroll
                for (int t = 0; t < S::kTiles; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (!((bits >> (t * 16 + e)) & 1)) x[t * 4 + e] = -INFINITY;
            }
            float sum = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                w[e] = __builtin_amdgcn_exp2f(x[e] - m[k]);
                sum += w[e];
            }
            if (__builtin_expect(__ballot(sum > most_weight(DSKV_BF16)) != 0, 0)) {
                float top = x[0];
#pragma unroll
                for (int e = 1; e < 8; e++) top = fmaxf(top, x[e]);
                top = fmaxf(m[k], quad_rows_max(top));
                const float keep = __builtin_amdgcn_exp2f(m[k] - top);
                m[k] = top;
                l[k] *= keep;
#pragma unroll
                for (int d = 0; d < S::kDimTiles; d++) o[k][d] *= keep;
                sum = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    w[e] = __builtin_amdgcn_exp2f(x[e] - top);
                    sum += w[e];
                }
            }
            l[k] += sum;
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] *= v_scale[e >> 2][e & 3];
            split8<S::kPTerms>(w, p[k]);
        }
        // ---- output
#pragma unroll
        for (int d = 0; d < S::kDimTiles; d++) {
            const u32x4 x = operand_of<DSKV_BF16>(value[d]);
#pragma unroll
            for (int k = 0; k < kBlocks; k++)
#pragma unroll
                for (int i = 0; i < S::kPTerms; i++) o[k][d] = Elt<DSKV_BF16>::mfma_k32(x, p[k][i], o[k][d]);
        }
        st += kTreeWaves;
    };
    auto finish_item = [&]() {
        // the waves' results meet
        float *const o_lds = reinterpret_cast<float *>(lds);
        float *const ml_lds = o_lds + kTreeWaves * S::kCols * S::kOPitch;
        __syncthreads();                                       // all waves are through with their K and V
#pragma unroll
        for (int k = 0; k < kBlocks; k++) {
            l[k] = quad_rows_sum(l[k]);
            const int col = wave * S::kCols + k * 16 + c;
            if (g == 0) {
                ml_lds[col * 2] = m[k];
                ml_lds[col * 2 + 1] = l[k];
            }
#pragma unroll
            for (int d = 0; d < S::kDimTiles; d++)
                *reinterpret_cast<f32x4 *>(o_lds + col * S::kOPitch + d * 16 + 4 * g) = o[k][d];
        }
        __syncthreads();
        const bool cut = it.st0 > 0 || it.st1 < it.r.subtiles;
        const PartSlot<S::kCols, kD> part(a, head, 2u * (uint32_t)share + (it.first ? 0u : 1u));
        constexpr int kQuads = kD / 4;
        for (int x = threadIdx.x; x < cols * kQuads; x += kTreeThreads) {
            const int col = x / kQuads, quad = x % kQuads;
            float top = ml_lds[col * 2];
#pragma unroll
            for (int w = 1; w < kTreeWaves; w++) top = fmaxf(top, ml_lds[(w * S::kCols + col) * 2]);
            float sum = 0;
            f32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < kTreeWaves; w++) {
                const float weight = __builtin_amdgcn_exp2f(ml_lds[(w * S::kCols + col) * 2] - top);
                sum += ml_lds[(w * S::kCols + col) * 2 + 1] * weight;
                acc += *reinterpret_cast<const f32x4 *>(o_lds + (w * S::kCols + col) * S::kOPitch + quad * 4) * weight;
            }
            if (cut) {
                part.put_o(col, quad * 4, acc);
                if (quad == 0) part.put_ml(col, top, sum);
            } else {
                put_result<DT, kD>(a, it.r.first, head, it.ct * S::kCols + col, quad * 4, acc, sum);
            }
        }
        if (cut) {
            const int item = it.base + it.ct * it.r.subtiles;
            join_parts<DT, kD, S::kCols, kTreeThreads>(a, place, it.r, parts_of(a, place, item, it.r.subtiles, it.ct), head, it.ct,
                                                       cols, &last_part);
        }
        __syncthreads();
    };
    start_item(begin);                                          // (its loads in front of those that wait for page ids)
    const Ids second = next_ids();
    request(ids, held);
    ids = second;
    for (;;) {
        settle_item();
        while (st < it.st1) subtile();
        finish_item();
        if (it.next >= end) return;
        start_item(it.next);
    }
}

}  // namespace dskv
