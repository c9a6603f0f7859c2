// The matrix form of the tree attention: head_dim 64 and 128, all three types.  See tree_attn.hip for what is computed.
//
// The columns of a kv head are its (row, q head of the group) pairs; S^T = K Q^T and O^T = V^T P^T keep a column in the
// lanes that share lane % 16, so its maximum and sum never cross more than four lanes.
// The work is cut without a host plan: request b has ct_b column tiles of kBlocks * 16 columns and st_b subtiles
// of kSub tokens; all (request, column tile, subtile) units lie end to end, every workgroup takes the sums over the requests for
// itself, and takes one of n shares of them, equal to one unit whatever the lengths (see tree_place for small batches).  One
// workgroup per (share, kv head); its four waves take the share's subtiles in turn, each with a running maximum, sum and O of
// its own, and meet in LDS where an item (request, column tile) ends.  An item that a share boundary cuts leaves
// a partial (maximum, sum, O in fp32) that tree_merge_kernel adds up.
// K and V go by whole rows through registers and a wave's own LDS: rows of 256 bytes are what
// HBM delivers best, and a row's page is looked up once per subtile, by lane, so pages may have any size.
//
// Bound by HBM where there is work enough: 64 requests of 5 rows over 256 - 4096 tokens (32 heads over 8, bf16, 0.6 GB) 117 us, of
// which the launch for cut items takes 5: 5.0 TB/s; its loads alone run in 96.  In short calls by latency: one request over
// 1.8 K tokens 13.9 us, 10.3 - 11 for the first launch (place of the share 2.6, page ids and requests 3, K and V 1.2, products 2, waves
// meet 2).  fp32: the matrix instruction takes 32 products a cycle and SIMD, 3.2 of the 4.5 us of a wave's subtile for 48 columns; 8
// requests over 300 - 700 tokens 28 us.
#pragma once

#include "kv_tile.h"
#include "rope_math.h"

namespace dskv {

constexpr int kTreeWaves = 4;
constexpr int kTreeThreads = kTreeWaves * 64;
// The running maximum of a column is raised only when a subtile's (block's) weights under it sum to more than most_weight in a lane.
// It is set headroom under the largest score then: float16 has normal numbers from 2^-14 to 2^16 only, and weights of 2^8 to 2^15 at the
// top leave those down to 2^-22 of the largest their eleven bits and are off by 2^-33 of it below.  (With 1 at the top, where a model parks its
// attention on few keys without a V, the others at 2^-22 of their weight gave results 2 % off, and none at all under 2^-25.)
constexpr float most_weight(int dtype) { return dtype == DSKV_F16 ? 32768.f : 256.f; }
constexpr float headroom(int dtype) { return dtype == DSKV_F16 ? 8.f : 0.f; }
constexpr int kMostTokens = 1 << 30;        // of a request in the matrix forms: what n_page_indices pages hold
constexpr int kTreeMostRows = 1024;         // of a request in the matrix forms; longer chunks are a prefill's

struct TreeArgs {
    const int32_t *qo_indptr, *kv_page_indptr, *kv_page_indices, *kv_last_page_lens;
    const int64_t *masks;
    char *out;
    const char *q, *pages;
    long q_stride, n_page_indices;        // q_stride in bytes
    int batch, nnz, max_rows, n_qo_heads, n_kv_heads, head_dim, page_size, num_pages;
    float scale;                          // sm_scale / log 2
    // matrix forms
    uint32_t page_magic;                  // ceil(2^page_shift / page_size): t / page_size = t * page_magic >> page_shift
    int page_shift;
    float *part_o, *part_ml;              // (2 * n_shares, n_kv_heads, columns of a tile, head_dim | 2)
    int32_t *units_before;                // (batch + 4): units (parts) of the requests in front; see tree_place
    int n_shares, group;
    int sides;                            // see side_by_side
};

// Workgroups a compute unit: two where the registers allow it.  Else one, with one wave a SIMD: 128 dims take 256 VGPRs and 80 - 230
// accumulation registers, 64 dims with 48 or 64 columns 256 and 80 - 140; 64 dims with fewer 175 - 228 in all.
constexpr int tree_workgroups(int dim, int blocks) { return dim == 64 && blocks <= 2 ? 2 : 1; }

// Columns of a tile at most: what a wave's registers hold beside the K and V on their way.
// (64 of 128 dims spill: 64 requests of 16 rows over 4 K tokens each 253 us, the wide form 214.)
constexpr int tree_columns(int dim) { return dim == 64 ? 64 : 48; }
// Subtiles a wave has in flight, in registers: two where there is room for them.  64 requests over 256 - 4096 tokens, bf16, 32 heads
// over 8: of 8 rows 121 us, with one set 122; 64 dims, of 12 rows 79 and 91.  With less to compute per subtile one set is no worse: of 5
// rows 118 and 117, of one row 105 and 102; 64 dims, of 5 rows 72 and 67; one request over 1.8 K tokens 14.7 and 13.8.
constexpr int tree_depth(int dim, int blocks) { return dim == 64 || blocks <= 2 ? 2 : 1; }

template <int DT, int kD, int kBlocks> struct TreeShape {
    static constexpr int kElt = DT == DSKV_F32 ? 4 : 2;
    static constexpr int kSub = DT == DSKV_F32 ? 16 : 32;            // tokens of a subtile
    static constexpr int kTiles = kSub / 16;
    static constexpr int kRow = kD * kElt;                           // bytes
    static constexpr int kChunks = kRow / 16;                        // 16-byte chunks of a row
    static constexpr int kRowsPerLoad = 64 / kChunks;
    static constexpr int kLoads = kSub / kRowsPerLoad;
    static constexpr int kSteps = kD * kElt / 64;                    // 16-byte operand chunks of a lane along the dims
    static constexpr int kDimTiles = kD / 16;
    static constexpr int kCols = kBlocks * 16;
    static constexpr int kKPitch = kRow + 16;                        // 16 rows' chunks at one offset meet no bank twice
    static constexpr int kVPitch = DT == DSKV_F32 ? kRow + 16 : kRow + 32;
    static constexpr int kWaveLds = kSub * (kKPitch + kVPitch);
    static constexpr int kOPitch = kD + 4;                           // floats
    static constexpr int kMergeLds = kTreeWaves * kCols * (kOPitch + 2) * 4;
    static constexpr int kLds = kTreeWaves * kWaveLds > kMergeLds ? kTreeWaves * kWaveLds : kMergeLds;
};

// Tokens of a request by the index arrays.  Those may promise more than the tensors hold: an entry behind the last of kv_page_indices is
// no page, and where a table begins in front of the first there is none either.
struct TreeTokens {
    long len;            // cached and new ones
    long walk;           // from here on no token lies in a page
};
__device__ __forceinline__ TreeTokens tree_tokens(int page0, int page_end, int last, int page_size, long n_page_indices)
{
    const long pages = (long)page_end - page0, entries = page0 < 0 ? 0L : max(n_page_indices - page0, 0L);
    TreeTokens x;
    x.len = pages > 0 ? max((pages - 1) * page_size + min(last, page_size), 0L) : 0L;
    x.walk = min(x.len, entries * page_size);
    return x;
}

struct TreeRequest {
    long first;          // its first row
    long kv_len;         // tokens that its rows may see
    int prior;           // tokens in front of its rows
    int page0;
    int n;               // rows that are computed
    int col_tiles, subtiles;
    int tile;            // columns of a tile: its tiles are as even as 32 columns a wave allow
};

// What the arrays say about request b, within the bounds of the tensors.
template <int kCols, int kSub> __device__ __forceinline__ TreeRequest tree_request(const TreeArgs &a, int b)
{
    // (through the constant address space: scalar loads where b is uniform, also after the kernel has stored)
    const const_i32_ptr qo = as_const(a.qo_indptr) + b, kv = as_const(a.kv_page_indptr) + b;
    TreeRequest r;
    r.first = qo[0];
    const long rows = (long)qo[1] - r.first;
    r.page0 = kv[0];
    const TreeTokens tokens = tree_tokens(kv[0], kv[1], as_const(a.kv_last_page_lens)[b], a.page_size, a.n_page_indices);
    r.n = r.first < 0 ? 0 : (int)max(min(min(rows, (long)a.max_rows), (long)a.nnz - r.first), 0L);
    const long prior = tokens.len - rows;
    r.kv_len = max(min(tokens.walk, prior + (a.masks ? DSKV_MAX_TREE_ROWS : r.n)), 0L);
    r.prior = (int)max(min(prior, (long)kMostTokens), -(long)kMostTokens);       // (further off than any token that is walked)
    r.col_tiles = (r.n * a.group + kCols - 1) / kCols;
    r.tile = kCols;
    if (kCols > tree_columns(64) && r.col_tiles > 1) r.tile = (r.n * a.group + 32 * r.col_tiles - 1) / (32 * r.col_tiles) * 32;
    r.subtiles = max((int)((r.kv_len + kSub - 1) / kSub), 1);        // a row that sees nothing is written too
    return r;
}

// Equal shares: `each` units, the first `longer` shares one more.  Units are counted in 32 bits (what the arrays can hold fits; a
// batch whose arrays contradict themselves so that it does not is left out): divisions of 64 bits cost a short call a
// microsecond.
struct Shares {
    int each, longer, used;
};
__device__ __forceinline__ Shares shares_of(int units, int used)                  // used > 0
{
    Shares s;
    s.used = used;
    s.each = (int)((unsigned)units / (unsigned)used);
    s.longer = units - s.each * used;
    return s;
}
__device__ __forceinline__ int share_begin(const Shares &s, int share) { return share * s.each + min(share, s.longer); }
__device__ __forceinline__ int share_with(const Shares &s, int unit)              // units >= used
{
    const int of_longer = s.longer * (s.each + 1);
    return unit < of_longer ? (int)((unsigned)unit / (unsigned)(s.each + 1))
                            : s.longer + (int)((unsigned)(unit - of_longer) / (unsigned)s.each);
}

// Share and kv head of a workgroup.  Workgroups go round the eight XCDs in turn; the heads of a share belong on
// one, since their rows of a token lie side by side: with a head per XCD every one of its L2s would be
// asked for every eighth 256 bytes, by two of its sixteen channels.
__device__ __forceinline__ void share_and_head(const TreeArgs &a, int &share, int &head)
{
    const int wg = blockIdx.x;
    if (a.n_shares % 8 == 0) {
        share = wg % 8 + wg / 8 / a.n_kv_heads * 8;        // (few shares in use are spread over the XCDs)
        head = wg / 8 % a.n_kv_heads;
    } else {
        share = wg / a.n_kv_heads;
        head = wg % a.n_kv_heads;
    }
}

// Column tiles side by side.  Where (nearly) all requests have a.sides column tiles, their workgroups walk the same
// tokens at the same time, on one XCD: K and V then come from its L2 for all but one of them (16 trees of 33 - 64 rows, two
// tiles: 0.34 instead of 1.08 GB from HBM, 288 us instead of 305).  Units are subtiles there, and
// share (x + 8 j) takes column tile j % sides of span x + 8 (j / sides).  (n_shares is a multiple of 8 * sides.)
__device__ __forceinline__ int share_of_span(int span, int side, int sides) { return span % 8 + 8 * (span / 8 * sides + side); }
__device__ __forceinline__ bool side_by_side(const TreeArgs &a, long units, long spans)
{
    // idle workgroups cost what they save beyond a quarter
    return a.sides > 1 && 4 * a.sides * spans <= 5 * units;
}
__device__ __forceinline__ long units_of(const TreeRequest &r, bool beside)
{
    return beside ? (r.col_tiles > 0 ? r.subtiles : 0) : (long)r.col_tiles * r.subtiles;
}

// Sums up to and with this lane's over a wave, by moves between lanes that do not go through LDS.
template <int kCtrl, int kRows> __device__ __forceinline__ long lanes_below(long v)
{
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, kCtrl, kRows, 0xf, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)((uint64_t)v >> 32), kCtrl, kRows, 0xf, true);
    return (long)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ long wave_scan(long v)
{
    v += lanes_below<0x111, 0xf>(v);       // row_shr 1, 2, 4, 8 within 16 lanes
    v += lanes_below<0x112, 0xf>(v);
    v += lanes_below<0x114, 0xf>(v);
    v += lanes_below<0x118, 0xf>(v);
    v += lanes_below<0x142, 0xa>(v);       // the last lane of rows 0 and 2 to rows 1 and 3
    v += lanes_below<0x143, 0xc>(v);       // lane 31 to rows 2 and 3
    return v;
}

// Where the workgroup's share begins and ends, by all of its kThreads threads; the first workgroup leaves the
// sums for the merge launch.
struct TreePlace {
    int begin, end;      // units; equal: nothing to do
    int base;            // units in front of request b
    int b;
    bool beside;
    int side;
    TreeRequest r;       // request b
};
// A share that goes over from one item to another starts twice and joins its waves' results twice, which a small batch notices: if
// parts of a common number of units, whole turns (kTurn) and at most two turns more than equal shares have, take no more
// shares than there are, no part crosses an item's end.  Measured against equal shares (32 heads over 8, bf16): 3 requests of 5 rows over
// 50 - 500 tokens 14.5 for 18.4 us, 8 over 1 - 4 K 26.6 for 29.5, 8 over 4 - 16 K 65.0 for 67.1, 8 trees of 64 rows over 1 - 4 K
// 54 for 64.5; at 16 over 2 - 8 K they take too many shares.
template <int kCols, int kSub, int kThreads, bool kSides, int kLeast, int kTurn>
__device__ __forceinline__ void tree_place(const TreeArgs &a, int share, TreePlace &at)
{
    __shared__ long scan[2][kThreads / 64], scan_parts[kThreads / 64];
    __shared__ int busy_of[kThreads / 64];
    __shared__ int found_base, found_b, found_begin, found_end;
    __shared__ TreeRequest found_r;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int per = (a.batch + kThreads - 1) / kThreads;
    const int b0 = threadIdx.x * per, b1 = min(b0 + per, a.batch);
    long mine[2] = {0, 0}, upto[2];        // units; with column tiles side by side
    TreeRequest r;
    for (int b = b0; b < b1; b++) {
        r = tree_request<kCols, kSub>(a, b);
        mine[0] += units_of(r, false);
        if (kSides) mine[1] += units_of(r, true);
    }
    long total[2] = {0, 0};
    const unsigned long long busy = __ballot(b0 < b1 && r.n > 0);
    if (lane == 0) busy_of[wave] = __popcll(busy);
#pragma unroll
    for (int i = 0; i < (kSides ? 2 : 1); i++) {
        upto[i] = wave_scan(mine[i]);
        if (lane == 63) scan[i][wave] = upto[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < (kSides ? 2 : 1); i++)
#pragma unroll
        for (int w = 0; w < kThreads / 64; w++) {
            if (w == wave) upto[i] += total[i];
            total[i] += scan[i][w];
        }
    at.beside = kSides && side_by_side(a, total[0], total[1]);
    const int which = kSides && at.beside ? 1 : 0;
    const long sum = which ? total[1] : total[0];
    const int units = sum <= INT32_MAX ? (int)sum : 0;
    int span = share, spans = a.n_shares;
    at.side = 0;
    if (which) {
        const int j = share / 8;
        at.side = j % a.sides;
        span = share % 8 + 8 * (j / a.sides);
        spans = a.n_shares / a.sides;
    }
    // Shares in use: of no fewer units than kLeast, but as many as there are requests with rows, if there are as many (40 requests of
    // 8 rows over 3 - 21 tokens 21 us, with kLeast alone 33; 70 of 64 rows over 3 - 60 tokens 72 and 75, of 5 rows 33.5 and 32.5; where
    // parts take no more shares than there are, these decide, and both are the same).
    int requests = per > 1 ? spans : 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; w++) requests += busy_of[w];
    const int used = max(min(min(spans, units), max((int)(((unsigned)units + kLeast - 1) / kLeast), requests)), 1);
    const Shares shares = shares_of(units, used);
    at.begin = at.end = 0;
    if (span < shares.used) {
        at.begin = share_begin(shares, span);
        at.end = share_begin(shares, span + 1);
    }
    int before = (int)((which ? upto[1] : upto[0]) - (which ? mine[1] : mine[0]));
    const bool tells = blockIdx.x == 0;
    if constexpr (kTurn > 0) {
        if (a.batch > 1 && a.batch <= spans && per == 1 && units > 0) {     // (`parts` is of one request a thread)
            const int most = shares.each + (shares.longer > 0);
            const int cut = most <= kLeast ? kLeast : (most + kTurn - 1) / kTurn * kTurn, cut_more = (cut + 2 * kTurn - 1) / kTurn * kTurn;
            const int tiles = which ? (r.col_tiles > 0) : r.col_tiles;
            long parts = 0;                                                 // of `cut` units and, in the upper half, a turn more
            if (b0 < b1)
                parts = (long)tiles * ((unsigned)(r.subtiles + cut - 1) / (unsigned)cut) |
                        (long)tiles * ((unsigned)(r.subtiles + cut_more - 1) / (unsigned)cut_more) << 32;
            long parts_upto = wave_scan(parts), parts_total = 0;
            if (lane == 63) scan_parts[wave] = parts_upto;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kThreads / 64; w++) {
                if (w == wave) parts_upto += parts_total;
                parts_total += scan_parts[w];
            }
            const bool fits = (int)parts_total <= spans;
            const int half = fits ? 0 : 32, total_parts = (int)(parts_total >> half), part = fits ? cut : cut_more;
            if (total_parts <= spans) {
                const int p = (int)(parts >> half), first = (int)(parts_upto >> half) - p;
                if (p > 0 && first <= span && span < first + p) {
                    const int of_item = (int)((unsigned)p / (unsigned)tiles), ct = (span - first) / of_item;
                    const int item = before + ct * r.subtiles;
                    found_begin = item + (span - first - ct * of_item) * part;
                    found_end = found_begin + min(part, item + r.subtiles - found_begin);
                    found_b = b0;
                    found_base = before;
                    found_r = r;
                }
                if (tells && b0 < b1) a.units_before[b0] = first;
                if (tells && b1 == a.batch) {
                    a.units_before[a.batch] = units;
                    a.units_before[a.batch + 1] = which;
                    a.units_before[a.batch + 2] = part;
                }
                __syncthreads();
                at.begin = span < total_parts ? found_begin : 0;
                at.end = span < total_parts ? found_end : 0;
                at.b = __builtin_amdgcn_readfirstlane(found_b);
                at.base = found_base;
                at.r = found_r;
                return;
            }
        }
    }
    if (tells || (before <= at.begin && at.begin < (int)(which ? upto[1] : upto[0]))) {
        for (int b = b0; b < b1; b++) {
            if (per > 1) r = tree_request<kCols, kSub>(a, b);
            const int u = (int)units_of(r, which);
            if (tells) a.units_before[b] = before;
            if (before <= at.begin && at.begin < before + u) {
                found_b = b;
                found_base = before;
                found_r = r;
            }
            before += u;
        }
        if (tells && b1 == a.batch) {
            a.units_before[a.batch] = units;
            a.units_before[a.batch + 1] = which;
            a.units_before[a.batch + 2] = 0;
            a.units_before[a.batch + 3] = used;
        }
    }
    __syncthreads();
    at.b = __builtin_amdgcn_readfirstlane(found_b);
    at.base = found_base;
    at.r = found_r;
}
// (LDS words are vectors for the compiler: an index that is the same for all lanes is said to be)
__device__ __forceinline__ long uniform(long x)
{
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)x), hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)((uint64_t)x >> 32));
    return (long)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ void make_uniform(TreePlace &at)
{
    at.begin = __builtin_amdgcn_readfirstlane(at.begin);
    at.end = __builtin_amdgcn_readfirstlane(at.end);
    at.base = __builtin_amdgcn_readfirstlane(at.base);
    at.r.first = uniform(at.r.first);
    at.r.kv_len = uniform(at.r.kv_len);
    at.r.prior = __builtin_amdgcn_readfirstlane(at.r.prior);
    at.r.page0 = __builtin_amdgcn_readfirstlane(at.r.page0);
    at.r.n = __builtin_amdgcn_readfirstlane(at.r.n);
    at.r.col_tiles = __builtin_amdgcn_readfirstlane(at.r.col_tiles);
    at.r.subtiles = __builtin_amdgcn_readfirstlane(at.r.subtiles);
    at.r.tile = __builtin_amdgcn_readfirstlane(at.r.tile);
}

// t / page_size for 0 <= t < 2^31: with s = 31 + ceil(log2 P) and M = ceil(2^s / P) < 2^32 the error of t M / 2^s is under
// t / 2^s <= 1 / P.
__device__ __forceinline__ int page_number(const TreeArgs &a, int t)
{
    return (int)((uint64_t)(uint32_t)t * a.page_magic >> a.page_shift);
}
// Page of token t of a request, and its row of the pool (page * 2 P + place: K; V lies P rows on), -1 where there is none.
__device__ __forceinline__ int page_of(const TreeArgs &a, const TreeRequest &r, int t)
{
    const int entry = r.page0 + page_number(a, t);
    return t < (int)r.kv_len && entry >= 0 && entry < (int)a.n_page_indices ? a.kv_page_indices[entry] : -1;
}
__device__ __forceinline__ int pool_row(const TreeArgs &a, int t, int page)
{
    return page >= 0 && page < a.num_pages ? page * 2 * a.page_size + t - page_number(a, t) * a.page_size : -1;
}

static __device__ const u32x4 kNoRow[32] = {};          // what a token that there is not reads as
// (a pointer that may be to it or to the pool would be loaded from as a flat one, which waits for LDS, too)
typedef const __attribute__((address_space(1))) u32x4 *global_chunk_ptr;

// Which of the `count` <= 32 tokens from t on a column sees, as bits: `prior` tokens lie in front of the new ones, of which its
// mask names some (all: no mask), and none from `limit` on.
__device__ __forceinline__ uint32_t seen_bits(int t, int prior, int limit, unsigned long long mask, bool all)
{
    const int from = t - prior, left = limit - t;
    uint32_t bits;
    if (all || from <= -32) bits = ~0u;
    else if (from >= 0) bits = from < 64 ? (uint32_t)(mask >> from) : 0u;
    else bits = (uint32_t)(mask << -from) | ((1u << -from) - 1);
    return left <= 0 ? 0u : left >= 32 ? bits : bits & ((1u << left) - 1);
}

// Whether some of 16 bytes of elements is infinite or no number: its exponent is all ones, and one more carries into the sign.
template <int DT> __device__ __forceinline__ bool no_number(u32x4 x)
{
    constexpr uint32_t kExponent = DT == DSKV_F32 ? 0x7F800000u : DT == DSKV_BF16 ? 0x7F807F80u : 0x7C007C00u;
    constexpr uint32_t kOne = DT == DSKV_F32 ? 0x00800000u : DT == DSKV_BF16 ? 0x00800080u : 0x04000400u;
    constexpr uint32_t kSign = DT == DSKV_F32 ? 0x80000000u : 0x80008000u;
    uint32_t any = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) any |= (x[w] & kExponent) + kOne;
    return (any & kSign) != 0;
}

template <int DT, int kD, int kBlocks> struct TreeRegs {
    typedef TreeShape<DT, kD, kBlocks> S;
    u32x4 k[S::kLoads], v[S::kLoads];
};

// A share's walk through its items; one item at a time.
struct TreeItem {
    TreeRequest r;
    int base;            // units in front of request b
    int next;            // the first unit behind the item's part
    int b, ct, st0, st1; // column tile; subtiles of the part
    bool first;          // of the share
};
template <int kCols, int kSub>
__device__ __forceinline__ void open_item(const TreeArgs &a, int unit, int begin, int end, TreeItem &it)
{
    while (unit >= it.base + (int)units_of(it.r, false)) {         // on to the next request that has rows
        it.base += (int)units_of(it.r, false);
        it.b++;
        it.r = tree_request<kCols, kSub>(a, it.b);
    }
    it.ct = (int)((unsigned)(unit - it.base) / (unsigned)it.r.subtiles);
    const int item = it.base + it.ct * it.r.subtiles;
    it.st0 = (int)(unit - item);
    it.st1 = min(end - item, it.r.subtiles);
    it.next = item + it.st1;
    it.first = unit == begin;
}

template <int DT, int kD, int kBlocks>
__global__ __launch_bounds__(kTreeThreads, tree_workgroups(kD, kBlocks)) void tree_matrix_kernel(TreeArgs a)
{
    typedef TreeShape<DT, kD, kBlocks> S;
    __shared__ __align__(16) char lds[S::kLds];
    __shared__ unsigned bad_at[kTreeMostRows / S::kSub + 2 + 2 * kTreeWaves];    // bit per token of a subtile with new rows: its V is no number
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, c = lane & 15;
    int share, head;
    share_and_head(a, share, head);
    TreePlace place;
    tree_place<S::kCols, S::kSub, kTreeThreads, false, kTreeWaves, kTreeWaves * tree_depth(kD, kBlocks)>(a, share, place);
    make_uniform(place);
    const int begin = place.begin, end = place.end;
    if (begin >= end) return;

    char *const k_lds = lds + wave * S::kWaveLds, *const v_lds = k_lds + S::kSub * S::kKPitch;
    const int row_bytes = a.n_kv_heads * S::kRow;
    const long half_bytes = (long)a.page_size * row_bytes;
    const int load_row = lane / S::kChunks, load_chunk = lane % S::kChunks;
    const char *const pool = a.pages + head * S::kRow + load_chunk * 16;
    const char *const none = reinterpret_cast<const char *>(kNoRow) + load_chunk * 16;

    // ---- what is requested: the wave's subtiles through all items of the share, kDepth in flight, their page ids one step
    // further ahead (a wave's loads return in order: an id that is requested in front of the rows before it does not wait for those)
    TreeItem ahead;
    ahead.b = place.b;
    ahead.base = place.base;
    ahead.r = place.r;
    open_item<S::kCols, S::kSub>(a, begin, begin, end, ahead);
    // A wave takes a whole number of turns through its register sets per item, the last perhaps for subtiles that there are not: which set is
    // whose turn is known at compile time then, and the waits for one leave the other on its way.
    constexpr int kDepth = tree_depth(kD, kBlocks);
    auto walk_end = [&](const TreeItem &x) {                    // of the wave's subtiles st0 + wave, + kTreeWaves ..
        constexpr int kTurn = kDepth * kTreeWaves;
        return x.st0 + wave + max((x.st1 - x.st0 - wave + kTurn - 1) / kTurn, 0) * kTurn;
    };
    int ahead_st = ahead.st0 + wave, ahead_end = walk_end(ahead);
    bool more = true;
    auto settle = [&]() {                                       // on to a subtile that there is
        if (__builtin_expect(ahead_st < ahead_end, 1)) return;
        while (more && ahead_st >= ahead_end) {
            more = ahead.next < end;
            if (more) {
                open_item<S::kCols, S::kSub>(a, ahead.next, begin, end, ahead);
                ahead_st = ahead.st0 + wave;
                ahead_end = walk_end(ahead);
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
        x.page = more && ahead_st < ahead.st1 ? page_of(a, ahead.r, x.t) : -1;
        ahead_st += kTreeWaves;
        return x;
    };
    TreeRegs<DT, kD, kBlocks> regs[kDepth];
    unsigned long long held_of[kDepth];
    auto request = [&](const Ids &x, TreeRegs<DT, kD, kBlocks> &to, unsigned long long &held) {
        const int rows = pool_row(a, x.t, x.page);
        held = __ballot(rows >= 0);                             // tokens that there are (lanes repeat)
        int row[S::kLoads];
#pragma unroll
        for (int i = 0; i < S::kLoads; i++) row[i] = __shfl(rows, load_row + S::kRowsPerLoad * i);
#pragma unroll
        for (int i = 0; i < S::kLoads; i++) {
            const char *k = pool + (uint64_t)(uint32_t)row[i] * (uint32_t)row_bytes, *v = k + half_bytes;
            k = row[i] >= 0 ? k : none;
            v = row[i] >= 0 ? v : none;
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
    int cols, prior, new_from, st;
    u32x4 q[kBlocks][S::kSteps];
    unsigned long long mask[kBlocks];
    int limit[kBlocks];
    f32x4 o[kBlocks][S::kDimTiles];
    float m[kBlocks], l[kBlocks];
    auto start_item = [&](int unit) {
        open_item<S::kCols, S::kSub>(a, unit, begin, end, it);
        cols = min(it.r.n * a.group - it.ct * S::kCols, S::kCols);
        prior = it.r.prior;
        new_from = max(prior, 0) / S::kSub;                     // first subtile with new rows
        st = it.st0 + wave;
#pragma unroll
        for (int k = 0; k < kBlocks; k++) {
            const int col = it.ct * S::kCols + k * 16 + c;
            const int i = (int)((unsigned)col / (unsigned)a.group), hq = head * a.group + col - i * a.group;
            const bool there = k * 16 + c < cols;
            const char *row = there ? a.q + (it.r.first + i) * a.q_stride + hq * S::kRow + g * 16
                                    : reinterpret_cast<const char *>(kNoRow) + g * 16;
#pragma unroll
            for (int s = 0; s < S::kSteps; s++) q[k][s] = *(global_chunk_ptr)(row + s * 64);
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
            for (int s = 0; s < S::kSteps; s++) asm volatile("" : "+v"(q[k][s]));
            asm volatile("" : "+v"(mask[k]));
        }
    };
    auto subtile = [&](TreeRegs<DT, kD, kBlocks> &mine, unsigned long long &held_here) {
        const unsigned long long held = held_here;
        const bool whole = held == ~0ull && (st + 1) * S::kSub <= prior + (a.masks ? 0 : 1);
        const bool there = st < it.st1;                         // (else a turn without a subtile)
        u32x4 key[S::kTiles][S::kSteps];
        if (there) {
            __builtin_amdgcn_wave_barrier();
            // A weight of 0 times a V that is no number would reach columns that do not see the token: such tokens among the
            // new ones are taken out here and added behind the walk.
            if (st >= new_from) {
                unsigned bad = 0;
                bool odd[S::kLoads], any = false;
#pragma unroll
                for (int i = 0; i < S::kLoads; i++) {
                    odd[i] = no_number<DT>(mine.v[i]);
                    any |= odd[i];
                }
                if (__builtin_expect(__ballot(any) != 0, 0)) {
#pragma unroll
                    for (int i = 0; i < S::kLoads; i++) {
                        const unsigned long long odd_lanes = __ballot(odd[i]);
#pragma unroll
                        for (int j = 0; j < S::kRowsPerLoad; j++) {
                            const unsigned long long of_row = ((1ull << S::kChunks) - 1) << (j * S::kChunks);
                            if (odd_lanes & of_row) bad |= 1u << (j + S::kRowsPerLoad * i);
                        }
                        if ((bad >> (load_row + S::kRowsPerLoad * i)) & 1) mine.v[i] = u32x4{0, 0, 0, 0};
                    }
                }
                if (lane == 0) bad_at[st - new_from] = bad;
            }
#pragma unroll
            for (int i = 0; i < S::kLoads; i++) {
                const int row = load_row + S::kRowsPerLoad * i;
                *reinterpret_cast<u32x4 *>(k_lds + row * S::kKPitch + load_chunk * 16) = mine.k[i];
                *reinterpret_cast<u32x4 *>(v_lds + row * S::kVPitch + load_chunk * 16) = mine.v[i];
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            // LDS operands are read together and ahead: one wave a SIMD has nobody to wait for them in its place
#pragma unroll
            for (int t = 0; t < S::kTiles; t++)
#pragma unroll
                for (int e = 0; e < S::kSteps; e++)
                    key[t][e] = *reinterpret_cast<const u32x4 *>(k_lds + (t * 16 + c) * S::kKPitch + e * 64 + g * 16);
        }
        __builtin_amdgcn_sched_barrier(0);
        const Ids ids_next = next_ids();
        request(ids, mine, held_here);
        ids = ids_next;
        if (!there) {
            st += kTreeWaves;
            return;
        }

        // ---- scores
        f32x4 s[kBlocks][S::kTiles];
#pragma unroll
        for (int t = 0; t < S::kTiles; t++) {
#pragma unroll
            for (int k = 0; k < kBlocks; k++) s[k][t] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < S::kSteps; e++) {
#pragma unroll
                for (int k = 0; k < kBlocks; k++) {
                    if constexpr (DT == DSKV_F32) {
                        const f32x4 kf = __builtin_bit_cast(f32x4, key[t][e]), qf = __builtin_bit_cast(f32x4, q[k][e]);
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            s[k][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j], qf[j], s[k][t], 0, 0, 0);
                    } else {
                        s[k][t] = Elt<DT>::mfma_k32(key[t][e], q[k][e], s[k][t]);
                    }
                }
            }
        }
        // V's operands: four of a lane along the tokens for every 16 dims
        u32x4 value[S::kDimTiles];
#pragma unroll
        for (int d = 0; d < S::kDimTiles; d++) {
            if constexpr (DT == DSKV_F32) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    value[d][e] = *reinterpret_cast<const uint32_t *>(v_lds + (4 * g + e) * S::kVPitch + (d * 16 + c) * 4);
            } else {
                const char *at = v_lds + (4 * g + (c >> 2)) * S::kVPitch + d * 32 + (c & 3) * 8;
                const u32x2 lo = read_transposed(at), hi = read_transposed(at + 16 * S::kVPitch);
                value[d] = u32x4{lo.x, lo.y, hi.x, hi.y};
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        // ---- weights, under a maximum that is raised only where they ask for it
        u32x4 p[kBlocks];                                  // 16-bit: the operand; fp32: four floats
#pragma unroll
        for (int k = 0; k < kBlocks; k++) {
            float x[S::kTiles * 4], w[S::kTiles * 4];
#pragma unroll
            for (int t = 0; t < S::kTiles; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) x[t * 4 + e] = s[k][t][e] * a.scale;
            if (!whole) {
                const uint32_t bits = ((uint32_t)held & seen_bits(st * S::kSub, prior, limit[k], mask[k], !a.masks)) >> (4 * g);
#pragma unroll
                for (int t = 0; t < S::kTiles; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (!((bits >> (t * 16 + e)) & 1)) x[t * 4 + e] = -INFINITY;
            }
            float sum = 0;
#pragma unroll
            for (int e = 0; e < S::kTiles * 4; e++) {
                w[e] = __builtin_amdgcn_exp2f(x[e] - m[k]);
                sum += w[e];
            }
            if (__builtin_expect(__ballot(sum > most_weight(DT)) != 0, 0)) {
                float top = x[0];
#pragma unroll
                for (int e = 1; e < S::kTiles * 4; e++) top = fmaxf(top, x[e]);
                top = fmaxf(m[k], quad_rows_max(top) - headroom(DT));
                const float keep = __builtin_amdgcn_exp2f(m[k] - top);
                m[k] = top;
                l[k] *= keep;
#pragma unroll
                for (int d = 0; d < S::kDimTiles; d++) o[k][d] *= keep;
                sum = 0;
#pragma unroll
                for (int e = 0; e < S::kTiles * 4; e++) {
                    w[e] = __builtin_amdgcn_exp2f(x[e] - top);
                    sum += w[e];
                }
            }
            l[k] += sum;
            if constexpr (DT == DSKV_F32) {
                p[k] = __builtin_bit_cast(u32x4, f32x4{w[0], w[1], w[2], w[3]});
            } else {
                // rounded to 16 bits for the matrix product: half a step of each weight (see headroom); bf16 results are off by
                // 0.0020 - 0.0023 of their norm, with weights in 32 bits by 0.0017, their own rounding
#pragma unroll
                for (int e = 0; e < 4; e++) p[k][e] = Elt<DT>::pack2(w[2 * e], w[2 * e + 1]);
            }
        }
        // ---- output
#pragma unroll
        for (int d = 0; d < S::kDimTiles; d++)
#pragma unroll
            for (int e = 0; e < (DT == DSKV_F32 ? 4 : 1); e++)
#pragma unroll
                for (int k = 0; k < kBlocks; k++) {
                    if constexpr (DT == DSKV_F32)
                        o[k][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, value[d])[e],
                                                                       __builtin_bit_cast(f32x4, p[k])[e], o[k][d], 0, 0, 0);
                    else o[k][d] = Elt<DT>::mfma_k32(value[d], p[k], o[k][d]);
                }
        st += kTreeWaves;
    };
    auto finish_item = [&]() {
        // ---- the wave's tokens that were taken out, for the columns that see them
        for (st = it.st0 + wave; st < it.st1; st += kTreeWaves) {
            if (st < new_from) continue;
            unsigned bad = __builtin_amdgcn_readfirstlane(bad_at[st - new_from]);
            while (__builtin_expect(bad != 0, 0)) {
                const int token = __builtin_ctz(bad);
                bad &= bad - 1;
                const int t = st * S::kSub + token;
                const int row = pool_row(a, t, page_of(a, it.r, t));
                if (row < 0) continue;
                const char *key = a.pages + (uint64_t)(uint32_t)row * (uint32_t)row_bytes + head * S::kRow;
                const char *value = key + half_bytes;
#pragma unroll
                for (int k = 0; k < kBlocks; k++) {
                    float s = 0;
#pragma unroll
                    for (int e = 0; e < S::kSteps; e++) {
                        constexpr int E = Chunk<DT>::kElems;
                        float x[E], y[E];
                        Chunk<DT>::unpack(*reinterpret_cast<const u32x4 *>(key + e * 64 + g * 16), x);
                        Chunk<DT>::unpack(q[k][e], y);
#pragma unroll
                        for (int d = 0; d < E; d++) s = fmaf(x[d], y[d], s);
                    }
                    const float weight = __builtin_amdgcn_exp2f(quad_rows_sum(s) * a.scale - m[k]);
                    if ((seen_bits(st * S::kSub, prior, limit[k], mask[k], !a.masks) >> token) & 1) {
#pragma unroll
                        for (int d = 0; d < S::kDimTiles; d++)
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                o[k][d][e] += weight * LoadElt<DT>::get(value, d * 16 + 4 * g + e);
                    }
                }
            }
        }

        // ---- the waves' results meet
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
        const long slot = 2L * share + (it.first ? 0 : 1);
        const long part = (slot * a.n_kv_heads + head) * S::kCols;
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
                *reinterpret_cast<f32x4 *>(a.part_o + (part + col) * kD + quad * 4) = acc;
                if (quad == 0) {
                    a.part_ml[(part + col) * 2] = top;
                    a.part_ml[(part + col) * 2 + 1] = sum;
                }
            } else {
                const int at = it.ct * S::kCols + col, i = (int)((unsigned)at / (unsigned)a.group), hq = head * a.group + at - i * a.group;
                const float inv = sum == 0 ? 0.f : 1.f / sum;
                char *dst = a.out + ((it.r.first + i) * a.n_qo_heads + hq) * S::kRow + quad * 4 * S::kElt;
                if constexpr (DT == DSKV_F32) *reinterpret_cast<f32x4 *>(dst) = acc * inv;
                else *reinterpret_cast<u32x2 *>(dst) = u32x2{Elt<DT>::pack2(acc.x * inv, acc.y * inv), Elt<DT>::pack2(acc.z * inv, acc.w * inv)};
            }
        }
        __syncthreads();
    };
    start_item(begin);                                          // (its loads in front of those that wait for page ids)
#pragma unroll
    for (int i = 0; i < kDepth; i++) {
        const Ids ids_next = next_ids();
        request(ids, regs[i], held_of[i]);
        ids = ids_next;
    }
    for (;;) {
        settle_item();
        while (st < it.st1) {
#pragma unroll
            for (int i = 0; i < kDepth; i++) subtile(regs[i], held_of[i]);
        }
        finish_item();
        if (it.next >= end) return;
        start_item(it.next);
    }
}

// Items that were cut: a thread per (column, four dims) and group of parts.  kGroups > 1, for items in many parts: each takes
// every kGroups-th part, and they meet in LDS.  kEach > 1, for many columns: columns that a thread takes at once (66
// MB of partials, 16 trees of 33 - 64 rows: 16 us with four, 24 with one).
template <int DT, int kD, int kCols, int kSub, int kGroups, int kEach>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a, int max_col_tiles)
{
    constexpr int kElt = DT == DSKV_F32 ? 4 : 2;
    constexpr int kQuads = kD / 4, kColumns = 256 / (kQuads * kGroups);
    const int b = blockIdx.x / max_col_tiles, ct = blockIdx.x % max_col_tiles, head = blockIdx.y;
    const int quad = threadIdx.x % kQuads, column = threadIdx.x / kQuads % kColumns, group = threadIdx.x / (kQuads * kColumns);
    const TreeRequest r = tree_request<kCols, kSub>(a, b);
    const int before = a.units_before[b], units = a.units_before[a.batch];
    const bool beside = a.units_before[a.batch + 1] != 0;
    const int part_units = a.units_before[a.batch + 2];        // 0: equal shares
    const int cols = min(r.n * a.group - ct * r.tile, r.tile), col0 = (int)blockIdx.z * kColumns * kEach + column;
    if (ct >= r.col_tiles || (int)blockIdx.z * kColumns * kEach >= cols || units == 0) return;
    const int first = before + (beside ? 0 : ct * r.subtiles), last = first + r.subtiles - 1;
    int s0, s1;
    bool second = false;                                       // in the first of its shares the item is the second
    if (part_units > 0) {
        const int parts = (int)((unsigned)(r.subtiles + part_units - 1) / (unsigned)part_units);
        s0 = before + (beside ? 0 : ct * parts);
        s1 = s0 + parts - 1;
    } else {
        const Shares shares = shares_of(units, a.units_before[a.batch + 3]);
        s0 = share_with(shares, first);
        s1 = share_with(shares, last);
        second = share_begin(shares, s0) < first;
    }
    if (s0 == s1) return;
    float top[kEach], sum[kEach];
    f32x4 acc[kEach];
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        top[e] = -INFINITY;
        sum[e] = 0;
        acc[e] = f32x4{0, 0, 0, 0};
    }
    auto add = [&](int e, float pm, float pl, f32x4 po) {
        const float m = fmaxf(top[e], pm), from = m == -INFINITY ? 0.f : m;
        const float w0 = __builtin_amdgcn_exp2f(top[e] - from), w1 = __builtin_amdgcn_exp2f(pm - from);
        top[e] = m;
        sum[e] = sum[e] * w0 + pl * w1;
        acc[e] = acc[e] * w0 + po * w1;
    };
    constexpr int kAhead = kEach > 1 ? 2 : 4;          // parts requested together
    for (int s = s0 + group; s <= s1; s += kAhead * kGroups) {
        float pm[kAhead][kEach], pl[kAhead][kEach];
        f32x4 po[kAhead][kEach];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const int si = min(s + i * kGroups, s1);
            const long slot = 2L * (beside ? share_of_span(si, ct, a.sides) : si) + (si == s0 && second ? 1 : 0);
#pragma unroll
            for (int e = 0; e < kEach; e++) {
                const long part = (slot * a.n_kv_heads + head) * kCols + min(col0 + e * kColumns, cols - 1);
                pm[i][e] = a.part_ml[part * 2];
                pl[i][e] = a.part_ml[part * 2 + 1];
                po[i][e] = *reinterpret_cast<const f32x4 *>(a.part_o + part * kD + quad * 4);
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead; i++)
            if (s + i * kGroups <= s1) {
#pragma unroll
                for (int e = 0; e < kEach; e++) add(e, pm[i][e], pl[i][e], po[i][e]);
            }
    }
    if constexpr (kGroups > 1) {
        static_assert(kEach == 1, "the groups meet over one column a thread");
        __shared__ f32x4 acc_of[kGroups][kColumns * kQuads];
        __shared__ float ml_of[kGroups][kColumns][2];
        acc_of[group][column * kQuads + quad] = acc[0];
        if (quad == 0) {
            ml_of[group][column][0] = top[0];
            ml_of[group][column][1] = sum[0];
        }
        __syncthreads();
        if (group > 0) return;
#pragma unroll
        for (int w = 1; w < kGroups; w++) add(0, ml_of[w][column][0], ml_of[w][column][1], acc_of[w][column * kQuads + quad]);
    }
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        const int col = col0 + e * kColumns;
        if (col >= cols) break;
        const int at = ct * r.tile + col, i = at / a.group, hq = head * a.group + at - i * a.group;
        const float inv = sum[e] == 0 ? 0.f : 1.f / sum[e];
        char *dst = a.out + (((r.first + i) * a.n_qo_heads + hq) * kD + quad * 4) * kElt;
        if constexpr (DT == DSKV_F32) *reinterpret_cast<f32x4 *>(dst) = acc[e] * inv;
        else *reinterpret_cast<u32x2 *>(dst) = u32x2{Elt<DT>::pack2(acc[e].x * inv, acc[e].y * inv), Elt<DT>::pack2(acc[e].z * inv, acc[e].w * inv)};
    }
}

}  // namespace dskv
