// The tree attention for more columns than fit a wave (head_dim 64 and 128, 16 bits): the columns are split over the waves of
// a workgroup, 32 each, and all of them read the same 32-token blocks of K and V from LDS, which go there straight from
// memory.  See tree_kernel.h for how the work is cut.  sm_scale is positive: a masked score is -infinity before it is
// scaled.
//
// Bound by the matrix pipeline and the vector instructions beside it: 16 of 32x32x16 per block and wave, 16 exponentials and some 75
// other instructions (128 dims).  16 requests over 1 - 16 K tokens, 64 heads over 8, bf16, when the board's power has settled: with 64 rows
// each, over 160 K tokens in all, 370 us, 905 TFLOP/s; with 33 to 64 rows over 136 K 281 - 296, 750 - 790 TFLOP/s, since a block lasts as
// long as its units with two busy waves, and columns come in thirty-twos; of that 15 us are the launch for cut items (66 MB of
// partials).  The first thirty calls behind a pause take 330 - 340.
// With 64 dims a stage holds two blocks side by side, so that a load fetches whole kilobytes there, too, and both sizes share one
// layout of LDS: 16 requests of 48 rows, 64 heads, over 160 K tokens in all 205 us, 610 TFLOP/s (the narrow form: 396): half the
// products of 128 dims for the same exponentials.
// Measured and left out: priority for the matrix instructions (2 % slower), exponentials free to move through the iteration (3 %).
//
// Iteration j of a walk multiplies P(j - 1) into V(j - 1), turns S(j) into P(j) and computes S(j + 1), so that all of
// its matrix instructions are independent of its exponentials.  Blocks lie in kStages stages of K and of V; iteration j
// requests K(j + kStages) and V(j + kStages - 2) behind its only barrier, and reads the operands of K(j + 2) at its end; with eight
// stages there is room for two iterations to a barrier (48 rows as above 324 us, with one 327), V one block later.  The running maximum
// of a column is raised only when a block's weights under it sum to more than most_weight in a lane.  Weights are rounded to 16
// bits for the matrix product, half a step of each (see headroom); sums, maxima and O stay in 32.
// Where a token lies in the pool is looked up for some thousand tokens at a time and kept in LDS (row numbers, a bit per token that
// there is), so that pages may have any size and the loop's loads wait for nothing but LDS.
#pragma once

#include "tree_kernel.h"

namespace dskv {

constexpr int kWideBlock = 32;
constexpr int kWideRegion = 1088;           // 1 KB that a wave's load fetches, (4 chunk + row) * 16 of four rows, and 64 bytes of padding
constexpr int kWideStage = kWideBlock / 4 * kWideRegion;
constexpr int kWideLeast = 8;               // units a share has at least: what fills the stages takes about as long
constexpr int kBadBlocks = kTreeMostRows / kWideBlock + 2;       // that new rows reach into

template <int kD, int kWaves> struct WideShape {
    static constexpr int kThreads = kWaves * 64;
    static constexpr int kCols = kWaves * 32;
    static constexpr int kPack = 128 / kD;               // blocks of a stage: rows of 128 bytes lie side by side with the next block's
    static constexpr int kChunks = kD / 8;               // 16-byte chunks of a row
    static constexpr int kSteps = kD / 16, kDims = kD / 32;      // matrix instructions of a block's scores; 32-dim tiles of O
    static constexpr int kGroups = 8 / kWaves;           // regions of a stage that a wave requests
    static constexpr int kHalf = kWaves == 8 ? 64 : 32;  // blocks that are looked up at a time; two such halves are kept
    static constexpr int kTokens = 2 * kHalf * kWideBlock;
    static constexpr int kPair = kWaves == 8 || kPack == 2 ? 2 : 1;      // iterations between barriers
    static constexpr int kAsked = kPair / kPack;         // stages of K, and of V, that are requested there
    static constexpr int kStages = kWaves == 8 && kPack == 1 ? 8 : 4;    // of K, and of V, in LDS: as many as fit beside the other workgroup
    // a wave's loads that may be on their way behind a barrier's wait: all but those of K(j + 2) .., V(j - 1) ..
    static constexpr int kInFlight = (2 * kStages - 2 - 3 * kAsked - (kPack - 1)) * kGroups;
};

template <int DT, int kD, int kWaves>
__global__ __launch_bounds__(kWaves * 64, 2) void tree_wide_kernel(TreeArgs a)
{
    typedef Elt<DT> E;
    typedef WideShape<kD, kWaves> W;
    __shared__ __align__(16) char lds[2 * W::kStages * kWideStage];
    __shared__ int32_t row_at[W::kTokens];               // row of the pool (page * 2 P + place), -1: none
    __shared__ uint32_t held_at[2 * W::kHalf];           // bit per token of a block: there is one
    __shared__ uint32_t bad_at[kBadBlocks];              // bit per token of a block with new rows: its V is no number
    __shared__ int holes;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, c = lane & 15, h = lane >> 5, r32 = lane & 31;
    int share, head;
    share_and_head(a, share, head);
    TreePlace place;
    tree_place<W::kCols, kWideBlock, W::kThreads, true, kWideLeast, kWideLeast>(a, share, place);
    make_uniform(place);
    const int begin = place.begin, end = place.end;
    const bool beside = place.beside;
    int unit = begin, base = place.base;
    int b = place.b;
    TreeRequest r = place.r;

    auto k_stage = [&](int i) { return lds + i * kWideStage; };
    auto v_stage = [&](int i) { return lds + (W::kStages + i) * kWideStage; };
    constexpr int kLast = W::kStages - 1;
    // block j + n - j % 4 (of the walk, n a literal) in its stage of K or V
    auto block_at = [&](auto &stage, int j, int n) -> char * {
        if (W::kPack == 2) return stage((((j >> 2) << 1) + (n >> 1)) & kLast) + (n & 1) * 512;
        return stage((n + (W::kStages == 8 ? j & 4 : 0)) & kLast);
    };
    const int row_bytes = a.n_kv_heads * kD * 2;
    const long half_bytes = (long)a.page_size * row_bytes;
    // lane p of a load fetches chunk p / 4 of row p % 4 of a region
    const char *const pool = a.pages + head * kD * 2 + (lane >> 2) % W::kChunks * 16;
    const char *const none = reinterpret_cast<const char *>(kNoRow) + (lane >> 2) % W::kChunks * 16;

    while (unit < end) {
        if (unit >= base + (int)units_of(r, beside)) {             // on to the next request that has rows
            base += (int)units_of(r, beside);
            b++;
            r = tree_request<W::kCols, kWideBlock>(a, b);
            continue;
        }
        const int ct = beside ? place.side : (int)((unsigned)(unit - base) / (unsigned)r.subtiles);
        const int item = base + (beside ? 0 : ct * r.subtiles);
        const int st0 = unit - item, st1 = min(end - item, r.subtiles);
        if (ct >= r.col_tiles) {                              // (beside: a request of fewer column tiles)
            unit = item + st1;
            continue;
        }
        const int blocks = st1 - st0;
        const int cols = min(r.n * a.group - ct * r.tile, r.tile);
        const int prior = r.prior;
        const int t_end = (int)min(r.kv_len, (long)st1 * kWideBlock);
        const bool works = wave * 32 < cols;

        // ---- the column
        const int col = ct * r.tile + wave * 32 + r32, row_i = col / a.group;
        const bool there = wave * 32 + r32 < cols;
        const long q_row = r.first + (there ? row_i : 0);
        const int hq = head * a.group + (there ? col - row_i * a.group : 0);
        unsigned long long mask = ~0ull;
        int limit = 0;                                  // tokens from here on are not seen
        if (there) {
            if (a.masks) mask = (unsigned long long)a.masks[q_row];
            const long lim = a.masks ? (long)prior + DSKV_MAX_TREE_ROWS : (long)prior + row_i + 1;
            limit = (int)max(min(lim, (long)t_end), 0L);
        }
        u32x4 q[W::kSteps];
        {
            const char *row = a.q + q_row * a.q_stride + hq * kD * 2 + h * 16;
#pragma unroll
            for (int s = 0; s < W::kSteps; s++) {
                q[s] = u32x4{0, 0, 0, 0};
                if (there) q[s] = *reinterpret_cast<const u32x4 *>(row + s * 32);
            }
        }
        // blocks that reach behind here need their scores masked
        const int first_i = (ct * r.tile + wave * 32) / a.group;
        int mask_from = min(a.masks ? prior : prior + first_i + 1, t_end);

        f32x16 acc[W::kDims], xs[2];
        float m_run = -__FLT_MAX__, l_run = 0;
        u32x4 pb[2][2];
#pragma unroll
        for (int d = 0; d < W::kDims; d++)
#pragma unroll
            for (int v = 0; v < 16; v++) acc[d][v] = 0;
        pb[1][0] = pb[1][1] = u32x4{0, 0, 0, 0};

        // ---- rows of the pool, kHalf blocks at a time: half x of the walk into half x % 2
        auto look_up = [&](int x) {
            for (int i = threadIdx.x; i < W::kHalf * kWideBlock; i += W::kThreads) {
                const int t = (st0 + x * W::kHalf) * kWideBlock + i;
                int row = -1;
                if (t < t_end) {
                    row = pool_row(a, t, page_of(a, r, t));
                    if (row < 0) holes = 1;
                }
                const int at = (x & 1) * W::kHalf * kWideBlock + i;
                row_at[at] = row;
                const unsigned long long there64 = __ballot(row >= 0);
                if ((lane & 31) == 0) held_at[at / kWideBlock] = (uint32_t)(there64 >> (lane & 32));
            }
        };
        // rows of the pool that the lane requests 16 bytes of for stage u of the walk
        struct Where {
            int row[W::kGroups];
        };
        auto where = [&](int u, Where &w) {
            const int j = W::kPack == 2 ? 2 * u + (lane >> 5) : u;
#pragma unroll
            for (int i = 0; i < W::kGroups; i++) {
                const int at = (j & (2 * W::kHalf - 1)) * kWideBlock + (wave * W::kGroups + i) * 4 + (lane & 3);
                w.row[i] = j < blocks ? row_at[at] : -1;           // (behind the walk nothing was looked up)
            }
        };
        typedef __attribute__((address_space(3))) void *lds_ptr;
        // Written out as instructions: through the compiler's builtin every later LDS read waits for all of these loads.  What it does
        // not know it does not wait for: the waits are the explicit ones below.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
        auto request = [&](const Where &w, char *stage, long more) {
#pragma unroll
            for (int i = 0; i < W::kGroups; i++) {
                const uint32_t to = (uint32_t)(uintptr_t)(lds_ptr)(stage + (wave * W::kGroups + i) * kWideRegion);
                const char *p = pool + (unsigned long)(unsigned)w.row[i] * (unsigned)row_bytes + more;
                p = w.row[i] >= 0 ? p : none;
                asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off"
                             :
                             : "s"(__builtin_amdgcn_readfirstlane(to)), "v"(p)
                             : "memory", "m0");
            }
        };
#pragma clang diagnostic pop
        // until at most n of the wave's vector-memory operations are on their way
#define DSKV_WAIT_VMEM(n) __builtin_amdgcn_s_waitcnt(((n) & 15) | 0x70 | 0xF00 | (((n) >> 4) << 14))

        // ---- parts of an iteration
        u32x4 key[W::kSteps];                                    // K operand: token r32, dims 16 s + 8 h ..
        auto read_keys = [&](const char *stage) {
            // token r32 = row r32 & 3 of region r32 >> 2; chunk 2 s + h
            const char *rows = stage + (r32 >> 2) * kWideRegion + h * 64 + (r32 & 3) * 16;
#pragma unroll
            for (int s = 0; s < W::kSteps; s++) key[s] = *reinterpret_cast<const u32x4 *>(rows + s * 128);
        };
        auto scores = [&](f32x16 &x) {
#pragma unroll
            for (int v = 0; v < 16; v++) x[v] = 0;
#pragma unroll
            for (int s = 0; s < W::kSteps; s++) x = E::mfma_32x32(key[s], q[s], x);
        };
        // bits of block j's tokens that the column sees
        auto seen_of = [&](int j) { return seen_bits((st0 + j) * kWideBlock, prior, limit, mask, !a.masks); };
        auto seen = [&](int j) { return j < blocks ? seen_of(j) & held_at[j & (2 * W::kHalf - 1)] : 0u; };
        auto mask_scores = [&](int j, f32x16 &x) {
            asm volatile("" : "+v"(x));                 // keeps this a branch that most blocks do not take
            uint32_t bits = seen(j) >> (4 * h);
            asm volatile("" : "+v"(bits));
#pragma unroll
            for (int v = 0; v < 16; v++)
                if (!((bits >> (8 * (v >> 2) + (v & 3))) & 1)) x[v] = -INFINITY;
        };
        auto weights = [&](const f32x16 &x, int s, u32x4 &out, float &sum) {
            float p[8];
#pragma unroll
            for (int v = 0; v < 8; v++) {
                p[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * s + v], a.scale, -m_run));
                sum += p[v];
            }
            out = u32x4{E::pack2(p[0], p[1]), E::pack2(p[2], p[3]), E::pack2(p[4], p[5]), E::pack2(p[6], p[7])};
            asm volatile("" ::"v"(out), "v"(sum));      // keeps them in their half of the iteration
        };
        auto raise = [&](const f32x16 &x) {
            float m = x[0] * a.scale;
#pragma unroll
            for (int v = 1; v < 16; v++) m = fmaxf(m, x[v] * a.scale);
            float other = m;
            swap_halves32(m, other);
            const float m_new = fmaxf(m_run, fmaxf(m, other) - headroom(DT));
            const float keep = __builtin_amdgcn_exp2f(m_run - m_new);
            m_run = m_new;
            l_run *= keep;
#pragma unroll
            for (int d = 0; d < W::kDims; d++) acc[d] *= keep;
        };
        const int v_off = h * kWideRegion + (2 * (g & 1) + ((c & 3) >> 1)) * 64 + (c >> 2) * 16 + (c & 1) * 8;
        // A weight of 0 times a V that is no number would reach columns that do not see the token: such tokens among the new
        // ones are taken out of the block here, by the wave that requested them, and added behind the walk.
        const int new_from = max((max(prior, 0) >> 5) - st0, 0), new_to = min(((int)r.kv_len + 31) / 32 - st0, blocks);
        auto set_aside = [&](int u) {                    // of stage u
            const int j = W::kPack == 2 ? 2 * u + (lane >> 5) : u;
            const bool is_new = j >= new_from && j < new_to;
#pragma unroll
            for (int i = 0; i < W::kGroups; i++) {
                const int region = wave * W::kGroups + i;
                u32x4 *at = reinterpret_cast<u32x4 *>(v_stage(u & kLast) + region * kWideRegion + lane * 16);
                const bool odd = is_new && no_number<DT>(*at);
                const unsigned long long lanes = __ballot(odd);
                if (__builtin_expect(lanes != 0, 0)) {
                    const unsigned long long of_block = W::kPack == 1 ? lanes : lane < 32 ? lanes & 0xffffffff : lanes >> 32 << 32;
                    uint32_t rows = 0;
#pragma unroll
                    for (int row = 0; row < 4; row++)
                        if (of_block & (0x1111111111111111ull << row)) rows |= 1u << row;
                    if ((rows >> (lane & 3)) & 1) *at = u32x4{0, 0, 0, 0};
                    if (rows != 0 && (W::kPack == 1 ? lane : lane & 31) == 0) atomicOr(&bad_at[j - new_from], rows << (4 * region));
                }
            }
        };
        // ---- the walk
        __syncthreads();                                 // the item before is through with LDS
        if (threadIdx.x == 0) holes = 0;
        for (int i = threadIdx.x; i < kBadBlocks; i += W::kThreads) bad_at[i] = 0;
        __syncthreads();
        look_up(0);
        for (int i = threadIdx.x; i < kWideStage / 16; i += W::kThreads)
            reinterpret_cast<u32x4 *>(v_stage(kLast))[i] = u32x4{0, 0, 0, 0};          // V(-1), which P(-1) = 0 is multiplied by
        __syncthreads();
        if (holes) mask_from = 0;
        // q and the mask are waited for here: left to the loop, that would be a wait for all of its loads
#pragma unroll
        for (int s = 0; s < W::kSteps; s++) asm volatile("" : "+v"(q[s]));
        asm volatile("" : "+v"(mask));
        Where at_v[W::kAsked], at_between, at_k[W::kAsked];     // of the stages that the next requests are for
        {
            // as if there were iterations in front
            Where w[W::kStages];
#pragma unroll
            for (int i = 0; i < W::kStages; i++) where(i, w[i]);
#pragma unroll
            for (int i = 0; i < W::kStages; i += W::kAsked) {
#pragma unroll
                for (int x = i; x < i + W::kAsked; x++) request(w[x], k_stage(x), 0);
#pragma unroll
                for (int x = max(i - W::kAsked - 1, 0); x < i - 1; x++) request(w[x], v_stage(x), half_bytes);
            }
#pragma unroll
            for (int x = 0; x < W::kAsked; x++) {
                at_v[x] = w[W::kStages - 1 - W::kAsked + x];
                where(W::kStages + x, at_k[x]);
            }
            at_between = w[W::kStages - 1];
            DSKV_WAIT_VMEM((2 * W::kStages - 3 - W::kAsked) * W::kGroups);              // the first two stages of K
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (works) {
            read_keys(block_at(k_stage, 0, 0));
            scores(xs[0]);
            if ((st0 + 1) * kWideBlock > mask_from) mask_scores(0, xs[0]);
            read_keys(block_at(k_stage, 0, 1));
        }
        // in front of iterations j .. j + kPair - 1; phase = j % 4, a literal
        auto advance = [&](int j, int phase) {
            const int u = j / W::kPack;                  // the stage that block j is in
            // this wave's rows of K(j + 2), V(j - 1) and, for a pair, K(j + 3) and V(j) have landed
            DSKV_WAIT_VMEM(W::kInFlight);
            asm volatile("" ::: "memory");
            if (W::kPack == 2) {
                if (j + 1 >= new_from && j < new_to) set_aside(u);
            } else {
#pragma unroll
                for (int x = u - 1; x < u - 1 + W::kPair; x++)
                    if (x >= new_from && x < new_to) set_aside(x);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
#pragma unroll
            for (int x = 0; x < W::kAsked; x++) request(at_k[x], block_at(k_stage, j, phase + x), 0);          // stage u + kStages + x of K
#pragma unroll
            for (int x = 0; x < W::kAsked; x++)                                  // and u + kStages - 1 - kAsked + x of V
                request(at_v[x], W::kPack == 2 ? v_stage((u + 2) & kLast) : block_at(v_stage, j, phase + kLast - W::kAsked + x), half_bytes);
            at_v[0] = at_between;
            if (W::kAsked == 2) at_v[W::kAsked - 1] = at_k[0];
            at_between = at_k[W::kAsked - 1];
#pragma unroll
            for (int x = 0; x < W::kAsked; x++) where(u + W::kStages + W::kAsked + x, at_k[x]);
        };
        auto iteration = [&](int j, int phase) {
            if (W::kPair == 1 || (phase & 1) == 0) advance(j, phase);
            if (!works || j > blocks) return;
            const int cur = phase & 1, nxt = cur ^ 1;
            const char *rows = block_at(v_stage, j, phase - 1) + v_off;                        // V(j - 1)
            u32x4 va[W::kDims][2];
#pragma unroll
            for (int d = 0; d < W::kDims; d++)
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    const char *p = rows + s * 4 * kWideRegion + d * 256;
                    const u32x2 lo = read_transposed(p), hi = read_transposed(p + 2 * kWideRegion);
                    va[d][s] = u32x4{lo.x, lo.y, hi.x, hi.y};
                }
            scores(xs[nxt]);                                                        // S(j + 1)
            float sum = 0;
            weights(xs[cur], 0, pb[cur][0], sum);
            if ((st0 + j + 2) * kWideBlock > mask_from) mask_scores(j + 1, xs[nxt]);
#pragma unroll
            for (int d = 0; d < W::kDims; d++)
#pragma unroll
                for (int s = 0; s < 2; s++) acc[d] = E::mfma_32x32(va[d][s], pb[nxt][s], acc[d]);   // P(j - 1)
            read_keys(block_at(k_stage, j, phase + 2));                                  // K(j + 2)
            weights(xs[cur], 1, pb[cur][1], sum);
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(sum > most_weight(DT)) != 0, 0)) {
                raise(xs[cur]);
                __builtin_amdgcn_sched_barrier(0);
                sum = 0;
                weights(xs[cur], 0, pb[cur][0], sum);
                weights(xs[cur], 1, pb[cur][1], sum);
            }
            l_run += sum;
        };
        for (int j = 0; j <= blocks; j += 4) {
            if (j % W::kHalf == W::kHalf / 2 && j + W::kHalf / 2 < blocks) look_up(j / W::kHalf + 1);
            iteration(j, 0);
            if (holes) mask_from = 0;
            iteration(j + 1, 1);
            iteration(j + 2, 2);
            iteration(j + 3, 3);
        }
        DSKV_WAIT_VMEM(0);                               // nothing of this wave is still on its way into LDS

        // ---- tokens that were taken out, for the columns that see them
        for (int j = new_from; j < new_to; j++) {
            uint32_t bad = bad_at[j - new_from];
            if (__builtin_expect(bad == 0, 1)) continue;
            const uint32_t bits = seen_of(j);
            while (bad) {
                const int token = __builtin_ctz(bad);
                bad &= bad - 1;
                const int t = (st0 + j) * kWideBlock + token;
                const int row = pool_row(a, t, page_of(a, r, t));
                if (row < 0) continue;
                const char *key = a.pages + (unsigned long)(unsigned)row * (unsigned)row_bytes + head * kD * 2;
                float s = 0;
                for (int k = 0; k < W::kSteps; k++) {
                    float x[8], y[8];
                    Chunk<DT>::unpack(*reinterpret_cast<const u32x4 *>(key + k * 32 + h * 16), x);
                    u32x4 mine = q[0];
#pragma unroll
                    for (int i = 1; i < W::kSteps; i++) mine = k == i ? q[i] : mine;
                    Chunk<DT>::unpack(mine, y);
#pragma unroll
                    for (int e = 0; e < 8; e++) s = fmaf(x[e], y[e], s);
                }
                float other = s;
                swap_halves32(s, other);
                const float weight = __builtin_amdgcn_exp2f(fmaf(s + other, a.scale, -m_run));
                if ((bits >> token) & 1)
#pragma unroll
                    for (int d = 0; d < W::kDims; d++)
#pragma unroll
                        for (int v = 0; v < 16; v++)
                            acc[d][v] += weight * LoadElt<DT>::get(key + half_bytes, d * 32 + 8 * (v >> 2) + 4 * h + (v & 3));
            }
        }

        // ---- the item's result
        float l_other = l_run;
        swap_halves32(l_run, l_other);
        const float l = l_run + l_other;
        const bool cut = st0 > 0 || st1 < r.subtiles;
        if (there && cut) {
            const long slot = 2L * share + (unit > begin ? 1 : 0);
            const long part = (slot * a.n_kv_heads + head) * W::kCols + wave * 32 + r32;
#pragma unroll
            for (int d = 0; d < W::kDims; d++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    *reinterpret_cast<f32x4 *>(a.part_o + part * kD + d * 32 + 8 * i + 4 * h) =
                        f32x4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
            if (h == 0) {
                a.part_ml[part * 2] = m_run;
                a.part_ml[part * 2 + 1] = l;
            }
        } else if (there) {
            const float inv = l == 0 ? 0.f : 1.f / l;
            char *dst = a.out + ((q_row * a.n_qo_heads + hq) * kD + 4 * h) * 2;
#pragma unroll
            for (int d = 0; d < W::kDims; d++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    *reinterpret_cast<u32x2 *>(dst + (d * 32 + 8 * i) * 2) =
                        u32x2{E::pack2(acc[d][4 * i] * inv, acc[d][4 * i + 1] * inv),
                              E::pack2(acc[d][4 * i + 2] * inv, acc[d][4 * i + 3] * inv)};
        }
        unit = item + st1;
    }
}
#undef DSKV_WAIT_VMEM

}  // namespace dskv
