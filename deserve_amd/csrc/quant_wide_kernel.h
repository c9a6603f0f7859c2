// The attention over 8-bit pages for more columns than fit a wave (head_dim 64 and 128, 16-bit types): the columns are split over the
// waves of a workgroup, 32 each, and all of them read the same 32-token blocks of K and V from LDS, where these lie in the type of q,
// multiplied by their scales.  See tree_kernel.h for how the work is cut.  A lane fetches 16 or 32 bytes of a stage's codes (one block of
// K or V, or two), some stages ahead, makes numbers of them - two an instruction, which applies the scale; exact in bf16, in f16 but for
// what f16 itself does not hold - and writes them to LDS, so that every code is converted once a workgroup.
//
// Iteration j of a walk multiplies P(j - 1) into V(j - 1), turns S(j) into P(j) and computes S(j + 1), so that all of
// its matrix instructions are independent of its exponentials.  Behind its only barrier the next stages of K and V are written to LDS and those
// kAhead further on requested (see kFirst, kBehind), and at its end the operands of K(j + 2) are read; where a stage holds two blocks, this is once
// in two iterations.  The running maximum of a column is raised only when a block's weights under it
// sum to more than most_weight in a lane.  Weights are rounded to 16 bits for the matrix product, half a step of each (see headroom).
// Bound by the matrix and vector pipelines at the board's power cap: 16 chunks of 512 rows over up to 8 K tokens, 32 heads over 8, 128 dims, bf16, 840 us
// with the merge, 965 TFLOP/s.
// At 128 dims, where all waves fetch, 6 or 7 registers of an item's start (rows of q and out, its place) are in scratch until its end, none of the walk's.
// Where a token lies in the pool, and its scales, are looked up for some thousand tokens at a time and kept in LDS, so that pages may
// have any size.
#pragma once

#include "quant_kernel.h"

namespace dskv {

constexpr int kWideBlock = 32;
constexpr int kWideRegion = 1088;           // 64 chunks of 16 bytes, (4 chunk + row) * 16 of four rows, and 64 bytes of padding
constexpr int kWideStage = kWideBlock / 4 * kWideRegion;
constexpr int kWideLeast = 8;               // units a share has at least: what fills the stages takes about as long

// kFetch: waves without columns that fetch for the others, more stages ahead than there would be registers for beside O and q; 0: all do
// both.  64 requests of 12 rows over 256 - 4096 tokens, 128 dims, two waves of columns and two that fetch: 106 us; 113 in the narrow form with three
// blocks of columns a tile, and one such request over 4000 tokens 20.0 and 40.
template <int kD, int kWaves, int kFetch> struct QuantWide {
    static constexpr int kThreads = kWaves * 64;
    static constexpr int kCompute = kWaves - kFetch, kCols = kCompute * 32;
    static constexpr int kFetchThreads = (kFetch ? kFetch : kWaves) * 64;
    // A stage is what the workgroup's lanes fetch at once, kLane bytes each: one block or two, which lie one after the other in LDS, or, with
    // 64 dims, side by side in rows of 128
    static constexpr int kPack = kD == 128 && kWaves == 4 ? 1 : 2;
    static constexpr int kLane = kPack * kWideBlock * kD / kFetchThreads;
    static constexpr int kLaneRows = 64 * kLane / kD;    // tokens that a wave fetches
    static constexpr int kStageBytes = kD == 128 ? kPack * kWideStage : kWideStage;
    static constexpr int kSteps = kD / 16, kDims = kD / 32;      // matrix instructions of a block's scores; 32-dim tiles of O
    static constexpr int kHalf = kWaves == 8 ? 64 : 32;  // blocks that are looked up at a time; two such halves are kept
    static constexpr int kTokens = 2 * kHalf * kWideBlock, kBeyond = 12;
    static constexpr int kKStages = kPack == 2 ? 2 : 4, kVStages = kPack == 2 ? 4 : 2;      // in LDS
    static constexpr int kAhead = kFetch ? 8 : kD == 128 && kPack == 2 ? 1 : 2;      // stages of K, and of V, on their way in registers
    // what turn u (in front of the iterations of stage u) writes: K(u + kFirst) and V(u + kBehind)
    static constexpr int kFirst = kPack == 2 ? 2 : 3, kBehind = kPack - 1;
};

// An item that begins in a share and ends in another.
struct QuantCut {
    int first, col0, cols, ct;      // row of q that the request begins with; the tile's first column and how many it has
    bool beside;
    QuantParts parts;               // n < 2: none
};

template <int DT, int kD, int kWaves, int kFetch>
__global__ __launch_bounds__(kWaves * 64, 2) void quant_wide_kernel(QuantArgs a)
{
    typedef Elt<DT> E;
    typedef QuantWide<kD, kWaves, kFetch> W;
    __shared__ __align__(16) char lds[(W::kKStages + W::kVStages) * W::kStageBytes];
    // Where a token's K lies (see quant_row), and the exponents of its scales, V's in the second byte; behind the two halves the first
    // kBeyond blocks again, so that what a turn reads lies at fixed distances
    __shared__ u32x2 token_at[W::kTokens + W::kBeyond * kWideBlock];
    __shared__ uint32_t held_at[2 * W::kHalf];           // bit per token of a block: there is one
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
    if (head == 0 && threadIdx.x < 2) a.cuts[2 * share + threadIdx.x].parts.n = 0;

    auto k_stage = [&](int i) { return lds + (i & (W::kKStages - 1)) * W::kStageBytes; };
    auto v_stage = [&](int i) { return lds + (W::kKStages + (i & (W::kVStages - 1))) * W::kStageBytes; };
    // block j in its stage of K or V
    auto block_at = [&](auto &stage, int j) -> char * {
        return W::kPack == 2 ? stage(j >> 1) + (j & 1) * (kD == 128 ? kWideStage : 512) : stage(j);
    };
    // lane p of a wave fetches part p / kLaneRows of token p % kLaneRows of its tokens of a stage
    const bool fetches = kFetch == 0 || wave >= W::kCompute;
    const int my_token = (kFetch == 0 ? wave : fetches ? wave - W::kCompute : 0) * W::kLaneRows + lane % W::kLaneRows;
    const int my_part = lane / W::kLaneRows;
    const char *const pool = a.pages + head * a.head_bytes + my_part * W::kLane;
    const int my_row = my_token % kWideBlock, my_block = my_token / kWideBlock, my_chunk = my_part * (W::kLane / 8);
    const int my_place = kD == 128 ? my_block * kWideStage + my_row / 4 * kWideRegion + (4 * my_chunk + my_row % 4) * 16
                                   : my_row / 4 * kWideRegion + (4 * (my_chunk + 8 * my_block) + my_row % 4) * 16;
    const char *const none = reinterpret_cast<const char *>(kNoRow);
    const char *const scales = a.pages + 2 * a.half_bytes + head * 4;

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
        const int cols = min(r.n * a.group - ct * r.tile, r.tile);
        const int prior = r.prior;
        // (what lies behind the tile's last row is not walked, though it was counted)
        const long last_seen = a.masks ? r.kv_len : min(r.kv_len, (long)prior + (ct * r.tile + cols - 1) / a.group + 1);
        const int t_end = (int)max(min(last_seen, (long)st1 * kWideBlock), 0L);
        const int blocks = max((t_end + kWideBlock - 1) / kWideBlock - st0, 0);
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

        // ---- places in the pool, kHalf blocks at a time: half x of the walk into half x % 2
        auto look_up = [&](int x) {
            for (int i = threadIdx.x; i < W::kHalf * kWideBlock; i += W::kThreads) {
                const int t = (st0 + x * W::kHalf) * kWideBlock + i;
                uint32_t row = kNoQuantRow;
                uint32_t exponents = 0;
                if (t < t_end) {
                    const int page = page_of(a, r, t);
                    row = quant_row(a, t, page);
                    if (row == kNoQuantRow) holes = 1;
                    else {
                        const uint32_t *s = reinterpret_cast<const uint32_t *>(scales + page * a.page_bytes);
                        exponents = (s[0] >> 23 & 0xFF) | (s[a.n_kv_heads] >> 15 & 0xFF00);
                    }
                }
                const int at = (x & 1) * W::kHalf * kWideBlock + i;
                token_at[at] = u32x2{row, exponents};
                if (at < W::kBeyond * kWideBlock) token_at[W::kTokens + at] = u32x2{row, exponents};
                const unsigned long long there64 = __ballot(row != kNoQuantRow);
                if ((lane & 31) == 0) held_at[at / kWideBlock] = (uint32_t)(there64 >> (lane & 32));
            }
        };
        // what the tables say of the token that the lane fetches of stage u + more
        const u32x2 *const mine_at = token_at + my_token;
        auto token_of = [&](int u, int more) -> const u32x2 & {
            return mine_at[((u * W::kPack & (2 * W::kHalf - 1)) + more * W::kPack) * kWideBlock];
        };
        typedef uint32_t Codes __attribute__((ext_vector_type(W::kLane / 4)));
        Codes k_codes[W::kAhead], v_codes[W::kAhead];
        auto request = [&](uint32_t row, Codes &codes, long more) {
            const char *p = pool + (uint64_t)row * 16 + more;
            p = row != kNoQuantRow ? p : none;
            codes = *(const __attribute__((address_space(1))) Codes *)p;
        };
        auto write = [&](const Codes &codes, uint32_t exponent, char *stage) {
            const float scale = __builtin_bit_cast(float, exponent << 23);
#pragma unroll
            for (int c = 0; c < W::kLane / 8; c++) {
                u32x4 x;
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    const uint32_t four = codes[2 * c + w];
                    if constexpr (DT == DSKV_F16) {
                        x[2 * w] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(four, scale, false));
                        x[2 * w + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(four, scale, true));
                    } else {
                        x[2 * w] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, scale, false));
                        x[2 * w + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, scale, true));
                    }
                }
                *reinterpret_cast<u32x4 *>(stage + my_place + c * 64) = x;
            }
        };
        // what turn u needs of the tables: exponents of what it writes, places of what it requests
        struct Known {
            uint32_t k_exponent, v_exponent, k_row, v_row;
        };
        auto know = [&](int u, Known &x) {
            x.k_exponent = *(reinterpret_cast<const uint8_t *>(&token_of(u, W::kFirst)) + 4);
            x.v_exponent = *(reinterpret_cast<const uint8_t *>(&token_of(u, W::kBehind)) + 5);
            x.k_row = token_of(u, W::kFirst + W::kAhead).x;
            x.v_row = token_of(u, W::kBehind + W::kAhead).x;
        };
        static_assert((W::kFirst + W::kAhead + 1) * W::kPack <= W::kBeyond, "a turn reads behind what is there twice");

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
        auto seen = [&](int j) {
            return j < blocks ? seen_bits((st0 + j) * kWideBlock, prior, limit, mask, !a.masks) & held_at[j & (2 * W::kHalf - 1)] : 0u;
        };
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
        // ---- the walk
        __syncthreads();                                 // the item before is through with LDS
        if (threadIdx.x == 0) holes = 0;
        __syncthreads();
        look_up(0);
        for (int i = threadIdx.x; i < W::kStageBytes / 16; i += W::kThreads)
            reinterpret_cast<u32x4 *>(v_stage(-1))[i] = u32x4{0, 0, 0, 0};     // V(-1), which P(-1) = 0 is multiplied by
        __syncthreads();
        if (holes) mask_from = 0;
        // q and the mask are waited for here: left to the loop, that would be a wait for its loads
#pragma unroll
        for (int s = 0; s < W::kSteps; s++) asm volatile("" : "+v"(q[s]));
        asm volatile("" : "+v"(mask));
        Known known;
        auto fill = [&]() {                              // as if there were turns in front
#pragma unroll
            for (int u = 0; u < W::kAhead; u++) {
                const uint32_t row = token_of(0, u).x;
                request(row, k_codes[u], 0);
                request(row, v_codes[u], a.half_bytes);
            }
#pragma unroll
            for (int u = 0; u < W::kFirst; u++) {
                write(k_codes[u % W::kAhead], token_of(0, u).y & 0xFF, k_stage(u));
                request(token_of(0, u + W::kAhead).x, k_codes[u % W::kAhead], 0);
            }
#pragma unroll
            for (int u = 0; u < W::kBehind; u++) {
                write(v_codes[u], token_of(0, u).y >> 8, v_stage(u));
                request(token_of(0, u + W::kAhead).x, v_codes[u], a.half_bytes);
            }
            know(0, known);
        };
        // phase: u up to a multiple of kAhead, a literal
        auto turn = [&](int u, int phase) {
            constexpr int kMask = W::kAhead - 1;
            const int k_at = (phase + W::kFirst) & kMask, v_at = (phase + W::kBehind) & kMask;
            write(k_codes[k_at], known.k_exponent, k_stage(u + W::kFirst));
            write(v_codes[v_at], known.v_exponent, v_stage(u + W::kBehind));
            request(known.k_row, k_codes[k_at], 0);
            request(known.v_row, v_codes[v_at], a.half_bytes);
            know(u + 1, known);
        };
        auto meet = [&](int phase) {
            const bool turns = W::kPack == 1 || (phase & 1) == 0;
            if (turns) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            }
            return turns;
        };
        auto iteration = [&](int j, int phase) {
            const bool turns = meet(phase);
            const int cur = phase & 1, nxt = cur ^ 1;
            const char *rows = block_at(v_stage, j - 1) + v_off;                        // V(j - 1)
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
            if (kFetch == 0 && turns) turn(j / W::kPack, phase / W::kPack);
            float sum = 0;
            weights(xs[cur], 0, pb[cur][0], sum);
            if ((st0 + j + 2) * kWideBlock > mask_from) mask_scores(j + 1, xs[nxt]);
#pragma unroll
            for (int d = 0; d < W::kDims; d++)
#pragma unroll
                for (int s = 0; s < 2; s++) acc[d] = E::mfma_32x32(va[d][s], pb[nxt][s], acc[d]);   // P(j - 1)
            read_keys(block_at(k_stage, j + 2));                                         // K(j + 2)
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
        auto look_ahead = [&](int j) {                   // (the turns look up to 12 blocks behind the last one, too)
            if (j % W::kHalf == W::kHalf / 2 && j + W::kHalf / 2 < blocks + 16) look_up(j / W::kHalf + 1);
        };
        if constexpr (kFetch == 0) fill();
        if (kFetch == 0 || !fetches) __syncthreads();
        if (works) {
            read_keys(block_at(k_stage, 0));
            scores(xs[0]);
            if ((st0 + 1) * kWideBlock > mask_from) mask_scores(0, xs[0]);
            read_keys(block_at(k_stage, 1));
            for (int j = 0;; j += 4) {
                look_ahead(j);
                iteration(j, 0);
                if (holes) mask_from = 0;
                if (j >= blocks) break;
                iteration(j + 1, 1);
                if (j + 1 >= blocks) break;
                iteration(j + 2, 2);
                if (j + 2 >= blocks) break;
                iteration(j + 3, 3);
                if (j + 3 >= blocks) break;
            }
        } else if (fetches) {
            // a wave without columns only fetches
            if constexpr (kFetch != 0) {
                fill();
                __syncthreads();
            }
            auto passes = [&](int j, int phase) {
                if (meet(phase)) turn(j / W::kPack, phase / W::kPack);
                return j >= blocks;
            };
            for (int j = 0;; j += kFetch ? 8 : 4) {
                look_ahead(j);
                if (passes(j, 0) || passes(j + 1, 1) || passes(j + 2, 2) || passes(j + 3, 3)) break;
                if constexpr (kFetch != 0) {
                    look_ahead(j + 4);
                    if (passes(j + 4, 4) || passes(j + 5, 5) || passes(j + 6, 6) || passes(j + 7, 7)) break;
                }
            }
        } else {
            // a wave that would have columns, of a tile that has fewer
            for (int j = 0; j <= blocks; j++) {
                look_ahead(j);
                meet(0);
            }
        }

        // ---- the item's result
        float l_other = l_run;
        swap_halves32(l_run, l_other);
        const float l = l_run + l_other;
        const bool cut = st0 > 0 || st1 < r.subtiles;
        if (there && cut) {
            const long part = ((2L * share + (unit > begin ? 1 : 0)) * a.n_kv_heads + head) * W::kCols + wave * 32 + r32;
#pragma unroll
            for (int d = 0; d < W::kDims; d++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    *reinterpret_cast<f32x4 *>(a.part_o + part * kD + d * 32 + 8 * i + 4 * h) =
                        f32x4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
            if (h == 0) *reinterpret_cast<f32x2 *>(a.part_ml + part * 2) = f32x2{m_run, l};
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
        // an item that goes on in another share is the merge launch's
        if (cut && st0 == 0 && head == 0 && threadIdx.x == 0)
            a.cuts[2 * share + (unit > begin ? 1 : 0)] = {(int)r.first, ct * r.tile, cols, ct, beside, parts_of(a, place, item, r.subtiles, ct)};
        unit = item + st1;
    }
}

// Items that were cut, two for each share that they begin in: a thread per four dims of kEach columns and kAhead parts requested together, workgroups along the columns (in
// front, so that those of few items lie on all XCDs: 437 rows in 7 tiles 9.2 us, 16.3 with the items in front).  A chain of three trips and as
// many more as there are pairs of parts.
template <int DT, int kD, int kCols, int kEach, int kAhead>
__global__ __launch_bounds__(256) void quant_merge_kernel(QuantArgs a)
{
    constexpr int kQuads = kD / 4, kColumns = 256 / kQuads;           // columns side by side
    const QuantCut cut = a.cuts[blockIdx.z];
    if (cut.parts.n < 2) return;
    const int head = blockIdx.y, quad = threadIdx.x % kQuads, column = threadIdx.x / kQuads;
    const int cols = cut.cols, col0 = (int)blockIdx.x * kColumns * kEach + column;
    if ((int)blockIdx.x * kColumns * kEach >= cols) return;
    TreePlace place;
    place.beside = cut.beside;
    float top[kEach], sum[kEach];
    f32x4 acc[kEach];
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        top[e] = -INFINITY;
        sum[e] = 0;
        acc[e] = f32x4{0, 0, 0, 0};
    }
    for (int i0 = 0; i0 < cut.parts.n; i0 += kAhead) {
        f32x4 o[kAhead][kEach];
        f32x2 ml[kAhead][kEach];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
#pragma unroll
            for (int e = 0; e < kEach; e++) {
                ml[i][e] = f32x2{-INFINITY, 0};
                o[i][e] = f32x4{0, 0, 0, 0};
            }
            if (i0 + i >= cut.parts.n) continue;
            const long slot = part_slot(a, place, cut.parts, cut.ct, i0 + i);
#pragma unroll
            for (int e = 0; e < kEach; e++) {
                const long part = (slot * a.n_kv_heads + head) * kCols + min(col0 + e * kColumns, cols - 1);
                ml[i][e] = *reinterpret_cast<const f32x2 *>(a.part_ml + part * 2);
                o[i][e] = *reinterpret_cast<const f32x4 *>(a.part_o + part * kD + quad * 4);
            }
        }
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            float m = top[e];
#pragma unroll
            for (int i = 0; i < kAhead; i++) m = fmaxf(m, ml[i][e].x);
            const float keep = __builtin_amdgcn_exp2f(top[e] - m);
            top[e] = m;
            sum[e] *= keep;
            acc[e] *= keep;
#pragma unroll
            for (int i = 0; i < kAhead; i++)
                if (i0 + i < cut.parts.n) {
                    const float w = __builtin_amdgcn_exp2f(ml[i][e].x - m);
                    sum[e] += ml[i][e].y * w;
                    acc[e] += o[i][e] * w;
                }
        }
    }
#pragma unroll
    for (int e = 0; e < kEach; e++)
        if (col0 + e * kColumns < cols) put_result<DT, kD>(a, cut.first, head, cut.col0 + col0 + e * kColumns, quad * 4, acc[e], sum[e]);
}

}  // namespace dskv
