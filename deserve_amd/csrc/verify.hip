// Verification of drafted tokens against the target's probabilities.
//
// The walk from a request's row 0 down needs single probabilities only: row i's token at its parent's row, p_i, and
// with the draft's distributions q_i.  All are gathered at once, a lane per row, and the walk itself is scalar: the
// children of the row reached are a ballot.  Then one row of the vocabulary is left, the weights w of the token behind the
// walk (see dskv_verify_drafts): first its sum, then the first index whose cumulated weight passes uniform * sum.
// Sums and comparisons are in 64 bits: an index is drawn among 1e5 weights of 1e-5, which sums in 32 bits would
// move by whole tokens, and a product of two 32-bit numbers is exact in 64.
//
// Bound by reading that row (of p, and of q) where there are requests enough, by the chain of two launches otherwise: 64 chains
// over a vocabulary of 128000 in fp32 (65 MB) 14.6 and 4.5 us, one tree of 40 rows 5.3 and 4.4.
// Two launches: in the first every workgroup takes the walk for itself (a few hundred bytes from L2) and sums a part of kPart
// weights; a request's first workgroup writes the walk down.  The second finds the part by the parts' sums and the token in it.
#include "common.h"

namespace dskv {

constexpr int kVerifyThreads = 256;
constexpr int kPart = 4096;                                  // weights a workgroup sums
constexpr int kPerThread = kPart / kVerifyThreads;

template <int DT> struct Prob;
template <> struct Prob<DSKV_F32> {
    typedef float T;
    static __device__ __forceinline__ float widen(float x) { return x; }
};
template <> struct Prob<DSKV_F16> {
    typedef _Float16 T;
    static __device__ __forceinline__ float widen(_Float16 x) { return (float)x; }
};
template <> struct Prob<DSKV_BF16> {
    typedef uint16_t T;
    static __device__ __forceinline__ float widen(uint16_t x) { return __builtin_bit_cast(float, (uint32_t)x << 16); }
};

struct VerifyArgs {
    const void *target, *draft;
    long target_stride, draft_stride;      // elements
    const int32_t *tokens, *qo_indptr, *parents;
    const float *uniforms;
    int32_t *counts, *path, *out_tokens;
    double *sums;                          // (batch, parts): sum of w, then the same of p
    struct SharedWalk *walks;              // (batch)
    int batch, nnz, vocab, parts;
};

// What the workgroups need to know of a walk.
struct SharedWalk {
    long row, first;                       // the row reached, and the request's row 0, of all rows
    int count, n_refused;
    int minus_draft;
    float uniform;                         // of row 0
    int refused[DSKV_MAX_TREE_ROWS];       // tokens
};

// What is no probability counts as none.
template <int DT> __device__ __forceinline__ float weight_of(typename Prob<DT>::T x)
{
    const float f = Prob<DT>::widen(x);
    return f > 0.f && f <= __FLT_MAX__ ? f : 0.f;
}

struct Walk {
    long row;                      // the row reached, of all rows
    int count, n;                  // rows of the walk; rows of the request
    long first;
    bool minus_draft;              // w = max(p - q, 0)
    unsigned long long refused;    // children refused there
    float uniform;                 // of row 0
    int path;                      // lane j: j-th row of the walk
    int token, token_of_path;      // lane i: token of row i; lane j: token of the j-th row of the walk
};

// By one whole wave.
template <int DT> __device__ __forceinline__ Walk walk_drafts(const VerifyArgs &a, int b)
{
    typedef typename Prob<DT>::T T;
    const int lane = threadIdx.x & 63;
    Walk w = {0, 0, 0, 0, false, 0, 0.f, -1, -1, -1};
    const long first = a.qo_indptr[b], n = a.qo_indptr[b + 1] - first;
    w.first = first;
    if (first < 0 || n <= 0 || n > DSKV_MAX_TREE_ROWS || first + n > a.nnz) return w;
    w.n = (int)n;
    int up = -1, token = -1;
    double p = 0, q = 0;
    float u32 = 0;
    if (lane < n) {
        token = a.tokens[first + lane];
        u32 = a.uniforms[first + lane];
        up = lane == 0 ? -1 : a.parents ? a.parents[first + lane] : lane - 1;
        if (up >= lane) up = -1;
        if (up >= 0 && token >= 0 && token < a.vocab) {
            p = weight_of<DT>(((const T *)a.target)[(first + up) * a.target_stride + token]);
            if (a.draft) q = weight_of<DT>(((const T *)a.draft)[(first + up) * a.draft_stride + token]);
        }
    }
    const double u = u32;
    w.uniform = __shfl(u32, 0);
    const bool drafted = a.draft != nullptr;
    const bool chain_passes = drafted && up >= 0 && u * q < p;
    int at = 0, count = 1;
    int path = lane == 0 ? 0 : -1;
    for (;;) {
        const unsigned long long children = __ballot(up == at && lane > at);
        unsigned long long left = children, refused = 0;
        double rest = 1;
        int follow = -1;
        while (left) {
            const int c = __builtin_ctzll(left);
            left &= left - 1;
            bool pass;
            if (drafted) {
                pass = __shfl((int)chain_passes, c);
            } else {
                const int x = __shfl(token, c);
                const bool again = __ballot(((refused >> lane) & 1) && token == x) != 0;
                const double pc = __shfl(p, c);
                pass = !again && __shfl(u, c) * rest < pc;
                if (!again) rest -= pc;
            }
            if (pass) {
                follow = c;
                break;
            }
            refused |= 1ull << c;
        }
        if (follow < 0) {
            w.refused = refused;
            w.minus_draft = drafted && refused != 0;
            break;
        }
        at = follow;
        if (lane == count) path = at;
        count++;
    }
    w.row = first + at;
    w.count = count;
    w.path = path;
    w.token = token;
    w.token_of_path = __shfl(token, max(path, 0));
    return w;
}

// The walk for the workgroup's other waves.
__device__ __forceinline__ void share_walk(const Walk &w, SharedWalk &s, bool drafted)
{
    const int lane = threadIdx.x & 63;
    if (lane == 0) {
        s.row = w.row;
        s.first = w.first;
        s.count = w.count;
        s.minus_draft = w.minus_draft;
        s.uniform = w.uniform;
        s.n_refused = drafted ? 0 : __popcll(w.refused);
    }
    if (!drafted && ((w.refused >> lane) & 1)) s.refused[__popcll(w.refused & ((1ull << lane) - 1))] = w.token;
}

// Weights e0 .. e0 + 15 bytes' worth of the row, as many as a 16-byte load holds; rows start at any element.
template <int DT>
__device__ __forceinline__ void load_probs(const typename Prob<DT>::T *row, long e0, int vocab, float *p)
{
    typedef typename Prob<DT>::T T;
    constexpr int kN = 16 / sizeof(T);
    T x[kN];
    if (e0 + kN <= vocab) {
        __builtin_memcpy(x, row + e0, 16);
    } else {
#pragma unroll
        for (int i = 0; i < kN; i++) x[i] = e0 + i < vocab ? row[e0 + i] : T(0);
    }
#pragma unroll
    for (int i = 0; i < kN; i++) p[i] = weight_of<DT>(x[i]);
}

// The thread's weights of a part: kPerThread / kN runs of kN, the first at e0, kStep elements apart.
template <int DT, int kStep>
__device__ __forceinline__ void load_weights(const VerifyArgs &a, const SharedWalk &s, long e0, float (&p)[kPerThread],
                                             double (&w)[kPerThread])
{
    typedef typename Prob<DT>::T T;
    constexpr int kN = 16 / sizeof(T);
    const T *target = (const T *)a.target + s.row * a.target_stride;
    const T *draft = (const T *)a.draft + s.row * a.draft_stride;
#pragma unroll
    for (int i = 0; i < kPerThread / kN; i++) load_probs<DT>(target, e0 + i * kStep, a.vocab, p + i * kN);
    if (s.minus_draft) {
        float q[kPerThread];
#pragma unroll
        for (int i = 0; i < kPerThread / kN; i++) load_probs<DT>(draft, e0 + i * kStep, a.vocab, q + i * kN);
#pragma unroll
        for (int i = 0; i < kPerThread; i++) w[i] = p[i] > q[i] ? (double)p[i] - (double)q[i] : 0.0;
    } else {
#pragma unroll
        for (int i = 0; i < kPerThread; i++) w[i] = p[i];
        for (int r = 0; r < s.n_refused; r++) {
            const long at = s.refused[r] - e0;
#pragma unroll
            for (int i = 0; i < kPerThread; i++)
                if (at == i / kN * kStep + i % kN) w[i] = 0;
        }
    }
}

// Sums up to and with this lane's over a wave, by moves between lanes that do not go through LDS.
template <int kCtrl, int kRows> __device__ __forceinline__ double lanes_below(double v)
{
    const uint64_t x = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, kCtrl, kRows, 0xf, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), kCtrl, kRows, 0xf, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_scan64(double v)
{
    v += lanes_below<0x111, 0xf>(v);       // row_shr 1, 2, 4, 8 within 16 lanes
    v += lanes_below<0x112, 0xf>(v);
    v += lanes_below<0x114, 0xf>(v);
    v += lanes_below<0x118, 0xf>(v);
    v += lanes_below<0x142, 0xa>(v);       // the last lane of rows 0 and 2 to rows 1 and 3
    v += lanes_below<0x143, 0xc>(v);       // lane 31 to rows 2 and 3
    return v;
}
__device__ __forceinline__ double wave_sum64(double v)
{
    const uint64_t x = __builtin_bit_cast(uint64_t, wave_scan64(v));
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)x, 63), hi = __builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), 63);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

template <int DT> __global__ __launch_bounds__(kVerifyThreads) void verify_sums_kernel(VerifyArgs a)
{
    __shared__ SharedWalk s;
    __shared__ double of_wave[kVerifyThreads / 64][2];
    const int b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool tells = blockIdx.x == 0;
    // rows behind the last request
    if (tells && b >= a.batch - 1) {
        const long end = max((long)a.qo_indptr[a.batch], 0L);
        for (long t = end + threadIdx.x; t < a.nnz; t += kVerifyThreads) a.path[t] = a.out_tokens[t] = -1;
    }
    if (b >= a.batch) return;                                      // no requests at all: no entry of theirs, no workspace
    if (wave == 0) {
        const Walk w = walk_drafts<DT>(a, b);
        share_walk(w, s, a.draft != nullptr);
        if (tells) {
            share_walk(w, a.walks[b], a.draft != nullptr);
            const int next = __shfl(w.token_of_path, min(lane + 1, 63));
            if (lane < w.n) {
                a.path[w.first + lane] = lane < w.count ? w.path : -1;
                if (lane != w.count - 1) a.out_tokens[w.first + lane] = lane < w.count ? next : -1;
            }
            if (lane == 0) a.counts[b] = w.count;
        }
    }
    __syncthreads();
    if (s.count == 0) {                                            // no rows, or too many
        const long lo = max((long)a.qo_indptr[b], 0L), hi = min((long)a.qo_indptr[b + 1], (long)a.nnz);
        if (tells)
            for (long t = lo + threadIdx.x; t < hi; t += kVerifyThreads) a.path[t] = a.out_tokens[t] = -1;
        return;
    }
    constexpr int kN = 16 / sizeof(typename Prob<DT>::T);
    float p[kPerThread];
    double w[kPerThread], sw = 0, sp = 0;
    load_weights<DT, kVerifyThreads * kN>(a, s, (long)blockIdx.x * kPart + threadIdx.x * kN, p, w);
#pragma unroll
    for (int i = 0; i < kPerThread; i++) {
        sw += w[i];
        sp += p[i];
    }
    sw = wave_sum64(sw);
    sp = wave_sum64(sp);
    if (lane == 0) {
        of_wave[wave][0] = sw;
        of_wave[wave][1] = sp;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        double sum = 0;
#pragma unroll
        for (int i = 0; i < kVerifyThreads / 64; i++) sum += of_wave[i][threadIdx.x];
        a.sums[((long)threadIdx.x * a.batch + b) * a.parts + blockIdx.x] = sum;
    }
}

template <int DT> __global__ __launch_bounds__(kVerifyThreads) void verify_draw_kernel(VerifyArgs a)
{
    __shared__ SharedWalk s;
    __shared__ double of_wave[kVerifyThreads / 64];
    __shared__ int hit_of[kVerifyThreads / 64], mass_of[kVerifyThreads / 64];
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    static_assert(sizeof(SharedWalk) % 4 == 0 && sizeof(SharedWalk) / 4 <= kVerifyThreads, "a word a thread");
    if (threadIdx.x < sizeof(SharedWalk) / 4) ((int *)&s)[threadIdx.x] = ((const int *)(a.walks + b))[threadIdx.x];
    // sums of the parts, of w and of p, 64 at a time by every wave alike
    const double *of_w = a.sums + (long)b * a.parts, *of_p = of_w + (long)a.batch * a.parts;
    double first_w = lane < a.parts ? of_w[lane] : 0, first_p = lane < a.parts ? of_p[lane] : 0;
    __syncthreads();
    if (s.count == 0) return;
    const double u = s.uniform;
    double scan_w = wave_scan64(first_w), total = __shfl(scan_w, 63);
    for (int i = 64; i < a.parts; i += 64) total += wave_sum64(i + lane < a.parts ? of_w[i + lane] : 0);
    const bool from_p = !(total > 0);            // w has no mass
    const double *sums = from_p ? of_p : of_w;
    if (from_p) {
        scan_w = wave_scan64(first_p);
        total = __shfl(scan_w, 63);
        for (int i = 64; i < a.parts; i += 64) total += wave_sum64(i + lane < a.parts ? of_p[i + lane] : 0);
    }
    const double target = u < 0 ? 0 : u * total;
    // the first part whose sum passes the target; if rounding or u lets none, the last with mass
    double before = 0, before_part = 0;
    int part = -1;
    for (int i = 0; i < a.parts; i += 64) {
        const double sum = i == 0 ? (from_p ? first_p : first_w) : i + lane < a.parts ? sums[i + lane] : 0;
        const double upto = i == 0 ? scan_w : before + wave_scan64(sum);
        const unsigned long long mass = __ballot(sum > 0), over = __ballot(sum > 0 && upto > target);
        if (mass) {
            const int at = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(mass);
            part = i + at;
            before_part = __shfl(upto - sum, at);
        }
        if (over) break;
        before = __shfl(upto, 63);
    }
    int token = 0;
    if (part >= 0) {
        constexpr int kN = 16 / sizeof(typename Prob<DT>::T);
        float p[kPerThread];
        double w[kPerThread], mine = 0;
        load_weights<DT, kN>(a, s, (long)part * kPart + threadIdx.x * kPerThread, p, w);
#pragma unroll
        for (int i = 0; i < kPerThread; i++) {
            if (from_p) w[i] = p[i];
            mine += w[i];
        }
        const double upto = wave_scan64(mine);
        if (lane == 63) of_wave[wave] = upto;
        __syncthreads();
        double cum = before_part + upto - mine;
#pragma unroll
        for (int i = 0; i < kVerifyThreads / 64; i++)
            if (i < wave) cum += of_wave[i];
        const int e0 = threadIdx.x * kPerThread;
        int hit = -1, mass = -1;               // first weight that passes the target; last with weight at all
#pragma unroll
        for (int i = 0; i < kPerThread; i++) {
            cum += w[i];
            if (w[i] > 0) {
                mass = e0 + i;
                if (hit < 0 && cum > target) hit = e0 + i;
            }
        }
        const unsigned long long hits = __ballot(hit >= 0), masses = __ballot(mass >= 0);
        hit = __shfl(hit, hits ? __builtin_ctzll(hits) : 0);
        mass = __shfl(mass, masses ? 63 - __builtin_clzll(masses) : 0);
        if (lane == 0) {
            hit_of[wave] = hits ? hit : -1;
            mass_of[wave] = masses ? mass : -1;
        }
        __syncthreads();
        int drawn = -1, last = 0;
#pragma unroll
        for (int i = 0; i < kVerifyThreads / 64; i++) {
            if (drawn < 0) drawn = hit_of[i];
            last = max(last, mass_of[i]);
        }
        // rounding may leave the sum of the part below what its whole sum promised
        token = part * kPart + (drawn >= 0 ? drawn : last);
    }
    if (threadIdx.x == 0) a.out_tokens[s.first + s.count - 1] = token;
}

static int verify_parts(int vocab) { return (vocab - 1) / kPart + 1; }

}  // namespace dskv

extern "C" int64_t dskv_verify_workspace(int32_t batch, int32_t vocab)
{
    if (batch <= 0 || vocab <= 0) return 0;
    return batch * (dskv::verify_parts(vocab) * 2 * (int64_t)sizeof(double) + (int64_t)sizeof(dskv::SharedWalk));
}

extern "C" int dskv_verify_drafts(int32_t *counts, int32_t *path, int32_t *out_tokens, const void *target_probs,
                                  int64_t target_stride, const void *draft_probs, int64_t draft_stride,
                                  const int32_t *tokens, const float *uniforms, const int32_t *qo_indptr,
                                  const int32_t *parents, void *workspace, int64_t workspace_bytes, int32_t batch,
                                  int32_t nnz, int32_t vocab, int32_t dtype, void *stream)
{
    using namespace dskv;
    DSKV_REQUIRE(batch >= 0 && nnz >= 0, "verify_drafts: negative batch/nnz");
    DSKV_REQUIRE(vocab > 0, "verify_drafts: vocab must be positive");
    if (batch == 0 && nnz == 0) return 0;
    DSKV_REQUIRE((counts || batch == 0) && qo_indptr, "verify_drafts: null pointer argument");
    DSKV_REQUIRE(nnz == 0 || (path && out_tokens && target_probs && tokens && uniforms), "verify_drafts: null pointer argument");
    DSKV_REQUIRE(dtype == DSKV_F32 || dtype == DSKV_F16 || dtype == DSKV_BF16, "verify_drafts: unknown dtype %d", dtype);
    DSKV_REQUIRE(!draft_probs || !parents, "verify_drafts: draft_probs belong to chains, parents to trees of proposed tokens");
    DSKV_REQUIRE(target_stride >= vocab && (!draft_probs || draft_stride >= vocab), "verify_drafts: rows overlap");
    DSKV_REQUIRE(batch <= 65535, "verify_drafts: at most 65535 requests a call");
    if (batch > 0 && (!workspace || workspace_bytes < dskv_verify_workspace(batch, vocab))) {
        set_error("verify_drafts: workspace of %lld bytes, %lld are needed", (long long)workspace_bytes,
                  (long long)dskv_verify_workspace(batch, vocab));
        return DSKV_E_NOMEM;
    }
    DSKV_REQUIRE((uintptr_t)workspace % 16 == 0, "verify_drafts: the workspace must be 16-byte aligned");
    const int parts = verify_parts(vocab);
    VerifyArgs a = {target_probs, draft_probs, (long)target_stride, (long)draft_stride, tokens, qo_indptr, parents,
                    uniforms, counts, path, out_tokens, (double *)workspace,
                    (SharedWalk *)((double *)workspace + (int64_t)batch * parts * 2), batch, nnz, vocab, parts};
    hipStream_t s = (hipStream_t)stream;
#define DSKV_LAUNCH_VERIFY(DT)                                                                                      \
    do {                                                                                                            \
        hipLaunchKernelGGL((verify_sums_kernel<DT>), dim3((unsigned)parts, (unsigned)(batch > 0 ? batch : 1)),      \
                           dim3(kVerifyThreads), 0, s, a);                                                          \
        DSKV_LAUNCH_CHECK("verify_sums_kernel");                                                                    \
        if (batch > 0) {                                                                                            \
            hipLaunchKernelGGL((verify_draw_kernel<DT>), dim3((unsigned)batch), dim3(kVerifyThreads), 0, s, a);     \
            DSKV_LAUNCH_CHECK("verify_draw_kernel");                                                                \
        }                                                                                                           \
    } while (0)
    if (dtype == DSKV_F32) DSKV_LAUNCH_VERIFY(DSKV_F32);
    else if (dtype == DSKV_F16) DSKV_LAUNCH_VERIFY(DSKV_F16);
    else DSKV_LAUNCH_VERIFY(DSKV_BF16);
#undef DSKV_LAUNCH_VERIFY
    return 0;
}
