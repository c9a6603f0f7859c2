// Verification of drafted tokens against the target's probabilities.
//
// The walk from a request's row 0 down needs single probabilities only: row i's token at its parent's row, p_i, and
// with the draft's distributions q_i.  All are gathered at once, a lane per row, and the walk itself is scalar: the
// children of the row reached are a ballot.  Then one row of the vocabulary is left, the weights w of the token behind the
// walk (see dskv_verify_drafts): first its sum, then the first index whose cumulated weight passes uniform * sum.
// Sums and comparisons are in 64 bits: an index is drawn among 1e5 weights of 1e-5, which sums in 32 bits would
// move by whole tokens, and a product of two 32-bit numbers is exact in 64.
//
// Bound by reading that row (of p, and of q) where there are requests enough, by the chain of two launches otherwise.
// Two launches: the first sums parts of kPart weights, each workgroup taking the walk for itself (a few hundred
// bytes from L2), the second finds the part by the parts' sums and the token in it.
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
    int batch, nnz, vocab, parts;
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
    int path;                      // lane j: j-th row of the walk
    int token, token_of_path;      // lane i: token of row i; lane j: token of the j-th row of the walk
};

// By one whole wave.
template <int DT> __device__ __forceinline__ Walk walk_drafts(const VerifyArgs &a, int b)
{
    typedef typename Prob<DT>::T T;
    const int lane = threadIdx.x & 63;
    Walk w = {0, 0, 0, 0, false, 0, -1, -1, -1};
    const long first = a.qo_indptr[b], n = a.qo_indptr[b + 1] - first;
    w.first = first;
    if (first < 0 || n <= 0 || n > DSKV_MAX_TREE_ROWS || first + n > a.nnz) return w;
    w.n = (int)n;
    int up = -1, token = -1;
    double p = 0, q = 0, u = 0;
    if (lane < n) {
        token = a.tokens[first + lane];
        u = a.uniforms[first + lane];
        up = lane == 0 ? -1 : a.parents ? a.parents[first + lane] : lane - 1;
        if (up >= lane) up = -1;
        if (up >= 0 && token >= 0 && token < a.vocab) {
            p = weight_of<DT>(((const T *)a.target)[(first + up) * a.target_stride + token]);
            if (a.draft) q = weight_of<DT>(((const T *)a.draft)[(first + up) * a.draft_stride + token]);
        }
    }
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
struct SharedWalk {
    long row;
    int count, n_refused;
    bool minus_draft;
    int refused[DSKV_MAX_TREE_ROWS];       // tokens
};
__device__ __forceinline__ void share_walk(const Walk &w, SharedWalk &s, bool drafted)
{
    const int lane = threadIdx.x & 63;
    if (lane == 0) {
        s.row = w.row;
        s.count = w.count;
        s.minus_draft = w.minus_draft;
        s.n_refused = drafted ? 0 : __popcll(w.refused);
    }
    if (!drafted && ((w.refused >> lane) & 1)) s.refused[__popcll(w.refused & ((1ull << lane) - 1))] = w.token;
}

// Thread t's weights of a part: elements t * kPerThread .. of it.
template <int DT>
__device__ __forceinline__ void load_weights(const VerifyArgs &a, const SharedWalk &s, long part, float (&p)[kPerThread],
                                             double (&w)[kPerThread])
{
    typedef typename Prob<DT>::T T;
    const long e0 = part * kPart + threadIdx.x * kPerThread;
    const T *target = (const T *)a.target + s.row * a.target_stride;
    const T *draft = (const T *)a.draft + s.row * a.draft_stride;
#pragma unroll
    for (int i = 0; i < kPerThread; i++) p[i] = e0 + i < a.vocab ? weight_of<DT>(target[e0 + i]) : 0.f;
    if (s.minus_draft) {
#pragma unroll
        for (int i = 0; i < kPerThread; i++) {
            const float q = e0 + i < a.vocab ? weight_of<DT>(draft[e0 + i]) : 0.f;
            w[i] = fmax((double)p[i] - (double)q, 0.0);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPerThread; i++) w[i] = p[i];
        for (int r = 0; r < s.n_refused; r++) {
            const long at = s.refused[r] - e0;
#pragma unroll
            for (int i = 0; i < kPerThread; i++)
                if (at == i) w[i] = 0;
        }
    }
}

__device__ __forceinline__ double wave_sum64(double v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

template <int DT> __global__ __launch_bounds__(kVerifyThreads) void verify_sums_kernel(VerifyArgs a)
{
    __shared__ SharedWalk s;
    __shared__ double of_wave[kVerifyThreads / 64][2];
    const int b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (wave == 0) share_walk(walk_drafts<DT>(a, b), s, a.draft != nullptr);
    __syncthreads();
    if (s.count == 0) return;
    float p[kPerThread];
    double w[kPerThread], sw = 0, sp = 0;
    load_weights<DT>(a, s, blockIdx.x, p, w);
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
    __shared__ int drawn, last_with_mass;
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Walk walk = {};
    if (wave == 0 && b < a.batch) {
        walk = walk_drafts<DT>(a, b);
        share_walk(walk, s, a.draft != nullptr);
    }
    if (threadIdx.x == 0) drawn = 0x7fffffff, last_with_mass = -1;
    // rows behind the last request, and those of requests that are left out
    if (b >= a.batch - 1) {
        const long end = max((long)a.qo_indptr[a.batch], 0L);
        for (long t = end + threadIdx.x; t < a.nnz; t += kVerifyThreads) a.path[t] = a.out_tokens[t] = -1;
    }
    if (b >= a.batch) return;                  // no requests at all
    __syncthreads();
    if (s.count == 0) {
        const long lo = max((long)a.qo_indptr[b], 0L), hi = min((long)a.qo_indptr[b + 1], (long)a.nnz);
        for (long t = lo + threadIdx.x; t < hi; t += kVerifyThreads) a.path[t] = a.out_tokens[t] = -1;
        if (threadIdx.x == 0) a.counts[b] = 0;
        return;
    }
    // the part that the draw falls into: sums of the parts in order, by every thread alike
    const double *sums = a.sums + (long)b * a.parts;
    double total = 0;
    for (int i = 0; i < a.parts; i++) total += sums[i];
    const bool of_p = !(total > 0);            // w has no mass
    if (of_p) {
        sums += (long)a.batch * a.parts;
        total = 0;
        for (int i = 0; i < a.parts; i++) total += sums[i];
    }
    const double u = a.uniforms[a.qo_indptr[b]];
    const double target = u < 0 ? 0 : u * total;
    double before = 0;
    int part = -1;
    double before_part = 0;
    for (int i = 0; i < a.parts; i++) {
        const double sum = sums[i];
        if (sum > 0) {
            part = i;                          // the last with mass, if the draw is behind all of them
            before_part = before;
        }
        before += sum;
        if (before > target) break;
    }
    int token = 0;
    if (part >= 0) {
        float p[kPerThread];
        double w[kPerThread], mine = 0;
        load_weights<DT>(a, s, part, p, w);
#pragma unroll
        for (int i = 0; i < kPerThread; i++) {
            if (of_p) w[i] = p[i];
            mine += w[i];
        }
        double upto = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double v = __shfl_up(upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 63) of_wave[wave] = upto;
        __syncthreads();
        double cum = before_part + upto - mine;
#pragma unroll
        for (int i = 0; i < kVerifyThreads / 64; i++)
            if (i < wave) cum += of_wave[i];
        const int e0 = threadIdx.x * kPerThread;
        int hit = 0x7fffffff, mass = -1;
#pragma unroll
        for (int i = 0; i < kPerThread; i++) {
            cum += w[i];
            if (w[i] > 0) {
                mass = e0 + i;
                if (cum > target) hit = min(hit, e0 + i);
            }
        }
        if (hit != 0x7fffffff) atomicMin(&drawn, hit);
        if (mass >= 0) atomicMax(&last_with_mass, mass);
        __syncthreads();
        // rounding may leave the sum of the part below what its whole sum promised
        token = part * kPart + (drawn != 0x7fffffff ? drawn : max(last_with_mass, 0));
    }
    if (wave == 0 && lane < walk.n) {
        const int next = __shfl(walk.token_of_path, min(lane + 1, 63));
        a.path[walk.first + lane] = lane < walk.count ? walk.path : -1;
        a.out_tokens[walk.first + lane] = lane < walk.count - 1 ? next : lane == walk.count - 1 ? token : -1;
        if (lane == 0) a.counts[b] = walk.count;
    }
}

static int verify_parts(int vocab) { return (vocab + kPart - 1) / kPart; }

}  // namespace dskv

extern "C" int64_t dskv_verify_workspace(int32_t batch, int32_t vocab)
{
    if (batch <= 0 || vocab <= 0) return 0;
    return (int64_t)batch * dskv::verify_parts(vocab) * 2 * (int64_t)sizeof(double);
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
                    uniforms, counts, path, out_tokens, (double *)workspace, batch, nnz, vocab, parts};
    hipStream_t s = (hipStream_t)stream;
#define DSKV_LAUNCH_VERIFY(DT)                                                                                      \
    do {                                                                                                            \
        if (batch > 0) {                                                                                            \
            hipLaunchKernelGGL((verify_sums_kernel<DT>), dim3((unsigned)parts, (unsigned)batch),                    \
                               dim3(kVerifyThreads), 0, s, a);                                                      \
            DSKV_LAUNCH_CHECK("verify_sums_kernel");                                                                \
        }                                                                                                           \
        hipLaunchKernelGGL((verify_draw_kernel<DT>), dim3((unsigned)(batch > 0 ? batch : 1)),                       \
                           dim3(kVerifyThreads), 0, s, a);                                                          \
        DSKV_LAUNCH_CHECK("verify_draw_kernel");                                                                    \
    } while (0)
    if (dtype == DSKV_F32) DSKV_LAUNCH_VERIFY(DSKV_F32);
    else if (dtype == DSKV_F16) DSKV_LAUNCH_VERIFY(DSKV_F16);
    else DSKV_LAUNCH_VERIFY(DSKV_BF16);
#undef DSKV_LAUNCH_VERIFY
    return 0;
}
