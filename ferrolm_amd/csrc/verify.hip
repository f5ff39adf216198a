// Verification of drafted trees: the walk from a sequence's first row along the
// drafted tokens that the target's distributions accept, and the draw that ends
// it, from given uniform numbers.
//
// At a node with target distribution p and draft distribution q the children
// are tried in order; with P = p at first, child c passes when u q(c) < P(c)
// (and q(c) > 0), and a rejection leaves P <- max(0, P - q) / sum. After j
// rejections that is max(0, p - a q) / b with two numbers,
//   a' = a + b / d,  b' = sum over the vocabulary of max(0, p - a' q),
// d = 1 for independent draws, 1 - (q of the tokens drawn before) for draws
// without replacement: a token that was drawn before and rejected has
// p - a q < 0 already, so it needs no mark. Given drafts (no q) pass when
// u < P(c), and a rejected token's mass is removed. The emitted tokens then
// have exactly the target's distribution.
//
// Everything is in 64 bits: a sum over a vocabulary of 32-bit values and the
// place where a cumulative sum passes a threshold are as exact as the inputs.
#include "devutil.h"

namespace fg {

namespace {

constexpr int kVerifyThreads = 1024, kVerifyWaves = kVerifyThreads / 64;
// What q's tokens drawn so far leave of its sum, below which it is spent: a sum of f32 probabilities is 1 only to
// about that.
constexpr double kSpent = 0x1p-20;
constexpr int kKids = 256;  // children of a node taken at a time

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m);
    return x;
}

// What is left of a node's distribution.
struct Left {
    const float *p, *q;  // q: nullptr for given drafts
    double a;
    const uint32_t* gone;  // given drafts: the tokens removed
    int n_gone;
    __device__ __forceinline__ double at(int t) const {
        const float x = p[t];
        const double w = x > 0.0f ? (double)x : 0.0;  // a NaN counts as 0
        if (q) {
            const float y = q[t];
            const double r = w - a * (y > 0.0f ? (double)y : 0.0);
            return r > 0.0 ? r : 0.0;
        }
        for (int i = 0; i < n_gone; i++)
            if (gone[i] == (uint32_t)t) return 0.0;
        return w;
    }
};

// Sums of 16 consecutive shares of [first, last), one a wave; every thread returns their total.
__device__ __forceinline__ int share_len(int n) { return (n + kVerifyWaves - 1) / kVerifyWaves; }
__device__ double shares(const Left& f, int first, int last, double* sums) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, len = share_len(last - first);
    const int t0 = first + wave * len, t1 = min(last, t0 + len);
    double x = 0.0;
    for (int t = t0 + lane; t < t1; t += 64) x += f.at(t);
    x = wave_sum(x);
    __syncthreads();  // the sums of the call before have been read
    if (lane == 0) sums[wave] = x;
    __syncthreads();
    double total = 0.0;
    for (int w = 0; w < kVerifyWaves; w++) total += sums[w];
    return total;
}
// The share in which the cumulative sum passes `target`, which becomes relative to the share's start; where
// rounding leaves none, the last share with any mass.
__device__ __forceinline__ int pick(const double* sums, double& target) {
    double c = 0.0, start = 0.0;
    int last = 0;
    for (int w = 0; w < kVerifyWaves; w++) {
        if (c + sums[w] > target) {
            target -= c;
            return w;
        }
        if (sums[w] > 0.0) {
            last = w;
            start = c;
        }
        c += sums[w];
    }
    target -= start;
    return last;
}

}  // namespace

// One workgroup per sequence.
__global__ __launch_bounds__(kVerifyThreads) void k_tree_verify(RowArgs a, VerifyArgs v) {
    __shared__ double sums[kVerifyWaves];
    __shared__ uint32_t ctok[kKids];
    __shared__ float cp[kKids], cq[kKids], cu[kKids];
    __shared__ int seen[kKids];  // an earlier sibling has the token
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const int row0 = a.seqs[(size_t)s * kSeqWords], V = v.vocab;
    uint32_t* out = v.out_tokens + (size_t)s * v.ld;
    int32_t* path = v.out_path + (size_t)s * v.ld;
    int node = row0, count = 1, known = 0;  // known: sums holds the shares of what is left
    Left left{};
    double total = 0.0;
    if (tid == 0) path[0] = 0;
    for (;;) {
        const int c0 = a.cstart[node], nc = a.cstart[node + 1] - c0;
        left = Left{v.p + (size_t)node * V, v.kind == DRAFT_FIXED ? nullptr : v.q + (size_t)node * V, 0.0, nullptr, 0};
        known = 0;
        double b = 1.0, d = 1.0;
        int passed = -1;
        for (int j0 = 0; j0 < nc && passed < 0 && b > 0.0; j0 += kKids) {
            const int m = min(kKids, nc - j0);
            __syncthreads();
            for (int j = tid; j < m; j += kVerifyThreads) {
                const int row = a.clist[c0 + j0 + j];
                const uint32_t t = v.tokens[row];
                const bool in = t < (uint32_t)V;  // a token outside the vocabulary never passes
                const float x = in ? left.p[t] : 0.0f, y = in ? (left.q ? left.q[t] : 1.0f) : 0.0f;
                ctok[j] = t;
                cu[j] = v.u[row];
                cp[j] = x > 0.0f ? x : 0.0f;
                cq[j] = y > 0.0f ? y : 0.0f;
                int before = 0;
                if (v.kind != DRAFT_EACH)
                    for (int i = 0; i < j0 + j && !before; i++) before = v.tokens[a.clist[c0 + i]] == t;
                seen[j] = before;
            }
            __syncthreads();
            for (int j = 0; j < m; j++) {
                const double p = cp[j], q = cq[j], u = cu[j];
                double mass, rate;
                if (v.kind == DRAFT_FIXED) {
                    mass = seen[j] ? 0.0 : p / b;
                    rate = q;
                } else {
                    // without replacement: a token drawn before, or one that q had nothing left for, was not drawn
                    if (v.kind == DRAFT_DISTINCT && (seen[j] || d < kSpent || q == 0.0)) continue;
                    const double r = p - left.a * q;
                    rate = q / d;
                    mass = (r > 0.0 ? r : 0.0) / b;
                }
                if (u * rate < mass && rate > 0.0) {
                    passed = a.clist[c0 + j0 + j];
                    break;
                }
                if (v.kind == DRAFT_FIXED) {
                    if (!seen[j]) b -= p;
                } else {
                    left.a += b / d;
                    if (v.kind == DRAFT_DISTINCT) d -= q;
                    b = total = shares(left, 0, V, sums);
                    known = 1;
                    if (!(b > 0.0)) break;  // nothing is left: no child passes
                }
            }
        }
        if (passed < 0) {
            if (v.kind == DRAFT_FIXED && nc > 0) left.n_gone = nc;
            break;
        }
        if (tid == 0) {
            out[count - 1] = v.tokens[passed];
            path[count] = passed - row0;
        }
        node = passed;
        count++;
    }
    // the removed tokens of a node with given drafts
    __shared__ uint32_t gone[kKids];
    extern __shared__ uint32_t more[];
    if (left.n_gone) {
        uint32_t* g = left.n_gone <= kKids ? gone : more;
        for (int i = tid; i < left.n_gone; i += kVerifyThreads) g[i] = v.tokens[a.clist[a.cstart[node] + i]];
        left.gone = g;
        __syncthreads();
    }
    if (!known) total = shares(left, 0, V, sums);
    if (!(total > 0.0)) {  // nothing is left: the target's own distribution
        left.a = 0.0;
        left.q = nullptr;
        left.n_gone = 0;
        total = shares(left, 0, V, sums);
    }
    double target = (double)v.u[row0] * total;
    int first = 0, last = V;
    for (int round = 0; round < 2; round++) {
        if (round) (void)shares(left, first, last, sums);
        const int w = pick(sums, target), len = share_len(last - first);
        first += w * len;
        last = max(first, min(last, first + len));
    }
    if (tid >= 64) return;
    // one wave, in token order
    int found = -1, positive = 0;
    double c = 0.0;
    for (int t0 = first; t0 < last && found < 0; t0 += 64) {
        const int t = t0 + lane;
        const double w = t < last ? left.at(t) : 0.0;
        double x = w;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const double y = __shfl_up(x, m);
            if (lane >= m) x += y;
        }
        const uint64_t any = __ballot(w > 0.0), hit = __ballot(c + x > target && w > 0.0);
        if (hit) found = t0 + __builtin_ctzll(hit);
        if (any) positive = t0 + 63 - __builtin_clzll(any);
        c += __shfl(x, 63);
    }
    if (lane == 0) {
        out[count - 1] = (uint32_t)(found >= 0 ? found : positive);
        v.out_count[s] = count;
    }
    for (int i = count + lane; i < v.ld; i += 64) {
        out[i] = 0;
        path[i] = -1;
    }
}

void launch_tree_verify(hipStream_t st, const RowArgs& a, const VerifyArgs& v) {
    if (a.n_seqs <= 0) return;
    const size_t more = v.kind == DRAFT_FIXED && a.widest > kKids ? (size_t)a.widest * 4 : 0;
    hipLaunchKernelGGL(k_tree_verify, dim3(a.n_seqs), dim3(kVerifyThreads), more, st, a, v);
}

// One wave per sequence.
__global__ __launch_bounds__(64) void k_tree_accept(RowArgs a, const uint32_t* __restrict__ tokens,
                                                    const uint32_t* __restrict__ argmax, uint32_t* __restrict__ out_tokens,
                                                    int32_t* __restrict__ out_path, int32_t* __restrict__ out_count,
                                                    int ld) {
    const int s = blockIdx.x, lane = threadIdx.x, row0 = a.seqs[(size_t)s * kSeqWords];
    uint32_t* out = out_tokens + (size_t)s * ld;
    int32_t* path = out_path + (size_t)s * ld;
    int node = row0, count = 0;
    for (;;) {
        const uint32_t best = argmax[node];
        if (lane == 0) {
            out[count] = best;
            path[count] = node - row0;
        }
        count++;
        const int c0 = a.cstart[node], c1 = a.cstart[node + 1];
        int next = -1;
        for (int c = c0; c < c1 && next < 0; c += 64) {
            const uint64_t hit = __ballot(c + lane < c1 && tokens[a.clist[min(c + lane, c1 - 1)]] == best);
            if (hit) next = a.clist[c + __builtin_ctzll(hit)];
        }
        if (next < 0) break;
        node = next;
    }
    if (lane == 0) out_count[s] = count;
    for (int i = count + lane; i < ld; i += 64) {
        out[i] = 0;
        path[i] = -1;
    }
}

void launch_tree_accept(hipStream_t st, const RowArgs& a, const uint32_t* tokens, const uint32_t* argmax,
                        uint32_t* out_tokens, int32_t* out_path, int32_t* out_count, int ld) {
    if (a.n_seqs > 0)
        hipLaunchKernelGGL(k_tree_accept, dim3(a.n_seqs), dim3(64), 0, st, a, tokens, argmax, out_tokens, out_path,
                           out_count, ld);
}

// A row's distribution (launch_dist, prm[row]) by token; a greedy row's (temperature <= 0) is all on its argmax.
__global__ __launch_bounds__(256) void k_dense(SampleRows d, const SampleParams* __restrict__ prm,
                                               const uint32_t* __restrict__ argmax, float* __restrict__ p) {
    const int row = blockIdx.x;
    const SampleParams s = prm[row];
    float* y = p + (size_t)row * d.vocab;
    if (s.temperature > 0.0f && sample_wide(s)) {
        for (int i = threadIdx.x; i < d.vocab; i += 256) y[i] = d.dense[(size_t)row * d.cap + i];
        return;
    }
    for (int i = threadIdx.x; i < d.vocab; i += 256) y[i] = 0.0f;
    __syncthreads();
    if (s.temperature <= 0.0f) {
        if (threadIdx.x == 0) y[argmax[row]] = 1.0f;
        return;
    }
    for (int i = threadIdx.x; i < d.n[row]; i += 256)
        y[d.tok_id[(size_t)row * d.cap + i]] = d.pr_id[(size_t)row * d.cap + i];
}

void launch_dense(hipStream_t st, const SampleRows& d, int rows, const SampleParams* prm, const uint32_t* argmax,
                  float* p) {
    if (rows > 0) hipLaunchKernelGGL(k_dense, dim3(rows), dim3(256), 0, st, d, prm, argmax, p);
}

}  // namespace fg
