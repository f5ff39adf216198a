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

// Sums over aligned groups of 16 or 64 lanes without the LDS crossbar (devutil.h's lane swaps, a half at a time).
template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double row_sum(double x) {
    x += dpp_d<0xB1>(x);   // quad_perm [1,0,3,2]
    x += dpp_d<0x4E>(x);   // quad_perm [2,3,0,1]
    x += dpp_d<0x141>(x);  // row_half_mirror
    return x + dpp_d<0x140>(x);  // row_mirror
}
__device__ __forceinline__ double wave_sum(double x) {
    x = row_sum(x);
    uint64_t b = __builtin_bit_cast(uint64_t, x);
    const auto l = __builtin_amdgcn_permlane16_swap((uint32_t)b, (uint32_t)b, false, false);
    const auto h = __builtin_amdgcn_permlane16_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
    x = __builtin_bit_cast(double, (uint64_t)h[0] << 32 | l[0]) + __builtin_bit_cast(double, (uint64_t)h[1] << 32 | l[1]);
    b = __builtin_bit_cast(uint64_t, x);
    const auto m = __builtin_amdgcn_permlane32_swap((uint32_t)b, (uint32_t)b, false, false);
    const auto n = __builtin_amdgcn_permlane32_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
    return __builtin_bit_cast(double, (uint64_t)n[0] << 32 | m[0]) + __builtin_bit_cast(double, (uint64_t)n[1] << 32 | m[1]);
}
// x > 0, or 0: a NaN counts as 0
__device__ __forceinline__ double mass_of(float x) { return (double)fmaxf(x, 0.0f); }

// What is left of a node's distribution.
struct Left {
    const float *p, *q;  // q: nullptr for given drafts
    double a;
    template <bool Q>
    __device__ __forceinline__ double of(float x, float y) const {
        return Q ? fmax(mass_of(x) - a * mass_of(y), 0.0) : mass_of(x);
    }
};
// Given drafts: the tokens of the node's children, whose mass is removed.
struct Gone {
    const uint32_t* at;
    int n;
    // f(token) for those in [first, last), by whole waves
    template <class F>
    __device__ __forceinline__ void each(int first, int last, const F& f) const {
        const int lane = threadIdx.x & 63;
        for (int i = 0; i < n; i += 64) {
            const uint32_t g = at[min(i + lane, n - 1)];
            uint64_t in = __ballot(i + lane < n && g >= (uint32_t)first && g < (uint32_t)last);
            for (; in; in &= in - 1) f((int)__builtin_amdgcn_readlane(g, __builtin_ctzll(in)));
        }
    }
};

// Sums of 16 consecutive shares of [first, last), one a wave, into sums; every thread returns their total. V4: rows
// are 16-byte aligned and the shares whole groups of four.
template <bool V4>
__device__ __forceinline__ int share_len(int n) {
    const int len = (n + kVerifyWaves - 1) / kVerifyWaves;
    return V4 ? (len + 3) / 4 * 4 : len;
}
// A wave's share, UN loads of each row on their way per lane, of four values (V4) or one: they take no branch (past
// the end they read the last again), so that none waits for another.
template <bool V4, bool Q>
__device__ __forceinline__ double share_sum(const Left& f, const Gone& gone, int t0, int t1) {
    constexpr int UN = 8, E = V4 ? 4 : 1;
    const int lane = threadIdx.x & 63;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    for (int b = t0; b < t1; b += UN * E * 64) {
        float x[UN][E], y[UN][E];
#pragma unroll
        for (int k = 0; k < UN; k++) {
            const int t = min(b + (k * 64 + lane) * E, t1 - E);
            if constexpr (V4) {
                const f32x4 pv = *(const f32x4*)(f.p + t);
                f32x4 qv = (f32x4){0, 0, 0, 0};
                if (Q) qv = *(const f32x4*)(f.q + t);
#pragma unroll
                for (int e = 0; e < 4; e++) x[k][e] = pv[e], y[k][e] = qv[e];
            } else {
                x[k][0] = f.p[t];
                y[k][0] = Q ? f.q[t] : 0.0f;
            }
        }
        if constexpr (!Q)
            gone.each(b, b + UN * E * 64, [&](int g) {
#pragma unroll
                for (int k = 0; k < UN; k++)
#pragma unroll
                    for (int e = 0; e < E; e++) x[k][e] = b + (k * 64 + lane) * E + e == g ? 0.0f : x[k][e];
            });
        if (b + UN * E * 64 > t1) {
#pragma unroll
            for (int k = 0; k < UN; k++)
#pragma unroll
                for (int e = 0; e < E; e++) x[k][e] = b + (k * 64 + lane) * E < t1 ? x[k][e] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < UN; k++)
#pragma unroll
            for (int e = 0; e < E; e++) s[V4 ? e : k & 3] += f.of<Q>(x[k][e], y[k][e]);
    }
    return (s[0] + s[1]) + (s[2] + s[3]);
}
template <bool V4>
__device__ double shares(const Left& f, const Gone& gone, int first, int last, double* sums) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, len = share_len<V4>(last - first);
    const int t0 = first + wave * len, t1 = min(last, t0 + len);
    double x = 0.0;
    if (t0 < t1) x = f.q ? share_sum<V4, true>(f, gone, t0, t1) : share_sum<V4, false>(f, gone, t0, t1);
    x = wave_sum(x);
    __syncthreads();  // the sums of the call before have been read
    if (lane == 0) sums[wave] = x;
    __syncthreads();
    static_assert(kVerifyWaves == 16, "a row of lanes");
    return row_sum(sums[lane & 15]);
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

// A sequence's rows as the walk needs them: each row's children, and of each row its token, its probabilities at
// its parent, its random number and whether an earlier sibling has its token.
struct Tree {
    int32_t *cstart, *clist;  // relative to the sequence
    uint32_t* tok;
    float *p, *q, *u;
    int32_t* seen;
    static constexpr int kWords = kVerifyWords;  // of a row, and one word more
    __device__ Tree(int32_t* at, int n) {
        cstart = at;
        clist = cstart + n + 1;
        tok = (uint32_t*)(clist + n);
        p = (float*)(tok + n);
        q = p + n;
        u = q + n;
        seen = (int32_t*)(u + n);
    }
};

}  // namespace

// One workgroup per sequence, as each step of a walk needs the one before. Bound by what one CU reads from L2: a sum
// over 128256 tokens of p and q takes 7 to 9 us, one for a rejection (rows stay cached between them: reading past
// the cache took 72 us for 16 trees, 47 now). One tree of given drafts over 49152 tokens takes 13 us, of which the
// sum and the draw are most; 16 trees of independent drafts over 128256 47 to 55, 4 bushy ones of draws without
// replacement 52 to 110, by where their rows lie. The walk itself reads nothing from memory: what it can ask for is
// gathered first, all rows at once, into LDS (MEM: into v.tree, where some sequence has more than kVerifyLdsRows rows).
template <bool V4, bool MEM>
__global__ __launch_bounds__(kVerifyThreads) void k_tree_verify(RowArgs a, VerifyArgs v) {
    __shared__ double sums[kVerifyWaves];
    extern __shared__ int32_t mem[];
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, V = v.vocab;
    const int row0 = a.seqs[(size_t)s * kSeqWords], n = a.seqs[(size_t)s * kSeqWords + 1];
    const Tree tr(MEM ? v.tree + (size_t)Tree::kWords * row0 + s : mem, n);
    uint32_t* out = v.out_tokens + (size_t)s * v.ld;
    int32_t* path = v.out_path + (size_t)s * v.ld;
    const int c0 = a.cstart[row0];
    for (int i = tid; i <= n; i += kVerifyThreads) tr.cstart[i] = a.cstart[row0 + i] - c0;
    for (int i = tid; i < n; i += kVerifyThreads) {
        const uint32_t t = v.tokens[row0 + i];
        const int parent = a.parent[row0 + i];  // -1 for a first or unused row
        const bool in = parent >= 0 && t < (uint32_t)V;  // a token outside the vocabulary never passes
        const size_t at = in ? (size_t)(row0 + parent) * V + t : 0;
        tr.tok[i] = t;
        tr.u[i] = v.u[row0 + i];
        tr.p[i] = in ? v.p[at] : 0.0f;
        tr.q[i] = in ? (v.kind == DRAFT_FIXED ? 1.0f : v.q[at]) : 0.0f;
        tr.seen[i] = parent;
    }
    __syncthreads();
    for (int i = tid; i < tr.cstart[n]; i += kVerifyThreads) tr.clist[i] = a.clist[c0 + i] - row0;
    __syncthreads();
    if (v.kind != DRAFT_EACH) {
        for (int i = tid; i < n; i += kVerifyThreads) {
            const int parent = tr.seen[i];
            if (parent < 0) {
                tr.seen[i] = 0;
                continue;
            }
            int seen = 0;
            for (int k = tr.cstart[parent], c; (c = tr.clist[k]) != i; k++) seen |= tr.tok[c] == tr.tok[i];
            tr.seen[i] = seen;
        }
        __syncthreads();
    }
    int node = 0, count = 1;
    bool known = false;  // sums holds the shares of what is left
    Left left{};
    Gone gone{};
    double total = 0.0;
    if (tid == 0) path[0] = 0;
    for (;;) {
        const size_t row = (size_t)(row0 + node) * V;
        left = Left{v.p + row, v.kind == DRAFT_FIXED ? nullptr : v.q + row, 0.0};
        known = false;
        double b = 1.0, d = 1.0;
        int passed = -1;
        for (int j = tr.cstart[node]; j < tr.cstart[node + 1] && passed < 0; j++) {
            const int c = tr.clist[j];
            const bool seen = v.kind != DRAFT_EACH && tr.seen[c];
            const double p = mass_of(tr.p[c]), q = mass_of(tr.q[c]), u = tr.u[c];
            double mass, rate;
            if (v.kind == DRAFT_FIXED) {
                mass = seen || !(b > 0.0) ? 0.0 : p / b;
                rate = q;
            } else {
                // without replacement: a token drawn before, or one that q had nothing left for, was not drawn
                if (v.kind == DRAFT_DISTINCT && (seen || d < kSpent || q == 0.0)) continue;
                const double r = p - left.a * q;
                rate = q / d;
                mass = (r > 0.0 ? r : 0.0) / b;
            }
            if (u * rate < mass && rate > 0.0) {
                passed = c;
            } else if (v.kind == DRAFT_FIXED) {
                if (!seen) b -= p;
            } else {
                left.a += b / d;
                if (v.kind == DRAFT_DISTINCT) d -= q;
                b = total = shares<V4>(left, gone, 0, V, sums);
                known = true;
                if (!(b > 0.0)) break;  // nothing is left: no child passes
            }
        }
        if (passed < 0) break;
        if (tid == 0) {
            out[count - 1] = tr.tok[passed];
            path[count] = passed;
        }
        node = passed;
        count++;
    }
    if (v.kind == DRAFT_FIXED && tr.cstart[node + 1] > tr.cstart[node]) {
        // the removed tokens, over the probabilities, which have been used
        __syncthreads();
        uint32_t* g = (uint32_t*)tr.p;
        gone = Gone{g, tr.cstart[node + 1] - tr.cstart[node]};
        for (int i = tid; i < gone.n; i += kVerifyThreads) g[i] = tr.tok[tr.clist[tr.cstart[node] + i]];
        __syncthreads();
    }
    if (left.a == 0.0) left.q = nullptr;  // nothing was taken from p: its row alone
    if (!known) total = shares<V4>(left, gone, 0, V, sums);
    if (!(total > 0.0)) {  // nothing is left: the target's own distribution
        left.a = 0.0;
        left.q = nullptr;
        gone.n = 0;
        total = shares<V4>(left, gone, 0, V, sums);
    }
    // the share that the target falls in, then its tokens in order, eight a thread
    double target = (double)tr.u[0] * total;
    const int len = share_len<V4>(V), first = pick(sums, target) * len, last = min(V, first + len), wave = tid >> 6;
    __shared__ int found, positive;
    if (tid == 0) {
        found = INT32_MAX;
        positive = 0;
    }
    double before = 0.0;
    for (int c0 = first; c0 < last; c0 += 8 * kVerifyThreads) {
        float px[8], qx[8];
        const int t0 = c0 + 8 * tid;
        if constexpr (V4) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int t = min(t0 + 4 * k, last - 4);
                const f32x4 x = *(const f32x4*)(left.p + t);
                f32x4 y = (f32x4){0, 0, 0, 0};
                if (left.q) y = *(const f32x4*)(left.q + t);
#pragma unroll
                for (int e = 0; e < 4; e++) px[4 * k + e] = x[e], qx[4 * k + e] = y[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int t = min(t0 + e, last - 1);
                px[e] = left.p[t];
                qx[e] = left.q ? left.q[t] : 0.0f;
            }
        }
        const int w0 = c0 + 512 * wave;
        gone.each(w0, w0 + 512, [&](int g) {
#pragma unroll
            for (int e = 0; e < 8; e++) px[e] = t0 + e == g ? 0.0f : px[e];
        });
        double w[8], mine = 0.0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const double x = left.q ? left.of<true>(px[e], qx[e]) : left.of<false>(px[e], 0.0f);
            w[e] = t0 + e < last ? x : 0.0;
            mine += w[e];
        }
        double x = mine;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const double y = __shfl_up(x, m);
            if (lane >= m) x += y;
        }
        __syncthreads();  // the sums before have been read
        if (lane == 63) sums[wave] = x;
        __syncthreads();
        double run = before;
        for (int i = 0; i < wave; i++) run += sums[i];
        run += x - mine;
        int hit = INT32_MAX, top = -1;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            run += w[e];
            if (w[e] > 0.0) {
                top = t0 + e;
                if (hit == INT32_MAX && run > target) hit = top;
            }
        }
        const uint64_t hits = __ballot(hit != INT32_MAX), tops = __ballot(top >= 0);
        if (hits && lane == __builtin_ctzll(hits)) atomicMin(&found, hit);
        if (tops && lane == 63 - __builtin_clzll(tops)) atomicMax(&positive, top);
        for (int i = 0; i < kVerifyWaves; i++) before += sums[i];
        __syncthreads();
        if (found != INT32_MAX) break;
    }
    if (tid == 0) {
        out[count - 1] = (uint32_t)(found != INT32_MAX ? found : positive);
        v.out_count[s] = count;
    }
    for (int i = count + tid; i < v.ld; i += kVerifyThreads) {
        out[i] = 0;
        path[i] = -1;
    }
}

void launch_tree_verify(hipStream_t st, const RowArgs& a, const VerifyArgs& v0) {
    if (a.n_seqs <= 0) return;
    const VerifyArgs v = v0;
    const size_t lds = (size_t)(Tree::kWords * a.most_rows + 1) * 4;
    const bool v4 = v.vocab % 4 == 0 && ((uintptr_t)v.p | (uintptr_t)v.q) % 16 == 0;
    auto go = [&](auto k, size_t bytes) {
        hipLaunchKernelGGL(k, dim3(a.n_seqs), dim3(kVerifyThreads), bytes, st, a, v);
    };
    if (a.most_rows > kVerifyLdsRows) {
        if (v4)
            go(k_tree_verify<true, true>, 0);
        else
            go(k_tree_verify<false, true>, 0);
    } else if (v4) {
        go(k_tree_verify<true, false>, lds);
    } else {
        go(k_tree_verify<false, false>, lds);
    }
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
