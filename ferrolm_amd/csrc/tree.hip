// Attention of rows over a paged cache: chains, single tokens and trees of
// drafted tokens, over f32, int8 and fp8 caches.
//
// Row i of a sequence with `pos` cached tokens before its rows attends to
// those and to its own branch: o = sum_t softmax_t(q . k_t / sqrt(HD)) v_t,
// one pass with a running reference m and sum l per query: a token's probability
// is p = 2^(score - m), its weight w = p * (its value's scale), and the output
// sum w code / sum p, from which m cancels. m rises only when a weight would
// leave f16 (kMost) or a probability grow out of bounds, so most steps compare
// and branch once where a running maximum would reduce across lanes.
//
// A wave holds up to 16 QT queries (rows x grouped heads, a slot) of one kv
// head and takes pairs of pages. Both products run transposed on f16 MFMA
// (16x16x32): scores K q^T leave a lane with one query and four tokens of each
// page, which is the operand layout of V^T p^T, so scores and probabilities
// never leave their registers, and all of a query's state sits in its lanes.
// The cache's records are in operand layout (internal.h): loads go from memory
// to registers, with no LDS and no barrier before the shares of a workgroup's
// waves meet.
//
// Precision: int8 and fp8 codes are exact in f16. Queries are scaled by a power
// of two and split into two f16, to 2^-23 of each input or 2^-31 of the
// largest; probabilities times value scales likewise. f32 keys and values are
// scaled by row and split the same way (the product of the two small parts,
// at most 2^-22, is left out). Sums are f32.
#include "devutil.h"

namespace fg {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

namespace {

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
// Below every score; its exponential is 0 against any.
constexpr float kLowest = -3e38f;
// Once references pass kFused, scores are rounded before theirs is taken from them: what a fused product keeps of
// the score would be a whole step of the reference's rounding, and the largest score is to stay its reference.
constexpr float kFused = 0x1p20f;
// A weight past kMost, or a probability past kMostP (its value may be zero), raises the reference to where the
// largest weight is 2^kTop and no probability above 2^kTopP: weights keep their bits for value scales down to
// 2^(kTop - kTopP), and 2^30 probabilities have a sum.
constexpr float kMost = 32768.0f, kMostP = 0x1p90f, kTop = 9.0f, kTopP = 80.0f;

// Eight codes, of which d0 holds the first four, in f16.
template <int FMT>
__device__ __forceinline__ f16x8 codes8(uint32_t d0, uint32_t d1) {
    uint32_t h[4];
    if constexpr (FMT == KV_INT8) {
        // 0x6400 | (code + 128) is 1152 + code as f16
        h[0] = __builtin_amdgcn_perm(0x64646464u, d0, 0x04010400u);
        h[1] = __builtin_amdgcn_perm(0x64646464u, d0, 0x04030402u);
        h[2] = __builtin_amdgcn_perm(0x64646464u, d1, 0x04010400u);
        h[3] = __builtin_amdgcn_perm(0x64646464u, d1, 0x04030402u);
        f16x8 r;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const f16x2 y = __builtin_bit_cast(f16x2, h[i]) - (f16x2){(_Float16)1152.0f, (_Float16)1152.0f};
            r[2 * i] = y[0];
            r[2 * i + 1] = y[1];
        }
        return r;
    } else {
        f16x8 r;
        const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d0, 1.0f, false),
                    b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d0, 1.0f, true),
                    c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d1, 1.0f, false),
                    d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d1, 1.0f, true);
        r[0] = a[0], r[1] = a[1], r[2] = b[0], r[3] = b[1], r[4] = c[0], r[5] = c[1], r[6] = d[0], r[7] = d[1];
        return r;
    }
}

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// x = hi + lo to 2^-23 of x, or 2^-25 where that is more (half of f16's smallest step)
__device__ __forceinline__ void split2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    hi = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x0, x1}, f16x2));
    float y0, y1;  // x - hi, the f16 operand widened by the operation itself
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(y0) : "v"(hi), "v"(x0));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(y1) : "v"(hi), "v"(x1));
    lo = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){y0, y1}, f16x2));
}
__device__ __forceinline__ void split8(const float (&x)[8], f16x8& hi, f16x8& lo) {
    u32x4 h, l;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t a, b;
        split2(x[2 * i], x[2 * i + 1], a, b);
        h[i] = a, l[i] = b;
    }
    hi = __builtin_bit_cast(f16x8, h);
    lo = __builtin_bit_cast(f16x8, l);
}

// The exponent that brings values up to m below 2^6 (the two halves then hold them to 2^-31 of m, their products
// far from f32's ends); bounded, so that 2^-e stays finite. The lowest for zeros, so that values of 0 leave the
// weights' reference to others.
__device__ __forceinline__ int split_exp(float m) {
    int e = -100;
    if (m > 0.0f && m < INFINITY) frexpf(m, &e);
    return max(e, -100) - 6;
}

// What a lane takes of a page: the key of token lane % 16 at channels (lane / 16) HD / 4 .., and the values of
// tokens 4 (lane / 16) .. +3 at channels (lane % 16) HD / 16 .., each with the scales of those four tokens.
template <int HD, int FMT>
struct Half {  // 8-bit formats: the codes
    static constexpr int KD = HD / 16;
    uint32_t d[KD];
    float4 s;
    __device__ __forceinline__ void load(const uint8_t* p, const uint8_t* scales) {
        if constexpr (KD == 1) {
            d[0] = *(const uint32_t*)p;
        } else if constexpr (KD == 2) {
            const u32x2 x = *(const u32x2*)p;
            d[0] = x[0], d[1] = x[1];
        } else {
#pragma unroll
            for (int i = 0; i < KD / 4; i++) {
                const u32x4 x = *(const u32x4*)(p + 16 * i);
#pragma unroll
                for (int e = 0; e < 4; e++) d[4 * i + e] = x[e];
            }
        }
        s = *(const float4*)scales;
    }
};
template <int HD, int FMT>
struct KeyPage : Half<HD, FMT> {
    __device__ __forceinline__ void load(const KvLayer& kv, size_t block, int h, int lane) {
        const uint8_t* rec = kv.data + (block * kv.nkv + h) * kv_record(HD);
        Half<HD, FMT>::load(rec + (lane & 15) * HD + (lane >> 4) * (HD / 4), rec + 32 * HD + (lane >> 4) * 16);
    }
};
template <int HD, int FMT>
struct ValuePage : Half<HD, FMT> {
    __device__ __forceinline__ void load(const KvLayer& kv, size_t block, int h, int lane) {
        const uint8_t* rec = kv.data + (block * kv.nkv + h) * kv_record(HD) + 16 * HD;
        Half<HD, FMT>::load(rec + (lane >> 4) * (4 * HD) + (lane & 15) * (HD / 4), rec + 16 * HD + 64 + (lane >> 4) * 16);
    }
};
template <int HD>
struct KeyPage<HD, KV_F32> {
    float d[HD / 4];
    __device__ __forceinline__ void load(const KvLayer& kv, size_t block, int h, int lane) {
        const float* p = kv.k + (block * kv.nkv + h) * 16 * HD + (lane & 15) * HD + (lane >> 4) * (HD / 4);
#pragma unroll
        for (int i = 0; i < HD / 4; i += 4) {
            const float4 x = *(const float4*)(p + i);
            d[i] = x.x, d[i + 1] = x.y, d[i + 2] = x.z, d[i + 3] = x.w;
        }
    }
};
template <int HD>
struct ValuePage<HD, KV_F32> {
    static constexpr int C = HD / 16;  // channels of each of the four tokens
    float d[4][C];
    __device__ __forceinline__ void load(const KvLayer& kv, size_t block, int h, int lane) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const float* p = kv.v + ((block * kv.nkv + h) * 16 + 4 * (lane >> 4) + t) * HD + (lane & 15) * C;
            if constexpr (C >= 4) {
#pragma unroll
                for (int i = 0; i < C; i += 4) {
                    const float4 x = *(const float4*)(p + i);
                    d[t][i] = x.x, d[t][i + 1] = x.y, d[t][i + 2] = x.z, d[t][i + 3] = x.w;
                }
            } else if constexpr (C == 2) {
                const float2 x = *(const float2*)p;
                d[t][0] = x.x, d[t][1] = x.y;
            } else {
                d[t][0] = *p;
            }
        }
    }
};

// A page's keys as MFMA operands, by steps of 32 channels (lo for f32 caches only), and the scales of the lane's
// four tokens.
template <int HD, int FMT>
struct Keys {
    static constexpr int NS = HD >= 32 ? HD / 32 : 1;
    f16x8 hi[NS], lo[FMT == KV_F32 ? NS : 1];
    float s[4];
    __device__ __forceinline__ explicit Keys(const KeyPage<HD, FMT>& p, int lane) {
        if constexpr (FMT == KV_F32) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < HD / 4; i++) m = fmaxf(m, fabsf(p.d[i]) <= 3.4e38f ? fabsf(p.d[i]) : INFINITY);
            m = reduce_rows<true, true>(m);
            const bool fine = m < INFINITY;
            const int e = split_exp(m);
            const float f = ldexpf(1.0f, -e);
            const float sc = fine ? ldexpf(1.0f, e) : NAN;  // of key lane % 16
#pragma unroll
            for (int j = 0; j < NS; j++) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = 8 * j + i < HD / 4 && fine ? p.d[(8 * j + i) % (HD / 4)] * f : 0.0f;
                split8(x, hi[j], lo[j]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) s[i] = __shfl(sc, 4 * (lane >> 4) + i);
        } else {
#pragma unroll
            for (int j = 0; j < NS; j++)
                hi[j] = codes8<FMT>(p.d[(2 * j) % (HD / 16)], HD >= 32 ? p.d[(2 * j + 1) % (HD / 16)] : 0u);
            if constexpr (HD == 16) {  // only four channels a lane: the operand's other half is zero
#pragma unroll
                for (int i = 4; i < 8; i++) hi[0][i] = (_Float16)0.0f;
            }
            s[0] = p.s.x, s[1] = p.s.y, s[2] = p.s.z, s[3] = p.s.w;
        }
    }
};

// Scales of the lane's four values of a page, and for f32 the factors to split them by (0: not finite).
template <int HD, int FMT>
__device__ __forceinline__ void value_scales(const ValuePage<HD, FMT>& p, float* s, float* f) {
    if constexpr (FMT == KV_F32) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < HD / 16; i++) m = fmaxf(m, fabsf(p.d[t][i]) <= 3.4e38f ? fabsf(p.d[t][i]) : INFINITY);
            m = group_reduce<16, true>(m);
            const int e = split_exp(m);
            s[t] = m < INFINITY ? ldexpf(1.0f, e) : NAN;
            f[t] = m < INFINITY ? ldexpf(1.0f, -e) : 0.0f;
        }
    } else {
        s[0] = p.s.x, s[1] = p.s.y, s[2] = p.s.z, s[3] = p.s.w;
    }
}

// An item's geometry, the same for all of its waves.
struct Item {
    int seq0, n, pos, btab, mask0, mpages;  // the sequence's record
    int row0, page0, page1, wi, wi_step, slots, alone, next;  // next: the workgroup's next item, or -1
    bool chain;
    __device__ __forceinline__ bool read(const RowArgs& a, int item) {
        // scalar loads, also behind the stores of the item before
        typedef int words __attribute__((ext_vector_type(16)));
        const words w = *(const __attribute__((address_space(4))) words*)(uintptr_t)(a.items + (size_t)item * kItemWords);
        if (w[0] < 0) return false;  // an unused item of the launch's capacity
        row0 = w[1], page0 = w[2], page1 = w[3], wi = w[4], wi_step = w[5], slots = w[6], alone = w[7];
        seq0 = w[8], n = w[9], pos = w[10], btab = w[11], mask0 = w[12], mpages = w[13], next = w[14];
        chain = mask0 < 0;
        return true;
    }
};

// A wave's slot: 16 QT queries of one kv head, and what they have gathered.
template <int HD, int FMT, int QT>
struct Slot {
    static constexpr int KD = HD / 16, NS = Keys<HD, FMT>::NS, QM = HD >= 64 ? 32 : 64;
    static constexpr int ND = 4 * KD + 2;  // dwords a lane keeps of a tile
    static constexpr bool F32 = FMT == KV_F32;
    f16x8 qh[QT][NS], ql[QT][NS];
    float qf[QT], mq[QT], l[QT];  // score factor (log 2 units), reference, sum of probabilities
    int qrow[QT];                 // the query's row in its sequence
    f32x4 o[QT][KD];
    int h, G, r0, nr, last, full;  // first row and rows; pages that they see; tokens that all of them see
    bool on;

    __device__ __forceinline__ void place(const TreeAttn& t, const Item& it, int nkv, int head, int slot) {
        h = head;
        G = t.nh / nkv;
        r0 = it.row0 + slot * (QM / G);
        nr = min(QM / G, it.n - r0);
        on = slot < it.slots && nr > 0;
        last = it.chain ? min(it.page1, (it.pos + r0 + nr + 15) / 16) : it.page1;
        full = it.chain ? it.pos + r0 + 1 : it.pos;
#pragma unroll
        for (int i = 0; i < QT; i++) {
            mq[i] = kLowest;
            l[i] = 0.0f;
            qf[i] = 1.0f;
            qrow[i] = 0;
#pragma unroll
            for (int j = 0; j < KD; j++) o[i][j] = (f32x4){0, 0, 0, 0};
        }
    }

    __device__ __forceinline__ void queries(const RowArgs& a, const TreeAttn& t, const Item& it, int lane) {
        if (!on) return;
        const int r = lane & 15, g = lane >> 4, Q = nr * G;
#pragma unroll
        for (int i = 0; i < QT; i++) {
            const int qi = min(16 * i + r, Q - 1);  // lanes past the last query hold it again
            qrow[i] = r0 + qi / G;
            const int64_t row = it.seq0 + qrow[i];
            const float* qp = t.q + row * t.ldq + (h * G + qi % G) * HD;
            float x[HD / 4];
#pragma unroll
            for (int e = 0; e < HD / 4; e += 4) {
                const float4 w = *(const float4*)(qp + g * (HD / 4) + e);
                x[e] = w.x, x[e + 1] = w.y, x[e + 2] = w.z, x[e + 3] = w.w;
            }
            if (t.cos_t) {  // rotate-half, src/model.rs:451-459
                const float* cp = t.cos_t + (size_t)a.rpos[row] * (HD / 2) + (g & 1) * (HD / 4);
                const float* sp = t.sin_t + (size_t)a.rpos[row] * (HD / 2) + (g & 1) * (HD / 4);
#pragma unroll
                for (int e = 0; e < HD / 4; e++) {
                    const float y = qp[(g ^ 2) * (HD / 4) + e];
                    x[e] = __fadd_rn(__fmul_rn(x[e], cp[e]), __fmul_rn(g < 2 ? -y : y, sp[e]));
                }
            }
            float m = 0.0f;
#pragma unroll
            for (int e = 0; e < HD / 4; e++) m = fmaxf(m, fabsf(x[e]) <= 3.4e38f ? fabsf(x[e]) : INFINITY);
            m = reduce_rows<true, true>(m);
            const int ex = split_exp(m);
            const float f = m < INFINITY ? ldexpf(1.0f, -ex) : NAN;
            qf[i] = ldexpf(t.scale * kLog2e, ex);
#pragma unroll
            for (int s = 0; s < NS; s++) {
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = 8 * s + e < HD / 4 ? x[(8 * s + e) % (HD / 4)] * f : 0.0f;
                split8(y, qh[i][s], ql[i][s]);
            }
        }
    }

    // Scores of a pair of pages: raw[tile][page x 4 tokens], to be multiplied by qf. Products into one sum stand
    // apart, by the pages' and tiles' others.
    __device__ __forceinline__ void scores(const KeyPage<HD, FMT> (&kp)[2], float (&raw)[QT][8], int lane) const {
        const Keys<HD, FMT> k[2] = {Keys<HD, FMT>(kp[0], lane), Keys<HD, FMT>(kp[1], lane)};
        f32x4 acc[2][QT];
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int i = 0; i < QT; i++) acc[x][i] = (f32x4){0, 0, 0, 0};
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int s = 0; s < NS; s++) {
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int i = 0; i < QT; i++) acc[x][i] = mfma(k[x].hi[s], ql[i][s], acc[x][i]);
            if constexpr (F32) {
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int i = 0; i < QT; i++) acc[x][i] = mfma(k[x].lo[s], qh[i][s], acc[x][i]);
            }
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int i = 0; i < QT; i++) acc[x][i] = mfma(k[x].hi[s], qh[i][s], acc[x][i]);
        }
        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int i = 0; i < QT; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) raw[i][4 * x + e] = acc[x][i][e] * k[x].s[e];
    }

    // Whether some query does not see all of a pair of pages.
    __device__ __forceinline__ bool masked(int p0) const { return 16 * (p0 + 2) > full || p0 + 1 >= last; }

    // Scores of tokens that tile i's query does not see: -infinity.
    __device__ __forceinline__ void mask(const RowArgs& a, const Item& it, int p0, int i, float (&raw)[8], int lane) const {
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const int page = p0 + x, at = 16 * page + 4 * (lane >> 4), end = it.pos + qrow[i];  // end: a chain row's last
            uint32_t sees = page < last ? 15u : 0u;
            if (it.chain)
                sees &= at > end ? 0u : 15u >> max(0, 3 - (end - at));
            else if (page >= it.pos / 16 && page < last)
                sees &= (uint32_t)a.masks[it.mask0 + (size_t)qrow[i] * it.mpages + (page - it.pos / 16)] >> (lane >> 4 << 2);
#pragma unroll
            for (int e = 0; e < 4; e++) raw[4 * x + e] = sees >> e & 1 ? raw[4 * x + e] : -INFINITY;
        }
    }

    // The pair p0's weights, in two f16 each, from its scores and value scales; the reference and sums follow.
    __device__ __forceinline__ void weights(const RowArgs& a, const Item& it, int p0, float (&raw)[QT][8],
                                            const float (&vsc)[8], f16x8 (&hi)[QT], f16x8 (&lo)[QT], int lane) {
        const bool part = masked(p0);
#pragma unroll
        for (int i = 0; i < QT; i++) {
            float p[8], w[8];
            // true in a lane whose weights or probabilities are out of bounds; fused: the score's product is not
            // rounded before the reference, which was, is taken from it
            auto weigh = [&](bool fused) {
                float wm = 0.0f, pm = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    p[e] = __builtin_amdgcn_exp2f(fused ? fmaf(raw[i][e], qf[i], -mq[i])
                                                        : __fadd_rn(__fmul_rn(raw[i][e], qf[i]), -mq[i]));
                    w[e] = p[e] * vsc[e];
                    wm = fmaxf(wm, w[e]);
                    pm = fmaxf(pm, p[e]);
                }
                return wm > kMost || pm > kMostP;
            };
            if (part || __any(weigh(true))) {
                if (part) mask(a, it, p0, i, raw[i], lane);
                if (__any(weigh(false))) {
                    float top = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float sc = __fmul_rn(raw[i][e], qf[i]);
                        top = fmaxf(top, fmaxf(sc + __builtin_amdgcn_logf(vsc[e]) - kTop, sc - kTopP));
                    }
                    const float mn = fmaxf(mq[i], reduce_rows<true, true>(top)), f = __builtin_amdgcn_exp2f(mq[i] - mn);
                    l[i] *= f;
#pragma unroll
                    for (int j = 0; j < KD; j++) o[i][j] *= f;
                    mq[i] = mn;
                    if (__any(fabsf(mn) > kFused)) full = INT_MIN;  // every pair this way from now on
                    (void)weigh(false);
                }
                // a value that is not finite has a NaN scale, which must not reach the rows that don't see it
#pragma unroll
                for (int e = 0; e < 8; e++) w[e] = p[e] == 0.0f ? 0.0f : w[e];
            }
            split8(w, hi[i], lo[i]);
            l[i] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        }
    }

    // Adds a pair's weighted values; vf: value_scales' factors.
    __device__ __forceinline__ void gather(const f16x8 (&hi)[QT], const f16x8 (&lo)[QT], const ValuePage<HD, FMT> (&vp)[2],
                                           const float (&vf)[8]) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int j = 0; j < KD; j++) {
            f16x8 vh, vl;
            if constexpr (F32) {
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = vf[e] == 0.0f ? 0.0f : vp[e / 4].d[e % 4][j] * vf[e];
                split8(y, vh, vl);
            } else {
                vh = codes8<FMT>(vp[0].d[j], vp[1].d[j]);
            }
#pragma unroll
            for (int i = 0; i < QT; i++) {
                o[i][j] = mfma(vh, lo[i], o[i][j]);
                if constexpr (F32) o[i][j] = mfma(vl, hi[i], o[i][j]);
                o[i][j] = mfma(vh, hi[i], o[i][j]);
            }
        }
        __builtin_amdgcn_s_setprio(0);
    }

    // The sums of the pw position shares into share 0's, halving; a tile at a time, for the LDS that takes. Every
    // wave of the workgroup calls it; sh: pw / 2 * rw * ND * 64 floats.
    __device__ __forceinline__ void join(float* sh, int slot, int share, int rw, int pw, int lane) {
#pragma unroll
        for (int i = 0; i < QT; i++) l[i] = reduce_rows<false, true>(l[i]);
        for (int half = pw / 2; half > 0; half >>= 1) {
            float* x = sh + ((size_t)(share % half * rw + slot) * ND) * 64 + lane;
#pragma unroll
            for (int i = 0; i < QT; i++) {
                if (on && share >= half && share < 2 * half) {
                    x[0] = mq[i];
                    x[64] = l[i];
#pragma unroll
                    for (int j = 0; j < KD; j++)
#pragma unroll
                        for (int e = 0; e < 4; e++) x[(2 + 4 * j + e) * 64] = o[i][j][e];
                }
                __syncthreads();
                if (on && share < half) {
                    const float m2 = x[0], mn = fmaxf(mq[i], m2);
                    const float f1 = __builtin_amdgcn_exp2f(mq[i] - mn), f2 = __builtin_amdgcn_exp2f(m2 - mn);
                    l[i] = l[i] * f1 + x[64] * f2;
#pragma unroll
                    for (int j = 0; j < KD; j++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[i][j][e] = o[i][j][e] * f1 + x[(2 + 4 * j + e) * 64] * f2;
                    mq[i] = mn;
                }
                __syncthreads();
            }
        }
    }

    // Share 0: the outputs of rows that no other item has, partials of the others'.
    __device__ __forceinline__ void finish(const RowArgs& a, const TreeAttn& t, const Item& it, int nkv, int slot,
                                           int lane) {
        const int r = lane & 15, g = lane >> 4;
#pragma unroll
        for (int i = 0; i < QT; i++) {
            const int qi = 16 * i + r;
            if (qi >= nr * G) continue;
            float* dst;
            float f = 1.0f;
            if (t.out && it.alone) {
                // zeros where a row attends to nothing
                const bool none = l[i] == 0.0f || a.mrec[(size_t)(it.seq0 + qrow[i]) * 4 + 3];
                f = none ? 0.0f : 1.0f / l[i];
                if (none) {
#pragma unroll
                    for (int j = 0; j < KD; j++) o[i][j] = (f32x4){0, 0, 0, 0};
                }
                dst = t.out + (size_t)(it.seq0 + qrow[i]) * t.ldo + (size_t)(h * G + qi % G) * HD;
            } else {
                float* part = t.part + (((size_t)(it.wi + slot * it.wi_step) * nkv + h) * QM + qi) * (HD + 4);
                if (g == 0) {
                    part[0] = l[i] == 0.0f ? -INFINITY : t.out ? mq[i] : mq[i] * kLn2;
                    part[1] = l[i];
                }
                dst = part + 4;
            }
            dst += g * (HD / 4);
#pragma unroll
            for (int w = 0; w < KD; w++) {  // channel 4 w + e of the lane's: tile (4 w + e) % KD, register (4 w + e) / KD
                f32x4 y;
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = o[i][(4 * w + e) % KD][(4 * w + e) / KD] * f;
                *(f32x4*)(dst + 4 * w) = y;
            }
        }
    }
};

}  // namespace

// One workgroup per (kv head, first item of a list): rw row slots x pw position
// shares, a wave each, which takes its pages from memory straight to registers;
// the shares' sums meet in LDS. For one slot of rows, where no page is wanted
// twice, for f32 caches, and for heads of 16 and 32 channels. One token over
// 1030 cached int8 ones, 32 heads of 64: 7 us, nearly all of it latency (the
// item, its block ids, pages, the join, one after the other); a tree of 21 rows
// over as much in f32 14 us.
template <int HD, int FMT, int QT>
__global__ __launch_bounds__(512) void k_tree_attn(RowArgs a, KvLayer kv, TreeAttn t) {
    extern __shared__ float sh[];
    Item it;
    for (int item = blockIdx.x / kv.nkv; item >= 0; item = it.next) {
        if (!it.read(a, item)) return;
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));  // an item's addresses are not kept over the others
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // what depends on it stays scalar
        const int slot = wave % a.rw, share = wave / a.rw;
        Slot<HD, FMT, QT> s;
        s.place(t, it, kv.nkv, blockIdx.x % kv.nkv, slot);
        const int pairs = (s.last - it.page0 + 1) / 2, mine = s.on ? (pairs - share + a.pw - 1) / a.pw : 0;
        int ids = 0;  // a chunk's block ids, two pages a pair; past the last page the last again
        auto chunk = [&](int c0) {
            const int pg = it.page0 + 2 * (share + a.pw * (c0 + lane / 2)) + (lane & 1);
            ids = a.btab[it.btab + max(min(pg, s.last - 1), 0)];
        };
        auto block = [&](int c, int x) { return (size_t)(uint32_t)__builtin_amdgcn_readlane(ids, 2 * c + x); };
        // AHEAD: keys and values are asked for as soon as the registers of the pair before are free, the keys behind
        // the scores, the values behind the weighted sum. Otherwise the registers do not hold both: the values take
        // the keys' behind the scores. The first ones go out before the queries are read.
        constexpr bool AHEAD = HD < 128 || (QT == 1 && FMT != KV_F32);
        KeyPage<HD, FMT> kp[2];
        ValuePage<HD, FMT> vp[2];
        auto first = [&](int c0) {
            if (c0 >= mine) return;
            chunk(c0);
            if constexpr (AHEAD) {
#pragma unroll
                for (int x = 0; x < 2; x++) kp[x].load(kv, block(0, x), s.h, lane);
#pragma unroll
                for (int x = 0; x < 2; x++) vp[x].load(kv, block(0, x), s.h, lane);
            }
        };
        first(0);
        s.queries(a, t, it, lane);
        for (int c0 = 0; c0 < mine; c0 += 32) {
            const int np = min(32, mine - c0);
            if (c0) first(c0);
            for (int c = 0; c < np; c++) {
                const int next = min(c + 1, np - 1);
                float raw[QT][8], vsc[8], vf[8];
                if constexpr (!AHEAD)
#pragma unroll
                    for (int x = 0; x < 2; x++) kp[x].load(kv, block(c, x), s.h, lane);
                s.scores(kp, raw, lane);
#pragma unroll
                for (int x = 0; x < 2; x++)
                    if constexpr (AHEAD)
                        kp[x].load(kv, block(next, x), s.h, lane);
                    else
                        vp[x].load(kv, block(c, x), s.h, lane);
#pragma unroll
                for (int x = 0; x < 2; x++) value_scales<HD, FMT>(vp[x], &vsc[4 * x], &vf[4 * x]);
                f16x8 hi[QT], lo[QT];
                s.weights(a, it, it.page0 + 2 * (share + a.pw * (c0 + c)), raw, vsc, hi, lo, lane);
                s.gather(hi, lo, vp, vf);
                if constexpr (AHEAD)
#pragma unroll
                    for (int x = 0; x < 2; x++) vp[x].load(kv, block(next, x), s.h, lane);
            }
        }
        s.join(sh, slot, share, a.rw, a.pw, lane);
        if (s.on && share == 0) s.finish(a, t, it, kv.nkv, slot, lane);
    }
}

// The same for sequences of several slots over 8-bit caches: the slots' waves
// take each page once, through LDS. A ring of stages (a pair of pages for every
// position share) is filled by copies from memory straight to LDS, three stages ahead, so
// that enough bytes are on their way to cover the latency of memory: with every
// wave loading for itself a CU asks for the same 17 KB four times (270 us for
// the case below). 16-byte chunks lie in LDS by (chunk, row) so that 16 lanes
// read 256 consecutive bytes: no bank conflicts counted.
// A tree of 29 rows over 131069 fp8 tokens, 8 heads of 128 shared by four: 151
// us with the merge, 413 TFLOP/s, twice that in matrix work as each product takes
// two halves. Matrix instructions take 39% of the cycles and vector ones 49%, and
// with two waves on a SIMD they add up: without the scores the same takes 105
// us, without the values' product 121, without the weights 121, without the
// copies 127. Counters in LDS in place of the barriers took 158 against 148.
template <int HD, int FMT, int RW>
__global__ __launch_bounds__(512) void k_tree_attn_lds(RowArgs a, KvLayer kv, TreeAttn t) {
    constexpr int QT = 2, PW = RW == 2 ? 4 : 2, W = RW * PW, CPR = HD / 64;  // CPR: 16-byte chunks a lane takes of a page
    constexpr int SP = RW == 2 ? 1 : 2, PPS = 2 * SP * PW;  // pairs a share takes of a stage; pages of a stage
    constexpr int REC = 32 * HD + 128, STAGE = PPS * REC, NST = 4;
    constexpr int COPIES = (PPS * 2 * CPR + W - 1) / W;  // 1 KB copies a wave makes of a stage's codes
    constexpr int SCOPIES = (PPS + W - 1) / W;             // and copies of a page's scales
    constexpr int JOIN = PW / 2 * RW * Slot<HD, FMT, QT>::ND * 64 * 4;
    static_assert(HD == 64 || HD == 128, "whole chunks");
    static_assert(W <= 8 && NST * STAGE + 4 * kPartPages <= 160 * 1024 && JOIN <= NST * STAGE, "a CU's LDS");
    __shared__ __align__(1024) uint8_t ring[NST * STAGE];
    __shared__ int32_t ids[kPartPages];
    Item it;
    for (int item = blockIdx.x / kv.nkv; item >= 0; item = it.next) {
        if (!it.read(a, item)) return;
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));  // as above
        const int r = lane & 15, g = lane >> 4;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int slot = wave % RW, share = wave / RW;
        const int pages = it.page1 - it.page0, stages = (pages + PPS - 1) / PPS;
        for (int i = threadIdx.x; i < pages; i += 64 * W) ids[i] = a.btab[it.btab + it.page0 + i];
        Slot<HD, FMT, QT> s;
        s.place(t, it, kv.nkv, blockIdx.x % kv.nkv, slot);
        __syncthreads();
        // the wave's copies of a stage: codes copy i of page `page`, from byte `off` of its record to byte `to` of the
        // stage; more copies than there are repeat the last
        uint32_t off[COPIES];
        int page[COPIES], to[COPIES];
#pragma unroll
        for (int i = 0; i < COPIES; i++) {
            const int q = min(wave + W * i, PPS * 2 * CPR - 1), part = q % (2 * CPR), c = (part % CPR * 64 + lane) / 16;
            page[i] = q / (2 * CPR);
            to[i] = page[i] * REC + part * 1024;
            off[i] = part < CPR ? r * HD + c * 16 : 16 * HD + c / CPR * (4 * HD) + r * (HD / 4) + c % CPR * 16;
        }
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)ring;
        int held = 0, first = -64;  // a lane's block id, of 64 pages from `first` on
        auto copy = [&](int stage) {
            const uint32_t at = lds0 + stage % NST * STAGE;
            const int p0 = stage * PPS;
            if (p0 >= first + 64) {
                first = p0;
                held = ids[min(p0 + lane, pages - 1)];  // past the last page the last again
            }
            auto record = [&](int pg) {
                const uint32_t id = (uint32_t)__builtin_amdgcn_readlane(held, p0 - first + pg);
                return kv.data + ((size_t)id * kv.nkv + s.h) * REC;
            };
#pragma unroll
            for (int i = 0; i < COPIES; i++) copy_to_lds(at + to[i], record(page[i]), off[i]);
#pragma unroll
            for (int i = 0; i < SCOPIES; i++) {
                const int pg = (wave + W * i) % PPS;
                if (lane < 8) copy_to_lds(at + pg * REC + 32 * HD, record(pg) + 32 * HD, 16 * lane);
            }
        };
        // a pair's record in the ring: pair u of the share's
        auto pair = [&](int u) { return ring + u / SP % NST * STAGE + ((u % SP * PW + share) * 2) * REC; };
        auto keys = [&](int u, KeyPage<HD, FMT> (&k)[2]) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const uint8_t* base = pair(u) + x * REC;
#pragma unroll
                for (int j = 0; j < CPR; j++) {
                    const u32x4 y = *(const u32x4*)(base + ((g * CPR + j) * 16 + r) * 16);
#pragma unroll
                    for (int e = 0; e < 4; e++) k[x].d[4 * j + e] = y[e];
                }
                k[x].s = *(const float4*)(base + 32 * HD + 16 * g);
            }
        };
        auto values = [&](int u, ValuePage<HD, FMT> (&v)[2], float (&sc)[8]) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const uint8_t* base = pair(u) + x * REC;
                const float4 z = *(const float4*)(base + 32 * HD + 64 + 16 * g);
                sc[4 * x] = z.x, sc[4 * x + 1] = z.y, sc[4 * x + 2] = z.z, sc[4 * x + 3] = z.w;
#pragma unroll
                for (int j = 0; j < CPR; j++) {
                    const u32x4 y = *(const u32x4*)(base + 16 * HD + ((g * CPR + j) * 16 + r) * 16);
#pragma unroll
                    for (int e = 0; e < 4; e++) v[x].d[4 * j + e] = y[e];
                }
            }
        };
        for (int i = 0; i < NST - 1; i++) copy(i);
        s.queries(a, t, it, lane);
        // This wave's copies of all stages but the last `left` have landed, then everyone's.
#define LANDED(left)                                                                               \
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((left) * (COPIES + SCOPIES)) : "memory");              \
        __builtin_amdgcn_s_barrier();                                                                  \
        asm volatile("" ::: "memory")
        KeyPage<HD, FMT> kp[2];
        LANDED(NST - 2);
        keys(0, kp);
        for (int st = 0; st < stages; st++) {
            // the next stage is there too, for the keys that are read ahead, and everyone is past the stage before
            LANDED(NST - 3);
            const float none[8] = {};
#pragma unroll
            for (int i = 0; i < SP; i++) {
                const int u = st * SP + i, p0 = it.page0 + st * PPS + 2 * (i * PW + share);
                const bool mine = s.on && p0 < s.last;
                float raw[QT][8], vsc[8];
                ValuePage<HD, FMT> vp[2];
                f16x8 hi[QT], lo[QT];
                if (mine) s.scores(kp, raw, lane);
                if (i == 0) copy(st + NST - 1);  // over the stage before, its scalar work behind the products
                if (!mine) continue;
                values(u, vp, vsc);  // on their way behind the weights
                s.weights(a, it, p0, raw, vsc, hi, lo, lane);
                keys(u + 1, kp);  // behind the values' products
                s.gather(hi, lo, vp, none);
            }
        }
#undef LANDED
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy is left on its way when the ring is reused, or given up
        __syncthreads();
        s.join((float*)ring, slot, share, RW, PW, lane);
        if (s.on && share == 0) s.finish(a, t, it, kv.nkv, slot, lane);
    }
}

// The parts of each (row, query head), 4 channels a thread. Up to kFewParts: all of them asked for at once, 256
// threads for as many pairs as they hold. 3 us for a row, 6 us for 352 rows of 32 heads.
constexpr int kFewParts = 8;
template <int HD>
__global__ __launch_bounds__(256) void k_tree_merge_few(RowArgs a, TreeAttn t, int nkv) {
    constexpr int T = HD / 4, QM = HD >= 64 ? 32 : 64;
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) / T;
    const int d = threadIdx.x % T, G = t.nh / nkv, row = (int)(at / t.nh), hq = (int)(at % t.nh);
    if (row >= a.rows) return;
    const int4 mr = *(const int4*)(a.mrec + (size_t)row * 4);
    if (mr.z == 1) return;  // written by the attention
    const size_t stride = (size_t)nkv * QM * (HD + 4);
    const float* base = t.part + (((size_t)mr.y * nkv + hq / G) * QM + mr.x + hq % G) * (HD + 4);
    float2 st[kFewParts];
    float4 v[kFewParts];
#pragma unroll
    for (int s = 0; s < kFewParts; s++) {
        const float* p = base + min(s, mr.z - 1) * stride;
        st[s] = *(const float2*)p;
        v[s] = *(const float4*)(p + 4 + 4 * d);
    }
    float m = kLowest, l = 0.0f;
#pragma unroll
    for (int s = 0; s < kFewParts; s++) {
        if (s >= mr.z || st[s].x == -INFINITY) st[s] = make_float2(-INFINITY, 0.0f);
        m = fmaxf(m, st[s].x);
    }
    float4 y = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int s = 0; s < kFewParts; s++) {
        const float f = __builtin_amdgcn_exp2f(st[s].x - m);
        if (s >= mr.z) continue;
        l += st[s].y * f;
        y.x += v[s].x * f;
        y.y += v[s].y * f;
        y.z += v[s].z * f;
        y.w += v[s].w * f;
    }
    const float f = 1.0f / l;
    y = l == 0.0f || mr.w ? make_float4(0, 0, 0, 0) : make_float4(y.x * f, y.y * f, y.z * f, y.w * f);
    *(float4*)(t.out + (size_t)row * t.ldo + (size_t)hq * HD + 4 * d) = y;
}

// More: one workgroup per pair, the parts dealt over its threads. Tens of parts of 29 rows x 32 heads: 7 us.
template <int HD>
__global__ __launch_bounds__(256) void k_tree_merge(RowArgs a, TreeAttn t, int nkv) {
    constexpr int T = HD / 4, NP = 256 / T, QM = HD >= 64 ? 32 : 64;
    __shared__ float4 so[NP][T];
    __shared__ float sm[NP], sl[NP];
    const int row = blockIdx.x, hq = blockIdx.y, G = t.nh / nkv, h = hq / G;
    const int4 mr = *(const int4*)(a.mrec + (size_t)row * 4);
    if (mr.z == 1) return;  // written by the attention
    const int d = threadIdx.x % T, w = threadIdx.x / T;
    const size_t stride = (size_t)nkv * QM * (HD + 4);
    const float* base = t.part + (((size_t)mr.y * nkv + h) * QM + mr.x + hq % G) * (HD + 4);
    float m = kLowest, l = 0.0f;
    float4 o = make_float4(0, 0, 0, 0);
    for (int s = w; s < mr.z; s += NP) {
        const float* p = base + s * stride;
        const float2 st = *(const float2*)p;
        const float4 v = *(const float4*)(p + 4 + 4 * d);
        if (st.x == -INFINITY) continue;
        const float mn = fmaxf(m, st.x), f1 = __builtin_amdgcn_exp2f(m - mn), f2 = __builtin_amdgcn_exp2f(st.x - mn);
        l = l * f1 + st.y * f2;
        o.x = o.x * f1 + v.x * f2;
        o.y = o.y * f1 + v.y * f2;
        o.z = o.z * f1 + v.z * f2;
        o.w = o.w * f1 + v.w * f2;
        m = mn;
    }
    so[w][d] = o;
    if (d == 0) {
        sm[w] = m;
        sl[w] = l;
    }
    __syncthreads();
    if (w > 0) return;
    const int np = min(NP, mr.z);
    float M = kLowest, L = 0.0f;
    for (int i = 0; i < np; i++) M = fmaxf(M, sm[i]);
    float4 y = make_float4(0, 0, 0, 0);
    for (int i = 0; i < np; i++) {
        const float f = __builtin_amdgcn_exp2f(sm[i] - M);
        const float4 v = so[i][d];
        L += sl[i] * f;
        y.x += v.x * f;
        y.y += v.y * f;
        y.z += v.z * f;
        y.w += v.w * f;
    }
    const bool none = L == 0.0f || mr.w;
    const float f = 1.0f / L;
    y = none ? make_float4(0, 0, 0, 0) : make_float4(y.x * f, y.y * f, y.z * f, y.w * f);
    *(float4*)(t.out + (size_t)row * t.ldo + (size_t)hq * HD + 4 * d) = y;
}

template <int HD, int FMT>
static void tree_qt(hipStream_t st, const RowArgs& a, const KvLayer& kv, const TreeAttn& t) {
    const dim3 grid((unsigned)kv.nkv * a.n_items), block(64 * a.rw * a.pw);
    constexpr int QT = HD >= 64 ? 2 : 4;
    if constexpr (HD >= 64 && FMT != KV_F32) {
        // several slots, which then hold more than 16 queries each
        if (a.rw > 1) {
            if (a.rw == 2)
                hipLaunchKernelGGL((k_tree_attn_lds<HD, FMT, 2>), grid, block, 0, st, a, kv, t);
            else if (a.rw == 3)
                hipLaunchKernelGGL((k_tree_attn_lds<HD, FMT, 3>), grid, block, 0, st, a, kv, t);
            else
                hipLaunchKernelGGL((k_tree_attn_lds<HD, FMT, 4>), grid, block, 0, st, a, kv, t);
            return;
        }
    }
    const size_t join = (size_t)64 * 4 * Slot<HD, FMT, QT>::ND * (a.pw / 2) * a.rw;
    if (a.qt == 1)
        hipLaunchKernelGGL((k_tree_attn<HD, FMT, 1>), grid, block, join, st, a, kv, t);
    else
        hipLaunchKernelGGL((k_tree_attn<HD, FMT, QT>), grid, block, join, st, a, kv, t);
}

template <int HD>
static void tree_hd(hipStream_t st, const RowArgs& a, const KvLayer& kv, const TreeAttn& t) {
    if (kv.format == KV_F32)
        tree_qt<HD, KV_F32>(st, a, kv, t);
    else if (kv.format == KV_INT8)
        tree_qt<HD, KV_INT8>(st, a, kv, t);
    else
        tree_qt<HD, KV_FP8>(st, a, kv, t);
    if (!t.out || a.parts <= 1) return;
    const int64_t threads = (int64_t)a.rows * t.nh * (HD / 4);
    if (a.parts <= kFewParts)
        hipLaunchKernelGGL((k_tree_merge_few<HD>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, a, t, kv.nkv);
    else
        hipLaunchKernelGGL((k_tree_merge<HD>), dim3(a.rows, t.nh), dim3(256), 0, st, a, t, kv.nkv);
}

int launch_tree_attn(hipStream_t st, const RowArgs& a, const KvLayer& kv, const TreeAttn& t) {
    if (a.rows <= 0) return 0;
    switch (kv.hd) {
        case 16: tree_hd<16>(st, a, kv, t); return 0;
        case 32: tree_hd<32>(st, a, kv, t); return 0;
        case 64: tree_hd<64>(st, a, kv, t); return 0;
        case 128: tree_hd<128>(st, a, kv, t); return 0;
        default: return -1;
    }
}

}  // namespace fg
