// The 8-bit paged cache: rows quantized as they are written, read back in f32,
// and moved to the positions of an accepted branch. The f32 cache takes the
// same calls.
//
// A row of one head (HD channels of a token's key or value) has the scale
// s = max|x| * r, r = 1/127 (int8) or 1/448 (fp8 e4m3, whose largest value that
// is) as f32; its codes are x / s rounded to nearest, ties to even, and stand
// for code * s: off by at most half a step, s / 2 for int8 and 2^-4 of the
// value for normal fp8 codes. The division is an IEEE one, so the codes are
// the same wherever these steps are taken. A row of zeros, or whose scale
// underflows, has codes 0; a row that holds an infinity or a NaN has the scale
// NaN and codes 0, so that it reaches only what reads this row.
#include "devutil.h"

namespace fg {

namespace {

// The four channels of a thread (d, HD / 4 threads a row) of one token, as one
// dword of codes; amax is the row's largest |x|, infinite where a value is not finite.
template <int FMT>
__device__ __forceinline__ uint32_t codes4(const float (&x)[4], float s) {
    if (!(s > 0.0f)) return FMT == KV_INT8 ? 0x80808080u : 0u;  // zeros, or a NaN scale
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = x[e] / s;
    if constexpr (FMT == KV_INT8) {
        uint32_t c = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) c |= ((uint32_t)(int)rintf(fminf(fmaxf(y[e], -127.0f), 127.0f)) & 255u) << (8 * e);
        return c ^ 0x80808080u;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = fminf(fmaxf(y[e], -448.0f), 448.0f);
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
    }
}
template <int FMT>
__device__ __forceinline__ void values4(uint32_t c, float s, float (&x)[4]) {
    if constexpr (FMT == KV_INT8) {
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = ((float)(c >> (8 * e) & 255u) - 128.0f) * s;
    } else {
        x[0] = __builtin_amdgcn_cvt_f32_fp8(c, 0) * s;
        x[1] = __builtin_amdgcn_cvt_f32_fp8(c, 1) * s;
        x[2] = __builtin_amdgcn_cvt_f32_fp8(c, 2) * s;
        x[3] = __builtin_amdgcn_cvt_f32_fp8(c, 3) * s;
    }
}
// The scale of a row from its threads' largest |x|, over the HD / 4 lanes that hold it.
template <int FMT, int HD>
__device__ __forceinline__ float row_scale(const float (&x)[4]) {
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float a = fabsf(x[e]);
        m = fmaxf(m, a < INFINITY ? a : INFINITY);  // a NaN compares false
    }
    m = group_reduce<HD / 4, true>(m);
    if (m == INFINITY) return NAN;
    return m * (FMT == KV_INT8 ? 1.0f / 127.0f : 1.0f / 448.0f);
}
__device__ __forceinline__ void get4(const float* p, float (&x)[4]) {
    const float4 v = *(const float4*)p;
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
// Codes of four tokens' dwords (one token each, four channels) as four channels' dwords (one channel each, four tokens).
__device__ __forceinline__ uint4 transpose4(const uint32_t (&c)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(c[1], c[0], 0x05010400), b = __builtin_amdgcn_perm(c[3], c[2], 0x05010400);
    const uint32_t e = __builtin_amdgcn_perm(c[1], c[0], 0x07030602), f = __builtin_amdgcn_perm(c[3], c[2], 0x07030602);
    return make_uint4(__builtin_amdgcn_perm(b, a, 0x05040100), __builtin_amdgcn_perm(b, a, 0x07060302),
                      __builtin_amdgcn_perm(f, e, 0x05040100), __builtin_amdgcn_perm(f, e, 0x07060302));
}

// Where a (block, head)'s group of four tokens lies in an 8-bit record, for the thread's channels.
template <int HD>
struct Group {
    uint8_t *k, *v;  // k: its first token's dword, HD apart; v: 16 bytes, four channels of four tokens
    float *ks, *vs;  // four scales
    __device__ Group(uint8_t* rec, int tg, int d) {
        k = rec + (size_t)tg * 4 * HD + 4 * d;
        v = rec + 16 * HD + (size_t)tg * 4 * HD + 16 * d;
        ks = (float*)(rec + 32 * HD) + 4 * tg;
        vs = ks + 16;
    }
};

// Four tokens' keys and values of one head into their group; used: which of them.
template <int FMT, int HD>
__device__ __forceinline__ void put_group(const Group<HD>& g, int d, int used, float (&kx)[4][4], float (&vx)[4][4]) {
    uint32_t vc[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const float ks = row_scale<FMT, HD>(kx[t]), vs = row_scale<FMT, HD>(vx[t]);
        vc[t] = codes4<FMT>(vx[t], vs);
        if (!(used >> t & 1)) continue;
        *(uint32_t*)(g.k + t * HD) = codes4<FMT>(kx[t], ks);
        if (d == 0) {
            g.ks[t] = ks;
            g.vs[t] = vs;
        }
    }
    if (used == 15) {
        *(uint4*)g.v = transpose4(vc);
    } else {
#pragma unroll
        for (int t = 0; t < 4; t++)
            if (used >> t & 1)
#pragma unroll
                for (int e = 0; e < 4; e++) g.v[4 * e + t] = (uint8_t)(vc[t] >> (8 * e));
    }
}

template <int FMT, int HD>
__device__ __forceinline__ void get_group(const Group<HD>& g, float (&kx)[4][4], float (&vx)[4][4]) {
    uint32_t kc[4];
#pragma unroll
    for (int t = 0; t < 4; t++) kc[t] = *(const uint32_t*)(g.k + t * HD);
    const uint4 w = *(const uint4*)g.v;
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
    const uint4 tv = transpose4(ws);  // back to a dword per token
    const uint32_t vc[4] = {tv.x, tv.y, tv.z, tv.w};
    const float4 ks = *(const float4*)g.ks, vs = *(const float4*)g.vs;
    const float ksa[4] = {ks.x, ks.y, ks.z, ks.w}, vsa[4] = {vs.x, vs.y, vs.z, vs.w};
#pragma unroll
    for (int t = 0; t < 4; t++) {
        values4<FMT>(kc[t], ksa[t], kx[t]);
        values4<FMT>(vc[t], vsa[t], vx[t]);
    }
}

}  // namespace

// A thread takes four channels of one head over an aligned group of four tokens
// of a page (a quad), so that the values, which a record holds by channel, go
// out as one 16-byte store of a whole group. Bound by memory: six ragged
// chunks, 9500 rows in all, 8 heads of 128, fp8: 20.5 us (98 MB read and
// written, 4.8 TB/s); one row 3.6 us.
template <int FMT, int HD>
__global__ __launch_bounds__(256) void k_kv_append(RowArgs a, KvLayer kv, const float* __restrict__ k,
                                                   const float* __restrict__ v, int64_t ld,
                                                   const float* __restrict__ cos_t, const float* __restrict__ sin_t) {
    constexpr int T = HD / 4;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int d = (int)(at % T), h = (int)(at / T % kv.nkv);
    const int64_t qi = at / T / kv.nkv;
    if (qi >= a.n_quads) return;
    const int4 rec = *(const int4*)(a.quads + 4 * qi);
    float kx[4][4], vx[4][4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const bool on = rec.w >> t & 1;
        const int64_t row = on ? rec.x + t : 0;
        const float* kp = k + row * ld + h * HD;
        get4(kp + 4 * d, kx[t]);
        get4(v + row * ld + h * HD + 4 * d, vx[t]);
        if (cos_t) {  // rotate-half, src/model.rs:451-459
            const int dh = d % (T / 2);
            float y[4], c[4], s[4];
            get4(kp + 4 * (d < T / 2 ? d + T / 2 : d - T / 2), y);
            get4(cos_t + (size_t)a.rpos[row] * (HD / 2) + 4 * dh, c);
            get4(sin_t + (size_t)a.rpos[row] * (HD / 2) + 4 * dh, s);
#pragma unroll
            for (int e = 0; e < 4; e++)
                kx[t][e] = __fadd_rn(__fmul_rn(kx[t][e], c[e]), __fmul_rn(d < T / 2 ? -y[e] : y[e], s[e]));
        }
    }
    if constexpr (FMT == KV_F32) {
        const size_t o = (((size_t)(uint32_t)rec.y * kv.nkv + h) * 16 + 4 * rec.z) * HD + 4 * d;
#pragma unroll
        for (int t = 0; t < 4; t++)
            if (rec.w >> t & 1) {
                *(float4*)(kv.k + o + t * HD) = make_float4(kx[t][0], kx[t][1], kx[t][2], kx[t][3]);
                *(float4*)(kv.v + o + t * HD) = make_float4(vx[t][0], vx[t][1], vx[t][2], vx[t][3]);
            }
    } else {
        const Group<HD> g(kv.data + ((size_t)(uint32_t)rec.y * kv.nkv + h) * kv_record(HD), rec.z, d);
        put_group<FMT, HD>(g, d, rec.w, kx, vx);
    }
}

// CONTEXT: every token of a sequence (blockIdx.y); else the rows, unused ones as zeros. Bound by the f32 it writes:
// 16 contexts of 128 to 2048 tokens, 32 heads of 64, int8, 70 us (5.1 TB/s in all, of
// 6.2 that a copy reaches).
template <int FMT, int HD, bool CONTEXT>
__global__ __launch_bounds__(256) void k_kv_gather(RowArgs a, KvLayer kv, float* __restrict__ k,
                                                   float* __restrict__ v) {
    constexpr int T = HD / 4;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int d = (int)(at % T), h = (int)(at / T % kv.nkv);
    const int64_t qi = at / T / kv.nkv;
    int64_t out;  // first token's row of the output
    int used, tg;
    size_t block;
    if (CONTEXT) {
        const int32_t* s = a.seqs + (size_t)blockIdx.y * kSeqWords;
        const int left = s[7] - (int)min(4 * qi, (int64_t)s[7]);
        if (left <= 0) return;
        used = left >= 4 ? 15 : (1 << left) - 1;
        out = (int64_t)s[6] + 4 * qi;
        block = (uint32_t)a.btab[s[3] + qi / 4];
        tg = (int)(qi % 4);
    } else {
        if (qi >= a.n_quads) return;
        const int4 rec = *(const int4*)(a.quads + 4 * qi);
        out = rec.x;
        block = (uint32_t)rec.y;
        tg = rec.z;
        used = rec.w;
    }
    float kx[4][4], vx[4][4];
    if constexpr (FMT == KV_F32) {
        const size_t o = ((block * kv.nkv + h) * 16 + 4 * tg) * HD + 4 * d;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            get4(kv.k + o + t * HD, kx[t]);
            get4(kv.v + o + t * HD, vx[t]);
        }
    } else {
        get_group<FMT, HD>(Group<HD>(kv.data + (block * kv.nkv + h) * kv_record(HD), tg, d), kx, vx);
    }
#pragma unroll
    for (int t = 0; t < 4; t++)
        if (used >> t & 1) {
            const size_t o = ((size_t)(out + t) * kv.nkv + h) * HD + 4 * d;
            *(float4*)(k + o) = make_float4(kx[t][0], kx[t][1], kx[t][2], kx[t][3]);
            *(float4*)(v + o) = make_float4(vx[t][0], vx[t][1], vx[t][2], vx[t][3]);
        }
}

// Rows that no call wrote (unused rows of a tree) read back as zeros.
__global__ __launch_bounds__(256) void k_zero_unused(RowArgs a, int width, float* __restrict__ x, float* __restrict__ y) {
    if (!a.mrec[4 * (size_t)blockIdx.x + 3]) return;
    for (int i = threadIdx.x; i < width; i += 256) {
        x[(size_t)blockIdx.x * width + i] = 0.0f;
        if (y) y[(size_t)blockIdx.x * width + i] = 0.0f;
    }
}

// Whole layers, [block][head][16][HD] f32 and back.
template <int FMT, int HD, bool PACK>
__global__ __launch_bounds__(256) void k_kv_layer(KvLayer kv, int64_t groups, float* __restrict__ k,
                                                  float* __restrict__ v) {
    constexpr int T = HD / 4;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, gi = at / T;
    const int d = (int)(at % T);
    if (gi >= groups) return;
    const Group<HD> g(kv.data + (size_t)(gi / 4) * kv_record(HD), (int)(gi % 4), d);
    float kx[4][4], vx[4][4];
    const size_t o = (size_t)gi * 4 * HD + 4 * d;
    if (PACK) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
            get4(k + o + t * HD, kx[t]);
            get4(v + o + t * HD, vx[t]);
        }
        put_group<FMT, HD>(g, d, 15, kx, vx);
    } else {
        get_group<FMT, HD>(g, kx, vx);
#pragma unroll
        for (int t = 0; t < 4; t++) {
            *(float4*)(k + o + t * HD) = make_float4(kx[t][0], kx[t][1], kx[t][2], kx[t][3]);
            *(float4*)(v + o + t * HD) = make_float4(vx[t][0], vx[t][1], vx[t][2], vx[t][3]);
        }
    }
}

// One workgroup of HD / 4 threads per (sequence, head, layer); a thread moves its
// four channels of one row after the other. A branch's rows stand in order, row
// path[j] at or behind position j, so no row is overwritten before it is moved.
// Counts and rows outside the sequence's are not followed. A few rows: latency, one read and write after the other.
template <int FMT, int HD>
__global__ __launch_bounds__(64) void k_kv_commit(RowArgs a, KvLayer kv, size_t layer_bytes,
                                                  const int32_t* __restrict__ path, const int32_t* __restrict__ count,
                                                  int ld) {
    const int s = blockIdx.x, h = blockIdx.y, d = threadIdx.x;
    const int32_t* sr = a.seqs + (size_t)s * kSeqWords;
    const int n = sr[1], pos = sr[2], m = min(min(count[s], ld), n);
    const size_t lo = blockIdx.z * layer_bytes;
    const float *ck = (const float*)((const char*)kv.k + lo), *cv = (const float*)((const char*)kv.v + lo);
    for (int j = 0; j < m; j++) {
        const int r = path[(size_t)s * ld + j];
        if (r <= j || r >= n) continue;
        const int from = pos + r, to = pos + j;
        const size_t fb = (uint32_t)a.btab[sr[3] + from / 16], tb = (uint32_t)a.btab[sr[3] + to / 16];
        if constexpr (FMT == KV_F32) {
            const size_t fo = ((fb * kv.nkv + h) * 16 + from % 16) * HD + 4 * d;
            const size_t to_ = ((tb * kv.nkv + h) * 16 + to % 16) * HD + 4 * d;
            *(float4*)((float*)ck + to_) = *(const float4*)(ck + fo);
            *(float4*)((float*)cv + to_) = *(const float4*)(cv + fo);
        } else {
            const int ft = from % 4, tt = to % 4;
            const Group<HD> f(kv.data + lo + (fb * kv.nkv + h) * kv_record(HD), from % 16 / 4, d);
            const Group<HD> t(kv.data + lo + (tb * kv.nkv + h) * kv_record(HD), to % 16 / 4, d);
            *(uint32_t*)(t.k + tt * HD) = *(const uint32_t*)(f.k + ft * HD);
#pragma unroll
            for (int e = 0; e < 4; e++) t.v[4 * e + tt] = f.v[4 * e + ft];
            if (d == 0) {
                t.ks[tt] = f.ks[ft];
                t.vs[tt] = f.vs[ft];
            }
        }
    }
}

namespace {
// f(format, head dim) as constants.
template <class F>
int with_shape(int format, int hd, const F& f) {
    auto by_hd = [&](auto fmt) {
        switch (hd) {
            case 16: f(fmt, std::integral_constant<int, 16>()); return 0;
            case 32: f(fmt, std::integral_constant<int, 32>()); return 0;
            case 64: f(fmt, std::integral_constant<int, 64>()); return 0;
            case 128: f(fmt, std::integral_constant<int, 128>()); return 0;
            default: return -1;
        }
    };
    switch (format) {
        case KV_F32: return by_hd(std::integral_constant<int, KV_F32>());
        case KV_INT8: return by_hd(std::integral_constant<int, KV_INT8>());
        case KV_FP8: return by_hd(std::integral_constant<int, KV_FP8>());
        default: return -1;
    }
}
unsigned groups_of(int64_t threads) { return (unsigned)((threads + 255) / 256); }
}  // namespace

int launch_kv_append(hipStream_t st, const RowArgs& a, const KvLayer& kv, const float* k, const float* v, int64_t ld,
                     const float* cos_t, const float* sin_t) {
    if (a.n_quads <= 0) return 0;
    return with_shape(kv.format, kv.hd, [&](auto fmt, auto hd) {
        hipLaunchKernelGGL((k_kv_append<fmt.value, hd.value>),
                           dim3(groups_of((int64_t)a.n_quads * kv.nkv * (hd.value / 4))), dim3(256), 0, st, a, kv, k, v,
                           ld, cos_t, sin_t);
    });
}

int launch_kv_gather(hipStream_t st, const RowArgs& a, const KvLayer& kv, bool context, float* k, float* v) {
    if (context ? a.longest <= 0 : a.rows <= 0) return 0;
    return with_shape(kv.format, kv.hd, [&](auto fmt, auto hd) {
        const int64_t per = (int64_t)kv.nkv * (hd.value / 4);
        if (context) {
            hipLaunchKernelGGL((k_kv_gather<fmt.value, hd.value, true>),
                               dim3(groups_of((a.longest + 3) / 4 * per), a.n_seqs), dim3(256), 0, st, a, kv, k, v);
        } else {
            if (a.n_quads > 0)
                hipLaunchKernelGGL((k_kv_gather<fmt.value, hd.value, false>), dim3(groups_of(a.n_quads * per)),
                                   dim3(256), 0, st, a, kv, k, v);
            if (a.unused) hipLaunchKernelGGL(k_zero_unused, dim3(a.rows), dim3(256), 0, st, a, kv.nkv * kv.hd, k, v);
        }
    });
}

int launch_kv_unpack(hipStream_t st, const KvLayer& kv, int blocks, float* k, float* v) {
    return with_shape(kv.format, kv.hd, [&](auto fmt, auto hd) {
        if constexpr (fmt.value != KV_F32) {
            const int64_t groups = (int64_t)blocks * kv.nkv * 4;
            hipLaunchKernelGGL((k_kv_layer<fmt.value, hd.value, false>), dim3(groups_of(groups * (hd.value / 4))),
                               dim3(256), 0, st, kv, groups, k, v);
        }
    });
}

int launch_kv_pack(hipStream_t st, const KvLayer& kv, int blocks, const float* k, const float* v) {
    return with_shape(kv.format, kv.hd, [&](auto fmt, auto hd) {
        if constexpr (fmt.value != KV_F32) {
            const int64_t groups = (int64_t)blocks * kv.nkv * 4;
            hipLaunchKernelGGL((k_kv_layer<fmt.value, hd.value, true>), dim3(groups_of(groups * (hd.value / 4))),
                               dim3(256), 0, st, kv, groups, const_cast<float*>(k), const_cast<float*>(v));
        }
    });
}

int launch_kv_commit(hipStream_t st, const RowArgs& a, const KvLayer& first, int layers, size_t layer_bytes,
                     const int32_t* path, const int32_t* count, int ld) {
    if (a.n_seqs <= 0 || layers <= 0) return 0;
    return with_shape(first.format, first.hd, [&](auto fmt, auto hd) {
        hipLaunchKernelGGL((k_kv_commit<fmt.value, hd.value>), dim3(a.n_seqs, first.nkv, layers), dim3(hd.value / 4), 0,
                           st, a, first, layer_bytes, path, count, ld);
    });
}

}  // namespace fg
