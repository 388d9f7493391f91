// norm_rope.cu -- per-head norms of q and k, the position rotation and the cache append of packed
// tokens, in one pass.
//
// For head vector x of a q or k row at position p, with weight w (the same for every head):
//   r = 1 / sqrt(mean(x^2) + eps),  y = x * r * w,
//   (y_2i, y_2i+1) <- (y_2i c_i - y_2i+1 s_i, y_2i s_i + y_2i+1 c_i),  c_i, s_i = cos, sin(p theta_i)
// q goes to the packed output, k and v to the cache.  The angle is the float32 product p * theta_i
// and its cosine and sine are the correctly rounded ones, as in every rotation of this library.
// Sums, norms and products are in float32; the only rounding to fewer bits is the store in the
// output's or the cache's type.
//
// A warp takes a token, or a part of its heads when there are few tokens, and needs nothing from other
// warps.  A thread holds 16 bytes of a head, so a head is spread over D*sizeof(IO)/16 neighbouring
// lanes and its sum of squares takes log2 of that many shuffles; a pair never leaves its thread,
// and a thread's columns are the same for every head, so its weights and the token's cos/sin pairs
// stay in registers.  While the first loads are in flight (kAhead heads, kept as the 16 bytes
// they are), the warp finds the token's sequence (32 entries of cu a step) and evaluates the
// cos/sin pairs in double precision, D/64 a lane.  Earlier versions kept the pairs in shared memory for a block:
// they were bound by their instructions and by L1 (65% and 77% at 11384 tokens of 48 heads of 128) and took 97 to 109 us
// there; this one takes 64, 4.4 TB/s, and is bound by its instructions (two thirds of the issue slots).
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "internal.h"

namespace tl {
namespace {

constexpr int kWarps = 4;   // per block
constexpr int kAhead = 2;   // loads of a thread in flight

template <typename T>
__device__ __forceinline__ uint4 load16(const T *p, bool vec) {
    if (vec) return *reinterpret_cast<const uint4 *>(p);
    if constexpr (sizeof(T) == 4) {
        const uint32_t *u = reinterpret_cast<const uint32_t *>(p);
        return make_uint4(u[0], u[1], u[2], u[3]);
    } else {
        const uint16_t *u = reinterpret_cast<const uint16_t *>(p);
        return make_uint4(u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16, u[4] | (uint32_t)u[5] << 16,
                          u[6] | (uint32_t)u[7] << 16);
    }
}
template <typename T, int N>
__device__ __forceinline__ void widen(const uint4 &u, float (&x)[N]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            x[i] = __uint_as_float(w[i]);
        } else {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}

// N consecutive values; p is aligned to N * sizeof(T) bytes
template <typename T, int N>
__device__ __forceinline__ void store_row(T *p, const float (&x)[N]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            *reinterpret_cast<float4 *>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    } else {
        uint32_t w[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&b);
        }
        if constexpr (N == 8) *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        else *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
    }
}

// What is wrong with sequence b of the batch (then none of its rows is computed, as in the attention of
// packed rows).
__device__ __forceinline__ unsigned bad_seq(long long first, long long end, long long pos, int ntok, int max_len) {
    if (end < first || first < 0 || end > ntok) return TL_DEVERR_BAD_ARG;
    return end > first && (pos < 0 || pos + end - first > max_len) ? TL_DEVERR_POS_RANGE : 0u;
}
// Out of line, and before the warp holds anything: the first warps of a launch only.
__device__ __noinline__ void report_bad(const int *cu, const int *pos0, int nseq, int ntok, int max_len, int64_t b, int64_t step,
                                        unsigned *err) {
    for (; b < nseq; b += step)
        if (const unsigned bad = bad_seq(cu[b], cu[b + 1], pos0 ? pos0[b] : 0, ntok, max_len)) atomicOr(err, bad);
}

// UNI: a warp's heads of one turn are all q, all k or all v (nHead and nHeadKv are multiples of HPW),
// so what they are is decided once for the warp.
template <typename IO, typename KV, int D, bool UNI>
__global__ void __launch_bounds__(kWarps * 32, 8) norm_rope_kernel(const NormRopeArgs a, const RopeTab tab, int parts,
                                                                bool vec_q, bool vec_k, bool vec_v, bool vec_o) {
    constexpr int N = 16 / (int)sizeof(IO);  // values per thread
    constexpr int LPH = D / N;               // lanes per head
    constexpr int HPW = 32 / LPH;            // heads per turn of a warp
    static_assert(LPH <= 32 && 32 % LPH == 0, "a head stays within a warp");
    const int lane = threadIdx.x & 31, sub = lane % LPH, d = sub * N;
    const int heads = a.nHead + 2 * a.nHeadKv;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // known to be the same for its lanes
    const int64_t job = (int64_t)blockIdx.x * kWarps + warp;
    if (job >= (int64_t)a.ntok * parts) return;
    if (job * 32 < a.nseq)
        report_bad(a.cu, a.pos0, a.nseq, a.ntok, a.kv.maxLen, job * 32 + lane, (int64_t)a.ntok * parts * 32, a.err);
    const int tok = (int)(job / parts), part = (int)(job - (int64_t)tok * parts);
    const int t1 = part * HPW, step = parts * HPW, mine = lane / LPH;  // heads t1 + mine, + step, ...
    const IO *qr = reinterpret_cast<const IO *>(a.q) + tok * a.ldq + d;
    const IO *kr = reinterpret_cast<const IO *>(a.k) + tok * a.ldk + d;
    const IO *vr = reinterpret_cast<const IO *>(a.v) + tok * a.ldv + d;
    auto load = [&](int t) {
        const int hh = t + mine, kind = UNI ? t : hh;
        if (kind < a.nHead) return load16<IO>(qr + hh * D, vec_q);
        if (kind < a.nHead + a.nHeadKv) return load16<IO>(kr + (hh - a.nHead) * D, vec_k);
        if (kind < heads) return load16<IO>(vr + (hh - a.nHead - a.nHeadKv) * D, vec_v);
        return make_uint4(0u, 0u, 0u, 0u);
    };
    uint4 x[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) x[i] = load(t1 + i * step);
    // the token's sequence: the last b with cu[b] <= tok.  Rows from cu[nseq] on belong to none.
    int lo = 0, n = a.nseq;
    while (n > 1) {
        const int st = (n + 31) / 32, i = lane * st;
        const unsigned below = __ballot_sync(0xffffffffu, i < n && a.cu[lo + min(i, n - 1)] <= tok);
        const int c = max(__popc(below) - 1, 0);
        lo += c * st;
        n = min(st, n - c * st);
    }
    const int first = a.cu[lo], end = a.cu[lo + 1], pos0 = a.pos0 ? a.pos0[lo] : 0;
    if (tok < first || tok >= end || bad_seq(first, end, pos0, a.ntok, a.kv.maxLen)) return;
    const int pos = pos0 + (tok - first);
    // cos/sin of the pairs of this thread's columns, from the lanes that evaluated them
    float2 cs[N / 2];
    {
        float2 e[D / 64];
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            const int j = lane + 32 * i;
            e[i] = j < tab.pairs ? rope_cos_sin(a.pos_base + pos, tab.theta[j]) : make_float2(1.f, 0.f);
        }
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const int j = d / 2 + i;
            cs[i] = make_float2(0.f, 0.f);
#pragma unroll
            for (int k = 0; k < D / 64; ++k) {
                const float c = __shfl_sync(0xffffffffu, e[k].x, j & 31), s = __shfl_sync(0xffffffffu, e[k].y, j & 31);
                if (j / 32 == k) cs[i] = make_float2(c, s);
            }
        }
    }
    // this thread's weights: q's, and from the first k head on k's
    float w[N];
    bool w_is_q = t1 + (UNI ? 0 : mine) < a.nHead;
    auto weights = [&](const float *src) {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = src ? __ldg(src + d + i) : 1.f;
    };
    weights(w_is_q ? a.wq : a.wk);
    IO *qo = reinterpret_cast<IO *>(a.q_out) + (int64_t)tok * a.nHead * D + d;
    // head 0 of this position in the caches; heads are maxLen rows apart
    const int64_t row0 = a.kv.row(a.layer, a.slot0 + lo, 0, pos) * D + d, hs = (int64_t)a.kv.maxLen * D;
    // every lane of a warp takes the same number of turns, so the shuffles see all of them
    // (one long basic block for the sums of kAhead heads, so that their shuffles overlap)
    for (int t0 = t1; t0 < heads; t0 += kAhead * step) {
        uint4 cur[kAhead];
        float ss[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            cur[i] = x[i];
            x[i] = load(t0 + (kAhead + i) * step);
            float y[N];
            widen<IO, N>(cur[i], y);
            ss[i] = 0.f;
#pragma unroll
            for (int k = 0; k < N; ++k) ss[i] = fmaf(y[k], y[k], ss[i]);
        }
        if (t0 < a.nHead + a.nHeadKv) {
#pragma unroll
            for (int o = LPH / 2; o >= 1; o >>= 1)
#pragma unroll
                for (int i = 0; i < kAhead; ++i) ss[i] += __shfl_xor_sync(0xffffffffu, ss[i], o);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int hh = t0 + i * step + mine, kind = UNI ? t0 + i * step : hh;
            const bool is_q = kind < a.nHead, is_k = !is_q && kind < a.nHead + a.nHeadKv;
            float y[N];
            widen<IO, N>(cur[i], y);
            if (is_q || is_k) {
                if (is_q ? a.wq != nullptr : a.wk != nullptr) {
                    if (is_k && w_is_q) {
                        weights(a.wk);
                        w_is_q = false;
                    }
                    const float r = rsqrtf(ss[i] * (1.0f / D) + a.eps);
#pragma unroll
                    for (int k = 0; k < N; ++k) y[k] = y[k] * r * w[k];
                }
#pragma unroll
                for (int k = 0; k < N; k += 2)
                    if (d / 2 + k / 2 < tab.pairs)
                        rope_rotate(y[k], y[k + 1], cs[k / 2].x, cs[k / 2].y, y[k], y[k + 1]);
            }
            if (is_q) {
                if (vec_o) {
                    store_row<IO, N>(qo + hh * D, y);
                } else {
#pragma unroll
                    for (int k = 0; k < N; ++k) qo[hh * D + k] = KvT<IO>::from_f(y[k]);
                }
            } else if (kind < heads) {
                const int h = hh - a.nHead - (is_k ? 0 : a.nHeadKv);
                store_row<KV, N>(reinterpret_cast<KV *>(is_k ? a.kv.k : a.kv.v) + row0 + h * hs, y);
            }
        }
    }
}

template <typename IO, typename KV, int D>
cudaError_t launch_t(const NormRopeArgs &a, const RopeTab &tab, cudaStream_t s) {
    auto vec = [](const void *p, int64_t ld) {
        return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * (int64_t)sizeof(IO)) % 16 == 0;
    };
    // A token is cut into parts until the warps fill the device (16 a SM) or a part is one turn
    constexpr int HPW = 32 / (D * (int)sizeof(IO) / 16);
    const int turns = (a.nHead + 2 * a.nHeadKv + HPW - 1) / HPW;
    int parts = 1;
    while (parts * 2 <= turns && (int64_t)a.ntok * parts < 16 * (int64_t)a.sms) parts *= 2;
    const int64_t blocks = ((int64_t)a.ntok * parts + kWarps - 1) / kWarps;
    const bool uni = a.nHead % HPW == 0 && a.nHeadKv % HPW == 0;
    auto kern = uni ? norm_rope_kernel<IO, KV, D, true> : norm_rope_kernel<IO, KV, D, false>;
    kern<<<(unsigned)blocks, kWarps * 32, 0, s>>>(
        a, tab, parts, vec(a.q, a.ldq), vec(a.k, a.ldk), vec(a.v, a.ldv), vec(a.q_out, 8));
    return cudaGetLastError();
}

template <typename IO, typename KV>
cudaError_t launch_d(const NormRopeArgs &a, const RopeTab &tab, cudaStream_t s) {
    if (a.headDim == 64) return launch_t<IO, KV, 64>(a, tab, s);
    if (a.headDim == 128) return launch_t<IO, KV, 128>(a, tab, s);
    return cudaErrorNotSupported;
}

}  // namespace

cudaError_t launch_norm_rope(const NormRopeArgs &a, const RopeTab &tab, cudaStream_t s) {
    if (a.ntok <= 0) return cudaSuccess;
    if (a.io == TL_IO_BF16)
        return a.kv.dtype == TL_KV_BF16 ? launch_d<__nv_bfloat16, __nv_bfloat16>(a, tab, s) : cudaErrorNotSupported;
    return a.kv.dtype == TL_KV_BF16 ? launch_d<float, __nv_bfloat16>(a, tab, s) : launch_d<float, float>(a, tab, s);
}

}  // namespace tl
