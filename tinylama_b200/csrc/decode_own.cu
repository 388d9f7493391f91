// decode_own.cu -- one query token per sequence over its own cached positions: the part of a decode over a
// shared prefix that is not shared.
//
// The state of a q-head over positions 0..pos[b] of its sequence's slot: m = max_j s_j (log2 units),
// l = sum_j 2^(s_j - m), o = sum_j 2^(s_j - m) v_j, with s_j = log2(e)/sqrt(D) q . k_j.
//
// Own positions are few (a conversation turn behind a long prompt), so what counts is not the stream of
// one sequence but how many are under way.  The work is cut into (sequence, kv-head, chunk)
// jobs, and a warp takes a job alone, from its own ring of shared-memory tiles that its own lane 0
// fills by TMA: there is no other warp to wait for, and no merge inside the CTA.  The tiles of the next
// job are requested before the current one ends.  Jobs are numbered without gaps (a prefix sum of the
// sequences' chunks, which every CTA forms for itself) and dealt out in turn, so no warp has more
// than one job more than another.  One CTA per SM, kWarps warps of NS tiles of
// 16 KB: 192 KB in flight.  The G heads of the group are rows of mma.sync fragments as in
// decode_mma.cu: a bf16 cache takes q and the weights as bf16 high and low parts (rows 0-7 and 8-15
// of one m16n8k16), an f32 cache takes q, K, the weights and V as tf32 high and low parts, which hold a value to
// 2^-22 (a third part would be two more products for each two; the error of 48 sequences of up to 300 behind 2000,
// 32/8/128, is below that of a 32-bit softmax as it is).  f32 activations over
// a bf16 cache take a third bf16 part in a product of its own: two hold 16 bits of q, which left an
// error of 3.4e-6 where a 32-bit softmax has 5e-7 (48 sequences of up to 300, 32/8/128).  Such warp-level
// products reach HBM speed with G <= 8 rows; the 128 rows of a tcgen05 tile would be mostly empty.
// At 64 sequences of up to 512 positions (32/8/128 bf16, 87 MB with the prefix) a kernel with one
// unit per CTA of 4 warps took 37 us on 94 SMs; this one takes 23 on 100, and streams up to 50 GB/s to an SM.
#include <math.h>

#include "common.cuh"
#include "decode_common.cuh"
#include "internal.h"
#include "mma_common.cuh"
#include "tc_common.cuh"

namespace tl {
namespace {

constexpr int kWarps = 6, kStages = 2;

template <typename KV, int D>
struct OwnCfg {
    static constexpr bool F32 = sizeof(KV) == 4;
    static constexpr int STAGE = 16384;                              // K and V of a tile
    static constexpr int T = STAGE / (2 * D * (int)sizeof(KV));      // positions per tile
    static constexpr int R = F32 || T < 32 ? 1 : 2;                  // 16-position groups worked on together
    static constexpr int BOX_COLS = 128 / (int)sizeof(KV), HALVES = D / BOX_COLS, HALF = T * 128;
    static constexpr int KT = D / 16, NT = D / 8;
    static int smem(int nseq) { return 1024 + kWarps * kStages * STAGE + kWarps * kStages * 8 + 4 * (2 * nseq + 1 + kWarps); }
    static_assert(T % (16 * R) == 0, "whole groups");
};

struct OwnParams {
    const void *q;
    const void *k, *v;    // from (layer, slot0) on
    const int *pos;
    int nseq, nHead, nHeadKv, G, max_len;
    int chunk, nchunks;   // positions per job, jobs per (sequence, kv-head)
    float *state;         // [nchunks][nseq * nHead] of D values, then as many (m, l)
    unsigned *err;
};

// Where a warp is in its list of jobs: the tile to be requested or worked on next.
struct Cursor {
    int job;
    int b, g, c, n, t;    // sequence, kv-head, chunk, its positions, tiles done
};

// the bf16 rest of a pair behind its high and low parts
__device__ __forceinline__ uint32_t third2(float x0, float x1, uint32_t hi, uint32_t lo) {
    auto low = [](uint32_t u) { return __uint_as_float(u << 16); };
    auto high = [](uint32_t u) { return __uint_as_float(u & 0xffff0000u); };
    return pack_bf16(x0 - low(hi) - low(lo), x1 - high(hi) - high(lo));
}

// The state of one head over a job's n positions (rows k, v) by fp32 products, for one whose sums have
// come out not finite.  The matrix products take an infinity apart into parts (infinity - infinity) or
// multiply it with a low part of zero, and both are NaN.  Here a key of minus infinity has no
// weight, and an infinite value is what it is.  A warp takes a position at a time, D/32 columns a lane: about 25
// instructions a position, some 20 times a head's share of the products above, and no further than
// the first score that is not a number.
template <typename IO, typename KV, int D>
__device__ __noinline__ void own_again(const IO *q, const KV *k, const KV *v, int n, float *state, float2 *ml) {
    constexpr int N = D / 32;
    const int lane = threadIdx.x & 31;
    const float scale = kLog2e / sqrtf((float)D);
    q += lane * N;
    k += lane * N;
    v += lane * N;
    float x[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        x[i] = KvT<IO>::to_f(q[i]);
        o[i] = 0.f;
    }
    for (int j = 0; j < n && l == l; ++j, k += D, v += D) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) s = fmaf(x[i], KvT<KV>::to_f(k[i]), s);
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        s *= scale;
        if (s == -INFINITY) continue;
        const float M = fmaxf(m, s), alpha = safe_exp2_diff(m, M), w = exp2f(s - M);
        m = M;
        l = fmaf(l, alpha, w);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            o[i] *= alpha;
            if (w != 0.f) o[i] = fmaf(w, KvT<KV>::to_f(v[i]), o[i]);
        }
    }
    if (lane == 0) *ml = make_float2(m, l);
#pragma unroll
    for (int i = 0; i < N; ++i) state[lane * N + i] = o[i];
}

template <typename IO, typename KV, int D>
__global__ void __launch_bounds__(kWarps * 32, 1)
decode_own_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const OwnParams p) {
    using C = OwnCfg<KV, D>;
    constexpr bool IO32 = sizeof(IO) == 4, THREE = IO32 && !C::F32;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t *base = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    uint64_t *bars = reinterpret_cast<uint64_t *>(base + kWarps * kStages * C::STAGE);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int gid = lane >> 2, tq = lane & 3;  // fragment row (head) and column pair
    uint8_t *ring = base + warp * kStages * C::STAGE;
    uint64_t *full = bars + warp * kStages;
    if (lane == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(&full[i], 1);
        fence_mbar_init();
    }
    __syncwarp();
    pdl_launch_dependents();
    // own positions of the sequences, and the chunks of the sequences before each one
    int *len = reinterpret_cast<int *>(bars + kWarps * kStages), *pre = len + p.nseq, *sums = pre + p.nseq + 1;
    {
        const int tid = threadIdx.x, per = (p.nseq + kWarps * 32 - 1) / (kWarps * 32);
        const int b0 = min(tid * per, p.nseq), b1 = min(b0 + per, p.nseq);
        int mine = 0;
        for (int b = b0; b < b1; ++b) {
            const int pos = p.pos[b], n = min(max(pos + 1, 0), p.max_len);
            int c = (n + p.chunk - 1) / p.chunk;
            len[b] = n;
            if (blockIdx.x == 0 && (pos < -1 || pos >= p.max_len)) atomicOr(p.err, TL_DEVERR_POS_RANGE);
            if (c > p.nchunks) {  // the host sized the chunks from its copy of the positions
                if (blockIdx.x == 0) atomicOr(p.err, TL_DEVERR_BAD_ARG);
                c = p.nchunks;
            }
            pre[b] = c;
            mine += c;
        }
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) sums[warp] = incl;
        __syncthreads();
        int run = incl - mine;
        for (int w = 0; w < warp; ++w) run += sums[w];
        for (int b = b0; b < b1; ++b) {
            const int c = pre[b];
            pre[b] = run;
            run += c;
        }
        if (tid == kWarps * 32 - 1) pre[p.nseq] = run;
        __syncthreads();
    }
    const int jobs = pre[p.nseq] * p.nHeadKv, stride = gridDim.x * kWarps;
    auto start = [&](int job) {
        Cursor c{};
        c.job = job;
        if (job >= jobs) return c;
        const int x = job / p.nHeadKv;
        c.g = job - x * p.nHeadKv;
        int lo = 0, hi = p.nseq;  // pre[lo] <= x < pre[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (pre[mid] <= x) lo = mid; else hi = mid;
        }
        c.b = lo;
        c.c = x - pre[lo];
        c.n = min(len[lo] - c.c * p.chunk, p.chunk);
        return c;
    };
    const float scale = kLog2e / sqrtf((float)D);
    const uint64_t pol = policy_evict_first();
    int is = 0, us = 0;          // stage to be filled, stage to be used
    uint32_t uphase = 0;
    Cursor in = start(warp * gridDim.x + blockIdx.x), at = in;
    // the q rows of a job, towards L1: they are read only when the job starts, which would wait for them
    auto prefetch_q = [&](const Cursor &c) {
        if (c.job < jobs && lane * 128 < p.G * D * (int)sizeof(IO))
            asm volatile("prefetch.global.L1 [%0];" ::"l"(reinterpret_cast<const uint8_t *>(
                reinterpret_cast<const IO *>(p.q) + ((int64_t)c.b * p.nHead + (int64_t)c.g * p.G) * D) + lane * 128));
    };
    auto request = [&]() {
        if (in.job >= jobs) return;
        if (lane == 0) {
            uint8_t *st = ring + is * C::STAGE;
            const int row = (in.b * p.nHeadKv + in.g) * p.max_len + in.c * p.chunk + in.t * C::T;
            mbar_arrive_expect_tx(&full[is], C::STAGE);
#pragma unroll
            for (int hh = 0; hh < C::HALVES; ++hh) {
                tma_load_2d_hint(st + hh * C::HALF, &kmap, C::BOX_COLS * hh, row, &full[is], pol);
                tma_load_2d_hint(st + C::STAGE / 2 + hh * C::HALF, &vmap, C::BOX_COLS * hh, row, &full[is], pol);
            }
        }
        if (++is == kStages) is = 0;
        if (++in.t * C::T >= in.n) {
            in = start(in.job + stride);
            prefetch_q(in);
        }
    };
    prefetch_q(in);
    for (int i = 0; i < kStages; ++i) request();
    const bool row_ok = gid < p.G;
    while (at.job < jobs) {
        // ---- q fragments: bf16 high and low parts, or tf32 ones, of this thread's columns ----
        uint32_t qh[C::KT][C::F32 ? 4 : 2], ql[C::KT][C::F32 ? 4 : 2], qt[C::KT][2];
        const int64_t head = (int64_t)at.b * p.nHead + (int64_t)at.g * p.G + (row_ok ? gid : 0);
        {
            auto q2 = [&](int d) {
                if (!row_ok) return make_float2(0.f, 0.f);
                const IO *src = reinterpret_cast<const IO *>(p.q) + head * D + d;
                if constexpr (IO32) return *reinterpret_cast<const float2 *>(src);
                else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(src));
            };
#pragma unroll
            for (int kt = 0; kt < C::KT; ++kt) {
                if constexpr (C::F32) {
                    const int d = 32 * (kt >> 1) + 4 * (2 * tq + (kt & 1));
                    const float2 x = q2(d), y = q2(d + 2);
                    split_tf32(x.x, qh[kt][0], ql[kt][0]);
                    split_tf32(x.y, qh[kt][1], ql[kt][1]);
                    split_tf32(y.x, qh[kt][2], ql[kt][2]);
                    split_tf32(y.y, qh[kt][3], ql[kt][3]);
                } else {
                    const float2 x = q2(16 * kt + 2 * tq), y = q2(16 * kt + 2 * tq + 8);
                    split2(x.x, x.y, qh[kt][0], ql[kt][0]);
                    split2(y.x, y.y, qh[kt][1], ql[kt][1]);
                    if constexpr (THREE) {
                        qt[kt][0] = third2(x.x, x.y, qh[kt][0], ql[kt][0]);
                        qt[kt][1] = third2(y.x, y.y, qh[kt][1], ql[kt][1]);
                    }
                }
            }
        }
        float m = -INFINITY, l = 0.f, o[C::NT][4];
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt) o[nt][0] = o[nt][1] = o[nt][2] = o[nt][3] = 0.f;
        bool ok = true;
        for (int p0 = 0; p0 < at.n; p0 += C::T) {
            ok = __all_sync(0xffffffffu, mbar_wait(&full[us], uphase, p.err, nullptr));
            if (!ok) break;
            uint8_t *st = ring + us * C::STAGE;
            const uint32_t kbox = smem_u32(st), vbox = kbox + C::STAGE / 2;
            const bool tail = p0 + C::T > at.n;
            if (tail) {
                // V rows behind the last position hold leftovers; zero times an infinity is not zero
                for (int e = (at.n - p0) * 8 + lane; e < C::T * 8; e += 32)
#pragma unroll
                    for (int hh = 0; hh < C::HALVES; ++hh)
                        *reinterpret_cast<uint4 *>(st + C::STAGE / 2 + hh * C::HALF + e * 16) = make_uint4(0u, 0u, 0u, 0u);
                fence_proxy_async_smem();  // before the ring's next copy into these bytes
                __syncwarp();
            }
#pragma unroll 1
            for (int r0 = 0; r0 < C::T && p0 + r0 < at.n; r0 += 16 * C::R) {
                // ---- S = Q K^T for 16 R positions: n8 tiles 0 .. 2R-1 ----
                float s[2 * C::R][4];
#pragma unroll
                for (int i = 0; i < 2 * C::R; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
                if constexpr (C::F32) {
                    // the terms with K's low part are summed apart: two shorter chains of products
                    float t[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                    for (int kt = 0; kt < C::KT; ++kt)
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt) {
                            const float4 x = *reinterpret_cast<const float4 *>(
                                st + (swz(kbox + (kt >> 1) * C::HALF, r0 + 8 * nt + gid, 2 * tq + (kt & 1)) - kbox));
                            uint32_t kb[4], ks[4];
                            split_tf32(x.x, kb[0], ks[0]);
                            split_tf32(x.y, kb[1], ks[1]);
                            split_tf32(x.z, kb[2], ks[2]);
                            split_tf32(x.w, kb[3], ks[3]);
                            mma1688(t[nt], qh[kt][0], ql[kt][0], qh[kt][1], ql[kt][1], ks[0], ks[1]);
                            mma1688(s[nt], qh[kt][0], ql[kt][0], qh[kt][1], ql[kt][1], kb[0], kb[1]);
                            mma1688(t[nt], qh[kt][2], ql[kt][2], qh[kt][3], ql[kt][3], ks[2], ks[3]);
                            mma1688(s[nt], qh[kt][2], ql[kt][2], qh[kt][3], ql[kt][3], kb[2], kb[3]);
                        }
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[nt][i] += t[nt][i];
                } else {
                    const int krow = r0 + ((lane >> 4) << 3) + (lane & 7), kc = (lane >> 3) & 1;
#pragma unroll
                    for (int kt = 0; kt < C::KT; ++kt) {
                        const int dim = 16 * kt + 8 * kc;
#pragma unroll
                        for (int i = 0; i < C::R; ++i) {
                            uint32_t b00, b01, b10, b11;
                            ldsm_x4(swz(kbox + (dim >> 6) * C::HALF, krow + 16 * i, (dim & 63) >> 3), b00, b01, b10, b11);
                            mma16816(s[2 * i], qh[kt][0], ql[kt][0], qh[kt][1], ql[kt][1], b00, b01);
                            mma16816(s[2 * i + 1], qh[kt][0], ql[kt][0], qh[kt][1], ql[kt][1], b10, b11);
                            if constexpr (THREE) {
                                mma16816(s[2 * i], qt[kt][0], 0u, qt[kt][1], 0u, b00, b01);
                                mma16816(s[2 * i + 1], qt[kt][0], 0u, qt[kt][1], 0u, b10, b11);
                            }
                        }
                    }
                }
                // ---- online softmax of row gid; this thread has positions 2tq, 2tq+1 of each n8 tile ----
                float pr[4 * C::R];
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4 * C::R; ++i) {
                    const int at_p = p0 + r0 + 8 * (i >> 1) + 2 * tq + (i & 1);
                    pr[i] = at_p < at.n ? (s[i >> 1][i & 1] + s[i >> 1][2 + (i & 1)]) * scale : -INFINITY;
                    mx = fmaxf(mx, pr[i]);
                }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                if (mx > m + 8.0f || (m == -INFINITY && mx != -INFINITY)) {  // the same in a row's four lanes
                    const float alpha = (m == -INFINITY) ? 0.f : exp2f(m - mx);
                    m = mx;
                    l *= alpha;
#pragma unroll
                    for (int nt = 0; nt < C::NT; ++nt) {
                        o[nt][0] *= alpha;
                        o[nt][1] *= alpha;
                        o[nt][2] *= alpha;
                        o[nt][3] *= alpha;
                    }
                }
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4 * C::R; ++i) {
                    pr[i] = pr[i] == -INFINITY ? 0.f : exp2f(pr[i] - m);
                    sum += pr[i];
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                l += sum;
                // ---- O += P V ----
                if constexpr (C::F32) {
                    uint32_t pb[4], ps[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) split_tf32(pr[i], pb[i], ps[i]);
#pragma unroll
                    for (int j = 0; j < C::HALVES; ++j) {
                        const uint32_t box = vbox + j * C::HALF;
                        auto v4 = [&](int r) {
                            return *reinterpret_cast<const float4 *>(st + (swz(box, r0 + r, gid) - kbox));
                        };
                        const float4 x0 = v4(2 * tq), x1 = v4(2 * tq + 1), x8 = v4(2 * tq + 8), x9 = v4(2 * tq + 9);
                        const float a0[4] = {x0.x, x0.y, x0.z, x0.w}, a1[4] = {x1.x, x1.y, x1.z, x1.w};
                        const float a8[4] = {x8.x, x8.y, x8.z, x8.w}, a9[4] = {x9.x, x9.y, x9.z, x9.w};
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            uint32_t v0b, v0s, v1b, v1s, v8b, v8s, v9b, v9s;
                            split_tf32(a0[u], v0b, v0s);
                            split_tf32(a1[u], v1b, v1s);
                            split_tf32(a8[u], v8b, v8s);
                            split_tf32(a9[u], v9b, v9s);
                            mma1688(o[4 * j + u], pb[0], ps[0], pb[1], ps[1], v0b, v1b);
                            mma1688(o[4 * j + u], pb[0], ps[0], pb[1], ps[1], v0s, v1s);
                            mma1688(o[4 * j + u], pb[2], ps[2], pb[3], ps[3], v8b, v9b);
                            mma1688(o[4 * j + u], pb[2], ps[2], pb[3], ps[3], v8s, v9s);
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < C::R; ++i) {
                        uint32_t ph0, pl0, ph1, pl1, pt0 = 0u, pt1 = 0u;
                        split2(pr[4 * i], pr[4 * i + 1], ph0, pl0);
                        split2(pr[4 * i + 2], pr[4 * i + 3], ph1, pl1);
                        if constexpr (THREE) {
                            pt0 = third2(pr[4 * i], pr[4 * i + 1], ph0, pl0);
                            pt1 = third2(pr[4 * i + 2], pr[4 * i + 3], ph1, pl1);
                        }
                        const int vrow = r0 + 16 * i + (((lane >> 3) & 1) << 3) + (lane & 7), vc = lane >> 4;
#pragma unroll
                        for (int dp = 0; dp < C::NT / 2; ++dp) {
                            const int dim = 16 * dp + 8 * vc;
                            uint32_t b00, b01, b10, b11;
                            ldsm_x4_t(swz(vbox + (dim >> 6) * C::HALF, vrow, (dim & 63) >> 3), b00, b01, b10, b11);
                            mma16816(o[2 * dp], ph0, pl0, ph1, pl1, b00, b01);
                            mma16816(o[2 * dp + 1], ph0, pl0, ph1, pl1, b10, b11);
                            if constexpr (THREE) {
                                mma16816(o[2 * dp], pt0, 0u, pt1, 0u, b00, b01);
                                mma16816(o[2 * dp + 1], pt0, 0u, pt1, 0u, b10, b11);
                            }
                        }
                    }
                }
            }
            __syncwarp();  // every lane has read this stage
            request();
            if (++us == kStages) {
                us = 0;
                uphase ^= 1u;
            }
        }
        if (!ok) break;
        // ---- the job's state, rows gid < G ----
        const int64_t rows = (int64_t)p.nseq * p.nHead, row = at.c * rows + head;
        float z[4] = {l * 0.f, 0.f, 0.f, 0.f};  // NaN if a sum is not finite
        if (row_ok) {
            if (tq == 0) reinterpret_cast<float2 *>(p.state + p.nchunks * rows * D)[row] = make_float2(m, l);
            float *dst = p.state + row * D;
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt) {
                z[nt & 1] = fmaf(o[nt][0] + o[nt][2], 0.f, z[nt & 1]);
                z[2 + (nt & 1)] = fmaf(o[nt][1] + o[nt][3], 0.f, z[2 + (nt & 1)]);
                if constexpr (C::F32) {
                    const int c = 32 * (nt >> 2) + (nt & 3);  // column of n = 2tq is c + 8tq
                    dst[c + 8 * tq] = o[nt][0] + o[nt][2];
                    dst[c + 8 * tq + 4] = o[nt][1] + o[nt][3];
                } else {
                    *reinterpret_cast<float2 *>(dst + 8 * nt + 2 * tq) = make_float2(o[nt][0] + o[nt][2], o[nt][1] + o[nt][3]);
                }
            }
        }
        const unsigned again = __ballot_sync(0xffffffffu, row_ok && (z[0] + z[1]) + (z[2] + z[3]) != 0.f);
        if (again) {
            __syncwarp();  // these rows are written once more
            const int64_t first = (((int64_t)at.b * p.nHeadKv + at.g) * p.max_len + (int64_t)at.c * p.chunk) * D;
            for (int r = 0; r < p.G; ++r) {
                if (!(again >> (4 * r) & 15u)) continue;
                const int64_t i = (int64_t)at.b * p.nHead + (int64_t)at.g * p.G + r;
                own_again<IO, KV, D>(reinterpret_cast<const IO *>(p.q) + i * D, reinterpret_cast<const KV *>(p.k) + first,
                                     reinterpret_cast<const KV *>(p.v) + first, at.n, p.state + (at.c * rows + i) * D,
                                     reinterpret_cast<float2 *>(p.state + p.nchunks * rows * D) + at.c * rows + i);
            }
        }
        at = start(at.job + stride);
    }
    // an abandoned warp still waits (bounded) for its copies in flight
    if (at.job < jobs)
        for (int i = 0; i < kStages; ++i) {
            mbar_wait(&full[us], uphase, nullptr, nullptr);
            if (++us == kStages) {
                us = 0;
                uphase ^= 1u;
            }
        }
    // Beside a prefix kernel: nothing that it writes is read here, but the merge, which waits for
    // this kernel alone, reads both.
    pdl_wait();
}

template <typename IO, typename KV, int D>
cudaError_t launch_t(const OwnArgs &a, cudaStream_t s) {
    using C = OwnCfg<KV, D>;
    const uint64_t rows = (uint64_t)a.nseq * a.kv.nHeadKv * a.kv.maxLen;
    if (rows + C::T > INT32_MAX) return cudaErrorNotSupported;
    const size_t first = (size_t)a.kv.row(a.layer, a.slot0, 0, 0) * D * sizeof(KV);
    CUtensorMap km, vm;
    if (!map_rows(&km, reinterpret_cast<const uint8_t *>(a.kv.k) + first, rows, D, C::F32, C::T) ||
        !map_rows(&vm, reinterpret_cast<const uint8_t *>(a.kv.v) + first, rows, D, C::F32, C::T))
        return cudaErrorNotSupported;
    OwnParams p;
    p.q = a.q;
    p.k = reinterpret_cast<const uint8_t *>(a.kv.k) + first;
    p.v = reinterpret_cast<const uint8_t *>(a.kv.v) + first;
    p.pos = a.pos;
    p.nseq = a.nseq;
    p.nHead = a.nHead;
    p.nHeadKv = a.kv.nHeadKv;
    p.G = a.nHead / a.kv.nHeadKv;
    p.max_len = a.kv.maxLen;
    p.chunk = a.chunk;
    p.nchunks = a.nchunks;
    p.state = a.state;
    p.err = a.err;
    auto kern = decode_own_kernel<IO, KV, D>;
    static SmemLimit limit;
    const int smem = C::smem(a.nseq);
    const cudaError_t e = allow_smem(kern, smem, limit);
    if (e != cudaSuccess) return e;
    const int64_t jobs = (int64_t)a.nseq * p.nHeadKv * a.nchunks;
    if (jobs > INT32_MAX / 2) return cudaErrorNotSupported;
    // few jobs are spread over as many SMs as there are
    const int grid = (int)(jobs < a.sms ? jobs : a.sms);
    if (a.beside) return launch_pdl(kern, dim3(grid), dim3(kWarps * 32), smem, s, km, vm, p);
    kern<<<grid, kWarps * 32, smem, s>>>(km, vm, p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_decode_own(const OwnArgs &a, cudaStream_t s) {
    using bf16 = __nv_bfloat16;
    const bool kv32 = a.kv.dtype == TL_KV_F32, io32 = a.io == TL_IO_F32;
    if (kv32 && !io32) return cudaErrorNotSupported;
    if (a.kv.headDim == 64)
        return kv32 ? launch_t<float, float, 64>(a, s) : io32 ? launch_t<float, bf16, 64>(a, s) : launch_t<bf16, bf16, 64>(a, s);
    if (a.kv.headDim == 128)
        return kv32 ? launch_t<float, float, 128>(a, s) : io32 ? launch_t<float, bf16, 128>(a, s) : launch_t<bf16, bf16, 128>(a, s);
    return cudaErrorNotSupported;
}

}  // namespace tl
