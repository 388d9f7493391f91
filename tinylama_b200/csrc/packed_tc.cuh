// packed_tc.cuh -- what the two tensor-core kernels for packed batches share: parameters, the start
// of a CTA's share of the work, the end of a piece (partial states, merge, output rows), and the
// checks for values that are not finite.
#pragma once

#include <math.h>

#include "common.cuh"
#include "decode_common.cuh"
#include "internal.h"
#include "packed_sched.cuh"
#include "tc_common.cuh"

namespace tl {
namespace {

constexpr int kStgRow = 80;       // bytes of a staged row: 64 and a pad
constexpr float kRescale = 8.0f;  // log2 units: a sum is rescaled only when its maximum grows past 2^8

// Tile steps that a unit's start and end come to.  At headDim 64 2 (3: 475 us against 462 for 8 documents of up to
// 4096, 32/8 heads, and 110 against 102 for 4 f32 prompts of up to 1024, 32/4), at 128 3 (2: 276 against 257
// for 4 f32 prompts of up to 2048 over a bf16 cache, 32/8).
constexpr int unit_cost(int D) { return D == 64 ? 2 : 3; }

template <int D>
struct PkParams {
    SchedIn<unit_cost(D)> in;
    const void *q;
    void *out;
    int nHead, lg_g;
    int prefix_len, prefix_max_len;
    const void *k, *v;       // own K and V from (layer, slot0) on
    const void *pk, *pv;     // the prefix's K and V
    float *part;             // states of pieces: [2 * gridDim][rows of a unit] of D + 2 values, or of the
                             // parts of a prefix: [splits][ntok * nHead] of them
    unsigned *counter;       // [2 * gridDim], zero between launches
    unsigned *err;
};

// One arrival of a warp whose TMEM accesses are complete (after tcgen05.wait): 32 lanes arriving one by
// one on a barrier take longer than the wait they signal.
__device__ __forceinline__ void warp_arrive(uint64_t *bar, int lane) {
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
}

// ---- start: the line's length and the first sequence of this CTA ----------------------------------

struct SchedStart {
    long long warp_sum[32];
    long long s0;
    int b0;
};

// All THREADS threads.  Returns false when the CTA has no share (the same for all of them).
template <int THREADS, int D>
__device__ __forceinline__ bool sched_begin(const PkParams<D> &p, SchedStart *st, SchedCut<unit_cost(D)> &cut) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;
    if (p.in.cu == nullptr) return true;
    const int per = (p.in.nseq + THREADS - 1) / THREADS;
    const int sq0 = min(tid * per, p.in.nseq), sq1 = min(sq0 + per, p.in.nseq);
    long long mine = 0;
    for (int b = sq0; b < sq1; ++b) {
        const SeqSpan q = sched_seq(p.in, b);
        if (cta == 0 && q.bad_arg) atomicOr(p.err, TL_DEVERR_BAD_ARG);
        if (cta == 0 && q.bad_range) atomicOr(p.err, TL_DEVERR_POS_RANGE);
        mine += sched_seq_steps(p.in, q) * p.in.heads_kv;
    }
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) st->warp_sum[warp] = incl;
    __syncthreads();
    long long total = 0, before = incl - mine;
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += st->warp_sum[w];
        total += st->warp_sum[w];
    }
    cut = sched_cut(p.in, total, gridDim.x);
    const long long lo = cta * cut.share;
    if (lo >= total) return false;
    if (lo >= before && lo < before + mine) {
        long long s = before;
        for (int b = sq0; b < sq1; ++b) {
            const long long e = sched_seq_steps(p.in, sched_seq(p.in, b)) * p.in.heads_kv;
            if (lo < s + e) {
                st->b0 = b;
                st->s0 = s;
                break;
            }
            s += e;
        }
    }
    return true;  // b0 and s0 are there after the next __syncthreads
}

// ---- pieces, handed to the warps of a CTA through shared memory ----------------------------------------
// Warp 0 derives the CTA's pieces and publishes them; the others read them from here, so that none
// of them carries the schedule's state in registers.  One warp takes a slot with get() and gives it
// back with put(); w < 0 marks the end.
constexpr int kRing = 4;
template <int CONSUMERS>
struct PieceRing {
    uint64_t full[kRing], empty[kRing];
    Piece slot[kRing];
    unsigned bad[kRing][2];  // see clean_rows
    __device__ __forceinline__ void init() {
        for (int i = 0; i < kRing; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], CONSUMERS);
        }
    }
    // by a whole warp, `leader` set in one lane; false if the wait gave up
    __device__ __forceinline__ bool publish(int it, const Piece &pc, uint32_t leader, unsigned *err, volatile int *ab) {
        const int i = it % kRing;
        if (!__all_sync(0xffffffffu, mbar_wait(&empty[i], ((it / kRing) & 1) ^ 1, err, ab))) return false;
        if (leader) {
            slot[i] = pc;
            bad[i][0] = bad[i][1] = 0u;
            mbar_arrive(&full[i]);
        }
        __syncwarp();
        return true;
    }
    // by a whole warp; nullptr at the end or if the wait gave up (*ok false then)
    __device__ __forceinline__ const Piece *get(int it, unsigned *err, volatile int *ab, bool *ok) {
        const int i = it % kRing;
        if (!__all_sync(0xffffffffu, mbar_wait(&full[i], (it / kRing) & 1, err, ab))) {
            *ok = false;
            return nullptr;
        }
        return slot[i].w < 0 ? nullptr : &slot[i];
    }
    // a bit for every 1/64 of a piece's tiles (at least one): the word and the bit of tile j
    __device__ __forceinline__ static int bad_step(const Piece &pc) { return (pc.j1 - pc.j0 + 63) >> 6; }
    __device__ __forceinline__ unsigned *bad_word(int it, const Piece &pc, int j, unsigned &bit) {
        const int b = (j - pc.j0) / bad_step(pc);
        bit = 1u << (b & 31);
        return &bad[it % kRing][b >> 5];
    }
    __device__ __forceinline__ void put(int it, int lane) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[it % kRing]);
    }
};

// ---- end of a piece ---------------------------------------------------------------------------------

// Columns col0 .. col0+W-1 of rows r (packed [token][head] row row_at(r)) of a warp's 32, times inv, through `stg`
// (32 staged rows), 64 bytes of a row at a time; live(r) says which rows exist.
template <int D, int W, typename OUT, typename At, typename Live>
__device__ __forceinline__ void store_rows(OUT *out, const float (&o)[W], float inv, int row, int col0, uint8_t *stg,
                                           At row_at, Live live) {
    constexpr int N = 64 / (int)sizeof(OUT);  // columns per turn
    const int row0 = row & ~31, lane = row & 31;
    int64_t at[4];
    bool have[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int r = row0 + k * 8 + (lane >> 2);
        have[k] = live(r);
        at[k] = row_at(r) * D + col0 + N / 4 * (lane & 3);
    }
#pragma unroll
    for (int c = 0; c < W / N; ++c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint4 u;
            if constexpr (sizeof(OUT) == 4) {
                u = make_uint4(__float_as_uint(o[N * c + 4 * i] * inv), __float_as_uint(o[N * c + 4 * i + 1] * inv),
                               __float_as_uint(o[N * c + 4 * i + 2] * inv), __float_as_uint(o[N * c + 4 * i + 3] * inv));
            } else {
                u = make_uint4(pack_bf16(o[N * c + 8 * i] * inv, o[N * c + 8 * i + 1] * inv),
                               pack_bf16(o[N * c + 8 * i + 2] * inv, o[N * c + 8 * i + 3] * inv),
                               pack_bf16(o[N * c + 8 * i + 4] * inv, o[N * c + 8 * i + 5] * inv),
                               pack_bf16(o[N * c + 8 * i + 6] * inv, o[N * c + 8 * i + 7] * inv));
            }
            *reinterpret_cast<uint4 *>(stg + lane * kStgRow + 16 * i) = u;
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (have[k])
                *reinterpret_cast<uint4 *>(out + at[k] + N * c) =
                    *reinterpret_cast<const uint4 *>(stg + (k * 8 + (lane >> 2)) * kStgRow + 16 * (lane & 3));
        __syncwarp();
    }
}

// 16 bytes of a row as floats
template <typename T, int N>
__device__ __forceinline__ void load_floats(const T *p, float (&x)[N]) {
    const uint4 u = __ldg(reinterpret_cast<const uint4 *>(p));
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

// Values that are not finite.  In the matrix products a value of V that is infinite or not a number reaches every
// row of its tile: the weight of a row that does not see the key is zero, but zero times infinity is
// not.  So such values are set to zero in shared memory before the product, and their tile is marked; when a piece
// ends, each row adds those that it sees to its sum as they are (put_back).  Looked over are the keys that
// not every row of the unit sees, at most as many as the unit has tokens: the others are right as they are.  Of
// f32 activations over a bf16 cache all keys are: their weights come in parts of either sign, which makes NaN of
// an infinity also for the rows that see it.
// So the cost is bounded whatever the values.  8 documents of up to 4096 (32/8/64 bf16): a NaN in each one's first
// position takes no time (summing the rows again on the CUDA cores, each over all its keys, took 80 ms), NaN
// everywhere 1.2 ms instead of 0.47; the most is a bf16 cache under f32 activations, 4 prompts of up to 1024 (32/4/64):
// 14 times the 80 us with one such value in every tile of V, 29 times with a minus infinity in every key.

// four words of two bf16 values each: not a number (in one of two halves) if one of them is not finite
__device__ __forceinline__ uint32_t not_finite(uint4 u, uint32_t z) {
    const __nv_bfloat162 zero = __floats2bfloat162_rn(0.f, 0.f);
    __nv_bfloat162 a = *reinterpret_cast<__nv_bfloat162 *>(&z);
    a = __hfma2(*reinterpret_cast<__nv_bfloat162 *>(&u.x), zero, a);
    a = __hfma2(*reinterpret_cast<__nv_bfloat162 *>(&u.y), zero, a);
    a = __hfma2(*reinterpret_cast<__nv_bfloat162 *>(&u.z), zero, a);
    a = __hfma2(*reinterpret_cast<__nv_bfloat162 *>(&u.w), zero, a);
    return *reinterpret_cast<uint32_t *>(&a);
}
constexpr uint32_t kNotZero = 0x7fff7fffu;  // bits of such a word that a zero of either sign does not have

// bits of the values of a pair that are finite
__device__ __forceinline__ uint32_t finite_halves(uint32_t u) {
    return ((u & 0x7f80u) != 0x7f80u ? 0xffffu : 0u) | ((u & 0x7f800000u) != 0x7f800000u ? 0xffff0000u : 0u);
}

// Rows r0 .. r1-1 of a bf16 V tile, by a warp (two may do it at a time): values that are not finite to zero, and
// the tile's mark.  UNROLL > 1 takes fewer turns, but more of the instruction cache: bf16, 8 documents of up
// to 4096 (32/8/64) take 461 us with 1, 501 with 2, 512 with 4.
template <int HALVES, int BOX, int UNROLL>
__device__ __forceinline__ void clean_rows(uint8_t *tile, int r0, int r1, unsigned *word, unsigned bit) {
    const int lane = threadIdx.x & 31;
    uint32_t z[2] = {0u, 0u};
#pragma unroll
    for (int hh = 0; hh < HALVES; ++hh)
#pragma unroll UNROLL
        for (int e = r0 * 8 + lane; e < r1 * 8; e += 32)
            z[hh] = not_finite(*reinterpret_cast<const uint4 *>(tile + hh * BOX + e * 16), z[hh]);
    // (marked already: by the other warp, whose zeros this one may have found; they go to the product by this fence)
    if (__any_sync(0xffffffffu, ((z[0] | z[1]) & kNotZero) != 0u || (*reinterpret_cast<volatile unsigned *>(word) & bit))) {
        if (lane == 0) atomicOr(word, bit);
        __threadfence_block();  // the mark before the zeros
        __syncwarp();
#pragma unroll 1
        for (int hh = 0; hh < HALVES; ++hh)
#pragma unroll 1
            for (int e = r0 * 32 + lane; e < r1 * 32; e += 32) {
                uint32_t *w = reinterpret_cast<uint32_t *>(tile + hh * BOX + e * 4);
                const uint32_t keep = finite_halves(*w);
                if (keep != ~0u) *w &= keep;
            }
        fence_proxy_async_smem();
        __syncwarp();
    }
}

// The same for a V tile in three parts, without the mark: of a value that is not finite, the third part is not.
template <int HALVES, int BOX, int PART>
__device__ __noinline__ void clean_parts(uint8_t *tile, int r0, int r1) {
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int hh = 0; hh < HALVES; ++hh)
#pragma unroll 1
        for (int e = r0 * 32 + lane; e < r1 * 32; e += 32) {
            uint32_t *w = reinterpret_cast<uint32_t *>(tile + hh * BOX + e * 4);
            const uint32_t keep = finite_halves(w[2 * PART / 4]);
            if (keep == ~0u) continue;
            for (int k = 0; k < 3; ++k) w[k * PART / 4] &= keep;
        }
    fence_proxy_async_smem();
    __syncwarp();
}

// The cleaned values that row `row` of the unit sees, columns col0 .. col0+W-1, into its sum.  (Their weight
// is taken as positive: one that underflows to zero would make NaN of an infinity.)
template <int D, int W, bool ALL, typename KV>
__device__ __forceinline__ void put_back(const PkParams<D> &p, const Piece &pc, const volatile unsigned *bad, int step, int row,
                                         int col0, float (&o)[W]) {
    constexpr int NK = 16 / (int)sizeof(KV);
    const unsigned w0 = bad[0], w1 = bad[1];
    if ((w0 | w1) == 0u) return;
    const int tok = row >> p.lg_g;
    if (tok >= pc.ntok) return;
    for (int j = pc.j0; j < pc.j1; ++j) {
        const int b = (j - pc.j0) / step;
        if (!((b < 32 ? w0 : w1) >> (b & 31) & 1u)) continue;
        const bool pre = j < p.in.prefix_tiles;
        const int k0 = (pre ? j : j - p.in.prefix_tiles) << p.in.lg_kt;
        const int n = min(1 << p.in.lg_kt, (pre ? p.prefix_len : pc.pos + tok + 1) - k0);
        const int64_t first = (pre ? (int64_t)pc.g * p.prefix_max_len : ((int64_t)pc.b * p.in.heads_kv + pc.g) * p.in.max_len) + k0;
        const KV *v = reinterpret_cast<const KV *>(pre ? p.pv : p.v) + first * D + col0;
        for (int i = ALL ? 0 : pre ? n : max(pc.pos + 1 - k0, 0); i < n; ++i) {
#pragma unroll
            for (int d = 0; d < W; d += NK) {
                float x[NK];
                load_floats<KV, NK>(v + (int64_t)i * D + d, x);
#pragma unroll
                for (int c = 0; c < NK; ++c) o[d + c] += fabsf(x[c]) < INFINITY ? 0.f : x[c];
            }
        }
    }
}

// Is the score of q and a key that has come out not a number minus infinity?  Only elements of the key that
// are not finite count.
template <int D, typename KV>
__device__ __noinline__ bool weightless(const float *q, const KV *k) {
    constexpr int NK = 16 / (int)sizeof(KV);
    float s = 0.f;
#pragma unroll 1
    for (int d = 0; d < D; d += NK) {
        float x[NK];
        load_floats<KV, NK>(k + d, x);
#pragma unroll
        for (int c = 0; c < NK; ++c)
            if (!(fabsf(x[c]) < INFINITY)) s = fmaf(q[d + c], x[c], s);
    }
    return s == -INFINITY;
}

// Called by 128 threads that hold columns col0 .. col0+W-1 of rows 128*n .. 128*n+127 of a unit of ROWS
// rows: thread `row` has (o, m, l).  A piece that is not the whole unit leaves its state in p.part;
// the last piece of the unit to arrive (counter q of the unit's; nothing waits) merges them in the
// unit's order, so the result does not depend on who is last.  Parts of a prefix leave their states row
// by row for the merge kernel.  sync() is a bounded barrier of the 128 threads.
template <int D, int W, typename OUT, int ROWS, typename Sync>
__device__ __forceinline__ bool finish_rows(const PkParams<D> &p, const SchedCut<unit_cost(D)> &cut, const Piece &pc, int q, int row, int col0,
                                            float (&o)[W], float m, float l, Sync sync, volatile int *last_flag,
                                            uint8_t *stg) {
    const int cta = blockIdx.x;
    auto row_at = [&](int r) {
        return (int64_t)(pc.tok0 + (r >> p.lg_g)) * p.nHead + (pc.g << p.lg_g) + (r & ((1 << p.lg_g) - 1));
    };
    auto live = [&](int r) { return (r >> p.lg_g) < pc.ntok; };
    if (p.in.cu == nullptr) {
        const int64_t rows = (int64_t)p.in.ntok * p.nHead, first = pc.start * rows;
        store_rows<D, W>(p.part + first * D, o, 1.f, row, col0, stg, row_at, live);
        if (live(row) && col0 == 0)
            reinterpret_cast<float2 *>(p.part + p.in.splits * rows * D)[first + row_at(row)] = make_float2(m, l);
        return true;
    }
    if (!pc.whole()) {
        int first = -1, slot = -1;
        const int n = sched_pieces(cut, pc.start, pc.w, [&](int c, int s) {
            if (first < 0) first = c;
            if (c == cta) slot = s;
        });
        // [slot][D/4][ROWS] float4, then (m, l) as [slot][column half][ROWS]
        const int64_t c4 = col0 / 4, half = col0 > 0;
        float4 *dst = reinterpret_cast<float4 *>(p.part) + ((int64_t)slot * (D / 4) + c4) * ROWS + row;
        float2 *ml = reinterpret_cast<float2 *>(p.part + (int64_t)2 * gridDim.x * D * ROWS) + half * ROWS + row;
#pragma unroll
        for (int d = 0; d < W; d += 4) __stcg(dst + (d / 4) * ROWS, make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]));
        __stcg(ml + (int64_t)slot * 2 * ROWS, make_float2(m, l));
        __threadfence();
        if (!sync()) return false;
        if ((row & 127) == 0) {
            const unsigned old = atomicAdd(&p.counter[2 * first + q], 1u);
            *last_flag = old == (unsigned)(n - 1);
            if (old == (unsigned)(n - 1)) p.counter[2 * first + q] = 0u;
        }
        if (!sync()) return false;
        const bool last = *last_flag != 0;
        if (!sync()) return false;  // the flag is read before the next piece writes it
        if (!last) return true;
        __threadfence();
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int d = 0; d < W; ++d) o[d] = 0.f;
        // with a running maximum: one pass, a piece's (m, l) and values in flight together
        sched_pieces(cut, pc.start, pc.w, [&](int, int s) {
            const float2 x = __ldcg(ml + (int64_t)s * 2 * ROWS);
            const float4 *src = reinterpret_cast<const float4 *>(p.part) + ((int64_t)s * (D / 4) + c4) * ROWS + row;
            // 128 columns: eight loads kept ahead (685 us against 700 for 6 prompts of up to 4096 behind 1000);
            // 64: left to the compiler (459 against 490, 8 documents of up to 4096)
            constexpr bool AHEAD = W > 64;
            float4 v[8];
            if constexpr (AHEAD) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = __ldcg(src + i * ROWS);
            }
            const float M = fmaxf(m, x.x), w0 = safe_exp2_diff(m, M), w = safe_exp2_diff(x.x, M);
            m = M;
            l = fmaf(x.y, w, l * w0);
#pragma unroll
            for (int d0 = 0; d0 < W; d0 += 32) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int d = d0 + 4 * i;
                    const float4 u = AHEAD ? v[i] : __ldcg(src + (d / 4) * ROWS);
                    if (AHEAD && d0 + 32 < W) v[i] = __ldcg(src + (d / 4 + 8) * ROWS);
                    o[d] = fmaf(u.x, w, o[d] * w0);
                    o[d + 1] = fmaf(u.y, w, o[d + 1] * w0);
                    o[d + 2] = fmaf(u.z, w, o[d + 2] * w0);
                    o[d + 3] = fmaf(u.w, w, o[d + 3] * w0);
                }
            }
        });
    }
    store_rows<D, W>(reinterpret_cast<OUT *>(p.out), o, l > 0.f ? 1.f / l : l /* NaN stays */, row, col0, stg, row_at, live);
    return true;
}

// ---- tensor maps (host) ----------------------------------------------------------------------------

int ilog2(int x) {
    int n = 0;
    while (x > 1) x >>= 1, ++n;
    return n;
}

// Parameters of a call; rows = rows of a unit, kt = keys of a tile.  False if a coordinate would
// not fit.  The maps and pointers cover this call's slots only, so row numbers stay small however
// large the cache is.
template <int D>
bool pk_params(const PackedArgs &a, int rows, int kt, PkParams<D> &p) {
    const int G = a.nHead / a.nHeadKv;
    const size_t es = a.kv.dtype == TL_KV_BF16 ? 2 : 4;
    const uint64_t own_rows = (uint64_t)(a.cu ? a.nseq : 1) * a.nHeadKv * a.kv.maxLen;
    const uint64_t pre_rows = (uint64_t)a.nHeadKv * a.pkv.maxLen;
    if (own_rows + kt > INT32_MAX || pre_rows + kt > INT32_MAX) return false;
    const size_t own0 = (size_t)a.kv.row(a.layer, a.slot0, 0, 0) * a.headDim * es;
    const size_t pre0 = (size_t)a.pkv.row(a.layer, a.prefix_slot, 0, 0) * a.headDim * es;
    p = PkParams<D>{};
    p.in.cu = a.cu;
    p.in.ctas = a.ctas;
    p.in.splits = a.splits;
    p.in.pos0 = a.pos0;
    p.in.nseq = a.cu ? a.nseq : 1;
    p.in.ntok = a.ntok;
    p.in.heads_kv = a.nHeadKv;
    p.in.max_len = a.kv.maxLen;
    p.in.lg_kt = ilog2(kt);
    p.in.lg_tb = ilog2(rows / G);
    p.in.prefix_tiles = (a.prefix_len + kt - 1) / kt;
    p.q = a.q;
    p.out = a.out;
    p.nHead = a.nHead;
    p.lg_g = ilog2(G);
    p.prefix_len = a.prefix_len;
    p.prefix_max_len = a.pkv.maxLen;
    p.k = reinterpret_cast<const uint8_t *>(a.kv.k) + own0;
    p.v = reinterpret_cast<const uint8_t *>(a.kv.v) + own0;
    p.pk = reinterpret_cast<const uint8_t *>(a.pkv.k) + pre0;
    p.pv = reinterpret_cast<const uint8_t *>(a.pkv.v) + pre0;
    p.part = a.part;
    p.counter = a.counter;
    p.err = a.err;
    return true;
}

}  // namespace
}  // namespace tl
