// packed_tc32.cu -- attention of packed f32 query rows with 32-bit products, on the bf16 tensor cores.
//
// The same operator as packed_tc.cu for f32 activations, over an f32 or a bf16 cache.  A float32 x is the
// sum of three bf16 values, x = x1 + x2 + x3, each the rounding of what the ones before leave (8
// bits of the 24 apiece), and a product of two such sums needs the six terms above 2^-24:
//   x y = x1 y1 + (x1 y2 + x2 y1) + (x1 y3 + x2 y2 + x3 y1)
// (a bf16 cache value is exact in one part: three terms).  Six bf16 products on the tensor cores are
// 280 TFLOP/s at the measured peak, against about 70 for fp32 multiply-adds on the CUDA cores.  The
// small terms are summed first, while the fp32 accumulator is small, and the sums over the keys
// leave the tensor core after every tile and are carried in registers with rounded additions, so
// no long chain of accumulations of the tensor core enters the result.
//
// A unit is 128 rows (the G heads of a kv-head for 128/G tokens); shares of the work as in
// packed_tc.cu.  The A operand of both products comes from TMEM: a thread of the softmax
// warpgroup holds one row, splits its q (scaled by log2(e)/sqrt(D)) and its weights into parts, and
// stores them to the lanes it owns.  So shared memory holds K and V only.  Tiles are 8192 values: 128
// keys of 64 or 64 keys of 128.  TMEM columns: Q parts 3 D/2, S kt, P parts 3 kt/2, T (= P V of
// one tile) D: 480 for both head sizes.
//   warp 0     derives the pieces of work, and brings K and V tiles of a bf16 cache (TMA)
//   warp 1     issues S(j+1) = Q K^T, then T(j) = P V
//   warp 3     bf16 cache: zeroes the rows of a V tile that hold leftovers, and values that are not finite;
//              f32 cache: looks over, in the cache, the new V rows of which not every row of a unit sees all, and
//              tells warp 1, which cleans the tile (once for each such tile: with a turn of this warp on every tile
//              the softmax lost issue slots to it, 111 us against 104, 4 prompts of up to 1024, 32/4/64)
//   warps 4-7  f32 cache: read K and V, split them and write the parts in the swizzled layout (8 warps for
//              it took registers from the softmax: 557 us against 451, 8 x up to 2048, 32/8/64)
//   the last 8 softmax, two threads a row (half the keys of a tile, and half the columns of T, each; they
//              exchange the tile's maximum): S(j) to registers (which frees S for j+1), weights, then, once
//              T(j-1) is there, o += T(j-1) and P(j) to TMEM.  With one thread a row its chain of
//              instructions, 7700 clocks a tile, was what took the time; the products take 3100.
// While the group works on one tile the tensor core has S of the next one to do, and each piece's q
// is in place before the one ahead has been written out.
//
// Measured: 103 us for 4 prompts of up to 1024 (32/4/64), 450 for 8 of up to 2048 (32/8/64), 455 for 4 of up to 2048
// (32/8/128), and over a bf16 cache 76 for the first and 260 for the last.  The tensor pipe is 36% busy in the
// first (46% on the busiest SM) and waits for the parts that the softmax threads write.
//
// Masked keys and leftovers: V rows that no row of the unit sees are zero in shared memory.  Values of the
// sequence itself that are not finite: an f32 cache's infinities go through the products as what they are
// (split3_cache), a bf16 cache's meet parts of either sign and are looked after (clean_rows in packed_tc.cuh for V,
// keep_weights for K).
#include <type_traits>

#include "packed_tc.cuh"

namespace tl {
namespace {

template <int D, bool KV32>
struct P32 {
    static constexpr int KT = D == 64 ? 128 : 64;    // keys per tile
    static constexpr int NP = KV32 ? 3 : 1;          // parts of a cache value
    static constexpr int HALVES = D / 64;
    static constexpr int BOX = KT * 128;             // 64 columns of a tile
    static constexpr int PART = HALVES * BOX;        // 16 KB: one part of a tile
    static constexpr int TILE = NP * PART;
    static constexpr int NS = KV32 ? 2 : 4;
    static constexpr int CONV = KV32 ? 128 : 0;      // threads that split K and V
    static constexpr int THREADS = 384 + CONV;
    static constexpr int SOFT0 = THREADS / 32 - 8;   // first softmax warp
    static constexpr int CONSUMERS = 1 + 1 + CONV / 32 + 8;  // warps that read the ring of pieces
    static constexpr int OFF_V = NS * TILE;
    static constexpr int OFF_STG = 2 * NS * TILE;
    static constexpr int OFF_BARS = OFF_STG + 8 * 32 * kStgRow;
    static constexpr int COL_Q = 0, COL_S = 3 * D / 2, COL_P = COL_S + KT, COL_T = COL_P + 3 * KT / 2;
    static_assert(COL_T + D <= 512, "TMEM columns");
    // registers of the warpgroups: dec only goes down and inc only up, and together they stay within the
    // launch's.  112 for the warps that split an f32 cache at headDim 128 (4 prompts of up to 2048, 32/8: 452 us
    // against 482 with 104), 104 at 64 (8 of up to 2048, 32/8: 437 against 441 with 112).
    static constexpr int REG_LAUNCH = 65536 / THREADS / 8 * 8, REG_CTRL = KV32 ? 64 : 104, REG_CONV = D == 64 ? 104 : 112,
                         REG_SOFT = KV32 ? 168 : 200;
    static_assert(REG_CTRL <= REG_LAUNCH && REG_CONV <= REG_LAUNCH && REG_SOFT >= REG_LAUNCH, "direction of the change");
    static_assert(REG_CTRL + CONV / 128 * REG_CONV + 2 * REG_SOFT <= THREADS / 128 * REG_LAUNCH,
                  "register split exceeds the launch");
};

template <int D, bool KV32>
struct P32Bars {
    static constexpr int NS = P32<D, KV32>::NS;
    uint64_t k_full[NS], k_empty[NS], v_raw[NS], v_full[NS], v_empty[NS];
    uint64_t v_clean, v_taken, q_ready, s_full, s_free, p_ready, o_bar, x_bar, g_bar[2], mma_final;
    PieceRing<P32<D, KV32>::CONSUMERS> ring;
    SchedStart start;
    uint32_t tmem_base;
    int abort;
    int last_flag[2];
    volatile int verdict;  // rows of a V tile that are to be cleaned, or 0
    float xch[2][2][BM];  // a row's maximum (or sum) over each half of the keys, two turns of it
};

// one K = 16 step, A from TMEM
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate,
                                       uint32_t issue) {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\t"
        "setp.ne.b32 e, %5, 0;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(issue)
        : "memory");
}

// parts of a pair of floats as packed bf16
__device__ __forceinline__ void split3(float x0, float x1, uint32_t &a, uint32_t &b, uint32_t &c) {
    a = pack_bf16(x0, x1);
    const float2 r = fsub2(make_float2(x0, x1), make_float2(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u)));
    b = pack_bf16(r.x, r.y);
    const float2 q = fsub2(r, make_float2(__uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u)));
    c = pack_bf16(q.x, q.y);
}

// The same for values of the cache, of which an infinity has to stay one: the first two parts are clamped to the
// largest bf16 value, so that only the third is infinite.  It meets only the first part of q or of the weights,
// whose sign is theirs: a score or a sum comes out as the infinity that it is.  (A finite value that rounds to
// infinity in bf16 is the exact sum of its clamped parts.)
__device__ __forceinline__ uint32_t pack_clamped(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void split3_cache(float x0, float x1, uint32_t &a, uint32_t &b, uint32_t &c) {
    a = pack_clamped(x0, x1);
    const float2 r = fsub2(make_float2(x0, x1), make_float2(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u)));
    b = pack_clamped(r.x, r.y);
    const float2 q = fsub2(r, make_float2(__uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u)));
    c = pack_bf16(q.x, q.y);
}

// A row's weights w of KH keys, of which some are not a number (`lost`; all lanes of the warp take part).  Such a
// key has no weight if its score is minus infinity; then w and their sum are put right, and the result is true.
// Otherwise the row has no softmax: the sum stays what it is, and the row is not looked at again.
template <int D, int KH, typename KV>
__device__ __noinline__ bool keep_weights(uint32_t *w, bool lost, const float *q, const KV *k, float &sum) {
    bool none = false;
    float s = 0.f;
#pragma unroll 1
    for (int c = 0; c < KH; ++c) {
        const float x = __uint_as_float(w[c]);
        const bool mine = lost && x != x;
        if (__any_sync(0xffffffffu, mine && !none)) {
            const bool out = weightless<D, KV>(q, k + (int64_t)c * D);
            none |= mine && !out;
        }
        if (mine) w[c] = 0u;
        else s += x;
    }
    if (!lost || none) return false;
    sum = s;
    return true;
}

// The terms of a product, small ones first: the parts of A and of B, four bits each from the low end.
// The loop over them is not unrolled: with every term of both products written out (and the other
// long loops of this kernel) the code outgrew the instruction caches, and waiting for instructions
// took three times the issue slots.
template <int NP>
struct Terms {
    static constexpr int N = NP == 3 ? 6 : 3;
    static constexpr uint32_t A = NP == 3 ? 0x001102u : 0x012u, B = NP == 3 ? 0x010120u : 0u;
};

// the parts of D/2 values of a row of q, times scale, into TMEM: D/4 columns from `col`, + D/2 and + D
template <int D>
__device__ __noinline__ void store_q(const float *src, bool live, float scale, uint32_t col) {
#pragma unroll 1
    for (int c = 0; c < D / 64; ++c) {
        uint32_t a[16], b[16], d[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (live) x = __ldg(reinterpret_cast<const float4 *>(src + 32 * c + 4 * i));
            split3(x.x * scale, x.y * scale, a[2 * i], b[2 * i], d[2 * i]);
            split3(x.z * scale, x.w * scale, a[2 * i + 1], b[2 * i + 1], d[2 * i + 1]);
        }
        TL_ST16(col + 16 * c, a);
        TL_ST16(col + D / 2 + 16 * c, b);
        TL_ST16(col + D + 16 * c, d);
    }
    tmem_wait_st();
}

template <int D, bool KV32>
__global__ void __launch_bounds__((P32<D, KV32>::THREADS), 1)
packed_tc32_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                   const __grid_constant__ CUtensorMap pkmap, const __grid_constant__ CUtensorMap pvmap, const PkParams<D> p) {
    using C = P32<D, KV32>;
    using B_ = P32Bars<D, KV32>;
    using KV = std::conditional_t<KV32, float, __nv_bfloat16>;
    constexpr int NS = C::NS, KT = C::KT;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t *base = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    uint8_t *sK = base, *sV = base + C::OFF_V;
    B_ *bars = reinterpret_cast<B_ *>(base + C::OFF_BARS);
    volatile int *abort_flag = &bars->abort;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(&bars->k_full[i], KV32 ? C::CONV / 32 : 1);
            mbar_init(&bars->k_empty[i], 1);
            mbar_init(&bars->v_raw[i], 1);
            mbar_init(&bars->v_full[i], KV32 ? C::CONV / 32 : 1);
            mbar_init(&bars->v_empty[i], 1);
        }
        mbar_init(&bars->v_clean, 1);
        mbar_init(&bars->v_taken, 1);
        mbar_init(&bars->q_ready, 8);
        mbar_init(&bars->s_full, 1);
        mbar_init(&bars->s_free, 8);
        mbar_init(&bars->p_ready, 8);
        mbar_init(&bars->o_bar, 1);
        mbar_init(&bars->x_bar, 8);
        mbar_init(&bars->g_bar[0], BM);
        mbar_init(&bars->g_bar[1], BM);
        mbar_init(&bars->mma_final, 1);
        bars->ring.init();
        bars->abort = 0;
        bars->start.b0 = p.in.nseq;
        bars->start.s0 = 0;
        fence_mbar_init();
    }
    if (p.in.cu == nullptr) pdl_launch_dependents();  // the own positions' kernel runs beside this one
    SchedCut<unit_cost(D)> cut;
    if (!sched_begin<C::THREADS>(p, &bars->start, cut)) return;
    if (warp == 1) {
        tmem_alloc(&bars->tmem_base, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars->tmem_base;
    auto wait_all = [&](uint64_t *bar, uint32_t parity, unsigned *err, volatile int *ab) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, ab));
    };
    // keys [k0, k0 + KT) of tile j: the first row of its cache, k0, how many of them some row of the
    // unit sees, and the first key (from k0) that not every row sees
    struct TileAt {
        int64_t row;
        int k0, n, all;
        bool pre;
    };
    auto tile_at = [&](const Piece &pc, int j) {
        TileAt t;
        t.pre = j < p.in.prefix_tiles;
        t.k0 = (t.pre ? j : j - p.in.prefix_tiles) * KT;
        t.row = (t.pre ? (int64_t)pc.g * p.prefix_max_len : ((int64_t)pc.b * p.in.heads_kv + pc.g) * p.in.max_len) + t.k0;
        t.n = min(KT, (t.pre ? p.prefix_len : pc.pos + pc.ntok) - t.k0);
        t.all = t.pre ? KT : pc.pos + 1 - t.k0;
        return t;
    };

    // the first tile of which not every row of the unit sees every key
    auto first_diagonal = [&](const Piece &pc) {
        return p.in.cu != nullptr && pc.ntok > 1 ? p.in.prefix_tiles + ((pc.pos + 1) >> p.in.lg_kt) : pc.j1;
    };

    if (warp < 4) {
        setmaxnreg_dec<C::REG_CTRL>();
        const uint32_t leader = elect_one();
        if (warp == 0) {
            // ---------------- pieces, and the tiles of a bf16 cache (TMA) ----------------
            SchedIter<unit_cost(D)> iter;
            iter.init(p.in, cut, blockIdx.x, bars->start.b0, bars->start.s0);
            int kvit = 0, it = 0;
            bool ok = true;
            Piece pc;
            while (ok && iter.next(p.in, pc)) {
                if (!bars->ring.publish(it, pc, leader, p.err, abort_flag)) { ok = false; break; }
                ++it;
                if constexpr (!KV32) {
                    for (int j = pc.j0; j < pc.j1; ++j, ++kvit) {
                        const TileAt t = tile_at(pc, j);
                        const CUtensorMap *km = t.pre ? &pkmap : &kmap, *vm = t.pre ? &pvmap : &vmap;
                        const int st = kvit % NS;
                        const uint32_t par = ((kvit / NS) & 1) ^ 1;
                        if (!wait_all(&bars->k_empty[st], par, p.err, abort_flag)) { ok = false; break; }
                        if (leader) mbar_arrive_expect_tx(&bars->k_full[st], C::TILE);
                        __syncwarp();
#pragma unroll
                        for (int hh = 0; hh < C::HALVES; ++hh)
                            tma_load_2d(sK + st * C::TILE + hh * C::BOX, km, 64 * hh, (int)t.row, &bars->k_full[st], leader);
                        if (!wait_all(&bars->v_empty[st], par, p.err, abort_flag)) {
                            wait_all(&bars->k_full[st], (kvit / NS) & 1, nullptr, nullptr);  // the K in flight
                            ok = false;
                            break;
                        }
                        if (leader) mbar_arrive_expect_tx(&bars->v_raw[st], C::TILE);
                        __syncwarp();
#pragma unroll
                        for (int hh = 0; hh < C::HALVES; ++hh)
                            tma_load_2d(sV + st * C::TILE + hh * C::BOX, vm, 64 * hh, (int)t.row, &bars->v_raw[st], leader);
                    }
                }
            }
            pc.w = -1;
            if (ok) bars->ring.publish(it, pc, leader, p.err, abort_flag);
            for (int j = max(0, kvit - NS); j < kvit; ++j) {
                wait_all(&bars->k_full[j % NS], (j / NS) & 1, nullptr, nullptr);
                wait_all(&bars->v_raw[j % NS], (j / NS) & 1, nullptr, nullptr);
            }
        } else if (warp == 1) {
            // ---------------- MMA issuer ----------------
            const uint32_t idesc_s = idesc_bf16(KT, false), idesc_o = idesc_bf16(D, true);
            using T_ = Terms<C::NP>;
            int it = 0, ks = 0, ps = 0;  // pieces, S tiles issued, P V tiles issued
            int diag = 0;                // tiles that warp 3 has had a say on
            bool ok = true;
            // S of the next tile
            auto issue_s = [&]() {
                const int st = ks % NS;
                if (!wait_all(&bars->k_full[st], (ks / NS) & 1, p.err, abort_flag)) return false;
                if (ks > 0 && !wait_all(&bars->s_free, (ks - 1) & 1, p.err, abort_flag)) return false;
                tc_fence_after();
                const uint32_t ka = smem_u32(sK + st * C::TILE);
#pragma unroll 1
                for (int t = 0; t < T_::N; ++t) {
                    const uint32_t qa = tmem + C::COL_Q + ((T_::A >> (4 * t)) & 3u) * (D / 2);
                    const uint64_t kd = sw128_desc(ka + ((T_::B >> (4 * t)) & 3u) * C::PART, 16);
#pragma unroll
                    for (int s = 0; s < D / 16; ++s)
                        mma_ts(tmem + C::COL_S, qa + 8 * s, kd + (s / 4) * (C::BOX / 16) + 2 * (s % 4), idesc_s,
                               (t > 0 || s > 0) ? 1u : 0u, leader);
                }
                tc_commit(&bars->s_full, leader);
                tc_commit(&bars->k_empty[st], leader);
                ++ks;
                return true;
            };
            for (; ok; ++it) {
                const Piece *slot = bars->ring.get(it, p.err, abort_flag, &ok);
                if (!slot) break;
                const int n = slot->j1 - slot->j0;
                const int clean = KV32 ? first_diagonal(*slot) - slot->j0 : n;  // the first tile that warp 3 has a say on
                bars->ring.put(it, lane);
                ok = wait_all(&bars->q_ready, it & 1, p.err, abort_flag);
                if (!ok) break;
                ok = issue_s();
                for (int j = 0; j < n && ok; ++j) {
                    if (j + 1 < n) ok = issue_s();
                    if (!ok) break;
                    const int st = ps % NS;
                    ok = wait_all(&bars->v_full[st], (ps / NS) & 1, p.err, abort_flag);
                    if (ok && j >= clean) {
                        ok = wait_all(&bars->v_clean, diag++ & 1, p.err, abort_flag);
                        const int verdict = bars->verdict;
                        __syncwarp();
                        if (ok && leader) mbar_arrive(&bars->v_taken);
                        if (ok && verdict != 0) clean_parts<C::HALVES, C::BOX, C::PART>(sV + st * C::TILE, verdict >> 16, verdict & 0xffff);
                    }
                    if (ok) ok = wait_all(&bars->p_ready, ps & 1, p.err, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t va = smem_u32(sV + st * C::TILE);
#pragma unroll 1
                    for (int t = 0; t < T_::N; ++t) {
                        const uint32_t pa = tmem + C::COL_P + ((T_::A >> (4 * t)) & 3u) * (KT / 2);
                        const uint64_t vd = sw128_desc(va + ((T_::B >> (4 * t)) & 3u) * C::PART, C::BOX);
#pragma unroll
                        for (int s = 0; s < KT / 16; ++s)
                            mma_ts(tmem + C::COL_T, pa + 8 * s, vd + s * 128, idesc_o, (t > 0 || s > 0) ? 1u : 0u, leader);
                    }
                    tc_commit(&bars->o_bar, leader);
                    tc_commit(&bars->v_empty[st], leader);
                    ++ps;
                }
            }
            tc_commit(&bars->mma_final, leader);
            wait_all(&bars->mma_final, 0, p.err, nullptr);
        } else if (warp == 3) {
            // ---------------- leftovers and values that are not finite in V tiles ----------------
            int kvit = 0, it = 0, diag = 0;
            bool ok = true;
            for (; ok; ++it) {
                const Piece *slot = bars->ring.get(it, p.err, abort_flag, &ok);
                if (!slot) break;
                const Piece pc = *slot;
                bars->ring.put(it, lane);
                if constexpr (KV32) {
                    // Only tiles of which not every row sees every key, and from the cache itself, ahead of their
                    // conversion: warp 1 takes the verdict when it comes to such a tile, and cleans it if need be.
                    for (int j = max(pc.j0, first_diagonal(pc)); j < pc.j1 && ok; ++j, ++diag) {
                        const TileAt t = tile_at(pc, j);
                        const int from = max(t.all, 0);
                        const uint4 *src = reinterpret_cast<const uint4 *>(reinterpret_cast<const float *>(p.v) + (t.row + from) * D);
                        float z = 0.f;
#pragma unroll 2
                        for (int e = lane; e < (t.n - from) * (D / 4); e += 32) {
                            const uint4 u = __ldg(src + e);
                            z = fmaf(__uint_as_float(u.x), 0.f, fmaf(__uint_as_float(u.y), 0.f, z));
                            z = fmaf(__uint_as_float(u.z), 0.f, fmaf(__uint_as_float(u.w), 0.f, z));
                        }
                        const bool bad = __any_sync(0xffffffffu, z != 0.f);
                        ok = wait_all(&bars->v_taken, (diag & 1) ^ 1, p.err, abort_flag);
                        if (ok && lane == 0) {
                            bars->verdict = bad ? from << 16 | t.n : 0;
                            if (bad) {
                                unsigned bit;
                                unsigned *word = bars->ring.bad_word(it, pc, j, bit);
                                atomicOr(word, bit);
                            }
                            mbar_arrive(&bars->v_clean);
                        }
                    }
                } else {
                    for (int j = pc.j0; j < pc.j1 && ok; ++j, ++kvit) {
                        const TileAt t = tile_at(pc, j);
                        const int st = kvit % NS;
                        uint8_t *vt = sV + st * C::TILE;
                        ok = wait_all(&bars->v_raw[st], (kvit / NS) & 1, p.err, abort_flag);
                        if (!ok) break;
                        if (t.n < KT) {
#pragma unroll
                            for (int hh = 0; hh < C::HALVES; ++hh)
                                for (int e = t.n * 8 + lane; e < KT * 8; e += 32)
                                    *reinterpret_cast<uint4 *>(vt + hh * C::BOX + e * 16) = make_uint4(0u, 0u, 0u, 0u);
                            fence_proxy_async_smem();
                        }
                        unsigned bit;
                        unsigned *word = bars->ring.bad_word(it, pc, j, bit);
                        clean_rows<C::HALVES, C::BOX, 4>(vt, 0, t.n, word, bit);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bars->v_full[st]);
                    }
                }
            }
        }
    } else if (KV32 && warp < 4 + C::CONV / 32) {
        setmaxnreg_dec<C::REG_CONV>();
        // ---------------- f32 cache: K and V in three parts ----------------
        constexpr int CH = D / 8, CONV = KV32 ? C::CONV : 128, PER = KT * CH / CONV;  // 8-value chunks of a row, and per thread
        const int me = tid - 128;
        // K and V tiles in turn, through the same code (see Terms).  Each 8 values are split and stored, and
        // then their place in registers takes the same ones of the next tile.
        float x[PER][8];
        auto load = [&](int i, const void *cache, const TileAt &t) {
            const int e = me + CONV * i, row = e / CH, c = e % CH;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
            if (row < t.n) {
                const float *src = reinterpret_cast<const float *>(cache) + (t.row + row) * D + 8 * c;
                a = __ldg(reinterpret_cast<const float4 *>(src));
                b = __ldg(reinterpret_cast<const float4 *>(src + 4));
            }
            x[i][0] = a.x; x[i][1] = a.y; x[i][2] = a.z; x[i][3] = a.w;
            x[i][4] = b.x; x[i][5] = b.y; x[i][6] = b.z; x[i][7] = b.w;
        };
        int n2 = 0, it = 0;  // tiles done (K and V counted), pieces
        bool ok = true;
        const Piece *slot = bars->ring.get(0, p.err, abort_flag, &ok);
        Piece pc;
        TileAt tn;
        int j = 0;
        if (slot) {
            pc = *slot;
            bars->ring.put(0, lane);
            j = pc.j0;
            tn = tile_at(pc, j);
#pragma unroll
            for (int i = 0; i < PER; ++i) load(i, tn.pre ? p.pk : p.k, tn);
        }
        while (ok && slot) {
            const bool is_v = n2 & 1;
            const int st = (n2 >> 1) % NS;
            const uint32_t par = ((n2 >> 1) / NS & 1) ^ 1;
            // the next tile: V of this one, or K of the one after
            if (is_v && ++j == pc.j1) {
                slot = bars->ring.get(++it, p.err, abort_flag, &ok);
                if (slot) {
                    pc = *slot;
                    bars->ring.put(it, lane);
                    j = pc.j0;
                }
            }
            if (is_v && slot) tn = tile_at(pc, j);
            const void *next = is_v ? (tn.pre ? p.pk : p.k) : (tn.pre ? p.pv : p.v);
            if (!wait_all(is_v ? &bars->v_empty[st] : &bars->k_empty[st], par, p.err, abort_flag)) { ok = false; break; }
            uint8_t *tile = (is_v ? sV : sK) + st * C::TILE;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int e = me + CONV * i, row = e / CH, c = e % CH;
                uint32_t w[3][4];
#pragma unroll
                for (int k = 0; k < 4; ++k) split3_cache(x[i][2 * k], x[i][2 * k + 1], w[0][k], w[1][k], w[2][k]);
                if (slot) load(i, next, tn);
                uint8_t *at = tile + (c >> 3) * C::BOX + row * 128 + (((c & 7) ^ (row & 7)) << 4);
#pragma unroll
                for (int k = 0; k < 3; ++k)
                    *reinterpret_cast<uint4 *>(at + k * C::PART) = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(is_v ? &bars->v_full[st] : &bars->k_full[st]);
            ++n2;
        }
    } else {
        setmaxnreg_inc<C::REG_SOFT>();
        // ---------------- softmax: thread = half a row ----------------
        constexpr int KH = KT / 2, DH = D / 2;  // keys and columns of a thread
        const int half = (warp - C::SOFT0) >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const float scale = kLog2e / (D == 64 ? 8.0f : 11.313708498984761f);
        int js = 0;  // S tiles taken; P V tiles awaited are js - 1 at the same place
        uint32_t gph = 0, xph = 0;
        auto group_sync = [&]() -> bool {
            mbar_arrive(&bars->g_bar[half]);
            return __all_sync(0xffffffffu, mbar_wait(&bars->g_bar[half], gph++ & 1, p.err, abort_flag));
        };
        // the other half's value for this row
        auto exchange = [&](float mine, float &other) -> bool {
            bars->xch[xph & 1][half][r] = mine;
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->x_bar);
            const bool ok = __all_sync(0xffffffffu, mbar_wait(&bars->x_bar, xph & 1, p.err, abort_flag));
            other = *reinterpret_cast<volatile float *>(&bars->xch[xph & 1][half ^ 1][r]);
            ++xph;
            return ok;
        };
        auto put_q = [&](const Piece &pc) {
            const int tok = r >> p.lg_g;
            const bool live = tok < pc.ntok;
            const int64_t row = (int64_t)(pc.tok0 + (live ? tok : 0)) * p.nHead + (pc.g << p.lg_g) + (r & ((1 << p.lg_g) - 1));
            store_q<D>(reinterpret_cast<const float *>(p.q) + row * D + half * DH, live, scale,
                       tmem + lane_base + C::COL_Q + half * (D / 4));
            warp_arrive(&bars->q_ready, lane);
        };
        bool ok = true;
        const Piece *next = bars->ring.get(0, p.err, abort_flag, &ok);
        if (next) put_q(*next);
        for (int it = 0; ok && next; ++it) {
            const Piece &pc = *next;
            const int kpos = pc.pos + (r >> p.lg_g);
            float m = -INFINITY, l = 0.f;
            float o[DH];
#pragma unroll
            for (int d = 0; d < DH; ++d) o[d] = 0.f;
            // step j: S(j) to registers and weights; then, with T(j-1) there, o += T(j-1) and P(j) to
            // TMEM.  The last step only adds the last T.
            for (int j = pc.j0;; ++j) {
                const bool more = j < pc.j1;
                uint32_t sr[KH];
                float alpha = 1.f, sum = 0.f;
                bool grow = false;
                if (more) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&bars->s_full, js & 1, p.err, abort_flag));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < KH / 32; ++c) {
                        uint32_t *rr = sr + 32 * c;
                        TL_LD32(tmem + lane_base + C::COL_S + half * KH + 32 * c, rr);
                    }
                    tmem_wait_ld();
                    warp_arrive(&bars->s_free, lane);
                    const TileAt t = tile_at(pc, j);
                    if (t.pre ? t.n < KT : t.all < KT) {
                        const int seen = (t.pre ? t.n - 1 : kpos - t.k0) - half * KH;  // last key this row sees
#pragma unroll
                        for (int c = 0; c < KH; ++c)
                            if (c > seen) sr[c] = __float_as_uint(-INFINITY);
                    }
                    float mq[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < KH; c += 8)
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            mq[u] = max3f(mq[u], __uint_as_float(sr[c + 2 * u]), __uint_as_float(sr[c + 2 * u + 1]));
                    float mx = max3f(mq[0], mq[1], fmaxf(mq[2], mq[3])), mo;
                    ok = exchange(mx, mo);
                    if (!ok) break;
                    mx = fmaxf(mx, mo);
                    grow = mx > m + kRescale || m == -INFINITY;  // the same in both halves
                    if (grow) {
                        alpha = m == -INFINITY ? 0.f : exp2f(m - mx);
                        m = mx;
                        l *= alpha;
                    }
                    const float nm = m == -INFINITY ? 0.f : -m;
                    const float2 n2 = make_float2(nm, nm);
                    float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                    for (int c = 0; c < KH; c += 2) {
                        const float2 d = fadd2(make_float2(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), n2);
                        const float2 e = make_float2(ex2(d.x), ex2(d.y));
                        acc[(c >> 1) & 1] = fadd2(acc[(c >> 1) & 1], e);
                        sr[c] = __float_as_uint(e.x);
                        sr[c + 1] = __float_as_uint(e.y);
                    }
                    const float2 sums = fadd2(acc[0], acc[1]);
                    sum = sums.x + sums.y;
                    ++js;
                } else {
                    // every S of this piece has been read (s_full of the last one, and its exchange): the
                    // next one's q may take the place of its q
                    next = bars->ring.get(it + 1, p.err, abort_flag, &ok);
                    if (next) put_q(*next);
                    if (!ok) break;
                }
                if (j > pc.j0) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&bars->o_bar, (js - (more ? 2 : 1)) & 1, p.err, abort_flag));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < DH / 32; ++c) {
                        uint32_t t[32];
                        TL_LD32(tmem + lane_base + C::COL_T + half * DH + 32 * c, t);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[32 * c + i] += __uint_as_float(t[i]);
                    }
                    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                        for (int d = 0; d < DH; ++d) o[d] *= alpha;
                    }
                }
                if (!more) break;
                // A weight that is not a number over a bf16 cache: the parts of q times an infinite key cancel.
                if (!KV32 && __builtin_expect(__any_sync(0xffffffffu, sum != sum && l == l), 0)) {
                    const TileAt t = tile_at(pc, j);
                    uint32_t w[KH];  // in local memory, to keep this path short
#pragma unroll
                    for (int c = 0; c < KH; ++c) w[c] = sr[c];
                    float kept = sum;
                    const bool lost = sum != sum && l == l && (r >> p.lg_g) < pc.ntok;
                    const int64_t row = (int64_t)(pc.tok0 + (lost ? r >> p.lg_g : 0)) * p.nHead + (pc.g << p.lg_g) + (r & ((1 << p.lg_g) - 1));
                    if (keep_weights<D, KH, KV>(w, lost, reinterpret_cast<const float *>(p.q) + row * D,
                                                reinterpret_cast<const KV *>(t.pre ? p.pk : p.k) + (t.row + half * KH) * D, kept)) {
                        sum = kept;
#pragma unroll
                        for (int c = 0; c < KH; ++c) sr[c] = w[c];
                    }
                }
                l += sum;
#pragma unroll
                for (int c = 0; c < KH / 32; ++c) {
                    uint32_t a[16], b[16], d[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        split3(__uint_as_float(sr[32 * c + 2 * i]), __uint_as_float(sr[32 * c + 2 * i + 1]), a[i], b[i], d[i]);
                    const uint32_t col = tmem + lane_base + C::COL_P + half * (KH / 2) + 16 * c;
                    TL_ST16(col, a);
                    TL_ST16(col + KT / 2, b);
                    TL_ST16(col + KT, d);
                }
                tmem_wait_st();
                warp_arrive(&bars->p_ready, lane);
            }
            if (!ok) break;
            tc_fence_before();
            float lo;
            ok = exchange(l, lo);
            if (!ok) break;
            l = half == 0 ? l + lo : lo + l;  // the same sum in both halves
            put_back<D, DH, !KV32, KV>(p, pc, bars->ring.bad[it % kRing], bars->ring.bad_step(pc), r, half * DH, o);
            ok = finish_rows<D, DH, float, BM>(p, cut, pc, half, r, half * DH, o, m, l, group_sync, &bars->last_flag[half],
                                               base + C::OFF_STG + (warp - C::SOFT0) * 32 * kStgRow);
            bars->ring.put(it, lane);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int D, bool KV32>
cudaError_t launch_t(const PackedArgs &a, cudaStream_t s) {
    using C = P32<D, KV32>;
    PkParams<D> p;
    if (!pk_params(a, BM, C::KT, p)) return cudaErrorNotSupported;
    CUtensorMap km{}, vm{}, pkm{}, pvm{};
    if constexpr (!KV32) {
        const uint64_t own_rows = (uint64_t)p.in.nseq * a.nHeadKv * a.kv.maxLen;
        if (!map_rows(&km, p.k, own_rows, D, false, C::KT) || !map_rows(&vm, p.v, own_rows, D, false, C::KT))
            return cudaErrorNotSupported;
        pkm = km;
        pvm = vm;
        if (a.prefix_len > 0) {
            const uint64_t pre_rows = (uint64_t)a.nHeadKv * a.pkv.maxLen;
            if (!map_rows(&pkm, p.pk, pre_rows, D, false, C::KT) || !map_rows(&pvm, p.pv, pre_rows, D, false, C::KT))
                return cudaErrorNotSupported;
        }
    }
    const int smem = C::OFF_BARS + (int)sizeof(P32Bars<D, KV32>) + 1024;
    auto kern = packed_tc32_kernel<D, KV32>;
    static SmemLimit limit;
    const cudaError_t e = allow_smem(kern, smem, limit);
    if (e != cudaSuccess) return e;
    kern<<<a.ctas, C::THREADS, smem, s>>>(km, vm, pkm, pvm, p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_packed_tc32(const PackedArgs &a, cudaStream_t s) {
    if (a.ntok <= 0) return cudaSuccess;
    if (a.io != TL_IO_F32) return cudaErrorNotSupported;
    const bool f = a.kv.dtype == TL_KV_F32;
    if (a.headDim == 64) return f ? launch_t<64, true>(a, s) : launch_t<64, false>(a, s);
    if (a.headDim == 128) return f ? launch_t<128, true>(a, s) : launch_t<128, false>(a, s);
    return cudaErrorNotSupported;
}

}  // namespace tl
