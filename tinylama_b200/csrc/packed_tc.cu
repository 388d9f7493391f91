// packed_tc.cu -- attention of packed query rows on the 5th-generation tensor cores (bf16 activations
// over a bf16 cache): prompts of different lengths behind a shared prefix, and the prefix part of
// a decode over it.
//
// Row (token t of sequence b, head h) attends the P prefix positions, then own positions
// 0..pos0[b]+t:  o = sum_j 2^(c s_j - m) v_j / sum_j 2^(c s_j - m),  c = log2(e)/sqrt(D).
//
// A unit is 256 rows -- the G heads of a kv-head for 256/G consecutive tokens -- in two MMA tiles
// of 128, against 128-key tiles.  Taking the group's heads as rows of one tile lets short prompts and
// single tokens fill a tile that a tile per head would leave empty, halves the keys a causal
// tile computes in vain (the diagonal crosses 128/G tokens), and reads K/V once per group.  The Q
// tile is one 3-D TMA box (64 columns x G heads x 128/G tokens).  Units are shared out in
// equal pieces (packed_sched.cuh); a unit cut in pieces is merged by the piece that ends last.
//
// One CTA per SM, 12 warps, as the prefill kernel: warp 0 brings Q, K and V (TMA, 128-byte swizzle),
// warp 1 issues S_q = Q_q K^T, warps 2 and 3 issue O_q += P_q V (A = P from TMEM), and two
// softmax warpgroups (thread = row = TMEM lane) turn S_q into P_q with the running maximum and
// sum in fp32.  P is rounded to bf16 for the tensor cores (half a step of 2^-8 of each weight,
// as much as the output's own rounding); everything else is kept in fp32.  TMEM, 512 columns:
//   D = 64:   S0 S1 (128 each), P0 P1 (64 each), O0 O1 (64 each)
//   D = 128:  S (128, taken in turns by the two tiles), P0 P1, O0 O1 (128 each)
// What bounds it is the softmax.  With D = 64 the exponentials of a unit's tile (256 x 128) take 2048 clocks of the
// MUFU unit, its products 512 of the tensor core; a tile takes about 2950, and a unit 2 to 3.5 us more.  8 documents
// of up to 4096 (32/8/64): 465 us, 625 TFLOP/s; 6 prompts of up to 4096 behind 1000 shared positions (32/8/128): 681 us, 980
// TFLOP/s.  One exponential in 4 or 8 as a polynomial on the FMA pipe was slower (486, 502 us against 461).
//
// With D = 128 a tile's S is free again as soon as its group has it in registers, so one S serves both
// tiles while each P keeps its own columns and S(j+1) does not wait for P(j) V.
//
// Masked keys.  A slot's rows behind the last position hold leftovers; the warps that issue P V set
// those rows of V to zero in shared memory.  Values of the sequence itself that are not finite: see
// clean_rows (packed_tc.cuh).
//
// Every mbarrier wait is bounded (common.cuh); TMEM is released on every path after all issued MMAs
// have completed.
#include "packed_tc.cuh"

namespace tl {
namespace {

constexpr int kThreads = 384;
constexpr int kKeyTile = 128;
constexpr int kIssuers = 3;
constexpr int kLeadClocks = 2500;
constexpr unsigned kLeadUnit = 1u << 16;
constexpr int kConsumers = 11;  // warps that read the ring of pieces: 1, 2, 3 and the softmax warps

template <int D>
struct PkShape {
    static constexpr int HALVES = D / 64;
    static constexpr int BOX = 128 * 128;            // one 64-column box of 128 rows
    static constexpr int TILE = HALVES * BOX;        // a Q, K or V tile
    static constexpr int NQB = D == 64 ? 2 : 1;      // Q buffers (of two tiles)
    static constexpr int NS = D == 64 ? 4 : 2;       // K/V stages
    static constexpr int OFF_K = 2 * NQB * TILE;
    static constexpr int OFF_V = OFF_K + NS * TILE;
    static constexpr int OFF_STG = OFF_V + NS * TILE;
    static constexpr int OFF_BARS = OFF_STG + 8 * 32 * kStgRow;
    static constexpr bool S_SHARED = D == 128;
    __host__ __device__ static constexpr int col_s(int q) { return S_SHARED ? 0 : q * 128; }
    __host__ __device__ static constexpr int col_p(int q) { return (S_SHARED ? 128 : 256) + q * 64; }
    __host__ __device__ static constexpr int col_o(int q) { return (S_SHARED ? 256 : 384) + q * D; }
    static_assert(col_o(1) + D <= 512, "TMEM columns");
    static constexpr int REG_CTRL = 104, REG_SOFT = 200;
    static_assert(REG_CTRL + 2 * REG_SOFT <= 3 * (65536 / kThreads / 8 * 8), "register split exceeds the launch");
};

template <int D>
struct PkBars {
    static constexpr int NS = PkShape<D>::NS;
    uint64_t q_full[2], q_empty[2], k_full[NS], k_empty[NS], v_full[NS], v_empty[NS];
    uint64_t s_full[2], s_free[2], p_ready[2], o_bar[2], o_done[2], o_free[2], g_bar[2], mma_final;
    PieceRing<kConsumers> ring;
    SchedStart start;
    uint32_t tmem_base;
    int abort;
    int last_flag[2];
    volatile unsigned lead[4];  // by scheduler: how far group 0's exponentials are, kLeadUnit a piece
};

__device__ __forceinline__ void tma_load3(void *dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar,
                                          uint32_t issue) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "setp.ne.b32 e, %6, 0;\n\t"
        "@e cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n\t}" ::
            "r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)), "r"(issue)
        : "memory");
}

// D (+)= A B over K = 64: both operands K-major in shared memory, four K = 16 steps of 32 bytes
__device__ __forceinline__ void mma_ss_k64(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate,
                                           uint32_t issue) {
    asm volatile(
        "{\n\t.reg .pred e, t, p;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
        "setp.ne.b32 e, %5, 0;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.eq.b32 t, %5, %5;\n\t"
        "add.s64 a1, %1, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 a3, %1, 6;\n\t"
        "add.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(issue)
        : "memory");
}

// what a role needs of a piece
struct PieceTiles {
    int nt[2];  // tiles that the rows of MMA tile 0 / 1 see, counted from the unit's first (0: no rows)
    template <int UC>
    __device__ __forceinline__ PieceTiles(const SchedIn<UC> &in, const Piece &p) {
        const int tt = in.tb() / 2;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            if (p.ntok <= q * tt) nt[q] = 0;
            else if (in.cu == nullptr) nt[q] = in.prefix_tiles;
            else nt[q] = in.prefix_tiles + ((p.pos + min(p.ntok, (q + 1) * tt) + kKeyTile - 1) >> 7);
        }
    }
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
packed_tc_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                 const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap pkmap,
                 const __grid_constant__ CUtensorMap pvmap, const PkParams<D> p) {
    using S_ = PkShape<D>;
    using B_ = PkBars<D>;
    constexpr int NS = S_::NS, NQB = S_::NQB;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t *base = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    uint8_t *sQ = base, *sK = base + S_::OFF_K, *sV = base + S_::OFF_V;
    B_ *bars = reinterpret_cast<B_ *>(base + S_::OFF_BARS);
    volatile int *abort_flag = &bars->abort;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // ---- the line's length and this CTA's first sequence --------------------------------------
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars->q_full[i], 1);
            mbar_init(&bars->q_empty[i], 1);
            mbar_init(&bars->s_full[i], 1);
            mbar_init(&bars->s_free[i], 4);
            mbar_init(&bars->p_ready[i], 4);
            mbar_init(&bars->o_bar[i], 1);
            mbar_init(&bars->o_done[i], 1);
            mbar_init(&bars->o_free[i], 4);
            mbar_init(&bars->g_bar[i], BM);
        }
        for (int i = 0; i < NS; ++i) {
            mbar_init(&bars->k_full[i], 1);
            mbar_init(&bars->k_empty[i], 1);
            mbar_init(&bars->v_full[i], 1);
            mbar_init(&bars->v_empty[i], 2);
        }
        mbar_init(&bars->mma_final, kIssuers);
        bars->ring.init();
        bars->abort = 0;
        for (int i = 0; i < 4; ++i) bars->lead[i] = 0;
        bars->start.b0 = p.in.nseq;
        bars->start.s0 = 0;
        fence_mbar_init();
    }
    if (p.in.cu == nullptr) pdl_launch_dependents();  // the own positions' kernel runs beside this one
    SchedCut<unit_cost(D)> cut;
    if (!sched_begin<kThreads>(p, &bars->start, cut)) return;
    if (warp == 1) {
        tmem_alloc(&bars->tmem_base, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars->tmem_base;
    const int tt = p.in.tb() / 2;  // tokens of an MMA tile

    if (warp < 4) {
        setmaxnreg_dec<S_::REG_CTRL>();
        auto wait_all = [&](uint64_t *bar, uint32_t parity, unsigned *err, volatile int *ab) {
            return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, ab));
        };
        const uint32_t leader = elect_one();
        if (warp == 0) {
            // ---------------- TMA producer ----------------
            SchedIter<unit_cost(D)> iter;
            iter.init(p.in, cut, blockIdx.x, bars->start.b0, bars->start.s0);
            int it = 0, kvit = 0, pieces = 0;
            bool ok = true;
            Piece pc;
            while (ok && iter.next(p.in, pc)) {
                if (!bars->ring.publish(pieces, pc, leader, p.err, abort_flag)) { ok = false; break; }
                ++pieces;
                const PieceTiles pt(p.in, pc);
                const int qb = it % NQB;
                if (!wait_all(&bars->q_empty[qb], ((it / NQB) & 1) ^ 1, p.err, abort_flag)) { ok = false; break; }
                const int live = pt.nt[1] > 0 ? 2 : 1;
                if (leader) mbar_arrive_expect_tx(&bars->q_full[qb], live * S_::TILE);
                __syncwarp();
                for (int q = 0; q < live; ++q)
#pragma unroll
                    for (int hh = 0; hh < S_::HALVES; ++hh)
                        tma_load3(sQ + (qb * 2 + q) * S_::TILE + hh * S_::BOX, &qmap, 64 * hh, pc.g << p.lg_g,
                                  pc.tok0 + q * tt, &bars->q_full[qb], leader);
                ++it;
                for (int j = pc.j0; j < pc.j1; ++j, ++kvit) {
                    const bool pre = j < p.in.prefix_tiles;
                    const CUtensorMap *km = pre ? &pkmap : &kmap, *vm = pre ? &pvmap : &vmap;
                    const int row = pre ? pc.g * p.prefix_max_len + j * kKeyTile
                                        : (pc.b * p.in.heads_kv + pc.g) * p.in.max_len + (j - p.in.prefix_tiles) * kKeyTile;
                    const int st = kvit % NS;
                    const uint32_t par = ((kvit / NS) & 1) ^ 1;
                    if (!wait_all(&bars->k_empty[st], par, p.err, abort_flag)) { ok = false; break; }
                    if (leader) mbar_arrive_expect_tx(&bars->k_full[st], S_::TILE);
                    __syncwarp();
#pragma unroll
                    for (int hh = 0; hh < S_::HALVES; ++hh)
                        tma_load_2d(sK + st * S_::TILE + hh * S_::BOX, km, 64 * hh, row, &bars->k_full[st], leader);
                    if (!wait_all(&bars->v_empty[st], par, p.err, abort_flag)) {
                        // K of this stage is in flight, V is not: wait for the K alone
                        wait_all(&bars->k_full[st], (kvit / NS) & 1, nullptr, nullptr);
                        ok = false;
                        break;
                    }
                    if (leader) mbar_arrive_expect_tx(&bars->v_full[st], S_::TILE);
                    __syncwarp();
#pragma unroll
                    for (int hh = 0; hh < S_::HALVES; ++hh)
                        tma_load_2d(sV + st * S_::TILE + hh * S_::BOX, vm, 64 * hh, row, &bars->v_full[st], leader);
                }
            }
            pc.w = -1;
            if (ok) bars->ring.publish(pieces, pc, leader, p.err, abort_flag);
            // wait (bounded) until every copy issued into this CTA's shared memory has landed
            for (int i = max(0, it - NQB); i < it; ++i)
                wait_all(&bars->q_full[i % NQB], (i / NQB) & 1, nullptr, nullptr);
            for (int j = max(0, kvit - NS); j < kvit; ++j) {
                wait_all(&bars->k_full[j % NS], (j / NS) & 1, nullptr, nullptr);
                wait_all(&bars->v_full[j % NS], (j / NS) & 1, nullptr, nullptr);
            }
        } else if (warp == 1) {
            // ---------------- S issuer: S_q(j) = Q_q K_j^T ----------------
            const uint32_t idesc_s = idesc_bf16(kKeyTile, false);
            int it = 0, kvit = 0, ns[2] = {0, 0}, prev = -1;
            bool ok = true;
            while (ok) {
                const Piece *slot = bars->ring.get(it, p.err, abort_flag, &ok);
                if (!slot) break;
                const Piece pc = *slot;
                bars->ring.put(it, lane);
                const PieceTiles pt(p.in, pc);
                const int qb = it % NQB;
                ok = wait_all(&bars->q_full[qb], (it / NQB) & 1, p.err, abort_flag);
                for (int j = pc.j0; j < pc.j1 && ok; ++j, ++kvit) {
                    const int st = kvit % NS;
                    ok = wait_all(&bars->k_full[st], (kvit / NS) & 1, p.err, abort_flag);
                    if (!ok) break;
                    const uint32_t ka = smem_u32(sK + st * S_::TILE);
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        if (!ok || j >= pt.nt[q]) continue;
                        // the S that these columns held must be in its group's registers
                        if constexpr (S_::S_SHARED) {
                            if (prev >= 0)
                                ok = wait_all(&bars->s_free[prev], ((prev == 0 ? ns[0] : ns[1]) - 1) & 1, p.err, abort_flag);
                        } else {
                            if (ns[q] > 0) ok = wait_all(&bars->s_free[q], (ns[q] - 1) & 1, p.err, abort_flag);
                        }
                        if (!ok) continue;
                        tc_fence_after();
                        const uint32_t qa = smem_u32(sQ + (qb * 2 + q) * S_::TILE);
#pragma unroll
                        for (int hh = 0; hh < S_::HALVES; ++hh)
                            mma_ss_k64(tmem + S_::col_s(q), sw128_desc(qa + hh * S_::BOX, 16), sw128_desc(ka + hh * S_::BOX, 16),
                                       idesc_s, hh > 0 ? 1u : 0u, leader);
                        tc_commit(&bars->s_full[q], leader);
                        ++ns[q];
                        prev = q;
                    }
                    if (ok) tc_commit(&bars->k_empty[st], leader);
                }
                if (ok) tc_commit(&bars->q_empty[qb], leader);
                ++it;
            }
            tc_commit(&bars->mma_final, leader);
            wait_all(&bars->mma_final, 0, p.err, nullptr);
        } else {
            // ---------------- P V issuer for MMA tile q ----------------
            // While the group forms P(j), this warp zeroes the rows of V(j) that no row of the unit sees
            // (both P V warps do).
            auto zero_v = [&](const Piece &pc, int j, uint8_t *vt) {
                const bool pre = j < p.in.prefix_tiles;
                const int row0 = (pre ? p.prefix_len - j * kKeyTile : pc.pos + pc.ntok - (j - p.in.prefix_tiles) * kKeyTile);
                if (row0 >= kKeyTile) return;
#pragma unroll
                for (int hh = 0; hh < S_::HALVES; ++hh)
                    for (int e = row0 * 8 + lane; e < kKeyTile * 8; e += 32)
                        *reinterpret_cast<uint4 *>(vt + hh * S_::BOX + e * 16) = make_uint4(0u, 0u, 0u, 0u);
                fence_proxy_async_smem();
                __syncwarp();
            };
            const int q = warp - 2;
            const uint32_t idesc_o = idesc_bf16(D, true);
            int it = 0, kvit = 0, npv = 0, nto = 0;
            bool ok = true;
            for (; ok; ++it) {
                const Piece *slot = bars->ring.get(it, p.err, abort_flag, &ok);
                if (!slot) break;
                const Piece pc = *slot;
                bars->ring.put(it, lane);
                const PieceTiles pt(p.in, pc);
                const int end = min(pc.j1, q == 0 ? pt.nt[0] : pt.nt[1]);
                for (int j = pc.j0; j < pc.j1 && ok; ++j, ++kvit) {
                    const int st = kvit % NS;
                    ok = wait_all(&bars->v_full[st], (kvit / NS) & 1, p.err, abort_flag);
                    if (!ok) break;
                    if (j < end) {
                        uint8_t *vt = sV + st * S_::TILE;
                        zero_v(pc, j, vt);
                        const int seen = pc.pos + 1 - (j - p.in.prefix_tiles) * kKeyTile;  // own keys that every row sees
                        if (p.in.cu != nullptr && j >= p.in.prefix_tiles && seen < kKeyTile) {
                            unsigned bit;
                            unsigned *word = bars->ring.bad_word(it, pc, j, bit);
                            clean_rows<S_::HALVES, S_::BOX, 1>(vt, max(seen, 0), min(seen - 1 + pc.ntok, kKeyTile), word, bit);
                        }
                        if (j == pc.j0 && nto > 0) ok = wait_all(&bars->o_free[q], (nto - 1) & 1, p.err, abort_flag);
                        if (ok) ok = wait_all(&bars->p_ready[q], npv & 1, p.err, abort_flag);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t va = smem_u32(vt);
#pragma unroll
                        for (int kb = 0; kb < kKeyTile / 64; ++kb)
                            mma_pv_k64(tmem + S_::col_o(q), tmem + S_::col_p(q) + kb * 32,
                                       sw128_desc(va + kb * 4 * 2048, S_::BOX), idesc_o,
                                       (j > pc.j0 || kb > 0) ? 1u : 0u, leader);
                        tc_commit(&bars->o_bar[q], leader);
                        if (j == end - 1) tc_commit(&bars->o_done[q], leader);
                        ++npv;
                    }
                    tc_commit(&bars->v_empty[st], leader);
                }
                if (end > pc.j0) ++nto;
            }
            tc_commit(&bars->mma_final, leader);
        }
    } else {
        setmaxnreg_inc<S_::REG_SOFT>();
        // ---------------- softmax of MMA tile q ----------------
        const int q = (warp - 4) >> 2;
        const int r = (warp & 3) * 32 + lane;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const float C = kLog2e / (D == 64 ? 8.0f : 11.313708498984761f);
        int ns = 0, npv = 0, nto = 0, it = 0;
        bool ok = true;
        uint32_t gph = 0;
        // the group's 128 threads, by an mbarrier so that the wait is bounded
        auto group_sync = [&]() -> bool {
            mbar_arrive(&bars->g_bar[q]);
            return __all_sync(0xffffffffu, mbar_wait(&bars->g_bar[q], gph++ & 1, p.err, abort_flag));
        };
        for (; ok; ++it) {
            const Piece *slot = bars->ring.get(it, p.err, abort_flag, &ok);
            if (!slot) break;
            const Piece &pc = *slot;
            const PieceTiles pt(p.in, pc);
            const int ntq = q == 0 ? pt.nt[0] : pt.nt[1];
            const int end = min(pc.j1, ntq);
            if (ntq == 0) {
                bars->ring.put(it, lane);
                continue;
            }
            const int kfirst = pc.pos + q * tt;          // own position of the tile's first token
            const int kpos = kfirst + (r >> p.lg_g);     // and of this row's
            float m_run = -INFINITY, l = 0.f;
            for (int j = pc.j0; j < end && ok; ++j) {
                ok = __all_sync(0xffffffffu, mbar_wait(&bars->s_full[q], ns & 1, p.err, abort_flag));
                if (!ok) break;
                ++ns;
                tc_fence_after();
                uint32_t sr[kKeyTile];
#pragma unroll
                for (int c = 0; c < kKeyTile / 32; ++c) {
                    uint32_t *rr = sr + 32 * c;
                    TL_LD32(tmem + lane_base + S_::col_s(q) + 32 * c, rr);
                }
                tmem_wait_ld();
                warp_arrive(&bars->s_free[q], lane);
                const bool pre = j < p.in.prefix_tiles;
                const int k0 = (pre ? j : j - p.in.prefix_tiles) * kKeyTile;
                const int seen = (pre ? p.prefix_len - 1 : kpos) - k0;  // last key of the tile that this row sees
                if (pre ? seen < kKeyTile - 1 : kfirst - k0 < kKeyTile - 1) {
#pragma unroll
                    for (int c = 0; c < kKeyTile; ++c)
                        if (c > seen) sr[c] = __float_as_uint(-INFINITY);
                }
                float mq[8] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < kKeyTile; c += 16) {
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        mq[u] = max3f(mq[u], __uint_as_float(sr[c + 2 * u]), __uint_as_float(sr[c + 2 * u + 1]));
                }
                const float mx = max3f(max3f(mq[0], mq[1], mq[2]), max3f(mq[3], mq[4], mq[5]), fmaxf(mq[6], mq[7]));
                const float ms = mx * C;
                const bool grow = ms > m_run + kRescale || m_run == -INFINITY;
                float alpha = 1.f;
                if (grow) {
                    alpha = (m_run == -INFINITY) ? 0.f : ex2(m_run - ms);
                    m_run = ms;
                    l *= alpha;
                }
                // Group 1's warp lets group 0's warp of the same scheduler form its exponentials of the
                // tile first: in step the two would share the MUFU unit and then leave it idle
                // together.  Only a hint: the wait is short and whatever it finds is right.
                if (q == 1) {
                    const unsigned want = (unsigned)it * kLeadUnit + (unsigned)min(j - pc.j0 + 1, (int)kLeadUnit - 1);
                    const long long t0 = clock64();
                    while ((int)(bars->lead[warp & 3] - want) < 0 && clock64() - t0 < kLeadClocks) {}
                    __syncwarp();
                }
                // a row that has seen no key yet keeps every exponent at -infinity
                const float nm = m_run == -INFINITY ? 0.f : -m_run;
                const float2 c2 = make_float2(C, C), n2 = make_float2(nm, nm);
                float2 acc[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                uint32_t pk[kKeyTile / 2];
#pragma unroll
                for (int c = 0; c < kKeyTile; c += 2) {
                    const float2 x = ffma2(make_float2(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), c2, n2);
                    const float2 pp = make_float2(ex2(x.x), ex2(x.y));
                    acc[(c >> 1) & 3] = fadd2(acc[(c >> 1) & 3], pp);
                    pk[c / 2] = pack_bf16(pp.x, pp.y);
                }
                const float2 a = fadd2(fadd2(acc[0], acc[1]), fadd2(acc[2], acc[3]));
                l += a.x + a.y;
                if (q == 0 && lane == 0)
                    bars->lead[warp & 3] = (unsigned)it * kLeadUnit + (unsigned)min(j - pc.j0 + 1, (int)kLeadUnit - 1);
                if (j > pc.j0) {
                    // P_q V(j-1) is complete: P_q may be overwritten and O_q rescaled
                    ok = __all_sync(0xffffffffu, mbar_wait(&bars->o_bar[q], (npv - 1) & 1, p.err, abort_flag));
                    if (!ok) break;
                    tc_fence_after();
                }
                if (__any_sync(0xffffffffu, grow && j > pc.j0)) {
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t orr[16];
                        TL_LD16(tmem + lane_base + S_::col_o(q) + 16 * c, orr);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) orr[i] = __float_as_uint(__uint_as_float(orr[i]) * alpha);
                        TL_ST16(tmem + lane_base + S_::col_o(q) + 16 * c, orr);
                    }
                }
#pragma unroll
                for (int c = 0; c < kKeyTile / 64; ++c) {
                    uint32_t *rr = pk + 32 * c;
                    TL_ST32(tmem + lane_base + S_::col_p(q) + 32 * c, rr);
                }
                tmem_wait_st();
                warp_arrive(&bars->p_ready[q], lane);
                ++npv;
            }
            if (!ok) break;
            if (q == 0 && lane == 0) bars->lead[warp & 3] = (unsigned)(it + 1) * kLeadUnit;
            // ---- the piece's state: O_q out of TMEM ----
            float o[D];
            if (end > pc.j0) {
                ok = __all_sync(0xffffffffu, mbar_wait(&bars->o_done[q], nto & 1, p.err, abort_flag));
                if (!ok) break;
                ++nto;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t *rr = reinterpret_cast<uint32_t *>(o) + 32 * c;
                    TL_LD32(tmem + lane_base + S_::col_o(q) + 32 * c, rr);
                }
                tmem_wait_ld();
                warp_arrive(&bars->o_free[q], lane);
            } else {
#pragma unroll
                for (int d = 0; d < D; ++d) o[d] = 0.f;
            }
            put_back<D, D, false, __nv_bfloat16>(p, pc, bars->ring.bad[it % kRing], bars->ring.bad_step(pc), q * BM + r, 0, o);
            ok = finish_rows<D, D, __nv_bfloat16, 2 * BM>(p, cut, pc, q, q * BM + r, 0, o, m_run, l, group_sync,
                                                          &bars->last_flag[q],
                                                          base + S_::OFF_STG + (warp - 4) * 32 * kStgRow);
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

// ---- host side ------------------------------------------------------------------------------
// q as [token][head][D]: a box is 64 columns of G heads of 128/G tokens
bool map_q(CUtensorMap *m, const void *ptr, int ntok, int heads, int D, int G) {
    auto enc = get_encode();
    if (!enc) return false;
    cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)ntok};
    cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)heads * D * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)(BM / G)};
    cuuint32_t estr[3] = {1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(ptr), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D>
cudaError_t launch_t(const PackedArgs &a, cudaStream_t s) {
    using S_ = PkShape<D>;
    const int G = a.nHead / a.nHeadKv;
    PkParams<D> p;
    if (!pk_params(a, 2 * BM, kKeyTile, p)) return cudaErrorNotSupported;
    const uint64_t own_rows = (uint64_t)p.in.nseq * a.nHeadKv * a.kv.maxLen;
    CUtensorMap qm, km, vm, pkm, pvm;
    if (!map_q(&qm, a.q, a.ntok, a.nHead, D, G) || !map_rows(&km, p.k, own_rows, D, false, kKeyTile) ||
        !map_rows(&vm, p.v, own_rows, D, false, kKeyTile))
        return cudaErrorNotSupported;
    pkm = km;
    pvm = vm;
    if (a.prefix_len > 0) {
        const uint64_t pre_rows = (uint64_t)a.nHeadKv * a.pkv.maxLen;
        if (!map_rows(&pkm, p.pk, pre_rows, D, false, kKeyTile) || !map_rows(&pvm, p.pv, pre_rows, D, false, kKeyTile))
            return cudaErrorNotSupported;
    }
    const int smem = S_::OFF_BARS + (int)sizeof(PkBars<D>) + 1024;
    auto kern = packed_tc_kernel<D>;
    static SmemLimit limit;
    const cudaError_t e = allow_smem(kern, smem, limit);
    if (e != cudaSuccess) return e;
    kern<<<a.ctas, kThreads, smem, s>>>(qm, km, vm, pkm, pvm, p);
    return cudaGetLastError();
}

// One warp per row, a lane holding D/32 columns.  Few rows, so each row's parts are loaded
// together (up to 8 in flight) before they are added.
template <typename IO, int D>
__global__ void __launch_bounds__(128) merge_kernel(const MergeArgs a) {
    constexpr int N = D / 32, UN = 8;
    const int lane = threadIdx.x & 31;
    const int64_t rows = (int64_t)a.nseq * a.nHead, i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    pdl_wait();
    if (i >= rows) return;
    const int pos = min(a.pos[i / a.nHead], a.max_len - 1);
    const int nown = pos < 0 ? 0 : min(pos / a.chunk + 1, a.nchunks), n = a.nparts + nown;
    const float2 *ml0 = reinterpret_cast<const float2 *>(a.part + a.nparts * rows * D) + i;
    const float2 *ml1 = reinterpret_cast<const float2 *>(a.own + a.nchunks * rows * D) + i;
    const float *o0 = a.part + i * D + lane * N, *o1 = a.own + i * D + lane * N;
    float m = -INFINITY, l = 0.f, o[N];
#pragma unroll
    for (int k = 0; k < N; ++k) o[k] = 0.f;
    for (int p0 = 0; p0 < n; p0 += UN) {
        float2 s[UN];
        float x[UN][N];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            s[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int k = 0; k < N; ++k) x[u][k] = 0.f;
            const int k0 = p0 + u, k1 = k0 - a.nparts;
            if (k0 >= n) continue;
            s[u] = k1 < 0 ? ml0[k0 * rows] : ml1[k1 * rows];
            const float *src = k1 < 0 ? o0 + k0 * rows * D : o1 + k1 * rows * D;
            if constexpr (N == 4) {
                const float4 v = *reinterpret_cast<const float4 *>(src);
                x[u][0] = v.x; x[u][1] = v.y; x[u][2] = v.z; x[u][3] = v.w;
            } else {
                const float2 v = *reinterpret_cast<const float2 *>(src);
                x[u][0] = v.x; x[u][1] = v.y;
            }
        }
        float M = m;
#pragma unroll
        for (int u = 0; u < UN; ++u) M = fmaxf(M, s[u].x);
        const float w0 = safe_exp2_diff(m, M);
        l *= w0;
#pragma unroll
        for (int k = 0; k < N; ++k) o[k] *= w0;
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const float w = safe_exp2_diff(s[u].x, M);
            l = fmaf(s[u].y, w, l);
#pragma unroll
            for (int k = 0; k < N; ++k) o[k] = fmaf(x[u][k], w, o[k]);
        }
        m = M;
    }
    const float inv = l > 0.f ? 1.f / l : l;  // NaN stays
    if constexpr (sizeof(IO) == 4) {
        float *dst = reinterpret_cast<float *>(a.out) + i * D + lane * N;
#pragma unroll
        for (int k = 0; k < N; k += 2) *reinterpret_cast<float2 *>(dst + k) = make_float2(o[k] * inv, o[k + 1] * inv);
    } else {
        uint32_t *dst = reinterpret_cast<uint32_t *>(a.out) + (i * D + lane * N) / 2;
#pragma unroll
        for (int k = 0; k < N; k += 2) dst[k / 2] = pack_bf16(o[k] * inv, o[k + 1] * inv);
    }
}

}  // namespace

size_t packed_part_floats(int headDim, int ctas) { return (size_t)2 * ctas * (headDim + 4) * 256; }

void packed_unit(int headDim, int io, int *rows, int *keys) {
    *rows = io == TL_IO_BF16 ? 256 : 128;
    *keys = io == TL_IO_BF16 || headDim == 64 ? 128 : 64;
}

cudaError_t launch_packed_merge(const MergeArgs &a, cudaStream_t s) {
    const unsigned grid = (unsigned)(((int64_t)a.nseq * a.nHead + 3) / 4);
    if (a.headDim == 64)
        return launch_pdl(a.io == TL_IO_BF16 ? merge_kernel<__nv_bfloat16, 64> : merge_kernel<float, 64>, dim3(grid), dim3(128),
                          0, s, a);
    return launch_pdl(a.io == TL_IO_BF16 ? merge_kernel<__nv_bfloat16, 128> : merge_kernel<float, 128>, dim3(grid), dim3(128), 0,
                      s, a);
}

cudaError_t launch_packed_tc(const PackedArgs &a, cudaStream_t s) {
    if (a.ntok <= 0) return cudaSuccess;
    if (a.io != TL_IO_BF16 || a.kv.dtype != TL_KV_BF16) return cudaErrorNotSupported;
    if (a.headDim == 64) return launch_t<64>(a, s);
    if (a.headDim == 128) return launch_t<128>(a, s);
    return cudaErrorNotSupported;
}

}  // namespace tl
