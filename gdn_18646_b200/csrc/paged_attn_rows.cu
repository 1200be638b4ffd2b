// paged_attn_rows.cu -- paged attention where an item has few rows (a decode step, a few
// drafted tokens: tokens x query heads of a kv head <= 64), on tcgen05.
//
// The mathematics, the rows and the line of work are those of paged_attn.cu.  Here the
// keys stand in the MMA's wide dimension and the rows in its narrow one:
//   S^T = K Q^T      M 128 positions, N rows (16, 32 or 64), SS        -> TMEM, lane = position
//   P^T (bf16)       thread = position, written to shared memory as the next B operand
//   O^T += V^T P^T   M = D, N rows, SS (V as it lies, MN-major)    -> TMEM, lane = value index
// so a tile of 128 keys costs N/128 of the tensor work of a 128-row tile, and its softmax
// 256 threads x N / 2 exponentials instead of one warp x 128 a row (with rows in the wide
// dimension a tile took 2050 cycles, near the 2800 in which HBM delivers one, and the clock fell).  The running
// maximum is the same for all threads; only when some weight would pass 2^8 do they
// reduce a new one and rescale.  The sums l stay per thread until the item ends.
//
// Bound by HBM: K and V are read once, 32 KB (D 128) per ring stage.  256 decode steps over up to
// 8192 positions, 16 heads on 2: 160 us, 6.4 TB/s; 2 over up to 131072, 32 heads on 4: 72 us,
// 5.5 TB/s, of which about 8 us are the start of the pieces and the join.
#include <mutex>

#include "common.cuh"
#include "paged_work.cuh"

namespace gdn {
namespace {

// A warp issues a copy in about 60 cycles, and a tile is 2 x 128 / page size x D / 64 of them, so
// with small pages the issue sets the pace of one warp while the ring fills.  With 1 / 2 / 4 warps,
// us: 1 token over 1000 positions in pages of 16, head dim 128, 16.5 / 13.0 / 12.3; 256 sequences of
// up to 8192 159.8 / 162.5 / 164.3; 2 of up to 131072 in pages of 64 72.2 / 72.7 / 73.0.
constexpr int kLoadWarps = 2;
constexpr int kRowsThreads = 288 + 32 * kLoadWarps;      // 2 x 4 softmax warps, MMA, load

template <int D, int N>
struct RowsShape {
    static constexpr int HALVES = D / 64;
    static constexpr int STAGE = kTile * D * 2;
    static constexpr int Q_BYTES = HALVES * N * 128;            // one of two buffers
    static constexpr int P_BYTES = 2 * N * 128;                 // 128 positions as two halves; one of two buffers
    // D 64: the MMA (M 128) reads 16 KB past a V tile for result lanes that nobody uses
    static constexpr int USED = 2 * Q_BYTES + 2 * P_BYTES + 3072;
    static constexpr int AFTER = USED > 16384 ? USED : 16384;
    static constexpr int FIT = (232448 - 1024 - AFTER) / STAGE;
    static constexpr int STAGES = FIT < 12 ? FIT : 12;
    static constexpr int OFF_Q = STAGES * STAGE;
    static constexpr int OFF_P = OFF_Q + 2 * Q_BYTES;
    static constexpr int OFF_BAR = OFF_P + 2 * P_BYTES;
    static constexpr int SMEM = 1024 + OFF_Q + AFTER;
    static constexpr int COLS = N == 16 ? 64 : N == 32 ? 128 : 256;             // TMEM: two S buffers, O
    static constexpr int T_O = 2 * N;
    static_assert(SMEM <= 232448, "shared memory");
};

struct RowsBars {
    uint64_t full[16], empty[16];
    uint64_t q_full[2], q_empty[2];
    uint64_t s_full[2], p_full[2];
    uint64_t o_full, pv_done;
    PieceScratch scratch;
    alignas(16) float m[64];
    float f[64];                      // per row: reference maximum, factor of a rescale
    float red[4][64];                 // per warp and row: tile maxima, then sums
    uint32_t tmem;
    int abort;
};
static_assert(sizeof(RowsBars) <= 3072, "barrier block");

// whether any of the 128 threads that meet at barrier `id` says so
__device__ __forceinline__ bool any_of_128(int id, bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbarrier.cta.red.or.pred p, %2, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r)
        : "r"(static_cast<uint32_t>(x)), "r"(id)
        : "memory");
    return r != 0;
}

// 8 columns of the thread's lane
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float (&v)[8]) {
    uint32_t r[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const float (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr),
                 "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])),
                 "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7]))
                 : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_ld_rows(uint32_t taddr, float (&v)[N]) {
    if constexpr (N == 8) {
        tmem_ld8(taddr, v);
        return;
    } else if constexpr (N == 16) {
        uint32_t r[16];
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
              "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(taddr));
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N / 32; ++i) tmem_ld32(taddr + i * 32, reinterpret_cast<float(&)[32]>(v[i * 32]));
    }
    tmem_ld_wait();
}
// eight values of shared memory (16-byte aligned)
__device__ __forceinline__ void rows8(const float* at, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(at), b = *reinterpret_cast<const float4*>(at + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
// Eight rows' maxima (or sums) over the warp's lanes: halves of the rows go to halves of the
// lanes, so lanes 4 i .. 4 i + 3 end with row i's.
template <bool MAX>
__device__ __forceinline__ float reduce8(float (&v)[8]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 4, o = 16; n >= 1; n >>= 1, o >>= 1) {
        const bool up = (lane & o) != 0;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float send = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
            const float got = __shfl_xor_sync(0xffffffffu, send, o);
            v[i] = MAX ? fmaxf(keep, got) : keep + got;
        }
    }
#pragma unroll
    for (int o = 2; o >= 1; o >>= 1) {
        const float got = __shfl_xor_sync(0xffffffffu, v[0], o);
        v[0] = MAX ? fmaxf(v[0], got) : v[0] + got;
    }
    return v[0];
}

template <int D, int N>
__global__ void __launch_bounds__(kRowsThreads, 1)
paged_attn_rows_kernel(const __grid_constant__ AttnMaps maps, const __grid_constant__ AttnArgs a) {
    using S = RowsShape<D, N>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    RowsBars* sh = reinterpret_cast<RowsBars*>(sm + S::OFF_BAR);
    volatile int* dead = &sh->abort;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int MMA_WARP = 8, LOAD_WARP = 9;
    const int tt = a.tile_tokens, cta = blockIdx.x;

    if (tid == 0) {
        for (int i = 0; i < S::STAGES; ++i) {
            mbar_init(&sh->full[i], kLoadWarps);
            mbar_init(&sh->empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh->q_full[i], 1);
            mbar_init(&sh->q_empty[i], 1);
            mbar_init(&sh->s_full[i], 1);
            mbar_init(&sh->p_full[i], 8);
        }
        mbar_init(&sh->o_full, 1);
        mbar_init(&sh->pv_done, 1);
        sh->abort = 0;
        fence_mbar_init();
        tma_prefetch_desc(&maps.q);
        tma_prefetch_desc(&maps.k);
        tma_prefetch_desc(&maps.v);
    }
    if (warp == MMA_WARP) {
        tmem_alloc(&sh->tmem, S::COLS);
        tmem_relinquish();
    }
    pdl_launch_dependents();
    pdl_wait_prior();                                           // q, the cache and the lengths come from earlier kernels
    find_piece(a, &sh->scratch, tt);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh->tmem;
    const Piece piece = sh->scratch.piece;

    uint32_t q_loads = 0, issued = 0;                           // of the producer
    int stage = 0;                                              // the kv ring, as the producer or the MMA warp walks it
    uint32_t phase = 0;
    auto step = [&]() {
        if (++stage == S::STAGES) {
            stage = 0;
            phase ^= 1u;
        }
    };
    if (warp >= LOAD_WARP) {
        // ---------------- TMA producers, each with a share of every tile's copies; the first also loads Q
        Walk w;
        for (w.start(a, piece, tt); w.valid(); w.next(a, tt)) {
            if (w.t0 >= w.t1) continue;
            if (warp == LOAD_WARP) {
                const int qb = q_loads & 1;
                if (!warp_wait(&sh->q_empty[qb], ((q_loads >> 1) & 1u) ^ 1u, a.err, dead)) break;
                ++q_loads;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&sh->q_full[qb], S::HALVES * tt * a.group * 128);
                    for (int h = 0; h < S::HALVES; ++h)
                        tma_load_3d(sm + S::OFF_Q + qb * S::Q_BYTES + h * N * 128, &maps.q, &sh->q_full[qb], h * 64,
                                    w.head * a.group, w.s.c0 + w.item * tt);
                }
            }
            if (!load_tiles<D, S::STAGES, kLoadWarps>(a, maps, w, sm, sh->full, sh->empty, stage, phase, issued, dead,
                                                      warp - LOAD_WARP))
                break;
        }
    } else if (warp == MMA_WARP) {
        // ---------------- MMA issuer (one lane; the warp together clears unseen value rows)
        constexpr uint32_t id_s = idesc_bf16(128, N, false, false);
        constexpr uint32_t id_o = idesc_bf16(128, N, true, false);
        const uint32_t k_lo = desc_lo(smem_u32(sm), 16), v_lo = desc_lo(smem_u32(sm), 16384);
        const uint32_t q_lo = desc_lo(smem_u32(sm) + S::OFF_Q, 16), p_lo = desc_lo(smem_u32(sm) + S::OFF_P, 16);
        uint32_t items = 0, done = 0;                           // done: kv tiles finished so far
        auto mma_s = [&](uint32_t qb, uint32_t buf, int st) {   // S^T[buf] = K Q^T
            const uint32_t k = uniform(k_lo + st * (S::STAGE >> 4)), q = uniform(q_lo + qb * (S::Q_BYTES >> 4));
            const uint32_t d = uniform(tmem + buf * N);
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    umma_bf16_ss(d, desc_of(k + (kk >> 2) * 1024 + (kk & 3) * 2), desc_of(q + (kk >> 2) * (N * 8) + (kk & 3) * 2),
                                 id_s, kk > 0);
                umma_commit(&sh->s_full[buf]);
            }
        };
        auto mma_o = [&](uint32_t buf, int st, bool add) {      // O^T (+)= V^T P^T[buf]
            const uint32_t v = uniform(v_lo + st * (S::STAGE >> 4)), p = uniform(p_lo + buf * (S::P_BYTES >> 4));
            const uint32_t d = uniform(tmem + S::T_O), acc = uniform(add);
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < kTile / 16; ++kk)
                    umma_bf16_ss(d, desc_of(v + kk * 128), desc_of(p + (kk >> 2) * (N * 8) + (kk & 3) * 2), id_o,
                                 kk > 0 ? 1u : acc);
            }
        };
        auto commit = [&](uint64_t* bar) {
            if (elect_one()) umma_commit(bar);
        };
        Walk w;
        for (w.start(a, piece, tt); w.valid(); w.next(a, tt)) {
            if (w.t0 >= w.t1) continue;
            const uint32_t qb = items & 1;
            if (!warp_wait(&sh->q_full[qb], (items >> 1) & 1u, a.err, dead)) break;
            ++items;
            const int n = w.t1 - w.t0;
            if (!warp_wait(&sh->full[stage], phase, a.err, dead)) break;
            tc_fence_after();
            mma_s(qb, done & 1u, stage);
            commit(&sh->empty[stage]);
            if (n == 1) commit(&sh->q_empty[qb]);
            step();
            bool stop = false;
            for (int j = 0; j < n; ++j) {
                const int vst = stage;
                const uint32_t vph = phase;
                step();
                if (j + 1 < n) {
                    if (!warp_wait(&sh->full[stage], phase, a.err, dead)) { stop = true; break; }
                    tc_fence_after();
                    mma_s(qb, (done + 1) & 1u, stage);
                    commit(&sh->empty[stage]);
                    if (j + 2 == n) commit(&sh->q_empty[qb]);
                    step();
                }
                if (!warp_wait(&sh->full[vst], vph, a.err, dead)) { stop = true; break; }
                clear_rows<D>(w, w.t0 + j, sm + vst * S::STAGE);
                if (!warp_wait(&sh->p_full[done & 1u], (done >> 1) & 1u, a.err, dead)) { stop = true; break; }
                tc_fence_after();
                mma_o(done & 1u, vst, j > 0);
                commit(&sh->empty[vst]);
                commit(&sh->pv_done);
                if (j + 1 == n) commit(&sh->o_full);
                ++done;
            }
            if (stop) break;
        }
    } else {
        // ---------------- softmax and epilogue: thread = position of the tile, then value index.
        // Two groups of 128 threads, a half of the rows each: they share nothing but the MMAs.
        // What a tile always does is unrolled over the rows; the new maximum, the rescale and the
        // end of an item are loops over eight rows, because with those unrolled the code did not
        // stay in the instruction cache (an item of one tile took 11 us at N 16).
        // No early way out of a tile: a wait that gave up returns, and all warps keep
        // meeting at the barriers until their walk ends.
        constexpr int R = N / 2;
        const int group = tid >> 7, th = tid & 127, wg = warp & 3, r0 = group * R, bar = 1 + group;
        const uint32_t lanes = static_cast<uint32_t>(wg * 32) << 16;
        const float c = a.scale * 1.4426950408889634f;
        uint8_t* const p_base = sm + S::OFF_P + (th >> 6) * (N * 128);
        uint32_t done = 0, items = 0;
        if (tid == 0)
            for (int i = 0; i < 8; ++i) a.part_state[cta * 8 + i] = 0;
        if (th < R) sh->m[r0 + th] = -INFINITY;
        named_bar(bar, 128);
        Walk w;
        for (w.start(a, piece, tt); w.valid();) {
            const int toks = min(tt, w.s.n - w.item * tt), rows = toks * a.group;   // of the item
            const long at0 = static_cast<long>(w.s.c0 + w.item * tt) * a.Hq + w.head * a.group;
            const int nr = min(max(rows - r0, 0), R);           // rows of this half
            auto row_at = [&](int r) {                          // (token, head) row of the output
                const int tok = r / a.group;
                return at0 + static_cast<long>(tok) * a.Hq + (r - tok * a.group);
            };
            if (w.t0 >= w.t1) {
                if (w.count == 0) {                             // sees nothing
                    for (int r = r0; r < r0 + nr; ++r) {
                        const long at = row_at(r);
                        if (th < D) a.out[at * D + th] = 0;
                        if (a.lse && th == 0) a.lse[at] = -INFINITY;
                    }
                }
                w.next(a, tt);
                continue;
            }
            int lo0, hi0, lo1, hi1;                             // what the first and the last token see
            w.s.range(a, w.item * tt, w.item * tt, lo0, hi0);
            w.s.range(a, w.item * tt + toks - 1, w.item * tt + toks - 1, lo1, hi1);
            float l[R];                                         // this thread's part of the rows' sums
#pragma unroll
            for (int r = 0; r < R; ++r) l[r] = 0.f;
#pragma unroll 1
            for (int j = w.t0; j < w.t1; ++j, ++done) {
                const uint32_t buf = done & 1u, s_col = tmem + lanes + buf * N + r0;
                const int j0 = (w.first + j) * kTile, pos = j0 + th;
                // rows [from, to) of the half see this position: those of the token that stands here and of the
                // tokens after it, up to the window's end
                int from = 0, to = R;
                if (j0 + kTile > hi0 || j0 < lo1) {
                    const int tok = pos - (w.s.kv - w.s.n + w.item * tt);
                    if (a.causal) from = min(max(tok, 0) * a.group, N) - r0;
                    if (a.window > 0) to = min(max(tok + a.window, 0), N) * a.group - r0;
                    if (pos >= w.s.kv) from = R;
                }
                wait_at(smem_u32(&sh->s_full[buf]), (done >> 1) & 1u, a.err, dead);
                tc_fence_after();
                float s[R];
                tmem_ld_rows<R>(s_col, s);
                if (from > 0 || to < R) {
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        if (r < from || r >= to) s[r] = -INFINITY;
                }
                bool grow = false;                              // m = -inf: true for any finite s
#pragma unroll
                for (int q = 0; q < R; q += 8) {
                    if (q >= nr) break;
                    float m[8];
                    rows8(sh->m + r0 + q, m);
#pragma unroll
                    for (int i = 0; i < 8; ++i) grow |= q + i < nr && (s[q + i] - m[i]) * c > 8.f;
                }
                if (any_of_128(bar, grow)) {
#pragma unroll 1
                    for (int q = 0; q < nr; q += 8) {
                        float x[8];
                        tmem_ld8(s_col + q, x);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (q + i < from || q + i >= to) x[i] = -INFINITY;
                        const float top = reduce8<true>(x);
                        if ((lane & 3) == 0) sh->red[wg][r0 + q + (lane >> 2)] = top;
                    }
                    named_bar(bar, 128);
                    if (th < nr) {
                        const int r = r0 + th;
                        const float x = fmaxf(fmaxf(sh->red[0][r], sh->red[1][r]), fmaxf(sh->red[2][r], sh->red[3][r]));
                        const float m = sh->m[r];
                        sh->f[r] = x > m ? ex2_approx((m - x) * c) : 1.f;
                        if (x > m) sh->m[r] = x;
                    }
                    named_bar(bar, 128);
                    if (j > w.t0) {                             // O once P V(j - 1) is in it
                        wait_at(smem_u32(&sh->pv_done), (done - 1) & 1u, a.err, dead);
                        tc_fence_after();
#pragma unroll 1
                        for (int q = 0; q < nr; q += 8) {
                            float o[8];
                            tmem_ld8(tmem + lanes + S::T_O + r0 + q, o);
#pragma unroll
                            for (int i = 0; i < 8; ++i) o[i] *= q + i < nr ? sh->f[r0 + q + i] : 1.f;   // rows past the item's: any
                            tmem_st8(tmem + lanes + S::T_O + r0 + q, o);
                        }
                        tmem_st_wait();
#pragma unroll
                        for (int r = 0; r < R; ++r)
                            if (r < nr) l[r] *= sh->f[r0 + r];
                    }
                }
                uint8_t* const pb = p_base + buf * S::P_BYTES;
                // rows past the item's go with the last eight (their columns go nowhere)
#pragma unroll
                for (int q = 0; q < R; q += 8) {
                    if (q >= nr) break;
                    float m[8], p[8];                           // all loads before the stores, which might alias them
                    rows8(sh->m + r0 + q, m);
#pragma unroll
                    for (int i = 0; i < 8; ++i) p[i] = ex2_approx(fmaf(s[q + i], c, m[i] == -INFINITY ? 0.f : -m[i] * c));
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        l[q + i] += p[i];
                        *reinterpret_cast<uint16_t*>(pb + sw128_off(r0 + q + i, th & 63)) = f32_to_bf16_bits(p[i]);
                    }
                }
                fence_async_smem();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh->p_full[buf]);
            }
            // the sums of the threads, in order
#pragma unroll
            for (int q = 0; q < R; q += 8) {
                if (q >= nr) break;
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = l[q + i];
                const float sum = reduce8<false>(x);
                if ((lane & 3) == 0) sh->red[wg][r0 + q + (lane >> 2)] = sum;
            }
            const bool begins = w.t0 == 0, ends = w.t1 == w.count, whole = begins && ends;
            const int tok0 = w.s.c0 + w.item * tt, head = w.head;
            const long slot = (static_cast<long>(cta) * 2 + (begins ? 1 : 0)) * a.part_rows;
            w.next(a, tt);                                      // beside the last P V
            named_bar(bar, 128);
            wait_at(smem_u32(&sh->o_full), items & 1u, a.err, dead);
            ++items;
            tc_fence_after();
#pragma unroll 1
            for (int q = 0; q < nr; q += 8) {
                float o[8], sum[8];                             // loads before stores here too
                tmem_ld8(tmem + lanes + S::T_O + r0 + q, o);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = r0 + q + i;
                    sum[i] = (sh->red[0][r] + sh->red[1][r]) + (sh->red[2][r] + sh->red[3][r]);
                }
                int tok = (r0 + q) / a.group, g = r0 + q - tok * a.group;
                if (th < D)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (q + i < nr) {
                            if (whole)
                                a.out[(at0 + static_cast<long>(tok) * a.Hq + g) * D + th] =
                                    f32_to_bf16_bits(sum[i] == 0.f ? 0.f : __fdividef(o[i], sum[i]));
                            else
                                a.part_o[(slot + r0 + q + i) * D + th] = o[i];
                        }
                        if (++g == a.group) {
                            g = 0;
                            ++tok;
                        }
                    }
            }
            tc_fence_before();
            if (th < nr) {
                const int r = r0 + th;
                const float sum = (sh->red[0][r] + sh->red[1][r]) + (sh->red[2][r] + sh->red[3][r]), m = sh->m[r];
                if (!whole)
                    *reinterpret_cast<float2*>(a.part_ml + (slot + r) * 2) = make_float2(m, sum);
                else if (a.lse)
                    a.lse[row_at(r)] = sum == 0.f ? -INFINITY : m * a.scale + logf(sum);
            }
            if (th < R) sh->m[r0 + th] = -INFINITY;             // for the next item
            if (tid == 0 && !whole) {
                int* ps = a.part_state + cta * 8;
                if (begins) {
                    ps[1] = 1;
                    ps[2] = tok0;                                // first token
                    ps[3] = toks;
                    ps[4] = head;
                } else {
                    ps[0] = ends ? 2 : 1;                        // 2: the item's last part
                }
            }
            named_bar(bar, 128);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (sh->abort && warp >= LOAD_WARP) {
        drain_ring(a, sh->full, S::STAGES, issued);
        for (uint32_t i = q_loads > 2 ? q_loads - 2 : 0; i < q_loads; ++i) mbar_wait(&sh->q_full[i & 1], (i >> 1) & 1u, a.err);
    }
    if (warp == MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem, S::COLS);
    }
}

// Joins the parts of the items that pieces cut: blocks (x, y) take the item that CTA x began and
// did not finish, 16 rows each, a warp per row, the lanes along its values.
// Six parts in flight and two blocks per SM, against 16 and one: 44.7 / 49.2 us (whole call) for 64
// rows over 32768 positions, 8 kv heads (8 items of 19 parts), 70 / 75.5 for 256 items of 2048.
template <int D>
__global__ void __launch_bounds__(512, 2) paged_attn_rows_join_kernel(const __grid_constant__ AttnArgs a, int ctas) {
    pdl_wait_prior();
    constexpr int V = D / 32, BATCH = 6;
    const int x = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // the states of this CTA and of the 31 after it in one go
    const int4 mine = __ldcg(reinterpret_cast<const int4*>(a.part_state + x * 8));
    const int head = __ldcg(a.part_state + x * 8 + 4);
    int st = x + 1 + lane < ctas ? __ldcg(a.part_state + (x + 1 + lane) * 8) : 0;
    if (mine.y == 0) return;
    int parts = 1;                                              // CTAs x, x + 1, ...: up to the one with the last part
    for (int at = x + 1;;) {
        const uint32_t end = __ballot_sync(0xffffffffu, st != 1);
        if (end) {
            const int k = __ffs(end) - 1;
            parts += k + (__shfl_sync(0xffffffffu, st, k) == 2 ? 1 : 0);
            break;
        }
        parts += 32;
        at += 32;
        st = at + lane < ctas ? __ldcg(a.part_state + (at + lane) * 8) : 0;
    }
    const float c = a.scale * 1.4426950408889634f;
    const int r = blockIdx.y * 16 + warp;
    if (r < mine.w * a.group) {
        // part 0 is CTA x's slot 1, part p the slot 0 of CTA x + p
        auto row = [&](int p) { return (static_cast<long>(x) * 2 + (p == 0 ? 1 : 2 * p)) * a.part_rows + r; };
        float m = -INFINITY, l = 0.f, o[V] = {};
        for (int p0 = 0; p0 < parts; p0 += BATCH) {             // loads of a batch under a predicate, all in flight
            float2 v[BATCH];
            float u[BATCH][V];
            float mn = m;
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
                v[k] = make_float2(0.f, 0.f);
#pragma unroll
                for (int i = 0; i < V; ++i) u[k][i] = 0.f;
                if (p0 + k < parts) {
                    v[k] = __ldcg(reinterpret_cast<const float2*>(a.part_ml) + row(p0 + k));
                    const float* src = a.part_o + row(p0 + k) * D + lane * V;
                    if constexpr (V == 4) {
                        const float4 f = __ldcg(reinterpret_cast<const float4*>(src));
                        u[k][0] = f.x; u[k][1] = f.y; u[k][2] = f.z; u[k][3] = f.w;
                    } else {
                        const float2 f = __ldcg(reinterpret_cast<const float2*>(src));
                        u[k][0] = f.x; u[k][1] = f.y;
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < BATCH; ++k) mn = fmaxf(mn, v[k].y == 0.f ? -INFINITY : v[k].x);
            const float mc = mn == -INFINITY ? 0.f : mn * c, keep = ex2_approx(m * c - mc);
            m = mn;
            l *= keep;
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] *= keep;
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
                const float f = v[k].y == 0.f ? 0.f : ex2_approx(v[k].x * c - mc);
                l += v[k].y * f;
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] += u[k][i] * f;
            }
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int tok = r / a.group;
        const long at = static_cast<long>(mine.z + tok) * a.Hq + head * a.group + (r - tok * a.group);
        uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + at * D + lane * V);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) dst[i] = l == 0.f ? 0u : cvt_bf16x2(o[2 * i] * inv, o[2 * i + 1] * inv);
        if (a.lse && lane == 0) a.lse[at] = l == 0.f ? -INFINITY : m * a.scale + logf(l);
    }
}

template <int D, int N>
int launch(const AttnMaps& maps, const AttnArgs& a, cudaStream_t st) {
    using S = RowsShape<D, N>;
    const char* name = "gdn_paged_attn_fwd";
    static std::once_flag once[64];                             // once per device
    static cudaError_t attr[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(GDN_ERR_CUDA, "%s: no current device", name);
    std::call_once(once[dev], [dev] {
        attr[dev] = cudaFuncSetAttribute(paged_attn_rows_kernel<D, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    });
    if (attr[dev] != cudaSuccess)
        return fail(GDN_ERR_CUDA, "%s: cudaFuncSetAttribute: %s", name, cudaGetErrorString(attr[dev]));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = pdl;
    cfg.numAttrs = launch_overlap() ? 1 : 0;
    cfg.stream = st;
    cfg.gridDim = dim3(a.whole ? a.whole : kMaxCtas);
    cfg.blockDim = dim3(kRowsThreads);
    cfg.dynamicSmemBytes = S::SMEM;
    cudaError_t e = cudaLaunchKernelEx(&cfg, paged_attn_rows_kernel<D, N>, maps, a);
    if (e != cudaSuccess) return fail(GDN_ERR_CUDA, "%s: launch failed: %s", name, cudaGetErrorString(e));
    if (a.whole) return launch_status(name);
    cfg.gridDim = dim3(kMaxCtas, N / 16);
    cfg.numAttrs = 1;                                           // starts while the first kernel ends
    cfg.blockDim = dim3(512);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, paged_attn_rows_join_kernel<D>, a, static_cast<int>(kMaxCtas));
    if (e != cudaSuccess) return fail(GDN_ERR_CUDA, "%s: join launch failed: %s", name, cudaGetErrorString(e));
    return launch_status(name);
}

}  // namespace

int launch_attn_rows(const AttnMaps& maps, const AttnArgs& a, int D, cudaStream_t st) {
    if (D == 64)
        return a.part_rows == 16   ? launch<64, 16>(maps, a, st)
               : a.part_rows == 32 ? launch<64, 32>(maps, a, st)
                                   : launch<64, 64>(maps, a, st);
    return a.part_rows == 16   ? launch<128, 16>(maps, a, st)
           : a.part_rows == 32 ? launch<128, 32>(maps, a, st)
                               : launch<128, 64>(maps, a, st);
}

}  // namespace gdn
