// paged_attn.cu -- softmax attention of new tokens over a paged key/value cache, on tcgen05.
//
// Token i of sequence b stands at position p = kv_len - q_len + i and sees the positions
// lo .. hi of its mask.  One pass over them in tiles of 128, with a running reference
// maximum m and sum l per row (fp32; c = scale log2 e):
//   p_j = 2^(c (s_j - m)),   l = l a + sum p_j,   o = o a + sum p_j v_j,   s_j = q . k_j
//   out = o / l,  lse = scale m + ln l;   a row that sees nothing keeps l = 0: out 0, lse -inf.
// a = 2^(c (m_old - m_new)) is 1 unless the maximum grew by more than 2^8 in p: the sums
// are exact for any m near the maximum, so a smaller growth leaves m and o where they are.
//
// Rows.  The G query heads that share a kv head are packed with their tokens into rows
// (row = token G + g), floor(128 / G) tokens to a tile of 128, so that a key is read once
// for its whole group.
//
// Work.  An item is (sequence, kv head, two row tiles); its kv tiles are the ones that some
// row of it sees.  All kv tiles of all items, with a constant cost per item, form one line
// that is cut into equal pieces, one per CTA: a long sequence is split over many CTAs and a
// CTA may take many short ones.  An item cut by a piece's end leaves its o, m, l in the
// workspace, and a second small kernel joins such parts in a fixed order.  The pieces follow
// from the lengths on the device, so a captured launch serves every length.
//
// Roles.  A producer warp loads q, k, v by TMA (128-byte swizzle, a ring of stages; a
// lane per page); one thread issues the MMAs; a warpgroup per row tile does the softmax,
// a thread per row:
//   S = Q K^T   M 128, N 128 (SS)      -> TMEM, 128 columns per S buffer
//   P (bf16) overwrites S in TMEM      (rounded to bf16: 2^-9 rms of each weight)
//   O += P V    M 128, N D (TS)        -> TMEM, fp32 over the whole pass
// The tensor core works for one row tile while the softmax of the other runs.  Items of
// at most 64 rows (a decode step) go to paged_attn_rows.cu.
//
// What bounds it.  A kv tile of both row tiles is 32 MMAs of about 61 cycles and 128 x 256
// exponentials, 2048 cycles either if nothing else ran.  The softmax takes 3400 cycles of its
// warps, two to a scheduler: loads of S, maxima, exponentials, conversions and stores of P one
// after the other, 128 scores of a row in 168 registers (264 bytes a thread spilled), and 600 to
// 900 cycles of waiting for the MMAs.  2048 new tokens over 32768, 16 heads on 2, head dim 128:
// 430 us (1.24 PFLOP/s) at 1.97 GHz, 487 (1.09) in sustained passes, where the power cap lowers
// the clock to 1.64 GHz.
#include <cstddef>
#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "paged_work.cuh"
#include "tensormap.h"

namespace gdn {
namespace {

constexpr int QT = 2;                 // row tiles of 128 per item
// kv tiles that starting and ending an item is worth, beside its tiles.  With 1 / 2 / 3, us: 40 chunks of up to
// 130 tokens over 500 36.9 / 32.8 / 35.5, 16 of 300 over 3000 73 / 62 / 62, 32 of 200 over 200 31 / 28.7 / 27
constexpr int kItemCost = 2;
constexpr int kJoinThreads = 256, kJoinBlocks = 2;  // of the join kernel, per SM
constexpr int kWholeTiles = 8;        // items of so many kv tiles are not cut when there are few
constexpr int kEarly = 3;             // quarters of a tile's P after which P V starts
// pairs of weights in every so many that take the polynomial on the FMA pipe, the others the MUFU
// (2048 tokens over 32768: 486 us with three of eight, 495 with a quarter or two fifths)
constexpr int kPolyPairs = 3, kPolyOf = 8;

// umma_commit to a barrier given by its shared-memory address
__device__ __forceinline__ void commit_to(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 2^x for two x <= 128 on the FMA pipe: x = n + f, |f| <= 1/2, n by adding 1.5 2^23; 2^f by
// the degree-4 polynomial of least relative error (2.7e-6, found by linear programming
// over Chebyshev nodes); n goes into the exponent bits, so results below 2^-126 are off by up
// to 2^-127.  x below -127 + 2^-10 (a masked position's -inf) counts as that, whose bits, 8e-42,
// are 0 in bf16.  The integer add makes a NaN (0x7fffffff) the largest finite number, which the
// caller has to look for.
__device__ __forceinline__ void exp2_poly2(float& x0, float& x1) {
    constexpr float kRound = 12582912.f, kLeast = -126.9990234375f;
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x0) : "f"(kLeast));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x1) : "f"(kLeast));
    const uint64_t x = pack2(x0, x1);
    const uint64_t t = add2(x, pack2(kRound, kRound));
    const uint64_t n = add2(t, pack2(-kRound, -kRound));
    const uint64_t f = fma2(n, pack2(-1.f, -1.f), x);
    uint64_t r = fma2(f, pack2(9.570102207362652e-3f, 9.570102207362652e-3f), pack2(5.591785907745361e-2f, 5.591785907745361e-2f));
    r = fma2(f, r, pack2(0.240247443318367f, 0.240247443318367f));
    r = fma2(f, r, pack2(0.6931217908859253f, 0.6931217908859253f));
    r = fma2(f, r, pack2(0.9999992847442627f, 0.9999992847442627f));
    float t0, t1, r0, r1;
    unpack2(t, t0, t1);
    unpack2(r, r0, r1);
    x0 = __uint_as_float(__float_as_uint(r0) + (__float_as_uint(t0) << 23));
    x1 = __uint_as_float(__float_as_uint(r1) + (__float_as_uint(t1) << 23));
}

template <int D>
struct Shape {
    static constexpr int HALVES = D / 64;
    static constexpr int Q_BYTES = QT * kTile * D * 2;
    static constexpr int STAGE = kTile * D * 2;                 // one K or V tile
    static constexpr int OUT_BYTES = QT * 4 * 4096;             // 32 rows x 64 values per softmax warp
    static constexpr int STAGES_FIT = (232448 - 2048 - Q_BYTES - OUT_BYTES) / STAGE;
    static constexpr int STAGES = STAGES_FIT < 10 ? STAGES_FIT : 10;
    static constexpr int OFF_KV = Q_BYTES;
    static constexpr int OFF_OUT = OFF_KV + STAGES * STAGE;
    static constexpr int OFF_BAR = OFF_OUT + OUT_BYTES;
    static constexpr int SMEM = OFF_BAR + 1024 + 1024;          // barriers and state; alignment
    static constexpr int THREADS = QT * 128 + 64;
    // TMEM columns: S buffers of 128, then O
    static constexpr int T_O = 2 * kTile;
    static constexpr int O_COLS = D;
    static_assert(SMEM <= 232448, "shared memory");
    static_assert(T_O + QT * O_COLS <= 512, "TMEM");
};

struct Bars {
    uint64_t full[16], empty[16];     // kv ring
    uint64_t q_full, q_empty;
    uint64_t s_full[2], p_part[2], p_full[2];
    uint64_t o_full[2];
    PieceScratch scratch;
    uint32_t tmem;
    int abort;
};
static_assert(sizeof(Bars) <= 1024, "barrier block");

template <int D>
__global__ void __launch_bounds__(Shape<D>::THREADS, 1)
paged_attn_kernel(const __grid_constant__ AttnMaps maps, const __grid_constant__ AttnArgs a) {
    using S = Shape<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Bars* sh = reinterpret_cast<Bars*>(sm + S::OFF_BAR);
    volatile int* dead = &sh->abort;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int MMA_WARP = QT * 4, LOAD_WARP = QT * 4 + 1;
    const int tt = QT * a.tile_tokens;                          // tokens per item
    const int cta = blockIdx.x;

    if (tid == 0) {
        for (int i = 0; i < S::STAGES; ++i) {
            mbar_init(&sh->full[i], 1);
            mbar_init(&sh->empty[i], 1);
        }
        mbar_init(&sh->q_full, 1);
        mbar_init(&sh->q_empty, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh->s_full[i], 1);
            mbar_init(&sh->p_part[i], 4);
            mbar_init(&sh->p_full[i], 4);
            mbar_init(&sh->o_full[i], 1);
        }
        sh->abort = 0;
        fence_mbar_init();
        tma_prefetch_desc(&maps.q);
        tma_prefetch_desc(&maps.k);
        tma_prefetch_desc(&maps.v);
    }
    if (warp == MMA_WARP) {
        tmem_alloc(&sh->tmem, 512);
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
    if (warp == LOAD_WARP) {
        // ---------------- TMA producer
        int stage = 0;
        uint32_t phase = 0;
        Walk w;
        for (w.start(a, piece, tt); w.valid(); w.next(a, tt)) {
            if (w.t0 >= w.t1) continue;
            // q: rows of the item's tokens, `group` heads each
            if (!warp_wait(&sh->q_empty, (q_loads & 1u) ^ 1u, a.err, dead)) break;
            ++q_loads;
            if (lane == 0) {
                mbar_arrive_expect_tx(&sh->q_full, QT * S::HALVES * a.tile_tokens * a.group * 128);
                for (int t = 0; t < QT; ++t)
                    for (int h = 0; h < S::HALVES; ++h)
                        tma_load_3d(sm + (t * S::HALVES + h) * 16384, &maps.q, &sh->q_full, h * 64, w.head * a.group,
                                    w.s.c0 + w.item * tt + t * a.tile_tokens);
            }
            if (!load_tiles<D, S::STAGES, 1>(a, maps, w, sm + S::OFF_KV, sh->full, sh->empty, stage, phase, issued, dead)) break;
        }
    } else if (warp == MMA_WARP) {
        // ---------------- MMA issuer (one lane; the warp together clears unseen value rows).
        // The tensor core takes about one MMA in 64 cycles and queues few, so what this warp does
        // between MMAs is time lost: one shuffle a tile makes the stages uniform (descriptors then
        // stay in uniform registers), barriers go by shared-memory addresses.
        constexpr uint32_t id_s = idesc_bf16(128, kTile, false, false);
        constexpr uint32_t id_o = idesc_bf16(128, D, false, true);
        const uint32_t sm0 = uniform(smem_u32(sm)), tm = uniform(tmem), bars = smem_u32(sh);
        const uint32_t q_lo = desc_lo(sm0, 16), k_lo = desc_lo(sm0 + S::OFF_KV, 16), v_lo = desc_lo(sm0 + S::OFF_KV, 16384);
        const uint32_t full = bars + offsetof(Bars, full), empty = bars + offsetof(Bars, empty);
        const uint32_t s_full = bars + offsetof(Bars, s_full), p_part = bars + offsetof(Bars, p_part);
        const uint32_t p_full = bars + offsetof(Bars, p_full), o_full = bars + offsetof(Bars, o_full);
        const uint32_t q_full = bars + offsetof(Bars, q_full), q_empty = bars + offsetof(Bars, q_empty);
        uint32_t stage = 0, phase = 0, items = 0, done = 0;     // done: kv tiles finished so far
        auto step = [&]() {
            if (++stage == S::STAGES) {
                stage = 0;
                phase ^= 1u;
            }
        };
        // inside an elected lane's branch: S[t] = Q[t] K^T;  O[t] (+)= P[t] V over k-steps k0 .. k1 - 1
        auto mma_s = [&](int t, uint32_t st) {
            const uint32_t q = q_lo + t * (S::HALVES * 1024), k = k_lo + st * (S::STAGE >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                const uint32_t o = (kk >> 2) * 1024 + (kk & 3) * 2;
                umma_bf16_ss(tm + t * kTile, desc_of(q + o), desc_of(k + o), id_s, kk > 0);
            }
            commit_to(s_full + t * 8);
        };
        auto mma_o = [&](int t, uint32_t st, uint32_t add, auto k0, auto k1) {
            const uint32_t v = v_lo + st * (S::STAGE >> 4);
#pragma unroll
            for (int kk = decltype(k0)::value; kk < decltype(k1)::value; ++kk)
                umma_bf16_ts(tm + S::T_O + t * S::O_COLS, tm + t * kTile + kk * 8, desc_of(v + kk * 128), id_o, kk > 0 ? 1u : add);
        };
        constexpr std::integral_constant<int, 0> k_first{};
        constexpr std::integral_constant<int, kEarly * 2> k_early{};
        constexpr std::integral_constant<int, kTile / 16> k_last{};
        Walk w;
        for (w.start(a, piece, tt); w.valid(); w.next(a, tt)) {
            if (w.t0 >= w.t1) continue;
            const int n = w.t1 - w.t0;
            // only the item's first and last tile hold positions that no row of it sees
            const int clear_lo = (w.first + w.t0) * kTile < w.lo ? 0 : -1;
            const int clear_hi = (w.first + w.t1) * kTile > w.hi ? n - 1 : -1;
            wait_at(q_full, items & 1u, a.err, dead);
            ++items;
            wait_at(full + stage * 8, phase, a.err, dead);
            tc_fence_after();
            {
                const uint32_t k = uniform(stage);
                if (elect_one()) {
                    mma_s(0, k);
                    mma_s(1, k);
                    commit_to(empty + k * 8);
                    if (n == 1) commit_to(q_empty);
                }
            }
            step();
            for (int j = 0; j < n; ++j) {
                const uint32_t vst = stage, vph = phase;
                step();
                const uint32_t kst = stage, kph = phase;
                const bool more = j + 1 < n;
                if (more) step();
                const uint32_t both = uniform(vst | kst << 8 | (j > 0 ? 1u << 16 : 0u));
                const uint32_t v = both & 0xff, k = (both >> 8) & 0xff, add = both >> 16, ph = done & 1u;
                wait_at(full + vst * 8, vph, a.err, dead);
                if (j == clear_lo || j == clear_hi) clear_rows<D>(w, w.t0 + j, sm + S::OFF_KV + vst * S::STAGE);
                wait_at(p_part, ph, a.err, dead);
                tc_fence_after();
                if (elect_one()) mma_o(0, v, add, k_first, k_early);
                wait_at(p_full, ph, a.err, dead);
                tc_fence_after();
                if (more) wait_at(full + kst * 8, kph, a.err, dead);
                if (elect_one()) {
                    mma_o(0, v, add, k_early, k_last);
                    if (more)
                        mma_s(0, k);
                    else
                        commit_to(o_full);
                }
                wait_at(p_part + 8, ph, a.err, dead);
                tc_fence_after();
                if (elect_one()) mma_o(1, v, add, k_first, k_early);
                wait_at(p_full + 8, ph, a.err, dead);
                tc_fence_after();
                if (elect_one()) {
                    mma_o(1, v, add, k_early, k_last);
                    commit_to(empty + v * 8);
                    if (more) {
                        mma_s(1, k);
                        commit_to(empty + k * 8);
                        if (j + 2 == n) commit_to(q_empty);
                    } else {
                        commit_to(o_full + 8);
                    }
                }
                ++done;
            }
        }
    } else {
        // ---------------- softmax and epilogue: a thread per row
        const int t = warp >> 2;                                // row tile
        const int row = tid & 127;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const int tok = row / a.group, g = row - tok * a.group; // token within the row tile, head within the group
        const float c = a.scale * 1.4426950408889634f;
        const uint32_t o_col = tmem + lanes + S::T_O + t * S::O_COLS;
        const uint32_t s_full = smem_u32(&sh->s_full[t]), o_full = smem_u32(&sh->o_full[t]);
        uint32_t done = 0, items = 0;
        if (tid == 0)
            for (int i = 0; i < 8; ++i) a.part_state[cta * 8 + i] = 0;
        Walk w;
        for (w.start(a, piece, tt); w.valid();) {
            const int rel = w.item * tt + t * a.tile_tokens + tok;      // token within the chunk
            const bool real = tok < a.tile_tokens && rel < w.s.n;
            const int first_tok = w.item * tt + t * a.tile_tokens;
            const int last_tok = min(first_tok + a.tile_tokens, w.s.n) - 1;
            const bool busy = __any_sync(0xffffffffu, real);
            const long at = static_cast<long>(w.s.c0 + rel) * a.Hq + w.head * a.group + g;
            if (w.t0 >= w.t1) {
                if (w.count == 0 && real) {                             // sees nothing
                    uint4* o = reinterpret_cast<uint4*>(a.out + at * D);
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) o[i] = make_uint4(0, 0, 0, 0);
                    if (a.lse) a.lse[at] = -INFINITY;
                }
                w.next(a, tt);
                continue;
            }
            int lo, hi, dummy, hi_first, lo_last;
            w.s.range(a, rel, rel, lo, hi);
            w.s.range(a, first_tok, first_tok, dummy, hi_first);
            w.s.range(a, last_tok, last_tok, lo_last, dummy);
            float m = -INFINITY, l = 0.f;
            for (int j = w.t0; j < w.t1; ++j) {
                wait_at(s_full, done & 1u, a.err, dead);
                tc_fence_after();
                if (busy) {
                    const uint32_t s_col = tmem + lanes + t * kTile;
                    const int j0 = (w.first + j) * kTile;
                    float s[kTile];
                    // once, or, after a rescale (a row of S and one of O do not fit the registers), twice: a
                    // loop, because the code of an item's rare parts would push the rest out of the
                    // instruction cache
#pragma unroll 1
                    for (;;) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) tmem_ld32(s_col + q * 32, reinterpret_cast<float(&)[32]>(s[q * 32]));
                        tmem_ld_wait();
                        if (j0 + kTile > hi_first || j0 < lo_last) {     // bits of the positions this row sees
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const int e = min(max(hi - j0 - q * 32, 0), 32), b = min(max(lo - j0 - q * 32, 0), 32);
                                const uint32_t bits = (e == 32 ? ~0u : (1u << e) - 1u) & ~(b == 32 ? ~0u : (1u << b) - 1u);
#pragma unroll
                                for (int i = 0; i < 32; ++i)
                                    if (!(bits & (1u << i))) s[q * 32 + i] = -INFINITY;
                            }
                        }
                        // four chains, two values an instruction
                        float mx4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                        for (int i = 4; i < kTile; i += 8)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                mx4[e] = i + 4 + e < kTile ? max3(mx4[e], s[i + e], s[i + 4 + e]) : fmaxf(mx4[e], s[i + e]);
                        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                        if (j == w.t0) {
                            m = mx;
                            break;
                        }
                        const bool grow = real && (mx - m) * c > 8.f;    // m = -inf: true for any finite mx
                        if (!__any_sync(0xffffffffu, grow)) break;
                        const float r = grow ? ex2_approx((m - mx) * c) : 1.f;
                        if (grow) m = mx;
                        l *= r;
                        // O is at rest: S(j) was issued after P V(j - 1)
#pragma unroll 1
                        for (int q = 0; q < D / 32; ++q) {
                            float o[32];
                            tmem_ld32(o_col + q * 32, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] *= r;
                            tmem_st32(o_col + q * 32, o);
                        }
                    }
                    const float mc = m == -INFINITY ? 0.f : m * c;
                    const uint64_t c2 = pack2(c, c), mc2 = pack2(-mc, -mc);
                    uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint32_t p[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            float x0, x1;
                            unpack2(fma2(pack2(s[q * 32 + 2 * i], s[q * 32 + 2 * i + 1]), c2, mc2), x0, x1);
                            if ((i % kPolyOf) < kPolyPairs) {
                                exp2_poly2(x0, x1);
                            } else {
                                x0 = ex2_approx(x0);
                                x1 = ex2_approx(x1);
                            }
                            sum[i & 3] = add2(sum[i & 3], pack2(x0, x1));
                            p[i] = cvt_bf16x2(x0, x1);
                        }
                        tmem_st16(s_col + q * 16, p);
                        if (q == kEarly - 1) {                   // the first part of P V may start
                            tmem_st_wait();
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(&sh->p_part[t]);
                        }
                    }
                    float l0, l1;
                    unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), l0, l1);
                    // a NaN score (or inf - inf) makes the row NaN: its weight is one too, or, from the polynomial,
                    // the largest number, where all others are at most 2^8
                    l = l0 + l1 < 1e30f ? l + (l0 + l1) : __int_as_float(0x7fffffff);
                    tmem_st_wait();
                } else {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh->p_part[t]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh->p_full[t]);
                ++done;
            }
            const bool begins = w.t0 == 0, ends = w.t1 == w.count, whole = begins && ends;
            const int tok0 = w.s.c0 + w.item * tt, toks = min(tt, w.s.n - w.item * tt), head = w.head;
            w.next(a, tt);                                              // beside the last P V
            wait_at(o_full, items & 1u, a.err, dead);
            ++items;
            tc_fence_after();
            if (m == -INFINITY && l < 1.f) l = 0.f;                     // saw nothing (the polynomial gives 8e-42 for 2^-inf)
            if (busy) {
                if (whole) {
                    // through shared memory, so that a store instruction writes whole lines: 64
                    // values of the warp's 32 rows at a time, 16-byte pieces swizzled by the row
                    const float inv = l == 0.f ? 0.f : 1.f / l;          // NaN for a NaN
                    const long mine = real ? at : -1;
                    uint8_t* buf = sm + S::OFF_OUT + warp * 4096;
#pragma unroll 1
                    for (int hf = 0; hf < S::HALVES; ++hf) {
#pragma unroll 1
                        for (int q = 0; q < 2; ++q) {
                            float o[32];
                            tmem_ld32(o_col + hf * 64 + q * 32, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float x[8];
#pragma unroll
                                for (int e = 0; e < 8; ++e) x[e] = l == 0.f ? 0.f : o[i * 8 + e] * inv;
                                *reinterpret_cast<uint4*>(buf + sw128_chunk(lane, q * 4 + i)) =
                                    make_uint4(cvt_bf16x2(x[0], x[1]), cvt_bf16x2(x[2], x[3]), cvt_bf16x2(x[4], x[5]),
                                               cvt_bf16x2(x[6], x[7]));
                            }
                        }
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int r = i * 4 + (lane >> 3);
                            const long to = __shfl_sync(0xffffffffu, mine, r);
                            if (to >= 0)
                                reinterpret_cast<uint4*>(a.out + to * D + hf * 64)[lane & 7] =
                                    *reinterpret_cast<const uint4*>(buf + sw128_chunk(r, lane & 7));
                        }
                        __syncwarp();
                    }
                    if (a.lse && real) a.lse[at] = l == 0.f ? -INFINITY : m * a.scale + logf(l);
                } else {
                    // slot 0: a part that does not hold the item's first tile; 1: the first part
                    const long part = static_cast<long>(cta) * 2 + (begins ? 1 : 0), slot = part * a.part_rows + t * 128 + row;
                    float4* dst = reinterpret_cast<float4*>(a.part_o) + part * (D / 4) * a.part_rows + t * 128 + row;
#pragma unroll 1
                    for (int q = 0; q < D / 32; ++q) {
                        float o[32];
                        tmem_ld32(o_col + q * 32, o);
                        tmem_ld_wait();
                        if (real)
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                dst[(q * 8 + i) * a.part_rows] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                    if (real) {
                        a.part_ml[slot * 2] = m;
                        a.part_ml[slot * 2 + 1] = l;
                    }
                }
                tc_fence_before();
            }
            if (tid == 0 && !whole) {
                int* ps = a.part_state + cta * 8;
                if (begins) {
                    ps[1] = 1;
                    ps[2] = tok0;                                        // first token
                    ps[3] = toks;
                    ps[4] = head;
                } else {
                    ps[0] = ends ? 2 : 1;                                // 2: the item's last part
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (sh->abort && warp == LOAD_WARP) {
        drain_ring(a, sh->full, S::STAGES, issued);
        if (q_loads > 0) mbar_wait(&sh->q_full, (q_loads - 1) & 1u, a.err);
    }
    if (warp == MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// What the join kernel knows of an item that CTA x began and did not finish.
struct Cut {
    int x, parts, tok0, toks, head;
};

// Joins 32 rows (a lane each, as the parts lie in memory) of a cut item, C float4 of their
// values from float4 c0 on: one pass over the parts with a running maximum, loads in batches of
// N parts under a predicate (a remainder loop would wait for each of them).
template <int D, int C, int N>
__device__ __forceinline__ void join_rows(const AttnArgs& a, const Cut& w, int slice, int c0) {
    const int rows = a.part_rows, row = slice * 32 + (threadIdx.x & 31), r = row & 127;
    const int tl = r / a.group, tok = (row >> 7) * a.tile_tokens + tl;
    if (tl >= a.tile_tokens || tok >= w.toks) return;
    const float c = a.scale * 1.4426950408889634f;
    // part 0 is CTA x's slot 1, part p the slot 0 of CTA x + p
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + static_cast<long>(w.x) * 2 * rows + row;
    const float4* po = reinterpret_cast<const float4*>(a.part_o) + (static_cast<long>(w.x) * 2 * (D / 4) + c0) * rows + row;
    auto slot = [](int p) { return p == 0 ? 1 : 2 * p; };
    float m = -INFINITY, l = 0.f;
    float4 o[C];
#pragma unroll
    for (int i = 0; i < C; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int p0 = 0; p0 < w.parts; p0 += N) {
        float2 v[N];
        float4 u[N][C];
        float mn = m;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            v[k] = p0 + k < w.parts ? __ldcg(ml + slot(p0 + k) * rows) : make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < C; ++i)
                u[k][i] = p0 + k < w.parts ? __ldcg(po + (static_cast<long>(slot(p0 + k)) * (D / 4) + i) * rows)
                                           : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int k = 0; k < N; ++k) mn = fmaxf(mn, v[k].y == 0.f ? -INFINITY : v[k].x);
        const float mc = mn == -INFINITY ? 0.f : mn * c, keep = ex2_approx(m * c - mc);
        m = mn;
        l *= keep;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            o[i].x *= keep; o[i].y *= keep; o[i].z *= keep; o[i].w *= keep;
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const float f = v[k].y == 0.f ? 0.f : ex2_approx(v[k].x * c - mc);
            l += v[k].y * f;
#pragma unroll
            for (int i = 0; i < C; ++i) {
                o[i].x += u[k][i].x * f; o[i].y += u[k][i].y * f; o[i].z += u[k][i].z * f; o[i].w += u[k][i].w * f;
            }
        }
    }
    const long at = static_cast<long>(w.tok0 + tok) * a.Hq + w.head * a.group + (r - tl * a.group);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint2* dst = reinterpret_cast<uint2*>(a.out + at * D) + c0;
#pragma unroll
    for (int i = 0; i < C; ++i)
        dst[i] = l == 0.f ? make_uint2(0u, 0u)
                          : make_uint2(cvt_bf16x2(o[i].x * inv, o[i].y * inv), cvt_bf16x2(o[i].z * inv, o[i].w * inv));
    if (a.lse && c0 == 0) a.lse[at] = l == 0.f ? -INFINITY : m * a.scale + logf(l);
}

// Joins the parts of the items that pieces cut.  Every block lists the cut items (up to one per
// CTA), then the warps of the grid share them: 32 rows x 16 values each, or, where the items are
// too few for that to fill the GPU, which is also where they have many parts, 32 rows x 4 values
// with four times the parts in flight (5 tokens over 32768, 8 kv heads,
// 19 parts each: 9 us; 22 with 16 values).  Registers for the loads in flight count more than warps:
// 256 threads twice per SM 13.6 us for 148 items of head dim 128, 512 threads with 64 registers 18.
template <int D>
__global__ void __launch_bounds__(kJoinThreads, kJoinBlocks) paged_attn_join_kernel(const __grid_constant__ AttnArgs a, int ctas) {
    constexpr int WORDS = (kMaxCtas + 31) / 32;
    __shared__ Cut cut[kMaxCtas];
    __shared__ uint32_t begun[WORDS], more[WORDS], last[WORDS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait_prior();
    int4 st = make_int4(0, 0, 0, 0);
    int head = 0;
    if (warp < WORDS) {                                         // thread x: CTA x's state
        if (tid < ctas) {
            st = __ldcg(reinterpret_cast<const int4*>(a.part_state + tid * 8));
            head = __ldcg(a.part_state + tid * 8 + 4);
        }
        const uint32_t b = __ballot_sync(0xffffffffu, st.y != 0), m = __ballot_sync(0xffffffffu, st.x == 1),
                       e = __ballot_sync(0xffffffffu, st.x == 2);
        if (lane == 0) {
            begun[warp] = b;
            more[warp] = m;
            last[warp] = e;
        }
    }
    __syncthreads();
    int n = 0, mine = 0;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
        const int k = __popc(begun[i]);
        if (i < warp) mine += k;
        n += k;
    }
    if (st.y != 0) {
        mine += __popc(begun[warp] & ((1u << lane) - 1));
        int at = tid + 1;                                       // CTAs x + 1, ...: up to the one with the last part
        while (at < ctas && (more[at >> 5] >> (at & 31) & 1)) ++at;
        const int ends = at < ctas ? static_cast<int>(last[at >> 5] >> (at & 31) & 1) : 0;
        cut[mine] = Cut{tid, at - tid + ends, st.z, st.w, head};
    }
    __syncthreads();
    const int slices = a.part_rows / 32, warps = gridDim.x * (kJoinThreads / 32);
    const bool wide = n * slices * (D / 16) * 2 >= warps;
    const int cols = wide ? D / 16 : D / 4;
    for (int u = blockIdx.x * (kJoinThreads / 32) + warp; u < n * slices * cols; u += warps) {
        const int c = u % cols, slice = u / cols % slices;
        const Cut& w = cut[u / cols / slices];
        if (wide)
            join_rows<D, 4, 4>(a, w, slice, c * 4);
        else
            join_rows<D, 1, 8>(a, w, slice, c);
    }
}

// Kernel by the rows (tokens x heads of a group) of the longest chunk: up to 64 the one for
// few rows, which keeps them in the MMA's narrow dimension, else the one with 128-row tiles.
// Both sides, us: 25 rows (16 x 5 tokens over 4096, head dim 64) 43 / 65; 40 (5 tokens over 32768)
// 41 / 51, (32 x 5 over 4096, head dim 64) 96 / 115; 64 (8 tokens x 8 heads over 32768) 45 / 52,
// (4 x 16 over 4096) 44 / 51, (1 x 64 over 100000, head dim 64) 40 / 54.
bool few_rows(int max_q, int group) { return static_cast<long>(max_q > 1 ? max_q : 1) * group <= 64; }

// Rows of an unfinished item's part.
int part_rows(int max_q, int group) {
    return !few_rows(max_q, group) ? QT * 128 : max_q * group <= 16 && group <= 16 ? 16 : max_q * group <= 32 && group <= 32 ? 32 : 64;
}

// CTAs for a call whose items are few and short enough to be left whole, one per item, so
// that no second launch has to join parts; 0: the work is cut.  Both sides on the device, us,
// whole / cut: 1 token over 1000 positions 13.0 / 13.2 (and 3 less on the host), 8 x 1 over 1000
// 13.1 / 14.8, 100 over 1000 23.5 / 29.7, 1 over 2000 19.2 / 12.7, 100 over 2000 38 / 33.
int whole_items(int B, int T, int n_kv, int item_tokens, int max_kv) {
    const long most = static_cast<long>(n_kv) * (static_cast<long>(B) + T / item_tokens);
    return most <= kMaxCtas && max_kv <= kWholeTiles * kTile ? static_cast<int>(most) : 0;
}

template <int D>
int launch(const AttnMaps& maps, const AttnArgs& a, cudaStream_t st) {
    using S = Shape<D>;
    const char* name = "gdn_paged_attn_fwd";
    static std::once_flag once[64];                             // once per device
    static cudaError_t attr[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(GDN_ERR_CUDA, "%s: no current device", name);
    std::call_once(once[dev], [dev] {
        attr[dev] = cudaFuncSetAttribute(paged_attn_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    });
    if (attr[dev] != cudaSuccess)
        return fail(GDN_ERR_CUDA, "%s: cudaFuncSetAttribute: %s", name, cudaGetErrorString(attr[dev]));
    paged_attn_kernel<D><<<a.whole ? a.whole : kMaxCtas, S::THREADS, S::SMEM, st>>>(maps, a);
    int rc = launch_status(name);
    if (rc != GDN_OK || a.whole) return rc;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3(kJoinBlocks * kMaxCtas);                         // one wave
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = st;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_attn_join_kernel<D>, a, static_cast<int>(kMaxCtas));
    if (e != cudaSuccess) return fail(GDN_ERR_CUDA, "%s: join launch failed: %s", name, cudaGetErrorString(e));
    return launch_status(name);
}

}  // namespace
}  // namespace gdn

extern "C" size_t gdn_paged_attn_workspace_bytes(int B, int Ttot, int Hq, int n_kv, int head_dim, int max_q, int max_kv,
                                                 int window) {
    using namespace gdn;
    (void)window;
    if (B < 1 || Ttot < 1 || Hq < 1 || n_kv < 1 || Hq % n_kv != 0 || Hq / n_kv > 64 || max_q < 0 || max_kv < 0 ||
        (head_dim != 64 && head_dim != 128))
        return 0;
    const int rows = part_rows(max_q, Hq / n_kv);
    return part_state_bytes() + part_ml_bytes(rows) + part_o_bytes(rows, head_dim);
}

extern "C" int gdn_paged_attn_fwd(const void* q, long q_ld, const gdn_paged_cache* cache, const int* cu_seqlens,
                                  const int* kv_lens, void* out, float* lse, int B, int Ttot, int Hq, int max_q,
                                  int max_kv, int causal, int window, float scale, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    using namespace gdn;
    const char* name = "gdn_paged_attn_fwd";
    PagedView pv;
    int st = check_cache(name, cache, &pv);
    if (st != GDN_OK) return st;
    if (!q || !cu_seqlens || !kv_lens || !out)
        return fail(GDN_ERR_NULL, "%s: q, cu_seqlens, kv_lens and out are required", name);
    const int D = cache->head_dim;
    if (D != 64 && D != 128) return fail(GDN_ERR_UNSUPPORTED, "%s: head dim %d (64 or 128)", name, D);
    if (B < 1 || Ttot < 0 || Hq < 1 || max_q < 0 || max_kv < 0)
        return fail(GDN_ERR_SHAPE, "%s: B=%d Ttot=%d Hq=%d max_q=%d max_kv=%d", name, B, Ttot, Hq, max_q, max_kv);
    if (Hq % cache->n_kv != 0 || Hq / cache->n_kv > 64)
        return fail(GDN_ERR_SHAPE, "%s: Hq=%d must be a multiple, at most 64 times, of n_kv=%d", name, Hq, cache->n_kv);
    if (max_kv > cache->max_pages * cache->page_size)
        return fail(GDN_ERR_SHAPE, "%s: max_kv=%d exceeds the %d positions of a block_table row", name, max_kv,
                    cache->max_pages * cache->page_size);
    if (Ttot > 1 && q_ld < static_cast<long>(Hq) * D) return fail(GDN_ERR_SHAPE, "%s: q rows of %ld elements overlap", name, q_ld);
    if (window < 0 || (window > 0 && !causal)) return fail(GDN_ERR_ARG, "%s: a window needs causal, and must not be negative", name);
    if (!(scale >= 0.f) || scale > 3e38f) return fail(GDN_ERR_ARG, "%s: scale must be positive (0: 1/sqrt(D)), got %g", name, scale);
    if (!aligned16(q) || !aligned16(out) || q_ld % 8 != 0)
        return fail(GDN_ERR_ALIGN, "%s: q, its rows and out must be 16-byte aligned", name);
    const size_t need = gdn_paged_attn_workspace_bytes(B, Ttot, Hq, cache->n_kv, D, max_q, max_kv, window);
    if (Ttot > 0 && (!workspace || workspace_bytes < need))
        return fail(GDN_ERR_SHAPE, "%s: workspace of %zu bytes is smaller than %zu", name, workspace ? workspace_bytes : 0, need);
    if (!aligned16(workspace)) return fail(GDN_ERR_ALIGN, "%s: workspace must be 16-byte aligned", name);
    if ((st = check_sm100()) != GDN_OK) return st;
    if (Ttot == 0) return GDN_OK;
    if (max_kv > kMaxPositions) max_kv = kMaxPositions;         // a longer sequence is one outside the cache
    AttnArgs a = {};
    a.out = static_cast<uint16_t*>(out);
    a.lse = lse;
    a.cu = cu_seqlens;
    a.kv_lens = kv_lens;
    a.table = pv.table;
    a.table_ld = pv.table_ld;
    a.num_pages = pv.num_pages;
    a.page_shift = pv.page_shift;
    a.B = B;
    a.T = Ttot;
    a.Hq = Hq;
    a.n_kv = pv.n_kv;
    a.group = Hq / pv.n_kv;
    const bool few = few_rows(max_q, a.group);
    a.part_rows = part_rows(max_q, a.group);
    a.tile_tokens = (few ? a.part_rows : 128) / a.group;        // at least 1: group <= 64, and <= part_rows for few rows
    a.max_q = max_q;
    a.max_kv = max_kv;
    a.causal = causal != 0;
    a.window = window >= max_kv ? 0 : window;                   // as wide as the cache: none (and no sum overflows)
    a.scale = scale == 0.f ? 1.f / sqrtf(static_cast<float>(D)) : scale;
    a.err = device_error_word();
    a.item_cost = few ? 1 : kItemCost;
    a.whole = whole_items(B, Ttot, pv.n_kv, few ? a.tile_tokens : QT * a.tile_tokens, max_kv);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    a.part_state = reinterpret_cast<int*>(ws);
    a.part_ml = reinterpret_cast<float*>(ws + part_state_bytes());
    a.part_o = reinterpret_cast<float*>(ws + part_state_bytes() + part_ml_bytes(a.part_rows));

    AttnMaps maps;
    {
        const uint64_t ld = static_cast<uint64_t>(Ttot > 1 ? q_ld : static_cast<long>(Hq) * D) * 2;
        const uint64_t dims[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(Hq), static_cast<uint64_t>(Ttot)};
        const uint64_t strides[2] = {static_cast<uint64_t>(D) * 2, ld};
        const uint32_t box[3] = {64, static_cast<uint32_t>(a.group), static_cast<uint32_t>(a.tile_tokens)};
        if ((st = make_map_bf16(&maps.q, q, 3, dims, strides, box, true)) != GDN_OK) return st;
    }
    {
        const uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(cache->page_size),
                                  static_cast<uint64_t>(pv.n_kv), static_cast<uint64_t>(pv.num_pages)};
        const uint64_t strides[3] = {static_cast<uint64_t>(pv.token_stride) * 2, static_cast<uint64_t>(pv.head_stride) * 2,
                                     static_cast<uint64_t>(pv.page_stride) * 2};
        const uint32_t box[4] = {64, static_cast<uint32_t>(cache->page_size < kTile ? cache->page_size : kTile), 1, 1};
        if ((st = make_map_bf16(&maps.k, pv.k, 4, dims, strides, box, true)) != GDN_OK) return st;
        if ((st = make_map_bf16(&maps.v, pv.v, 4, dims, strides, box, true)) != GDN_OK) return st;
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (few) return launch_attn_rows(maps, a, D, s);
    return D == 64 ? launch<64>(maps, a, s) : launch<128>(maps, a, s);
}
