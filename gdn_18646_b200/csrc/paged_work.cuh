// paged_work.cuh -- what the paged attention kernels share: their arguments, the line of
// work (items of a sequence's new tokens and a kv head, their kv tiles) and its cut into one
// piece per CTA, the loading of kv tiles by TMA, and helpers around the MMAs.
#pragma once
#include "common.cuh"
#include "paged.cuh"

namespace gdn {

constexpr int kTile = 128;            // positions per kv tile
constexpr int kMaxCtas = 148;         // pieces of the work line: one CTA per SM of a B200
constexpr int kMaxPositions = 0x7fffffff - 511;   // of a sequence: sums with a tile's and an item's size stay ints
// Shortest piece.  Finer ones save tiles in a row where there are few items, and cost more to join where
// an item ends up in many.  With 2 / 4 / 8, us (1 token unless noted, 16 heads): over 1100 positions, 2 kv
// heads 10.1 / 12.1 / 14.7; over 8000 13.5 / 13.6 / 15.6, with 8 kv heads 15.8 / 15.1 / 17.5; over 20000
// 18.9 / 16.5 / 17.5; 100 tokens over 2000 20.9 / 23.3 / 29.9.
constexpr int kMinPiece = 4;

struct AttnArgs {
    uint16_t* out;
    float* lse;
    const int* cu;
    const int* kv_lens;
    const int* table;
    long table_ld;
    int num_pages, page_shift;
    int B, T, Hq, n_kv, group;        // group: query heads per kv head
    int tile_tokens;                  // tokens of a row tile: floor(its rows / group)
    int max_q, max_kv, causal, window;
    float scale;
    int item_cost;                    // kv tiles that an item is worth beside its tiles
    int whole;                        // a CTA per item, no cut: few items of few tiles
    unsigned int* err;
    int* part_state;                  // [ctas][8]: what a CTA left unfinished
    int part_rows;                    // rows of a part
    float* part_ml;                   // [ctas][2][part_rows][2]: m, l
    float* part_o;                    // [ctas][2][D / 4][part_rows][4], or [ctas][2][part_rows][D] (few rows)
};

struct alignas(64) AttnMaps {
    CUtensorMap q, k, v;
};

// sum over i in [0, n) of floor((a i + b) / 128) for a <= 256 (the Euclid-like reduction);
// after the first reduction every operand is small, so the divisions are 32-bit
__host__ __device__ __forceinline__ long long floor_sum(uint32_t n, uint32_t a, uint32_t b) {
    uint32_t m = kTile;
    long long s = 0;
    while (n > 0) {
        const uint32_t qa = a / m, qb = b / m;
        s += static_cast<long long>(n - 1) * n / 2 * qa + static_cast<long long>(n) * qb;
        a -= qa * m;
        b -= qb * m;
        const uint32_t y = a * n + b;                           // a < 128, n <= 2^24
        if (y < m) break;
        n = y / m;
        b = y - n * m;
        const uint32_t t = m;
        m = a;
        a = t;
    }
    return s;
}

// One lane of the warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
// lane 0's value: tells the compiler that it is the same in the whole warp, so that MMA
// descriptors built from it stay in uniform registers
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
// sdesc_sw128 from its low word
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint64_t desc_of(uint32_t lo) {
    return static_cast<uint64_t>(kDescHi) << 32 | lo;
}
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo_bytes) { return ((saddr & 0x3FFFFu) >> 4) | (lbo_bytes >> 4) << 16; }

// Waits at a barrier given by its shared-memory address, for warps whose every step counts: the
// way of a barrier that is ready has no clock and no loop.
__device__ __forceinline__ bool try_at(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
static __device__ __noinline__ bool wait_slowly(uint32_t bar, uint32_t parity, unsigned int* err, volatile int* dead) {
    const long long t0 = clock64(), budget = wait_budget();
    while (!try_at(bar, parity)) {
        if (*dead) return false;
        if (clock64() - t0 > budget) {
            if (err) atomicOr(err, DERR_TIMEOUT);
            *dead = 1;
            return false;
        }
    }
    return true;
}
// Ends with the warp together and says nothing when it gave up (the error word and *dead are
// set then, all later waits return at once, and the warp runs on to its end over garbage).
__device__ __forceinline__ void wait_at(uint32_t bar, uint32_t parity, unsigned int* err, volatile int* dead) {
    if (!try_at(bar, parity)) wait_slowly(bar, parity, err, dead);
    __syncwarp();
}
// One that all lanes of a warp leave alike; false: gave up.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, unsigned int* err, volatile int* dead) {
    const bool ok = try_at(bar, parity);
    return __all_sync(0xffffffffu, ok) || __all_sync(0xffffffffu, ok || wait_slowly(bar, parity, err, dead));
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, unsigned int* err, volatile int* dead) {
    return warp_wait(smem_u32(bar), parity, err, dead);
}

// One sequence as the kernel sees it; tt: tokens per item.
struct Seq {
    int c0, n, kv, items;             // first packed token, new tokens, positions, row-tile groups
    __device__ __forceinline__ void load(const AttnArgs& a, int b, int tt, bool report) {
        c0 = a.cu[b];
        const int c1 = a.cu[b + 1];
        kv = a.kv_lens[b];
        n = c1 - c0;
        if (c0 < 0 || c1 > a.T || n < 0 || n > a.max_q || kv < 0 || kv > a.max_kv) {
            if (report) atomicOr(a.err, DERR_PAGED);
            c0 = n = kv = 0;
        }
        items = (n + tt - 1) / tt;
    }
    // positions [lo, hi) that tokens first .. last of the chunk see between them
    __host__ __device__ __forceinline__ void range(const AttnArgs& a, int first, int last, int& lo, int& hi) const {
        const int p = kv - n;
        hi = a.causal ? max(0, min(p + last + 1, kv)) : kv;
        lo = a.window > 0 ? max(0, p + first + 1 - a.window) : 0;
        if (hi <= lo) lo = hi = 0;
    }
    __host__ __device__ __forceinline__ void tiles(const AttnArgs& a, int item, int tt, int& first, int& count, int& lo, int& hi) const {
        range(a, item * tt, min((item + 1) * tt, n) - 1, lo, hi);
        first = lo / kTile;
        count = hi > 0 ? (hi + kTile - 1) / kTile - first : 0;
    }
    // cost of the items before `q` of one kv head
    __host__ __device__ __forceinline__ long long cost(const AttnArgs& a, int q, int tt) const {
        if (q == 0) return 0;
        if (a.whole) return q;
        long long s = static_cast<long long>(q) * a.item_cost;
        if (q <= 6) {                                           // as they are: the closed form costs as much as six
            for (int i = 0; i < q; ++i) {
                int first, count, lo, hi;
                tiles(a, i, tt, first, count, lo, hi);
                s += count;
            }
            return s;
        }
        const int full = (kv + kTile - 1) / kTile;
        if (!a.causal) return s + static_cast<long long>(q) * full;
        const int p = kv - n;
        const int m = min(q, items - 1);
        const int i0 = p + tt > 0 ? 0 : (-p) / tt;              // first item with p + (i + 1) tt > 0
        if (i0 < m) s += floor_sum(m - i0, tt, p + (i0 + 1) * tt + kTile - 1);
        if (q == items) s += full;
        if (a.window > 0) {
            const int w = p + 1 - a.window;                     // lo of item i: max(0, w + i tt)
            const int i1 = w >= 0 ? 0 : (-w + tt - 1) / tt;
            if (i1 < q) s -= floor_sum(q - i1, tt, w + i1 * tt);
        }
        return s;
    }
    // Whether unit `off` of one kv head lies in its item i, and how far into it.  A head's units pass
    // 32 bits (a chunk of 2^21 tokens at 64 query heads a kv head has 2^32), an item's do not.
    __host__ __device__ __forceinline__ bool holds(const AttnArgs& a, int i, int tt, long long off, int& skip) const {
        const long long before = cost(a, i, tt);
        if (off < before || off >= cost(a, i + 1, tt)) return false;
        skip = static_cast<int>(off - before);
        return true;
    }
};

// Where a CTA's piece of the work line starts, and its length.
struct Piece {
    Seq s;
    int b, head, item;
    int skip;                         // units of the first item that belong to earlier CTAs
    long long units;
};

// Walks the items of a piece; every role of the CTA does so on its own.
struct Walk {
    Seq s;
    int b, head, item, skip;
    long long left;
    int first, count, lo, hi;         // the item's kv tiles and positions
    int t0, t1;                       // this CTA's part of its tiles: [t0, t1) of [0, count)
    __device__ __forceinline__ void start(const AttnArgs& a, const Piece& p, int tt) {
        b = p.b;
        head = p.head;
        item = p.item;
        skip = p.skip;
        left = p.units;
        if (left > 0) {
            s = p.s;
            set(a, tt);
        }
    }
    __device__ __forceinline__ bool valid() const { return left > 0; }
    __device__ __forceinline__ void set(const AttnArgs& a, int tt) {
        s.tiles(a, item, tt, first, count, lo, hi);
        if (a.whole) {
            t0 = 0;
            t1 = count;
            return;
        }
        const long long end = min(static_cast<long long>(count + a.item_cost), skip + left);
        t0 = max(skip - a.item_cost, 0);
        t1 = max(static_cast<int>(end) - a.item_cost, 0);
    }
    __device__ __forceinline__ void next(const AttnArgs& a, int tt) {
        left -= a.whole ? 1 : count + a.item_cost - skip;
        skip = 0;
        if (left <= 0) return;
        if (++item == s.items) {
            item = 0;
            if (++head == a.n_kv) {
                head = 0;
                do {
                    ++b;
                    s.load(a, b, tt, false);
                } while (s.items == 0);
            }
        }
        set(a, tt);
    }
};

// Scratch of find_piece in shared memory.
struct PieceScratch {
    Piece piece;
    long long off;                    // where the piece starts, in units of its kv head
    long long scan[16];
};

// This CTA's piece: a thread sums the costs of its share of the sequences, a scan over the
// threads finds the sequence in which the piece starts, and all threads together the item in it.
__device__ __forceinline__ void find_piece(const AttnArgs& a, PieceScratch* sh, int tt) {
    const int tid = threadIdx.x, nt = blockDim.x, warp = tid >> 5, lane = tid & 31, nw = nt >> 5;
    if (tid == 0) sh->piece.units = 0;
    const int each = (a.B + nt - 1) / nt, b0 = tid * each, b1 = min(b0 + each, a.B);
    long long mine = 0, u = 0;
    Seq s = {};
#pragma unroll 4
    for (int b = b0; b < b1; ++b) {
        s.load(a, b, tt, blockIdx.x == 0);
        u = s.cost(a, s.items, tt);
        mine += u * a.n_kv;
    }
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) sh->scan[warp] = inc;
    __syncthreads();
    long long start = inc - mine, total = 0;
    for (int w = 0; w < nw; ++w) {
        const long long v = sh->scan[w];
        if (w < warp) start += v;
        total += v;
    }
    const long long most = a.whole ? total : (total + kMinPiece - 1) / kMinPiece;
    const int pieces = most < gridDim.x ? static_cast<int>(most) : static_cast<int>(gridDim.x);
    if (static_cast<int>(blockIdx.x) < pieces) {
        // total x / pieces without a wide product; the quotient in two short divisions (total < 2^48)
        const uint32_t top = static_cast<uint32_t>(total >> 24), q1 = top / pieces;
        const uint32_t low = (top - q1 * pieces) << 24 | static_cast<uint32_t>(total & 0xffffff), q0 = low / pieces;
        const long long q = static_cast<long long>(q1) << 24 | q0;
        const int r = static_cast<int>(low - q0 * pieces), x = blockIdx.x;
        const long long from = q * x + r * x / pieces, to = q * (x + 1) + r * (x + 1) / pieces;
        if (from >= start && from < start + mine) {
            int b = b0;
            if (each > 1) {
                for (;; ++b) {
                    s.load(a, b, tt, false);
                    u = s.cost(a, s.items, tt);
                    if (from < start + u * a.n_kv) break;
                    start += u * a.n_kv;
                }
            }
            long long off = from - start;
            int head = 0;
            for (; off >= u; off -= u) ++head;
            Piece& p = sh->piece;
            p.s = s;
            p.b = b;
            p.head = head;
            p.item = 0;
            p.skip = static_cast<int>(off);                     // of a head's only item; else found below
            p.units = to - from;
            sh->off = off;
        }
    }
    __syncthreads();
    if (sh->piece.units == 0) return;
    s = sh->piece.s;
    if (s.items == 1) return;
    const long long off = sh->off;
    for (int i = tid; i < s.items; i += nt) {
        int skip;
        if (s.holds(a, i, tt, off, skip)) {
            sh->piece.item = i;
            sh->piece.skip = skip;
        }
    }
    __syncthreads();
}

// A copy of one page's rows of a kv tile, 64 values wide.
__device__ __forceinline__ void load_page(uint32_t dst, const CUtensorMap* map, uint32_t bar, int value, int in_page, int head, int page) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(value), "r"(in_page), "r"(head), "r"(page)
        : "memory");
}

// Loads the K and V tiles of the walk's item into the kv ring (warp together, a lane per page of
// the tile); only pages that hold a position somebody sees.  False: gave up.  WARPS warps share
// the copies of every tile, this one is `which`; each arrives at its barrier.  The lanes' copies
// go out one by one, so whatever they have in common is made uniform before.
template <int D, int STAGES, int WARPS>
__device__ __forceinline__ bool load_tiles(const AttnArgs& a, const AttnMaps& maps, const Walk& w, uint8_t* kv_ring,
                                           uint64_t* full, uint64_t* empty, int& stage, uint32_t& phase, uint32_t& issued,
                                           volatile int* dead, int which = 0) {
    constexpr int HALVES = D / 64, STAGE = kTile * D * 2;
    constexpr int MINE = WARPS >= HALVES ? 1 : HALVES;          // halves of a tile (64 values each) that this warp loads
    constexpr int STEP = WARPS >= HALVES ? WARPS / HALVES : 1;  // of them every STEP-th page
    const int lane = threadIdx.x & 31;
    const int page_rows = min(1 << a.page_shift, kTile);
    const int half0 = MINE == 1 && HALVES > 1 ? uniform(which % HALVES) : 0;
    const int my_page = lane * STEP + (MINE == 1 ? which / HALVES : 0);
    const int* row = a.table + w.b * a.table_ld;
    const int head = uniform(w.head);
    const uint32_t ring = smem_u32(kv_ring) + half0 * 16384, fulls = smem_u32(full), empties = smem_u32(empty);
    const uint32_t mine_at = my_page * page_rows * 128;
    // the table is read a tile ahead, so that its latency is not between the copies
    int at = uniform((w.first + w.t0) * kTile);                 // the tile's first position
    auto seen = [&]() {
        const int pos = at + my_page * page_rows;
        return my_page * page_rows < kTile && pos + page_rows > w.lo && pos < w.hi;
    };
    auto look_up = [&]() { return row[(at + my_page * page_rows) >> a.page_shift]; };
    int ahead = seen() ? look_up() : 0;
    for (int j = w.t0; j < w.t1; ++j) {
        const bool mine = seen();
        const int in_page = at & ((1 << a.page_shift) - 1);     // 0 where a tile has several pages
        int page = ahead;
        at += kTile;
        if (j + 1 < w.t1 && seen()) ahead = look_up();
        if (mine && (page < 0 || page >= a.num_pages)) {
            page = a.num_pages;                                 // outside: the copy fills zeros
            atomicOr(a.err, DERR_PAGED);
        }
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, mine)) * page_rows * MINE * 128;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            const uint32_t st = uniform(stage), bar = fulls + st * 8, dst = ring + st * STAGE + mine_at;
            if (!warp_wait(empties + st * 8, phase ^ 1u, a.err, dead)) return false;
            if (lane == 0)
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
            __syncwarp();
#pragma unroll
            for (int h = 0; h < MINE; ++h)
                if (mine) load_page(dst + h * 16384, kv ? &maps.v : &maps.k, bar, (half0 + h) * 64, in_page, head, page);
            ++issued;
            if (++stage == STAGES) {
                stage = 0;
                phase ^= 1u;
            }
        }
    }
    return true;
}

// Zeroes the value rows of a tile that no row of the item sees (warp together): a weight of 0
// times what the cache holds there (NaN included) has to be 0.
template <int D>
__device__ __forceinline__ void clear_rows(const Walk& w, int j, uint8_t* v) {
    const int j0 = (w.first + j) * kTile;
    if (j0 >= w.lo && j0 + kTile <= w.hi) return;
    const int below = max(0, w.lo - j0), above = min(kTile, w.hi - j0);
    for (int c = threadIdx.x & 31; c < kTile * 8 * (D / 64); c += 32) {
        const int r = (c >> 3) & (kTile - 1);
        if (r < below || r >= above) *reinterpret_cast<uint4*>(v + c * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_async_smem();
    __syncwarp();
}

// After a CTA gave up: waits (bounded) until its copies in flight have landed.
__device__ __forceinline__ void drain_ring(const AttnArgs& a, uint64_t* full, uint32_t stages, uint32_t issued) {
    for (uint32_t i = issued > stages ? issued - stages : 0; i < issued; ++i)
        mbar_wait(&full[i % stages], (i / stages) & 1u, a.err);
}

inline size_t part_state_bytes() { return static_cast<size_t>(kMaxCtas) * 8 * sizeof(int); }
inline size_t part_ml_bytes(int rows) { return static_cast<size_t>(kMaxCtas) * 2 * rows * 2 * sizeof(float); }
inline size_t part_o_bytes(int rows, int D) { return static_cast<size_t>(kMaxCtas) * 2 * rows * D * sizeof(float); }

// paged_attn_rows.cu: at most 64 rows per item (a decode step, a few drafted tokens)
int launch_attn_rows(const AttnMaps& maps, const AttnArgs& a, int D, cudaStream_t st);

}  // namespace gdn
