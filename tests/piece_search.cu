// Host program: the search for the item in which a piece of the attention's work line starts
// (Seq::holds), against a walk over the items.  Prints "ok <checks>" or the first difference.
#include <cstdio>
#include <random>
#include <vector>

#include "../gdn_18646_b200/csrc/paged_work.cuh"

using namespace gdn;

static long checks = 0;

static bool run(int n, int kv, int group, int causal, int window, int item_cost, bool all, std::mt19937_64& rng) {
    AttnArgs a = {};
    a.causal = causal;
    a.window = window;
    a.item_cost = item_cost;
    a.tile_tokens = 128 / group;
    const int tt = 2 * a.tile_tokens;
    Seq s = {};
    s.n = n;
    s.kv = kv;
    s.items = (n + tt - 1) / tt;
    std::vector<long long> before(s.items + 1, 0);
    for (int i = 0; i < s.items; ++i) {
        int first, count, lo, hi;
        s.tiles(a, i, tt, first, count, lo, hi);
        before[i + 1] = before[i] + count + item_cost;
    }
    const long long total = before[s.items];
    PieceScratch sh = {};
    std::vector<long long> offs = {0, total - 1, total / 2};
    for (long long x : {1ll << 31, 1ll << 32})
        for (long long d = -1; d <= 1; ++d)
            if (x + d < total) offs.push_back(x + d);
    for (int i = 0; i < 4; ++i) offs.push_back(static_cast<long long>(rng() % static_cast<unsigned long long>(total)));
    if (all)
        for (long long x = 0; x < total && x < 3000; ++x) offs.push_back(x);
    for (long long off : offs) {
        sh.off = off;                                           // as find_piece hands it on
        int found = 0;
        for (int i = 0; i < s.items; ++i) {
            int skip = -1;
            if (!s.holds(a, i, tt, sh.off, skip)) continue;
            ++found;
            if (before[i] > off || off >= before[i + 1] || skip != off - before[i]) {
                std::printf("n %d kv %d group %d causal %d window %d: unit %lld given to item %d + %d\n", n, kv, group, causal,
                            window, off, i, skip);
                return false;
            }
        }
        if (found != 1) {
            std::printf("n %d kv %d group %d causal %d window %d: unit %lld of %lld lies in %d items\n", n, kv, group, causal,
                        window, off, total, found);
            return false;
        }
        ++checks;
    }
    return true;
}

int main() {
    std::mt19937_64 rng(1);
    // a head's units past 2^31 and 2^32
    if (!run(1 << 21, 1 << 21, 64, 1, 0, 2, false, rng) || !run(1600000, 1900001, 64, 1, 0, 2, false, rng) ||
        !run(3300000, 3300000, 16, 1, 0, 2, false, rng) || !run(600000, 2000000, 40, 0, 0, 2, false, rng) ||
        !run(1 << 20, 1 << 22, 64, 1, 3000000, 2, false, rng))
        return 1;
    for (int k = 0; k < 300; ++k) {
        const int groups[] = {1, 2, 3, 5, 8, 16, 31, 64}, group = groups[rng() % 8];
        const int n = 1 + static_cast<int>(rng() % 900);
        const int kv = static_cast<int>(rng() % 2 ? n + rng() % 4000 : rng() % 900);
        const int causal = rng() % 4 != 0;
        const int window = causal && rng() % 2 ? 1 + static_cast<int>(rng() % 1500) : 0;
        if (!run(n, kv, group, causal, window, 1 + static_cast<int>(rng() % 2), true, rng)) return 1;
    }
    std::printf("ok %ld\n", checks);
    return 0;
}
