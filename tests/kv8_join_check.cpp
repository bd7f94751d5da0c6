// Host build of quantr-in-c_b200/csrc/kv8_join.cuh: CTAs that share row tiles
// count themselves in, in random orders, as the kernel does.  Built and run by
// tests/test_kv8_join.py.  Prints "wrong N of M": schedules in which a row tile
// was joined early, twice or never, or a counter was left non-zero.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "kv8_join.cuh"

namespace {

struct Tile {
    int c0, c1;
    std::vector<char> have;  // by CTA - c0: its part (or its group's result) is there
    int joined = 0;
};

// The row tiles of a flat list of tiles cut into runs of `share`; nt: tiles of
// each row tile.
std::vector<Tile> spans(const std::vector<int>& nt, int ctas)
{
    long long total = 0;
    for (int n : nt) total += n;
    const long long share = (total + ctas - 1) / ctas;
    std::vector<Tile> t;
    long long at = 0;
    for (int n : nt) {
        Tile x;
        x.c0 = (int)(at / share), x.c1 = (int)((at + n - 1) / share);
        x.have.assign(x.c1 - x.c0 + 1, 0);
        t.push_back(x);
        at += n;
    }
    return t;
}

bool play(std::vector<Tile> tiles, int ctas, std::mt19937& rng, bool ordered)
{
    std::vector<int> counters(2 * qr::kJoinCtas, 0);
    struct Todo {
        std::vector<int> tiles;
        size_t at = 0;
        int step = -1;
    };
    std::vector<Todo> todo(ctas);
    for (size_t i = 0; i < tiles.size(); ++i)
        for (int c = tiles[i].c0; c <= tiles[i].c1 && tiles[i].c0 < tiles[i].c1; ++c) todo[c].tiles.push_back((int)i);
    std::vector<int> live;
    for (int c = 0; c < ctas; ++c)
        if (!todo[c].tiles.empty()) live.push_back(c);
    bool right = true;
    while (!live.empty()) {
        const size_t pick = ordered ? 0 : rng() % live.size();
        const int me = live[pick];
        Todo& d = todo[me];
        Tile& t = tiles[d.tiles[d.at]];
        if (d.step < 0) {
            if (d.at == 0)  // all of a CTA's parts are written before it counts
                for (int i : d.tiles) tiles[i].have[me - tiles[i].c0] = 1;
            d.step = qr::join_first(t.c0, t.c1, me);
        }
        const qr::JoinStep s = qr::join_step(d.step, t.c0, t.c1, me);
        const bool last = counters[s.counter]++ == s.n - 1;
        if (last) {
            counters[s.counter] = 0;
            if (d.step == 0) {
                const int g0 = qr::join_group(t.c0, me);
                for (int i = 0; i < s.n; ++i) right &= t.have[g0 - t.c0 + i] == 1;
                for (int i = 0; i < s.n; ++i) t.have[g0 - t.c0 + i] = 2;
            } else {
                const bool g = qr::join_grouped(t.c0, t.c1);
                for (int c = t.c0; c <= t.c1; ++c) {
                    const int g0 = qr::join_group(t.c0, c), end = g0 + qr::kJoinGroup - 1;
                    const bool alone = g0 == (t.c1 < end ? t.c1 : end);
                    right &= t.have[c - t.c0] == 2 || (!(g && !alone) && t.have[c - t.c0] == 1);
                }
                ++t.joined;
            }
        }
        if (last && d.step == 0) {
            d.step = 1;
        } else {
            d.step = -1;
            if (++d.at == d.tiles.size()) live.erase(live.begin() + pick);
        }
    }
    for (const Tile& t : tiles) right &= t.joined == (t.c0 < t.c1 ? 1 : 0);
    for (int c : counters) right &= c == 0;
    return right;
}

} // namespace

int main()
{
    std::mt19937 rng(1);
    long long wrong = 0, all = 0;
    auto look = [&](const std::vector<int>& nt, int ctas) {
        const std::vector<Tile> t = spans(nt, ctas);
        for (int i = 0; i < 12; ++i, ++all) wrong += !play(t, ctas, rng, i == 0);
    };
    auto each = [](int heads, const std::vector<int>& lens) {  // 128-token tiles of every head
        std::vector<int> nt;
        for (int n : lens)
            for (int h = 0; h < heads; ++h) nt.push_back((n + 127) / 128);
        return nt;
    };
    // One long context among short ones; two long ones; chance.
    std::vector<int> a(22, 2000), b(30, 2000), c(6, 2000);
    a[0] = 100000, b[0] = 131072, c[0] = 100000;
    look(each(4, a), 296), look(each(4, b), 296), look(each(8, c), 296);
    look(each(4, {65600, 1000}), 296), look(each(4, {131072, 64000}), 296);
    for (int i = 0; i < 3000; ++i) {
        const int ctas = i % 2 ? 296 : 148, heads = 1 << rng() % 4;
        std::vector<int> lens{(int)(20000 + rng() % 200000)};
        for (int k = rng() % 12; k > 0; --k) lens.push_back(1 + rng() % (rng() % 2 ? 4000 : 100000));
        look(each(heads, lens), ctas);
    }
    std::printf("wrong %lld of %lld\n", wrong, all);
    return wrong != 0;
}
