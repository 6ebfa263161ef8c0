// What kernels over an 8-bit paged cache make of the numbers that device memory holds (kv8_units.h), on the CPU: every number is checked against the arrays it indexes.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>

#include "../../crane_b200/csrc/kv8_units.h"

using namespace cb;
#define CHECK(c) do { if (!(c)) { std::fprintf(stderr, "%s:%d: %s\n", __FILE__, __LINE__, #c); std::exit(1); } } while (0)

struct Case { std::vector<int> table, lens, starts; Kv8Seqs s; Kv8Pool p; };

static Case make(std::mt19937& g, bool wild) {
    auto in = [&](int lo, int hi) { return (int)(lo + g() % (unsigned)(hi - lo + 1)); };
    Case c;
    const int seqs = in(1, 40), width = in(1, 9), pages = in(1, 60), page = 16 << in(0, 3), kv = in(1, 4);
    const int wildest[] = {-2147483647 - 1, -1, 2147483647, 1 << 30, 7};
    auto rare = [&](int v) { return wild && g() % 4 == 0 ? wildest[g() % 5] : v; };
    int at = wild ? in(0, 2) : 0;
    for (int b = 0; b < seqs; ++b) {
        const int n = g() % 3 ? in(0, 3) : in(0, 3 * page);
        c.starts.push_back(rare(at));
        c.lens.push_back(rare(wild ? in(0, width * page + 40) : in(n, n + 5 * page)));
        at += n;
        for (int i = 0; i < width + 2; ++i) c.table.push_back(rare(in(-1, pages)));
    }
    c.starts.push_back(rare(at));
    c.s = Kv8Seqs{c.table.data(), width + 2, width, c.lens.data(), c.starts.data(), seqs, at};
    c.p = Kv8Pool{nullptr, nullptr, nullptr, pages, kv, page, 64};
    return c;
}

static void pieces(const Case& c, bool wild) {
    const Kv8Seqs& s = c.s;
    const int P = c.p.page;
    for (int by_row = 0; by_row < 2; ++by_row) {
        std::map<std::pair<int, int>, int> seen;                   // (sequence, position) -> row
        const int slots = by_row ? s.rows : s.rows / P + 2 * s.seqs;
        for (int at = 0; at < slots; ++at) {
            int b = 0;                                             // the largest whose key is at most `at` (the kernel's search gives some sequence where starts do not ascend)
            for (int i = 0; i < s.seqs; ++i) if (kv8_piece_key(s, P, i, by_row) <= at) b = i;
            for (int t = 0; t < (wild ? s.seqs : 1); ++t, b = (b + 1) % s.seqs) {
                const Kv8Seq q = kv8_seq(s, b);
                CHECK(q.s0 >= 0 && q.n >= 0 && q.s0 + q.n <= s.rows && q.len >= 0);
                const Kv8Piece k = kv8_piece(s, q, P, b, at, by_row);
                if (!k.count) continue;
                CHECK(k.count > 0 && k.pos >= 0 && k.pos / P == k.block && (k.pos + k.count - 1) / P == k.block && k.pos + k.count <= q.len);
                const int row = q.s0 + (k.pos - q.first);
                CHECK(row >= q.s0 && row + k.count <= q.s0 + q.n);
                const int page = kv8_page(s, c.p, b, k.block);
                CHECK(page >= -1 && page < c.p.pages);
                if (!wild) for (int i = 0; i < k.count; ++i) CHECK(seen.emplace(std::make_pair(b, k.pos + i), row + i).second);
            }
        }
        if (wild) continue;
        size_t rows = 0;
        for (int b = 0; b < s.seqs; ++b) {
            const Kv8Seq q = kv8_seq(s, b);
            for (int i = 0; i < q.n; ++i)
                if (q.first + i >= 0) { ++rows; CHECK(seen.at({b, q.first + i}) == q.s0 + i); }
        }
        CHECK(rows == seen.size());                                // every row once, in its place
    }
}

template <int M, int TILE, int OWN>
static void units(const Case& c, int group, int ctas, long long lo, long long hi) {
    using U = Kv8Units<M, TILE, OWN>;
    const Kv8Deal d = {c.s, c.p, group, lo, hi};
    long long total = 0;
    for (int b = 0; b < c.s.seqs; ++b) {
        U u; u.b = b; u.shape(d);
        CHECK(u.groups >= 0 && (long long)u.groups * M < (long long)u.q.n * group + M);
        CHECK(!u.groups == (u.q.n == 0 || (long long)u.q.n * group < lo || (long long)u.q.n * group > hi));
        total += u.head_steps(d) * c.p.kv_heads;
    }
    if (total > 2000000) return;
    std::map<std::tuple<int, int, int>, std::vector<std::pair<int, std::pair<int, int>>>> parts;      // unit -> (slot, tiles), in order; slot -1: whole
    std::map<std::tuple<int, int, int>, int> tiles;
    long long next = 0;
    std::set<int> slots;
    for (int k = 0; k < ctas; ++k) {
        const long long begin = kv8_range(total, ctas, k), end = kv8_range(total, ctas, k + 1);
        CHECK(begin == next && end >= begin && end <= total && end - begin <= total / ctas + 1);
        next = end;
        if (begin == end) continue;
        CHECK(kv8_owner(total, ctas, begin) == k && kv8_owner(total, ctas, end - 1) == k);
        U u;
        u.seek(d, 0, 0, begin);
        for (long long step = begin; step < end;) {
            CHECK(u.first <= step && step < u.first + u.size() && u.head >= 0 && u.head < c.p.kv_heads && u.grp >= 0 && u.grp < u.groups && u.b < c.s.seqs);
            CHECK(u.tiles >= 1 && (long long)(u.tiles - 1) * TILE < (long long)c.s.width * c.p.page);
            const long long row = least((long long)u.q.n * group, (u.grp + 1LL) * M) - 1;            // the group's last row and what it sees
            const long long seen = least((long long)u.q.first + row / group + 1, (long long)c.s.width * c.p.page);
            CHECK((long long)u.tiles * TILE >= seen && ((long long)(u.tiles - 1) * TILE < seen || u.tiles == 1));
            const int t0 = u.tile_at(step), t1 = u.tile_at(u.stop(end));
            const bool whole = u.whole(step, end);
            CHECK(t0 <= t1 && t1 <= u.tiles && u.size() == u.tiles + OWN && (!whole || (t0 == 0 && t1 == u.tiles)));
            const int slot = whole ? -1 : kv8_slot(k, begin, step);
            if (!whole) CHECK(slot < 2 * ctas && slots.insert(slot).second);
            parts[{u.b, u.head, u.grp}].push_back({slot, {t0, t1}});
            tiles[{u.b, u.head, u.grp}] = u.tiles;
            step = u.stop(end);
            if (step < end) CHECK(u.next(d));
        }
    }
    CHECK(next == total);
    // what joins them: the unit that a CTA began and did not end
    std::set<std::tuple<int, int, int>> joined;
    for (int k = 0; k < ctas; ++k) {
        const long long begin = kv8_range(total, ctas, k), end = kv8_range(total, ctas, k + 1);
        if (begin == end) continue;
        U u;
        u.seek(d, 0, 0, begin);
        int here = 0;
        for (long long step = begin; step < end;) {
            if (u.begins(step, end)) {
                const Kv8Join j = kv8_join(d, u, M, total, ctas, k, begin);
                CHECK(!here++ && j.rows >= 1 && j.rows <= M && j.last > k && j.last < ctas);
                const auto& p = parts.at({u.b, u.head, u.grp});
                CHECK((int)p.size() == j.last - k + 1);
                for (int i = k; i <= j.last; ++i) CHECK(p[i - k].first == (i == k ? j.slot : kv8_slot(i, 0, 0)));
                CHECK(joined.insert({u.b, u.head, u.grp}).second);
            }
            step = u.stop(end);
            if (step < end) CHECK(u.next(d));
        }
    }
    for (const auto& e : parts) {
        int at = 0;
        for (const auto& p : e.second) { CHECK(p.second.first == at); at = p.second.second; }
        CHECK(at == tiles.at(e.first));
        CHECK((e.second.size() > 1) == (joined.count(e.first) == 1));
        if (e.second.size() == 1) CHECK(e.second[0].first == -1);
    }
    size_t want = 0;
    for (int b = 0; b < c.s.seqs; ++b) { U u; u.b = b; u.shape(d); want += (size_t)u.groups * c.p.kv_heads; }
    CHECK(parts.size() == want);                                    // every unit once
}

int main() {
    std::mt19937 g(7);
    for (int i = 0; i < 600; ++i) {
        const Case tame = make(g, false), wild = make(g, true);
        pieces(tame, false);
        pieces(wild, true);
        for (int ctas : {1, 3, 148, 296}) {
            const int group = 1 + i % 7;
            units<16, 64, 4>(tame, group, ctas, 0, 1LL << 62);
            units<16, 64, 4>(tame, group, ctas, 0, 64);
            units<32, 32, 4>(wild, group, ctas, 0, 1LL << 62);
            units<256, 128, 4>(tame, group, ctas, 65, 1LL << 62);
            units<256, 128, 4>(wild, group, ctas, 65, 1LL << 62);
        }
    }
    std::puts("ok");
}
