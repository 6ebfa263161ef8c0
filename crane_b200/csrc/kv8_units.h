// How the work over an 8-bit paged cache (kv8.cuh) is found in what device memory says, and dealt out.  Host and device code: tests run it on the CPU.
#pragma once

#ifdef __CUDACC__
#define CB_HD __host__ __device__ __forceinline__
#else
#define CB_HD inline
#endif

namespace cb {

struct Kv8Pool { unsigned char* k; unsigned char* v; float* scales; int pages, kv_heads, page, dim; };
// Sequence b holds lens[b] positions, position i on page table[b * ldt + i / page]; its new rows are rows starts[b] .. starts[b + 1] - 1, at its last positions.
// Everything here is device memory that the host does not look at: kernels clamp starts to the rows there are and leave out pages and positions that do not exist.
struct Kv8Seqs { const int* table; long long ldt; int width; const int* lens; const int* starts; int seqs, rows; };

template <typename T> CB_HD T least(T a, T b) { return b < a ? b : a; }
template <typename T> CB_HD T most(T a, T b) { return a < b ? b : a; }

// a / b for numbers that are not negative, by 32 bits where they do (64-bit division is a hundred instructions one behind the other)
CB_HD long long quotient(long long a, long long b) {
    if (((a | b) >> 32) == 0) return (long long)((unsigned)a / (unsigned)b);
    return a / b;
}

// What a sequence brings
struct Kv8Seq { int s0, n, len, first; };                           // first: position of row s0 (negative: rows ahead of position 0 are not in the cache)
CB_HD int kv8_start(const Kv8Seqs& s, int b) { return least(most(s.starts[b], 0), s.rows); }
CB_HD Kv8Seq kv8_seq(const Kv8Seqs& s, int b) {
    Kv8Seq q;
    q.s0 = kv8_start(s, b);
    q.n = most(kv8_start(s, b + 1), q.s0) - q.s0;
    q.len = least(most(s.lens[b], 0), 1 << 30);
    q.first = q.len - q.n;
    return q;
}
CB_HD int kv8_page(const Kv8Seqs& s, const Kv8Pool& p, int b, int block) {      // -1: none
    if (block < 0 || block >= s.width) return -1;
    const int page = s.table[b * s.ldt + block];
    return (unsigned)page < (unsigned)p.pages ? page : -1;
}

// ---- rows into pages: the pieces of a sequence's new rows that lie on one page each ------------------------------------------------
// Piece number `at` is either a row, the first of its page's (by_row), or a number that sequence b has kv8_piece_key(b) and on: n rows touch at most n / page + 2 pages.
CB_HD int kv8_piece_key(const Kv8Seqs& s, int page, int b, bool by_row) { const int r = kv8_start(s, b); return by_row ? r : r / page + 2 * b; }
struct Kv8Piece { int block, pos, count; };                        // block of the sequence's table, first position, positions (none: 0)
CB_HD Kv8Piece kv8_piece(const Kv8Seqs& s, const Kv8Seq& q, int page, int b, int at, bool by_row) {
    const int begin = most(q.first, 0);
    int block;
    if (by_row) {
        const int pos = q.first + (at - q.s0);
        if (at < q.s0 || at >= q.s0 + q.n || pos < 0 || (pos != begin && pos % page)) return {0, 0, 0};
        block = pos / page;
    } else {
        block = begin / page + (at - kv8_piece_key(s, page, b, false));
    }
    if (block < 0 || (long long)block * page >= q.len) return {0, 0, 0};
    const int pos = most(begin, block * page);
    return {block, pos, most((int)least((long long)q.len, (long long)block * page + page) - pos, 0)};
}

// ---- attention: how the steps are dealt out ----------------------------------------------------------------------------------------
// A unit is a sequence, a kv head and a group of M rows of its queries (row = token * group + head of the group); its steps are the tiles of TILE positions that the group's last
// row sees, one at least, behind OWN more that stand for what a unit costs by itself.  All steps, unit after unit, are dealt out evenly to the CTAs, whatever the lengths: a unit may lie with several CTAs, which then leave their parts of
// the sums to be joined.  A kernel takes the sequences that bring from `lo` to `hi` rows.
struct Kv8Deal { Kv8Seqs s; Kv8Pool p; int group; long long lo, hi; };
template <int M, int TILE, int OWN>
struct Kv8Units {
    int b, head, grp;                          // the unit
    Kv8Seq q;
    int tiles, groups;                         // its tiles, the sequence's groups
    long long first;                           // number of its first step
    CB_HD void shape(const Kv8Deal& d) {
        q = kv8_seq(d.s, b);
        const long long rows = (long long)q.n * d.group;
        groups = rows < d.lo || rows > d.hi ? 0 : (int)quotient(rows + M - 1, M);
    }
    CB_HD int tiles_of(const Kv8Deal& d, int g) const {
        const long long last = least((long long)q.n, quotient(((long long)g + 1) * M - 1, d.group) + 1);      // tokens up to the group's last
        const long long seen = least(q.first + last, (long long)d.s.width * d.p.page);
        return most(1, (int)(seen + TILE - 1) / TILE);
    }
    CB_HD long long head_steps(const Kv8Deal& d) const {
        long long n = 0;
        for (int g = 0; g < groups; ++g) n += tiles_of(d, g) + OWN;
        return n;
    }
    CB_HD int size() const { return tiles + OWN; }
    CB_HD long long stop(long long end) const { return least(first + size(), end); }       // where the part of a CTA whose steps run up to `end` ends
    CB_HD int tile_at(long long step) const { return most(0, (int)(step - first) - OWN); }       // tiles ahead of a step
    CB_HD bool whole(long long step, long long end) const { return step == first && stop(end) == first + size(); }
    CB_HD bool begins(long long step, long long end) const { return step == first && stop(end) < first + size(); }      // ... and goes on with the next CTA
    CB_HD bool next(const Kv8Deal& d) {        // false: behind the last
        first += size();
        if (++grp >= groups) {
            grp = 0;
            if (++head >= d.p.kv_heads) {
                head = 0;
                do {
                    if (++b >= d.s.seqs) return false;
                    shape(d);
                } while (!groups);
            }
        }
        tiles = tiles_of(d, grp);
        return true;
    }
    // The unit that holds a step; sequences are counted off from `from` on, which begins with step `at`
    CB_HD void seek(const Kv8Deal& d, int from, long long at, long long step) {
        long long each;
        for (b = from;; ++b) {
            shape(d);
            each = head_steps(d);
            if (step < at + each * d.p.kv_heads || b + 1 >= d.s.seqs) break;
            at += each * d.p.kv_heads;
        }
        head = (int)quotient(step - at, most(each, 1LL));
        first = at + head * each;
        for (grp = 0; tiles = tiles_of(d, grp), first + size() <= step && grp + 1 < groups; ++grp) first += size();
    }
};
CB_HD long long kv8_range(long long total, int ctas, int c) { const long long base = quotient(total, ctas); return base * c + least((long long)c, total - base * ctas); }       // a CTA's first step
CB_HD int kv8_owner(long long total, int ctas, long long step) {
    const long long base = quotient(total, ctas), rem = total - base * ctas, big = rem * (base + 1);
    return (int)(step < big ? quotient(step, base + 1) : rem + quotient(step - big, most(base, 1LL)));
}
// Where a CTA leaves its part of a unit that it shares: 0 for the one that its range begins with, 1 for the one that it ends with
CB_HD int kv8_slot(int cta, long long begin, long long part) { return 2 * cta + (part == begin ? 0 : 1); }

// A unit that a CTA begins and does not end: what is needed to add up its parts, which lie with this CTA and those up to `last` (none: rows = 0)
struct Kv8Join { int s0, head, grp, rows, last, slot, pad[2]; };
template <typename U>
CB_HD Kv8Join kv8_join(const Kv8Deal& d, const U& u, int m, long long total, int ctas, int c, long long begin) {
    return Kv8Join{u.q.s0, u.head, u.grp, (int)least((long long)m, (long long)u.q.n * d.group - (long long)u.grp * m), kv8_owner(total, ctas, u.first + u.size() - 1), kv8_slot(c, begin, u.first), {0, 0}};
}

}  // namespace cb
