// paged_book.cpp -- which pages belong to whom, and how a batch's attention is cut into work (paged_book.h).
#include "paged_book.h"

#include <algorithm>
#include <climits>
#include <iterator>

#include "../../include/mechta_kv.h"

namespace mkv {
namespace paged {

void Book::init(int pages_, int page_, int seqs_, int ctx_) {
    pages = free = pages_;
    page = page_;
    seqs = seqs_;
    ctx = ctx_;
    owners.assign(pages, 0);
    open.assign(((size_t)pages + 63) / 64, ~0ull);
    if (pages % 64) open.back() = (1ull << (pages % 64)) - 1;
    low = 0;
    table.assign(seqs, {});
    len.assign(seqs, 0);
    fresh.assign(seqs, 0);
    shift.assign(seqs, 0);
    floor.assign(seqs, 0);
    moved.assign(seqs, 0);
}

int Book::take() {  // the free page of the lowest number; one is free
    while (!open[low]) low++;
    const int p = (int)(low * 64 + __builtin_ctzll(open[low]));
    open[low] &= open[low] - 1;
    free--;
    owners[p] = 1;
    return p;
}

void Book::drop(int p) {
    if (--owners[p]) return;
    open[p / 64] |= 1ull << (p % 64);
    low = std::min(low, (size_t)p / 64);
    free++;
}

int Book::distinct(const char* who, int n, const int* seq) const {
    if (n < 0) return fail(MKV_E_ARG, "%s: %d sequences", who, n);
    if (n && !seq) return fail(MKV_E_ARG, "%s: NULL argument", who);
    std::vector<bool> seen(seqs, false);
    for (int i = 0; i < n; i++) {
        if (seq[i] < 0 || seq[i] >= seqs) return fail(MKV_E_ARG, "%s: sequence %d outside [0, %d)", who, seq[i], seqs);
        if (seen[seq[i]]) return fail(MKV_E_ARG, "%s: sequence %d twice", who, seq[i]);
        seen[seq[i]] = true;
    }
    return MKV_OK;
}

int Book::reserve(const char* who, int n, const int* seq, const int* count) {
    if (int rc = distinct(who, n, seq)) return rc;
    if (n && !count) return fail(MKV_E_ARG, "%s: NULL argument", who);
    long long want = 0;
    for (int i = 0; i < n; i++) {
        if (count[i] < 0) return fail(MKV_E_ARG, "%s: %d positions for sequence %d", who, count[i], seq[i]);
        if (count[i] > ctx - len[seq[i]])
            return fail(MKV_E_POS, "%s: sequence %d of %d positions plus %d: more than the context %d", who, seq[i],
                        len[seq[i]], count[i], ctx);
        if (count[i] > INT_MAX - len[seq[i]] - shift[seq[i]])
            return fail(MKV_E_POS, "%s: sequence %d at position %lld plus %d: past 32 bits", who, seq[i],
                        (long long)len[seq[i]] + shift[seq[i]], count[i]);
        want += need(len[seq[i]] + count[i]) - (int)table[seq[i]].size();
    }
    if (want > free) return fail(MKV_E_NOMEM, "%s: %lld pages needed, %d free", who, want, free);
    for (int i = 0; i < n; i++) {  // nothing throws behind this
        std::vector<int>& t = table[seq[i]];
        const size_t m = need(len[seq[i]] + count[i]);
        if (m > t.capacity()) t.reserve(std::max(m, 2 * t.capacity()));
    }
    for (int i = 0; i < n; i++) {
        std::vector<int>& t = table[seq[i]];
        len[seq[i]] += count[i];
        stale(seq[i], (int)t.size());
        while ((int)t.size() < need(len[seq[i]])) t.push_back(take());
    }
    return MKV_OK;
}

int Book::fork(const char* who, int n, const int* src, const int* dst, const int* upto, bool own,
               std::vector<Pair>& copies) {
    if (int rc = distinct(who, n, dst)) return rc;
    if (n && !src) return fail(MKV_E_ARG, "%s: NULL argument", who);
    std::vector<bool> is_dst(seqs, false);
    for (int i = 0; i < n; i++) is_dst[dst[i]] = true;
    long long want = 0;
    for (int i = 0; i < n; i++) {
        if (src[i] < 0 || src[i] >= seqs) return fail(MKV_E_ARG, "%s: sequence %d outside [0, %d)", who, src[i], seqs);
        if (is_dst[src[i]]) return fail(MKV_E_ARG, "%s: sequence %d is both source and destination", who, src[i]);
        if (!table[dst[i]].empty()) return fail(MKV_E_ARG, "%s: destination %d is not empty", who, dst[i]);
        const int m = upto ? upto[i] : len[src[i]];
        if (m < 0 || m > len[src[i]])
            return fail(MKV_E_POS, "%s: %d positions of sequence %d, which has %d", who, m, src[i], len[src[i]]);
        if (m && m < floor[src[i]])
            return fail(MKV_E_POS, "%s: %d positions of sequence %d, of which eviction has left %d", who, m, src[i], floor[src[i]]);
        want += own ? need(m) : m % page ? 1 : 0;
    }
    if (want > free) return fail(MKV_E_NOMEM, "%s: %lld pages needed, %d free", who, want, free);
    copies.reserve(want);  // nothing throws behind these
    for (int i = 0; i < n; i++) table[dst[i]].reserve(need(upto ? upto[i] : len[src[i]]));
    for (int i = 0; i < n; i++) {
        const int m = upto ? upto[i] : len[src[i]], full = own ? 0 : m / page;
        const std::vector<int>& from = table[src[i]];
        std::vector<int>& t = table[dst[i]];
        t.assign(from.begin(), from.begin() + full);
        for (int p : t) owners[p]++;
        for (int k = full; k < need(m); k++) {
            t.push_back(take());
            copies.push_back({from[k], t[k]});
        }
        len[dst[i]] = m;
        stale(dst[i], 0);
        if (m) move(dst[i], shift[src[i]], floor[src[i]]);
    }
    return MKV_OK;
}

void Book::undo_reserve(int n, const int* seq, const int* count) {
    for (int i = 0; i < n; i++) {  // (the new pages belong to these sequences alone)
        std::vector<int>& t = table[seq[i]];
        len[seq[i]] -= count[i];
        while ((int)t.size() > need(len[seq[i]])) {
            drop(t.back());
            t.pop_back();
        }
        stale(seq[i], (int)t.size());
    }
}

void Book::clear(int n, const int* seq) {
    for (int i = 0; i < n; i++) {
        for (int p : table[seq[i]]) drop(p);
        table[seq[i]].clear();
        len[seq[i]] = 0;
        fresh[seq[i]] = 0;
        move(seq[i], 0, 0);
    }
}

int Book::release(const char* who, int n, const int* seq, const std::function<int()>& before) {
    if (int rc = distinct(who, n, seq)) return rc;
    if (before)
        if (int rc = before()) return rc;
    clear(n, seq);
    return MKV_OK;
}

int Book::set_len(const char* who, int seq, int n, std::vector<Pair>& copies, Cut* cut) {
    if (int rc = distinct(who, 1, &seq)) return rc;
    if (n < 0 || n > len[seq])
        return fail(MKV_E_POS, "%s: length %d of sequence %d, which has %d", who, n, seq, len[seq]);
    if (n && n < floor[seq])
        return fail(MKV_E_POS, "%s: length %d of sequence %d, of which eviction has left %d", who, n, seq, floor[seq]);
    std::vector<int>& t = table[seq];
    const int keep = need(n);
    const bool shared = n % page && owners[t[keep - 1]] > 1;
    if (shared) {
        bool given = false;  // the pages given back may serve as the copy
        for (int k = keep; k < (int)t.size(); k++) given |= owners[t[k]] == 1;
        if (!free && !given) return fail(MKV_E_NOMEM, "%s: no free page for a copy of a shared one", who);
    }
    if (shared) copies.reserve(1);
    if (cut) {
        const int from = shared ? keep - 1 : keep;
        *cut = Cut{len[seq], from, shared, std::vector<int>(t.begin() + from, t.end()), shift[seq], floor[seq]};
    }
    while ((int)t.size() > keep) {  // nothing throws from here on
        drop(t.back());
        t.pop_back();
    }
    if (shared) {
        const int was = t.back();
        t.back() = take();
        copies.push_back({was, t.back()});
        owners[was]--;
        stale(seq, keep - 1);
    }
    stale(seq, keep);
    len[seq] = n;
    if (!n) move(seq, 0, 0);
    return MKV_OK;
}

void Book::undo_set_len(int seq, const Cut& cut) {
    std::vector<int>& t = table[seq];
    if (cut.copied) {
        drop(t.back());
        t.pop_back();
    }
    for (int p : cut.pages) {  // the table has room for what it had
        own_again(p);
        t.push_back(p);
    }
    len[seq] = cut.len;
    stale(seq, cut.from);
    move(seq, cut.shift, cut.floor);
}

void Book::own_again(int p) {  // a page that has been given back, or that others own
    if (owners[p]++) return;
    open[p / 64] &= ~(1ull << (p % 64));
    free--;
}

int Book::can_evict(const char* who, int n, const int* seq, const int* keep) const {
    if (int rc = distinct(who, n, seq)) return rc;
    if (n && !keep) return fail(MKV_E_ARG, "%s: NULL argument", who);
    long long want = 0;
    for (int i = 0; i < n; i++) {
        if (keep[i] < 1) return fail(MKV_E_ARG, "%s: %d positions kept of sequence %d", who, keep[i], seq[i]);
        if (len[seq[i]] > keep[i]) want += need(keep[i]);
    }
    return want > free ? fail(MKV_E_NOMEM, "%s: %lld pages needed, %d free", who, want, free) : (int)MKV_OK;
}

int Book::evict(const char* who, int n, const int* seq, const int* keep, std::vector<Evicted>& cut) {
    if (int rc = can_evict(who, n, seq, keep)) return rc;
    std::vector<std::vector<int>> fresh_pages(n);  // nothing throws behind these
    cut.reserve(n);
    for (int i = 0; i < n; i++)
        if (len[seq[i]] > keep[i]) fresh_pages[i].reserve(need(keep[i]));
    for (int i = 0; i < n; i++) {
        const int s = seq[i];
        if (len[s] <= keep[i]) continue;
        for (int k = 0; k < need(keep[i]); k++) fresh_pages[i].push_back(take());
        cut.push_back({s, len[s], shift[s], floor[s], {}});
        cut.back().pages.swap(table[s]);
        table[s].swap(fresh_pages[i]);
        fresh[s] = 0;
        move(s, shift[s] + len[s] - keep[i], keep[i]);
        len[s] = keep[i];
    }
    for (const Evicted& e : cut)  // only now: what is taken is never what is given back
        for (int p : e.pages) drop(p);
    return MKV_OK;
}

void Book::undo_evict(std::vector<Evicted>& cut) {
    for (Evicted& e : cut)
        for (int p : e.pages) own_again(p);
    for (Evicted& e : cut) {
        for (int p : table[e.seq]) drop(p);
        table[e.seq].swap(e.pages);
        fresh[e.seq] = 0;
        move(e.seq, e.shift, e.floor);
        len[e.seq] = e.len;
    }
}

int Book::compact(std::vector<Pair>& copies) {
    const int used = pages - free;
    std::vector<int> to(pages);
    copies.reserve(std::min(used, free));  // nothing throws behind these
    int hole = 0;
    for (int p = 0; p < pages; p++) to[p] = p;
    for (int p = used; p < pages; p++) {
        if (!owners[p]) continue;
        while (owners[hole]) hole++;  // there are as many holes below `used` as pages in use behind it
        to[p] = hole;
        owners[hole] = owners[p];
        owners[p] = 0;
        copies.push_back({p, hole});
    }
    for (int s = 0; s < seqs; s++)
        for (int k = 0; k < (int)table[s].size(); k++)
            if (to[table[s][k]] != table[s][k]) {
                stale(s, k);
                table[s][k] = to[table[s][k]];
            }
    reopen();
    return (int)copies.size();
}

void Book::undo_compact(const std::vector<Pair>& copies) {
    for (const Pair& c : copies) {
        owners[c.src] = owners[c.dst];
        owners[c.dst] = 0;
    }
    for (int s = 0; s < seqs; s++)
        for (int k = 0; k < (int)table[s].size(); k++) {  // the holes are in order
            const auto c = std::lower_bound(copies.begin(), copies.end(), table[s][k],
                                            [](const Pair& a, int page) { return a.dst < page; });
            if (c == copies.end() || c->dst != table[s][k]) continue;
            stale(s, k);
            table[s][k] = c->src;
        }
    reopen();
}

void Book::reopen() {  // the free pages, by their owners
    std::fill(open.begin(), open.end(), 0);
    for (int p = 0; p < pages; p++)
        if (!owners[p]) open[p / 64] |= 1ull << (p % 64);
    low = 0;
}

// ---- plans ----

constexpr int XCDS = 8;  // the dispatcher deals consecutive work-groups round robin to the dies, each with its own L2

size_t most_items(const Shape& g, int tokens, int seqs) {
    const size_t rows = (size_t)tokens * (g.q_heads / g.kv_heads);
    return (rows / TILE_ROWS[FEW] + seqs) * g.kv_heads + SPLITS_MOST;
}
size_t most_joins(const Shape& g, int tokens, int seqs) { return most_items(g, tokens, seqs) - SPLITS_MOST; }

namespace {
struct Tile {
    int member, tok0, row0, k0, k1, kind;
    int range;  // of a shared range, -1: of the member
};
constexpr int LEAST_KEYS = 128;  // of a piece: a tile for each wave of few rows
// Pieces of a kind's tiles: about as many as CUs. Few rows stream fastest from 216 work-groups (1 token at 131,072
// positions of 2 x 256: 128 / 192 / 216 / 240 / 256 / 512 of them 59.1 / 51.4 / 51.3 / 52.0 / 52.6 / 59.8 us; 64 sequences of 4 x 128 at
// 3,000: 256 / 512 / 768 64.1 / 69.5 / 71.9) -- or from 256 where 216 would leave a quarter of them without work.
constexpr int STREAMS = 216;
// Few rows that none of the tiles is worth a join for: 512 keys of 64 or 128 dims, 256 of 256. (Whole / split, us: a token of
// 4 x 128 at 400 / 513 / 700 positions 5.8, 6.1, 8.9 / 6.9, 6.9, 7.6; of 12 sequences 9.1, 9.2, 11.6 / 9.1, 9.5, 11.0; of
// 2 x 256 at 200 / 300 / 400 9.1, 10.9, 12.7 / 10.0, 9.7, 9.5; of 12 9.7, 11.8, 13.6 / 11.1, 11.5, 11.8.)
constexpr int WHOLE = 512 * 128;
constexpr int WIDE_SPLITS = 8, WIDE_ROWS = 512;
// Rows of a shared batch, times their dims, that are joined by 64 dims a work-group. (Whole calls, us, by 64 dims / row by row,
// sequences of a token on a prompt of 4,096 of 4 x 128: 4 12.2 / 14.7, 8 13.4 / 14.6, 16 18.0 / 14.7; 8 and 16 of 2 x 256 15.8 / 17.9,
// 20.1 / 18.9.)
constexpr int WIDE_SHARED = 512 * 64;
// Rows and splits of a shared batch that are joined a row a work-group. (Whole calls, us, so / D / 4 lanes a row: 8 verifies of 4
// tokens at 65,536, 2 x 256, 512 rows of 54 splits 61.2 / 66; 16 tokens on 16,384 of 4 x 128 23.9 / 26.9; 64 tokens, 2,048 rows of
// up to 40 42.5 / 39.6, of 8 x 64 35.7 / 31.)
constexpr int ROW_SPLITS = 16, ROW_ROWS = 1024;
}  // namespace

// Dies take the items of a list in turn (position i: die i % 8). The tiles of one (sequence, head, split) stream the same
// keys, so they go to one die, dealt over several where they are more than a die's share of the work; on a die the longest
// comes first.
static void deal(std::vector<Item>& items) {
    struct Bunch {
        long long work;
        std::vector<int> at;
    };
    std::vector<Bunch> bunches;
    long long all = 0;
    auto work = [&](const Item& i) { return (long long)(i.k1 - i.k0) + 2 * KEYS; };
    for (const Item& i : items) all += work(i);
    for (size_t i = 0; i < items.size();) {  // items of a bunch lie together
        size_t e = i;
        long long w = 0;
        while (e < items.size() && items[e].seq == items[i].seq && items[e].head == items[i].head && items[e].split == items[i].split)
            w += work(items[e++]);
        const int ways = (int)std::min<long long>(e - i, std::max<long long>(1, (w * XCDS + all - 1) / std::max(1ll, all)));
        for (int k = 0; k < ways; k++) {
            Bunch b{0, {}};
            for (size_t x = i + k; x < e; x += ways) {
                b.work += work(items[x]);
                b.at.push_back((int)x);
            }
            bunches.push_back(std::move(b));
        }
        i = e;
    }
    std::stable_sort(bunches.begin(), bunches.end(), [](const Bunch& a, const Bunch& b) { return a.work > b.work; });
    long long load[XCDS] = {};
    std::vector<int> mine[XCDS];
    for (const Bunch& b : bunches) {
        const int x = (int)(std::min_element(load, load + XCDS) - load);
        load[x] += b.work;
        mine[x].insert(mine[x].end(), b.at.begin(), b.at.end());
    }
    std::vector<Item> out;
    out.reserve(items.size());
    size_t next[XCDS] = {};
    for (auto& m : mine)
        std::stable_sort(m.begin(), m.end(), [&](int a, int b) { return work(items[a]) > work(items[b]); });
    for (size_t i = 0; i < items.size(); i++) {
        int x = i % XCDS;
        if (next[x] == mine[x].size())  // that die has all of its own: the one with the most left gives
            for (int y = 0; y < XCDS; y++)
                if (mine[y].size() - next[y] > mine[x].size() - next[x]) x = y;
        out.push_back(items[mine[x][next[x]++]]);
    }
    items.swap(out);
}

namespace {
int pieces_of(const Tile& t, long long length) {  // of at most so many KEYS
    return (int)(((t.k1 - t.k0 + KEYS - 1) / KEYS + length - 1) / length);
}

// The least length of a piece (in KEYS) that gives no more pieces than places.
long long shortest(const std::vector<Tile>& tiles, int kv_heads, int places) {
    long long lo = LEAST_KEYS / KEYS, hi = lo;
    for (const Tile& t : tiles) hi = std::max(hi, (long long)(t.k1 - t.k0 + KEYS - 1) / KEYS);
    while (lo < hi) {
        const long long mid = (lo + hi) / 2;
        long long n = 0;
        for (const Tile& t : tiles) n += (long long)pieces_of(t, mid) * kv_heads;
        if (n <= places) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// Few rows: whole where they are short; else as many pieces as stream fastest, unless that leaves one much longer than a
// CU's share of the keys: then, and where the tiles are more than the CUs, pieces of three quarters of a share, dealt out as
// CUs fall free. (A token each of sequences at 500 .. 8,001 positions, 4 x 128, 64 of them: as many pieces as CUs 85 us,
// pieces of 1/2, 3/4, 1, 3/2 and 2 shares 65 / 63 / 66 / 68 / 76; 50 of them 73 and 56 / 54 / 57 / 59 / 58; 30 of them,
// where the longest piece is 1.6 shares of 1,147 keys, 32 and 35 for 3/4; 64 at 2,000 .. 4,000, the longest 1.4 of 2,858,
// 66 and 68.)
long long few_length(const std::vector<Tile>& tiles, const Shape& g) {
    const int kv_heads = g.kv_heads;
    const long long whole = (long long)tiles.size() * kv_heads;
    long long keys = 0, n = 0, longest = 0;
    for (const Tile& t : tiles) {
        keys += (long long)(t.k1 - t.k0) * kv_heads;
        longest = std::max<long long>(longest, t.k1 - t.k0);
    }
    if (longest <= WHOLE / std::max(g.head_dim, 128)) return std::max(1ll, (longest + KEYS - 1) / KEYS);
    const long long share = (keys + CUS - 1) / CUS, dealt = std::max<long long>(LEAST_KEYS, share * 3 / 4) / KEYS;
    if (whole > CUS) return dealt;
    auto count = [&](long long length) {
        n = longest = 0;
        for (const Tile& t : tiles) {
            const int p = pieces_of(t, length);
            n += (long long)p * kv_heads;
            longest = std::max<long long>(longest, (t.k1 - t.k0 + p - 1) / p);
        }
    };
    long long length = shortest(tiles, kv_heads, whole <= STREAMS ? STREAMS : CUS);
    count(length);
    if (n < STREAMS * 3 / 4) count(length = shortest(tiles, kv_heads, CUS));
    return longest * 5 > share * 7 + 5 * 512 ? dealt : length;
}

// us per key of a work-group: tiles of 128 and 256 rows, heads of 64, 128 and 256
constexpr double CHUNK_US[2][3] = {{.0107, .0162, .0295}, {.0155, .029, .062}};
// Chunks: the cheapest length of a piece by a model of the call in us: a piece's keys, 9 for its beginning and end, the split
// partials written and read back at 5 TB/s and 3 for the launch that joins them. (Pieces that are more than the CUs run in
// rounds; half a mean piece is added for the last one. Where CUs stand idle behind short pieces the card, limited by its
// power, runs the others faster: up to .65 of the time.) Tiles of shared ranges are much longer than the others: with them
// the call may be as long as its longest piece.
// (The call's cost for one length; returns the split partials' rows.)
long long chunk_cost(const std::vector<Tile>& tiles, const Shape& g, int kind, long long length, double& c) {
    const double key = CHUNK_US[kind == MANY][g.head_dim / 128];
    long long n = 0, sum = 0, rows = 0, most = 0;
    bool shared = false;
    for (const Tile& t : tiles) {
        const int p = pieces_of(t, length);
        const long long keys = t.k1 - t.k0;
        n += (long long)p * g.kv_heads;
        sum += keys * g.kv_heads;
        most = std::max(most, (keys + p - 1) / p);
        shared |= t.range >= 0;
        if (p > 1 || t.range >= 0) rows += (long long)p * TILE_ROWS[kind] * g.kv_heads;
    }
    const double busy = (double)sum / ((double)CUS * most);
    c = n <= CUS ? most * key * (.65 + .35 * std::min(1., busy)) + 9
                 : (double)sum / CUS * key + 9. * n / CUS + .5 * sum / n * key;
    if (shared) c = std::max(c, most * key + 9);
    if (rows) c += 3 + 8. * g.head_dim * rows / 5e6;
    return rows;
}
long long chunk_length(const std::vector<Tile>& tiles, const Shape& g, int kind, double& cost) {
    long long longest = LEAST_KEYS / KEYS, best = longest;
    for (const Tile& t : tiles) longest = std::max(longest, (long long)(t.k1 - t.k0 + KEYS - 1) / KEYS);
    cost = 1e30;
    for (long long length = longest;; length = length * 7 / 8) {  // from whole tiles down
        if (length < LEAST_KEYS / KEYS) break;
        double c;
        const long long rows = chunk_cost(tiles, g, kind, length, c);
        if (c < cost) {
            cost = c;
            best = length;
        }
        if (rows > PART_ROWS) break;  // no room for more
    }
    return best;
}
// What a launch for few rows adds to one for chunks, us: 3 before its first product, the keys at 5.5 TB/s or the longest
// piece, 4 where the pieces have to be joined.
double few_cost(const std::vector<Tile>& tiles, const Shape& g, long long length) {
    if (tiles.empty()) return 0;
    long long keys = 0, longest = 0;
    bool split = false;
    for (const Tile& t : tiles) {
        const int p = pieces_of(t, length);
        keys += (long long)(t.k1 - t.k0) * g.kv_heads;
        longest = std::max<long long>(longest, (t.k1 - t.k0 + p - 1) / p);
        split |= p > 1;
    }
    return 3 + std::max(keys * g.head_dim * 4 / 5.5e6, longest * g.head_dim * 7e-5) + (split ? 4 : 0);
}

// The least that tiles of few rows among a chunk's can take, us: their keys through LDS at 3.2 TB/s; where the pieces are
// more than the CUs, some CU has two of those that are at least the last CU's.
double mixed_least(const std::vector<Tile>& tiles, const Shape& g, long long length) {
    long long keys = 0;
    std::vector<int> pieces;
    for (const Tile& t : tiles) {
        const int p = pieces_of(t, length);
        pieces.insert(pieces.end(), (size_t)p * g.kv_heads, (t.k1 - t.k0 + p - 1) / p);
        if (t.kind == FEW || t.kind == SOME) keys += (long long)(t.k1 - t.k0) * g.kv_heads;
    }
    double least = keys * g.head_dim * 4 / 3.2e6;
    if ((int)pieces.size() > CUS) {
        std::nth_element(pieces.begin(), pieces.begin() + CUS, pieces.end(), std::greater<int>());
        const int next = pieces[CUS], last = *std::min_element(pieces.begin(), pieces.begin() + CUS);
        least = std::max(least, (next + last) * CHUNK_US[0][g.head_dim / 128] + 18);
    }
    return least;
}

// Chunks whose tiles are all about as long and some more than the CUs take in whole rounds: those of the last round cut into
// pieces for all CUs, where the model above makes that cheaper. The number of tiles cut (the first ones; 0: none), and the
// length of their pieces in KEYS. (1,050 / 1,100 / 1,200 tokens at 8,000 positions of 4 x 128, 264 to 300 tiles: 202 / 201 /
// 176 us, cut so 152 / 154 / 168; 2,100 at 16,000 of 2 x 256 589 / 468.)
int last_round(const std::vector<Tile>& tiles, const Shape& g, int kind, double& cost, long long& length) {
    const int n = (int)tiles.size() * g.kv_heads, rounds = n / CUS, cut = (int)tiles.size() - rounds * CUS / g.kv_heads;
    if (!rounds || cut <= 0) return 0;
    long long sum = 0, longest = 0, last = 0;
    for (const Tile& t : tiles) {
        sum += t.k1 - t.k0;
        longest = std::max<long long>(longest, t.k1 - t.k0);
    }
    if (longest * (long long)tiles.size() > sum * 5 / 4) return 0;
    for (int i = 0; i < cut; i++) last = std::max<long long>(last, (tiles[i].k1 - tiles[i].k0 + KEYS - 1) / KEYS);
    const int p = CUS / (cut * g.kv_heads);
    if (p < 3) return 0;  // (of two pieces a tile: 1,500 tokens at 8,000 positions 198 us, 184 with all tiles cut alike)
    const long long piece = std::max<long long>(LEAST_KEYS / KEYS, (last + p - 1) / p);
    long long pieces = 0;
    for (int i = 0; i < cut; i++) pieces += (long long)pieces_of(tiles[i], piece) * g.kv_heads;
    const double key = CHUNK_US[kind == MANY][g.head_dim / 128], rows = (double)pieces * TILE_ROWS[kind];
    const double c = rounds * (longest * key + 9) + piece * KEYS * key + 9 + 3 + 8. * g.head_dim * rows / 5e6;
    if (rows > PART_ROWS || c >= .97 * cost) return 0;
    cost = c;
    length = piece;
    return cut;
}
}  // namespace

int splits_room(int rows, int kv_heads, int part, int more) {
    return std::min({SPLITS_MOST, (PART_ROWS - part) / (rows * kv_heads), 1 + (SPLITS_MOST - more) / kv_heads});
}

namespace {
// Which of a batch's common positions are attended once for all that have them. Apart they are read once for each (though the
// later readings may find them in a cache); together they cost a launch more, or tiles among those there, and their partials.
// What is found here is worth a draft; whether it is attended so, the model of the whole call says (cost_of).
struct Sharer {
    static constexpr int LEAST = 128;         // positions of a range
    static constexpr int LEAST_SPARED = 512;  // positions that a range spares its sequences, in all
    static constexpr int ROWS = 256;          // of a sequence with more rows no tile is worth sharing
    static constexpr int DEEP = 64;           // forks of forks that are looked through
    const Book& b;
    const std::vector<Member>& batch;
    Share& out;
    const std::vector<int>& table(int i) const { return b.table[batch[i].seq]; }
    int whole(int i) const { return (batch[i].len - batch[i].count) / b.page; }  // pages before the new tokens
    // pages that i and j have in common
    int common(int i, int j) const {
        const std::vector<int>&x = table(i), &y = table(j);
        int lo = 0, hi = std::min(whole(i), whole(j));
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (x[mid - 1] == y[mid - 1]) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    }
    void leaf(int i, int start, int range) {
        out.from[i] = start * b.page;
        out.range[i] = range;
        out.members.push_back(i);
    }
    // who: sequences that have pages [0, probe) in common, of which those before `start` are done by `range` and what it is in
    void split(std::vector<int>& who, int start, int probe, int range, int level, int deep) {
        auto page = [&](int i) { return whole(i) > probe ? table(i)[probe] : -1 - i; };
        if (level == LEVELS || deep == DEEP) {
            for (int i : who) leaf(i, start, range);
            return;
        }
        std::stable_sort(who.begin(), who.end(), [&](int i, int j) { return page(i) < page(j); });
        for (size_t x = 0; x < who.size();) {
            size_t y = x + 1;
            int end = whole(who[x]);
            for (; y < who.size() && page(who[y]) == page(who[x]); y++) end = std::min(end, common(who[x], who[y]));
            if (y - x == 1) {
                leaf(who[x], start, range);
            } else {
                std::vector<int> group(who.begin() + x, who.begin() + y);
                const long long span = (long long)(end - start) * b.page;
                const bool pays = span >= LEAST && span * (long long)(group.size() - 1) >= LEAST_SPARED;
                if (pays) out.ranges.push_back({start * b.page, end * b.page, (int)out.members.size(), (int)group.size(), range});
                if (pays) split(group, end, end, (int)out.ranges.size() - 1, level + 1, deep + 1);
                else split(group, start, end, range, level, deep + 1);
            }
            x = y;
        }
    }
};
}  // namespace

void share(const Book& b, const Shape& g, const std::vector<Member>& batch, Share& out) {
    const int n = (int)batch.size(), group = g.q_heads / g.kv_heads;
    out = Share{};
    out.from.assign(n, 0);
    out.range.assign(n, -1);
    out.at.assign(n, 0);
    std::vector<int> who;
    for (int i = 0; i < n; i++)
        if (batch[i].count > 0 && (long long)batch[i].count * group <= Sharer::ROWS) who.push_back(i);
    Sharer s{b, batch, out};
    s.split(who, 0, 0, -1, 0, 0);
    if (out.ranges.empty()) return;
    std::vector<int> tok(n);
    for (int i = 0, t = 0; i < n; t += batch[i++].count) tok[i] = t;
    for (int i : out.members) {
        out.at[i] = (int)out.order.size();
        for (int t = 0; t < batch[i].count; t++) out.order.push_back({tok[i] + t, batch[i].len - batch[i].count + t});
    }
}

namespace {
// A shared range in a window: its rows, their first entry in the order, the first key that any of them sees (rows 0: none sees
// any); its splits and partials.
struct Common {
    int rows = 0, tok0 = 0, k0 = 0, splits = 0, part = 0;
};
// How a batch's work may be cut. APART: every sequence by itself. STREAMED: what they share in tiles of 32 rows beside their own, all
// by few_rows (or, where few rows go among a chunk's tiles, with them). TILED: what they share in a chunk's tiles where it has more than
// 32 rows. (Whole calls, us, 2 / 4 / 8 / 16 / 64 tokens on
// a prompt of 16,384 of 4 x 128, 32 heads: apart 16.7 / 23.4 / 38.9 / 55 / 123, where the later readings come out of the L2s at 17 TB/s;
// streamed 14.8 / 15.8 / 19.1 / 30.9 / 48; tiled 13.8 / 21 / 20.6 / 26.8 / 39.)
enum Way { APART, STREAMED, TILED };
struct Draft {
    std::vector<Tile> tiles[KINDS];
    long long length[KINDS], piece[KINDS] = {};  // of a piece of each kind's tiles; of those in the last round of CUs
    int cut[KINDS] = {};                         // tiles of that round
    std::vector<Common> common;
    double cost = 0;  // us, of a batch with pages in common
};

// What a launch for few rows takes where sequences have keys in common: `distinct` bytes from memory, all of them from the L2s, or
// the longest piece of a work-group alone on its CU (several share it where there are more), and 9 for its beginning, its
// end and the join (5 without one).
double stream_cost(const std::vector<Tile>& tiles, const Shape& g, int kind, long long length, double distinct, bool joined) {
    if (tiles.empty()) return 0;
    double keys = 0, n = 0, longest = 0;
    for (const Tile& t : tiles) {
        const int p = pieces_of(t, length);
        n += (double)p * g.kv_heads;
        keys += (double)(t.k1 - t.k0) * g.kv_heads;
        longest = std::max<double>(longest, (t.k1 - t.k0 + p - 1) / p);
        joined |= p > 1;
    }
    const double bytes = 4. * g.head_dim, us = g.head_dim * (kind == SOME ? 1.25e-4 : 7e-5);  // of a key
    const double work = n <= CUS ? longest * us : (keys / CUS * (g.head_dim <= 128 ? .7 : 1.) + .5 * longest) * us;
    return (joined ? 9 : 5) + std::max({distinct * bytes / 5.5e6, keys * bytes / 17e6, work});
}

void draft(const Shape& g, const std::vector<Member>& batch, const Share* share, int window, Way way, Draft& out) {
    const int group = g.q_heads / g.kv_heads;
    std::vector<Tile>(&by_kind)[KINDS] = out.tiles;
    if (way == APART) share = nullptr;
    auto add = [&](int i, int tok0, int kind) {
        const Member& m = batch[i];
        const int rows = m.count * group, pos0 = m.len - m.count, from = share ? share->from[i] : 0;
        for (int r = 0; r < rows; r += TILE_ROWS[kind]) {
            const int last = (std::min(r + TILE_ROWS[kind], rows) - 1) / group;
            const int lo = window ? std::max(0, pos0 + r / group - window + 1) : 0;
            by_kind[kind].push_back({i, tok0, r, std::max(from, lo / KEYS * KEYS), pos0 + last + 1, kind, -1});
        }
    };
    int tok0 = 0;
    for (int i = 0; i < (int)batch.size(); i++) {
        const int rows = batch[i].count * group;
        if (rows <= TILE_ROWS[SOME]) {
            add(i, tok0, rows <= TILE_ROWS[FEW] && way != STREAMED ? FEW : SOME);
        } else {  // either size of tile is a candidate
            add(i, tok0, HALF);
            add(i, tok0, MANY);
        }
        tok0 += batch[i].count;
    }
    out.common.resize(share ? share->ranges.size() : 0);
    bool any = false;
    for (size_t x = 0; x < out.common.size(); x++) {
        const Range& r = share->ranges[x];
        Common& c = out.common[x];
        c.tok0 = share->at[share->members[r.first]];
        int lo = r.k1;
        for (int i = r.first; i < r.first + r.count; i++) {
            const Member& m = batch[share->members[i]];
            c.rows += m.count * group;
            lo = std::min(lo, window ? std::max(0, m.len - m.count - window + 1) : 0);
        }
        c.k0 = std::max(r.k0, lo / KEYS * KEYS);
        if (c.k0 >= r.k1) {
            c.rows = 0;
            continue;
        }
        any = true;
        auto tiles = [&](int kind) {
            for (int row = 0; row < c.rows; row += TILE_ROWS[kind])
                by_kind[kind].push_back({share->members[r.first], c.tok0, row, c.k0, r.k1, kind, (int)x});
        };
        if (c.rows <= TILE_ROWS[SOME] || way == STREAMED) {
            tiles(c.rows <= TILE_ROWS[FEW] && way != STREAMED ? FEW : SOME);
        } else {
            tiles(HALF);
            tiles(MANY);
        }
    }
    long long(&length)[KINDS] = out.length;
    for (int k : {FEW, SOME}) length[k] = few_length(by_kind[k], g);
    double half, many;
    length[HALF] = chunk_length(by_kind[HALF], g, HALF, half);
    length[MANY] = chunk_length(by_kind[MANY], g, MANY, many);
    if (!any) {  // (the tiles of a shared range are split alike)
        out.cut[HALF] = last_round(by_kind[HALF], g, HALF, half, out.piece[HALF]);
        out.cut[MANY] = last_round(by_kind[MANY], g, MANY, many, out.piece[MANY]);
    }
    // Few rows among a chunk's tiles fill CUs that its last ones leave idle, and spare a launch, often two. (us apart / among:
    // 512 tokens and 12 decodes at 500 .. 4,000 positions 31.8 / 23.9 of 4 x 128, 40.8 / 30.6 of 2 x 256; 100 and 20 at 100
    // .. 400 21.9 / 13.9, 31.8 / 19.8. 64 tokens and 60 decodes at 500 .. 8,000 of 4 x 128 92.7 / 114: those stay apart.)
    std::vector<Tile> both = by_kind[HALF];  // (of a streamed range's tiles of 32 rows those that a chunk's tiles begin with)
    for (int k : {FEW, SOME})
        std::copy_if(by_kind[k].begin(), by_kind[k].end(), std::back_inserter(both), [](const Tile& t) { return t.row0 % TILE_ROWS[HALF] == 0; });
    double together = 1e30;
    const bool mixed = !by_kind[HALF].empty() && both.size() > by_kind[HALF].size();
    const long long joint = mixed ? chunk_length(both, g, HALF, together) : 0;
    if (mixed) together = std::max(together, mixed_least(both, g, joint));
    const double apart = std::min(half, many) + few_cost(by_kind[FEW], g, length[FEW]) + few_cost(by_kind[SOME], g, length[SOME]);
    if (mixed && together <= apart) {
        for (Tile& t : both) t.kind = HALF;
        by_kind[HALF] = std::move(both);
        length[HALF] = joint;
        out.cut[HALF] = 0;
        for (int k : {FEW, SOME, MANY}) by_kind[k].clear();
    } else {
        by_kind[half <= many ? MANY : HALF].clear();
    }
}

// What a draft takes, where sequences have keys in common.
double cost_of(const Shape& g, const Share& share, const Draft& d) {
    double distinct[KINDS] = {};  // keys of the lists for few rows, what several tiles have counted once
    for (int k : {FEW, SOME}) {
        std::vector<char> seen(share.ranges.size(), 0);
        for (const Tile& t : d.tiles[k]) {
            if (t.range >= 0) {
                if (t.row0 == 0) distinct[k] += (double)(t.k1 - t.k0) * g.kv_heads;
                continue;
            }
            distinct[k] += (double)(t.k1 - t.k0) * g.kv_heads;
            for (int x = share.range[t.member]; x >= 0; x = share.ranges[x].parent) {  // of ranges that it takes by itself
                const int have = std::min(t.k1, share.ranges[x].k1) - std::max(t.k0, share.ranges[x].k0);
                if (have <= 0) continue;
                if (seen[x]) distinct[k] -= (double)have * g.kv_heads;
                seen[x] = 1;
            }
        }
    }
    bool joined = false;
    for (const Common& c : d.common) joined |= c.rows > 0;
    double chunks = 0;
    for (int k : {HALF, MANY})
        if (!d.tiles[k].empty()) chunk_cost(d.tiles[k], g, k, d.length[k], chunks);
    const double few = stream_cost(d.tiles[FEW], g, FEW, d.length[FEW], distinct[FEW], joined);
    const double some = stream_cost(d.tiles[SOME], g, SOME, d.length[SOME], distinct[SOME], joined);
    return chunks + few + some - (chunks > 0 && few + some > 0 ? 4 : 0) - (few > 0 && some > 0 ? 4 : 0);
}
}  // namespace

static void plan(const Shape& g, const std::vector<Member>& batch, const Share* share, int window, Plan& out) {
    for (auto& v : out.items) v.clear();
    out.joins.clear();
    out.segs.clear();
    const int group = g.q_heads / g.kv_heads;
    Draft best;
    draft(g, batch, share, window, APART, best);
    if (share) {
        best.cost = cost_of(g, *share, best);
        for (Way way : {STREAMED, TILED}) {
            Draft d;
            draft(g, batch, share, window, way, d);
            d.cost = cost_of(g, *share, d);
            if (d.cost < best.cost) best = std::move(d);
        }
    }
    std::vector<Common>& common = best.common;
    // the shared ranges that a member's rows have keys in, the outermost first
    auto chain = [&](int i) {
        std::vector<int> c;
        for (int x = common.empty() ? -1 : share->range[i]; x >= 0; x = share->ranges[x].parent)
            if (common[x].rows) c.insert(c.begin(), x);
        return c;
    };
    bool any = false;
    for (const Common& c : common) any |= c.rows > 0;
    std::vector<Tile> tiles;
    std::vector<long long> most;  // KEYS of a piece of the tile
    for (int k = 0; k < KINDS; k++)
        for (int i = 0; i < (int)best.tiles[k].size(); i++) {
            tiles.push_back(best.tiles[k][i]);
            most.push_back(best.cut[k] ? i < best.cut[k] ? best.piece[k] : 1 << 20 : best.length[k]);
        }
    int part = 0, more = 0;  // partials and work items that splits have taken
    // What shared ranges and the rows in them cannot do without: a split's partials each, and the ranges' work items.
    long long least = 0, items = 0;
    if (any) {
        for (const Common& c : common) least += (long long)c.rows * g.kv_heads;
        for (const Tile& t : tiles) {
            if (t.range >= 0) items += g.kv_heads;
            else if (!chain(t.member).empty())
                least += (long long)std::min(TILE_ROWS[t.kind], batch[t.member].count * group - t.row0) * g.kv_heads;
        }
        if (least > PART_ROWS || items > SPLITS_MOST / 2) {
            plan(g, batch, nullptr, window, out);
            return;
        }
        more = (int)items;
        for (size_t i = 0; i < tiles.size(); i++) {
            const Tile& t = tiles[i];
            if (t.range < 0) continue;
            Common& c = common[t.range];
            if (!c.splits) {  // its first tile
                const int count = (c.rows + TILE_ROWS[t.kind] - 1) / TILE_ROWS[t.kind];
                least -= (long long)c.rows * g.kv_heads;
                c.splits = std::min({pieces_of(t, most[i]), splits_room(c.rows, g.kv_heads, part + (int)least, more), SPLITS_MOST / (LEVELS + 1),
                                     1 + (SPLITS_MOST - more) / (g.kv_heads * count)});
                c.splits = std::max(c.splits, 1);
                more += (c.splits - 1) * g.kv_heads * count;
                c.part = part;
                part += c.splits * c.rows * g.kv_heads;
            }
            const Range& r = share->ranges[t.range];
            const int units = (t.k1 - t.k0 + KEYS - 1) / KEYS, last = std::min(t.row0 + TILE_ROWS[t.kind], c.rows) - 1;
            int top = 0;
            for (int x = t.row0 / group; x <= last / group; x++) top = std::max(top, share->order[c.tok0 + x].pos + 1);
            for (int head = 0; head < g.kv_heads; head++)
                for (int s = 0; s < c.splits; s++)
                    out.items[t.kind].push_back({batch[t.member].seq, head, c.tok0, t.row0, c.rows, r.k1,
                                                 t.k0 + (int)((long long)units * s / c.splits) * KEYS,
                                                 s + 1 < c.splits ? t.k0 + (int)((long long)units * (s + 1) / c.splits) * KEYS : t.k1,
                                                 c.part + (head * c.splits + s) * c.rows + t.row0, s, top, 0});
        }
    }
    for (size_t i = 0; i < tiles.size(); i++) {
        const Tile& t = tiles[i];
        if (t.range >= 0) continue;
        const Member& m = batch[t.member];
        const int rows = m.count * group, count = std::min(TILE_ROWS[t.kind], rows - t.row0);
        const int units = (t.k1 - t.k0 + KEYS - 1) / KEYS;
        const std::vector<int> in = any ? chain(t.member) : std::vector<int>();
        if (!in.empty()) least -= (long long)count * g.kv_heads;
        int splits = std::min(pieces_of(t, most[i]), splits_room(count, g.kv_heads, part + (int)least, more));
        if (!in.empty()) splits = std::min(splits, SPLITS_MOST / (LEVELS + 1));
        if (splits < 2) splits = 1;
        more += (splits - 1) * g.kv_heads;
        const bool joined = splits > 1 || !in.empty();
        for (int head = 0; head < g.kv_heads; head++) {
            for (int s = 0; s < splits; s++) {
                const int a = t.k0 + (int)((long long)units * s / splits) * KEYS;
                const int b = s + 1 < splits ? t.k0 + (int)((long long)units * (s + 1) / splits) * KEYS : t.k1;
                out.items[t.kind].push_back({m.seq, head, t.tok0, t.row0, rows, m.len - m.count, a, b,
                                             joined ? part + s * count : -1, s, 0, 0});
            }
            if (joined) {
                out.joins.push_back({head, t.tok0, t.row0, count, part, splits, 0, (int)in.size()});
                part += splits * count;
                for (int x = 0; any && x < LEVELS; x++) {
                    Seg seg{0, 0, 0, 0};
                    if (x < (int)in.size()) {
                        const Common& c = common[in[x]];
                        const int row = (share->at[t.member] - c.tok0) * group + t.row0;
                        seg = {c.part + head * c.splits * c.rows + row, c.rows, c.splits, 0};
                    }
                    out.segs.push_back(seg);
                }
            }
        }
    }
    // Many splits of few rows are read by many work-groups at once; of many rows the rows are work enough (3,200 rows of 9
    // splits by 64 dims each: 45 us, row by row 14).
    long long rows = 0;
    for (const Join& j : out.joins) rows += j.count;
    for (size_t n = 0; n < out.joins.size(); n++) {
        Join& j = out.joins[n];
        int splits = j.splits;
        for (int x = 0; x < j.segs; x++) splits += out.segs[n * LEVELS + x].splits;
        j.wide = splits > WIDE_SPLITS && (any ? rows * g.head_dim <= WIDE_SHARED : rows <= WIDE_ROWS);
        if (any && !j.wide && splits > ROW_SPLITS && rows <= ROW_ROWS) j.wide = ROW_WIDE;
    }
    for (auto& list : out.items) {
        std::stable_sort(list.begin(), list.end(), [](const Item& a, const Item& b) {
            return a.seq != b.seq ? a.seq < b.seq : a.head != b.head ? a.head < b.head : a.split < b.split;
        });
        deal(list);
    }
}

void plan_window(const Shape& g, const std::vector<Member>& batch, int window, Plan& out) { plan(g, batch, nullptr, window, out); }
void plan_shared(const Shape& g, const std::vector<Member>& batch, const Share& s, int window, Plan& out) {
    plan(g, batch, s.ranges.empty() ? nullptr : &s, window, out);
}

// ---- accumulated attention weights ----

bool may_weigh(const Shape& g, int tokens, int seqs, int ctx, int window, int last, const WeighRoom& room, int list) {
    const long long rows = (long long)(last ? std::min(last, tokens) : tokens) * (g.q_heads / g.kv_heads);
    // (a sequence's scores are of whole blocks of keys)
    const double scores = (double)std::min(seqs, tokens) * ((ctx + KEYS - 1) / KEYS * KEYS) * rows * g.kv_heads;
    const bool many = rows > TILE_ROWS[SOME] || scores > room.work - WEIGH_PARTS;
    switch (list) {
        case SCORE_SOME: return rows > TILE_ROWS[FEW];
        case SCORE_MANY: case MERGES: case SUM_MANY: return many;
        case FADES: return many || window;
        default: return true;
    }
}

size_t weigh_entries(const Shape& g, int tokens, int seqs) {
    const size_t group = g.q_heads / g.kv_heads;
    return ((size_t)tokens * group / SCORE_ROWS + 2 * (size_t)std::min(seqs, tokens)) * g.kv_heads + WEIGH_MOST;
}

void plan_weigh(const Shape& g, const std::vector<Member>& batch, int window, int last, const WeighRoom& room, WeighPlan& out) {
    for (auto& v : out.scores) v.clear();
    for (auto& v : out.sums) v.clear();
    out.merges.clear();
    out.fades.clear();
    const int group = g.q_heads / g.kv_heads, heads = g.kv_heads;
    struct Weighed {  // a sequence with counted tokens
        int seq, tok0, rows, pos0, k0, len, scores;
    };
    std::vector<Weighed> few, many;
    long long stats = 0, work = 0, few_keys = 0, tile_keys = 0, rows_left = 0;
    int tok = 0;
    for (const Member& m : batch) {
        const int n = last ? std::min(last, m.count) : m.count, tok0 = tok + m.count - n;
        tok += m.count;
        if (!n) continue;
        const int pos0 = m.len - n, k0 = (window ? std::max(0, pos0 - window + 1) : 0) / KEYS * KEYS, rows = n * group;
        const long long blocks = (m.len - k0 + KEYS - 1) / KEYS, kept = blocks * KEYS * rows * heads;
        rows_left += (long long)rows * heads;
        Weighed w{m.seq, tok0, rows, pos0, k0, m.len, -1};
        if (rows <= TILE_ROWS[SOME] && work + kept <= room.work - WEIGH_PARTS) {
            w.scores = (int)work;
            work += kept;
            few_keys += (long long)(m.len - k0) * heads;
            few.push_back(w);
        } else {
            tile_keys += (long long)((rows + SCORE_ROWS - 1) / SCORE_ROWS) * (m.len - k0) * heads;
            many.push_back(w);
        }
        if (k0 > 0)
            for (int h = 0; h < heads; h++) out.fades.push_back({m.seq, h, 0, k0, 0, 0, 0, 0});
    }
    // rows x pieces of statistics, at least one piece for all that is left
    auto pieces_in = [&](int rows, long long units, long long length) {
        const long long p = (units + length - 1) / length, most = (room.stats - stats - rows_left) / rows;
        return (int)std::max(1ll, std::min(p, most));
    };
    int more = 0;
    // Few rows: bound by the keys' stream. Whole where they are short, which spares the launch for their sums (a token at 300
    // positions of 2 x 256 6.2 us, in three pieces 8.4; 12 windows of 545 keys of 4 x 128 9.3 and 9.2); else in about four pieces a
    // CU. (The statistics of 64 sequences at 500 .. 8,001 positions of 4 x 128 in 428 / 640 / 1,160 / 2,300 work-groups: 45.5 / 44.1
    // / 42.3 / 41.5 us.)
    constexpr int WHOLE_FEW = 512;
    const long long few_length = std::max<long long>(LEAST_KEYS, (few_keys + 4 * CUS - 1) / (4 * CUS)) / KEYS;
    for (const Weighed& w : few) {
        const int units = (w.len - w.k0 + KEYS - 1) / KEYS;
        for (int h = 0; h < heads; h++) {
            rows_left -= w.rows;
            int pieces = units * KEYS <= WHOLE_FEW ? 1 : pieces_in(w.rows, units, few_length);
            pieces = std::min(pieces, 1 + (WEIGH_MOST / 2 - std::min(more, WEIGH_MOST / 2)));
            more += pieces - 1;
            const int scores = w.scores + h * units * KEYS * w.rows, stat = (int)stats;
            stats += (long long)pieces * w.rows;
            for (int p = 0; p < pieces; p++) {
                const int a = (int)((long long)units * p / pieces), b = (int)((long long)units * (p + 1) / pieces);
                out.scores[w.rows <= TILE_ROWS[FEW] ? SCORE_FEW : SCORE_SOME].push_back(
                    {w.seq, h, w.tok0, w.rows, 0, w.pos0, w.k0 + a * KEYS, std::min(w.len, w.k0 + b * KEYS), stat + p * w.rows,
                     scores + a * KEYS * w.rows, pieces == 1, 0});
            }
            if (pieces > 1)
                out.sums[0].push_back({w.seq, h, w.tok0, w.rows, w.pos0, w.k0, w.len, 0, w.rows, stat, pieces, scores, w.k0, -1, {0, 0}});
        }
    }
    // their sums by ranges of keys
    {
        std::vector<Sum> whole;
        whole.swap(out.sums[0]);
        const long long keys = std::min(1ll << 30, std::max<long long>(512, (few_keys / (WEIGH_MOST / 4) + 255) / 256 * 256));
        for (Sum s : whole) {
            const int end = s.k1;
            for (int k = s.k0; k < end; k += (int)keys) {
                s.k0 = k;
                s.k1 = (int)std::min<long long>(end, k + keys);
                out.sums[0].push_back(s);
            }
        }
    }
    // Many rows: bound by the matrix units and the exponentials. Tiles of rows against all their keys, split where they are few.
    more = 0;
    constexpr int PLACES = 2 * CUS;  // (32 tokens of 16 heads at 16,000 positions of 2 x 256: 32.6 us, with 256 / 384 / 768 34.5 / 32.6 / 32.4)
    const long long many_length = std::max<long long>(LEAST_KEYS, (tile_keys + PLACES - 1) / PLACES) / KEYS;
    long long key_tiles = 0, row_tiles = 0;
    for (const Weighed& w : many) {
        key_tiles += (long long)((w.len - w.k0 + SUM_KEYS - 1) / SUM_KEYS) * heads;
        for (int k = w.k0; k < w.len; k += SUM_KEYS) {
            const int r0 = (int)std::max(0ll, (long long)(k - w.pos0) * group);
            row_tiles += (long long)(w.rows - r0 + KEYS - 1) / KEYS * heads;
        }
    }
    const int per = (int)std::max(1ll, (key_tiles + WEIGH_MOST / 2 - 1) / (WEIGH_MOST / 2));  // key tiles of a work-group
    // rows of one (at least 4 tiles of them: 15 sequences in a window of 513, prompts of 33 .. 700 among them, 35.3 us; 8 and 16 tiles
    // 38.7 and 45.9, where a batch has fewer parts to add up)
    const long long chunk = per > 1 ? 1ll << 40 : std::max<long long>(4, (row_tiles + SUM_PLACES - 1) / SUM_PLACES) * KEYS;
    for (const Weighed& w : many) {
        const int units = (w.len - w.k0 + KEYS - 1) / KEYS;
        int pieces = 0;
        for (int h = 0; h < heads; h++) {
            rows_left -= w.rows;
            const int tiles = (w.rows + SCORE_ROWS - 1) / SCORE_ROWS;
            if (!h) {
                rows_left -= (long long)w.rows * (heads - 1);
                pieces = pieces_in(w.rows * heads, units, many_length);
                rows_left += (long long)w.rows * (heads - 1);
                pieces = std::min(pieces, 1 + std::max(0, WEIGH_MOST - more) / (tiles * heads));
                more += (pieces - 1) * tiles * heads;
            }
            const int stat = (int)stats;
            stats += (long long)pieces * w.rows;
            for (int r = 0; pieces > 1 && r < w.rows; r += SCORE_ROWS)
                out.merges.push_back({h, w.tok0, w.rows, r, std::min(r + SCORE_ROWS, w.rows), stat, pieces, 0});
            for (int r = 0; r < w.rows; r += SCORE_ROWS) {
                const int end = std::min(w.len, w.pos0 + (std::min(r + SCORE_ROWS, w.rows) - 1) / group + 1);
                const int lo = window ? std::max(0, w.pos0 + r / group - window + 1) / KEYS * KEYS : 0;
                for (int p = 0; p < pieces; p++) {  // (a piece without keys leaves its rows' statistics empty)
                    const int a = std::max(lo, w.k0 + (int)((long long)units * p / pieces) * KEYS);
                    const int b = std::min(end, w.k0 + (int)((long long)units * (p + 1) / pieces) * KEYS);
                    out.scores[SCORE_MANY].push_back(
                        {w.seq, h, w.tok0, w.rows, r, w.pos0, a, std::max(a, b), stat + p * w.rows + r, -1, pieces == 1, 0});
                }
            }
            for (int k = w.k0; k < w.len; k += SUM_KEYS * per) {
                const int end = std::min(w.len, k + SUM_KEYS * per);
                const int r0 = (int)std::min<long long>(w.rows, std::max(0ll, (long long)(k - w.pos0) * group)) / KEYS * KEYS;
                const long long seen = std::max(0ll, ((long long)end - 1 + window - w.pos0) * group);
                const int r1 = window ? (int)std::min<long long>(w.rows, seen) : w.rows;
                int sums = (int)std::max(1ll, (std::max(0, r1 - r0) + chunk - 1) / chunk);
                if (sums > 1 && work + (long long)sums * SUM_KEYS > room.work) sums = 1;
                for (int x = 0; x < sums; x++) {
                    const int units_of = (std::max(0, r1 - r0) + KEYS - 1) / KEYS;
                    const int a = r0 + (int)((long long)units_of * x / sums) * KEYS;
                    const int b = std::min(std::max(r0, r1), r0 + (int)((long long)units_of * (x + 1) / sums) * KEYS);
                    out.sums[1].push_back({w.seq, h, w.tok0, w.rows, w.pos0, k, end, a, b, stat, pieces, -1, 0,
                                           sums > 1 ? (int)work + x * SUM_KEYS : -1, {0, 0}});
                }
                if (sums > 1) {
                    out.fades.push_back({w.seq, h, k, end, (int)work, sums, SUM_KEYS, 0});
                    work += (long long)sums * SUM_KEYS;
                }
            }
        }
    }
    // All tiles of rows run at once, several on a CU, which takes every CUS-th of them: the longest beside the shortest.
    auto& tiles = out.scores[SCORE_MANY];
    std::stable_sort(tiles.begin(), tiles.end(), [](const Score& x, const Score& y) { return x.k1 - x.k0 > y.k1 - y.k0; });
    for (size_t i = CUS; i < tiles.size(); i += 2 * CUS) std::reverse(tiles.begin() + i, tiles.begin() + std::min(tiles.size(), i + CUS));
}

}  // namespace paged
}  // namespace mkv
