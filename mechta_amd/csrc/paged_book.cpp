// paged_book.cpp -- which pages belong to whom, and how a batch's attention is cut into work (paged_book.h).
#include "paged_book.h"

#include <algorithm>
#include <climits>

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
        *cut = Cut{len[seq], from, shared, std::vector<int>(t.begin() + from, t.end())};
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
    return MKV_OK;
}

void Book::undo_set_len(int seq, const Cut& cut) {
    std::vector<int>& t = table[seq];
    if (cut.copied) {
        drop(t.back());
        t.pop_back();
    }
    for (int p : cut.pages) {  // the table has room for what it had
        if (!owners[p]++) {
            open[p / 64] &= ~(1ull << (p % 64));
            free--;
        }
        t.push_back(p);
    }
    len[seq] = cut.len;
    stale(seq, cut.from);
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
};
constexpr int LEAST_KEYS = 128;  // of a piece: a tile for each wave of few rows
// Pieces of a kind's tiles: about as many as CUs. Few rows stream fastest from 216 work-groups (1 token at 131,072
// positions of 2 x 256: 128 / 192 / 216 / 240 / 256 / 512 of them 59.1 / 51.4 / 51.3 / 52.0 / 52.6 / 59.8 us; 64 sequences of 4 x 128 at
// 3,000: 256 / 512 / 768 64.1 / 69.5 / 71.9) -- or from 256 where 216 would leave a quarter of them without work.
constexpr int CUS = 256, STREAMS = 216;
// Few rows that none of the tiles is worth a join for: 512 keys of 64 or 128 dims, 256 of 256. (Whole / split, us: a token of
// 4 x 128 at 400 / 513 / 700 positions 5.8, 6.1, 8.9 / 6.9, 6.9, 7.6; of 12 sequences 9.1, 9.2, 11.6 / 9.1, 9.5, 11.0; of
// 2 x 256 at 200 / 300 / 400 9.1, 10.9, 12.7 / 10.0, 9.7, 9.5; of 12 9.7, 11.8, 13.6 / 11.1, 11.5, 11.8.)
constexpr int WHOLE = 512 * 128;
constexpr int WIDE_SPLITS = 8, WIDE_ROWS = 512;
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
// power, runs the others faster: up to .65 of the time.)
long long chunk_length(const std::vector<Tile>& tiles, const Shape& g, int kind, double& cost) {
    const double key = CHUNK_US[kind == MANY][g.head_dim / 128];
    long long longest = LEAST_KEYS / KEYS, best = longest;
    for (const Tile& t : tiles) longest = std::max(longest, (long long)(t.k1 - t.k0 + KEYS - 1) / KEYS);
    cost = 1e30;
    for (long long length = longest;; length = length * 7 / 8) {  // from whole tiles down
        if (length < LEAST_KEYS / KEYS) break;
        long long n = 0, sum = 0, rows = 0, most = 0;
        for (const Tile& t : tiles) {
            const int p = pieces_of(t, length);
            const long long keys = t.k1 - t.k0;
            n += (long long)p * g.kv_heads;
            sum += keys * g.kv_heads;
            most = std::max(most, (keys + p - 1) / p);
            if (p > 1) rows += (long long)p * TILE_ROWS[kind] * g.kv_heads;
        }
        const double busy = (double)sum / ((double)CUS * most);
        double c = n <= CUS ? most * key * (.65 + .35 * std::min(1., busy)) + 9
                            : (double)sum / CUS * key + 9. * n / CUS + .5 * sum / n * key;
        if (rows) c += 3 + 8. * g.head_dim * rows / 5e6;
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

void plan_window(const Shape& g, const std::vector<Member>& batch, int window, Plan& out) {
    for (auto& v : out.items) v.clear();
    out.joins.clear();
    const int group = g.q_heads / g.kv_heads;
    std::vector<Tile> by_kind[KINDS];
    auto add = [&](int i, int tok0, int kind) {
        const Member& m = batch[i];
        const int rows = m.count * group, pos0 = m.len - m.count;
        for (int r = 0; r < rows; r += TILE_ROWS[kind]) {
            const int last = (std::min(r + TILE_ROWS[kind], rows) - 1) / group;
            const int lo = window ? std::max(0, pos0 + r / group - window + 1) : 0;
            by_kind[kind].push_back({i, tok0, r, lo / KEYS * KEYS, pos0 + last + 1, kind});
        }
    };
    int tok0 = 0;
    for (int i = 0; i < (int)batch.size(); i++) {
        const int rows = batch[i].count * group;
        if (rows <= TILE_ROWS[SOME]) {
            add(i, tok0, rows <= TILE_ROWS[FEW] ? FEW : SOME);
        } else {  // either size of tile is a candidate
            add(i, tok0, HALF);
            add(i, tok0, MANY);
        }
        tok0 += batch[i].count;
    }
    long long length[KINDS];
    for (int k : {FEW, SOME}) length[k] = few_length(by_kind[k], g);
    double half, many;
    length[HALF] = chunk_length(by_kind[HALF], g, HALF, half);
    length[MANY] = chunk_length(by_kind[MANY], g, MANY, many);
    long long piece[KINDS] = {};
    int cut[KINDS] = {};
    cut[HALF] = last_round(by_kind[HALF], g, HALF, half, piece[HALF]);
    cut[MANY] = last_round(by_kind[MANY], g, MANY, many, piece[MANY]);
    // Few rows among a chunk's tiles fill CUs that its last ones leave idle, and spare a launch, often two. (us apart / among:
    // 512 tokens and 12 decodes at 500 .. 4,000 positions 31.8 / 23.9 of 4 x 128, 40.8 / 30.6 of 2 x 256; 100 and 20 at 100
    // .. 400 21.9 / 13.9, 31.8 / 19.8. 64 tokens and 60 decodes at 500 .. 8,000 of 4 x 128 92.7 / 114: those stay apart.)
    std::vector<Tile> both = by_kind[HALF];
    for (int k : {FEW, SOME}) both.insert(both.end(), by_kind[k].begin(), by_kind[k].end());
    double together = 1e30;
    const bool mixed = !by_kind[HALF].empty() && both.size() > by_kind[HALF].size();
    const long long joint = mixed ? chunk_length(both, g, HALF, together) : 0;
    if (mixed) together = std::max(together, mixed_least(both, g, joint));
    const double apart = std::min(half, many) + few_cost(by_kind[FEW], g, length[FEW]) + few_cost(by_kind[SOME], g, length[SOME]);
    if (mixed && together <= apart) {
        for (Tile& t : both) t.kind = HALF;
        by_kind[HALF] = std::move(both);
        length[HALF] = joint;
        cut[HALF] = 0;
        for (int k : {FEW, SOME, MANY}) by_kind[k].clear();
    } else {
        by_kind[half <= many ? MANY : HALF].clear();
    }
    std::vector<Tile> tiles;
    std::vector<long long> most;  // KEYS of a piece of the tile
    for (int k = 0; k < KINDS; k++)
        for (int i = 0; i < (int)by_kind[k].size(); i++) {
            tiles.push_back(by_kind[k][i]);
            most.push_back(cut[k] ? i < cut[k] ? piece[k] : 1 << 20 : length[k]);
        }
    int part = 0, more = 0;  // partials and work items that splits have taken
    for (size_t i = 0; i < tiles.size(); i++) {
        const Tile& t = tiles[i];
        const Member& m = batch[t.member];
        const int rows = m.count * group, count = std::min(TILE_ROWS[t.kind], rows - t.row0);
        const int units = (t.k1 - t.k0 + KEYS - 1) / KEYS;
        int splits = std::min(pieces_of(t, most[i]), splits_room(count, g.kv_heads, part, more));
        if (splits < 2) splits = 1;
        more += (splits - 1) * g.kv_heads;
        for (int head = 0; head < g.kv_heads; head++) {
            for (int s = 0; s < splits; s++) {
                const int a = t.k0 + (int)((long long)units * s / splits) * KEYS;
                const int b = s + 1 < splits ? t.k0 + (int)((long long)units * (s + 1) / splits) * KEYS : t.k1;
                out.items[t.kind].push_back({m.seq, head, t.tok0, t.row0, rows, m.len - m.count, a, b,
                                             splits > 1 ? part + s * count : -1, s, {0, 0}});
            }
            if (splits > 1) {
                out.joins.push_back({head, t.tok0, t.row0, count, part, splits, 0, 0});
                part += splits * count;
            }
        }
    }
    // Many splits of few rows are read by many work-groups at once; of many rows the rows are work enough (3,200 rows of 9
    // splits by 64 dims each: 45 us, row by row 14).
    long long rows = 0;
    for (const Join& j : out.joins) rows += j.count;
    for (Join& j : out.joins) j.wide = j.splits > WIDE_SPLITS && rows <= WIDE_ROWS;
    for (auto& list : out.items) {
        std::stable_sort(list.begin(), list.end(), [](const Item& a, const Item& b) {
            return a.seq != b.seq ? a.seq < b.seq : a.head != b.head ? a.head < b.head : a.split < b.split;
        });
        deal(list);
    }
}

}  // namespace paged
}  // namespace mkv
