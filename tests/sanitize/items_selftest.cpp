// Host-side checks of the items that the attention over a batch is cut into
// (mx230_amd/csrc/fa_batch_items.h), under AddressSanitizer and
// UndefinedBehaviorSanitizer; nothing touches a device. Exit status 0 = all
// checks passed.
//  * Sensible batches, many rows: every unit of every sequence and head is an
//    item, or all its shares are, once each; shares cover the unit's stages; the
//    slots of split units are inside the workspace and nobody else's; the join's
//    items are the split units; the launch's work-groups are enough for all.
//  * Few rows: the work-groups' pieces cover every sequence's stages once, none
//    has more than its run; the slots of a sequence in pieces are those its join
//    reads, nobody else's; every such sequence is joined once.
//  * Arrays that hold anything: rows, positions, heads, units and slots of every
//    item that is found lie inside the buffers.
#include <algorithm>
#include <cstdio>
#include <cstring>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>

#include "../../mx230_amd/csrc/fa_batch_items.h"

using namespace mxfa;

static int g_fail = 0;
#define CHECK(cond, ...)                                              \
    do {                                                              \
        if (!(cond)) {                                                \
            if (g_fail < 20) {                                        \
                std::fprintf(stderr, "FAIL %s:%d: ", __FILE__, __LINE__); \
                std::fprintf(stderr, __VA_ARGS__);                    \
                std::fputc('\n', stderr);                             \
            }                                                         \
            ++g_fail;                                                 \
        }                                                             \
    } while (0)

// find_item of the kernels with a loop in the place of a wave, and the count of
// split units.
template <int ROWS>
static bool find(const BatchParams &p, int w, BatchItem &it, int *total = nullptr) {
    float all = 0, units = 0;
    for (int s = 0; s < p.n_seq; ++s) {
        const BatchSeq b = batch_seq<false, ROWS>(p, s);
        all += seq_stages<ROWS>(p, b);
        units += (float)b.units;
    }
    auto count = [&](unsigned q) {
        int n = 0;
        for (int s = 0; s < p.n_seq; ++s) n += seq_items<ROWS>(p, batch_seq<false, ROWS>(p, s), q).items;
        return (float)n;
    };
    auto longer = [&](unsigned x) {
        for (int s = 0; s < p.n_seq; ++s) {
            if ((unsigned)batch_seq<false, ROWS>(p, s).stages > x) return true;
        }
        return false;
    };
    const unsigned quota = batch_quota(p, all, units, count, longer);
    int before = 0, slots = 0, splits = 0;
    bool found = false;
    for (int s = 0; s < p.n_seq; ++s) {
        const BatchSeq b = batch_seq<false, ROWS>(p, s);
        const SeqItems n = seq_items<ROWS>(p, b, quota);
        if (w >= before && w < before + n.items) {
            it.seq = s;
            it.s = b;
            found = batch_item(p, n, slots, splits, w - before, it);
            if (total == nullptr) return found;
        }
        before += n.items;
        slots += n.slots;
        splits += n.split;
    }
    if (total != nullptr) *total = splits;
    return found;
}

static void check_bounds(const BatchParams &p, const BatchForm &f, const BatchItem &it) {
    const long long cap = ((long long)p.max_blocks) << p.bs_shift;
    CHECK(it.seq >= 0 && it.seq < p.n_seq && it.head >= 0 && it.head < p.Hkv, "seq %d head %d", it.seq, it.head);
    CHECK(it.s.rows > 0 && it.unit >= 0 && it.unit < it.s.units && (long long)it.unit * f.rows < it.s.rows,
          "unit %d of %d, %d rows", it.unit, it.s.units, it.s.rows);
    CHECK(it.s.q0 >= 0 && it.s.q0 + (long long)(it.s.rows - 1) / p.group < p.n_tok, "rows %d from %d of %d", it.s.rows,
          it.s.q0, p.n_tok);
    CHECK(it.s.keys >= 0 && it.s.keys <= cap, "keys %d of %lld", it.s.keys, cap);
    CHECK((long long)it.s.pos + it.s.rows / p.group + 1 < INT_MAX, "position %d", it.s.pos);
    CHECK(it.shares >= 1 && it.share >= 0 && it.share < it.shares, "share %d of %d", it.share, it.shares);
    if (it.shares > 1) CHECK(it.slot >= 0 && it.slot < f.slots, "slot %d of %lld", it.slot, f.slots);
}

template <int ROWS>
static void check_many(BatchParams p, int bf16, bool sound) {
    const BatchForm f = batch_many_form(&p, bf16);
    const long long groups = f.groups;
    std::map<std::tuple<int, int, int>, std::vector<BatchItem>> units;
    std::set<int> slots;
    const long long step = sound ? 1 : std::max(1LL, groups / 400);
    for (long long w = 0; w < groups; w += step) {
        BatchItem it{};
        if (!find<ROWS>(p, batch_order(p, (int)w), it)) continue;
        check_bounds(p, f, it);
        int lo, hi;
        share_stages(it, it.s.stages, lo, hi);
        CHECK(lo >= 0 && lo <= hi && hi <= it.s.stages, "stages %d..%d of %d", lo, hi, it.s.stages);
        if (!sound) continue;
        units[{it.seq, it.head, it.unit}].push_back(it);
        if (it.shares > 1) CHECK(slots.insert(it.slot).second, "slot %d twice", it.slot);
    }
    const long long joins = f.joins;
    if (!sound) {
        // what a note may hold is checked before it is used
        std::mt19937 r(3);
        for (int i = 0; i < 2000; ++i) {
            ManyNote n;
            for (int *x = &n.shares; x < &n.shares + 8; ++x) {
                const int k = (int)(r() % 4);
                *x = k == 0 ? (int)r() : k == 1 ? (int)(r() % 300) : k == 2 ? 0 : INT_MAX;
            }
            if (!note_holds(p, n)) continue;
            CHECK(n.slot >= 0 && n.slot + (n.shares - 1LL) * p.Hkv < f.slots, "slots %d + %d", n.slot, n.shares);
            CHECK(n.q0 >= 0 && n.q0 + (long long)(n.rows - 1) / p.group < p.n_tok, "rows %d from %d", n.rows, n.q0);
        }
        return;
    }
    BatchItem past{};
    size_t want = 0, split = 0;
    for (int s = 0; s < p.n_seq; ++s) want += (size_t)batch_seq<false, ROWS>(p, s).units * p.Hkv;
    CHECK(units.size() == want, "%zu units of %zu", units.size(), want);
    int total = 0;
    find<ROWS>(p, 0, past, &total);
    CHECK(total <= joins, "%d split units, %lld joins", total, joins);
    std::map<int, BatchItem> joined;  // by number: what share 0 notes
    for (auto &[key, v] : units) {
        for (auto &x : v) {
            if (x.shares < 2 || x.share != 0) continue;
            CHECK(x.split >= 0 && x.split < total, "split unit %d of %d", x.split, total);
            CHECK(joined.emplace(x.split, x).second, "split unit %d twice", x.split);
            const ManyNote n{x.shares, x.slot, x.s.q0, x.s.rows, x.unit, x.head, {0, 0}};
            CHECK(note_holds(p, n), "the note of split unit %d", x.split);
        }
    }
    CHECK((int)joined.size() == total, "%zu joins for %d split units", joined.size(), total);
    for (auto &[key, v] : units) {
        const BatchItem &a = v[0];
        CHECK((int)v.size() == a.shares, "%zu of %d shares", v.size(), a.shares);
        int end = 0;
        for (int i = 0; i < (int)v.size(); ++i) {
            const BatchItem *s = nullptr;
            for (auto &x : v) {
                if (x.share == i) s = &x;
            }
            CHECK(s != nullptr, "share %d is missing", i);
            if (s == nullptr) continue;
            int lo, hi;
            share_stages(*s, s->s.stages, lo, hi);
            CHECK(lo == end, "share %d from %d, not %d", i, lo, end);
            end = hi;
            if (a.shares > 1 && i == 0) {
                ++split;
            }
        }
        CHECK(end == a.s.stages, "stages to %d of %d", end, a.s.stages);
        for (auto &x : v) {
            const BatchItem *first = &v[0];
            for (auto &y : v) {
                if (y.share == 0) first = &y;
            }
            if (a.shares > 1) CHECK(x.slot == first->slot + x.share * p.Hkv, "slots %d and %d", first->slot, x.slot);
        }
    }
    CHECK(joined.size() == split, "%zu joins for %zu split units", joined.size(), split);
}

// The few-row form as its kernels walk its line (and the join its cuts).
static void check_few(BatchParams p, bool sound) {
    const BatchForm f = batch_few_form(&p);
    std::vector<BatchSeq> seq;
    std::vector<unsigned> u{0};
    for (int s = 0; s < p.n_seq; ++s) {
        seq.push_back(batch_seq<true, kBatchFew>(p, s));
        u.push_back(u.back() + few_weight(seq.back()));
        const BatchSeq &b = seq.back();
        CHECK(b.rows >= 0 && b.rows <= kBatchFew && (b.rows == 0 || b.units == 1), "%d rows", b.rows);
        if (b.rows == 0) continue;
        const BatchItem it{b, s, 0, 0, 0, 1, 0};
        check_bounds(p, f, it);
    }
    const unsigned all = u.back(), run = few_run(p, all);
    CHECK((unsigned long long)run * p.few_groups >= all, "%d runs of %u on a line of %u", p.few_groups, run, all);
    std::map<std::pair<int, int>, std::vector<FewPiece>> pieces;  // (sequence, head)
    std::map<int, std::pair<int, int>> owner;
    for (int g = 0; g < f.groups; ++g) {
        const int head = g % p.Hkv;
        unsigned x = (unsigned)(g / p.Hkv) * run;
        const unsigned x1 = std::min(x + run, all);
        int stages = 0;
        for (int s = 0; s < p.n_seq && x < x1; ++s) {
            if (u[s + 1] == u[s] || u[s + 1] <= x) continue;
            const FewPiece c = few_piece(x, x1, u[s], u[s + 1], g);
            CHECK(c.lo >= 0 && c.lo <= c.hi && c.hi <= seq[s].stages, "stages %d..%d of %d", c.lo, c.hi, seq[s].stages);
            CHECK(c.end > x && c.end <= x1, "a piece from %u to %u", x, c.end);
            if (c.slot >= 0) {
                CHECK(c.slot < f.slots, "slot %d of %lld", c.slot, f.slots);
                CHECK(owner.emplace(c.slot, std::make_pair(s, head)).second, "slot %d twice", c.slot);
            }
            pieces[{s, head}].push_back(c);
            stages += c.hi - c.lo;
            x = c.end;
        }
        CHECK(stages <= (int)run, "%d stages in a run of %u", stages, run);
    }
    std::map<std::pair<int, int>, int> joined;
    for (int j = 0; j < f.joins; ++j) {
        const int cut = j / p.Hkv, head = j % p.Hkv;
        const unsigned long long x = (unsigned long long)(cut + 1) * run;
        // the note of work-group j: the sequence its run ends in, if it begins there
        if (x >= all) continue;
        int s = 0;
        while (u[s + 1] <= x) ++s;
        if (u[s] >= x || u[s] / run != (unsigned)cut) continue;
        const int S = few_parts(run, u[s], u[s + 1]);
        ++joined[{s, head}];
        const auto &v = pieces[{s, head}];
        CHECK((int)v.size() == S, "%zu pieces, the join reads %d", v.size(), S);
        for (int i = 0; i < S && i < (int)v.size(); ++i) {
            const int at = i == 0 ? few_first_slot(cut, p.Hkv, head) : few_next_slot(cut, p.Hkv, head) + 2 * p.Hkv * (i - 1);
            CHECK(v[i].slot == at, "piece %d in slot %d, the join reads %d", i, v[i].slot, at);
        }
    }
    if (!sound && all == 0) return;
    for (int s = 0; s < p.n_seq; ++s) {
        if (seq[s].rows == 0) continue;
        for (int h = 0; h < p.Hkv; ++h) {
            const auto &v = pieces[{s, h}];
            int end = 0;
            for (const FewPiece &c : v) {
                CHECK(c.lo == end, "a piece from stage %d, not %d", c.lo, end);
                end = c.hi;
            }
            CHECK(!v.empty() && end == seq[s].stages, "stages to %d of %d", end, seq[s].stages);
            CHECK((v.size() == 1) == (v.empty() || v[0].slot < 0), "%zu pieces, slot %d", v.size(), v.empty() ? 0 : v[0].slot);
            CHECK((joined[{s, h}]) == (v.size() > 1 ? 1 : 0), "%zu pieces joined %d times", v.size(), (joined[{s, h}]));
        }
    }
}

int main() {
    std::mt19937 r(7);
    auto pick = [&](int lo, int hi) { return (int)(lo + r() % (unsigned)(hi - lo + 1)); };
    const int ends[] = {INT_MIN, -(1 << 30), -1, 0, 1, 63, 64, 65, 1 << 20, INT_MAX - 1, INT_MAX};
    for (int t = 0; t < 900; ++t) {
        const bool sound = t % 3 != 0;
        BatchParams p{};
        const int bf16 = pick(0, 2) > 0;
        p.d = bf16 && pick(0, 1) ? 128 : 64;
        p.Hkv = (int[]){1, 2, 3, 8}[pick(0, 3)];
        p.group = (int[]){1, 4, 7, 8, 16, 17, 40}[pick(0, 6)];
        p.Hq = p.Hkv * p.group;
        p.n_seq = pick(0, 2) ? pick(1, 12) : pick(1, 150);
        p.bs_shift = (int[]){0, 4, 7}[pick(0, 2)];
        std::vector<int> cu{0}, lens;
        const int longest = (int[]){70, 700, 5000, 70000}[pick(0, 3)], chunk = (int[]){1, 2, 40, 700}[pick(0, 3)];
        int most = 1;
        for (int s = 0; s < p.n_seq; ++s) {
            const int n = pick(0, 3) == 0 ? pick(0, chunk) : pick(0, 1);
            cu.push_back(cu.back() + n);
            lens.push_back(pick(0, 9) == 0 ? pick(0, 3) : std::max(n, pick(1, longest)));
            most = std::max(most, n);
        }
        p.n_tok = cu.back() + pick(0, 3);
        if (p.n_tok == 0) p.n_tok = 1;
        p.max_q = most + pick(0, 1);
        p.max_blocks = (longest >> p.bs_shift) + 1;
        p.table_stride = p.max_blocks;
        p.n_blocks = 10;
        if (!sound) {
            if (pick(0, 1)) p.max_q = pick(0, 1) ? INT_MAX : pick(1, 50);
            if (pick(0, 1)) p.max_blocks = pick(1, 40);
            for (int &x : cu) {
                if (pick(0, 3) == 0) x = pick(0, 1) ? ends[pick(0, 10)] : pick(0, p.n_tok);
            }
            for (int &x : lens) {
                if (pick(0, 2) == 0) x = ends[pick(0, 10)];
            }
        }
        p.cu_q = cu.data();
        p.lens = lens.data();
        batch_plan(&p, bf16);
        if (p.few_rows > 0) check_few(p, sound);
        if (batch_may_be_many(p)) {
            if (p.many_rows == 64) check_many<64>(p, bf16, sound);
            else check_many<128>(p, bf16, sound);
        } else if (sound) {
            for (int s = 0; s < p.n_seq; ++s) CHECK((batch_seq<false, 64>(p, s).rows == 0), "rows that no form takes");
        }
    }
    if (g_fail == 0) std::printf("items: all checks passed\n");
    return g_fail == 0 ? 0 : 1;
}
