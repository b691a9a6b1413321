// The work of the attention over a batch (fa_batch.hip): which rows and keys each
// work-group takes. Plain arithmetic on the batch's lengths, used by the kernels
// and by the launcher, and compiled for the host by its tests.
#pragma once

#include <limits.h>

#include <algorithm>

#include "fa_cache.h"
#include "fa_device.h"

namespace mxfa {

constexpr int kBatchFew = 16;  // rows of the few-row form's units
constexpr int kCusPerXcd = 32;  // of 8 XCDs
// Rows of a work-group of the join: as many of the many-row form's as it has
// groups of D / 4 threads; a quarter of the few-row form's, whose sequences may be
// in a hundred pieces.
__host__ __device__ constexpr int join_rows(int d) { return 1024 / d; }
constexpr int kFewJoins = 4;
// Waves of the few-row form's work-groups over a microscaled cache.
constexpr int kMxFewWaves = 8;
// Waves of the many-row form's work-groups in fp32, of 16 rows each (bf16: 4, of 16
// or 32: batch_many_rows).
constexpr int kBatchF32Waves = 8;

// The workspace holds the shares of split units: `slots` of them, each ROWS rows
// of D floats and their (max, sum) pairs; then what the join reads about them,
// `notes` ints.
__host__ __device__ constexpr size_t batch_slot_floats(long long slots, int rows, int d) {
    return (size_t)slots * rows * (d + 2);
}
// The join's notes. Few rows: per work-group the pieces of the sequence that its
// run ends in (0: none), its rows and first position. Many rows: the count of split
// units, then each.
struct FewNote {
    int parts, q0, rows, pos;
};
struct ManyNote {
    int shares, slot, q0, rows, unit, head, pos[2];  // (pos[1]: to 32 bytes)
};

template <class X>
__host__ __device__ inline X less_of(X a, X b) {
    return a < b ? a : b;
}
template <class X>
__host__ __device__ inline X more_of(X a, X b) {
    return a < b ? b : a;
}

// What a sequence brings to a form.
struct BatchSeq {
    int q0;      // its first row of q
    int pos;     // position of that row's token
    int rows;    // new tokens x query heads per KV head (0: none for this form)
    int keys;    // positions that its last token sees
    int units, stages;  // units, and stages of the last one, which has the most
};

template <bool FEW, int ROWS>  // (FEW: ROWS = kBatchFew, one unit)
__host__ __device__ inline BatchSeq batch_seq(const BatchParams &p, int s) {
    BatchSeq b{0, 0, 0, 0, 0, 0};
    if (s >= p.n_seq) return b;
    const int c0 = p.cu_q[s], c1 = p.cu_q[s + 1], len = p.lens[s];
    b.q0 = less_of(more_of(c0, 0), p.n_tok);
    const int count = less_of(less_of(more_of(c1, b.q0), p.n_tok) - b.q0, p.max_q);
    const long long rows = (long long)count * p.group;
    const bool mine = FEW ? rows <= p.few_rows : rows > p.few_rows;
    if (!mine || count == 0) return b;
    b.rows = (int)rows;
    // positions stay within int with a stage to spare, whatever the arrays hold
    const long long cap = less_of((long long)p.max_blocks << p.bs_shift, (long long)INT_MAX - 256);
    const long long pos = (long long)len - ((long long)c1 - b.q0);
    b.pos = (int)less_of(more_of(pos, -(1LL << 30)), cap);
    b.keys = (int)more_of(less_of(less_of((long long)b.pos + count, (long long)len), cap), 0LL);
    b.units = (int)((rows + ROWS - 1) / ROWS);
    b.stages = (b.keys + 63) / 64;
    return b;
}

// ---- the few-row form. The sequences' stages, and one more for each sequence,
// lie on a line in their order (the extra one first: it stands for what a
// piece costs besides its stages, and gives a sequence without keys a place). A
// KV head's p.few_groups work-groups cut the line into equal runs, so all have
// the same work; a sequence that a cut goes through is in pieces, which the
// join puts together. A work-group has two slots of the workspace: one for a
// piece that its run ends in, one for a piece that its run begins in or is in.
__host__ __device__ inline unsigned few_weight(const BatchSeq &b) { return b.rows > 0 ? (unsigned)b.stages + 1u : 0u; }
// The run of each work-group, of a line of `all`.
__host__ __device__ inline unsigned few_run(const BatchParams &p, unsigned all) {
    return more_of((all + (unsigned)p.few_groups - 1) / (unsigned)p.few_groups, (unsigned)p.least[0]);
}
struct FewPiece {
    int lo, hi;   // stages
    int slot;     // -1: all of the sequence's stages, finished in place
    unsigned end; // where the next piece begins
};
// The piece of the sequence at [u0, u1) of the line that work-group g (of all KV
// heads') has from x on, its run ending at x1.
__host__ __device__ inline FewPiece few_piece(unsigned x, unsigned x1, unsigned u0, unsigned u1, int g) {
    FewPiece f;
    f.end = less_of(x1, u1);
    f.lo = (int)(x > u0 ? x - u0 - 1 : 0);
    f.hi = (int)(f.end - u0 - 1);
    f.slot = x > u0 ? 2 * g : f.end < u1 ? 2 * g + 1 : -1;
    return f;
}
// The pieces of the sequence at [u0, u1).
__host__ __device__ inline int few_parts(unsigned run, unsigned u0, unsigned u1) {
    return (int)((u1 - 1) / run - u0 / run) + 1;
}
// The slots of a sequence's pieces, by the run it begins in: the first piece's
// and then one each 2 Hkv on from the second's.
__host__ __device__ inline int few_first_slot(int run, int heads, int head) { return 2 * (run * heads + head) + 1; }
__host__ __device__ inline int few_next_slot(int run, int heads, int head) { return 2 * ((run + 1) * heads + head); }

// ---- the many-row form.

// About the stages of all its units: those of the first and of the last one
// each count for half of them.
template <int ROWS>
__host__ __device__ inline float seq_stages(const BatchParams &p, const BatchSeq &b) {
    const int last = more_of(b.stages, 1);
    const int tokens = (int)((unsigned)less_of(ROWS, b.rows) / (unsigned)p.group);
    const int first = less_of(more_of((b.pos + tokens + 63) / 64, 1), last);
    return (float)b.units * 0.5f * (float)(first + last);
}

// A sequence's items at a quota, the most stages of a share: its first `whole`
// units are whole items, the others are cut into `shares` each. Counts over all
// KV heads: `split` units that are cut, their `slots` shares, and all items.
struct SeqItems {
    int whole, shares, split, slots, items;
};
template <int ROWS>
__host__ __device__ inline SeqItems seq_items(const BatchParams &p, const BatchSeq &b, unsigned quota) {
    SeqItems n{b.units, 1, 0, 0, 0};
    if (b.units > 0 && (unsigned)b.stages > quota) {
        n.shares = (int)(((unsigned)b.stages + quota - 1) / quota);
        // unit u ends with row (u + 1) ROWS - 1, which sees more than 64 quota
        // positions from row t group on, t = 64 quota - pos; the last one does
        const long long t = 64LL * quota - b.pos;
        n.whole = t <= 0 ? 0 : (int)less_of((unsigned long long)t * (unsigned)p.group / ROWS, (unsigned long long)(b.units - 1));
    }
    n.split = (b.units - n.whole) * p.Hkv;
    n.slots = n.split * n.shares;
    n.items = n.whole * p.Hkv + n.slots;
    return n;
}

// The quota, from the sums of seq_stages and of the units over the sequences (of
// one KV head), the count of all items at a quota, and whether a sequence has
// more stages than a number. It is about the least one, up to two even shares, by
// which all shares fit the work-groups that are resident at once (p.resident), found
// by raising an even share's; without one, one and a half even shares, if the launch
// has room for those (p.roomy; else the search goes on). INT_MAX: no split. It depends
// on lengths alone.
//
// A split costs a join of about p.whole stages' time and p.per_item stages' for
// each share's part written and read again; where the longest unit is over a
// share's by no more, all units stay whole. us, whole and split: bf16, 14/2 heads,
// 4 chunks of 700 tokens after 700 32 and 39, one of 500 after 1500 31 and 23,
// 1000 tokens 19 and 21; 32/8 heads, d = 128, 1000 tokens 27 and 35; fp32, 14/2
// heads, 500 tokens 28 and 29, 1000 51 and 35.
constexpr float kManySplit = 1.5f;
template <class Count, class Longer>
__host__ __device__ inline unsigned batch_quota(const BatchParams &p, float all, float units, Count count, Longer longer) {
    if (p.slots == 0) return INT_MAX;
    all = less_of(all * (float)p.Hkv * 1.001f, 1e18f);  // (more than its rounding)
    const float resident = (float)p.resident, even = less_of(all * p.per_resident + 1.0f, 1e8f);
    const float least = (float)p.least[1];
    auto worth = [&](unsigned q, float items) {
        return longer(q + p.whole + (unsigned)(p.per_item * items)) ? q : (unsigned)INT_MAX;
    };
    unsigned q = (unsigned)more_of(even, least);
    for (int i = 0; i < 12 && units * (float)p.Hkv <= resident; ++i) {
        const float items = count(q);
        if (items <= resident) return worth(q, items);
        q = (unsigned)more_of((float)q * 1.125f + 1.0f, (float)q * items * p.per_resident);
        if (p.roomy && (float)q > 2.0f * even) break;
    }
    if (!p.roomy) return INT_MAX;
    q = (unsigned)more_of(kManySplit * even, least);
    return worth(q, count(q));
}

struct BatchItem {
    BatchSeq s;
    int seq, head, unit, share, shares;
    int slot;   // of this share, where shares > 1
    int split;  // the unit's number among the split ones
};

// Item i of a sequence whose shares' slots begin at `slot` and split units at
// `split`. Items: the split units (the last, heaviest one first) x shares x KV
// heads, then the whole ones x KV heads, so that neighbouring work-groups, which
// the dispatcher spreads over the XCDs, have the heads and an XCD's share of
// them the same head's keys. False where the share has no slot, which only a
// cu_q that gives rows to several sequences can bring about.
__host__ __device__ inline bool batch_item(const BatchParams &p, const SeqItems &n, int slot, int split, int item,
                                           BatchItem &it) {
    const unsigned heads = p.Hkv;
    unsigned i = item;
    it.share = it.split = 0;
    it.shares = n.shares;
    it.slot = slot + item;
    if (i >= (unsigned)n.slots) {
        i -= n.slots;
        it.shares = 1;
        it.unit = n.whole - 1 - (int)(i / heads);
        it.head = i % heads;
        return true;
    }
    const unsigned per_unit = i / heads;
    it.head = i - per_unit * heads;
    const unsigned u = per_unit / (unsigned)n.shares;
    it.share = per_unit - u * n.shares;
    it.unit = it.s.units - 1 - (int)u;
    it.split = split + (int)(u * heads) + it.head;
    return it.slot < p.slots;
}

// The item of the many-row form's work-group `block`, in the order by which a CU's
// resident ones have long and short units (cu_order_wg); neighbours in eights
// (the XCDs) stay together. It permutes the resident ones: a launch of more than
// one a CU has them all (batch_many_form).
__host__ __device__ inline int batch_order(const BatchParams &p, int block) {
    return cu_order_wg(block >> 3, kCusPerXcd, p.resident / (8 * kCusPerXcd)) * 8 + (block & 7);
}

// Whether a note of the join is one that find_item's items write (whatever the
// workspace holds where none was written).
__host__ __device__ inline bool note_holds(const BatchParams &p, const ManyNote &n) {
    return n.shares > 1 && n.slot >= 0 && (long long)n.slot + (long long)(n.shares - 1) * p.Hkv < p.slots && n.q0 >= 0 &&
           n.rows > 0 && n.q0 + (long long)(n.rows - 1) / p.group < p.n_tok && n.unit >= 0 &&
           (long long)n.unit * p.many_rows < n.rows && n.head >= 0 && n.head < p.Hkv;
}

// The share's stages of the unit's n.
__host__ __device__ inline void share_stages(const BatchItem &it, int n, int &lo, int &hi) {
    // n < 2^25 stages and at most 2^11 shares: the products pass 32 bits
    if (it.shares == 1) {
        lo = 0;
        hi = n;
    } else {
        lo = (int)((unsigned long long)(unsigned)it.share * (unsigned)n / (unsigned)it.shares);
        hi = (int)((unsigned long long)(unsigned)(it.share + 1) * (unsigned)n / (unsigned)it.shares);
    }
}

// ---- the launcher's side

// Work-groups resident at once: the few-row form's have a CU each, the many-row
// form's share one in twos, threes or fours (the kernels' registers and LDS).
constexpr int kBatchCus = 256;
inline int batch_resident(int dtype_bf16, int d, int rows, bool both) {
    return kBatchCus * (!dtype_bf16 || d == 128 ? 2 : rows == 64 && !both ? 4 : 3);
}

// Which forms a call launches, by what the host knows: the few-row form alone
// where no sequence can have more rows; the many-row form alone where one
// sequence has the rows; else both, each taking its own sequences.
inline int batch_few_rows(const BatchParams &p) {
    const bool may_exceed = (long long)p.max_q * p.group > kBatchFew;
    return may_exceed && p.n_seq == 1 ? 0 : kBatchFew;
}
inline bool batch_may_be_many(const BatchParams &p) {
    return (long long)less_of(p.max_q, p.n_tok) * p.group > kBatchFew || p.few_rows == 0;
}

// Units of the many-row form at most.
inline long long batch_units(const BatchParams &p, int rows) {
    return ((long long)p.n_tok * p.group / rows + less_of(p.n_seq, p.n_tok)) * p.Hkv;
}

// Whether most sequences are of few rows, by what the host knows: the others have
// max_q tokens at most.
inline bool batch_mostly_few(const BatchParams &p) {
    if (p.few_rows == 0) return false;
    const long long few_tok = p.few_rows / p.group;
    return 2 * (more_of((long long)p.n_tok - p.n_seq * few_tok, 0LL) / p.max_q) < p.n_seq;
}

// Stages that a sequence has at most, by its table.
inline long long batch_most_stages(const BatchParams &p) { return (((long long)p.max_blocks << p.bs_shift) + 63) / 64; }

// Rows of its units (bf16: 4 waves of 16 or of 32). 32 a wave halve the LDS reads of
// K and V for each product, 16 give twice the work-groups: taken where units of 128
// rows are at most one and a half (d = 128: one) per CU. us, by 64 and by 128 rows:
// 14/2 heads, 1000 tokens 14 and 19, 2000 25 and 34, 4 chunks of 700 after 700 28 and
// 33, 8 of 512 after 3584 111 and 92; 32/8 heads, d = 128, 1000 tokens 23 and 28,
// 2 chunks of 1000 after 2000 134 and 106. Beside the few-row form's work-groups, which
// leave a CU room for two more of either, 128: 4 chunks and 28 tokens 58 and 52.
//
// Over a microscaled cache, whose keys each work-group converts, 64 rows also cost
// twice the conversions, and where there are stages enough to share out a unit's keys
// fill the CUs as well: 128 where a row of the longest chunk sees more than 20 stages
// on average. us, 4 bits, by 64 and by 128 rows: 14/2 heads, d = 64, 2000 tokens from
// the start (16) 29 and 33, 4 chunks of 700 to 1400 (16) 29 and 34, 1000 to 2048 (24) 31
// and 28, 4 of 512 to 8192 (124) 137 and 95; 32/8 heads, d = 128, 500 to 1000 (12) 24 and 30,
// 500 to 2048 (28) 45 and 38, to 8192 112 and 82.
inline int batch_many_rows(const BatchParams &p, int dtype_bf16) {
    if (!dtype_bf16) return 16 * kBatchF32Waves;
    if (p.bits != 0 && 2 * batch_most_stages(p) - less_of(p.max_q, p.n_tok) / 64 > 40) return 128;
    return !batch_mostly_few(p) && batch_units(p, 128) <= (p.d == 64 ? 3 * kBatchCus / 2 : kBatchCus) ? 64 : 128;
}

// A form's launch: its work-groups and the join's, and the workspace's slots.
struct BatchForm {
    int rows;
    long long groups, joins, slots, notes;
};

// Few rows: a CU's work-group for each run of the line, at least one per KV head;
// no more than give each `least` stages of the longest line there can be.
inline BatchForm batch_few_form(BatchParams *p) {
    const long long line = less_of(p->n_seq, p->n_tok) * (batch_most_stages(*p) + 1);
    const long long each = more_of(kBatchCus / p->Hkv, 1);
    p->few_groups = (int)less_of(each, (line + p->least[0] - 1) / p->least[0]);
    BatchForm f;
    f.rows = kBatchFew;
    f.groups = (long long)p->few_groups * p->Hkv;
    // a cut between each two runs
    f.joins = p->few_groups > 1 ? f.groups - p->Hkv : 0;
    f.slots = f.joins > 0 ? 2 * f.groups : 0;
    f.notes = f.joins > 0 ? f.groups * (long long)(sizeof(FewNote) / sizeof(int)) : 0;
    return f;
}

// Many rows. The units are full but for a sequence's last. Where they are up to
// half of the resident work-groups, all items fit those, the shares of split units
// among them. Else the quota may be at least one and a half even shares, and find_item's sum of
// stages at least half of units x the last one's in each sequence: then the
// shares of split units, ceil(last one's / quota) each, are at most 4/3 of the
// resident + the split units, those at most 4/3 of the resident and the units.
inline BatchForm batch_many_form(BatchParams *p, int dtype_bf16) {
    BatchForm f;
    f.rows = p->many_rows;
    p->roomy = 0;
    p->resident = batch_resident(dtype_bf16, p->d, p->many_rows, p->few_rows > 0);
    // Beside the few-row form's work-groups a CU holds two of these. us, 14/2 heads,
    // d = 64: 4 chunks and 28 tokens 57.6 (61 by three a CU); 8 chunks 84 by three
    // (104 by two)
    if (batch_mostly_few(*p)) p->resident = 2 * kBatchCus;
    p->per_resident = 1.0f / (float)p->resident;
    const long long units = batch_units(*p, f.rows);
    const long long more = (long long)p->resident * 4 / 3 + 1;
    // nothing is split, and no join launched, where batch_quota would hardly ever
    // find it worth it: some 3 shares of a unit
    const float shares = 3.0f * (float)less_of(units, (long long)p->resident / 2);
    if ((float)batch_most_stages(*p) <= (float)(p->least[1] + p->whole) + p->per_item * shares) {
        f.groups = units <= kBatchCus ? units : more_of(units, (long long)p->resident);  // (batch_order)
        f.joins = f.slots = 0;
    } else {
        p->roomy = units > p->resident / 2;
        f.groups = p->roomy ? units + more : p->resident;
        const long long split = less_of(units, more);
        f.slots = p->roomy ? more + split : p->resident;
        f.joins = split;
    }
    p->slots = (int)f.slots;
    p->splits = (int)f.joins;
    f.notes = f.joins > 0 ? (f.joins + 1) * (long long)(sizeof(ManyNote) / sizeof(int)) : 0;
    return f;
}

// The least stages of a share or run: one for each of the few-row form's waves; 4
// of the many-row form's.
inline void batch_plan(BatchParams *p, int dtype_bf16) {
    p->few_rows = batch_few_rows(*p);
    p->many_rows = batch_many_rows(*p, dtype_bf16);
    p->least[0] = p->bits != 0 ? kMxFewWaves : dtype_bf16 && p->d == 64 ? 8 : 4;
    p->least[1] = 4;
    p->whole = dtype_bf16 ? 6 : 4;
    p->per_item = dtype_bf16 ? 0.024f : 0.007f;
}

// The forms of a call; groups = 0: not launched. many_rows: 0, or other units than its own.
inline void batch_forms(BatchParams *p, int dtype_bf16, BatchForm (&f)[2], int many_rows = 0) {
    batch_plan(p, dtype_bf16);
    if (many_rows > 0) p->many_rows = many_rows;
    f[0] = f[1] = BatchForm{0, 0, 0, 0, 0};
    if (p->few_rows > 0) f[0] = batch_few_form(p);
    if (batch_may_be_many(*p)) f[1] = batch_many_form(p, dtype_bf16);
}

}  // namespace mxfa
