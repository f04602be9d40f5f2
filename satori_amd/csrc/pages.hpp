// Host bookkeeping of a paged key/value cache that sequences share, and the plan of one batch over it: which page
// holds what, which tokens several rows have in common, and how their attention is cut into workgroups. Plain C++
// without device calls; the device code reads the plan's image (PlanHeader and the arrays behind it).
#pragma once

#include <cstdint>
#include <shared_mutex>
#include <vector>

struct satori_hip_pages;

namespace satori {

struct PageMove {
    int source, destination;
};

inline bool valid_page_tokens(int n) { return n == 32 || n == 64 || n == 128 || n == 256; }

// Reference-counted pages of `page_tokens` positions and the sequences that hold them. Every change is all or nothing:
// a call that fails leaves everything as it was. New pages and sequence numbers are the lowest free ones, so that the
// same calls always give the same tables.
class PageTables {
public:
    PageTables(int pages, int page_tokens);

    int open();
    // Makes room for tokens[i] more positions of sequences[i] that nobody else sees: a last page that is part full and
    // shared is replaced by a copy of its own (a move), and pages are added behind it.
    void extend(const int* sequences, const int* tokens, int count, std::vector<PageMove>& moves);
    void truncate(int sequence, int tokens);
    // `count` sequences that hold the same pages.
    void fork(int sequence, int count, int* forks);
    // A sequence with the same tokens in pages of its own.
    int copy(int sequence, std::vector<PageMove>& moves);
    void release(const int* sequences, int count);
    // Moves every page behind the first n (n pages being in use) into a gap among those, in ascending order of both.
    void compact(std::vector<PageMove>& moves);

    int pages() const { return static_cast<int>(references_.size()); }
    int page_tokens() const { return page_tokens_; }
    int free_pages() const { return free_; }
    int references(int page) const { return references_[page]; }
    int tokens(int sequence) const { return at(sequence).tokens; }
    const std::vector<int>& table(int sequence) const { return at(sequence).table; }

    // For the handle that holds it: calls are made under `lock` (shared: those that change nothing, so that a list can be
    // read while a plan is being made), and none but live() after close().
    std::shared_mutex lock;
    bool live() const { return live_; }
    void close();

private:
    struct Sequence {
        bool open = false;
        int tokens = 0;
        std::vector<int> table;
    };
    const Sequence& at(int sequence) const;
    int pages_of(int64_t tokens) const { return static_cast<int>((tokens + page_tokens_ - 1) / page_tokens_); }
    void require_distinct(const int* sequences, int count) const;
    int take_page();
    void drop_page(int page);
    int next_sequence();

    bool live_ = true;
    int page_tokens_;
    int free_;
    int lowest_ = 0;  // no page below this one is free
    std::vector<int> references_;
    std::vector<Sequence> sequences_;
};

// ---- the plan of a batch ----

// One query row: attends positions 0 .. position of its sequence, or, as a row of a tree (position < 0), the first
// -1 - position ones, its context, and what its words name (PlanTrees). Its attention is the joined result of `slots` partial
// ones, slot .. slot + slots - 1 (one: written as the output by the workgroup that computes it).
struct PlanRow {
    int position, slot, slots, row;
};

// One workgroup's attention: key/value head `kv`, tokens [first, first + tokens) of the pages listed from `pages` on
// (the first of them holds token `first`, a multiple of 32), for the (row, query head) pairs pair .. pair + pairs - 1 of
// the rows listed from `rows` on (pair p: row p / group, head p % group of the key/value head). `slot` counts from the
// rows' first slots; `limit` is the least position of the rows, so tokens up to it are seen by all of them.
// What a workgroup would otherwise have to read before it can ask for its first keys and queries, each some 0.7 us behind the
// item itself, is in the item: the pages of its first tokens (tile[i]: of tokens 32 i on, the last one's where it has fewer),
// and its rows where they are one sequence's (row_slots != 0): row and position of pair p are then those of the item's first
// pair, `row` and `limit`, and p's distance from it in rows, and its slots begin at row_slot + that distance * row_slots.
// Rows of a tree have -row_slots, and all of them the context 0 .. limit.
struct PlanItem {
    int pages, first, tokens, rows;
    int pair, pairs, slot, kv;
    int limit, row, row_slot, row_slots;
    int tile[4];
};

// Consecutive rows of one sequence whose positions lie in one page: row .. row + tokens - 1, from `position` on, at `offset`
// of the page.
struct PlanRun {
    int row, tokens, page, offset;
    int position, pad[3];
};

// At the start of the image. Rows of several slots are `joined`; their slots come first, `partials` of them, and only those
// are memory: a row of one slot has a number behind them, and its result goes straight to the output.
struct PlanHeader {
    int rows, narrow, wide, runs;
    int joined, slots, longest_run, partials;
    int tree_stride, most_slots, most_position, pad;  // most_slots: of a row; most_position: that a row stands for
};

// Where a batch has trees, tree_stride numbers for every row: the position that it stands for (its context and its depth in
// the tree; where rows are no tree's, the one it lies at), and for a row of a tree a bit for each position from its context's
// last multiple of 32 on, 32 a number: whether the row sees it. Bits in the order of positions, so that a tile of 32 has
// one number; a row's own is its last one.
constexpr int kMostTree = 1024;  // rows of a tree (33 numbers each)

// Where the arrays lie in the image (in 4-byte words from its start) and how many entries each has room for. Launches
// take it by value, so that a launch finds an array without reading where it is; room only grows.
struct PlanLayout {
    int rows_at = 0, narrow_at = 0, wide_at = 0, runs_at = 0, pages_at = 0, list_at = 0, trees_at = 0, words = 0;
    int rows = 0, narrow = 0, wide = 0, runs = 0, pages = 0, list = 0, trees = 0;
    // Room for at least these; whether anything moved.
    bool grow(const PlanLayout& least);
    bool holds(const PlanLayout& least) const;
    // Room for plain divisions as well (PlanImage::plain), unless the image would be very large.
    void grow_plain(const PlanLayout& plain);
    // What a plan begins with: a batch of a few hundred rows over long sequences, so that a captured step has room to
    // follow it.
    static PlanLayout first();
};

struct PlanShape {
    int kv_heads, group;  // group: query heads of a key/value head
    int wide_pairs;       // pairs of a wide workgroup; a narrow one takes 16
    int token_bytes;      // a position's key and value of one head
};

// A plan's arrays, and what its launches need to know.
struct PlanImage {
    PlanHeader header{};
    std::vector<PlanRow> rows, list;  // list: the rows of every item's part of the tree
    std::vector<PlanItem> narrow, wide;
    std::vector<PlanRun> runs;
    std::vector<int> pages, trees;
    bool writable = true;  // no page that the rows lie in is shared
    PlanLayout least() const;  // the room they take
    // What kPlainDivision can take of any batch of no more rows, sequences with rows and pages in their lists, none of them
    // longer: both grow with the batch, unlike what the usual division takes.
    PlanLayout plain{};
    int64_t plain_partials = 0;
    void write(const PlanLayout& layout, int* words) const;
};

// How a batch's attention is divided: chunks for about so many workgroups, and whether runs of pages are attended once for all
// sequences that share them. Plain: every sequence by itself in one chunk (of kMostTokens), so that what it takes follows from the
// numbers of rows, sequences and pages alone.
struct PlanDivision {
    int workgroups = 256;
    bool plain = false;
};
constexpr PlanDivision kPlainDivision{1, true};

// Rows: the last new_tokens[i] positions of sequences[i], in this order. `parents`: of every row the one of the same sequence
// that it follows, by its number among those, or -1 for the context; null: each the one before it. (Rows that follow one
// another so are no tree, whether said or not.)
PlanImage plan_batch(const PageTables& tables, const int* sequences, const int* new_tokens, int count,
                     const PlanShape& shape, const PlanDivision& division = {}, const int* parents = nullptr);

// The batch in the room that a plan has: in the usual division, or the first coarser one that fits. Whether one does.
bool plan_batch_within(const PageTables& tables, const int* sequences, const int* new_tokens, int count,
                       const PlanShape& shape, const PlanLayout& room, int64_t partials, PlanImage& image,
                       const int* parents = nullptr);

// The tables behind a handle (satori_hip_pages_*).
PageTables& page_tables(satori_hip_pages* handle);

}  // namespace satori
