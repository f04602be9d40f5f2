// Pages of a shared key/value cache (PageTables), the plan of a batch over them (plan_batch) and the host-only entry
// points satori_hip_pages_*. No device code.
#include "pages.hpp"

#include <algorithm>
#include <climits>
#include <cstring>
#include <mutex>
#include <new>
#include <string>
#include <unordered_map>

#include "../../include/satori_hip.h"
#include "host_shapes.hpp"

namespace satori {

namespace {

[[noreturn]] void out_of_range(const char* name) {
    fail(SATORI_HIP_E_ARGUMENT_OUT_OF_RANGE,
         std::string("Specified argument was out of the range of valid values. (Parameter '") + name + "')");
}

// push_back after this does not allocate.
template <class T>
void reserve_for(std::vector<T>& v, size_t n) {
    if (v.capacity() < n) v.reserve(std::max(n, 2 * v.capacity()));
}

}  // namespace

PageTables::PageTables(int pages, int page_tokens) : page_tokens_(page_tokens), free_(pages) {
    if (pages <= 0) out_of_range("pageCount");
    if (!valid_page_tokens(page_tokens))
        fail(SATORI_HIP_E_ARGUMENT_OUT_OF_RANGE, "Supported page sizes: 32, 64, 128 and 256 tokens.");
    if (static_cast<int64_t>(pages) * page_tokens > INT32_MAX)
        fail(SATORI_HIP_E_OVERFLOW, "Arithmetic operation resulted in an overflow.");
    references_.resize(pages);
}

const PageTables::Sequence& PageTables::at(int sequence) const {
    if (sequence < 0 || static_cast<size_t>(sequence) >= sequences_.size() || !sequences_[sequence].open)
        fail(SATORI_HIP_E_ARGUMENT, "There is no open sequence " + std::to_string(sequence) + ".");
    return sequences_[sequence];
}

void PageTables::require_distinct(const int* sequences, int count) const {
    std::vector<int> sorted(sequences, sequences + count);
    std::sort(sorted.begin(), sorted.end());
    if (std::adjacent_find(sorted.begin(), sorted.end()) != sorted.end())
        fail(SATORI_HIP_E_ARGUMENT, "A sequence is listed twice.");
    for (int s : sorted) at(s);
}

int PageTables::take_page() {
    while (references_[lowest_] != 0) ++lowest_;
    references_[lowest_] = 1;
    --free_;
    return lowest_++;
}

void PageTables::drop_page(int page) {
    if (--references_[page] == 0) {
        ++free_;
        lowest_ = std::min(lowest_, page);
    }
}

int PageTables::next_sequence() {
    for (size_t i = 0; i < sequences_.size(); ++i)
        if (!sequences_[i].open) return static_cast<int>(i);
    if (sequences_.size() >= INT32_MAX) fail(SATORI_HIP_E_OVERFLOW, "Arithmetic operation resulted in an overflow.");
    sequences_.emplace_back();
    return static_cast<int>(sequences_.size() - 1);
}

void PageTables::close() {
    live_ = false;
    std::vector<int>().swap(references_);
    std::vector<Sequence>().swap(sequences_);
}

int PageTables::open() {
    const int s = next_sequence();
    sequences_[s].open = true;
    return s;
}

void PageTables::extend(const int* sequences, const int* tokens, int count, std::vector<PageMove>& moves) {
    require_distinct(sequences, count);
    // What the call takes, before anything changes: sequences that share a part full page are asked in order, and
    // the last holder left keeps it.
    int64_t need = 0;
    std::unordered_map<int, int> left;
    for (int i = 0; i < count; ++i) {
        if (tokens[i] < 0) out_of_range("tokens");
        Sequence& s = sequences_[sequences[i]];
        const int64_t total = static_cast<int64_t>(s.tokens) + tokens[i];
        if (total > INT32_MAX) fail(SATORI_HIP_E_OVERFLOW, "Arithmetic operation resulted in an overflow.");
        const int pages = pages_of(total);
        need += pages - static_cast<int>(s.table.size());
        if (tokens[i] > 0 && s.tokens % page_tokens_ != 0 && references_[s.table.back()] > 1) {
            auto it = left.emplace(s.table.back(), references_[s.table.back()]).first;
            if (it->second > 1) {
                --it->second;
                ++need;
            }
        }
    }
    if (need > free_)
        fail(SATORI_HIP_E_OUT_OF_MEMORY, "The cache has " + std::to_string(free_) + " free pages; " +
                                             std::to_string(need) + " are needed.");
    reserve_for(moves, moves.size() + count);
    for (int i = 0; i < count; ++i) {
        Sequence& s = sequences_[sequences[i]];
        reserve_for(s.table, pages_of(static_cast<int64_t>(s.tokens) + tokens[i]));
    }
    for (int i = 0; i < count; ++i) {
        Sequence& s = sequences_[sequences[i]];
        if (tokens[i] > 0 && s.tokens % page_tokens_ != 0 && references_[s.table.back()] > 1) {
            const int page = take_page();
            moves.push_back({s.table.back(), page});
            drop_page(s.table.back());
            s.table.back() = page;
        }
        s.tokens += tokens[i];
        while (static_cast<int>(s.table.size()) < pages_of(s.tokens)) s.table.push_back(take_page());
    }
}

void PageTables::truncate(int sequence, int tokens) {
    at(sequence);
    Sequence& s = sequences_[sequence];
    if (tokens < 0 || tokens > s.tokens) out_of_range("tokens");
    s.tokens = tokens;
    while (static_cast<int>(s.table.size()) > pages_of(tokens)) {
        drop_page(s.table.back());
        s.table.pop_back();
    }
}

void PageTables::fork(int sequence, int count, int* forks) {
    at(sequence);
    if (count < 0) out_of_range("count");
    const Sequence parent = sequences_[sequence];
    std::vector<Sequence> made(count, parent);  // what allocates comes first
    size_t free_numbers = 0;
    for (const Sequence& s : sequences_) free_numbers += !s.open;
    if (static_cast<size_t>(count) > free_numbers) reserve_for(sequences_, sequences_.size() + count - free_numbers);
    for (int i = 0; i < count; ++i) {
        const int s = next_sequence();
        sequences_[s] = std::move(made[i]);
        forks[i] = s;
    }
    for (int page : parent.table) references_[page] += count;
}

int PageTables::copy(int sequence, std::vector<PageMove>& moves) {
    at(sequence);
    const size_t pages = sequences_[sequence].table.size();
    if (static_cast<int64_t>(pages) > free_)
        fail(SATORI_HIP_E_OUT_OF_MEMORY, "The cache has " + std::to_string(free_) + " free pages; " +
                                             std::to_string(pages) + " are needed.");
    reserve_for(moves, moves.size() + pages);
    std::vector<int> table;
    table.reserve(pages);
    const int s = next_sequence();
    for (int page : sequences_[sequence].table) {
        table.push_back(take_page());
        moves.push_back({page, table.back()});
    }
    sequences_[s].open = true;
    sequences_[s].tokens = sequences_[sequence].tokens;
    sequences_[s].table = std::move(table);
    return s;
}

void PageTables::release(const int* sequences, int count) {
    require_distinct(sequences, count);
    for (int i = 0; i < count; ++i) {
        for (int page : sequences_[sequences[i]].table) drop_page(page);
        sequences_[sequences[i]] = Sequence{};
    }
}

void PageTables::compact(std::vector<PageMove>& moves) {
    const int used = pages() - free_;
    std::vector<int> to(pages() - used, -1);  // of the pages behind
    int moved = 0;
    for (int p = used; p < pages(); ++p) moved += references_[p] != 0;
    reserve_for(moves, moves.size() + moved);
    int gap = 0;
    for (int p = used; p < pages(); ++p) {
        if (references_[p] == 0) continue;
        while (references_[gap] != 0) ++gap;
        references_[gap] = references_[p];
        references_[p] = 0;
        to[p - used] = gap;
        moves.push_back({p, gap});
    }
    if (moved == 0) return;
    for (Sequence& s : sequences_)
        for (int& page : s.table)
            if (page >= used) page = to[page - used];
    lowest_ = used;
}

// ---- the plan ----

namespace {

constexpr int kTile = 32;         // tokens a wave attends at once
constexpr int kWaves = 4;         // of a workgroup, which take tiles in turn
constexpr int kNarrowPairs = 16;  // pairs of a narrow workgroup
constexpr int64_t kNarrowBytes = 128 << 20;
constexpr int kMostTokens = 1 << 20;  // of an item
// A layout larger than this is not made larger still for plain divisions to come.
constexpr int64_t kMostPlainWords = 64 << 20;

// Tokens [begin, end) of the pages of `sequence`, seen by the rows of the sequences members[0 .. count).
struct Node {
    int begin, end;
    std::vector<int> members;  // positions in the batch
    int ancestors;             // node that the members share before this one, or -1
    int chunks = 0, slot = 0, chunk = 0;
    int pages = 0, rows = 0;   // where its lists begin
    bool wide = false;
};

// Runs of pages that sequences share but that are shorter than this are read by each of them: one more partial result
// per row and head (and its joining) costs about what reading so many tokens again does (16 sequences of 12 heads and 300 to
// 400 positions, shared against not, F16: 64 positions 11.6 us and 11.9, 256 12.0 and 12.0, 1024 12.3 and 13.3, 4096 13.6 and
// 17.8; 20 of 32 heads and 100 to 200: 128 positions 14.9 and 14.1, 256 14.8 and 15.4, 512 13.8 and 20.6).
constexpr int kLeastShared = 128;
// The card holds so many workgroups at once (two a CU, up to 128 lanes), each of some 7 us for the chain of its reads alone. Where the items of
// the sequences' own fill that and those of a shared run would come behind them, the run is shared if that saves this much
// reading: 64 sequences of 8 key/value heads and 100 to 200 positions, F16, over 256 shared ones (50 MB) 24.6 us shared and
// 17.5 not, 512 (100 MB) 24.4 and 21.9, 1024 (201 MB) 27.5 and 32.0. Heads of 192 and 256 lanes fit one workgroup a CU, but half
// the number serves them no better: F16, 256 lanes, 32 + 8 heads over 256 shared positions, 30 sequences take 31.1 us with 512
// here and 38.8 with 256, 32 take 30.8 and 23.7, 40 take 32.5 with either; FP32, 30 sequences, 45.4 and 73.7.
constexpr int64_t kPlaces = 512, kRoundBytes = 128 << 20;

}  // namespace

PlanImage plan_batch(const PageTables& tables, const int* sequences, const int* new_tokens, int count,
                     const PlanShape& shape, const PlanDivision& division) {
    PlanImage image;
    const int P = tables.page_tokens();
    std::vector<int> sorted(sequences, sequences + count);
    std::sort(sorted.begin(), sorted.end());
    if (std::adjacent_find(sorted.begin(), sorted.end()) != sorted.end())
        fail(SATORI_HIP_E_ARGUMENT, "A sequence is listed twice.");
    std::vector<int> first_row(count + 1);
    std::vector<PlanRow>& rows = image.rows;
    std::vector<PlanRun>& runs = image.runs;
    for (int i = 0; i < count; ++i) {
        const int tokens = tables.tokens(sequences[i]);
        if (new_tokens[i] < 0 || new_tokens[i] > tokens)
            fail(SATORI_HIP_E_ARGUMENT_OUT_OF_RANGE, "A sequence has fewer tokens than rows.");
        const int64_t total = static_cast<int64_t>(first_row[i]) + new_tokens[i];
        if (total * shape.group > INT32_MAX / 2)
            fail(SATORI_HIP_E_OVERFLOW, "Arithmetic operation resulted in an overflow.");
        first_row[i + 1] = static_cast<int>(total);
        const std::vector<int>& table = tables.table(sequences[i]);
        for (int p = tokens - new_tokens[i]; p < tokens; ++p) {
            if (p % P == 0 || p == tokens - new_tokens[i]) {
                runs.push_back({static_cast<int>(rows.size()), 0, table[p / P], p % P, p, {}});
                image.writable &= tables.references(table[p / P]) == 1;
            }
            image.header.longest_run = std::max(image.header.longest_run, ++runs.back().tokens);
            rows.push_back({p, 0, 0, static_cast<int>(rows.size())});
        }
    }

    const auto blocks_of = [](int64_t pairs) { return (pairs + kNarrowPairs - 1) / kNarrowPairs; };
    int64_t own = 0;  // items of the sequences by themselves, at least
    for (int i = 0; i < count; ++i) own += blocks_of(static_cast<int64_t>(new_tokens[i]) * shape.group) * shape.kv_heads;
    const auto worth_sharing = [&](const std::vector<int>& members, int64_t tokens) {
        if (division.plain || tokens < kLeastShared) return false;
        int64_t pairs = 0, apart = 0;
        for (int m : members) {
            pairs += static_cast<int64_t>(new_tokens[m]) * shape.group;
            apart += blocks_of(static_cast<int64_t>(new_tokens[m]) * shape.group);
        }
        const int64_t together = blocks_of(pairs);
        const auto rounds = [](int64_t items) { return (items + kPlaces - 1) / kPlaces; };
        return rounds(own + together * shape.kv_heads) == rounds(own) ||
               (apart - together) * tokens * shape.kv_heads >= kRoundBytes / shape.token_bytes;
    };

    // The trie of the tables: a node for every run of pages that the same sequences share.
    std::vector<Node> nodes;
    struct Open {
        std::vector<int> members;
        int page, ancestors;
    };
    std::vector<Open> open(1);
    open[0].page = 0;
    open[0].ancestors = -1;
    for (int i = 0; i < count; ++i)
        if (new_tokens[i] > 0) open[0].members.push_back(i);
    while (!open.empty()) {
        Open o = std::move(open.back());
        open.pop_back();
        if (o.members.empty()) continue;
        const std::vector<int>& lead = tables.table(sequences[o.members[0]]);
        if (o.members.size() == 1) {
            const int end = tables.tokens(sequences[o.members[0]]);
            if (o.page * P < end) nodes.push_back({o.page * P, end, o.members, o.ancestors});
            continue;
        }
        size_t common = lead.size();
        int longest = 0;
        for (int m : o.members) {
            const std::vector<int>& t = tables.table(sequences[m]);
            size_t same = o.page;
            while (same < std::min(common, t.size()) && t[same] == lead[same]) ++same;
            common = same;
            longest = std::max(longest, tables.tokens(sequences[m]));
        }
        const int begin = o.page * P, end = std::min(static_cast<int>(common) * P, longest);
        int from = o.page, ancestors = o.ancestors;
        if (worth_sharing(o.members, end - begin)) {
            nodes.push_back({begin, end, o.members, o.ancestors});
            from = static_cast<int>(common);
            ancestors = static_cast<int>(nodes.size()) - 1;
        }
        // Its members by the page that follows, in the order of their first appearance.
        std::vector<Open> parts;
        std::unordered_map<int, size_t> by_page;
        for (int m : o.members) {
            const std::vector<int>& t = tables.table(sequences[m]);
            if (common >= t.size()) {  // nothing follows: what is left of it, if anything, is its own part
                if (from < static_cast<int>(t.size())) parts.push_back({{m}, from, ancestors});
                continue;
            }
            auto it = by_page.find(t[common]);
            if (it == by_page.end()) {
                it = by_page.emplace(t[common], parts.size()).first;
                parts.push_back({{}, from, ancestors});
            }
            parts[it->second].members.push_back(m);
        }
        for (auto it = parts.rbegin(); it != parts.rend(); ++it) open.push_back(std::move(*it));
    }

    // Which nodes' items are wide. A wide workgroup reads a tile once for all its pairs but takes them through it in four
    // waves; narrow ones, 16 pairs each, read it again for each of their blocks (from L2, mostly) but give every wave tokens of
    // its own. So narrow items serve up to half a wide workgroup's pairs, and all of them while the blocks together read no
    // more than kNarrowBytes. Wide against narrow, F16 heads of 128 lanes, 96 pairs over 4096, 16384 and 65536 tokens of 2
    // key/value heads (25, 100 and 400 MB): 19.7 us and 13.5, 24.7 and 22.6, 38.7 and 46.9; 128 pairs of 8 heads over 4096 and
    // 8192 (134 and 268 MB): 26.1 and 27.0, 31.0 and 37.4; FP32, 144 pairs of 2 heads over 4000 and 8192 (74 and 151 MB): 25.7
    // and 23.1, 35.5 and 50.3. One number for all types and widths leaves prompts on the slower side just behind it: 4 x 128
    // rows of 14 + 2 heads of 80 F16 lanes over 1128 positions (194 MB) take 38.9 wide and 20.0 narrow, 512 rows of 32 + 8 heads
    // of 128 over themselves (268 MB) 49.9 and 28.3 (over 4512, 2.4 GB, 121 and 187); FP32 turns earlier, 128 rows of 12 + 2 heads
    // of 128 lanes over 1128 (111 MB) taking 27.4 and 44.9.
    int64_t narrow_tokens = 0, wide_tokens = 0, again = 0;
    std::vector<int64_t> pairs_of(nodes.size());
    for (size_t i = 0; i < nodes.size(); ++i) {
        Node& n = nodes[i];
        for (int m : n.members) pairs_of[i] += static_cast<int64_t>(new_tokens[m]) * shape.group;
        n.wide = pairs_of[i] > shape.wide_pairs / 2;
        if (n.wide) again += blocks_of(pairs_of[i]) * shape.kv_heads * (n.end - n.begin);
    }
    const auto pairs_a_block = [&](const Node& n) { return n.wide ? shape.wide_pairs : kNarrowPairs; };
    for (size_t i = 0; i < nodes.size(); ++i) {
        Node& n = nodes[i];
        n.wide &= division.plain || again > kNarrowBytes / shape.token_bytes;
        const int64_t blocks = (pairs_of[i] + pairs_a_block(n) - 1) / pairs_a_block(n);
        (n.wide ? wide_tokens : narrow_tokens) += blocks * shape.kv_heads * (n.end - n.begin);
    }
    // Chunks of tokens: as many as give every CU work (kv heads and blocks of pairs count too), and no shorter than
    // one tile per wave. (Few pairs in 256, 512 and 1024 workgroups: 24 rows over 4000 positions, FP32, 23.0, 28.9 and 31.6 us, 64
    // of 32 + 8 heads and 1000 to 2000 each, F16, 68, 78 and 80, 9 x 5 over 4000 16.9, 15.4 and 19.3. Many in 256 and 512: 64 rows over 8192, F16, 46
    // and 58, over 32768 103 and 102, 24 over 8192, FP32, 35 and 31: the more chunks, the more partial results.)
    const auto chunk_for = [&](int64_t tokens) {
        if (division.plain) return kMostTokens;
        const int64_t step = kTile * kWaves;
        const int64_t c = (tokens / division.workgroups + step - 1) / step * step;
        return static_cast<int>(std::min<int64_t>(std::max<int64_t>(c, step), kMostTokens));
    };
    const int narrow_chunk = chunk_for(narrow_tokens), wide_chunk = chunk_for(wide_tokens);

    std::vector<int>& page_list = image.pages;
    std::vector<int> row_list;
    for (Node& n : nodes) {
        n.chunk = n.wide ? wide_chunk : narrow_chunk;
        n.chunks = (n.end - n.begin - 1) / n.chunk + 1;  // (a sum with the chunk could pass 32 bits)
        n.slot = n.ancestors < 0 ? 0 : nodes[n.ancestors].slot + nodes[n.ancestors].chunks;
        n.pages = static_cast<int>(page_list.size());
        const std::vector<int>& table = tables.table(sequences[n.members[0]]);
        page_list.insert(page_list.end(), table.begin() + n.begin / P, table.begin() + ((n.end - 1) / P + 1));
        n.rows = static_cast<int>(row_list.size());
        for (int m : n.members)
            for (int r = first_row[m]; r < first_row[m + 1]; ++r) {
                row_list.push_back(r);
                rows[r].slots = n.slot + n.chunks;  // a deeper node comes later
            }
    }
    int64_t slots = 0;
    const auto number = [&](PlanRow& r) {
        if (slots + r.slots > INT32_MAX) fail(SATORI_HIP_E_OVERFLOW, "Arithmetic operation resulted in an overflow.");
        r.slot = static_cast<int>(slots);
        slots += r.slots;
    };
    for (PlanRow& r : rows)
        if (r.slots > 1) {
            number(r);
            ++image.header.joined;
        }
    image.header.partials = static_cast<int>(slots);
    for (PlanRow& r : rows)
        if (r.slots == 1) number(r);
    image.header.slots = static_cast<int>(slots);

    // The workgroups. Consecutive workgroups run on different XCDs (eight, each with an L2 of its own), so the blocks of
    // pairs that read the same tokens are put eight apart.
    std::vector<PlanItem>&narrow = image.narrow, &wide = image.wide;
    for (size_t i = 0; i < nodes.size(); ++i) {
        const Node& n = nodes[i];
        // Blocks of pairs, as even as whole matrix tiles of 16 make them.
        const int most = pairs_a_block(n);
        const int64_t least = (pairs_of[i] + most - 1) / most;
        const int step = static_cast<int>((pairs_of[i] + 16 * least - 1) / (16 * least) * 16);
        const int blocks = static_cast<int>((pairs_of[i] + step - 1) / step);
        const int64_t units = static_cast<int64_t>(n.chunks) * shape.kv_heads;
        std::vector<PlanItem>& list = n.wide ? wide : narrow;
        if (static_cast<int64_t>(list.size()) + units * blocks > INT32_MAX / 32)
            fail(SATORI_HIP_E_OVERFLOW, "Arithmetic operation resulted in an overflow.");
        for (int64_t u0 = 0; u0 < units; u0 += 8)
            for (int b = 0; b < blocks; ++b)
                for (int64_t u = u0; u < std::min<int64_t>(u0 + 8, units); ++u) {
                    const int chunk = static_cast<int>(u / shape.kv_heads);
                    PlanItem item{};
                    item.first = n.begin + chunk * n.chunk;
                    item.tokens = std::min(n.chunk, n.end - item.first);
                    item.pages = n.pages + item.first / P - n.begin / P;
                    item.rows = n.rows;
                    item.pair = b * step;
                    item.pairs = static_cast<int>(std::min<int64_t>(step, pairs_of[i] - item.pair));
                    item.slot = n.slot + chunk;
                    item.kv = static_cast<int>(u % shape.kv_heads);
                    int least = INT_MAX, most = 0;
                    for (int r = item.pair / shape.group; r <= (item.pair + item.pairs - 1) / shape.group; ++r) {
                        const int position = rows[row_list[n.rows + r]].position;
                        least = std::min(least, position);
                        most = std::max(most, position);
                    }
                    item.limit = least;
                    // Tokens behind all rows of the block are not read (an empty item still writes its partials).
                    item.tokens = std::max(0, std::min(item.tokens, most + 1 - item.first));
                    for (int i = 0; i < 4; ++i)
                        item.tile[i] = page_list[item.pages + (item.first % P + std::min(i * kTile, std::max(0, item.tokens - 1))) / P];
                    if (n.members.size() == 1) {
                        const PlanRow& row = rows[row_list[n.rows + item.pair / shape.group]];
                        item.row = row.row;
                        item.row_slot = row.slot;
                        item.row_slots = row.slots;
                    }
                    list.push_back(item);
                }
    }

    image.list.reserve(row_list.size());
    for (int r : row_list) image.list.push_back(rows[r]);
    PlanHeader& h = image.header;
    h.rows = static_cast<int>(rows.size());
    h.narrow = static_cast<int>(narrow.size());
    h.wide = static_cast<int>(wide.size());
    h.runs = static_cast<int>(runs.size());

    // What plain divisions take at most: a sequence's pairs fill their blocks but for the last one, sequences of up to half a
    // wide workgroup's pairs (no more than that many blocks each) are narrow, those of more (so many there can be) wide; a run
    // ends at a page's end or the sequence's.
    int64_t of_rows = 0, list_pages = 0, longest = 0;
    for (int i = 0; i < count; ++i)
        if (new_tokens[i] > 0) {
            ++of_rows;
            list_pages += static_cast<int64_t>(tables.table(sequences[i]).size());
            longest = std::max<int64_t>(longest, tables.tokens(sequences[i]));
        }
    const int64_t all = static_cast<int64_t>(h.rows) * shape.group, chunks = (longest + kMostTokens - 1) / kMostTokens;
    const int64_t units = chunks * shape.kv_heads;
    const int64_t narrow_blocks = std::min(all / kNarrowPairs + of_rows, of_rows * blocks_of(shape.wide_pairs / 2));
    const int64_t wide_blocks = all / shape.wide_pairs + std::min(of_rows, 2 * all / shape.wide_pairs);
    const auto entries = [](int64_t n) { return static_cast<int>(std::min<int64_t>(n, INT32_MAX / 64)); };
    image.plain.rows = image.plain.list = h.rows;
    image.plain.runs = entries(std::min<int64_t>(h.rows, h.rows / P + 2 * of_rows));
    image.plain.pages = entries(list_pages);
    image.plain.narrow = entries(narrow_blocks * units);
    image.plain.wide = entries(wide_blocks * units);
    image.plain_partials = chunks > 1 ? h.rows * chunks : 0;
    return image;
}

bool plan_batch_within(const PageTables& tables, const int* sequences, const int* new_tokens, int count,
                       const PlanShape& shape, const PlanLayout& room, int64_t partials, PlanImage& image) {
    PlanDivision division;
    for (;;) {
        image = plan_batch(tables, sequences, new_tokens, count, shape, division);
        if (room.holds(image.least()) && image.header.partials <= partials) return true;
        if (division.plain || image.header.rows > room.rows) return false;
        division.workgroups > 1 ? void(division.workgroups /= 2) : void(division = kPlainDivision);
    }
}

bool PlanLayout::holds(const PlanLayout& l) const {
    return l.rows <= rows && l.narrow <= narrow && l.wide <= wide && l.runs <= runs && l.pages <= pages && l.list <= list;
}

bool PlanLayout::grow(const PlanLayout& least) {
    bool moved = words == 0;
    const auto room = [&](int& have, int need) {
        if (need <= have) return;
        have = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(need) + need / 2 + 16, INT32_MAX / 64));
        have = std::max(have, need);
        moved = true;
    };
    room(rows, least.rows);
    room(narrow, least.narrow);
    room(wide, least.wide);
    room(runs, least.runs);
    room(pages, least.pages);
    room(list, least.list);
    if (!moved) return false;
    int64_t at = sizeof(PlanHeader) / 4;
    const auto place = [&](int& where, int64_t entries, size_t size) {
        where = static_cast<int>(at);
        at = (at + entries * static_cast<int64_t>(size / 4) + 3) / 4 * 4;  // 16-byte aligned
        if (at > INT32_MAX / 8) fail(SATORI_HIP_E_OVERFLOW, "Arithmetic operation resulted in an overflow.");
    };
    place(rows_at, rows, sizeof(PlanRow));
    place(narrow_at, narrow, sizeof(PlanItem));
    place(wide_at, wide, sizeof(PlanItem));
    place(runs_at, runs, sizeof(PlanRun));
    place(pages_at, pages, sizeof(int));
    place(list_at, list, sizeof(PlanRow));
    words = static_cast<int>(at);
    return true;
}

void PlanLayout::grow_plain(const PlanLayout& plain) {
    const int64_t most = 2 * (static_cast<int64_t>(plain.rows + int64_t(plain.list)) * (sizeof(PlanRow) / 4) +
                              (plain.narrow + int64_t(plain.wide)) * (sizeof(PlanItem) / 4) +
                              int64_t(plain.runs) * (sizeof(PlanRun) / 4) + plain.pages);
    if (words + most <= kMostPlainWords) grow(plain);
}

PlanLayout PlanLayout::first() {
    PlanLayout least, layout;
    least.rows = least.runs = 256;
    least.narrow = least.wide = 1024;
    least.pages = 32768;
    least.list = 1024;
    layout.grow(least);
    return layout;
}

PlanLayout PlanImage::least() const {
    PlanLayout l;
    l.rows = static_cast<int>(rows.size());
    l.narrow = static_cast<int>(narrow.size());
    l.wide = static_cast<int>(wide.size());
    l.runs = static_cast<int>(runs.size());
    l.pages = static_cast<int>(pages.size());
    l.list = static_cast<int>(list.size());
    return l;
}

void PlanImage::write(const PlanLayout& layout, int* words) const {
    static_assert(sizeof(PlanHeader) % 16 == 0 && sizeof(PlanRow) % 16 == 0 && sizeof(PlanItem) % 16 == 0 &&
                      sizeof(PlanRun) % 16 == 0,
                  "16-byte entries");
    std::memcpy(words, &header, sizeof header);
    const auto put = [&](int at, const auto& v) {
        if (!v.empty()) std::memcpy(words + at, v.data(), v.size() * sizeof(v[0]));
    };
    put(layout.rows_at, rows);
    put(layout.narrow_at, narrow);
    put(layout.wide_at, wide);
    put(layout.runs_at, runs);
    put(layout.pages_at, pages);
    put(layout.list_at, list);
}

}  // namespace satori

struct satori_hip_pages {
    satori::PageTables tables;
    satori_hip_pages(int pages, int page_tokens) : tables(pages, page_tokens) {}
};

namespace satori {

PageTables& page_tables(satori_hip_pages* handle) { return handle->tables; }

namespace {

template <class F>
int host_call(F&& body) {
    try {
        body();
        record_error("");
        return SATORI_HIP_OK;
    } catch (const Failure& f) {
        record_error(f.message);
        return f.status;
    } catch (const std::bad_alloc&) {
        record_error("Out of host memory.");
        return SATORI_HIP_E_OUT_OF_MEMORY;
    } catch (...) {
        record_error("Unexpected failure.");
        return SATORI_HIP_E_DEVICE;
    }
}

void require_pointer(const void* p, const char* name) {
    if (!p) fail(SATORI_HIP_E_ARGUMENT_NULL, std::string("Value cannot be null. (Parameter '") + name + "')");
}

// Lock: std::unique_lock, or std::shared_lock where the tables stay as they are.
template <template <class> class Lock = std::unique_lock, class F>
int pages_call(satori_hip_pages* handle, F&& body) {
    return host_call([&] {
        require_pointer(handle, "pages");
        const Lock<std::shared_mutex> guard(handle->tables.lock);
        if (!handle->tables.live())
            fail(SATORI_HIP_E_OBJECT_DISPOSED, "Cannot access a disposed object. Object name: 'satori_hip_pages'.");
        body(handle->tables);
    });
}

// The caller's arrays hold `capacity` moves. `most` is what the call can need: checked before anything changes.
void require_capacity(int64_t most, int capacity, const int* sources, const int* destinations) {
    if (capacity < 0) out_of_range("capacity");
    if (most > capacity)
        fail(SATORI_HIP_E_ARGUMENT, "The move arrays hold " + std::to_string(capacity) + " of up to " +
                                        std::to_string(most) + " moves.");
    if (most > 0) {
        require_pointer(sources, "sources");
        require_pointer(destinations, "destinations");
    }
}

void give(const std::vector<PageMove>& moves, int* sources, int* destinations, int* count) {
    for (size_t i = 0; i < moves.size(); ++i) {
        sources[i] = moves[i].source;
        destinations[i] = moves[i].destination;
    }
    *count = static_cast<int>(moves.size());
}

}  // namespace
}  // namespace satori

using namespace satori;

extern "C" {

int satori_hip_pages_create(int page_count, int page_tokens, satori_hip_pages** pages) {
    return host_call([&] {
        require_pointer(pages, "pages");
        *pages = nullptr;
        *pages = new satori_hip_pages(page_count, page_tokens);
    });
}

int satori_hip_pages_destroy(satori_hip_pages* pages) {
    return host_call([&] {
        if (!pages) return;
        const std::unique_lock<std::shared_mutex> guard(pages->tables.lock);
        pages->tables.close();  // the handle stays valid as a tombstone so a second destroy is a no-op
    });
}

int satori_hip_pages_open(satori_hip_pages* pages, int* sequence) {
    return pages_call(pages, [&](PageTables& t) {
        require_pointer(sequence, "sequence");
        *sequence = t.open();
    });
}

int satori_hip_pages_extend(satori_hip_pages* pages, const int* sequences, const int* tokens, int count, int* sources,
                            int* destinations, int capacity, int* moves) {
    return pages_call(pages, [&](PageTables& t) {
        require_pointer(moves, "moves");
        *moves = 0;
        if (count < 0) out_of_range("count");
        if (count > 0) {
            require_pointer(sequences, "sequences");
            require_pointer(tokens, "tokens");
        }
        require_capacity(count, capacity, sources, destinations);
        std::vector<PageMove> made;
        t.extend(sequences, tokens, count, made);
        give(made, sources, destinations, moves);
    });
}

int satori_hip_pages_truncate(satori_hip_pages* pages, int sequence, int tokens) {
    return pages_call(pages, [&](PageTables& t) { t.truncate(sequence, tokens); });
}

int satori_hip_pages_fork(satori_hip_pages* pages, int sequence, int count, int* forks) {
    return pages_call(pages, [&](PageTables& t) {
        if (count > 0) require_pointer(forks, "forks");
        t.fork(sequence, count, forks);
    });
}

int satori_hip_pages_copy(satori_hip_pages* pages, int sequence, int* copy, int* sources, int* destinations,
                          int capacity, int* moves) {
    return pages_call(pages, [&](PageTables& t) {
        require_pointer(copy, "copy");
        require_pointer(moves, "moves");
        *moves = 0;
        require_capacity(static_cast<int64_t>(t.table(sequence).size()), capacity, sources, destinations);
        std::vector<PageMove> made;
        *copy = t.copy(sequence, made);
        give(made, sources, destinations, moves);
    });
}

int satori_hip_pages_free(satori_hip_pages* pages, const int* sequences, int count) {
    return pages_call(pages, [&](PageTables& t) {
        if (count < 0) out_of_range("count");
        if (count > 0) require_pointer(sequences, "sequences");
        t.release(sequences, count);
    });
}

int satori_hip_pages_compact(satori_hip_pages* pages, int* sources, int* destinations, int capacity, int* moves) {
    return pages_call(pages, [&](PageTables& t) {
        require_pointer(moves, "moves");
        *moves = 0;
        const int used = t.pages() - t.free_pages();
        int64_t most = 0;
        for (int p = used; p < t.pages(); ++p) most += t.references(p) != 0;
        require_capacity(most, capacity, sources, destinations);
        std::vector<PageMove> made;
        t.compact(made);
        give(made, sources, destinations, moves);
    });
}

int satori_hip_pages_free_count(satori_hip_pages* pages, int* free_pages) {
    return pages_call<std::shared_lock>(pages, [&](PageTables& t) {
        require_pointer(free_pages, "freePages");
        *free_pages = t.free_pages();
    });
}

int satori_hip_pages_sequence(satori_hip_pages* pages, int sequence, int* tokens, int* table, int capacity,
                              int* count) {
    return pages_call<std::shared_lock>(pages, [&](PageTables& t) {
        const std::vector<int>& list = t.table(sequence);
        if (tokens) *tokens = t.tokens(sequence);
        if (count) *count = static_cast<int>(list.size());
        if (!table) return;
        if (capacity < static_cast<int>(list.size()))
            fail(SATORI_HIP_E_ARGUMENT, "The table holds " + std::to_string(capacity) + " of " +
                                            std::to_string(list.size()) + " pages.");
        std::copy(list.begin(), list.end(), table);
    });
}

}  // extern "C"
