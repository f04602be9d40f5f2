// The paged cache's host code (satori_amd/csrc/pages.cpp) under AddressSanitizer and UndefinedBehaviorSanitizer (built and
// run by tests/test_pages_sanitize.py with g++): random sequences of calls over small caches, and after each the plan of a
// random batch, whose image is checked against what the kernels assume of it:
//  * every row's attention covers each position up to its own exactly once, in the page and place that the sequence's
//    table says, over all key/value heads and query heads of a group;
//  * a row's partial results have numbers of their own, 0 .. slots - 1, and those of all rows do not overlap;
//  * items start at multiples of 32 positions and hold at most 16 (narrow) or wide_pairs (wide) pairs;
//  * runs cover each row once, each within one page;
//  * every offset and list lies inside the image.
#include <algorithm>
#include <cstdio>
#include <cstring>
#include <map>
#include <random>
#include <set>
#include <string>
#include <tuple>
#include <vector>

#include "../include/satori_hip.h"
#include "../satori_amd/csrc/host_shapes.hpp"
#include "../satori_amd/csrc/pages.hpp"

namespace satori {
void record_error(const std::string&) {}
}  // namespace satori

using namespace satori;

namespace {

int failures = 0;

void expect(bool ok, const char* what, int round) {
    if (!ok && ++failures <= 20) std::fprintf(stderr, "FAILED: %s (round %d)\n", what, round);
}

template <class T>
std::vector<T> section(const std::vector<int>& words, int at, int count, int round) {
    const size_t n = static_cast<size_t>(count) * (sizeof(T) / 4);
    expect(at % 4 == 0 && at >= 0 && at + n <= words.size(), "a section lies outside the image", round);
    std::vector<T> out(count);
    if (count) std::memcpy(out.data(), words.data() + at, n * 4);
    return out;
}

void check_plan(const PageTables& tables, const std::vector<int>& sequences, const std::vector<int>& fresh,
                const PlanShape& shape, PlanLayout& at, int round) {
    const PlanImage image = plan_batch(tables, sequences.data(), fresh.data(), static_cast<int>(sequences.size()), shape);
    const PlanLayout before = at;
    if (!at.grow(image.least())) expect(std::memcmp(&before, &at, sizeof at) == 0, "a layout that stays", round);
    std::vector<int> words(at.words);
    image.write(at, words.data());
    PlanHeader h;
    std::memcpy(&h, words.data(), sizeof h);
    expect(words.size() % 4 == 0, "whole 16-byte words", round);
    expect(h.rows <= at.rows && h.narrow <= at.narrow && h.wide <= at.wide && h.runs <= at.runs, "room", round);
    const auto rows = section<PlanRow>(words, at.rows_at, h.rows, round);
    for (size_t r = 0; r < rows.size(); ++r) expect(rows[r].row == static_cast<int>(r), "a row's number", round);
    const int P = tables.page_tokens();
    std::vector<std::pair<int, int>> of_row;  // sequence, position
    for (size_t i = 0; i < sequences.size(); ++i)
        for (int p = tables.tokens(sequences[i]) - fresh[i]; p < tables.tokens(sequences[i]); ++p)
            of_row.push_back({sequences[i], p});
    expect(of_row.size() == rows.size(), "rows", round);
    // Runs.
    std::vector<int> written(rows.size());
    bool writable = true;
    for (const PlanRun& run : section<PlanRun>(words, at.runs_at, h.runs, round)) {
        expect(run.tokens > 0 && run.offset >= 0 && run.offset + run.tokens <= P, "a run within a page", round);
        expect(run.position == of_row.at(run.row).second && run.tokens <= h.longest_run, "a run's positions", round);
        for (int t = 0; t < run.tokens; ++t) {
            const auto [s, p] = of_row.at(run.row + t);
            expect(rows[run.row + t].position == p, "a row's position", round);
            expect(tables.table(s).at(p / P) == run.page && p % P == run.offset + t, "a run's place", round);
            written[run.row + t]++;
            writable &= tables.references(run.page) == 1;
        }
    }
    for (int w : written) expect(w == 1, "runs cover every row once", round);
    expect(writable == image.writable, "whether the pages are the rows' own", round);
    // Items: (row, kv, head of the group) -> positions seen, and slots written.
    std::map<std::tuple<int, int, int>, std::pair<std::vector<int>, std::set<int>>> seen;
    static int singles = 0;
    for (int wide = 0; wide < 2; ++wide)
        for (const PlanItem& item : section<PlanItem>(words, wide ? at.wide_at : at.narrow_at, wide ? h.wide : h.narrow, round)) {
            expect(item.first % 32 == 0 && item.tokens >= 0, "an item's tokens", round);
            expect(item.pairs > 0 && item.pairs <= (wide ? shape.wide_pairs : 16), "an item's pairs", round);
            expect(item.kv >= 0 && item.kv < shape.kv_heads, "an item's head", round);
            for (int i = 0; i < 4; ++i) {
                const int token = item.first % P + std::min(32 * i, std::max(0, item.tokens - 1));
                expect(item.tile[i] == words.at(at.pages_at + item.pages + token / P), "the page of a first tile", round);
            }
            int least = INT32_MAX;
            for (int p = item.pair; p < item.pair + item.pairs; ++p) {
                const int entry = item.rows + p / shape.group;
                expect(entry >= 0 && entry < at.list, "a row list inside its room", round);
                PlanRow listed;
                std::memcpy(&listed, words.data() + at.list_at + 4 * entry, sizeof listed);
                const int r = listed.row;
                if (item.row_slots > 0) {
                    const int behind = p / shape.group - item.pair / shape.group;
                    const PlanRow derived{item.limit + behind, item.row_slot + behind * item.row_slots, item.row_slots,
                                          item.row + behind};
                    expect(std::memcmp(&derived, &listed, sizeof derived) == 0, "rows of one sequence follow one another", round);
                    singles++;
                }
                expect(std::memcmp(&listed, &rows.at(r), sizeof listed) == 0, "a listed row", round);
                const auto [s, position] = of_row.at(r);
                least = std::min(least, position);
                auto& [positions, slots] = seen[{r, item.kv, p % shape.group}];
                expect(item.slot >= 0 && item.slot < rows[r].slots, "a slot of the row", round);
                expect(slots.insert(item.slot).second, "a slot is written once", round);
                for (int t = item.first; t < item.first + item.tokens; ++t) {
                    const int entry = item.pages + t / P - item.first / P;
                    expect(entry >= 0 && entry < at.pages, "a page list inside its room", round);
                    const int page = words.at(at.pages_at + entry);
                    expect(page >= 0 && page < tables.pages(), "a page of the pool", round);
                    if (t > position) continue;  // hidden
                    expect(page == tables.table(s).at(t / P), "the page of a position", round);
                    positions.push_back(t);
                }
            }
            expect(item.limit == least, "an item's limit", round);
        }
    std::set<int> all;
    for (size_t r = 0; r < rows.size(); ++r) {
        for (int s = 0; s < rows[r].slots; ++s) {
            expect(rows[r].slot + s < h.slots, "slots within their number", round);
            expect(all.insert(rows[r].slot + s).second, "rows have slots of their own", round);
        }
        for (int kv = 0; kv < shape.kv_heads; ++kv)
            for (int g = 0; g < shape.group; ++g) {
                auto& [positions, slots] = seen[{static_cast<int>(r), kv, g}];
                std::sort(positions.begin(), positions.end());
                bool each = static_cast<int>(positions.size()) == rows[r].position + 1;
                for (size_t i = 0; each && i < positions.size(); ++i) each = positions[i] == static_cast<int>(i);
                expect(each, "every position is attended once", round);
                expect(static_cast<int>(slots.size()) == rows[r].slots, "every slot is written", round);
            }
    }
}

}  // namespace

int main() {
    std::mt19937 g(1729);
    const auto up_to = [&](int n) { return static_cast<int>(g() % (n + 1)); };
    for (int round = 0; round < 80; ++round) {
        const int P = 32 << up_to(3), pages = 4 + up_to(60);
        PageTables tables(pages, P);
        std::vector<int> open;
        PlanLayout layout;
        for (int step = 0; step < 25; ++step) {
            try {
                std::vector<PageMove> moves;
                const int what = up_to(9);
                if (open.empty() || what == 0) {
                    open.push_back(tables.open());
                } else if (what <= 4) {
                    std::vector<int> s, n;
                    for (int id : open)
                        if (up_to(1)) {
                            s.push_back(id);
                            n.push_back(up_to(3) ? up_to(3) : up_to(P * 5));
                        }
                    tables.extend(s.data(), n.data(), static_cast<int>(s.size()), moves);
                } else if (what <= 6) {
                    int forks[3];
                    const int count = up_to(3);
                    tables.fork(open[up_to(static_cast<int>(open.size()) - 1)], count, forks);
                    open.insert(open.end(), forks, forks + count);
                } else if (what == 7) {
                    const int s = open[up_to(static_cast<int>(open.size()) - 1)];
                    tables.truncate(s, up_to(tables.tokens(s)));
                } else if (what == 8) {
                    open.push_back(tables.copy(open[up_to(static_cast<int>(open.size()) - 1)], moves));
                } else {
                    const size_t i = up_to(static_cast<int>(open.size()) - 1);
                    tables.release(&open[i], 1);
                    open.erase(open.begin() + i);
                    tables.compact(moves);
                    for (int p = 0; p < tables.pages(); ++p)
                        expect((tables.references(p) > 0) == (p < tables.pages() - tables.free_pages()), "compacted", round);
                }
            } catch (const Failure& f) {
                expect(f.status == SATORI_HIP_E_OUT_OF_MEMORY, "only pages run out", round);
            }
            std::vector<int> held(pages);
            for (int id : open)
                for (int page : tables.table(id)) held[page]++;
            int used = 0;
            for (int p = 0; p < pages; ++p) {
                expect(held[p] == tables.references(p), "reference counts", round);
                used += held[p] > 0;
            }
            expect(used == pages - tables.free_pages(), "free pages", round);
            std::vector<int> batch, fresh;
            for (int id : open)
                if (up_to(2)) {
                    batch.push_back(id);
                    fresh.push_back(std::min(tables.tokens(id), up_to(2) ? 1 : up_to(40)));
                }
            check_plan(tables, batch, fresh, PlanShape{1 + up_to(2), 1 + up_to(6), 16 << up_to(2), 1 << (round % 2 ? 22 : 9)}, layout, round);
        }
    }
    // Long sequences, many chunks.
    for (int round = 1000; round < 1004; ++round) {
        PageTables tables(1 << 12, 32 << (round % 4));
        std::vector<PageMove> moves;
        const int first = tables.open(), tokens = 20000;
        tables.extend(&first, &tokens, 1, moves);
        std::vector<int> batch{first}, fresh{1};
        int forks[9];
        tables.fork(first, 9, forks);
        for (int f : forks) {
            const int n = 1 + up_to(900);
            tables.extend(&f, &n, 1, moves);
            batch.push_back(f);
            fresh.push_back(1 + up_to(2));
            if (fresh.back() > n) fresh.back() = n;
        }
        PlanLayout layout;
        check_plan(tables, batch, fresh, PlanShape{2, 3, 64, 1 << (round % 2 ? 12 : 20)}, layout, round);
    }
    if (failures) return 1;
    std::puts("ok");
    return 0;
}
