// Plans of trees (satori_amd/csrc/pages.cpp) under AddressSanitizer and UndefinedBehaviorSanitizer (built and run by
// tests/test_trees.py with g++): random trees and prompts over sequences that share pages, every plan's image read as the
// kernels read it:
//  * what the items' tiles show of each row's positions is its context, the rows that it follows and itself, each once;
//  * rows of one sequence are derived as listed, and a tree's words lie inside the image;
//  * every row has the position that it stands for, and its place.
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

int failures = 0, trees = 0, singles = 0, shared = 0;

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
                const std::vector<int>& parents, const PlanShape& shape, const PlanDivision& division, PlanLayout& at, int round) {
    const int count = static_cast<int>(sequences.size());
    const PlanImage image = plan_batch(tables, sequences.data(), fresh.data(), count, shape, division, parents.data());
    at.grow(image.least());
    std::vector<int> words(at.words, -7);
    image.write(at, words.data());
    PlanHeader h;
    std::memcpy(&h, words.data(), sizeof h);
    const int P = tables.page_tokens();
    // What each row is and sees.
    std::vector<std::tuple<int, int, int>> of_row;  // sequence, place, position
    std::vector<std::set<int>> sees;
    std::vector<bool> tree;
    bool any = false;
    for (int i = 0, first = 0; i < count; first += fresh[i++]) {
        const int context = tables.tokens(sequences[i]) - fresh[i];
        bool chain = true;
        for (int j = 0; j < fresh[i]; ++j) chain &= parents[first + j] == j - 1;
        any |= !chain;
        for (int j = 0; j < fresh[i]; ++j) {
            const int parent = parents[first + j];
            const int depth = parent < 0 ? 0 : std::get<2>(of_row[first + parent]) - context + 1;
            of_row.push_back({sequences[i], context + j, context + depth});
            std::set<int> mine;
            if (parent < 0)
                for (int p = 0; p < context; ++p) mine.insert(p);
            else
                mine = sees[first + parent];
            mine.insert(context + j);
            sees.push_back(mine);
            tree.push_back(!chain);
        }
    }
    expect((h.tree_stride > 0) == any, "numbers of trees where there are some", round);
    expect(h.rows == static_cast<int>(of_row.size()), "rows", round);
    expect(at.trees_at % 4 == 0 && at.trees_at + h.rows * h.tree_stride <= at.words, "the trees' numbers lie inside", round);
    expect(h.rows * h.tree_stride == static_cast<int>(image.trees.size()), "as many numbers as rows say", round);
    const auto rows = section<PlanRow>(words, at.rows_at, h.rows, round);
    for (int r = 0; r < h.rows; ++r) {
        const auto [s, place, position] = of_row[r];
        (void)s;
        if (h.tree_stride) expect(words.at(at.trees_at + r * h.tree_stride) == position, "the position a row stands for", round);
        const int context = sees[r].size() ? place : 0;
        (void)context;
        if (tree[r]) {
            expect(rows[r].position < 0, "a row of a tree", round);
            trees++;
        } else {
            expect(rows[r].position == place, "a row of no tree", round);
        }
    }
    for (const PlanRun& run : section<PlanRun>(words, at.runs_at, h.runs, round))
        for (int t = 0; t < run.tokens; ++t) {
            const auto [s, place, position] = of_row.at(run.row + t);
            (void)position;
            expect(run.position + t == place && tables.table(s).at(place / P) == run.page && place % P == run.offset + t,
                   "a run's place", round);
        }
    std::map<std::tuple<int, int, int>, std::pair<std::vector<int>, std::set<int>>> seen;
    for (int wide = 0; wide < 2; ++wide)
        for (const PlanItem& item : section<PlanItem>(words, wide ? at.wide_at : at.narrow_at, wide ? h.wide : h.narrow, round))
            for (int p = item.pair; p < item.pair + item.pairs; ++p) {
                PlanRow listed;
                std::memcpy(&listed, words.data() + at.list_at + 4 * (item.rows + p / shape.group), sizeof listed);
                const int behind = p / shape.group - item.pair / shape.group;
                PlanRow row = listed;
                if (item.row_slots > 0)
                    row = PlanRow{item.limit + behind, item.row_slot + behind * item.row_slots, item.row_slots, item.row + behind};
                else if (item.row_slots < 0)
                    row = PlanRow{-2 - item.limit, item.row_slot - behind * item.row_slots, -item.row_slots, item.row + behind};
                singles += item.row_slots < 0;
                shared += item.row_slots == 0 && row.position < 0;
                expect(std::memcmp(&row, &listed, sizeof row) == 0, "rows of one sequence are derived as listed", round);
                const int r = row.row;
                auto& [positions, slots] = seen[{r, item.kv, p % shape.group}];
                expect(item.slot >= 0 && item.slot < rows.at(r).slots && slots.insert(item.slot).second, "a slot", round);
                const int limit = (row.position < 0 ? -2 - row.position : row.position) - item.first;
                for (int t = 0; t < item.tokens; t += 32) {
                    const int end = item.tokens - t;
                    const bool hides = item.first + t + 31 > item.limit;
                    unsigned bits = end >= 32 ? ~0u : (1u << end) - 1;
                    if (hides && row.position >= 0) {
                        const int n = std::min(limit - t + 1, end);
                        bits = n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1;
                    } else if (hides) {
                        const int k = (item.first + t) / 32 - (item.first + limit + 1) / 32;
                        if (k >= 0)
                            bits &= k < h.tree_stride - 1
                                        ? static_cast<unsigned>(words.at(at.trees_at + r * h.tree_stride + 1 + k))
                                        : 0u;
                    }
                    for (int i = 0; i < 32; ++i)
                        if (bits >> i & 1) {
                            const int token = item.first + t + i;
                            positions.push_back(token);
                            const int page = words.at(at.pages_at + item.pages + token / P - item.first / P);
                            expect(page == tables.table(std::get<0>(of_row[r])).at(token / P), "the page of a position", round);
                        }
                }
            }
    for (int r = 0; r < h.rows; ++r)
        for (int kv = 0; kv < shape.kv_heads; ++kv)
            for (int g = 0; g < shape.group; ++g) {
                auto& [positions, slots] = seen[{r, kv, g}];
                std::sort(positions.begin(), positions.end());
                expect(positions == std::vector<int>(sees[r].begin(), sees[r].end()), "a row sees its own, once", round);
                expect(static_cast<int>(slots.size()) == rows[r].slots, "every slot is written", round);
            }
}

}  // namespace

int main() {
    std::mt19937 g(4104);
    const auto up_to = [&](int n) { return static_cast<int>(g() % (n + 1)); };
    for (int round = 0; round < 300; ++round) {
        const int P = 32 << up_to(3);
        PageTables tables(200, P);
        std::vector<PageMove> moves;
        std::vector<int> open{tables.open()};
        int tokens = up_to(2) ? up_to(700) : 0;
        tables.extend(open.data(), &tokens, 1, moves);
        int forks[3];
        const int count = up_to(3);
        tables.fork(open[0], count, forks);
        open.insert(open.end(), forks, forks + count);
        PlanLayout layout;
        for (int step = 0; step < 3; ++step) {
            std::vector<int> batch, fresh, parents;
            for (int id : open) {
                const int n = up_to(4) ? up_to(20) : up_to(200);
                // (some rows stay in pages that others hold)
                if (up_to(3)) tables.extend(&id, &n, 1, moves);
                const int rows = std::min(tables.tokens(id), n);
                batch.push_back(id);
                fresh.push_back(rows);
                const int kind = up_to(3);
                for (int j = 0; j < rows; ++j) parents.push_back(kind == 0 ? j - 1 : kind == 1 ? up_to(j) - 1 : std::max(-1, (j - 1) / 3 - (j == 0)));
            }
            const PlanShape shape{1 + up_to(1), 1 + up_to(4), 16 << up_to(2), 1 << (round % 2 ? 22 : 9)};
            check_plan(tables, batch, fresh, parents, shape, step == 2 ? kPlainDivision : PlanDivision{1 << up_to(9)}, layout, round);
        }
    }
    // The largest tree, and rows that follow one another in any number.
    {
        PageTables tables(300, 32);
        std::vector<PageMove> moves;
        const int s = tables.open(), tokens = 3000;
        tables.extend(&s, &tokens, 1, moves);
        for (int rows : {kMostTree, kMostTree + 1}) {
            std::vector<int> parents(rows);
            for (int j = 0; j < rows; ++j) parents[j] = j ? (j - 1) / 2 : -1;
            PlanLayout layout;
            try {
                check_plan(tables, {s}, {rows}, parents, PlanShape{1, 2, 64, 512}, {}, layout, rows);
                expect(rows == kMostTree, "a tree that is too large", rows);
            } catch (const Failure& f) {
                expect(rows > kMostTree && f.status == SATORI_HIP_E_NOT_SUPPORTED, "only larger trees are refused", rows);
            }
            for (int j = 0; j < rows; ++j) parents[j] = j - 1;
            check_plan(tables, {s}, {rows}, parents, PlanShape{1, 2, 64, 512}, {}, layout, rows);
        }
        for (int bad : {-2, 1, 5}) {
            const int parents[] = {-1, bad};
            const int two = 2;
            try {
                plan_batch(tables, &s, &two, 1, PlanShape{1, 2, 64, 512}, {}, parents);
                expect(false, "a row that follows a later one", bad);
            } catch (const Failure& f) {
                expect(f.status == SATORI_HIP_E_ARGUMENT_OUT_OF_RANGE, "its error", bad);
            }
        }
        // A batch that does not fit the room of a plan without trees.
        PlanLayout room = PlanLayout::first();
        PlanImage image;
        const int parents[] = {-1, -1}, two = 2;
        expect(!plan_batch_within(tables, &s, &two, 1, PlanShape{1, 2, 64, 512}, room, 0, image, parents), "no room for trees", 0);
    }
    expect(trees > 1000 && singles > 1000 && shared > 100, "rows of trees of all kinds", -1);
    if (failures) return 1;
    std::puts("ok");
    return 0;
}
