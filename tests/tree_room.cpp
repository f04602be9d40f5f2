// A tree beside prompts of any length (plan_batch of satori_amd/csrc/pages.cpp): as many rows as an image counts are planned, with
// room in a layout; more are refused before anything is made for them. Built and run by tests/test_tree_room.py.
#include <cstdio>
#include <string>
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

void expect(bool ok, const char* what, int rows) {
    if (!ok) std::fprintf(stderr, "FAILED: %s (%d rows)\n", what, rows), ++failures;
}

}  // namespace

int main() {
    const PlanShape shape{1, 1, 64, 512};
    const int tree = kMostTree, context = 1000;
    for (int prompt : {16000, 1'100'000, 8'200'000}) {
        PageTables tables(40000, 256);
        std::vector<PageMove> moves;
        const int ids[] = {tables.open(), tables.open()};
        const int tokens[] = {prompt, context + tree};
        tables.extend(ids, tokens, 2, moves);
        const int rows[] = {prompt, tree};
        std::vector<int> parents(prompt + tree);
        for (int j = 0; j < prompt; ++j) parents[j] = j - 1;
        for (int j = 0; j < tree; ++j) parents[prompt + j] = j / 2 - 1;
        try {
            const PlanImage image = plan_batch(tables, ids, rows, 2, shape, {}, parents.data());
            expect(prompt < 8'000'000, "more rows than an image counts", prompt);
            const int stride = image.header.tree_stride;
            expect(stride == 2 + (context % 32 + tree - 1) / 32, "a number for every 32 positions of the tree, and one", prompt);
            expect(image.trees.at(static_cast<size_t>(prompt - 1) * stride) == prompt - 1, "the prompt's last position", prompt);
            expect(image.trees.at(static_cast<size_t>(prompt) * stride) == context, "the tree's first position", prompt);
            expect(image.rows.at(prompt).position == -1 - context && image.rows.at(prompt - 1).position == prompt - 1,
                   "rows of a tree and of none", prompt);
            PlanLayout layout = PlanLayout::first();
            layout.grow(image.least());
            layout.grow_plain(image.plain);
            expect(layout.holds(image.least()), "a layout holds it", prompt);
            if (prompt == 16000) expect(layout.holds(image.plain), "and as many rows of any trees no larger", prompt);
        } catch (const Failure& f) {
            expect(prompt > 8'000'000 && f.status == SATORI_HIP_E_OVERFLOW, "rows that follow one another may be any number", prompt);
        }
    }
    if (failures) return 1;
    std::puts("ok");
    return 0;
}
