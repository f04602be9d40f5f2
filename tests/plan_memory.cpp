// The memory that a batch's plan asks for and the ranges it counts in (plan_batch of satori_amd/csrc/pages.cpp), one check a
// run, named by the argument; built with the sanitizers and run by tests/test_plan_memory.py.
#include <cstdio>
#include <cstring>
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

void expect(bool ok, const char* what) {
    if (!ok && ++failures <= 20) std::fprintf(stderr, "FAILED: %s\n", what);
}

// Key/value heads, query heads of each, pairs of a wide item, bytes of a position of one head.
constexpr PlanShape kShape{8, 4, 128, 512};

// Rows of one slot write the output themselves: they ask for no partial results, and rows of several have the first numbers.
void partials() {
    PageTables tables(4096, 32);
    std::vector<PageMove> moves;
    const int prompt = tables.open(), long_one = tables.open();
    int tokens = 8192;
    tables.extend(&prompt, &tokens, 1, moves);
    PlanImage image = plan_batch(tables, &prompt, &tokens, 1, kShape);
    expect(image.header.joined == 0 && image.header.partials == 0, "a prompt in one chunk joins nothing");
    tokens = 40000;
    tables.extend(&long_one, &tokens, 1, moves);
    const int short_one = tables.open(), batch[3] = {short_one, long_one, prompt}, fresh[3] = {1, 1, 1};
    tokens = 20;
    tables.extend(&short_one, &tokens, 1, moves);
    image = plan_batch(tables, batch, fresh, 3, kShape);
    expect(image.rows[0].slots == 1 && image.rows[0].slot == image.header.partials, "the short one goes behind");
    expect(image.rows[1].slots > 1 && image.rows[1].slot == 0, "the long one comes first");
    int joined = 0;
    for (const PlanRow& r : image.rows) joined += r.slots > 1 ? r.slots : 0;
    expect(image.header.partials == joined, "partial results of the joined rows alone");
}

}  // namespace

int main(int count, char** arguments) {
    const std::string what = count > 1 ? arguments[1] : "";
    if (what == "partials")
        partials();
    else
        expect(false, "no such check");
    if (failures) return 1;
    std::puts("ok");
    return 0;
}
