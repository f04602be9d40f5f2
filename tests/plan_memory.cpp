// The memory that a batch's plan asks for and the ranges it counts in (plan_batch of satori_amd/csrc/pages.cpp), one check a
// run, named by the argument; built with the sanitizers and run by tests/test_plan_memory.py.
#include <algorithm>
#include <chrono>
#include <climits>
#include <cstdio>
#include <cstring>
#include <future>
#include <random>
#include <shared_mutex>
#include <string>
#include <thread>
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

// Every (row, key/value head, query head) sees each of its positions once, in the page that its table names, in as many parts as
// its row says.
void check_division(const PageTables& tables, const std::vector<int>& sequences, const std::vector<int>& fresh,
                    const PlanShape& shape, const PlanImage& image) {
    std::vector<int> sequence_of;
    for (size_t i = 0; i < sequences.size(); ++i) sequence_of.insert(sequence_of.end(), fresh[i], sequences[i]);
    expect(sequence_of.size() == image.rows.size(), "rows");
    const int P = tables.page_tokens(), heads = shape.kv_heads * shape.group;
    std::vector<int64_t> seen(image.rows.size() * heads), sums(seen.size());
    std::vector<int> parts(seen.size());
    for (int wide = 0; wide < 2; ++wide)
        for (const PlanItem& item : wide ? image.wide : image.narrow)
            for (int p = item.pair; p < item.pair + item.pairs; ++p) {
                const PlanRow& row = image.list.at(item.rows + p / shape.group);
                const size_t at = static_cast<size_t>(row.row) * heads + item.kv * shape.group + p % shape.group;
                parts.at(at)++;
                expect(item.slot < row.slots, "a part's number");
                expect(row.slots == 1 || row.slot + row.slots <= image.header.partials, "a part's memory");
                const int end = std::min(item.first + item.tokens, row.position + 1);
                for (int t = item.first; t < end; t += P - t % P) {
                    const int next = std::min(end, t + P - t % P);
                    expect(image.pages.at(item.pages + t / P - item.first / P) == tables.table(sequence_of[row.row]).at(t / P),
                           "the page of a position");
                    seen[at] += next - t;
                    sums[at] += (static_cast<int64_t>(t) + next - 1) * (next - t) / 2;
                }
            }
    for (size_t at = 0; at < seen.size(); ++at) {
        const PlanRow& row = image.rows[at / heads];
        const int64_t n = row.position + 1;
        expect(seen[at] == n && sums[at] == n * (n - 1) / 2, "every position once");
        expect(parts[at] == row.slots, "every part once");
    }
}

struct Room {
    PlanLayout layout = PlanLayout::first();
    int64_t partials = 0;
    // As a plan grows with a batch that is set while no step reads it (without the margin that partial results get).
    explicit Room(const PlanImage& image) {
        layout.grow(image.least());
        layout.grow_plain(image.plain);
        partials = std::max<int64_t>(image.header.partials, image.plain_partials);
    }
};

// A plan that held a batch takes every smaller one, whatever its lengths and shared pages: 32 sequences over 2000 positions ask
// for more partial results with 10 positions of their own than with 390.
void smaller_batches() {
    int coarser = 0;
    {
        const PlanShape shape{8, 4, 128, 1024};
        std::vector<PlanImage> images;
        for (const int own : {390, 10}) {
            PageTables tables(4096, 32);
            std::vector<PageMove> moves;
            std::vector<int> batch{tables.open()}, fresh(32, 1);
            int tokens = 2000;
            tables.extend(batch.data(), &tokens, 1, moves);
            batch.resize(32);
            tables.fork(batch[0], 31, batch.data() + 1);
            const std::vector<int> more(32, own);
            tables.extend(batch.data(), more.data(), 32, moves);
            images.push_back(plan_batch(tables, batch.data(), fresh.data(), 32, shape));
            const Room room(images[0]);
            PlanImage image;
            expect(plan_batch_within(tables, batch.data(), fresh.data(), 32, shape, room.layout, room.partials, image), "fits");
            check_division(tables, batch, fresh, shape, image);
        }
        expect(images[1].header.partials > images[0].header.partials, "the shorter batch asks for more");
    }
    std::mt19937 g(97);
    const auto up_to = [&](int n) { return static_cast<int>(g() % (n + 1)); };
    for (int round = 0; round < 60; ++round) {
        const int P = 32 << up_to(3), count = 1 + up_to(20);
        const PlanShape shape{1 + up_to(3), 1 + up_to(7), 32 << up_to(2), round % 2 ? 1 << 22 : 512};
        // Sequences of a tree of forks, batches of them; every one that is no larger than the first fits its room.
        PageTables tables(1 << 14, P);
        std::vector<PageMove> moves;
        std::vector<int> ids{tables.open()};
        int tokens = up_to(6000);
        tables.extend(ids.data(), &tokens, 1, moves);
        while (static_cast<int>(ids.size()) < count) {
            int made = 0;
            tables.fork(ids[up_to(static_cast<int>(ids.size()) - 1)], 1, &made);
            tokens = up_to(3) ? up_to(700) : up_to(6000);
            tables.extend(&made, &tokens, 1, moves);
            ids.push_back(made);
        }
        std::vector<int> fresh(count);
        for (int i = 0; i < count; ++i) fresh[i] = std::min(tables.tokens(ids[i]), up_to(1) ? 1 : up_to(60));
        const Room room(plan_batch(tables, ids.data(), fresh.data(), count, shape));
        for (int smaller = 0; smaller < 6; ++smaller) {
            for (int i = 0; i < count; ++i) {
                const int least = tables.tokens(ids[i]) - up_to(400) * up_to(1);
                if (least >= fresh[i] && least > 0) tables.truncate(ids[i], least);
                if (!up_to(5) && fresh[i] > 0) --fresh[i];
            }
            PlanImage image;
            const bool fits = plan_batch_within(tables, ids.data(), fresh.data(), count, shape, room.layout, room.partials, image);
            expect(fits, "a smaller batch fits");
            if (fits) check_division(tables, ids, fresh, shape, image);
            const PlanImage usual = plan_batch(tables, ids.data(), fresh.data(), count, shape);
            coarser += !room.layout.holds(usual.least()) || usual.header.partials > room.partials;
        }
        // The rows of the batch dealt out otherwise, over sequences that share nothing.
        const PlanImage plain = plan_batch(tables, ids.data(), fresh.data(), count, shape, kPlainDivision);
        check_division(tables, ids, fresh, shape, plain);
        expect(plain.plain.rows >= plain.least().rows && plain.plain.narrow >= plain.least().narrow &&
                   plain.plain.wide >= plain.least().wide && plain.plain.runs >= plain.least().runs &&
                   plain.plain.pages >= plain.least().pages && plain.plain.list >= plain.least().list &&
                   plain.plain_partials >= plain.header.partials,
               "what plain divisions take");
    }
    expect(coarser > 10, "some had to be divided otherwise");
    // What cannot fit is refused.
    PageTables tables(4096, 32);
    std::vector<PageMove> moves;
    const int s = tables.open(), tokens = 3000, rows = 3000, one = 1;
    tables.extend(&s, &tokens, 1, moves);
    const Room room(plan_batch(tables, &s, &one, 1, kShape));
    PlanImage image;
    expect(!plan_batch_within(tables, &s, &rows, 1, kShape, room.layout, room.partials, image), "more rows do not fit");
}

// As many positions as a cache can count.
void longest() {
    const PlanShape shape{1, 1, 128, 128};
    PageTables tables(INT32_MAX / 256, 256);
    std::vector<PageMove> moves;
    const int s = tables.open(), tokens = INT32_MAX / 256 * 256, one = 1;
    tables.extend(&s, &tokens, 1, moves);
    for (const bool plain : {false, true}) {
        const PlanImage image = plan_batch(tables, &s, &one, 1, shape, plain ? kPlainDivision : PlanDivision{});
        expect(image.rows[0].slots == 2048, "chunks of 2^20 positions");
        expect(plain == false || image.plain_partials >= image.header.partials, "their partial results");
        check_division(tables, {s}, {1}, shape, image);
    }
}

// A list is read while a plan is being made, which holds the tables without changing them.
void readers() {
    satori_hip_pages* pages = nullptr;
    expect(satori_hip_pages_create(8, 32, &pages) == SATORI_HIP_OK, "create");
    int sequence = -1, tokens = -1, count = -1, free_pages = -1;
    expect(satori_hip_pages_open(pages, &sequence) == SATORI_HIP_OK, "open");
    PageTables& tables = page_tables(pages);
    std::promise<void> held, release;
    std::thread plan([&] {
        const std::shared_lock<std::shared_mutex> lock(tables.lock);
        held.set_value();
        release.get_future().wait();
    });
    held.get_future().wait();
    auto read = std::async(std::launch::async, [&] {
        return satori_hip_pages_sequence(pages, sequence, &tokens, nullptr, 0, &count) == SATORI_HIP_OK &&
               satori_hip_pages_free_count(pages, &free_pages) == SATORI_HIP_OK;
    });
    const bool done = read.wait_for(std::chrono::seconds(20)) == std::future_status::ready;
    expect(done, "a read beside a plan");
    release.set_value();
    plan.join();
    expect(read.get() && tokens == 0 && count == 0 && free_pages == 8, "what it reads");
    satori_hip_pages_destroy(pages);
}

}  // namespace

int main(int count, char** arguments) {
    const std::string what = count > 1 ? arguments[1] : "";
    if (what == "partials")
        partials();
    else if (what == "smaller")
        smaller_batches();
    else if (what == "longest")
        longest();
    else if (what == "readers")
        readers();
    else
        expect(false, "no such check");
    if (failures) return 1;
    std::puts("ok");
    return 0;
}
