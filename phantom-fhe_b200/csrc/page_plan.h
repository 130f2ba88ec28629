// page_plan.h - host side of b2_pages_move: the order in which the pages of a pool are read and written so that every page that
// is read still holds what it held before the call. No CUDA in here: the tests compile it for the host.
#pragma once
#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <vector>

namespace b2 {

// A step stores the words of page `src` to page `dst`. Two names stand for no page: PAGE_ZERO as a source is a page of zeros,
// PAGE_KEPT is a value that a thread holds on to: as a destination it takes the source's word, as a source it gives it back.
constexpr int PAGE_BATCH = 4;  // steps whose loads go out before their stores
constexpr uint32_t PAGE_ZERO = 0xFFFFFFFFu, PAGE_KEPT = 0xFFFFFFFEu, PAGE_MAX = 0xFFFFFFF0u;
struct PageStep {
    uint32_t src, dst;
};

// Runs of steps that may be worked on at the same time; within a run the order counts, and a value is kept within one run only.
struct PagePlan {
    std::vector<PageStep> steps;
    std::vector<uint32_t> ends;  // of the runs, in steps
};

// "new dst[i] := old src[i] for all i at once" (dst distinct, src[i] < 0: zeros) as runs of at most `cap` steps (cap >= 3), the
// runs of one component one after the other. A page has one writer at most, so that the moves of a pool onto itself form trees
// that hang off at most one cycle each: the moves whose destination nobody reads any more go first, which frees their source to
// be written; what then is left are cycles, opened by keeping one page. A cycle longer than a run is closed early, with the kept
// page in its last place, and goes on from there: one page more is moved. `apart`: the sources are in another pool.
// Returns the index of the first run of each component in `first` (runs of different components touch no common page).
inline PagePlan plan_pages(size_t n, const int64_t *dst, const int64_t *src, bool apart, size_t cap, std::vector<uint32_t> &first) {
    PagePlan p;
    p.steps.reserve(n + n / 2 + 1);
    std::vector<uint32_t> op;
    op.reserve(n);
    for (uint32_t i = 0; i < n; i++)
        if (apart || dst[i] != src[i]) op.push_back(i);
    const auto source = [&](uint32_t i) { return src[i] < 0 ? PAGE_ZERO : (uint32_t)src[i]; };
    bool free_of_order = apart;
    std::vector<int64_t> pages;  // the destinations, sorted: a page's place in them names it below
    if (!apart) {
        for (uint32_t i : op) pages.push_back(dst[i]);
        std::sort(pages.begin(), pages.end());
        free_of_order = std::none_of(op.begin(), op.end(), [&](uint32_t i) { return src[i] >= 0 && std::binary_search(pages.begin(), pages.end(), src[i]); });
    }
    if (free_of_order) {  // steps of one source side by side: it is read once for each batch of a run
        std::stable_sort(op.begin(), op.end(), [&](uint32_t a, uint32_t b) { return source(a) < source(b); });
        for (uint32_t i : op) {
            first.push_back((uint32_t)p.ends.size());
            p.steps.push_back(PageStep{source(i), (uint32_t)dst[i]});
            p.ends.push_back((uint32_t)p.steps.size());
        }
        return p;
    }
    const auto place = [&](int64_t page) -> int64_t {  // among the destinations; -1: only read, or zeros
        if (page < 0) return -1;
        const auto it = std::lower_bound(pages.begin(), pages.end(), page);
        return it != pages.end() && *it == page ? it - pages.begin() : -1;
    };
    const size_t m = op.size();
    std::vector<uint32_t> writer(m), readers(m, 0), comp(m);
    for (uint32_t k = 0; k < m; k++) comp[k] = k;
    const auto root = [&](uint32_t k) {
        while (comp[k] != k) k = comp[k] = comp[comp[k]];
        return k;
    };
    std::vector<int64_t> from(m);  // by place: the place of the source of the move that writes it
    for (uint32_t i : op) {
        const size_t k = (size_t)place(dst[i]);
        writer[k] = i, from[k] = place(src[i]);
        if (from[k] >= 0) {
            readers[from[k]]++;
            comp[root((uint32_t)k)] = root((uint32_t)from[k]);
        }
    }
    // places in the order in which they are written, the leaves first; -1 - k opens the cycle through place k
    std::vector<int64_t> order;
    std::vector<uint8_t> done(m, 0);
    order.reserve(m);
    for (uint32_t k = 0; k < m; k++)
        if (!readers[k]) order.push_back(k), done[k] = 1;
    for (size_t at = 0; at < order.size(); at++) {
        const int64_t f = from[order[at]];
        if (f >= 0 && --readers[f] == 0 && !done[f]) order.push_back(f), done[f] = 1;
    }
    for (uint32_t k = 0; k < m; k++)
        if (!done[k]) {
            order.push_back(-1 - (int64_t)k);
            for (int64_t j = k; !done[j]; j = from[j]) done[j] = 1;
        }
    // by component; within one the order stays
    std::vector<std::pair<uint32_t, uint32_t>> by(order.size());
    for (uint32_t a = 0; a < order.size(); a++) by[a] = {root((uint32_t)(order[a] < 0 ? -1 - order[a] : order[a])), a};
    std::sort(by.begin(), by.end());
    size_t run = 0;  // steps in the open run
    const auto close = [&] {
        if (run) p.ends.push_back((uint32_t)p.steps.size());
        run = 0;
    };
    const auto step = [&](uint32_t s, uint32_t d) { p.steps.push_back(PageStep{s, d}), run++; };
    for (size_t a = 0; a < by.size(); a++) {
        if (!a || by[a].first != by[a - 1].first) {
            close();
            first.push_back((uint32_t)p.ends.size());
        }
        const int64_t k = order[by[a].second];
        if (k >= 0) {
            if (run == cap) close();
            step(source(writer[k]), (uint32_t)pages[k]);
            continue;
        }
        const int64_t open = -1 - k;
        int64_t at = open;  // the next place to be written; its old value is the kept one
        do {
            if (run + 3 > cap) close();
            step((uint32_t)pages[at], PAGE_KEPT);
            while (from[at] != open && run + 1 < cap) {
                step((uint32_t)pages[from[at]], (uint32_t)pages[at]);
                at = from[at];
            }
            step(PAGE_KEPT, (uint32_t)pages[at]);
        } while (from[at] != open);
    }
    close();
    return p;
}

// Packs the runs of a plan into launches of at most `cap` steps, each spread over lanes that are worked on at the same time:
// as many whole components as fit, `lanes_of(components)` lanes at most, about equally long. The runs of a longer component
// follow one another, each in a launch of its own. emit(first step, ends of the lanes counted from it).
template <class Lanes, class Emit>
void pack_pages(const PagePlan &p, const std::vector<uint32_t> &first, size_t cap, Lanes &&lanes_of, Emit &&emit) {
    const auto begin = [&](size_t run) { return run ? p.ends[run - 1] : 0u; };
    const auto runs_end = [&](size_t k) { return k + 1 < first.size() ? (size_t)first[k + 1] : p.ends.size(); };
    std::vector<uint32_t> ends;
    for (size_t k = 0; k < first.size();) {
        if (runs_end(k) - first[k] > 1) {
            for (size_t r = first[k]; r < runs_end(k); r++) {
                ends.assign(1, p.ends[r] - begin(r));
                emit(begin(r), ends);
            }
            k++;
            continue;
        }
        size_t to = k;
        const uint32_t b = begin(first[k]);
        while (to < first.size() && runs_end(to) - first[to] == 1 && p.ends[first[to]] - b <= cap) to++;
        const uint64_t steps = p.ends[first[to - 1]] - b, lanes = lanes_of(to - k);
        ends.clear();
        for (size_t j = k; j < to; j++) {
            const uint32_t e = p.ends[first[j]] - b;
            if (j + 1 == to || e * lanes >= steps * (ends.size() + 1)) ends.push_back(e);
        }
        emit(b, ends);
        k = to;
    }
}

}  // namespace b2
