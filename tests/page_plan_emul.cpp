// What pages_move_kernel does with the plans of page_plan.h, word for word on the host: a page is one number. Lanes run one after
// another, last one first; within a lane the loads of `batch` steps come before their stores, as in the kernel.
// Returns the pages read (a run of steps of one source within a batch counts once), -1 where two lanes of a launch touch a page
// that one of them writes, -2 where a launch or a lane is larger than the kernel's parameters.
#include "../phantom-fhe_b200/csrc/page_plan.h"

using namespace b2;

extern "C" long emul_pages(size_t n, const int64_t *dst, const int64_t *src, int apart, size_t cap, size_t lanes, size_t batch, int64_t *pool, size_t pages,
                           const int64_t *other) {
    std::vector<uint32_t> first;
    const PagePlan p = plan_pages(n, dst, src, apart != 0, cap, first);
    long reads = 0;
    bool clash = false, large = false;
    pack_pages(
        p, first, cap, [&](size_t parts) { return std::min(parts, lanes); },
        [&](uint32_t begin, const std::vector<uint32_t> &ends) {
            if (ends.empty() || ends.back() > cap || ends.size() > lanes) large = true;
            std::vector<int> writer(pages, -1), reader(pages, -1);
            for (int pass = 0; pass < 2; pass++)
                for (size_t l = 0; l < ends.size(); l++)
                    for (uint32_t k = l ? ends[l - 1] : 0; k < ends[l]; k++) {
                        const PageStep s = p.steps[begin + k];
                        if (pass == 0 && s.dst != PAGE_KEPT) {
                            clash = clash || (writer[s.dst] >= 0 && writer[s.dst] != (int)l);
                            writer[s.dst] = (int)l;
                        }
                        if (pass == 1 && !apart && s.src < PAGE_KEPT) clash = clash || (writer[s.src] >= 0 && writer[s.src] != (int)l);
                    }
            for (size_t l = ends.size(); l-- > 0;) {
                int64_t kept = -77;
                for (uint32_t k = l ? ends[l - 1] : 0; k < ends[l]; k += batch) {
                    std::vector<int64_t> v(batch, 0);
                    for (size_t u = 0; u < batch && k + u < ends[l]; u++) {
                        const PageStep s = p.steps[begin + k + u];
                        if (s.src >= PAGE_KEPT) continue;
                        v[u] = (apart ? other : pool)[s.src];
                        reads += !(u && p.steps[begin + k + u - 1].src == s.src);
                    }
                    for (size_t u = 0; u < batch && k + u < ends[l]; u++) {
                        const PageStep s = p.steps[begin + k + u];
                        if (s.dst == PAGE_KEPT) kept = v[u];
                        else pool[s.dst] = s.src == PAGE_KEPT ? kept : v[u];
                    }
                }
            }
        });
    return clash ? -1 : large ? -2 : reads;
}

// steps in a batch of the kernel
extern "C" int kernel_batch() { return PAGE_BATCH; }
