// page_groups.h -- which sequences of a batch share their first pages (host only;
// defined in pages.hip, used by crane_hip_group_prefixes and the paged cache manager).
#pragma once

#include <stdint.h>

#include <vector>

namespace crane {

struct PageList {
    const int32_t* ids;
    size_t n;
};

struct PageGroups {
    std::vector<int32_t> shared;     // pages each list shares with its group (0: none)
    std::vector<int32_t> start{0};   // group g: members[start[g] .. start[g + 1])
    std::vector<int32_t> members;
    int count() const { return (int)start.size() - 1; }
};

// The groups whose members read the fewest pages: a group of n lists with c leading
// pages in common reads (n - 1) c pages fewer than its members alone.
PageGroups group_pages(const std::vector<PageList>& lists);

}  // namespace crane
