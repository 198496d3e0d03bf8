// How the group norm kernels divide their work: pure host arithmetic on sizes.
#pragma once

#include <algorithm>
#include <cstdint>

namespace mfh {

constexpr int GROUP_NORM_POSITIONS_LIMIT = 1 << 30;  // the kernels' row numbers go a few thousand beyond the last

struct GroupNormShape {
    std::int64_t n;
    int positions, channels, groups;
};

// A block is what one workgroup takes of a row: `groups` whole groups, or, where a group is wider than a
// workgroup, one of `parts` pieces of a group. Threads lie over it in `lanes` side by side, a pack of `vw`
// channels each (those beyond the block idle), threads / lanes rows at a time (those beyond idle). Lanes are a
// power of two up to 32, so that the rows of a wave join across its lanes; from 33 packs on as many as there are.
struct GroupNormPlan {
    bool held;       // a workgroup holds its block over all positions
    int threads;
    int vw;          // channels of a pack: a pack lies within a row and within a block
    int per;         // channels of a group
    int groups;      // whole groups of a block (1 when parts > 1)
    int parts;       // blocks of a group
    int width;       // channels of a block (the last part of a group may hold fewer)
    int blocks;      // blocks of a sample
    int lanes;
    int runs, rows;  // split: runs of a sample's positions, and positions of a run
    std::int64_t grid() const { return blocks * static_cast<std::int64_t>(held ? 1 : runs); }  // workgroups of a sample
};

constexpr int GROUP_NORM_BLOCK_GROUPS = 256;  // at most, so that a thread a group suffices
constexpr int GROUP_NORM_SPLIT_THREADS = 256, GROUP_NORM_SPLIT_AHEAD = 4;  // rows that a thread reads ahead
constexpr int GROUP_NORM_COLUMN_SPAN = 64, GROUP_NORM_COLUMN_RUNS = 16;  // columns and runs of rows of a summing workgroup
constexpr std::int64_t GROUP_NORM_LAUNCH_THREADS = (1LL << 32) - 1;      // threads of a launch, at most

// Packs that a thread holds of x (and, backward, of dy). 256 threads take up to 8 in turn: 26 single elements each
// took 9.2 and 13.1 us forward and backward where four times the threads with 7 each took 7.9 and 9.2 (33 x 405 x
// 90 float16). 1024 threads hold as many as leave them their 128 registers without spills.
constexpr int group_norm_hold(int type_size, int vw, bool backward, int threads) {
    if (threads <= 256) return 8;
    if (vw * type_size < 16) return 32;
    return type_size == 2 && backward ? 5 : 8;
}

// A pack of 16 bytes, a 4-byte pair of a half type, or one element: the widest that divides `channels`.
inline int group_norm_pack(int type_size, int channels) {
    const int wide = 16 / type_size;
    if (channels % wide == 0) return wide;
    return type_size == 2 && channels % 2 == 0 ? 2 : 1;
}

inline int group_norm_lanes(int packs) {
    if (packs > 32) return packs;
    int lanes = 1;
    while (lanes < packs) lanes *= 2;
    return lanes;
}

inline void group_norm_block(const GroupNormShape& s, int groups, int vw, GroupNormPlan* plan) {
    plan->vw = vw, plan->per = s.channels / s.groups, plan->groups = groups, plan->parts = 1;
    plan->width = groups * plan->per, plan->blocks = s.groups / groups;
    plan->lanes = group_norm_lanes(plan->width / vw);
}

// Whether `threads` threads hold a block of `groups` groups over all positions.
inline bool group_norm_holds(const GroupNormShape& s, int type_size, bool backward, int groups, int threads,
                             GroupNormPlan* plan) {
    const int width = groups * (s.channels / s.groups), vw = group_norm_pack(type_size, width);
    if (width / vw > threads || groups > GROUP_NORM_BLOCK_GROUPS) return false;
    // Where the blocks leave half of the CUs idle, up to 16 narrow packs a thread: 64 blocks of 32 each took 28 us
    // backward (2 x 4096 x 320 float16), by runs of positions over all CUs 19.
    int hold = group_norm_hold(type_size, vw, backward, threads);
    if (s.n * (s.groups / groups) < 128) hold = std::min(hold, 16);
    if (threads / group_norm_lanes(width / vw) * hold < s.positions) return false;
    group_norm_block(s, groups, vw, plan);
    plan->held = true, plan->threads = threads;
    return true;
}

inline GroupNormPlan group_norm_plan(const GroupNormShape& s, int type_size, bool backward) {
    constexpr int FILL = 256;        // workgroups that fill the CUs
    constexpr int LINE_BYTES = 128;  // a cache line
    constexpr int RUN_GROUPS = 1024; // workgroups of a split pass: four a CU
    GroupNormPlan plan{};
    const int per = s.channels / s.groups;
    // Held: whole groups side by side until a block's row fills a cache line and the block two packs a thread of
    // 256, as long as the blocks fill the CUs.
    for (int groups = 1; groups <= s.groups; ++groups) {
        if (s.groups % groups) continue;
        if (groups > 1 && s.n * (s.groups / groups) < FILL) break;
        if (!group_norm_holds(s, type_size, backward, groups, 256, &plan) &&
            !group_norm_holds(s, type_size, backward, groups, 1024, &plan))
            break;
        if (groups * per * type_size >= LINE_BYTES && static_cast<std::int64_t>(s.positions) * (plan.width / plan.vw) >= 512)
            break;
    }
    if (plan.held) return plan;
    // Split: as many whole groups as a workgroup's row takes, in the widest pack that allows one; else parts.
    plan.threads = GROUP_NORM_SPLIT_THREADS;
    int groups = 0, vw = 0;
    for (const int pack : {group_norm_pack(type_size, s.channels), group_norm_pack(type_size, per)}) {
        if (groups) break;
        vw = pack;
        for (int g = 1; g <= std::min(s.groups, GROUP_NORM_BLOCK_GROUPS); ++g)
            if (s.groups % g == 0 && static_cast<std::int64_t>(g) * per <= plan.threads * vw && (g * per) % vw == 0) groups = g;
    }
    group_norm_block(s, std::max(groups, 1), vw, &plan);
    if (!groups) {
        plan.width = plan.threads * vw;
        plan.parts = (per + plan.width - 1) / plan.width;
        plan.blocks = s.groups * plan.parts;
        plan.lanes = plan.threads;
    }
    const int step = plan.threads / plan.lanes * 2 * GROUP_NORM_SPLIT_AHEAD;  // a thread reads ahead twice at least
    const std::int64_t most = (s.positions + static_cast<std::int64_t>(step) - 1) / step;
    const std::int64_t wanted = std::max<std::int64_t>(1, RUN_GROUPS / (s.n * plan.blocks));
    const std::int64_t count = std::min(most, wanted);
    plan.rows = static_cast<int>((s.positions + count - 1) / count);
    plan.runs = static_cast<int>((s.positions + static_cast<std::int64_t>(plan.rows) - 1) / plan.rows);
    return plan;
}

// Samples that one launch of any of a call's kernels takes: a call with more of them goes in slices of this many.
// A sample takes at most 65536 workgroups of 1024 threads.
inline std::int64_t group_norm_slice(const GroupNormShape& s, const GroupNormPlan& plan, bool backward) {
    std::int64_t threads = plan.grid() * plan.threads;
    if (!plan.held) {
        const std::int64_t tiles = (2LL * s.channels + GROUP_NORM_COLUMN_SPAN - 1) / GROUP_NORM_COLUMN_SPAN;
        const std::int64_t join = backward ? tiles * GROUP_NORM_COLUMN_SPAN * GROUP_NORM_COLUMN_RUNS
                                           : static_cast<std::int64_t>(s.groups) * GROUP_NORM_SPLIT_THREADS;
        threads = std::max(threads, join);
    }
    return GROUP_NORM_LAUNCH_THREADS / threads;
}

}  // namespace mfh
