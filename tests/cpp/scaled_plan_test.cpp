// Host-only test of the work decomposition of the 8-bit products (composable_kernel_b200/csrc/ckb_scaled_plan.h): for a
// sweep of sizes, groupings, offsets and pinned tiles, every tile is decoded exactly as the kernel decodes it, and the test
// asserts that
//   - tiles start inside the problem and lie on their grid;
//   - every element of E that a group owns is covered by exactly one tile of that group, no other one by any (in 16 x 16
//     units where the sizes allow no finer check in reasonable time);
//   - the K blocks of a tile are the group's, and the parts of a K split cover them once;
//   - offsets of any value (negative, too large, decreasing) lead to no row, column or K block outside the tensors;
//   - the launch is no larger than the device and never empty.
// Build: g++ -std=c++17 -I composable_kernel_b200/csrc tests/cpp/scaled_plan_test.cpp
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "ckb_scaled_plan.h"

using namespace ckb;

static long g_checks = 0, g_plans = 0;

#define REQUIRE(cond)                                                             \
    do                                                                            \
    {                                                                             \
        ++g_checks;                                                               \
        if(!(cond))                                                               \
        {                                                                         \
            std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond);         \
            std::exit(1);                                                         \
        }                                                                         \
    } while(0)

static ScaledPlanInput input(int64_t M, int64_t N, int num_kb, int mode, int groups)
{
    ScaledPlanInput in{};
    in.M = M, in.N = N, in.num_kb = num_kb, in.mode = mode, in.groups = groups;
    in.a_block = 1, in.b_block = 128, in.sm_count = 148;
    in.cluster_cap[0] = 74, in.cluster_cap[1] = 36, in.cluster_cap[2] = 17;
    return in;
}

// offsets == nullptr: a plain product
static void check(const ScaledPlanInput& in, const std::vector<int32_t>& offsets)
{
    ScaledPlan p;
    if(!plan_scaled(in, &p))
        return;
    ++g_plans;
    const ScaledTiles& t = p.t;
    REQUIRE(p.grid >= 1 && p.grid % (p.cg == 2 ? 2 : t.ksplit) == 0);
    REQUIRE(t.ksplit > 1 || p.grid <= in.sm_count);
    const int64_t M = in.M, N = in.N;
    std::vector<int> times(static_cast<std::size_t>(M * N), 0); // tiles that cover an element (all groups)
    // the starts of the groups, as the kernel builds them
    std::vector<int32_t> starts{0}, row0, row1;
    int total = p.num_tiles;
    if(in.mode == SCALED_GROUP_ROWS)
    {
        for(int g = 0; g < in.groups; ++g)
        {
            int32_t lo, hi;
            scaled_group_span(offsets.data(), g, static_cast<int32_t>(M), &lo, &hi);
            REQUIRE(0 <= lo && lo <= hi && hi <= M);
            row0.push_back(lo), row1.push_back(hi);
            starts.push_back(starts.back() + scaled_group_tiles(t, hi - lo) * (t.swapped ? t.tiles_u : t.tiles_v));
        }
        total = starts.back();
        REQUIRE(total <= p.num_tiles);
    }
    else
        REQUIRE(total == in.groups * t.tiles_u * t.tiles_v);
    if(t.ksplit > 1)
    {
        REQUIRE(p.grid == total * t.ksplit && in.num_kb >= 2 * t.ksplit);
    }
    std::vector<int> per_group(in.groups, 0);
    for(int i = 0; i < total; ++i)
    {
        const ScaledItem it = in.mode == SCALED_GROUP_ROWS ? scaled_group_item(t, i, starts.data(), row0.data(), row1.data())
                                                           : scaled_item(t, i, offsets.data());
        REQUIRE(it.group >= 0 && it.group < in.groups);
        REQUIRE(it.kb0 >= 0 && it.kb0 <= it.kb1 && it.kb1 <= in.num_kb);
        ++per_group[it.group];
        if(in.mode == SCALED_GROUP_K)
        {
            int32_t lo, hi;
            scaled_group_span(offsets.data(), it.group, in.num_kb, &lo, &hi);
            REQUIRE(it.kb0 == lo && it.kb1 == hi);
        }
        else
            REQUIRE(it.kb0 == 0 && it.kb1 == in.num_kb);
        REQUIRE(it.u0 >= 0 && it.u0 < it.u_end && it.v0 >= 0 && it.v0 < it.v_end);
        REQUIRE(it.u_end <= t.ext_u && it.v_end <= t.ext_v);
        if(in.mode == SCALED_GROUP_ROWS)
            REQUIRE((t.swapped ? it.v_end : it.u_end) == row1[it.group] && (t.swapped ? it.v0 : it.u0) >= row0[it.group]);
        const int u1 = std::min<int>(it.u0 + t.u_rows, it.u_end), v1 = std::min<int>(it.v0 + t.width, it.v_end);
        for(int u = it.u0; u < u1; ++u)
            for(int v = it.v0; v < v1; ++v)
                ++times[t.swapped ? static_cast<int64_t>(v) * N + u : static_cast<int64_t>(u) * N + v];
    }
    if(in.mode == SCALED_GROUP_K)
        for(int g = 0; g < in.groups; ++g)
            REQUIRE(per_group[g] == t.tiles_u * t.tiles_v);
    for(int64_t m = 0; m < M; ++m)
    {
        int want = in.mode == SCALED_GROUP_K ? in.groups : 1;
        if(in.mode == SCALED_GROUP_ROWS)
        {
            want = 0;
            for(int g = 0; g < in.groups; ++g)
                want += row0[g] <= m && m < row1[g];
        }
        for(int64_t n = 0; n < N; ++n)
            if(times[m * N + n] != want)
                REQUIRE(times[m * N + n] == want);
        ++g_checks;
    }
}

int main()
{
    std::mt19937 rng(1);
    auto draw = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
    struct Pin
    {
        int cols, cg, ksplit;
    };
    const Pin pins[] = {{0, 0, 0}, {128, 2, 1}, {192, 2, 1}, {224, 2, 1}, {256, 2, 1}, {16, 1, 1}, {32, 1, 2}, {64, 1, 4}, {128, 1, 8}, {128, 1, 1}};
    for(const Pin& pin : pins)
        for(int round = 0; round < 40; ++round)
        {
            const int64_t M = draw(1, round % 4 == 0 ? 1500 : 300), N = draw(1, round % 4 == 1 ? 2600 : 500);
            auto pinned = [&](ScaledPlanInput in) {
                in.cols = pin.cols, in.cg = pin.cg, in.ksplit = pin.ksplit;
                in.a_mn = draw(0, 3) == 0, in.b_mn = draw(0, 1);
                in.a_block = draw(0, 1) ? 1 : 128, in.b_block = draw(0, 1) ? 1 : 128;
                return in;
            };
            check(pinned(input(M, N, draw(1, 60), SCALED_PLAIN, 1)), {});
            const int groups = draw(1, 12);
            for(int kind = 0; kind < 3; ++kind) // sorted; with empty groups and rows in front and behind; anything
            {
                const int num_kb = draw(1, 20);
                for(const int mode : {SCALED_GROUP_ROWS, SCALED_GROUP_K})
                {
                    const int extent = mode == SCALED_GROUP_ROWS ? static_cast<int>(M) : num_kb;
                    std::vector<int32_t> offsets(groups + 1);
                    for(auto& o : offsets)
                        o = kind == 2 ? draw(-extent - 5, 2 * extent + 5) : draw(0, extent);
                    if(kind != 2)
                        std::sort(offsets.begin(), offsets.end());
                    if(kind == 0)
                        offsets.front() = 0, offsets.back() = extent;
                    if(kind == 2 && round % 2)
                        offsets[draw(0, groups)] = draw(0, 1) ? 0x7fffffff : -0x7fffffff - 1;
                    ScaledPlanInput in = pinned(input(M, N, num_kb, mode, groups));
                    if(mode == SCALED_GROUP_ROWS)
                        in.a_mn = false, in.a_block = 1;
                    check(in, offsets);
                }
            }
        }
    // more tiles than the kernel counts: refused
    ScaledPlan p;
    REQUIRE(!plan_scaled(input(0x7ffff000ll, 0x7ffff000ll, 1, SCALED_PLAIN, 1), &p));
    REQUIRE(g_plans > 1500);
    std::printf("scaled plan checks passed (%ld plans, %ld checks)\n", g_plans, g_checks);
    return 0;
}
