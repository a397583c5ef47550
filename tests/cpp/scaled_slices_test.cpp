// Host-only test of the K split of the 8-bit products: the slices of a tile, as the CTAs of a cluster take them, start where
// the one before ends, hold at least two K blocks each where the planner makes a split, differ by one block at most, and cover
// the tile's K blocks once.
// Build: g++ -std=c++17 -I composable_kernel_b200/csrc tests/cpp/scaled_slices_test.cpp
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#include "ckb_scaled_plan.h"

using namespace ckb;

static long g_checks = 0;

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

static void check(int32_t kb0, int32_t kb1, int ksplit)
{
    int32_t at = kb0, shortest = kb1 - kb0, longest = 0;
    for(int r = 0; r < ksplit; ++r)
    {
        ScaledItem it{};
        it.u0 = 1, it.v0 = 2, it.u_end = 3, it.v_end = 4, it.group = 5;
        it.kb0 = kb0, it.kb1 = kb1;
        scaled_slice(&it, r, ksplit);
        REQUIRE(it.kb0 == at && it.kb1 >= it.kb0);
        REQUIRE(it.u0 == 1 && it.v0 == 2 && it.u_end == 3 && it.v_end == 4 && it.group == 5);
        shortest = std::min(shortest, it.kb1 - it.kb0);
        longest  = std::max(longest, it.kb1 - it.kb0);
        at       = it.kb1;
    }
    REQUIRE(at == kb1);
    REQUIRE(longest - shortest <= 1);
    if(kb1 - kb0 >= 2 * ksplit)
        REQUIRE(shortest >= 2);
}

int main()
{
    for(const int ksplit : {1, 2, 4, 8})
    {
        for(int n = 0; n <= 300; ++n)
            for(const int first : {0, 1, 77})
                check(first, first + n, ksplit);
        check(0, 0x7ffff000 / SCALED_BLOCK, ksplit); // the longest K
        check(0, 0x7fffffff, ksplit);
    }
    // every split that the planner makes gives each CTA two K blocks at least
    long splits = 0;
    for(int M = 1; M <= 128; M += 9)
        for(int num_kb = 1; num_kb <= 70; ++num_kb)
            for(const int pin : {0, 2, 4, 8})
            {
                ScaledPlanInput in{};
                in.M = M, in.N = 512, in.num_kb = num_kb, in.mode = SCALED_PLAIN, in.groups = 1;
                in.a_block = 1, in.b_block = 128, in.sm_count = 148;
                in.cluster_cap[0] = 64, in.cluster_cap[1] = 32, in.cluster_cap[2] = 16;
                if(pin)
                    in.cols = 16, in.cg = 1, in.ksplit = pin;
                ScaledPlan p;
                if(!plan_scaled(in, &p))
                {
                    REQUIRE(pin && num_kb < 2 * pin);
                    continue;
                }
                REQUIRE(!pin || p.t.ksplit == pin);
                splits += p.t.ksplit > 1;
                for(int t = 0; t < p.num_tiles; ++t)
                {
                    const ScaledItem it = scaled_item(p.t, t, nullptr);
                    check(it.kb0, it.kb1, p.t.ksplit);
                    REQUIRE(p.t.ksplit == 1 || it.kb1 - it.kb0 >= 2 * p.t.ksplit);
                }
            }
    REQUIRE(splits > 1000);
    std::printf("scaled slice checks passed (%ld splits, %ld checks)\n", splits, g_checks);
    return 0;
}
