// Every place that place_in_list gives lies in the list, whatever its numbers are, and of
// a choice that adds up the places are those of the pages taken, in their order.
#include "gq8_paged_list.hpp"

#include <climits>
#include <cstdio>
#include <vector>

int main()
{
    const int counts[] = {0, 1, 2, 7, 63, 64, 255, 4096, 1 << 20, 1 << 30};
    const int wanteds[] = {INT_MIN, INT_MIN + 1, -(1 << 30), -4096, -255, -8, -7, -2, -1, 0, 1, 2, 8, 255, 1 << 30, INT_MAX};
    const int tops[] = {1, 2, 8, 64, 4096, 1 << 30};
    long outside = 0, tried = 0;
    for (int above : counts)
        for (int before : counts)
            for (int wanted : wanteds)
                for (int top : tops)
                    for (int kind = 0; kind < 4; ++kind) {
                        const int to = gq8::place_in_list(kind & 1, kind & 2, above, before, wanted, top);
                        outside += to < -1 || to >= top;
                        ++tried;
                    }
    long wrong = 0;
    for (unsigned seed = 1; seed <= 200; ++seed) {
        std::vector<int> kinds; // 0 not taken, 1 above, 2 equal
        unsigned x = seed;
        int more = 0, equal = 0;
        for (int i = 0; i < 300; ++i) {
            x = x * 1664525u + 1013904223u;
            kinds.push_back((int) (x >> 24) % 3);
            more += kinds.back() == 1;
            equal += kinds.back() == 2;
        }
        const int wanted = equal / 2, top = more + wanted;
        int above = 0, before = 0, next = 0;
        for (int kind : kinds) {
            const bool taken = kind == 1 || (kind == 2 && before < wanted);
            wrong += gq8::place_in_list(kind == 1, kind == 2, above, before, wanted, top) != (taken ? next : -1);
            next += taken;
            above += kind == 1;
            before += kind == 2;
        }
        wrong += next != top;
    }
    std::printf("tried %ld outside %ld wrong %ld\n", tried, outside, wrong);
    return outside || wrong;
}
