// The search for a slice's largest values (largest.h) on the CPU, as a group of waves runs it: the bound from 128 sets of the slice's values, counts that the
// waves add up in one word, at the borders of what a group holds, for rows that are alike or have no order.
#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <algorithm>
#include <vector>

#include "../../excalibur_amd/csrc/largest.h"

namespace {

constexpr int kRanked = 128, kMostReadings = 80;

unsigned order_of(float v) {
    if (v != v) return 0xffffffffu;
    v += 0.f;
    unsigned b;
    memcpy(&b, &v, 4);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Group {
    int waves, per_thread, run;  // values of a thread, neighbouring ones of a run
};
Group group_of(int len, int run) {
    if (len <= 512) return {1, 8, run};
    if (len <= 2048) return {1, 32, run};
    return {len <= 8192 ? 4 : len <= 16384 ? 8 : 16, 32, run};
}

// What a group would find: false if it reads the slice too often, or takes too many, or not the `top` first.
bool finds(const std::vector<float>& x, int top, int run, long long* readings) {
    const int len = (int)x.size();
    const Group g = group_of(len, run);
    const int threads = 64 * g.waves, held = threads * g.per_thread;
    std::vector<unsigned> order(held);
    std::vector<float> sets(128, -INFINITY);
    for (int i = 0; i < held; ++i) {
        const float v = i < len ? x[i] : -INFINITY;
        order[i] = order_of(v);
        const int thread = i / run % threads, lane = thread % 64, wave = thread / 64;
        const int set = g.waves > 1 ? wave * (128 / g.waves) + lane / (g.waves / 2) : i / run / threads % 2 * 64 + lane;
        sets[set] = fmaxf(sets[set], v);
    }
    const int want = std::min(top, len);
    std::vector<unsigned> of_sets;
    for (float s : sets) of_sets.push_back(order_of(s));
    std::sort(of_sets.begin(), of_sets.end(), [](unsigned a, unsigned b) { return a > b; });
    int turns = 0;
    const Cut cut = find_cut(of_sets[want - 1], want, kRanked, len, [&](unsigned o, auto takes) {
        if (++turns > kMostReadings) {
            printf("FAILED: %d values, the %d largest: read more than %d times\n", len, top, kMostReadings);
            exit(1);
        }
        unsigned sum = 0;
        for (int w = 0; w < g.waves; ++w) {
            int here = 0, more = 0;
            for (int i = 0; i < g.per_thread / run; ++i)
                for (int e = 0; e < 64 * run; ++e) {
                    const int at = (i * threads + w * 64) * run + e;
                    here += takes(order[at], at);
                    more += order[at] > o;
                }
            sum += two_counts(here, more);
        }
        return sum;
    });
    *readings += turns;
    std::vector<int> taken, first(len);
    for (int i = 0; i < held; ++i)
        if (order[i] > cut.order || (order[i] == cut.order && i < cut.end)) taken.push_back(i);
    for (int i = 0; i < len; ++i) first[i] = i;
    const auto in_front = [&](int a, int b) { return order[a] != order[b] ? order[a] > order[b] : a < b; };
    std::partial_sort(first.begin(), first.begin() + want, first.end(), in_front);
    if ((int)taken.size() < want || (int)taken.size() > kRanked) return false;
    std::partial_sort(taken.begin(), taken.begin() + want, taken.end(), in_front);
    return std::equal(first.begin(), first.begin() + want, taken.begin());
}

}  // namespace

int main() {
    int failures = 0;
    long long readings = 0;
    unsigned seed = 1;
    const auto random = [&] { return (seed = seed * 1664525u + 1013904223u) >> 8; };
    for (int border : {64, 512, 2048, 8192, 16384, 32768})
        for (int len : {border - 1, border, border + 1, border - 300}) {
            if (len < 1 || len > 32768) continue;
            for (int kind = 0; kind < 12; ++kind) {
                std::vector<float> x(len);
                for (int i = 0; i < len; ++i) {
                    const float spread = (float)random() / 65536.f - 128.f;
                    switch (kind) {
                    case 0: x[i] = NAN; break;
                    case 1: x[i] = i % 1000 == 3 ? spread : NAN; break;       // a few numbers
                    case 2: x[i] = i == len / 2 ? spread : NAN; break;
                    case 3: x[i] = i % 2 ? spread : NAN; break;
                    case 4: x[i] = 0.f; break;
                    case 5: x[i] = -65504.f; break;
                    case 6: x[i] = -INFINITY; break;
                    case 7: x[i] = INFINITY; break;
                    case 8: x[i] = i % 7 ? INFINITY : NAN; break;
                    case 9: x[i] = (float)i; break;
                    case 10: x[i] = (float)(random() % 4); break;
                    default: x[i] = i < len - 50 ? 1.f : 0.5f; break;
                    }
                }
                for (int top : {1, 8, 20, 64})
                    for (int run : {4, 8}) {
                        if (finds(x, top, run, &readings)) continue;
                        ++failures;
                        printf("FAILED: %d values of kind %d, the %d largest, runs of %d\n", len, kind, top, run);
                    }
            }
        }
    printf("%d failures, %lld readings\n", failures, readings);
    return failures != 0;
}
