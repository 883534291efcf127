#pragma once
#include <hip/hip_runtime.h>

// Which values of a slice are its largest, where a bound alone leaves too many of them: the search counts readings of the slice and knows nothing of how
// they are made, so that it also runs on the host.

// Two counts of a slice's values in one word, which the words of its waves are added up in: each is up to the slice's length, and the upper one takes the
// word's last bit from 32768 on, so the word has no sign.
constexpr int kMostCounted = 0xffff;
__host__ __device__ __forceinline__ unsigned two_counts(int lower, int upper) { return (unsigned)lower | (unsigned)upper << 16; }
__host__ __device__ __forceinline__ int lower_count(unsigned two) { return (int)(two & 0xffffu); }
__host__ __device__ __forceinline__ int upper_count(unsigned two) { return (int)(two >> 16); }

struct Cut {  // the values of a higher order than this one, and of this one those in front of `end`
    unsigned order;
    int end;
};
// A cut that between `want` and `ranked` of a slice's `len` values stand in front of, if `want` of them reach o. (want <= len, want <= ranked.)
// reading(o, takes) is a reading of the slice: two_counts(values with takes(order, index), values of a higher order than o).
// The bound is raised by halves until few enough reach it; where more are alike, as many of these as come first. Every turn of either loop takes something off
// what it halves, whatever the counts are: 32 turns at most of the first, and two for each halving of the second.
template <typename Reading>
__host__ __device__ __forceinline__ Cut find_cut(unsigned o, int want, int ranked, int len, Reading reading) {
    const unsigned first = reading(o, [o](unsigned order, int) { return order >= o; });
    int reach = lower_count(first), above = upper_count(first);
    unsigned most_o = ~0u;
    while (reach > ranked && above >= want && o < most_o) {
        const unsigned up = o + (most_o - o) / 2 + 1;
        const unsigned two = reading(o, [up](unsigned order, int) { return order >= up; });
        if (lower_count(two) < want) {
            most_o = up - 1;
            above = upper_count(two);
        } else {
            o = up;
            reach = lower_count(two);
            above = want;  // or more, unless there is nothing above
            if (o == most_o) above = upper_count(reading(o, [](unsigned, int) { return false; }));
        }
    }
    int begin = 0, end = len;  // of those alike, what stands in front of `end`
    for (int step = 0, n_begin = above, n_end = reach; n_end > ranked && end - begin > 1; ++step) {
        // where they would be spread evenly, and the middle, by turns
        const int even = (end - begin) * ((want + ranked) / 2 - n_begin) / (n_end - n_begin);
        const int to = begin + (step % 2 == 0 && even > 0 && even < end - begin ? even : (end - begin) / 2);
        const int n_to = above + lower_count(reading(o, [o, to](unsigned order, int i) { return order == o && i < to; }));
        if (n_to < want) {
            begin = to;
            n_begin = n_to;
        } else {
            end = to;
            n_end = n_to;
        }
    }
    return Cut{o, end};
}
