// Of many keys, a threshold that lets at least the k first through and no more than
// can be sorted. A key is an order (the larger first, 0: no key) and among equal ones a
// place (the lower first; all different). The search sees no keys, only numbers of them.
//
// Compiles as host C++ and as HIP device code (KTH_KEY_FN).
#pragma once
#include <stdint.h>

#ifndef KTH_KEY_FN
#define KTH_KEY_FN static inline
#endif

namespace wpcg {

struct KthKey {
    uint32_t order;
    int place;  // of that order the keys up to here
};
// from(o): how many keys have an order from o on; at(o, p): how many have the order o and
// a place up to p. least: the lowest order of those that are known to hold the k first;
// they are more than `most` >= k. Places are below `places`.
template <class FROM, class AT>
KTH_KEY_FN KthKey kth_key(int k, int most, uint32_t least, int places, FROM from, AT at)
{
    // the k-th key's order: mostly the least, else by bisection, which may end above it
    // once no more than `most` are left. `above`: no more than the keys above `of`, and
    // fewer than k.
    uint32_t of = least;
    int above = from(of + 1);
    if (above >= k) {
        of = 0;
        above = 0;
        bool few = false;
        for (int bit = 31; bit >= 0 && !few; bit--) {
            const int n = from(of | 1u << bit);
            if (n < k) above = n;
            else of |= 1u << bit;
            few = n >= k && n <= most;
        }
        if (!few) above = from(of + 1);
    }
    // of this order the lowest places
    int first = 0, last = places - 1;
    while (first < last) {
        const int mid = (int)((uint32_t)(first + last) / 2), n = above + at(of, mid);
        if (n < k) first = mid + 1;
        else last = mid;
        if (n >= k && n <= most) break;
    }
    return {of, last};
}

}  // namespace wpcg
