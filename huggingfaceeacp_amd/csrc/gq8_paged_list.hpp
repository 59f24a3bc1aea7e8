// gq8_paged_list.hpp -- where a chosen page stands in its row's list.
//
// Plain C++ so the host tests can build it without HIP; GQ8_HD (of gq8_numerics.hpp)
// makes it a host and device function under hipcc.
#pragma once

#ifndef GQ8_HD
#define GQ8_HD inline
#endif

namespace gq8 {

// A page ranked above the last one to take (`more`), or equal to it (`equal`), of which the
// lowest `wanted` are taken: `above` pages of the first kind and `before` of the second
// precede it.  -1: it is not taken.  Numbers that belong to no choice (ranks that
// another call wrote over, of which more are always taken than a list holds) place
// nothing outside a list of `top`.
GQ8_HD int place_in_list(bool more, bool equal, int above, int before, int wanted, int top)
{
    const int to = above + (before < wanted ? before : wanted);
    return (more || (equal && before < wanted)) && (unsigned) to < (unsigned) top ? to : -1; // below zero: past any top
}

} // namespace gq8
