// shared_list.h -- the list of block_kernel's items over shared tokens (kv8_shared.hip): which places a group's items take, and which
// ones say that there is no item. No HIP: also built by the host compiler.
#pragma once

namespace ixg {

// Places 0 .. room; block_kernel reads all of them, so each is written, the last never as an item. Groups that do not overlap have at
// most `room` items; of others, which are not allowed, the numbers are any, and what has no place is left out.

// How many of a group's `items` items, the first at place `first`, are listed.
constexpr int items_listed(int first, int items, int room) {
    return first < 0 || first >= room || items < 0 ? 0 : items < room - first ? items : room - first;
}
// The first place behind all groups' `items`.
constexpr int list_end(int items, int room) { return items < 0 ? 0 : items < room ? items : room; }

}  // namespace ixg
