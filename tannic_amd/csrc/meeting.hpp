// Parts of a group of rows that blocks leave for each other meet in a tree: `most` parts that lie beside each other are put together by the last of their blocks to
// get there, what comes of them by the last of those that have `most` of these, and so on.  Every meeting counts its blocks in a word of its own.
#pragma once

#include <cstdint>

namespace th {

// The word, among as many as the group has parts, of the meeting whose first member is number `first` of its level; members of a level are `apart` parts from each
// other, most^level.  It is that of the second member's first part (whoever meets is not alone, so there is one): `first` is a multiple of `most`, so the number ends, to the
// base of `most`, in a 1 and as many zeros as the level, and no other meeting of the group has it.  Word 0, where a neighbouring group's last part may lie, is nobody's.
constexpr uint32_t meeting_count(uint32_t first, uint32_t apart) { return (first + 1) * apart; }

}  // namespace th
