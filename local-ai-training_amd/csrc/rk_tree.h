// The trees of drafted tokens, as their plan (rk_draft_tree) leaves them.
#pragma once

namespace rk {

constexpr int kTreeNodes = 256;  // of a tree at most: four words of lineage
constexpr int kTreeOff = -2;     // the parent of a node that does not belong to the tree

}  // namespace rk
