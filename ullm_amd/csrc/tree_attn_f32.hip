// attn_tree over f32 caches (tree_attn.hpp).
#include "tree_attn.hpp"

namespace ullm {
void launch_tree_f32(const TreeCall &c) { launch_dims<F32, ULLM_DT_F32>(c); }
}  // namespace ullm
