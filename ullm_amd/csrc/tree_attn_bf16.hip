// attn_tree over bf16 caches (tree_attn.hpp).
#include "tree_attn.hpp"

namespace ullm {
void launch_tree_bf16(const TreeCall &c) { c.f32_out ? launch_dims<BF16, ULLM_DT_F32>(c) : launch_dims<BF16, ULLM_DT_BF16>(c); }
}  // namespace ullm
