// attn_tree over f16 caches (tree_attn.hpp).
#include "tree_attn.hpp"

namespace ullm {
void launch_tree_f16(const TreeCall &c) { c.f32_out ? launch_dims<F16, ULLM_DT_F32>(c) : launch_dims<F16, ULLM_DT_F16>(c); }
}  // namespace ullm
