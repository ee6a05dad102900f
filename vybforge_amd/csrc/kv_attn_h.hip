// Attention over the 8-bit cache, fp16 and bf16 queries (kernel: kv_attn.h).
#include "kv_attn.h"

namespace vybdq {

template <int D, int NCT>
static void launch_rows(const KvAttnArgs &a, dim3 grid, hipStream_t s) {
  hipLaunchKernelGGL((k_kv_attn_rows<D, NCT, false>), grid, dim3(256), 0, s, a);
  if (grid.y > 1)
    hipLaunchKernelGGL((k_kv_attn_join<D, 64 * NCT, false>), dim3(grid.x, 8 * NCT), dim3(256), 0, s, a, static_cast<int>(grid.y));
}

template <int D>
static void launch(int variant, const KvAttnArgs &a, dim3 grid, hipStream_t s) {
  if (variant == 0) hipLaunchKernelGGL((k_kv_attn_keys<D, 1, false>), grid, dim3(256), 0, s, a);
  else if (variant == 1) hipLaunchKernelGGL((k_kv_attn_keys<D, 2, false>), grid, dim3(256), 0, s, a);
  else if (variant == 2) launch_rows<D, 1>(a, grid, s);
  else if constexpr (D == 128) launch_rows<D, 2>(a, grid, s);
}

void kv_attn_launch_h(int D, int variant, const KvAttnArgs &a, dim3 grid, hipStream_t s) {
  switch (D) {
    case 64: launch<64>(variant, a, grid, s); break;
    case 128: launch<128>(variant, a, grid, s); break;
    case 192: launch<192>(variant, a, grid, s); break;
    default: launch<256>(variant, a, grid, s); break;
  }
}

}  // namespace vybdq
