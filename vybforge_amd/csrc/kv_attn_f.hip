// Attention over the 8-bit cache, float32 queries as two fp16 terms (kernel: kv_attn.h).
#include "kv_attn.h"

namespace vybdq {

template <int D, int NCT>
static void launch_rows(const KvAttnArgs &a, dim3 grid, hipStream_t s) {
  hipLaunchKernelGGL((k_kv_attn_rows<D, NCT, true>), grid, dim3(256), 0, s, a);
  if (grid.y > 1)
    hipLaunchKernelGGL((k_kv_attn_join<D, 64 * NCT, true>), dim3(grid.x, 8 * NCT), dim3(256), 0, s, a, static_cast<int>(grid.y));
}

template <int D>
static void launch(int variant, const KvAttnArgs &a, dim3 grid, hipStream_t s) {
  if (variant == 0) hipLaunchKernelGGL((k_kv_attn_keys<D, 1, true>), grid, dim3(256), 0, s, a);
  else if (variant == 1) hipLaunchKernelGGL((k_kv_attn_keys<D, 2, true>), grid, dim3(256), 0, s, a);
  else launch_rows<D, 1>(a, grid, s);
}

void kv_attn_launch_f(int D, int variant, const KvAttnArgs &a, dim3 grid, hipStream_t s) {
  switch (D) {
    case 64: launch<64>(variant, a, grid, s); break;
    case 128: launch<128>(variant, a, grid, s); break;
    case 192: launch<192>(variant, a, grid, s); break;
    default: launch<256>(variant, a, grid, s); break;
  }
}

}  // namespace vybdq
