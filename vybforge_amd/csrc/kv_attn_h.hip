// Attention over the 8-bit cache, fp16 and bf16 queries (kernel: kv_attn.h).
#include "kv_attn.h"

namespace vybdq {

template <int D>
static void launch(int variant, const KvAttnArgs &a, dim3 grid, hipStream_t s) {
  if (variant == 0) hipLaunchKernelGGL((k_kv_attn<D, 1, 4, 1, false>), grid, dim3(256), 0, s, a);
  else if (variant == 1) hipLaunchKernelGGL((k_kv_attn<D, 2, 4, 1, false>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((k_kv_attn<D, 2, 1, 4, false>), grid, dim3(256), 0, s, a);
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
