// Flash attention forward on modified scores (tanh cap, distance bias, prefix masks): fa_fwd3_kernel's MOD forms.
#include "flash_attn_kernels.h"

namespace llmt {

hipError_t launch_mod_fwd(const AttnArgs& a, int D, int mod, unsigned grid, hipStream_t stream) {
#define LLMT_MOD(DD, M)                                                       \
  if (M == kModCap || a.olo)                                                  \
    fa_fwd3_kernel<DD, 2, 1, 4, false, true, M><<<grid, 256, 0, stream>>>(a); \
  else /* (kModCap has no such form: it is not instantiated a second time) */ \
    fa_fwd3_kernel<DD, 2, 1, 4, false, M == kModCap, M><<<grid, 256, 0, stream>>>(a)
  LLMT_MOD_KERNELS(LLMT_MOD)
#undef LLMT_MOD
  return hipGetLastError();
}

}  // namespace llmt
