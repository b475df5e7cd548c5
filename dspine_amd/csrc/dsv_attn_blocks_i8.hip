// The kernels of attention over selected blocks of the int8 caches.
#include "dsv_attn.h"

namespace dsv {

template void launch_attn<DSV_BF16, DSV_I8, true>(const AttnParams&, const AttnShape&, unsigned, hipStream_t);
template void launch_attn<DSV_F16, DSV_I8, true>(const AttnParams&, const AttnShape&, unsigned, hipStream_t);

}  // namespace dsv
