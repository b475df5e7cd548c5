// The attention kernels of the e4m3 caches.
#include "dsv_attn.h"

namespace dsv {

template void launch_attn<DSV_BF16, DSV_E4M3>(const AttnParams&, const AttnShape&, unsigned, hipStream_t);
template void launch_attn<DSV_F16, DSV_E4M3>(const AttnParams&, const AttnShape&, unsigned, hipStream_t);

}  // namespace dsv
