// Linear attention: the kernels for K' heads of up to 256 channels.
#include "gdn_linatt.h"

namespace gdn {
namespace la {

void pass_d256(const Pass &a, Kind kind, hipStream_t st) {
    if (a.dt == DT_BF16) launch_pass<bf16, 256, 1>(a, kind, st);
    else launch_pass<float, 256, 1>(a, kind, st);
}
void seg_d256(const Seg &a, bool rev, hipStream_t st) {
    if (a.dt == DT_BF16) launch_seg<bf16, 256, 1>(a, rev, st);
    else launch_seg<float, 256, 1>(a, rev, st);
}

}  // namespace la
}  // namespace gdn
