// Linear attention: the kernels for K' heads of up to 128 channels.
#include "gdn_linatt.h"

namespace gdn {
namespace la {

void pass_d128(const Pass &a, Kind kind, hipStream_t st) {
    if (a.dt == DT_BF16) cols_of(128, a.dv) == 64 ? launch_pass<bf16, 128, 1>(a, kind, st) : launch_pass<bf16, 128, 2>(a, kind, st);
    else cols_of(128, a.dv) == 64 ? launch_pass<float, 128, 1>(a, kind, st) : launch_pass<float, 128, 2>(a, kind, st);
}
void seg_d128(const Seg &a, bool rev, hipStream_t st) {
    if (a.dt == DT_BF16) cols_of(128, a.dv) == 64 ? launch_seg<bf16, 128, 1>(a, rev, st) : launch_seg<bf16, 128, 2>(a, rev, st);
    else cols_of(128, a.dv) == 64 ? launch_seg<float, 128, 1>(a, rev, st) : launch_seg<float, 128, 2>(a, rev, st);
}

}  // namespace la
}  // namespace gdn
