// Linear attention: the kernels for K' heads of up to 64 channels.
#include "gdn_linatt.h"

namespace gdn {
namespace la {

void pass_d64(const Pass &a, Kind kind, hipStream_t st) {
    if (a.dt == DT_BF16) cols_of(64, a.dv) == 64 ? launch_pass<bf16, 64, 1>(a, kind, st) : launch_pass<bf16, 64, 2>(a, kind, st);
    else cols_of(64, a.dv) == 64 ? launch_pass<float, 64, 1>(a, kind, st) : launch_pass<float, 64, 2>(a, kind, st);
}
void seg_d64(const Seg &a, bool rev, hipStream_t st) {
    if (a.dt == DT_BF16) cols_of(64, a.dv) == 64 ? launch_seg<bf16, 64, 1>(a, rev, st) : launch_seg<bf16, 64, 2>(a, rev, st);
    else cols_of(64, a.dv) == 64 ? launch_seg<float, 64, 1>(a, rev, st) : launch_seg<float, 64, 2>(a, rev, st);
}

}  // namespace la
}  // namespace gdn
