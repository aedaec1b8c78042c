// Linear attention: the kernels for K' heads of up to 128 channels.
#include "gdn_linatt.h"

namespace gdn {
namespace la {

GDN_LINATT(d128, 128, true)

}  // namespace la
}  // namespace gdn
