// Linear attention: the kernels for K' heads of up to 256 channels.
#include "gdn_linatt.h"

namespace gdn {
namespace la {

GDN_LINATT(d256, 256, true)

}  // namespace la
}  // namespace gdn
