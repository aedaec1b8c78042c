// Linear attention: the kernels for K' heads of up to 64 channels.
#include "gdn_linatt.h"

namespace gdn {
namespace la {

GDN_LINATT(d64, 64, true)

}  // namespace la
}  // namespace gdn
