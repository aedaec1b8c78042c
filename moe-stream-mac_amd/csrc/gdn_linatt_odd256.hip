// Linear attention: the kernels for K' heads of up to 256 channels, sizes that are no multiple of 8.
#include "gdn_linatt.h"

namespace gdn {
namespace la {

GDN_LINATT(odd256, 256, false)

}  // namespace la
}  // namespace gdn
