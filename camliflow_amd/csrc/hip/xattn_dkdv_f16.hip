// Cross attention, dkdv, f16 elements: the instantiations of xattn.h (one file each, so that they compile side by side).
#include "xattn.h"

namespace xattn {
XATTN_DEFINE_DKDV(_Float16)
XATTN_DEFINE_SUM(_Float16)
}
