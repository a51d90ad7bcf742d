// Cross attention, dkdv, f32 elements: the instantiations of xattn.h (one file each, so that they compile side by side).
#include "xattn.h"

namespace xattn {
XATTN_DEFINE_DKDV(float)
XATTN_DEFINE_SUM(float)
}
