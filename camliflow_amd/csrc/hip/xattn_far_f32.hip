// Cross attention, both adjoints of far rows, f32 elements: the instantiations of xattn.h (one file each, so that they compile side by side).
#include "xattn.h"

namespace xattn {
XATTN_DEFINE_FAR(float)
}
