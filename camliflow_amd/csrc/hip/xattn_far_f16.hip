// Cross attention, both adjoints of far rows, f16 elements: the instantiations of xattn.h (one file each, so that they compile side by side).
#include "xattn.h"

namespace xattn {
XATTN_DEFINE_FAR(_Float16)
XATTN_DEFINE_VALUES(_Float16)
}
