// Cross attention, fwd, bf16 elements: the instantiations of xattn.h (one file each, so that they compile side by side).
#include "xattn.h"

namespace xattn {
XATTN_DEFINE_FWD(__bf16)
}
