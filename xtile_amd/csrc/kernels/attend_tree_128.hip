// attend kernels of drafted trees for heads of 128 and 160 columns.
#define XTK_ATTEND_KERNELS
#include "attend_kernels.h"

namespace xtk {

template hipError_t run_attend_tree<128>(bool, bool, const AttendArgs&, const TreeCap&, bool, hipStream_t);
template hipError_t run_attend_tree<160>(bool, bool, const AttendArgs&, const TreeCap&, bool, hipStream_t);

}  // namespace xtk
