// attend kernels of drafted trees for heads of 192, 224 and 256 columns.
#define XTK_ATTEND_KERNELS
#include "attend_kernels.h"

namespace xtk {

template hipError_t run_attend_tree<192>(bool, bool, const AttendArgs&, const TreeCap&, bool, hipStream_t);
template hipError_t run_attend_tree<224>(bool, bool, const AttendArgs&, const TreeCap&, bool, hipStream_t);
template hipError_t run_attend_tree<256>(bool, bool, const AttendArgs&, const TreeCap&, bool, hipStream_t);

}  // namespace xtk
