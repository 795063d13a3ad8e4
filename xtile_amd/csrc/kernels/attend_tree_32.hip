// attend kernels of drafted trees for heads of 32, 64 and 96 columns.
#define XTK_ATTEND_KERNELS
#include "attend_kernels.h"

namespace xtk {

template hipError_t run_attend_tree<32>(bool, bool, const AttendArgs&, const TreeCap&, bool, hipStream_t);
template hipError_t run_attend_tree<64>(bool, bool, const AttendArgs&, const TreeCap&, bool, hipStream_t);
template hipError_t run_attend_tree<96>(bool, bool, const AttendArgs&, const TreeCap&, bool, hipStream_t);

}  // namespace xtk
