// attend kernels for heads of 192, 224 and 256 columns.
#define XTK_ATTEND_KERNELS
#include "attend_kernels.h"

namespace xtk {

template hipError_t run_attend<192>(bool, bool, const AttendArgs&, const FineCap*, hipStream_t);
template hipError_t run_attend<224>(bool, bool, const AttendArgs&, const FineCap*, hipStream_t);
template hipError_t run_attend<256>(bool, bool, const AttendArgs&, const FineCap*, hipStream_t);

}  // namespace xtk
