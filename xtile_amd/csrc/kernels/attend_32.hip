// attend kernels for heads of 32, 64 and 96 columns.
#define XTK_ATTEND_KERNELS
#include "attend_kernels.h"

namespace xtk {

template hipError_t run_attend<32>(bool, bool, const AttendArgs&, const FineCap*, hipStream_t);
template hipError_t run_attend<64>(bool, bool, const AttendArgs&, const FineCap*, hipStream_t);
template hipError_t run_attend<96>(bool, bool, const AttendArgs&, const FineCap*, hipStream_t);

}  // namespace xtk
