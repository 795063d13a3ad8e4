// attend kernels for heads of 128 and 160 columns.
#define XTK_ATTEND_KERNELS
#include "attend_kernels.h"

namespace xtk {

template hipError_t run_attend<128>(bool, bool, const AttendArgs&, const FineCap*, hipStream_t);
template hipError_t run_attend<160>(bool, bool, const AttendArgs&, const FineCap*, hipStream_t);

}  // namespace xtk
