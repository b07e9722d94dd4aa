// recur_bf16.hip -- the kernels of recur.hpp for one element type.
#include "recur.hpp"

namespace fr {
template int rec_run<__hip_bfloat16>(fr_ctx*, RecArgs&, int, int, bool, OpWorkspace&);
}
