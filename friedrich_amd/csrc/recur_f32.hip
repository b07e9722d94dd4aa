// recur_f32.hip -- the kernels of recur.hpp for one element type.
#include "recur.hpp"

namespace fr {
template int rec_run<float>(fr_ctx*, RecArgs&, int, int, bool, OpWorkspace&);
}
