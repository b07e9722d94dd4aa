// recur_f16.hip -- the kernels of recur.hpp for one element type.
#include "recur.hpp"

namespace fr {
template int rec_run<__half>(fr_ctx*, RecArgs&, int, int, bool, OpWorkspace&);
}
