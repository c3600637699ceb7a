// The kernels of attention with capped scores (ba_kv_attend.h), in a source of their own: they take as long to build as
// all others of a mode.
#include "ba_kv_attend.h"

namespace ba {

template int launch_attend<AT_CAPPED>(const AtArgs<AT_CAPPED>&, AtShape, unsigned, int, int, int, hipStream_t);

}  // namespace ba
