// The kernels of attention with scores that fall with the distance (ba_kv_attend.h), in a source of their own: they take as long to build as
// all others of a mode.
#include "ba_kv_attend.h"

namespace ba {

template int launch_attend<AT_SLOPES>(const AtArgs<AT_SLOPES>&, AtShape, unsigned, int, int, int, hipStream_t);

}  // namespace ba
