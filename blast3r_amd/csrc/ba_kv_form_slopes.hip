// The kernels of attention that AT_SLOPES names (ba_kv_attend.h), in a source of their own because of the time that they take to build.
#include "ba_kv_attend.h"

namespace ba {

template int launch_tiles<AT_SLOPES>(const AtArgs<AT_SLOPES>&, const AtShape&, const AtGrid&, int, hipStream_t);

}  // namespace ba
