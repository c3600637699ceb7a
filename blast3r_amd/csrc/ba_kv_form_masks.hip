// The kernels of attention that AT_MASKS names (ba_kv_attend.h), in a source of their own because of the time that they take to build.
#include "ba_kv_attend.h"

namespace ba {

template int launch_tiles<AT_MASKS>(const AtArgs<AT_MASKS>&, const AtShape&, const AtGrid&, int, hipStream_t);

}  // namespace ba
