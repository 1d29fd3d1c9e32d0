#include "half_tile.h"

namespace phx {
template void launch_half_tiles<false, false>(hipStream_t, const HalfMat&, const HalfArgs&, int);
}
