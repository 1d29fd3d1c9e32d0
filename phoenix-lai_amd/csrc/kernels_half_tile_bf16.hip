#include "half_tile.h"

namespace phx {
template void launch_half_tiles<true, false>(hipStream_t, const HalfMat&, const HalfArgs&, int);
}
