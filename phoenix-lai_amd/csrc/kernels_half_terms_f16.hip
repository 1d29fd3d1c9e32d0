#include "half_tile.h"

namespace phx {
template void launch_half_tiles<false, true>(hipStream_t, const HalfMat&, const HalfArgs&, int);
}
