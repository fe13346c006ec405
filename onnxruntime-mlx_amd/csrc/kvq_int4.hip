// The matrix-core kernels of kvq_tile.h for int4 caches.
#include "kvq_tile.h"

namespace ortmi {
namespace kvq {

int tiles_int4(const Params& p, bool paged, hipStream_t st) { return launch_code<kInt4>(p, paged, st); }

}  // namespace kvq
}  // namespace ortmi
