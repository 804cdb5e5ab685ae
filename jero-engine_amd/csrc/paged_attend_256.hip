// paged_attend_256.hip -- attention over a paged key/value cache, heads of up to 256.
#include "paged_attend.h"

namespace jero {

int paged_attend_256(const PagedCall& c, const PagedPlan& p, bool x16, bool kv16, const void* q, void* out, float* part_o,
                    float2* part_ml, hipStream_t s) {
  return launch_paged_types<256>(c, p, x16, kv16, q, out, part_o, part_ml, s);
}

}  // namespace jero
