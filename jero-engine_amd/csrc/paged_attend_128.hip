// paged_attend_128.hip -- attention over a paged key/value cache, heads of up to 128.
#include "paged_attend.h"

namespace jero {

int paged_attend_128(const PagedCall& c, const PagedPlan& p, bool x16, bool kv16, const void* q, void* out, float* part_o,
                    float2* part_ml, hipStream_t s) {
  return launch_paged_types<128>(c, p, x16, kv16, q, out, part_o, part_ml, s);
}

}  // namespace jero
