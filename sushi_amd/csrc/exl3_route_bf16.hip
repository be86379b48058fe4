#include "exl3_route.h"

namespace exl3 {
hipError_t run_route_bf16(const RouteArgs &a, hipStream_t s) { return route_of_type<DT_BF16>(a, s); }
}  // namespace exl3
