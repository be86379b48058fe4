#include "exl3_route.h"

namespace exl3 {
hipError_t run_route_f32(const RouteArgs &a, hipStream_t s) { return route_of_type<DT_F32>(a, s); }
}  // namespace exl3
