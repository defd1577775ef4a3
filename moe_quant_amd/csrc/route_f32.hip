#include "route_kernels.hpp"

int mq_route_f32(const RouteArgs& a, hipStream_t st) {
  route_any<DT_F32>(a, st);
  return mq_check_launch();
}
