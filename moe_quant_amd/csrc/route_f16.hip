#include "route_kernels.hpp"

int mq_route_f16(const RouteArgs& a, hipStream_t st) {
  route_any<DT_F16>(a, st);
  return mq_check_launch();
}
