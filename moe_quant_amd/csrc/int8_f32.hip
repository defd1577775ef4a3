#include "int8_kernels.hpp"

int mq_int8_product_f32(const Int8Args& a, int swiglu, hipStream_t st) {
  return swiglu ? int8_launch<DT_F32, true>(a, st) : int8_launch<DT_F32, false>(a, st);
}
int mq_int8_rows_f32(const Int8Args& a, hipStream_t st) { return vector_launch<DT_F32, false, DT_F32>(a, st); }
