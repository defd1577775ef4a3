#include "int8_kernels.hpp"

int mq_int8_product_bf16(const Int8Args& a, int swiglu, hipStream_t st) {
  return swiglu ? int8_launch<DT_BF16, true>(a, st) : int8_launch<DT_BF16, false>(a, st);
}
int mq_int8_rows_bf16(const Int8Args& a, hipStream_t st) { return vector_launch<DT_BF16, false, DT_BF16>(a, st); }
