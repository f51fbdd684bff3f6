#include "ops_products_kernels.h"

template int launch_rows<f16_t>(const RowsArgs &, bool, bool, bool, i64, hipStream_t);
template int launch_weight<f16_t>(const WeightArgs &, bool, i64, hipStream_t);
template int launch_combine<f16_t>(const CombineArgs &, bool, hipStream_t);
