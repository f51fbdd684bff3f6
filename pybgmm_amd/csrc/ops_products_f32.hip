#include "ops_products_kernels.h"

template int launch_rows<float>(const RowsArgs &, bool, bool, bool, i64, hipStream_t);
template int launch_weight<float>(const WeightArgs &, bool, i64, hipStream_t);
template int launch_combine<float>(const CombineArgs &, bool, hipStream_t);
