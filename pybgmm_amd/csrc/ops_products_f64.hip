#include "ops_products_kernels.h"

template int launch_rows<double>(const RowsArgs &, bool, bool, bool, i64, hipStream_t);
template int launch_weight<double>(const WeightArgs &, bool, i64, hipStream_t);
template int launch_combine<double>(const CombineArgs &, bool, hipStream_t);
