#include "ops_products_kernels.h"

template int launch_rows<double>(const RowsArgs &, bool, int, int, i64, hipStream_t);
template int launch_weight<double>(const WeightArgs &, int, int, i64, hipStream_t);
template int launch_combine<double>(const CombineArgs &, hipStream_t);
template int launch_gates<double>(const GatesArgs &, hipStream_t);
