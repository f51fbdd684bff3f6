#include "ops_products_kernels.h"

template int launch_rows<float>(const RowsArgs &, bool, int, int, i64, hipStream_t);
template int launch_weight<float>(const WeightArgs &, int, int, i64, hipStream_t);
template int launch_combine<float>(const CombineArgs &, hipStream_t);
template int launch_gates<float>(const GatesArgs &, hipStream_t);
