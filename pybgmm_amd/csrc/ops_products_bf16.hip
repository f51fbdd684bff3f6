#include "ops_products_kernels.h"

template int launch_rows<bf16_t>(const RowsArgs &, bool, int, int, i64, hipStream_t);
template int launch_weight<bf16_t>(const WeightArgs &, int, int, i64, hipStream_t);
template int launch_combine<bf16_t>(const CombineArgs &, hipStream_t);
template int launch_gates<bf16_t>(const GatesArgs &, hipStream_t);
