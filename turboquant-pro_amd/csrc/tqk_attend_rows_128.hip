// Instances of tqk_attend_rows.h for head_dim 128.
#include "tqk_attend_rows.h"

void tqk_launch_rows_128(const MoreArgs& a, unsigned groups, hipStream_t st) { launch_rows<128>(a, groups, st); }
