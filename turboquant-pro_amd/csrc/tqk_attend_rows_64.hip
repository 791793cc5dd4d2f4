// Instances of tqk_attend_rows.h for head_dim 64.
#include "tqk_attend_rows.h"

void tqk_launch_rows_64(const MoreArgs& a, unsigned groups, hipStream_t st) { launch_rows<64>(a, groups, st); }
