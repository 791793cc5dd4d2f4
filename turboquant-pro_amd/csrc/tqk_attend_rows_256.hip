// Instances of tqk_attend_rows.h for head_dim 256.
#include "tqk_attend_rows.h"

void tqk_launch_rows_256(const MoreArgs& a, unsigned groups, hipStream_t st) { launch_rows<256>(a, groups, st); }
