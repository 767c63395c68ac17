// The group norm's kernels (group_norm.h) for fp32 maps.
#define GROUP_NORM_TYPE float
#include "group_norm.h"
