// The group norm's kernels (group_norm.h) for fp16 maps.
#define GROUP_NORM_TYPE _Float16
#include "group_norm.h"
