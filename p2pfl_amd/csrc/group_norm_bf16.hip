// The group norm's kernels (group_norm.h) for bf16 maps.
#define GROUP_NORM_TYPE __bf16
#include "group_norm.h"
