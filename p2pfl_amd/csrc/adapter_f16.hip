// The adapters' kernels (adapter.h) for fp16 rows.
#define ADAPTER_TYPE _Float16
#include "adapter.h"
