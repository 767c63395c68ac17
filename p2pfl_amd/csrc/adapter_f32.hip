// The adapters' kernels (adapter.h) for fp32 rows.
#define ADAPTER_TYPE float
#include "adapter.h"
