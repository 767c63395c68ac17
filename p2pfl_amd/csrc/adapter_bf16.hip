// The adapters' kernels (adapter.h) for bf16 rows.
#define ADAPTER_TYPE __bf16
#include "adapter.h"
