// The paged-attention kernels with a sliding window: instances of paged_attention.hip in an object of their own.
#define KVH_WINDOW_OBJECT
#include "paged_attention.hip"
