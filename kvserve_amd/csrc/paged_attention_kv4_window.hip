// The paged-attention kernels over MXFP4 caches with a sliding window: instances of paged_attention.hip in an object of
// their own.
#define KVH_KV4_OBJECT
#define KVH_WINDOW_OBJECT
#include "paged_attention.hip"
