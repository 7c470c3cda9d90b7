// The paged-attention kernels over MXFP4 caches: instances of paged_attention.hip in an object of their own, so that
// both compile at once.
#define KVH_KV4_OBJECT
#include "paged_attention.hip"
