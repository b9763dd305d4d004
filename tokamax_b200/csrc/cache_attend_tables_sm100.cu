// Attention over the quantised key / value cache with a page table for each kv head and query.
#include "cache_attend.cuh"

extern "C" {

int splash_cache_attend_tables(const SplashCacheAttendArgs* args, void* cuda_stream) {
  return args == nullptr ? SPLASH_ERR_INVALID_ARGUMENT : sb::cache_attend<true>(*args, static_cast<cudaStream_t>(cuda_stream));
}

size_t splash_cache_attend_tables_workspace_bytes(const SplashCacheAttendArgs* args) {
  return args == nullptr ? 0 : sb::cache_attend_workspace(*args, true);
}

}  // extern "C"
