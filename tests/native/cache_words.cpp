// Test-only host build: what a context holds for the calls on cache pages.
#include "../../juno_b200/csrc/common.cuh"

// Where decode attention leaves the number of a call that gave up a wait (device memory, 64 bits), and how many calls there were.
extern "C" void *cache_gave_up(void *ctx) { return static_cast<juno_ctx *>(ctx)->cache_arrived; }
extern "C" unsigned long long cache_calls(void *ctx) { return static_cast<juno_ctx *>(ctx)->cache_calls; }
extern "C" long long cache_scratch_bytes(void *ctx) { return (long long)static_cast<juno_ctx *>(ctx)->cache_scratch_bytes; }
