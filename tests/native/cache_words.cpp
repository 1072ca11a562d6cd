// Test-only host build: what a context holds for the calls on cache pages.
#include "../../juno_b200/csrc/common.cuh"

extern "C" long long cache_scratch_bytes(void *ctx) { return (long long)static_cast<juno_ctx *>(ctx)->cache_scratch_bytes; }
