/* Which part of the work a workgroup of the 8-bit decode attention takes. */
#include "../gb300-rl-runtime_amd/csrc/hip/kv8_runs.h"

uint32_t kv8_probe_run(uint32_t block, uint32_t grid, uint32_t n) { return kv8_run_of(block, grid, n); }
uint64_t kv8_probe_bytes(uint64_t cost, uint32_t rows, uint32_t head_dim) { return kv8_bytes_of(cost, rows, head_dim); }
