// kv8_runs.h - which part of the work a workgroup of the 8-bit decode attention
// takes. Workgroup b of a grid runs on XCD b % 8, and each XCD has an L2 of its
// own: neighbouring parts, whose rollouts may share prefix blocks, go to one XCD,
// and the parts that have work to all XCDs alike. Plain C, also for the host.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define KV8_HD __host__ __device__ __forceinline__
#else
#define KV8_HD static inline
#endif

#define KV8_NO_RUN UINT32_MAX
#define KV8_UNIT 32u     // tokens per unit
#define KV8_ROW_COST 8u  // units that turning to a row is worth

// Bytes of the cache that rows of `cost` units in all hold, `rows` of them not empty:
// the row costs are nothing that is read.
KV8_HD uint64_t kv8_bytes_of(uint64_t cost, uint32_t rows, uint32_t head_dim)
{
    return (cost - (uint64_t)rows * KV8_ROW_COST) * (2u * KV8_UNIT * head_dim);
}

// Workgroup `block` of `grid`: a contiguous eighth of the grid's parts per XCD.
KV8_HD uint32_t kv8_contiguous(uint32_t block, uint32_t grid)
{
    return grid % 8 != 0 ? block : block % 8 * (grid / 8) + block / 8;
}

// The run, of the n <= grid that have work, of workgroup `block`; KV8_NO_RUN: none. A
// contiguous eighth of the n per XCD (of the grid, few runs would lie on few XCDs: n
// follows the contexts, the grid their bound).
KV8_HD uint32_t kv8_run_of(uint32_t block, uint32_t grid, uint32_t n)
{
    if (grid % 8 != 0)
        return block < n ? block : KV8_NO_RUN;
    const uint32_t x = block % 8, run = x * n / 8 + block / 8;
    return run < (x + 1) * n / 8 ? run : KV8_NO_RUN;
}
