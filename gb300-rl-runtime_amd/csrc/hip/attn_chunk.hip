// attn_chunk.hip - causal attention of chunks of new tokens over the 16-bit paged
// arena (the kernels, what bounds them and what they measure are in prompt_core.h).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cmath>

#include "kv_layout.h"
#include "prompt_core.h"
#include "rl_hip.h"
#include "rl_hip_internal.h"

namespace {

int validate(const rl_attn_chunk_args_t *a, const char *who)
{
    if (!a || !a->arena_base || !a->block_table || !a->ctx_lens || !a->q_starts || !a->q || !a->out) {
        rl_set_error("%s: NULL argument", who);
        return -1;
    }
    if (kv_layout_check_paged(&a->layout) != 0) {
        rl_set_error("%s: unsupported KV layout (token_count %u, head_dim %u, scalar %u, block of %u bytes)", who,
                     a->layout.token_count, a->layout.head_dim, a->layout.scalar_bytes, a->layout.block_bytes);
        return -1;
    }
    if (a->dtype != RL_DTYPE_BF16 && a->dtype != RL_DTYPE_FP16) {
        rl_set_error("%s: dtype %u", who, a->dtype);
        return -1;
    }
    if (a->kv_heads == 0 || a->q_heads == 0 || a->q_heads % a->kv_heads != 0 || a->q_heads > 65535) {
        rl_set_error("%s: q_heads %u not a multiple of kv_heads %u (up to 65,535)", who, a->q_heads, a->kv_heads);
        return -1;
    }
    if (a->batch == 0 || a->batch > 65535) {
        rl_set_error("%s: batch %u (1 to 65,535)", who, a->batch);
        return -1;
    }
    if (a->arena_bytes < a->layout.block_bytes) {
        rl_set_error("%s: arena of %llu bytes holds no block", who, (unsigned long long)a->arena_bytes);
        return -1;
    }
    if (a->max_ctx >= (1u << 31) || (uint64_t)a->max_ctx > (uint64_t)a->table_stride * a->layout.token_count) {
        rl_set_error("%s: max_ctx %u exceeds table_stride %u x %u tokens (or is 2^31 and above)", who, a->max_ctx,
                     a->table_stride, a->layout.token_count);
        return -1;
    }
    const uint64_t group = a->q_heads / a->kv_heads;
    if (a->max_q * group >= (1ull << 31) || a->q_tokens >= (1u << 31)) {
        rl_set_error("%s: max_q %u x %llu heads per KV head / q_tokens %u of 2^31 and above", who, a->max_q,
                     (unsigned long long)group, a->q_tokens);
        return -1;
    }
    // (a launch holds less than 2^32 work-items)
    const uint64_t blocks = (uint64_t)a->batch * a->kv_heads * ((a->max_q * group + ROWS - 1) / ROWS);
    if (blocks >= (1u << 24)) {
        rl_set_error("%s: %llu blocks of %u rows (%u sequences of up to %u queries, %u KV heads; less than 2^24)", who,
                     (unsigned long long)blocks, ROWS, a->batch, a->max_q, a->kv_heads);
        return -1;
    }
    if (!(a->scale >= 0.f) || std::isinf(a->scale)) {
        rl_set_error("%s: scale %g (positive, or 0 for 1/sqrt(head_dim))", who, (double)a->scale);
        return -1;
    }
    const uint64_t row = (uint64_t)a->q_heads * a->layout.head_dim;
    const uint32_t strides[2] = {a->q_stride, a->out_stride};
    for (int i = 0; i < 2; i++)
        if (strides[i] != 0 && (strides[i] < row || strides[i] % 8 != 0 || strides[i] > (1u << 24))) {
            rl_set_error("%s: stride %u (0, or a multiple of 8 from the row's %llu elements to 2^24)", who, strides[i],
                         (unsigned long long)row);
            return -1;
        }
    if (row > (1u << 24)) {
        rl_set_error("%s: rows of %llu elements (up to 2^24)", who, (unsigned long long)row);
        return -1;
    }
    if (((uintptr_t)a->arena_base | (uintptr_t)a->q | (uintptr_t)a->out) % 16 != 0) {
        rl_set_error("%s: arena_base, q and out must be 16-byte aligned", who);
        return -1;
    }
    return 0;
}

PromptPlan plan_of(const rl_attn_chunk_args_t *a)
{
    return plan_of(a->batch, a->max_q, a->max_ctx, a->q_heads, a->kv_heads, a->layout.head_dim);
}

}  // namespace

extern "C" size_t rl_hip_attn_chunk_workspace(const rl_attn_chunk_args_t *a)
{
    if (validate(a, "rl_hip_attn_chunk_workspace") || rl_require_open("rl_hip_attn_chunk_workspace"))
        return 0;
    return plan_of(a).most;
}

extern "C" int rl_hip_attn_chunk(const rl_attn_chunk_args_t *a)
{
    const char *who = "rl_hip_attn_chunk";
    if (validate(a, who) || rl_require_open(who))
        return -1;
    if (a->max_q == 0 || a->q_tokens == 0)
        return 0;  // no query
    const PromptPlan pl = plan_of(a);
    if (!a->workspace || a->workspace_bytes < pl.workspace) {
        rl_set_error("%s: workspace %zu bytes < %zu required", who, a->workspace_bytes, pl.workspace);
        return -1;
    }
    const uint32_t row = a->q_heads * a->layout.head_dim;
    PromptParams p = {};
    p.q = (const uint16_t *)a->q;
    p.out = (uint16_t *)a->out;
    p.q_stride = a->q_stride ? a->q_stride : row;
    p.out_stride = a->out_stride ? a->out_stride : row;
    p.q_starts = a->q_starts;
    p.q_tokens = a->q_tokens;
    p.max_q = a->max_q;
    p.arena = (const uint8_t *)a->arena_base;
    p.block_bytes = a->layout.block_bytes;
    p.arena_blocks = (uint32_t)std::min<uint64_t>(a->arena_bytes / a->layout.block_bytes, 0xFFFFFFFFu);
    p.table = a->block_table;
    p.table_stride = a->table_stride;
    p.tpb = a->layout.token_count;
    p.tpb_shift = p.tpb == 32 ? 5 : 4;
    p.ctx = a->ctx_lens;
    p.max_ctx = a->max_ctx;
    set_plan(p, pl, a->batch, a->max_ctx, a->q_heads, a->kv_heads, a->layout.head_dim, a->scale, a->workspace);
    if (a->layout.head_dim == 128)
        return a->dtype == RL_DTYPE_BF16 ? prompt_launch<128, 0, true>(p) : prompt_launch<128, 1, true>(p);
    return a->dtype == RL_DTYPE_BF16 ? prompt_launch<64, 0, true>(p) : prompt_launch<64, 1, true>(p);
}
