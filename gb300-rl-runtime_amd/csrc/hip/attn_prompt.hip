// attn_prompt.hip - causal attention over whole prompts, packed sequences with
// grouped heads (the kernels are in prompt_core.h).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cmath>

#include "prompt_core.h"
#include "rl_hip.h"
#include "rl_hip_internal.h"

namespace {

int validate(const rl_attn_prompt_args_t *a, const char *who)
{
    if (!a || !a->q || !a->k || !a->v || !a->out || !a->q_starts) {
        rl_set_error("%s: NULL argument", who);
        return -1;
    }
    if (a->head_dim != 64 && a->head_dim != 128) {
        rl_set_error("%s: head_dim %u not in {64, 128}", who, a->head_dim);
        return -1;
    }
    if (a->kv_heads == 0 || a->q_heads == 0 || a->q_heads % a->kv_heads != 0 || a->q_heads > 65535) {
        rl_set_error("%s: q_heads %u not a multiple of kv_heads %u (up to 65,535)", who, a->q_heads, a->kv_heads);
        return -1;
    }
    if (a->dtype != RL_DTYPE_BF16 && a->dtype != RL_DTYPE_FP16) {
        rl_set_error("%s: dtype %u", who, a->dtype);
        return -1;
    }
    if (a->seqs == 0 || a->seqs > 65535) {
        rl_set_error("%s: %u sequences (1 to 65,535)", who, a->seqs);
        return -1;
    }
    const uint64_t group = a->q_heads / a->kv_heads;
    if ((uint64_t)a->max_q * group >= (1ull << 31) || a->max_kv >= (1u << 31)) {
        rl_set_error("%s: max_q %u x %llu heads per KV head / max_kv %u of 2^31 and above", who, a->max_q,
                     (unsigned long long)group, a->max_kv);
        return -1;
    }
    if (a->q_tokens >= (1u << 31) || a->kv_tokens >= (1u << 31)) {
        rl_set_error("%s: q_tokens %u / kv_tokens %u of 2^31 and above", who, a->q_tokens, a->kv_tokens);
        return -1;
    }
    // (a launch holds less than 2^32 work-items)
    const uint64_t blocks = (uint64_t)a->seqs * a->kv_heads * ((a->max_q * group + ROWS - 1) / ROWS);
    if (blocks >= (1u << 24)) {
        rl_set_error("%s: %llu blocks of %u rows (%u sequences of up to %u queries, %u KV heads; less than 2^24)", who,
                     (unsigned long long)blocks, ROWS, a->seqs, a->max_q, a->kv_heads);
        return -1;
    }
    if (!(a->scale >= 0.f) || std::isinf(a->scale)) {
        rl_set_error("%s: scale %g (positive, or 0 for 1/sqrt(head_dim))", who, (double)a->scale);
        return -1;
    }
    const uint64_t qrow = (uint64_t)a->q_heads * a->head_dim, kvrow = (uint64_t)a->kv_heads * a->head_dim;
    const uint32_t strides[4] = {a->q_stride, a->k_stride, a->v_stride, a->out_stride};
    for (int i = 0; i < 4; i++) {
        const uint64_t row = i == 0 || i == 3 ? qrow : kvrow;
        if (strides[i] != 0 && (strides[i] < row || strides[i] % 8 != 0 || strides[i] > (1u << 24))) {
            rl_set_error("%s: stride %u (0, or a multiple of 8 from the row's %llu elements to 2^24)", who, strides[i],
                         (unsigned long long)row);
            return -1;
        }
    }
    if (qrow > (1u << 24)) {
        rl_set_error("%s: rows of %llu elements (up to 2^24)", who, (unsigned long long)qrow);
        return -1;
    }
    if (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out) % 16 != 0) {
        rl_set_error("%s: q, k, v and out must be 16-byte aligned", who);
        return -1;
    }
    return 0;
}

}  // namespace

extern "C" size_t rl_hip_attn_prompt_workspace(const rl_attn_prompt_args_t *a)
{
    if (validate(a, "rl_hip_attn_prompt_workspace") || rl_require_open("rl_hip_attn_prompt_workspace"))
        return 0;
    return plan_of(a->seqs, a->max_q, a->max_kv, a->q_heads, a->kv_heads, a->head_dim).most;
}

extern "C" int rl_hip_attn_prompt(const rl_attn_prompt_args_t *a)
{
    const char *who = "rl_hip_attn_prompt";
    if (validate(a, who) || rl_require_open(who))
        return -1;
    if (a->max_q == 0 || a->q_tokens == 0)
        return 0;  // no query
    const PromptPlan pl = plan_of(a->seqs, a->max_q, a->max_kv, a->q_heads, a->kv_heads, a->head_dim);
    if (!a->workspace || a->workspace_bytes < pl.workspace) {
        rl_set_error("%s: workspace %zu bytes < %zu required", who, a->workspace_bytes, pl.workspace);
        return -1;
    }
    PromptParams p;
    p.q = (const uint16_t *)a->q;
    p.k = (const uint16_t *)a->k;
    p.v = (const uint16_t *)a->v;
    p.out = (uint16_t *)a->out;
    p.q_stride = a->q_stride ? a->q_stride : a->q_heads * a->head_dim;
    p.k_stride = a->k_stride ? a->k_stride : a->kv_heads * a->head_dim;
    p.v_stride = a->v_stride ? a->v_stride : a->kv_heads * a->head_dim;
    p.out_stride = a->out_stride ? a->out_stride : a->q_heads * a->head_dim;
    p.q_starts = a->q_starts;
    p.kv_starts = a->kv_starts ? a->kv_starts : a->q_starts;
    p.q_tokens = a->q_tokens;
    p.kv_tokens = a->kv_tokens;
    p.max_q = a->max_q;
    set_plan(p, pl, a->seqs, a->max_kv, a->q_heads, a->kv_heads, a->head_dim, a->scale, a->workspace);
    if (a->head_dim == 128)
        return a->dtype == RL_DTYPE_BF16 ? prompt_launch<128, 0, false>(p) : prompt_launch<128, 1, false>(p);
    return a->dtype == RL_DTYPE_BF16 ? prompt_launch<64, 0, false>(p) : prompt_launch<64, 1, false>(p);
}
