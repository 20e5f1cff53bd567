/* Sizes and offsets of the 8-bit cache's and the prompt attention's arguments, for the ctypes mirror. */
#include "rl_hip.h"

size_t kv8_probe(int what)
{
    switch (what) {
    case 0: return sizeof(rl_kv8_append_args_t);
    case 1: return offsetof(rl_kv8_append_args_t, tokens);
    case 2: return offsetof(rl_kv8_append_args_t, v_stride);
    case 3: return sizeof(rl_attn_prompt_args_t);
    case 4: return offsetof(rl_attn_prompt_args_t, q_starts);
    case 5: return offsetof(rl_attn_prompt_args_t, scale);
    case 6: return offsetof(rl_attn_prompt_args_t, workspace_bytes);
    default: return 0;
    }
}

int kv8_layout(unsigned t, unsigned d, KvLayoutDesc *out)
{
    *out = kv_layout_desc_paged8(t, d);
    return kv_layout_check_paged8(out);
}
