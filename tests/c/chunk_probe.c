/* Sizes and offsets of the chunk attention's arguments, for the ctypes mirror. */
#include "rl_hip.h"

size_t chunk_probe(int what)
{
    switch (what) {
    case 0: return sizeof(rl_attn_chunk_args_t);
    case 1: return offsetof(rl_attn_chunk_args_t, max_ctx);
    case 2: return offsetof(rl_attn_chunk_args_t, q_tokens);
    case 3: return offsetof(rl_attn_chunk_args_t, scale);
    case 4: return offsetof(rl_attn_chunk_args_t, workspace_bytes);
    default: return 0;
    }
}
