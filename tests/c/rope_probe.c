/* Sizes and offsets of the rotating append's arguments, for the ctypes mirror. */
#include "rl_hip.h"

size_t rope_probe(int what)
{
    switch (what) {
    case 0: return sizeof(rl_rope_append_args_t);
    case 1: return offsetof(rl_rope_append_args_t, tokens);
    case 2: return offsetof(rl_rope_append_args_t, rot_dim);
    case 3: return offsetof(rl_rope_append_args_t, k_out);
    case 4: return offsetof(rl_rope_append_args_t, k_out_stride);
    default: return 0;
    }
}
