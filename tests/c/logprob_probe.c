/* Sizes and offsets of the token logprobs' arguments, for the ctypes mirror. */
#include "rl_hip.h"

size_t logprob_probe(int what)
{
    switch (what) {
    case 0: return sizeof(rl_token_logprob_args_t);
    case 1: return offsetof(rl_token_logprob_args_t, scale);
    case 2: return offsetof(rl_token_logprob_args_t, workspace_bytes);
    case 3: return sizeof(rl_token_logprob_grad_args_t);
    case 4: return offsetof(rl_token_logprob_grad_args_t, lse);
    case 5: return offsetof(rl_token_logprob_grad_args_t, dw_stride);
    case 6: return offsetof(rl_token_logprob_grad_args_t, workspace_bytes);
    default: return 0;
    }
}
