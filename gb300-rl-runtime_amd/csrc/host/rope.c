/* rope.c - frequencies of the position rotation (rl_hip_rope_append). */
#include <math.h>

#include "rl_hip.h"

int rl_rope_freqs(double *freqs, uint32_t rot_dim, double theta)
{
    if (!freqs || rot_dim % 2 != 0 || !(theta > 0.0))
        return -1;
    for (uint32_t i = 0; i < rot_dim / 2; i++)
        freqs[i] = pow(theta, -2.0 * i / rot_dim);
    return 0;
}
