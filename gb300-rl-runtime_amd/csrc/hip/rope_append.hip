// rope_append.hip - new tokens' queries and keys turned by their positions, and
// keys and values into the 16-bit paged arena, whole prompts or one token per
// row, on gfx950.
//
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t),  t = position freqs[i]
//
// for the i-th pair of every query and key head's first rot_dim elements.
//
//  angle  t is formed in 64 bits (in 32 a position of 100,000 would be off by
//         0.004 rad), reduced to within an eighth of a turn, and only then
//         rounded to 32 bits, where the Taylor series of sine (to the 9th power)
//         and cosine (to the 10th) are within 2^-24.
//  bound  the bytes: 64 prompts of 512-1,024 tokens, 32 query and 8 KV heads of d128,
//         211-226 us (5.3-5.7 TB/s, a copy's rate); one token of 64 rows 3.1-4.0 us, a
//         launch and the chain position, table entry, store. Copies on write, each a
//         wave's, add 0.2-0.3 us to 64 rows of 8 KV heads (one token 3.2 to 3.4, 200
//         tokens 62.8 to 63.1).
//  split  a lane holds two 16-byte chunks of a head, those that are turned into
//         each other, of one token; a wave D / 16 lanes for each of its 8 (d128)
//         or 16 (d64) tokens, and goes through some of their heads, so that
//         the angles are formed once for several heads.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "attn_core.h"
#include "rl_hip.h"
#include "rl_hip_internal.h"

namespace {

constexpr int kWaves = 4;

struct RopeParams {
    uint8_t *arena;        // NULL: nothing is appended
    uint64_t block_bytes, arena_blocks;
    const uint32_t *table;
    uint32_t table_stride, tpb, tpb_shift;  // blocks of tpb = 2^tpb_shift tokens
    uint32_t q_heads, kv_heads;  // q_heads 0: no queries
    uint32_t heads;        // of a token in all: q_heads, then kv_heads of K (unless nobody wants them) and of V
    uint32_t slices;       // waves sharing a token's heads
    uint32_t batch, tokens;
    uint32_t items;        // waves that turn and append; behind them one per (row, KV head) that copies on write
    uint32_t copies;
    const uint32_t *positions, *starts;
    const int32_t *cow_src;
    const double *freqs;
    uint32_t units;        // of a head, each 16 elements, that are turned: rot_dim / 16
    uint32_t neighbours;   // pairs are neighbours, not halves
    const uint16_t *q, *k, *v;
    uint16_t *q_out, *k_out;
    uint64_t q_stride, q_out_stride, k_stride, v_stride, k_out_stride;  // elements between tokens
};

// How many of starts[0 .. batch] are at most t, 64 at a time.
__device__ __forceinline__ uint32_t starts_up_to(const uint32_t *starts, uint32_t batch, uint32_t t, int lane)
{
    uint32_t lo = 0, n = batch + 1;
    while (n > 64) {
        const uint32_t step = (n + 63) / 64, i = (uint32_t)lane * step;
        const uint32_t k = (uint32_t)__builtin_popcountll(
            __builtin_amdgcn_ballot_w64(i < n && starts[lo + min(i, n - 1)] <= t));
        if (k == 0)
            return lo;
        const uint32_t past = (k - 1) * step + 1;  // (the k-th of those that were looked at counts)
        lo += past;
        n = min(step - 1, n - past);
    }
    const bool has = (uint32_t)lane < n && starts[lo + min((uint32_t)lane, max(n, 1u) - 1)] <= t;
    return lo + (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(has));
}

// Sine and cosine of pos f.
__device__ __forceinline__ void turn_of(double pos, double f, float &sine, float &cosine)
{
    constexpr double kQuarters = 0.63661977236758134308, kQuarter = 1.57079632679489661923;  // 2 / pi, pi / 2
    constexpr double kRound = 6755399441055744.0;  // 1.5 x 2^52: the sum's last bits are the nearest whole number
    const double quarters = pos * f * kQuarters, sum = quarters + kRound;
    const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, sum);
    const float y = (float)((quarters - (sum - kRound)) * kQuarter), z = y * y;
    const float s = y + y * z * fmaf(z, fmaf(z, fmaf(z, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6);
    const float c4 = fmaf(z, fmaf(z, fmaf(z, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24);
    const float c = fmaf(z, fmaf(z, c4, -0.5f), 1.f);
    const float a = n & 1 ? c : s, b = n & 1 ? s : c;
    sine = n & 2 ? -a : a;
    cosine = (n + 1) & 2 ? -b : b;
}

// The turned chunks x, y: element e of x with element e of y, or neighbours of
// each (the pairs 0 .. 3 in x, 4 .. 7 in y).
template <int DT, bool NB>
__device__ __forceinline__ void turn(rl_u32x4 &x, rl_u32x4 &y, const float (&s)[8], const float (&c)[8])
{
    rl_u32x4 r[2];
#pragma unroll
    for (int w = 0; w < 4; w++) {
        float x0, x1, y0, y1, o[4];
        rl_unpack2<DT>(x[w], x0, x1);
        rl_unpack2<DT>(y[w], y0, y1);
        if constexpr (NB) {
            o[0] = fmaf(x0, c[w], -(x1 * s[w]));
            o[1] = fmaf(x0, s[w], x1 * c[w]);
            o[2] = fmaf(y0, c[4 + w], -(y1 * s[4 + w]));
            o[3] = fmaf(y0, s[4 + w], y1 * c[4 + w]);
        } else {
            o[0] = fmaf(x0, c[2 * w], -(y0 * s[2 * w]));
            o[1] = fmaf(x1, c[2 * w + 1], -(y1 * s[2 * w + 1]));
            o[2] = fmaf(x0, s[2 * w], y0 * c[2 * w]);
            o[3] = fmaf(x1, s[2 * w + 1], y1 * c[2 * w + 1]);
        }
#pragma unroll
        for (int h = 0; h < 2; h++)
            r[h][w] = (uint32_t)to16<DT>(o[2 * h]) | (uint32_t)to16<DT>(o[2 * h + 1]) << 16;
    }
    x = r[0];
    y = r[1];
}

// The filled slots of the shared block that row b's first new token falls into,
// into its own block.
template <int D>
__device__ __forceinline__ void copy_on_write(const RopeParams &p, uint32_t b, uint32_t g, int lane)
{
    uint32_t n = b < p.tokens ? 1u : 0u;
    if (p.starts) {
        const uint32_t first = rl_sload(p.starts + b), end = min(rl_sload(p.starts + b + 1), p.tokens);
        n = end > first ? end - first : 0u;
    }
    const uint32_t pos = rl_sload(p.positions + b), slot = pos % p.tpb, row = b * p.kv_heads + g;
    const int32_t from = rl_sload(p.cow_src + row);
    if (n == 0 || pos / p.tpb >= p.table_stride || from < 0 || (uint64_t)from >= p.arena_blocks)
        return;
    const uint32_t blk = rl_sload(p.table + (size_t)row * p.table_stride + pos / p.tpb);
    if (blk >= p.arena_blocks || blk == (uint32_t)from)
        return;
    const uint8_t *src = p.arena + (uint64_t)(uint32_t)from * p.block_bytes;
    uint8_t *dst = p.arena + (uint64_t)blk * p.block_bytes;
    constexpr uint32_t kRow = D / 8;  // 16-byte chunks of a row
    for (uint32_t i = (uint32_t)lane; i < 2 * slot * kRow; i += 64) {
        const uint32_t v = i >= slot * kRow, at = (v * p.tpb * kRow + (i - v * slot * kRow)) * 16;
        *(rl_u32x4 *)(dst + at) = *(const rl_u32x4 *)(src + at);
    }
}

template <int D, int DT, bool NB, int HEADS>
__global__ __launch_bounds__(kWaves * 64) void rope_append_kernel(RopeParams p)
{
    constexpr uint32_t UNITS = D / 16, TOKENS = 64 / UNITS;
    const int lane = threadIdx.x & 63;
    uint32_t item = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (item >= p.items) {
        item -= p.items;
        if (item < p.copies)
            copy_on_write<D>(p, item / p.kv_heads, item % p.kv_heads, lane);
        return;
    }
    const uint32_t h0 = item % p.slices * HEADS, t0 = item / p.slices * TOKENS;
    const uint32_t u = (uint32_t)lane % UNITS, r = (uint32_t)lane / UNITS, t = t0 + r;
    uint32_t b = t, i = 0;
    bool has = t < p.tokens;
    if (p.starts) {
        const uint32_t c = starts_up_to(p.starts, p.batch, t0, lane);
        uint32_t up_to = c;
        for (uint32_t at = c;; at += 64) {
            const uint32_t s = at + lane <= p.batch ? p.starts[at + lane] : 0xFFFFFFFFu;
            uint64_t in = 0;
#pragma unroll
            for (uint32_t j = 0; j < TOKENS; j++) {
                in = __builtin_amdgcn_ballot_w64(s <= t0 + j);
                up_to += r == j ? (uint32_t)__builtin_popcountll(in) : 0u;
            }
            if (in >> 63 == 0)
                break;  // (no start further on is as small as the last of these tokens)
        }
        has = has && up_to >= 1 && up_to <= p.batch;
        b = has ? up_to - 1 : 0u;
        i = t - p.starts[b];
    }
    if (!has)
        return;
    const uint64_t pos = (uint64_t)p.positions[b] + i;
    const uint32_t k0 = p.q_heads, v0 = k0 + p.kv_heads;
    float s[8], c[8];
    if (u < p.units && h0 < v0) {
#pragma unroll
        for (int e = 0; e < 8; e++)
            turn_of((double)pos, p.freqs[8 * u + e], s[e], c[e]);
    }
    // this lane's chunks of a head
    uint32_t c0 = 2 * u, c1 = 2 * u + 1;
    if (!NB && u < p.units) {
        c0 = u;
        c1 = u + p.units;
    }
    const uint32_t e0 = c0 * 8, e1 = c1 * 8;
    const uint32_t lb = (uint32_t)min<uint64_t>(pos >> p.tpb_shift, 0xFFFFFFFFu), slot = (uint32_t)pos & (p.tpb - 1);
    const bool held = p.arena != nullptr && lb < p.table_stride;
    rl_u32x4 x[HEADS], y[HEADS];
    uint32_t blk[HEADS];
#pragma unroll
    for (int j = 0; j < HEADS; j++) {
        const uint32_t h = h0 + j;
        if (h >= p.heads)
            break;
        const uint16_t *src;
        if (h < k0)
            src = p.q + t * p.q_stride + (uint64_t)h * D;
        else
            src = h < v0 ? p.k + t * p.k_stride + (uint64_t)(h - k0) * D : p.v + t * p.v_stride + (uint64_t)(h - v0) * D;
        x[j] = *(const rl_u32x4 *)(src + e0);
        y[j] = *(const rl_u32x4 *)(src + e1);
        blk[j] = 0xFFFFFFFFu;
        if (h >= k0 && held)
            blk[j] = p.table[((size_t)b * p.kv_heads + (h < v0 ? h - k0 : h - v0)) * p.table_stride + lb];
    }
#pragma unroll
    for (int j = 0; j < HEADS; j++) {
        const uint32_t h = h0 + j;
        if (h >= p.heads)
            break;
        if (h < v0 && u < p.units)
            turn<DT, NB>(x[j], y[j], s, c);
        if (h < k0 || (h < v0 && p.k_out)) {
            uint16_t *out = h < k0 ? p.q_out + t * p.q_out_stride + (uint64_t)h * D
                                   : p.k_out + t * p.k_out_stride + (uint64_t)(h - k0) * D;
            *(rl_u32x4 *)(out + e0) = x[j];
            *(rl_u32x4 *)(out + e1) = y[j];
        }
        if (h >= k0 && blk[j] < p.arena_blocks) {
            uint16_t *out = (uint16_t *)(p.arena + (uint64_t)blk[j] * p.block_bytes) +
                            ((h >= v0 ? p.tpb : 0u) + slot) * (uint32_t)D;
            *(rl_u32x4 *)(out + e0) = x[j];
            *(rl_u32x4 *)(out + e1) = y[j];
        }
    }
}

template <int D, int DT, bool NB, int HEADS>
int launch(const RopeParams &p)
{
    const uint32_t grid = (uint32_t)(((uint64_t)p.items + p.copies + kWaves - 1) / kWaves);
    hipLaunchKernelGGL((rope_append_kernel<D, DT, NB, HEADS>), dim3(grid), dim3(kWaves * 64), 0, rl_stream(), p);
    return rl_check_launch("rope_append_kernel launch");
}

template <int D, int DT>
int launch(const RopeParams &p, uint32_t per)
{
    if (p.neighbours)
        return per == 1 ? launch<D, DT, true, 1>(p) : per == 2 ? launch<D, DT, true, 2>(p) : launch<D, DT, true, 4>(p);
    return per == 1 ? launch<D, DT, false, 1>(p) : per == 2 ? launch<D, DT, false, 2>(p) : launch<D, DT, false, 4>(p);
}

int validate(const rl_rope_append_args_t *a)
{
    const char *who = "rl_hip_rope_append";
    if (!a || !a->positions || (!a->q != !a->q_out) || (!a->q && !a->k_out && !a->arena_base) ||
        ((a->k_out || a->arena_base) && !a->k_new) || (a->arena_base && (!a->block_table || !a->v_new)) ||
        (a->rot_dim && !a->freqs)) {
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
    if (a->rot_dim % 16 != 0 || a->rot_dim > a->layout.head_dim) {
        rl_set_error("%s: rot_dim %u (a multiple of 16 up to head_dim %u)", who, a->rot_dim, a->layout.head_dim);
        return -1;
    }
    if (a->pairing != RL_ROPE_HALVES && a->pairing != RL_ROPE_NEIGHBOURS) {
        rl_set_error("%s: pairing %u", who, a->pairing);
        return -1;
    }
    const bool keys = a->k_out || a->arena_base;
    if (a->batch == 0 || a->batch > 65535 || (a->q && a->q_heads == 0) || a->q_heads > 65535 ||
        (keys && a->kv_heads == 0) || a->kv_heads > 65535) {
        rl_set_error("%s: batch %u, q_heads %u or kv_heads %u out of range", who, a->batch, a->q_heads, a->kv_heads);
        return -1;
    }
    if ((!a->starts && a->tokens != a->batch) || a->tokens >= (1u << 31)) {
        rl_set_error("%s: %u tokens for %u rows%s", who, a->tokens, a->batch,
                     a->starts ? " (less than 2^31)" : " of one token each");
        return -1;
    }
    if (a->cow_src && !a->arena_base) {
        rl_set_error("%s: cow_src without an arena", who);
        return -1;
    }
    if (a->arena_base && a->arena_bytes < a->layout.block_bytes) {
        rl_set_error("%s: arena of %llu bytes holds no block", who, (unsigned long long)a->arena_bytes);
        return -1;
    }
    const uint64_t qrow = (uint64_t)a->q_heads * a->layout.head_dim, kvrow = (uint64_t)a->kv_heads * a->layout.head_dim;
    const uint32_t strides[5] = {a->q_stride, a->q_out_stride, a->k_stride, a->v_stride, a->k_out_stride};
    for (int i = 0; i < 5; i++) {
        const uint64_t row = i < 2 ? qrow : kvrow;
        if (strides[i] != 0 && (strides[i] < row || strides[i] % 8 != 0)) {
            rl_set_error("%s: stride %u (0, or a multiple of 8 of at least the row's %llu elements)", who, strides[i],
                         (unsigned long long)row);
            return -1;
        }
    }
    if (a->q && a->q == a->q_out && (a->q_stride ? a->q_stride : qrow) != (a->q_out_stride ? a->q_out_stride : qrow)) {
        rl_set_error("%s: q_out is q with another stride (%u and %u)", who, a->q_stride, a->q_out_stride);
        return -1;
    }
    if (((uintptr_t)a->arena_base | (uintptr_t)a->q | (uintptr_t)a->q_out | (uintptr_t)a->k_new | (uintptr_t)a->v_new |
         (uintptr_t)a->k_out) % 16 != 0 || (uintptr_t)a->freqs % 8 != 0) {
        rl_set_error("%s: arena_base and rows must be 16-byte aligned, freqs 8-byte aligned", who);
        return -1;
    }
    return 0;
}

}  // namespace

extern "C" int rl_hip_rope_append(const rl_rope_append_args_t *a)
{
    const char *who = "rl_hip_rope_append";
    if (validate(a) || rl_require_open(who))
        return -1;
    if (a->tokens == 0)
        return 0;
    const uint32_t d = a->layout.head_dim;
    RopeParams p;
    p.arena = (uint8_t *)a->arena_base;
    p.block_bytes = a->layout.block_bytes;
    p.arena_blocks = a->arena_base ? std::min<uint64_t>(a->arena_bytes / a->layout.block_bytes, 0xFFFFFFFFu) : 0;
    p.table = a->block_table;
    p.table_stride = a->table_stride;
    p.tpb = a->layout.token_count;
    p.tpb_shift = p.tpb == 32 ? 5 : 4;
    p.q_heads = a->q ? a->q_heads : 0;
    p.kv_heads = a->kv_heads;
    p.heads = p.q_heads + (p.arena ? 2 * a->kv_heads : a->k_out ? a->kv_heads : 0);
    p.batch = a->batch;
    p.tokens = a->tokens;
    p.positions = a->positions;
    p.starts = a->starts;
    p.cow_src = a->cow_src;
    p.freqs = a->freqs;
    p.units = a->rot_dim / 16;
    p.neighbours = a->pairing == RL_ROPE_NEIGHBOURS;
    p.q = (const uint16_t *)a->q;
    p.k = (const uint16_t *)a->k_new;
    p.v = (const uint16_t *)a->v_new;
    p.q_out = (uint16_t *)a->q_out;
    p.k_out = (uint16_t *)a->k_out;
    const uint64_t qrow = (uint64_t)a->q_heads * d, kvrow = (uint64_t)a->kv_heads * d;
    p.q_stride = a->q_stride ? a->q_stride : qrow;
    p.q_out_stride = a->q_out_stride ? a->q_out_stride : qrow;
    p.k_stride = a->k_stride ? a->k_stride : kvrow;
    p.v_stride = a->v_stride ? a->v_stride : kvrow;
    p.k_out_stride = a->k_out_stride ? a->k_out_stride : kvrow;
    const uint64_t groups = ((uint64_t)a->tokens * (d / 16) + 63) / 64;
    // Heads per wave: as many as leave two waves for each SIMD (24 x 1-301 tokens of 24 heads, d64: 7.0 us; with one
    // wave 7.7, with four 7.4).
    const uint64_t enough = 8ull * rl_cu_count();
    const uint32_t per = groups * ((p.heads + 3) / 4) >= enough ? 4 : groups * ((p.heads + 1) / 2) >= enough ? 2 : 1;
    p.slices = (p.heads + per - 1) / per;
    const uint64_t copies = a->cow_src ? (uint64_t)a->batch * a->kv_heads : 0;
    // (a launch holds less than 2^32 work-items, 64 for each of these)
    if (groups * p.slices + copies >= (1u << 26) - kWaves) {
        rl_set_error("%s: %u tokens of %u heads (with %u x %u copies) exceed 2^26 waves", who, a->tokens, p.heads, a->batch,
                     a->kv_heads);
        return -1;
    }
    p.items = (uint32_t)(groups * p.slices);
    p.copies = (uint32_t)copies;
    if (d == 128)
        return a->dtype == RL_DTYPE_BF16 ? launch<128, 0>(p, per) : launch<128, 1>(p, per);
    return a->dtype == RL_DTYPE_BF16 ? launch<64, 0>(p, per) : launch<64, 1>(p, per);
}
