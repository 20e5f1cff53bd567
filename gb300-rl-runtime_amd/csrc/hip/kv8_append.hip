// kv8_append.hip - K/V rows into the 8-bit paged arena, whole prompts or one
// token per row, on gfx950.
//
// For every block that a row's new tokens reach, and each plane (K, V) of it:
//   s = the smallest power of two with 448 s >= every finite new value's
//       magnitude, and not below the scale the block already has when it
//       holds earlier tokens of the row;
//   new bytes  e4m3(x / s); earlier bytes e4m3(value s_old / s) where s grew.
// e4m3 keeps four significant bits at any exponent, so a scale that is no
// power of two would round no better; with powers of two the division is
// exact and a growing scale only moves the earlier values' exponents (values
// that end below 2^-6 s are rounded again).
//
// One wave per (row, block, KV head): a lane holds eight elements of every
// 512 / head_dim-th token of both planes, so that a block is read once, its
// largest magnitudes are reduced across the wave in registers, and the bytes
// leave in 8-byte stores. The rows are read past the caches, for this is their
// last use (60.9 us against 65.2 below, 57 against 62 for rows that were just
// written); the blocks are not written past them (58.2), for the next decode
// step reads them. Bound: the bytes, 2 in and 1 out per element (64 prompts of
// 512-1,024 tokens, 302 MB in 60.9 us: 4.95 TB/s, 97% of a plain copy); for one
// token per row the chain position, table entry, scale, store (64 rows x 8
// heads: 4.2 us).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "attn_core.h"
#include "kv8_core.h"
#include "rl_hip.h"
#include "rl_hip_internal.h"

namespace {

constexpr int kWaves = 4;
constexpr float kMostFinite = 3.4028234663852886e38f;

struct Append8Params {
    uint8_t *arena;
    uint64_t block_bytes;
    uint64_t arena_blocks;
    const uint32_t *table;
    uint32_t table_stride;
    uint32_t kv_heads;
    uint32_t touched;   // blocks of a row that max_new tokens may reach
    uint32_t items;     // batch * touched * kv_heads
    const uint32_t *positions;
    const uint32_t *starts;  // NULL: one token per row
    uint32_t tokens;
    uint32_t max_new;
    const int32_t *cow_src;
    const uint16_t *k_new;
    const uint16_t *v_new;
    uint64_t k_stride, v_stride;  // elements between tokens
};

template <int DT>
__device__ __forceinline__ void unpack8(const rl_u32x4 &w, float (&f)[8])
{
#pragma unroll
    for (int i = 0; i < 4; i++)
        rl_unpack2<DT>(w[i], f[2 * i], f[2 * i + 1]);
}

// The larger of x over the wave's 64 lanes, in every lane.
__device__ __forceinline__ float wave_max(float x) { return tile_max(rl_row_max(x)); }

template <int D, int TPB, int DT>
__global__ __launch_bounds__(kWaves * 64) void kv8_append_kernel(Append8Params p)
{
    constexpr int LPR = D / 8;             // lanes per token
    constexpr int RPP = 64 / LPR;          // tokens per pass
    constexpr int PASSES = TPB / RPP;
    const int lane = threadIdx.x & 63;
    const uint32_t item = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (item >= p.items)
        return;
    const uint32_t g = item % p.kv_heads, bj = item / p.kv_heads;
    const uint32_t b = bj / p.touched, j = bj % p.touched;

    const uint32_t pos = rl_sload(p.positions + b);
    uint32_t first = b, n = b < p.tokens ? 1u : 0u;
    if (p.starts) {
        first = rl_sload(p.starts + b);
        const uint32_t end = min(rl_sload(p.starts + b + 1), p.tokens);
        n = end > first ? min(end - first, p.max_new) : 0u;
    }
    const uint32_t lb = pos / TPB + j;
    if (n == 0 || lb >= p.table_stride)
        return;
    // slots [lo, hi) of this block are new; those below lo hold earlier tokens
    const uint32_t lo = j == 0 ? pos % TPB : 0u;
    const uint64_t end = (uint64_t)pos + n;
    if (end <= (uint64_t)lb * TPB)
        return;
    const uint32_t hi = (uint32_t)min<uint64_t>(end - (uint64_t)lb * TPB, TPB);
    const uint32_t blk = rl_sload(p.table + ((size_t)b * p.kv_heads + g) * p.table_stride + lb);
    if (blk >= p.arena_blocks)
        return;
    uint8_t *dst = p.arena + (uint64_t)blk * p.block_bytes;

    const uint32_t r0 = (uint32_t)lane / LPR, c = (uint32_t)lane % LPR;
    const uint32_t tok0 = first + (uint32_t)((uint64_t)lb * TPB + lo - pos);  // token of slot lo
    rl_u32x4 kw[PASSES], vw[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const uint32_t slot = r0 + i * RPP;
        kw[i] = vw[i] = rl_u32x4{0, 0, 0, 0};
        if (slot >= lo && slot < hi) {
            const uint64_t t = tok0 + (slot - lo);
            kw[i] = __builtin_nontemporal_load((const rl_u32x4 *)(p.k_new + t * p.k_stride + g * D + c * 8));
            vw[i] = __builtin_nontemporal_load((const rl_u32x4 *)(p.v_new + t * p.v_stride + g * D + c * 8));
        }
    }
    // the block that holds the earlier tokens: this one, or the shared one that is copied
    const uint8_t *src = dst;
    if (p.cow_src && j == 0 && lo > 0) {
        const int32_t s = p.cow_src[(size_t)b * p.kv_heads + g];
        if (s >= 0 && (uint64_t)s < p.arena_blocks)
            src = p.arena + (uint64_t)(uint32_t)s * p.block_bytes;
    }
    uint32_t old_exp[2] = {0, 0};
    if (lo > 0) {
        const rl_f32x2 old = *(const rl_f32x2 *)(src + 2 * TPB * D);
#pragma unroll
        for (int q = 0; q < 2; q++)  // (bounded also for a block that was never written)
            old_exp[q] = min(max((__float_as_uint(old[q]) >> 23) & 0xFFu, 1u), 247u);
    }
    uint32_t exps[2];
#pragma unroll
    for (int q = 0; q < 2; q++) {
        const rl_u32x4(&w)[PASSES] = q ? vw : kw;
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < PASSES; i++) {
            float f[8];
            unpack8<DT>(w[i], f);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float a = fabsf(f[e]);
                amax = fmaxf(amax, a <= kMostFinite ? a : 0.f);  // infinities and NaN set no scale
            }
        }
        exps[q] = max(kv8_scale_exponent(wave_max(amax)), old_exp[q]);
        const float inv = kv8_inverse(exps[q]);
        uint8_t *plane = dst + q * TPB * D + c * 8;
        if (lo > 0 && (exps[q] != old_exp[q] || src != dst)) {
            // earlier tokens: to the new scale (times 1 when only copied)
            const float ratio = kv8_scale(old_exp[q]) * inv;
            const uint8_t *from = src + q * TPB * D + c * 8;
#pragma unroll
            for (int i = 0; i < PASSES; i++) {
                const uint32_t slot = r0 + i * RPP;
                if (slot < lo) {
                    const rl_u32x2 o = *(const rl_u32x2 *)(from + slot * D);
                    rl_u32x2 r;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const rl_f32x2 x = __builtin_amdgcn_cvt_pk_f32_fp8((int)o[h], false);
                        const rl_f32x2 y = __builtin_amdgcn_cvt_pk_f32_fp8((int)o[h], true);
                        r[h] = kv8_pack4(x[0] * ratio, x[1] * ratio, y[0] * ratio, y[1] * ratio);
                    }
                    *(rl_u32x2 *)(plane + slot * D) = r;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < PASSES; i++) {
            const uint32_t slot = r0 + i * RPP;
            if (slot >= lo && slot < hi) {
                float f[8];
                unpack8<DT>(w[i], f);
#pragma unroll
                for (int e = 0; e < 8; e++)  // e4m3 has no infinity: both become NaN
                    f[e] = fabsf(f[e]) <= kMostFinite ? f[e] * inv : __builtin_nanf("");
                rl_u32x2 r;
                r[0] = kv8_pack4(f[0], f[1], f[2], f[3]);
                r[1] = kv8_pack4(f[4], f[5], f[6], f[7]);
                *(rl_u32x2 *)(plane + slot * D) = r;
            }
        }
    }
    if (lane == 0)
        *(rl_f32x2 *)(dst + 2 * TPB * D) = rl_f32x2{kv8_scale(exps[0]), kv8_scale(exps[1])};
}

template <int D, int TPB>
int launch(const Append8Params &p, uint32_t dtype)
{
    const uint32_t grid = (p.items + kWaves - 1) / kWaves;
    if (dtype == RL_DTYPE_BF16)
        hipLaunchKernelGGL((kv8_append_kernel<D, TPB, 0>), dim3(grid), dim3(kWaves * 64), 0, rl_stream(), p);
    else
        hipLaunchKernelGGL((kv8_append_kernel<D, TPB, 1>), dim3(grid), dim3(kWaves * 64), 0, rl_stream(), p);
    return rl_check_launch("kv8_append_kernel launch");
}

// Blocks of a row that max_new tokens may reach: the worst first position is a
// block's last slot, and the table has no more.
uint64_t touched_of(const rl_kv8_append_args_t *a)
{
    const uint64_t tpb = a->layout.token_count;
    return std::min<uint64_t>(((uint64_t)a->max_new + tpb - 2) / tpb + 1, a->table_stride);
}

int validate(const rl_kv8_append_args_t *a)
{
    const char *who = "rl_hip_kv8_append";
    if (!a || !a->arena_base || !a->block_table || !a->positions || !a->k_new || !a->v_new) {
        rl_set_error("%s: NULL argument", who);
        return -1;
    }
    if (kv_layout_check_paged8(&a->layout) != 0) {
        rl_set_error("%s: unsupported KV layout (token_count %u, head_dim %u, scalar %u, block of %u bytes)", who,
                     a->layout.token_count, a->layout.head_dim, a->layout.scalar_bytes, a->layout.block_bytes);
        return -1;
    }
    if (a->dtype != RL_DTYPE_BF16 && a->dtype != RL_DTYPE_FP16) {
        rl_set_error("%s: dtype %u", who, a->dtype);
        return -1;
    }
    if (a->batch == 0 || a->kv_heads == 0 || a->batch > 65535 || a->kv_heads > 65535) {
        rl_set_error("%s: batch %u kv_heads %u out of range", who, a->batch, a->kv_heads);
        return -1;
    }
    if (a->max_new == 0 || (!a->starts && a->max_new != 1)) {
        rl_set_error("%s: max_new %u (1 without starts, at least 1 with them)", who, a->max_new);
        return -1;
    }
    // (a launch holds less than 2^32 work-items, 64 for each of these)
    if ((uint64_t)a->batch * a->kv_heads * touched_of(a) > (1u << 25)) {
        rl_set_error("%s: batch %u x kv_heads %u x the blocks of max_new %u tokens exceed 2^25", who, a->batch,
                     a->kv_heads, a->max_new);
        return -1;
    }
    if (!a->starts && a->tokens != a->batch) {
        rl_set_error("%s: %u tokens for %u rows of one token each", who, a->tokens, a->batch);
        return -1;
    }
    if (a->arena_bytes < a->layout.block_bytes) {
        rl_set_error("%s: arena of %llu bytes holds no block", who, (unsigned long long)a->arena_bytes);
        return -1;
    }
    const uint64_t row = (uint64_t)a->kv_heads * a->layout.head_dim;
    const uint32_t strides[2] = {a->k_stride, a->v_stride};
    for (int i = 0; i < 2; i++)
        if (strides[i] != 0 && (strides[i] < row || strides[i] % 8 != 0)) {
            rl_set_error("%s: k_stride %u / v_stride %u (0, or multiples of 8 of at least kv_heads x head_dim = %llu)",
                         who, a->k_stride, a->v_stride, (unsigned long long)row);
            return -1;
        }
    if (((uintptr_t)a->arena_base | (uintptr_t)a->k_new | (uintptr_t)a->v_new) % 16 != 0) {
        rl_set_error("%s: arena_base, k_new and v_new must be 16-byte aligned", who);
        return -1;
    }
    return 0;
}

}  // namespace

extern "C" int rl_hip_kv8_append(const rl_kv8_append_args_t *a)
{
    if (validate(a) || rl_require_open("rl_hip_kv8_append"))
        return -1;
    const uint32_t tpb = a->layout.token_count, d = a->layout.head_dim;
    Append8Params p;
    p.arena = (uint8_t *)a->arena_base;
    p.block_bytes = a->layout.block_bytes;
    p.arena_blocks = a->arena_bytes / a->layout.block_bytes;
    p.table = a->block_table;
    p.table_stride = a->table_stride;
    p.kv_heads = a->kv_heads;
    p.touched = (uint32_t)touched_of(a);
    if (p.touched == 0)
        return 0;  // a table without entries: every position lies past it
    p.items = a->batch * p.touched * a->kv_heads;
    p.positions = a->positions;
    p.starts = a->starts;
    p.tokens = a->tokens;
    p.max_new = a->max_new;
    p.cow_src = a->cow_src;
    p.k_new = (const uint16_t *)a->k_new;
    p.v_new = (const uint16_t *)a->v_new;
    p.k_stride = a->k_stride ? a->k_stride : (uint64_t)a->kv_heads * d;
    p.v_stride = a->v_stride ? a->v_stride : (uint64_t)a->kv_heads * d;
    if (d == 128)
        return tpb == 16 ? launch<128, 16>(p, a->dtype) : launch<128, 32>(p, a->dtype);
    return tpb == 16 ? launch<64, 16>(p, a->dtype) : launch<64, 32>(p, a->dtype);
}
