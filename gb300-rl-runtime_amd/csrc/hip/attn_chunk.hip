// attn_chunk.hip - causal attention of chunks of new tokens over the 16-bit paged
// arena. The kernels of many rows or long contexts, what bounds them and what they
// measure are in prompt_core.h; here is the one of few rows behind short contexts, for
// which latency counts:
//
//  split  a workgroup has 32 rows of a (sequence, KV head), and its four waves share
//         their keys, 32 at a time in turn, each with copies and sums of its own and
//         no barrier until the sums are joined in LDS (1 x 37 queries of 32 heads, 8
//         KV heads, d128, behind 480 tokens 9.9 us; four waves of 32 rows each that go
//         through all keys together 12.5; behind 1,000 14.8 against 17.5; 16 x 8
//         behind 2,000 30.0 against 37.0).
//  bound  the chain launch, context, block id, keys, sums, joined sums; of a wave's
//         units each about 1.1 us, with the next one's copies in flight. Two sums for
//         the scores, so that matrix instructions wait less, changed nothing.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cmath>

#include "kv_layout.h"
#include "prompt_core.h"
#include "rl_hip.h"
#include "rl_hip_internal.h"

namespace {

constexpr uint32_t kFewRows = 256;  // of a sequence and KV head

template <int D, int DT>
__global__ __launch_bounds__(256, 1) void attn_chunk_few_kernel(PromptParams p)
{
    using C = PCfg<D>;
    constexpr int UNIT = 32;                     // keys
    constexpr int PLANE = UNIT * C::RB;
    constexpr int OPS = PLANE / 1024;            // copies of a unit's keys, or values
    constexpr int PER = 64 / C::NC;              // rows of a copy
    constexpr int OWN = 2 * 2 * PLANE;           // a wave's LDS: two stages
    __shared__ __attribute__((aligned(1024))) uint8_t smem[4 * OWN];
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t hf = (uint32_t)lane >> 5, lr = (uint32_t)lane & 31u;
    const Place x = place_of<true>(p, blockIdx.x, lane);
    const uint32_t lq = x.lq, lk = x.lk;
    const uint32_t rows = min(lq, p.max_q) * p.group, row0 = x.tile * 32;
    if (row0 >= rows)
        return;
    auto seen = [&](uint32_t t) { return (uint32_t)max((int32_t)(t - lq + 1) + (int32_t)lk, 0); };
    const uint32_t tok0 = quotient(row0, p.by_group), h0 = row0 - tok0 * p.group;
    const uint32_t most = seen(quotient(min(row0 + 32, rows) - 1, p.by_group)), least = seen(tok0);
    // (rows past the last repeat it)
    const uint32_t my_x = h0 + min(row0 + lr, rows - 1) - row0, my_dt = quotient(my_x, p.by_group);
    const uint32_t my_seen = seen(tok0 + my_dt);
    const uint32_t all = (most + UNIT - 1) / UNIT, units = all > wave ? (all - wave + 3) / 4 : 0u;

    // ---- the copies: unit i of this wave has the keys 32 (wave + 4 i) on, two runs of 16 that lie in a block each.
    // Lane j knows the block of run j % 2 of unit ids_from + j / 2.
    const uint32_t *table = p.table + ((uint64_t)x.seq * p.kv_heads + x.g) * p.table_stride;
    const uint32_t last16 = lk > 0 ? (lk - 1) & ~15u : 0u;
    uint32_t ids = 0xFFFFFFFFu, ids_from = 0;
    auto look_up = [&](uint32_t i) {
        ids_from = i;
        const uint32_t token = min((wave + 4 * (i + (uint32_t)lane / 2)) * UNIT + (lane & 1) * 16u, last16);
        ids = x.lost ? 0xFFFFFFFFu : table[token >> p.tpb_shift];
        asm volatile("" : "+v"(ids));  // (settled here: the compiler does not see the copies' waits)
    };
    auto plane_of = [&](uint32_t id, int plane, uint32_t slot) {
        const uint8_t *at = p.arena + (uint64_t)id * p.block_bytes + (plane * p.tpb + slot) * (uint32_t)C::RB;
        return id < p.arena_blocks ? at : (const uint8_t *)(plane ? g_lost.value : g_lost.key);
    };
    RL_LDS uint8_t *own = (RL_LDS uint8_t *)smem + wave * OWN;
    const uint32_t cr = (uint32_t)lane / C::NC, pos = (uint32_t)lane % C::NC;
    auto copy = [&](uint32_t i) {
        if (i - ids_from > 31)
            look_up(i);
        RL_LDS uint8_t *dst = own + i % 2 * (2 * PLANE);
#pragma unroll
        for (int j = 0; j < OPS; j++) {
            const uint32_t run = j / (OPS / 2), token = min((wave + 4 * i) * UNIT + 16 * run, last16);
            const uint32_t row = j * PER + cr, in = min(row & 15u, lk - token - 1);  // (past the last key: that again)
            const uint32_t id = rl_readlane(ids, (int)(2 * (i - ids_from) + run)), slot = token & (p.tpb - 16u);
            rl_g2lds_16_off(plane_of(id, 0, slot), in * C::RB + ((pos ^ C::kswz(row)) << 4), dst + j * 1024);
            rl_g2lds_16_off(plane_of(id, 1, slot), in * C::RB + ((pos ^ C::vswz(row)) << 4), dst + PLANE + j * 1024);
        }
    };
    if (units > 0) {
        look_up(0);
        copy(0);
    }
    s16x8 qf[C::KS];
    {
        const uint16_t *q = p.q + (uint64_t)(x.qs + tok0 + my_dt) * p.q_stride +
                            (uint64_t)(x.g * p.group + my_x - my_dt * p.group) * D + 8 * hf;
#pragma unroll
        for (int s = 0; s < C::KS; s++)
            qf[s] = *(const s16x8 *)(q + 16 * s);
#pragma unroll
        for (int s = 0; s < C::KS; s++)
            asm volatile("" : "+v"(qf[s]));
    }
    if (units > 1)
        copy(1);
    f32x16 o[C::DB];
#pragma unroll
    for (int d = 0; d < C::DB; d++)
        o[d] = f32x16{};
    float m = -INFINITY, l = 0.f;
    const uint32_t vr = 4u * hf + (((uint32_t)lane & 15u) >> 2);
    const uint32_t vc = 2u * (((uint32_t)lane >> 4) & 1u) + (((uint32_t)lane & 3u) >> 1);
    for (uint32_t i = 0; i < units; i++) {
        if (i + 1 < units)
            rl_wait_vmcnt<2 * OPS>();
        else
            rl_wait_vmcnt<0>();
        RL_LDS const uint8_t *ks = own + i % 2 * (2 * PLANE), *vs = ks + PLANE;
        const uint32_t k0 = (wave + 4 * i) * UNIT;
        // (operands as in prompt_core.h: S^T leaves this lane with row lr and the keys 8 a + 4 hf .. + 3)
        f32x16 s{};
#pragma unroll
        for (int e = 0; e < C::KS; e++)
            s = mfma32<DT>(*(RL_LDS const s16x8 *)(ks + lr * C::RB + (((2u * e + hf) ^ C::kswz(lr)) << 4)), qf[e], s);
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            if (k0 + UNIT > least)
                s[e] = k0 + 8 * (e / 4) + 4 * hf + e % 4 < my_seen ? s[e] : -INFINITY;
            top = fmaxf(top, s[e]);
        }
        top = half_max(top) * p.scale_log2;
        if (__builtin_amdgcn_ballot_w64(top > m + kSlack) != 0) {
            // (a row's reference rises by its own scores alone, so that its output does not depend on its neighbours)
            const float m_new = top > m + kSlack ? top : m, alpha = m_new == -INFINITY ? 1.f : exp2f(m - m_new);
            l *= alpha;
#pragma unroll
            for (int d = 0; d < C::DB; d++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    o[d][e] *= alpha;
            m = m_new;
        }
        const float neg = m == -INFINITY ? 0.f : -m;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], p.scale_log2, neg));
            l += s[e];
        }
        // Infinities and NaN among the values spoil the matrix product for rows that do not see them (0 times NaN), and
        // in fp16, whose weights may round to 0, for those that do: such units are summed key by key.
        uint32_t spoilt = 0;
        if (DT != 0 || k0 + UNIT > least) {
            constexpr uint32_t kExp = DT == 0 ? 0x7F807F80u : 0x7C007C00u, kOne = DT == 0 ? 0x00800080u : 0x04000400u;
#pragma unroll
            for (int j = 0; j < OPS; j++) {
                const rl_u32x4 w = *(RL_LDS const rl_u32x4 *)(vs + j * 1024 + lane * 16);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    spoilt |= ((w[e] & kExp) + kOne) & 0x80008000u;  // (all exponent bits set)
            }
        }
        if (__builtin_amdgcn_ballot_w64(spoilt != 0) == 0) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const s16x8 pf = __builtin_bit_cast(
                    s16x8, (rl_u32x4{pack2<DT>(s[8 * u], s[8 * u + 1]), pack2<DT>(s[8 * u + 2], s[8 * u + 3]),
                                     pack2<DT>(s[8 * u + 4], s[8 * u + 5]), pack2<DT>(s[8 * u + 6], s[8 * u + 7])}));
#pragma unroll
                for (int d = 0; d < C::DB; d++) {
                    RL_LDS const uint8_t *at = vs + (vr + 16 * u) * C::RB + 8 * (lane & 1);
                    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (RL_LDS s16x4 *)(at + (((4u * d + vc) ^ C::vswz(vr)) << 4)));
                    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (RL_LDS s16x4 *)(at + 8 * C::RB + (((4u * d + vc) ^ C::vswz(vr + 8)) << 4)));
                    o[d] = mfma32<DT>(__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7), pf, o[d]);
                }
            }
        } else {
            // the weights to where the keys were, [key][row], then each key's values for the rows that see it
            RL_LDS float *w = (RL_LDS float *)(own + i % 2 * (2 * PLANE));
            rl_wait_lgkmcnt0();
#pragma unroll
            for (int e = 0; e < 16; e++)
                w[(8 * (e / 4) + 4 * hf + e % 4) * 32 + lr] = s[e];
            rl_wave_lds_fence();
            for (uint32_t k = 0; k < UNIT && k0 + k < most; k++) {
                const float f = w[k * 32 + lr];
#pragma unroll
                for (int d = 0; d < C::DB; d++)
#pragma unroll
                    for (int a = 0; a < 4; a++) {
                        const s16x4 v =
                            *(RL_LDS const s16x4 *)(vs + k * C::RB + (((4u * d + a) ^ C::vswz(k)) << 4) + 8 * hf);
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            o[d][4 * a + e] = k0 + k < my_seen
                                                  ? fmaf(f, from16<DT>((uint16_t)v[e]), o[d][4 * a + e])
                                                  : o[d][4 * a + e];
                    }
            }
        }
        rl_wait_lgkmcnt0();  // (nothing of the stage is still being read)
        if (i + 2 < units)
            copy(i + 2);
    }
    // ---- the waves' sums joined: wave d the dims 32 d .. 32 d + 31 --------------------
    rl_wait_vmcnt<0>();
    const float L = half_sum(l);
    float *sums = (float *)(smem + wave * OWN);
#pragma unroll
    for (int d = 0; d < C::DB; d++)
#pragma unroll
        for (int a = 0; a < 4; a++)
            *(rl_f32x4 *)(sums + ((4 * d + a) * 64 + lane) * 4) =
                rl_f32x4{o[d][4 * a], o[d][4 * a + 1], o[d][4 * a + 2], o[d][4 * a + 3]};
    sums[C::DB * 16 * 64 + lane] = m;
    sums[(C::DB * 16 + 1) * 64 + lane] = L;
    __syncthreads();
    if (wave >= C::DB)
        return;
    float top = -INFINITY, total = 0.f, y[16];
#pragma unroll
    for (int e = 0; e < 16; e++)
        y[e] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++)
        top = fmaxf(top, ((const float *)(smem + w * OWN))[C::DB * 16 * 64 + lane]);
#pragma unroll
    for (int w = 0; w < 4; w++) {
        const float *in = (const float *)(smem + w * OWN);
        const float mw = in[C::DB * 16 * 64 + lane], f = mw == -INFINITY ? 0.f : exp2f(mw - top);
        const float lw = in[(C::DB * 16 + 1) * 64 + lane];
        total = fmaf(lw, f, total);
#pragma unroll
        for (int a = 0; a < 4; a++) {
            const rl_f32x4 z = *(const rl_f32x4 *)(in + ((4 * wave + a) * 64 + lane) * 4);
            // (a wave without a key that the row sees has sums of 0, or what is no number)
#pragma unroll
            for (int e = 0; e < 4; e++)
                y[4 * a + e] = fmaf(z[e], f, y[4 * a + e]);
        }
    }
    const float inv = my_seen == 0 ? 0.f : 1.f / total;
    uint16_t *out = p.out + (uint64_t)(x.qs + tok0 + my_dt) * p.out_stride +
                    (uint64_t)(x.g * p.group + my_x - my_dt * p.group) * D + 32 * wave + 8 * hf;
#pragma unroll
    for (int a = 0; a < 4; a += 2) {
        // lanes l and l + 32 hold four dims each of both 8-dim chunks: each takes a whole one
        rl_u32x4 w;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const uint32_t c = pack2<DT>(y[4 * a + 2 * e] * inv, y[4 * a + 2 * e + 1] * inv);
            const uint32_t b = pack2<DT>(y[4 * a + 4 + 2 * e] * inv, y[4 * a + 5 + 2 * e] * inv);
            const auto h = __builtin_amdgcn_permlane32_swap(c, b, false, false);
            w[e] = h[0];
            w[2 + e] = h[1];
        }
        if (row0 + lr < rows)
            *(rl_u32x4 *)(out + 8 * a) = w;
    }
}

template <int D, int DT>
int launch_few(const PromptParams &p)
{
    hipLaunchKernelGGL((attn_chunk_few_kernel<D, DT>), dim3(p.pairs * p.tiles), dim3(256), 0, rl_stream(), p);
    return rl_check_launch("attn_chunk_few_kernel launch");
}

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
    // Few rows, at most one workgroup per compute unit, where the keys of a wave, 1.1 us for 32, take less than those of
    // a share among the other kernel's workgroups, 0.9 us for 64, and the launch that joins the shares, 5 us.
    const uint64_t group = a->q_heads / a->kv_heads, tiles = (a->max_q * group + 31) / 32;
    const uint64_t units = ((uint64_t)a->max_ctx + 31) / 32, per_share = ((units + 1) / 2 + pl.split - 1) / pl.split;
    const bool few = a->max_q * group <= kFewRows && tiles * a->batch * a->kv_heads <= rl_cu_count() &&
                     11 * ((units + 3) / 4) < 9 * per_share + (pl.split > 1 ? 50 : 0);
    PromptPlan plan = pl;
    if (few) {
        plan.tiles = (uint32_t)tiles;
        plan.split = 1;
    }
    set_plan(p, plan, a->batch, a->max_ctx, a->q_heads, a->kv_heads, a->layout.head_dim, a->scale, a->workspace);
    if (few && a->layout.head_dim == 128)
        return a->dtype == RL_DTYPE_BF16 ? launch_few<128, 0>(p) : launch_few<128, 1>(p);
    if (few)
        return a->dtype == RL_DTYPE_BF16 ? launch_few<64, 0>(p) : launch_few<64, 1>(p);
    if (a->layout.head_dim == 128)
        return a->dtype == RL_DTYPE_BF16 ? prompt_launch<128, 0, true>(p) : prompt_launch<128, 1, true>(p);
    return a->dtype == RL_DTYPE_BF16 ? prompt_launch<64, 0, true>(p) : prompt_launch<64, 1, true>(p);
}
