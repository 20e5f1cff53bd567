// attn_prompt.hip - causal attention over whole prompts, packed sequences with
// grouped heads, written for gfx950.
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j <= i + Lk - Lq
//
// of a sequence with Lq queries and Lk >= Lq keys (the queries are its last
// tokens). Bound: the matrix cores from some hundred tokens on, 4 head_dim
// operations per head and visible pair; K and V come from L2.
//
//  rows   a workgroup of NW waves takes 32 NW rows of one (sequence, KV head);
//         row r is query token r / G, head r % G of the group, so that a
//         group's heads share every K and V tile and a wave's rows span few
//         tokens (little masked work on the diagonal).
//  stage  64 tokens of K and V are copied to LDS with global_load_lds (16 B per
//         lane), double-buffered, one barrier per tile. The 16-byte chunks of
//         a row are permuted so that the operand reads below meet no bank
//         conflict.
//  QK     v_mfma_f32_32x32x16: A = K rows, B = q^T (in registers for the whole
//         row block). S^T leaves lane l with row l % 32 and tokens 8 a + 4 (l /
//         32) .. + 3: the softmax of a row is in two lanes' registers, and
//         S^T, rounded to 16 bits, is the B operand of
//  PV     O^T += V^T P^T, whose A operand ds_read_b64_tr_b16 takes from the
//         row-major V tile in the same token order. P in the inputs' type: its
//         rounding, 2^-9 of each weight with bf16, is of the order of the
//         output's own.
//  softmax online; the maximum a row's weights refer to is raised only when it
//         is exceeded by more than 2^8, which the fp32 sums and 16-bit weights
//         hold without loss, so the output is rarely rescaled.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "attn_core.h"
#include "rl_dev_common.h"
#include "rl_hip.h"
#include "rl_hip_internal.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int BT = 64;         // keys per tile
constexpr float kSlack = 8.f;  // log2 of what a weight may exceed its reference by

struct PromptParams {
    const uint16_t *q, *k, *v;
    uint16_t *out;
    uint64_t q_stride, k_stride, v_stride, out_stride;  // elements between tokens
    const uint32_t *q_starts, *kv_starts;
    uint32_t q_tokens, kv_tokens;
    uint32_t kv_heads, group;
    uint32_t pairs;   // sequences x KV heads
    uint32_t tiles;   // row blocks of the longest sequence
    uint32_t by_xcd;  // a pair's row blocks all on one XCD
    float scale_log2;
};

template <int D>
struct PCfg {
    static constexpr int RB = 2 * D;             // bytes of a K or V row
    static constexpr int NC = D / 8;             // 16-byte chunks of a row
    static constexpr int PLANE = BT * RB;
    static constexpr int OPS = PLANE / 1024;     // 1 KiB copies per plane
    static constexpr int KS = D / 16;            // k-steps of QK
    static constexpr int DB = D / 32;            // 32-dim blocks of the output
    // LDS position of chunk c of row t is c ^ swizzle(t). K is read 16 rows x
    // one chunk at a time, V (transposed) four rows x four chunks.
    static __device__ __forceinline__ uint32_t kswz(uint32_t t) { return D == 128 ? t & 15u : (t >> 1) & 7u; }
    static __device__ __forceinline__ uint32_t vswz(uint32_t t)
    {
        return D == 128 ? ((t & 3u) << 2) | ((t >> 2) & 3u) : ((t >> 1) & 1u) << 2;
    }
};

template <int DT>
__device__ __forceinline__ f32x16 mfma32(s16x8 a, s16x8 b, f32x16 c)
{
    if constexpr (DT == 0)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b)
{
    if constexpr (DT == 0) {
        rl_bf16x2 w;
        w[0] = (__bf16)a;
        w[1] = (__bf16)b;
        return __builtin_bit_cast(uint32_t, w);
    } else {
        rl_f16x2 w;
        w[0] = (_Float16)a;
        w[1] = (_Float16)b;
        return __builtin_bit_cast(uint32_t, w);
    }
}

// The larger (the sum) of lanes l and l ^ 32, in both.
__device__ __forceinline__ float half_max(float x)
{
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
}
__device__ __forceinline__ float half_sum(float x)
{
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}

template <int D, int DT, int NW>
__global__ __launch_bounds__(NW * 64, 2) void attn_prompt_kernel(PromptParams p)
{
    using C = PCfg<D>;
    constexpr int WOPS = C::OPS / NW;  // copies of a plane per wave
    static_assert(WOPS * NW == C::OPS, "whole copies per wave");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[2][2 * C::PLANE];
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t hf = (uint32_t)lane >> 5;

    // heavy row blocks (the last ones) first
    uint32_t pair, tile;
    if (p.by_xcd) {  // workgroup b runs on XCD b % 8
        const uint32_t local = blockIdx.x / 8;
        pair = blockIdx.x % 8 + 8 * (local / p.tiles);
        tile = p.tiles - 1 - local % p.tiles;
    } else {
        pair = blockIdx.x % p.pairs;
        tile = p.tiles - 1 - blockIdx.x / p.pairs;
    }
    const uint32_t seq = pair / p.kv_heads, g = pair % p.kv_heads;
    const uint32_t qs = rl_sload(p.q_starts + seq), qe = min(rl_sload(p.q_starts + seq + 1), p.q_tokens);
    const uint32_t ks = rl_sload(p.kv_starts + seq), ke = min(rl_sload(p.kv_starts + seq + 1), p.kv_tokens);
    const uint32_t lq = qe > qs ? qe - qs : 0u, lk = ke > ks ? ke - ks : 0u;
    const uint64_t rows = (uint64_t)lq * p.group;
    const uint64_t wg_row = (uint64_t)tile * (NW * 32);
    if (wg_row >= rows)
        return;
    // keys that query token t sees: t + lk - lq + 1, not below 0
    auto seen = [&](uint32_t t) { return (uint32_t)max<int64_t>((int64_t)t + lk - lq + 1, 0); };
    const uint32_t wg_seen = seen((uint32_t)(min<uint64_t>(wg_row + NW * 32, rows) - 1) / p.group);
    const uint64_t w_row = wg_row + wave * 32;
    const bool w_has = w_row < rows;
    const uint32_t w_least = w_has ? seen((uint32_t)(w_row / p.group)) : 0u;
    const uint32_t w_most = w_has ? seen((uint32_t)((min<uint64_t>(w_row + 32, rows) - 1) / p.group)) : 0u;
    const uint64_t my_row = w_row + (lane & 31);
    const uint32_t my = (uint32_t)min<uint64_t>(my_row, rows - 1);
    const uint32_t my_tok = my / p.group, my_head = g * p.group + my % p.group;
    const uint32_t my_seen = seen(my_tok);

    s16x8 qf[C::KS];
    {
        const uint16_t *q = p.q + (uint64_t)(qs + my_tok) * p.q_stride + (uint64_t)my_head * D + 8 * hf;
#pragma unroll
        for (int s = 0; s < C::KS; s++)
            qf[s] = *(const s16x8 *)(q + 16 * s);
    }
    f32x16 o[C::DB];
#pragma unroll
    for (int d = 0; d < C::DB; d++)
        o[d] = f32x16{};
    float m = -INFINITY, l = 0.f;

    // ---- the tiles -------------------------------------------------------------
    const uint16_t *kbase = p.k + (uint64_t)ks * p.k_stride + (uint64_t)g * D;
    const uint16_t *vbase = p.v + (uint64_t)ks * p.v_stride + (uint64_t)g * D;
    auto stage = [&](uint32_t t) {
        RL_LDS uint8_t *kd = (RL_LDS uint8_t *)smem[t & 1];
        RL_LDS uint8_t *vd = kd + C::PLANE;
        const uint32_t left = lk - t * BT;  // keys from this tile on; rows past them repeat the last
        const uint16_t *kt = kbase + (uint64_t)t * BT * p.k_stride;
        const uint16_t *vt = vbase + (uint64_t)t * BT * p.v_stride;
#pragma unroll
        for (int i = 0; i < WOPS; i++) {
            const uint32_t op = wave * WOPS + i;
            const uint32_t r = op * (64 / C::NC) + (uint32_t)lane / C::NC, pos = (uint32_t)lane % C::NC;
            const uint32_t rc = min(r, left - 1);
            rl_g2lds_16_off(kt, rc * (uint32_t)p.k_stride * 2u + ((pos ^ C::kswz(r)) << 4), kd + op * 1024);
            rl_g2lds_16_off(vt, rc * (uint32_t)p.v_stride * 2u + ((pos ^ C::vswz(r)) << 4), vd + op * 1024);
        }
    };
    const uint32_t nt = (wg_seen + BT - 1) / BT;
    if (nt > 0)
        stage(0);
    for (uint32_t t = 0; t < nt; t++) {
        rl_wait_vmcnt<0>();
        __syncthreads();  // tile t is there, and nobody reads tile t - 1 any more
        if (t + 1 < nt)
            stage(t + 1);
        RL_LDS uint8_t *kt = (RL_LDS uint8_t *)smem[t & 1];
        RL_LDS uint8_t *vt = kt + C::PLANE;
        const uint32_t t0 = t * BT;
        if (t0 + BT > lk) {  // rows past the last key: zero weights must meet zeros, not NaN
            for (uint32_t i = threadIdx.x + (lk - t0) * C::NC; i < (uint32_t)(BT * C::NC); i += NW * 64)
                *(RL_LDS rl_u32x4 *)(vt + i * 16) = rl_u32x4{0, 0, 0, 0};
            __syncthreads();
        }
        if (t0 >= w_most)
            continue;
        // ---- S^T = K q^T ---------------------------------------------------------
        f32x16 sc[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            sc[i] = f32x16{};
            const uint32_t r = 32u * i + (lane & 31);
            RL_LDS const uint8_t *row = kt + r * C::RB;
#pragma unroll
            for (int s = 0; s < C::KS; s++) {
                const s16x8 a = *(RL_LDS const s16x8 *)(row + (((2u * s + hf) ^ C::kswz(r)) << 4));
                sc[i] = mfma32<DT>(a, qf[s], sc[i]);
            }
        }
        if (t0 + BT > w_least) {
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (t0 + 32 * i + 8 * (r / 4) + 4 * hf + r % 4 >= my_seen)
                        sc[i][r] = -INFINITY;
        }
        // ---- softmax -------------------------------------------------------------
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int r = 0; r < 16; r++)
                mx = fmaxf(mx, sc[i][r]);
        mx = half_max(mx) * p.scale_log2;
        if (__builtin_amdgcn_ballot_w64(mx > m + kSlack) != 0) {
            const float m_new = fmaxf(m, mx);
            const float alpha = m_new == -INFINITY ? 1.f : exp2f(m - m_new);
            l *= alpha;
#pragma unroll
            for (int d = 0; d < C::DB; d++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    o[d][r] *= alpha;
            m = m_new;
        }
        const float neg = m == -INFINITY ? 0.f : -m;
        s16x8 pf[4];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                rl_u32x4 w;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float a = __builtin_amdgcn_exp2f(fmaf(sc[i][8 * u + 2 * e], p.scale_log2, neg));
                    const float b = __builtin_amdgcn_exp2f(fmaf(sc[i][8 * u + 2 * e + 1], p.scale_log2, neg));
                    l += a + b;
                    w[e] = pack2<DT>(a, b);
                }
                pf[2 * i + u] = __builtin_bit_cast(s16x8, w);
            }
        // ---- O^T += V^T P^T --------------------------------------------------------
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const uint32_t r = 16u * s + 4u * hf + (((uint32_t)lane & 15u) >> 2);  // and r + 8
            RL_LDS const uint8_t *row = vt + r * C::RB + 8 * (lane & 1);
#pragma unroll
            for (int d = 0; d < C::DB; d++) {
                const uint32_t c = 4u * d + 2u * (((uint32_t)lane >> 4) & 1u) + (((uint32_t)lane & 3u) >> 1);
                const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((RL_LDS s16x4 *)(row + ((c ^ C::vswz(r)) << 4)));
                const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (RL_LDS s16x4 *)(row + 8 * C::RB + ((c ^ C::vswz(r + 8)) << 4)));
                o[d] = mfma32<DT>(__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7), pf[s], o[d]);
            }
        }
    }
    // ---- the rows' outputs -------------------------------------------------------
    const float L = half_sum(l);
    const float inv = my_seen == 0 ? 0.f : 1.f / L;
    uint16_t *orow = p.out + (uint64_t)(qs + my_tok) * p.out_stride + (uint64_t)my_head * D;
    float odd = 0.f;
#pragma unroll
    for (int d = 0; d < C::DB; d++)
#pragma unroll
        for (int a = 0; a < 4; a++) {
            rl_u32x2 w;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float x = o[d][4 * a + 2 * e], y = o[d][4 * a + 2 * e + 1];
                odd = fmaf(x, 0.f, fmaf(y, 0.f, odd));
                w[e] = pack2<DT>(x * inv, y * inv);
            }
            if (my_row < rows)
                *(rl_u32x2 *)(orow + 32 * d + 8 * a + 4 * hf) = w;
        }
    // A value of V that is no number spoils its whole 64-key tile in the matrix
    // product, also for the rows that do not see it (0 times NaN). Rows with
    // such an output are computed again, key by key, over what they see. (A
    // row whose sum is no number is right as it is: NaN.)
    uint64_t again = __builtin_amdgcn_ballot_w64(odd != 0.f && L == L && my_row < rows);
    again = (again | again >> 32) & 0xFFFFFFFFu;
    while (again) {
        const int r = __builtin_ctzll(again);
        again &= again - 1;
        const uint32_t tok = rl_readlane(my_tok, r), head = rl_readlane(my_head, r), n = rl_readlane(my_seen, r);
        const float mr = __uint_as_float(rl_readlane(__float_as_uint(m), r));
        const float lr = __uint_as_float(rl_readlane(__float_as_uint(L), r));
        constexpr int E = D / 64;  // dims per lane
        const uint16_t *q = p.q + (uint64_t)(qs + tok) * p.q_stride + (uint64_t)head * D + lane * E;
        float qv[E], acc[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            qv[e] = from16<DT>(q[e]);
            acc[e] = 0.f;
        }
        for (uint32_t j = 0; j < n; j++) {
            const uint16_t *kr = kbase + (uint64_t)j * p.k_stride + lane * E;
            const uint16_t *vr = vbase + (uint64_t)j * p.v_stride + lane * E;
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < E; e++)
                s = fmaf(qv[e], from16<DT>(kr[e]), s);
#pragma unroll
            for (int x = 1; x < 64; x *= 2)
                s += __shfl_xor(s, x);
            const float w = __builtin_amdgcn_exp2f(fmaf(s, p.scale_log2, -mr));
#pragma unroll
            for (int e = 0; e < E; e++)
                acc[e] = fmaf(w, from16<DT>(vr[e]), acc[e]);
        }
        uint16_t *dst = p.out + (uint64_t)(qs + tok) * p.out_stride + (uint64_t)head * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; e++)
            dst[e] = n ? to16<DT>(acc[e] / lr) : (uint16_t)0;
    }
}

template <int D, int DT, int NW>
int launch(PromptParams p, uint32_t seqs, uint32_t max_q)
{
    p.tiles = (uint32_t)(((uint64_t)max_q * p.group + NW * 32 - 1) / (NW * 32));
    p.pairs = seqs * p.kv_heads;
    p.by_xcd = p.pairs % 8 == 0;
    const uint64_t grid = (uint64_t)p.pairs * p.tiles;
    if (grid > 0x7FFFFFFFull) {
        rl_set_error("rl_hip_attn_prompt: %llu workgroups", (unsigned long long)grid);
        return -1;
    }
    hipLaunchKernelGGL((attn_prompt_kernel<D, DT, NW>), dim3((uint32_t)grid), dim3(NW * 64), 0, rl_stream(), p);
    return rl_check_launch("attn_prompt_kernel launch");
}

template <int D, int DT>
int dispatch(const PromptParams &p, uint32_t seqs, uint32_t max_q)
{
    return launch<D, DT, 4>(p, seqs, max_q);
}

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
    return 256;
}

extern "C" int rl_hip_attn_prompt(const rl_attn_prompt_args_t *a)
{
    const char *who = "rl_hip_attn_prompt";
    if (validate(a, who) || rl_require_open(who))
        return -1;
    if (a->max_q == 0 || a->q_tokens == 0)
        return 0;  // no query
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
    p.kv_heads = a->kv_heads;
    p.group = a->q_heads / a->kv_heads;
    const float scale = a->scale != 0.f ? a->scale : 1.0f / sqrtf((float)a->head_dim);
    p.scale_log2 = scale * 1.4426950408889634f;
    if (a->head_dim == 128)
        return a->dtype == RL_DTYPE_BF16 ? dispatch<128, 0>(p, a->seqs, a->max_q) : dispatch<128, 1>(p, a->seqs, a->max_q);
    return a->dtype == RL_DTYPE_BF16 ? dispatch<64, 0>(p, a->seqs, a->max_q) : dispatch<64, 1>(p, a->seqs, a->max_q);
}
