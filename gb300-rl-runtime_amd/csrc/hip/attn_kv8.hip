// attn_kv8.hip - single-query GQA decode attention over the 8-bit paged arena
// (kv_layout.h: e4m3 blocks with a scale per plane), written for gfx950.
//
//   o_h = sum_t softmax_t(scale sK(t) q_h . k8_t) sV(t) v8_t,  t < ctx
//
// with sK(t), sV(t) the scales of token t's block. Bound: the bytes of the
// cache, 2 head_dim per token and KV head; for few rows the chain context,
// table, block, MFMA, merge.
//
//  work   a row (rollout, KV head) is ceil(ctx / 32) units of 32 tokens. A row
//         has up to `split` workgroups that take equal shares of its units;
//         the workgroup's waves take its units in turn.
//  loads  straight to registers, one unit ahead of the one that is consumed:
//         no LDS, no barriers in the loop. A lane's K bytes are one token's,
//         its V bytes eight tokens'.
//  QK     v_mfma_f32_16x16x32: A = 16 tokens' K, B = q^T with the heads of the
//         group as columns (up to 16). A lane's 16 consecutive K bytes are two
//         k-steps of the product; q's dims are permuted the same way. The
//         bytes become bf16 or fp16 (both hold every e4m3 value exactly, two
//         per instruction); K's scale multiplies the score.
//  PV     O^T = V^T P^T: a lane's scores S^T (head lane % 16, tokens 4 (lane /
//         16) .. + 3 of both 16-token tiles) are already the B operand; A is
//         V with lane % 16 naming D / 16 neighbouring dims, transposed four
//         tokens at a time with byte permutes and widened to bf16 with V's
//         scale (exact: a power of two). P is split in a bf16 high part and
//         the bf16 remainder, so that the products keep 16 bits of it.
//  merge  online softmax per wave, the waves' partials through LDS, the
//         workgroups' through the workspace and a second kernel.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "attn_core.h"
#include "kv8_core.h"
#include "rl_hip.h"
#include "rl_hip_internal.h"

namespace {

constexpr int kUnit = 32;           // tokens per unit
constexpr uint32_t kMaxSplit = 64;  // workgroups per row at most
constexpr int kWavesPerWg = 4;

struct Kv8Params {
    const uint8_t *arena;
    uint64_t block_bytes;
    uint64_t arena_blocks;
    const uint32_t *table;
    uint32_t table_stride;
    const uint32_t *ctx;
    uint32_t max_ctx;
    uint32_t q_heads, kv_heads, group;
    const uint16_t *q;
    uint16_t *out;
    float *out_f32;
    float scale_log2;
    uint32_t split;      // workgroups per row
    uint32_t min_units;  // units per workgroup, at least, where a row has several
    float *part;         // [rows][split][group * D + 2 * group]
};

// The workgroups that share a row of nu units.
__device__ __forceinline__ uint32_t row_wgs(const Kv8Params &p, uint32_t nu)
{
    return max(1u, min(p.split, nu / p.min_units));
}

// One unit as it was loaded: K of two 16-token tiles, V of eight tokens per
// lane, both tiles' scales.
template <int D>
struct Unit {
    rl_u32x4 k[2][D / 64];
    uint32_t v[8][D / 64];
    rl_f32x2 scale[2];
    bool bad;
};

template <int D, int DT>
struct Row8 {
    s16x8 qf[D / 32];      // B operand: q[head][64 i + 16 (lane / 16) + 8 half ..] for k-step 2 i + half
    rl_f32x4 acc[D / 16];  // O^T: head lane % 16, dim (D / 16) (4 (lane / 16) + r) + j
    float m, l;            // running max (log2 domain) of the head; this lane's share of the sum
};

template <int D, int DT, bool FULL>
__device__ __forceinline__ void consume8(Row8<D, DT> &rs, const Unit<D> &u, float scale_log2, uint32_t tokens, int lane)
{
    constexpr int NJ = D / 16;
    const int c = lane >> 4;
    // ---- S^T = K q^T, both tiles -------------------------------------------------
    rl_f32x4 sc[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        sc[i] = rl_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < D / 32; s++) {
            const uint32_t w0 = u.k[i][s / 2][2 * (s % 2)], w1 = u.k[i][s / 2][2 * (s % 2) + 1];
            const rl_u32x4 a = {kv8_unpack2<DT, false>(w0), kv8_unpack2<DT, true>(w0), kv8_unpack2<DT, false>(w1),
                                kv8_unpack2<DT, true>(w1)};
            sc[i] = mfma_qk<DT>(__builtin_bit_cast(s16x8, a), rs.qf[s], sc[i]);
        }
    }
    // ---- online softmax ----------------------------------------------------------
    float sv[8], mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const float f = scale_log2 * u.scale[i][0];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const bool ok = FULL || (uint32_t)(16 * i + 4 * c + r) < tokens;
            sv[4 * i + r] = ok ? sc[i][r] * f : -INFINITY;
            mx = fmaxf(mx, sv[4 * i + r]);
        }
    }
    mx = tile_max(mx);
    const bool grow = mx > rs.m;
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
        const float m_new = fmaxf(rs.m, mx);
        const float alpha = grow ? exp2f(rs.m - m_new) : 1.f;  // (0 the first time: rs.m is -inf)
        rs.l *= alpha;
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                rs.acc[j][r] *= alpha;
        rs.m = m_new;
    }
    const float m_use = rs.m == -INFINITY ? 0.f : rs.m;
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float p0 = exp2f(sv[2 * e] - m_use), p1 = exp2f(sv[2 * e + 1] - m_use);
        rs.l += p0 + p1;
        rl_bf16x2 h, w;
        h[0] = (__bf16)p0;
        h[1] = (__bf16)p1;
        hi[e] = __builtin_bit_cast(uint32_t, h);
        w[0] = (__bf16)(p0 - rl_bf16_lo(hi[e]));
        w[1] = (__bf16)(p1 - rl_bf16_hi(hi[e]));
        lo[e] = __builtin_bit_cast(uint32_t, w);
    }
    const s16x8 phi = __builtin_bit_cast(s16x8, (rl_u32x4{hi[0], hi[1], hi[2], hi[3]}));
    const s16x8 plo = __builtin_bit_cast(s16x8, (rl_u32x4{lo[0], lo[1], lo[2], lo[3]}));
    // ---- O^T += V^T P^T ----------------------------------------------------------
#pragma unroll
    for (int q = 0; q < D / 64; q++) {
        uint32_t t[2][4];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            uint32_t rows[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                // slots past the context may hold anything, NaN included
                const bool ok = FULL || (uint32_t)(16 * i + 4 * c + r) < tokens;
                rows[r] = ok ? u.v[4 * i + r][q] : 0u;
            }
            kv8_transpose4(rows, t[i]);
        }
#pragma unroll
        for (int jj = 0; jj < 4; jj++) {
            const int j = 4 * q + jj;
            const rl_u32x4 a = {kv8_unpack2_scaled<false>(t[0][jj], u.scale[0][1]),
                                kv8_unpack2_scaled<true>(t[0][jj], u.scale[0][1]),
                                kv8_unpack2_scaled<false>(t[1][jj], u.scale[1][1]),
                                kv8_unpack2_scaled<true>(t[1][jj], u.scale[1][1])};
            const s16x8 vf = __builtin_bit_cast(s16x8, a);
            rs.acc[j] = mfma_qk<0>(vf, phi, rs.acc[j]);
            rs.acc[j] = mfma_qk<0>(vf, plo, rs.acc[j]);
        }
    }
}

// Workgroup b of the grid runs on XCD b % 8; each XCD gets a contiguous eighth
// of the rows, so that rollouts that share prefix blocks read them through one L2.
__device__ __forceinline__ uint32_t xcd_contiguous(uint32_t n)
{
    return n % 8 != 0 ? blockIdx.x : (blockIdx.x % 8) * (n / 8) + blockIdx.x / 8;
}

template <int D, int DT, int TPB, int W>
__global__ __launch_bounds__(W * 64) void attn_kv8_kernel(Kv8Params p)
{
    constexpr int BPU = kUnit / TPB;  // blocks per unit
    constexpr int NJ = D / 16;
    extern __shared__ float lds[];    // [W][G * D + 2 G]
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wg = xcd_contiguous(gridDim.x);
    const uint32_t row = wg / p.split, s = wg % p.split;
    const uint32_t b = row / p.kv_heads, g = row % p.kv_heads, G = p.group;
    const int h = lane & 15, c = lane >> 4;
    const uint32_t PART = G * D + 2 * G;

    const uint32_t cin = rl_sload(p.ctx + b);
    const uint32_t ctx = min(cin, p.max_ctx);
    const uint32_t nu = (uint32_t)(((uint64_t)ctx + kUnit - 1) / kUnit);
    const uint32_t nwg = row_wgs(p, nu);
    if (s >= nwg)
        return;
    const size_t obase = ((size_t)b * p.q_heads + (size_t)g * G) * D;
    if (nu == 0) {  // no token: zeros (NaN where max_ctx is 0 and the context is not)
        for (uint32_t e = threadIdx.x; e < G * D; e += W * 64) {
            const float v = cin > p.max_ctx ? __builtin_nanf("") : 0.f;
            p.out[obase + e] = rl_from_f32<DT>(v);
            if (p.out_f32)
                p.out_f32[obase + e] = v;
        }
        return;
    }
    const uint32_t u0 = (uint32_t)((uint64_t)s * nu / nwg), u1 = (uint32_t)((uint64_t)(s + 1) * nu / nwg);
    const uint32_t n = u1 - u0 > wave ? (u1 - u0 - wave + W - 1) / W : 0u;  // this wave's units
    bool bad = cin > p.max_ctx;

    Row8<D, DT> rs;
    rs.m = -INFINITY;
    rs.l = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; j++)
        rs.acc[j] = rl_f32x4{0.f, 0.f, 0.f, 0.f};

    if (n > 0) {
        const uint32_t *trow = p.table + (size_t)row * p.table_stride;
        const uint32_t nblk = (uint32_t)(((uint64_t)ctx + TPB - 1) / TPB);
        uint32_t win[BPU], wfirst = 0;
        auto window = [&](uint32_t first) {
            wfirst = first;
#pragma unroll
            for (int i = 0; i < BPU; i++) {
                const uint64_t at = ((uint64_t)u0 + wave + (uint64_t)(first + lane) * W) * BPU + i;
                // (the last unit's second block may not exist: its first one again, all masked)
                win[i] = at < nblk ? trow[at] : (i > 0 && at == nblk ? trow[at - 1] : 0u);
            }
        };
        window(0);
        {
            const int hq = min(h, (int)G - 1);
            const uint16_t *q = p.q + obase + (size_t)hq * D;
#pragma unroll
            for (int t = 0; t < D / 32; t++) {
                const s16x8 v = *(const s16x8 *)(q + 64 * (t / 2) + 16 * c + 8 * (t % 2));
                rs.qf[t] = h < (int)G ? v : s16x8{0, 0, 0, 0, 0, 0, 0, 0};
            }
        }
        const uint32_t koff = (uint32_t)h * D + 16u * c;
        const uint32_t voff = (uint32_t)TPB * D + 4u * c * D + (uint32_t)h * NJ;
        auto load = [&](uint32_t k, Unit<D> &u) {
            k = min(k, n - 1);
            if (k - wfirst >= 64u)
                window(k);
            u.bad = false;
            const uint8_t *base[BPU];
#pragma unroll
            for (int i = 0; i < BPU; i++) {
                uint32_t blk = rl_readlane(win[i], (int)(k - wfirst));
                if (blk >= p.arena_blocks) {  // never read outside the arena
                    u.bad = true;
                    blk = 0;
                }
                base[i] = p.arena + (uint64_t)blk * p.block_bytes;
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint8_t *at = BPU == 2 ? base[i % BPU] : base[0] + i * 16 * D;
#pragma unroll
                for (int q = 0; q < D / 64; q++)
                    u.k[i][q] = *(const rl_u32x4 *)(at + koff + 64 * q);
                u.scale[i] = rl_sload((const rl_f32x2 *)(base[i % BPU] + 2 * TPB * D));
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint8_t *at = BPU == 2 ? base[i % BPU] : base[0] + i * 16 * D;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if constexpr (D == 128) {
                        const rl_u32x2 x = *(const rl_u32x2 *)(at + voff + r * D);
                        u.v[4 * i + r][0] = x[0];
                        u.v[4 * i + r][D / 64 - 1] = x[1];
                    } else {
                        u.v[4 * i + r][0] = *(const uint32_t *)(at + voff + r * D);
                    }
                }
            }
        };
        auto consume = [&](uint32_t k, const Unit<D> &u) {
            const uint64_t t0 = ((uint64_t)u0 + wave + (uint64_t)k * W) * kUnit;
            bad |= u.bad;
            if (t0 + kUnit <= ctx)
                consume8<D, DT, true>(rs, u, p.scale_log2, kUnit, lane);
            else
                consume8<D, DT, false>(rs, u, p.scale_log2, (uint32_t)(ctx - t0), lane);
        };
        // two register stages; past the last unit the loads repeat it, so that
        // every turn has the same number in flight
        Unit<D> ua, ub;
        load(0, ua);
        for (uint32_t k = 0; k < n; k += 2) {
            load(k + 1, ub);
            consume(k, ua);
            if (k + 1 >= n)
                break;
            load(k + 2, ua);
            consume(k + 1, ub);
        }
    }
    // ---- merge the waves -----------------------------------------------------------
    float lt = rs.l + __shfl_xor(rs.l, 16);
    lt += __shfl_xor(lt, 32);
    if (bad)
        lt = __builtin_nanf("");
    float *mine = lds + wave * PART;
    if (h < (int)G) {
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int j = 0; j < NJ; j++)
                mine[h * D + NJ * (4 * c + r) + j] = rs.acc[j][r];
        if (c == 0) {
            mine[G * D + 2 * h] = rs.m;
            mine[G * D + 2 * h + 1] = lt;
        }
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < G * D; e += W * 64) {
        const uint32_t hh = e / D;
        float mm[W], M = -INFINITY;
#pragma unroll
        for (int i = 0; i < W; i++) {
            mm[i] = lds[i * PART + G * D + 2 * hh];
            M = fmaxf(M, mm[i]);
        }
        float L = 0.f, O = 0.f;
#pragma unroll
        for (int i = 0; i < W; i++) {
            const float f = mm[i] == -INFINITY ? 0.f : exp2f(mm[i] - M);
            L += lds[i * PART + G * D + 2 * hh + 1] * f;
            O += lds[i * PART + e] * f;
        }
        if (nwg > 1) {
            float *part = p.part + ((size_t)row * p.split + s) * PART;
            part[e] = O;
            if (e % D == 0) {
                part[G * D + 2 * hh] = M;
                part[G * D + 2 * hh + 1] = L;
            }
            continue;
        }
        const float v = O / L;
        p.out[obase + e] = rl_from_f32<DT>(v);
        if (p.out_f32)
            p.out_f32[obase + e] = v;
    }
}

// Merges the partials of the rows that several workgroups shared: thread e of
// workgroup (x, row) output element 256 x + e of the row.
template <int DT, int D>
__global__ __launch_bounds__(256) void attn_kv8_merge_kernel(Kv8Params p)
{
    const uint32_t G = p.group, PART = G * D + 2 * G, NE = G * D;
    const uint32_t blocks = (NE + 255) / 256;
    const uint32_t row = blockIdx.x / blocks, e = blockIdx.x % blocks * 256 + threadIdx.x;
    const uint32_t b = row / p.kv_heads, g = row % p.kv_heads;
    const uint32_t cin = rl_sload(p.ctx + b);
    const uint32_t nwg = row_wgs(p, (uint32_t)(((uint64_t)min(cin, p.max_ctx) + kUnit - 1) / kUnit));
    if (nwg < 2 || e >= NE)
        return;
    const float *part = p.part + (size_t)row * p.split * PART;
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (uint32_t i0 = 0; i0 < nwg; i0 += 8) {
        float o[8], mm[8], ll[8], mx = M;
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const float *pp = part + (size_t)min(i0 + i, nwg - 1) * PART;
            o[i] = pp[e];
            mm[i] = pp[NE + 2 * (e / D)];
            ll[i] = pp[NE + 2 * (e / D) + 1];
        }
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            mm[i] = i0 + i < nwg ? mm[i] : -INFINITY;
            mx = fmaxf(mx, mm[i]);
        }
        const float keep = M == -INFINITY ? 0.f : exp2f(M - mx);
        L *= keep;
        O *= keep;
        M = mx;
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const float f = mm[i] == -INFINITY ? 0.f : exp2f(mm[i] - M);
            L = i0 + i < nwg ? L + ll[i] * f : L;
            O = i0 + i < nwg ? O + o[i] * f : O;
        }
    }
    const float v = O / L;
    const size_t at = ((size_t)b * p.q_heads + (size_t)g * G) * D + e;
    p.out[at] = rl_from_f32<DT>(v);
    if (p.out_f32)
        p.out_f32[at] = v;
}

// ---- launcher ------------------------------------------------------------------

struct Plan8 {
    uint32_t split, min_units;
};

Plan8 plan_of(const rl_attn_decode_args_t *a)
{
    Plan8 pl;
    pl.min_units = 2 * kWavesPerWg;
    const uint64_t rows = (uint64_t)a->batch * a->kv_heads;
    const uint64_t most = std::max<uint64_t>(1, ((uint64_t)a->max_ctx + kUnit - 1) / kUnit / pl.min_units);
    const uint64_t want = std::max<uint64_t>(1, 4096 / rows);
    pl.split = (uint32_t)std::min<uint64_t>(std::min<uint64_t>(most, want), kMaxSplit);
    return pl;
}

size_t workspace_of(const rl_attn_decode_args_t *a)
{
    const uint32_t G = a->q_heads / a->kv_heads;
    const Plan8 pl = plan_of(a);
    const size_t rows = (size_t)a->batch * a->kv_heads;
    return 256 + (pl.split > 1 ? rows * pl.split * (G * a->layout.head_dim + 2 * G) * sizeof(float) : 0);
}

template <int D, int DT, int TPB>
int launch(const Kv8Params &p, uint64_t rows)
{
    const size_t lds = (size_t)kWavesPerWg * (p.group * D + 2 * p.group) * sizeof(float);
    hipLaunchKernelGGL((attn_kv8_kernel<D, DT, TPB, kWavesPerWg>), dim3((uint32_t)(rows * p.split)),
                       dim3(kWavesPerWg * 64), lds, rl_stream(), p);
    if (rl_check_launch("attn_kv8_kernel launch"))
        return -1;
    if (p.split < 2)
        return 0;
    const uint32_t blocks = (p.group * D + 255) / 256;
    hipLaunchKernelGGL((attn_kv8_merge_kernel<DT, D>), dim3((uint32_t)(rows * blocks)), dim3(256), 0, rl_stream(), p);
    return rl_check_launch("attn_kv8_merge_kernel launch");
}

template <int D, int DT>
int dispatch(const Kv8Params &p, uint64_t rows, uint32_t tpb)
{
    return tpb == 16 ? launch<D, DT, 16>(p, rows) : launch<D, DT, 32>(p, rows);
}

int validate(const rl_attn_decode_args_t *a, const char *who)
{
    if (!a) {
        rl_set_error("%s: NULL args", who);
        return -1;
    }
    if (kv_layout_check_paged8(&a->layout) != 0) {
        rl_set_error("%s: unsupported KV layout (token_count %u, head_dim %u, scalar %u, block of %u bytes)", who,
                     a->layout.token_count, a->layout.head_dim, a->layout.scalar_bytes, a->layout.block_bytes);
        return -1;
    }
    if (a->kv_heads == 0 || a->q_heads == 0 || a->q_heads % a->kv_heads != 0 || a->q_heads / a->kv_heads > 16) {
        rl_set_error("%s: q_heads %u not 1 to 16 times kv_heads %u", who, a->q_heads, a->kv_heads);
        return -1;
    }
    if (a->dtype != RL_DTYPE_BF16 && a->dtype != RL_DTYPE_FP16) {
        rl_set_error("%s: dtype %u", who, a->dtype);
        return -1;
    }
    if (!a->arena_base || !a->block_table || !a->ctx_lens || !a->q || !a->out) {
        rl_set_error("%s: NULL device pointer", who);
        return -1;
    }
    if (((uintptr_t)a->arena_base | (uintptr_t)a->q) % 16 != 0) {
        rl_set_error("%s: arena_base and q must be 16-byte aligned", who);
        return -1;
    }
    if (a->arena_bytes < a->layout.block_bytes) {
        rl_set_error("%s: arena of %llu bytes holds no block", who, (unsigned long long)a->arena_bytes);
        return -1;
    }
    if (a->batch == 0 || a->batch > 65535 || a->kv_heads > 65535 || (uint64_t)a->batch * a->kv_heads > (1u << 24)) {
        rl_set_error("%s: batch %u / kv_heads %u out of range", who, a->batch, a->kv_heads);
        return -1;
    }
    if (a->grid_waves != 0) {
        rl_set_error("%s: grid_waves %u (only 0, the library's own split)", who, a->grid_waves);
        return -1;
    }
    const uint64_t table_need = ((uint64_t)a->max_ctx + a->layout.token_count - 1) / a->layout.token_count;
    if (a->table_stride < table_need) {
        rl_set_error("%s: table_stride %u < %llu blocks needed for max_ctx %u", who, a->table_stride,
                     (unsigned long long)table_need, a->max_ctx);
        return -1;
    }
    return 0;
}

}  // namespace

extern "C" size_t rl_hip_attn_decode_kv8_workspace(const rl_attn_decode_args_t *a)
{
    if (validate(a, "rl_hip_attn_decode_kv8_workspace") || rl_require_open("rl_hip_attn_decode_kv8_workspace"))
        return 0;
    return workspace_of(a);
}

extern "C" int rl_hip_attn_decode_kv8(const rl_attn_decode_args_t *a)
{
    const char *who = "rl_hip_attn_decode_kv8";
    if (validate(a, who) || rl_require_open(who))
        return -1;
    const size_t need = workspace_of(a);
    if (!a->workspace || a->workspace_bytes < need) {
        rl_set_error("%s: workspace %zu bytes < %zu required", who, a->workspace_bytes, need);
        return -1;
    }
    const Plan8 pl = plan_of(a);
    Kv8Params p;
    p.arena = (const uint8_t *)a->arena_base;
    p.block_bytes = a->layout.block_bytes;
    p.arena_blocks = a->arena_bytes / a->layout.block_bytes;
    p.table = a->block_table;
    p.table_stride = a->table_stride;
    p.ctx = a->ctx_lens;
    p.max_ctx = a->max_ctx;
    p.q_heads = a->q_heads;
    p.kv_heads = a->kv_heads;
    p.group = a->q_heads / a->kv_heads;
    p.q = (const uint16_t *)a->q;
    p.out = (uint16_t *)a->out;
    p.out_f32 = a->out_f32;
    const float scale = a->scale != 0.f ? a->scale : 1.0f / sqrtf((float)a->layout.head_dim);
    p.scale_log2 = scale * 1.4426950408889634f;
    p.split = pl.split;
    p.min_units = pl.min_units;
    p.part = (float *)a->workspace;
    const uint64_t rows = (uint64_t)a->batch * a->kv_heads;
    const uint32_t tpb = a->layout.token_count;
    if (a->layout.head_dim == 128)
        return a->dtype == RL_DTYPE_BF16 ? dispatch<128, 0>(p, rows, tpb) : dispatch<128, 1>(p, rows, tpb);
    return a->dtype == RL_DTYPE_BF16 ? dispatch<64, 0>(p, rows, tpb) : dispatch<64, 1>(p, rows, tpb);
}
