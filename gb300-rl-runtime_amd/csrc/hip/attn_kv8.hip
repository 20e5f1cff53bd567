// attn_kv8.hip - single-query GQA decode attention over the 8-bit paged arena
// (kv_layout.h: e4m3 blocks with a scale per plane), written for gfx950.
//
//   o_h = sum_t softmax_t(scale sK(t) q_h . k8_t) sV(t) v8_t,  t < ctx
//
// with sK(t), sV(t) the scales of token t's block. Bound: the bytes of the
// cache, 2 head_dim per token and KV head; for few rows the chain context,
// table, block, MFMA, merge. Measured, bf16, GQA 4, 8 KV heads, d128: 8 x 32,768
// tokens (539 MB) 95.2 us, 64 x 512-4,096 (304 MB) 62.6 us; 5.8 us of it are there
// for the shortest contexts too. 1 x 517 tokens 8.0 us, 24 x 64-2,048 of d64 11.0 us.
//
//  work   a row (rollout, KV head) is ceil(ctx / 32) units of 32 tokens. Few
//         rows have workgroups of their own, many rows are cut in even shares
//         (the two kernels below); a workgroup's waves take its units in turn.
//  loads  straight to registers, one unit ahead of the one that is consumed:
//         no LDS, no barriers in the loop. A lane's K bytes are one token's,
//         its V bytes eight tokens'. Every load of the loop is a vector load,
//         counted in order: scalar loads of the scales, which return in any
//         order, cost the whole latency per unit (124 us against 102 at 8 x
//         32,768 tokens).
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
#include "kv8_runs.h"
#include "rl_hip.h"
#include "rl_hip_internal.h"

namespace {

constexpr int kUnit = KV8_UNIT;
constexpr uint32_t kRowCost = KV8_ROW_COST;
constexpr uint64_t kKeptBytes = 256u << 20;  // what the last cache before HBM holds

struct Kv8Params {
    const uint8_t *arena;
    uint64_t block_bytes;
    uint64_t arena_blocks;
    const uint32_t *table;
    uint32_t table_stride;
    const uint32_t *ctx;
    uint32_t max_ctx;
    uint32_t batch;
    uint32_t q_heads, kv_heads, group;
    const uint16_t *q;
    uint16_t *out;
    float *out_f32;
    float scale_log2;
    uint32_t split;      // rows kernel: workgroups per row; even kernel: workgroups
    uint32_t min_units;  // units per workgroup, at least, where there are several
    float *part;         // partials, [group * D + 2 * group] each
    uint32_t *cum;       // even kernel: [batch + 1] units of all rows before rollout b
};

__device__ __forceinline__ uint32_t units_of(const Kv8Params &p, uint32_t ctx)
{
    return (uint32_t)(((uint64_t)min(ctx, p.max_ctx) + kUnit - 1) / kUnit);
}

// What a row costs a workgroup, in units: its units, and the latencies of
// turning to it.
__device__ __forceinline__ uint32_t cost_of(uint32_t units) { return units ? units + kRowCost : 0u; }

// Of the workgroups there are, those that share n units.
__device__ __forceinline__ uint32_t sharing(const Kv8Params &p, uint32_t n)
{
    return max(1u, min(p.split, n / p.min_units));
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

// The table entries of 64 of a wave's units (one per lane), from its first-th on:
// units u0 + wave, u0 + wave + W, ... of a row. They are asked for without a look
// at the context; what lies past it is never used.
template <int TPB>
struct Window8 {
    uint32_t e[kUnit / TPB];
};

template <int TPB, int W>
__device__ __forceinline__ Window8<TPB> window8(const Kv8Params &p, uint32_t row, uint32_t u0, uint32_t first)
{
    constexpr int BPU = kUnit / TPB;  // blocks per unit
    const uint32_t *trow = p.table + (size_t)row * p.table_stride;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Window8<TPB> win;
#pragma unroll
    for (int i = 0; i < BPU; i++) {
        const uint64_t at = ((uint64_t)u0 + wave + (uint64_t)(first + (threadIdx.x & 63)) * W) * BPU + i;
        win.e[i] = at < p.table_stride ? trow[at] : 0u;
    }
    return win;
}

// A load of the cache; ONCE: of bytes that nobody reads again soon, which the
// caches need not keep.
template <bool ONCE, class T>
__device__ __forceinline__ T cache_load(const uint8_t *p)
{
    if constexpr (ONCE)
        return __builtin_nontemporal_load((const T *)p);
    else
        return *(const T *)p;
}

// Units u0 .. u1 - 1 of row (rollout b, KV head g) by the W waves of a
// workgroup: the row's output when part is NULL, else a partial. lds: [W][G * D
// + 2 G] floats, free again when the last wave returns from a later barrier.
// win: the wave's first table entries (window8), loaded by the caller as early
// as it can.
template <int D, int DT, int TPB, int W, bool ONCE>
__device__ __forceinline__ void attend8(const Kv8Params &p, uint32_t b, uint32_t g, uint32_t cin, uint32_t u0,
                                        uint32_t u1, Window8<TPB> win, float *part, float *lds)
{
    constexpr int BPU = kUnit / TPB;  // blocks per unit
    constexpr int NJ = D / 16;
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = lane & 15, c = lane >> 4;
    const uint32_t G = p.group, PART = G * D + 2 * G, row = b * p.kv_heads + g;
    const uint32_t ctx = min(cin, p.max_ctx);
    const size_t obase = ((size_t)b * p.q_heads + (size_t)g * G) * D;
    const uint32_t n = u1 - u0 > wave ? (u1 - u0 - wave + W - 1) / W : 0u;  // this wave's units
    bool bad = cin > p.max_ctx;

    Row8<D, DT> rs;
    rs.m = -INFINITY;
    rs.l = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; j++)
        rs.acc[j] = rl_f32x4{0.f, 0.f, 0.f, 0.f};

    if (n > 0) {
        const uint32_t nblk = (uint32_t)(((uint64_t)ctx + TPB - 1) / TPB);
        {
            const int hq = min(h, (int)G - 1);
            const uint16_t *q = p.q + obase + (size_t)hq * D;
#pragma unroll
            for (int t = 0; t < D / 32; t++) {
                const s16x8 v = *(const s16x8 *)(q + 64 * (t / 2) + 16 * c + 8 * (t % 2));
                rs.qf[t] = h < (int)G ? v : s16x8{0, 0, 0, 0, 0, 0, 0, 0};
            }
        }
        uint32_t wfirst = 0;
        // Settled once per 64 units: else every reading of an entry would wait
        // for all loads in flight. The last unit's second block may not exist:
        // its first one again, all masked.
        auto settle = [&] {
#pragma unroll
            for (int i = 0; i < BPU; i++)
                asm volatile("" : "+v"(win.e[i]));
            if constexpr (BPU == 2) {
                const uint64_t at = ((uint64_t)u0 + wave + (uint64_t)(wfirst + lane) * W) * 2 + 1;
                win.e[BPU - 1] = at < nblk ? win.e[BPU - 1] : win.e[0];
            }
        };
        settle();
        const uint32_t koff = (uint32_t)h * D + 16u * c;
        uint32_t zero = 0;
        asm volatile("" : "+v"(zero));
        const uint32_t voff = (uint32_t)TPB * D + 4u * c * D + (uint32_t)h * NJ;
        auto load = [&](uint32_t k, Unit<D> &u) {
            k = min(k, n - 1);
            if (k - wfirst >= 64u) {
                wfirst = k;
                win = window8<TPB, W>(p, row, u0, k);
                settle();
            }
            u.bad = false;
            const uint8_t *base[BPU];
#pragma unroll
            for (int i = 0; i < BPU; i++) {
                uint32_t blk = rl_readlane(win.e[i], (int)(k - wfirst));
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
                    u.k[i][q] = cache_load<ONCE, rl_u32x4>(at + koff + 64 * q);
                // (a vector load: these return in order, so the unit in flight is not waited for)
                u.scale[i] = *(const rl_f32x2 *)(base[i % BPU] + 2 * TPB * D + zero);
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint8_t *at = BPU == 2 ? base[i % BPU] : base[0] + i * 16 * D;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if constexpr (D == 128) {
                        const rl_u32x2 x = cache_load<ONCE, rl_u32x2>(at + voff + r * D);
                        u.v[4 * i + r][0] = x[0];
                        u.v[4 * i + r][D / 64 - 1] = x[1];
                    } else {
                        u.v[4 * i + r][0] = cache_load<ONCE, uint32_t>(at + voff + r * D);
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
        if (part) {
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

// A row without tokens: zeros (NaN where max_ctx is 0 and the context is not).
template <int D, int DT>
__device__ __forceinline__ void empty8(const Kv8Params &p, uint32_t b, uint32_t g, uint32_t cin, uint32_t e)
{
    const size_t at = ((size_t)b * p.q_heads + (size_t)g * p.group) * D + e;
    const float v = cin > p.max_ctx ? __builtin_nanf("") : 0.f;
    p.out[at] = rl_from_f32<DT>(v);
    if (p.out_f32)
        p.out_f32[at] = v;
}

// ---- few rows: workgroups that own their rows ----------------------------------
// `split` workgroups per row. Nothing but the row's own context decides its
// work, so the chain of loads is short: context, table, units.
// A row's shares lie on one XCD, or a few: spread over all of them, where few have
// work, the merge reads them from other L2s than they were written to (1 x 2,000
// tokens, 4 KV heads, max_ctx 32,768: 12.8 us against 9.5).
template <int D, int DT, int TPB, int W>
__global__ __launch_bounds__(W * 64) void attn_kv8_rows_kernel(Kv8Params p)
{
    extern __shared__ float lds[];
    const uint32_t wg = kv8_contiguous(blockIdx.x, gridDim.x);
    const uint32_t row = wg / p.split, s = wg % p.split;
    const uint32_t b = row / p.kv_heads, g = row % p.kv_heads;
    Window8<TPB> win;
    if (p.split == 1)  // the row's first units are this workgroup's, whatever the context
        win = window8<TPB, W>(p, row, 0, 0);
    const uint32_t cin = rl_sload(p.ctx + b), nu = units_of(p, cin), n = sharing(p, nu);
    if (s >= n)
        return;
    if (nu == 0) {
        for (uint32_t e = threadIdx.x; e < p.group * D; e += W * 64)
            empty8<D, DT>(p, b, g, cin, e);
        return;
    }
    const uint32_t u0 = (uint32_t)((uint64_t)s * nu / n), u1 = (uint32_t)((uint64_t)(s + 1) * nu / n);
    if (p.split > 1)
        win = window8<TPB, W>(p, row, u0, 0);
    attend8<D, DT, TPB, W, false>(p, b, g, cin, u0, u1, win,
                                  n > 1 ? p.part + (size_t)wg * (p.group * D + 2 * p.group) : nullptr, lds);
}

// Whether a rollout beside b begins with the same block, as those that share a
// prompt do.
__device__ __forceinline__ bool shares_blocks(const Kv8Params &p, uint32_t b, uint32_t g)
{
    const uint32_t *first = p.table + (size_t)g * p.table_stride;
    const size_t step = (size_t)p.kv_heads * p.table_stride;
    const uint32_t here = rl_sload(first + b * step);
    return (b > 0 && rl_sload(first + (b - 1) * step) == here) ||
           (b + 1 < p.batch && rl_sload(first + (b + 1) * step) == here);
}

// ---- many rows: the units of all rows in even shares -----------------------------
// The units of all rows, rows in (b, g) order, form one sequence; the
// workgroups, two per compute unit, take equal runs of it, whatever the
// contexts are; where these are short of max_ctx and the runs are fewer than the
// workgroups, they still lie on all XCDs (8 x 500 tokens, max_ctx 32,768: 11.2 us
// against 13.5 on the first three). A run that covers a row writes its output; a
// row that several share is merged from their partials. A workgroup has at most
// two of those, of the rows its run starts and ends in: number 2 w when the row's
// part starts the run, else 2 w + 1.
// Where the rows' bytes, those of shared blocks once for each rollout, are more
// than the last cache keeps for a next call, the rows of rollouts whose first
// block is not that of the rollout before or after them are read past the caches:
// 8 x 32,768 tokens (539 MB) 95 us against 104, and 109 against 116 behind a
// product with 1 GiB of weights, as in a model's step; 64 x 512-4,096 (304 MB) 62.5
// against 67. What is kept pays below (64 x 1,800 again and again 42.8 against
// 48.0, 512 x 200 64.8 against 79.1; where three such sets are read in turn 49.6
// against 46.5 and 75.7 against 81.2), with shared prompts (64 x 4,096, three
// quarters shared by eight neighbours, 64 to 68 against 82; where the eight lie
// apart, which is not looked for, 88), and right behind 1 GiB of writes, which the
// last cache still has to put away (107 against 140): that the kernel cannot see.
template <int D, int DT, int TPB, int W>
__global__ __launch_bounds__(W * 64) void attn_kv8_even_kernel(Kv8Params p)
{
    extern __shared__ float lds[];
    const int lane = threadIdx.x & 63;
    const uint32_t PART = p.group * D + 2 * p.group;
    auto cost64 = [&](uint32_t b0) {  // of the rows of rollout b0 + lane
        return b0 + lane < p.batch ? cost_of(units_of(p, p.ctx[b0 + lane])) * p.kv_heads : 0u;
    };
    const uint32_t t0 = cost64(0);
    uint32_t total = rl_wave_sum_u32(t0), filled = (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(t0 != 0));
    for (uint32_t b0 = 64; b0 < p.batch; b0 += 64) {
        const uint32_t t = cost64(b0);
        total += rl_wave_sum_u32(t);
        filled += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(t != 0));
    }
    const uint32_t n = sharing(p, total);
    // (the wave, not its threads, decides: what follows stays in scalar registers)
    const uint32_t wg = __builtin_amdgcn_readfirstlane(kv8_run_of(blockIdx.x, gridDim.x, n));
    const bool writes = blockIdx.x == 0 && __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) == 0;
    if (wg == KV8_NO_RUN && !writes)
        return;
    const uint32_t first = (uint32_t)((uint64_t)wg * total / n), last = (uint32_t)((uint64_t)(wg + 1) * total / n);
    // the rollout that the run begins in, and the cost before it
    uint32_t b = 0, before = 0, sum = 0;
    bool found = false;
    for (uint32_t b0 = 0; b0 < p.batch && (writes || !found); b0 += 64) {
        const uint32_t t = b0 == 0 ? t0 : cost64(b0);
        const uint32_t inc = sum + rl_wave_incl_scan_u32(t);
        if (writes && b0 + lane < p.batch)
            p.cum[b0 + lane] = inc - t;
        const uint64_t in = __builtin_amdgcn_ballot_w64(inc > first);
        if (!found && in) {
            const int l = __builtin_ctzll(in);
            found = true;
            b = b0 + l;
            before = rl_readlane(inc - t, l);
        }
        sum = rl_readlane(inc, 63);
    }
    if (writes && lane == 0)
        p.cum[p.batch] = total;
    if (wg == KV8_NO_RUN || total == 0)
        return;
    uint32_t cin = rl_sload(p.ctx + b), nu = units_of(p, cin);
    uint32_t g = (first - before) / cost_of(nu), x = (first - before) % cost_of(nu);  // x: of this row's cost
    const bool once = kv8_bytes_of(total, filled * p.kv_heads, D) > kKeptBytes;
    uint32_t parts = 0;
    for (uint32_t at = first; at < last;) {
        const uint32_t m = min(cost_of(nu) - x, last - at);
        const uint32_t u0 = max(x, kRowCost) - kRowCost, u1 = max(x + m, kRowCost) - kRowCost;
        if (u1 > u0) {
            const Window8<TPB> win = window8<TPB, W>(p, b * p.kv_heads + g, u0, 0);
            float *part = u1 - u0 < nu ? p.part + (size_t)(2 * wg + min(parts, 1u)) * PART : nullptr;
            if (once && !shares_blocks(p, b, g))
                attend8<D, DT, TPB, W, true>(p, b, g, cin, u0, u1, win, part, lds);
            else
                attend8<D, DT, TPB, W, false>(p, b, g, cin, u0, u1, win, part, lds);
            parts++;
            __syncthreads();
        }
        at += m;
        x = 0;
        if (++g == p.kv_heads && at < last) {
            g = 0;
            do {
                cin = rl_sload(p.ctx + ++b);
                nu = units_of(p, cin);
            } while (nu == 0);  // (cost remains, so a later rollout has some)
        }
    }
}

// Merges the partials of the rows that several workgroups shared: thread e of
// workgroup (x, row) output element 256 x + e of the row.
template <int D, int DT, bool EVEN>
__global__ __launch_bounds__(256) void attn_kv8_merge_kernel(Kv8Params p)
{
    const uint32_t G = p.group, PART = G * D + 2 * G, NE = G * D;
    const uint32_t blocks = (NE + 255) / 256;
    const uint32_t row = blockIdx.x / blocks, e = blockIdx.x % blocks * 256 + threadIdx.x;
    const uint32_t b = row / p.kv_heads, g = row % p.kv_heads;
    const uint32_t cin = rl_sload(p.ctx + b), nu = units_of(p, cin);
    if (e >= NE)
        return;
    const float *part, *start;  // the later ones follow each other, the first may lie elsewhere
    uint32_t n, step;
    if constexpr (EVEN) {
        if (nu == 0) {
            empty8<D, DT>(p, b, g, cin, e);
            return;
        }
        // the places of the row's units in the sequence, and of the runs that hold the first and the last
        const uint32_t total = rl_sload(p.cum + p.batch), row0 = rl_sload(p.cum + b) + g * cost_of(nu);
        const uint64_t wgs = sharing(p, total), r0 = (uint64_t)row0 + kRowCost;
        const uint32_t w0 = (uint32_t)(((r0 + 1) * wgs - 1) / total), w1 = (uint32_t)(((r0 + nu) * wgs - 1) / total);
        n = w1 - w0 + 1;
        step = 2 * PART;
        part = p.part + (size_t)w0 * step;
        start = part + ((uint64_t)w0 * total / wgs < row0 ? PART : 0u);
    } else {
        n = sharing(p, nu);
        step = PART;
        start = part = p.part + (size_t)row * p.split * PART;
    }
    if (n < 2)
        return;
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (uint32_t i0 = 0; i0 < n; i0 += 8) {
        float o[8], mm[8], ll[8], mx = M;
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const float *pp = i0 + i == 0 ? start : part + (size_t)min(i0 + i, n - 1) * step;
            o[i] = pp[e];
            mm[i] = pp[NE + 2 * (e / D)];
            ll[i] = pp[NE + 2 * (e / D) + 1];
        }
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            mm[i] = i0 + i < n ? mm[i] : -INFINITY;
            mx = fmaxf(mx, mm[i]);
        }
        const float keep = M == -INFINITY ? 0.f : exp2f(M - mx);
        L *= keep;
        O *= keep;
        M = mx;
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const float f = mm[i] == -INFINITY ? 0.f : exp2f(mm[i] - M);
            L = i0 + i < n ? L + ll[i] * f : L;
            O = i0 + i < n ? O + o[i] * f : O;
        }
    }
    const float v = O / L;
    const size_t at = ((size_t)b * p.q_heads + (size_t)g * G) * D + e;
    p.out[at] = rl_from_f32<DT>(v);
    if (p.out_f32)
        p.out_f32[at] = v;
}

// ---- launcher ------------------------------------------------------------------

// Which kernel and how many workgroups, by sizes alone (times in us, GQA 4,
// 8 KV heads, d128 unless said):
//  - the even shares from 100 units of the longest context and 16,384 units in
//    all on: 16 x 4,000-16,000 tokens 68.2 against 73.4 of the rows kernel, 64 x
//    1-4,000 59.7 against 64.7, 128 x 512-4,096 122 against 127; below, turning to
//    the next row costs more than uneven rows do: 64 x 512-2,048 43.4 against
//    39.8, 128 x 64-1,024 43.2 against 37.4, 256 x 100-200 39.0 against 27.3.
//  - rows of few units whole, in one launch: 1 x 517 tokens (17 units) 8.1
//    against 9.2 with the row in two.
//  - one row per compute unit, with eight waves: 24 x 64-2,048 tokens of d64,
//    192 rows, 11.4 against 12.6 with four waves and rows in two.
//  - else as many workgroups per row as two per compute unit allow, of 8 units
//    and more: 1 x 1,024 9.4 against 10.6 with 16 and more, 4 x 100-1,024 10.4
//    against 11.7.
constexpr uint64_t kEvenContext = 100, kEvenUnits = 16384, kWholeUnits = 24, kShareUnits = 8;

struct Plan8 {
    bool even;
    uint32_t split, min_units, waves;
    size_t part_off, total;  // of the workspace
    size_t most;             // the largest total of calls up to this one's batch and max_ctx
};

Plan8 plan_of(const rl_attn_decode_args_t *a)
{
    Plan8 pl;
    const uint64_t rows = (uint64_t)a->batch * a->kv_heads;
    const uint64_t units = std::max<uint64_t>(1, ((uint64_t)a->max_ctx + kUnit - 1) / kUnit);
    const uint32_t cus = rl_cu_count();
    pl.waves = 4;
    pl.even = units >= kEvenContext && rows * units >= kEvenUnits;
    pl.min_units = kShareUnits;
    if (pl.even) {
        pl.split = 2 * cus;
    } else if (rows > cus / 2 && rows <= cus && units >= kWholeUnits) {
        pl.split = 1;
        pl.waves = 8;
    } else {
        const uint64_t most = units < kWholeUnits ? 1 : units / pl.min_units;
        pl.split = (uint32_t)std::min<uint64_t>(most, std::max<uint64_t>(1, 2 * cus / rows));
    }
    const uint32_t G = a->q_heads / a->kv_heads;
    const size_t part = (size_t)(G * a->layout.head_dim + 2 * G) * sizeof(float);
    pl.part_off = pl.even ? (((size_t)a->batch + 1) * 4 + 255) / 256 * 256 : 0;
    pl.total = 256 + pl.part_off + (pl.even ? 2 * (size_t)pl.split * part : pl.split > 1 ? rows * pl.split * part : 0);
    // no more for any smaller batch and max_ctx: the rows kernel's shares are at most these
    const uint64_t shares = units < kWholeUnits ? 0 : std::min<uint64_t>(2 * cus, rows * (units / kShareUnits));
    pl.most = pl.even ? pl.total : 256 + shares * part;
    return pl;
}

template <int D, int DT, int TPB>
int launch(const Kv8Params &p, uint64_t rows, const Plan8 &pl)
{
    const size_t lds = (size_t)pl.waves * (p.group * D + 2 * p.group) * sizeof(float);
    const dim3 threads(pl.waves * 64), merge((uint32_t)(rows * ((p.group * D + 255) / 256)));
    if (pl.even) {
        hipLaunchKernelGGL((attn_kv8_even_kernel<D, DT, TPB, 4>), dim3(p.split), threads, lds, rl_stream(), p);
        if (rl_check_launch("attn_kv8_even_kernel launch"))
            return -1;
        hipLaunchKernelGGL((attn_kv8_merge_kernel<D, DT, true>), merge, dim3(256), 0, rl_stream(), p);
        return rl_check_launch("attn_kv8_merge_kernel launch");
    }
    const dim3 grid((uint32_t)(rows * p.split));
    if (pl.waves == 8)
        hipLaunchKernelGGL((attn_kv8_rows_kernel<D, DT, TPB, 8>), grid, threads, lds, rl_stream(), p);
    else
        hipLaunchKernelGGL((attn_kv8_rows_kernel<D, DT, TPB, 4>), grid, threads, lds, rl_stream(), p);
    if (rl_check_launch("attn_kv8_rows_kernel launch"))
        return -1;
    if (p.split < 2)
        return 0;
    hipLaunchKernelGGL((attn_kv8_merge_kernel<D, DT, false>), merge, dim3(256), 0, rl_stream(), p);
    return rl_check_launch("attn_kv8_merge_kernel launch");
}

template <int D, int DT>
int dispatch(const Kv8Params &p, uint64_t rows, const Plan8 &pl, uint32_t tpb)
{
    return tpb == 16 ? launch<D, DT, 16>(p, rows, pl) : launch<D, DT, 32>(p, rows, pl);
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
    // (a launch holds less than 2^32 work-items: the merge 256 for each 256 output elements of a row)
    const uint64_t elements = (uint64_t)(a->q_heads / a->kv_heads) * a->layout.head_dim;
    if (a->batch == 0 || a->batch > 65535 || a->kv_heads > 65535 ||
        (uint64_t)a->batch * a->kv_heads * ((elements + 255) / 256) >= (1u << 24)) {
        rl_set_error("%s: batch %u / kv_heads %u out of range (%llu output elements per row)", who, a->batch,
                     a->kv_heads, (unsigned long long)elements);
        return -1;
    }
    if (a->grid_waves != 0) {
        rl_set_error("%s: grid_waves %u (only 0, the library's own split)", who, a->grid_waves);
        return -1;
    }
    // (the even kernel counts a row's units and its cost in 32 bits)
    if ((uint64_t)a->batch * a->kv_heads * (((uint64_t)a->max_ctx + kUnit - 1) / kUnit + kRowCost) >= (1ull << 32)) {
        rl_set_error("%s: batch %u x kv_heads %u of max_ctx %u exceeds 2^32 units of %d tokens", who, a->batch,
                     a->kv_heads, a->max_ctx, kUnit);
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
    return plan_of(a).most;
}

extern "C" int rl_hip_attn_decode_kv8(const rl_attn_decode_args_t *a)
{
    const char *who = "rl_hip_attn_decode_kv8";
    if (validate(a, who) || rl_require_open(who))
        return -1;
    const Plan8 pl = plan_of(a);
    if (!a->workspace || a->workspace_bytes < pl.total) {
        rl_set_error("%s: workspace %zu bytes < %zu required", who, a->workspace_bytes, pl.total);
        return -1;
    }
    Kv8Params p;
    p.arena = (const uint8_t *)a->arena_base;
    p.block_bytes = a->layout.block_bytes;
    p.arena_blocks = a->arena_bytes / a->layout.block_bytes;
    p.table = a->block_table;
    p.table_stride = a->table_stride;
    p.ctx = a->ctx_lens;
    p.max_ctx = a->max_ctx;
    p.batch = a->batch;
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
    p.cum = (uint32_t *)a->workspace;
    p.part = (float *)((uint8_t *)a->workspace + pl.part_off);
    const uint64_t rows = (uint64_t)a->batch * a->kv_heads;
    const uint32_t tpb = a->layout.token_count;
    if (a->layout.head_dim == 128)
        return a->dtype == RL_DTYPE_BF16 ? dispatch<128, 0>(p, rows, pl, tpb) : dispatch<128, 1>(p, rows, pl, tpb);
    return a->dtype == RL_DTYPE_BF16 ? dispatch<64, 0>(p, rows, pl, tpb) : dispatch<64, 1>(p, rows, pl, tpb);
}
