// token_logprob.hip - log probabilities of given tokens under a vocabulary
// projection, and their gradients, without keeping the logits, on gfx950.
//
//   z[r][v] = scale x_r . w_v      lse_r = log sum_v exp z[r][v]      logprob_r = z[r][t_r] - lse_r
//   D[r][v] = scale g_r (1[v = t_r] - exp(z[r][v] - lse_r))           dx = D w      dw = D^T x
//
//  forward   the product's tiles (gemm_core.h) end in each row's maximum and sum
//            of exponentials over a wave's columns; a second launch joins them.
//            Bound by W's stream up to some 100 rows (24 x 32,000 x 4,096 50.6 us, 46 of
//            them the stream, 5.7 TB/s), by the chip's power with thousands (2,048 x
//            128,256 x 4,096 1,655-1,755 us, 1,230-1,300 TFLOP/s). A logit's fp32 sum is
//            formed 512 products at a time in all but the largest tiles: of 4,096 normal
//            products, logprobs near -5 are then off by 0.6e-6 (root mean square), not
//            1.8e-6, at no cost to 24 rows and 3 of 350 us to the gradients' 200.
//  gradient  in pieces of the vocabulary, of which D (bf16) takes up to 256 MiB:
//            the logits of the piece again, from them D, then its shares of dx and
//            its rows of dw, both products of D. dx is summed in fp32 over pieces,
//            and over shares of a piece's vocabulary where its tiles are few.
//            D's rounding, up to 2^-8 of each element, is of the order of the
//            outputs' own. What it takes from D at a row's target, where D is
//            largest, is put back into dx and dw, whose error is then about that of
//            their own rounding: into dw of more than 128 rows by a product of the rows
//            that have a target in a tile, however many rows an entry has (tokens are
//            not spread evenly); up to 128 rows by a second part of D.
//            With the forward pass, 4,096 rows x 32,000 x 4,096 take 3,420-3,650 us,
//            200 rows 347-357; with all rows of one target 5% and 2% more.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "gemm_core.h"
#include "rl_hip.h"
#include "rl_hip_internal.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// The larger (the sum) of lanes l and l ^ 32, in both.
__device__ __forceinline__ float pair_max(float x)
{
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
}
__device__ __forceinline__ float pair_sum(float x)
{
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}

// Maximum and sum of exponentials of two sets together.
__device__ __forceinline__ rl_f32x2 join(rl_f32x2 x, rl_f32x2 y)
{
    // (an equal maximum is no difference: two infinities have none that is a number)
    const float top = fmaxf(x[0], y[0]);
    return rl_f32x2{top, x[1] * (x[0] == top ? 1.f : __builtin_amdgcn_exp2f((x[0] - top) * kLog2e)) +
                             y[1] * (y[0] == top ? 1.f : __builtin_amdgcn_exp2f((y[0] - top) * kLog2e))};
}

struct LogitParams {
    GemmOperand w, x;        // w: the piece's rows
    const uint32_t *targets;
    float scale;
    uint32_t rows, vocab, v0;  // v0: the piece's first entry; vocab: of all
    uint32_t m_tiles, n_tiles;
    // statistics
    rl_f32x2 *part;          // [n_tiles][rows]: maximum and sum
    float *hit;              // [rows]: the target's logit
    // gradient
    const float *lse, *grad;
    uint16_t *d;             // [rows_pad][pitch], and behind it what rounding left of it, if `parts` is 2
    uint32_t rows_pad, parts;
    uint64_t pitch;
    float *rest;             // [rows]: what rounding left of D at the row's target
};

template <typename G, bool ROT>
__device__ __forceinline__ bool logits_of(const LogitParams &p, uint8_t *smem, typename G::Acc &acc, uint32_t &m0,
                                          uint32_t &nt)
{
    uint32_t t, mt;
    if (!gemm_run_of(blockIdx.x, p.m_tiles * p.n_tiles, t))
        return false;
    gemm_tile_of(t, p.m_tiles, p.n_tiles, mt, nt);
    m0 = mt * G::BM;
    const uint32_t steps = p.x.k / kGemmK;
    // Each workgroup starts at another k: all starting at 0, they would read the same columns of rows that lie a
    // power of two apart together.
    // (the largest tiles' waves have no registers for a second set of sums)
    G::template run<G::TN * G::TM <= 4>(p.w, p.x, nt * G::BN, m0, 0, steps, ROT ? blockIdx.x / 8 * 5u % steps : 0u, smem,
                                        acc);
    return true;
}

template <typename G, bool ROT>
__global__ __launch_bounds__(G::WAVES * 64) void token_stats_kernel(LogitParams p)
{
    __shared__ __attribute__((aligned(1024))) uint8_t smem[G::LDS];
    typename G::Acc acc;
    uint32_t m0, nt;
    if (!logits_of<G, ROT>(p, smem, acc, m0, nt))
        return;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hf = lane >> 5;
    const uint32_t wn = wave % G::WN, wm = wave / G::WN, n0 = nt * G::BN + wn * G::TN * 32;
    const bool whole = n0 + G::TN * 32 <= p.vocab;
    rl_f32x2 *all = (rl_f32x2 *)smem;  // [WN][BM]
    __syncthreads();                   // (nobody reads operands any more)
#pragma unroll
    for (int b = 0; b < G::TM; b++) {
        const uint32_t at_row = (wm * G::TM + b) * 32 + (lane & 31), row = m0 + at_row;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int a = 0; a < G::TN; a++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                float z = acc[a][b][r] * p.scale;
                if (!whole && n0 + 32 * a + 8 * (r / 4) + 4 * hf + r % 4 >= p.vocab)
                    z = -INFINITY;
                acc[a][b][r] = z;
                top = fmaxf(top, z);
            }
        top = pair_max(top);
        const float ref = fabsf(top) == INFINITY ? 0.f : top;  // (the exponentials are then 0 and infinity)
#pragma unroll
        for (int a = 0; a < G::TN; a++)
#pragma unroll
            for (int r = 0; r < 16; r++)
                sum += __builtin_amdgcn_exp2f((acc[a][b][r] - ref) * kLog2e);
        sum = pair_sum(sum);
        if (hf == 0)
            all[wn * G::BM + at_row] = rl_f32x2{top, sum};
        if (row < p.rows) {
            const uint32_t t = p.targets[row], at = t - n0;
            if (t < p.vocab && at < G::TN * 32 && (at >> 2 & 1) == hf) {
#pragma unroll
                for (int a = 0; a < G::TN; a++)
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        if (at == 32u * a + 8 * (r / 4) + 4 * hf + r % 4)
                            p.hit[row] = acc[a][b][r];
            }
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < G::BM && m0 + i < p.rows; i += G::WAVES * 64) {
        rl_f32x2 x = all[i];
#pragma unroll
        for (int w = 1; w < G::WN; w++)
            x = join(x, all[w * G::BM + i]);
        p.part[(uint64_t)nt * p.rows + m0 + i] = x;
    }
}

// Joins the tiles' statistics of R rows per workgroup: 256 / R threads a row, each with eight tiles' at a time.
template <int R>
__global__ __launch_bounds__(256) void token_logprob_kernel(const rl_f32x2 *part, const float *hit,
                                                            const uint32_t *targets, uint32_t rows, uint32_t vocab,
                                                            uint32_t slots, float *logprob, float *lse)
{
    constexpr uint32_t PER = 256 / R;
    __shared__ rl_f32x2 all[4][R];
    const uint32_t r = threadIdx.x % R, y = threadIdx.x / R, row = blockIdx.x * R + r, at = min(row, rows - 1);
    rl_f32x2 x = {-INFINITY, 0.f};
    for (uint32_t s = y; s < slots; s += 8 * PER) {
        rl_f32x2 in[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; i++)
            in[i] = part[(uint64_t)min(s + PER * i, slots - 1) * rows + at];
#pragma unroll
        for (uint32_t i = 0; i < 8; i++)
            if (s + PER * i < slots)
                x = join(x, in[i]);
    }
#pragma unroll
    for (int d = R; d < 64; d *= 2)
        x = join(x, rl_f32x2{__shfl_xor(x[0], d), __shfl_xor(x[1], d)});
    if ((threadIdx.x & 63) < R)
        all[threadIdx.x >> 6][r] = x;
    __syncthreads();
    if (threadIdx.x >= R || row >= rows)
        return;
#pragma unroll
    for (int i = 1; i < 4; i++)
        x = join(x, all[i][r]);
    // (all of them -infinity: so is the logarithm)
    const float z = x[0] == -INFINITY ? (x[1] == 0.f ? -INFINITY : x[1]) : x[0] + logf(x[1]);
    lse[row] = z;
    logprob[row] = targets[row] < vocab ? hit[row] - z : 0.f;
}

template <typename G, bool ROT>
__global__ __launch_bounds__(G::WAVES * 64) void token_delta_kernel(LogitParams p)
{
    __shared__ __attribute__((aligned(1024))) uint8_t smem[G::LDS];
    typename G::Acc acc;
    uint32_t m0, nt;
    if (!logits_of<G, ROT>(p, smem, acc, m0, nt))
        return;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hf = lane >> 5;
    const uint32_t wn = wave % G::WN, wm = wave / G::WN, n0 = nt * G::BN + wn * G::TN * 32;
    const bool whole = p.v0 + n0 + G::TN * 32 <= p.vocab;
#pragma unroll
    for (int b = 0; b < G::TM; b++) {
        const uint32_t row = m0 + (wm * G::TM + b) * 32 + (lane & 31);
        const uint32_t t = row < p.rows ? p.targets[row] : 0xFFFFFFFFu;
        const bool has = t < p.vocab;  // rows without a target: zeros, whatever their logits are
        const float g = has ? p.grad[row] * p.scale : 0.f, lse = has ? p.lse[row] : 0.f;
        const uint32_t at = has ? t - p.v0 - n0 : 0xFFFFFFFFu;
#pragma unroll
        for (int a = 0; a < G::TN; a++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const uint32_t n = 32u * a + 8 * (r / 4) + 4 * hf + r % 4;
                const float e = __builtin_amdgcn_exp2f((acc[a][b][r] * p.scale - lse) * kLog2e);
                const float x = g * ((n == at ? 1.f : 0.f) - e);
                acc[a][b][r] = !has || (!whole && p.v0 + n0 + n >= p.vocab) ? 0.f : x;
                if (n == at)
                    p.rest[row] = x - from16<0>(to16<0>(x));
            }
    }
    for (uint32_t part = 0; part < p.parts; part++) {
        if (part)
#pragma unroll
            for (int b = 0; b < G::TM; b++)
#pragma unroll
                for (int a = 0; a < G::TN; a++)
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        acc[a][b][r] -= from16<0>(to16<0>(acc[a][b][r]));
        uint16_t *d = p.d + (uint64_t)part * p.rows_pad * p.pitch + nt * G::BN;
        __syncthreads();  // (nobody reads operands any more)
        G::template each<false>(acc, smem, [&](uint32_t m, uint32_t n, rl_u32x4 w) {
            if (m0 + m < p.rows_pad)
                *(rl_u32x4 *)(d + (uint64_t)(m0 + m) * p.pitch + n) = w;
            if (G::BM == 32 && m0 + 32 >= p.rows && m0 + 32 < p.rows_pad)  // (rows_pad is a multiple of 64)
                *(rl_u32x4 *)(d + (uint64_t)(m0 + m + 32) * p.pitch + n) = rl_u32x4{0, 0, 0, 0};
        });
    }
}

// x with zeros for the rows without a target and those up to rows_pad, which D's zeros alone would not keep out where
// they are no numbers; `parts` times one behind the other. A workgroup copies a row at a time.
__global__ __launch_bounds__(256) void token_rows_kernel(const uint16_t *x, uint64_t ld, const uint32_t *targets,
                                                         uint32_t rows, uint32_t rows_pad, uint32_t parts,
                                                         uint32_t vocab, uint32_t hidden, uint16_t *out)
{
    for (uint32_t i = blockIdx.x; i < parts * rows_pad; i += gridDim.x) {
        const uint32_t row = i < rows_pad ? i : i - rows_pad;
        const bool has = row < rows && targets[row] < vocab;
        for (uint32_t c = threadIdx.x; c < hidden / 8; c += 256)
            *(rl_u32x4 *)(out + (uint64_t)i * hidden + c * 8) =
                has ? *(const rl_u32x4 *)(x + row * ld + c * 8) : rl_u32x4{0, 0, 0, 0};
    }
}

struct DxParams {
    GemmOperand w, d;
    const uint32_t *targets;
    uint32_t rows, vocab, hidden;
    uint32_t m_tiles, n_tiles, steps, split;
    uint32_t add;     // to what an earlier piece left in part
    float *part;      // [split][rows][hidden], or NULL: to dx
    uint16_t *dx;
    uint64_t dx_ld;
    const uint16_t *w_all;  // the projection, for the targets' rows
    uint64_t w_ld;
    const float *rest;
};

// Four elements from c on of what rounding D at the target took from row `row` of dx (which has a target): there D is
// largest, and its rounding alone would be up to 2^-8 of the row.
__device__ __forceinline__ rl_f32x4 target_rest(const DxParams &p, uint32_t row, uint32_t c)
{
    const rl_u32x2 w = *(const rl_u32x2 *)(p.w_all + p.targets[row] * p.w_ld + c);
    const float f = p.rest[row];
    return rl_f32x4{f * rl_bf16_lo(w[0]), f * rl_bf16_hi(w[0]), f * rl_bf16_lo(w[1]), f * rl_bf16_hi(w[1])};
}

template <typename G>
__global__ __launch_bounds__(G::WAVES * 64) void token_dx_kernel(DxParams p)
{
    __shared__ __attribute__((aligned(1024))) uint8_t smem[G::LDS];
    // (an XCD's workgroups have the same share of the vocabulary, or two)
    uint32_t t, mt, nt;
    if (!gemm_run_of(blockIdx.x, p.m_tiles * p.n_tiles * p.split, t))
        return;
    const uint32_t share = t / (p.m_tiles * p.n_tiles);
    gemm_tile_of(t - share * (p.m_tiles * p.n_tiles), p.m_tiles, p.n_tiles, mt, nt);
    const uint32_t m0 = mt * G::BM, n0 = nt * G::BN;
    const uint32_t k0 = (uint32_t)((uint64_t)share * p.steps / p.split);
    const uint32_t k1 = (uint32_t)((uint64_t)(share + 1) * p.steps / p.split);
    typename G::Acc acc;
    G::run(p.w, p.d, n0, m0, k0, k1, 0, smem, acc);
    __syncthreads();  // (nobody reads operands any more)
    if (p.part) {
        float *part = p.part + (uint64_t)share * p.rows * p.hidden;
        G::template each<true>(acc, smem, [&](uint32_t m, uint32_t n, rl_u32x4 w) {
            rl_f32x4 x = __builtin_bit_cast(rl_f32x4, w);
            if (m0 + m < p.rows && n0 + n < p.hidden) {
                float *at = part + (uint64_t)(m0 + m) * p.hidden + n0 + n;
                if (p.add) {
                    const rl_f32x4 y = *(const rl_f32x4 *)at;
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        x[e] += y[e];
                }
                *(rl_f32x4 *)at = x;
            }
        });
        return;
    }
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int b = 0; b < G::TM; b++) {
        const uint32_t row = m0 + (wave / G::WN * G::TM + b) * 32 + (lane & 31);
        if (row >= p.rows || p.targets[row] >= p.vocab)
            continue;
#pragma unroll
        for (int a = 0; a < G::TN; a++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const uint32_t n = n0 + (wave % G::WN * G::TN + a) * 32 + 8 * c + 4 * (lane >> 5);
                if (n < p.hidden) {
                    const rl_f32x4 x = target_rest(p, row, n);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        acc[a][b][4 * c + e] += x[e];
                }
            }
    }
    G::template each<false>(acc, smem, [&](uint32_t m, uint32_t n, rl_u32x4 w) {
        if (m0 + m < p.rows && n0 + n < p.hidden) {
            if (p.targets[m0 + m] >= p.vocab)
                w = rl_u32x4{0, 0, 0, 0};
            *(rl_u32x4 *)(p.dx + (m0 + m) * p.dx_ld + n0 + n) = w;
        }
    });
}

// dx from its shares: 1,024 elements of a row per workgroup, in turn.
__global__ __launch_bounds__(256) void token_dx_sum_kernel(DxParams p)
{
    const uint32_t across = (p.hidden + 1023) / 1024;
    for (uint32_t i = blockIdx.x; i < p.rows * across; i += gridDim.x) {
        const uint32_t row = i / across, c = (i - row * across) * 1024 + threadIdx.x * 4;
        if (c >= p.hidden)
            continue;
        rl_f32x4 x = {0.f, 0.f, 0.f, 0.f};
        const float *at = p.part + (uint64_t)row * p.hidden + c;
        for (uint32_t s = 0; s < p.split; s += 8) {
            rl_f32x4 y[8];
#pragma unroll
            for (uint32_t k = 0; k < 8; k++)
                y[k] = *(const rl_f32x4 *)(at + (uint64_t)min(s + k, p.split - 1) * p.rows * p.hidden);
#pragma unroll
            for (uint32_t k = 0; k < 8; k++)
                if (s + k < p.split)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        x[e] += y[k][e];
        }
        rl_u32x2 w = {0, 0};
        if (p.targets[row] < p.vocab) {
            const rl_f32x4 y = target_rest(p, row, c);
#pragma unroll
            for (int e = 0; e < 4; e++)
                x[e] += y[e];
            w = rl_u32x2{(uint32_t)to16<0>(x[0]) | (uint32_t)to16<0>(x[1]) << 16,
                         (uint32_t)to16<0>(x[2]) | (uint32_t)to16<0>(x[3]) << 16};
        }
        *(rl_u32x2 *)(p.dx + row * p.dx_ld + c) = w;
    }
}

struct DwParams {
    GemmOperand x, d;
    uint32_t entries, hidden;  // of the piece
    uint32_t m_tiles, n_tiles, steps;
    uint16_t *dw;
    uint64_t dw_ld;
    uint32_t past;    // dw is written past the caches
    const float *rest;        // what rounding left of D at the rows' targets, or NULL: D has a second part
    const uint32_t *targets;
    uint32_t rows, v0;        // v0: the piece's first entry
};

// Puts back what rounding took from D at the targets, for the entries m0 .. of a tile: the product of x with a matrix
// that has one element in each row with a target here. Such rows are listed in order, so that the sums are the same
// every time, and taken 64 at a time: their x through LDS as an operand of D's product is, the elements from registers, in
// two bf16 parts, which hold all of an element's at most 16 bits. An entry may have any number of rows.
template <typename G>
__device__ __forceinline__ void add_rest(const DwParams &p, uint32_t m0, uint32_t n0, uint8_t *smem_,
                                         typename G::Acc &acc)
{
    using X = typename G::NT;
    constexpr uint32_t THREADS = G::WAVES * 64, SPAN = 4 * THREADS, MASKS = SPAN / 64, NONE = 0xFFFFFFFFu;
    static_assert(MASKS <= 64, "a mask for each lane at the most");
    static_assert(X::BYTES + SPAN * 4 + (SPAN + 64) * 8 + MASKS * 8 <= G::LDS, "room for the lists");
    RL_LDS uint8_t *stage = (RL_LDS uint8_t *)smem_;
    RL_LDS rl_u32x2 *what = (RL_LDS rl_u32x2 *)(stage + X::BYTES);  // entry, both parts
    RL_LDS uint32_t *rows = (RL_LDS uint32_t *)(what + SPAN + 64);
    RL_LDS uint64_t *masks = (RL_LDS uint64_t *)(rows + SPAN);
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wn = wave % G::WN, wm = wave / G::WN, hf = lane >> 5;
    uint32_t at[G::TN];
    X::template places<G::TN>(wn * G::TN, (int)lane, at);
    for (uint32_t r0 = 0; r0 < p.rows; r0 += SPAN) {
        uint32_t v[4];
        uint64_t has[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; i++)
            v[i] = p.targets[min(r0 + i * THREADS + threadIdx.x, p.rows - 1)] - p.v0 - m0;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const uint32_t r = r0 + i * THREADS + threadIdx.x;
            v[i] = r < p.rows && v[i] < G::BM && m0 + v[i] < p.entries ? v[i] : NONE;
            has[i] = __builtin_amdgcn_ballot_w64(v[i] != NONE);
            if (lane == 0)
                masks[i * G::WAVES + wave] = has[i];
        }
        __syncthreads();
        uint32_t upto = lane < MASKS ? (uint32_t)__builtin_popcountll(masks[lane]) : 0u;
#pragma unroll
        for (uint32_t d = 1; d < 64; d *= 2) {
            const uint32_t before = __shfl_up(upto, d);
            upto += lane >= d ? before : 0u;
        }
        const uint32_t n = rl_readlane(upto, 63);
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const uint32_t mask = i * G::WAVES + wave, first = mask ? rl_readlane(upto, (int)mask - 1) : 0u;
            if (v[i] != NONE) {
                const uint32_t to = first + __builtin_amdgcn_mbcnt_hi((uint32_t)(has[i] >> 32),
                                                                      __builtin_amdgcn_mbcnt_lo((uint32_t)has[i], 0));
                const uint32_t r = r0 + i * THREADS + threadIdx.x;
                const float f = p.rest[r];
                const uint32_t high = to16<0>(f);
                rows[to] = r;
                what[to] = rl_u32x2{v[i], high | (uint32_t)to16<0>(f - from16<0>((uint16_t)high)) << 16};
            }
        }
        if (threadIdx.x < 64)  // (up to a whole step: no row's)
            what[n + threadIdx.x] = rl_u32x2{NONE, 0u};
        __syncthreads();
        for (uint32_t k0 = 0; k0 < n; k0 += 64) {
            const uint32_t slices = min(4u, (n - k0 + 15) / 16);  // of 16 rows
#pragma unroll
            for (uint32_t i = 0; i < X::OPS; i++) {
                const uint32_t first = (wave * X::OPS + i) * X::PER, k = first + lane / X::NC;
                if (first >= 16 * slices)
                    break;
                // (past the last row it again, beside elements of 0)
                const uint32_t c = n0 + 8 * ((lane % X::NC) ^ X::swz(k));
                rl_g2lds_16_at(p.x.base + rows[min(k0 + k, n - 1)] * p.x.ld + min(c, p.hidden - 8),
                            stage + (wave * X::OPS + i) * 1024);
            }
            rl_wait_vmcnt<0>();
            __syncthreads();
            for (uint32_t s = 0; s < slices; s++) {
                RL_LDS const rl_u32x2 *of = what + k0 + 16 * s + 8 * hf;
                RL_LDS const uint8_t *from = stage + 16 * s * (G::BN * 2);
                s16x8 fn[G::TN];
#pragma unroll
                for (int a = 0; a < G::TN; a++)
                    fn[a] = X::read(from, at, a, 0);
#pragma unroll
                for (int b = 0; b < G::TM; b++) {
                    const uint32_t m = (wm * G::TM + b) * 32 + (lane & 31);
                    rl_u32x4 high, low;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint32_t x = of[2 * e][0] == m ? of[2 * e][1] : 0u;
                        const uint32_t y = of[2 * e + 1][0] == m ? of[2 * e + 1][1] : 0u;
                        high[e] = (x & 0xFFFFu) | y << 16;
                        low[e] = x >> 16 | (y & 0xFFFF0000u);
                    }
#pragma unroll
                    for (int a = 0; a < G::TN; a++) {
                        acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                            __builtin_bit_cast(bf16x8, fn[a]), __builtin_bit_cast(bf16x8, high), acc[a][b], 0, 0, 0);
                        acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                            __builtin_bit_cast(bf16x8, fn[a]), __builtin_bit_cast(bf16x8, low), acc[a][b], 0, 0, 0);
                    }
                }
            }
            __syncthreads();  // (nobody reads this step's rows any more)
        }
    }
}

__device__ __forceinline__ void store16(uint16_t *at, rl_u32x4 w, uint32_t past)
{
    if (past)
        __builtin_nontemporal_store(w, (rl_u32x4 *)at);
    else
        *(rl_u32x4 *)at = w;
}

template <typename G>
__global__ __launch_bounds__(G::WAVES * 64) void token_dw_kernel(DwParams p)
{
    __shared__ __attribute__((aligned(1024))) uint8_t smem[G::LDS];
    uint32_t t, mt, nt;
    if (!gemm_run_of(blockIdx.x, p.m_tiles * p.n_tiles, t))
        return;
    gemm_tile_of(t, p.m_tiles, p.n_tiles, mt, nt);
    const uint32_t m0 = mt * G::BM, n0 = nt * G::BN;
    typename G::Acc acc;
    G::run(p.x, p.d, n0, m0, 0, p.steps, 0, smem, acc);
    __syncthreads();  // (nobody reads operands any more)
    if (p.rest)
        add_rest<G>(p, m0, n0, smem, acc);
    G::template each<false>(acc, smem, [&](uint32_t m, uint32_t n, rl_u32x4 w) {
        if (m0 + m < p.entries && n0 + n < p.hidden)
            store16(p.dw + (m0 + m) * p.dw_ld + n0 + n, w, p.past);
    });
}

// ---- the host's side ----------------------------------------------------------------
// Tiles of the logits (n along the vocabulary x m along the rows), and what a workgroup's step of one takes beside how
// many run at a time: measured at hidden 2,048, one round of each, in us: 46-50, 31-35, 21-25, 17-20 and 14.5-17, some 4.5
// of them the launch; the rest are as 26 to 17, 11, 8 and 6.
using Logits256 = Gemm<4, 2, 2, 4, 2, false, false>;  // 256 x 256
using Logits128x256 = Gemm<2, 2, 2, 4, 3, false, false>;
using Logits128 = Gemm<1, 4, 2, 2, 4, false, false>;
using Logits64 = Gemm<1, 2, 2, 1, 4, false, false>;
using Logits64x32 = Gemm<1, 2, 1, 1, 4, false, false>;
// (n along hidden)
using Dx32 = Gemm<1, 4, 1, 1, 4, true, false>;       // 128 x 32
using Dx64 = Gemm<1, 4, 2, 1, 3, true, false>;       // 128 x 64
using Dx128 = Gemm<1, 4, 2, 2, 4, true, false>;      // 128 x 128
using DxMany = Gemm<4, 2, 2, 4, 2, true, false>;     // 256 x 256
// (n along hidden, m along the vocabulary)
using Dw256 = Gemm<4, 2, 2, 4, 2, true, true>;       // 256 x 256
using Dw128 = Gemm<1, 4, 2, 2, 4, true, true>;       // 128 x 128

uint32_t tiles_of(uint64_t n, uint32_t per) { return (uint32_t)((n + per - 1) / per); }
uint32_t grid_of(uint32_t tiles) { return (tiles + 7) / 8 * 8; }

// The rounds of workgroups that tiles of a kind take, times a round's duration in 1/26 of the largest tiles'.
template <typename G>
uint64_t cost_of(uint64_t n, uint64_t m, uint32_t per_cu, uint32_t duration)
{
    const uint64_t tiles = (n + G::BN - 1) / G::BN * ((m + G::BM - 1) / G::BM), at_once = per_cu * rl_cu_count();
    return (tiles + at_once - 1) / at_once * duration;
}

// Which tiles the logits of so many rows and entries take: those with the fewest rounds for their duration, the largest
// of them. (At hidden 2,048, in us, the choice and the next best: 100 rows x 16,000 entries 20.7, 23.1; x 32,000 35,
// 36; 300 x 9,000 26.5, 35; 500 x 16,000 42.8, 52; 1,000 x 4,500 37, 49.)
int logits_kind(uint32_t rows, uint32_t vocab)
{
    const uint64_t cost[5] = {cost_of<Logits256>(vocab, rows, 1, 26), cost_of<Logits128x256>(vocab, rows, 1, 17),
                              cost_of<Logits128>(vocab, rows, 1, 11), cost_of<Logits64>(vocab, rows, 2, 8),
                              cost_of<Logits64x32>(vocab, rows, 3, 6)};
    return (int)(std::min_element(cost, cost + 5) - cost);
}

uint32_t slots_of(uint32_t rows, uint32_t vocab)
{
    const uint32_t wide[5] = {Logits256::BN, Logits128x256::BN, Logits128::BN, Logits64::BN, Logits64x32::BN};
    return tiles_of(vocab, wide[logits_kind(rows, vocab)]);
}

// At least as many statistics as any call up to these rows and entries has: with the largest tiles their own; smaller
// ones are taken only where they are no slower, so they have at most 26 / duration times the largest's rounds, of all
// workgroups at a time: up to 430 rows' statistics for each compute unit (the 64 x 64 and 64 x 32 tiles).
uint64_t most_statistics(uint32_t rows, uint32_t vocab)
{
    const uint64_t rounds = cost_of<Logits256>(vocab, rows, 1, 1);
    return std::max<uint64_t>((uint64_t)tiles_of(vocab, 256) * rows, 430ull * rl_cu_count() * rounds);
}

template <typename G, bool ROT>
int launch_stats(LogitParams &p)
{
    p.m_tiles = tiles_of(p.rows, G::BM);
    p.n_tiles = tiles_of(p.w.rows, G::BN);
    hipLaunchKernelGGL((token_stats_kernel<G, ROT>), dim3(grid_of(p.m_tiles * p.n_tiles)), dim3(G::WAVES * 64), 0,
                       rl_stream(), p);
    return rl_check_launch("token_stats_kernel launch");
}

template <typename G, bool ROT>
int launch_delta(LogitParams &p)
{
    p.m_tiles = tiles_of(p.rows, G::BM);
    p.n_tiles = tiles_of(p.w.rows, G::BN);
    hipLaunchKernelGGL((token_delta_kernel<G, ROT>), dim3(grid_of(p.m_tiles * p.n_tiles)), dim3(G::WAVES * 64), 0,
                       rl_stream(), p);
    return rl_check_launch("token_delta_kernel launch");
}

int launch_stats(LogitParams &p)
{
    switch (logits_kind(p.rows, p.w.rows)) {
    case 0: return launch_stats<Logits256, false>(p);
    case 1: return launch_stats<Logits128x256, true>(p);
    case 2: return launch_stats<Logits128, true>(p);
    case 3: return launch_stats<Logits64, true>(p);
    default: return launch_stats<Logits64x32, true>(p);
    }
}

int launch_delta(LogitParams &p)
{
    switch (logits_kind(p.rows, p.w.rows)) {
    case 0: return launch_delta<Logits256, false>(p);
    case 1: return launch_delta<Logits128x256, true>(p);
    case 2: return launch_delta<Logits128, true>(p);
    case 3: return launch_delta<Logits64, true>(p);
    default: return launch_delta<Logits64x32, true>(p);
    }
}

template <typename G>
int launch_dx(DxParams p)
{
    p.m_tiles = tiles_of(p.rows, G::BM);
    p.n_tiles = tiles_of(p.hidden, G::BN);
    hipLaunchKernelGGL(token_dx_kernel<G>, dim3(grid_of(p.m_tiles * p.n_tiles * p.split)), dim3(G::WAVES * 64), 0,
                       rl_stream(), p);
    return rl_check_launch("token_dx_kernel launch");
}

template <typename G>
int launch_dw(DwParams p)
{
    p.m_tiles = tiles_of(p.entries, G::BM);
    p.n_tiles = tiles_of(p.hidden, G::BN);
    hipLaunchKernelGGL(token_dw_kernel<G>, dim3(grid_of(p.m_tiles * p.n_tiles)), dim3(G::WAVES * 64), 0, rl_stream(),
                       p);
    return rl_check_launch("token_dw_kernel launch");
}

struct GradPlan {
    uint32_t rows_pad, width;  // rows of D, and its columns: entries of a piece, a multiple of 256
    uint32_t parts;            // of D for dw: with few rows also what its rounding left
    uint32_t split;            // shares of a piece's vocabulary for dx
    bool direct;               // dx from the product itself
    size_t d, x, rest, part;   // bytes of the workspace's parts
    size_t most;               // the largest workspace of calls up to this one's rows, vocab and hidden
};

constexpr uint64_t kDeltaElements = 1ull << 27;  // of D, unless a piece of 1,024 entries has more

// tiles of dx along rows and hidden, and workgroups that run at a time
template <typename G>
void dx_shape(uint32_t rows, uint32_t hidden, uint32_t per_cu, uint32_t &tiles, uint32_t &at_once)
{
    tiles = tiles_of(rows, G::BM) * tiles_of(hidden, G::BN);
    at_once = per_cu * rl_cu_count();
}

size_t up256(uint64_t n) { return (size_t)((n + 255) / 256 * 256); }

GradPlan plan_of(uint32_t rows, uint32_t vocab, uint32_t hidden)
{
    GradPlan pl;
    pl.rows_pad = tiles_of(rows, 64) * 64;
    const uint32_t all = tiles_of(vocab, 256) * 256;
    // With few rows dw itself is what moves, and twice the products cost little: D in two parts (forward and gradients of
    // 24 rows x 32,000 x 4,096 244 us against 232, of 120 292 against 265; of 200 404 against 346).
    pl.parts = rows <= 128 ? 2 : 1;
    const uint32_t d_rows = pl.parts * pl.rows_pad;
    pl.width = std::min(all, std::max<uint32_t>(1024, (uint32_t)(kDeltaElements / d_rows) / 256 * 256));
    uint32_t tiles, at_once;
    if (rows <= 32)
        dx_shape<Dx32>(rows, hidden, 2, tiles, at_once);
    else if (rows <= 64)
        dx_shape<Dx64>(rows, hidden, 2, tiles, at_once);
    else if (rows <= 128)
        dx_shape<Dx128>(rows, hidden, 1, tiles, at_once);
    else
        dx_shape<DxMany>(rows, hidden, 1, tiles, at_once);
    // shares of eight steps at least, of the last piece too
    const uint32_t last = vocab % pl.width ? vocab % pl.width : std::min(pl.width, vocab);
    pl.split = std::max(1u, std::min(at_once / tiles, last / kGemmK / 8));
    pl.direct = pl.split == 1 && pl.width >= vocab;
    pl.d = up256((uint64_t)d_rows * pl.width * 2);
    pl.x = up256((uint64_t)d_rows * hidden * 2);
    pl.rest = up256(rows * 4ull);
    pl.part = pl.direct ? 0 : up256((uint64_t)pl.split * rows * hidden * 4);
    // D's bound, and as many sums as there are in all tiles at once, or rows
    const uint64_t most_rows = std::max(d_rows, std::min(256u, 2 * pl.rows_pad));
    const uint64_t d = std::min(most_rows * all, std::max(kDeltaElements, most_rows * 1024));
    const uint64_t at_most = (uint64_t)rl_cu_count() * (rows <= 128 ? 128 * 128 : 256 * 256);
    pl.most = up256(2 * d) + up256(most_rows * hidden * 2) + pl.rest +
              up256(4 * std::max<uint64_t>((uint64_t)rows * hidden, at_most));
    return pl;
}

// What both calls have to have.
int validate(const char *who, const void *x, const void *w, const void *targets, uint32_t rows, uint32_t vocab,
             uint32_t hidden, uint32_t x_stride, uint32_t w_stride, float scale)
{
    if (!x || !w || !targets) {
        rl_set_error("%s: NULL argument", who);
        return -1;
    }
    if (rows == 0 || rows > (1u << 20) || vocab == 0 || vocab > (1u << 24) || hidden == 0 || hidden % kGemmK != 0 ||
        hidden > (1u << 16)) {
        rl_set_error("%s: rows %u (1 to 2^20), vocab %u (1 to 2^24), hidden %u (a multiple of %d up to 2^16)", who, rows,
                     vocab, hidden, kGemmK);
        return -1;
    }
    // (a launch holds less than 2^32 work-items, 512 for each tile of 256 x 256)
    if ((uint64_t)((rows + 255) / 256) * ((vocab + 255) / 256) >= (1u << 23) - 8) {
        rl_set_error("%s: rows %u x vocab %u exceed 2^23 tiles of 256 x 256", who, rows, vocab);
        return -1;
    }
    if (x_stride < hidden || w_stride < hidden || x_stride % 8 != 0 || w_stride % 8 != 0 || x_stride > (1u << 22) ||
        w_stride > (1u << 22)) {
        rl_set_error("%s: strides x %u w %u (multiples of 8 from hidden to 2^22)", who, x_stride, w_stride);
        return -1;
    }
    if (!(scale >= 0.f) || std::isinf(scale)) {
        rl_set_error("%s: scale %g (positive, or 0 for 1)", who, (double)scale);
        return -1;
    }
    if (((uintptr_t)x | (uintptr_t)w) % 16 != 0) {
        rl_set_error("%s: x and w must be 16-byte aligned", who);
        return -1;
    }
    return 0;
}

int validate(const rl_token_logprob_args_t *a, const char *who)
{
    if (!a || !a->logprob || !a->lse) {
        rl_set_error("%s: NULL argument", who);
        return -1;
    }
    return validate(who, a->x, a->w, a->targets, a->rows, a->vocab, a->hidden, a->x_stride, a->w_stride, a->scale);
}

int validate(const rl_token_logprob_grad_args_t *a, const char *who)
{
    if (!a || !a->lse || !a->grad_logprob || (!a->dx && !a->dw)) {
        rl_set_error("%s: NULL argument", who);
        return -1;
    }
    if (validate(who, a->x, a->w, a->targets, a->rows, a->vocab, a->hidden, a->x_stride, a->w_stride, a->scale))
        return -1;
    if ((a->dx && (a->dx_stride < a->hidden || a->dx_stride % 8 != 0)) ||
        (a->dw && (a->dw_stride < a->hidden || a->dw_stride % 8 != 0))) {
        rl_set_error("%s: strides dx %u dw %u (multiples of 8 from hidden on)", who, a->dx_stride, a->dw_stride);
        return -1;
    }
    if (((uintptr_t)a->dx | (uintptr_t)a->dw) % 16 != 0) {
        rl_set_error("%s: dx and dw must be 16-byte aligned", who);
        return -1;
    }
    return 0;
}

int short_workspace(const char *who, const void *ws, size_t bytes, size_t need)
{
    if (ws && bytes >= need && (uintptr_t)ws % 16 == 0)
        return 0;
    rl_set_error("%s: workspace %zu bytes < %zu required (16-byte aligned)", who, bytes, need);
    return -1;
}

}  // namespace

extern "C" size_t rl_hip_token_logprob_workspace(const rl_token_logprob_args_t *a)
{
    if (validate(a, "rl_hip_token_logprob_workspace") || rl_require_open("rl_hip_token_logprob_workspace"))
        return 0;
    return up256(8 * most_statistics(a->rows, a->vocab)) + up256(a->rows * 4ull);
}

extern "C" int rl_hip_token_logprob(const rl_token_logprob_args_t *a)
{
    const char *who = "rl_hip_token_logprob";
    if (validate(a, who) || rl_require_open(who))
        return -1;
    const uint32_t slots = slots_of(a->rows, a->vocab);
    const size_t part = up256((uint64_t)slots * a->rows * 8);
    if (short_workspace(who, a->workspace, a->workspace_bytes, part + up256(a->rows * 4ull)))
        return -1;
    LogitParams p = {};
    p.w = GemmOperand{(const uint16_t *)a->w, a->w_stride, a->vocab, a->hidden};
    p.x = GemmOperand{(const uint16_t *)a->x, a->x_stride, a->rows, a->hidden};
    p.targets = a->targets;
    p.scale = a->scale != 0.f ? a->scale : 1.f;
    p.rows = a->rows;
    p.vocab = a->vocab;
    p.part = (rl_f32x2 *)a->workspace;
    p.hit = (float *)((uint8_t *)a->workspace + part);
    if (launch_stats(p))
        return -1;
    if (slots > 128)
        hipLaunchKernelGGL(token_logprob_kernel<4>, dim3(tiles_of(a->rows, 4)), dim3(256), 0, rl_stream(), p.part, p.hit,
                           a->targets, a->rows, a->vocab, slots, a->logprob, a->lse);
    else
        hipLaunchKernelGGL(token_logprob_kernel<16>, dim3(tiles_of(a->rows, 16)), dim3(256), 0, rl_stream(), p.part,
                           p.hit, a->targets, a->rows, a->vocab, slots, a->logprob, a->lse);
    return rl_check_launch("token_logprob_kernel launch");
}

extern "C" size_t rl_hip_token_logprob_grad_workspace(const rl_token_logprob_grad_args_t *a)
{
    if (validate(a, "rl_hip_token_logprob_grad_workspace") || rl_require_open("rl_hip_token_logprob_grad_workspace"))
        return 0;
    return plan_of(a->rows, a->vocab, a->hidden).most;
}

extern "C" int rl_hip_token_logprob_grad(const rl_token_logprob_grad_args_t *a)
{
    const char *who = "rl_hip_token_logprob_grad";
    if (validate(a, who) || rl_require_open(who))
        return -1;
    const GradPlan pl = plan_of(a->rows, a->vocab, a->hidden);
    if (short_workspace(who, a->workspace, a->workspace_bytes, pl.d + pl.x + pl.rest + pl.part))
        return -1;
    uint16_t *d = (uint16_t *)a->workspace, *x = (uint16_t *)((uint8_t *)d + pl.d);
    float *rest = (float *)((uint8_t *)x + pl.x), *part = (float *)((uint8_t *)rest + pl.rest);
    if (a->dw) {
        hipLaunchKernelGGL(token_rows_kernel, dim3(std::min(pl.parts * pl.rows_pad, 65535u)), dim3(256), 0, rl_stream(),
                           (const uint16_t *)a->x, a->x_stride, a->targets, a->rows, pl.rows_pad, pl.parts, a->vocab,
                           a->hidden, x);
        if (rl_check_launch("token_rows_kernel launch"))
            return -1;
    }
    LogitParams p = {};
    p.x = GemmOperand{(const uint16_t *)a->x, a->x_stride, a->rows, a->hidden};
    p.targets = a->targets;
    p.scale = a->scale != 0.f ? a->scale : 1.f;
    p.rows = a->rows;
    p.vocab = a->vocab;
    p.lse = a->lse;
    p.grad = a->grad_logprob;
    p.d = d;
    p.rows_pad = pl.rows_pad;
    p.parts = a->dw ? pl.parts : 1;
    p.pitch = pl.width;
    p.rest = rest;
    DxParams dx = {};
    dx.targets = a->targets;
    dx.rows = a->rows;
    dx.vocab = a->vocab;
    dx.hidden = a->hidden;
    dx.part = pl.direct ? nullptr : part;
    dx.dx = (uint16_t *)a->dx;
    dx.dx_ld = a->dx_stride;
    dx.w_all = (const uint16_t *)a->w;
    dx.w_ld = a->w_stride;
    dx.rest = rest;
    for (uint32_t v0 = 0; v0 < a->vocab; v0 += pl.width) {
        const uint32_t n = std::min(pl.width, a->vocab - v0);
        const uint16_t *w = (const uint16_t *)a->w + (uint64_t)v0 * a->w_stride;
        p.w = GemmOperand{w, a->w_stride, n, a->hidden};
        p.v0 = v0;
        if (launch_delta(p))
            return -1;
        if (a->dx) {
            dx.w = GemmOperand{w, a->w_stride, a->hidden, n};
            dx.d = GemmOperand{d, pl.width, pl.rows_pad, n};
            dx.steps = tiles_of(n, kGemmK);
            dx.split = pl.split;
            dx.add = v0 != 0;
            if (a->rows <= 32    ? launch_dx<Dx32>(dx)
                : a->rows <= 64  ? launch_dx<Dx64>(dx)
                : a->rows <= 128 ? launch_dx<Dx128>(dx)
                                 : launch_dx<DxMany>(dx))
                return -1;
        }
        if (a->dw) {
            DwParams dw;
            dw.x = GemmOperand{x, a->hidden, a->hidden, pl.parts * pl.rows_pad};
            dw.d = GemmOperand{d, pl.width, pl.width, pl.parts * pl.rows_pad};
            dw.entries = n;
            dw.hidden = a->hidden;
            dw.steps = pl.parts * pl.rows_pad / kGemmK;
            dw.dw = (uint16_t *)a->dw + (uint64_t)v0 * a->dw_stride;
            dw.dw_ld = a->dw_stride;
            // Few rows: little but dw itself moves (200 rows: 326 us for both gradients and the forward pass against
            // 342). With many, the operands that the caches lose cost more (4,096 rows: 3,590 against 3,512).
            dw.past = a->rows <= 512;
            dw.rest = pl.parts == 1 ? rest : nullptr;
            dw.targets = a->targets;
            dw.rows = a->rows;
            dw.v0 = v0;
            // (as for the logits; at 200 rows x 32,000 x 4,096, what rounding took put back, 256 x 256 tiles take 111 us,
            // 128 x 128 188; at 4,096 rows 923 and 1,534)
            if (cost_of<Dw128>(dw.hidden, n, 1, 11) < cost_of<Dw256>(dw.hidden, n, 1, 26) ? launch_dw<Dw128>(dw)
                                                                                         : launch_dw<Dw256>(dw))
                return -1;
        }
    }
    if (a->dx && !pl.direct) {
        hipLaunchKernelGGL(token_dx_sum_kernel, dim3(std::min(a->rows * tiles_of(a->hidden, 1024), 1u << 16)), dim3(256),
                           0, rl_stream(), dx);
        if (rl_check_launch("token_dx_sum_kernel launch"))
            return -1;
    }
    return 0;
}
