// prompt_core.h - the kernels of causal attention with grouped heads, written for
// gfx950: over whole prompts whose keys and values are packed rows
// (attn_prompt.hip), and of chunks of tokens over the blocks of a paged arena
// (attn_chunk.hip).
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j <= i + Lk - Lq
//
// of a sequence with Lq queries and Lk >= Lq keys (the queries are its last
// tokens). Bound: the matrix cores from some hundred tokens on, 4 head_dim
// operations per head and visible pair; K and V come from L2. Measured, bf16,
// GQA 4, 8 KV heads, d128: 1 x 8,192 tokens 482 us, 1,140 TFLOP/s (372 with
// zeros: the chip's power sets the clock), 64 x 512-1,024 446 us, 720 TFLOP/s (382
// with zeros; 6.8 key tiles per row block, each block with its own start and
// end), 1 x 517 12.3 us (136 row blocks on 256 compute units, up to nine tiles one
// after the other).
//
//  rows   a workgroup of NW waves takes 32 NW rows of one (sequence, KV head);
//         row r is query token r / G, head r % G of the group, so that a
//         group's heads share every K and V tile and a wave's rows span few
//         tokens (little masked work on the diagonal).
//         Eight waves per workgroup, two groups of keys in one, or several row
//         blocks one after the other in one (each's first tile copied during the
//         last step of the one before) were no faster.
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
//         rounding, up to 2^-8 of each weight with bf16, is of the order of the
//         output's own (against 64 bits 2.0e-3 of the output's norm where 32 bits
//         rounded once have 1.6e-3); in two parts, as the decode kernels keep it,
//         it would double PV's products.
//  LDS    a step of a d128 workgroup reads 128 KiB of operands and stores 32 KiB of
//         tiles: 1,280 cycles at 128 bytes each, against 1,024 of matrix
//         instructions per wave. 32 rows per wave thus keep the matrix cores below
//         80%.
//  paged  the same with K and V found through a block table: of each tile a wave copies
//         16 tokens, which lie in one block of 16 or 32, and its lanes hold the block
//         ids of the next 64 tiles, so that a copy waits for no table entry. A block
//         that the arena does not have reads as keys that are no numbers and values
//         of 0. Measured, bf16, d128: 2,048 queries of 64 heads behind 30,000 tokens
//         1,820-1,860 us (1,120-1,145 TFLOP/s of visible pairs), 64 x 1-512 of 32 heads
//         behind 512 shared ones 236, 64 x 4 behind 512-4,096 120-122 (5.0 TB/s).
//  softmax online; the maximum a row's weights refer to is raised only when it
//         is exceeded by more than 2^8, which the fp32 sums and 16-bit weights
//         hold without loss, so the output is rarely rescaled.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attn_core.h"
#include "rl_dev_common.h"
#include "rl_hip.h"
#include "rl_hip_internal.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int BT = 64;         // keys per tile
constexpr int NW = 4;          // waves per workgroup, 32 rows each
constexpr uint32_t ROWS = NW * 32;
// tiles per workgroup, at least, where several share a row block's keys: one and two workgroups per compute unit
constexpr uint32_t kShareTiles = 6, kLongShareTiles = 48;
constexpr int kPlain = 0, kMasked = 1, kFinal = 2;  // what a step's next scores are: all seen, some hidden, none
constexpr float kSlack = 8.f;  // log2 of what a weight may exceed its reference by

// Division of n < 2^31 by d: with 2^(shift - 1) < d <= 2^shift and mul the ceiling
// of 2^(31 + shift) / d, floor(n mul / 2^(31 + shift)) is the quotient.
struct Divisor {
    uint32_t mul, shift;
};

Divisor divisor_of(uint32_t d)
{
    Divisor v = {0, 0};
    while ((1ull << v.shift) < d)
        v.shift++;
    v.mul = (uint32_t)(((1ull << (31 + v.shift)) + d - 1) / d);
    return v;
}

__device__ __forceinline__ uint32_t quotient(uint32_t n, const Divisor &v)
{
    return (uint32_t)((uint64_t)(n << 1) * v.mul >> 32) >> v.shift;
}

struct PromptParams {
    const uint16_t *q, *k, *v;  // (k, v: rows, unless paged)
    uint16_t *out;
    uint64_t q_stride, k_stride, v_stride, out_stride;  // elements between tokens
    const uint32_t *q_starts, *kv_starts;
    uint32_t q_tokens, kv_tokens, max_q;
    // paged: sequence s has ctx[s] keys, in the blocks table[(s kv_heads + g) table_stride ..] of the arena
    const uint8_t *arena;
    uint64_t block_bytes;
    uint32_t arena_blocks, table_stride, tpb, tpb_shift, max_ctx;  // blocks of tpb = 2^tpb_shift tokens: 16 or 32
    const uint32_t *table, *ctx;
    uint32_t kv_heads, group;
    uint32_t pairs;   // sequences x KV heads
    uint32_t tiles;   // row blocks of the longest sequence
    uint32_t by_xcd;  // a pair's row blocks all on one XCD
    uint32_t ranked;  // the longest sequences first, by ...
    uint32_t rank_shift;  // ... their keys divided by 2^rank_shift, up to 63
    uint32_t seqs;
    uint32_t split;   // workgroups per row block, at most
    Divisor by_group, by_pairs, by_heads, by_tiles;
    float scale_log2;
    float *part;      // [pairs x tiles][split][NW][PART] sums of split row blocks
};

template <int D>
struct PCfg {
    static constexpr int RB = 2 * D;             // bytes of a K or V row
    static constexpr int NC = D / 8;             // 16-byte chunks of a row
    static constexpr int PLANE = BT * RB;
    static constexpr int OPS = PLANE / 1024;     // 1 KiB copies per plane
    static constexpr int KS = D / 16;            // k-steps of QK
    static constexpr int DB = D / 32;            // 32-dim blocks of the output
    static constexpr int PART = (DB * 16 + 2) * 64;  // words of a wave's sums in the workspace
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

// The workgroups that share the keys of a row block of nt tiles.
__device__ __forceinline__ uint32_t shares_of(const PromptParams &p, uint32_t nt)
{
    return max(1u, min(p.split, nt / kShareTiles));
}

// The lane whose key, 0 to 63, is the rank-th largest of the first n lanes (ties
// in lane order): the largest value that more than `rank` keys reach, bit by bit.
__device__ __forceinline__ uint32_t lane_of_rank(uint32_t key, uint32_t n, uint32_t rank)
{
    const uint64_t lanes = ~0ull >> (64 - n);
    uint32_t least = 0;
#pragma unroll
    for (uint32_t bit = 32; bit > 0; bit /= 2)
        if ((uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(key >= (least | bit)) & lanes) > rank)
            least |= bit;
    const uint64_t same = __builtin_amdgcn_ballot_w64(key == least) & lanes;
    const uint32_t more = (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(key > least) & lanes);
    const uint32_t before = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0));
    return (uint32_t)__builtin_ctzll(__builtin_amdgcn_ballot_w64(before == rank - more) & same);
}

// A workgroup's row block (of 128 rows): the tile-th of sequence seq and KV head g,
// whose queries start at qs, lq of them, and the keys at ks (0 where paged).
// lost: no key can be read (the sequence has more than max_ctx).
struct Place {
    uint32_t seq, g, tile, qs, lq, ks, lk;
    bool lost;
};

// What stands for the rows of a block that the arena does not have: keys that are
// no numbers, so that neither are the outputs of rows that see them, and values of
// 0, which say nothing to the others. (Both read as rows of 16 tokens, d128.)
constexpr uint32_t kPage = 16 * 256;
struct LostPages {
    uint32_t key[kPage / 4], value[kPage / 4];
};
constexpr LostPages lost_pages()
{
    LostPages p = {};
    for (uint32_t i = 0; i < kPage / 4; i++)
        p.key[i] = 0xFFFFFFFFu;
    return p;
}
__device__ const LostPages g_lost = lost_pages();

// Which one workgroup `at` of the grid has: the last ones, which see the most,
// first, the longest sequences first, and all of a pair's on one XCD (workgroup
// b runs on XCD b % 8), behind whose L2 they share K and V.
template <bool PAGED>
__device__ __forceinline__ Place place_of(const PromptParams &p, uint32_t at, int lane)
{
    Place x;
    uint32_t pair;
    if (p.by_xcd) {
        const uint32_t local = at / 8, n = quotient(local, p.by_tiles);
        pair = at % 8 + 8 * n;
        x.tile = p.tiles - 1 - (local - n * p.tiles);
    } else {
        const uint32_t n = quotient(at, p.by_pairs);
        pair = at - n * p.pairs;
        x.tile = p.tiles - 1 - n;
    }
    const uint32_t seq = quotient(pair, p.by_heads);
    x.g = pair - seq * p.kv_heads;
    uint32_t qe, ke;
    if (p.ranked) {
        const uint32_t i = min((uint32_t)lane, p.seqs - 1);
        const uint32_t q0 = p.q_starts[i], q1 = p.q_starts[i + 1];
        const uint32_t k0 = PAGED ? 0u : p.kv_starts[i], k1 = PAGED ? p.ctx[i] : p.kv_starts[i + 1];
        const uint32_t n = PAGED ? k1 : min(k1, p.kv_tokens);
        const int l = (int)lane_of_rank(min((n > k0 ? n - k0 : 0u) >> p.rank_shift, 63u), p.seqs, seq);
        x.seq = (uint32_t)l;
        x.qs = rl_readlane(q0, l);
        qe = rl_readlane(q1, l);
        x.ks = rl_readlane(k0, l);
        ke = rl_readlane(k1, l);
    } else {
        x.seq = seq;
        x.qs = rl_sload(p.q_starts + seq);
        qe = rl_sload(p.q_starts + seq + 1);
        x.ks = PAGED ? 0u : rl_sload(p.kv_starts + seq);
        ke = PAGED ? rl_sload(p.ctx + seq) : rl_sload(p.kv_starts + seq + 1);
    }
    qe = min(qe, p.q_tokens);
    x.lq = qe > x.qs ? qe - x.qs : 0u;
    x.lost = PAGED && ke > p.max_ctx;
    if constexpr (PAGED) {
        x.lk = x.lost ? x.lq : ke;  // (lost: enough for every row to see one)
    } else {
        ke = min(ke, p.kv_tokens);
        x.lk = ke > x.ks ? ke - x.ks : 0u;
    }
    return x;
}

// One row block; SPLIT: or a share of its keys, its sums to the workspace; PAGED:
// the keys and values in the blocks of an arena.
template <int D, int DT, bool SPLIT, bool PAGED>
__global__ __launch_bounds__(NW * 64, 2) void attn_prompt_kernel(PromptParams p)
{
    using C = PCfg<D>;
    constexpr int WOPS = C::OPS / NW;  // copies of a plane per wave
    static_assert(WOPS * NW == C::OPS, "whole copies per wave");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[4 * C::PLANE];
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t hf = (uint32_t)lane >> 5;
    const uint32_t blocks = p.pairs * p.tiles, at = SPLIT ? blockIdx.x % blocks : blockIdx.x;
    const Place x = place_of<PAGED>(p, at, lane);
    const uint32_t g = x.g, tile = x.tile, qs = x.qs, lq = x.lq, ks = x.ks, lk = x.lk;
    const uint32_t rows = min(lq, p.max_q) * p.group, wg_row = tile * ROWS;
    if (wg_row >= rows)
        return;
    // keys that query token t < lq sees: t + lk - lq + 1, not below 0
    auto seen = [&](uint32_t t) { return (uint32_t)max((int32_t)(t - lq + 1) + (int32_t)lk, 0); };
    const uint32_t wg_seen = seen(quotient(min(wg_row + ROWS, rows) - 1, p.by_group));
    // the wave's rows: from head h0 of token tok0 on (those past the last row repeat it)
    const uint32_t w_row = wg_row + wave * 32, w0 = min(w_row, rows - 1);
    const uint32_t tok0 = quotient(w0, p.by_group), h0 = w0 - tok0 * p.group;
    // this workgroup's tiles of the keys: first .. first + steps - 1
    const uint32_t nt = (wg_seen + BT - 1) / BT;
    uint32_t first = 0, last = nt;
    if constexpr (SPLIT) {
        const uint32_t n = shares_of(p, nt), share = blockIdx.x / blocks;
        if (share >= n)
            return;
        first = (uint32_t)((uint64_t)share * nt / n);
        last = (uint32_t)((uint64_t)(share + 1) * nt / n);
    }
    const uint32_t steps = last - first, most = (uint32_t)min<uint64_t>((uint64_t)last * BT, lk);
    const bool w_has = w_row < rows;
    const uint32_t w_least = w_has ? min(most, seen(tok0)) : 0u;
    const uint32_t w_most = w_has ? min(most, seen(quotient(min(w_row + 32, rows) - 1, p.by_group))) : 0u;
    const uint32_t my_x = h0 + min(w_row + ((uint32_t)lane & 31u), rows - 1) - w0, my_dt = quotient(my_x, p.by_group);
    const uint32_t my_seen = min(most, seen(tok0 + my_dt));

    // ---- the copies --------------------------------------------------------------
    const uint16_t *kbase = nullptr, *vbase = nullptr;
    const uint32_t *table = nullptr;
    if constexpr (PAGED) {
        table = p.table + ((uint64_t)x.seq * p.kv_heads + g) * p.table_stride;
    } else {
        kbase = p.k + (uint64_t)ks * p.k_stride + (uint64_t)g * D;
        vbase = p.v + (uint64_t)ks * p.v_stride + (uint64_t)g * D;
    }
    // Paged: the plane (0: keys, 1: values) of block id from in-block token `slot`
    // (0 or 16) on.
    auto plane_of = [&](uint32_t id, int plane, uint32_t slot) {
        const uint8_t *at = p.arena + (uint64_t)id * p.block_bytes + (plane * p.tpb + slot) * (uint32_t)C::RB;
        return (const uint16_t *)(id < p.arena_blocks ? at : (const uint8_t *)(plane ? g_lost.value : g_lost.key));
    };
    // The row of key or value j (below lk), for what is read from memory once more.
    auto row_of = [&](int plane, uint32_t j) {
        if constexpr (PAGED)
            return plane_of(x.lost ? 0xFFFFFFFFu : table[j >> p.tpb_shift], plane, j & (p.tpb - 16u)) +
                   (j & 15u) * (uint32_t)D;
        else
            return plane ? vbase + (uint64_t)j * p.v_stride : kbase + (uint64_t)j * p.k_stride;
    };
    // Paged: a wave copies 16 tokens of each tile, which lie in one block; the 16
    // after the last key's are that key's again. Lane i knows the block of tile
    // ids_from + i.
    uint32_t ids = 0xFFFFFFFFu, ids_from = first;
    const uint32_t last16 = lk > 0 ? (lk - 1) & ~15u : 0u;
    auto look_up = [&](uint32_t t) {
        ids_from = t;
        const uint32_t token = min((t + (uint32_t)lane) * BT + wave * 16u, last16);
        ids = x.lost ? 0xFFFFFFFFu : table[token >> p.tpb_shift];
        asm volatile("" : "+v"(ids));  // (settled here, as the queries below)
    };
    auto kbuf = [&](uint32_t s) { return (RL_LDS uint8_t *)smem + s % 2 * C::PLANE; };
    auto vbuf = [&](uint32_t s) { return (RL_LDS uint8_t *)smem + (2 + s % 2) * C::PLANE; };
    // row and source chunk of this lane in copy i of a plane
    const uint32_t r0 = wave * WOPS * (64 / C::NC) + (uint32_t)lane / C::NC, pos = (uint32_t)lane % C::NC;
    uint32_t koff[WOPS], voff[WOPS];
#pragma unroll
    for (int i = 0; i < WOPS; i++) {
        const uint32_t r = r0 + i * (64 / C::NC);
        koff[i] = (PAGED ? (r & 15u) * (uint32_t)C::RB : r * (uint32_t)p.k_stride * 2u) + ((pos ^ C::kswz(r)) << 4);
        voff[i] = (PAGED ? (r & 15u) * (uint32_t)C::RB : r * (uint32_t)p.v_stride * 2u) + ((pos ^ C::vswz(r)) << 4);
    }
    static_assert(WOPS * (64 / C::NC) == 16, "a wave copies 16 tokens of a tile");
    // One of the wave's copies of tile t of a plane; rows past the last key
    // repeat it (a tile that is whole needs no such look).
    auto copy1 = [&](auto whole, const uint16_t *base, uint64_t stride, const uint32_t (&off)[WOPS], RL_LDS uint8_t *dst,
                     uint32_t t, int i) {
        uint32_t o = off[i];
        if constexpr (!decltype(whole)::value) {
            const uint32_t r = r0 + i * (64 / C::NC);
            o -= (r - min(r, lk - t * BT - 1)) * (uint32_t)stride * 2u;
        }
        rl_g2lds_16_off(base + (uint64_t)t * BT * stride, o, dst + (wave * WOPS + i) * 1024);
    };
    auto copy1_paged = [&](auto whole, int plane, const uint32_t (&off)[WOPS], RL_LDS uint8_t *dst, uint32_t t, int i) {
        const uint32_t token = decltype(whole)::value ? t * BT + wave * 16u : min(t * BT + wave * 16u, last16);
        uint32_t o = off[i];
        if constexpr (!decltype(whole)::value) {
            const uint32_t r = (r0 + i * (64 / C::NC)) & 15u;
            o -= (r - min(r, lk - token - 1)) * (uint32_t)C::RB;
        }
        rl_g2lds_16_off(plane_of(rl_readlane(ids, (int)(t - ids_from)), plane, token & (p.tpb - 16u)), o,
                        dst + (wave * WOPS + i) * 1024);
    };
    // (past the last tile the copies repeat it)
    auto copy_k = [&](auto whole, uint32_t s, int i) {
        if constexpr (PAGED)
            copy1_paged(whole, 0, koff, kbuf(s), min(first + s, last - 1), i);
        else
            copy1(whole, kbase, p.k_stride, koff, kbuf(s), min(first + s, last - 1), i);
    };
    auto copy_v = [&](auto whole, uint32_t s, int i) {
        if constexpr (PAGED)
            copy1_paged(whole, 1, voff, vbuf(s), min(first + s, last - 1), i);
        else
            copy1(whole, vbase, p.v_stride, voff, vbuf(s), min(first + s, last - 1), i);
    };
    constexpr std::false_type maybe{};
    if constexpr (PAGED)
        if (steps > 0)
            look_up(first);
    if (steps > 0)
#pragma unroll
        for (int i = 0; i < WOPS; i++)
            copy_k(maybe, 0, i);

    s16x8 qf[C::KS];
    {
        const uint16_t *q = p.q + (uint64_t)(qs + tok0) * p.q_stride + (uint64_t)g * p.group * D;
        q += my_dt * (uint32_t)p.q_stride + (my_x - my_dt * p.group) * D + 8 * hf;
#pragma unroll
        for (int s = 0; s < C::KS; s++)
            qf[s] = *(const s16x8 *)(q + 16 * s);
        // Settled here: the compiler does not see the copies' waits, and would
        // otherwise wait for these loads, and with them for the copies in
        // flight, at their first use in every step.
#pragma unroll
        for (int s = 0; s < C::KS; s++)
            asm volatile("" : "+v"(qf[s]));
    }
    f32x16 o[C::DB];
#pragma unroll
    for (int d = 0; d < C::DB; d++)
        o[d] = f32x16{};
    float m = -INFINITY, l = 0.f, l2 = 0.f;  // (the sum in two halves)

    // ---- operands ----------------------------------------------------------------
    // K: row 32 i + lane % 32, chunk 2 s + lane / 32. V: the tokens 32 i + 16 s + 4
    // (lane / 32) .. + 3 and those 8 further, dims 32 d + lane % 32. The step's
    // parity, the half and s are immediate offsets.
    const uint32_t kr = (uint32_t)lane & 31u, vr = 4u * hf + (((uint32_t)lane & 15u) >> 2);
    const uint32_t vc = 2u * (((uint32_t)lane >> 4) & 1u) + (((uint32_t)lane & 3u) >> 1);
    RL_LDS const uint8_t *kat[C::KS], *vat[2][C::DB];
#pragma unroll
    for (int s = 0; s < C::KS; s++)
        kat[s] = kbuf(0) + kr * C::RB + (((2u * s + hf) ^ C::kswz(kr)) << 4);
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
        for (int d = 0; d < C::DB; d++)
            vat[e][d] = vbuf(0) + (vr + 8 * e) * C::RB + 8 * (lane & 1) + (((4u * d + vc) ^ C::vswz(vr + 8 * e)) << 4);
    auto read_k = [&](int parity, int i, int s) {
        return *(RL_LDS const s16x8 *)(kat[s] + parity * C::PLANE + 32 * i * C::RB);
    };
    auto read_v = [&](int parity, int i, int s, int d) {
        const int at = parity * C::PLANE + (32 * i + 16 * s) * C::RB;
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((RL_LDS s16x4 *)(vat[0][d] + at));
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((RL_LDS s16x4 *)(vat[1][d] + at));
        return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    // the scores of the keys k0 .. k0 + 31 that the row does not see
    auto hide = [&](float x, uint32_t k0, int r) { return k0 + 8 * (r / 4) + 4 * hf + r % 4 < my_seen ? x : -INFINITY; };
    auto raise = [&](float top) {
        if (__builtin_amdgcn_ballot_w64(top * p.scale_log2 > m + kSlack) != 0) {
            const float m_new = fmaxf(m, half_max(top) * p.scale_log2);
            const float alpha = m_new == -INFINITY ? 1.f : exp2f(m - m_new);
            l *= alpha;
            l2 *= alpha;
#pragma unroll
            for (int d = 0; d < C::DB; d++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    o[d][r] *= alpha;
            m = m_new;
        }
    };

    // One step: of tile t (scores in cur) the weights and V's product, of the
    // next one the scores and their maximum. The matrix instructions, the reads
    // of their operands AHEAD instructions earlier and the vector work are laid
    // out here one by one: left to itself the compiler gathers each kind, and
    // then matrix cores and vector units take turns instead of working side by
    // side. AHEAD: 2 is best, 3 costs 2%, 1 much more. The sum in plain adds: a
    // dot product instruction does not run beside a matrix one (73-76 cycles
    // per matrix instruction and its share of the weights, 46-49 with adds).
    auto step = [&](auto parity_, auto kind_, f32x16 (&cur)[2], f32x16 (&next)[2], uint32_t k_next) {
        constexpr int parity = decltype(parity_)::value;
        constexpr int kind = decltype(kind_)::value;
        constexpr int QK = kind == kFinal ? 0 : C::KS;  // matrix instructions per 32 keys: of the next scores, ...
        constexpr int PER = QK + 2 * C::DB;              // ... and in all
        constexpr int AHEAD = 2;
        const float neg = m == -INFINITY ? 0.f : -m;
        float top = -INFINITY;
        s16x8 ring[AHEAD + 1];
        uint32_t w[8];
        auto fetch = [&](int n) {
            const int i = n / PER, j = n % PER;
            ring[n % (AHEAD + 1)] = j < QK ? read_k(1 - parity, i, j) : read_v(parity, i, (j - QK) / C::DB, (j - QK) % C::DB);
        };
        // the pairs e0 .. e1 - 1 of the weights of half i
        auto weights = [&](int i, int e0, int e1) {
#pragma unroll
            for (int e = e0; e < e1; e++) {
                const float a = __builtin_amdgcn_exp2f(fmaf(cur[i][2 * e], p.scale_log2, neg));
                const float b = __builtin_amdgcn_exp2f(fmaf(cur[i][2 * e + 1], p.scale_log2, neg));
                l += a;
                l2 += b;
                w[e] = pack2<DT>(a, b);
            }
        };
#pragma unroll
        for (int n = 0; n < AHEAD; n++)
            fetch(n);
#pragma unroll
        for (int n = 0; n < 2 * PER; n++) {
            const int i = n / PER, j = n % PER;
            if (kind == kFinal && n == PER && k_next - 32 >= w_most)
                break;  // (no row of the wave sees the tile's second half)
            if (kind == kFinal && j == 0)
                weights(i, 0, 8);
            if (j < QK) {
                next[i] = mfma32<DT>(ring[n % (AHEAD + 1)], qf[j], j == 0 ? f32x16{} : next[i]);
            } else {
                const int u = (j - QK) / C::DB, d = (j - QK) % C::DB;
                const s16x8 pf = __builtin_bit_cast(s16x8, (rl_u32x4{w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]}));
                o[d] = mfma32<DT>(ring[n % (AHEAD + 1)], pf, o[d]);
            }
            if (n + AHEAD < 2 * PER)
                fetch(n + AHEAD);
            if (j < QK) {
                weights(i, 8 / C::KS * j, 8 / C::KS * (j + 1));
            } else if (kind != kFinal) {
                constexpr int E = 16 / (2 * C::DB);
#pragma unroll
                for (int r = E * (j - QK); r < E * (j - QK + 1); r++) {
                    if (kind == kMasked)
                        next[i][r] = hide(next[i][r], k_next + 32 * i, r);
                    top = fmaxf(top, next[i][r]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (kind != kFinal)
            raise(top);
    };

    // ---- the tiles -------------------------------------------------------------
    f32x16 sa[2], sb[2];
    if (steps > 0) {
        rl_wait_vmcnt<0>();
        __syncthreads();  // K of step 0
#pragma unroll
        for (int i = 0; i < WOPS; i++)
            copy_v(maybe, 0, i);
#pragma unroll
        for (int i = 0; i < WOPS; i++)
            copy_k(maybe, 1, i);
        if (first * BT < w_most) {
            float top = -INFINITY;
#pragma unroll
            for (int s = 0; s < C::KS; s++)
#pragma unroll
                for (int i = 0; i < 2; i++)
                    sa[i] = mfma32<DT>(read_k(0, i, s), qf[s], s == 0 ? f32x16{} : sa[i]);
#pragma unroll
            for (int i = 0; i < 2; i++) {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    sa[i][r] = hide(sa[i][r], first * BT + 32 * i, r);
                    top = fmaxf(top, sa[i][r]);
                }
            }
            raise(top);
        }
    }
    auto meet = [&](auto whole, uint32_t s, bool more) {
        rl_wait_vmcnt<0>();
        rl_wait_lgkmcnt0();
        __builtin_amdgcn_s_barrier();  // K of step s + 1 and V of step s are there; nobody reads K of step s or V of s - 1
        asm volatile("" ::: "memory");
        if (!more)
            return;
        if constexpr (PAGED)
            if (min(first + s + 2, last - 1) - ids_from > 63)  // (the tile before it is needed too)
                look_up(first + s + 1);
#pragma unroll
        for (int i = 0; i < WOPS; i++)
            copy_k(whole, s + 2, i);
#pragma unroll
        for (int i = 0; i < WOPS; i++)
            copy_v(whole, s + 1, i);
    };
    constexpr std::integral_constant<int, 0> even{};
    constexpr std::integral_constant<int, 1> uneven{};
    constexpr std::integral_constant<int, kPlain> plain{};
    constexpr std::integral_constant<int, kMasked> masked{};
    constexpr std::integral_constant<int, kFinal> final{};
    auto turn = [&](auto parity, auto kind, uint32_t s, f32x16 (&cur)[2], f32x16 (&next)[2]) {
        meet(std::bool_constant<decltype(kind)::value == kPlain>{}, s, decltype(kind)::value != kFinal || s + 1 < steps);
        step(parity, kind, cur, next, (first + s + 1) * BT);
    };
    // The steps, two by two: those whose next scores every row of the wave sees
    // whole (and whose copies are of whole tiles), those whose next scores have
    // some to hide, the wave's last one or two, and those of the other waves.
    const uint32_t mine = w_most > first * BT ? (w_most + BT - 1) / BT - first : 0u;
    uint32_t s = 0;
    for (; (uint64_t)(first + s + 3) * BT <= w_least && (uint64_t)min(first + s + 4, last) * BT <= lk; s += 2) {
        turn(even, plain, s, sa, sb);
        turn(uneven, plain, s + 1, sb, sa);
    }
    if constexpr (SPLIT) {
        // (without the steps that have no next scores: with them the compiler
        // spills the shares' kernel, 10 us more at 16 queries behind 6,000 keys)
        auto turn_if = [&](auto parity, uint32_t s, f32x16 (&cur)[2], f32x16 (&next)[2]) {
            meet(maybe, s, s + 1 < steps);
            if ((first + s) * BT < w_most)
                step(parity, masked, cur, next, (first + s + 1) * BT);
        };
        for (; s < steps; s += 2) {
            turn_if(even, s, sa, sb);
            if (s + 1 < steps)
                turn_if(uneven, s + 1, sb, sa);
        }
    } else {
        for (; s + 2 < mine; s += 2) {
            turn(even, masked, s, sa, sb);
            turn(uneven, masked, s + 1, sb, sa);
        }
        if (s + 2 == mine) {
            turn(even, masked, s, sa, sb);
            turn(uneven, final, s + 1, sb, sa);
            s += 2;
        } else if (s + 1 == mine) {
            turn(even, final, s, sa, sb);
            s += 1;
        }
        for (; s < steps; s++)
            meet(maybe, s, s + 1 < steps);
    }
    rl_wait_vmcnt<0>();
    const float L = half_sum(l + l2);
    float odd = 0.f;
#pragma unroll
    for (int d = 0; d < C::DB; d++)
#pragma unroll
        for (int r = 0; r < 16; r++)
            odd = fmaf(o[d][r], 0.f, odd);
    // ---- the rows' outputs -------------------------------------------------------
    auto put = [&] {
        if constexpr (SPLIT) {
            if (shares_of(p, nt) > 1) {
                float *part = p.part + (((size_t)at * p.split + blockIdx.x / blocks) * NW + wave) * C::PART;
#pragma unroll
                for (int d = 0; d < C::DB; d++)
#pragma unroll
                    for (int a = 0; a < 4; a++)
                        *(rl_f32x4 *)(part + ((4 * d + a) * 64 + lane) * 4) =
                            rl_f32x4{o[d][4 * a], o[d][4 * a + 1], o[d][4 * a + 2], o[d][4 * a + 3]};
                part[C::DB * 16 * 64 + lane] = m;
                part[(C::DB * 16 + 1) * 64 + lane] = L;
                return;
            }
        }
        const float inv = my_seen == 0 ? 0.f : 1.f / L;
        uint16_t *out = p.out + (uint64_t)(qs + tok0) * p.out_stride + (uint64_t)g * p.group * D;
        const uint32_t r = (uint32_t)lane & 31u, dt = quotient(h0 + r, p.by_group);
        const uint32_t to = dt * (uint32_t)p.out_stride + (h0 + r - dt * p.group) * D + 8 * hf;
        const bool has = w_row + r < rows;
#pragma unroll
        for (int d = 0; d < C::DB; d++)
#pragma unroll
            for (int a = 0; a < 4; a += 2) {
                // lanes l and l + 32 hold four dims each of both 8-dim chunks: each takes a whole one
                rl_u32x4 w;
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const uint32_t x = pack2<DT>(o[d][4 * a + 2 * e] * inv, o[d][4 * a + 2 * e + 1] * inv);
                    const uint32_t y = pack2<DT>(o[d][4 * a + 4 + 2 * e] * inv, o[d][4 * a + 5 + 2 * e] * inv);
                    const auto h = __builtin_amdgcn_permlane32_swap(x, y, false, false);
                    w[e] = h[0];
                    w[2 + e] = h[1];
                }
                if (has)
                    *(rl_u32x4 *)(out + to + 32 * d + 8 * a) = w;
            }
    };
    if (w_has)
        put();
    // ---- values that are no numbers -------------------------------------------------
    // (a row whose sum is no number is right as it is: NaN)
    if (__builtin_amdgcn_ballot_w64(odd != 0.f && L == L && w_row + (lane & 31) < rows) != 0) {
        // An infinity or NaN in V spoils its whole tile in the matrix product, also
        // for the rows that do not see it (0 times NaN). Below `whole` every row sees
        // every key, so what came of those tiles is right; the places from there to
        // `held`, where those past the last key repeat it, are at most two tiles' and
        // are looked through. Where they hold only
        // numbers the outputs stand. (In fp16 a weight below 2^-25 is rounded to 0, and
        // 0 times a seen infinity is NaN instead: such outputs are computed again too.)
        // 1 x 8,192 tokens, 480-500 us (fp16 520) without any: a NaN in the first token
        // 501 (fp16 4,700), in the last 2,070 (fp16 2,600), an infinity in a dim of every
        // token 3,800 (fp16 4,700); 16 queries behind 6,000 keys 18 without, 28 (fp16 90),
        // 70 (fp16 116), 69 (fp16 115).
        const uint32_t whole = max(w_least, first * BT), held = (w_most + BT - 1) / BT * BT;
        constexpr int E = D / 64;  // dims per lane
        float spoilt = 0.f;
        for (uint32_t j = whole; j < held; j += 8)
#pragma unroll
            for (uint32_t i = 0; i < 8; i++) {
                const uint16_t *v = row_of(1, min(j + i, min(held, lk) - 1)) + lane * E;
#pragma unroll
                for (int e = 0; e < E; e++)
                    spoilt = fmaf(from16<DT>(v[e]), 0.f, spoilt);
            }
        if constexpr (DT != 0) {
#pragma unroll
            for (int d = 0; d < C::DB; d++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    spoilt = L == L && o[d][r] != o[d][r] ? o[d][r] : spoilt;
        }
        if (__builtin_amdgcn_ballot_w64(spoilt != 0.f) != 0) {
            // The wave's rows again, from memory: 32 keys at a time by the matrix
            // cores while all rows see them, then key by key for those that do.
            const float neg = m == -INFINITY ? 0.f : -m;
#pragma unroll
            for (int d = 0; d < C::DB; d++)
                o[d] = f32x16{};
            uint32_t j = first * BT;
            for (; j + 32 <= whole; j += 32) {
                const uint16_t *kp = row_of(0, j + kr) + 8 * hf;
                f32x16 x{};
#pragma unroll
                for (int s = 0; s < C::KS; s++)
                    x = mfma32<DT>(*(const s16x8 *)(kp + 16 * s), qf[s], x);
                float w[16];
#pragma unroll
                for (int r = 0; r < 16; r++)
                    w[r] = __builtin_amdgcn_exp2f(fmaf(x[r], p.scale_log2, neg));
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    // Weights and values as bf16, whose exponents reach every weight: the
                    // weights' high and low parts (low ones times numbers only), fp16 values'
                    // too, so that nothing of them is lost.
                    s16x8 wh, wl;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        wh[e] = (short)to16<0>(w[8 * u + e]);
                        wl[e] = (short)to16<0>(w[8 * u + e] - from16<0>((uint16_t)wh[e]));
                    }
                    const uint16_t *vp = row_of(1, j + 16 * u + 4 * hf) + (lane & 31);
                    const uint64_t v_stride = PAGED ? (uint64_t)D : p.v_stride;
#pragma unroll
                    for (int d = 0; d < C::DB; d++) {
                        s16x8 vh, vl, vn;
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const float v = from16<DT>(vp[(uint64_t)(e % 4 + 8 * (e / 4)) * v_stride + 32 * d]);
                            vh[e] = (short)to16<0>(v);
                            const bool number = v * 0.f == 0.f;
                            vn[e] = number ? vh[e] : (short)0;
                            vl[e] = number ? (short)to16<0>(v - from16<0>((uint16_t)vh[e])) : (short)0;
                        }
                        o[d] = mfma32<0>(vh, wh, o[d]);
                        o[d] = mfma32<0>(vn, wl, o[d]);
                        if constexpr (DT != 0)
                            o[d] = mfma32<0>(vl, wh, o[d]);
                    }
                }
            }
            for (; j < w_most; j++) {
                const uint16_t *kp = row_of(0, j) + 8 * hf, *vp = row_of(1, j) + 4 * hf;
                float x = 0.f;
#pragma unroll
                for (int s = 0; s < C::KS; s++) {
                    const s16x8 k = *(const s16x8 *)(kp + 16 * s);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        x = fmaf(from16<DT>((uint16_t)k[e]), from16<DT>((uint16_t)qf[s][e]), x);
                }
                const float w = __builtin_amdgcn_exp2f(fmaf(half_sum(x), p.scale_log2, neg));
                if (j < my_seen) {
#pragma unroll
                    for (int d = 0; d < C::DB; d++)
#pragma unroll
                        for (int a = 0; a < 4; a++) {
                            const s16x4 v = *(const s16x4 *)(vp + 32 * d + 8 * a);
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                o[d][4 * a + e] = fmaf(w, from16<DT>((uint16_t)v[e]), o[d][4 * a + e]);
                        }
                }
            }
            put();  // (each lane to the places it wrote before)
        }
    }
}

// Joins the shares of the row blocks that have several: a workgroup the 32 rows
// that wave w of theirs had, and 32 of the dims. Lane l holds, of row l % 32, the
// dims 32 d + 8 j + 4 (l / 32) .. + 3 in its 4 d + j-th four words, which wave j
// joins, eight shares' loads at a time (one after the other: 23.8 us against 18.7
// for 16 queries behind 6,000 keys).
template <int D, int DT, bool PAGED>
__global__ __launch_bounds__(256) void attn_prompt_merge_kernel(PromptParams p)
{
    using C = PCfg<D>;
    const int lane = threadIdx.x & 63;
    const uint32_t j = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t d = blockIdx.x % C::DB, w = blockIdx.x / C::DB % NW, at = blockIdx.x / (C::DB * NW);
    const Place place = place_of<PAGED>(p, at, lane);
    const uint32_t g = place.g, tile = place.tile, qs = place.qs, lq = place.lq, lk = place.lk;
    const uint32_t rows = min(lq, p.max_q) * p.group;
    const uint32_t wg_row = tile * ROWS, row = wg_row + w * 32 + (lane & 31);
    if (wg_row >= rows)
        return;
    const uint32_t last_tok = quotient(min(wg_row + ROWS, rows) - 1, p.by_group);
    const uint32_t wg_seen = (uint32_t)max((int32_t)(last_tok - lq + 1) + (int32_t)lk, 0);
    const uint32_t n = shares_of(p, (wg_seen + BT - 1) / BT);
    if (n < 2 || row >= rows)
        return;
    const float *part = p.part + ((size_t)at * p.split * NW + w) * C::PART;
    const float *tops = part + C::DB * 16 * 64 + lane, *words = part + ((4 * d + j) * 64 + lane) * 4;
    float M = -INFINITY, L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t i0 = 0; i0 < n; i0 += 8) {
        rl_f32x4 x[8];
        float m[8], l[8], top = M;
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const size_t off = (size_t)min(i0 + i, n - 1) * NW * C::PART;
            x[i] = *(const rl_f32x4 *)(words + off);
            m[i] = tops[off];
            l[i] = tops[off + 64];
        }
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            m[i] = i0 + i < n ? m[i] : -INFINITY;
            top = fmaxf(top, m[i]);
        }
        const float keep = M == -INFINITY ? 1.f : exp2f(M - top);  // (before a maximum, sums are 0 or no number)
        M = top;
        L *= keep;
#pragma unroll
        for (int e = 0; e < 4; e++)
            o[e] *= keep;
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const float f = m[i] == -INFINITY ? 0.f : exp2f(m[i] - M);
            if (i0 + i < n) {
                L = fmaf(l[i], f, L);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    o[e] = fmaf(x[i][e], f, o[e]);
            }
        }
    }
    const uint32_t tok = quotient(row, p.by_group), head = g * p.group + row - tok * p.group;
    const bool none = (int32_t)(tok - lq + 1) + (int32_t)lk <= 0;
    const float inv = none ? 0.f : 1.f / L;
    uint16_t *dst = p.out + (uint64_t)(qs + tok) * p.out_stride + (uint64_t)head * D + 32 * d + 8 * j + 4 * (lane >> 5);
    *(rl_u32x2 *)dst = rl_u32x2{pack2<DT>(o[0] * inv, o[1] * inv), pack2<DT>(o[2] * inv, o[3] * inv)};
}

// Few row blocks share their keys, in shares of six tiles and more, as many as
// compute units are left: 16 queries behind 6,000 keys 17.5 us against 80.4 of one
// workgroup per row block, 300 behind 2,000 28.9 against 39.1. In shares of eight
// tiles 18.6 us (16 behind 6,000), of four 18.9. Two shares per compute unit where
// each still has 48 tiles: 512 behind 32,000 260 us against 280, 2 x 300 behind
// 16,000 154 against 242 (152 row blocks on 256 compute units); shorter ones
// cost: 2 x 300 behind 600 23.2 against 18.1. So does it to split more than 256
// row blocks: 2 x 1,000 behind 4,000 145 against 113.
struct PromptPlan {
    uint32_t tiles, pairs, split;
    size_t workspace;
    size_t most;  // the largest workspace of calls up to this one's seqs, max_q and max_kv
};

inline PromptPlan plan_of(uint32_t seqs, uint32_t max_q, uint32_t max_kv, uint32_t q_heads, uint32_t kv_heads,
                          uint32_t head_dim)
{
    PromptPlan pl;
    const uint32_t group = q_heads / kv_heads;
    pl.tiles = (uint32_t)(((uint64_t)max_q * group + ROWS - 1) / ROWS);
    pl.pairs = seqs * kv_heads;
    const uint64_t blocks = (uint64_t)pl.tiles * pl.pairs;
    const uint64_t keys = ((uint64_t)max_kv + BT - 1) / BT, cus = rl_cu_count();
    uint64_t shares = 1;
    if (blocks > 0 && blocks <= cus) {
        shares = cus / blocks;
        if (keys >= kLongShareTiles * (2 * cus / blocks))
            shares = 2 * cus / blocks;
    }
    pl.split = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(shares, keys / kShareTiles));
    const size_t part = (size_t)NW * (head_dim / 32 * 16 + 2) * 64 * sizeof(float);
    pl.workspace = 256 + (pl.split > 1 ? (size_t)blocks * pl.split * part : 0);
    // no more for any fewer row blocks and keys: at most one share, or two, per compute unit
    const uint64_t few = std::min(blocks, cus), each = keys / kShareTiles;
    pl.most = 256;
    if (few > 0 && each > 1)
        pl.most += std::min(keys >= kLongShareTiles * (2 * cus / few) ? 2 * cus : cus, few * each) * part;
    return pl;
}


// The rest of a call's parameters, which follow from its plan and its sizes.
inline void set_plan(PromptParams &p, const PromptPlan &pl, uint32_t seqs, uint32_t max_kv, uint32_t q_heads,
                     uint32_t kv_heads, uint32_t head_dim, float scale, void *workspace)
{
    p.kv_heads = kv_heads;
    p.group = q_heads / kv_heads;
    p.scale_log2 = (scale != 0.f ? scale : 1.0f / sqrtf((float)head_dim)) * 1.4426950408889634f;
    p.seqs = seqs;
    p.tiles = pl.tiles;
    p.pairs = pl.pairs;
    p.split = pl.split;
    p.by_group = divisor_of(p.group);
    p.by_pairs = divisor_of(p.pairs);
    p.by_heads = divisor_of(p.kv_heads);
    p.by_tiles = divisor_of(p.tiles);
    p.part = (float *)workspace;
    p.by_xcd = p.pairs % 8 == 0;
    // (each workgroup finds its place for itself. In us, in this order and in batch order, by row blocks:
    // of 3-2,047 tokens, d64, 1,152 33 / 38, 2,048 44 / 50, 4,096 75 / 81, 6,144 113 / 116, 8,192 144 / 146;
    // d128, GQA 4, of 3-1,000 tokens 4,096 75 / 78, 8,192 143 / 142, of 3-700 8,448 127 / 123, 11,264
    // 166 / 162, of 512-1,024 8,192 225 / 224, 16,384 455 / 446)
    p.ranked = p.seqs > 1 && p.seqs <= 64 && (uint64_t)p.pairs * p.tiles <= 4096;
    p.rank_shift = 0;
    while (max_kv >> p.rank_shift > 63)
        p.rank_shift++;
}

template <int D, int DT, bool PAGED>
int prompt_launch(const PromptParams &p)
{
    const uint32_t grid = p.pairs * p.tiles * p.split;
    if (p.split == 1) {
        hipLaunchKernelGGL((attn_prompt_kernel<D, DT, false, PAGED>), dim3(grid), dim3(NW * 64), 0, rl_stream(), p);
        return rl_check_launch("attn_prompt_kernel launch");
    }
    hipLaunchKernelGGL((attn_prompt_kernel<D, DT, true, PAGED>), dim3(grid), dim3(NW * 64), 0, rl_stream(), p);
    if (rl_check_launch("attn_prompt_kernel launch"))
        return -1;
    hipLaunchKernelGGL((attn_prompt_merge_kernel<D, DT, PAGED>), dim3(p.pairs * p.tiles * NW * PCfg<D>::DB), dim3(256), 0,
                       rl_stream(), p);
    return rl_check_launch("attn_prompt_merge_kernel launch");
}

}  // namespace
