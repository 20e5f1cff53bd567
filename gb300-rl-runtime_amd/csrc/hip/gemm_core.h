// gemm_core.h - bf16 matrix products on gfx950 with the operands in either order
// and the caller's own use of the results:
//
//   acc[m][n] = sum_k M[m][k] N[n][k], fp32
//
//  tiles    BM x BN results per workgroup, K in steps of 64, copied HBM -> LDS with
//           global_load_lds_dwordx4 into a ring of NS stages.
//  orders   an operand's rows may follow k (row r's k contiguous) or be the
//           columns of a matrix whose rows are k (k-major). The first is read with
//           ds_read_b128, the second with ds_read_b64_tr_b16, which transposes on
//           the way; 16-byte chunks are permuted on the way in so that neither
//           meets a bank conflict.
//  MFMA     v_mfma_f32_32x32x16_bf16 with N's rows as the A operand: lane l ends up
//           with one row m (l % 32 of a block) and four consecutive columns n at a
//           time, so that sums along n stay in a lane and results leave in
//           16-byte pieces.
//  schedule a step is four slices of 16 k. While one slice is multiplied the
//           next one's operands are read from LDS, one read between two matrix
//           instructions; the barrier of a step stands before its last slice, whose
//           operands are then in registers, so that the next step's first reads and
//           the copies into the freed stage run beside matrix instructions too: half of
//           them in that slice, half in the next (all in one 3 to 5% slower, in three
//           worse). A wave that has passed the barrier goes first until it has issued
//           them (2%).
//  bound    256 x 256 tiles at 2,048 x 128,256 x 4,096: 1,655 us for the statistics,
//           1,300 TFLOP/s, the chip's power (zeros 1,340 us); there the copies, 64 KiB
//           a step and compute unit, whose path alone takes 1,410 us (without its
//           matrix instructions; the matrix instructions alone 1,050). Deeper rings of
//           32-k steps, prefetching lines into L2 and four waves of 128 x 128 were
//           slower.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attn_core.h"
#include "rl_dev_common.h"

namespace {

typedef float gemm_f32x16 __attribute__((ext_vector_type(16)));

constexpr int kGemmK = 64;  // k per step

// One operand: its rows are row0 .. of a matrix with `rows` rows (columns where it
// is k-major) and the pitch ld, in elements; past the last row, and the last k of a
// k-major one, the last is read again (in bounds; results are not used, or are
// products with the other operand's zeros).
struct GemmOperand {
    const uint16_t *base;
    uint64_t ld;
    uint32_t rows;
    uint32_t k;  // of a k-major one
};

template <int ROWS, bool KM, int WAVES>
struct GemmTile {
    static constexpr int BYTES = ROWS * kGemmK * 2;
    static constexpr int OPS = BYTES / 1024 / WAVES;  // 1 KiB copies per wave and step
    static constexpr int NC = KM ? ROWS / 8 : 8;      // 16-byte chunks of an LDS row
    static constexpr int PER = 64 / NC;               // LDS rows per copy
    static_assert(OPS * 1024 * WAVES == BYTES, "whole copies per wave");
    static_assert(!KM || ROWS >= 128, "four 64-byte granules of a k-major row");

    static __device__ __forceinline__ uint32_t swz(uint32_t r) { return KM ? (r & 3u) << 2 : (r >> 1) & 7u; }

    // Byte offsets of this lane's chunks of a step from the tile's first row at its first k.
    static __device__ __forceinline__ void offsets(const GemmOperand &a, uint32_t row0, int wave, int lane,
                                                   uint32_t (&off)[OPS])
    {
#pragma unroll
        for (int i = 0; i < OPS; i++) {
            const uint32_t r = (uint32_t)(wave * OPS + i) * PER + (uint32_t)lane / NC;
            const uint32_t c = ((uint32_t)lane % NC) ^ swz(r);
            if constexpr (KM)
                off[i] = r * (uint32_t)a.ld * 2u + (min(row0 + c * 8u, a.rows - 8u) - row0) * 2u;
            else
                off[i] = (min(row0 + r, a.rows - 1) - row0) * (uint32_t)a.ld * 2u + c * 16u;
        }
    }
    static __device__ __forceinline__ const uint16_t *first(const GemmOperand &a, uint32_t row0)
    {
        return KM ? a.base + row0 : a.base + row0 * a.ld;
    }
    // Copy i of this wave of step kt.
    static __device__ __forceinline__ void copy(const GemmOperand &a, const uint16_t *at, const uint32_t (&off)[OPS],
                                                uint32_t kt, RL_LDS uint8_t *dst, int wave, int lane, int i)
    {
        uint32_t o = off[i];
        if constexpr (KM) {
            if ((kt + 1) * kGemmK > a.k) {
                const uint32_t r = (uint32_t)(wave * OPS + i) * PER + (uint32_t)lane / NC;
                o -= (r - min(r, a.k - 1 - kt * kGemmK)) * (uint32_t)a.ld * 2u;
            }
            at += (uint64_t)kt * kGemmK * a.ld;
        } else {
            at += kt * kGemmK;
        }
        rl_g2lds_16_off(at, o, dst + (wave * OPS + i) * 1024);
    }
    // This lane's addresses inside a stage for the blocks b0 .. of 32 rows.
    // k contiguous: one for each slice, blocks 4 KiB apart; k-major: one for each block, slices 16 rows apart.
    template <int BLOCKS>
    static __device__ __forceinline__ void places(uint32_t b0, int lane, uint32_t (&at)[KM ? BLOCKS : 4])
    {
        const uint32_t hf = (uint32_t)lane >> 5;
        if constexpr (KM) {
            const uint32_t k = ((uint32_t)lane & 15u) >> 2;
#pragma unroll
            for (int b = 0; b < BLOCKS; b++)
                at[b] = (8u * hf + k) * (ROWS * 2u) + (((b0 + b) ^ k) << 6) + 32u * (((uint32_t)lane >> 4) & 1u) +
                        8u * ((uint32_t)lane & 3u);
        } else {
            const uint32_t r = (uint32_t)lane & 31u;
#pragma unroll
            for (int s = 0; s < 4; s++)
                at[s] = (b0 * 32u + r) * 128u + (((2u * s + hf) ^ swz(r)) << 4);
        }
    }
    template <int N>
    static __device__ __forceinline__ s16x8 read(RL_LDS const uint8_t *stage, const uint32_t (&at)[N], int b, int s)
    {
        if constexpr (KM) {
            RL_LDS const uint8_t *from = stage + at[b] + 16 * s * (ROWS * 2);
            const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((RL_LDS s16x4 *)from);
            const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((RL_LDS s16x4 *)(from + 4 * (ROWS * 2)));
            return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            return *(RL_LDS const s16x8 *)(stage + at[s] + b * 4096);
        }
    }
};

// TN x TM blocks of 32 x 32 per wave, WN x WM waves.
template <int TN_, int WN_, int TM_, int WM_, int NS_, bool NKM_, bool MKM_>
struct Gemm {
    static constexpr int TN = TN_, WN = WN_, TM = TM_, WM = WM_, NS = NS_;
    static constexpr int BN = TN * WN * 32, BM = TM * WM * 32, WAVES = WN * WM;
    using NT = GemmTile<BN, NKM_, WAVES>;
    using MT = GemmTile<BM, MKM_, WAVES>;
    static constexpr int OPS = NT::OPS + MT::OPS;
    static constexpr int LDS = NS * (NT::BYTES + MT::BYTES);
    using Acc = gemm_f32x16[TN][TM];

    // The steps kt0 .. kt1 - 1 of the tile at m0, n0 (kt0 < kt1); `rot`: the step to begin with, from which it wraps.
    // SUMS: eight steps at a time are summed by themselves, so that a sum of 4,096 products is rounded 32 times on its
    // way and not 256 times.
    template <bool SUMS = false>
    static __device__ __forceinline__ void run(const GemmOperand &n, const GemmOperand &m, uint32_t n0, uint32_t m0,
                                               uint32_t kt0, uint32_t kt1, uint32_t rot, uint8_t *smem_, Acc &acc)
    {
        RL_LDS uint8_t *smem = (RL_LDS uint8_t *)smem_;
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t wn = (uint32_t)wave % WN, wm = (uint32_t)wave / WN;
        uint32_t noff[NT::OPS], moff[MT::OPS], nat[NKM_ ? TN : 4], mat[MKM_ ? TM : 4];
        NT::offsets(n, n0, wave, lane, noff);
        MT::offsets(m, m0, wave, lane, moff);
        NT::template places<TN>(wn * TN, lane, nat);
        MT::template places<TM>(wm * TM, lane, mat);
        const uint16_t *nbase = NT::first(n, n0), *mbase = MT::first(m, m0);
        auto nstage = [&](uint32_t i) { return smem + i * NT::BYTES; };
        auto mstage = [&](uint32_t i) { return smem + NS * NT::BYTES + i * MT::BYTES; };
        const uint32_t steps = kt1 - kt0;
        // copy i of step s
        auto copy = [&](uint32_t s, int i) {
            uint32_t kt = kt0 + s + rot;
            kt = kt < kt1 ? kt : kt - steps;
            if (i < NT::OPS)
                NT::copy(n, nbase, noff, kt, nstage(s % NS), wave, lane, i);
            else
                MT::copy(m, mbase, moff, kt, mstage(s % NS), wave, lane, i - NT::OPS);
        };
#pragma unroll
        for (int a = 0; a < TN; a++)
#pragma unroll
            for (int b = 0; b < TM; b++)
                acc[a][b] = gemm_f32x16{};
#pragma unroll
        for (int s = 0; s < NS; s++)
            if ((uint32_t)s < steps)
#pragma unroll
                for (int i = 0; i < OPS; i++)
                    copy(s, i);
        // Step s + 1's copies have landed once at most those of the NS - 2 steps behind it are outstanding, if they
        // were all issued.
        auto wait = [&](uint32_t s) {
            if (NS > 2 && s + NS - 1 < steps)
                rl_wait_vmcnt<(NS - 2) * OPS>();
            else
                rl_wait_vmcnt<0>();
        };
        if (NS - 1 < steps)
            rl_wait_vmcnt<(NS - 1) * OPS>();
        else
            rl_wait_vmcnt<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        Acc total;
        if constexpr (SUMS)
#pragma unroll
            for (int a = 0; a < TN; a++)
#pragma unroll
                for (int b = 0; b < TM; b++)
                    total[a][b] = gemm_f32x16{};
        auto add = [&] {
#pragma unroll
            for (int a = 0; a < TN; a++)
#pragma unroll
                for (int b = 0; b < TM; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        total[a][b][e] += acc[a][b][e];
        };
        s16x8 fn[2][TN], fm[2][TM];
#pragma unroll
        for (int a = 0; a < TN; a++)
            fn[0][a] = NT::read(nstage(0), nat, a, 0);
#pragma unroll
        for (int b = 0; b < TM; b++)
            fm[0][b] = MT::read(mstage(0), mat, b, 0);
        for (uint32_t s = 0; s < steps; s++) {
            RL_LDS const uint8_t *ns = nstage(s % NS), *ms = mstage(s % NS);
            RL_LDS const uint8_t *ns1 = nstage((s + 1) % NS), *ms1 = mstage((s + 1) % NS);
            const bool more = s + NS < steps;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if (q == 3) {
                    rl_wait_lgkmcnt0();
                    wait(s);
                    __builtin_amdgcn_s_barrier();  // step s + 1 is there, and nobody reads step s any more
                    asm volatile("" ::: "memory");
                    __builtin_amdgcn_s_setprio(1);
                }
                if (q == 1)
                    __builtin_amdgcn_s_setprio(0);
                constexpr int ALL = TN * TM, READS = TN + TM;
#pragma unroll
                for (int i = 0; i < ALL; i++) {
                    const int a = i / TM, b = i % TM;
                    acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, fn[q & 1][a]),
                                                                        __builtin_bit_cast(bf16x8, fm[q & 1][b]),
                                                                        acc[a][b], 0, 0, 0);
                    // the next slice's operands
#pragma unroll
                    for (int j = i * READS / ALL; j < (i + 1) * READS / ALL; j++) {
                        if (j < TM)
                            fm[(q + 1) & 1][j] = MT::read(q < 3 ? ms : ms1, mat, j, (q + 1) & 3);
                        else
                            fn[(q + 1) & 1][j - TM] = NT::read(q < 3 ? ns : ns1, nat, j - TM, (q + 1) & 3);
                    }
                    // (the copies in two parts: all of them behind the barrier are a burst that the matrix
                    // instructions wait behind)
                    constexpr int HALF = OPS / 2;
                    if (q == 3 && more)
#pragma unroll
                        for (int j = i * HALF / ALL; j < (i + 1) * HALF / ALL; j++)
                            copy(s + NS, j);
                    if (q == 0 && s > 0 && s - 1 + NS < steps)
#pragma unroll
                        for (int j = HALF + i * (OPS - HALF) / ALL; j < HALF + (i + 1) * (OPS - HALF) / ALL; j++)
                            copy(s - 1 + NS, j);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (SUMS && s % 8 == 7) {
                add();
#pragma unroll
                for (int a = 0; a < TN; a++)
#pragma unroll
                    for (int b = 0; b < TM; b++)
                        acc[a][b] = gemm_f32x16{};
            }
        }
        if constexpr (SUMS) {
            add();
#pragma unroll
            for (int a = 0; a < TN; a++)
#pragma unroll
                for (int b = 0; b < TM; b++)
                    acc[a][b] = total[a][b];
        }
        rl_wait_lgkmcnt0();  // (the reads behind the last step)
    }

    // Hands the results out in 16-byte pieces of rows, f(m, n, w): row m and column n of the tile on, as bf16 (eight
    // columns) or as floats (four), so that a wave's pieces lie 64 * TN (floats: 128 * TN) bytes one behind the other in
    // each row. They change lanes in LDS, which must be free of operands: 32 rows of a wave at a time.
    template <bool FLOATS, typename F>
    static __device__ __forceinline__ void each(const Acc &acc, uint8_t *smem_, F f)
    {
        constexpr uint32_t NC = TN * (FLOATS ? 8 : 4), OUT = 32 * NC / 64;  // 16-byte chunks of a row; pieces per lane
        static_assert(WAVES * 32 * NC * 16 <= LDS, "room for the waves' rows");
        const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t wn = wave % WN, wm = wave / WN, hf = lane >> 5, r = lane & 31u;
        RL_LDS uint8_t *own = (RL_LDS uint8_t *)smem_ + wave * (32 * NC * 16);
        // (16 neighbouring lanes write the same chunk of 16 rows, and read chunks that follow each other: both meet
        // every bank once)
        auto place = [&](uint32_t row, uint32_t c) {
            const uint32_t swz = NC >= 16 ? row & 15u : NC == 8 ? (row >> 1) & 7u : (row >> 2) & 3u;
            return (RL_LDS rl_u32x4 *)(own + row * (NC * 16) + ((c ^ swz) << 4));
        };
#pragma unroll
        for (int b = 0; b < TM; b++) {
#pragma unroll
            for (int a = 0; a < TN; a++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    if constexpr (FLOATS) {
                        *place(r, 8 * a + 2 * c + hf) = rl_u32x4{
                            __float_as_uint(acc[a][b][4 * c]), __float_as_uint(acc[a][b][4 * c + 1]),
                            __float_as_uint(acc[a][b][4 * c + 2]), __float_as_uint(acc[a][b][4 * c + 3])};
                    } else if (c % 2 == 0) {
                        // lanes l and l + 32 hold four columns each of both eights: each takes a whole one
                        rl_u32x4 w;
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const uint32_t x = pack(acc[a][b][4 * c + 2 * e], acc[a][b][4 * c + 2 * e + 1]);
                            const uint32_t y = pack(acc[a][b][4 * c + 4 + 2 * e], acc[a][b][4 * c + 5 + 2 * e]);
                            const auto h = __builtin_amdgcn_permlane32_swap(x, y, false, false);
                            w[e] = h[0];
                            w[2 + e] = h[1];
                        }
                        *place(r, 4 * a + c + hf) = w;
                    }
                }
            rl_wave_lds_fence();
#pragma unroll
            for (uint32_t j = 0; j < OUT; j++) {
                const uint32_t row = (j * 64 + lane) / NC, c = (j * 64 + lane) % NC;
                f((wm * TM + b) * 32 + row, wn * TN * 32 + c * (FLOATS ? 4 : 8), *place(row, c));
            }
            rl_wave_lds_fence();
        }
    }

    static __device__ __forceinline__ uint32_t pack(float x, float y)
    {
        rl_bf16x2 w;
        w[0] = (__bf16)x;
        w[1] = (__bf16)y;
        return __builtin_bit_cast(uint32_t, w);
    }
};

// Workgroup b runs on XCD b % 8, each with its own L2. Each XCD gets a run of `all` pieces of work that follow each
// other (false: none is left).
__device__ __forceinline__ bool gemm_run_of(uint32_t b, uint32_t all, uint32_t &t)
{
    const uint32_t per = (all + 7) / 8;
    t = b % 8 * per + b / 8;
    return b / 8 < per && t < all;
}

// The tiles in columns of up to 8 along m, so that the 32 that an XCD has at a time are about 8 x 4 and share their
// operands.
__device__ __forceinline__ void gemm_tile_of(uint32_t t, uint32_t m_tiles, uint32_t n_tiles, uint32_t &mt, uint32_t &nt)
{
    const uint32_t group = t / (8 * n_tiles), first = group * 8, high = min(8u, m_tiles - first);
    const uint32_t r = t - group * 8 * n_tiles;
    mt = first + r % high;
    nt = r / high;
}

}  // namespace
