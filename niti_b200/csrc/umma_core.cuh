// What the tensor-core kernels share: problem description, tile order, the TMA producer and MMA issuer roles, and the host side of
// a launch (tensor maps, shared-memory grants).  umma_kernels.cu explains the structure of these kernels.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <atomic>
#include <cstdint>
#include <cstdio>

#include "../../include/niti_b200.h"
#include "internal.h"
#include "ptx.cuh"

namespace niti {
#ifdef NITI_PARKED_TIMING
static __device__ unsigned long long g_dbg_stamps[32];
#define PARK_STAMP(i) do { if (blockIdx.x == 0) g_dbg_stamps[i] = global_timer_ns(); } while (0)
#define DBG_CLK(v) const long long v = clock64()
#define DBG_DECL long long dbg_acc[4] = {0, 0, 0, 0}
#define DBG_ACC(i, d) dbg_acc[(i) & 3] += (d)
#define DBG_OUT(base) do { if (blockIdx.x == 0 && (threadIdx.x & 31) == 0) for (int q_ = 0; q_ < 4; ++q_) g_dbg_stamps[(base) + q_] = dbg_acc[q_]; } while (0)
#else
#define DBG_CLK(v) do { } while (0)
#define DBG_DECL do { } while (0)
#define DBG_ACC(i, d) do { } while (0)
#define DBG_OUT(base) do { } while (0)
#define PARK_STAMP(i) do { } while (0)
#endif

// Pin a value in a register: kernel parameters live in the constant bank, and under register pressure the compiler
// re-reads them at every use; in the producer / MMA loops each such load sits on one warp's serial critical path.
__device__ __forceinline__ int keep_reg(int v) { asm volatile("" : "+r"(v)); return v; }

constexpr int BLOCK_M = 128;
constexpr int ROW_BYTES = 128;               // bytes per shared-memory row of an operand tile
constexpr int PANEL_BYTES = 128 * ROW_BYTES; // one 128-row operand panel
constexpr int UMMA_THREADS = 192;
constexpr uint32_t SWIZZLE_128B_CODE = 2;
constexpr uint32_t SWIZZLE_64B_CODE = 4;
constexpr uint32_t SWIZZLE_32B_CODE = 6;
constexpr int EPI_CHUNK_BYTES = 128 * 32 * 4;  // 128 rows x 32 int32 columns, one TMA store box
constexpr int EPI_BARRIER = 1;                 // named barrier of the 128 epilogue threads

// Epilogue staging: each thread owns one accumulator row of 32 int32 (128 bytes) and writes it as
// eight 16-byte chunks at the 128-byte-swizzled position the TMA store expects (chunk ^ row%8);
// that placement is also free of shared-memory bank conflicts.
__device__ __forceinline__ void stage_row(uint32_t buf, int row, const uint32_t (&v)[32]) {
    const uint32_t base = buf + static_cast<uint32_t>(row) * 128u;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        st_shared_v4(base + (static_cast<uint32_t>(j ^ (row & 7)) << 4), v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
}

// ------------------------------------------------------------------------------------------------
// GEMM / convolution forward / error-backward
// ------------------------------------------------------------------------------------------------
// Division of a non-negative int by a divisor fixed at launch: q = (umulhi(mul, n) + n) >> shift with
// shift = ceil(log2 d) and mul = floor(2^32 (2^shift - d) / d) + 1, exact for 0 <= n < 2^31.  The tile loops turn a
// tile number into coordinates once per tile; eight hardware-less 32-bit divisions there were a quarter of an epilogue.
struct FastDiv { unsigned mul, shift; int d; };
static FastDiv make_fastdiv(int d) {
    FastDiv f{1u, 0u, d < 1 ? 1 : d};
    while ((1ull << f.shift) < static_cast<unsigned long long>(f.d)) ++f.shift;
    f.mul = static_cast<unsigned>(((1ull << 32) * ((1ull << f.shift) - static_cast<unsigned long long>(f.d))) / static_cast<unsigned long long>(f.d) + 1ull);
    return f;
}
__device__ __forceinline__ int fdiv(int n, const FastDiv& f) {
    return static_cast<int>((__umulhi(f.mul, static_cast<unsigned>(n)) + static_cast<unsigned>(n)) >> f.shift);
}

struct GemmParams {
    int conv;              // 0: plain GEMM, 1: implicit-GEMM convolution (A tile = 4-D box of pixels)
    int M, N;              // output rows (GEMM rows or pixels) and columns
    int num_kb;            // reduction blocks of the whole problem
    int splits;            // split-K: each output tile is produced `splits` times over disjoint reduction ranges
    int m_tiles, n_tiles;
    int a_mn, b_mn;        // operand majors (0 = K-major, 1 = MN-major)
    int a_bytes;           // bytes one A stage receives from TMA
    int mma_n;             // columns of one MMA: the tile's, or of the only column tile those that exist (in sixteens)
    int b_bytes;           // bytes of one tap's B tile (of this CTA's half of it): fewer than the tile where the box is lower
    // Operands of 32-byte rows that lie in memory as the MMA reads them (32-byte swizzle: see patch_half), loaded with
    // one untiled bulk copy instead of a box of 128 rows.  1: A [M][32] and B [N][32], one reduction block;
    // 2: B [reduction][32] as 32 MN-major columns.
    int rows32;
    const int8_t* a32; const int8_t* b32;
    int K;                 // rows32 == 2: reduction length
    // convolution geometry
    int H, W, S, pad, Nimg;
    int flip;              // 1: error-backward, taps are read mirrored (offset pad - r instead of r - pad)
    int tapstride;         // elements between consecutive taps in a filter row
    int BW, BH, BI;        // pixels of one tile along w, h and images; BW*BH*BI <= 128
    int tiles_w, tiles_h;
    FastDiv fd_mn, fd_n, fd_tw, fd_th;  // by m_tiles * n_tiles, n_tiles, tiles_w, tiles_h (set by finish_params)
    int cblocks;           // 128-byte blocks per tap: ceil(reduction channels / 128)
    int red;               // reduction channels per tap (conv) -- the last block of a tap may be partial
    unsigned* maxabs;      // max|acc| is reduced into this word; may be null (split-K partials)
    int32_t* status;
    int group_m;           // GEMM tile order: row tiles per group (0 / 1: plain row-major)
    int nstages;           // stages of the ring actually used (<= the compiled maximum; tuning / experiments)
    int accumulate;        // plain products: tiles are added to the result
    int32_t* plain_out;    // plain products: the result [M][N] where its rows are no whole 16-byte groups (null: through the tensor map)
    int split_cols;        // 1: both epilogue warpgroups share every tile (alternate 128-column groups); 0: they alternate tiles
    // fused requantisation (FUSED kernels): int8 output narrowed by the shift in state[0].
    // state = {shift, max|acc|, redo flag, redo count, finished-CTA ticket}; the last CTA of a first
    // launch derives the true shift from max|acc|, publishes it with the exponent / shift outputs and
    // raises the redo flag when the applied shift was wrong.
    int32_t* state;
    int only_if_redo;      // 1: this launch does nothing unless state[2] != 0, and verifies nothing
    int kind, target_bits;
    const int32_t* exp_a; const int32_t* exp_b; int32_t* exp_out; int32_t* shift_out;
    int mode, relu;
    int8_t* out8;          // fused kernels: the int8 output as a plain pointer (rows = row_lin, pitch N bytes)
    const int8_t* mask;    // fused kernels: optional ReLU-backward mask, same shape as the output (zero where mask <= 0)
    int8_t* pool_out;      // parked kernel, forward convolutions: optional 2x2 / stride-2 max-pooled copy of the output [N][H/2][W/2][K]
    uint32_t* side;        // streaming fused kernel, round-to-nearest without ReLU: two more bits per output (16 per word, rows of
                           // N / 4 bytes) from which the output for the next LOWER shift follows exactly (requant_step_down)
    const unsigned long long* seed;
    unsigned rng_stream;
    unsigned long long rng_offset;
};

// a call of its own: its dozen instructions at every wait lay between the ones that a launch fetches and runs once
static __device__ __noinline__ void report_abort(int32_t* status, int code, int role) {
    if (status != nullptr && atomicCAS(status, 0, code) == 0) {
        status[1] = static_cast<int32_t>(blockIdx.x + blockIdx.y * gridDim.x);
        status[2] = role;
    }
}

// Output tile (row tile, column tile) of the mn-th tile in launch order.  Convolutions: row-major (the few column
// tiles of a row tile run together and share its activation tile).  GEMMs: row tiles in groups of 8, column-major
// inside a group, so the ~148 tiles in flight at any time cover a compact block of the output (8 x ~18 tiles) instead
// of 2-3 whole rows: a wave then re-reads ~36 MB of operands instead of all of B.  Only when the operands do not fit
// in L2 anyway (group_m is set on the host): 8192^3 406 -> 376 us, 16384^3 3679 -> 2977 us, 4096^3 unchanged.
__device__ __forceinline__ void tile_coords(const GemmParams& p, int mn, int* m_pair, int* n_t) {
    if (p.group_m <= 1) { *m_pair = fdiv(mn, p.fd_n); *n_t = mn - *m_pair * p.n_tiles; return; }
    const int GM = p.group_m;
    const int per_group = GM * p.n_tiles;
    const int group = mn / per_group, in_group = mn % per_group;
    const int first = group * GM;
    const int rows = min(GM, p.m_tiles - first);
    *m_pair = first + in_group % rows;
    *n_t = in_group / rows;
}

// ---- warp roles shared by the streaming kernel and the accumulator-parking kernel -------------
// stages of the ring in use (NITI_OPT_STAGE_CAP)
__device__ __forceinline__ int ring_stages(const GemmParams& p, int compiled) { return (p.nstages > 0 && p.nstages < compiled) ? p.nstages : compiled; }

// TMA producer: fills the stage ring for every tile of this CTA, in tile order.  The WHOLE warp runs the loop and
// an elected lane issues.  TMA and MMA instructions take their operands from uniform registers, and the compiler keeps
// addresses, coordinates and descriptors there only while every branch around them is provably warp-uniform: waits
// therefore spin INSIDE one asm statement and hand back a voted verdict (mbar_wait_uniform), values read from shared
// memory or special registers pass through a shuffle, and the issuing lane comes from elect.sync.  Measured on B200
// (clock64 around the instructions): 50 cycles per tcgen05.mma and ~20 per TMA instruction this way; 85-90 and ~50 when
// a loop-carried value depends on a per-lane asm result or the issuer is chosen by `lane == 0`; a loop entered by a
// single lane sits in between.  Per-tile integer divisions are skipped when the reduction is not split.
// TWO: this CTA is half of a CTA pair (cluster ranks 0/1).  Tiles are 256 rows high: rank r owns rows
// [128 r, 128 r + 128) of the pair's tile (m tile 2*pair_m + r) and columns [r BN/2, (r+1) BN/2) of the B
// operand; all byte counts are reported to rank 0's "full" barrier, which its MMA thread waits on.
// ROWS32: operands of 32-byte rows (p.rows32).  A variant of its own: as a branch of the one loop its byte counts and
// sources made every other product's issue slower (2048 x 128 x 4096: 20.5 us with the branch, 18.5 without; 8x8x8, 512 -> 256: 20.5, 18.5).
template <int BN, int STAGES, int STAGE_BYTES, bool TWO, bool ROWS32>
__device__ __forceinline__ void producer_role(uint8_t* smem, uint64_t* full_bar, uint64_t* empty_bar, const CUtensorMap* tmA,
                                              const CUtensorMap* tmB, const GemmParams& p, const int first, const int step,
                                              volatile int* abort_flag) {
    const int mn_tiles = p.m_tiles * p.n_tiles;
    const int total_tiles = mn_tiles * p.splits;
    const uint32_t rank = TWO ? __shfl_sync(0xFFFFFFFFu, cluster_ctarank(), 0) : 0u;  // a special register: make it provably uniform
    constexpr int BNH = TWO ? BN / 2 : BN;  // B columns this CTA loads
    const int nst = ring_stages(p, STAGES);
    const uint32_t abort_addr = smem_u32(const_cast<int*>(abort_flag));
    const uint32_t smem0 = smem_u32(smem), full0 = smem_u32(full_bar), empty0 = smem_u32(empty_bar);
    const int conv = keep_reg(p.conv), flip = keep_reg(p.flip), pad = keep_reg(p.pad), S = keep_reg(p.S), cblocks = keep_reg(p.cblocks);
    const int tapstride = keep_reg(p.tapstride), b_mn = keep_reg(p.b_mn), a_mn = keep_reg(p.a_mn);
    const int rows32 = ROWS32 ? keep_reg(p.rows32) : 0;
    const uint32_t tx_full = static_cast<uint32_t>(keep_reg((TWO ? 2 : 1) * (p.a_bytes + p.b_bytes)));
    int s = 0; uint32_t ph = 0;
    uint32_t sa = smem0, fb_cur = full0, eb_cur = empty0;  // running stage pointers, wrapping with the ring
    DBG_DECL;
    DBG_CLK(c_begin);
    for (int tile = first; tile < total_tiles; tile += step) {
        int mn = tile, kb_lo = 0, kb_hi = p.num_kb;
        if (p.splits > 1) {
            const int split = fdiv(tile, p.fd_mn);
            mn = tile - split * mn_tiles;
            kb_lo = static_cast<int>(static_cast<long long>(split) * p.num_kb / p.splits);
            kb_hi = static_cast<int>(static_cast<long long>(split + 1) * p.num_kb / p.splits);
        }
        int m_pair, n_t;
        tile_coords(p, mn, &m_pair, &n_t);
        const int m_t = TWO ? 2 * m_pair + static_cast<int>(rank) : m_pair;
        int tw = 0, th = 0, tn = 0;
        if (conv) { const int q1 = fdiv(m_t, p.fd_tw); tw = m_t - q1 * p.tiles_w; tn = fdiv(q1, p.fd_th); th = q1 - tn * p.tiles_h; }
        const int ncol = n_t * BN + static_cast<int>(rank) * BNH;  // first B column of this CTA
        const int px = tw * p.BW, py = th * p.BH, pn = tn * p.BI;
        // This loop is one warp's serial instruction stream and sets the pace of the whole pipeline: the tap
        // (r, sx) and channel block cb of a reduction block are kept as running counters (four integer divisions per
        // block cost more than the block's MMAs), waits return nothing to branch on, pointers advance by addition.
        int cb = 0, sx = 0, r = 0;
        if (conv && kb_lo != 0) { const int tap0 = kb_lo / cblocks; cb = kb_lo % cblocks; r = tap0 / S; sx = tap0 % S; }
        for (int kb = kb_lo; kb < kb_hi; ++kb) {
            mbar_wait_quiet(eb_cur, ph ^ 1u, abort_addr);
            DBG_ACC(22, 1);
            const uint32_t sb = sa + PANEL_BYTES;
            uint32_t fb = fb_cur;
            uint32_t tx_bytes = tx_full, tx_b = 0;
            if (ROWS32) {  // the last rows of an operand may be fewer than a tile's; what they leave in the stage meets zeros or rows nobody stores
                const int b_rows = rows32 == 1 ? min(BN, p.N - ncol) : min(128, p.K - kb * 128);
                tx_b = static_cast<uint32_t>(b_rows) * 32u;
                tx_bytes = tx_b + (rows32 == 1 ? static_cast<uint32_t>(min(BLOCK_M, p.M - m_t * BLOCK_M)) * 32u : static_cast<uint32_t>(PANEL_BYTES));
            }
            if (elect_one()) {
                if (TWO) {
                    if (rank == 0) mbar_arrive_expect_tx(fb, tx_bytes);
                    fb = mapa_u32(fb, 0);
                } else {
                    mbar_arrive_expect_tx(fb, tx_bytes);
                }
                if (conv) {
                    const int tap = r * S + sx;
                    const int dx = flip ? pad - sx : sx - pad, dy = flip ? pad - r : r - pad;
                    if (TWO) tma_load_4d_pair(sa, tmA, fb, cb * ROW_BYTES, px + dx, py + dy, pn);
                    else     tma_load_4d(sa, tmA, fb, cb * ROW_BYTES, px + dx, py + dy, pn);
                    if (b_mn) {
#pragma unroll
                        for (int q = 0; q < (BNH + 127) / 128; ++q) {
                            if (TWO) tma_load_2d_pair(sb + q * PANEL_BYTES, tmB, fb, tap * tapstride + ncol + q * 128, cb * 128);
                            else     tma_load_2d(sb + q * PANEL_BYTES, tmB, fb, tap * tapstride + ncol + q * 128, cb * 128);
                        }
                    } else {
                        if (TWO) tma_load_2d_pair(sb, tmB, fb, tap * tapstride + cb * ROW_BYTES, ncol);
                        else     tma_load_2d(sb, tmB, fb, tap * tapstride + cb * ROW_BYTES, ncol);
                    }
                } else if (ROWS32 && rows32 == 1) {
                    bulk_load(sa, p.a32 + static_cast<long long>(m_t) * (BLOCK_M * 32), tx_bytes - tx_b, fb);
                    bulk_load(sb, p.b32 + static_cast<long long>(ncol) * 32, tx_b, fb);
                } else if (ROWS32) {
                    tma_load_2d(sa, tmA, fb, m_t * BLOCK_M, kb * 128);
                    bulk_load(sb, p.b32 + static_cast<long long>(kb) * (128 * 32), tx_b, fb);
                } else {
                    if (TWO) {
                        if (a_mn) tma_load_2d_pair(sa, tmA, fb, m_t * BLOCK_M, kb * 128);
                        else      tma_load_2d_pair(sa, tmA, fb, kb * ROW_BYTES, m_t * BLOCK_M);
                    } else {
                        if (a_mn) tma_load_2d(sa, tmA, fb, m_t * BLOCK_M, kb * 128);
                        else      tma_load_2d(sa, tmA, fb, kb * ROW_BYTES, m_t * BLOCK_M);
                    }
                    if (b_mn) {
#pragma unroll
                        for (int q = 0; q < BNH / 128; ++q) {
                            if (TWO) tma_load_2d_pair(sb + q * PANEL_BYTES, tmB, fb, ncol + q * 128, kb * 128);
                            else     tma_load_2d(sb + q * PANEL_BYTES, tmB, fb, ncol + q * 128, kb * 128);
                        }
                    } else {
                        if (TWO) tma_load_2d_pair(sb, tmB, fb, kb * ROW_BYTES, ncol);
                        else     tma_load_2d(sb, tmB, fb, kb * ROW_BYTES, ncol);
                    }
                }
            }
            if (conv && ++cb == cblocks) { cb = 0; if (++sx == S) { sx = 0; ++r; } }
            sa += STAGE_BYTES; fb_cur += 8u; eb_cur += 8u;
            if (++s == nst) { s = 0; ph ^= 1u; sa = smem0; fb_cur = full0; eb_cur = empty0; }
        }
    }
    if (*abort_flag) report_abort(p.status, 1, 0);  // a quiet wait of this role (or another role) gave up
    DBG_CLK(c_end); DBG_ACC(20, c_end - c_begin);
    DBG_OUT(20);
}

// MMA issuer: the whole warp runs the loop with warp-uniform control flow (see the producer), one elected lane issues
// the MMAs and the commits.  Streaming: NACC accumulators used in turn, each handed back by the
// epilogue (tempty).  Parked (NACC = 0): tile i of this CTA accumulates into TMEM columns [i*BN, (i+1)*BN) and
// stays there until the kernel ends, so no accumulator is ever waited for.
// TWO: run by rank 0 of a CTA pair only; M = 256 MMAs over both CTAs' shared and tensor memory, and every
// completion (stage free, accumulator full) is signalled to both CTAs.
template <bool TWO>
__device__ __forceinline__ void umma_issue(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if (TWO) umma_i8_pair(d_tmem, a, b, idesc, accumulate); else umma_i8(d_tmem, a, b, idesc, accumulate);
}
template <int BN, int STAGES, int STAGE_BYTES, int NACC, bool TWO, bool ROWS32>
__device__ __forceinline__ void mma_role(uint8_t* smem, uint64_t* full_bar, uint64_t* empty_bar, uint64_t* tfull_bar,
                                         uint64_t* tempty_bar, uint32_t tmem_base_in, const GemmParams& p, const int first, const int step,
                                         volatile int* abort_flag) {
    constexpr bool PARKED = NACC == 0;
    const int rows32 = ROWS32 ? keep_reg(p.rows32) : 0;
    const int mn_tiles = p.m_tiles * p.n_tiles;
    const int total_tiles = mn_tiles * p.splits;
    const uint32_t idesc = make_idesc_i8(TWO ? 2 * BLOCK_M : BLOCK_M, p.mma_n, p.a_mn, p.b_mn);
    const int nst = ring_stages(p, STAGES);
    const uint32_t tmem_base = __shfl_sync(0xFFFFFFFFu, tmem_base_in, 0);  // read from shared memory: make it provably uniform
    const uint32_t abort_addr = smem_u32(const_cast<int*>(abort_flag));
    const uint32_t full0 = smem_u32(full_bar), empty0 = smem_u32(empty_bar);
    // operand descriptors of stage 0 (a stage's are these advanced by the stage offset) and the K = 32 steps
    const uint32_t s0 = smem_u32(smem);
    const uint64_t a_base = rows32 == 1 ? make_smem_desc(s0, 16, 256, SWIZZLE_32B_CODE) : p.a_mn ? make_smem_desc(s0, PANEL_BYTES, 1024, SWIZZLE_128B_CODE) : make_smem_desc(s0, 16, 1024, SWIZZLE_128B_CODE);
    // a 64-column MN-major operand has rows of 64 bytes: 64-byte swizzle, 8-row groups of 512 bytes
    const uint64_t b_base = ROWS32 ? make_smem_desc(s0 + PANEL_BYTES, 1024, 256, SWIZZLE_32B_CODE) : p.b_mn ? (BN == 64 ? make_smem_desc(s0 + PANEL_BYTES, 64 * ROW_BYTES, 512, SWIZZLE_64B_CODE)
                                               : make_smem_desc(s0 + PANEL_BYTES, PANEL_BYTES, 1024, SWIZZLE_128B_CODE))
                                   : make_smem_desc(s0 + PANEL_BYTES, 16, 1024, SWIZZLE_128B_CODE);
    const uint32_t a_step = static_cast<uint32_t>(keep_reg((p.a_mn ? 32 * ROW_BYTES : 32) >> 4));  // in descriptor units of 16 bytes
    const uint32_t b_step = static_cast<uint32_t>(keep_reg((rows32 == 2 ? 32 * 32 : p.b_mn ? 32 * (BN == 64 ? 64 : ROW_BYTES) : 32) >> 4));
    const int conv = keep_reg(p.conv), red = keep_reg(p.red), cblocks = keep_reg(p.cblocks), num_kb = keep_reg(p.num_kb), splits = keep_reg(p.splits);
    int s = 0; uint32_t ph = 0; bool ok = true; int it = 0;
    // every reduction block has four MMAs unless a conv tap's channel count ends in a partial 128-byte block
    const bool all4 = conv ? (red & 127) == 0 : rows32 != 1;
    // running stage pointers: descriptors and barrier addresses advance by one stage per block and wrap with the ring
    const uint64_t stage_step = STAGE_BYTES >> 4;
    uint64_t a_cur = a_base, b_cur = b_base;
    uint32_t full_cur = full0, empty_cur = empty0;
    DBG_DECL;
#ifdef NITI_PARKED_TIMING
    long long c_first = 0;
#endif
    for (int tile = first; ok && tile < total_tiles; tile += step, ++it) {
        const int acc = PARKED ? it : it % (PARKED ? 1 : NACC);
        if (!PARKED) {
            const uint32_t aph = (it / (PARKED ? 1 : NACC)) & 1u;
            ok = mbar_wait_uniform(smem_u32(&tempty_bar[acc]), aph ^ 1u, abort_addr);
            if (!ok) { *abort_flag = 1; report_abort(p.status, 2, 1); break; }
            tc_fence_after();
        }
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
        int kb_lo = 0, kb_hi = num_kb;
        if (splits > 1) {
            const int split = tile / mn_tiles;
            kb_lo = static_cast<int>(static_cast<long long>(split) * num_kb / splits);
            kb_hi = static_cast<int>(static_cast<long long>(split + 1) * num_kb / splits);
        }
        int cb = (conv && kb_lo != 0) ? kb_lo % cblocks : 0;  // channel block within the tap: a running counter, no division per block
        for (int kb = kb_lo; kb < kb_hi; ++kb) {
            DBG_ACC(19, 1);
#ifdef NITI_PARKED_TIMING
            if (it == 0 && kb == kb_lo) { c_first = clock64(); if (PARKED) PARK_STAMP(2); }
#endif
            if (all4) {
                // wait for the stage, four MMAs, commit: one asm statement, nothing for the loop to branch on
                umma_block4_wait<TWO>(d_tmem, a_cur, b_cur, a_step, b_step, idesc, static_cast<uint32_t>(kb != kb_lo), empty_cur,
                                      full_cur, ph, abort_addr);
            } else {
                // a partial block: issue only the MMAs (K = 32 each) that cover real channels (the rest is TMA zero fill)
                const int left = red - cb * 128;
                const int nmma = !conv ? 1 : left >= 128 ? 4 : (left + 31) >> 5;  // rows32 == 1: the one block is 32 deep
                if (++cb == cblocks) cb = 0;
                mbar_wait_quiet(full_cur, ph, abort_addr);
                if (elect_one()) {
                    for (int k = 0; k < nmma; ++k)
                        umma_issue<TWO>(d_tmem, a_cur + k * a_step, b_cur + k * b_step, idesc, static_cast<uint32_t>(kb != kb_lo || k != 0));
                    if (TWO) umma_commit_pair(empty_cur); else umma_commit(empty_cur);
                }
            }
            a_cur += stage_step; b_cur += stage_step; full_cur += 8u; empty_cur += 8u;
            if (++s == nst) { s = 0; ph ^= 1u; a_cur = a_base; b_cur = b_base; full_cur = full0; empty_cur = empty0; }
        }
        if (ok && elect_one()) { if (TWO) umma_commit_pair(smem_u32(&tfull_bar[acc])); else umma_commit(smem_u32(&tfull_bar[acc])); }
    }
    if (*abort_flag) report_abort(p.status, 3, 1);  // a quiet wait of this role (or another role) gave up
    if (PARKED) PARK_STAMP(3);
#ifdef NITI_PARKED_TIMING
    DBG_ACC(16, clock64() - c_first);
#endif
    DBG_OUT(16);
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static void* driver_entry(const char* name) {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult qres;
    return cudaGetDriverEntryPoint(name, &sym, cudaEnableDefault, &qres) == cudaSuccess && qres == cudaDriverEntryPointSuccess ? sym : nullptr;
}
static EncodeTiledFn get_encode() {
    static const EncodeTiledFn fn = reinterpret_cast<EncodeTiledFn>(driver_entry("cuTensorMapEncodeTiled"));
    return fn;
}
// A number for the current context that no other one has had or will have; 0: not known.
static unsigned long long context_number() {
    static const auto get_id = reinterpret_cast<CUresult (*)(CUcontext, unsigned long long*)>(driver_entry("cuCtxGetId"));
    unsigned long long id = 0;
    return get_id != nullptr && get_id(nullptr, &id) == CUDA_SUCCESS ? id + 1 : 0;
}

// Tensor map with 128-byte swizzle over uint8 (operands) or int32 (outputs) elements; dims/box
// innermost first, in elements; strides of dims 1.. in bytes.
static int encode_map(CUtensorMap* map, const void* ptr, bool int32_elems, int rank, const uint64_t* dims,
                      const uint64_t* strides, const uint32_t* box, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B,
                      CUtensorMapL2promotion promotion = CU_TENSOR_MAP_L2_PROMOTION_L2_256B) {
    EncodeTiledFn enc = get_encode();
    if (!enc) return set_cuda_error_text("cuTensorMapEncodeTiled is not available from this driver");
    cuuint64_t gdim[4]; cuuint64_t gstr[3]; cuuint32_t bx[4]; cuuint32_t es[4];
    for (int i = 0; i < rank; ++i) { gdim[i] = dims[i]; bx[i] = box[i]; es[i] = 1; }
    for (int i = 0; i + 1 < rank; ++i) gstr[i] = strides[i];
    CUresult r = enc(map, int32_elems ? CU_TENSOR_MAP_DATA_TYPE_INT32 : CU_TENSOR_MAP_DATA_TYPE_UINT8, rank,
                     const_cast<void*>(ptr), gdim, gstr, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     swizzle, promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        char buf[160];
        snprintf(buf, sizeof buf, "cuTensorMapEncodeTiled failed with CUresult %d (rank %d)", static_cast<int>(r), rank);
        return set_cuda_error_text(buf);
    }
    return 0;
}

// The dynamic shared memory of a kernel, granted once per context: asked for at every launch it was about a microsecond of the host's
// time, and a single image's layers are bound by that.  Not once per device: a second context of a device, or its first one after a
// reset, starts without the grant, and a launch there would be refused.
template <auto KERNEL>
static cudaError_t allow_shared(int bytes) {
    static std::atomic<unsigned long long> granted[16];  // context numbers; two that share a place ask in turn
    const unsigned long long now = context_number();
    std::atomic<unsigned long long>& place = granted[now % 16];
    if (now != 0 && place.load(std::memory_order_acquire) == now) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && now != 0) place.store(now, std::memory_order_release);
    return e;
}

// The result of a launch whose thread blocks have to be resident together: see LAUNCH_REFUSED.
static int launched_together(cudaError_t e) {
    if (e != cudaErrorCooperativeLaunchTooLarge && e != cudaErrorInvalidClusterSize && e != cudaErrorLaunchOutOfResources) return launched(e);
    cudaGetLastError();
    return LAUNCH_REFUSED;
}

static int sm_count() {
    static int n = 0;
    if (n == 0) {
        int dev = 0;
        cudaGetDevice(&dev);
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        if (n <= 0) n = 148;
    }
    return n;
}

}  // namespace niti
