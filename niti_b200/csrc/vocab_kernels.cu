// A last layer with a vocabulary of classes and the losses over it: softmax cross entropy against one class a row and against a
// teacher's top logits, with the error and the weight gradient, without the logits ever reaching memory (training on up to four
// tokens keeps theirs).
//
// The reference ends in TiLinear.forward (ti_torch.py:241-253), TiLoss.forward (ti_loss.py:6-36) and TiLinear.backward (:255-266),
// which write [rows][classes] logits and errors out and whose softmax has 11 bits: with 2048 equal classes every error is zero.
// Here the softmax works on the int32 accumulators themselves:
//
//   a[t][v] = sum_f x[t][f] w[v][f],  e = exp_x + exp_w - temperature_log2
//   E(d)    = 2^30 exp(-d 2^e) for whole d >= 0, in integers (exp_weight below; a quartic, |relative error| < 2.9e-6)
//   pieces of 64 classes:  m_c = max a,  S_c = (sum E(m_c - a)) >> 6          (2^24 is 1)
//   a row:  M = max m_c,  S = sum_c (S_c E(M - m_c)) >> 20                    (2^34 is 1; for p)
//           L = sum_c (S_c q) >> (10 + I),  q >> I being E(M - m_c)           (2^44 is 1; for the loss)
//   loss  = (M - a_y) 2^e + ln(L 2^-44)                                       (double, stored as float32)
//   p     = hi32(E(M - a) R) >> (n - 3),  R = (2^63 - 1) / (S >> n), 2^31 <= S >> n < 2^32    (2^30 is 1; S >= 2^34, so n >= 3)
//   err   = p - target share, narrowed by 23 bits to int8 (2^-7), NITI's roundings (pseudo-stochastically, by p's own low bits,
//           equal classes are rounded alike)
//
// E ends at 2^-30, so S loses up to 2^-30 of each class of a piece far below the maximum: p is up to V 2^-30 (2.4e-4 for 2^18 classes) of
// itself too large, a thirtieth of err's unit.  As a loss that would be all there is where one class stands alone (16 nats above 131072
// others 0.7 % of it, from 21.5 on everything), so L shifts the product, not E.
//
// Sums of integers do not depend on their order, so tiles, splits and thread blocks change no bit of any result.
//
// Launches, each setting up under the one before:
//   vocab_align_kernel     operands whose rows are no multiples of 16 bytes, copied to such a pitch
//   vocab_kernel           the product; each piece's maximum and sum            (up to four tokens: vocab_thin_kernel)
//   vocab_finish_kernel    the wanted classes' logits, row sums, losses, reciprocals, the wanted classes' errors
// and for training, a piece of the vocabulary (up to 96 MB of errors) at a time,
//   vocab_kernel           the product again, its errors as int8 into the workspace
//   vocab_patch_kernel     a teacher's classes' errors over them
//   umma_gemm_two          error and weight gradient                            (up to four tokens: vocab_back_thin_kernel)
// and vocab_narrow_kernel, err_calc of the error.
//
// What bounds it: beyond a few hundred tokens vocab_kernel's epilogue up to about 2500 features (the integer pipes: E), the tensor
// cores above; the two products the tensor cores; up to 128 tokens memory; a few small launches their number.
#include <cuda.h>
#include <cuda_runtime.h>
#include <climits>
#include <cstdint>

#include "umma_core.cuh"
#include "requant.cuh"
#include "grid_barrier.cuh"

namespace niti {
namespace {

constexpr int PIECE = 64;            // classes whose exponentials are summed relative to their own maximum: part of the definition
constexpr int VBN = 256;             // columns of the widest output tile
// Loading warp, MMA warp and four epilogue warps for each 64 columns of a tile; a thread works on one row of them: one piece.
constexpr int vocab_threads(int bn) { return 64 + bn / PIECE * 128; }
constexpr int FINISH_THREADS = 256;
constexpr int MAX_ENTRIES = 128;     // a teacher's logits per row

// ---------------------------------------------------------------------------------------------- E(d)
// u = d 2^e log2(e) in units of 2^-25, plus a half: its whole part I is the shift, its fraction less a half the polynomial's
// argument in [-1/2, 1/2).  d 2^(26+e) has at most 31 bits once d is cut at D, where E is 0 (31 powers of two and more).
struct ExpScale { unsigned D, K; int sl; };
__device__ __forceinline__ ExpScale exp_scale(int e) {
    ExpScale s;
    if (e > 5) e = 5;  // from here on every d >= 1 gives 0
    s.D = e >= 0 ? static_cast<unsigned>((21 + (1 << e)) >> e) : e <= -28 ? 0xFFFFFFFFu : 43u << (-e - 1);
    s.sl = e >= -26 ? 26 + e : 0;
    s.K = e >= -26 ? 0xB8AA3B29u : e <= -58 ? 0u : 0xB8AA3B29u >> (-26 - e);  // log2(e) 2^31
    return s;
}
// The high words of 32 x 32 bit products.  As the upper half of a 64-bit product with a separate addition: mad.hi, four cycles of the
// multiplier as well, held back the instructions beside it (64 E's of a row: 37 cycles per 128 with mad.hi, 32 so).
__device__ __forceinline__ uint32_t mul_hi(uint32_t a, uint32_t b) {
    uint64_t d;
    asm("mul.wide.u32 %0, %1, %2;" : "=l"(d) : "r"(a), "r"(b));
    return static_cast<uint32_t>(d >> 32);
}
__device__ __forceinline__ int32_t mul_hi(int32_t a, int32_t b) {
    int64_t d;
    asm("mul.wide.s32 %0, %1, %2;" : "=l"(d) : "r"(a), "r"(b));
    return static_cast<int32_t>(d >> 32);
}
__device__ __forceinline__ uint32_t shift_right(uint32_t a, uint32_t n) {  // 0 for n >= 32, which the operator >> leaves undefined
    uint32_t d;
    asm("shr.u32 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(n));
    return d;
}
// E before its shift; h: u without its half
__device__ __forceinline__ uint32_t exp_mantissa(uint32_t h) {
    const int32_t phi = static_cast<int32_t>(h << 7);  // the fraction of h + 2^24, less a half, with 2^32 as 1
    int32_t q = mul_hi(phi, 10289510) - 60029066;
    q = mul_hi(phi, q) + 257956795;
    q = mul_hi(phi, q) - 744236436;
    return static_cast<uint32_t>(mul_hi(phi, q) + (1 << 30));
}
// xs = min(d, D) << sl
__device__ __forceinline__ uint32_t exp_weight_shifted(uint32_t xs, uint32_t K) {
    const uint32_t h = mul_hi(xs, K);
    return shift_right(exp_mantissa(h), (h + (1u << 24)) >> 25);
}
__device__ __forceinline__ uint32_t exp_weight(uint32_t d, const ExpScale& s) { return exp_weight_shifted(min(d, s.D) << s.sl, s.K); }

// The largest d that a row's sums tell from no term at all: 64 nats and more, where d 2^(26+e) has 32 bits.  Of units above 32 nats (which
// exp_scale takes for 32) it is 0.
__device__ __forceinline__ unsigned far_limit(int e, const ExpScale& s) { return e > 5 ? 0u : 0xFFFFFFFFu >> s.sl; }
// A piece's part of its row's sums; S is for training alone.  No branch, which would hold back the loads behind it: beside one sum of
// cut E's, the two cost 8192 x 1024 x 32768 with an early return 5 us of 337, this way nothing that shows.
template <bool TRAIN>
__device__ __forceinline__ void add_piece(uint32_t sum, uint32_t d, const ExpScale& s, unsigned far, unsigned long long* S, unsigned long long* L) {
    if (d > far) sum = 0;
    const uint32_t h = mul_hi(min(d, far) << s.sl, s.K), q = exp_mantissa(h), I = (h + (1u << 24)) >> 25;
    if (TRAIN) *S += (static_cast<unsigned long long>(sum) * shift_right(q, I)) >> 20;
    *L += (static_cast<unsigned long long>(sum) * q) >> min(10u + I, 63u);  // 30 and 31 bits: none is left behind 63
}

// A row's view of E: E(M - a) for its accumulators a <= M.  max(a, floor) cuts d at D; the difference is taken in the
// multiply-add that shifts it (modulo 2^32, which the result stays below).
struct RowExp { int32_t floor_a; uint32_t base; };
__device__ __forceinline__ RowExp row_exp(int32_t M, const ExpScale& s) {
    const long long f = static_cast<long long>(M) - s.D;
    return {f < INT_MIN ? INT_MIN : static_cast<int32_t>(f), static_cast<uint32_t>(M) << s.sl};
}
__device__ __forceinline__ uint32_t exp_weight_row(int32_t a, const RowExp& r, uint32_t minus_unit, uint32_t K) {
    return exp_weight_shifted(static_cast<uint32_t>(max(a, r.floor_a)) * minus_unit + r.base, K);
}

// A row's wanted class and its error in a word, where a row has one: bits 0 to 17, bit 23 and bits 24 to 31.
__device__ __forceinline__ int one_entry(int cls, int err) { return cls | (1 << 23) | (err << 24); }

struct VocabParams {
    GemmParams g;
    const int32_t* exp_x; const int32_t* exp_w; int temperature;
    int rows;                 // tokens
    int copies_log2;          // of the tokens in a row tile (see vocab_copies)
    int first, classes;       // of the piece of the vocabulary this launch covers (multiple of 256); classes of the whole vocabulary
    int32_t* piece_max; uint32_t* piece_sum;  // [pieces][rows]
    const int4* row_stat;     // {M, R, n - 3, the wanted class where there is one: see one_entry}; R = 0: a row without an error
    int8_t* err; long long err_pitch;
    const unsigned long long* seed; unsigned rng_stream; unsigned long long rng_offset;
};

// A stage of the ring holds 256 bytes of every row for a pair of thread blocks (two panels of A, two of the half of B) and 128 for a
// single one.
template <bool TWO, int BN>
struct VocabCfg {
    static constexpr int BLOCKS = TWO ? 2 : 1;  // 128-byte reduction blocks of a stage
    static constexpr int B_PANEL_BYTES = (TWO ? BN / 2 : BN) * ROW_BYTES;
    static constexpr int STAGE_BYTES = BLOCKS * (PANEL_BYTES + B_PANEL_BYTES);
    static constexpr int PER_SM = BN == 64 ? 3 : 1;  // thread blocks
    static constexpr int STAGES = 224 * 1024 / PER_SM / STAGE_BYTES;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 /*alignment slack*/ + 256 /*barriers*/;
};

// ---------------------------------------------------------------------------------------------- loads and MMAs
// The roles of umma_core.cuh for this one layout (both operands along the reduction), in half the instructions: the sixteen
// epilogue warps keep the schedulers so busy that what the issuing warps execute per reduction block, not the tensor pipe, set
// the pace (2048 features: 12400 cycles a tile with the general roles, 8900 where the epilogue computed nothing).
template <bool TWO, int BN>
__device__ __forceinline__ void vocab_load(uint8_t* smem, uint64_t* full_bar, uint64_t* empty_bar, const CUtensorMap* tmA, const CUtensorMap* tmB,
                                           const GemmParams& p, int copies_log2, int first, int step, volatile int* abort_flag) {
    using Cfg = VocabCfg<TWO, BN>;
    const int total = keep_reg(p.m_tiles * p.n_tiles), num_kb = keep_reg(p.num_kb);
    const uint32_t rank = TWO ? __shfl_sync(0xFFFFFFFFu, cluster_ctarank(), 0) : 0u;
    const uint32_t abort_addr = smem_u32(const_cast<int*>(abort_flag));
    const uint32_t smem0 = smem_u32(smem), full0 = smem_u32(full_bar), empty0 = smem_u32(empty_bar);
    const uint32_t block_tx = static_cast<uint32_t>(keep_reg((TWO ? 2 : 1) * (p.a_bytes + Cfg::B_PANEL_BYTES)));
    uint32_t s = 0, ph = 1;
    for (int tile = first; tile < total; tile += step) {
        int m_pair, n_t;
        tile_coords(p, tile, &m_pair, &n_t);
        const int ya = (TWO ? 2 * m_pair + static_cast<int>(rank) : m_pair) * BLOCK_M;
        const int yb = n_t * BN + static_cast<int>(rank) * (BN / 2);
        for (int kb = 0; kb < num_kb; kb += Cfg::BLOCKS) {
            mbar_wait_quiet(empty0 + 8 * s, ph, abort_addr);
            const uint32_t sa = smem0 + s * Cfg::STAGE_BYTES;
            if (elect_one()) {
                const bool two = TWO && kb + 1 < num_kb;
                uint32_t fb = full0 + 8 * s;
                if (TWO) {
                    if (rank == 0) mbar_arrive_expect_tx(fb, two ? 2 * block_tx : block_tx);
                    fb = mapa_u32(fb, 0);
                    tma_load_2d_pair(sa, tmA, fb, kb * ROW_BYTES, ya);
                    tma_load_2d_pair(sa + 2 * PANEL_BYTES, tmB, fb, kb * ROW_BYTES, yb);
                    if (two) {
                        tma_load_2d_pair(sa + PANEL_BYTES, tmA, fb, (kb + 1) * ROW_BYTES, ya);
                        tma_load_2d_pair(sa + 3 * PANEL_BYTES, tmB, fb, (kb + 1) * ROW_BYTES, yb);
                    }
                } else {
                    mbar_arrive_expect_tx(fb, block_tx);
#pragma unroll 1
                    for (int c = 0; c < 1 << copies_log2; ++c) tma_load_2d(sa + c * (PANEL_BYTES >> copies_log2), tmA, fb, kb * ROW_BYTES, ya);
                    tma_load_2d(sa + PANEL_BYTES, tmB, fb, kb * ROW_BYTES, yb);
                }
            }
            if (++s == Cfg::STAGES) { s = 0; ph ^= 1u; }
        }
    }
    if (*abort_flag) report_abort(p.status, 1, 0);
}

// wait for a stage, MMAs of 32 reduction elements each (their descriptors differ in the low word), commit: one statement
#define VOCAB_MMA(GROUP, AT, PRED)                                               \
    "add.u32 x, %1, " AT ";\n\tmov.b64 a, {x, %3};\n\t"                         \
    "add.u32 x, %2, " AT ";\n\tmov.b64 b, {x, %3};\n\t"                         \
    "@E tcgen05.mma.cta_group::" GROUP ".kind::i8 [%0], a, b, %4, " PRED ";\n\t"
template <bool TWO>
__device__ __forceinline__ void vocab_mma_stage(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate,
                                                uint32_t empty_bar, uint32_t full_bar, uint32_t parity, uint32_t abort_addr) {
    if (TWO) {
        asm volatile(
            "{\n\t.reg .pred P, Q, E, T;\n\t.reg .b32 r, ab, x;\n\t.reg .u64 t0, t1;\n\t.reg .b64 a, b;\n\t"
            NITI_QUIET_WAIT_ASM("VWP", "%7", "%8", "%9", "%10")
            "elect.sync r|E, 0xFFFFFFFF;\n\tsetp.ne.b32 P, %5, 0;\n\tsetp.eq.b32 T, 0, 0;\n\t"
            VOCAB_MMA("2", "0", "P") VOCAB_MMA("2", "2", "T") VOCAB_MMA("2", "4", "T") VOCAB_MMA("2", "6", "T")
            VOCAB_MMA("2", "1024", "T") VOCAB_MMA("2", "1026", "T") VOCAB_MMA("2", "1028", "T") VOCAB_MMA("2", "1030", "T")
            "@E tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%6], %11;\n\t}"
            :: "r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate), "r"(empty_bar), "r"(full_bar), "r"(parity), "r"(abort_addr),
               "l"(WAIT_LIMIT_NS), "h"(static_cast<uint16_t>(3))
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred P, Q, E, T;\n\t.reg .b32 r, ab, x;\n\t.reg .u64 t0, t1;\n\t.reg .b64 a, b;\n\t"
            NITI_QUIET_WAIT_ASM("VW", "%7", "%8", "%9", "%10")
            "elect.sync r|E, 0xFFFFFFFF;\n\tsetp.ne.b32 P, %5, 0;\n\tsetp.eq.b32 T, 0, 0;\n\t"
            VOCAB_MMA("1", "0", "P") VOCAB_MMA("1", "2", "T") VOCAB_MMA("1", "4", "T") VOCAB_MMA("1", "6", "T")
            "@E tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%6];\n\t}"
            :: "r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate), "r"(empty_bar), "r"(full_bar), "r"(parity), "r"(abort_addr),
               "l"(WAIT_LIMIT_NS)
            : "memory");
    }
}
template <bool TWO, int BN>
__device__ __forceinline__ void vocab_mma(uint8_t* smem, uint64_t* full_bar, uint64_t* empty_bar, uint64_t* tfull_bar, uint64_t* tempty_bar,
                                          uint32_t tmem_base_in, const GemmParams& p, int first, int step, volatile int* abort_flag) {
    using Cfg = VocabCfg<TWO, BN>;
    constexpr int STEPS = 4 * Cfg::BLOCKS;  // MMAs of a full stage
    const int total = keep_reg(p.m_tiles * p.n_tiles), all_steps = keep_reg((p.K + 31) / 32);
    const uint32_t idesc = make_idesc_i8(TWO ? 2 * BLOCK_M : BLOCK_M, BN, 0, 0);
    const uint32_t tmem_base = __shfl_sync(0xFFFFFFFFu, tmem_base_in, 0);
    const uint32_t abort_addr = smem_u32(const_cast<int*>(abort_flag));
    const uint32_t full0 = smem_u32(full_bar), empty0 = smem_u32(empty_bar);
    const uint64_t a0 = make_smem_desc(smem_u32(smem), 16, 1024, SWIZZLE_128B_CODE);
    const uint32_t lo0 = static_cast<uint32_t>(a0), hi = static_cast<uint32_t>(a0 >> 32);
    uint32_t s = 0, ph = 0, it = 0;
    for (int tile = first; tile < total; tile += step, ++it) {
        const uint32_t acc = it & 1;
        if (!mbar_wait_uniform(smem_u32(&tempty_bar[acc]), ((it >> 1) & 1u) ^ 1u, abort_addr)) { *abort_flag = 1; report_abort(p.status, 2, 1); break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        for (int k = 0; k < all_steps; k += STEPS) {
            const uint32_t a_lo = lo0 + s * (Cfg::STAGE_BYTES >> 4), b_lo = a_lo + ((Cfg::BLOCKS * PANEL_BYTES) >> 4);
            if (all_steps - k >= STEPS) {
                vocab_mma_stage<TWO>(d_tmem, a_lo, b_lo, hi, idesc, static_cast<uint32_t>(k), empty0 + 8 * s, full0 + 8 * s, ph, abort_addr);
            } else {  // the reduction's end inside a stage
                mbar_wait_quiet(full0 + 8 * s, ph, abort_addr);
                if (elect_one()) {
                    for (int j = 0; k + j < all_steps; ++j) {
                        const uint32_t at = (j & 3) * 2 + (j >> 2) * (PANEL_BYTES >> 4);
                        umma_issue<TWO>(d_tmem, (static_cast<uint64_t>(hi) << 32) | (a_lo + at), (static_cast<uint64_t>(hi) << 32) | (b_lo + at), idesc, static_cast<uint32_t>(k + j));
                    }
                    if (TWO) umma_commit_pair(empty0 + 8 * s); else umma_commit(empty0 + 8 * s);
                }
            }
            if (++s == Cfg::STAGES) { s = 0; ph ^= 1u; }
        }
        if (elect_one()) { if (TWO) umma_commit_pair(smem_u32(&tfull_bar[acc])); else umma_commit(smem_u32(&tfull_bar[acc])); }
    }
    if (*abort_flag) report_abort(p.status, 3, 1);
}

// 64 columns of one row: the piece's maximum and its sum of exponentials.
__device__ __forceinline__ void piece_stats(const uint32_t (&v)[64], int lim, const ExpScale& sc, uint32_t minus_unit, int32_t* m_out, uint32_t* s_out) {
    int32_t m = INT_MIN;
    unsigned long long sum = 0;
    if (lim >= PIECE) {
#pragma unroll
        for (int i = 0; i < PIECE; i += 2) m = __vimax3_s32(m, static_cast<int>(v[i]), static_cast<int>(v[i + 1]));
        const RowExp r = row_exp(m, sc);
#pragma unroll
        for (int i = 0; i < PIECE; i += 2)  // two of at most 2^30.5 fit in a word
            sum += exp_weight_row(static_cast<int>(v[i]), r, minus_unit, sc.K) + exp_weight_row(static_cast<int>(v[i + 1]), r, minus_unit, sc.K);
    } else {  // the vocabulary's last piece
#pragma unroll
        for (int i = 0; i < PIECE; ++i)
            if (i < lim) m = max(m, static_cast<int>(v[i]));
        const RowExp r = row_exp(m, sc);
#pragma unroll
        for (int i = 0; i < PIECE; ++i)
            if (i < lim) sum += exp_weight_row(static_cast<int>(v[i]), r, minus_unit, sc.K);
    }
    *m_out = m;
    *s_out = static_cast<uint32_t>(sum >> 6);
}

// p (2^30 is 1, never negative) in units of 2^-7, 128 still to be cut to 127: the same values as narrow(p, 23, ...).  Pseudo-
// stochastically p is rounded up where its twelve upper dropped bits A exceed twice the eleven lower ones, B: where A + 4095 - B
// carries.
template <int ROUND>
__device__ __forceinline__ int narrow_p(uint32_t p, uint32_t rnd) {
    if (ROUND == ROUND_NEAREST) return static_cast<int>((p + (1u << 22)) >> 23);
    if (ROUND == ROUND_STOCHASTIC) return static_cast<int>((p + (~rnd & 0x7FFFFFu)) >> 23);  // up where the dropped bits exceed the word's
    return static_cast<int>((p + 0x7FF800u - ((p << 12) & 0x7FF000u)) >> 23);
}

enum { VOCAB_STATS = 3 };  // beside the three roundings of the error kernel

// The product x w^T, tile by tile in tensor memory, and per row and 64 columns either the piece's statistics (WHAT == VOCAB_STATS) or
// the errors as int8 in the workspace (WHAT: their rounding).  Roles, ring and accumulators are those of umma_gemm_kernel; the
// epilogue warps (sixteen for 256 columns) take a tile's 64-column groups out of tensor memory into registers, hand the accumulator
// back at once and work on the registers under the next tile's MMAs.
template <bool TWO, int WHAT, int BN>
__global__ void __launch_bounds__(vocab_threads(BN), (VocabCfg<TWO, BN>::PER_SM))
vocab_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const VocabParams vp) {
    using Cfg = VocabCfg<TWO, BN>;
    constexpr int STAGES = Cfg::STAGES;
    const GemmParams& p = vp.g;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * Cfg::STAGE_BYTES);
    uint64_t* full_bar = bars;
    uint64_t* empty_bar = bars + STAGES;
    uint64_t* tfull_bar = bars + 2 * STAGES;
    uint64_t* tempty_bar = bars + 2 * STAGES + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 4);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = TWO ? cluster_ctarank() : 0u;

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) { mbar_init(smem_u32(&full_bar[i]), 1); mbar_init(smem_u32(&empty_bar[i]), 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(smem_u32(&tfull_bar[i]), 1); mbar_init(smem_u32(&tempty_bar[i]), BN / PIECE * 4 * (TWO ? 2 : 1)); }
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
    }
    if (warp == 1) {
        if (TWO) { tmem_alloc_pair(smem_u32(tmem_slot), 2 * BN); tmem_relinquish_pair(); }
        else     { tmem_alloc(smem_u32(tmem_slot), 2 * BN); tmem_relinquish(); }
    }
    tc_fence_before();
    __syncthreads();
    if (TWO) cluster_sync_all();
    tc_fence_after();
    dependents_wait();
    dependents_start();
    const uint32_t tmem_base = *tmem_slot;
    const int total_tiles = p.m_tiles * p.n_tiles;
    const int cta_first = TWO ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
    const int cta_step = TWO ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);

    if (warp == 0) {
        vocab_load<TWO, BN>(smem, full_bar, empty_bar, &tmA, &tmB, p, vp.copies_log2, cta_first, cta_step, abort_flag);
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0)
            vocab_mma<TWO, BN>(smem, full_bar, empty_bar, tfull_bar, tempty_bar, tmem_base, p, cta_first, cta_step, abort_flag);
        __syncwarp();
    } else {
        const int piece = (warp - 2) >> 2, q = warp & 3;  // its 64 columns and 32 rows of every tile
        const uint32_t abort_addr = smem_u32(const_cast<int*>(abort_flag));
        const ExpScale sc = exp_scale(*vp.exp_x + *vp.exp_w - vp.temperature);
        const uint32_t minus_unit = 0u - (1u << sc.sl);
        unsigned long long seed = 0;
        if (WHAT == ROUND_STOCHASTIC) seed = *vp.seed;
        int it = 0;
        for (int tile = cta_first; tile < total_tiles; tile += cta_step, ++it) {
            const int acc = it & 1; const uint32_t aph = (it >> 1) & 1u;
            int m_pair, n_t;
            tile_coords(p, tile, &m_pair, &n_t);
            const int m_t = TWO ? 2 * m_pair + static_cast<int>(rank) : m_pair;
            const int cl = TWO ? 0 : vp.copies_log2;
            const int row = m_t * BLOCK_M + (q & ((4 >> cl) - 1)) * 32 + lane;
            const int col = n_t * BN + piece * PIECE;  // within this launch's classes
            const bool mine = ((piece + n_t) & ((1 << cl) - 1)) == q >> (2 - cl);  // this copy's rows see to these columns
            const bool valid = mine && row < vp.rows;
            int4 stat = make_int4(0, 0, 0, 0);
            if (WHAT != VOCAB_STATS && valid) stat = vp.row_stat[row];
            if (!mbar_wait_uniform(smem_u32(&tfull_bar[acc]), aph, abort_addr)) {
                *abort_flag = 1;
                if (lane == 0) report_abort(p.status, 4, 2);
                break;
            }
            tc_fence_after();
            const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(acc * BN + piece * PIECE);
            uint32_t v[PIECE];
            if (mine && col < p.N) {
                tmem_ld_32x32(taddr, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
                tmem_ld_32x32(taddr + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
                tmem_ld_wait();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (TWO) mbar_arrive_cluster_relaxed(mapa_u32(smem_u32(&tempty_bar[acc]), 0));
                else     mbar_arrive(smem_u32(&tempty_bar[acc]));
            }
            if (col >= p.N || !valid) continue;
            if (WHAT == VOCAB_STATS) {
                int32_t m; uint32_t s;
                piece_stats(v, p.N - col, sc, minus_unit, &m, &s);
                const long long at = static_cast<long long>(col / PIECE) * vp.rows + row;
                vp.piece_max[at] = m;
                vp.piece_sum[at] = s;
            } else {
                const RowExp r = row_exp(stat.x, sc);
                const uint32_t R = static_cast<uint32_t>(stat.y), sh = static_cast<uint32_t>(stat.z);
                int8_t* out = vp.err + row * vp.err_pitch + col;
                const unsigned long long block0 =
                    WHAT == ROUND_STOCHASTIC ? (vp.rng_offset + row) * static_cast<unsigned long long>((vp.classes + 3) >> 2) + ((vp.first + col) >> 2) : 0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        uint32_t rnd[4] = {0, 0, 0, 0};
                        int y[4];
                        if (WHAT == ROUND_STOCHASTIC) random_block(seed, vp.rng_stream, block0 + h * 8 + j, rnd);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t E = exp_weight_row(static_cast<int>(v[h * 32 + j * 4 + k]), r, minus_unit, sc.K);
                            y[k] = narrow_p<WHAT>(mul_hi(E, R) >> sh, rnd[k]);
                        }
                        w[j] = pack2_sat_s8(y[1], y[0], pack2_sat_s8(y[3], y[2], 0u));
                    }
                    st_global_v8(out + h * 32, w);
                }
                const int at = (stat.w & 0x3FFFF) - vp.first - col;
                if ((stat.w & (1 << 23)) && at >= 0 && at < PIECE) out[at] = static_cast<int8_t>(stat.w >> 24);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (TWO) cluster_sync_all();
    if (warp == 1) {
        if (*abort_flag) __nanosleep(200000);  // let copies and MMAs already in flight land
        tc_fence_after();
        __syncwarp();
        if (TWO) tmem_dealloc_pair(tmem_base, 2 * BN); else tmem_dealloc(tmem_base, 2 * BN);
    }
}

// ---------------------------------------------------------------------------------------------- operands of odd rows
// Rows of `bytes` bytes, one behind the other from any address, to rows of a pitch of 16 bytes, the rest of each zeroed.  A thread to
// 16 bytes: five aligned words and four funnel shifts; what lies across the tensor's ends is read byte by byte.
// Two tensors with rows of the same length in one launch.
__global__ void __launch_bounds__(256) vocab_align_kernel(const int8_t* src0, long long rows0, const int8_t* src1, long long rows1,
                                                          uint4* dst0, uint4* dst1, int bytes, int pitch16) {
    const long long pieces0 = rows0 * pitch16, pieces = pieces0 + rows1 * pitch16;
    dependents_wait();
    dependents_start();
    for (long long n0 = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; n0 < pieces; n0 += static_cast<long long>(gridDim.x) * 256) {
        const bool second = n0 >= pieces0;
        const long long i = second ? n0 - pieces0 : n0;
        const int8_t* const src = second ? src1 : src0;
        const uintptr_t begin = reinterpret_cast<uintptr_t>(src), end = begin + (second ? rows1 : rows0) * bytes;
        const long long row = i / pitch16;
        const int c = static_cast<int>(i - row * pitch16) * 16, n = min(16, bytes - c);
        const uintptr_t at = begin + row * bytes + c, word0 = at & ~uintptr_t(3);
        uint32_t o[4];
        if (word0 >= begin && word0 + 20 <= end) {
            const uint32_t* p = reinterpret_cast<const uint32_t*>(word0);
            const uint32_t shift = static_cast<uint32_t>(at - word0) * 8;
            uint32_t w[5];
#pragma unroll
            for (int k = 0; k < 5; ++k) w[k] = p[k];
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = __funnelshift_r(w[k], w[k + 1], shift);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                o[k] = 0;
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    if (4 * k + b < n) o[k] |= static_cast<uint32_t>(static_cast<uint8_t>(src[row * bytes + c + 4 * k + b])) << (8 * b);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // zeros behind the row's end
            const int left = n - 4 * k;
            if (left < 4) o[k] = left <= 0 ? 0u : o[k] & ((1u << (8 * left)) - 1u);
        }
        (second ? dst1 : dst0)[i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
}
// Every launch of a call may begin while the kernel before it ends (see dependents_wait, with which each of these kernels begins): a
// training step of seven launches takes five to seven microseconds less. What an earlier launch wrote is read by plain loads: those through
// the read-only path may be moved in front of the wait.
template <class... P, class... A>
int launch_next(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, const A&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    return launched(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
}
int align_rows(const int8_t* src0, long long rows0, void* dst0, const int8_t* src1, long long rows1, void* dst1, int bytes, int pitch, cudaStream_t st) {
    const long long blocks = ((rows0 + rows1) * (pitch / 16) + 255) / 256, most = 16ll * sm_count();
    return launch_next(vocab_align_kernel, dim3(static_cast<unsigned>(blocks < most ? blocks : most)), 256, 0, st, src0, rows0, src1, rows1, static_cast<uint4*>(dst0),
                       static_cast<uint4*>(dst1), bytes, pitch / 16);
}

// ---------------------------------------------------------------------------------------------- a few tokens
__device__ __forceinline__ int dot16(const uint4& u, const uint4& v, int sum) {
    sum = __dp4a(static_cast<int>(u.x), static_cast<int>(v.x), sum);
    sum = __dp4a(static_cast<int>(u.y), static_cast<int>(v.y), sum);
    sum = __dp4a(static_cast<int>(u.z), static_cast<int>(v.z), sum);
    return __dp4a(static_cast<int>(u.w), static_cast<int>(v.w), sum);
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}
__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// Up to THIN_TOKENS tokens: w passes once, at the rate of memory, and a 128-row tile of the tensor cores would hold next to nothing
// (1 x 2048 x 131072: 48 us, 0.85 of the measured rate; as tiles 64).  A block takes pieces of 64 classes, a warp eight of them side by side; the features lie in
// shared memory.  Rows of w that start off a 16-byte boundary are read from the boundary before, against a copy of the
// features that starts as far behind one (zeros around it): no copy of w is needed.
constexpr int THIN_TOKENS = 4, THIN_THREADS = 256, THIN_ROWS = PIECE / (THIN_THREADS / 32);
constexpr size_t THIN_MAX_SMEM = 100 * 1024;  // two blocks to an SM (4 x 2047 x 65536, one block of 131 KB: 115 us; through the tensor cores 94)
struct ThinParams {
    const int8_t* x; long long x_pitch;       // [rows][x_pitch]
    const int8_t* w; long long pitch;         // [classes][pitch], any address and pitch
    int F, rows, classes, pieces, entries;
    int step, copies, chunks;                 // rows of w start at (w + k step) mod 16; copies of the features; 16-byte chunks of a copy
    const int32_t* exp_x; const int32_t* exp_w; int temperature;
    int32_t* piece_max; uint32_t* piece_sum;
    const long long* index; int32_t* logit;
    int32_t* all_logits;                      // training: [rows][classes]; null: they are not kept
};
template <int T, bool ALIGNED>
__global__ void __launch_bounds__(THIN_THREADS) vocab_thin_kernel(const ThinParams p) {
    extern __shared__ __align__(16) uint8_t thin_smem[];
    __shared__ int32_t s_logit[T][PIECE];
    uint4* sx = reinterpret_cast<uint4*>(thin_smem);  // [copies][T][chunks]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uintptr_t begin = reinterpret_cast<uintptr_t>(p.w), end = begin + static_cast<uintptr_t>(p.classes - 1) * p.pitch + p.F;
    const int base = static_cast<int>(begin & 15);
    dependents_wait();
    dependents_start();
    // The tokens' copies: as they are where rows are multiples of 16 bytes from such an address; otherwise five aligned words and four
    // funnel shifts for a chunk, four chunks in flight, what lies outside the row zeroed (3 x 2046 x 20000: 43.7 us by bytes, 38.9 so).
    if (ALIGNED) for (int i = tid; i < T * p.chunks; i += THIN_THREADS) sx[i] = reinterpret_cast<const uint4*>(p.x)[i];
    const uintptr_t x_begin = reinterpret_cast<uintptr_t>(p.x), x_end = x_begin + static_cast<uintptr_t>(T - 1) * p.x_pitch + p.F;
    const int chunks = p.copies * T * p.chunks;
    constexpr int AT_ONCE = 4;
    for (int i0 = tid; !ALIGNED && i0 < chunks; i0 += AT_ONCE * THIN_THREADS) {
        uint32_t w[AT_ONCE][5], shift[AT_ONCE];
        int at[AT_ONCE];  // the feature in the chunk's first byte
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int i = i0 + u * THIN_THREADS;
            if (i >= chunks) break;
            const int c = i % p.chunks, t = i / p.chunks % T, copy = i / p.chunks / T;
            at[u] = c * 16 - ((base + copy * p.step) & 15);
            const uintptr_t from = x_begin + static_cast<uintptr_t>(t) * p.x_pitch + at[u], word0 = from & ~uintptr_t(3);
            shift[u] = static_cast<uint32_t>(from - word0) * 8;
            if (word0 >= x_begin && word0 + 20 <= x_end) {
#pragma unroll
                for (int k = 0; k < 5; ++k) w[u][k] = reinterpret_cast<const uint32_t*>(word0)[k];
            } else {
#pragma unroll
                for (int k = 0; k < 5; ++k) {
                    w[u][k] = 0;
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const uintptr_t byte = word0 + 4 * k + b;
                        if (byte >= x_begin && byte < x_end) w[u][k] |= static_cast<uint32_t>(*reinterpret_cast<const uint8_t*>(byte)) << (8 * b);
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int i = i0 + u * THIN_THREADS;
            if (i >= chunks) break;
            uint32_t o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int before = -at[u] - 4 * k, rest = p.F - at[u] - 4 * k;  // bytes in front of the row; bytes up to its end
                o[k] = __funnelshift_r(w[u][k], w[u][k + 1], shift[u]);
                if (before > 0) o[k] = before >= 4 ? 0u : o[k] & (0xFFFFFFFFu << (8 * before));
                if (rest < 4) o[k] = rest <= 0 ? 0u : o[k] & ((1u << (8 * rest)) - 1u);
            }
            sx[i] = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
    const ExpScale sc = exp_scale(*p.exp_x + *p.exp_w - p.temperature);
    __syncthreads();
    for (int piece = blockIdx.x; piece < p.pieces; piece += gridDim.x) {
        const int row0 = piece * PIECE + warp * THIN_ROWS;
        int sum[THIN_ROWS][T];
        uintptr_t at[THIN_ROWS];
        int copy[THIN_ROWS];
        bool inside = true;  // no chunk of these rows crosses the tensor's ends
#pragma unroll
        for (int r = 0; r < THIN_ROWS; ++r) {
            const uintptr_t start = begin + static_cast<uintptr_t>(min(row0 + r, p.classes - 1)) * p.pitch;  // rows behind the last: not looked at
            at[r] = start & ~uintptr_t(15);
            copy[r] = ALIGNED ? 0 : ((static_cast<int>(start & 15) - base) & 15) / p.step * T * p.chunks;
            inside = inside && at[r] >= begin && at[r] + 16 * static_cast<uintptr_t>(p.chunks) <= end;
#pragma unroll
            for (int t = 0; t < T; ++t) sum[r][t] = 0;
        }
        if (inside) {
#pragma unroll 1
            for (int c = lane; c < p.chunks; c += 32) {
                uint4 v[THIN_ROWS];
#pragma unroll
                for (int r = 0; r < THIN_ROWS; ++r) v[r] = reinterpret_cast<const uint4*>(at[r])[c];
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    uint4 u = sx[t * p.chunks + c];
#pragma unroll
                    for (int r = 0; r < THIN_ROWS; ++r) {
                        if (!ALIGNED) u = sx[copy[r] + t * p.chunks + c];
                        sum[r][t] = dot16(u, v[r], sum[r][t]);
                    }
                }
            }
        } else {
            for (int c = lane; c < p.chunks; c += 32)
#pragma unroll
                for (int r = 0; r < THIN_ROWS; ++r) {
                    uint32_t o[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int b = 0; b < 16; ++b) {
                        const uintptr_t a = at[r] + 16 * c + b;
                        if (a >= begin && a < end) o[b >> 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint8_t*>(a)) << (8 * (b & 3));
                    }
#pragma unroll
                    for (int t = 0; t < T; ++t) sum[r][t] = dot16(sx[copy[r] + t * p.chunks + c], make_uint4(o[0], o[1], o[2], o[3]), sum[r][t]);
                }
        }
#pragma unroll
        for (int r = 0; r < THIN_ROWS; ++r)
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const int v = __reduce_add_sync(0xFFFFFFFFu, sum[r][t]);
                if (lane == 0) s_logit[t][warp * THIN_ROWS + r] = v;
            }
        __syncthreads();
        if (warp < p.rows) {  // a warp to each token: the piece's statistics, and the wanted classes in it
            const int lim = p.classes - piece * PIECE;
            const int32_t a = lane < lim ? s_logit[warp][lane] : INT_MIN, b = lane + 32 < lim ? s_logit[warp][lane + 32] : INT_MIN;
            if (p.all_logits != nullptr) {
                int32_t* to = p.all_logits + static_cast<long long>(warp) * p.classes + static_cast<long long>(piece) * PIECE;
                if (lane < lim) to[lane] = a;
                if (lane + 32 < lim) to[lane + 32] = b;
            }
            const int32_t m = __reduce_max_sync(0xFFFFFFFFu, max(a, b));
            unsigned long long e = 0;
            if (lane < lim) e = exp_weight(static_cast<unsigned>(m) - static_cast<unsigned>(a), sc);
            if (lane + 32 < lim) e += exp_weight(static_cast<unsigned>(m) - static_cast<unsigned>(b), sc);
            e = warp_sum(e);
            if (lane == 0) {
                p.piece_max[static_cast<long long>(piece) * p.rows + warp] = m;
                p.piece_sum[static_cast<long long>(piece) * p.rows + warp] = static_cast<uint32_t>(e >> 6);
            }
            for (int k = lane; k < p.entries; k += 32) {
                const long long j = p.index[static_cast<long long>(warp) * p.entries + k] - static_cast<long long>(piece) * PIECE;
                if (j >= 0 && j < PIECE && j < lim) p.logit[warp * p.entries + k] = s_logit[warp][j];
            }
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------- row sums and losses
struct FinishParams {
    const int32_t* exp_x; const int32_t* exp_w; const int32_t* exp_top; int temperature;
    int rows, classes, pieces, entries, rows_log2;  // a block's rows: 2^rows_log2
    const int32_t* piece_max; const uint32_t* piece_sum;
    const long long* index; long long ignore;  // ignore: rows of this class are left out (a teacher's: every negative one is)
    const void* top; int top32;                // teacher's logits [rows][entries], int32 or int8; null: all on the one entry
    const int8_t* x; const int8_t* w; int F16; // for the wanted classes' logits; null: they lie in logit, [rows][entries]
    const int32_t* logit;
    float* loss;
    int4* row_stat; int* entry_err;            // training; entry_err [entries][rows], see one_entry
    int32_t* err_exp; uint32_t* clear[3];      // training: written and zeroed for the launches behind
    uint4* zero; long long zero_count;         // training: zeroed as well
    int round_mode;
    const unsigned long long* seed; unsigned rng_stream; unsigned long long rng_offset;
};
__device__ __forceinline__ double pow2(int e) { return __hiloint2double((1023 + max(-1022, min(1023, e))) << 20, 0); }
// Row sums, losses, and for training what vocab_kernel needs of each row.  Up to eight rows to a block: a thread takes every G-th
// piece of one of them, the first eight at once and into registers, so that a short vocabulary costs one trip to memory.
// ONE: a class to each row, finished by a thread; otherwise a warp to each row, its lanes to the entries.
constexpr int FINISH_HELD = 8;
template <bool ONE, bool TRAIN>
__global__ void __launch_bounds__(FINISH_THREADS) vocab_finish_kernel(const FinishParams p) {
    constexpr int WARPS = FINISH_THREADS / 32, MAX_ROWS = 8;
    __shared__ unsigned long long s_sum[WARPS][MAX_ROWS], s_loss_sum[WARPS][MAX_ROWS];
    __shared__ int32_t s_max[WARPS][MAX_ROWS], s_logit[MAX_ROWS][ONE ? 1 : MAX_ENTRIES];
    __shared__ unsigned s_share[ONE ? 1 : WARPS][ONE ? 1 : MAX_ENTRIES];
    __shared__ int s_class[ONE ? 1 : WARPS][ONE ? 1 : MAX_ENTRIES];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int RB = 1 << p.rows_log2, G = FINISH_THREADS >> p.rows_log2;
    const int r = tid & (RB - 1), g = tid >> p.rows_log2;
    const int row0 = static_cast<int>(blockIdx.x) << p.rows_log2, row = row0 + r;
    const bool there = row < p.rows;
    // The wanted classes' logits, a warp to four of a row's: of tensors that were there before the launch in front of this one passed its
    // own wait, so this one need not wait for it.  What a negative index or one behind the last class gets is not looked at.
    constexpr int AT_ONCE = ONE ? 1 : 4;
    if (p.x != nullptr) {
        const int groups = (p.entries + AT_ONCE - 1) / AT_ONCE, tasks = groups << p.rows_log2;
        for (int i = warp; i < tasks; i += WARPS) {
            const int k0 = (i >> p.rows_log2) * AT_ONCE, ri = i & (RB - 1);
            const long long t = row0 + ri;
            if (t >= p.rows) continue;
            const uint4 *a = reinterpret_cast<const uint4*>(p.x) + t * p.F16, *b[AT_ONCE];
            int sum[AT_ONCE];
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                const long long j = k0 + k < p.entries ? __ldcg(p.index + t * p.entries + k0 + k) : -1;
                b[k] = reinterpret_cast<const uint4*>(p.w) + (j >= 0 && j < p.classes ? j : 0) * p.F16;
                sum[k] = 0;
            }
#pragma unroll 2
            for (int c = lane; c < p.F16; c += 32) {
                uint4 v[AT_ONCE];
                const uint4 u = __ldcg(a + c);
#pragma unroll
                for (int k = 0; k < AT_ONCE; ++k) v[k] = __ldcg(b[k] + c);
#pragma unroll
                for (int k = 0; k < AT_ONCE; ++k) sum[k] = dot16(u, v[k], sum[k]);
            }
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                const int v = __reduce_add_sync(0xFFFFFFFFu, sum[k]);
                if (lane == 0 && k0 + k < p.entries) s_logit[ri][k0 + k] = v;
            }
        }
    }
    dependents_wait();
    dependents_start();
    if (p.x == nullptr)
        for (int i = tid; i < p.entries << p.rows_log2; i += FINISH_THREADS)
            if (row0 + (i & (RB - 1)) < p.rows) s_logit[i & (RB - 1)][i >> p.rows_log2] = p.logit[static_cast<long long>(row0 + (i & (RB - 1))) * p.entries + (i >> p.rows_log2)];

    int32_t hm[FINISH_HELD];
    uint32_t hs[FINISH_HELD];
#pragma unroll
    for (int u = 0; u < FINISH_HELD; ++u) {
        const int c = g + u * G;
        const bool in = there && c < p.pieces;
        const long long at = static_cast<long long>(c) * p.rows + row;
        hm[u] = in ? p.piece_max[at] : INT_MIN;
        hs[u] = in ? p.piece_sum[at] : 0u;
    }
    const int e = *p.exp_x + *p.exp_w - p.temperature;
    const long long mine = ONE && tid < RB && there ? p.index[row] : -1;
    if (p.err_exp != nullptr && blockIdx.x == 0 && tid == 0) { *p.err_exp = p.temperature - 7; *p.clear[0] = 0; *p.clear[1] = 0; *p.clear[2] = 0; }
    for (long long i = static_cast<long long>(blockIdx.x) * FINISH_THREADS + tid; i < p.zero_count; i += static_cast<long long>(gridDim.x) * FINISH_THREADS)
        p.zero[i] = make_uint4(0, 0, 0, 0);

    // the row's maximum over its pieces, then its sum relative to it
    int32_t m = hm[0];
#pragma unroll
    for (int u = 1; u < FINISH_HELD; ++u) m = max(m, hm[u]);
    if (there) {
#pragma unroll 8
        for (int c = g + FINISH_HELD * G; c < p.pieces; c += G) m = max(m, p.piece_max[static_cast<long long>(c) * p.rows + row]);
    }
    for (int o = RB; o < 32; o <<= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if (lane < RB) s_max[warp][lane] = m;
    __syncthreads();
    m = s_max[0][r];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) m = max(m, s_max[w][r]);
    const int32_t M = m;
    const ExpScale sc = exp_scale(e);
    const unsigned far = far_limit(e, sc);
    unsigned long long S = 0, L = 0;
#pragma unroll 1
    for (int u = 0; u < FINISH_HELD; ++u) {
        // (a loop around one copy of E: this code runs once, and what a thread block has to fetch of it takes longer than it runs)
        int32_t mu = hm[0]; uint32_t su = hs[0];
#pragma unroll
        for (int k = 1; k < FINISH_HELD; ++k) if (k == u) { mu = hm[k]; su = hs[k]; }
        if (g + u * G >= p.pieces) break;
        add_piece<TRAIN>(su, static_cast<unsigned>(M) - static_cast<unsigned>(mu), sc, far, &S, &L);
    }
    if (there) {
#pragma unroll 4
        for (int c = g + FINISH_HELD * G; c < p.pieces; c += G) {
            const long long at = static_cast<long long>(c) * p.rows + row;
            add_piece<TRAIN>(p.piece_sum[at], static_cast<unsigned>(M) - static_cast<unsigned>(p.piece_max[at]), sc, far, &S, &L);
        }
    }
    for (int o = RB; o < 32; o <<= 1) {
        if (TRAIN) S += __shfl_xor_sync(0xFFFFFFFFu, S, o);
        L += __shfl_xor_sync(0xFFFFFFFFu, L, o);
    }
    if (lane < RB) { s_sum[warp][lane] = S; s_loss_sum[warp][lane] = L; }
    __syncthreads();

    const double unit = pow2(e);
    if (ONE) {
        if (tid >= RB || !there) return;
        S = L = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) { S += s_sum[w][tid]; L += s_loss_sum[w][tid]; }
        const bool used = mine >= 0 && mine < p.classes && mine != p.ignore, wrong = !used && mine != p.ignore;
        const unsigned d = static_cast<unsigned>(M) - static_cast<unsigned>(s_logit[tid][0]);
        float loss = wrong ? __int_as_float(0x7FC00000) : 0.0f;
        if (used) loss = static_cast<float>(static_cast<double>(d) * unit + log(static_cast<double>(L) * pow2(-44)));
        p.loss[row] = loss;
        if (!TRAIN) return;
        const int n = 32 - __clzll(static_cast<long long>(S));
        const uint32_t R = static_cast<uint32_t>(((1ull << 63) - 1) / (S >> n)), sh = static_cast<uint32_t>(n - 3);
        int one = 0;
        if (used) {
            const int32_t v = static_cast<int32_t>(mul_hi(exp_weight(d, sc), R) >> sh) - (1 << 30);
            uint32_t rnd = 0;
            if (p.round_mode == ROUND_STOCHASTIC) rnd = random_word(*p.seed, p.rng_stream, (p.rng_offset + row) * static_cast<unsigned long long>((p.classes + 3) / 4 * 4) + static_cast<unsigned long long>(mine));
            one = one_entry(static_cast<int>(mine), narrow(v, 23, p.round_mode, rnd));
        }
        p.row_stat[row] = make_int4(M, used ? static_cast<int32_t>(R) : 0, static_cast<int32_t>(sh), one);
        return;
    }
    // a teacher's entries: a warp to each row
    const int i = warp, t = row0 + warp;
    if (i >= RB || t >= p.rows) return;
    unsigned long long Si = 0, Li = 0;
    int32_t Mi = INT_MIN;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) { Si += s_sum[w][i]; Li += s_loss_sum[w][i]; Mi = max(Mi, s_max[w][i]); }
    const long long first = static_cast<long long>(t) * p.entries;
    const int et = *p.exp_top - p.temperature;
    const ExpScale st = exp_scale(et);
    const auto teacher = [&](int k) {
        return p.top32 ? static_cast<const int32_t*>(p.top)[first + k] : static_cast<int32_t>(static_cast<const int8_t*>(p.top)[first + k]);
    };
    // which entries there are, and the teacher's largest
    bool any = false, wrong = false;
    int32_t best = INT_MIN;
    for (int k = lane; k < p.entries; k += 32) {
        const long long j = p.index[first + k];
        const bool used = j >= 0 && j < p.classes;
        wrong |= j >= p.classes;
        any |= used;
        s_class[warp][k] = used ? static_cast<int>(j) : -1;
        if (used) best = max(best, teacher(k));
    }
    any = __any_sync(0xFFFFFFFFu, any);
    wrong = __any_sync(0xFFFFFFFFu, wrong);
    best = __reduce_max_sync(0xFFFFFFFFu, best);
    unsigned long long total = 0;
    for (int k = lane; k < p.entries; k += 32) {
        const unsigned share = s_class[warp][k] >= 0 ? exp_weight(static_cast<unsigned>(best) - static_cast<unsigned>(teacher(k)), st) : 0u;
        s_share[warp][k] = share;
        total += share;
    }
    total = warp_sum(total);
    const double ln_l = log(static_cast<double>(Li) * pow2(-44)), ln_q = log(static_cast<double>(total) * pow2(-30)), teacher_unit = pow2(et);
    double loss = 0.0;
    for (int k = lane; k < p.entries; k += 32) {
        const unsigned share = s_share[warp][k];
        if (share == 0) continue;
        const double lnp = -(static_cast<double>(static_cast<long long>(Mi) - s_logit[i][k]) * unit + ln_l);
        const double lnq = -(static_cast<double>(static_cast<long long>(best) - teacher(k)) * teacher_unit + ln_q);
        loss += static_cast<double>(share) / static_cast<double>(total) * (lnq - lnp);
        s_share[warp][k] = static_cast<unsigned>((static_cast<unsigned long long>(share) << 30) / total);
    }
    loss = warp_sum(loss) * pow2(2 * p.temperature);
    const bool learns = any && !wrong;
    if (lane == 0) p.loss[t] = wrong ? __int_as_float(0x7FC00000) : any ? static_cast<float>(loss) : 0.0f;
    if (!TRAIN) return;
    const int n = 32 - __clzll(static_cast<long long>(Si));
    const uint32_t R = static_cast<uint32_t>(((1ull << 63) - 1) / (Si >> n)), sh = static_cast<uint32_t>(n - 3);
    if (lane == 0) p.row_stat[t] = make_int4(Mi, learns ? static_cast<int32_t>(R) : 0, static_cast<int32_t>(sh), 0);
    __syncwarp();
    const unsigned long long seed = p.round_mode == ROUND_STOCHASTIC ? *p.seed : 0;
    for (int k = lane; k < p.entries; k += 32) {
        const int j = s_class[warp][k];
        int& out = p.entry_err[static_cast<long long>(k) * p.rows + t];
        if (j < 0) { out = 0; continue; }
        int err = 0;
        if (learns) {
            unsigned q = 0;  // a class may be listed more than once
            for (int o = 0; o < p.entries; ++o) q += s_class[warp][o] == j ? s_share[warp][o] : 0u;
            const uint32_t E = exp_weight(static_cast<unsigned>(Mi) - static_cast<unsigned>(s_logit[i][k]), sc);
            const int32_t v = static_cast<int32_t>(mul_hi(E, R) >> sh) - static_cast<int32_t>(q);
            const unsigned long long at = (p.rng_offset + t) * static_cast<unsigned long long>((p.classes + 3) / 4 * 4) + j;
            err = narrow(v, 23, p.round_mode, p.round_mode == ROUND_STOCHASTIC ? random_word(seed, p.rng_stream, at) : 0u);
        }
        out = one_entry(j, err);
    }
}

// A teacher's entries in a piece of the vocabulary, over what vocab_kernel wrote there.  (Looked through by vocab_kernel's epilogue, every
// piece of 64 classes for itself, they cost 333 x 640 x 20011 with 50 entries 16 us more and won two with one.)
__global__ void __launch_bounds__(256) vocab_patch_kernel(const int* entries, long long n, int rows, int first, int count, int8_t* err, long long pitch) {
    dependents_wait();
    dependents_start();
    const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= n) return;
    const int w = entries[i], j = (w & 0x3FFFF) - first;
    if ((w & (1 << 23)) && j >= 0 && j < count) err[(i % rows) * pitch + j] = static_cast<int8_t>(w >> 24);
}

// ---------------------------------------------------------------------------------------------- a few tokens' way back
// Both products that lead back for the tokens of vocab_thin_kernel, from the logits it kept (4 T / F of w's bytes): w read once, the gradient written once, which is nearly all there is to do (an outer product of a few rows).  A thread
// owns four features and sixteen classes of a batch, whose w it fetches at once (stores in between would hold the later ones back);
// their errors with the features' tokens (dp4a over tokens) are the gradient, which leaves at once; with w (dp4a over classes) they add
// up to the features' error, which is added to e32 at the end.  Rows shorter than 1024 features leave room for several groups of
// sixteen classes in a block.  Training with one group and four classes at a time, and so: 2 x 256 x 89596 63.0 and 42.6 us, 1 x 64 x
// 131072 48.1 and 27.7, 1 x 2048 x 30000 91.4 and 77.5.  Rows that are no multiple of four are fetched in up to four parts; four classes at
// a time and four blocks an SM are ahead there (3 x 2046 x 20000: 120 us, sixteen at a time 136).  The tiles of umma_gemm_two, all epilogue
// here, are ahead from five tokens on.
constexpr int BACK_THREADS = 256, BACK_ROWS = 16, BACK_MIN_COLS = 32, BACK_MAX_GROUPS = BACK_THREADS / BACK_MIN_COLS;
struct BackParams {
    const int32_t* logits;                    // [T][V]
    const int8_t* x; const int8_t* w;         // rows of F bytes
    int T, F, V, F4;
    int cols_log2;                            // threads side by side along the features
    int32_t* e32; int32_t* g32; unsigned* g_max;
    const int32_t* exp_x; const int32_t* exp_w; int temperature;
    const int4* row_stat; const int* entries; int num_entries;
    int mode; const unsigned long long* seed; unsigned rng_stream; unsigned long long rng_offset;
};
// One class's error from its logit: what vocab_kernel computes, a value at a time.
__device__ __forceinline__ int8_t error_of(int32_t a, const int4& stat, const ExpScale& sc, const BackParams& p, int t, int v) {
    if ((stat.w & (1 << 23)) && (stat.w & 0x3FFFF) == v) return static_cast<int8_t>(stat.w >> 24);
    const uint32_t E = exp_weight(static_cast<unsigned>(stat.x) - static_cast<unsigned>(a), sc);
    const int32_t y = static_cast<int32_t>(mul_hi(E, static_cast<uint32_t>(stat.y)) >> stat.z);
    uint32_t rnd = 0;
    if (p.mode == ROUND_STOCHASTIC) rnd = random_word(*p.seed, p.rng_stream, (p.rng_offset + t) * static_cast<unsigned long long>((p.V + 3) / 4 * 4) + v);
    return narrow(y, 23, p.mode, rnd);
}
// VEC: features side by side that a thread loads and stores at once (4, or 2 or 1 where rows are no multiples of four)
constexpr int back_per_sm(int vec) { return vec == 4 ? 2 : 4; }
template <int NT, int VEC>
__global__ void __launch_bounds__(BACK_THREADS, back_per_sm(VEC)) vocab_back_thin_kernel(const BackParams p) {
    constexpr int AT_ONCE = VEC == 4 ? BACK_ROWS : 4;  // classes whose w is fetched together
    constexpr int MAX_ROWS = BACK_ROWS * BACK_MAX_GROUPS, TOKENS = 4, VALUES = MAX_ROWS * TOKENS / BACK_THREADS;
    __shared__ uint32_t s_tokens[MAX_ROWS];             // a class's errors, a byte to each token
    __shared__ uint32_t s_classes[MAX_ROWS / 4][TOKENS]; // a token's errors, four classes to a word
    __shared__ int s_entries[MAX_ENTRIES * TOKENS], s_acc[NT * 4][BACK_THREADS];
    __shared__ unsigned s_max[BACK_THREADS / 32];
    const int tid = threadIdx.x, cols = 1 << p.cols_log2, ct = tid & (cols - 1), group = tid >> p.cols_log2;
    const int rows_log2 = 4 + 8 - p.cols_log2, rows = 1 << rows_log2;  // classes of a batch: sixteen to each group
    static_assert(BACK_ROWS == 16 && BACK_THREADS == 256, "rows_log2");
    const int f0 = static_cast<int>(blockIdx.y) * 4 * cols;
    dependents_wait();
    dependents_start();
    const ExpScale sc = exp_scale(*p.exp_x + *p.exp_w - p.temperature);
    for (int i = tid; i < p.num_entries * p.T; i += BACK_THREADS) s_entries[i] = p.entries[i];  // [entries][T]
    int f[4];
    uint32_t xq[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[j] = f0 + j / VEC * (VEC * cols) + VEC * ct + j % VEC;
        xq[j] = 0;
#pragma unroll
        for (int k = 0; k < TOKENS; ++k)
            if (k < p.T && f[j] < p.F) xq[j] |= static_cast<uint32_t>(static_cast<uint8_t>(p.x[static_cast<long long>(k) * p.F + f[j]])) << (8 * k);
    }
    // a thread's errors of a batch: value u is class (tid + 256 u) % rows of token (tid + 256 u) / rows
    int4 stat[VALUES];
#pragma unroll
    for (int u = 0; u < VALUES; ++u) {
        const int t = (tid + u * BACK_THREADS) >> rows_log2;
        stat[u] = t < p.T ? p.row_stat[t] : make_int4(0, 0, 0, 0);
    }
    const auto logit = [&](int u, int v0) {
        const int i = tid + u * BACK_THREADS, t = i >> rows_log2, v = v0 + (i & (rows - 1));
        return t < p.T && v < p.V ? p.logits[static_cast<long long>(t) * p.V + v] : 0;
    };
    int acc[NT][4], hi = 0, lo = 0;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[t][j] = 0;
    const int batches = (p.V + rows - 1) >> rows_log2;
    int32_t a[VALUES];
#pragma unroll
    for (int u = 0; u < VALUES; ++u) a[u] = logit(u, static_cast<int>(blockIdx.x) << rows_log2);
    for (int batch = blockIdx.x; batch < batches; batch += gridDim.x) {
        const int v0 = batch << rows_log2, mine = v0 + group * BACK_ROWS;
        uint32_t row[AT_ONCE];
        const auto fetch = [&](int first) {
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                row[k] = 0;
                if (first + k < p.V) {
                    const int8_t* at = p.w + static_cast<long long>(first + k) * p.F;
#pragma unroll
                    for (int j = 0; j < 4; j += VEC)
                        if (f[j] < p.F) {
                            if (VEC == 4) row[k] = *reinterpret_cast<const uint32_t*>(at + f[j]);
                            else if (VEC == 2) row[k] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(at + f[j])) << (8 * j);
                            else row[k] |= static_cast<uint32_t>(static_cast<uint8_t>(at[f[j]])) << (8 * j);
                        }
                }
            }
        };
        if (AT_ONCE == BACK_ROWS) fetch(mine);
        __syncthreads();  // the batch before is done with the errors
#pragma unroll
        for (int u = 0; u < VALUES; ++u) {
            const int i = tid + u * BACK_THREADS, t = i >> rows_log2, r = i & (rows - 1);
            if (t >= TOKENS) break;
            const int8_t e = t < p.T && v0 + r < p.V ? error_of(a[u], stat[u], sc, p, t, v0 + r) : int8_t(0);
            reinterpret_cast<int8_t*>(s_tokens)[r * TOKENS + t] = e;
            reinterpret_cast<int8_t*>(s_classes)[(r >> 2) * (4 * TOKENS) + t * 4 + (r & 3)] = e;
            a[u] = logit(u, (batch + static_cast<int>(gridDim.x) < batches ? batch + static_cast<int>(gridDim.x) : batch) << rows_log2);
        }
        __syncthreads();
        if (p.num_entries > 0) {  // a teacher's classes
            for (int i = tid; i < p.num_entries * p.T; i += BACK_THREADS) {
                const int w = s_entries[i], t = i % p.T, r = (w & 0x3FFFF) - v0;
                if (!(w & (1 << 23)) || r < 0 || r >= rows) continue;
                reinterpret_cast<int8_t*>(s_tokens)[r * TOKENS + t] = static_cast<int8_t>(w >> 24);
                reinterpret_cast<int8_t*>(s_classes)[(r >> 2) * (4 * TOKENS) + t * 4 + (r & 3)] = static_cast<int8_t>(w >> 24);
            }
            __syncthreads();
        }
        if (f[0] >= p.F) continue;
#pragma unroll (AT_ONCE / 4)
        for (int rq = 0; rq < BACK_ROWS / 4; ++rq) {
            if (AT_ONCE != BACK_ROWS) fetch(mine + 4 * rq);
            // four classes of a feature to a word
            const uint32_t* four = row + (AT_ONCE == BACK_ROWS ? 4 * rq : 0);
            const uint32_t b0 = __byte_perm(four[0], four[1], 0x5140), b1 = __byte_perm(four[2], four[3], 0x5140);
            const uint32_t b2 = __byte_perm(four[0], four[1], 0x7362), b3 = __byte_perm(four[2], four[3], 0x7362);
            const uint32_t col[4] = {__byte_perm(b0, b1, 0x5410), __byte_perm(b0, b1, 0x7632), __byte_perm(b2, b3, 0x5410), __byte_perm(b2, b3, 0x7632)};
            const int rl = group * BACK_ROWS + 4 * rq;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int e = static_cast<int>(s_classes[rl >> 2][t]);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[t][j] = __dp4a(static_cast<int>(col[j]), e, acc[t][j]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (mine + 4 * rq + k >= p.V) break;
                const int e = static_cast<int>(s_tokens[rl + k]);
                int g[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) g[j] = __dp4a(static_cast<int>(xq[j]), e, 0);
                hi = __vimax3_s32(__vimax3_s32(hi, g[0], g[1]), g[2], g[3]);
                lo = __vimin3_s32(__vimin3_s32(lo, g[0], g[1]), g[2], g[3]);
                int32_t* to = p.g32 + static_cast<long long>(mine + 4 * rq + k) * p.F;
#pragma unroll
                for (int j = 0; j < 4; j += VEC)
                    if (f[j] < p.F) {
                        if (VEC == 4) *reinterpret_cast<int4*>(to + f[j]) = make_int4(g[0], g[1], g[2], g[3]);
                        else if (VEC == 2) *reinterpret_cast<int2*>(to + f[j]) = make_int2(g[j], g[j + 1]);
                        else to[f[j]] = g[j];
                    }
            }
        }
    }
    // the groups' sums, then one addition a feature and token
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) s_acc[t * 4 + j][tid] = acc[t][j];
    const unsigned m = __reduce_max_sync(0xFFFFFFFFu, max(static_cast<unsigned>(hi), static_cast<unsigned>(-lo)));
    if ((tid & 31) == 0) s_max[tid >> 5] = m;
    __syncthreads();
    if (group == 0) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                int sum = 0;
                for (int i = ct; i < BACK_THREADS; i += cols) sum += s_acc[t * 4 + j][i];
                if (t < p.T && f[j] < p.F && sum != 0) atomicAdd(p.e32 + static_cast<long long>(t) * p.F4 + f[j], sum);
            }
    }
    if (tid == 0) {
        unsigned largest = 0;
#pragma unroll
        for (int w = 0; w < BACK_THREADS / 32; ++w) largest = max(largest, s_max[w]);
        if (largest != 0) atomicMax(p.g_max, largest);
    }
}

// ---------------------------------------------------------------------------------------------- the error's narrowing
struct NarrowParams {
    const int32_t* e32; int F, F4, rows;      // [rows][F4], F of them written
    int8_t* out;                              // [rows][F]
    unsigned* max_word; int32_t* barrier;     // both zero before the first launch that finds the maximum
    int find, narrow;                         // find: max |e32| into its word; narrow: by it.  Both: a cooperative launch
    const int32_t* exp_a; const int32_t* exp_b; int32_t* exp_out;
    int bits, mode;
    const unsigned long long* seed; unsigned rng_stream; unsigned long long rng_offset;
    int32_t* status;
};
// err_calc (ti_torch.py:119-133) of an error that came in parts, so that nobody has seen its maximum yet.  A thread's first four words
// stay in registers over the barrier: a small error is read once, and its two passes cost one launch.
// CLUSTER: an error that one cluster of up to eight blocks holds whole; its maximum goes through their shared memory, and the launch
// need not be a cooperative one (whole training steps: 8 tokens, 256 features x 4096 classes 28.7 -> 25.5 us, 128 tokens, 1024 x 5000
// 35.3 -> 32.5).
constexpr int NARROW_HELD = 4, NARROW_CLUSTER = 8;
template <int THREADS, bool CLUSTER>
__global__ void __launch_bounds__(THREADS) vocab_narrow_kernel(const NarrowParams p) {
    __shared__ unsigned s_max[THREADS / 32], s_all[NARROW_CLUSTER];
    __shared__ int s_flag;
    if (CLUSTER) cluster_arrive();  // every block is there before one writes to it
    const int tid = threadIdx.x, per_row = p.F4 / 4;
    dependents_wait();
    dependents_start();
    const bool dense = p.F4 == p.F;
    const long long words = static_cast<long long>(p.rows) * per_row, step = static_cast<long long>(gridDim.x) * THREADS;
    const long long first = static_cast<long long>(blockIdx.x) * THREADS + tid;
    const int4* src = reinterpret_cast<const int4*>(p.e32);
    const auto load = [&](long long i) {
        int4 v = __ldcg(src + i);
        if (!dense) {
            const int left = p.F - static_cast<int>(i % per_row) * 4;  // what lies behind a row is anything
            if (left < 4) v.w = 0;
            if (left < 3) v.z = 0;
            if (left < 2) v.y = 0;
        }
        return v;
    };
    int4 held[NARROW_HELD];
#pragma unroll
    for (int u = 0; u < NARROW_HELD; ++u) held[u] = first + u * step < words ? load(first + u * step) : make_int4(0, 0, 0, 0);
    unsigned largest = 0;
    if (CLUSTER) {
        unsigned m = 0;
#pragma unroll
        for (int u = 0; u < NARROW_HELD; ++u) m = max(m, absmax4(held[u]));
        m = __reduce_max_sync(0xFFFFFFFFu, m);
        if ((tid & 31) == 0) s_max[tid >> 5] = m;
        __syncwarp();
        cluster_wait();
        __syncthreads();
        if (tid < 32) {
            m = __reduce_max_sync(0xFFFFFFFFu, tid < THREADS / 32 ? s_max[tid] : 0u);
            if (tid < static_cast<int>(gridDim.x)) st_cluster_u32(mapa_u32(smem_u32(s_all + blockIdx.x), tid), m);
            __syncwarp();
        }
        cluster_sync_all();
        for (int b = 0; b < static_cast<int>(gridDim.x); ++b) largest = max(largest, s_all[b]);
    } else if (p.find) {
        unsigned m = 0;
#pragma unroll
        for (int u = 0; u < NARROW_HELD; ++u) m = max(m, absmax4(held[u]));
        for (long long i = first + NARROW_HELD * step; i < words; i += step) m = max(m, absmax4(load(i)));
        m = __reduce_max_sync(0xFFFFFFFFu, m);
        if ((tid & 31) == 0) s_max[tid >> 5] = m;
        __syncthreads();
        if (tid == 0) {
#pragma unroll
            for (int w = 1; w < THREADS / 32; ++w) m = max(m, s_max[w]);
            if (m != 0) red_relaxed_max(p.max_word, m);
        }
        if (!p.narrow) return;
        if (!bounded_grid_barrier(p.barrier, static_cast<int>(gridDim.x), p.status, 6, &s_flag)) return;
    }
    bool zero;
    const int shift = shift_for(CLUSTER ? largest : __ldcg(p.max_word), CALC_ERR, p.bits, &zero);
    if (blockIdx.x == 0 && tid == 0) *p.exp_out = shift + *p.exp_a + *p.exp_b;
    const bool stochastic = p.mode == ROUND_STOCHASTIC && shift > 0;
    const unsigned long long seed = stochastic ? *p.seed : 0;
    const auto emit = [&](long long i, const int4& v) {
        const int x[4] = {v.x, v.y, v.z, v.w};
        if (dense) {
            uint32_t rnd[4] = {0, 0, 0, 0}, o = 0;
            if (stochastic) random_block(seed, p.rng_stream, (p.rng_offset >> 2) + i, rnd);
#pragma unroll
            for (int j = 0; j < 4; ++j) o |= static_cast<uint32_t>(static_cast<uint8_t>(narrow(x[j], shift, p.mode, rnd[j]))) << (8 * j);
            reinterpret_cast<uint32_t*>(p.out)[i] = o;
        } else {
            const long long row = i / per_row;
            const int f = static_cast<int>(i - row * per_row) * 4;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (f + j < p.F) {
                    const long long at = row * p.F + f + j;
                    p.out[at] = narrow(x[j], shift, p.mode, stochastic ? random_word(seed, p.rng_stream, p.rng_offset + at) : 0u);
                }
        }
    };
#pragma unroll
    for (int u = 0; u < NARROW_HELD; ++u) if (first + u * step < words) emit(first + u * step, held[u]);
    if constexpr (!CLUSTER) {
#pragma unroll 2
        for (long long i = first + NARROW_HELD * step; i < words; i += step) emit(i, load(i));
    }
}

// ---------------------------------------------------------------------------------------------- host side
template <int NT>
int launch_back_inst(BackParams p, cudaStream_t st) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.w);
    const int vec = p.F % 4 == 0 && at % 4 == 0 ? 4 : p.F % 2 == 0 && at % 2 == 0 ? 2 : 1;
    int cols = BACK_MIN_COLS;
    p.cols_log2 = 5;
    while (cols < BACK_THREADS && 4 * cols < p.F) { cols *= 2; ++p.cols_log2; }
    const int rows = BACK_ROWS * (BACK_THREADS / cols), y = (p.F + 4 * cols - 1) / (4 * cols), batches = (p.V + rows - 1) / rows, most = (back_per_sm(vec) * sm_count() + y - 1) / y;
    const dim3 grid(static_cast<unsigned>(batches < most ? batches : most), static_cast<unsigned>(y));
    const auto kernel = vec == 4 ? vocab_back_thin_kernel<NT, 4> : vec == 2 ? vocab_back_thin_kernel<NT, 2> : vocab_back_thin_kernel<NT, 1>;
    return launch_next(kernel, grid, BACK_THREADS, 0, st, p);
}
int launch_back(const BackParams& p, cudaStream_t st) {
    return p.T == 1 ? launch_back_inst<1>(p, st) : p.T == 2 ? launch_back_inst<2>(p, st) : launch_back_inst<THIN_TOKENS>(p, st);
}
// err_calc of the whole error; `summed`: its maximum is still to be found
int narrow_error(NarrowParams p, bool summed, cudaStream_t st) {
    const long long words = static_cast<long long>(p.rows) * (p.F4 / 4), blocks = (words + 1023) / 1024, most = 4ll * sm_count();
    const unsigned grid = static_cast<unsigned>(blocks < 1 ? 1 : blocks < most ? blocks : most);
    constexpr int WHOLE = 1024;
    if (summed && words <= static_cast<long long>(NARROW_CLUSTER) * WHOLE * NARROW_HELD) {
        unsigned size = 1;
        while (static_cast<long long>(size) * WHOLE * NARROW_HELD < words) size *= 2;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(size); cfg.blockDim = dim3(WHOLE); cfg.stream = st;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = size; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr; cfg.numAttrs = 2;
        return launched(cudaLaunchKernelEx(&cfg, vocab_narrow_kernel<WHOLE, true>, p));
    }
    if (summed && g_cooperative) {
        p.find = p.narrow = 1;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(grid); cfg.blockDim = dim3(256); cfg.stream = st;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeCooperative; attr[0].val.cooperative = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr; cfg.numAttrs = 2;
        const int e = launched_together(cudaLaunchKernelEx(&cfg, vocab_narrow_kernel<256, false>, p));
        if (e != LAUNCH_REFUSED) return e;
    }
    if (summed) {
        p.find = 1; p.narrow = 0;
        if (int e = launch_next(vocab_narrow_kernel<256, false>, dim3(grid), 256, 0, st, p)) return e;
    }
    p.find = 0; p.narrow = 1;
    return launch_next(vocab_narrow_kernel<256, false>, dim3(grid), 256, 0, st, p);
}

template <bool TWO, int WHAT, int BN>
int launch_vocab_inst(const CUtensorMap& a, const CUtensorMap& b, const VocabParams& p, cudaStream_t st) {
    using Cfg = VocabCfg<TWO, BN>;
    cudaError_t e = allow_shared<vocab_kernel<TWO, WHAT, BN>>(Cfg::SMEM_BYTES);
    if (e != cudaSuccess) return set_cuda_error(e);
    const int units = sm_count() * Cfg::PER_SM / (TWO ? 2 : 1), tiles = p.g.m_tiles * p.g.n_tiles, grid = tiles < units ? tiles : units;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(TWO ? 2 * grid : grid); cfg.blockDim = dim3(vocab_threads(BN)); cfg.dynamicSmemBytes = Cfg::SMEM_BYTES; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = TWO ? 2 : 1;
    return launched(cudaLaunchKernelEx(&cfg, vocab_kernel<TWO, WHAT, BN>, a, b, p));
}
template <bool TWO, int BN>
int launch_vocab(int what, const CUtensorMap& a, const CUtensorMap& b, const VocabParams& p, cudaStream_t st) {
    switch (what) {
        case ROUND_NEAREST: return launch_vocab_inst<TWO, ROUND_NEAREST, BN>(a, b, p, st);
        case ROUND_STOCHASTIC: return launch_vocab_inst<TWO, ROUND_STOCHASTIC, BN>(a, b, p, st);
        case ROUND_PSEUDO_STOCHASTIC: return launch_vocab_inst<TWO, ROUND_PSEUDO_STOCHASTIC, BN>(a, b, p, st);
        default: return launch_vocab_inst<TWO, VOCAB_STATS, BN>(a, b, p, st);
    }
}
// The tile of a launch: 256 columns of 128 rows (or of 256, to a pair of thread blocks), or 64 columns in up to three thread blocks to an SM,
// for launches whose last wave of wide tiles would be far from full.  Cycles: an epilogue of 256 columns, one and two of 64 on an SM; a
// 128-byte reduction block of each; the first tile's blocks lie in front of every epilogue.  A box that the rows' end cuts short takes the
// TMA unit 10 to 30 cycles a row.  48 x 256 x 4096 (64 SMs instead of 16): 11.8 -> 8.2 us.  In a graph, the loss in wide tiles and in
// narrow ones: 128 x 128 x 8000 9.6 and 7.2 us, 128 x 128 x 17664 10.5 and 9.3, 200 x 128 x 60000 34.0 and 31.3; with part of a box 200 x
// 80 x 60000 36.3 and 47.7, 200 x 400 x 17664 15.1 and 21.4; 32 x 128 x 17664 7.4 and 9.2.  A pair fetches half of w for each of its
// thread blocks, but computes a row tile for nothing where their number is odd: training on 777 x 1000 x 10007 took 91.6 us in pairs
// (three waves) and takes 78.5 in single blocks (two).
struct VocabTile { int bn; bool pair; };
// A warp reads the tensor-memory lanes of its place in a group of four, which are the places on the four schedulers: 32 tokens' rows in
// one quarter of a tile would leave all the work to one scheduler.  Up to 64 tokens lie in a tile twice, up to 32 four times, and
// every copy's warps see to their share of the columns (the loss, 1024 features x 30000 classes: 32 tokens 18.6 -> 13.8 us, 64 18.6 ->
// 14.6; 256 x 60000: 5 tokens 20.8 -> 13.4, 32 tokens 22.0 -> 17.4).
int vocab_copies(int T) { return T <= 32 ? 2 : T <= 64 ? 1 : 0; }
VocabTile vocab_tile(int T, int F, int count) {
    const int m128 = (T + 127) / 128, wide_epilogue = 10400 >> vocab_copies(T);
    const long long kb = (F + 127) / 128, sms = sm_count();
    const auto larger = [](long long a, long long b) { return a > b ? a : b; };
    const long long part = F % 128 != 0;  // the last box of a row is cut short
    const auto wide = [&](bool pair) {
        const long long tiles = static_cast<long long>(pair ? (m128 + 1) / 2 : m128) * ((count + VBN - 1) / VBN), units = pair ? sms / 2 : sms, load = kb * (pair ? 600 : 700);
        return load + part * 1000 + wide_epilogue + (tiles - 1) / units * larger(wide_epilogue, load + part * (pair ? 3200 : 5000));
    };
    const long long single_cost = wide(false), pair_cost = (g_two_cta & 1) && m128 >= 2 ? wide(true) : single_cost + 1, wide_cost = pair_cost < single_cost ? pair_cost : single_cost;
    const long long narrow = static_cast<long long>(m128) * ((count + 63) / 64), whole = narrow / (2 * sms), rest = narrow - whole * 2 * sms;
    const long long full = larger(vocab_copies(T) != 0 ? 6000 : 5800, 2 * (kb * 650 + part * 5400)), last = rest == 0 ? 0 : rest <= sms ? larger(4200, kb * 400) + part * 2500 : full;
    const long long narrow_cost = kb * 400 + whole * full + last;
    return narrow_cost < wide_cost ? VocabTile{64, false} : VocabTile{VBN, pair_cost < single_cost};
}
// x [T][pitch] times `count` rows of w [V][pitch] from p->first on
int run_vocab(int what, const int8_t* x, const int8_t* w, int T, int F, int pitch, int count, VocabParams* p, int32_t* status, cudaStream_t st) {
    const int m128 = (T + 127) / 128;
    const VocabTile tile = vocab_tile(T, F, count);
    const int bn = tile.bn;
    const bool pair = tile.pair;
    CUtensorMap ma, mb;
    uint64_t dims[2] = {static_cast<uint64_t>(F), static_cast<uint64_t>(T)}, str[1] = {static_cast<uint64_t>(pitch)};
    // a single row tile's box is no higher than its tokens (in eights): what the MMAs read of the other rows ends in rows nobody looks at
    const int a_rows = m128 == 1 ? (T + 7) / 8 * 8 : BLOCK_M;
    p->copies_log2 = vocab_copies(T);
    uint32_t box[2] = {128, static_cast<uint32_t>(a_rows)};
    if (int e = encode_map(&ma, x, false, 2, dims, str, box)) return e;
    dims[1] = count; box[1] = pair ? VBN / 2 : bn;
    if (int e = encode_map(&mb, w + static_cast<long long>(p->first) * pitch, false, 2, dims, str, box)) return e;
    GemmParams& g = p->g;
    g = GemmParams{};
    g.M = T; g.N = count; g.K = F; g.num_kb = (F + 127) / 128; g.splits = 1;
    g.m_tiles = pair ? (m128 + 1) / 2 : m128; g.n_tiles = (count + bn - 1) / bn;
    g.a_bytes = (a_rows << p->copies_log2) * ROW_BYTES; g.status = status;
    g.group_m = (static_cast<long long>(T) + count) * F > (48ll << 20) ? 8 : 0;  // as umma_gemm orders its tiles
    g.fd_mn = make_fastdiv(g.m_tiles * g.n_tiles); g.fd_n = make_fastdiv(g.n_tiles); g.fd_tw = make_fastdiv(1); g.fd_th = make_fastdiv(1);
    if (pair) return launch_vocab<true, VBN>(what, ma, mb, *p, st);
    return bn == 64 ? launch_vocab<false, 64>(what, ma, mb, *p, st) : launch_vocab<false, VBN>(what, ma, mb, *p, st);
}

size_t up(size_t v, size_t a) { return (v + a - 1) / a * a; }

template <int T>
int launch_thin_inst(const ThinParams& p, size_t smem, cudaStream_t st) {
    const bool aligned = p.copies == 1;
    cudaError_t e = aligned ? allow_shared<vocab_thin_kernel<T, true>>(THIN_MAX_SMEM) : allow_shared<vocab_thin_kernel<T, false>>(THIN_MAX_SMEM);
    if (e != cudaSuccess) return set_cuda_error(e);
    // one piece to a block, dealt out by the hardware, unless the block has copies of the features to lay out first
    const int most = sm_count() * (smem <= 48 * 1024 ? 4 : 2), grid = aligned || p.pieces < most ? p.pieces : most;
    return launch_next(aligned ? vocab_thin_kernel<T, true> : vocab_thin_kernel<T, false>, dim3(static_cast<unsigned>(grid)), THIN_THREADS, smem, st, p);
}
// How w's rows (of F bytes, `pitch` apart) lie to 16-byte boundaries, and the shared memory their features take.
size_t thin_layout(int T, int F, long long pitch, const int8_t* w, ThinParams* p) {
    p->step = 16;
    for (int g = 8; g >= 1; g >>= 1) if (pitch % (2 * g) != 0) p->step = g;
    p->copies = 16 / p->step;
    p->chunks = (F + 15 + (p->copies == 1 && reinterpret_cast<uintptr_t>(w) % 16 == 0 ? 0 : 15)) / 16;
    return static_cast<size_t>(p->copies) * T * p->chunks * 16;
}
int launch_thin(int T, const ThinParams& p, size_t smem, cudaStream_t st) {
    switch (T) {
        case 1: return launch_thin_inst<1>(p, smem, st);
        case 2: return launch_thin_inst<2>(p, smem, st);
        case 3: return launch_thin_inst<3>(p, smem, st);
        default: return launch_thin_inst<4>(p, smem, st);
    }
}

// The workspace of a call, from the first 32-byte boundary on: vocab_kernel stores a row's errors 32 bytes at a time.
constexpr size_t SCRATCH_ALIGN = 32, SCRATCH_SLACK = SCRATCH_ALIGN - 16;  // a caller's is 16-byte aligned
struct VocabPlan {
    int pieces, pitch, piece;   // row pitch of the operands; classes whose errors are in the workspace at a time
    size_t max_at, sum_at, stat_at, logit_at, entry_at, err_at, e32_at, word_at, x_at, w_at, logits_at, bytes;
};
// Errors in the workspace at a time.  Pieces of 37 column tiles: 148 SMs are 74 pairs of thread blocks, so the errors' tiles and the weight
// gradient's come in whole waves where the tokens, or the features, fill an even number of 256-row tiles.
constexpr long long ERR_BYTES = 96ll << 20;
constexpr int PIECE_TILES = 37;
int vocab_piece(int T, int V) {
    const long long whole = (V + VBN - 1) / VBN, most = ERR_BYTES / VBN / T;  // column tiles
    const long long tiles = most >= whole ? whole : most >= PIECE_TILES ? most / PIECE_TILES * PIECE_TILES : most < 1 ? 1 : most;
    return static_cast<int>(tiles) * VBN;
}
bool thin_serves(int T, int F) { ThinParams t{}; return T <= THIN_TOKENS && thin_layout(T, F, F, nullptr, &t) + 16 * 16 * T <= THIN_MAX_SMEM; }
VocabPlan vocab_plan(int T, int F, int V, int entries, bool train) {
    VocabPlan p{};
    p.pieces = (V + PIECE - 1) / PIECE;
    p.pitch = (F + 15) / 16 * 16;
    p.piece = vocab_piece(T, V);
    size_t at = 0;
    const auto take = [&](size_t n) { const size_t here = at; at = up(at + n, 256); return here; };
    const size_t t = T, k = entries;
    p.max_at = take(4 * t * p.pieces);
    p.sum_at = take(4 * t * p.pieces);
    const bool thin = thin_serves(T, F);
    if (thin) p.logit_at = take(4 * t * k);
    p.word_at = take(16);
    if (p.pitch != F && !thin) { p.x_at = take(t * p.pitch); p.w_at = take(static_cast<size_t>(V) * p.pitch); }
    if (train) {
        p.stat_at = take(16 * t);
        p.entry_at = take(4 * t * k);
        if (thin) p.logits_at = take(4 * t * V);
        else p.err_at = take(t * p.piece);
        p.e32_at = take(4 * t * up(F, 4));
    }
    p.bytes = at + SCRATCH_SLACK;
    return p;
}

bool vocab_sizes_ok(long long T, long long F, long long V, long long entries) {
    return T > 0 && F > 0 && V > 0 && entries > 0 && T < (1 << 17) && F < (1 << 17) && V <= (1 << 18) && entries <= MAX_ENTRIES;
}
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace niti

using namespace niti;

extern "C" int niti_vocab_supported(int T, int F, int V, int entries) { return vocab_sizes_ok(T, F, V, entries) ? 1 : 0; }

extern "C" size_t niti_vocab_scratch_bytes(int T, int F, int V, int entries, int train) {
    return vocab_sizes_ok(T, F, V, entries) ? vocab_plan(T, F, V, entries, train != 0).bytes : 0;
}

extern "C" int niti_vocab_piece(int T, int V) { return T > 0 && V > 0 ? vocab_piece(T, V) : 0; }

extern "C" int niti_vocab_loss_i8(const niti_vocab_args* a, void* stream) {
    if (a == nullptr) return NITI_ERR_BAD_ARG;
    const bool train = a->g32 != nullptr;
    if (!(a->x && a->exp_x && a->w && a->exp_w && a->index && a->loss && a->scratch && a->T > 0 && a->F > 0 && a->V > 0 && a->entries > 0))
        return NITI_ERR_BAD_ARG;
    if ((a->top == nullptr) != (a->exp_top == nullptr) || (a->top == nullptr && a->entries != 1)) return NITI_ERR_BAD_ARG;
    if (train && !(a->e8 && a->exp_err && a->grad_maxabs)) return NITI_ERR_BAD_ARG;
    if (train && (!aligned16(a->e8) || !aligned16(a->g32))) return NITI_ERR_BAD_ARG;
    if (train && (a->bits < 1 || a->bits > 7)) return NITI_ERR_BAD_ARG;
    if (train && (a->loss_round < 0 || a->loss_round > 2 || a->err_round < 0 || a->err_round > 2 ||
                  (a->seed == nullptr && (a->loss_round == ROUND_STOCHASTIC || a->err_round == ROUND_STOCHASTIC))))
        return NITI_ERR_BAD_ARG;
    if (!vocab_sizes_ok(a->T, a->F, a->V, a->entries) || a->temperature_log2 < -30 || a->temperature_log2 > 30) return NITI_ERR_UNSUPPORTED;
    const int T = a->T, F = a->F, V = a->V, K = a->entries;
    const VocabPlan pl = vocab_plan(T, F, V, K, train);
    if (!aligned16(a->scratch) || a->scratch_bytes < pl.bytes) return NITI_ERR_SCRATCH;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    char* ws = reinterpret_cast<char*>(up(reinterpret_cast<uintptr_t>(a->scratch), SCRATCH_ALIGN));

    // operands whose rows are no multiples of 16 bytes go through copies that are
    const int8_t *x = a->x, *w = a->w;
    const bool thin = thin_serves(T, F);
    if (pl.pitch != F && !thin) {
        x = reinterpret_cast<int8_t*>(ws + pl.x_at);
        w = reinterpret_cast<int8_t*>(ws + pl.w_at);
        if (int e = align_rows(a->x, T, ws + pl.x_at, a->w, V, ws + pl.w_at, F, pl.pitch, st)) return e;
    } else if (pl.pitch == F && (!aligned16(x) || !aligned16(w))) {
        return NITI_ERR_BAD_ARG;
    }

    VocabParams vp{};
    vp.exp_x = a->exp_x; vp.exp_w = a->exp_w; vp.temperature = a->temperature_log2;
    vp.rows = T; vp.first = 0; vp.classes = V;
    vp.piece_max = reinterpret_cast<int32_t*>(ws + pl.max_at); vp.piece_sum = reinterpret_cast<uint32_t*>(ws + pl.sum_at);
    const long long* index = reinterpret_cast<const long long*>(a->index);
    int32_t* logit = reinterpret_cast<int32_t*>(ws + pl.logit_at);
    const long long wanted = static_cast<long long>(T) * K;
    if (thin) {
        ThinParams tp{};
        tp.x = x; tp.w = w; tp.x_pitch = tp.pitch = F;
        if (train) tp.all_logits = reinterpret_cast<int32_t*>(ws + pl.logits_at);
        tp.F = F; tp.rows = T; tp.classes = V; tp.pieces = pl.pieces; tp.entries = K;
        tp.exp_x = a->exp_x; tp.exp_w = a->exp_w; tp.temperature = a->temperature_log2;
        tp.piece_max = vp.piece_max; tp.piece_sum = vp.piece_sum; tp.index = index; tp.logit = logit;
        const size_t smem = thin_layout(T, F, tp.pitch, w, &tp);
        if (int e = launch_thin(T, tp, smem, st)) return e;
    } else if (int e = run_vocab(VOCAB_STATS, x, w, T, F, pl.pitch, V, &vp, a->status, st)) {
        return e;
    }

    FinishParams fp{};
    fp.exp_x = a->exp_x; fp.exp_w = a->exp_w; fp.exp_top = a->exp_top; fp.temperature = a->temperature_log2;
    fp.rows = T; fp.classes = V; fp.pieces = pl.pieces; fp.entries = K;
    fp.rows_log2 = T >= 2048 ? 3 : T >= 1024 ? 2 : T >= 256 ? 1 : 0;  // two to four blocks an SM, up to eight words of a piece: a sector
    fp.piece_max = vp.piece_max; fp.piece_sum = vp.piece_sum;
    fp.index = index; fp.ignore = a->ignore_index; fp.top = a->top; fp.top32 = a->top_is_int32; fp.logit = logit; fp.loss = a->loss;
    if (!thin) { fp.x = x; fp.w = w; fp.F16 = pl.pitch / 16; }
    int32_t* words = reinterpret_cast<int32_t*>(ws + pl.word_at);  // {exponent of the logits' error, max |e32|, barrier}
    // e32 (+)= err w and g32 = err^T x of a piece of the vocabulary
    const int F4 = static_cast<int>(up(F, 4));
    int32_t* e32 = reinterpret_cast<int32_t*>(ws + pl.e32_at);
    unsigned* e32_max = reinterpret_cast<unsigned*>(words + 1);
    int8_t* err = reinterpret_cast<int8_t*>(ws + pl.err_at);
    GemmCall to_x{}, to_w{};
    const auto piece_calls = [&](int v0, int count) {
        to_x = GemmCall{err, w + static_cast<long long>(v0) * pl.pitch, e32, e32_max, T, F, count, 0, 0, 1, pl.piece, pl.pitch, F4, v0 > 0, a->status};
        to_w = GemmCall{err, x, a->g32 + static_cast<long long>(v0) * F, a->grad_maxabs, count, F, T, 1, 0, 1, pl.piece, pl.pitch, F, 0, a->status};
        const GemmTwoPlan plan = umma_gemm_two_plan(to_x, to_w);
        if (plan.splits > 1) to_x.accumulate = 1;
        if (plan.splits > 1 || pl.piece < V) to_x.maxabs = nullptr;  // a part's maximum is not the error's, which may be smaller
        return plan;
    };
    GemmTwoPlan plan{};
    if (train && !thin) plan = piece_calls(0, pl.piece < V ? pl.piece : V);
    const bool summed = train && (thin || plan.splits > 1 || pl.piece < V);  // e32 comes in several parts
    if (train) {
        fp.row_stat = reinterpret_cast<int4*>(ws + pl.stat_at);
        fp.entry_err = reinterpret_cast<int*>(ws + pl.entry_at);
        fp.err_exp = words; fp.clear[0] = reinterpret_cast<uint32_t*>(words + 1); fp.clear[1] = reinterpret_cast<uint32_t*>(words + 2); fp.clear[2] = a->grad_maxabs;
        if (thin || plan.splits > 1) { fp.zero = reinterpret_cast<uint4*>(ws + pl.e32_at); fp.zero_count = static_cast<long long>(T) * F4 / 4; }
        fp.round_mode = a->loss_round;
        fp.seed = reinterpret_cast<const unsigned long long*>(a->seed); fp.rng_stream = a->loss_stream; fp.rng_offset = a->sample_offset;
    }
    const int rb = 1 << fp.rows_log2;
    const auto finish = a->top == nullptr ? (train ? vocab_finish_kernel<true, true> : vocab_finish_kernel<true, false>)
                                          : (train ? vocab_finish_kernel<false, true> : vocab_finish_kernel<false, false>);
    if (int e = launch_next(finish, dim3(static_cast<unsigned>((T + rb - 1) / rb)), FINISH_THREADS, 0, st, fp)) return e;
    if (!train) return NITI_OK;

    vp.row_stat = fp.row_stat;
    vp.err = err; vp.err_pitch = pl.piece;
    vp.seed = fp.seed; vp.rng_stream = a->loss_stream; vp.rng_offset = a->sample_offset;
    if (thin) {
        BackParams bp{};
        bp.logits = reinterpret_cast<const int32_t*>(ws + pl.logits_at);
        bp.x = x; bp.w = w; bp.T = T; bp.F = F; bp.V = V; bp.F4 = F4;
        bp.e32 = e32; bp.g32 = a->g32; bp.g_max = a->grad_maxabs;
        bp.exp_x = a->exp_x; bp.exp_w = a->exp_w; bp.temperature = a->temperature_log2;
        bp.row_stat = fp.row_stat; bp.mode = a->loss_round;
        if (a->top != nullptr) { bp.entries = fp.entry_err; bp.num_entries = K; }
        bp.seed = fp.seed; bp.rng_stream = a->loss_stream; bp.rng_offset = a->sample_offset;
        if (int e = launch_back(bp, st)) return e;
    }
    for (int v0 = 0; v0 < V && !thin; v0 += pl.piece) {
        const int count = V - v0 < pl.piece ? V - v0 : pl.piece;
        vp.first = v0;
        if (int e = run_vocab(a->loss_round, x, w, T, F, pl.pitch, count, &vp, a->status, st)) return e;
        if (a->top != nullptr) {
            if (int e = launch_next(vocab_patch_kernel, dim3(static_cast<unsigned>((wanted + 255) / 256)), 256, 0, st, fp.entry_err, wanted, T, v0, count, vp.err, vp.err_pitch)) return e;
        }
        if (v0 > 0) plan = piece_calls(v0, count);
        if (int e = umma_gemm_two(to_x, to_w, plan, st)) return e;
    }
    NarrowParams np{};
    np.e32 = e32; np.F = F; np.F4 = F4; np.rows = T; np.out = a->e8;
    np.max_word = e32_max; np.barrier = words + 2;
    np.exp_a = words; np.exp_b = a->exp_w; np.exp_out = a->exp_err;
    np.bits = a->bits; np.mode = a->err_round;
    np.seed = fp.seed; np.rng_stream = a->err_stream; np.rng_offset = a->sample_offset * static_cast<unsigned long long>(F);
    np.status = a->status;
    return narrow_error(np, summed, st);
}
