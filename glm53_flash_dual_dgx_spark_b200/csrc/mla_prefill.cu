// Causal MLA attention of a ragged batch of new tokens over the NVFP4 paged pool.
//
//   x[r, t] = bmm1_scale (q[r, :512] . k[t] + q[r, 512:] . k_rope[t]),  t <= L - n + i(r)
//   out[r] = bmm2_scale sum_t softmax(x[r])_t k[t],   lse[r] = log sum_t exp(x[r, t])
//
// With a window W and sinks S only t > p - W or t < S counts, p = L - n + i(r).  What follows is the form
// without; the windowed one (kDirect) differs in the tiles of a unit (unit_gap), the image, Q and how
// the MMA warp learns of the next part, and calls of few rows have kernels of their own at the end.
//
// Rows r = (new token i, head) of one sequence share the latent rows k, which are both keys and
// values, so the kernel is two chained matrix products over 128 rows: S = Q K^T (512 or 576 deep)
// and O = P K (512 wide), about 2.2 kFLOP per row and token, on the tensor cores.
//
// A unit is 128 rows of one sequence.  It is run by a pair of CTAs (a cluster of two) with
// cta_group::2 MMAs of M = 128, 64 rows in each CTA.  What decides that is tensor memory: fp32 O of
// 64 rows x 512 is half of an SM's 256 KB, and S of two tiles the other half.  M = 128 over a pair
// runs at the full rate (measured 32 / 64 cycles for N = 128 / 256 at K = 16, 4090 multiply-adds a
// cycle and SM): each CTA supplies its rows of A and half of B.  A single CTA with 64 rows on N
// takes 48 cycles where 32 are due, because its operands saturate shared memory.
//   QK: B = tokens: CTA c holds tokens [128 c, 128 c + 128) of a 256-token tile
//   PV: B = latent dims: CTA c holds dims [256 c, 256 c + 256) of all 256 tokens
// in 16 KB ring stages (64 dims x 128 tokens, or 128 dims x 64 tokens), each 128 rows of 128 bytes,
// 128-byte swizzled, and four MMAs of 64 cycles.
//
// The stages are bulk copies from an image of the context in the workspace: a kernel before the
// attention dequantises every token once, into the very bytes of the stages (1,152 a token).  A pair
// needs every latent byte twice (K and V lie in different CTAs), and 64 heads make a unit of every
// two new tokens, so dequantising in the attention kernel repeats the work once per unit and twice
// in it: producer warps that did so held a tile to 13,000 cycles (issue slots), and a batch of single
// tokens gained nothing by them.  Copies from L2 reach 70 bytes a cycle and SM with two warps issuing
// (46 with one).
//
// What bounds it: a tile's 17 stages are 4,352 cycles of MMAs and, at 40 KB written and read each,
// 5,440 cycles of shared memory; it measures 5,800.  2,048 new tokens x 64 heads over 16,384: 3.2 ms
// in a short run (1.37 PFLOP/s), 3.5 ms back to back, where the GPU is at its power limit (1.25
// PFLOP/s; a large library product sustains 1.39 there).  A part's first tile and its epilogue add
// about 8,700 cycles.
//
// The work of a call, all (unit, tile) pairs in order and one and a half more per unit, is cut into
// one equal range per CTA pair, so that no pair waits for another's longer sequence; a unit cut
// by a range's end leaves its parts in the workspace for the combine kernel.  The ranges come from
// the device-side lengths in closed form, in every CTA.
//
// Dims are permuted within each half h of the latent: column 8 p + e of dim atom 4 h + s is dim
// 256 h + 32 p + 8 s + e, so that 16 code bytes (32 dims) of a row give 16 bytes to each of four
// atoms; the queries and the output use the same order.
//
// Numbers: a code times its e4m3 scale is exact in fp16, q is scaled per row by a power of two and
// then exact in fp16 (but for parts below 2^-35 of the row's largest), the rope part stays bf16;
// products accumulate in fp32 (beside a rope part 2^50 times larger, the latent part keeps what is
// above 2^-85 of it).  Probabilities are fp16 (11 bits; bf16 would add as much error as the output's
// own rounding), their sums fp32 and of the unrounded values.  A row's reference is 2^7 below its
// maximum and moves only when a tile exceeds that by 2^8, so O is rarely rescaled, P
// stays at or below 2^15 (fp16's largest is 65504), and a long flat tail under one high score keeps
// its mass: what fp16 rounds away of a probability is at most 2^-32 of the largest (with P = 1 at the
// maximum it is 2^-25, and 131,072 tokens at exp(-18) of one score lost all of theirs).
//
// Warps: 0-7 softmax (a row's 256 scores over four of them) and epilogue, 8-11 Q, 12 issues the
// MMAs (in the leading CTA), 13-14 image copies, 15 hands landed copies to the leader.  Every wait is
// bounded (common.cuh).
#include <math.h>

#include "../../include/nvfp4kv_serving.h"
#include "abi_common.h"
#include "common.cuh"
#include "decode_shared.h"

namespace nvfp4kv {
namespace {

constexpr int kRope = NVFP4KV_ROPE;
// The kernels' forms.  kAll: every token up to a row's own.  kDirect: a window and sinks; units are short,
// so Q stays bf16 and goes from q straight into its operand (converted as in kAll, it was what they waited
// for: 10,000 cycles of 32,600 a unit of three tiles), and the image holds every latent twice, in bf16
// for QK and in fp16 for PV.  Without a power of two per row, products of the latent part stay within fp32 for
// queries up to 2^106 (values up to 2,688, 512 of them) and keep all their bits down to 2^-92.
enum Form { kAll, kDirect };
constexpr int kDim = kLatent + kRope;
constexpr int kUnitRows = 128;                  // query rows of a unit
constexpr int kCtaRows = 64;
constexpr int kTile = 256;                      // tokens per tile
constexpr int kStages = 7;
constexpr int kStageBytes = 16384;              // 128 rows x 128 B
constexpr int kVStages = 8;                     // V stages of a tile: 4 x 64 tokens x 2 x 128 dims a CTA
constexpr int kSoftmaxWarps = 8, kQWarp0 = 8, kQWarps = 4, kMmaWarp = 12, kCopyWarp0 = 13, kRelayWarp = 15;
constexpr int kThreads = 16 * 32;
constexpr uint32_t kRegsLaunch = 128, kRegsSoftmax = 160, kRegsQ = 128, kRegsCtl = 64;
constexpr int kQRows = 4;                       // rows of Q a warp converts at a time
static_assert(256 * kRegsSoftmax + 128 * kRegsQ + 128 * kRegsCtl <= kThreads * kRegsLaunch,
              "the register split stays within what the block is launched with");
constexpr float kRescaleLog2 = 8.0f;             // how far scores may pass the maximum that set the reference,
constexpr float kTopLog2 = 7.0f;                // and log2 of P there
constexpr int kMaxPairs = 128;
constexpr int kImageTok = 128;                  // tokens of an image block
constexpr int kImagePieces = kImageTok / 32;    // a block of the image kernel does 32 at a time

constexpr int kQBytes = 9 * kCtaRows * 128;
constexpr int SM_Q = 0;                                      // 9 dim atoms x [64 rows x 128 B]
constexpr int SM_P = SM_Q + 9 * kCtaRows * 128;              // 4 token atoms x [64 rows x 128 B]
constexpr int SM_RING = SM_P + 4 * kCtaRows * 128;
constexpr int SM_RED = SM_RING + kStages * kStageBytes;      // 2 x 4 x 64 f32: row maxima of the token quarters
constexpr int SM_LSUM = SM_RED + 2 * 4 * 64 * 4;             // 4 x 64 f32
constexpr int SM_QS = SM_LSUM + 4 * 64 * 4;                  // 4 x 64 f32: score factor (log2 units) of a row
constexpr int SM_FLAGS = SM_QS + 4 * 64 * 4;                 // [0] TMEM base, [1] abort
constexpr int SM_WORK = SM_FLAGS + 16;                       // a Work per warp, and one with the range's first part
constexpr int kWorkBytes = 192;
constexpr int SM_BARS = SM_WORK + (kThreads / 32 + 1) * kWorkBytes;
constexpr int B_FULL = 0;                      // [kStages] leader: stage landed in both CTAs
constexpr int B_EMPTY = B_FULL + kStages;      // [kStages] both: the MMAs have read the stage
constexpr int B_LAND = B_EMPTY + kStages;      // [kStages] own: an image copy landed
constexpr int B_S_FULL = B_LAND + kStages;     // [2] both: S of a tile complete
constexpr int B_S_FREE = B_S_FULL + 2;         // [2] leader: S read by both CTAs
constexpr int B_P_FULL = B_S_FREE + 2;         // leader: P written in both CTAs
constexpr int B_PV_DONE = B_P_FULL + 1;        // both: O stable, P free
constexpr int B_Q_FULL = B_PV_DONE + 1;        // leader: Q written in both CTAs
constexpr int B_Q_FREE = B_Q_FULL + 1;         // both: the last QK of a part complete
constexpr int B_Q_LAND = B_Q_FREE + 1;         // own: Q copied
constexpr int B_O_FREE = B_Q_LAND + 1;         // leader: O read by both CTAs
constexpr int B_DRAIN = B_O_FREE + 1;          // both: every MMA complete
constexpr int kNumBars = B_DRAIN + 1;
constexpr int kSmemBytes = SM_BARS + kNumBars * 8 + 1024;    // slack to align the base
static_assert(SM_BARS % 8 == 0 && kSmemBytes <= 232448, "shared memory budget");

// Tensor memory: S of two tiles (lane l < 64: row l, tokens 0..127; lane 64 + l: row l, tokens
// 128..255) and O in two blocks n (lane l < 64: row l, latent half 0; lane 64 + l: half 1; column
// 64 a + 8 p + e of block n: dim 32 p + 16 n + 8 a + e of the half).
constexpr uint32_t kTS = 0, kTO = 256, kTmemCols = 512;

// A part of a unit that another pair's part completes: what the combine kernel reads.
struct __align__(16) PartInfo {
    int32_t used, head, tail, pad;
    int32_t first, rows, block, pad2;
};

struct PrefillParams {
    const __nv_bfloat16* q;
    int64_t q_st, q_sh;
    const uint8_t* pool;
    const uint16_t* rope;
    int64_t num_pages;
    const int32_t* tables;
    int64_t tables_stride;
    const int32_t* cu;
    const int32_t* seq_lens;
    int batch, total_q, heads, page_shift, max_q_len, max_seq_len;
    int window, sinks;         // position p sees t > p - window and t < sinks (window 0: every t <= p)
    int sink_rows, max_tiles;  // sinks rounded up to 64; tiles of a unit far into its sequence
    uint32_t heads_magic;      // ceil(2^32 / heads)
    int pairs;
    float scale_log2, out_scale;
    float factor;              // kDirect: what turns a score into log2 units, and what it is turned by before that
    float turn;                // (1, -1 for a negative scale, 0 for none)
    __nv_bfloat16* out;
    int64_t o_st, o_sh;
    float* lse;
    PartInfo* parts;    // [pairs][2]: the range's first part of a unit, and its last one
    float* part_ml;     // [pairs][2][128][2]: reference (log2 units), sum
    float* part_o;      // [pairs][2][64 chunks of 8 dims][128 rows][8]
    uint8_t* q_scratch; // [pairs][2 CTAs][kQBytes]: the next part's Q
    uint8_t* image;     // [blocks][8 or 9 atoms; kDirect: and 8 for PV][128 tokens x 128 B]
    uint32_t* image_bits;   // [blocks][8]: 128 bits of tokens that exist, 128 of those that hold a NaN
    int32_t* err;
};

// ------------------------------------------------------------------ pair (cta_group::2) wrappers
__device__ __forceinline__ void pair_tmem_alloc(uint32_t smem_dst, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "r"(ncols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void pair_mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// Arrive on the barrier at this shared address in both CTAs once every MMA issued so far completes.
__device__ __forceinline__ void pair_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
}
// mbar_wait whose polls sleep until the phase completes, or for about 20 us.
__device__ __forceinline__ bool try_wait_asleep(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity), "r"(20000u) : "memory");
    return ok != 0;
}
// Whether the phase has completed, without waiting.
__device__ __forceinline__ bool test_phase(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* err) {
    if (try_wait_asleep(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    while (!try_wait_asleep(bar, parity)) {
        if (*abort_flag) return false;
        if (globaltimer_ns() - t0 > NVFP4KV_WAIT_TIMEOUT_NS) {
            *abort_flag = 1;
            set_error(err, NVFP4KV_DEVERR_TIMEOUT);
            return false;
        }
    }
    return true;
}
// Arrive on the leading CTA's barrier.  What the arrival publishes is this CTA's own shared and
// tensor memory, ordered before it by fence.proxy.async or tcgen05.fence and read by the tensor
// core only, so the plain (CTA-scoped) release does; a cluster-scoped one is a full fence that
// takes about 900 cycles (measured: one per stage held the kernel to 0.38 of its rate).
__device__ __forceinline__ void leader_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_map(bar, 0)) : "memory");
}
// One 32-byte store (dst 32-byte aligned).
__device__ __forceinline__ void st_global_v8(void* dst, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
// Pairs of fp32: one instruction for two.
__device__ __forceinline__ uint64_t pair_of(float2 v) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
    return r;
}
__device__ __forceinline__ float2 of_pair(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pair_of(a)), "l"(pair_of(b)), "l"(pair_of(c)));
    return of_pair(r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_of(a)), "l"(pair_of(b)));
    return of_pair(r);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Instruction descriptors: fp32 accumulators, M = 128 (a pair's rows), N = 256.
constexpr uint32_t kIdescQk = idesc_f16_f32(128, 256, false, false);
constexpr uint32_t kIdescBf16 = kIdescQk | (1u << 7) | (1u << 10);      // both operands bf16
constexpr uint32_t kIdescPv = idesc_f16_f32(128, 256, false, true);

// A warpgroup's registers per thread from here on (a decrease may not go up, nor an increase down).
template <uint32_t kRegs>
__device__ __forceinline__ void set_registers() {
    if constexpr (kRegs > kRegsLaunch) warpgroup_reg_alloc<kRegs>();
    if constexpr (kRegs < kRegsLaunch) warpgroup_reg_dealloc<kRegs>();
}

// ------------------------------------------------------------------ the work and its ranges
struct Seq {
    int first, n, L;        // first new token in q, their number, tokens of the sequence (clamped to max_seq_len)
    int rows, units;        // of its first max_q_len new tokens
};
__device__ __forceinline__ Seq load_seq(const PrefillParams& p, int b) {
    Seq s;
    const int lo = max(0, min(__ldg(p.cu + b), p.total_q)), hi = max(lo, min(__ldg(p.cu + b + 1), p.total_q));
    const int len = __ldg(p.seq_lens + b);
    s.first = lo;
    s.n = hi - lo;
    s.L = max(0, min(len, p.max_seq_len));
    if (hi - lo > p.max_q_len || len > p.max_seq_len) set_error(p.err, NVFP4KV_DEVERR_SEQ_LEN);
    s.rows = min(s.n, p.max_q_len) * p.heads;
    s.units = (s.rows + kUnitRows - 1) / kUnitRows;
    return s;
}
// The new token of a row of the sequence: row / heads.
__device__ __forceinline__ int token_of(const PrefillParams& p, int row) {
    int tok = p.heads == 1 ? row : static_cast<int>(__umulhi(row, p.heads_magic));      // the quotient, or one more
    tok -= tok * p.heads > row;
    return tok;
}
// Tokens that unit k of the sequence sees: those of its last row.
__device__ __forceinline__ int unit_end(const PrefillParams& p, const Seq& s, int k) {
    const int last = min(s.rows, (k + 1) * kUnitRows) - 1;
    return max(0, min(s.L, s.L - s.n + token_of(p, last) + 1));
}
template <bool kWindow>
__device__ __forceinline__ int tiles_to(const PrefillParams& p, int end) {
    const int tiles = (end + kTile - 1) / kTile;
    return kWindow ? min(tiles, p.max_tiles) : tiles;
}
template <bool kWindow>
__device__ __forceinline__ int unit_tiles(const PrefillParams& p, const Seq& s, int k) {
    return tiles_to<kWindow>(p, unit_end(p, s, k));
}
// A window's unit covers, in max_tiles tiles, the first sink_rows tokens and the last ones up to its
// end (rounded up to 64); positions it leaves out in between.  0 for a unit that covers everything.
__device__ __forceinline__ int unit_gap(const PrefillParams& p, int end) {
    return end > p.max_tiles * kTile ? (end + 63) / 64 * 64 - p.max_tiles * kTile : 0;
}
// Rows of the sequence's image: its tokens, or with a window those that its units cover (without the gap
// of the first one, which is the smallest).
template <bool kWindow>
__device__ __forceinline__ int image_rows_of(const PrefillParams& p, const Seq& s) {
    if (s.units == 0) return 0;
    return kWindow ? unit_end(p, s, s.units - 1) - unit_gap(p, unit_end(p, s, 0)) : s.L;
}
template <bool kWindow>
__device__ __forceinline__ int image_blocks_of(const PrefillParams& p, const Seq& s) {
    return (image_rows_of<kWindow>(p, s) + kImageTok - 1) / kImageTok;
}
// Weights of the work: a tile, and what a unit adds (its first tile's and its epilogue's latency, about
// 8,700 cycles of a tile's 5,800).  With one tile's weight for a unit, pairs with short units took 9 %
// longer than the mean in a batch of chunks, now 6.
constexpr int kTileWeight = 2, kUnitWeight = 3;
// Weight of the sequence's first K units.  A unit's tiles do not fall with k, so the sum goes over
// tile counts (at most n / 256 + 2 of them), not over units.
template <bool kWindow>
__device__ __forceinline__ int64_t weight_before(const PrefillParams& p, const Seq& s, int K) {
    if (K <= 0) return 0;
    const int t0 = unit_tiles<kWindow>(p, s, 0), t1 = unit_tiles<kWindow>(p, s, s.units - 1);
    int64_t w = static_cast<int64_t>(K) * (kTileWeight * t0 + kUnitWeight);
    for (int t = t0; t < t1; ++t) {
        // units of at most t tiles: those whose last row's token is at most y
        const int64_t y1 = static_cast<int64_t>(t) * kTile - (s.L - s.n);      // y + 1
        const int64_t rows = y1 * p.heads;
        int64_t c = y1 <= 0 ? 0 : rows >= s.rows ? s.units : rows / kUnitRows;
        w += kTileWeight * (K - (c < K ? c : K));
    }
    return w;
}

template <typename T>
__device__ __forceinline__ T warp_inclusive_sum(T x, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T y = __shfl_up_sync(0xFFFFFFFFu, x, o);
        if (lane >= o) x += y;
    }
    return x;
}

// A pair's place in its range.
struct Range {
    int64_t left;       // weight still to do
    int b, k, offset;   // sequence, unit, weight of the unit done before
    int image0;         // image blocks of the sequences before b
    int loaded;         // whether what follows is sequence b's
    Seq seq;
    int image_rows, gap0;
};
// Where pair `pair` of p.pairs begins.  Run by one warp, a sequence per lane (and pass, past 32).
template <bool kWindow>
__device__ __forceinline__ Range find_range(const PrefillParams& p, int pair) {
    const int lane = threadIdx.x & 31;
    Seq s{};
    int64_t w = 0, total = 0;
    for (int b = lane; b < p.batch; b += 32) {
        s = load_seq(p, b);
        w = weight_before<kWindow>(p, s, s.units);
        total += w;
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
    int64_t lo, hi;
    if (total <= 0xFFFFFFFFll / kMaxPairs) {      // (64-bit divisions take hundreds of cycles)
        lo = static_cast<uint32_t>(total) * pair / p.pairs;
        hi = static_cast<uint32_t>(total) * (pair + 1) / p.pairs;
    } else {
        lo = total * pair / p.pairs;
        hi = total * (pair + 1) / p.pairs;
    }
    Range r{hi - lo, 0, 0, 0, 0, 0, {}, 0, 0};
    if (hi <= lo) return r;
    int64_t before = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
        if (p.batch > 32) {       // (else the first pass left them here)
            s = Seq{};
            if (b0 + lane < p.batch) s = load_seq(p, b0 + lane);
            w = weight_before<kWindow>(p, s, s.units);
        }
        const int blocks = image_blocks_of<kWindow>(p, s);
        const int64_t upto = before + warp_inclusive_sum(w, lane);
        const int img = r.image0 + warp_inclusive_sum(blocks, lane);
        const uint32_t hit = __ballot_sync(0xFFFFFFFFu, lo < upto);
        if (hit) {
            const int src = __ffs(hit) - 1;
            r.b = b0 + src;
            r.image0 = __shfl_sync(0xFFFFFFFFu, img - blocks, src);
            const int64_t x = lo - __shfl_sync(0xFFFFFFFFu, upto - w, src);
            Seq t;
            t.n = __shfl_sync(0xFFFFFFFFu, s.n, src);
            t.L = __shfl_sync(0xFFFFFFFFu, s.L, src);
            t.rows = __shfl_sync(0xFFFFFFFFu, s.rows, src);
            t.units = __shfl_sync(0xFFFFFFFFu, s.units, src);
            t.first = 0;
            int k = 0, len = t.units;
            while (len > 1) {                          // the last unit that begins at or before x, 32 candidates a step
                const int step = (len + 31) / 32, cand = k + lane * step;
                const uint32_t ok = __ballot_sync(0xFFFFFFFFu, cand < k + len && weight_before<kWindow>(p, t, cand) <= x);
                const int at = 31 - __clz(ok);
                len = min(step, k + len - (k + at * step));
                k += at * step;
            }
            r.k = k;
            r.offset = static_cast<int>(x - weight_before<kWindow>(p, t, k));
            return r;
        }
        before = __shfl_sync(0xFFFFFFFFu, upto, 31);
        r.image0 = __shfl_sync(0xFFFFFFFFu, img, 31);
    }
    r.left = 0;
    return r;
}

// A run of tiles of one unit.
struct Part {
    int b, block;           // sequence, unit of it
    int first, n, L, rows;  // of the sequence
    int end;                // tokens the unit sees
    int tile0, n_tiles;
    int image;              // the sequence's first image block
    int head, tail;         // it begins / ends the unit
    int half;               // rows in the leading CTA (the unit's others are in the second)
    int image_rows;         // of the sequence
    int gap, lift;          // with a window: positions, and image rows, left out after sink_rows
};
// Tiles in a unit's first `weight`.
__device__ __forceinline__ int tiles_in(int weight) { return max(weight - kUnitWeight, 0) / kTileWeight; }
// The next part of the range; parts without tiles are given only where they are a whole unit (one
// that sees no token).
template <bool kWindow>
__device__ __forceinline__ bool next_part_of(const PrefillParams& p, Range& r, Part& t) {
    while (r.left > 0) {
        if (!r.loaded) {
            r.seq = load_seq(p, r.b);
            r.image_rows = image_rows_of<kWindow>(p, r.seq);
            r.gap0 = kWindow && r.seq.units > 0 ? unit_gap(p, unit_end(p, r.seq, 0)) : 0;
            r.loaded = 1;
        }
        const Seq& s = r.seq;
        if (r.k >= s.units) {
            ++r.b;
            r.k = 0;
            r.offset = 0;
            r.image0 += (r.image_rows + kImageTok - 1) / kImageTok;
            r.loaded = 0;
            continue;
        }
        t.image_rows = r.image_rows;
        t.end = unit_end(p, s, r.k);
        const int tiles = tiles_to<kWindow>(p, t.end);
        if (kWindow) {
            t.gap = unit_gap(p, t.end);
            t.lift = t.gap - r.gap0;
        }
        const int weight = kTileWeight * tiles + kUnitWeight, begin = r.offset;
        const int take = static_cast<int>(r.left < weight - begin ? r.left : weight - begin);
        t.tile0 = tiles_in(begin);
        t.n_tiles = tiles_in(begin + take) - t.tile0;
        t.b = r.b; t.block = r.k;
        t.first = s.first; t.n = s.n; t.L = s.L; t.rows = s.rows;
        t.image = r.image0;
        // 64 rows or fewer (one token of 64 heads): 32 in each CTA, so that both store O
        t.half = s.rows - r.k * kUnitRows <= kCtaRows ? kCtaRows / 2 : kCtaRows;
        t.head = t.tile0 == 0;
        t.tail = t.tile0 + t.n_tiles == tiles;
        r.left -= take;
        r.offset += take;
        if (r.offset == weight) {
            ++r.k;
            r.offset = 0;
        }
        if (t.n_tiles > 0 || (tiles == 0 && begin == 0)) return true;
    }
    return false;
}
// A warp's place in its pair's range and its current part, in shared memory: read where they are
// used, they cost no registers in the loops over tiles.
struct Work {
    Range range;
    int more;
    Part part;
    Part ahead;
};
static_assert(sizeof(Work) <= kWorkBytes, "a warp's work record");
// The search for a part takes a microsecond of dependent loads and divisions, so a warp may look for
// the next one (ahead) while it waits for something else, and move on to it later (advance_part).
template <bool kWindow>
__device__ __forceinline__ void look_ahead(const PrefillParams& p, Work* w) {
    if ((threadIdx.x & 31) == 0) {
        Range r = w->range;
        Part t;
        const bool more = next_part_of<kWindow>(p, r, t);
        w->range = r;
        w->more = more;
        if (more) w->ahead = t;
    }
}
__device__ __forceinline__ bool advance_part(Work* w) {
    __syncwarp();
    const bool more = *reinterpret_cast<volatile int*>(&w->more) != 0;
    if (more) {
        const int* src = reinterpret_cast<const int*>(&w->ahead);
        int* dst = reinterpret_cast<int*>(&w->part);
        static_assert(sizeof(Part) <= 128 && sizeof(Part) % 4 == 0, "a word per lane");
        const int lane = threadIdx.x & 31;
        if (lane < static_cast<int>(sizeof(Part) / 4)) dst[lane] = src[lane];
    }
    __syncwarp();
    return more;
}
template <bool kWindow>
__device__ __forceinline__ bool next_part(const PrefillParams& p, Work* w) {
    __syncwarp();
    look_ahead<kWindow>(p, w);
    return advance_part(w);
}

// Pool row of position pos < end of a sequence, -1 for a missing page or past the end.
__device__ __forceinline__ int64_t pool_row(const PrefillParams& p, const int32_t* table, int pos, int end) {
    if (pos >= end) return -1;
    const int pg = __ldg(table + (pos >> p.page_shift));
    if (pg < 0 || pg >= p.num_pages) return -1;
    return (static_cast<int64_t>(pg) << p.page_shift) | (pos & ((1 << p.page_shift) - 1));
}

// Stages in the order the MMAs take them: K of tile 0, then K of tile i and V of tile i - 1.
struct Cursor {
    int u, i, s;      // stage number; s < k_stages: K stage s of tile i, else V stage s - k_stages of tile i - 1
};
__device__ __forceinline__ void advance(Cursor& c, int k_stages, int n_tiles) {
    ++c.u;
    ++c.s;
    if (c.i == 0 ? c.s == k_stages : c.s == k_stages + kVStages) {
        ++c.i;
        c.s = c.i < n_tiles ? 0 : k_stages;
    }
}

// 8 latent dims (a word of codes, their block scale twice) as fp16.
__device__ __forceinline__ uint4 dequant8(uint32_t code, uint32_t scale2) {
    uint32_t h[4];
    e2m1x8_to_f16x2x4(code, h);
    return make_uint4(hmul2_u32(h[0], scale2), hmul2_u32(h[1], scale2), hmul2_u32(h[2], scale2), hmul2_u32(h[3], scale2));
}

// Two fp16 as bf16; exact for a code (2 bits) times its scale (4 bits): 6 of bf16's 8 bits, and well within its range.
__device__ __forceinline__ uint32_t half2_to_bf162(uint32_t h) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    const __nv_bfloat162 b = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&b);
}

// ------------------------------------------------------------------ image
// The image: every token of the sequences with new ones dequantised, as the ring stages the attention
// kernel copies.  Block = 128 tokens: [8 latent atoms (+ the rope part)][128 tokens x 128 B], 128-byte
// swizzled, zeros for tokens that do not exist and for blocks with a NaN scale (the token's bit says
// so instead: a NaN in V would reach rows that do not see it).  Eight lanes read a row's half (128
// code bytes), a thread writes its 32 dims as 16 bytes to each of four atoms, a warp whole 128-byte
// rows.  The blocks of the grid take pieces of 32 tokens in turn (their number is on the device), a
// row per thread, six blocks on an SM: 24.2 us for 91K tokens (143 MB read and written, 5.9 TB/s;
// with four rows a thread and two blocks 26.6, and 5.4 against 3.4 for 2.4K tokens).
template <Form kForm>
__global__ void __launch_bounds__(256, 6) prefill_image_kernel(const __grid_constant__ PrefillParams p) {
    constexpr bool kWindow = kForm == kDirect;
    __shared__ uint32_t bits[2];      // of the piece's tokens: those that exist, those that hold a NaN
    __shared__ int b_s, pos_s, total_s;
    griddep_wait();                   // first: what starts now counts on all before this grid being done
    griddep_launch_dependents();
    const int tid = threadIdx.x, lp = tid & 7, r0 = tid >> 3;
    int total = 0x7FFFFFFF;
    for (int item = blockIdx.x; item < total; item += gridDim.x) {
        const int block = item / kImagePieces, piece = item % kImagePieces;
        if (tid < 32) {
            const int lane = tid;
            int base = 0, b = -1, pos = 0;
            for (int b0 = 0; b0 < p.batch; b0 += 32) {
                int blocks = 0;
                if (b0 + lane < p.batch) blocks = image_blocks_of<kWindow>(p, load_seq(p, b0 + lane));
                const int upto = base + warp_inclusive_sum(blocks, lane);
                const uint32_t hit = __ballot_sync(0xFFFFFFFFu, block < upto);
                if (hit && b < 0) {
                    const int src = __ffs(hit) - 1;
                    b = b0 + src;
                    pos = kImageTok * (block - __shfl_sync(0xFFFFFFFFu, upto - blocks, src)) + 32 * piece;
                }
                base = __shfl_sync(0xFFFFFFFFu, upto, 31);
            }
            if (lane == 0) {
                b_s = b;
                pos_s = pos;
                total_s = base;
            }
            if (lane < 2) bits[lane] = 0;
        }
        __syncthreads();
        if (b_s < 0) return;
        total = total_s * kImagePieces;
        const Seq seq = load_seq(p, b_s);
        int L = seq.L, t = pos_s + r0;
        bool seen = true;
        if (kWindow) {      // (a token that no row sees is not read: its page may be gone)
            L = unit_end(p, seq, seq.units - 1);
            if (t >= p.sink_rows) t += unit_gap(p, unit_end(p, seq, 0));
            seen = t < p.sinks || t > seq.L - seq.n - p.window;
        }
        const int64_t row = seen ? pool_row(p, p.tables + b_s * p.tables_stride, t, L) : -1;
        uint4 code[2], rope = make_uint4(0, 0, 0, 0);
        uint16_t scale[2] = {0, 0};
        code[0] = code[1] = rope;
        if (row >= 0) {
            const uint8_t* src = p.pool + row * kRowBytes;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                code[h] = ldg_nc_v4(src + 128 * h + 16 * lp);
                scale[h] = __ldg(reinterpret_cast<const uint16_t*>(src + 256 + 16 * h + 2 * lp));
            }
            if (p.rope) rope = ldg_nc_v4(p.rope + row * kRope + 8 * lp);
        }
        const int k_atoms = p.rope ? 9 : 8, atoms = k_atoms + (kForm == kDirect ? 8 : 0);
        uint8_t* dst = p.image + static_cast<int64_t>(block) * atoms * kStageBytes + piece * 4096 + r0 * 128 + ((lp ^ (r0 & 7)) << 4);
        bool nan = false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t word[4] = {code[h].x, code[h].y, code[h].z, code[h].w};
            const uint32_t s2 = e4m3x2_to_f16x2(scale[h]);
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const bool bad = ((scale[h] >> (s & 2 ? 8 : 0)) & 0x7F) == 0x7F;
                nan |= bad;
                const uint4 v = dequant8(word[s], __byte_perm(s2, s2, s & 2 ? 0x3232 : 0x1010));
                const uint4 w = bad ? make_uint4(0, 0, 0, 0) : v;
                if constexpr (kForm == kDirect) {
                    *reinterpret_cast<uint4*>(dst + (k_atoms + 4 * h + s) * kStageBytes) = w;
                    *reinterpret_cast<uint4*>(dst + (4 * h + s) * kStageBytes) =
                        make_uint4(half2_to_bf162(w.x), half2_to_bf162(w.y), half2_to_bf162(w.z), half2_to_bf162(w.w));
                } else {
                    *reinterpret_cast<uint4*>(dst + (4 * h + s) * kStageBytes) = w;
                }
            }
        }
        if (p.rope) *reinterpret_cast<uint4*>(dst + 8 * kStageBytes) = rope;
        if (nan) atomicOr(&bits[1], 1u << r0);
        if (lp == 0) {
            if (row >= 0) atomicOr(&bits[0], 1u << r0);
            else if (seen && t < L) set_error(p.err, NVFP4KV_DEVERR_BAD_PAGE);
        }
        __syncthreads();
        if (tid < 2) p.image_bits[8 * static_cast<int64_t>(block) + 4 * tid + piece] = bits[tid];
        __syncthreads();      // (the next item's words)
    }
}

// ------------------------------------------------------------------ attention
// Q of a unit: rows -> fp16 after a power of two per row that brings its largest |q| to [2^10, 2^11)
// (the rope part by the same factor, in bf16).  A rope part far larger than the rest sets the power
// itself, kRopeLog2 above what the latent part would: with 2^100 for a tiny latent part its products
// passed fp32's range.  A warp per row, 16 + 2 dims per lane, kQRows rows at a time: r, r + step, ...
// of the CTA's 64.
constexpr uint32_t kRopeLog2 = 50;
struct QRows {
    uint4 u[kQRows][2];
    uint32_t rope[kQRows];
};
__device__ __forceinline__ void load_q(const PrefillParams& p, const volatile Part& t, int cta, int r, int step, QRows& q) {
    const int lane = threadIdx.x & 31, half = t.half, row0 = t.block * kUnitRows + half * cta, rows = t.rows, first = t.first;
#pragma unroll
    for (int j = 0; j < kQRows; ++j) {
        q.u[j][0] = q.u[j][1] = make_uint4(0, 0, 0, 0);
        q.rope[j] = 0;
        const int row = row0 + r + j * step;
        if (row < rows && r + j * step < half) {
            const int tok = token_of(p, row);
            const __nv_bfloat16* src = p.q + static_cast<int64_t>(first + tok) * p.q_st + static_cast<int64_t>(row - tok * p.heads) * p.q_sh;
            q.u[j][0] = ldg_nc_v4(src + 16 * lane);
            q.u[j][1] = ldg_nc_v4(src + 16 * lane + 8);
            if (p.rope) q.rope[j] = __ldg(reinterpret_cast<const uint32_t*>(src + kLatent) + lane);
        }
    }
}
// (base: the operand's place, or its copy in the workspace)
__device__ __forceinline__ void store_q(const PrefillParams& p, uint8_t* base, float* qs, int r0, int step, const QRows& q) {
    const int lane = threadIdx.x & 31;
    uint32_t w[kQRows][8], amax[kQRows];
#pragma unroll
    for (int j = 0; j < kQRows; ++j) {
        w[j][0] = q.u[j][0].x; w[j][1] = q.u[j][0].y; w[j][2] = q.u[j][0].z; w[j][3] = q.u[j][0].w;
        w[j][4] = q.u[j][1].x; w[j][5] = q.u[j][1].y; w[j][6] = q.u[j][1].z; w[j][7] = q.u[j][1].w;
        uint32_t hi = 0, lo = 0;      // the largest |q| of the pairs' halves: as integers, the order of |x|
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            hi = max(hi, w[j][i] & 0x7FFF0000u);
            lo = max(lo, w[j][i] & 0x7FFFu);
        }
        const int rope = static_cast<int>(max(q.rope[j] & 0x7FFF0000u, (q.rope[j] & 0x7FFFu) << 16));
        amax[j] = max(max(hi, lo << 16), static_cast<uint32_t>(max(rope - static_cast<int>(kRopeLog2 << 23), 0)));
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1)
#pragma unroll
        for (int j = 0; j < kQRows; ++j) amax[j] = max(amax[j], __shfl_xor_sync(0xFFFFFFFFu, amax[j], o));
#pragma unroll
    for (int j = 0; j < kQRows; ++j) {
        const int r = r0 + j * step;
        const int eb = static_cast<int>((amax[j] >> 23) & 0xFFu);      // 255: inf or NaN
        const int e = eb > 0 && eb < 255 ? max(eb - 127 - 10, -100) : 0;
        float factor = fabsf(p.scale_log2) * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
        float mul = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        mul = p.scale_log2 < 0.0f ? -mul : mul;
        if (factor == 0.0f) {          // every score 0: zero queries, and a factor that keeps a hidden score's -inf
            factor = 1.0f;
            mul = 0.0f;
        }
        uint32_t h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            h[i] = pack_half2(__uint_as_float(w[j][i] << 16) * mul, __uint_as_float(w[j][i] & 0xFFFF0000u) * mul);
        // dims 16 lane + 8 c: half lane / 16, piece (lane / 2) % 8, chunk 2 (lane % 2) + c
        uint8_t* dst = base + ((lane >> 4) * 4 + 2 * (lane & 1)) * (kCtaRows * 128) + r * 128 + ((((lane >> 1) & 7) ^ (r & 7)) << 4);
        *reinterpret_cast<uint4*>(dst) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(dst + kCtaRows * 128) = make_uint4(h[4], h[5], h[6], h[7]);
        if (p.rope) {
            const __nv_bfloat162 two = __floats2bfloat162_rn(__uint_as_float(q.rope[j] << 16) * mul, __uint_as_float(q.rope[j] & 0xFFFF0000u) * mul);
            *reinterpret_cast<uint32_t*>(base + 8 * (kCtaRows * 128) + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + 4 * (lane & 3)) =
                *reinterpret_cast<const uint32_t*>(&two);
        }
        if (lane == 0) qs[r] = factor;
    }
}

// The first n bits of a word.
__device__ __forceinline__ uint32_t bits_below(int n) { return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u; }

// kDirect: the unit's rows of q into the operand as they are, 16 bytes at a time, zeros past the unit.  Run by
// the threads tid, tid + nt, ... ; they wait for their copies and make them visible to the tensor core.
__device__ __forceinline__ void copy_q(const PrefillParams& p, const volatile Part& t, int cta, uint8_t* base, int tid, int nt) {
    const int half = t.half, row0 = t.block * kUnitRows + half * cta, rows = t.rows, first = t.first, pieces = p.rope ? 72 : 64;
    const uint32_t dst0 = smem_u32(base);
    for (int u = tid; u < kCtaRows * 8; u += nt) {      // (a piece of all atoms at a time: eight threads a row)
        const int r = u >> 3, c0 = u & 7, row = row0 + r;
        const bool real = r < half && row < rows;
        const int tok = real ? token_of(p, row) : 0;
        const __nv_bfloat16* src = p.q + static_cast<int64_t>(first + tok) * p.q_st + static_cast<int64_t>(real ? row - tok * p.heads : 0) * p.q_sh;
        const uint32_t bytes = real ? 16 : 0;
#pragma unroll
        for (int k = 0; k < 9; ++k) {
            const int c = c0 + 8 * k;                    // dims 8 c .. of the row
            if (c >= pieces) break;
            // latent half c / 32, piece (c / 4) % 8 of atom c % 4; the rope part in order
            const int atom = k < 8 ? 4 * (c >> 5) + (c & 3) : 8, at = k < 8 ? (c >> 2) & 7 : c0;
            cp_async16_zfill(dst0 + atom * (kCtaRows * 128) + r * 128 + ((at ^ (r & 7)) << 4), src + 8 * c, bytes);
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    fence_proxy_async_smem();
}
// The same rows into L2.
__device__ __forceinline__ void prefetch_q(const PrefillParams& p, const volatile Part& t, int cta, int tid) {
    const int row = t.block * kUnitRows + t.half * cta + tid;
    if (tid >= t.half || row >= t.rows) return;
    const int tok = token_of(p, row);
    const __nv_bfloat16* src = p.q + static_cast<int64_t>(t.first + tok) * p.q_st + static_cast<int64_t>(row - tok * p.heads) * p.q_sh;
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"((p.rope ? kDim : kLatent) * 2) : "memory");
}

template <Form kForm>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
mla_prefill_kernel(const __grid_constant__ PrefillParams p) {
    constexpr bool kWindow = kForm == kDirect;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const uint32_t sbase = smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cta = static_cast<int>(cluster_rank()), pair = blockIdx.x >> 1;
    volatile int* flags = reinterpret_cast<volatile int*>(smem + SM_FLAGS);
    volatile int* abort_flag = flags + 1;
    auto bar = [&](int i) -> uint32_t { return sbase + SM_BARS + 8 * i; };

    if (warp == 0) {
        const Range r = find_range<kWindow>(p, pair);
        if (lane == 0) {
            flags[1] = 0;
            // the range's first part, for every warp, and in `part` the first one with tiles: its Q and
            // its first stages are fetched before the roles begin
            Work* w = reinterpret_cast<Work*>(smem + SM_WORK + kThreads / 32 * kWorkBytes);
            Range r0 = r;
            Part t0;
            const bool more = next_part_of<kWindow>(p, r0, t0);
            w->range = r0;
            w->more = more;
            if (more) w->ahead = t0;
            bool tiles = more && t0.n_tiles > 0;
            while (more && !tiles && next_part_of<kWindow>(p, r0, t0)) tiles = t0.n_tiles > 0;
            if (!tiles) t0.n_tiles = 0;
            w->part = t0;
            if (cta == 0) p.parts[2 * pair].used = p.parts[2 * pair + 1].used = 0;
        }
    }
    if (threadIdx.x == 32) {
        for (int k = 0; k < kStages; ++k) {
            mbar_init(bar(B_FULL + k), 2);
            mbar_init(bar(B_EMPTY + k), 1);
            mbar_init(bar(B_LAND + k), 1);
        }
        for (int k = 0; k < 2; ++k) {
            mbar_init(bar(B_S_FULL + k), 1);
            mbar_init(bar(B_S_FREE + k), 2 * kSoftmaxWarps);
        }
        mbar_init(bar(B_P_FULL), 2 * kSoftmaxWarps);
        mbar_init(bar(B_PV_DONE), 1);
        mbar_init(bar(B_Q_FULL), 2);
        mbar_init(bar(B_Q_FREE), 1);
        mbar_init(bar(B_Q_LAND), 1);
        mbar_init(bar(B_O_FREE), 2 * kSoftmaxWarps);
        mbar_init(bar(B_DRAIN), 1);
        mbar_fence_init();
    }
    __syncthreads();
    Work* work = reinterpret_cast<Work*>(smem + SM_WORK + warp * kWorkBytes);
    const volatile Part& t = work->part;
    const Work* first = reinterpret_cast<const Work*>(smem + SM_WORK + kThreads / 32 * kWorkBytes);
    if (!first->more) {               // nothing for this pair: the whole cluster
        griddep_wait();               // (this grid ends after the image kernel)
        return;
    }
    {
        static_assert(sizeof(Work) % 4 == 0 && sizeof(Work) <= 256, "two words per lane");
        for (int k = lane; k < static_cast<int>(sizeof(Work) / 4); k += 32)
            reinterpret_cast<int*>(work)[k] = reinterpret_cast<const int*>(first)[k];
    }
    if (warp == kMmaWarp) pair_tmem_alloc(sbase + SM_FLAGS, kTmemCols);
    const int k_stages = p.rope ? 9 : 8;
    // A stage of a part's ring: K stage c.s of tile c.i, or V stage c.s - k_stages of tile c.i - 1.
    const int64_t image_bytes = static_cast<int64_t>(k_stages + (kForm == kDirect ? kVStages : 0)) * kStageBytes;
    const int v_atom = kForm == kDirect ? k_stages : 0;      // the image's first one for PV
    // (with a window, `last` is the sequence's last run of 64 image rows, `lift` in such runs)
    auto copy_stage = [&](const Cursor& c, int image, int last, int tile0, int lift, int slot) {
        const uint32_t dst = sbase + SM_RING + slot * kStageBytes, landed = bar(B_LAND + slot);
        if (elect_one()) {
            mbar_arrive_expect_tx(landed, kStageBytes);
            if constexpr (kWindow) {
                auto run = [&](int g) {      // 64 tokens of the unit: where their rows of atom 0 lie
                    if (64 * g >= p.sink_rows) g += lift;
                    g = min(g, last);
                    return p.image + (image + (g >> 1)) * image_bytes + (g & 1) * 8192;
                };
                if (c.s < k_stages) {
                    const int g = 4 * (tile0 + c.i) + 2 * cta;
                    bulk_copy_g2s(dst, run(g) + c.s * kStageBytes, 8192, landed);
                    bulk_copy_g2s(dst + 8192, run(g + 1) + c.s * kStageBytes, 8192, landed);
                } else {
                    const int v = c.s - k_stages;
                    const uint8_t* src = run(4 * (tile0 + c.i - 1) + (v >> 1)) + (v_atom + 4 * cta + 2 * (v & 1)) * kStageBytes;
                    bulk_copy_g2s(dst, src, 8192, landed);
                    bulk_copy_g2s(dst + 8192, src + kStageBytes, 8192, landed);
                }
            } else if (c.s < k_stages) {
                const int blk = min(image + 2 * (tile0 + c.i) + cta, last);
                bulk_copy_g2s(dst, p.image + blk * image_bytes + c.s * kStageBytes, kStageBytes, landed);
            } else {
                const int v = c.s - k_stages;      // tokens 64 (v / 2) .., dim atoms 4 c + 2 (v % 2), + 1
                const int blk = min(image + 2 * (tile0 + c.i - 1) + (v >> 2), last);
                const uint8_t* src = p.image + blk * image_bytes + (4 * cta + 2 * (v & 1)) * kStageBytes + ((v >> 1) & 1) * 8192;
                bulk_copy_g2s(dst, src, 8192, landed);
                bulk_copy_g2s(dst + 8192, src + kStageBytes, 8192, landed);
            }
        }
        __syncwarp();
    };
    auto last_block = [&](int image, int rows) {      // (tokens past it are masked)
        const int blocks = (rows + kImageTok - 1) / kImageTok;
        return kWindow ? 2 * blocks - 1 : image + blocks - 1;
    };
    int early = 0;                    // stages copied before the roles begin
    if (first->part.n_tiles > 0) {
        const Part& t1 = first->part;
        QRows q;
        constexpr int kWarps = kThreads / 32;
        static_assert(kWarps * kQRows == kCtaRows, "one round of rows");
        if constexpr (kForm != kDirect) load_q(p, t1, cta, warp, kWarps, q);
        if (warp == kCopyWarp0 || warp == kCopyWarp0 + 1) {
            griddep_wait();           // the image kernel's writes
            early = kStages;          // (a tile has more)
            static_assert(kStages < 8 + kVStages, "stages of one tile");
            Cursor c{0, 0, 0};
            for (int u = 0; u < kStages; ++u, advance(c, k_stages, t1.n_tiles))
                if ((u & 1) == warp - kCopyWarp0) copy_stage(c, t1.image, last_block(t1.image, t1.image_rows), t1.tile0, t1.lift / 64, u);
        }
        if constexpr (kForm == kDirect) {      // (the other warps)
            if (warp < kCopyWarp0 || warp == kRelayWarp)
                copy_q(p, t1, cta, smem + SM_Q, warp == kRelayWarp ? threadIdx.x - 64 : threadIdx.x, kThreads - 64);
        } else {
            store_q(p, smem + SM_Q, reinterpret_cast<float*>(smem + SM_QS), warp, kWarps, q);
            fence_proxy_async_smem();
        }
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = static_cast<uint32_t>(flags[0]);

    if (warp >= kMmaWarp) {
        set_registers<kRegsCtl>();
        if (warp == kMmaWarp) {
            if (cta == 0) {
                // ==================================================== MMA issue
                const uint64_t dq = smem_desc_sw128(sbase + SM_Q, 16, 1024);
                const uint64_t dp = smem_desc_sw128(sbase + SM_P, 16, 1024);
                const uint64_t dk = smem_desc_sw128(sbase + SM_RING, 16, 1024);
                const uint64_t dv = smem_desc_sw128(sbase + SM_RING, 8192, 1024);
                int stages = 0, parts = 0, tile = 0;      // so far
                // (kDirect: the Q warps say how many tiles the next part has, 0 after the last, when its Q is there;
                // looking parts up here took 2,000 to 5,000 cycles a part between its MMAs)
                int told = kForm == kDirect ? first->part.n_tiles : 0;
                bool more = kForm == kDirect ? told > 0 : advance_part(work);
#pragma unroll 1
                for (; more && !*abort_flag; more = kForm == kDirect ? told > 0 : next_part<kWindow>(p, work)) {
                    const int n_tiles = kForm == kDirect ? told : t.n_tiles;
                    if (n_tiles == 0) continue;
                    if (kForm != kDirect && parts > 0) mbar_wait(bar(B_Q_FULL), (parts - 1) & 1, abort_flag, p.err);
                    // One thread runs the part.  Only about one MMA is queued behind the running one, so all that
                    // comes between two MMAs has 64 cycles to hide in: the next stage's barrier is looked at in
                    // the middle of a stage.  (A wait per stage by the whole warp: 375 cycles a stage where the
                    // MMAs take 256.)
                    if (elect_one()) {
                        int slot = stages % kStages;
                        uint32_t phase = (stages / kStages) & 1;
                        bool landed = false;
                        auto stage = [&](uint32_t d, uint64_t a, uint64_t b, uint32_t step, uint32_t id, bool first) {
                            if (!landed) mbar_wait(bar(B_FULL + slot), phase, abort_flag, p.err);
                            const uint32_t done = bar(B_EMPTY + slot);
                            if (++slot == kStages) {
                                slot = 0;
                                phase ^= 1;
                            }
                            pair_mma_f16(d, a, b, id, !first);
                            pair_mma_f16(d, a + 2, b + step, id, 1);
                            landed = test_phase(bar(B_FULL + slot), phase);
                            pair_mma_f16(d, a + 4, b + 2 * step, id, 1);
                            pair_mma_f16(d, a + 6, b + 3 * step, id, 1);
                            pair_commit(done);
                        };
#pragma unroll 1
                        for (int i = 0; i <= n_tiles; ++i) {
                            // (the output of the part before is read faster while no QK writes, so a part's second
                            // waits for it: 3 chunks of up to 777 tokens x 32 heads in a window of 512 109.4 ->
                            // 107.8 us; with the first waiting too 112.5)
                            if (kForm == kDirect && i == 1 && parts > 0) mbar_wait(bar(B_O_FREE), (parts - 1) & 1, abort_flag, p.err);
                            if (i < n_tiles) {
                                const int at = tile + i;
                                const uint32_t d = tmem + kTS + 128 * (at & 1);
                                if (at >= 2) mbar_wait(bar(B_S_FREE + (at & 1)), ((at >> 1) - 1) & 1, abort_flag, p.err);
                                tc_fence_after();
#pragma unroll 1
                                for (int j = 0; j < k_stages; ++j)
                                    stage(d, dq + ((j * kCtaRows * 128) >> 4), dk + ((slot * kStageBytes) >> 4), 2, kForm == kDirect || j == 8 ? kIdescBf16 : kIdescQk, j == 0);
                                pair_commit(bar(B_S_FULL + (at & 1)));
                                if (i == n_tiles - 1) pair_commit(bar(B_Q_FREE));
                            }
                            if (i > 0) {
                                mbar_wait(bar(B_P_FULL), (tile + i - 1) & 1, abort_flag, p.err);
                                if (kForm != kDirect && i == 1 && parts > 0) mbar_wait(bar(B_O_FREE), (parts - 1) & 1, abort_flag, p.err);
                                tc_fence_after();
#pragma unroll 1
                                for (int s = 0; s < kVStages; ++s)
                                    stage(tmem + kTO + 128 * (s & 1), dp + (((s >> 1) * kCtaRows * 128) >> 4), dv + ((slot * kStageBytes) >> 4), 128, kIdescPv,
                                          i == 1 && s < 2);
                                pair_commit(bar(B_PV_DONE));
                            }
                        }
                    }
                    __syncwarp();
                    stages += n_tiles * (k_stages + kVStages);
                    tile += n_tiles;
                    ++parts;
                    if constexpr (kForm == kDirect) {
                        if (!mbar_wait(bar(B_Q_FULL), (parts - 1) & 1, abort_flag, p.err)) break;
                        told = flags[2 + (parts & 1)];
                    }
                }
                if (elect_one()) pair_commit(bar(B_DRAIN));
                __syncwarp();
            }
            griddep_wait();       // this grid ends after the image kernel, whatever its units read
            mbar_drain_wait(bar(B_DRAIN), 0);
        } else {
            // ======================================================== image copies and their relay
            // Two warps take the stages in turn, a third hands each landed stage to the leader.
            const bool relay = warp == kRelayWarp;
            const int mine = warp - kCopyWarp0;
            int u = 0, slot = 0;                  // stage number and its ring slot
            uint32_t phase = 0;
            bool ok = true;
            griddep_wait();                       // the image kernel's writes
#pragma unroll 1
            for (bool more = advance_part(work); ok && more; more = next_part<kWindow>(p, work)) {
                const int n_tiles = t.n_tiles, total = n_tiles * (k_stages + kVStages), image = t.image, tile0 = t.tile0;
                const int last = last_block(image, t.image_rows), lift = kWindow ? t.lift / 64 : 0;
                Cursor c{0, 0, 0};
#pragma unroll 1
                for (; c.u < total; advance(c, k_stages, n_tiles)) {
                    if (relay) {
                        if (!(ok = mbar_wait(bar(B_LAND + slot), phase, abort_flag, p.err))) break;
                        if (lane == 0) leader_arrive(bar(B_FULL + slot));
                        __syncwarp();
                    } else if ((u & 1) == mine && u >= early) {
                        // (a release waited for by the other warp in between is earlier than this one's: no
                        // phase is skipped unseen)
                        if (u >= kStages && !(ok = mbar_wait(bar(B_EMPTY + slot), phase ^ 1, abort_flag, p.err))) break;
                        copy_stage(c, image, last, tile0, lift, slot);
                    }
                    ++u;
                    if (++slot == kStages) {
                        slot = 0;
                        phase ^= 1;
                    }
                }
            }
            // Every copy has landed once the MMAs that read it are done; after a timed-out wait the ones in
            // flight (the stages before u) are awaited here, so that the CTA does not exit under them.
            if (!relay && *abort_flag)
                for (int k = max(0, max(u, early) - kStages); k < max(u, early); ++k) mbar_drain_wait(bar(B_LAND + k % kStages), (k / kStages) & 1);
        }
    } else if (warp >= kQWarp0) {
        set_registers<kRegsQ>();
        // ============================================================ Q of each part
        // The factors have four places: part k's are written once the last QK of part k - 2 is complete, so
        // (S has two buffers) S of the tile two before it has been read, a tile of part k - 4 at the
        // earliest, whose factors the softmax warps read before.
        float* qs = reinterpret_cast<float*>(smem + SM_QS);
        int parts = 0;
#pragma unroll 1
        for (bool more = advance_part(work); more; more = next_part<kWindow>(p, work)) {
            if (t.n_tiles == 0) continue;
            if (kForm == kDirect && parts > 0) {
                prefetch_q(p, t, cta, threadIdx.x - 32 * kQWarp0);
                wait_phase(bar(B_Q_FREE), (parts - 1) & 1, abort_flag, p.err);
                copy_q(p, t, cta, smem + SM_Q, threadIdx.x - 32 * kQWarp0, 32 * kQWarps);
                named_bar_sync(3, 32 * kQWarps);
                if (warp == kQWarp0 && lane == 0) {
                    if (cta == 0) flags[2 + (parts & 1)] = t.n_tiles;
                    leader_arrive(bar(B_Q_FULL));
                }
                __syncwarp();
            } else if (kForm != kDirect && parts > 0) {      // (the first part's is there)
                // Converted into the workspace while the last part runs, and copied from there once its last QK
                // is done: converted only then, the MMAs waited 10,000 cycles a part for it (8 chunks of 777
                // tokens took 6 % longer).
                uint8_t* scratch = p.q_scratch + static_cast<int64_t>(2 * pair + cta) * kQBytes;
                QRows q;
                load_q(p, t, cta, warp - kQWarp0, kQWarps, q);
#pragma unroll 1
                for (int r = warp - kQWarp0; r < kCtaRows; r += kQRows * kQWarps) {
                    const QRows now = q;
                    load_q(p, t, cta, r + kQRows * kQWarps, kQWarps, q);
                    store_q(p, scratch, qs + 64 * (parts & 3), r, kQWarps, now);
                }
                __threadfence();
                asm volatile("fence.proxy.async;" ::: "memory");
                named_bar_sync(3, 32 * kQWarps);
                wait_phase(bar(B_Q_FREE), (parts - 1) & 1, abort_flag, p.err);
                if (warp == kQWarp0 && __all_sync(0xFFFFFFFFu, !*abort_flag)) {
                    if (elect_one()) {
                        const uint32_t bytes = k_stages * kCtaRows * 128;
                        mbar_arrive_expect_tx(bar(B_Q_LAND), bytes);
                        bulk_copy_g2s(sbase + SM_Q, scratch, bytes, bar(B_Q_LAND));
                    }
                    __syncwarp();
                    mbar_drain_wait(bar(B_Q_LAND), (parts - 1) & 1);      // whatever else fails: the CTA does not exit under it
                } else {
                    wait_phase(bar(B_Q_LAND), (parts - 1) & 1, abort_flag, p.err);
                }
                if (warp == kQWarp0 && lane == 0) leader_arrive(bar(B_Q_FULL));
                __syncwarp();
            }
            ++parts;
        }
        if (kForm == kDirect && parts > 0) {         // no more
            wait_phase(bar(B_Q_FREE), (parts - 1) & 1, abort_flag, p.err);      // (the last Q's arrival has been seen)
            if (warp == kQWarp0 && lane == 0) {
                if (cta == 0) flags[2 + (parts & 1)] = 0;
                leader_arrive(bar(B_Q_FULL));
            }
            __syncwarp();
        }
    } else {
        set_registers<kRegsSoftmax>();
        // ============================================================ softmax
        // warp: TMEM lanes 32 sp .., columns 64 ch .. of a tile's 128: row 32 (sp & 1) + lane, token
        // quarter q4; the four warps of a row exchange their maxima in shared memory
        const int sp = warp & 3, ch = warp >> 2;
        const int row = 32 * (sp & 1) + lane, q4 = 2 * (sp >> 1) + ch;
        const uint32_t lanes = static_cast<uint32_t>(32 * sp) << 16;
        float* red = reinterpret_cast<float*>(smem + SM_RED);
        float* lsum = reinterpret_cast<float*>(smem + SM_LSUM);
        int parts = 0, tile = 0;                 // parts with tiles, and tiles, so far
        bool first_part = true;
        griddep_wait();                          // the image kernel's token bits
        // bits of the quarter's tokens that exist, and of those that hold a NaN: loaded a tile ahead, a part's
        // first ones while the last PV of the part before runs (without a window with the part's place in
        // registers: read from `t` it held up every tile, 2,048 tokens of 64 heads over 16,384 2,898 us against 2,891)
        auto load_bits = [&](const volatile Part& t, int tile0, int image, int L, int i, uint2 (&w)[2]) {
            const int tok0 = ((kWindow ? t.tile0 : tile0) + i) * kTile + 64 * q4;
            if constexpr (kWindow) {
                const int row0 = min(tok0 < p.sink_rows ? tok0 : tok0 + t.lift, t.image_rows - 1);
                const uint32_t* src = p.image_bits + 8 * static_cast<int64_t>(t.image + row0 / kImageTok) + (row0 & 64) / 32;
                w[0] = *reinterpret_cast<const uint2*>(src);
                w[1] = *reinterpret_cast<const uint2*>(src + 4);
                return;
            }
            const uint32_t* src = p.image_bits + 8 * static_cast<int64_t>(image + min(tok0, L - 1) / kImageTok) + ((tok0 & (kImageTok - 1)) >> 5);
            w[0] = *reinterpret_cast<const uint2*>(src);
            w[1] = *reinterpret_cast<const uint2*>(src + 4);
        };
        uint2 ahead[2];
        const volatile Part& next = work->ahead;
#pragma unroll 1
        while (advance_part(work)) {
            const int n_tiles = t.n_tiles, tile0 = t.tile0, image = t.image, L = t.L, gap = kWindow ? t.gap : 0;
            int lim = 0;                                                      // tokens the row sees
            {
                const int grow = t.block * kUnitRows + t.half * cta + row;    // row of the sequence
                if (grow < t.rows && row < t.half) lim = min(t.L, t.L - t.n + token_of(p, grow) + 1);
            }
            float factor = kForm == kDirect ? p.factor : 1.0f, m_ref = -INFINITY, l = 0.0f;
            if (first_part && n_tiles > 0) load_bits(t, tile0, image, L, 0, ahead);
#pragma unroll 1
            for (int i = 0; i < n_tiles; ++i, ++tile) {
                uint2 have = ahead[0];
                const uint2 nan = ahead[1];
                if (i + 1 < n_tiles) load_bits(t, tile0, image, L, i + 1, ahead);
                int see = lim - ((tile0 + i) * kTile + 64 * q4);     // tokens of the quarter the row sees
                if constexpr (kWindow) {
                    if (lim - see >= p.sink_rows) see -= gap;
                    const int skip = see - p.window, keep = min(see, p.sinks - (lim - see));      // (lim - see: the quarter's first)
                    have.x &= (bits_below(see) & ~bits_below(skip)) | bits_below(keep);
                    have.y &= (bits_below(see - 32) & ~bits_below(skip - 32)) | bits_below(keep - 32);
                    see = 64;      // (all in the bits)
                }
                wait_phase(bar(B_S_FULL + (tile & 1)), (tile >> 1) & 1, abort_flag, p.err);
                tc_fence_after();
                if (kForm != kDirect && i == 0) factor = reinterpret_cast<const float*>(smem + SM_QS)[64 * (parts & 3) + row];
                float x[64];
                tmem_ld32(tmem + kTS + 128 * (tile & 1) + 64 * ch + lanes, reinterpret_cast<uint32_t*>(x));
                tmem_ld32(tmem + kTS + 128 * (tile & 1) + 64 * ch + 32 + lanes, reinterpret_cast<uint32_t*>(x) + 32);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) leader_arrive(bar(B_S_FREE + (tile & 1)));
                if (kForm == kDirect && p.turn != 1.0f) {
#pragma unroll
                    for (int k = 0; k < 64; ++k) x[k] *= p.turn;
                }
                if (!__all_sync(0xFFFFFFFFu, see >= 64 && (have.x & have.y) == 0xFFFFFFFFu && (nan.x | nan.y) == 0)) {
#pragma unroll
                    for (int k = 0; k < 64; ++k) {
                        if (((k < 32 ? nan.x : nan.y) >> (k & 31)) & 1u) x[k] = __int_as_float(0x7FFFFFFF);
                        if (k >= see || !(((k < 32 ? have.x : have.y) >> (k & 31)) & 1u)) x[k] = -INFINITY;
                    }
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int k = 0; k < 32; ++k) mx[k & 3] = max3(mx[k & 3], x[2 * k], x[2 * k + 1]);
                float* slot = red + (tile & 1) * 256;
                slot[64 * q4 + row] = factor * fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                named_bar_sync(1 + (sp & 1), 128);
                const float m = fmaxf(fmaxf(slot[row], slot[64 + row]), fmaxf(slot[128 + row], slot[192 + row]));
                float alpha = 1.0f;
                // (a difference: exact near the limit, true of a row's first score, false of equal infinities)
                if (m - m_ref > kRescaleLog2 + kTopLog2) {
                    const float next = m - kTopLog2;
                    alpha = m_ref == -INFINITY ? 0.0f : ex2_approx(m_ref - next);
                    l *= alpha;
                    m_ref = next;
                }
                const float base = m_ref == -INFINITY ? 0.0f : m_ref;
                uint32_t pk[32];
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
                const float2 factor2 = make_float2(factor, factor), base2 = make_float2(-base, -base);
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                    const float2 e = fma2(make_float2(x[2 * k], x[2 * k + 1]), factor2, base2);
                    const float2 w = make_float2(ex2_approx(e.x), ex2_approx(e.y));
                    sum[k & 1] = add2(sum[k & 1], w);
                    pk[k] = pack_half2(w.x, w.y);
                }
                sum[0] = add2(sum[0], sum[1]);
                l += sum[0].x + sum[0].y;
                if (i > 0) {
                    wait_phase(bar(B_PV_DONE), (tile - 1) & 1, abort_flag, p.err);
                    if (__any_sync(0xFFFFFFFFu, alpha != 1.0f)) {          // the row's O: this warp's lanes, block ch
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < 128; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(tmem + kTO + 128 * ch + c + lanes, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                            tmem_st16(tmem + kTO + 128 * ch + c + lanes, o);
                        }
                        tmem_wait_st();
                        tc_fence_before();
                    }
                }
                uint8_t* dst = smem + SM_P + q4 * (kCtaRows * 128) + row * 128;
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    *reinterpret_cast<uint4*>(dst + ((c ^ (row & 7)) << 4)) = make_uint4(pk[4 * c], pk[4 * c + 1], pk[4 * c + 2], pk[4 * c + 3]);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) leader_arrive(bar(B_P_FULL));
            }
            look_ahead<kWindow>(p, work);                        // (the last PV is running)
            __syncwarp();
            if (*reinterpret_cast<volatile int*>(&work->more) && next.n_tiles > 0) load_bits(next, next.tile0, next.image, next.L, 0, ahead);
            // ---- epilogue: sums over the row's four warps, O out of TMEM
            named_bar_sync(1 + (sp & 1), 128);          // the last part's sums are read
            lsum[64 * q4 + row] = l;
            named_bar_sync(1 + (sp & 1), 128);
            l = (lsum[row] + lsum[64 + row]) + (lsum[128 + row] + lsum[192 + row]);
            if (n_tiles > 0) wait_phase(bar(B_PV_DONE), (tile - 1) & 1, abort_flag, p.err);
            tc_fence_after();
            const bool any = l > 0.0f || l != l, whole = t.head && t.tail;
            const int unit_row = t.half * cta + row, grow = t.block * kUnitRows + unit_row;
            const bool real = grow < t.rows && row < t.half;
            const int tok = real ? token_of(p, grow) : 0, head = grow - tok * p.heads;
            const int64_t part_row = (2 * pair + (first_part ? 0 : 1)) * kUnitRows + unit_row;
            const float mul = whole ? (any ? p.out_scale / l : 0.0f) : 1.0f;
            if (q4 == 0 && real) {
                if (!whole)
                    *reinterpret_cast<float2*>(p.part_ml + 2 * part_row) = make_float2(m_ref, l);
                else if (p.lse)
                    p.lse[static_cast<int64_t>(t.first + tok) * p.heads + head] = any ? 0.69314718055994531f * (m_ref + log2f(l)) : -INFINITY;
            }
            if (!whole && threadIdx.x == 0 && cta == 0)
                p.parts[2 * pair + (first_part ? 0 : 1)] = PartInfo{1, t.head, t.tail, 0, t.first, t.rows, t.block, 0};
            // Two pieces a step, 16 dims of each as 32-byte stores by the lanes that hold the rows, the next two
            // on their way from tensor memory.  Rolled up: this code runs once per part, and unrolled its
            // instructions took longer to arrive than to run.  (Whole rows of the output staged in shared
            // memory and stored by warps were no faster.)
            __nv_bfloat16* out = p.out + static_cast<int64_t>(t.first + tok) * p.o_st + static_cast<int64_t>(head) * p.o_sh + 256 * (sp >> 1) + 16 * ch;
            // (chunks of 8 dims, each of all rows: a warp's store is 1 KB in one piece; 4,400 cycles, as rows 6,800)
            float* part_o = p.part_o + (static_cast<int64_t>(2 * pair + (first_part ? 0 : 1)) * 64 + 32 * (sp >> 1) + 2 * ch) * (8 * kUnitRows) + 8 * unit_row;
            const bool wide = (reinterpret_cast<uintptr_t>(p.out) % 32 == 0) && p.o_st % 16 == 0 && p.o_sh % 16 == 0;
            const uint32_t o_addr = tmem + kTO + 128 * ch + lanes;
            uint32_t ahead_o[2][16];      // columns 8 j .. + 16 (dims a = 0 of pieces j, j + 1) and 64 + 8 j .. (a = 1)
            if (n_tiles > 0) {
                tmem_ld16(o_addr, ahead_o[0]);
                tmem_ld16(o_addr + 64, ahead_o[1]);
                tmem_wait_ld();
            }
#pragma unroll 1
            for (int j = 0; j < 8; j += 2) {
                uint32_t o[2][16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    o[0][k] = any ? __float_as_uint(__uint_as_float(ahead_o[0][k]) * mul) : 0u;
                    o[1][k] = any ? __float_as_uint(__uint_as_float(ahead_o[1][k]) * mul) : 0u;
                }
                if (n_tiles > 0 && j < 6) {
                    tmem_ld16(o_addr + 8 * j + 16, ahead_o[0]);
                    tmem_ld16(o_addr + 8 * j + 80, ahead_o[1]);
                }
                if (real) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (whole) {
                            uint32_t w[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                const uint32_t* src = &o[k >> 2][8 * h + 2 * (k & 3)];
                                const __nv_bfloat162 two = __floats2bfloat162_rn(__uint_as_float(src[0]), __uint_as_float(src[1]));
                                w[k] = *reinterpret_cast<const uint32_t*>(&two);
                            }
                            __nv_bfloat16* dst = out + 32 * (j + h);
                            if (wide) {
                                st_global_v8(dst, w);
                            } else {
                                *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
                                *reinterpret_cast<uint4*>(dst + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                            }
                        } else if (any) {
                            st_global_v8(part_o + 4 * (j + h) * (8 * kUnitRows), &o[0][8 * h]);
                            st_global_v8(part_o + (4 * (j + h) + 1) * (8 * kUnitRows), &o[1][8 * h]);
                        }
                    }
                }
                tmem_wait_ld();
            }
            if (n_tiles > 0) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) leader_arrive(bar(B_O_FREE));
                ++parts;
            }
            first_part = false;
        }
        tc_fence_before();
    }
    cluster_sync();
    if (warp == kMmaWarp) pair_tmem_dealloc(tmem, kTmemCols);
}

// Merges the parts of the units that a range's end cut: out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s -
// M) l_s.  A pair whose last part begins a unit has 32 row groups x 4 / kQ blocks here; the unit's
// other parts are the first ones of the pairs after it, up to the one that ends it.  A block takes 4
// rows x 128 kQ dims, so that the chunks it reads are whole 128-byte lines; it is bound by the latency
// of three dependent loads (the parts' records, a pair per thread; their maxima, a row per warp; O).
// kQ = 4 where there are many pairs (8 chunks of new tokens, 74 pairs: 11.5 us against 18.5), kQ = 1
// where four times the blocks find idle SMs (12 pairs: 4.1 against 5.4).
template <int kQ>
__global__ void __launch_bounds__(128) prefill_combine_kernel(const __grid_constant__ PrefillParams p) {
    static_assert(kMaxPairs <= 128, "a pair per thread");
    __shared__ uint32_t used_bits[4], tail_bits[4];
    __shared__ PartInfo head;
    __shared__ int head_part, count_s, parts[kMaxPairs + 1];
    __shared__ float wts[kMaxPairs + 1][4], invs[4];
    const int pair = blockIdx.x / (kUnitRows / kQ), row0 = blockIdx.x % (kUnitRows / kQ) / (4 / kQ) * 4, dim0 = blockIdx.x % (4 / kQ) * 128 * kQ;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    griddep_wait();
    int4 flags = make_int4(0, 0, 0, 0);      // used, head, tail of a later pair's first part
    if (tid > pair && tid < p.pairs) flags = *reinterpret_cast<const int4*>(p.parts + 2 * tid);
    const bool used = flags.x != 0;
    const uint32_t ub = __ballot_sync(0xFFFFFFFFu, used), tb = __ballot_sync(0xFFFFFFFFu, used && flags.z);
    if (lane == 0) {
        used_bits[warp] = ub;
        tail_bits[warp] = tb;
    }
    if (tid == pair) {
        const PartInfo a = p.parts[2 * pair], b = p.parts[2 * pair + 1];
        head = b.used ? b : a;
        head_part = 2 * pair + (b.used ? 1 : 0);
        count_s = 0;
    }
    __syncthreads();
    if (!head.used || !head.head || head.tail) return;
    const int unit_row = head.block * kUnitRows + row0, rows = head.rows;
    if (unit_row >= rows) return;
    // part 0: the head; then the used first parts up to the first that ends the unit (a pair whose
    // range is empty has none)
    bool after_tail = false;
    int rank = 1;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const uint32_t below = w < warp ? 0xFFFFFFFFu : w == warp ? (1u << lane) - 1u : 0u;
        after_tail |= (tail_bits[w] & below) != 0;
        rank += __popc(used_bits[w] & below);
    }
    const bool mine = used && !after_tail;
    if (mine) parts[rank] = 2 * tid;
    if (mine && flags.z) count_s = rank + 1;
    if (tid == 0) parts[0] = head_part;
    __syncthreads();
    // (without a tail, after a timed-out wait, all there are)
    const int count = count_s > 0 ? count_s : 1 + __popc(used_bits[0]) + __popc(used_bits[1]) + __popc(used_bits[2]) + __popc(used_bits[3]);
    {
        // a row per warp: its weights, and what divides it
        const int row = unit_row + warp;
        const int n = row < rows ? count : 0;
        auto ml_of = [&](int i) { return *reinterpret_cast<const float2*>(p.part_ml + 2 * (static_cast<int64_t>(parts[i]) * kUnitRows + row0 + warp)); };
        float m = -INFINITY, l = 0.0f;
#pragma unroll 1
        for (int i = lane; i < n; i += 32) {
            const float2 ml = ml_of(i);
            if (ml.y > 0.0f) m = fmaxf(m, ml.x);
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
#pragma unroll 1
        for (int i = lane; i < count; i += 32) {
            float w = 0.0f;
            if (i < n) {
                const float2 ml = ml_of(i);
                if (ml.y > 0.0f) w = exp2f(ml.x - m);
                if (ml.y != ml.y) w = ml.y;      // a NaN counts whatever its part's maximum, which no NaN raises
                if (w != 0.0f) l += w * ml.y;
            }
            wts[i][warp] = w;
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
        if (lane == 0) {
            const bool any = l > 0.0f || l != l;
            invs[warp] = any ? p.out_scale / l : 0.0f;
            if (p.lse && dim0 == 0 && row < rows)      // (row = token x heads + head)
                p.lse[static_cast<int64_t>(head.first) * p.heads + row] = any ? 0.69314718055994531f * (m + log2f(l)) : -INFINITY;
        }
    }
    __syncthreads();
    const int j = (tid >> 1) & 3, row = unit_row + j, dim = dim0 + 8 * (tid >> 3) + 4 * (tid & 1);      // and dim + 128 q
    const int64_t at = static_cast<int64_t>(dim >> 3) * (8 * kUnitRows) + 8 * (row0 + j) + (dim & 7);
    float4 acc[kQ];
#pragma unroll
    for (int q = 0; q < kQ; ++q) acc[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int kParts = kQ == 1 ? 4 : 2;      // in flight
    for (int k0 = 0; k0 < count; k0 += kParts) {
        float4 v[kParts][kQ];
        float wk[kParts];
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
            wk[k] = k0 + k < count ? wts[k0 + k][j] : 0.0f;
#pragma unroll
            for (int q = 0; q < kQ; ++q) v[k][q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (wk[k] != 0.0f) {      // (a part that saw no token wrote no O)
                const float* src = p.part_o + static_cast<int64_t>(parts[k0 + k]) * (kUnitRows * kLatent) + at;
#pragma unroll
                for (int q = 0; q < kQ; ++q) v[k][q] = *reinterpret_cast<const float4*>(src + q * (16 * 8 * kUnitRows));
            }
        }
#pragma unroll
        for (int k = 0; k < kParts; ++k)
#pragma unroll
            for (int q = 0; q < kQ; ++q) {
                acc[q].x = fmaf(wk[k], v[k][q].x, acc[q].x);
                acc[q].y = fmaf(wk[k], v[k][q].y, acc[q].y);
                acc[q].z = fmaf(wk[k], v[k][q].z, acc[q].z);
                acc[q].w = fmaf(wk[k], v[k][q].w, acc[q].w);
            }
    }
    if (row >= rows) return;
    const float inv = invs[j];
    const int tok = row / p.heads, h = row - tok * p.heads;
    __nv_bfloat16* dst = p.out + static_cast<int64_t>(head.first + tok) * p.o_st + static_cast<int64_t>(h) * p.o_sh + dim;
#pragma unroll
    for (int q = 0; q < kQ; ++q) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(acc[q].x * inv, acc[q].y * inv), hi = __floats2bfloat162_rn(acc[q].z * inv, acc[q].w * inv);
        *reinterpret_cast<uint2*>(dst + 128 * q) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
}

// ------------------------------------------------------------------ few rows in a window
// Single tokens and short drafts over windows leave the kernels above waiting for one another: an image
// that is read once, ranges, and 256-token tiles in pairs.  Here a CTA takes 64 query rows of one sequence
// and a range of the tokens that any of them sees, 128 at a time, from the pool's rows to its part of the
// output: latents and Q to shared memory as fp16, S = Q K^T with M = 128 (its upper half is whatever lies
// behind the rows, and not read), and O^T += V^T P^T, 128 dims at a time, whose 64 columns are the rows:
// the same tile is B of the first product and A of the second.  Parts of a unit meet in a second kernel,
// or in the cluster that they are (few_joined).
//
// What bounds it is the latency of that chain: of 22,600 cycles for 16 single tokens of 64 heads with a
// window of 1,024 (144 CTAs, a tile each), 4,600 until Q and the pool's rows are asked for, 4,800 for them
// to come and be converted, 2,700 for QK, 3,300 for the softmax, 2,000 for PV and 4,600 for the parts (19
// MB) into L2.  With O = P V and 64 rows on M, the upper half of PV was wasted and half of the warps held
// no row of O: 28.3 us a call, now 23.3 (the second kernel's look at the lengths before it waits, and eight
// parts in flight, are 1.1 of that).  The pool's rows of a tile are asked for under the tile before; a
// further tile takes 10,300 cycles (2,200 dequantising, 2,800 QK, 2,500 softmax, whose rows lie in the
// lanes of half of the warps, 2,100 PV).
constexpr int kFewTokens = 128, kFewThreads = 512, kFewMaxParts = 64;
constexpr int SF_Q = 0;                                       // 9 dim atoms x [64 rows x 128 B]
constexpr int SF_KV = SF_Q + 9 * kCtaRows * 128;              // 9 dim atoms x [128 tokens x 128 B]
constexpr int SF_P = SF_KV + 8 * kFewTokens * 128;            // 2 token atoms x [64 rows x 128 B], where the rope part was
constexpr int SF_RED = SF_KV + 9 * kFewTokens * 128;          // 4 x 64 f32: row maxima of the token quarters; 4 x 64: their sums
constexpr int SF_QS = SF_RED + 2 * 4 * 64 * 4;                // 64 f32: score factor of a row, then what O is multiplied by
constexpr int SF_ALPHA = SF_QS + 64 * 4;                      // 64 f32: what O is multiplied by before a tile
constexpr int SF_BITS = SF_ALPHA + 64 * 4;                    // 4 words of tokens that exist, 4 of those with a NaN
constexpr int SF_FLAGS = SF_BITS + 32;                        // [0] TMEM base, [1] abort
constexpr int SF_BARS = SF_FLAGS + 16;                        // [0] S complete, [1] O complete, [2] everything
constexpr int kFewSmemBytes = SF_BARS + 24 + 1024;
static_assert(kFewSmemBytes <= 232448, "shared memory budget");
static_assert(2 * kCtaRows * 128 <= kFewTokens * 128, "P takes the rope part's place");
constexpr uint32_t kIdescFewQk = idesc_f16_f32(128, kFewTokens, false, false);
constexpr uint32_t kIdescFewRope = kIdescFewQk | (1u << 7) | (1u << 10);
constexpr uint32_t kIdescFewPv = idesc_f16_f32(128, kCtaRows, true, false);
constexpr uint32_t kTFewO = 128;                              // TMEM: S, then O^T in four blocks of 128 dims x 64 rows
constexpr int kFewGroup = 8;                                  // rows that lie together in a part, and of a block that merges
// The dim of lane l of O^T's block m: atom c / 64, column c % 64 of c = 128 m + l.
__device__ __forceinline__ int few_dim(int c) { return 256 * (c >> 8) + 32 * ((c >> 3) & 7) + 8 * ((c >> 6) & 3) + (c & 7); }

// What 64 rows from row 64 k on see: the first `sinks` tokens, then [lo, end).
struct FewUnit {
    int rows;             // of the unit
    int sinks, lo, end;
    int tokens, tiles, parts;    // both >= 1; part s: tiles [s tiles / parts, (s + 1) tiles / parts)
};
__device__ __forceinline__ FewUnit few_unit(const PrefillParams& p, const Seq& s, int k, int most) {
    FewUnit u;
    const int r0 = kCtaRows * k, last = min(s.rows, r0 + kCtaRows) - 1;
    u.rows = last + 1 - r0;
    u.end = max(0, min(s.L, s.L - s.n + token_of(p, last) + 1));
    u.lo = max(0, min(u.end, s.L - s.n + token_of(p, r0) + 1 - p.window));
    u.sinks = min(p.sinks, u.lo);
    u.tokens = u.sinks + u.end - u.lo;
    u.tiles = max(1, (u.tokens + kFewTokens - 1) / kFewTokens);
    u.parts = min(u.tiles, most);
    return u;
}

constexpr int kFewJoined = 8;                                 // parts of a unit whose CTAs are a cluster, at most
constexpr int kFewPieces = 8;                                 // a CTA's share of the merge: eight rows of another's part each
__device__ __forceinline__ void tmem_ld8(uint32_t addr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(addr));
}

// Block x = part + few_parts (unit + few_units sequence).  Part s of a unit, when there are several, goes
// to part_o [unit][few_parts][8 groups of rows][512 (as few_dim)][8 rows] and part_ml [unit][few_parts][64][2].
// kJoined: the parts of a unit are a cluster, and each merges its share of the unit's rows.
template <bool kJoined>
__global__ void __launch_bounds__(kFewThreads, 1) mla_window_few_kernel(const __grid_constant__ PrefillParams p, int few_units, int few_parts) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const uint32_t sbase = smem_u32(smem);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int part = blockIdx.x % few_parts, unit = blockIdx.x / few_parts, k = unit % few_units, b = unit / few_units;
    volatile int* flags = reinterpret_cast<volatile int*>(smem + SF_FLAGS);
    volatile int* abort_flag = flags + 1;
    uint32_t* bits = reinterpret_cast<uint32_t*>(smem + SF_BITS);
    const uint32_t bar = sbase + SF_BARS;
    // (what needs no input comes before the wait: 0.5 us of 16)
    if (tid < 8) bits[tid] = 0;
    if (tid == 32) {
        flags[1] = 0;
        mbar_init(bar, 1);
        mbar_init(bar + 8, 1);
        mbar_init(bar + 16, 1);
        mbar_fence_init();
    }
    if (warp == 2) {
        tmem_alloc(sbase + SF_FLAGS, kTmemCols);
        tmem_relinquish();
    }
    __syncthreads();
    const uint32_t tmem = static_cast<uint32_t>(flags[0]);
    griddep_wait();                   // first: the kernel that starts now reads the lengths at once
    griddep_launch_dependents();
    const Seq seq = load_seq(p, b);
    FewUnit u;
    u.parts = 0;
    if (kCtaRows * k < seq.rows) u = few_unit(p, seq, k, few_parts);
    if (part >= u.parts) {
        if (warp == 2) tmem_dealloc(tmem, kTmemCols);
        return;
    }
    const int tile0 = part * u.tiles / u.parts, tile1 = (part + 1) * u.tiles / u.parts;
    // Q on its way
    Part t;
    t.block = k >> 1;
    t.half = kCtaRows;
    t.rows = seq.rows;
    t.first = seq.first;
    QRows q;
    load_q(p, t, k & 1, warp, kFewThreads / 32, q);
    // a tile's pool rows: eight threads a row, two rows a thread
    const int lp = tid & 7, r0 = tid >> 3;
    uint4 code[2][2], rope[2];
    uint16_t scale[2][2];
    bool have[2];
    auto load_rows = [&](int tile) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int l = kFewTokens * tile + r0 + 64 * i, pos = l < u.sinks ? l : u.lo + l - u.sinks;
            const int64_t row = l < u.tokens ? pool_row(p, p.tables + b * p.tables_stride, pos, u.end) : -1;
            have[i] = row >= 0;
            if (l < u.tokens && row < 0 && lp == 0) set_error(p.err, NVFP4KV_DEVERR_BAD_PAGE);
            rope[i] = code[i][0] = code[i][1] = make_uint4(0, 0, 0, 0);
            scale[i][0] = scale[i][1] = 0;
            if (have[i]) {
                const uint8_t* src = p.pool + row * kRowBytes;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    code[i][h] = ldg_nc_v4(src + 128 * h + 16 * lp);
                    scale[i][h] = __ldg(reinterpret_cast<const uint16_t*>(src + 256 + 16 * h + 2 * lp));
                }
                if (p.rope) rope[i] = ldg_nc_v4(p.rope + row * kRope + 8 * lp);
            }
        }
    };
    load_rows(tile0);
    store_q(p, smem + SF_Q, reinterpret_cast<float*>(smem + SF_QS), warp, kFewThreads / 32, q);
    // softmax: eight warps, 32 rows x 32 tokens each (a row's quarters in warps 4 apart)
    const int sp = warp & 3, cg = warp >> 2, row = 32 * (sp & 1) + lane;
    const uint32_t lanes = static_cast<uint32_t>(32 * (sp & 1)) << 16;
    // O: a dim of 64 rows a thread (warp: lanes 32 sp .. of block cg)
    const int c = 128 * cg + 32 * sp + lane;
    const uint32_t o_addr = tmem + kTFewO + kCtaRows * cg + (static_cast<uint32_t>(32 * sp) << 16);
    float* red = reinterpret_cast<float*>(smem + SF_RED);
    float* alphas = reinterpret_cast<float*>(smem + SF_ALPHA);
    int lim = 0;
    if (row < u.rows) lim = min(seq.L, seq.L - seq.n + token_of(p, kCtaRows * k + row) + 1);
    float factor = 1.0f, m_ref = -INFINITY, l = 0.0f;
    const bool any_tokens = u.tokens > 0;      // (without, one tile of nothing, and no PV)
#pragma unroll 1
    for (int tile = tile0; tile < tile1; ++tile) {
        const int u0 = kFewTokens * tile;
        const uint32_t phase = (tile - tile0) & 1;
        // the first tile by halves of the latent dims, the first one's QK under the second's conversion (a call of
        // one tile a CTA 17.3 -> 16.9 us; later tiles so too were slower, 256 single tokens 115 -> 119)
        const bool halves = tile == tile0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = r0 + 64 * i;
                uint8_t* dst = smem + SF_KV + r * 128 + ((lp ^ (r & 7)) << 4);
                const uint32_t word[4] = {code[i][h].x, code[i][h].y, code[i][h].z, code[i][h].w};
                const uint32_t s2 = e4m3x2_to_f16x2(scale[i][h]);
                bool nan = false;
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const bool bad = ((scale[i][h] >> (a & 2 ? 8 : 0)) & 0x7F) == 0x7F;
                    nan |= bad;
                    const uint4 v = dequant8(word[a], __byte_perm(s2, s2, a & 2 ? 0x3232 : 0x1010));
                    *reinterpret_cast<uint4*>(dst + (4 * h + a) * (kFewTokens * 128)) = bad ? make_uint4(0, 0, 0, 0) : v;
                }
                if (nan) atomicOr(&bits[4 + (r >> 5)], 1u << (r & 31));
                if (h == 0) {
                    if (p.rope) *reinterpret_cast<uint4*>(dst + 8 * (kFewTokens * 128)) = rope[i];
                    if (lp == 0 && have[i]) atomicOr(&bits[r >> 5], 1u << (r & 31));
                }
            }
            if (h == 0 && !halves) continue;
            fence_proxy_async_smem();
            tc_fence_before();
            __syncthreads();
            tc_fence_after();
            if (warp == 2) {
                if (elect_one()) {
                    const uint64_t dq = smem_desc_sw128(sbase + SF_Q, 16, 1024), dk = smem_desc_sw128(sbase + SF_KV, 16, 1024);
                    auto atom = [&](int j) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            tc_mma_f16(tmem, dq + ((j * kCtaRows * 128) >> 4) + 2 * i, dk + ((j * kFewTokens * 128) >> 4) + 2 * i,
                                       j == 8 ? kIdescFewRope : kIdescFewQk, j > 0 || i > 0);
                    };
                    for (int j = halves ? 4 * h : 0; j < 4 * h + 4; ++j) atom(j);
                    if (h == 1) {
                        if (p.rope) atom(8);
                        tc_commit(bar);
                    }
                }
                __syncwarp();
            }
        }
        if (tile + 1 < tile1) load_rows(tile + 1);
        mbar_wait(bar, phase, abort_flag, p.err);
        tc_fence_after();
        float alpha = 1.0f;
        if (sp < 2) {
            if (tile == tile0) factor = reinterpret_cast<const float*>(smem + SF_QS)[row];
            float x[32];
            tmem_ld32(tmem + 32 * cg + lanes, reinterpret_cast<uint32_t*>(x));
            tmem_wait_ld();
            // local tokens before `sinks` lie at their own positions, the others `off` further
            const int l0 = u0 + 32 * cg, off = l0 + u.lo - u.sinks;
            const uint32_t first = bits_below(u.sinks - l0);
            const uint32_t see = bits[cg] & ((first & bits_below(lim - l0)) |
                                             (~first & bits_below(lim - off) & (~bits_below(lim - p.window - off) | bits_below(p.sinks - off))));
            const uint32_t nan = bits[4 + cg];
            if (!__all_sync(0xFFFFFFFFu, see == 0xFFFFFFFFu && nan == 0)) {
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    if ((nan >> i) & 1u) x[i] = __int_as_float(0x7FFFFFFF);
                    if (!((see >> i) & 1u)) x[i] = -INFINITY;
                }
            }
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 16; ++i) mx[i & 1] = max3(mx[i & 1], x[2 * i], x[2 * i + 1]);
            float m = fmaxf(mx[0], mx[1]);
            red[64 * cg + row] = factor * m;
            named_bar_sync(1, 256);
            m = fmaxf(fmaxf(red[row], red[64 + row]), fmaxf(red[128 + row], red[192 + row]));
            // (as in the kernel above: the reference moves when a tile passes it by 2^8)
            if (m - m_ref > kRescaleLog2 + kTopLog2) {
                const float next = m - kTopLog2;
                alpha = m_ref == -INFINITY ? 0.0f : ex2_approx(m_ref - next);
                l *= alpha;
                m_ref = next;
            }
            const float base = m_ref == -INFINITY ? 0.0f : m_ref;
            uint32_t pk[16];
            float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
            const float2 factor2 = make_float2(factor, factor), base2 = make_float2(-base, -base);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 e = fma2(make_float2(x[2 * i], x[2 * i + 1]), factor2, base2);
                const float2 w = make_float2(ex2_approx(e.x), ex2_approx(e.y));
                sum[i & 1] = add2(sum[i & 1], w);
                pk[i] = pack_half2(w.x, w.y);
            }
            sum[0] = add2(sum[0], sum[1]);
            l += sum[0].x + sum[0].y;
            uint8_t* dst = smem + SF_P + (cg >> 1) * (kCtaRows * 128) + row * 128;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<uint4*>(dst + (((4 * (cg & 1) + i) ^ (row & 7)) << 4)) = make_uint4(pk[4 * i], pk[4 * i + 1], pk[4 * i + 2], pk[4 * i + 3]);
            if (cg == 0) alphas[row] = alpha;
            fence_proxy_async_smem();
        }
        tc_fence_before();
        const bool moved = __syncthreads_or(tile > tile0 && alpha != 1.0f);
        tc_fence_after();
        if (tid < 8) bits[tid] = 0;       // (read by all; the next tile's are set behind a barrier)
        if (moved) {                      // (the PV before is complete: the tile's latents came after it)
#pragma unroll 1
            for (int g = 0; g < kCtaRows; g += 16) {
                uint32_t o[16];
                tmem_ld16(o_addr + g, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alphas[g + i]);
                tmem_st16(o_addr + g, o);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncthreads();
            tc_fence_after();
        }
        if (!any_tokens) break;
        if (warp == 2) {
            if (elect_one()) {
                const uint64_t dp = smem_desc_sw128(sbase + SF_P, 16, 1024);
                const int steps = (min(kFewTokens, u.tokens - u0) + 15) / 16;
#pragma unroll 1
                for (int m = 0; m < 4; ++m) {
                    const uint64_t dv = smem_desc_sw128(sbase + SF_KV + 2 * m * (kFewTokens * 128), kFewTokens * 128, 1024);
                    for (int i = 0; i < steps; ++i)
                        tc_mma_f16(tmem + kTFewO + kCtaRows * m, dv + 128 * i, dp + (((i >> 2) * kCtaRows * 128) >> 4) + 2 * (i & 3), kIdescFewPv,
                                   tile > tile0 || i > 0);
                }
                tc_commit(bar + 8);
            }
            __syncwarp();
        }
        if (tile + 1 < tile1) {
            mbar_wait(bar + 8, phase, abort_flag, p.err);
            tc_fence_after();
            __syncthreads();              // (the bits are clear)
        }
    }
    if (sp < 2) red[256 + 64 * cg + row] = l;
    __syncthreads();
    const bool whole = u.parts == 1;
    const int64_t slot = static_cast<int64_t>(unit) * few_parts + part;
    float* mul = reinterpret_cast<float*>(smem + SF_QS);
    if (sp < 2 && cg == 0) {
        l = (red[256 + row] + red[320 + row]) + (red[384 + row] + red[448 + row]);
        const bool any = l > 0.0f || l != l;
        mul[row] = any ? p.out_scale / l : 0.0f;
        if (row < u.rows) {
            if (!whole) *reinterpret_cast<float2*>(p.part_ml + 2 * (slot * kCtaRows + row)) = make_float2(m_ref, l);
            else if (p.lse)      // (row = token x heads + head)
                p.lse[static_cast<int64_t>(seq.first) * p.heads + kCtaRows * k + row] = any ? 0.69314718055994531f * (m_ref + log2f(l)) : -INFINITY;
        }
    }
    if (any_tokens) mbar_wait(bar + 8, (tile1 - 1 - tile0) & 1, abort_flag, p.err);
    tc_fence_after();
    __syncthreads();
    // kJoined: CTA `part` merges row groups part, part + parts ...: its own share of them is still in tensor
    // memory, the others' are asked for, up to eight pieces at a time, before the weights are known.
    auto join_parts = [&] {
        const int parts = u.parts, others = parts - 1, groups = (u.rows + kFewGroup - 1) / kFewGroup;
        const int mine = groups > part ? (groups - part + parts - 1) / parts : 0, pieces = mine * others;
        const int64_t slot0 = static_cast<int64_t>(unit) * few_parts;
        float* wts = reinterpret_cast<float*>(smem + SF_Q);      // [row][part]
        float* invs = wts + kCtaRows * kFewJoined;
        __nv_bfloat16* rows = reinterpret_cast<__nv_bfloat16*>(smem + SF_KV);
        float4 v[kFewPieces][2];
        int at_g = 0, at_s = 0;         // of the next piece
        auto ask = [&](int first) {
#pragma unroll
            for (int j = 0; j < kFewPieces; ++j) {
                if (first + j < pieces) {
                    const int s = at_s + (at_s >= part);
                    const float4* src = reinterpret_cast<const float4*>(
                        p.part_o + (((slot0 + s) * (kCtaRows / kFewGroup) + part + at_g * parts) * kLatent + c) * kFewGroup);
                    v[j][0] = __ldcg(src);
                    v[j][1] = __ldcg(src + 1);
                }
                if (++at_s == others) {
                    at_s = 0;
                    ++at_g;
                }
            }
        };
        ask(0);
        {      // weights of all rows: eight parts of four rows a warp
            const int r = 4 * warp + (lane >> 3), s = lane & 7;
            const bool real = r < u.rows;
            float2 ml = make_float2(-INFINITY, 0.0f);
            if (real && s < parts) ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml + 2 * ((slot0 + s) * kCtaRows + r)));
            float m = ml.y > 0.0f ? ml.x : -INFINITY;
#pragma unroll
            for (int o = 4; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
            float w = ml.y > 0.0f ? exp2f(ml.x - m) : 0.0f;
            if (ml.y != ml.y) w = ml.y;      // a NaN counts whatever its part's maximum, which no NaN raises
            float sum = w != 0.0f ? w * ml.y : 0.0f;
#pragma unroll
            for (int o = 4; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            wts[r * kFewJoined + s] = w;
            if (s == 0) {
                const bool any = sum > 0.0f || sum != sum;
                invs[r] = any ? p.out_scale / sum : 0.0f;
                if (p.lse && real && part == 0)      // (row = token x heads + head)
                    p.lse[static_cast<int64_t>(seq.first) * p.heads + kCtaRows * k + r] = any ? 0.69314718055994531f * (m + log2f(sum)) : -INFINITY;
            }
        }
        __syncthreads();
        float acc[kFewGroup];
        int g = 0, s = 0;
#pragma unroll 1
        for (int first = 0; first < pieces; first += kFewPieces) {
            if (first > 0) ask(first);
#pragma unroll
            for (int j = 0; j < kFewPieces; ++j) {
                if (first + j < pieces) {
                    const float* w = wts + kFewGroup * (part + g * parts) * kFewJoined;
                    if (s == 0) {
                        uint32_t o[8];
                        tmem_ld8(o_addr + kFewGroup * (part + g * parts), o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < kFewGroup; ++i) acc[i] = w[i * kFewJoined + part] * __uint_as_float(o[i]);
                    }
                    const int from = s + (s >= part);
                    const float x[kFewGroup] = {v[j][0].x, v[j][0].y, v[j][0].z, v[j][0].w, v[j][1].x, v[j][1].y, v[j][1].z, v[j][1].w};
#pragma unroll
                    for (int i = 0; i < kFewGroup; ++i) acc[i] = fmaf(w[i * kFewJoined + from], x[i], acc[i]);
                    if (++s == others) {
#pragma unroll
                        for (int i = 0; i < kFewGroup; ++i)
                            rows[(kFewGroup * g + i) * kLatent + few_dim(c)] = __float2bfloat16_rn(acc[i] * invs[kFewGroup * (part + g * parts) + i]);
                        s = 0;
                        ++g;
                    }
                }
            }
        }
        __syncthreads();
        for (int i = tid; i < mine * kFewGroup * (kLatent / 8); i += kFewThreads) {
            const int r = i / (kLatent / 8), d = 8 * (i % (kLatent / 8)), row = kFewGroup * (part + r / kFewGroup * parts) + r % kFewGroup;
            if (row >= u.rows) continue;
            const int grow = kCtaRows * k + row, tok = token_of(p, grow), head = grow - tok * p.heads;
            *reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(seq.first + tok) * p.o_st + static_cast<int64_t>(head) * p.o_sh + d) =
                *reinterpret_cast<const uint4*>(rows + r * kLatent + d);
        }
    };
    if (!whole) {
        float* dst = p.part_o + (slot * (kCtaRows / kFewGroup) * kLatent + c) * kFewGroup;
#pragma unroll
        for (int g = 0; g < kCtaRows / kFewGroup; g += 4) {
            uint32_t o[32];
            tmem_ld32(o_addr + kFewGroup * g, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!kJoined || (g + i) % u.parts != part) st_global_v8(dst + (g + i) * (kLatent * kFewGroup), o + 8 * i);
        }
        if constexpr (kJoined) {
            cluster_sync();
            join_parts();
        }
    } else {
        // through shared memory (the latents' place: every product is done) to rows of the output
        __nv_bfloat16* rows = reinterpret_cast<__nv_bfloat16*>(smem + SF_KV);
        const int dim = few_dim(c);
#pragma unroll
        for (int g = 0; g < kCtaRows; g += 32) {
            uint32_t o[32];
            tmem_ld32(o_addr + g, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i)
                rows[(g + i) * kLatent + dim] = __float2bfloat16_rn(any_tokens ? __uint_as_float(o[i]) * mul[g + i] : 0.0f);
        }
        __syncthreads();
        for (int i = tid; i < u.rows * (kLatent / 8); i += kFewThreads) {
            const int r = i / (kLatent / 8), d = 8 * (i % (kLatent / 8)), grow = kCtaRows * k + r, tok = token_of(p, grow), head = grow - tok * p.heads;
            *reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(seq.first + tok) * p.o_st + static_cast<int64_t>(head) * p.o_sh + d) =
                *reinterpret_cast<const uint4*>(rows + r * kLatent + d);
        }
    }
    tc_fence_before();
    if (warp == 2) {      // (after a timed-out wait products may be in flight: they end before their memory goes)
        if (elect_one()) tc_commit(bar + 16);
        __syncwarp();
        mbar_drain_wait(bar + 16, 0);
    }
    __syncthreads();
    if (warp == 2) tmem_dealloc(tmem, kTmemCols);
}

// Merges the parts of the units that have several: eight rows of a unit a block, a row's weights by a warp,
// a dim of the rows by a thread.
__global__ void __launch_bounds__(kLatent) mla_window_few_combine_kernel(const __grid_constant__ PrefillParams p, int few_units, int few_parts) {
    __shared__ float wts[kFewMaxParts][kFewGroup], invs[kFewGroup];
    __shared__ __align__(16) __nv_bfloat16 rows[kFewGroup][kLatent];
    constexpr int kGroups = kCtaRows / kFewGroup;
    const int unit = blockIdx.x / kGroups, group = blockIdx.x % kGroups, k = unit % few_units, b = unit / few_units;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    griddep_launch_dependents();
    // (the lengths were there before the kernel before this one)
    const Seq seq = load_seq(p, b);
    const int grow0 = kCtaRows * k + kFewGroup * group;
    FewUnit u;
    u.parts = 1;
    if (grow0 < seq.rows) u = few_unit(p, seq, k, few_parts);
    griddep_wait();                   // whatever there is to merge: this grid ends after the one before it
    if (u.parts == 1) return;
    const int64_t slot0 = static_cast<int64_t>(unit) * few_parts;
    if (warp < kFewGroup) {
        const bool real = grow0 + warp < seq.rows;
        float2 ml[kFewMaxParts / 32];
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int i = 0; i < kFewMaxParts / 32; ++i) {
            const int s = 32 * i + lane;
            ml[i] = make_float2(-INFINITY, 0.0f);
            if (real && s < u.parts) ml[i] = *reinterpret_cast<const float2*>(p.part_ml + 2 * ((slot0 + s) * kCtaRows + kFewGroup * group + warp));
            if (ml[i].y > 0.0f) m = fmaxf(m, ml[i].x);
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
#pragma unroll
        for (int i = 0; i < kFewMaxParts / 32; ++i) {
            float w = ml[i].y > 0.0f ? exp2f(ml[i].x - m) : 0.0f;
            if (ml[i].y != ml[i].y) w = ml[i].y;      // a NaN counts whatever its part's maximum, which no NaN raises
            if (w != 0.0f) l += w * ml[i].y;
            wts[32 * i + lane][warp] = w;
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
        if (lane == 0) {
            const bool any = l > 0.0f || l != l;
            invs[warp] = any ? p.out_scale / l : 0.0f;
            if (p.lse && real)      // (row = token x heads + head)
                p.lse[static_cast<int64_t>(seq.first) * p.heads + grow0 + warp] = any ? 0.69314718055994531f * (m + log2f(l)) : -INFINITY;
        }
    }
    __syncthreads();
    float acc[kFewGroup] = {};
    const float* src = p.part_o + ((slot0 * kGroups + group) * kLatent + tid) * kFewGroup;
#pragma unroll 8
    for (int s = 0; s < u.parts; ++s) {
        const float4 a = *reinterpret_cast<const float4*>(src + static_cast<int64_t>(s) * (kCtaRows * kLatent));
        const float4 c = *reinterpret_cast<const float4*>(src + static_cast<int64_t>(s) * (kCtaRows * kLatent) + 4);
        const float v[kFewGroup] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < kFewGroup; ++i) acc[i] = fmaf(wts[s][i], v[i], acc[i]);
    }
#pragma unroll
    for (int i = 0; i < kFewGroup; ++i) rows[i][few_dim(tid)] = __float2bfloat16_rn(acc[i] * invs[i]);
    __syncthreads();
    const int r = tid / (kLatent / 8), d = 8 * (tid % (kLatent / 8)), row = grow0 + r;
    if (row >= seq.rows) return;
    const int tok = token_of(p, row), head = row - tok * p.heads;
    *reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(seq.first + tok) * p.o_st + static_cast<int64_t>(head) * p.o_sh + d) =
        *reinterpret_cast<const uint4*>(&rows[r][d]);
}

struct PrefillPlan {
    int group;               // sequences per pass over the workspace
    int pairs, image_blocks;
    int sink_rows, max_tiles;
    Form form;
    int few_units, few_parts;   // > 0: units a sequence and parts a unit of the kernels for few rows
    size_t image_bytes, bits_bytes, q_bytes, o_bytes, ml_bytes, ws_bytes;
};

// Images take at most this, or one sequence's; a larger batch runs in groups of sequences.
constexpr size_t kImageCap = size_t(1) << 30;

constexpr int64_t kFewWaves = 2;

// Sequences end here at the latest: a position and what its tile, its image block or the rounding of a unit's end
// adds to it (up to 256) stay an int.  A multiple of every page size.
constexpr int kMostTokens = 0x7FFFF000;

size_t round256(size_t x) { return (x + 255) / 256 * 256; }

PrefillPlan make_prefill_plan(int batch, int total_q, int num_heads, int max_q_len, int max_seq_len, int window, int sinks) {
    PrefillPlan pl{};
    const int64_t longest = max_q_len < total_q ? max_q_len : total_q;
    int64_t tiles = (static_cast<int64_t>(max_seq_len) + kTile - 1) / kTile, image_rows = max_seq_len;
    if (window > 0) {
        // a unit's rows belong to at most `span` tokens, and see no more than the sinks and the window - 1 +
        // span last tokens up to its end, which is rounded up to a multiple of 64
        const int64_t by_rows = (num_heads + kUnitRows - 2) / num_heads + 1, span = by_rows < longest ? by_rows : longest;
        // The kernels for few rows: where no sequence has more than one unit of 64 (single tokens of 64 heads with a
        // window of 1,024: 1 takes 17.0 us there and 19.0 with an image, 16 23.5 and 32, 64 40 and 84, 256 115 and
        // 312; with a window of 16,384 a token takes 40 us either way and 16 of them 103 and 187), or there are no
        // more than kFewWaves tiles an SM (4 x 8 tokens of 16 heads, 512: 16.8 us against 22.3; 8 x 16 of 32, 256,
        // 192 tiles: 22.3 and 27.5; 4 x 16 of 64, 512, 320 tiles: 28.4 and 28.4).  As many parts as there are SMs for.
        const int64_t rows = longest * num_heads, few_units = (rows + kCtaRows - 1) / kCtaRows;
        const int64_t of_64 = (num_heads + kCtaRows - 2) / num_heads + 1, few_span = of_64 < longest ? of_64 : longest;
        int64_t seen = static_cast<int64_t>(sinks) + window - 1 + few_span;
        seen = seen < max_seq_len ? seen : max_seq_len;
        const int64_t few_tiles = seen > kFewTokens ? (seen + kFewTokens - 1) / kFewTokens : 1, all_units = batch * few_units;
        if (few_units == 1 || (few_units > 1 && all_units <= kFewWaves * device_sm_count() / few_tiles)) {
            int64_t parts = all_units > 0 ? device_sm_count() / all_units : 1;
            parts = parts < 1 ? 1 : parts > kFewMaxParts ? kFewMaxParts : parts;
            pl.few_parts = static_cast<int>(parts < few_tiles ? parts : few_tiles);
            pl.few_units = static_cast<int>(few_units);
            const size_t slots = pl.few_parts > 1 ? static_cast<size_t>(all_units) * pl.few_parts : 0;
            pl.group = batch;
            pl.o_bytes = slots * kCtaRows * kLatent * sizeof(float);
            pl.ml_bytes = round256(slots * kCtaRows * 2 * sizeof(float));
            pl.ws_bytes = pl.o_bytes + pl.ml_bytes;
            return pl;
        }
        pl.sink_rows = (sinks + 63) / 64 * 64;
        const int64_t most = (pl.sink_rows + static_cast<int64_t>(window) - 1 + span + 63 + kTile - 1) / kTile;
        tiles = most < tiles ? most : tiles;
        image_rows = kTile * most + longest < image_rows ? kTile * most + longest : image_rows;
    }
    tiles = tiles < 0x7FFFFFFF / kTile ? tiles : 0x7FFFFFFF / kTile;      // (their tokens are an int on the device)
    pl.max_tiles = static_cast<int>(tiles);
    pl.form = window > 0 ? kDirect : kAll;
    const size_t block_bytes = static_cast<size_t>(pl.form == kDirect ? 17 : 9) * kStageBytes;
    const int64_t one = (image_rows + kImageTok - 1) / kImageTok;
    const int64_t cap = static_cast<int64_t>(kImageCap / block_bytes);
    const int64_t fit = one > 0 ? cap / one : batch;
    pl.group = static_cast<int>(fit < 1 ? 1 : (fit < batch ? fit : batch));
    // no more pairs than leave each less than a tile's weight: what a group can have
    const int64_t by_seq = (longest * num_heads + kUnitRows - 1) / kUnitRows * pl.group;
    const int64_t by_rows = (static_cast<int64_t>(total_q) * num_heads + static_cast<int64_t>(pl.group) * (kUnitRows - 1)) / kUnitRows;
    const int64_t units = by_seq < by_rows ? by_seq : by_rows;
    const int64_t most = units * (kUnitWeight + kTileWeight * tiles) / kTileWeight + 1;
    int64_t pairs = device_sm_count() / 2;
    pairs = pairs > kMaxPairs ? kMaxPairs : pairs;
    pairs = pairs > most ? most : pairs;
    pl.pairs = static_cast<int>(pairs < 1 ? 1 : pairs);
    const int64_t blocks = one * pl.group;
    pl.image_blocks = static_cast<int>(blocks);
    pl.image_bytes = static_cast<size_t>(blocks) * block_bytes;
    pl.bits_bytes = round256(static_cast<size_t>(blocks) * 32);
    pl.o_bytes = static_cast<size_t>(pl.pairs) * 2 * kUnitRows * kLatent * sizeof(float);
    pl.ml_bytes = static_cast<size_t>(pl.pairs) * 2 * kUnitRows * 2 * sizeof(float);
    pl.q_bytes = pl.form == kDirect ? 0 : static_cast<size_t>(pl.pairs) * 2 * kQBytes;
    pl.ws_bytes = pl.image_bytes + pl.bits_bytes + pl.q_bytes + pl.o_bytes + pl.ml_bytes + round256(static_cast<size_t>(pl.pairs) * 2 * sizeof(PartInfo));
    return pl;
}

template <auto kKernel>
int set_smem_limit(int bytes) {
    static int done[64] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return fail(NVFP4KV_ECUDA, "cudaGetDevice failed");
    if (dev >= 0 && dev < 64 && done[dev]) return NVFP4KV_OK;
    const cudaError_t e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "mla_prefill: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) done[dev] = 1;
    return NVFP4KV_OK;
}

// The launches of a call, a group of sequences at a time.
template <Form kForm>
int launch_prefill(const PrefillParams& all, const PrefillPlan& pl, cudaStream_t st) {
    int rc = set_smem_limit<mla_prefill_kernel<kForm>>(kSmemBytes);
    if (rc != NVFP4KV_OK) return rc;
    for (int b0 = 0; b0 < all.batch; b0 += pl.group) {
        PrefillParams p = all;
        p.batch = all.batch - b0 < pl.group ? all.batch - b0 : pl.group;
        p.tables = all.tables + b0 * all.tables_stride;
        p.cu = all.cu + b0;
        p.seq_lens = all.seq_lens + b0;
        const dim3 grid(2 * pl.pairs);
        cudaError_t e = cudaSuccess;
        if (pl.image_blocks > 0) {
            const int most = 8 * device_sm_count();
            const int blocks = kImagePieces * pl.image_blocks;
            e = launch_dependent(prefill_image_kernel<kForm>, dim3(blocks < most ? blocks : most), dim3(256), 0, st, p);
            if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "nvfp4kv_mla_prefill image launch failed: %s", cudaGetErrorString(e));
            // its set-up overlaps the image kernel; all else it reads was there before that one
            e = launch_dependent(mla_prefill_kernel<kForm>, grid, dim3(kThreads), kSmemBytes, st, p);
        } else {
            mla_prefill_kernel<kForm><<<grid, kThreads, kSmemBytes, st>>>(p);
        }
        if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "nvfp4kv_mla_prefill launch failed: %s", cudaGetErrorString(e));
        if ((rc = check_launch("nvfp4kv_mla_prefill")) != NVFP4KV_OK) return rc;
        if (pl.pairs == 1 || pl.max_tiles <= 1) continue;      // no unit can be cut
        if (8 * pl.pairs <= device_sm_count()) e = launch_dependent(prefill_combine_kernel<1>, dim3(pl.pairs * kUnitRows), dim3(128), 0, st, p);
        else e = launch_dependent(prefill_combine_kernel<4>, dim3(pl.pairs * (kUnitRows / 4)), dim3(128), 0, st, p);
        if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "nvfp4kv_mla_prefill combine launch failed: %s", cudaGetErrorString(e));
        if ((rc = check_launch("nvfp4kv_mla_prefill combine")) != NVFP4KV_OK) return rc;
    }
    return NVFP4KV_OK;
}

// How many clusters of n blocks of the kernel for few rows run at once (0: none, or not known).
int few_clusters(int n) {
    static int known[64][kFewJoined + 1];      // (one more than the number)
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    if (known[dev][n] == 0) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(n);
        cfg.blockDim = dim3(kFewThreads);
        cfg.dynamicSmemBytes = kFewSmemBytes;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = n;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int clusters = 0;
        if (cudaOccupancyMaxActiveClusters(&clusters, mla_window_few_kernel<true>, &cfg) != cudaSuccess) {
            (void)cudaGetLastError();
            clusters = 0;
        }
        known[dev][n] = clusters + 1;
    }
    return known[dev][n] - 1;
}

// Whether the parts of a unit run as a cluster and merge themselves.  Where the CTAs fill most of the SMs, the
// second kernel waits for the slowest of all and reads every part while no SM computes: 64 single tokens
// of 64 heads in 2 parts 18.1 us against 20.6, 30 in 4 parts 18.3 against 19.3, 15 in 8 parts 18.6
// against 22.1.  With fewer CTAs it is faster, its rows spread over more SMs (12 CTAs 15.7 against 16.9, 64
// 17.3 against 17.9), and where a CTA's share is more than kFewPieces pieces (16 tokens in 6 parts 19.3
// against 19.6).
bool few_joined(int units, int parts) {
    constexpr int kGroups = kCtaRows / kFewGroup;
    return parts > 1 && parts <= kFewJoined && (kGroups + parts - 1) / parts * (parts - 1) <= kFewPieces &&
           8 * units * parts >= 5 * device_sm_count() && units <= few_clusters(parts);
}

int launch_few(const PrefillParams& p, const PrefillPlan& pl, cudaStream_t st) {
    int rc = set_smem_limit<mla_window_few_kernel<false>>(kFewSmemBytes);
    if (rc == NVFP4KV_OK) rc = set_smem_limit<mla_window_few_kernel<true>>(kFewSmemBytes);
    if (rc != NVFP4KV_OK) return rc;
    const int units = p.batch * pl.few_units;
    cudaError_t e;
    if (few_joined(units, pl.few_parts)) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(units * pl.few_parts);
        cfg.blockDim = dim3(kFewThreads);
        cfg.dynamicSmemBytes = kFewSmemBytes;
        cfg.stream = st;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = pl.few_parts;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        e = cudaLaunchKernelEx(&cfg, mla_window_few_kernel<true>, p, pl.few_units, pl.few_parts);
    } else {
        e = launch_dependent(mla_window_few_kernel<false>, dim3(units * pl.few_parts), dim3(kFewThreads), kFewSmemBytes, st, p, pl.few_units, pl.few_parts);
        if (e == cudaSuccess && pl.few_parts > 1)
            e = launch_dependent(mla_window_few_combine_kernel, dim3(units * (kCtaRows / kFewGroup)), dim3(kLatent), 0, st, p, pl.few_units, pl.few_parts);
    }
    if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "nvfp4kv_mla_prefill_window launch failed: %s", cudaGetErrorString(e));
    return check_launch("nvfp4kv_mla_prefill_window");
}

int workspace_call(int batch, int total_q, int num_heads, int max_q_len, int max_seq_len, int window, int sinks, size_t* bytes) {
    if (!bytes) return fail(NVFP4KV_EINVAL, "mla_prefill_workspace_size: null output");
    if (batch < 0 || total_q < 0 || num_heads < 1 || max_q_len < 0 || max_seq_len < 0)
        return fail(NVFP4KV_EINVAL, "mla_prefill_workspace_size: batch, total_q, max_q_len and max_seq_len must be >= 0, num_heads >= 1");
    *bytes = batch == 0 || total_q == 0 ? 0 : make_prefill_plan(batch, total_q, num_heads, max_q_len, max_seq_len, window, sinks).ws_bytes;
    return NVFP4KV_OK;
}

// nvfp4kv_mla_prefill (window 0) and nvfp4kv_mla_prefill_window
int prefill_call(const void* q, int64_t q_stride_t, int64_t q_stride_h, const uint8_t* pool, int64_t pool_rows,
                 const void* rope_pool, const int32_t* tables, int64_t tables_stride, const int32_t* cu_seqlens_q,
                 const int32_t* seq_lens, int batch, int total_q, int num_heads, int head_dim_qk, int kv_lora_rank,
                 int page_size, int max_q_len, int max_seq_len, int window, int sinks, float bmm1_scale,
                 float bmm2_scale, void* out, int64_t out_stride_t, int64_t out_stride_h, float* lse, void* workspace,
                 size_t workspace_bytes, int32_t* err_flag, nvfp4kv_stream_t stream) {
    if (batch < 0 || total_q < 0) return fail(NVFP4KV_EINVAL, "mla_prefill: batch or total_q < 0");
    if (num_heads < 1 || max_q_len < 0 || max_seq_len < 0)
        return fail(NVFP4KV_EINVAL, "mla_prefill: num_heads must be >= 1, max_q_len and max_seq_len >= 0");
    if (kv_lora_rank != kLatent) return fail(NVFP4KV_EINVAL, "mla_prefill: kv_lora_rank must be 512 (got %d)", kv_lora_rank);
    if (head_dim_qk < (rope_pool ? kDim : kLatent))
        return fail(NVFP4KV_EINVAL, "mla_prefill: head_dim_qk %d too small", head_dim_qk);
    if (page_size <= 0 || (page_size & (page_size - 1)) != 0 || page_size > 4096)
        return fail(NVFP4KV_EINVAL, "mla_prefill: page_size must be a power of two <= 4096 (got %d)", page_size);
    if (batch == 0 || total_q == 0) return NVFP4KV_OK;
    if (!q || !pool || !tables || !cu_seqlens_q || !seq_lens || !out) return fail(NVFP4KV_EINVAL, "mla_prefill: null pointer");
    if (pool_rows <= 0 || pool_rows % page_size || pool_rows > 0x7FFFFFFFll)
        return fail(NVFP4KV_EINVAL, "mla_prefill: pool_rows %lld not a multiple of page_size %d in [1, 2^31)",
                    (long long)pool_rows, page_size);
    if (static_cast<int64_t>(max_q_len) * num_heads > 0x3FFFFFFF || static_cast<int64_t>(total_q) * num_heads > 0x7FFFFFFF)
        return fail(NVFP4KV_EINVAL, "mla_prefill: too many query rows");
    if (reinterpret_cast<uintptr_t>(pool) % 16 || reinterpret_cast<uintptr_t>(q) % 16 ||
        reinterpret_cast<uintptr_t>(rope_pool) % 16 || q_stride_t % 8 || q_stride_h % 8)
        return fail(NVFP4KV_EINVAL, "mla_prefill: pools and q must be 16-byte aligned and q strides multiples of 8");
    if (reinterpret_cast<uintptr_t>(out) % 16 || out_stride_t % 8 || out_stride_h % 8)
        return fail(NVFP4KV_EINVAL, "mla_prefill: out must be 16-byte aligned and its strides multiples of 8");
    const PrefillPlan pl = make_prefill_plan(batch, total_q, num_heads, max_q_len, max_seq_len, window, sinks);
    const size_t need = pl.ws_bytes;
    if (need && (!workspace || workspace_bytes < need))
        return fail(NVFP4KV_EWORKSPACE, "mla_prefill: workspace %zu bytes < %zu required", workspace_bytes, need);
    if (reinterpret_cast<uintptr_t>(workspace) % 256)
        return fail(NVFP4KV_EINVAL, "mla_prefill: workspace must be 256-byte aligned");
    PrefillParams p{};
    p.q = static_cast<const __nv_bfloat16*>(q); p.q_st = q_stride_t; p.q_sh = q_stride_h;
    p.pool = pool; p.rope = static_cast<const uint16_t*>(rope_pool); p.num_pages = pool_rows / page_size;
    p.tables = tables; p.tables_stride = tables_stride; p.cu = cu_seqlens_q; p.seq_lens = seq_lens;
    p.batch = batch; p.total_q = total_q; p.heads = num_heads; p.max_q_len = max_q_len;
    p.max_seq_len = max_seq_len < kMostTokens ? max_seq_len : kMostTokens;
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    p.scale_log2 = bmm1_scale * 1.4426950408889634f; p.out_scale = bmm2_scale;
    p.out = static_cast<__nv_bfloat16*>(out); p.o_st = out_stride_t; p.o_sh = out_stride_h;
    p.lse = lse; p.err = err_flag; p.pairs = pl.pairs;
    p.heads_magic = num_heads > 1 ? static_cast<uint32_t>(((1ull << 32) + num_heads - 1) / num_heads) : 0xFFFFFFFFu;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    p.image = ws;
    p.image_bits = reinterpret_cast<uint32_t*>(ws += pl.image_bytes);
    p.q_scratch = ws += pl.bits_bytes;
    p.part_o = reinterpret_cast<float*>(ws += pl.q_bytes);
    p.part_ml = reinterpret_cast<float*>(ws += pl.o_bytes);
    p.parts = reinterpret_cast<PartInfo*>(ws += pl.ml_bytes);
    p.window = window; p.sinks = sinks; p.sink_rows = pl.sink_rows; p.max_tiles = pl.max_tiles;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    p.turn = p.scale_log2 > 0.0f ? 1.0f : p.scale_log2 < 0.0f ? -1.0f : 0.0f;
    p.factor = p.scale_log2 == 0.0f ? 1.0f : fabsf(p.scale_log2);
    if (pl.few_units > 0) return launch_few(p, pl, st);
    if (pl.form == kDirect) return launch_prefill<kDirect>(p, pl, st);
    return launch_prefill<kAll>(p, pl, st);
}

// A window that hides nothing is none; otherwise it and the sinks lie within max_seq_len.  (2^30 rows are more
// than a GPU's memory holds, so a longer window hides no more, and positions less a window stay an int.)
constexpr int kMaxWindow = 1 << 30;
int check_window(const char* what, int max_seq_len, int* window, int* sinks) {
    if (*window < 1 || *sinks < 0) return fail(NVFP4KV_EINVAL, "%s: window must be >= 1 and sinks >= 0", what);
    *window = *window < kMaxWindow ? *window : kMaxWindow;
    *sinks = *sinks < kMaxWindow ? *sinks : kMaxWindow;
    if (max_seq_len >= 0 && static_cast<int64_t>(*window) + *sinks >= max_seq_len) *window = *sinks = 0;
    return NVFP4KV_OK;
}

}  // namespace
}  // namespace nvfp4kv

extern "C" int nvfp4kv_mla_prefill_workspace_size(int batch, int total_q, int num_heads, int max_q_len,
                                                  int max_seq_len, size_t* bytes) {
    return nvfp4kv::workspace_call(batch, total_q, num_heads, max_q_len, max_seq_len, 0, 0, bytes);
}

extern "C" int nvfp4kv_mla_prefill(const void* q, int64_t q_stride_t, int64_t q_stride_h, const uint8_t* pool,
                                   int64_t pool_rows, const void* rope_pool, const int32_t* tables,
                                   int64_t tables_stride, const int32_t* cu_seqlens_q, const int32_t* seq_lens,
                                   int batch, int total_q, int num_heads, int head_dim_qk, int kv_lora_rank,
                                   int page_size, int max_q_len, int max_seq_len, float bmm1_scale,
                                   float bmm2_scale, void* out, int64_t out_stride_t, int64_t out_stride_h,
                                   float* lse, void* workspace, size_t workspace_bytes, int32_t* err_flag,
                                   nvfp4kv_stream_t stream) {
    return nvfp4kv::prefill_call(q, q_stride_t, q_stride_h, pool, pool_rows, rope_pool, tables, tables_stride, cu_seqlens_q, seq_lens, batch,
                                 total_q, num_heads, head_dim_qk, kv_lora_rank, page_size, max_q_len, max_seq_len, 0, 0,
                                 bmm1_scale, bmm2_scale, out, out_stride_t, out_stride_h, lse, workspace, workspace_bytes, err_flag,
                                 stream);
}

extern "C" int nvfp4kv_mla_prefill_window_workspace_size(int batch, int total_q, int num_heads, int max_q_len,
                                                         int max_seq_len, int window, int sinks, size_t* bytes) {
    const int rc = nvfp4kv::check_window("mla_prefill_window_workspace_size", max_seq_len, &window, &sinks);
    return rc != NVFP4KV_OK ? rc : nvfp4kv::workspace_call(batch, total_q, num_heads, max_q_len, max_seq_len, window, sinks, bytes);
}

extern "C" int nvfp4kv_mla_prefill_window(const void* q, int64_t q_stride_t, int64_t q_stride_h, const uint8_t* pool,
                                          int64_t pool_rows, const void* rope_pool, const int32_t* tables,
                                          int64_t tables_stride, const int32_t* cu_seqlens_q, const int32_t* seq_lens,
                                          int batch, int total_q, int num_heads, int head_dim_qk, int kv_lora_rank,
                                          int page_size, int max_q_len, int max_seq_len, int window, int sinks, float bmm1_scale,
                                          float bmm2_scale, void* out, int64_t out_stride_t, int64_t out_stride_h,
                                          float* lse, void* workspace, size_t workspace_bytes, int32_t* err_flag,
                                          nvfp4kv_stream_t stream) {
    const int rc = nvfp4kv::check_window("mla_prefill_window", max_seq_len, &window, &sinks);
    if (rc != NVFP4KV_OK) return rc;
    return nvfp4kv::prefill_call(q, q_stride_t, q_stride_h, pool, pool_rows, rope_pool, tables, tables_stride, cu_seqlens_q, seq_lens, batch,
                                 total_q, num_heads, head_dim_qk, kv_lora_rank, page_size, max_q_len, max_seq_len, window, sinks,
                                 bmm1_scale, bmm2_scale, out, out_stride_t, out_stride_h, lse, workspace, workspace_bytes, err_flag,
                                 stream);
}
