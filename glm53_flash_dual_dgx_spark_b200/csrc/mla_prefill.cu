// Causal MLA attention of a ragged batch of new tokens over the NVFP4 paged pool.
//
//   x[r, t] = bmm1_scale (q[r, :512] . k[t] + q[r, 512:] . k_rope[t]),  t <= L - n + i(r)
//   out[r] = bmm2_scale sum_t softmax(x[r])_t k[t],   lse[r] = log sum_t exp(x[r, t])
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
constexpr int kWorkBytes = 144;
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
    uint32_t heads_magic;      // ceil(2^32 / heads)
    int pairs;
    float scale_log2, out_scale;
    __nv_bfloat16* out;
    int64_t o_st, o_sh;
    float* lse;
    PartInfo* parts;    // [pairs][2]: the range's first part of a unit, and its last one
    float* part_ml;     // [pairs][2][128][2]: reference (log2 units), sum
    float* part_o;      // [pairs][2][64 chunks of 8 dims][128 rows][8]
    uint8_t* q_scratch; // [pairs][2 CTAs][kQBytes]: the next part's Q
    uint8_t* image;     // [blocks][8 or 9 atoms][128 tokens x 128 B]
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
constexpr uint32_t kIdescRope = kIdescQk | (1u << 7) | (1u << 10);      // both operands bf16
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
__device__ __forceinline__ int image_blocks_of(const Seq& s) {
    return s.units > 0 ? (s.L + kImageTok - 1) / kImageTok : 0;
}
// Tokens that unit k of the sequence sees: those of its last row.
__device__ __forceinline__ int unit_end(const PrefillParams& p, const Seq& s, int k) {
    const int last = min(s.rows, (k + 1) * kUnitRows) - 1;
    return max(0, min(s.L, s.L - s.n + last / p.heads + 1));
}
__device__ __forceinline__ int unit_tiles(const PrefillParams& p, const Seq& s, int k) {
    return (unit_end(p, s, k) + kTile - 1) / kTile;
}
// Weights of the work: a tile, and what a unit adds (its first tile's and its epilogue's latency, about
// 8,700 cycles of a tile's 5,800).  With one tile's weight for a unit, pairs with short units took 9 %
// longer than the mean in a batch of chunks, now 6.
constexpr int kTileWeight = 2, kUnitWeight = 3;
// Weight of the sequence's first K units.  A unit's tiles do not fall with k, so the sum goes over
// tile counts (at most n / 256 + 2 of them), not over units.
__device__ __forceinline__ int64_t weight_before(const PrefillParams& p, const Seq& s, int K) {
    if (K <= 0) return 0;
    const int t0 = unit_tiles(p, s, 0), t1 = unit_tiles(p, s, s.units - 1);
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
};
// Where pair `pair` of p.pairs begins.  Run by one warp, a sequence per lane (and pass, past 32).
__device__ __forceinline__ Range find_range(const PrefillParams& p, int pair) {
    const int lane = threadIdx.x & 31;
    Seq s{};
    int64_t w = 0, total = 0;
    for (int b = lane; b < p.batch; b += 32) {
        s = load_seq(p, b);
        w = weight_before(p, s, s.units);
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
    Range r{hi - lo, 0, 0, 0, 0};
    if (hi <= lo) return r;
    int64_t before = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
        if (p.batch > 32) {       // (else the first pass left them here)
            s = Seq{};
            if (b0 + lane < p.batch) s = load_seq(p, b0 + lane);
            w = weight_before(p, s, s.units);
        }
        const int blocks = image_blocks_of(s);
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
                const uint32_t ok = __ballot_sync(0xFFFFFFFFu, cand < k + len && weight_before(p, t, cand) <= x);
                const int at = 31 - __clz(ok);
                len = min(step, k + len - (k + at * step));
                k += at * step;
            }
            r.k = k;
            r.offset = static_cast<int>(x - weight_before(p, t, k));
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
};
// Tiles in a unit's first `weight`.
__device__ __forceinline__ int tiles_in(int weight) { return max(weight - kUnitWeight, 0) / kTileWeight; }
// The next part of the range; parts without tiles are given only where they are a whole unit (one
// that sees no token).
__device__ __forceinline__ bool next_part_of(const PrefillParams& p, Range& r, Part& t) {
    while (r.left > 0) {
        const Seq s = load_seq(p, r.b);
        const int blocks = image_blocks_of(s);
        if (r.k >= s.units) {
            ++r.b;
            r.k = 0;
            r.offset = 0;
            r.image0 += blocks;
            continue;
        }
        t.end = unit_end(p, s, r.k);
        const int tiles = (t.end + kTile - 1) / kTile;
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
__device__ __forceinline__ void look_ahead(const PrefillParams& p, Work* w) {
    if ((threadIdx.x & 31) == 0) {
        Range r = w->range;
        Part t;
        const bool more = next_part_of(p, r, t);
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
__device__ __forceinline__ bool next_part(const PrefillParams& p, Work* w) {
    __syncwarp();
    look_ahead(p, w);
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

// ------------------------------------------------------------------ image
// The image: every token of the sequences with new ones dequantised, as the ring stages the attention
// kernel copies.  Block = 128 tokens: [8 latent atoms (+ the rope part)][128 tokens x 128 B], 128-byte
// swizzled, zeros for tokens that do not exist and for blocks with a NaN scale (the token's bit says
// so instead: a NaN in V would reach rows that do not see it).  Eight lanes read a row's half (128
// code bytes), a thread writes its 32 dims as 16 bytes to each of four atoms, a warp whole 128-byte
// rows.  The blocks of the grid take pieces of 32 tokens in turn (their number is on the device), a
// row per thread, six blocks on an SM: 24.2 us for 91K tokens (143 MB read and written, 5.9 TB/s;
// with four rows a thread and two blocks 26.6, and 5.4 against 3.4 for 2.4K tokens).
__global__ void __launch_bounds__(256, 6) prefill_image_kernel(const __grid_constant__ PrefillParams p) {
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
                if (b0 + lane < p.batch) blocks = image_blocks_of(load_seq(p, b0 + lane));
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
        const int L = load_seq(p, b_s).L, t = pos_s + r0;
        const int64_t row = pool_row(p, p.tables + b_s * p.tables_stride, t, L);
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
        const int atoms = p.rope ? 9 : 8;
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
                *reinterpret_cast<uint4*>(dst + (4 * h + s) * kStageBytes) = bad ? make_uint4(0, 0, 0, 0) : v;
            }
        }
        if (p.rope) *reinterpret_cast<uint4*>(dst + 8 * kStageBytes) = rope;
        if (nan) atomicOr(&bits[1], 1u << r0);
        if (lp == 0) {
            if (row >= 0) atomicOr(&bits[0], 1u << r0);
            else if (t < L) set_error(p.err, NVFP4KV_DEVERR_BAD_PAGE);
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
            int tok = p.heads == 1 ? row : static_cast<int>(__umulhi(row, p.heads_magic));      // row / heads, or one more
            tok -= tok * p.heads > row;
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

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
mla_prefill_kernel(const __grid_constant__ PrefillParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const uint32_t sbase = smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cta = static_cast<int>(cluster_rank()), pair = blockIdx.x >> 1;
    volatile int* flags = reinterpret_cast<volatile int*>(smem + SM_FLAGS);
    volatile int* abort_flag = flags + 1;
    auto bar = [&](int i) -> uint32_t { return sbase + SM_BARS + 8 * i; };

    if (warp == 0) {
        const Range r = find_range(p, pair);
        if (lane == 0) {
            flags[1] = 0;
            // the range's first part, for every warp, and in `part` the first one with tiles: its Q and
            // its first stages are fetched before the roles begin
            Work* w = reinterpret_cast<Work*>(smem + SM_WORK + kThreads / 32 * kWorkBytes);
            Range r0 = r;
            Part t0;
            const bool more = next_part_of(p, r0, t0);
            w->range = r0;
            w->more = more;
            if (more) w->ahead = t0;
            bool tiles = more && t0.n_tiles > 0;
            while (more && !tiles && next_part_of(p, r0, t0)) tiles = t0.n_tiles > 0;
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
    const int64_t image_bytes = static_cast<int64_t>(k_stages) * kStageBytes;
    auto copy_stage = [&](const Cursor& c, int image, int last, int tile0, int slot) {
        const uint32_t dst = sbase + SM_RING + slot * kStageBytes, landed = bar(B_LAND + slot);
        if (elect_one()) {
            mbar_arrive_expect_tx(landed, kStageBytes);
            if (c.s < k_stages) {
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
    auto last_block = [&](int image, int L) { return image + (L + kImageTok - 1) / kImageTok - 1; };      // (tokens past it are masked)
    int early = 0;                    // stages copied before the roles begin
    if (first->part.n_tiles > 0) {
        const Part& t1 = first->part;
        QRows q;
        constexpr int kWarps = kThreads / 32;
        static_assert(kWarps * kQRows == kCtaRows, "one round of rows");
        load_q(p, t1, cta, warp, kWarps, q);
        if (warp == kCopyWarp0 || warp == kCopyWarp0 + 1) {
            griddep_wait();           // the image kernel's writes
            early = kStages;          // (a tile has more)
            static_assert(kStages < 8 + kVStages, "stages of one tile");
            Cursor c{0, 0, 0};
            for (int u = 0; u < kStages; ++u, advance(c, k_stages, t1.n_tiles))
                if ((u & 1) == warp - kCopyWarp0) copy_stage(c, t1.image, last_block(t1.image, t1.L), t1.tile0, u);
        }
        store_q(p, smem + SM_Q, reinterpret_cast<float*>(smem + SM_QS), warp, kWarps, q);
        fence_proxy_async_smem();
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
#pragma unroll 1
                for (bool more = advance_part(work); more && !*abort_flag; more = next_part(p, work)) {
                    const int n_tiles = t.n_tiles;
                    if (n_tiles == 0) continue;
                    if (parts > 0) mbar_wait(bar(B_Q_FULL), (parts - 1) & 1, abort_flag, p.err);
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
                            if (i < n_tiles) {
                                const int at = tile + i;
                                const uint32_t d = tmem + kTS + 128 * (at & 1);
                                if (at >= 2) mbar_wait(bar(B_S_FREE + (at & 1)), ((at >> 1) - 1) & 1, abort_flag, p.err);
                                tc_fence_after();
#pragma unroll 1
                                for (int j = 0; j < k_stages; ++j)
                                    stage(d, dq + ((j * kCtaRows * 128) >> 4), dk + ((slot * kStageBytes) >> 4), 2, j == 8 ? kIdescRope : kIdescQk, j == 0);
                                pair_commit(bar(B_S_FULL + (at & 1)));
                                if (i == n_tiles - 1) pair_commit(bar(B_Q_FREE));
                            }
                            if (i > 0) {
                                mbar_wait(bar(B_P_FULL), (tile + i - 1) & 1, abort_flag, p.err);
                                if (i == 1 && parts > 0) mbar_wait(bar(B_O_FREE), (parts - 1) & 1, abort_flag, p.err);
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
            for (bool more = advance_part(work); ok && more; more = next_part(p, work)) {
                const int n_tiles = t.n_tiles, total = n_tiles * (k_stages + kVStages), image = t.image, tile0 = t.tile0;
                const int last = last_block(image, t.L);
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
                        copy_stage(c, image, last, tile0, slot);
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
        for (bool more = advance_part(work); more; more = next_part(p, work)) {
            if (t.n_tiles == 0) continue;
            if (parts > 0) {                     // (the first part's is there)
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
#pragma unroll 1
        while (advance_part(work)) {
            const int n_tiles = t.n_tiles, tile0 = t.tile0, image = t.image;
            int lim = 0;                                                      // tokens the row sees
            {
                const int grow = t.block * kUnitRows + t.half * cta + row;    // row of the sequence
                if (grow < t.rows && row < t.half) lim = min(t.L, t.L - t.n + grow / p.heads + 1);
            }
            float factor = 1.0f, m_ref = -INFINITY, l = 0.0f;
            // bits of the quarter's tokens that exist, and of those that hold a NaN, loaded a tile ahead
            auto load_bits = [&](int i, uint2 (&w)[2]) {
                const int tok0 = (tile0 + i) * kTile + 64 * q4;
                const uint32_t* src = p.image_bits + 8 * static_cast<int64_t>(image + min(tok0, t.L - 1) / kImageTok) + ((tok0 & (kImageTok - 1)) >> 5);
                w[0] = *reinterpret_cast<const uint2*>(src);
                w[1] = *reinterpret_cast<const uint2*>(src + 4);
            };
            uint2 ahead[2];
            if (n_tiles > 0) load_bits(0, ahead);
#pragma unroll 1
            for (int i = 0; i < n_tiles; ++i, ++tile) {
                const uint2 have = ahead[0], nan = ahead[1];
                if (i + 1 < n_tiles) load_bits(i + 1, ahead);
                const int see = lim - ((tile0 + i) * kTile + 64 * q4);     // tokens of the quarter the row sees
                wait_phase(bar(B_S_FULL + (tile & 1)), (tile >> 1) & 1, abort_flag, p.err);
                tc_fence_after();
                if (i == 0) factor = reinterpret_cast<const float*>(smem + SM_QS)[64 * (parts & 3) + row];
                float x[64];
                tmem_ld32(tmem + kTS + 128 * (tile & 1) + 64 * ch + lanes, reinterpret_cast<uint32_t*>(x));
                tmem_ld32(tmem + kTS + 128 * (tile & 1) + 64 * ch + 32 + lanes, reinterpret_cast<uint32_t*>(x) + 32);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) leader_arrive(bar(B_S_FREE + (tile & 1)));
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
            look_ahead(p, work);                        // (the last PV is running)
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
            const int tok = real ? grow / p.heads : 0, head = grow - tok * p.heads;
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

struct PrefillPlan {
    int group;               // sequences per pass over the workspace
    int pairs, image_blocks;
    size_t image_bytes, bits_bytes, q_bytes, o_bytes, ml_bytes, ws_bytes;
};

// Images take at most this, or one sequence's; a larger batch runs in groups of sequences.
constexpr size_t kImageCap = size_t(1) << 30;

size_t round256(size_t x) { return (x + 255) / 256 * 256; }

PrefillPlan make_prefill_plan(int batch, int total_q, int num_heads, int max_q_len, int max_seq_len) {
    PrefillPlan pl{};
    const int64_t one = (static_cast<int64_t>(max_seq_len) + kImageTok - 1) / kImageTok;
    const int64_t cap = static_cast<int64_t>(kImageCap / (9 * kStageBytes));
    const int64_t fit = one > 0 ? cap / one : batch;
    pl.group = static_cast<int>(fit < 1 ? 1 : (fit < batch ? fit : batch));
    // no more pairs than leave each less than a tile's weight: what a group can have
    const int64_t longest = max_q_len < total_q ? max_q_len : total_q;
    const int64_t by_seq = (longest * num_heads + kUnitRows - 1) / kUnitRows * pl.group;
    const int64_t by_rows = (static_cast<int64_t>(total_q) * num_heads + static_cast<int64_t>(pl.group) * (kUnitRows - 1)) / kUnitRows;
    const int64_t units = by_seq < by_rows ? by_seq : by_rows;
    const int64_t most = units * (kUnitWeight + kTileWeight * ((static_cast<int64_t>(max_seq_len) + kTile - 1) / kTile)) / kTileWeight + 1;
    int64_t pairs = device_sm_count() / 2;
    pairs = pairs > kMaxPairs ? kMaxPairs : pairs;
    pairs = pairs > most ? most : pairs;
    pl.pairs = static_cast<int>(pairs < 1 ? 1 : pairs);
    const int64_t blocks = one * pl.group;
    pl.image_blocks = static_cast<int>(blocks);
    pl.image_bytes = static_cast<size_t>(blocks) * 9 * kStageBytes;
    pl.bits_bytes = round256(static_cast<size_t>(blocks) * 32);
    pl.o_bytes = static_cast<size_t>(pl.pairs) * 2 * kUnitRows * kLatent * sizeof(float);
    pl.ml_bytes = static_cast<size_t>(pl.pairs) * 2 * kUnitRows * 2 * sizeof(float);
    pl.q_bytes = static_cast<size_t>(pl.pairs) * 2 * kQBytes;
    pl.ws_bytes = pl.image_bytes + pl.bits_bytes + pl.q_bytes + pl.o_bytes + pl.ml_bytes + round256(static_cast<size_t>(pl.pairs) * 2 * sizeof(PartInfo));
    return pl;
}

int set_smem_limit() {
    static int done[64] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return fail(NVFP4KV_ECUDA, "cudaGetDevice failed");
    if (dev >= 0 && dev < 64 && done[dev]) return NVFP4KV_OK;
    const cudaError_t e = cudaFuncSetAttribute(mla_prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "mla_prefill: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) done[dev] = 1;
    return NVFP4KV_OK;
}

}  // namespace
}  // namespace nvfp4kv

extern "C" int nvfp4kv_mla_prefill_workspace_size(int batch, int total_q, int num_heads, int max_q_len,
                                                  int max_seq_len, size_t* bytes) {
    using namespace nvfp4kv;
    if (!bytes) return fail(NVFP4KV_EINVAL, "mla_prefill_workspace_size: null output");
    if (batch < 0 || total_q < 0 || num_heads < 1 || max_q_len < 0 || max_seq_len < 0)
        return fail(NVFP4KV_EINVAL, "mla_prefill_workspace_size: batch, total_q, max_q_len and max_seq_len must be >= 0, num_heads >= 1");
    *bytes = batch == 0 || total_q == 0 ? 0 : make_prefill_plan(batch, total_q, num_heads, max_q_len, max_seq_len).ws_bytes;
    return NVFP4KV_OK;
}

extern "C" int nvfp4kv_mla_prefill(const void* q, int64_t q_stride_t, int64_t q_stride_h, const uint8_t* pool,
                                   int64_t pool_rows, const void* rope_pool, const int32_t* tables,
                                   int64_t tables_stride, const int32_t* cu_seqlens_q, const int32_t* seq_lens,
                                   int batch, int total_q, int num_heads, int head_dim_qk, int kv_lora_rank,
                                   int page_size, int max_q_len, int max_seq_len, float bmm1_scale,
                                   float bmm2_scale, void* out, int64_t out_stride_t, int64_t out_stride_h,
                                   float* lse, void* workspace, size_t workspace_bytes, int32_t* err_flag,
                                   nvfp4kv_stream_t stream) {
    using namespace nvfp4kv;
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
    const PrefillPlan pl = make_prefill_plan(batch, total_q, num_heads, max_q_len, max_seq_len);
    const size_t need = pl.ws_bytes;
    if (need && (!workspace || workspace_bytes < need))
        return fail(NVFP4KV_EWORKSPACE, "mla_prefill: workspace %zu bytes < %zu required", workspace_bytes, need);
    if (reinterpret_cast<uintptr_t>(workspace) % 256)
        return fail(NVFP4KV_EINVAL, "mla_prefill: workspace must be 256-byte aligned");
    PrefillParams p{};
    p.q = static_cast<const __nv_bfloat16*>(q); p.q_st = q_stride_t; p.q_sh = q_stride_h;
    p.pool = pool; p.rope = static_cast<const uint16_t*>(rope_pool); p.num_pages = pool_rows / page_size;
    p.tables = tables; p.tables_stride = tables_stride; p.cu = cu_seqlens_q; p.seq_lens = seq_lens;
    p.batch = batch; p.total_q = total_q; p.heads = num_heads; p.max_q_len = max_q_len; p.max_seq_len = max_seq_len;
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
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    int rc = set_smem_limit();
    if (rc != NVFP4KV_OK) return rc;
    for (int b0 = 0; b0 < batch; b0 += pl.group) {
        p.batch = batch - b0 < pl.group ? batch - b0 : pl.group;
        p.tables = tables + b0 * tables_stride;
        p.cu = cu_seqlens_q + b0;
        p.seq_lens = seq_lens + b0;
        const dim3 grid(2 * pl.pairs);
        cudaError_t e = cudaSuccess;
        if (pl.image_blocks > 0) {
            const int most = 8 * device_sm_count();
            const int blocks = kImagePieces * pl.image_blocks;
            e = launch_dependent(prefill_image_kernel, dim3(blocks < most ? blocks : most), dim3(256), 0, st, p);
            if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "nvfp4kv_mla_prefill image launch failed: %s", cudaGetErrorString(e));
            // its set-up overlaps the image kernel; all else it reads was there before that one
            e = launch_dependent(mla_prefill_kernel, grid, dim3(kThreads), kSmemBytes, st, p);
        } else {
            mla_prefill_kernel<<<grid, kThreads, kSmemBytes, st>>>(p);
        }
        if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "nvfp4kv_mla_prefill launch failed: %s", cudaGetErrorString(e));
        if ((rc = check_launch("nvfp4kv_mla_prefill")) != NVFP4KV_OK) return rc;
        if (pl.pairs == 1 || max_seq_len <= kTile) continue;      // no unit can be cut
        if (8 * pl.pairs <= device_sm_count()) e = launch_dependent(prefill_combine_kernel<1>, dim3(pl.pairs * kUnitRows), dim3(128), 0, st, p);
        else e = launch_dependent(prefill_combine_kernel<4>, dim3(pl.pairs * (kUnitRows / 4)), dim3(128), 0, st, p);
        if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "nvfp4kv_mla_prefill combine launch failed: %s", cudaGetErrorString(e));
        if ((rc = check_launch("nvfp4kv_mla_prefill combine")) != NVFP4KV_OK) return rc;
    }
    return NVFP4KV_OK;
}
