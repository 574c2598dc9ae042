// Causal MLA attention of a ragged batch of new tokens over the NVFP4 paged pool.
//
//   x[r, t] = bmm1_scale (q[r, :512] . k[t] + q[r, 512:] . k_rope[t]),  t <= L - n + i(r)
//   out[r] = bmm2_scale sum_t softmax(x[r])_t k[t],   lse[r] = log sum_t exp(x[r, t])
//
// Rows r = (new token i, head) of one sequence share the latent rows k, which are both keys and
// values, so the kernel is two chained matrix products over 128 rows: S = Q K^T (512 or 576 deep)
// and O = P K (512 wide), 4.3 kFLOP per row and token, on the tensor cores.
//
// Work unit: 128 rows of one sequence x a range of its tokens, run by a pair of CTAs (a cluster
// of two) with cta_group::2 MMAs of M = 128: each CTA holds 64 of the rows.  What decides that is
// tensor memory: fp32 O of 64 rows x 512 is half of an SM's 256 KB, and S of two tiles the other
// half.  M = 128 over a pair runs at the full rate (measured 32 / 64 cycles for N = 128 / 256 at
// K = 16, 4090 multiply-adds a cycle and SM), reads A at half a single CTA's shared-memory traffic
// and each CTA supplies only half of B.  A single CTA with 64 rows on N reaches 48 cycles where 32
// are due: its operands saturate shared memory.
//   QK: B = tokens: CTA c dequantises tokens [128 c, 128 c + 128) of a 256-token tile
//   PV: B = latent dims: CTA c dequantises dims [256 c, 256 c + 256) of all 256 tokens
// so every pool byte is dequantised twice in a pair, by producer warps, straight from global memory
// into 16 KB ring stages (64 dims x 128 tokens, or 128 dims x 64 tokens: the same 128 rows of
// 128 bytes, 128-byte swizzled, one row per thread), four MMAs of 64 cycles a stage.
//
// Numbers: a code times its e4m3 scale is exact in fp16, q is scaled per row by a power of two and
// then exact in fp16 (subnormal tails aside: 2^-35 of the row's largest), the rope part stays
// bf16; products accumulate in fp32.  Probabilities are fp16 (11 bits; V is fp16 already, and
// bf16 would triple the output error), their sums fp32 and of the unrounded values.  A row's maximum moves only when a tile exceeds
// it by 2^8, so O is rarely rescaled and P stays far from fp16's largest value.
//
// Warps: 0-7 softmax (a row's 256 scores over four of them), 8-15 producers, 16 issues MMAs (in
// the leading CTA).  Every wait is bounded (common.cuh).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <math.h>

#include <mutex>

#include "../../include/nvfp4kv_serving.h"
#include "abi_common.h"
#include "common.cuh"
#include "decode_shared.h"

namespace nvfp4kv {
namespace {

constexpr int kRope = NVFP4KV_ROPE;
constexpr int kDim = kLatent + kRope;
constexpr int kUnitRows = 128;                  // query rows of a work unit
constexpr int kCtaRows = 64;
constexpr int kTile = 256;                      // tokens per tile
constexpr int kStages = 7;                      // ring stages with an image,
constexpr int kDirectStages = 3;                // and without: the rest of the ring holds raw rows
constexpr int kStageBytes = 16384;              // 128 rows x 128 B
constexpr int kRawSlots = 3;
constexpr int kRawBytes = 128 * (128 + 16);     // 128 rows: 256 dims' codes and scales (or 64 rope dims)
constexpr int kVStages = 8;                     // V stages of a tile: 4 x 64 tokens x 2 x 128 dims a CTA
static_assert(kRawSlots * kRawBytes + kDirectStages * kStageBytes <= kStages * kStageBytes, "ring area");
constexpr int kSoftmaxWarps = 8, kProducerWarp0 = 8, kProducerWarps = 8, kMmaWarp = 16;
constexpr int kThreads = 20 * 32;
constexpr uint32_t kRegsSoftmax = 152, kRegsProducer = 64, kRegsCtl = 48;
static_assert(256 * kRegsSoftmax + 256 * kRegsProducer + 128 * kRegsCtl <= kThreads * 96,
              "the register split stays within what the block is launched with");
constexpr float kRescaleLog2 = 8.0f;
constexpr int kMaxSplits = 64;
constexpr int kImageTok = 128;                  // tokens of an image block
constexpr int kImageUnits = 2;                  // sequences with at least this many units read an image

constexpr int SM_Q = 0;                                      // 9 dim atoms x [64 rows x 128 B]
constexpr int SM_P = SM_Q + 9 * kCtaRows * 128;              // 4 token atoms x [64 rows x 128 B]
constexpr int SM_RING = SM_P + 4 * kCtaRows * 128;
constexpr int SM_RED = SM_RING + kStages * kStageBytes;      // 2 x 4 x 64 f32: row maxima of the token quarters
constexpr int SM_LSUM = SM_RED + 2 * 4 * 64 * 4;             // 4 x 64 f32
constexpr int SM_QS = SM_LSUM + 4 * 64 * 4;                  // 64 f32: score factor (log2 units) of a row
constexpr int SM_FLAGS = SM_QS + 64 * 4;                     // [0] TMEM base, [1] abort, [2..6] work unit
constexpr int SM_BARS = SM_FLAGS + 32;
constexpr int B_FULL = 0;                      // [kStages] leader: stage written in both CTAs (image: each CTA's own copy landed)
constexpr int B_EMPTY = B_FULL + kStages;      // [kStages] both: the MMAs have read the stage
constexpr int B_S_FULL = B_EMPTY + kStages;    // [2] both: S of a tile complete
constexpr int B_S_FREE = B_S_FULL + 2;         // [2] leader: S read by both CTAs
constexpr int B_P_FULL = B_S_FREE + 2;         // leader: P written in both CTAs
constexpr int B_PV_DONE = B_P_FULL + 1;        // both: O stable, P free
constexpr int B_DRAIN = B_PV_DONE + 1;         // both: every MMA complete
constexpr int B_RAW_FULL = B_DRAIN + 1;        // [kRawSlots] own: raw rows landed
constexpr int B_RAW_EMPTY = B_RAW_FULL + kRawSlots;      // own: the producers have read them
constexpr int kNumBars = B_RAW_EMPTY + kRawSlots;
constexpr int kSmemBytes = SM_BARS + kNumBars * 8 + 1024;    // slack to align the base
static_assert(kSmemBytes <= 232448, "shared memory budget");

// Tensor memory: S of two tiles (lane l < 64: row l, tokens 0..127; lane 64 + l: row l, tokens
// 128..255) and O in two blocks n (lane l < 64: row l, dims 128 n ..; lane 64 + l: dims 256 + 128 n ..).
constexpr uint32_t kTS = 0, kTO = 256, kTmemCols = 512;

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
    int units, splits, box_rows;
    float scale_log2, out_scale;
    __nv_bfloat16* out;
    int64_t o_st, o_sh;
    float* lse;
    float* part_o;      // [splits][units][128][512] with splits > 1
    float* part_ml;     // [splits][units][128][2]: maximum (log2 units), sum
    uint8_t* image;     // [image_blocks][8 or 9 atoms][128 tokens x 128 B]
    uint32_t* image_bits;   // [image_blocks][8]: 128 bits of tokens that exist, 128 of those that hold a NaN
    int image_blocks;
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
// Arrive on the leading CTA's barrier.  What the arrival publishes is this CTA's own shared and
// tensor memory, ordered before it by fence.proxy.async or tcgen05.fence and read by the tensor
// core only, so the plain (CTA-scoped) release does; a cluster-scoped one is a full fence that
// takes about 900 cycles (measured: one per stage held the kernel to 0.38 of its rate).
__device__ __forceinline__ void leader_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_map(bar, 0)) : "memory");
}
__device__ __forceinline__ uint32_t max_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// Instruction descriptors: fp32 accumulators, M = 128 (a pair's rows), N = 256.
constexpr uint32_t kIdescQk = idesc_f16_f32(128, 256, false, false);
constexpr uint32_t kIdescRope = kIdescQk | (1u << 7) | (1u << 10);      // both operands bf16
constexpr uint32_t kIdescPv = idesc_f16_f32(128, 256, false, true);

// Sequence b's new tokens: their first index in q and their number, clamped to what the call says.
__device__ __forceinline__ void query_span(const PrefillParams& p, int b, int* first, int* n) {
    const int lo = max(0, min(__ldg(p.cu + b), p.total_q)), hi = max(lo, min(__ldg(p.cu + b + 1), p.total_q));
    *first = lo;
    *n = min(hi - lo, p.max_q_len);
    if (hi - lo > p.max_q_len) set_error(p.err, NVFP4KV_DEVERR_SEQ_LEN);
}

__device__ __forceinline__ int visible_len(const PrefillParams& p, int b) {
    return max(0, min(__ldg(p.seq_lens + b), p.max_seq_len));
}

// A sequence's share of the work: units, and the image blocks it reads.
__device__ __forceinline__ void shares(const PrefillParams& p, int b, int* first, int* n, int* units, int* blocks) {
    query_span(p, b, first, n);
    *units = (*n * p.heads + kUnitRows - 1) / kUnitRows;
    *blocks = *units >= kImageUnits && p.image_blocks > 0 ? (visible_len(p, b) + kImageTok - 1) / kImageTok : 0;
}

__device__ __forceinline__ int warp_inclusive_sum(int x, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xFFFFFFFFu, x, o);
        if (lane >= o) x += y;
    }
    return x;
}

struct Unit {
    int b, first, n;    // sequence, its first new token in q and their number
    int block;          // kImage: block of the image; else: block of rows
    int image;          // the sequence's first image block, -1 without an image
};

// The `item`-th unit (the last blocks of rows, which see the most tokens, first), or with kImage the
// `item`-th image block.  Run by one warp; false past the last one.
template <bool kImage>
__device__ __forceinline__ bool find_unit(const PrefillParams& p, int item, Unit* u) {
    const int lane = threadIdx.x & 31;
    int image0 = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
        int f = 0, c = 0, units = 0, blocks = 0;
        if (b0 + lane < p.batch) shares(p, b0 + lane, &f, &c, &units, &blocks);
        const int img = image0 + warp_inclusive_sum(blocks, lane);
        // a sequence whose blocks do not all fit has no image
        const bool fits = blocks > 0 && img <= p.image_blocks;
        const int sum = kImage ? img : warp_inclusive_sum(units, lane);
        const uint32_t hit = __ballot_sync(0xFFFFFFFFu, item < sum);
        if (hit) {
            const int w = __ffs(hit) - 1;
            u->b = b0 + w;
            u->first = __shfl_sync(0xFFFFFFFFu, f, w);
            u->n = __shfl_sync(0xFFFFFFFFu, c, w);
            u->image = __shfl_sync(0xFFFFFFFFu, fits ? img - blocks : -1, w);
            u->block = kImage ? item - u->image : __shfl_sync(0xFFFFFFFFu, sum, w) - 1 - item;
            return !kImage || u->image >= 0;
        }
        image0 = __shfl_sync(0xFFFFFFFFu, img, 31);
        if (!kImage) item -= __shfl_sync(0xFFFFFFFFu, sum, 31);
    }
    return false;
}

// Pool row of position pos < end of sequence b, -1 for a missing page or past the end.
__device__ __forceinline__ int64_t pool_row(const PrefillParams& p, const int32_t* table, int pos, int end) {
    if (pos >= end) return -1;
    const int pg = __ldg(table + (pos >> p.page_shift));
    if (pg < 0 || pg >= p.num_pages) return -1;
    return (static_cast<int64_t>(pg) << p.page_shift) | (pos & ((1 << p.page_shift) - 1));
}

// Pieces in the order the MMAs take them: the k_pieces of K of tile 0, then those of K of tile i and
// the v_pieces of V of tile i - 1.
struct Cursor {
    int u, i, s;      // piece number; s < k_pieces: K piece s of tile i, else V piece s - k_pieces of tile i - 1
};
__device__ __forceinline__ void advance(Cursor& c, int k_pieces, int v_pieces, int n_tiles) {
    ++c.u;
    ++c.s;
    if (c.i == 0 ? c.s == k_pieces : c.s == k_pieces + v_pieces) {
        ++c.i;
        c.s = c.i < n_tiles ? 0 : k_pieces;
    }
}

// The image of the sequences with many units: their tokens dequantised once for all of them, as
// the ring stages the attention kernel copies.  Block = 128 tokens: [8 latent atoms (+ the rope
// part)][128 tokens x 128 B], 128-byte swizzled, zeros for tokens that do not exist and for blocks
// with a NaN scale (the token's bit says so instead: a NaN in V would reach rows that do not see it).
__global__ void __launch_bounds__(256) prefill_image_kernel(const __grid_constant__ PrefillParams p) {
    __shared__ int64_t rows[kImageTok];
    __shared__ uint32_t bits[8];
    __shared__ int found_s, b_s, pos_s;
    griddep_launch_dependents();
    if (threadIdx.x < 32) {
        Unit u{};
        const bool found = find_unit<true>(p, blockIdx.x, &u);
        if (threadIdx.x == 0) {
            found_s = found;
            b_s = u.b;
            pos_s = u.block * kImageTok;
        }
    }
    if (threadIdx.x < 8) bits[threadIdx.x] = 0;
    __syncthreads();
    if (!found_s) return;
    const int L = visible_len(p, b_s), tid = threadIdx.x;
    if (tid < kImageTok) {
        const int pos = pos_s + tid;
        const int64_t row = pool_row(p, p.tables + b_s * p.tables_stride, pos, L);
        rows[tid] = row;
        if (row >= 0) atomicOr(&bits[tid >> 5], 1u << (tid & 31));
        else if (pos < L) set_error(p.err, NVFP4KV_DEVERR_BAD_PAGE);
    }
    __syncthreads();
    const int atoms = p.rope ? 9 : 8;
    uint4* dst = reinterpret_cast<uint4*>(p.image + static_cast<int64_t>(blockIdx.x) * atoms * kStageBytes);
#pragma unroll 4
    for (int k = tid; k < atoms * 1024; k += 256) {      // 16-byte chunk of the image
        const int atom = k >> 10, t = (k >> 3) & 127, c = (k & 7) ^ (t & 7);
        const int64_t row = rows[t];
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row >= 0) {
            if (atom == 8) {
                v = ldg_nc_v4(p.rope + row * kRope + 8 * c);
            } else {
                const uint8_t* src = p.pool + row * kRowBytes;
                const uint32_t code = __ldg(reinterpret_cast<const uint32_t*>(src + 32 * atom + 4 * c));
                const uint32_t sb = src[256 + 4 * atom + (c >> 1)];
                if ((sb & 0x7F) == 0x7F) {
                    atomicOr(&bits[4 + (t >> 5)], 1u << (t & 31));
                } else {
                    const uint32_t s2 = e4m3x2_to_f16x2(static_cast<uint16_t>(sb | sb << 8));
                    uint32_t h[4];
                    e2m1x8_to_f16x2x4(code, h);
                    v = make_uint4(hmul2_u32(h[0], s2), hmul2_u32(h[1], s2), hmul2_u32(h[2], s2), hmul2_u32(h[3], s2));
                }
            }
        }
        dst[k] = v;
    }
    __syncthreads();
    if (tid < 8) p.image_bits[8 * static_cast<int64_t>(blockIdx.x) + tid] = bits[tid];
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
mla_prefill_kernel(const __grid_constant__ PrefillParams p, const __grid_constant__ CUtensorMap tm_codes,
                   const __grid_constant__ CUtensorMap tm_scales, const __grid_constant__ CUtensorMap tm_rope) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const uint32_t sbase = smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cta = static_cast<int>(cluster_rank());
    volatile int* flags = reinterpret_cast<volatile int*>(smem + SM_FLAGS);
    volatile int* abort_flag = flags + 1;
    float* qs = reinterpret_cast<float*>(smem + SM_QS);
    auto bar = [&](int i) -> uint32_t { return sbase + SM_BARS + 8 * i; };

    const int item = blockIdx.x >> 1;
    const int unit = item / p.splits, split = item - unit * p.splits;
    if (warp == 0) {
        Unit u{};
        const bool found = find_unit<false>(p, unit, &u);
        if (lane == 0) {
            flags[1] = 0;
            flags[2] = found ? u.b : -1;
            flags[3] = u.first;
            flags[4] = u.n;
            flags[5] = u.block;
            flags[6] = u.image;
        }
    }
    __syncthreads();
    const int b = flags[2], first = flags[3], n_new = flags[4], block = flags[5], image0 = flags[6];
    if (b < 0) return;                 // past the last unit: the whole cluster
    const bool image = image0 >= 0;
    if (threadIdx.x == 0 && __ldg(p.seq_lens + b) > p.max_seq_len) set_error(p.err, NVFP4KV_DEVERR_SEQ_LEN);
    const int L = visible_len(p, b);
    const int32_t* table = p.tables + b * p.tables_stride;
    const int unit_rows = n_new * p.heads;                                    // rows of the sequence
    const int row0 = block * kUnitRows + kCtaRows * cta;                      // this CTA's first
    const int last_row = min(unit_rows, block * kUnitRows + kUnitRows) - 1;
    const int end = max(0, min(L, L - n_new + last_row / p.heads + 1));       // tokens the unit sees
    const int tiles = (end + kTile - 1) / kTile;
    const int tile0 = static_cast<int>(static_cast<int64_t>(split) * tiles / p.splits);
    const int n_tiles = static_cast<int>(static_cast<int64_t>(split + 1) * tiles / p.splits) - tile0;
    const int k_stages = p.rope ? 9 : 8, stages = image ? kStages : kDirectStages;
    const int ring = image ? SM_RING : SM_RING + kRawSlots * kRawBytes;
    const int image_last = image0 + (L + kImageTok - 1) / kImageTok - 1;      // (tokens past it are masked)

    if (threadIdx.x == 0) {
        for (int k = 0; k < kStages; ++k) {
            // dequantised here: four producer warps of each CTA; copied: the copy's issuer and, in the
            // leader, the other CTA's relay
            mbar_init(bar(B_FULL + k), image ? 2 - cta : 2 * 4);
            mbar_init(bar(B_EMPTY + k), 1);
        }
        for (int k = 0; k < 2; ++k) {
            mbar_init(bar(B_S_FULL + k), 1);
            mbar_init(bar(B_S_FREE + k), 2 * kSoftmaxWarps);
        }
        for (int k = 0; k < kRawSlots; ++k) {
            mbar_init(bar(B_RAW_FULL + k), 1);
            mbar_init(bar(B_RAW_EMPTY + k), kProducerWarps);
        }
        mbar_init(bar(B_P_FULL), 2 * kSoftmaxWarps);
        mbar_init(bar(B_PV_DONE), 1);
        mbar_init(bar(B_DRAIN), 1);
        mbar_fence_init();
    }
    if (warp == kMmaWarp) pair_tmem_alloc(sbase + SM_FLAGS, kTmemCols);
    // Q: 64 rows -> fp16 after a power of two per row that brings its largest |q| to [2^10, 2^11)
    // (the rope part by the same factor, in bf16); a warp per row, 16 + 2 dims per lane
    for (int r = warp; r < kCtaRows; r += kThreads / 32) {
        uint4 u[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        uint32_t rw = 0;
        const int row = row0 + r;
        if (row < unit_rows && n_tiles > 0) {
            const int tok = row / p.heads;
            const __nv_bfloat16* src = p.q + static_cast<int64_t>(first + tok) * p.q_st + static_cast<int64_t>(row - tok * p.heads) * p.q_sh;
            u[0] = ldg_nc_v4(src + 16 * lane);
            u[1] = ldg_nc_v4(src + 16 * lane + 8);
            if (p.rope) rw = __ldg(reinterpret_cast<const uint32_t*>(src + kLatent) + lane);
        }
        const uint32_t w[8] = {u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w};
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w[j] << 16)), fabsf(__uint_as_float(w[j] & 0xFFFF0000u))));
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
        const int eb = static_cast<int>((__float_as_uint(amax) >> 23) & 0xFFu);
        const int e = eb > 0 && eb < 255 ? max(eb - 127 - 10, -100) : 0;
        float factor = fabsf(p.scale_log2) * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
        float mul = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        mul = p.scale_log2 < 0.0f ? -mul : mul;
        if (factor == 0.0f) {              // every score 0: zero queries, and a factor that keeps a hidden score's -inf
            factor = 1.0f;
            mul = 0.0f;
        }
        uint32_t h[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = pack_half2(__uint_as_float(w[j] << 16) * mul, __uint_as_float(w[j] & 0xFFFF0000u) * mul);
        uint8_t* dst = smem + SM_Q + (lane >> 2) * (kCtaRows * 128) + r * 128;
#pragma unroll
        for (int c = 0; c < 2; ++c)
            *reinterpret_cast<uint4*>(dst + (((2 * (lane & 3) + c) ^ (r & 7)) << 4)) = make_uint4(h[4 * c], h[4 * c + 1], h[4 * c + 2], h[4 * c + 3]);
        if (p.rope) {
            const __nv_bfloat162 two = __floats2bfloat162_rn(__uint_as_float(rw << 16) * mul, __uint_as_float(rw & 0xFFFF0000u) * mul);
            *reinterpret_cast<uint32_t*>(smem + SM_Q + 8 * (kCtaRows * 128) + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + 4 * (lane & 3)) =
                *reinterpret_cast<const uint32_t*>(&two);
        }
        if (lane == 0) qs[r] = factor;
    }
    fence_proxy_async_smem();
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = static_cast<uint32_t>(flags[0]);

    if (warp >= kMmaWarp) {
        warpgroup_reg_dealloc<kRegsCtl>();
        if (warp == kMmaWarp) {
            if (cta == 0) {
                // ==================================================== MMA issue
                const uint64_t dq = smem_desc_sw128(sbase + SM_Q, 16, 1024);
                const uint64_t dp = smem_desc_sw128(sbase + SM_P, 16, 1024);
                const uint64_t dk = smem_desc_sw128(sbase + ring, 16, 1024);
                const uint64_t dv = smem_desc_sw128(sbase + ring, 8192, 1024);
                int slot = 0;
                uint32_t phase = 0;
                auto next = [&] {
                    if (++slot == stages) {
                        slot = 0;
                        phase ^= 1;
                    }
                };
#pragma unroll 1
                for (int i = 0; i <= n_tiles; ++i) {
                    if (i < n_tiles) {
                        const uint32_t d = tmem + kTS + 128 * (i & 1);
                        if (i >= 2) mbar_wait(bar(B_S_FREE + (i & 1)), ((i >> 1) - 1) & 1, abort_flag, p.err);
#pragma unroll 1
                        for (int j = 0; j < k_stages; ++j) {
                            mbar_wait(bar(B_FULL + slot), phase, abort_flag, p.err);
                            tc_fence_after();
                            const uint64_t a = dq + ((j * kCtaRows * 128) >> 4), bb = dk + ((slot * kStageBytes) >> 4);
                            const uint32_t id = j == 8 ? kIdescRope : kIdescQk;
                            if (elect_one()) {
#pragma unroll
                                for (int k = 0; k < 4; ++k) pair_mma_f16(d, a + 2 * k, bb + 2 * k, id, (j | k) != 0);
                                pair_commit(bar(B_EMPTY + slot));
                                if (j == k_stages - 1) pair_commit(bar(B_S_FULL + (i & 1)));
                            }
                            __syncwarp();
                            next();
                        }
                    }
                    if (i > 0) {
                        const int t = i - 1;
                        mbar_wait(bar(B_P_FULL), t & 1, abort_flag, p.err);
#pragma unroll 1
                        for (int s = 0; s < kVStages; ++s) {
                            mbar_wait(bar(B_FULL + slot), phase, abort_flag, p.err);
                            tc_fence_after();
                            const uint64_t a = dp + (((s >> 1) * kCtaRows * 128) >> 4), bb = dv + ((slot * kStageBytes) >> 4);
                            const uint32_t d = tmem + kTO + 128 * (s & 1);
                            if (elect_one()) {
#pragma unroll
                                for (int k = 0; k < 4; ++k) pair_mma_f16(d, a + 2 * k, bb + 128 * k, kIdescPv, (t | (s >> 1) | k) != 0);
                                pair_commit(bar(B_EMPTY + slot));
                                if (s == kVStages - 1) pair_commit(bar(B_PV_DONE));
                            }
                            __syncwarp();
                            next();
                        }
                    }
                }
                if (elect_one()) pair_commit(bar(B_DRAIN));
                __syncwarp();
            }
            griddep_wait();       // this grid ends after the image kernel, whatever its units read
            mbar_drain_wait(bar(B_DRAIN), 0);
        } else if (image && warp <= kMmaWarp + 2) {
            // ======================================================== image copies
            // Two warps take the stages in turn (one issues at most about 46 bytes a cycle).
            const int total = n_tiles * (k_stages + kVStages);
            const int64_t image_bytes = static_cast<int64_t>(k_stages) * kStageBytes;
            Cursor cur{0, 0, 0};
            int slot = warp - kMmaWarp - 1;
            uint32_t phase = 0;
            if (slot == 1) advance(cur, k_stages, kVStages, n_tiles);
            griddep_wait();                       // the image kernel's writes
            int issued = -1;                      // last stage copied
#pragma unroll 1
            while (cur.u < total) {
                if (cur.u >= kStages && !mbar_wait(bar(B_EMPTY + slot), phase ^ 1, abort_flag, p.err)) break;
                const uint32_t dst = sbase + SM_RING + slot * kStageBytes, full = bar(B_FULL + slot);
                if (elect_one()) {
                    mbar_arrive_expect_tx(full, kStageBytes);
                    if (cur.s < k_stages) {
                        const int blk = min(image0 + 2 * (tile0 + cur.i) + cta, image_last);
                        bulk_copy_g2s(dst, p.image + blk * image_bytes + cur.s * kStageBytes, kStageBytes, full);
                    } else {
                        const int v = cur.s - k_stages;      // tokens 64 (v / 2) .., dim atoms 4 c + 2 (v % 2), + 1
                        const int blk = min(image0 + 2 * (tile0 + cur.i - 1) + (v >> 2), image_last);
                        const uint8_t* src = p.image + blk * image_bytes + (4 * cta + 2 * (v & 1)) * kStageBytes + ((v >> 1) & 1) * 8192;
                        bulk_copy_g2s(dst, src, 8192, full);
                        bulk_copy_g2s(dst + 8192, src + kStageBytes, 8192, full);
                    }
                }
                __syncwarp();
                issued = cur.u;
                advance(cur, k_stages, kVStages, n_tiles);
                advance(cur, k_stages, kVStages, n_tiles);
                slot += 2;
                if (slot >= kStages) {
                    slot -= kStages;
                    phase ^= 1;
                }
            }
            // The last copies land before the CTA can exit (an earlier stage's slot was taken again, so
            // it has; after a timed-out wait, the last ones issued).
            const int from = max(0, cur.u >= total ? total - kStages : issued - kStages + 1);
            for (int u = from; u <= issued; ++u)
                if ((u & 1) == (issued & 1)) mbar_drain_wait(bar(B_FULL + u % kStages), (u / kStages) & 1);
        } else if (!image && warp == kMmaWarp + 1) {
            // ======================================================== raw rows
            // Piece: 128 tokens x 128 code bytes + their 16 scales (K: half of this CTA's tokens' dims; V:
            // half of the tile's tokens, this CTA's dims), or the 64 rope dims of the K tokens; boxes of up
            // to a page, a lane each.  A missing page, and a box past the end, is addressed out of range
            // and reads as zeros, so a slot always receives the same bytes.
            const int kp = p.rope ? 3 : 2, total = n_tiles * (kp + 2), box = p.box_rows, boxes = kImageTok / box;
            auto box_row = [&](const Cursor& c, int r) {
                const int pos = c.s < kp ? (tile0 + c.i) * kTile + 128 * cta : (tile0 + c.i - 1) * kTile + 128 * (c.s - kp);
                const int64_t row = pool_row(p, table, pos + r * box, end);
                return row < 0 ? -box : static_cast<int>(row);
            };
            if (lane == 0) {
                tma_prefetch_desc(&tm_codes);
                tma_prefetch_desc(&tm_scales);
            }
            Cursor cur{0, 0, 0};
            int slot = 0, y = total > 0 ? box_row(cur, min(lane, boxes - 1)) : 0;
            uint32_t phase = 0;
#pragma unroll 1
            while (cur.u < total) {
                if (cur.u >= kRawSlots && !mbar_wait(bar(B_RAW_EMPTY + slot), phase ^ 1, abort_flag, p.err)) break;
                fence_proxy_async_smem();
                const uint32_t dst = sbase + SM_RING + slot * kRawBytes, full = bar(B_RAW_FULL + slot);
                const bool rope = p.rope && cur.s == 2;
                const int half = cur.s < kp ? cur.s : cta;      // which 256 dims
                const bool scale_boxes = box >= 8;              // a copy starts on a multiple of 128 bytes
                if (!scale_boxes && !rope) {
                    for (int r = lane; r < kImageTok; r += 32) {
                        const int row = box_row(cur, r / box) + r % box;
                        *reinterpret_cast<uint4*>(smem + SM_RING + slot * kRawBytes + kStageBytes + 16 * r) =
                            row >= 0 ? ldg_nc_v4(p.pool + static_cast<int64_t>(row) * kRowBytes + 256 + 16 * half) : make_uint4(0, 0, 0, 0);
                    }
                    __syncwarp();
                }
                if (lane == 0) mbar_arrive_expect_tx(full, rope || !scale_boxes ? kStageBytes : kRawBytes);
                __syncwarp();
                for (int r = lane; r < boxes; r += 32) {
                    if (r >= 32) y = box_row(cur, r);
                    if (rope) {
                        tma_load_2d(dst + r * box * 128, &tm_rope, 0, y, full);
                    } else {
                        tma_load_2d(dst + r * box * 128, &tm_codes, 128 * half, y, full);
                        if (scale_boxes) tma_load_2d(dst + kStageBytes + r * box * 16, &tm_scales, 256 + 16 * half, y, full);
                    }
                }
                __syncwarp();
                advance(cur, kp, 2, n_tiles);
                if (cur.u < total) y = box_row(cur, min(lane, boxes - 1));
                if (++slot == kRawSlots) {
                    slot = 0;
                    phase ^= 1;
                }
            }
            for (int u = max(0, cur.u - kRawSlots); u < cur.u; ++u)      // every copy lands before the CTA can exit
                mbar_drain_wait(bar(B_RAW_FULL + u % kRawSlots), (u / kRawSlots) & 1);
        } else if (image && cta == 1 && warp == kMmaWarp + 3) {
            // ======================================================== relay: this CTA's copies, to the leader
            const int total = n_tiles * (k_stages + kVStages);
            int slot = 0;
            uint32_t phase = 0;
#pragma unroll 1
            for (int u = 0; u < total; ++u) {
                if (!mbar_wait(bar(B_FULL + slot), phase, abort_flag, p.err)) break;
                if (lane == 0) leader_arrive(bar(B_FULL + slot));
                __syncwarp();
                if (++slot == kStages) {
                    slot = 0;
                    phase ^= 1;
                }
            }
        }
    } else if (warp >= kProducerWarp0) {
        warpgroup_reg_dealloc<kRegsProducer>();
        if (!image) {
        // ============================================================ producers
        // Two groups of four warps take the stages in turn.  Thread t writes row t of a stage: K: token
        // 128 c + t of the tile, dims 64 s ..; V: token 64 (s / 2) + t % 64, dims 256 c + 128 (s % 2) +
        // 64 (t / 64) .. : 32 code bytes and 4 scales of a raw row.
        const int grp = (warp - kProducerWarp0) >> 2, t = threadIdx.x & 127;
        const int kp = p.rope ? 3 : 2, total = n_tiles * (kp + 2);
        Cursor cur{0, 0, 0};
        int raw = 0, slot = 0, n = 0;          // raw slot; ring slot and number of the next stage
        uint32_t raw_phase = 0, phase = 0;
        auto next = [&] {
            ++n;
            if (++slot == kDirectStages) {
                slot = 0;
                phase ^= 1;
            }
        };
#pragma unroll 1
        while (cur.u < total) {
            mbar_wait(bar(B_RAW_FULL + raw), raw_phase, abort_flag, p.err);
            const uint8_t* src = smem + SM_RING + raw * kRawBytes;
            if (p.rope && cur.s == 2) {
                if ((n & 1) == grp) {
                    uint4 v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = *reinterpret_cast<const uint4*>(src + t * 128 + 16 * j);
                    if (n >= kDirectStages) mbar_wait(bar(B_EMPTY + slot), phase ^ 1, abort_flag, p.err);
#pragma unroll
                    for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4*>(smem + ring + slot * kStageBytes + t * 128 + 16 * j) = v[j];
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) leader_arrive(bar(B_FULL + slot));
                }
                next();
            } else {
                const bool is_v = cur.s >= kp;
#pragma unroll 1
                for (int s = 0; s < 4; ++s, next()) {
                    if ((n & 1) != grp) continue;
                    // raw row, its 32-byte piece
                    const int r = is_v ? 64 * (s >> 1) + (t & 63) : t, piece = is_v ? 2 * (s & 1) + (t >> 6) : s;
                    const uint4 lo = *reinterpret_cast<const uint4*>(src + r * 128 + (((2 * piece) ^ (r & 7)) << 4));
                    const uint4 hi = *reinterpret_cast<const uint4*>(src + r * 128 + (((2 * piece + 1) ^ (r & 7)) << 4));
                    const uint32_t sc4 = *reinterpret_cast<const uint32_t*>(src + kStageBytes + r * 16 + 4 * piece);
                    const uint32_t code[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                    uint32_t s2[2] = {e4m3x2_to_f16x2(static_cast<uint16_t>(sc4)), e4m3x2_to_f16x2(static_cast<uint16_t>(sc4 >> 16))};
                    if (is_v) {
                        // a NaN block scale counts as 0 in V: rows that see the token are NaN by its score,
                        // rows that do not (probability 0) stay clear of it
                        s2[0] = max_f16x2(s2[0], 0u);
                        s2[1] = max_f16x2(s2[1], 0u);
                    }
                    if (n >= kDirectStages) mbar_wait(bar(B_EMPTY + slot), phase ^ 1, abort_flag, p.err);
                    uint8_t* dst = smem + ring + slot * kStageBytes + t * 128;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {                       // chunk j: dims 8 j .. of the 64
                        const uint32_t two = s2[j >> 2];
                        const uint32_t sc = (j & 2) ? __byte_perm(two, two, 0x3232) : __byte_perm(two, two, 0x1010);
                        uint32_t h[4];
                        e2m1x8_to_f16x2x4(code[j], h);
                        *reinterpret_cast<uint4*>(dst + ((j ^ (t & 7)) << 4)) =
                            make_uint4(hmul2_u32(h[0], sc), hmul2_u32(h[1], sc), hmul2_u32(h[2], sc), hmul2_u32(h[3], sc));
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) leader_arrive(bar(B_FULL + slot));
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_RAW_EMPTY + raw));
            advance(cur, kp, 2, n_tiles);
            if (++raw == kRawSlots) {
                raw = 0;
                raw_phase ^= 1;
            }
        }
        }
    } else {
        warpgroup_reg_alloc<kRegsSoftmax>();
        // ============================================================ softmax
        // warp: TMEM lanes 32 sp .., columns 64 ch .. of a tile's 128: row 32 (sp & 1) + lane, token
        // quarter q4; the four warps of a row exchange their maxima in shared memory
        const int sp = warp & 3, ch = warp >> 2;
        const int row = 32 * (sp & 1) + lane, q4 = 2 * (sp >> 1) + ch;
        const uint32_t lanes = static_cast<uint32_t>(32 * sp) << 16;
        float* red = reinterpret_cast<float*>(smem + SM_RED);
        const int grow = row0 + row;                                   // row of the sequence
        const bool real = grow < unit_rows;
        const int tok = real ? grow / p.heads : 0, head = grow - tok * p.heads;
        const int lim = real ? min(L, L - n_new + tok + 1) : 0;        // tokens the row sees
        const float factor = qs[row];
        float m_ref = -INFINITY, l = 0.0f;
        // What the next tile's token masks are made of, loaded a tile ahead.  Image: the bits of the
        // quarter's tokens that exist and of those that hold a NaN; else: the page ids of tokens lane
        // and 32 + lane.
        auto load_masks = [&](int i, uint32_t (&w)[4]) {
            const int tok0 = (tile0 + i) * kTile + 64 * q4;
            if (image) {
                const int blk = min(image0 + tok0 / kImageTok, image_last), k = (tok0 & (kImageTok - 1)) >> 5;
                const uint2 have = *reinterpret_cast<const uint2*>(p.image_bits + 8 * static_cast<int64_t>(blk) + k);
                const uint2 nans = *reinterpret_cast<const uint2*>(p.image_bits + 8 * static_cast<int64_t>(blk) + 4 + k);
                w[0] = have.x; w[1] = have.y; w[2] = nans.x; w[3] = nans.y;
            } else {
                w[0] = tok0 + lane < end ? __ldg(table + ((tok0 + lane) >> p.page_shift)) : 0;
                w[1] = tok0 + 32 + lane < end ? __ldg(table + ((tok0 + 32 + lane) >> p.page_shift)) : 0;
            }
        };
        if (image) griddep_wait();
        uint32_t ahead[4];
        load_masks(0, ahead);
#pragma unroll 1
        for (int i = 0; i < n_tiles; ++i) {
            uint32_t bits[4] = {ahead[0], ahead[1], 0, 0};
            if (image) {
                bits[2] = ahead[2];
                bits[3] = ahead[3];
            } else {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const bool missing = static_cast<int64_t>(ahead[k]) >= p.num_pages;      // (a negative id is a large one)
                    if (missing) set_error(p.err, NVFP4KV_DEVERR_BAD_PAGE);
                    bits[k] = __ballot_sync(0xFFFFFFFFu, !missing);
                }
            }
            load_masks(i + 1, ahead);
            const int see = lim - ((tile0 + i) * kTile + 64 * q4);     // tokens of the quarter the row sees
            mbar_wait(bar(B_S_FULL + (i & 1)), (i >> 1) & 1, abort_flag, p.err);
            tc_fence_after();
            float x[64];
            tmem_ld32(tmem + kTS + 128 * (i & 1) + 64 * ch + lanes, reinterpret_cast<uint32_t*>(x));
            tmem_ld32(tmem + kTS + 128 * (i & 1) + 64 * ch + 32 + lanes, reinterpret_cast<uint32_t*>(x) + 32);
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) leader_arrive(bar(B_S_FREE + (i & 1)));
            if (!__all_sync(0xFFFFFFFFu, see >= 64 && (bits[0] & bits[1]) == 0xFFFFFFFFu && (bits[2] | bits[3]) == 0)) {
#pragma unroll
                for (int k = 0; k < 64; ++k) {
                    if ((bits[2 + (k >> 5)] >> (k & 31)) & 1u) x[k] = __int_as_float(0x7FFFFFFF);
                    if (k >= see || !((bits[k >> 5] >> (k & 31)) & 1u)) x[k] = -INFINITY;
                }
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int k = 0; k < 64; ++k) mx[k & 3] = fmaxf(mx[k & 3], x[k]);
            float* slot = red + (i & 1) * 256;
            slot[64 * q4 + row] = factor * fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            named_bar_sync(1 + (sp & 1), 128);
            const float m = fmaxf(fmaxf(slot[row], slot[64 + row]), fmaxf(slot[128 + row], slot[192 + row]));
            float alpha = 1.0f;
            if (m > m_ref + kRescaleLog2 || (m_ref == -INFINITY && m > -INFINITY)) {
                alpha = m_ref == -INFINITY ? 0.0f : ex2_approx(m_ref - m);
                l *= alpha;
                m_ref = m;
            }
            const float base = m_ref == -INFINITY ? 0.0f : m_ref;
            uint32_t pk[32];
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < 32; ++k) {
                const float a = ex2_approx(fmaf(x[2 * k], factor, -base)), c = ex2_approx(fmaf(x[2 * k + 1], factor, -base));
                sum[k & 1] += a;
                sum[2 + (k & 1)] += c;
                pk[k] = pack_half2(a, c);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            if (i > 0) {
                mbar_wait(bar(B_PV_DONE), (i - 1) & 1, abort_flag, p.err);
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
        // ---- epilogue: sums over the row's four warps, O out of TMEM
        float* lsum = reinterpret_cast<float*>(smem + SM_LSUM);
        lsum[64 * q4 + row] = l;
        named_bar_sync(1 + (sp & 1), 128);
        l = (lsum[row] + lsum[64 + row]) + (lsum[128 + row] + lsum[192 + row]);
        if (n_tiles > 0) mbar_wait(bar(B_PV_DONE), (n_tiles - 1) & 1, abort_flag, p.err);
        tc_fence_after();
        const bool any = l > 0.0f || l != l;
        const int d0 = 256 * (sp >> 1) + 128 * ch;                     // the thread's 128 dims
        if (p.splits > 1) {
            const int64_t u = (static_cast<int64_t>(split) * p.units + unit) * kUnitRows + kCtaRows * cta + row;
            if (q4 == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * u) = make_float2(m_ref, l);
            if (n_tiles > 0) {
#pragma unroll 1
                for (int c = 0; c < 128; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(tmem + kTO + 128 * ch + c + lanes, o);
                    tmem_wait_ld();
                    if (real && any) {
                        uint4* dst = reinterpret_cast<uint4*>(p.part_o + u * kLatent + d0 + c);
#pragma unroll
                        for (int k = 0; k < 8; ++k) dst[k] = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                    }
                }
            }
        } else {
            const float inv = any ? p.out_scale / l : 0.0f;
            if (p.lse && real && q4 == 0)
                p.lse[static_cast<int64_t>(first + tok) * p.heads + head] =
                    any ? 0.69314718055994531f * (m_ref + log2f(l)) : -INFINITY;
            __nv_bfloat16* dst = p.out + static_cast<int64_t>(first + tok) * p.o_st + static_cast<int64_t>(head) * p.o_sh + d0;
#pragma unroll 1
            for (int c = 0; c < 128; c += 32) {
                uint32_t o[32];
                if (n_tiles > 0) {
                    tmem_ld32(tmem + kTO + 128 * ch + c + lanes, o);
                    tmem_wait_ld();
                }
                if (real) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t w[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float a = any ? __uint_as_float(o[8 * k + 2 * j]) * inv : 0.0f;
                            const float c2 = any ? __uint_as_float(o[8 * k + 2 * j + 1]) * inv : 0.0f;
                            const __nv_bfloat162 two = __floats2bfloat162_rn(a, c2);
                            w[j] = *reinterpret_cast<const uint32_t*>(&two);
                        }
                        *reinterpret_cast<uint4*>(dst + c + 8 * k) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
        }
        tc_fence_before();
    }
    cluster_sync();
    if (warp == kMmaWarp) pair_tmem_dealloc(tmem, kTmemCols);
}

// Merges the splits of a unit: out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s.  A block per row.
__global__ void __launch_bounds__(128) prefill_combine_kernel(const __grid_constant__ PrefillParams p) {
    __shared__ int where[3];
    __shared__ float wts[kMaxSplits];
    griddep_wait();
    const int unit = blockIdx.x / kUnitRows, r = blockIdx.x % kUnitRows;
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        Unit un{};
        const bool found = find_unit<false>(p, unit, &un);
        const int first = un.first, row = un.block * kUnitRows + r;
        const bool real = found && row < un.n * p.heads;
        if (real) {
            const int64_t step = static_cast<int64_t>(p.units) * kUnitRows;
            const int64_t u = static_cast<int64_t>(unit) * kUnitRows + r;
            float m[2], l[2], top = -INFINITY;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int s = lane + 32 * k;
                const float2 v = s < p.splits ? *reinterpret_cast<const float2*>(p.part_ml + 2 * (s * step + u)) : make_float2(-INFINITY, 0.0f);
                m[k] = v.x;
                l[k] = v.y;
                if (l[k] > 0.0f || l[k] != l[k]) top = fmaxf(top, m[k]);
            }
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            float w[2], sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                w[k] = l[k] > 0.0f || l[k] != l[k] ? exp2f(m[k] - top) : 0.0f;
                sum += w[k] > 0.0f || w[k] != w[k] ? w[k] * l[k] : 0.0f;
            }
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            const bool any = sum > 0.0f || sum != sum;
            const float inv = any ? p.out_scale / sum : 0.0f;
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (lane + 32 * k < p.splits) wts[lane + 32 * k] = w[k] != 0.0f ? w[k] * inv : 0.0f;
            const int tok = row / p.heads;
            if (p.lse && lane == 0)
                p.lse[static_cast<int64_t>(first + tok) * p.heads + (row - tok * p.heads)] =
                    any ? 0.69314718055994531f * (top + log2f(sum)) : -INFINITY;
            if (lane == 0) {
                where[1] = first + tok;
                where[2] = row - tok * p.heads;
            }
        }
        if (lane == 0) where[0] = real;
    }
    __syncthreads();
    if (!where[0]) return;
    const int64_t step = static_cast<int64_t>(p.units) * kUnitRows * kLatent;
    const float* src = p.part_o + (static_cast<int64_t>(unit) * kUnitRows + r) * kLatent + 4 * threadIdx.x;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
        const float w = wts[s];
        if (w != 0.0f) {      // a split that saw no token wrote no O
            const float4 v = *reinterpret_cast<const float4*>(src + s * step);
            acc.x = fmaf(w, v.x, acc.x);
            acc.y = fmaf(w, v.y, acc.y);
            acc.z = fmaf(w, v.z, acc.z);
            acc.w = fmaf(w, v.w, acc.w);
        }
    }
    const __nv_bfloat162 lo = __floats2bfloat162_rn(acc.x, acc.y), hi = __floats2bfloat162_rn(acc.z, acc.w);
    *reinterpret_cast<uint2*>(p.out + where[1] * p.o_st + where[2] * p.o_sh + 4 * threadIdx.x) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
    static std::once_flag once;
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    std::call_once(once, [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    });
    return fn;
}

// Map of [rows][row_bytes] bytes with boxes of box_x bytes x box_y rows.
int make_row_map(CUtensorMap* m, const void* base, int64_t rows, int row_bytes, int box_x, int box_y, bool swizzle) {
    auto enc = tensor_map_encoder();
    if (!enc) return fail(NVFP4KV_ECUDA, "mla_prefill: cuTensorMapEncodeTiled is unavailable");
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(row_bytes), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_bytes)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_x), static_cast<cuuint32_t>(box_y)}, step[2] = {1, 1};
    const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, step,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(NVFP4KV_ECUDA, "mla_prefill: cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
    return NVFP4KV_OK;
}

struct PrefillPlan {
    int units, splits, image_blocks;
    size_t image_bytes, part_bytes, ws_bytes;
};

constexpr size_t kImageCap = size_t(1) << 30;      // images take at most this, or one sequence's

// Units: 128-row blocks over all sequences, bounded from what the host knows.  With fewer units than
// CTA pairs the tokens of a unit are split over the idle pairs, and the parts merged.
PrefillPlan make_prefill_plan(int batch, int total_q, int num_heads, int max_q_len, int max_seq_len) {
    PrefillPlan pl{};
    const int64_t per_seq = (static_cast<int64_t>(max_q_len < total_q ? max_q_len : total_q) * num_heads + kUnitRows - 1) / kUnitRows;
    const int64_t by_seq = per_seq * batch;
    const int64_t by_rows = (static_cast<int64_t>(total_q) * num_heads + static_cast<int64_t>(batch) * (kUnitRows - 1)) / kUnitRows;
    const int64_t units = by_seq < by_rows ? by_seq : by_rows;
    pl.units = static_cast<int>(units < 1 ? 1 : units);
    const int pairs = device_sm_count() / 2;
    const int tiles = max_seq_len > 0 ? (max_seq_len + kTile - 1) / kTile : 1;
    int splits = pairs / pl.units;
    splits = splits > kMaxSplits ? kMaxSplits : splits;
    splits = splits > tiles ? tiles : splits;
    pl.splits = splits < 1 ? 1 : splits;
    pl.part_bytes = pl.splits > 1 ? static_cast<size_t>(pl.splits) * pl.units * kUnitRows * (kLatent + 2) * sizeof(float) : 0;
    // Images: only sequences of at least kImageUnits units have one
    const int64_t least = (static_cast<int64_t>(kImageUnits - 1) * kUnitRows) / num_heads + 1;      // their new tokens
    int64_t seqs = max_q_len >= least ? total_q / least : 0;
    seqs = seqs > batch ? batch : seqs;
    const int64_t one = (static_cast<int64_t>(max_seq_len) + kImageTok - 1) / kImageTok;
    const int64_t cap = static_cast<int64_t>(kImageCap / (9 * kStageBytes));
    int64_t blocks = seqs * one;
    if (blocks > cap) blocks = cap > one ? cap : one;
    pl.image_blocks = static_cast<int>(blocks);
    pl.image_bytes = static_cast<size_t>(blocks) * 9 * kStageBytes;
    pl.ws_bytes = pl.image_bytes + ((static_cast<size_t>(blocks) * 32 + 255) / 256) * 256 + pl.part_bytes;
    return pl;
}

}  // namespace
}  // namespace nvfp4kv

extern "C" int nvfp4kv_mla_prefill_workspace_size(int batch, int total_q, int num_heads, int max_q_len,
                                                  int max_seq_len, size_t* bytes) {
    using namespace nvfp4kv;
    if (!bytes) return fail(NVFP4KV_EINVAL, "mla_prefill_workspace_size: null output");
    if (batch < 0 || total_q < 0 || num_heads < 1 || max_q_len < 0 || max_seq_len < 0)
        return fail(NVFP4KV_EINVAL, "mla_prefill_workspace_size: bad shape");
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
    p.lse = lse; p.err = err_flag; p.units = pl.units; p.splits = pl.splits;
    p.image = static_cast<uint8_t*>(workspace); p.image_blocks = pl.image_blocks;
    p.image_bits = reinterpret_cast<uint32_t*>(p.image + pl.image_bytes);
    if (pl.splits > 1) {
        p.part_o = reinterpret_cast<float*>(p.image + pl.ws_bytes - pl.part_bytes);
        p.part_ml = p.part_o + static_cast<size_t>(pl.splits) * pl.units * kUnitRows * kLatent;
    }
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e = cudaFuncSetAttribute(mla_prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "mla_prefill: %s", cudaGetErrorString(e));
    p.box_rows = page_size < kImageTok ? page_size : kImageTok;
    CUtensorMap tm_codes{}, tm_scales{}, tm_rope{};
    int rc = make_row_map(&tm_codes, pool, pool_rows, kRowBytes, 128, p.box_rows, true);
    if (rc == NVFP4KV_OK) rc = make_row_map(&tm_scales, pool, pool_rows, kRowBytes, 16, p.box_rows, false);
    if (rc == NVFP4KV_OK && rope_pool) rc = make_row_map(&tm_rope, rope_pool, pool_rows, 2 * kRope, 2 * kRope, p.box_rows, true);
    if (rc != NVFP4KV_OK) return rc;
    if (pl.image_blocks > 0) {
        prefill_image_kernel<<<pl.image_blocks, 256, 0, st>>>(p);
        if ((rc = check_launch("nvfp4kv_mla_prefill image")) != NVFP4KV_OK) return rc;
    }
    const dim3 grid(static_cast<unsigned>(2 * pl.units * pl.splits));
    if (pl.image_blocks > 0)      // its set-up overlaps the image kernel, all else it reads was there before that one
        e = launch_dependent(mla_prefill_kernel, grid, dim3(kThreads), kSmemBytes, st, p, tm_codes, tm_scales, tm_rope);
    else
        mla_prefill_kernel<<<grid, kThreads, kSmemBytes, st>>>(p, tm_codes, tm_scales, tm_rope);
    if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "nvfp4kv_mla_prefill launch failed: %s", cudaGetErrorString(e));
    rc = check_launch("nvfp4kv_mla_prefill");
    if (rc != NVFP4KV_OK || pl.splits == 1) return rc;
    e = launch_dependent(prefill_combine_kernel, dim3(pl.units * kUnitRows), dim3(128), 0, st, p);
    if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "nvfp4kv_mla_prefill combine launch failed: %s", cudaGetErrorString(e));
    return check_launch("nvfp4kv_mla_prefill combine");
}
