// Upkeep of a paged cache whose pools share page ids: copying, forking, compacting and freeing
// pages, all on the device and in stream order (no count comes back to the host).
//
// The results are those of the sequential definition whatever order blocks run in: counts change
// by integer atomics, which commute, and every choice (which free page, which fork of a twice
// named slot) is the lowest index.  The data movement is bound by HBM, the bookkeeping by the
// latency of a few dependent launches.
#include "../../include/nvfp4kv_serving.h"
#include "abi_common.h"
#include "common.cuh"
#include "decode_shared.h"

namespace nvfp4kv {
namespace {

constexpr int kPlanThreads = 1024;

struct Caches {
    uint8_t* base[NVFP4KV_MAX_CACHES];
    int64_t page_bytes[NVFP4KV_MAX_CACHES];
    int num;
};

// Exclusive prefix sum of `v` over the block (kPlanThreads threads); *total receives the sum.
// `warp_sums`: 32 ints of shared memory, free again after the caller's next __syncthreads().
__device__ __forceinline__ int block_exclusive_scan(int v, int* warp_sums, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xFFFFFFFFu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    int w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xFFFFFFFFu, w, o);
        if (lane >= o) w += y;
    }
    *total = __shfl_sync(0xFFFFFFFFu, w, 31);
    const int before = __shfl_sync(0xFFFFFFFFu, w, warp > 0 ? warp - 1 : 0);
    return x - v + (warp > 0 ? before : 0);
}

// `bytes` from src to dst by the threads of a block, `tid` of `nt`, in the widest pieces that
// both addresses and the size allow; four pieces in flight per thread.
template <typename V>
__device__ __forceinline__ void copy_pieces(uint8_t* dst, const uint8_t* src, int64_t bytes, int tid, int nt) {
    const int64_t n = bytes / static_cast<int64_t>(sizeof(V));
    const V* s = reinterpret_cast<const V*>(src);
    V* d = reinterpret_cast<V*>(dst);
    for (int64_t i = tid; i < n; i += 4 * nt) {
        V v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k * nt < n) v[k] = __ldg(s + i + k * nt);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k * nt < n) d[i + k * nt] = v[k];
    }
}
__device__ __forceinline__ void copy_bytes(uint8_t* dst, const uint8_t* src, int64_t bytes, int tid, int nt) {
    const uint64_t a = reinterpret_cast<uint64_t>(dst) | reinterpret_cast<uint64_t>(src) | static_cast<uint64_t>(bytes);
    if (a % 16 == 0) copy_pieces<uint4>(dst, src, bytes, tid, nt);
    else if (a % 4 == 0) copy_pieces<uint32_t>(dst, src, bytes, tid, nt);
    else copy_pieces<uint8_t>(dst, src, bytes, tid, nt);
}

// Pairs (src[k], dst[k]): blockIdx.y = cache, blocks of x stride over the pairs, whose number is
// on the host (num) or on the device (num_dev).  For pages that bulk copies cannot move.
__global__ void __launch_bounds__(256)
copy_pages_kernel(const __grid_constant__ Caches c, int64_t num_pages, const int32_t* __restrict__ src,
                  const int32_t* __restrict__ dst, int64_t num, const int32_t* __restrict__ num_dev,
                  int32_t* __restrict__ err) {
    griddep_wait();
    const int64_t n = num_dev ? static_cast<int64_t>(*num_dev) : num;
    const int64_t pb = c.page_bytes[blockIdx.y];
    uint8_t* base = c.base[blockIdx.y];
    for (int64_t k = blockIdx.x; k < n; k += gridDim.x) {
        const int s = __ldg(src + k), d = __ldg(dst + k);
        if (s < 0 || d < 0) continue;
        if (s >= num_pages || d >= num_pages) {
            if (threadIdx.x == 0) set_error(err, NVFP4KV_DEVERR_BAD_PAGE);
            continue;
        }
        copy_bytes(base + d * pb, base + s * pb, pb, threadIdx.x, blockDim.x);
    }
}

// The same with bulk copies through shared memory: a block is one warp that keeps kCopyStages pieces
// in flight, loads ahead of stores, and no data passes registers.  A page is cut into equal pieces of
// at most kCopyBytes; the blocks take the pieces of all pairs in turn.  Compacting 42,405 pages of three
// caches (1.32 GB, 35 % in use) moves 0.60 GB, read and written, in 97.5 us: 6.1 TB/s, 95 % of a plain
// copy's rate.
constexpr int kCopyStages = 8, kCopyBytes = 9216;
struct CopyPieces {
    int first[NVFP4KV_MAX_CACHES + 1];      // a pair's first piece in each cache
    int bytes[NVFP4KV_MAX_CACHES];          // of a piece
};
__global__ void __launch_bounds__(32)
bulk_copy_pages_kernel(const __grid_constant__ Caches c, const __grid_constant__ CopyPieces pieces, int64_t num_pages,
                       const int32_t* __restrict__ src, const int32_t* __restrict__ dst, int64_t num,
                       const int32_t* __restrict__ num_dev, int32_t* __restrict__ err) {
    extern __shared__ __align__(128) uint8_t stage[];
    __shared__ __align__(8) uint64_t bars[kCopyStages];
    __shared__ int abort_flag;
    if (threadIdx.x != 0) return;
    for (int k = 0; k < kCopyStages; ++k) mbar_init(smem_u32(&bars[k]), 1);
    abort_flag = 0;
    mbar_fence_init();
    griddep_wait();
    const int per = pieces.first[c.num];
    const int64_t total = (num_dev ? static_cast<int64_t>(*num_dev) : num) * per;
    // piece i: where it comes from and goes to, 0 bytes for a pair that is skipped
    auto locate = [&](int64_t i, const uint8_t** from, uint8_t** to) -> uint32_t {
        const int64_t k = i / per;
        const int q = static_cast<int>(i - k * per);
        const int s = __ldg(src + k), d = __ldg(dst + k);
        if (s < 0 || d < 0) return 0;
        if (s >= num_pages || d >= num_pages) {
            set_error(err, NVFP4KV_DEVERR_BAD_PAGE);
            return 0;
        }
        int cache = 0;
        while (q >= pieces.first[cache + 1]) ++cache;
        const int size = pieces.bytes[cache];
        const int64_t pb = c.page_bytes[cache], at = static_cast<int64_t>(q - pieces.first[cache]) * size;
        *from = c.base[cache] + s * pb + at;
        *to = c.base[cache] + d * pb + at;
        return static_cast<uint32_t>(pb - at < size ? pb - at : size);
    };
    // Piece i of this block (blockIdx.x + i gridDim.x) uses stage i % kCopyStages.  Loads run kAhead
    // pieces ahead; the stage a load takes was last stored from kCopyStages - kAhead pieces ago.
    constexpr int kAhead = kCopyStages / 2;
    const int64_t mine = total > blockIdx.x ? (total - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
    uint8_t* to[kCopyStages];
    uint32_t bytes[kCopyStages];
    auto load = [&](int64_t i, int st) {
        bytes[st] = 0;
        if (i >= mine) return;
        const uint8_t* from = nullptr;
        bytes[st] = locate(blockIdx.x + i * gridDim.x, &from, &to[st]);
        mbar_arrive_expect_tx(smem_u32(&bars[st]), bytes[st]);      // (a skipped pair's phase completes at once)
        if (bytes[st]) bulk_copy_g2s(smem_u32(stage) + st * kCopyBytes, from, bytes[st], smem_u32(&bars[st]));
    };
#pragma unroll
    for (int st = 0; st < kAhead; ++st) load(st, st);
    uint32_t phase = 0;
    int64_t done = 0;      // pieces whose load has landed
    for (int64_t i0 = 0; i0 < mine; i0 += kCopyStages, phase ^= 1) {
#pragma unroll
        for (int st = 0; st < kCopyStages; ++st) {
            if (i0 + st >= mine) break;
            if (!mbar_wait(smem_u32(&bars[st]), phase, &abort_flag, err)) break;
            if (bytes[st]) bulk_copy_s2g(to[st], smem_u32(stage) + st * kCopyBytes, bytes[st]);
            bulk_commit_group();
            asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kCopyStages - kAhead) : "memory");
            load(i0 + st + kAhead, (st + kAhead) % kCopyStages);
            ++done;
        }
        if (abort_flag) break;
    }
    bulk_wait_group_read0();
    // (after a timed-out wait: the loads in flight, each in its own round's phase, land before the
    // block's shared memory goes; those before have landed and begin no other phase)
    if (abort_flag)
        for (int64_t i = done; i < done + kAhead && i < mine; ++i) mbar_drain_wait(smem_u32(&bars[i % kCopyStages]), (i / kCopyStages) & 1);
}

// ------------------------------------------------------------------ freeing
// Block = slot (32 samples of 16,000 tokens: 3 us).  A table entry is taken with an exchange, so that a slot named twice gives its
// pages back once; a decrement that finds no reference is undone and reported.
__global__ void __launch_bounds__(256)
free_pages_kernel(int32_t* tables, int64_t stride, int width, int64_t num_slots, int32_t* seq_lens,
                  const int32_t* __restrict__ slots, int32_t* refs, int64_t num_pages, int32_t* err) {
    griddep_wait();
    const int slot = __ldg(slots + blockIdx.x);
    if (slot < 0 || slot >= num_slots) {
        if (threadIdx.x == 0) set_error(err, NVFP4KV_DEVERR_BAD_SLOT);
        return;
    }
    int32_t* row = tables + slot * stride;
    for (int j = threadIdx.x; j < width; j += blockDim.x) {
        const int p = atomicExch(row + j, -1);
        if (p < 0) continue;
        if (p >= num_pages) {
            set_error(err, NVFP4KV_DEVERR_BAD_PAGE);
        } else if (atomicSub(refs + p, 1) <= 0) {
            atomicAdd(refs + p, 1);
            set_error(err, NVFP4KV_DEVERR_BAD_PAGE);
        }
    }
    if (threadIdx.x == 0) seq_lens[slot] = 0;
}

// ------------------------------------------------------------------ forking
struct ForkArgs {
    int32_t* tables;
    int64_t stride;
    int width, page_size;
    int64_t num_slots;
    int32_t* seq_lens;
    const int32_t* src;
    const int32_t* dst;
    int num;
    int32_t* refs;
    int64_t num_pages;
    int32_t* fresh;      // [num]: the new last page, -1 without one, -2 for a fork that is skipped
    int32_t* free_list;  // [num]: the lowest free pages
    int32_t* lens;       // [num]: the parents' lengths (a fork may fill a slot that another names as parent)
    int32_t* err;
};

// The parent's length; whether its last page has to be copied, and that page (*old).
__device__ __forceinline__ int fork_length(const ForkArgs& p, int src) {
    const int64_t most = static_cast<int64_t>(p.width) * p.page_size;
    const int len = p.seq_lens[src];
    return static_cast<int>(len < 0 ? 0 : (len > most ? most : len));
}
__device__ __forceinline__ bool fork_partial(const ForkArgs& p, int src, int len, int* old) {
    const int full = len / p.page_size;
    *old = -1;
    if (len % p.page_size == 0) return false;
    const int pg = p.tables[src * p.stride + full];
    if (pg < 0 || pg >= p.num_pages) return false;      // a missing page stays missing
    *old = pg;
    return true;
}

// One block: which forks count, how many free pages they need, the lowest free pages, and one of
// them for each fork in order.  Bound by the latency of its passes: 5.5 us for 28 forks over 1,024
// pages, 7 us for 480 over 42,405 (16 counts a thread and step; it stops at the last page it needs).
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const __grid_constant__ ForkArgs p) {
    __shared__ int sums[2][32];
    const int tid = threadIdx.x;
    griddep_wait();
    // claims: an empty slot's seq_len becomes the smallest -(num - k) of the forks that name it,
    // so the first of them wins; the forks write the real length afterwards
    for (int k = tid; k < p.num; k += kPlanThreads) {
        const int s = p.src[k], d = p.dst[k];
        const bool ok = s >= 0 && s < p.num_slots && d >= 0 && d < p.num_slots && p.seq_lens[d] == 0 && s != d;
        p.fresh[k] = ok ? 0 : -2;
        if (!ok) set_error(p.err, NVFP4KV_DEVERR_BAD_SLOT);
    }
    __syncthreads();
    for (int k = tid; k < p.num; k += kPlanThreads)
        if (p.fresh[k] == 0) atomicMin(p.seq_lens + p.dst[k], -(p.num - k));
    __syncthreads();
    int need_total = 0;
    for (int k0 = 0; k0 < p.num; k0 += kPlanThreads) {
        const int k = k0 + tid;
        bool need = false;
        int state = -2;
        if (k < p.num && p.fresh[k] == 0) {
            // (an empty parent that a fork of this call claims reads as length 0)
            if (p.seq_lens[p.dst[k]] == -(p.num - k)) {
                int old;
                const int len = fork_length(p, p.src[k]);
                p.lens[k] = len;
                need = fork_partial(p, p.src[k], len, &old);
                state = -1;
            } else {
                set_error(p.err, NVFP4KV_DEVERR_BAD_SLOT);
            }
        }
        int total;
        const int rank = need_total + block_exclusive_scan(need, sums[0], &total);
        if (k < p.num) p.fresh[k] = need ? rank : state;   // the rank, until the pages are known
        need_total += total;
        __syncthreads();
    }
    // the lowest need_total free pages, 16 counts a thread and step
    constexpr int kPer = 16;
    int found = 0;
    for (int64_t b0 = 0; b0 < p.num_pages && found < need_total; b0 += kPlanThreads * kPer) {
        const int64_t i0 = b0 + tid * kPer;
        uint32_t zero = 0;
        if (i0 + kPer <= p.num_pages && reinterpret_cast<uintptr_t>(p.refs) % 16 == 0) {
            int4 v[kPer / 4];
#pragma unroll
            for (int j = 0; j < kPer / 4; ++j) v[j] = *(reinterpret_cast<const int4*>(p.refs + i0) + j);
#pragma unroll
            for (int j = 0; j < kPer / 4; ++j)
                zero |= static_cast<uint32_t>((v[j].x == 0) | (v[j].y == 0) << 1 | (v[j].z == 0) << 2 | (v[j].w == 0) << 3) << (4 * j);
        } else {
            for (int j = 0; j < kPer; ++j)
                if (i0 + j < p.num_pages && p.refs[i0 + j] == 0) zero |= 1u << j;
        }
        int total;
        int at = found + block_exclusive_scan(__popc(zero), sums[1], &total);
        for (; zero && at < need_total; zero &= zero - 1, ++at) p.free_list[at] = static_cast<int>(i0) + __ffs(zero) - 1;
        found += total;
        __syncthreads();
    }
    for (int k = tid; k < p.num; k += kPlanThreads) {
        const int r = p.fresh[k];
        if (r >= 0) {
            if (r < found) {
                p.fresh[k] = p.free_list[r];
            } else {
                p.fresh[k] = -2;
                set_error(p.err, NVFP4KV_DEVERR_CAPACITY);
            }
        }
        if (p.fresh[k] == -2) {   // a skipped fork leaves an empty slot empty
            const int d = p.dst[k];
            if (d >= 0 && d < p.num_slots && p.seq_lens[d] == -(p.num - k)) p.seq_lens[d] = 0;
        }
    }
    griddep_launch_dependents();
}

// blockIdx.x = fork; y = 0: its table, counts and length, y = 1 + c: the filled rows of its last
// page in cache c.  480 forks of 16,000 tokens: 6 us, 17 MB of it last pages and tables.
__global__ void __launch_bounds__(256) fork_apply_kernel(const __grid_constant__ ForkArgs p, const __grid_constant__ Caches c) {
    griddep_wait();
    const int k = blockIdx.x;
    const int fresh = p.fresh[k];
    if (fresh == -2) return;
    const int src = __ldg(p.src + k), dst = __ldg(p.dst + k);
    const int len = p.lens[k];
    const int full = len / p.page_size;
    if (blockIdx.y == 0) {
        const int32_t* from = p.tables + src * p.stride;
        int32_t* to = p.tables + dst * p.stride;
        const int used = (len + p.page_size - 1) / p.page_size;
        for (int j = threadIdx.x; j < p.width; j += blockDim.x) {
            int pg = -1;
            if (j < used) {
                pg = from[j];
                if (pg < 0 || pg >= p.num_pages) {
                    pg = -1;
                    set_error(p.err, NVFP4KV_DEVERR_BAD_PAGE);
                } else if (j < full) {
                    atomicAdd(p.refs + pg, 1);
                } else {
                    pg = fresh;
                    atomicAdd(p.refs + pg, 1);
                }
            }
            to[j] = pg;
        }
        if (threadIdx.x == 0) p.seq_lens[dst] = len;
        return;
    }
    int old;
    if (fresh < 0 || !fork_partial(p, src, len, &old)) return;
    const int64_t pb = c.page_bytes[blockIdx.y - 1];
    uint8_t* base = c.base[blockIdx.y - 1];
    copy_bytes(base + fresh * pb, base + old * pb, pb / p.page_size * (len % p.page_size), threadIdx.x, blockDim.x);
}

// ------------------------------------------------------------------ compacting
struct CompactArgs {
    const int32_t* refs;
    int32_t* out_refs;
    int64_t num_pages;
    int32_t* num_live;
    int32_t* moves;      // number of pages that move
    int32_t* counts;     // [blocks]: live pages of each block's pages
    int32_t* src;        // [num_pages]
    int32_t* dst;
    int32_t* src_refs;
    int32_t* remap;      // page -> its new id, -1 for a free one, -2 - k for the k-th that moves
    const int32_t* tables;
    int64_t stride, num_slots, out_stride;
    int width;
    int32_t* out_tables;
    int32_t* err;
};
constexpr int kPer = 4, kBlockPages = kPlanThreads * kPer;      // pages of a thread, of a block

// kPer consecutive counts of a thread (0 past the end).
__device__ __forceinline__ void load_counts(const int32_t* refs, int64_t i0, int64_t num, int (&r)[kPer]) {
    if (i0 + kPer <= num && reinterpret_cast<uintptr_t>(refs) % 16 == 0) {
        const int4 v = *reinterpret_cast<const int4*>(refs + i0);
        r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
    } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) r[j] = i0 + j < num ? refs[i0 + j] : 0;
    }
}

__global__ void __launch_bounds__(kPlanThreads) compact_count_kernel(const __grid_constant__ CompactArgs p) {
    __shared__ int sums[32];
    int r[kPer], live = 0, total;
    griddep_wait();
    load_counts(p.refs, static_cast<int64_t>(blockIdx.x) * kBlockPages + threadIdx.x * kPer, p.num_pages, r);
#pragma unroll
    for (int j = 0; j < kPer; ++j) live += r[j] > 0;
    block_exclusive_scan(live, sums, &total);
    if (threadIdx.x == 0) p.counts[blockIdx.x] = total;
    griddep_launch_dependents();
}

// With n = live pages in all: the k-th live page past n goes to the k-th hole before it.  A page's
// number among the live ones is the live pages of the blocks before its own plus a scan; that of a
// hole before n is its index less that; that of a live page past n is that less the live pages
// before n, which every block counts for itself.  A pool of one block needs no counting kernel (42,405 pages: counting 2.6 us, this 7.4, the tables
// 4.2; one block alone took 70).  (In place, only counts of free pages and of
// pages past n change, which no other block's counting depends on.)
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const __grid_constant__ CompactArgs p) {
    __shared__ int sums[3][32];
    const int tid = threadIdx.x, blocks = gridDim.x;
    griddep_wait();
    const int64_t i0 = static_cast<int64_t>(blockIdx.x) * kBlockPages + tid * kPer;
    int r[kPer], live = 0, total, n, before = 0, part = 0, live_low;
    load_counts(p.refs, i0, p.num_pages, r);
#pragma unroll
    for (int j = 0; j < kPer; ++j) live += r[j] > 0;
    if (blocks == 1) {                                      // (nothing was counted before)
        block_exclusive_scan(live, sums[0], &n);
#pragma unroll
        for (int j = 0; j < kPer; ++j) part += r[j] > 0 && i0 + j < n;
    } else {
        int all = 0, below = 0;
        for (int b = tid; b < blocks; b += kPlanThreads) {
            const int c = p.counts[b];
            all += c;
            if (b < static_cast<int>(blockIdx.x)) below += c;
        }
        block_exclusive_scan(all, sums[0], &n);
        block_exclusive_scan(below, sums[1], &before);
        // live pages before page n: whole blocks, and the part of n's own
        const int nb = n / kBlockPages;
        for (int b = tid; b < nb; b += kPlanThreads) part += p.counts[b];
        int low[kPer];
        load_counts(p.refs, static_cast<int64_t>(nb) * kBlockPages + tid * kPer, n, low);
#pragma unroll
        for (int j = 0; j < kPer; ++j) part += low[j] > 0;
    }
    block_exclusive_scan(part, sums[2], &live_low);
    __syncthreads();
    int rank = before + block_exclusive_scan(live, sums[0], &total);      // live pages before the thread's first
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int64_t i = i0 + j;
        if (i >= p.num_pages) break;
        if (r[j] > 0) {
            if (i >= n) {
                const int k = rank - live_low;
                p.src[k] = static_cast<int>(i);
                p.src_refs[k] = r[j];
                p.remap[i] = -2 - k;
                p.out_refs[i] = 0;
            } else {
                p.remap[i] = static_cast<int>(i);
                p.out_refs[i] = r[j];
            }
            ++rank;
        } else {
            if (i < n) p.dst[i - rank] = static_cast<int>(i);      // (its count comes with the page that moves in)
            else p.out_refs[i] = 0;
            p.remap[i] = -1;
        }
    }
    if (blockIdx.x == 0 && tid == 0) {
        *p.num_live = n;
        *p.moves = n - live_low;
    }
    griddep_launch_dependents();
}

// The tables by the new ids, and the counts of the pages that moved.
__global__ void __launch_bounds__(256) compact_tables_kernel(const __grid_constant__ CompactArgs p) {
    griddep_wait();
    const int64_t first = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * blockDim.x;
    const int64_t n = p.num_slots * p.width;
    for (int64_t i = first; i < n; i += step) {
        const int64_t s = i / p.width, j = i - s * p.width;
        const int pg = p.tables[s * p.stride + j];
        int q = -1;
        if (pg >= 0) {
            if (pg < p.num_pages) q = p.remap[pg];
            if (q <= -2) q = p.dst[-2 - q];
            if (q < 0) set_error(p.err, NVFP4KV_DEVERR_BAD_PAGE);
        }
        p.out_tables[s * p.out_stride + j] = q;
    }
    const int moves = *p.moves;
    for (int64_t k = first; k < moves; k += step) p.out_refs[p.dst[k]] = p.src_refs[k];
}

int gather_caches(const char* what, const void* const* caches, const int64_t* page_bytes, int num, int page_size, Caches* c) {
    if (num < 0 || num > NVFP4KV_MAX_CACHES)
        return fail(NVFP4KV_EINVAL, "%s: %d caches (at most %d)", what, num, NVFP4KV_MAX_CACHES);
    if (num > 0 && (!caches || !page_bytes)) return fail(NVFP4KV_EINVAL, "%s: null cache list", what);
    *c = Caches{};
    for (int k = 0; k < num; ++k) {
        if (!caches[k]) return fail(NVFP4KV_EINVAL, "%s: null cache %d", what, k);
        if (page_bytes[k] < 1 || page_bytes[k] % page_size)
            return fail(NVFP4KV_EINVAL, "%s: page_bytes[%d] must be a positive multiple of the page size", what, k);
        c->base[k] = static_cast<uint8_t*>(const_cast<void*>(caches[k]));
        c->page_bytes[k] = page_bytes[k];
    }
    c->num = num;
    return NVFP4KV_OK;
}

int check_tables(const char* what, const void* tables, int64_t stride, int width, int64_t num_slots, const void* refs,
                 int64_t num_pages) {
    if (!tables || !refs) return fail(NVFP4KV_EINVAL, "%s: null pointer", what);
    if (width < 1 || stride < width || num_slots < 1)
        return fail(NVFP4KV_EINVAL, "%s: bad table shape (width %d, stride %lld, %lld slots)", what, width,
                    (long long)stride, (long long)num_slots);
    if (num_pages < 1 || num_pages >= 0x7FFFFFFFll) return fail(NVFP4KV_EINVAL, "%s: bad num_pages", what);
    return NVFP4KV_OK;
}

// Moves (with a pad), counts of the blocks, and four lists of pages.
int64_t compact_ints(int64_t num_pages) { return 4 + (num_pages + kBlockPages - 1) / kBlockPages + 4 * num_pages; }

int launch_copy(const Caches& c, int64_t num_pages, const int32_t* src, const int32_t* dst, int64_t num,
                const int32_t* num_dev, int64_t most_pairs, int32_t* err, cudaStream_t st) {
    if (c.num == 0) return NVFP4KV_OK;
    uint64_t align = 0;
    CopyPieces pieces{};
    for (int k = 0; k < c.num; ++k) {
        align |= reinterpret_cast<uint64_t>(c.base[k]) | static_cast<uint64_t>(c.page_bytes[k]);
        const int64_t cut = (c.page_bytes[k] + kCopyBytes - 1) / kCopyBytes;
        pieces.bytes[k] = static_cast<int>(((c.page_bytes[k] + cut - 1) / cut + 15) / 16 * 16);
        pieces.first[k + 1] = pieces.first[k] + static_cast<int>((c.page_bytes[k] + pieces.bytes[k] - 1) / pieces.bytes[k]);
    }
    cudaError_t e;
    if (align % 16 == 0) {      // what a bulk copy can move
        static_assert(kCopyStages * kCopyBytes * 3 <= 227 * 1024, "three blocks on an SM");
        static int done[64] = {0};      // (a device's limit, set once)
        int dev = 0;
        e = cudaGetDevice(&dev);
        if (e == cudaSuccess && (dev >= 64 || !done[dev])) {
            e = cudaFuncSetAttribute(bulk_copy_pages_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kCopyStages * kCopyBytes);
            if (e == cudaSuccess && dev < 64) done[dev] = 1;
        }
        int64_t blocks = 3 * device_sm_count();
        blocks = blocks < most_pairs * pieces.first[c.num] ? blocks : most_pairs * pieces.first[c.num];
        if (e == cudaSuccess)
            e = launch_dependent(bulk_copy_pages_kernel, dim3(static_cast<unsigned>(blocks)), dim3(32), kCopyStages * kCopyBytes, st, c,
                                 pieces, num_pages, src, dst, num, num_dev, err);
    } else {
        const int64_t blocks = most_pairs < 8 * device_sm_count() ? most_pairs : 8 * device_sm_count();
        e = launch_dependent(copy_pages_kernel, dim3(static_cast<unsigned>(blocks), c.num), dim3(256), 0, st, c, num_pages, src, dst,
                             num, num_dev, err);
    }
    if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "page copy launch failed: %s", cudaGetErrorString(e));
    return check_launch("page copy");
}

}  // namespace
}  // namespace nvfp4kv

extern "C" int nvfp4kv_copy_pages(const void* const* caches, const int64_t* page_bytes, int num_caches,
                                  int64_t num_pages, const int32_t* src, const int32_t* dst, int64_t num_pairs,
                                  int32_t* err_flag, nvfp4kv_stream_t stream) {
    using namespace nvfp4kv;
    if (num_pairs < 0) return fail(NVFP4KV_EINVAL, "nvfp4kv_copy_pages: num_pairs < 0");
    Caches c;
    int rc = gather_caches("nvfp4kv_copy_pages", caches, page_bytes, num_caches, 1, &c);
    if (rc != NVFP4KV_OK) return rc;
    if (num_pairs == 0) return NVFP4KV_OK;
    if (!src || !dst) return fail(NVFP4KV_EINVAL, "nvfp4kv_copy_pages: null pointer");
    if (num_pages < 1 || num_pages >= 0x7FFFFFFFll) return fail(NVFP4KV_EINVAL, "nvfp4kv_copy_pages: bad num_pages");
    return launch_copy(c, num_pages, src, dst, num_pairs, nullptr, num_pairs, err_flag, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int nvfp4kv_free_pages(int32_t* block_tables, int64_t tables_stride, int table_width, int64_t num_slots,
                                  int32_t* seq_lens, const int32_t* slots, int num, int32_t* ref_counts,
                                  int64_t num_pages, int32_t* err_flag, nvfp4kv_stream_t stream) {
    using namespace nvfp4kv;
    if (num < 0) return fail(NVFP4KV_EINVAL, "nvfp4kv_free_pages: num < 0");
    if (num == 0) return NVFP4KV_OK;
    if (!slots || !seq_lens) return fail(NVFP4KV_EINVAL, "nvfp4kv_free_pages: null pointer");
    int rc = check_tables("nvfp4kv_free_pages", block_tables, tables_stride, table_width, num_slots, ref_counts, num_pages);
    if (rc != NVFP4KV_OK) return rc;
    const cudaError_t e = launch_dependent(free_pages_kernel, dim3(num), dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), block_tables,
                                           tables_stride, table_width, num_slots, seq_lens, slots, ref_counts, num_pages, err_flag);
    if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "nvfp4kv_free_pages launch failed: %s", cudaGetErrorString(e));
    return check_launch("nvfp4kv_free_pages");
}

extern "C" int nvfp4kv_fork_pages(const void* const* caches, const int64_t* page_bytes, int num_caches, int page_size,
                                  int32_t* block_tables, int64_t tables_stride, int table_width, int64_t num_slots,
                                  int32_t* seq_lens, const int32_t* src, const int32_t* dst, int num,
                                  int32_t* ref_counts, int64_t num_pages, int32_t* workspace,
                                  int64_t workspace_ints, int32_t* err_flag, nvfp4kv_stream_t stream) {
    using namespace nvfp4kv;
    if (num < 0) return fail(NVFP4KV_EINVAL, "nvfp4kv_fork_pages: num < 0");
    if (page_size < 1) return fail(NVFP4KV_EINVAL, "nvfp4kv_fork_pages: page_size must be >= 1");
    Caches c;
    int rc = gather_caches("nvfp4kv_fork_pages", caches, page_bytes, num_caches, page_size, &c);
    if (rc != NVFP4KV_OK) return rc;
    if (num == 0) return NVFP4KV_OK;
    if (!src || !dst || !seq_lens) return fail(NVFP4KV_EINVAL, "nvfp4kv_fork_pages: null pointer");
    rc = check_tables("nvfp4kv_fork_pages", block_tables, tables_stride, table_width, num_slots, ref_counts, num_pages);
    if (rc != NVFP4KV_OK) return rc;
    if (!workspace || workspace_ints < 3ll * num)
        return fail(NVFP4KV_EWORKSPACE, "nvfp4kv_fork_pages: workspace %lld ints < %lld required",
                    (long long)workspace_ints, 3ll * num);
    ForkArgs a{};
    a.tables = block_tables; a.stride = tables_stride; a.width = table_width; a.page_size = page_size;
    a.num_slots = num_slots; a.seq_lens = seq_lens; a.src = src; a.dst = dst; a.num = num;
    a.refs = ref_counts; a.num_pages = num_pages; a.fresh = workspace; a.free_list = workspace + num; a.lens = a.free_list + num;
    a.err = err_flag;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e = launch_dependent(fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a);
    if (e == cudaSuccess) e = launch_dependent(fork_apply_kernel, dim3(num, 1 + num_caches), dim3(256), 0, st, a, c);
    if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "nvfp4kv_fork_pages launch failed: %s", cudaGetErrorString(e));
    return check_launch("nvfp4kv_fork_pages");
}

extern "C" int nvfp4kv_compact_workspace_ints(int64_t num_pages, int64_t* ints) {
    using namespace nvfp4kv;
    if (!ints) return fail(NVFP4KV_EINVAL, "nvfp4kv_compact_workspace_ints: null output");
    if (num_pages < 1) return fail(NVFP4KV_EINVAL, "nvfp4kv_compact_workspace_ints: bad num_pages");
    *ints = compact_ints(num_pages);
    return NVFP4KV_OK;
}

extern "C" int nvfp4kv_compact_pages(const void* const* caches, const int64_t* page_bytes, int num_caches,
                                     const int32_t* block_tables, int64_t tables_stride, int table_width,
                                     int64_t num_slots, const int32_t* ref_counts, int64_t num_pages,
                                     int32_t* out_tables, int64_t out_tables_stride, int32_t* out_ref_counts,
                                     int32_t* num_live, int32_t* workspace, int64_t workspace_ints,
                                     int32_t* err_flag, nvfp4kv_stream_t stream) {
    using namespace nvfp4kv;
    Caches c;
    int rc = gather_caches("nvfp4kv_compact_pages", caches, page_bytes, num_caches, 1, &c);
    if (rc != NVFP4KV_OK) return rc;
    rc = check_tables("nvfp4kv_compact_pages", block_tables, tables_stride, table_width, num_slots, ref_counts, num_pages);
    if (rc != NVFP4KV_OK) return rc;
    if (!out_tables || !out_ref_counts || !num_live || out_tables_stride < table_width)
        return fail(NVFP4KV_EINVAL, "nvfp4kv_compact_pages: null or too narrow output");
    if (!workspace || workspace_ints < compact_ints(num_pages))
        return fail(NVFP4KV_EWORKSPACE, "nvfp4kv_compact_pages: workspace %lld ints < %lld required",
                    (long long)workspace_ints, (long long)compact_ints(num_pages));
    CompactArgs a{};
    a.refs = ref_counts; a.out_refs = out_ref_counts; a.num_pages = num_pages; a.num_live = num_live;
    const int blocks = static_cast<int>((num_pages + kBlockPages - 1) / kBlockPages);
    a.moves = workspace; a.counts = workspace + 4; a.src = a.counts + blocks; a.dst = a.src + num_pages;
    a.src_refs = a.dst + num_pages; a.remap = a.src_refs + num_pages;
    a.tables = block_tables; a.stride = tables_stride; a.width = table_width; a.num_slots = num_slots;
    a.out_tables = out_tables; a.out_stride = out_tables_stride; a.err = err_flag;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int64_t want = (num_slots * table_width + 255) / 256, most = 8 * device_sm_count();
    cudaError_t e = cudaSuccess;
    if (blocks > 1) e = launch_dependent(compact_count_kernel, dim3(blocks), dim3(kPlanThreads), 0, st, a);
    if (e == cudaSuccess) e = launch_dependent(compact_plan_kernel, dim3(blocks), dim3(kPlanThreads), 0, st, a);
    if (e == cudaSuccess)
        e = launch_dependent(compact_tables_kernel, dim3(static_cast<unsigned>(want < most ? want : most)), dim3(256), 0, st, a);
    if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "nvfp4kv_compact_pages launch failed: %s", cudaGetErrorString(e));
    if ((rc = check_launch("nvfp4kv_compact_pages")) != NVFP4KV_OK) return rc;
    return launch_copy(c, num_pages, a.src, a.dst, 0, a.moves, num_pages, err_flag, st);
}
