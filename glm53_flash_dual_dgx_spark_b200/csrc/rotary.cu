// Rotary positions: nvfp4kv_rope (whole heads, any layout) and nvfp4kv_append_rope_rotated (the
// rope part of a step: rotated keys into the paged side-pool, queries rotated beside them), and
// both with positions on several axes (nvfp4kv_rope_axes, nvfp4kv_append_rope_rotated_axes).
//
// A pair (a, b) of a head turns by its token's angle: (a c - b s, b c + a s), in fp32, rounded
// once.  cos and sin come from the caller's table, so that scaled frequencies cost nothing here
// and no large angle is reduced on the device.  Both operators read and write each value once
// and are bound by HBM (latency for a few tokens); the table row is read by every head of its
// token and stays in L1.
#include "../../include/nvfp4kv_serving.h"
#include "abi_common.h"
#include "common.cuh"
#include "decode_shared.h"

namespace nvfp4kv {
namespace {

template <typename T> __device__ __forceinline__ float load_f32(const T* p) { return static_cast<float>(*p); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// 16 bytes of T as fp32 values and back.
template <typename T> struct Vec {
    static constexpr int kN = 16 / sizeof(T);
    T v[kN];
};
template <typename T, bool kStream = false> __device__ __forceinline__ Vec<T> load_vec(const T* p) {
    const uint4* src = reinterpret_cast<const uint4*>(p);
    const uint4 u = kStream ? __ldcs(src) : *src;
    Vec<T> r;
    memcpy(&r, &u, 16);
    return r;
}
template <typename T, bool kStream = false> __device__ __forceinline__ void store_vec(T* p, const Vec<T>& r) {
    uint4 u;
    memcpy(&u, &r, 16);
    if (kStream) __stcs(reinterpret_cast<uint4*>(p), u);
    else *reinterpret_cast<uint4*>(p) = u;
}

__device__ __forceinline__ int64_t load_index(const void* p, bool i64, int64_t i) {
    return i64 ? static_cast<int64_t>(__ldg(static_cast<const long long*>(p) + i))
               : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(p) + i));
}

__device__ __forceinline__ void rotate(float a, float b, float c, float s, float& u, float& v) {
    u = a * c - b * s;
    v = b * c + a * s;
}

// N consecutive cos (or sin) values, N a multiple of 4 or 2, 8-byte aligned, of the table or in shared memory.
template <int N, bool kShared> __device__ __forceinline__ void load_angles(const float* p, float (&r)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int k = 0; k < N / 4; ++k) {
            const float4* src = reinterpret_cast<const float4*>(p) + k;
            const float4 f = kShared ? *src : __ldg(src);
            r[4 * k] = f.x; r[4 * k + 1] = f.y; r[4 * k + 2] = f.z; r[4 * k + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int k = 0; k < N / 2; ++k) {
            const float2* src = reinterpret_cast<const float2*>(p) + k;
            const float2 f = kShared ? *src : __ldg(src);
            r[2 * k] = f.x; r[2 * k + 1] = f.y;
        }
    }
}

// Positions on several axes: the axis of each pair, two bits each, 32 pairs a word.
struct Axes {
    uint64_t pair_axes[NVFP4KV_MAX_AXES_DIM / 64];
    int64_t stride;      // between the axes of positions
    int num;
};
// The angles of a token: a row of cos | sin, from the table or gathered from the rows of its axes, and
// whether its positions are in the table.
struct Angles {
    const float* row;
    bool turn;
};
__device__ __forceinline__ Angles find_angles(const void* positions, bool i64, int64_t t, const float* table, int64_t max_positions, int rotary) {
    const int64_t pos = load_index(positions, i64, t);
    const bool turn = pos >= 0 && pos < max_positions;
    return {table + (turn ? pos : 0) * rotary, turn};
}
__device__ __forceinline__ uint32_t axis_of(const Axes& axes, int pair) {
    return static_cast<uint32_t>(axes.pair_axes[pair >> 5] >> (2 * (pair & 31))) & 3u;
}
__device__ __forceinline__ bool all_in_table(const void* positions, bool i64, int64_t t, const Axes& axes, int64_t max_positions) {
    bool in = true;
#pragma unroll
    for (int a = 0; a < NVFP4KV_MAX_AXES; ++a) {
        const int64_t pos = a < axes.num ? load_index(positions, i64, a * axes.stride + t) : 0;
        in &= pos >= 0 && pos < max_positions;
    }
    return in;
}

// One 16-byte vector of an interleaved rotation: pairs inside the vector.  cs -> cos of its first pair.
template <typename T, bool kShared>
__device__ __forceinline__ Vec<T> rotate_pairs(const Vec<T>& x, const float* cs, int half, float sign) {
    constexpr int N = Vec<T>::kN;
    float c[N / 2], s[N / 2];
    load_angles<N / 2, kShared>(cs, c);
    load_angles<N / 2, kShared>(cs + half, s);
    Vec<T> y;
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
        float u, v;
        rotate(load_f32(&x.v[2 * k]), load_f32(&x.v[2 * k + 1]), c[k], sign * s[k], u, v);
        y.v[2 * k] = from_f32<T>(u);
        y.v[2 * k + 1] = from_f32<T>(v);
    }
    return y;
}

// The two vectors of a half-layout rotation: dims i.. and i + half.. .
template <typename T, bool kShared>
__device__ __forceinline__ void rotate_halves(Vec<T>& xa, Vec<T>& xb, const float* cs, int half, float sign) {
    constexpr int N = Vec<T>::kN;
    float c[N], s[N];
    load_angles<N, kShared>(cs, c);
    load_angles<N, kShared>(cs + half, s);
#pragma unroll
    for (int k = 0; k < N; ++k) {
        float u, v;
        rotate(load_f32(&xa.v[k]), load_f32(&xb.v[k]), c[k], sign * s[k], u, v);
        xa.v[k] = from_f32<T>(u);
        xb.v[k] = from_f32<T>(v);
    }
}

// Quotients by a number the host knows, for the small dividends of one block (up to a few thousand
// plus the divisor): a multiplication by ceil(2^32 / d).
constexpr int kMostDivisor = 32768;
struct SmallDiv {
    uint32_t d, magic;
};
__device__ __forceinline__ uint32_t quotient(uint32_t n, const SmallDiv& v) { return v.d == 1 ? n : __umulhi(n, v.magic); }

// With several axes, a block gathers the cos | sin rows of its `num` tokens from t0 on in shared memory
// once, so that its units read them as 16-byte vectors like a row of the table, whichever way the
// axes are spread over the pairs (loaded pair by pair in every unit they took as many load slots as the
// values themselves: 8,192 tokens x 32 heads x 128 bf16 42 us; now 21.9, as much as a plain copy).  It
// comes before the units' own loads: behind them their addresses stay in registers, and fewer blocks fit
// (31.6 us against 28.3 before the vectors were marked as streaming; with the vectors through shared
// memory by asynchronous copies, asked for before the gathering, 34.5).  The schedulers issue in two of
// three cycles, so the index arithmetic counts.  rows [num][rotary], turns [num].
__device__ __forceinline__ void gather_rows(float* rows, uint8_t* turns, int num, int64_t t0, int64_t tokens, const void* positions,
                                            bool i64, const Axes& axes, const SmallDiv& half, const float* table, int64_t max_positions) {
    const int h = static_cast<int>(half.d);
    for (int l = threadIdx.x; l < num * h; l += blockDim.x) {
        const int k = static_cast<int>(quotient(l, half)), i = l - k * h;
        const int64_t t = t0 + k;
        if (t >= tokens) break;
        const int64_t pos = load_index(positions, i64, axis_of(axes, i) * axes.stride + t);
        const float* src = table + (pos >= 0 && pos < max_positions ? pos : 0) * (2 * h) + i;
        rows[2 * h * k + i] = __ldg(src);
        rows[2 * h * k + h + i] = __ldg(src + h);
    }
    // (by the threads that have no pair, where there are some: in the loop above, by the first pair's lane, every
    // warp waited for it; 65,536 tokens x 1 head x 128 bf16 took 32 us, so 24.4)
    for (int k = blockDim.x - 1 - threadIdx.x; k < num && t0 + k < tokens; k += blockDim.x)
        turns[k] = all_in_table(positions, i64, t0 + k, axes, max_positions);
    __syncthreads();
}

// The same for any dividend: the product's upper half is the quotient, or one more.
__device__ __forceinline__ uint32_t any_quotient(uint32_t n, const SmallDiv& v) {
    const uint32_t q = quotient(n, v);
    return q - (static_cast<int>(n - q * v.d) < 0);
}

inline SmallDiv small_div(uint32_t d) { return {d, static_cast<uint32_t>(((1ull << 32) + d - 1) / d)}; }

struct RopeArgs {
    const void* x;
    void* out;
    int64_t x_st, x_sh, o_st, o_sh;
    const void* positions;
    const float* cos_sin;
    int64_t max_positions, tokens, total;      // total: units of the call
    int heads, dim, rotary, offset;
    int before, rotated;    // units of a head: copies before the rotated part, rotated ones, copies after it
    SmallDiv units, by_heads;
    int pos_i64, inverse, in_place;
    int32_t* err;
    Axes axes;
    SmallDiv half;          // with several axes: rotary / 2, the tokens of a block at most
    int block_tokens;
};
constexpr int kRopeSteps = 2;

// A unit is a 16-byte vector of a head (a rotated one of the half layout: the pair of vectors that
// turn together).  The units of the call are dealt flat, two to a thread and 256 apart: every warp
// moves 512 contiguous bytes, every block is full, and two loads in flight per thread are enough at
// the occupancy that leaves (8,192 tokens x 64 heads x 576 bf16, 1.2 GB: 180 us = 6.7 TB/s, where a
// plain copy of the same tensors takes 184.5; 8 % more with one, 1 % more with four, 20 % more with
// blocks of whole heads, whose last steps are part empty).  The gradient of 2,049 tokens x 32 heads x 128 fp32 takes 10 us.
//
// With several axes the vectors are marked as streaming: with new inputs each time, 8,192 tokens x 32
// heads x 128 bf16 26.1 -> 24.4 us, the gradient of 2,049 x 20 x 192 fp32 14.9 -> 12.4 (marks on the
// loads or the stores alone gain a tenth of that); six blocks fit in the half layout, 27.6 -> 26.1.
template <typename T, bool kInterleaved, bool kAxes>
__global__ void __launch_bounds__(256, kAxes ? (kInterleaved ? 8 : 6) : (kInterleaved && sizeof(T) == 2 ? 8 : 4)) rope_vec_kernel(const __grid_constant__ RopeArgs p) {
    constexpr int N = Vec<T>::kN;
    const int64_t u0 = static_cast<int64_t>(blockIdx.x) * (256 * kRopeSteps);
    int64_t row0, t0;       // the block's first head row, its token
    if (p.total < (1ll << 32)) {
        row0 = any_quotient(static_cast<uint32_t>(u0), p.units);
        t0 = any_quotient(static_cast<uint32_t>(row0), p.by_heads);
    } else {
        row0 = u0 / p.units.d;
        t0 = row0 / p.by_heads.d;
    }
    const uint32_t j0 = static_cast<uint32_t>(u0 - row0 * p.units.d), h0 = static_cast<uint32_t>(row0 - t0 * p.by_heads.d);
    const int half = p.rotary / 2;
    griddep_wait();
    extern __shared__ __align__(16) float block_rows[];
    uint8_t* turns = reinterpret_cast<uint8_t*>(block_rows + p.block_tokens * p.rotary);
    if constexpr (kAxes)
        gather_rows(block_rows, turns, p.block_tokens, t0, p.tokens, p.positions, p.pos_i64, p.axes, p.half, p.cos_sin, p.max_positions);
    Vec<T> a[kRopeSteps], b[kRopeSteps];
    int64_t t[kRopeSteps], at[kRopeSteps];
    int r[kRopeSteps];      // dim within the rotated part, -1 for a copy, -2 past the end
#pragma unroll
    for (int k = 0; k < kRopeSteps; ++k) {
        const uint32_t l = j0 + threadIdx.x + 256 * k, lr = quotient(l, p.units);
        const int j = static_cast<int>(l - lr * p.units.d);
        const uint32_t lh = h0 + lr, lt = quotient(lh, p.by_heads), h = lh - lt * p.by_heads.d;
        t[k] = t0 + lt;
        const int q = j - p.before;
        r[k] = q < 0 || q >= p.rotated ? -1 : q * N;
        const int d = q < 0 ? j * N : q < p.rotated ? p.offset + q * N : p.offset + p.rotary + (q - p.rotated) * N;
        at[k] = t[k] * p.o_st + h * p.o_sh + d;
        if (u0 + threadIdx.x + 256 * k < p.total) {
            const T* xp = static_cast<const T*>(p.x) + t[k] * p.x_st + h * p.x_sh + d;
            a[k] = load_vec<T, kAxes>(xp);
            if (!kInterleaved && r[k] >= 0) b[k] = load_vec<T, kAxes>(xp + half);
        } else {
            r[k] = -2;
        }
    }
#pragma unroll
    for (int k = 0; k < kRopeSteps; ++k) {
        if (r[k] == -2) break;
        T* op = static_cast<T*>(p.out) + at[k];
        if (r[k] >= 0) {
            const int l = static_cast<int>(t[k] - t0);
            const Angles g = kAxes ? Angles{block_rows + l * p.rotary, turns[l] != 0}
                                   : find_angles(p.positions, p.pos_i64, t[k], p.cos_sin, p.max_positions, p.rotary);
            if (!g.turn) set_error(p.err, NVFP4KV_DEVERR_BAD_INDEX);
            const float* cs = g.row + (kInterleaved ? r[k] / 2 : r[k]);
            const float sign = p.inverse ? -1.0f : 1.0f;
            if (kInterleaved) {
                if (g.turn) a[k] = rotate_pairs<T, kAxes>(a[k], cs, half, sign);
            } else {
                if (g.turn) rotate_halves<T, kAxes>(a[k], b[k], cs, half, sign);
                store_vec<T, kAxes>(op + half, b[k]);
            }
        }
        store_vec<T, kAxes>(op, a[k]);
    }
}

// Any strides, alignment and sizes: one element (a rotated dim: its pair) per thread and step, for rows
// that no 16-byte access can take (views at an odd offset, heads of odd sizes).  It is bound by its
// 2- or 4-byte accesses and a division per element: 8,192 tokens x 64 heads x 192 bf16, shifted by 3,
// take 395 us where the bytes take 62 (1.0 TB/s; fp32 2.1), with three axes, whose positions every pair
// looks up, 510.  A caller that can align its rows should.
template <typename T, bool kInterleaved, bool kAxes>
__global__ void __launch_bounds__(256) rope_elem_kernel(const __grid_constant__ RopeArgs p, int head_blocks, int heads_per_block) {
    const int64_t t = blockIdx.x / head_blocks;
    const int h0 = static_cast<int>(blockIdx.x % head_blocks) * heads_per_block;
    const int heads = min(heads_per_block, p.heads - h0);
    Angles g = kAxes ? Angles{p.cos_sin, all_in_table(p.positions, p.pos_i64, t, p.axes, p.max_positions)}
                     : find_angles(p.positions, p.pos_i64, t, p.cos_sin, p.max_positions, p.rotary);
    if (!g.turn && threadIdx.x == 0) set_error(p.err, NVFP4KV_DEVERR_BAD_INDEX);
    const int half = p.rotary / 2;
    const float sign = p.inverse ? -1.0f : 1.0f;
    const T* x = static_cast<const T*>(p.x) + t * p.x_st + h0 * p.x_sh;
    T* o = static_cast<T*>(p.out) + t * p.o_st + h0 * p.o_sh;
    for (int u = threadIdx.x; u < heads * p.dim; u += blockDim.x) {
        const int h = u / p.dim, d = u - h * p.dim;
        const T* xp = x + h * p.x_sh;
        T* op = o + h * p.o_sh;
        const int r = d - p.offset;
        if (r < 0 || r >= p.rotary || !g.turn) {
            op[d] = xp[d];
            continue;
        }
        const int i = kInterleaved ? r / 2 : r;
        if (kInterleaved ? (r & 1) : r >= half) continue;      // done with its partner
        const int db = kInterleaved ? d + 1 : d + half;
        if (kAxes) g.row = p.cos_sin + load_index(p.positions, p.pos_i64, axis_of(p.axes, i) * p.axes.stride + t) * p.rotary;
        const float* cs = g.row;
        float u0, v0;
        rotate(load_f32(xp + d), load_f32(xp + db), __ldg(cs + i), sign * __ldg(cs + half + i), u0, v0);
        op[d] = from_f32<T>(u0);
        op[db] = from_f32<T>(v0);
    }
}

template <typename T, bool kAxes>
int launch_rope(RopeArgs a, int64_t tokens, bool interleaved, cudaStream_t st) {
    constexpr int N = Vec<T>::kN;
    const uintptr_t bases = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.out);
    // 16-byte vectors need every row, and each rotated vector's partner, on a 16-byte boundary
    const bool vec = bases % 16 == 0 && reinterpret_cast<uintptr_t>(a.cos_sin) % 16 == 0 && a.x_st % N == 0 &&
                     a.x_sh % N == 0 && a.o_st % N == 0 && a.o_sh % N == 0 && a.dim % N == 0 && a.offset % N == 0 &&
                     a.rotary % (interleaved ? N : 2 * N) == 0 &&
                     a.heads <= kMostDivisor && a.dim <= kMostDivisor;
    int64_t blocks;
    if (vec) {
        // in place only the rotated dims are visited
        a.rotated = a.rotary / (interleaved ? N : 2 * N);
        a.before = a.in_place ? 0 : a.offset / N;
        const uint32_t units = a.rotated + (a.in_place ? 0 : (a.dim - a.rotary) / N), heads = a.heads;
        a.units = small_div(units);
        a.by_heads = small_div(heads);
        a.total = tokens * heads * units;
        blocks = (a.total + 256 * kRopeSteps - 1) / (256 * kRopeSteps);
        size_t smem = 0;
        if (kAxes) {
            // a block's units begin anywhere in a token's; they touch at most 16 KB of rows (32 KB in the
            // half layout, whose units are two vectors) and two rows more
            const int64_t per_token = static_cast<int64_t>(heads) * units, most = (256 * kRopeSteps + per_token - 2) / per_token + 1;
            a.block_tokens = static_cast<int>(most < tokens ? most : tokens);
            a.half = small_div(a.rotary / 2);
            smem = a.block_tokens * (a.rotary * sizeof(float) + 1);
        }
        if (blocks > 0x7FFFFFFF) return fail(NVFP4KV_EINVAL, "nvfp4kv_rope: too many rows for one call");
        const cudaError_t e = launch_dependent(interleaved ? rope_vec_kernel<T, true, kAxes> : rope_vec_kernel<T, false, kAxes>, dim3(static_cast<unsigned>(blocks)), dim3(256), smem, st, a);
        if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "nvfp4kv_rope launch failed: %s", cudaGetErrorString(e));
    } else {
        int hb = 1024 / a.dim;
        hb = hb < 1 ? 1 : (hb > a.heads ? a.heads : hb);
        const int head_blocks = (a.heads + hb - 1) / hb, per_block = (a.heads + head_blocks - 1) / head_blocks;
        blocks = tokens * head_blocks;
        if (blocks > 0x7FFFFFFF) return fail(NVFP4KV_EINVAL, "nvfp4kv_rope: too many rows for one call");
        if (interleaved) rope_elem_kernel<T, true, kAxes><<<static_cast<unsigned>(blocks), 256, 0, st>>>(a, head_blocks, per_block);
        else rope_elem_kernel<T, false, kAxes><<<static_cast<unsigned>(blocks), 256, 0, st>>>(a, head_blocks, per_block);
    }
    return check_launch("nvfp4kv_rope");
}

constexpr int kAppendRows = 64, kHalfSteps = 2;      // rows of a block and step (four threads a row); steps in the half layout

struct RopeAppendArgs {
    const __nv_bfloat16* k;
    int64_t k_st, tokens;
    __nv_bfloat16* pool;
    int64_t rows;
    const void* slots;
    const void* positions;
    const float* cos_sin;
    int64_t max_positions;
    const __nv_bfloat16* q;
    __nv_bfloat16* qo;
    int64_t q_st, q_sh, qo_st, qo_sh;
    int heads;                 // 0 without queries
    SmallDiv rows_of_token;    // heads + 1
    int slot_i64, pos_i64;
    int32_t* err;
    Axes axes;
    int block_tokens;          // with several axes: the tokens of a block at most
};

// 8 bf16, as one 16-byte access or element by element.  The accesses are marked as streaming: a step's
// rows pass once, while the table rows of its positions come back with every layer, and should stay
// in L2 (32,768 tokens x 16 heads over a table of 77 MB: 28.0 us against 33.3 without the marks, and
// 29.8 with the next blocks' table rows prefetched instead; with the units below 25.2).
template <bool kVec> __device__ __forceinline__ Vec<__nv_bfloat16> get8(const __nv_bfloat16* p) {
    if constexpr (kVec) {
        const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
        Vec<__nv_bfloat16> r;
        memcpy(&r, &u, 16);
        return r;
    } else {
        Vec<__nv_bfloat16> r;
#pragma unroll
        for (int k = 0; k < 8; ++k) r.v[k] = p[k];
        return r;
    }
}
template <bool kVec> __device__ __forceinline__ void put8(__nv_bfloat16* p, const Vec<__nv_bfloat16>& r) {
    if constexpr (kVec) {
        uint4 u;
        memcpy(&u, &r, 16);
        __stcs(reinterpret_cast<uint4*>(p), u);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) p[k] = r.v[k];
    }
}

// The units (8 dims of a row and the 8 that lie 32 further) of all rows, dealt flat as in
// rope_vec_kernel, one a thread, in the half layout two (with several axes 31 us against 37 with one;
// interleaved, two units of 8 dims instead of one of 16 cost the index arithmetic twice, 33.8 against
// 32.2); a token's rows are its key and the heads of its query.  What bounds it is the issue of the
// index arithmetic and the latency of a block's dependent accesses (position, table row, store) at full
// occupancy, then HBM.
template <bool kInterleaved, bool kVec, bool kAxes>
__device__ __forceinline__ void rope_append_rotated(const RopeAppendArgs& p) {
    using V = Vec<__nv_bfloat16>;
    constexpr int kRows = kAppendRows, kU = 256 / kRows, kSteps = kInterleaved ? 1 : kHalfSteps;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * (kRows * kSteps);
    const int64_t t0 = row0 < (1ll << 32) ? static_cast<int64_t>(any_quotient(static_cast<uint32_t>(row0), p.rows_of_token)) : row0 / p.rows_of_token.d;
    const uint32_t first = static_cast<uint32_t>(row0 - t0 * p.rows_of_token.d);
    const int u = threadIdx.x % kU;
    griddep_wait();
    extern __shared__ __align__(16) float block_rows[];
    uint8_t* turns = reinterpret_cast<uint8_t*>(block_rows + p.block_tokens * NVFP4KV_ROPE);
    if constexpr (kAxes)
        gather_rows(block_rows, turns, p.block_tokens, t0, p.tokens, p.positions, p.pos_i64, p.axes,
                    SmallDiv{NVFP4KV_ROPE / 2, 1u << (32 - 5)}, p.cos_sin, p.max_positions);
    V a[kSteps], b[kSteps];
    int64_t t[kSteps];
    int h[kSteps];          // head, -1 for the key
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        const uint32_t l = first + threadIdx.x / kU + kRows * k, lt = quotient(l, p.rows_of_token);
        t[k] = t0 + lt;
        h[k] = static_cast<int>(l - lt * p.rows_of_token.d) - 1;
        if (t[k] >= p.tokens) continue;
        const __nv_bfloat16* src = h[k] < 0 ? p.k + t[k] * p.k_st : p.q + t[k] * p.q_st + h[k] * p.q_sh;
        a[k] = get8<kVec>(src + 8 * u);
        b[k] = get8<kVec>(src + 32 + 8 * u);
    }
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        if (t[k] >= p.tokens) break;
        const int l = static_cast<int>(t[k] - t0);
        const Angles g = kAxes ? Angles{block_rows + l * NVFP4KV_ROPE, turns[l] != 0}
                               : find_angles(p.positions, p.pos_i64, t[k], p.cos_sin, p.max_positions, NVFP4KV_ROPE);
        __nv_bfloat16* dst;
        if (h[k] < 0) {
            if (!g.turn && u == 0) set_error(p.err, NVFP4KV_DEVERR_BAD_INDEX);
            const int64_t slot = load_index(p.slots, p.slot_i64, t[k]);
            if (slot < 0) continue;
            if (slot >= p.rows) {
                if (u == 0) set_error(p.err, NVFP4KV_DEVERR_BAD_SLOT);
                continue;
            }
            dst = p.pool + slot * NVFP4KV_ROPE;
        } else {
            dst = p.qo + t[k] * p.qo_st + h[k] * p.qo_sh;
        }
        if (g.turn) {
            if (kInterleaved) {
                a[k] = rotate_pairs<__nv_bfloat16, kAxes>(a[k], g.row + 4 * u, 32, 1.0f);
                b[k] = rotate_pairs<__nv_bfloat16, kAxes>(b[k], g.row + 16 + 4 * u, 32, 1.0f);
            } else {
                rotate_halves<__nv_bfloat16, kAxes>(a[k], b[k], g.row + 8 * u, 32, 1.0f);
            }
        }
        put8<kVec>(dst + 32 + 8 * u, b[k]);
        put8<kVec>(dst + 8 * u, a[k]);
    }
}

template <bool kInterleaved, bool kVec>
__global__ void __launch_bounds__(256) rope_append_rotated_kernel(const __grid_constant__ RopeAppendArgs p) {
    rope_append_rotated<kInterleaved, kVec, false>(p);
}
// (more blocks on an SM hide the gathering: 43 us with the angles loaded pair by pair, 36 gathered
// beside the rows' loads with 5 blocks, 31.6 gathered before them with 8, now 27.7; one axis, which reads
// the table's own rows, 25)
template <bool kInterleaved, bool kVec>
__global__ void __launch_bounds__(256, kInterleaved && kVec ? 8 : kVec ? 6 : 4) rope_append_axes_kernel(const __grid_constant__ RopeAppendArgs p) {
    rope_append_rotated<kInterleaved, kVec, true>(p);
}

// The axes of a call (num 0: one, as nvfp4kv_rope).
int check_axes(const char* what, int64_t stride, int num, const uint8_t* pair_axes, int rotary_dim, Axes* out) {
    if (num < 1 || num > NVFP4KV_MAX_AXES) return fail(NVFP4KV_EINVAL, "%s: num_axes %d not in [1, %d]", what, num, NVFP4KV_MAX_AXES);
    if (!pair_axes) return fail(NVFP4KV_EINVAL, "%s: null pointer", what);
    if (rotary_dim > NVFP4KV_MAX_AXES_DIM)
        return fail(NVFP4KV_EINVAL, "%s: rotary_dim %d with several axes (at most %d)", what, rotary_dim, NVFP4KV_MAX_AXES_DIM);
    *out = Axes{};
    out->stride = stride;
    out->num = num;
    for (int i = 0; i < rotary_dim / 2; ++i) {
        if (pair_axes[i] >= num) return fail(NVFP4KV_EINVAL, "%s: pair %d has axis %d of %d", what, i, pair_axes[i], num);
        out->pair_axes[i >> 5] |= static_cast<uint64_t>(pair_axes[i]) << (2 * (i & 31));
    }
    return NVFP4KV_OK;
}

// nvfp4kv_rope (num_axes 0) and nvfp4kv_rope_axes
int rope_call(const char* what, const void* x, int dtype, int64_t num_tokens, int num_heads, int head_dim,
                            int64_t x_stride_t, int64_t x_stride_h, const void* positions, int pos_dtype,
                            int64_t positions_stride, int num_axes, const uint8_t* pair_axes,
                            const float* cos_sin, int64_t max_positions, int rotary_dim, int rope_offset,
                            int interleaved, int inverse, void* out, int64_t out_stride_t, int64_t out_stride_h,
                            int32_t* err_flag, nvfp4kv_stream_t stream) {
    if (num_tokens < 0) return fail(NVFP4KV_EINVAL, "%s: num_tokens < 0", what);
    if (dtype != NVFP4KV_DTYPE_BF16 && dtype != NVFP4KV_DTYPE_F16 && dtype != NVFP4KV_DTYPE_F32)
        return fail(NVFP4KV_EINVAL, "%s: dtype must be bf16, fp16 or fp32", what);
    if (pos_dtype != NVFP4KV_INDEX_I64 && pos_dtype != NVFP4KV_INDEX_I32)
        return fail(NVFP4KV_EINVAL, "%s: position dtype must be int64 or int32", what);
    if (num_heads < 1 || head_dim < 1) return fail(NVFP4KV_EINVAL, "%s: num_heads and head_dim must be >= 1", what);
    if (rotary_dim < 2 || rotary_dim % 2 || rope_offset < 0 || rope_offset > head_dim - rotary_dim)
        return fail(NVFP4KV_EINVAL, "%s: rotary_dim %d at offset %d does not fit head_dim %d (even, >= 2)", what,
                    rotary_dim, rope_offset, head_dim);
    if (max_positions < 1) return fail(NVFP4KV_EINVAL, "%s: empty cos_sin table", what);
    Axes axes{};
    if (num_axes != 0) {
        const int rc = check_axes(what, positions_stride, num_axes, pair_axes, rotary_dim, &axes);
        if (rc != NVFP4KV_OK) return rc;
    }
    if (num_tokens == 0) return NVFP4KV_OK;
    if (!x || !positions || !cos_sin || !out) return fail(NVFP4KV_EINVAL, "%s: null pointer", what);
    const uintptr_t size = dtype == NVFP4KV_DTYPE_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(x) % size || reinterpret_cast<uintptr_t>(out) % size ||
        reinterpret_cast<uintptr_t>(cos_sin) % 4)
        return fail(NVFP4KV_EINVAL, "%s: x, out and cos_sin must be aligned to their elements", what);
    if (x == out && (x_stride_t != out_stride_t || x_stride_h != out_stride_h))
        return fail(NVFP4KV_EINVAL, "%s: in place needs equal strides", what);
    RopeArgs a{};
    a.x = x; a.out = out; a.x_st = x_stride_t; a.x_sh = x_stride_h; a.o_st = out_stride_t; a.o_sh = out_stride_h;
    a.positions = positions; a.cos_sin = cos_sin; a.max_positions = max_positions; a.tokens = num_tokens;
    a.heads = num_heads; a.dim = head_dim; a.rotary = rotary_dim; a.offset = rope_offset;
    a.pos_i64 = pos_dtype == NVFP4KV_INDEX_I64; a.inverse = inverse != 0; a.in_place = x == out; a.err = err_flag;
    a.axes = axes;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const bool il = interleaved != 0;
    if (num_axes == 0) {
        if (dtype == NVFP4KV_DTYPE_BF16) return launch_rope<__nv_bfloat16, false>(a, num_tokens, il, st);
        if (dtype == NVFP4KV_DTYPE_F16) return launch_rope<__half, false>(a, num_tokens, il, st);
        return launch_rope<float, false>(a, num_tokens, il, st);
    }
    if (dtype == NVFP4KV_DTYPE_BF16) return launch_rope<__nv_bfloat16, true>(a, num_tokens, il, st);
    if (dtype == NVFP4KV_DTYPE_F16) return launch_rope<__half, true>(a, num_tokens, il, st);
    return launch_rope<float, true>(a, num_tokens, il, st);
}


// nvfp4kv_append_rope_rotated (num_axes 0) and nvfp4kv_append_rope_rotated_axes
int append_rotated_call(const char* what, const void* k_pe, int64_t num_tokens, int64_t k_stride, void* rope_pool,
                        int64_t pool_rows, const void* slot_mapping, int slot_dtype, const void* positions,
                        int pos_dtype, int64_t positions_stride, int num_axes, const uint8_t* pair_axes,
                        const float* cos_sin, int64_t max_positions, int interleaved, const void* q_pe,
                        int num_heads, int64_t q_stride_t, int64_t q_stride_h, void* q_out, int64_t qo_stride_t,
                        int64_t qo_stride_h, int32_t* err_flag, nvfp4kv_stream_t stream) {
    if (num_tokens < 0) return fail(NVFP4KV_EINVAL, "%s: num_tokens < 0", what);
    if ((slot_dtype != NVFP4KV_INDEX_I64 && slot_dtype != NVFP4KV_INDEX_I32) ||
        (pos_dtype != NVFP4KV_INDEX_I64 && pos_dtype != NVFP4KV_INDEX_I32))
        return fail(NVFP4KV_EINVAL, "%s: slots and positions must be int64 or int32", what);
    Axes axes{};
    if (num_axes != 0) {
        const int rc = check_axes(what, positions_stride, num_axes, pair_axes, NVFP4KV_ROPE, &axes);
        if (rc != NVFP4KV_OK) return rc;
    }
    if (num_tokens == 0) return NVFP4KV_OK;
    if (!k_pe || !rope_pool || !slot_mapping || !positions || !cos_sin || (q_pe && !q_out))
        return fail(NVFP4KV_EINVAL, "%s: null pointer", what);
    if (k_stride < NVFP4KV_ROPE)
        return fail(NVFP4KV_EINVAL, "%s: k_stride %lld < 64", what, (long long)k_stride);
    if (pool_rows <= 0 || max_positions < 1)
        return fail(NVFP4KV_EINVAL, "%s: empty rope pool or cos_sin table", what);
    if (q_pe && (num_heads < 1 || num_heads >= kMostDivisor))
        return fail(NVFP4KV_EINVAL, "%s: num_heads %d not in [1, %d)", what, num_heads, kMostDivisor);
    if (reinterpret_cast<uintptr_t>(rope_pool) % 16 || reinterpret_cast<uintptr_t>(cos_sin) % 16 ||
        (reinterpret_cast<uintptr_t>(k_pe) | reinterpret_cast<uintptr_t>(q_pe) | reinterpret_cast<uintptr_t>(q_out)) % 2)
        return fail(NVFP4KV_EINVAL, "%s: rope pool and cos_sin must be 16-byte aligned", what);
    if (q_pe && q_pe == q_out && (q_stride_t != qo_stride_t || q_stride_h != qo_stride_h))
        return fail(NVFP4KV_EINVAL, "%s: in place needs equal strides", what);
    RopeAppendArgs a{};
    a.k = static_cast<const __nv_bfloat16*>(k_pe); a.k_st = k_stride; a.tokens = num_tokens;
    a.pool = static_cast<__nv_bfloat16*>(rope_pool); a.rows = pool_rows;
    a.slots = slot_mapping; a.slot_i64 = slot_dtype == NVFP4KV_INDEX_I64;
    a.positions = positions; a.pos_i64 = pos_dtype == NVFP4KV_INDEX_I64;
    a.cos_sin = cos_sin; a.max_positions = max_positions; a.err = err_flag; a.axes = axes;
    a.q = static_cast<const __nv_bfloat16*>(q_pe); a.qo = static_cast<__nv_bfloat16*>(q_out);
    a.heads = q_pe ? num_heads : 0;
    a.q_st = q_stride_t; a.q_sh = q_stride_h; a.qo_st = qo_stride_t; a.qo_sh = qo_stride_h;
    const bool vec = reinterpret_cast<uintptr_t>(k_pe) % 16 == 0 && k_stride % 8 == 0 &&
                     (!q_pe || ((reinterpret_cast<uintptr_t>(q_pe) | reinterpret_cast<uintptr_t>(q_out)) % 16 == 0 &&
                                (q_stride_t | q_stride_h | qo_stride_t | qo_stride_h) % 8 == 0));
    const uint32_t per_token = a.heads + 1;
    a.rows_of_token = small_div(per_token);
    const int64_t per_block = kAppendRows * (interleaved ? 1 : kHalfSteps), blocks = (num_tokens * per_token + per_block - 1) / per_block;
    if (blocks > 0x7FFFFFFF) return fail(NVFP4KV_EINVAL, "%s: too many rows for one call", what);
    const dim3 grid(static_cast<unsigned>(blocks));
    size_t smem = 0;
    if (num_axes != 0) {
        const int64_t most = (per_block + per_token - 2) / per_token + 1;
        a.block_tokens = static_cast<int>(most < num_tokens ? most : num_tokens);
        smem = a.block_tokens * (NVFP4KV_ROPE * sizeof(float) + 1);      // (up to 129 tokens)
    }
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    constexpr void (*kKernels[2][2][2])(RopeAppendArgs) = {
        {{rope_append_rotated_kernel<false, false>, rope_append_axes_kernel<false, false>},
         {rope_append_rotated_kernel<false, true>, rope_append_axes_kernel<false, true>}},
        {{rope_append_rotated_kernel<true, false>, rope_append_axes_kernel<true, false>},
         {rope_append_rotated_kernel<true, true>, rope_append_axes_kernel<true, true>}}};
    void (*kernel)(RopeAppendArgs) = kKernels[interleaved != 0][vec][num_axes != 0];
    const cudaError_t e = launch_dependent(kernel, grid, dim3(256), smem, st, a);
    if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
    return check_launch(what);
}

}  // namespace
}  // namespace nvfp4kv

extern "C" int nvfp4kv_rope(const void* x, int dtype, int64_t num_tokens, int num_heads, int head_dim,
                            int64_t x_stride_t, int64_t x_stride_h, const void* positions, int pos_dtype,
                            const float* cos_sin, int64_t max_positions, int rotary_dim, int rope_offset,
                            int interleaved, int inverse, void* out, int64_t out_stride_t, int64_t out_stride_h,
                            int32_t* err_flag, nvfp4kv_stream_t stream) {
    return nvfp4kv::rope_call("nvfp4kv_rope", x, dtype, num_tokens, num_heads, head_dim, x_stride_t, x_stride_h, positions,
                              pos_dtype, 0, 0, nullptr, cos_sin, max_positions, rotary_dim, rope_offset, interleaved, inverse,
                              out, out_stride_t, out_stride_h, err_flag, stream);
}

extern "C" int nvfp4kv_rope_axes(const void* x, int dtype, int64_t num_tokens, int num_heads, int head_dim,
                                 int64_t x_stride_t, int64_t x_stride_h, const void* positions, int pos_dtype,
                                 int64_t positions_stride, int num_axes, const uint8_t* pair_axes,
                                 const float* cos_sin, int64_t max_positions, int rotary_dim, int rope_offset,
                                 int interleaved, int inverse, void* out, int64_t out_stride_t, int64_t out_stride_h,
                                 int32_t* err_flag, nvfp4kv_stream_t stream) {
    // (0 axes are refused here, where nvfp4kv_rope means one)
    return nvfp4kv::rope_call("nvfp4kv_rope_axes", x, dtype, num_tokens, num_heads, head_dim, x_stride_t, x_stride_h, positions,
                              pos_dtype, positions_stride, num_axes == 0 ? -1 : num_axes, pair_axes, cos_sin, max_positions,
                              rotary_dim, rope_offset, interleaved, inverse, out, out_stride_t, out_stride_h, err_flag, stream);
}

extern "C" int nvfp4kv_append_rope_rotated(const void* k_pe, int64_t num_tokens, int64_t k_stride, void* rope_pool,
                                           int64_t pool_rows, const void* slot_mapping, int slot_dtype,
                                           const void* positions, int pos_dtype, const float* cos_sin,
                                           int64_t max_positions, int interleaved, const void* q_pe, int num_heads,
                                           int64_t q_stride_t, int64_t q_stride_h, void* q_out, int64_t qo_stride_t,
                                           int64_t qo_stride_h, int32_t* err_flag, nvfp4kv_stream_t stream) {
    return nvfp4kv::append_rotated_call("nvfp4kv_append_rope_rotated", k_pe, num_tokens, k_stride, rope_pool, pool_rows,
                                        slot_mapping, slot_dtype, positions, pos_dtype, 0, 0, nullptr, cos_sin, max_positions,
                                        interleaved, q_pe, num_heads, q_stride_t, q_stride_h, q_out, qo_stride_t, qo_stride_h,
                                        err_flag, stream);
}

extern "C" int nvfp4kv_append_rope_rotated_axes(const void* k_pe, int64_t num_tokens, int64_t k_stride, void* rope_pool,
                                                int64_t pool_rows, const void* slot_mapping, int slot_dtype,
                                                const void* positions, int pos_dtype, int64_t positions_stride,
                                                int num_axes, const uint8_t* pair_axes, const float* cos_sin,
                                                int64_t max_positions, int interleaved, const void* q_pe, int num_heads,
                                                int64_t q_stride_t, int64_t q_stride_h, void* q_out, int64_t qo_stride_t,
                                                int64_t qo_stride_h, int32_t* err_flag, nvfp4kv_stream_t stream) {
    return nvfp4kv::append_rotated_call("nvfp4kv_append_rope_rotated_axes", k_pe, num_tokens, k_stride, rope_pool, pool_rows,
                                        slot_mapping, slot_dtype, positions, pos_dtype, positions_stride,
                                        num_axes == 0 ? -1 : num_axes, pair_axes, cos_sin, max_positions, interleaved, q_pe,
                                        num_heads, q_stride_t, q_stride_h, q_out, qo_stride_t, qo_stride_h, err_flag, stream);
}
