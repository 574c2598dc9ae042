// Rotary positions: nvfp4kv_rope (whole heads, any layout) and nvfp4kv_append_rope_rotated (the
// rope part of a step: rotated keys into the paged side-pool, queries rotated beside them).
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
template <typename T> __device__ __forceinline__ Vec<T> load_vec(const T* p) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    Vec<T> r;
    memcpy(&r, &u, 16);
    return r;
}
template <typename T> __device__ __forceinline__ void store_vec(T* p, const Vec<T>& r) {
    uint4 u;
    memcpy(&u, &r, 16);
    *reinterpret_cast<uint4*>(p) = u;
}

__device__ __forceinline__ int64_t load_index(const void* p, bool i64, int64_t i) {
    return i64 ? static_cast<int64_t>(__ldg(static_cast<const long long*>(p) + i))
               : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(p) + i));
}

__device__ __forceinline__ void rotate(float a, float b, float c, float s, float& u, float& v) {
    u = a * c - b * s;
    v = b * c + a * s;
}

// N consecutive cos (or sin) values, N a multiple of 4 or 2, 8-byte aligned.
template <int N> __device__ __forceinline__ void load_angles(const float* p, float (&r)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int k = 0; k < N / 4; ++k) {
            const float4 f = __ldg(reinterpret_cast<const float4*>(p) + k);
            r[4 * k] = f.x; r[4 * k + 1] = f.y; r[4 * k + 2] = f.z; r[4 * k + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int k = 0; k < N / 2; ++k) {
            const float2 f = __ldg(reinterpret_cast<const float2*>(p) + k);
            r[2 * k] = f.x; r[2 * k + 1] = f.y;
        }
    }
}

// One 16-byte vector of an interleaved rotation: pairs inside the vector.  cs -> cos of its first pair.
template <typename T>
__device__ __forceinline__ Vec<T> rotate_pairs(const Vec<T>& x, const float* cs, int half, float sign) {
    constexpr int N = Vec<T>::kN;
    float c[N / 2], s[N / 2];
    load_angles<N / 2>(cs, c);
    load_angles<N / 2>(cs + half, s);
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
template <typename T>
__device__ __forceinline__ void rotate_halves(Vec<T>& xa, Vec<T>& xb, const float* cs, int half, float sign) {
    constexpr int N = Vec<T>::kN;
    float c[N], s[N];
    load_angles<N>(cs, c);
    load_angles<N>(cs + half, s);
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
};
constexpr int kRopeSteps = 2;

// A unit is a 16-byte vector of a head (a rotated one of the half layout: the pair of vectors that
// turn together).  The units of the call are dealt flat, two to a thread and 256 apart: every warp
// moves 512 contiguous bytes, every block is full, and two loads in flight per thread are enough at
// the occupancy that leaves (8,192 tokens x 64 heads x 576 bf16, 1.2 GB: 188 us = 6.4 TB/s, as much
// as a plain copy; 8 % more with one, 1 % more with four, 20 % more with blocks of whole heads, whose
// last steps are part empty).  The gradient of 2,049 tokens x 32 heads x 128 fp32 takes 12 us.
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(256, kInterleaved && sizeof(T) == 2 ? 8 : 4) rope_vec_kernel(const __grid_constant__ RopeArgs p) {
    constexpr int N = Vec<T>::kN;
    const int64_t u0 = static_cast<int64_t>(blockIdx.x) * (256 * kRopeSteps);
    int64_t row0, t0;       // the block's first head row, its token
    if (p.total < (1ll << 32)) {
        row0 = static_cast<uint32_t>(u0) / p.units.d;
        t0 = static_cast<uint32_t>(row0) / p.by_heads.d;
    } else {
        row0 = u0 / p.units.d;
        t0 = row0 / p.by_heads.d;
    }
    const uint32_t j0 = static_cast<uint32_t>(u0 - row0 * p.units.d), h0 = static_cast<uint32_t>(row0 - t0 * p.by_heads.d);
    const int half = p.rotary / 2;
    griddep_wait();
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
            a[k] = load_vec(xp);
            if (!kInterleaved && r[k] >= 0) b[k] = load_vec(xp + half);
        } else {
            r[k] = -2;
        }
    }
#pragma unroll
    for (int k = 0; k < kRopeSteps; ++k) {
        if (r[k] == -2) break;
        T* op = static_cast<T*>(p.out) + at[k];
        if (r[k] >= 0) {
            const int64_t pos = load_index(p.positions, p.pos_i64, t[k]);
            const bool turn = pos >= 0 && pos < p.max_positions;
            if (!turn) set_error(p.err, NVFP4KV_DEVERR_BAD_INDEX);
            const float* cs = p.cos_sin + (turn ? pos : 0) * p.rotary + (kInterleaved ? r[k] / 2 : r[k]);
            const float sign = p.inverse ? -1.0f : 1.0f;
            if (kInterleaved) {
                if (turn) a[k] = rotate_pairs(a[k], cs, half, sign);
            } else {
                if (turn) rotate_halves(a[k], b[k], cs, half, sign);
                store_vec(op + half, b[k]);
            }
        }
        store_vec(op, a[k]);
    }
}

// Any strides, alignment and sizes: one element (a rotated dim: its pair) per thread and step, for rows
// that no 16-byte access can take (views at an odd offset, heads of odd sizes).  It is bound by its
// 2- or 4-byte accesses and a division per element: 8,192 tokens x 64 heads x 192 bf16, shifted by 3,
// take 388 us where the bytes take 62 (1.0 TB/s; fp32 2.1).  A caller that can align its rows should.
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(256) rope_elem_kernel(const __grid_constant__ RopeArgs p, int head_blocks, int heads_per_block) {
    const int64_t t = blockIdx.x / head_blocks;
    const int h0 = static_cast<int>(blockIdx.x % head_blocks) * heads_per_block;
    const int heads = min(heads_per_block, p.heads - h0);
    const int64_t pos = load_index(p.positions, p.pos_i64, t);
    const bool turn = pos >= 0 && pos < p.max_positions;
    if (!turn && threadIdx.x == 0) set_error(p.err, NVFP4KV_DEVERR_BAD_INDEX);
    const float* cs = p.cos_sin + (turn ? pos : 0) * p.rotary;
    const int half = p.rotary / 2;
    const float sign = p.inverse ? -1.0f : 1.0f;
    const T* x = static_cast<const T*>(p.x) + t * p.x_st + h0 * p.x_sh;
    T* o = static_cast<T*>(p.out) + t * p.o_st + h0 * p.o_sh;
    for (int u = threadIdx.x; u < heads * p.dim; u += blockDim.x) {
        const int h = u / p.dim, d = u - h * p.dim;
        const T* xp = x + h * p.x_sh;
        T* op = o + h * p.o_sh;
        const int r = d - p.offset;
        if (r < 0 || r >= p.rotary || !turn) {
            op[d] = xp[d];
            continue;
        }
        const int i = kInterleaved ? r / 2 : r;
        if (kInterleaved ? (r & 1) : r >= half) continue;      // done with its partner
        const int db = kInterleaved ? d + 1 : d + half;
        float u0, v0;
        rotate(load_f32(xp + d), load_f32(xp + db), __ldg(cs + i), sign * __ldg(cs + half + i), u0, v0);
        op[d] = from_f32<T>(u0);
        op[db] = from_f32<T>(v0);
    }
}

template <typename T>
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
        a.units = {units, static_cast<uint32_t>(((1ull << 32) + units - 1) / units)};
        a.by_heads = {heads, static_cast<uint32_t>(((1ull << 32) + heads - 1) / heads)};
        a.total = tokens * heads * units;
        blocks = (a.total + 256 * kRopeSteps - 1) / (256 * kRopeSteps);
        if (blocks > 0x7FFFFFFF) return fail(NVFP4KV_EINVAL, "nvfp4kv_rope: too many rows for one call");
        const cudaError_t e = launch_dependent(interleaved ? rope_vec_kernel<T, true> : rope_vec_kernel<T, false>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, a);
        if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "nvfp4kv_rope launch failed: %s", cudaGetErrorString(e));
    } else {
        int hb = 1024 / a.dim;
        hb = hb < 1 ? 1 : (hb > a.heads ? a.heads : hb);
        const int head_blocks = (a.heads + hb - 1) / hb, per_block = (a.heads + head_blocks - 1) / head_blocks;
        blocks = tokens * head_blocks;
        if (blocks > 0x7FFFFFFF) return fail(NVFP4KV_EINVAL, "nvfp4kv_rope: too many rows for one call");
        if (interleaved) rope_elem_kernel<T, true><<<static_cast<unsigned>(blocks), 256, 0, st>>>(a, head_blocks, per_block);
        else rope_elem_kernel<T, false><<<static_cast<unsigned>(blocks), 256, 0, st>>>(a, head_blocks, per_block);
    }
    return check_launch("nvfp4kv_rope");
}

constexpr int kAppendSteps = 2;

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
};

// 8 bf16, as one 16-byte access or element by element.  The accesses are marked as streaming: a step's
// rows pass once, while the table rows of its positions come back with every layer, and should stay
// in L2 (32,768 tokens x 16 heads over a table of 77 MB: 28.0 us against 33.3 without the marks, and
// 29.8 with the next blocks' table rows prefetched instead).
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

// The units (8 dims of a row, half layout: 8 and their partners) of all rows, dealt flat as in
// rope_vec_kernel, two a thread (37.7 us with one, 42 with four, before the streaming marks); a
// token's rows are its key and the heads of its query.  What bounds it is the latency of a block's
// three dependent accesses (position, table row, store) at full occupancy, then HBM.
template <bool kInterleaved, bool kVec>
__global__ void __launch_bounds__(256) rope_append_rotated_kernel(const __grid_constant__ RopeAppendArgs p) {
    using V = Vec<__nv_bfloat16>;
    constexpr int kU = kInterleaved ? 8 : 4, kSteps = kAppendSteps, kRows = 256 / kU;      // rows of a block and step
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * (kRows * kSteps);
    const int64_t t0 = row0 < (1ll << 32) ? static_cast<int64_t>(static_cast<uint32_t>(row0) / p.rows_of_token.d) : row0 / p.rows_of_token.d;
    const uint32_t first = static_cast<uint32_t>(row0 - t0 * p.rows_of_token.d);
    const int u = threadIdx.x % kU;
    griddep_wait();
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
        if (!kInterleaved) b[k] = get8<kVec>(src + 32 + 8 * u);
    }
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        if (t[k] >= p.tokens) break;
        const int64_t pos = load_index(p.positions, p.pos_i64, t[k]);
        const bool turn = pos >= 0 && pos < p.max_positions;
        const float* cs = p.cos_sin + (turn ? pos : 0) * NVFP4KV_ROPE;
        __nv_bfloat16* dst;
        if (h[k] < 0) {
            if (!turn && u == 0) set_error(p.err, NVFP4KV_DEVERR_BAD_INDEX);
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
        if (kInterleaved) {
            if (turn) a[k] = rotate_pairs(a[k], cs + 4 * u, 32, 1.0f);
        } else {
            if (turn) rotate_halves(a[k], b[k], cs + 8 * u, 32, 1.0f);
            put8<kVec>(dst + 32 + 8 * u, b[k]);
        }
        put8<kVec>(dst + 8 * u, a[k]);
    }
}

}  // namespace
}  // namespace nvfp4kv

extern "C" int nvfp4kv_rope(const void* x, int dtype, int64_t num_tokens, int num_heads, int head_dim,
                            int64_t x_stride_t, int64_t x_stride_h, const void* positions, int pos_dtype,
                            const float* cos_sin, int64_t max_positions, int rotary_dim, int rope_offset,
                            int interleaved, int inverse, void* out, int64_t out_stride_t, int64_t out_stride_h,
                            int32_t* err_flag, nvfp4kv_stream_t stream) {
    using namespace nvfp4kv;
    if (num_tokens < 0) return fail(NVFP4KV_EINVAL, "nvfp4kv_rope: num_tokens < 0");
    if (dtype != NVFP4KV_DTYPE_BF16 && dtype != NVFP4KV_DTYPE_F16 && dtype != NVFP4KV_DTYPE_F32)
        return fail(NVFP4KV_EINVAL, "nvfp4kv_rope: dtype must be bf16, fp16 or fp32");
    if (pos_dtype != NVFP4KV_INDEX_I64 && pos_dtype != NVFP4KV_INDEX_I32)
        return fail(NVFP4KV_EINVAL, "nvfp4kv_rope: position dtype must be int64 or int32");
    if (num_heads < 1 || head_dim < 1) return fail(NVFP4KV_EINVAL, "nvfp4kv_rope: num_heads and head_dim must be >= 1");
    if (rotary_dim < 2 || rotary_dim % 2 || rope_offset < 0 || rope_offset > head_dim - rotary_dim)
        return fail(NVFP4KV_EINVAL, "nvfp4kv_rope: rotary_dim %d at offset %d does not fit head_dim %d (even, >= 2)",
                    rotary_dim, rope_offset, head_dim);
    if (max_positions < 1) return fail(NVFP4KV_EINVAL, "nvfp4kv_rope: empty cos_sin table");
    if (num_tokens == 0) return NVFP4KV_OK;
    if (!x || !positions || !cos_sin || !out) return fail(NVFP4KV_EINVAL, "nvfp4kv_rope: null pointer");
    const uintptr_t size = dtype == NVFP4KV_DTYPE_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(x) % size || reinterpret_cast<uintptr_t>(out) % size ||
        reinterpret_cast<uintptr_t>(cos_sin) % 4)
        return fail(NVFP4KV_EINVAL, "nvfp4kv_rope: x, out and cos_sin must be aligned to their elements");
    if (x == out && (x_stride_t != out_stride_t || x_stride_h != out_stride_h))
        return fail(NVFP4KV_EINVAL, "nvfp4kv_rope: in place needs equal strides");
    RopeArgs a{};
    a.x = x; a.out = out; a.x_st = x_stride_t; a.x_sh = x_stride_h; a.o_st = out_stride_t; a.o_sh = out_stride_h;
    a.positions = positions; a.cos_sin = cos_sin; a.max_positions = max_positions;
    a.heads = num_heads; a.dim = head_dim; a.rotary = rotary_dim; a.offset = rope_offset;
    a.pos_i64 = pos_dtype == NVFP4KV_INDEX_I64; a.inverse = inverse != 0; a.in_place = x == out; a.err = err_flag;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == NVFP4KV_DTYPE_BF16) return launch_rope<__nv_bfloat16>(a, num_tokens, interleaved != 0, st);
    if (dtype == NVFP4KV_DTYPE_F16) return launch_rope<__half>(a, num_tokens, interleaved != 0, st);
    return launch_rope<float>(a, num_tokens, interleaved != 0, st);
}

extern "C" int nvfp4kv_append_rope_rotated(const void* k_pe, int64_t num_tokens, int64_t k_stride, void* rope_pool,
                                           int64_t pool_rows, const void* slot_mapping, int slot_dtype,
                                           const void* positions, int pos_dtype, const float* cos_sin,
                                           int64_t max_positions, int interleaved, const void* q_pe, int num_heads,
                                           int64_t q_stride_t, int64_t q_stride_h, void* q_out, int64_t qo_stride_t,
                                           int64_t qo_stride_h, int32_t* err_flag, nvfp4kv_stream_t stream) {
    using namespace nvfp4kv;
    if (num_tokens < 0) return fail(NVFP4KV_EINVAL, "nvfp4kv_append_rope_rotated: num_tokens < 0");
    if ((slot_dtype != NVFP4KV_INDEX_I64 && slot_dtype != NVFP4KV_INDEX_I32) ||
        (pos_dtype != NVFP4KV_INDEX_I64 && pos_dtype != NVFP4KV_INDEX_I32))
        return fail(NVFP4KV_EINVAL, "nvfp4kv_append_rope_rotated: slots and positions must be int64 or int32");
    if (num_tokens == 0) return NVFP4KV_OK;
    if (!k_pe || !rope_pool || !slot_mapping || !positions || !cos_sin || (q_pe && !q_out))
        return fail(NVFP4KV_EINVAL, "nvfp4kv_append_rope_rotated: null pointer");
    if (k_stride < NVFP4KV_ROPE)
        return fail(NVFP4KV_EINVAL, "nvfp4kv_append_rope_rotated: k_stride %lld < 64", (long long)k_stride);
    if (pool_rows <= 0 || max_positions < 1)
        return fail(NVFP4KV_EINVAL, "nvfp4kv_append_rope_rotated: empty rope pool or cos_sin table");
    if (q_pe && (num_heads < 1 || num_heads >= kMostDivisor))
        return fail(NVFP4KV_EINVAL, "nvfp4kv_append_rope_rotated: num_heads %d not in [1, %d)", num_heads, kMostDivisor);
    if (reinterpret_cast<uintptr_t>(rope_pool) % 16 || reinterpret_cast<uintptr_t>(cos_sin) % 16 ||
        (reinterpret_cast<uintptr_t>(k_pe) | reinterpret_cast<uintptr_t>(q_pe) | reinterpret_cast<uintptr_t>(q_out)) % 2)
        return fail(NVFP4KV_EINVAL, "nvfp4kv_append_rope_rotated: rope pool and cos_sin must be 16-byte aligned");
    if (q_pe && q_pe == q_out && (q_stride_t != qo_stride_t || q_stride_h != qo_stride_h))
        return fail(NVFP4KV_EINVAL, "nvfp4kv_append_rope_rotated: in place needs equal strides");
    RopeAppendArgs a{};
    a.k = static_cast<const __nv_bfloat16*>(k_pe); a.k_st = k_stride; a.tokens = num_tokens;
    a.pool = static_cast<__nv_bfloat16*>(rope_pool); a.rows = pool_rows;
    a.slots = slot_mapping; a.slot_i64 = slot_dtype == NVFP4KV_INDEX_I64;
    a.positions = positions; a.pos_i64 = pos_dtype == NVFP4KV_INDEX_I64;
    a.cos_sin = cos_sin; a.max_positions = max_positions; a.err = err_flag;
    a.q = static_cast<const __nv_bfloat16*>(q_pe); a.qo = static_cast<__nv_bfloat16*>(q_out);
    a.heads = q_pe ? num_heads : 0;
    a.q_st = q_stride_t; a.q_sh = q_stride_h; a.qo_st = qo_stride_t; a.qo_sh = qo_stride_h;
    const bool vec = reinterpret_cast<uintptr_t>(k_pe) % 16 == 0 && k_stride % 8 == 0 &&
                     (!q_pe || ((reinterpret_cast<uintptr_t>(q_pe) | reinterpret_cast<uintptr_t>(q_out)) % 16 == 0 &&
                                (q_stride_t | q_stride_h | qo_stride_t | qo_stride_h) % 8 == 0));
    const uint32_t per_token = a.heads + 1;
    a.rows_of_token = {per_token, static_cast<uint32_t>(((1ull << 32) + per_token - 1) / per_token)};
    const int64_t per_block = kAppendSteps * 256 / (interleaved ? 8 : 4), blocks = (num_tokens * per_token + per_block - 1) / per_block;
    if (blocks > 0x7FFFFFFF) return fail(NVFP4KV_EINVAL, "nvfp4kv_append_rope_rotated: too many rows for one call");
    const dim3 grid(static_cast<unsigned>(blocks));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    void (*kernel)(RopeAppendArgs) = interleaved ? (vec ? rope_append_rotated_kernel<true, true> : rope_append_rotated_kernel<true, false>)
                                                 : (vec ? rope_append_rotated_kernel<false, true> : rope_append_rotated_kernel<false, false>);
    const cudaError_t e = launch_dependent(kernel, grid, dim3(256), 0, st, a);
    if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "nvfp4kv_append_rope_rotated launch failed: %s", cudaGetErrorString(e));
    return check_launch("nvfp4kv_append_rope_rotated");
}
