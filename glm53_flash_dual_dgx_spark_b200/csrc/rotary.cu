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

struct RopeArgs {
    const void* x;
    void* out;
    int64_t x_st, x_sh, o_st, o_sh;
    const void* positions;
    const float* cos_sin;
    int64_t max_positions;
    int heads, dim, rotary, offset;
    int heads_per_block, head_blocks;
    int pos_i64, inverse, in_place;
    int32_t* err;
};

// One block: heads_per_block heads of one token, a 16-byte vector per thread and step.  In half
// layout the thread of a lower-half vector does its partner too.
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(256) rope_vec_kernel(const RopeArgs p) {
    constexpr int N = Vec<T>::kN;
    const int64_t t = blockIdx.x / p.head_blocks;
    const int h0 = static_cast<int>(blockIdx.x % p.head_blocks) * p.heads_per_block;
    const int heads = min(p.heads_per_block, p.heads - h0);
    const int64_t pos = load_index(p.positions, p.pos_i64, t);
    const bool turn = pos >= 0 && pos < p.max_positions;
    if (!turn && threadIdx.x == 0) set_error(p.err, NVFP4KV_DEVERR_BAD_INDEX);
    const float* cs = p.cos_sin + (turn ? pos : 0) * p.rotary;
    const int half = p.rotary / 2;
    const float sign = p.inverse ? -1.0f : 1.0f;
    // in place only the rotated dims are visited
    const int d0 = p.in_place ? p.offset : 0;
    const int per = (p.in_place ? p.rotary : p.dim) / N;
    const T* x = static_cast<const T*>(p.x) + t * p.x_st + h0 * p.x_sh + d0;
    T* o = static_cast<T*>(p.out) + t * p.o_st + h0 * p.o_sh + d0;
    for (int u = threadIdx.x; u < heads * per; u += blockDim.x) {
        const int h = u / per, d = (u - h * per) * N;
        const T* xp = x + h * p.x_sh + d;
        T* op = o + h * p.o_sh + d;
        const int r = d0 + d - p.offset;          // dim within the rotated part
        if (r < 0 || r >= p.rotary || !turn) {
            store_vec(op, load_vec(xp));
        } else if (kInterleaved) {
            store_vec(op, rotate_pairs(load_vec(xp), cs + r / 2, half, sign));
        } else if (r < half) {
            Vec<T> a = load_vec(xp), b = load_vec(xp + half);
            rotate_halves(a, b, cs + r, half, sign);
            store_vec(op, a);
            store_vec(op + half, b);
        }
    }
}

// Any strides, alignment and sizes: one element (a rotated dim: its pair) per thread and step.
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(256) rope_elem_kernel(const RopeArgs p) {
    const int64_t t = blockIdx.x / p.head_blocks;
    const int h0 = static_cast<int>(blockIdx.x % p.head_blocks) * p.heads_per_block;
    const int heads = min(p.heads_per_block, p.heads - h0);
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
                     a.rotary % (interleaved ? N : 2 * N) == 0;
    const int per_head = vec ? (a.in_place ? a.rotary : a.dim) / N : a.dim;
    // about four steps a thread: enough loads in flight, and blocks for every SM from a few tokens on
    int hb = 1024 / per_head;
    hb = hb < 1 ? 1 : (hb > a.heads ? a.heads : hb);
    a.head_blocks = (a.heads + hb - 1) / hb;
    a.heads_per_block = (a.heads + a.head_blocks - 1) / a.head_blocks;
    const int64_t blocks = tokens * a.head_blocks;
    if (blocks > 0x7FFFFFFF) return fail(NVFP4KV_EINVAL, "nvfp4kv_rope: too many rows for one call");
    const dim3 grid(static_cast<unsigned>(blocks));
    if (vec) {
        if (interleaved) rope_vec_kernel<T, true><<<grid, 256, 0, st>>>(a);
        else rope_vec_kernel<T, false><<<grid, 256, 0, st>>>(a);
    } else {
        if (interleaved) rope_elem_kernel<T, true><<<grid, 256, 0, st>>>(a);
        else rope_elem_kernel<T, false><<<grid, 256, 0, st>>>(a);
    }
    return check_launch("nvfp4kv_rope");
}

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
    int slot_i64, pos_i64;
    int32_t* err;
};

// 64 dims of a row from `x` to `o`, the part of them that belongs to unit `u` of 8 (interleaved:
// dims 8u..) or 4 (half layout: dims 8u.. and 32 + 8u..).
template <bool kInterleaved, bool kVec>
__device__ __forceinline__ void rotate_unit(const __nv_bfloat16* x, __nv_bfloat16* o, const float* cs, bool turn, int u) {
    using V = Vec<__nv_bfloat16>;
    auto get = [](const __nv_bfloat16* p) {
        if constexpr (kVec) {
            return load_vec(p);
        } else {
            V r;
#pragma unroll
            for (int k = 0; k < 8; ++k) r.v[k] = p[k];
            return r;
        }
    };
    auto put = [](__nv_bfloat16* p, const V& r) {
        if constexpr (kVec) {
            store_vec(p, r);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) p[k] = r.v[k];
        }
    };
    if constexpr (kInterleaved) {
        V a = get(x + 8 * u);
        if (turn) a = rotate_pairs(a, cs + 4 * u, 32, 1.0f);
        put(o + 8 * u, a);
    } else {
        V a = get(x + 8 * u), b = get(x + 32 + 8 * u);
        if (turn) rotate_halves(a, b, cs + 8 * u, 32, 1.0f);
        put(o + 8 * u, a);
        put(o + 32 + 8 * u, b);
    }
}

// Thread = unit of one row: the token's key (row 0) or a head of its query (rows 1..heads).
template <bool kInterleaved, bool kVec>
__global__ void __launch_bounds__(256) rope_append_rotated_kernel(const RopeAppendArgs p) {
    constexpr int kU = kInterleaved ? 8 : 4;
    const int64_t g = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    const int u = static_cast<int>(g % kU);
    const int64_t row = g / kU;
    const int64_t t = row / (p.heads + 1);
    const int h = static_cast<int>(row - t * (p.heads + 1)) - 1;
    if (t >= p.tokens) return;
    const int64_t pos = load_index(p.positions, p.pos_i64, t);
    const bool turn = pos >= 0 && pos < p.max_positions;
    const float* cs = p.cos_sin + (turn ? pos : 0) * NVFP4KV_ROPE;
    if (h >= 0) {
        rotate_unit<kInterleaved, kVec>(p.q + t * p.q_st + h * p.q_sh, p.qo + t * p.qo_st + h * p.qo_sh, cs, turn, u);
        return;
    }
    if (!turn && u == 0) set_error(p.err, NVFP4KV_DEVERR_BAD_INDEX);
    const int64_t slot = load_index(p.slots, p.slot_i64, t);
    if (slot < 0) return;
    if (slot >= p.rows) {
        if (u == 0) set_error(p.err, NVFP4KV_DEVERR_BAD_SLOT);
        return;
    }
    rotate_unit<kInterleaved, kVec>(p.k + t * p.k_st, p.pool + slot * NVFP4KV_ROPE, cs, turn, u);
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
    if (q_pe && num_heads < 1) return fail(NVFP4KV_EINVAL, "nvfp4kv_append_rope_rotated: num_heads must be >= 1");
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
    const int64_t threads = num_tokens * (a.heads + 1) * (interleaved ? 8 : 4);
    const int64_t blocks = (threads + 255) / 256;
    if (blocks > 0x7FFFFFFF) return fail(NVFP4KV_EINVAL, "nvfp4kv_append_rope_rotated: too many rows for one call");
    const dim3 grid(static_cast<unsigned>(blocks));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (interleaved) {
        if (vec) rope_append_rotated_kernel<true, true><<<grid, 256, 0, st>>>(a);
        else rope_append_rotated_kernel<true, false><<<grid, 256, 0, st>>>(a);
    } else {
        if (vec) rope_append_rotated_kernel<false, true><<<grid, 256, 0, st>>>(a);
        else rope_append_rotated_kernel<false, false><<<grid, 256, 0, st>>>(a);
    }
    return check_launch("nvfp4kv_append_rope_rotated");
}
