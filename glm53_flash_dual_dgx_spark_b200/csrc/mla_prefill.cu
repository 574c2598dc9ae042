// Causal MLA attention of a ragged batch of new tokens over the NVFP4 paged pool.
//
//   x[r, t] = bmm1_scale (q[r, :512] . k[t] + q[r, 512:] . k_rope[t]),  t <= L - n + i(r)
//   out[r] = bmm2_scale sum_t softmax(x[r])_t k[t],   lse[r] = log sum_t exp(x[r, t])
//
// Rows r = (new token i, head) of one sequence share the latent rows k, which are both keys and
// values.
#include <math.h>

#include "../../include/nvfp4kv_serving.h"
#include "abi_common.h"
#include "common.cuh"

namespace nvfp4kv {
namespace {

constexpr int kRope = NVFP4KV_ROPE;
constexpr int kDim = kLatent + kRope;
constexpr int kRows = 16;      // query rows per block
constexpr int kTok = 32;       // tokens per tile
constexpr int kLd = kDim + 1;  // key tile row in shared memory (no bank conflicts over tokens)

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
    float scale_log2, out_scale;
    __nv_bfloat16* out;
    int64_t o_st, o_sh;
    float* lse;
    int32_t* err;
};

// Sequence b's new tokens: their first index in q and their number, clamped to what the call says.
__device__ __forceinline__ void query_span(const PrefillParams& p, int b, int* first, int* n) {
    const int lo = max(0, min(p.cu[b], p.total_q)), hi = max(lo, min(p.cu[b + 1], p.total_q));
    *first = lo;
    *n = min(hi - lo, p.max_q_len);
    if (hi - lo > p.max_q_len) set_error(p.err, NVFP4KV_DEVERR_SEQ_LEN);
}

// Block of kRows rows: fp32 arithmetic on the CUDA cores, one running maximum per row.
__global__ void __launch_bounds__(256) mla_prefill_kernel(const PrefillParams p) {
    extern __shared__ float sm[];
    float* qs = sm;                        // [kRows][kDim]
    float* ks = qs + kRows * kDim;         // [kTok][kLd]
    float* ps = ks + kTok * kLd;           // [kRows][kTok]
    float* al = ps + kRows * kTok;         // [kRows] factor of the accumulators
    const int tid = threadIdx.x;
    int item = blockIdx.x, b = 0, first = 0, n = 0;
    for (; b < p.batch; ++b) {
        query_span(p, b, &first, &n);
        const int blocks = static_cast<int>((static_cast<int64_t>(n) * p.heads + kRows - 1) / kRows);
        if (item < blocks) break;
        item -= blocks;
    }
    if (b == p.batch) return;
    int L = p.seq_lens[b];
    if (L > p.max_seq_len) {
        if (tid == 0) set_error(p.err, NVFP4KV_DEVERR_SEQ_LEN);
        L = p.max_seq_len;
    }
    L = max(L, 0);
    const int r0 = item * kRows;
    const int rows = min(kRows, n * p.heads - r0);
    for (int k = tid; k < kRows * kDim; k += 256) {
        const int r = k / kDim, d = k - r * kDim;
        float v = 0.0f;
        if (r < rows && (d < kLatent || p.rope)) {
            const int tok = (r0 + r) / p.heads, h = (r0 + r) % p.heads;
            v = __bfloat162float(p.q[(first + tok) * p.q_st + h * p.q_sh + d]);
        }
        qs[k] = v;
    }
    const int row = tid >> 4, sub = tid & 15;
    const int lim = row < rows ? L - n + (r0 + row) / p.heads + 1 : 0;      // tokens this row sees
    const int end = min(L, L - n + (r0 + rows - 1) / p.heads + 1);
    float m = -INFINITY, l = 0.0f;
    float acc[kRows][2];
#pragma unroll
    for (int r = 0; r < kRows; ++r) acc[r][0] = acc[r][1] = 0.0f;
    for (int t0 = 0; t0 < end; t0 += kTok) {
        __syncthreads();
        for (int k = tid; k < kTok * 288; k += 256) {      // pairs of dims: 256 of the latent, 32 of the rope part
            const int t = k / 288, j = k - t * 288, pos = t0 + t;
            float a = 0.0f, c = 0.0f;
            if (pos < end) {
                const int pg = p.tables[b * p.tables_stride + (pos >> p.page_shift)];
                if (pg >= 0 && pg < p.num_pages) {
                    const int64_t slot = (static_cast<int64_t>(pg) << p.page_shift) | (pos & ((1 << p.page_shift) - 1));
                    if (j < 256) {
                        const uint8_t* kr = p.pool + slot * kRowBytes;
                        const uint32_t two = e2m1x2_to_f16x2(kr[j]);
                        const float s = e4m3_to_f32(kr[256 + j / 8]);
                        a = __half2float(__ushort_as_half(static_cast<unsigned short>(two & 0xFFFFu))) * s;
                        c = __half2float(__ushort_as_half(static_cast<unsigned short>(two >> 16))) * s;
                    } else if (p.rope) {
                        const uint32_t w = *reinterpret_cast<const uint32_t*>(p.rope + slot * kRope + 2 * (j - 256));
                        a = __uint_as_float(w << 16);
                        c = __uint_as_float(w & 0xFFFF0000u);
                    }
                }
            }
            ks[t * kLd + 2 * j] = a;
            ks[t * kLd + 2 * j + 1] = c;
        }
        __syncthreads();
        float x[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int t = sub + 16 * u, pos = t0 + t;
            float s = 0.0f;
            for (int d = 0; d < kDim; ++d) s = fmaf(qs[row * kDim + d], ks[t * kLd + d], s);
            bool see = pos < lim && pos < end;
            if (see) {
                const int pg = p.tables[b * p.tables_stride + (pos >> p.page_shift)];
                if (pg < 0 || pg >= p.num_pages) {
                    see = false;
                    set_error(p.err, NVFP4KV_DEVERR_BAD_PAGE);
                }
            }
            x[u] = see ? s * p.scale_log2 : -INFINITY;
        }
        float mt = fmaxf(m, fmaxf(x[0], x[1]));
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xFFFFFFFFu, mt, o));
        const float a = m == -INFINITY ? 0.0f : exp2f(m - mt);
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float e = x[u] == -INFINITY ? 0.0f : exp2f(x[u] - mt);
            ps[row * kTok + sub + 16 * u] = e;
            sum += e;
        }
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        l = l * a + sum;
        m = mt;
        if (sub == 0) al[row] = a;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            acc[r][0] *= al[r];
            acc[r][1] *= al[r];
        }
        for (int t = 0; t < kTok; ++t) {
            // a hidden token's values may be anything, even NaN: it does not take part
            const float v0 = ks[t * kLd + tid], v1 = ks[t * kLd + 256 + tid];
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const float e = ps[r * kTok + t];
                if (e != 0.0f) {
                    acc[r][0] = fmaf(e, v0, acc[r][0]);
                    acc[r][1] = fmaf(e, v1, acc[r][1]);
                }
            }
        }
    }
    __syncthreads();
    if (sub == 0) {
        al[row] = l > 0.0f || l != l ? p.out_scale / l : 0.0f;
        if (p.lse && row < rows) {
            const int tok = (r0 + row) / p.heads, h = (r0 + row) % p.heads;
            p.lse[static_cast<int64_t>(first + tok) * p.heads + h] =
                l > 0.0f || l != l ? 0.69314718055994531f * (m + log2f(l)) : -INFINITY;
        }
    }
    __syncthreads();
    for (int r = 0; r < rows; ++r) {
        const int tok = (r0 + r) / p.heads, h = (r0 + r) % p.heads;
        __nv_bfloat16* o = p.out + (first + tok) * p.o_st + h * p.o_sh;
        o[tid] = __float2bfloat16_rn(acc[r][0] * al[r]);
        o[256 + tid] = __float2bfloat16_rn(acc[r][1] * al[r]);
    }
}

}  // namespace
}  // namespace nvfp4kv

extern "C" int nvfp4kv_mla_prefill_workspace_size(int batch, int total_q, int num_heads, int max_q_len,
                                                  int max_seq_len, size_t* bytes) {
    using namespace nvfp4kv;
    if (!bytes) return fail(NVFP4KV_EINVAL, "mla_prefill_workspace_size: null output");
    if (batch < 0 || total_q < 0 || num_heads < 1 || max_q_len < 0 || max_seq_len < 0)
        return fail(NVFP4KV_EINVAL, "mla_prefill_workspace_size: bad shape");
    *bytes = 0;
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
    if (pool_rows <= 0 || pool_rows % page_size)
        return fail(NVFP4KV_EINVAL, "mla_prefill: pool_rows %lld not a positive multiple of page_size %d",
                    (long long)pool_rows, page_size);
    if (static_cast<int64_t>(max_q_len) * num_heads > 0x3FFFFFFF || static_cast<int64_t>(total_q) * num_heads > 0x7FFFFFFF)
        return fail(NVFP4KV_EINVAL, "mla_prefill: too many query rows");
    if (reinterpret_cast<uintptr_t>(pool) % 16 || reinterpret_cast<uintptr_t>(q) % 16 ||
        reinterpret_cast<uintptr_t>(rope_pool) % 16 || q_stride_t % 8 || q_stride_h % 8)
        return fail(NVFP4KV_EINVAL, "mla_prefill: pools and q must be 16-byte aligned and q strides multiples of 8");
    if (reinterpret_cast<uintptr_t>(out) % 16 || out_stride_t % 8 || out_stride_h % 8)
        return fail(NVFP4KV_EINVAL, "mla_prefill: out must be 16-byte aligned and its strides multiples of 8");
    size_t need = 0;
    int rc = nvfp4kv_mla_prefill_workspace_size(batch, total_q, num_heads, max_q_len, max_seq_len, &need);
    if (rc != NVFP4KV_OK) return rc;
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
    p.lse = lse; p.err = err_flag;
    const int smem = (kRows * kDim + kTok * kLd + kRows * kTok + kRows) * static_cast<int>(sizeof(float));
    cudaError_t e = cudaFuncSetAttribute(mla_prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return fail(NVFP4KV_ECUDA, "mla_prefill: %s", cudaGetErrorString(e));
    const int64_t blocks = static_cast<int64_t>(total_q) * num_heads / kRows + batch;
    mla_prefill_kernel<<<static_cast<unsigned>(blocks), 256, smem, reinterpret_cast<cudaStream_t>(stream)>>>(p);
    return check_launch("nvfp4kv_mla_prefill");
}
