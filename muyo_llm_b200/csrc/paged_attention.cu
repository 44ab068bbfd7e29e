// Attention of one new token per request over a paged key-value cache.
#include "paged.cuh"

namespace muyo {

constexpr int kPagedThreads = 256;
constexpr int kPagedMaxGroup = 16;

struct PagedAttnDev {
    PagedDev c;
    int seqs, table_stride, window;
    long long stride_q, stride_out;
    float scale;  // softmax scale * k_scale
};

template <typename KV>
__device__ __forceinline__ float pool_value(KV v);
template <>
__device__ __forceinline__ float pool_value<float>(float v)
{
    return v;
}
template <>
__device__ __forceinline__ float pool_value<__half>(__half v)
{
    return __half2float(v);
}
template <>
__device__ __forceinline__ float pool_value<__nv_fp8_e4m3>(__nv_fp8_e4m3 v)
{
    return float(v);
}

// One CTA per (request, KV head): each warp takes every eighth key with an online softmax per query head
// (lanes over the channels), and the warps' (m, l, o) are joined in shared memory.
template <typename KV, int HD>
__global__ void __launch_bounds__(kPagedThreads) k_paged_attention(PagedAttnDev p, const float* __restrict__ q,
                                                                   const KV* __restrict__ k_pool, const KV* __restrict__ v_pool,
                                                                   const int32_t* __restrict__ table,
                                                                   const int32_t* __restrict__ seq_lens,
                                                                   float* __restrict__ out, float* __restrict__ lse)
{
    constexpr int E = (HD + 31) / 32;  // channels per lane
    __shared__ float s_m[8][kPagedMaxGroup], s_l[8][kPagedMaxGroup], s_o[8][HD];
    pdl_wait();
    pdl_trigger();
    const int s = blockIdx.x, kvh = blockIdx.y, G = p.c.group;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n = min(max(seq_lens[s], 0), p.table_stride * p.c.page_size);
    const int begin = p.window > 0 ? max(0, n - p.window) : 0;
    const float* qs = q + s * p.stride_q + (long long)kvh * G * HD;
    float* os = out + s * p.stride_out + (long long)kvh * G * HD;
    float qv[kPagedMaxGroup][E], o[kPagedMaxGroup][E], m[kPagedMaxGroup], l[kPagedMaxGroup];
#pragma unroll
    for (int g = 0; g < kPagedMaxGroup; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int d = lane + 32 * e;
            qv[g][e] = g < G && d < HD ? qs[g * HD + d] * p.scale : 0.0f;
            o[g][e] = 0.0f;
        }
    }
    for (int t = begin + warp; t < n; t += 8) {
        const int page = table[(size_t)s * p.table_stride + t / p.c.page_size];
        if (page < 0 || page >= p.c.num_pages)
            continue;
        const long long row = page * p.c.page_stride + kvh * p.c.head_stride + (t % p.c.page_size) * p.c.slot_stride;
        float k[E], v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int d = lane + 32 * e;
            k[e] = d < HD ? pool_value<KV>(k_pool[row + d]) : 0.0f;
            v[e] = d < HD ? pool_value<KV>(v_pool[row + d]) : 0.0f;
        }
#pragma unroll
        for (int g = 0; g < kPagedMaxGroup; ++g) {
            if (g < G) {
                float x = 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e)
                    x = fmaf(qv[g][e], k[e], x);
                x = warp_sum(x);
                const float mn = fmaxf(m[g], x), a = expf(m[g] - mn), w = expf(x - mn);
                m[g] = mn;
                l[g] = fmaf(l[g], a, w);
#pragma unroll
                for (int e = 0; e < E; ++e)
                    o[g][e] = fmaf(o[g][e], a, w * v[e]);
            }
        }
    }
#pragma unroll
    for (int g = 0; g < kPagedMaxGroup; ++g) {
        if (g < G) {
            if (lane == 0) {
                s_m[warp][g] = m[g];
                s_l[warp][g] = l[g];
            }
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (lane + 32 * e < HD)
                    s_o[warp][lane + 32 * e] = o[g][e];
            __syncthreads();
            float M = -INFINITY;
            for (int w = 0; w < 8; ++w)
                M = fmaxf(M, s_m[w][g]);
            float L = 0.0f;
            for (int w = 0; w < 8; ++w)
                L += s_l[w][g] > 0.0f ? s_l[w][g] * expf(s_m[w][g] - M) : 0.0f;
            for (int d = threadIdx.x; d < HD; d += kPagedThreads) {
                float O = 0.0f;
                for (int w = 0; w < 8; ++w)
                    O += s_l[w][g] > 0.0f ? s_o[w][d] * expf(s_m[w][g] - M) : 0.0f;
                os[g * HD + d] = L > 0.0f ? O / L * p.c.v_scale : 0.0f;
            }
            if (lse && threadIdx.x == 0)
                lse[(size_t)s * p.c.heads + kvh * G + g] = L > 0.0f ? M + logf(L) : -INFINITY;
            __syncthreads();
        }
    }
}

static int paged_attention_prepare(const MuyoPagedAttentionParams* p, PagedAttnDev& d)
{
    MUYO_REQUIRE(p, "paged_attention: null parameter block");
    const int rc = paged_prepare(p->cache, "paged_attention", d.c);
    if (rc != MUYO_OK)
        return rc;
    MUYO_REQUIRE(p->seqs > 0 && p->seqs <= (uint32_t)INT_MAX, "paged_attention: seqs must be in [1, INT32_MAX]");
    MUYO_REQUIRE(p->table_stride > 0 && (uint64_t)p->cache.page_size * p->table_stride <= (uint64_t)INT_MAX,
                 "paged_attention: table_stride %u must be positive, and a row at most INT32_MAX slots", p->table_stride);
    MUYO_REQUIRE(p->window <= (uint32_t)INT_MAX, "paged_attention: window %u exceeds INT32_MAX", p->window);
    MUYO_REQUIRE(std::isfinite(p->scale), "paged_attention: scale must be finite");
    const uint32_t row = p->cache.heads * p->cache.head_dim;
    d.stride_q = p->stride_q ? p->stride_q : row;
    d.stride_out = p->stride_out ? p->stride_out : row;
    MUYO_REQUIRE(d.stride_q >= row && d.stride_out >= row, "paged_attention: a row stride is below the row of %u", row);
    MUYO_REQUIRE((d.stride_q | d.stride_out) % 4 == 0, "paged_attention: row strides must be multiples of 4");
    d.seqs = (int)p->seqs, d.table_stride = (int)p->table_stride, d.window = (int)p->window;
    d.scale = p->scale * d.c.k_scale;
    return MUYO_OK;
}

template <typename KV, int HD>
static int launch_paged_attention(const PagedAttnDev& d, const float* q, const void* k, const void* v, const int32_t* table,
                                  const int32_t* lens, float* out, float* lse, void* stream)
{
    MUYO_CUDA_TRY(launch_kernel(k_paged_attention<KV, HD>, dim3(d.seqs, d.c.kv_heads), dim3(kPagedThreads), 0,
                                as_stream(stream), true, d, q, static_cast<const KV*>(k), static_cast<const KV*>(v), table,
                                lens, out, lse));
    MUYO_LAUNCH_CHECK();
    return MUYO_OK;
}

template <typename KV>
static int launch_paged_attention_dim(const PagedAttnDev& d, const float* q, const void* k, const void* v,
                                      const int32_t* table, const int32_t* lens, float* out, float* lse, void* stream)
{
    switch (d.c.head_dim) {
        case 16: return launch_paged_attention<KV, 16>(d, q, k, v, table, lens, out, lse, stream);
        case 32: return launch_paged_attention<KV, 32>(d, q, k, v, table, lens, out, lse, stream);
        case 64: return launch_paged_attention<KV, 64>(d, q, k, v, table, lens, out, lse, stream);
        default: return launch_paged_attention<KV, 128>(d, q, k, v, table, lens, out, lse, stream);
    }
}

}  // namespace muyo

using namespace muyo;

extern "C" size_t muyo_cuda_paged_attention_workspace_size(const MuyoPagedAttentionParams* p)
{
    PagedAttnDev d{};
    return p && paged_attention_prepare(p, d) == MUYO_OK ? 256 : 0;
}

extern "C" int muyo_cuda_paged_attention_decode(const MuyoPagedAttentionParams* p, const float* q, const void* k_pool,
                                                const void* v_pool, const int32_t* block_table, const int32_t* seq_lens,
                                                float* out, float* lse, void* workspace, size_t workspace_bytes,
                                                void* stream)
{
    clear_error();
    PagedAttnDev d{};
    const int rc = paged_attention_prepare(p, d);
    if (rc != MUYO_OK)
        return rc;
    MUYO_REQUIRE(q && k_pool && v_pool && block_table && seq_lens && out, "paged_attention: null buffer");
    MUYO_REQUIRE(aligned16(q) && aligned16(out) && aligned16(k_pool) && aligned16(v_pool),
                 "paged_attention: q, out and the pools must be 16-byte aligned");
    const size_t need = muyo_cuda_paged_attention_workspace_size(p);
    MUYO_REQUIRE(workspace && workspace_bytes >= need, "paged_attention: workspace of %zu bytes needed, %zu given", need,
                 workspace_bytes);
    MUYO_REQUIRE(aligned16(workspace), "paged_attention: workspace must be 16-byte aligned");
    switch (p->cache.kv_dtype) {
        case MUYO_KV_F32:
            return launch_paged_attention_dim<float>(d, q, k_pool, v_pool, block_table, seq_lens, out, lse, stream);
        case MUYO_KV_F16:
            return launch_paged_attention_dim<__half>(d, q, k_pool, v_pool, block_table, seq_lens, out, lse, stream);
        default:
            return launch_paged_attention_dim<__nv_fp8_e4m3>(d, q, k_pool, v_pool, block_table, seq_lens, out, lse, stream);
    }
}
