// Log probabilities of given tokens with entropy, rank and the top alternatives.
#include <climits>
#include <cmath>

#include "common.cuh"

namespace muyo {

constexpr int kLogprobThreads = 256;
constexpr int kLogprobMaxTop = 32;

struct LogprobDev {
    int rows, vocab, top_k;
    long long stride;
    float inv_t;  // log2(e) / temperature
    float temperature;
};

// Order of the alternatives: larger logit first, then the lower id. -0 counts as +0; 0 stands for "no
// element" (also a NaN).
__device__ __forceinline__ unsigned long long order_key(float v, int id)
{
    unsigned b = __float_as_uint(v);
    if (b == 0x80000000u)
        b = 0u;
    const unsigned k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return v != v ? 0ull : ((unsigned long long)k << 32) | (unsigned)~id;
}

__device__ __forceinline__ float key_logit(unsigned long long key)
{
    const unsigned k = (unsigned)(key >> 32);
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

__device__ __forceinline__ unsigned long long block_max_key(unsigned long long v, unsigned long long* red)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long y = __shfl_xor_sync(0xffffffffu, v, o);
        v = y > v ? y : v;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0)
        red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < kLogprobThreads / 32; ++w)
        v = red[w] > v ? red[w] : v;
    return v;
}

// One CTA per row: the largest logit m, then r = the sum of 2^d over all but one largest and e = the sum
// of 2^d d, with d = (x - m) log2(e) / T, then one pass per alternative. log p = (x - m) / T - log(1 + r):
// nothing is lost of r when it is far below 1. H = log(1 + r) - ln 2 e / (1 + r).
__global__ void __launch_bounds__(kLogprobThreads) k_token_logprobs(LogprobDev p, const float* __restrict__ logits,
                                                                    const int32_t* __restrict__ tokens,
                                                                    float* __restrict__ logprob, float* __restrict__ entropy,
                                                                    int32_t* __restrict__ rank, int32_t* __restrict__ top_ids,
                                                                    float* __restrict__ top_logprobs)
{
    __shared__ unsigned long long s_key[kLogprobThreads / 32];
    __shared__ float red[32];
    pdl_wait();
    pdl_trigger();
    const int row = blockIdx.x, tid = threadIdx.x;
    const float* x = logits + row * p.stride;
    const int token = tokens[row];
    const bool inside = token >= 0 && token < p.vocab;
    const float xt = inside ? x[token] : 0.0f;
    float m = -INFINITY;
    int best = -1;  // the largest's first place in this thread
    for (int i = tid; i < p.vocab; i += kLogprobThreads) {
        if (x[i] > m) {
            m = x[i];
            best = i;
        }
    }
    const unsigned long long top = block_max_key(best >= 0 ? order_key(m, best) : 0ull, s_key);
    m = top ? key_logit(top) : -INFINITY;
    best = top ? (int)~(unsigned)top : -1;
    const float ms = m == -INFINITY ? 0.0f : m;
    float r = 0.0f, e = 0.0f, before = 0.0f;
    for (int i = tid; i < p.vocab; i += kLogprobThreads) {
        const float d = (x[i] - ms) * p.inv_t, w = exp2f(d);
        if (i != best)
            r += w;
        e = fmaf(w, fmaxf(d, -300.0f), e);
        before += x[i] > xt || (x[i] == xt && i < token) ? 1.0f : 0.0f;  // exact: a thread counts below 2^24
    }
    r = m == INFINITY ? NAN : block_sum(r, red);
    e = block_sum(e, red);
    __syncthreads();
    int count = (int)before;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        count += __shfl_xor_sync(0xffffffffu, count, o);
    int* s_count = reinterpret_cast<int*>(red);
    if ((tid & 31) == 0)
        s_count[tid >> 5] = count;
    __syncthreads();
    const float ln2 = 0.693147180559945f;
    const bool nothing = m == -INFINITY && r == r;
    const float log_sum = log1pf(r);
    if (tid == 0) {
        logprob[row] = !inside || nothing ? -INFINITY : __fdiv_rn(xt - ms, p.temperature) - log_sum;
        if (entropy)
            entropy[row] = nothing ? 0.0f : log_sum - ln2 * e / (1.0f + r);
        if (rank) {
            int c = 0;
            for (int w = 0; w < kLogprobThreads / 32; ++w)
                c += s_count[w];
            rank[row] = inside ? c : p.vocab;
        }
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < p.top_k; ++k) {
        unsigned long long next = 0ull;
        for (int i = tid; i < p.vocab; i += kLogprobThreads) {
            const unsigned long long key = order_key(x[i], i);
            next = key < last && key > next ? key : next;
        }
        last = block_max_key(next, s_key);
        if (tid == 0) {
            top_ids[(size_t)row * p.top_k + k] = last ? (int)~(unsigned)last : -1;
            const float v = last ? key_logit(last) : NAN;
            top_logprobs[(size_t)row * p.top_k + k] = nothing ? -INFINITY : __fdiv_rn(v - ms, p.temperature) - log_sum;
        }
    }
}

}  // namespace muyo

using namespace muyo;

static int logprobs_prepare(const MuyoTokenLogprobsParams* p, LogprobDev& d)
{
    MUYO_REQUIRE(p, "token_logprobs: null parameter block");
    MUYO_REQUIRE(p->rows > 0 && p->rows <= (uint32_t)INT_MAX, "token_logprobs: rows must be in [1, INT32_MAX]");
    MUYO_REQUIRE(p->vocab > 0 && p->vocab <= (1u << 28), "token_logprobs: vocab %u must be in [1, 2^28]", p->vocab);
    MUYO_REQUIRE(p->stride == 0 || p->stride >= p->vocab, "token_logprobs: stride %u is below vocab %u", p->stride, p->vocab);
    MUYO_REQUIRE(p->top_k <= (uint32_t)kLogprobMaxTop && p->top_k <= p->vocab,
                 "token_logprobs: top_k %u must be at most %d and at most vocab", p->top_k, kLogprobMaxTop);
    MUYO_REQUIRE(std::isfinite(p->temperature) && p->temperature > 0.0f, "token_logprobs: temperature must be positive");
    d.rows = (int)p->rows, d.vocab = (int)p->vocab, d.top_k = (int)p->top_k;
    d.stride = p->stride ? p->stride : p->vocab;
    d.temperature = p->temperature;
    d.inv_t = (float)(1.4426950408889634 / (double)p->temperature);
    return MUYO_OK;
}

extern "C" size_t muyo_cuda_token_logprobs_workspace_size(const MuyoTokenLogprobsParams* p)
{
    LogprobDev d{};
    return p && logprobs_prepare(p, d) == MUYO_OK ? 256 : 0;
}

extern "C" int muyo_cuda_token_logprobs(const MuyoTokenLogprobsParams* p, const float* logits, const int32_t* tokens,
                                        float* logprob, float* entropy, int32_t* rank, int32_t* top_ids, float* top_logprobs,
                                        void* workspace, size_t workspace_bytes, void* stream)
{
    clear_error();
    LogprobDev d{};
    const int rc = logprobs_prepare(p, d);
    if (rc != MUYO_OK)
        return rc;
    MUYO_REQUIRE(logits && tokens && logprob, "token_logprobs: null buffer");
    MUYO_REQUIRE((reinterpret_cast<uintptr_t>(logits) & 3u) == 0, "token_logprobs: logits must be 4-byte aligned");
    MUYO_REQUIRE(d.top_k == 0 || (top_ids && top_logprobs), "token_logprobs: top_ids and top_logprobs are needed with top_k");
    const size_t need = muyo_cuda_token_logprobs_workspace_size(p);
    MUYO_REQUIRE(workspace && workspace_bytes >= need, "token_logprobs: workspace of %zu bytes needed, %zu given", need,
                 workspace_bytes);
    MUYO_REQUIRE(aligned16(workspace), "token_logprobs: workspace must be 16-byte aligned");
    MUYO_CUDA_TRY(launch_kernel(k_token_logprobs, dim3(d.rows), dim3(kLogprobThreads), 0, as_stream(stream), true, d, logits,
                                tokens, logprob, entropy, rank, top_ids, top_logprobs));
    MUYO_LAUNCH_CHECK();
    return MUYO_OK;
}
