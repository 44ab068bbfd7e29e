// Log probabilities of given tokens with entropy, rank and the top alternatives.
#include <climits>
#include <cmath>

#include "common.cuh"

namespace muyo {

constexpr int kLogprobThreads = 256;
constexpr int kLogprobJoinThreads = 128;
constexpr int kLogprobMaxTop = 32;
constexpr int kLogprobGroups = 64;  // groups of 4 threads whose maxima give the threshold
constexpr int kLogprobList = 4096;  // at least (kLogprobMaxTop - 1) groups of 4 threads of 32 logits, and kLogprobMaxTop

struct LogprobDev {
    int rows, vocab, top_k;
    long long stride;
    float inv_t;  // log2(e) / temperature
    float temperature;
    int pieces;   // of a row
    bool small;   // pieces of 2048 logits
};

// What a piece of a row says: m its largest logit, r the sum of 2^d over all but one largest, e the sum of
// 2^d d with d = (x - m) log2(e) / T, before: the ids in front of the given token.
struct LogprobPiece {
    float m, r, e;
    int before;
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

__device__ __forceinline__ unsigned long long warp_max_key(unsigned long long v)
{
    const unsigned hi = (unsigned)(v >> 32), most = __reduce_max_sync(0xffffffffu, hi);
    const unsigned lo = __reduce_max_sync(0xffffffffu, hi == most ? (unsigned)v : 0u);
    return (unsigned long long)most << 32 | lo;
}

// 2^(x + 64): sums are formed 2^64 times as large, so that terms down to 2^-190 of the largest stay normal.
constexpr float kLogprobDown = 5.421010862427522e-20f;  // 2^-64
__device__ __forceinline__ float ex2_up(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x + 64.0f));
    return y;
}

// One piece of a row: V float4 per thread, read once and kept in registers. The largest logit first, then the
// sums of 2^d and 2^d d (the thread that holds the largest leaves one of it out of r), the count in front of the
// token, and the piece's first top_k ids: with the logits' maxima over 64 groups of threads, the top_k-th
// largest of them is a threshold that top_k logits reach and few others do (24 of 8192 on average for 20 of
// 64 groups); those go to a list that is ordered by counting. Rows of equal values (a mask's -inf, or a
// constant) pass the threshold in masses: then the logits above it are listed, and of those equal to it the lowest ids.
template <int V>
__global__ void __launch_bounds__(kLogprobThreads) k_logprob_pieces(LogprobDev p, const float* __restrict__ logits,
                                                                    const int32_t* __restrict__ tokens,
                                                                    LogprobPiece* __restrict__ stats,
                                                                    unsigned long long* __restrict__ tops)
{
    constexpr int WARPS = kLogprobThreads / 32;
    __shared__ float s_max[WARPS], s_r[WARPS], s_e[WARPS], s_group[kLogprobGroups], s_threshold;
    __shared__ int s_before[WARPS], s_equal[WARPS], s_count, s_above, s_ties[WARPS];
    __shared__ unsigned long long s_key[WARPS];
    extern __shared__ unsigned long long s_list[];  // [kLogprobList] when top_k > 0
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / p.pieces, piece = blockIdx.x - row * p.pieces;
    const float* x = logits + row * p.stride;
    const int token = tokens[row];
    const float xt = token >= 0 && token < p.vocab ? __ldg(x + token) : INFINITY;  // outside: nothing in front
    // float4 from the 16-byte border at or before the row's first logit
    const int shift = (int)((reinterpret_cast<uintptr_t>(x) >> 2) & 3);
    const int base = piece * (kLogprobThreads * 4 * V) - shift + tid * 4;
    float v[V][4];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int i = base + j * kLogprobThreads * 4;
        if (i >= 0 && i <= p.vocab - 4) {
            const float4 f = ld_stream16f(x + i);
            v[j][0] = f.x, v[j][1] = f.y, v[j][2] = f.z, v[j][3] = f.w;
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                v[j][c] = i + c >= 0 && i + c < p.vocab ? __ldg(x + i + c) : -INFINITY;
        }
    }
    float mine = -INFINITY;
#pragma unroll
    for (int j = 0; j < V; ++j)
        mine = fmaxf(mine, fmaxf(fmaxf(v[j][0], v[j][1]), fmaxf(v[j][2], v[j][3])));
    const float four = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
    const float group = fmaxf(four, __shfl_xor_sync(0xffffffffu, four, 2));
    float m = group;
#pragma unroll
    for (int o = 4; o < 32; o <<= 1)
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0)
        s_max[warp] = m;
    if ((tid & 3) == 0)
        s_group[tid >> 2] = group;
    if (tid == 0)
        s_count = s_above = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
        m = fmaxf(m, s_max[w]);
    // sums
    const float ms = m == -INFINITY ? 0.0f : m;
    float r = 0.0f, e = 0.0f;
    int before = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int i = base + j * kLogprobThreads * 4;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float d = (v[j][c] - ms) * p.inv_t, w = ex2_up(d);
            r += w;
            e = fmaf(w, fmaxf(d, -300.0f), e);
            before += v[j][c] > xt || (v[j][c] == xt && (unsigned)(i + c) < (unsigned)token);
        }
    }
    int equal = 0;
    if (mine == m && m > -INFINITY) {  // the sum again, without the largest: they are counted
        r = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                r += v[j][c] == m ? 0.0f : ex2_up((v[j][c] - ms) * p.inv_t);
                equal += v[j][c] == m;
            }
    }
    equal = __reduce_add_sync(0xffffffffu, equal);
    r = warp_sum(r);
    e = warp_sum(e);
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0)
        s_r[warp] = r, s_e[warp] = e, s_before[warp] = before, s_equal[warp] = equal;
    if (p.top_k > 0 && tid < kLogprobGroups) {  // the group whose maximum is the top_k-th largest
        const float g = s_group[tid];
        int place = 0;
#pragma unroll 8
        for (int i = 0; i < kLogprobGroups; ++i)
            place += s_group[i] > g || (s_group[i] == g && i < tid);
        if (place == p.top_k - 1)
            s_threshold = g;
    }
    __syncthreads();
    if (tid == 0) {
        LogprobPiece out{m, 0.0f, 0.0f, 0};
        equal = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w)
            out.r += s_r[w], out.e += s_e[w], out.before += s_before[w], equal += s_equal[w];
        out.r = fmaf(out.r, kLogprobDown, equal > 0 ? (float)(equal - 1) : 0.0f);
        out.e *= kLogprobDown;
        stats[blockIdx.x] = out;
    }
    if (p.top_k == 0)
        return;
    const float threshold = s_threshold;
    unsigned above = 0, equals = 0;  // bit 4 j + c
    if (mine >= threshold) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int i = base + j * kLogprobThreads * 4;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                above |= v[j][c] > threshold ? 1u << (4 * j + c) : 0u;
                equals |= v[j][c] == threshold && i + c >= 0 && i + c < p.vocab ? 1u << (4 * j + c) : 0u;
            }
        }
    }
    const auto id_of = [&](int bit) { return base + (bit >> 2) * kLogprobThreads * 4 + (bit & 3); };
    const auto list = [&](unsigned bits, int at) {
#pragma unroll 1
        for (; bits; bits &= bits - 1, ++at) {
            const int id = id_of(__ffs(bits) - 1);
            s_list[at] = order_key(__ldg(x + id), id);
        }
    };
    const unsigned reach = above | equals;
    int at = reach ? atomicAdd(&s_count, __popc(reach)) : 0;
    __syncthreads();
    int n = s_count;
    if (n <= kLogprobList) {
        list(reach, at);
    } else {  // too many equal ones
        if (above)
            list(above, atomicAdd(&s_above, __popc(above)));
        __syncthreads();
        n = s_above;  // of less than top_k groups of threads
        int have = 0;
#pragma unroll 1
        for (int j = 0; j < V && have < p.top_k; ++j) {  // by id: place j of every thread, then j + 1
            const unsigned bits = equals & (15u << (4 * j));
            int incl = __popc(bits);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o)
                    incl += y;
            }
            if (lane == 31)
                s_ties[warp] = incl;
            __syncthreads();
            at = have + incl - __popc(bits);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                at += w < warp ? s_ties[w] : 0;
                have += s_ties[w];
            }
#pragma unroll 1
            for (unsigned left = bits; left && at < p.top_k; left &= left - 1, ++at)
                s_list[n + at] = order_key(threshold, id_of(__ffs(left) - 1));
            __syncthreads();
        }
        n += min(have, p.top_k);
    }
    __syncthreads();
    unsigned long long* out = tops + (size_t)blockIdx.x * p.top_k;
    if (n <= kLogprobThreads) {  // a key's place is the number of larger ones
        if (tid < n) {
            const unsigned long long key = s_list[tid];
            int place = 0;
#pragma unroll 4
            for (int i = 0; i < n; ++i)
                place += s_list[i] > key;
            if (place < p.top_k)
                out[place] = key;
        }
        if (tid >= n && tid < p.top_k)
            out[tid] = 0ull;
    } else {  // one by one
        unsigned long long last = ~0ull;
#pragma unroll 1
        for (int k = 0; k < p.top_k; ++k) {
            unsigned long long next = 0ull;
#pragma unroll 1
            for (int i = tid; i < n; i += kLogprobThreads)
                next = s_list[i] < last && s_list[i] > next ? s_list[i] : next;
            next = warp_max_key(next);
            __syncthreads();
            if (lane == 0)
                s_key[warp] = next;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WARPS; ++w)
                next = s_key[w] > next ? s_key[w] : next;
            last = next;
            if (tid == 0)
                out[k] = next;
        }
    }
}

// Joins a row's pieces: one CTA per row, a piece per thread at a time. log p = (x - m) / T - log(1 + r), where
// nothing is lost of r when it is far below 1; H = log(1 + r) - ln 2 e / (1 + r).
__global__ void __launch_bounds__(kLogprobJoinThreads) k_logprob_join(LogprobDev p, const float* __restrict__ logits,
                                                                      const int32_t* __restrict__ tokens,
                                                                      const LogprobPiece* __restrict__ stats,
                                                                      const unsigned long long* __restrict__ tops,
                                                                      float* __restrict__ logprob, float* __restrict__ entropy,
                                                                      int32_t* __restrict__ rank, int32_t* __restrict__ top_ids,
                                                                      float* __restrict__ top_logprobs)
{
    constexpr int WARPS = kLogprobJoinThreads / 32;
    __shared__ float s_m[WARPS], s_r[WARPS], s_e[WARPS];
    __shared__ int s_before[WARPS], s_equal[WARPS];
    __shared__ unsigned long long s_key[2][WARPS];
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x;
    const LogprobPiece* mine = stats + (size_t)row * p.pieces;
    const int token = tokens[row];
    const bool inside = token >= 0 && token < p.vocab;
    const float xt = inside ? __ldg(logits + row * p.stride + token) : 0.0f;
    float m = -INFINITY;
#pragma unroll 1
    for (int c = tid; c < p.pieces; c += kLogprobJoinThreads)
        m = fmaxf(m, mine[c].m);
    m = warp_max(m);
    if (lane == 0)
        s_m[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
        m = fmaxf(m, s_m[w]);
    const float ms = m == -INFINITY ? 0.0f : m;
    float r = 0.0f, e = 0.0f;
    int before = 0, equal = 0;
#pragma unroll 1
    for (int c = tid; c < p.pieces; c += kLogprobJoinThreads) {
        const LogprobPiece q = mine[c];
        const bool top = q.m == m;
        const float d = (q.m - ms) * p.inv_t, w = ex2_up(d);
        r += top ? q.r : (1.0f + q.r) * w * kLogprobDown;
        equal += top;
        e += top ? q.e : fmaf(fmaxf(d, -300.0f), 1.0f + q.r, q.e) * w * kLogprobDown;
        before += q.before;
    }
    r = warp_sum(r);
    e = warp_sum(e);
    before = __reduce_add_sync(0xffffffffu, before);
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0)
        s_r[warp] = r, s_e[warp] = e, s_before[warp] = before, s_equal[warp] = equal;
    __syncthreads();
    r = e = 0.0f;
    before = equal = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
        r += s_r[w], e += s_e[w], before += s_before[w], equal += s_equal[w];
    const bool nothing = m == -INFINITY && r == r;
    r = m == INFINITY ? NAN : r + (float)(equal - 1);
    const float log_sum = log1pf(r);
    if (tid == 0) {
        logprob[row] = !inside || nothing ? -INFINITY : __fdiv_rn(xt - ms, p.temperature) - log_sum;
        if (entropy)
            entropy[row] = nothing ? 0.0f : log_sum - 0.693147180559945f * e / (1.0f + r);
        if (rank)
            rank[row] = inside ? before : p.vocab;
    }
    if (p.top_k == 0)
        return;
    // The pieces' lists, each in order: the largest head top_k times.
    const unsigned long long* list = tops + (size_t)row * p.pieces * p.top_k;
    int at = 0;  // of the thread's first list
    unsigned long long last = ~0ull, head = tid < p.pieces ? list[(size_t)tid * p.top_k] : 0ull;
#pragma unroll 1
    for (int k = 0; k < p.top_k; ++k) {
        unsigned long long best = head;
#pragma unroll 1
        for (int c = tid + kLogprobJoinThreads; c < p.pieces; c += kLogprobJoinThreads) {
            int i = 0;
            while (i < p.top_k && list[(size_t)c * p.top_k + i] >= last)
                ++i;
            const unsigned long long next = i < p.top_k ? list[(size_t)c * p.top_k + i] : 0ull;
            best = next > best ? next : best;
        }
        best = warp_max_key(best);
        if (lane == 0)
            s_key[k & 1][warp] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WARPS; ++w)
            best = s_key[k & 1][w] > best ? s_key[k & 1][w] : best;
        last = best;
        if (head == best && best != 0ull) {  // keys differ: one thread
            ++at;
            head = at < p.top_k ? list[(size_t)tid * p.top_k + at] : 0ull;
        }
        if (tid == 0) {
            top_ids[(size_t)row * p.top_k + k] = best ? (int)~(unsigned)best : -1;
            const float v = best ? key_logit(best) : NAN;
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
    // Pieces of 8192 logits; of 2048 where the larger ones would leave SMs without a CTA. A row may begin 3 logits
    // behind a 16-byte border.
    const long long large = (d.vocab + 3LL + 8191) / 8192;
    d.small = large * d.rows < sm_count();
    d.pieces = (int)(d.small ? (d.vocab + 3LL + 2047) / 2048 : large);
    if ((long long)d.pieces * d.rows > INT_MAX) {
        set_error("token_logprobs: %u rows of %u logits are more than 2^31 pieces", p->rows, p->vocab);
        return MUYO_EUNSUPPORTED;
    }
    return MUYO_OK;
}

static size_t logprobs_stats_bytes(const LogprobDev& d) { return (size_t)d.rows * d.pieces * sizeof(LogprobPiece); }

extern "C" size_t muyo_cuda_token_logprobs_workspace_size(const MuyoTokenLogprobsParams* p)
{
    LogprobDev d{};
    if (!p || logprobs_prepare(p, d) != MUYO_OK)
        return 0;
    return logprobs_stats_bytes(d) + (size_t)d.rows * d.pieces * d.top_k * sizeof(unsigned long long);
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
    LogprobPiece* stats = static_cast<LogprobPiece*>(workspace);
    unsigned long long* tops = reinterpret_cast<unsigned long long*>(static_cast<char*>(workspace) + logprobs_stats_bytes(d));
    const size_t smem = d.top_k ? kLogprobList * sizeof(unsigned long long) : 0;
    MUYO_CUDA_TRY(launch_kernel(d.small ? k_logprob_pieces<2> : k_logprob_pieces<8>, dim3(d.rows * d.pieces),
                                dim3(kLogprobThreads), smem, as_stream(stream), true, d, logits, tokens, stats, tops));
    MUYO_LAUNCH_CHECK();
    MUYO_CUDA_TRY(launch_kernel(k_logprob_join, dim3(d.rows), dim3(kLogprobJoinThreads), 0, as_stream(stream), true, d, logits,
                                tokens, stats, tops, logprob, entropy, rank, top_ids, top_logprobs));
    MUYO_LAUNCH_CHECK();
    return MUYO_OK;
}
