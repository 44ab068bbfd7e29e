// Log probabilities of given tokens with entropy, rank and the top alternatives.
#include <climits>
#include <cmath>

#include "common.cuh"

namespace muyo {

constexpr int kLogprobThreads = 256;
constexpr int kLogprobWarps = kLogprobThreads / 32;
constexpr int kLogprobJoinThreads = 128;
constexpr int kLogprobMaxTop = 32;
constexpr int kLogprobGroups = 64;   // groups of 4 threads whose maxima give the first threshold
constexpr int kLogprobKeep = 256;    // keys that the list may carry from tile to tile: a thread each
constexpr int kLogprobMaxTiles = 64; // of a piece

struct LogprobDev {
    int rows, vocab, top_k;
    long long stride;
    float inv_t;  // log2(e) / temperature
    float temperature;
    int pieces, tiles;  // of a row; of a piece
    bool small;         // tiles of 2048 logits instead of 4096
};

struct LogprobOut {
    float* logprob;
    float* entropy;
    int32_t* rank;
    int32_t* top_ids;
    float* top_logprobs;
};

// What a piece of a row says: m its largest logit, r the sum of w = exp((x - m) / T) over all but one largest, e the
// sum of w (x - m), before: the ids in front of the given token.
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

// exp(u / T) 2^64: the sums are formed 2^64 times as large, so that terms down to 2^-190 of the largest stay normal.
constexpr float kLogprobDown = 5.421010862427522e-20f;  // 2^-64
__device__ __forceinline__ float weight_up(float u, float inv_t)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaf(u, inv_t, 64.0f)));
    return y;
}
constexpr float kLogprobLeast = -1.0e29f;  // u where the weight is 0, so that 0 * -inf does not arise

// A row's results from its sums. log p = (x - m) / T - log(1 + r), where nothing is lost of r when it is far
// below 1; H = log(1 + r) - e / (T (1 + r)).
struct LogprobRow {
    float m, log_sum, temperature;
    bool nothing;  // no logit but -inf
    __device__ __forceinline__ LogprobRow(const LogprobDev& p, const LogprobPiece& q)
        : m(q.m == -INFINITY ? 0.0f : q.m), temperature(p.temperature), nothing(q.m == -INFINITY && q.r == q.r)
    {
        log_sum = q.m == INFINITY ? NAN : log1pf(q.r);
    }
    __device__ __forceinline__ float log_p(float x) const
    {
        return nothing ? -INFINITY : __fdiv_rn(x - m, temperature) - log_sum;
    }
    __device__ __forceinline__ void write(const LogprobDev& p, const LogprobOut& out, const LogprobPiece& q, int row, int token,
                                          float xt) const
    {
        const bool inside = token >= 0 && token < p.vocab;
        out.logprob[row] = inside ? log_p(xt) : -INFINITY;
        if (out.entropy)
            out.entropy[row] = nothing ? 0.0f : log_sum - __fdiv_rn(__fdiv_rn(q.e, temperature), 1.0f + q.r);
        if (out.rank)
            out.rank[row] = inside ? q.before : p.vocab;
    }
    __device__ __forceinline__ void write_top(const LogprobOut& out, size_t at, unsigned long long key) const
    {
        out.top_ids[at] = key ? (int)~(unsigned)key : -1;
        out.top_logprobs[at] = log_p(key ? key_logit(key) : NAN);
    }
};

// One piece of a row, read once: `tiles` tiles of V float4 per thread, the next one's loads under way while one is
// worked on. A thread keeps its largest logit so far and its sums of w and w (x - m) relative to it. An id
// below the token is in front of it at an equal logit too: it is compared with the next value below the token's.
//
// The first top_k ids: in the first tile the maxima of 64 groups of 4 threads give a threshold, the
// top_k-th largest of them, that top_k logits reach and few others do (24 on average for 20 of 64 groups);
// later tiles list what lies above it (an equal logit of a later id comes behind). A list past
// kLogprobKeep keys is cut to its first top_k, whose last is the new threshold. A first tile with masses
// at the threshold (a mask's -inf, a constant row) lists the logits above it, and of the equal ones the lowest ids.
//
// Bound by the read: 4 bytes a logit, 13 instructions.
template <int V>
__global__ void __launch_bounds__(kLogprobThreads, 4) k_logprob_pieces(LogprobDev p, const float* __restrict__ logits,
                                                                       const int32_t* __restrict__ tokens,
                                                                       LogprobPiece* __restrict__ stats,
                                                                       unsigned long long* __restrict__ tops, LogprobOut out)
{
    constexpr int WARPS = kLogprobWarps, TILE = kLogprobThreads * 4 * V;
    __shared__ float s_m[WARPS], s_r[WARPS], s_e[WARPS], s_group[kLogprobGroups], s_threshold;
    __shared__ int s_before[WARPS], s_equal[WARPS], s_count, s_above, s_ties[WARPS];
    __shared__ unsigned long long s_key[WARPS], s_top[kLogprobMaxTop];
    extern __shared__ unsigned long long s_list[];  // [kLogprobKeep + TILE] when top_k > 0
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / p.pieces, piece = blockIdx.x - row * p.pieces;
    const float* x = logits + row * p.stride;
    const int token = __ldg(tokens + row);  // not waited for before the first tile's loads are under way
    // float4 from the 16-byte border at or before the row's first logit
    const int shift = (int)((reinterpret_cast<uintptr_t>(x) >> 2) & 3);
    const int first = piece * p.tiles * TILE - shift, end = min(first + p.tiles * TILE, p.vocab);
    int base = first + tid * 4;  // of the tile at hand: id of bit 0
    const auto load = [&](float (&v)[V][4], int at) {
        const int tile = at - tid * 4;
        if (tile >= 0 && tile + TILE <= p.vocab) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float4 f = ld_stream16f(x + at + j * kLogprobThreads * 4);
                v[j][0] = f.x, v[j][1] = f.y, v[j][2] = f.z, v[j][3] = f.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int i = at + j * kLogprobThreads * 4;
                if (i >= 0 && i <= p.vocab - 4) {
                    const float4 f = ld_stream16f(x + i);
                    v[j][0] = f.x, v[j][1] = f.y, v[j][2] = f.z, v[j][3] = f.w;
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        v[j][c] = i + c >= 0 && i + c < p.vocab ? __ldg(x + i + c) : -INFINITY;
                }
            }
        }
    };
    float v[V][4];
    load(v, base);
    const float xt = token >= 0 && token < p.vocab ? __ldg(x + token) : INFINITY;  // outside: nothing in front
    const float below = nextafterf(xt, -INFINITY);
    float m = -INFINITY, r = 0.0f, e = 0.0f;  // r: 2^64 times the sum
    int before = 0;
    float threshold = -INFINITY;
    if (tid == 0)
        s_count = s_above = 0;
    // The list's keys in order into s_top, at most top_k of them; 0 behind them.
    const auto order = [&](int n) {
        if (n <= kLogprobThreads) {  // a key's place is the number of larger ones
            if (tid < n) {
                const unsigned long long key = s_list[tid];
                int place = 0;
#pragma unroll 4
                for (int i = 0; i < n; ++i)
                    place += s_list[i] > key;
                if (place < p.top_k)
                    s_top[place] = key;
            } else if (tid < p.top_k) {
                s_top[tid] = 0ull;
            }
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
                    s_top[k] = next;
            }
        }
        __syncthreads();
    };
    const auto id_of = [&](int bit) { return base + (bit >> 2) * kLogprobThreads * 4 + (bit & 3); };
    const auto list = [&](unsigned bits, int at) {
#pragma unroll 1
        for (; bits; bits &= bits - 1, ++at) {
            const int id = id_of(__ffs(bits) - 1);
            s_list[at] = order_key(__ldg(x + id), id);
        }
    };
    bool first_tile = true;
#pragma unroll 1
    for (;;) {
        const int next = base + TILE;
        float w4[V][4];
        const bool more = next - tid * 4 < end;
        if (more)
            load(w4, next);
        float mine = fmaxf(fmaxf(v[0][0], v[0][1]), fmaxf(v[0][2], v[0][3]));
#pragma unroll
        for (int j = 1; j < V; ++j)
            mine = fmaxf(fmaxf(mine, fmaxf(v[j][0], v[j][1])), fmaxf(v[j][2], v[j][3]));
        const float mn = fmaxf(m, mine), ms = mn == -INFINITY ? 0.0f : mn;
        float tr = 0.0f, te = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float border = base + j * kLogprobThreads * 4 + 3 < token ? below : xt;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float u = v[j][c] - ms, w = weight_up(u, p.inv_t);
                tr += w;
                te = fmaf(w, fmaxf(u, kLogprobLeast), te);
                before += v[j][c] > border;
            }
        }
        {  // the sums so far, relative to the new largest (at 0 before the first logit above -inf)
            const float u = fmaxf(m - ms, kLogprobLeast), w = weight_up(u, p.inv_t) * kLogprobDown;
            e = w > 0.0f ? fmaf(w, fmaf(u, r, e), te) : te;  // u * r is finite where w is not 0
            r = fmaf(w, r, tr);
            m = mn;
        }
        const int near = token - base;  // the token's place among the thread's: j * kLogprobThreads * 4 + c
        if (xt == -INFINITY || ((unsigned)near < (unsigned)TILE && (near & (kLogprobThreads * 4 - 1)) < 4)) {
            // nothing lies below -inf, and the four logits around the token have both kinds: counted one by one
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int i = base + j * kLogprobThreads * 4;
                const float border = i + 3 < token ? below : xt;
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    before += (v[j][c] > xt || (v[j][c] == xt && (unsigned)(i + c) < (unsigned)token)) - (v[j][c] > border);
            }
        }
        if (p.top_k > 0) {
            if (first_tile) {
                float group = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
                group = fmaxf(group, __shfl_xor_sync(0xffffffffu, group, 2));
                if ((tid & 3) == 0)
                    s_group[tid >> 2] = group;
                if (tid == 0)
                    s_above = s_count;
                __syncthreads();
                if (tid < kLogprobGroups) {
                    const float g = s_group[tid];
                    int place = 0;
#pragma unroll 8
                    for (int i = 0; i < kLogprobGroups; ++i)
                        place += s_group[i] > g || (s_group[i] == g && i < tid);
                    if (place == p.top_k - 1)
                        s_threshold = g;
                }
                __syncthreads();
                threshold = s_threshold;
            }
            unsigned reach = 0;  // bit 4 j + c
            if (first_tile ? mine >= threshold : mine > threshold) {
#pragma unroll
                for (int j = 0; j < V; ++j)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        reach |= (first_tile ? v[j][c] >= threshold : v[j][c] > threshold) ? 1u << (4 * j + c) : 0u;
                if (first_tile && threshold == -INFINITY) {  // keeps the row's ends out
#pragma unroll 1
                    for (int k = 0; k < 4 * V; ++k) {
                        const int id = id_of(k);
                        reach &= id >= 0 && id < p.vocab ? ~0u : ~(1u << k);
                    }
                }
            }
            const int at = reach ? atomicAdd(&s_count, __popc(reach)) : 0;
            bool cut;
            if (!first_tile) {
                list(reach, at);
                cut = __syncthreads_or(at + __popc(reach) > kLogprobKeep);
            } else {
                __syncthreads();
                if (s_count <= kLogprobKeep) {
                    list(reach, at);
                } else {  // masses at the threshold
                    unsigned equals = 0;
                    if (reach) {
#pragma unroll
                        for (int j = 0; j < V; ++j)
#pragma unroll
                            for (int c = 0; c < 4; ++c)
                                equals |= v[j][c] == threshold ? 1u << (4 * j + c) : 0u;
                        equals &= reach;
                    }
                    const unsigned above = reach & ~equals;
                    if (above)
                        list(above, atomicAdd(&s_above, __popc(above)));
                    __syncthreads();
                    const int n = s_above;  // less than top_k carried, and less than top_k groups of threads
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
                        int to = have + incl - __popc(bits);
#pragma unroll
                        for (int w = 0; w < WARPS; ++w) {
                            to += w < warp ? s_ties[w] : 0;
                            have += s_ties[w];
                        }
#pragma unroll 1
                        for (unsigned left = bits; left && to < p.top_k; left &= left - 1, ++to)
                            s_list[n + to] = order_key(threshold, id_of(__ffs(left) - 1));
                        __syncthreads();
                    }
                    if (tid == 0)
                        s_count = n + min(have, p.top_k);
                }
                __syncthreads();
                const int now = s_count;
                __syncthreads();  // everyone has read it before the next tile adds
                cut = now > kLogprobKeep;
                first_tile = now < p.top_k;  // a row's ends, or NaN: the next tile fills the list up
            }
            if (cut) {
                order(s_count);
                if (tid < p.top_k)
                    s_list[tid] = s_top[tid];
                if (tid == 0)
                    s_count = p.top_k;
                threshold = key_logit(s_top[p.top_k - 1]);
                __syncthreads();
            }
        }
        base = next;
        if (!more)
            break;
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                v[j][c] = w4[j][c];
    }

    // The block's sums: every thread's relative to the largest.
    float M = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if (lane == 0)
        s_m[warp] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
        M = fmaxf(M, s_m[w]);
    {
        const float u = fmaxf(m - (M == -INFINITY ? 0.0f : M), kLogprobLeast), w = weight_up(u, p.inv_t) * kLogprobDown;
        e = w > 0.0f ? fmaf(u, r, e) * w : 0.0f;
        r *= w;
    }
    float mine_r = r;
    r = warp_sum(r);
    e = warp_sum(e);
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0)
        s_r[warp] = r, s_e[warp] = e, s_before[warp] = before;
    __syncthreads();
    LogprobPiece sum{M, 0.0f, 0.0f, 0};
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
        sum.r += s_r[w], sum.e += s_e[w], sum.before += s_before[w];
    sum.r *= kLogprobDown;
    sum.e *= kLogprobDown;
    if (M > -INFINITY) {
        if (sum.r < 1.25f) {
            // Little beside the largest: its 1 has rounded the sum. The threads that hold a largest sum again,
            // without them.
            int equal = 0;
            if (m == M) {
                mine_r = 0.0f;
#pragma unroll 1
                for (int at = first + tid * 4; at - tid * 4 < end; at += TILE) {
                    load(v, at);
#pragma unroll
                    for (int j = 0; j < V; ++j)
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            mine_r += v[j][c] == M ? 0.0f : weight_up(v[j][c] - M, p.inv_t);
                            equal += v[j][c] == M;
                        }
                }
            }
            mine_r = warp_sum(mine_r);
            equal = __reduce_add_sync(0xffffffffu, equal);
            __syncthreads();
            if (lane == 0)
                s_r[warp] = mine_r, s_equal[warp] = equal;
            __syncthreads();
            sum.r = 0.0f;
            equal = 0;
#pragma unroll
            for (int w = 0; w < WARPS; ++w)
                sum.r += s_r[w], equal += s_equal[w];
            sum.r = fmaf(sum.r, kLogprobDown, (float)(equal - 1));
        } else {
            sum.r -= 1.0f;
        }
    }
    if (p.top_k > 0)
        order(s_count);
    if (p.pieces == 1) {
        const LogprobRow done(p, sum);
        if (tid == 0)
            done.write(p, out, sum, row, token, xt);
        if (tid < p.top_k)
            done.write_top(out, (size_t)row * p.top_k + tid, s_top[tid]);
        return;
    }
    if (tid == 0)
        stats[blockIdx.x] = sum;
    if (tid < p.top_k)
        tops[(size_t)blockIdx.x * p.top_k + tid] = s_top[tid];
}

// Joins a row's pieces: one CTA per row, a piece per thread at a time.
__global__ void __launch_bounds__(kLogprobJoinThreads) k_logprob_join(LogprobDev p, const float* __restrict__ logits,
                                                                      const int32_t* __restrict__ tokens,
                                                                      const LogprobPiece* __restrict__ stats,
                                                                      const unsigned long long* __restrict__ tops,
                                                                      LogprobOut out)
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
    const float xt = token >= 0 && token < p.vocab ? __ldg(logits + row * p.stride + token) : 0.0f;
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
        const float u = fmaxf(q.m - ms, kLogprobLeast), w = weight_up(u, p.inv_t);
        r += top ? q.r : (1.0f + q.r) * w * kLogprobDown;
        equal += top;
        e += top ? q.e : fmaf(u, 1.0f + q.r, q.e) * w * kLogprobDown;
        before += q.before;
    }
    r = warp_sum(r);
    e = warp_sum(e);
    before = __reduce_add_sync(0xffffffffu, before);
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0)
        s_r[warp] = r, s_e[warp] = e, s_before[warp] = before, s_equal[warp] = equal;
    __syncthreads();
    LogprobPiece sum{m, 0.0f, 0.0f, 0};
    equal = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
        sum.r += s_r[w], sum.e += s_e[w], sum.before += s_before[w], equal += s_equal[w];
    sum.r += (float)(equal - 1);
    const LogprobRow done(p, sum);
    if (tid == 0)
        done.write(p, out, sum, row, token, xt);
    if (p.top_k == 0)
        return;
    // The pieces' lists, each in order: the largest head top_k times.
    if (p.pieces <= 32) {  // one warp: a list per lane, its next key at hand
        if (warp > 0)
            return;
        const unsigned long long* list = tops + ((size_t)row * p.pieces + min(lane, p.pieces - 1)) * p.top_k;
        unsigned long long head = lane < p.pieces ? list[0] : 0ull, mine_out = 0ull;
        unsigned long long next = lane < p.pieces && p.top_k > 1 ? list[1] : 0ull;
        int at = 2;
#pragma unroll 1
        for (int k = 0; k < p.top_k; ++k) {
            const unsigned long long best = warp_max_key(head);
            mine_out = k == lane ? best : mine_out;
            if (head == best && best != 0ull) {  // keys differ: one lane
                head = next;
                next = at < p.top_k ? list[at] : 0ull;
                ++at;
            }
        }
        if (lane < p.top_k)
            done.write_top(out, (size_t)row * p.top_k + lane, mine_out);
        return;
    }
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
        if (tid == 0)
            done.write_top(out, (size_t)row * p.top_k + k, best);
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
    MUYO_REQUIRE(p->temperature >= 1e-6f && p->temperature <= 1e6f, "token_logprobs: temperature must be in [1e-6, 1e6]");
    d.rows = (int)p->rows, d.vocab = (int)p->vocab, d.top_k = (int)p->top_k;
    d.stride = p->stride ? p->stride : p->vocab;
    d.temperature = p->temperature;
    d.inv_t = (float)(1.4426950408889634 / (double)p->temperature);
    // Tiles of 4096 logits, of 2048 where the larger ones would leave SMs without a CTA; four CTAs on an SM at once, so a
    // row is cut into the pieces that fill them. A row may begin 3 logits behind a 16-byte border.
    const long long large = (d.vocab + 3LL + 4095) / 4096, room = 4LL * sm_count();
    d.small = large * d.rows < sm_count();
    const long long tiles = d.small ? (d.vocab + 3LL + 2047) / 2048 : large;
    const long long cut = room / d.rows < 1 ? 1 : room / d.rows < tiles ? room / d.rows : tiles;
    const long long each = (tiles + cut - 1) / cut;
    d.tiles = (int)(each < kLogprobMaxTiles ? each : kLogprobMaxTiles);
    d.pieces = (int)((tiles + d.tiles - 1) / d.tiles);
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
    const LogprobOut o{logprob, entropy, rank, top_ids, top_logprobs};
    const size_t smem = d.top_k ? (kLogprobKeep + (d.small ? 2048 : 4096)) * sizeof(unsigned long long) : 0;
    MUYO_CUDA_TRY(launch_kernel(d.small ? k_logprob_pieces<2> : k_logprob_pieces<4>, dim3(d.rows * d.pieces),
                                dim3(kLogprobThreads), smem, as_stream(stream), true, d, logits, tokens, stats, tops, o));
    MUYO_LAUNCH_CHECK();
    if (d.pieces > 1) {
        MUYO_CUDA_TRY(launch_kernel(k_logprob_join, dim3(d.rows), dim3(kLogprobJoinThreads), 0, as_stream(stream), true, d,
                                    logits, tokens, stats, tops, o));
        MUYO_LAUNCH_CHECK();
    }
    return MUYO_OK;
}
