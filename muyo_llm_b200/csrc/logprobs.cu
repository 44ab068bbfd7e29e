// Log probabilities of given tokens with entropy, rank and the top alternatives.
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace muyo {

// With alternatives a thread's part of a row is what is read again, and fewer threads would have longer ones; without,
// more and smaller CTAs on an SM begin and end beside the others' loops (2001 rows of 32001: 53.1 us, with 256 threads 56.8 us).
template <bool TOP>
constexpr int kLogprobThreads = TOP ? 256 : 128;
constexpr int kLogprobJoinThreads = 128;
constexpr int kLogprobMaxTop = 32;
constexpr int kLogprobGroups = 64;  // groups of 4 threads whose maxima give the threshold
constexpr int kLogprobList = 512;   // listed logits
constexpr int kLogprobMaxTiles = 64;  // of a piece
constexpr int kLogprobCluster = 8;

struct LogprobDev {
    int rows, vocab, top_k;
    long long stride;
    float inv_t;  // log2(e) / temperature
    float temperature;
    int pieces, tiles;  // of a row; of a piece
    bool small;         // tiles of two float4 per thread instead of four
    bool cluster;       // a row's pieces are one thread-block cluster, which joins them itself
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

// exp(u / T) is 0 from 2^-126 on. Where that could be missed, 2^64 times as large: near u = 0 the added 64 would round the
// exponent by 2^-18, so only where no weight is near 1, or where u is far.
constexpr float kLogprobDown = 5.421010862427522e-20f;  // 2^-64
__device__ __forceinline__ float weight_up(float u, float inv_t)
{
    return ex2(fmaf(u, inv_t, 64.0f));
}
// a exp(u / T), also where exp(u / T) alone would be 0
__device__ __forceinline__ float weighed(float a, float u, float inv_t)
{
    const float x = u * inv_t;
    const bool far = x < -64.0f;
    return a * ex2(far ? x + 64.0f : x) * (far ? kLogprobDown : 1.0f);
}
constexpr float kLogprobFew = 8.271806125530277e-25f;  // 2^-80
constexpr float kLogprobLeast = -1.0e29f;  // u where the weight is 0, so that 0 * -inf does not arise

// Four logits, which are read once: no L1 allocation. Not by the read-only path: an earlier kernel of the stream, whose
// end this one waits for, may have written them after this one began.
__device__ __forceinline__ float4 ld_logits(const float* p)
{
    float4 r;
    asm volatile("ld.global.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(r.x), "=f"(r.y), "=f"(r.z), "=f"(r.w)
                 : "l"(p)
                 : "memory");
    return r;
}

// The ids below `end` from `begin` on at which x is `value`, in order, by one warp: lanes have .. top_k - 1 receive them
// (-1 without one).
__device__ __forceinline__ int logprob_equal_ids(const float* x, float value, int begin, int end, int have, int top_k)
{
    const int lane = threadIdx.x & 31;
    int id = -1;
#pragma unroll 1
    for (int i = begin; have < top_k && i < end; i += 32) {
        const unsigned equal = __ballot_sync(0xffffffffu, i + lane < end && x[min(i + lane, end - 1)] == value);
        if (lane >= have && lane < top_k && lane - have < __popc(equal)) {
            unsigned bits = equal;
#pragma unroll 1
            for (int k = have; k < lane; ++k)
                bits &= bits - 1;
            id = i + __ffs(bits) - 1;
        }
        have = min(have + __popc(equal), top_k);
    }
    return id;
}

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
        if (nothing)
            return -INFINITY;
        const float d = x - m;
        // two finite logits may lie further apart than F32 reaches, and their difference by the temperature does not
        return (d == -INFINITY ? 2.0f * __fdiv_rn(0.5f * x - 0.5f * m, temperature) : __fdiv_rn(d, temperature)) - log_sum;
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
    // The first top_k ids by one warp, lane k the k-th; key 0 where no logit above -inf is left. Those places go to the
    // lowest ids at -inf, read from the row x; -1 where there are none (NaN).
    __device__ __forceinline__ void write_top(const LogprobDev& p, const LogprobOut& out, int row, unsigned long long key,
                                              const float* x) const
    {
        const int lane = threadIdx.x & 31;
        const int have = __popc(__ballot_sync(0xffffffffu, key != 0ull && lane < p.top_k));
        int id = key ? (int)~(unsigned)key : -1;
        float v = key ? key_logit(key) : NAN;
        const int masked = logprob_equal_ids(x, -INFINITY, 0, p.vocab, have, p.top_k);
        if (masked >= 0) {
            id = masked;
            v = -INFINITY;
        }
        if (lane < p.top_k) {
            out.top_ids[(size_t)row * p.top_k + lane] = id;
            out.top_logprobs[(size_t)row * p.top_k + lane] = log_p(v);
        }
    }
};

// Joins the sums of up to 32 pieces, by one warp: lane i has piece i's.
__device__ __forceinline__ LogprobPiece logprob_join_sums(const LogprobDev& p, LogprobPiece q, int pieces)
{
    const bool here = (int)(threadIdx.x & 31) < pieces;
    if (!here)
        q = LogprobPiece{-INFINITY, 0.0f, 0.0f, 0};
    const float m = warp_max(q.m), ms = m == -INFINITY ? 0.0f : m;
    const bool top = here && q.m == m;
    const float u = fmaxf(q.m - ms, kLogprobLeast);
    LogprobPiece sum{m, 0.0f, 0.0f, 0};
    sum.r = warp_sum(top ? q.r : here ? weighed(1.0f + q.r, u, p.inv_t) : 0.0f) + (float)(__popc(__ballot_sync(0xffffffffu, top)) - 1);
    sum.e = warp_sum(top ? q.e : here ? weighed(fmaf(u, 1.0f + q.r, q.e), u, p.inv_t) : 0.0f);
    sum.before = __reduce_add_sync(0xffffffffu, q.before);
    return sum;
}

// One piece of a row: tiles of V float4 per thread, two tiles' loads under way, no barrier. A thread keeps its largest
// logit so far, its sums of w and w (x - m) relative to it, and its count of ids in front of the token (looked
// at where a tile's largest is not below the token's logit). Where little lies beside the largest, its 1 has
// rounded the sum: then the sum is formed again without it, from a second read of its thread's logits; and where it is
// below 2^-80, sums and moments from a second read of all, with weights that do not end at 2^-126.
//
// The first top_k ids: the threads' maxima, taken over 64 groups of 4 threads, give a threshold, the top_k-th
// largest of them, that top_k logits reach and few others do (24 on average for 20 of 64). A warp
// reads the logits of one such thread at a time again, a float4 per lane; those that reach the threshold
// are ordered by counting. -inf is never listed, its places are filled in at the end. Masses at the threshold (a
// constant row, a mask of the lowest value) run the list over: then what lies above it is listed, and of the equal
// ones the lowest ids.
//
// Bound by the read, 4 bytes a logit: 2001 rows of 32001, 256 MB, take 51 us (5.0 TB/s, 0.76 of the copy rate; a CTA's
// first loads and its last sums are a third of its time, the count for the rank 2 us and the entropy's sum 3 us of the
// call), 97 rows of 151936 with 20 alternatives, 59 MB, 23.0 us (the
// loop ends at 40% of the kernel's time, the rest is the second reads and the cluster's join), one row 8.8 us. Listing
// tile by tile in the loop took 40 us for the 97 rows, whole pieces in shared memory 59 us.
//
// Slower contents, all exact: more than 512 logits of a piece above the threshold (whole tiles that rise by steps) take
// top_k passes over the piece, 97 rows 0.55 ms and 2001 rows 2.2 ms; constant rows 0.1 and 0.4 ms; a row with
// fewer than top_k logits that are not NaN is searched for masked ones by one warp, 1.5 ms for a row of 151936 and 2.5 ms for
// 97. Rows of almost certain tokens (the others' sum below 2^-80) take 2 to 4 us more.
template <bool TOP, int V>
__global__ void __launch_bounds__(kLogprobThreads<TOP>, 1024 / kLogprobThreads<TOP>)
                                                      k_logprob_pieces(LogprobDev p, const float* logits,
                                                                       const int32_t* tokens,
                                                                       LogprobPiece* stats,
                                                                       unsigned long long* tops, LogprobOut out)
{
    constexpr int THREADS = kLogprobThreads<TOP>, WARPS = THREADS / 32, Q = THREADS * 4, TILE = V * Q;
    __shared__ float s_m[WARPS], s_r[WARPS], s_e[WARPS], s_mine[TOP ? THREADS : 1], s_threshold;
    __shared__ int s_before[WARPS], s_count, s_threads, s_thread[TOP ? THREADS : 1];
    __shared__ unsigned long long s_key[WARPS], s_top[kLogprobMaxTop], s_list[TOP ? kLogprobList : 1];
    __shared__ LogprobPiece s_sum;
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / p.pieces, piece = blockIdx.x - row * p.pieces;
    const float* x = logits + row * p.stride;
    const int token = tokens[row];
    // float4 from the 16-byte border at or before the row's first logit; ids outside [begin, end) read as -inf
    const int origin = piece * p.tiles * TILE - (int)((reinterpret_cast<uintptr_t>(x) >> 2) & 3);
    const int begin = max(origin, 0), end = max(begin, min(origin + p.tiles * TILE, p.vocab));  // the last may be empty
    const int tiles = (end - origin + TILE - 1) / TILE;
    const auto quad = [&](int i) {
        if (i >= 0 && i <= p.vocab - 4)
            return ld_logits(x + i);
        float4 f = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
            const float y = i + c >= 0 && i + c < p.vocab ? x[i + c] : -INFINITY;
            f.x = c == 0 ? y : f.x, f.y = c == 1 ? y : f.y, f.z = c == 2 ? y : f.z, f.w = c == 3 ? y : f.w;
        }
        return f;
    };
    const auto load = [&](float4 (&v)[V], int tile) {
        const int i = origin + tile * TILE + tid * 4;
        if (i - tid * 4 >= 0 && i - tid * 4 + TILE <= p.vocab) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                v[j] = ld_logits(x + i + j * Q);
        } else {
#pragma unroll 1
            for (int j = 0; j < V; ++j) {
                const float4 f = quad(i + j * Q);
#pragma unroll
                for (int n = 0; n < V; ++n)
                    v[n] = j == n ? f : v[n];
            }
        }
    };
    float4 va[V], vb[V];
    load(va, 0);
    const float xt = token >= 0 && token < p.vocab ? x[token] : INFINITY;  // outside: nothing in front
    // An id below the token is in front of it at an equal logit too: it is compared with the next value below. Below -inf
    // there is none: of a masked token, all ids below it are in front (added after the loop) and those above it that are
    // not masked. The four logits around the token have both kinds: put right after the loop.
    const float below = xt == -INFINITY ? INFINITY : nextafterf(xt, -INFINITY);
    float m = -INFINITY, r = 0.0f, e = 0.0f;
    float front = 0.0f;  // ids in front of the token: exact, a thread has 1024 logits of a piece at most
    if (tid == 0)
        s_count = s_threads = 0;
    const auto work = [&](const float4 (&v)[V], int tile) {
        float mine = fmaxf(fmaxf(v[0].x, v[0].y), fmaxf(v[0].z, v[0].w));
#pragma unroll
        for (int j = 1; j < V; ++j)
            mine = fmaxf(fmaxf(mine, fmaxf(v[j].x, v[j].y)), fmaxf(v[j].z, v[j].w));
        const float mn = fmaxf(m, mine), ms = mn == -INFINITY ? 0.0f : mn;
        const float2 scale = make_float2(p.inv_t, p.inv_t), back = make_float2(-ms, -ms), zero = make_float2(0.0f, 0.0f);
        float2 sum = zero, moment = zero;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float2 u0 = add2(make_float2(v[j].x, v[j].y), back), u1 = add2(make_float2(v[j].z, v[j].w), back);
            const float2 x0 = fma2(u0, scale, zero), x1 = fma2(u1, scale, zero);
            const float2 w0 = make_float2(ex2(x0.x), ex2(x0.y)), w1 = make_float2(ex2(x1.x), ex2(x1.y));
            sum = add2(sum, add2(w0, w1));
            moment = fma2(w0, make_float2(fmaxf(u0.x, kLogprobLeast), fmaxf(u0.y, kLogprobLeast)), moment);
            moment = fma2(w1, make_float2(fmaxf(u1.x, kLogprobLeast), fmaxf(u1.y, kLogprobLeast)), moment);
        }
        const float tr = sum.x + sum.y, te = moment.x + moment.y;
        // the sums so far, relative to the new largest (at 0 before the first logit above -inf)
        const float u = fmaxf(m - ms, kLogprobLeast), w = ex2(u * p.inv_t);
        e = w > 0.0f ? fmaf(w, fmaf(u, r, e), te) : te;  // u * r is finite where w is not 0
        r = fmaf(w, r, tr);
        m = mn;
        if (mine >= xt) {
            const int i = origin + tile * TILE + tid * 4;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float border = i + j * Q + 3 < token ? below : xt;
                front += ((v[j].x > border ? 1.0f : 0.0f) + (v[j].y > border ? 1.0f : 0.0f)) +
                         ((v[j].z > border ? 1.0f : 0.0f) + (v[j].w > border ? 1.0f : 0.0f));
            }
        }
    };
#pragma unroll 1
    for (int tile = 0; tile < tiles; tile += 2) {
        if (tile + 1 < tiles)
            load(vb, tile + 1);
        work(va, tile);
        if (tile + 1 < tiles) {
            if (tile + 2 < tiles)
                load(va, tile + 2);
            work(vb, tile + 1);
        }
    }
    int before = (int)front;
    if (tid == 0) {
        if (token >= begin && token < end) {
#pragma unroll 1
            for (int i = max(token - ((token - origin) & 3), 0); i < token; ++i)
                before += xt == -INFINITY ? -(x[i] > xt) : x[i] == xt;
        }
        if (xt == -INFINITY)
            before += min(max(token - begin, 0), end - begin);
    }

    // The block's sums: every thread's relative to the largest.
    float M = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if (lane == 0)
        s_m[warp] = M;
    if (TOP)
        s_mine[tid] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
        M = fmaxf(M, s_m[w]);
    {
        const float u = fmaxf(m - (M == -INFINITY ? 0.0f : M), kLogprobLeast), w = ex2(u * p.inv_t);
        e = w > 0.0f ? fmaf(u, r, e) * w : 0.0f;
        r *= w;
    }
    const float own = r;
    r = warp_sum(r);
    e = warp_sum(e);
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0)
        s_r[warp] = r, s_e[warp] = e, s_before[warp] = before;
    if (TOP) {
        // a thread's group of 4, a quarter of the groups each
        const int mine = tid >> 2;
        const auto group = [&](int g) {
            return fmaxf(fmaxf(s_mine[4 * g], s_mine[4 * g + 1]), fmaxf(s_mine[4 * g + 2], s_mine[4 * g + 3]));
        };
        const float g = group(mine);
        int place = 0;
#pragma unroll 4
        for (int k = 0; k < kLogprobGroups / 4; ++k) {
            const int i = (tid & 3) + 4 * k;
            const float h = group(i);
            place += h > g || (h == g && i < mine);
        }
        place += __shfl_xor_sync(0xffffffffu, place, 1);
        place += __shfl_xor_sync(0xffffffffu, place, 2);
        if ((tid & 3) == 0 && place == p.top_k - 1)
            s_threshold = g;
    }
    __syncthreads();
    LogprobPiece sum{M, 0.0f, 0.0f, 0};
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
        sum.r += s_r[w], sum.e += s_e[w], sum.before += s_before[w];
    if (M == -INFINITY) {
        sum.r = sum.r == sum.r ? 0.0f : NAN;
        sum.e = 0.0f;
    } else if (sum.r < 1.25f) {
        // one logit is the largest, or the sum would be 2 or more: its thread's logits again, a float4 per lane
        const unsigned holder = __ballot_sync(0xffffffffu, m == M);
        float next = m == M ? -INFINITY : m;  // the largest of the others
        __syncthreads();
        if (holder) {
            const int from = __ffs(holder) - 1, i0 = origin + (warp * 32 + from) * 4;
            float rest = lane == from ? 0.0f : own;
            const auto add = [&](float y) {
                rest += y == M ? 0.0f : ex2((y - M) * p.inv_t);
                next = fmaxf(next, y == M ? -INFINITY : y);
            };
#pragma unroll 1
            for (int q = lane; q < V * tiles; q += 32) {
                const float4 f = quad(i0 + q / V * TILE + q % V * Q);
                add(f.x), add(f.y), add(f.z), add(f.w);
            }
            rest = warp_sum(rest);
            if (lane == 0)
                s_r[warp] = rest;
        }
        const bool more = __syncthreads_or(weight_up(next - M, p.inv_t) > 0.0f);
        sum.r = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w)
            sum.r += s_r[w];
        if (sum.r < kLogprobFew && more) {
            // The others' weights are all far below 1, and some have come out as 0 (less than 2^-107 together, which a
            // larger sum does not miss): every thread's logits again.
            r = e = 0.0f;
            const auto add = [&](float y) {
                const float u = y == M ? -INFINITY : y - M, w = weight_up(u, p.inv_t);
                r += w;
                e = fmaf(w, fmaxf(u, kLogprobLeast), e);
            };
#pragma unroll 1
            for (int q = 0; q < V * tiles; ++q) {
                const float4 f = quad(origin + q / V * TILE + q % V * Q + tid * 4);
                add(f.x), add(f.y), add(f.z), add(f.w);
            }
            r = warp_sum(r);
            e = warp_sum(e);
            __syncthreads();  // s_r is read
            if (lane == 0)
                s_r[warp] = r, s_e[warp] = e;
            __syncthreads();
            sum.r = sum.e = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w)
                sum.r += s_r[w], sum.e += s_e[w];
            sum.r *= kLogprobDown;
            sum.e *= kLogprobDown;
        }
    } else {
        sum.r -= 1.0f;
    }
    // The keys of s_list[0, n) in order: the first top_k into s_top, 0 behind them. A key's place is the number of
    // larger ones.
    const auto order = [&](int n) {
        if (tid < p.top_k)
            s_top[tid] = 0ull;
        __syncthreads();
#pragma unroll 1
        for (int k = tid; k < n; k += THREADS) {
            const unsigned long long key = s_list[k];
            int place = 0;
#pragma unroll 8
            for (int i = 0; i < n; ++i)
                place += s_list[i] > key;
            if (place < p.top_k && key)
                s_top[place] = key;
        }
        __syncthreads();
    };
    if (TOP) {
        const float threshold = s_threshold;
        const bool masked = threshold == -INFINITY;  // then every logit above it is listed
        if (masked ? m > threshold : m >= threshold)
            s_thread[atomicAdd(&s_threads, 1)] = tid;
        __syncthreads();
        // Lists the logits of the threads at hand that reach the threshold, or lie above it.
        const auto list = [&](bool above) {
            // a warp reads four threads' logits at once, a float4 of each per lane
            const int threads = s_threads;
#pragma unroll 1
            for (int k0 = warp; k0 < threads; k0 += 4 * WARPS)
#pragma unroll 1
                for (int q = lane; q < V * tiles; q += 32) {
                    float4 f[4];
                    int id[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        f[u].x = f[u].y = f[u].z = f[u].w = -INFINITY;
                        if (k0 + u * WARPS < threads) {
                            id[u] = origin + q / V * TILE + q % V * Q + s_thread[k0 + u * WARPS] * 4;
                            f[u] = quad(id[u]);
                        }
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const float most = fmaxf(fmaxf(f[u].x, f[u].y), fmaxf(f[u].z, f[u].w));
                        if (k0 + u * WARPS >= threads || (above ? most <= threshold : most < threshold))
                            continue;
#pragma unroll 1
                        for (int c = 0; c < 4; ++c) {
                            const float y = c == 0 ? f[u].x : c == 1 ? f[u].y : c == 2 ? f[u].z : f[u].w;
                            if (above ? y > threshold : y >= threshold) {
                                const int at = atomicAdd(&s_count, 1);
                                if (at < kLogprobList)
                                    s_list[at] = order_key(y, id[u] + c);
                            }
                        }
                    }
                }
        };
        list(masked);
        __syncthreads();
        int n = s_count;
        if (n > kLogprobList && !masked) {
            __syncthreads();
            if (tid == 0)
                s_count = 0;
            __syncthreads();
            list(true);
            if (warp == 0)
                s_top[lane] = 0ull;
            __syncthreads();
            n = s_count;
            if (n + kLogprobMaxTop <= kLogprobList) {
                if (warp == 0) {
                    const int id = logprob_equal_ids(x, threshold, begin, end, 0, p.top_k);
                    s_list[n + lane] = id >= 0 ? order_key(threshold, id) : 0ull;
                }
                __syncthreads();
                n += kLogprobMaxTop;
            }
        }
        if (n <= kLogprobList) {
            order(n);
        } else {  // rows of many logits above it after all: one by one
            unsigned long long last = ~0ull;
#pragma unroll 1
            for (int k = 0; k < p.top_k; ++k) {
                unsigned long long next = 0ull;
#pragma unroll 4
                for (int i = begin + tid; i < end; i += THREADS) {
                    const float y = x[i];
                    const unsigned long long key = y > -INFINITY ? order_key(y, i) : 0ull;
                    next = key < last && key > next ? key : next;
                }
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
            __syncthreads();
        }
    }
    if (p.pieces > 1) {
        if (!p.cluster) {
            if (tid == 0)
                stats[blockIdx.x] = sum;
            if (TOP && tid < p.top_k)
                tops[(size_t)blockIdx.x * p.top_k + tid] = s_top[tid];
            return;
        }
        cg::cluster_group cluster = cg::this_cluster();
        if (tid == 0)
            s_sum = sum;
        cluster.sync();
        if (piece == 0) {
            if (TOP && tid < p.pieces * p.top_k)  // at most 256 keys
                s_list[tid] = cluster.map_shared_rank(s_top, tid / p.top_k)[tid % p.top_k];
            if (warp == 0)
                sum = logprob_join_sums(
                    p, *cluster.map_shared_rank(&s_sum, min((unsigned)lane, (unsigned)p.pieces - 1)), p.pieces);
        }
        cluster.sync();  // the others' shared memory is read
        if (piece > 0)
            return;
        if (TOP)
            order(p.pieces * p.top_k);
    }
    if (warp == 0) {
        const LogprobRow done(p, sum);
        if (lane == 0)
            done.write(p, out, sum, row, token, xt);
        if (TOP)
            done.write_top(p, out, row, lane < p.top_k ? s_top[lane] : 0ull, x);
    }
}

// Joins a row's pieces where they are more than a cluster: one CTA per row, a piece per thread at a time.
__global__ void __launch_bounds__(kLogprobJoinThreads) k_logprob_join(LogprobDev p, const float* logits,
                                                                      const int32_t* tokens,
                                                                      const LogprobPiece* stats,
                                                                      const unsigned long long* tops,
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
    const float xt = token >= 0 && token < p.vocab ? logits[row * p.stride + token] : 0.0f;
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
        const float u = fmaxf(q.m - ms, kLogprobLeast);
        r += top ? q.r : weighed(1.0f + q.r, u, p.inv_t);
        equal += top;
        e += top ? q.e : weighed(fmaf(u, 1.0f + q.r, q.e), u, p.inv_t);
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
    const unsigned long long* list = tops + (size_t)row * p.pieces * p.top_k;
    int at = 0;  // of the thread's first list
    unsigned long long last = ~0ull, head = tid < p.pieces ? list[(size_t)tid * p.top_k] : 0ull, mine_out = 0ull;
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
        mine_out = tid == k ? best : mine_out;
    }
    if (warp == 0)
        done.write_top(p, out, row, mine_out, logits + row * p.stride);
}

}  // namespace muyo

using namespace muyo;

static int logprob_threads(const LogprobDev& d) { return d.top_k > 0 ? kLogprobThreads<true> : kLogprobThreads<false>; }

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
    // A row is cut into the pieces that come nearest to three CTAs on an SM (97 rows of 151936 with 20 alternatives: 5
    // pieces 23.5 us, 6 pieces 30 us, the ends of more pieces cost more than their loops gain; 150 rows: 2 pieces 44
    // us, 3 pieces 34 us), and not into more than a cluster joins where those are a CTA per SM (40 rows: 8 pieces 20
    // us, 14 pieces and a second kernel 22 us; one row: 8 pieces 13 us, 75 pieces 8 us); of the smaller CTAs, as many as
    // fill the same threads. A row may begin 3 logits behind a 16-byte border.
    const int threads = logprob_threads(d), per_sm = 768 / threads;
    const long long large = (d.vocab + 3LL + 16 * threads - 1) / (16 * threads);
    d.small = large * d.rows < sm_count();  // the larger tiles would leave SMs without a CTA
    const long long tiles = d.small ? (d.vocab + 3LL + 8 * threads - 1) / (8 * threads) : large;
    long long cut = std::max(1LL, std::min(((long long)per_sm * sm_count() + d.rows / 2) / d.rows, tiles));
    if (cut > kLogprobCluster && d.rows * (long long)kLogprobCluster >= sm_count())
        cut = kLogprobCluster;
    const long long each = std::min((tiles + cut - 1) / cut, (long long)kLogprobMaxTiles);
    d.tiles = (int)each;
    d.pieces = (int)((tiles + each - 1) / each);
    d.cluster = d.pieces > 1 && d.pieces <= kLogprobCluster;
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
    const auto kernel = d.small ? (d.top_k > 0 ? k_logprob_pieces<true, 2> : k_logprob_pieces<false, 2>)
                                : (d.top_k > 0 ? k_logprob_pieces<true, 4> : k_logprob_pieces<false, 4>);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(d.rows * d.pieces);
    cfg.blockDim = dim3(logprob_threads(d));
    cfg.stream = as_stream(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)d.pieces;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = d.cluster ? 2 : 1;
    MUYO_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, d, logits, tokens, stats, tops, o));
    MUYO_LAUNCH_CHECK();
    if (d.pieces > 1 && !d.cluster) {
        MUYO_CUDA_TRY(launch_kernel(k_logprob_join, dim3(d.rows), dim3(kLogprobJoinThreads), 0, as_stream(stream), true, d,
                                    logits, tokens, stats, tops, o));
        MUYO_LAUNCH_CHECK();
    }
    return MUYO_OK;
}
