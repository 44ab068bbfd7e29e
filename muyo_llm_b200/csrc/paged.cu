// The bookkeeping and the append of a paged key-value cache: block tables and slot maps from request
// lengths, and rotary positions fused with the store of keys and values into their slots.
#include <cooperative_groups.h>

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace muyo {

// ---- plan ------------------------------------------------------------------------------------------
// need_i = ceil((c_i + a_i) / P) - ceil(c_i / P) pages for a request that holds c_i tokens and asks for
// a_i; with stop_i and upto_i the inclusive sums of the asked tokens and of the needed pages, request i
// is admitted iff upto_i <= free pages and stop_i <= max_tokens (with MUYO_PLAN_ROOM, also iff need_i = 0 and
// stop_i <= max_tokens). Both sums are monotone, so the pages of
// the admitted requests are a contiguous run from the ring's head, and every token and every page
// finds its request by a binary search in the sums: all outputs are written in parallel from shared
// memory, whatever the mix of long prompts and single tokens. A cluster of 8 CTAs shares that work; each forms
// the sums for itself, and nothing is written before all have read what a step in place overwrites. Latency bound
// (the sums, a binary search and a page look-up per token): 1501 requests with 48000 new tokens take 12.1 us, with one CTA
// and divisions for pages and ring places 69 us; 250 single tokens 4.9 to 5.6 us, which is the call's own cost.
// Not separated by measurement: the sums, which every CTA forms in full, the barrier, and the tokens' searches.
constexpr int kPlanThreads = 1024;
constexpr int kPlanCtas = 8;
constexpr int kPlanMaxSeqs = 8192;
constexpr unsigned kPlanAdmitted = 0x80000000u, kPlanHeld = 0x7fffffffu;  // a row holds 2^30 tokens at most

struct PlanDev {
    int seqs, page_size, num_pages, table_stride, max_tokens;
    int page_shift;  // log2(page_size), or -1
    bool room;       // MUYO_PLAN_ROOM
};

struct PlanSums {
    long long tokens, pages, ended;
};

__device__ __forceinline__ PlanSums plan_add(PlanSums a, PlanSums b)
{
    return {a.tokens + b.tokens, a.pages + b.pages, a.ended + b.ended};
}

__device__ __forceinline__ PlanSums plan_shfl_up(PlanSums a, int o)
{
    return {__shfl_up_sync(0xffffffffu, a.tokens, o), __shfl_up_sync(0xffffffffu, a.pages, o),
            __shfl_up_sync(0xffffffffu, a.ended, o)};
}

__device__ __forceinline__ int saturated(long long v) { return v > INT_MAX ? INT_MAX : (int)v; }

// First i with sums[i] > x (sums ascending); n if none.
__device__ __forceinline__ int first_above(const int* sums, int n, int x)
{
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] > x)
            hi = mid;
        else
            lo = mid + 1;
    }
    return lo;
}

// Entry `by` places behind entry `from` of a ring of n (from < n, by <= n).
__device__ __forceinline__ int ring_index(int from, int by, int n)
{
    const unsigned r = (unsigned)from + (unsigned)by;
    return (int)(r < (unsigned)n ? r : r - (unsigned)n);
}

__device__ __forceinline__ int page_of(const PlanDev& p, int slot)
{
    return p.page_shift >= 0 ? slot >> p.page_shift : slot / p.page_size;
}

__global__ void __cluster_dims__(kPlanCtas, 1, 1) __launch_bounds__(kPlanThreads)
                                                k_paged_plan(PlanDev p, const int32_t* cached_lens, const int32_t* new_lens,
                                                             int32_t* table, int32_t* ring, const int64_t* state,
                                                             int32_t* seq_lens, int32_t* query_start, int32_t* positions,
                                                             int32_t* slots, int64_t* state_out)
{
    extern __shared__ int plan_smem[];
    int* stop = plan_smem;          // [seqs] tokens asked for up to and with this request
    int* upto = stop + p.seqs;      // [seqs] pages needed
    int* gone = upto + p.seqs;      // [seqs] pages of ended requests
    // [seqs] kPlanAdmitted and the tokens held before, else the tokens held after the step
    unsigned* held = reinterpret_cast<unsigned*>(gone + p.seqs);
    __shared__ PlanSums warp_sums[32];
    __shared__ int s_taken, s_refused;
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = blockIdx.x, all = rank * kPlanThreads + tid;  // of the cluster's threads
    if (tid == 0)
        s_taken = s_refused = 0;
    const long long head = state[0], tail = state[1];
    const long long span = tail - head;
    const int free_pages = span < 0 || span > p.num_pages ? (span < 0 ? 0 : p.num_pages) : (int)span;
    const int row_slots = p.table_stride * p.page_size;
    // Each thread sums its contiguous requests, the block scans the threads' sums.
    const int per = (p.seqs + kPlanThreads - 1) / kPlanThreads;
    const int i0 = min(tid * per, p.seqs), i1 = min(i0 + per, p.seqs);
    PlanSums mine{0, 0, 0};
    for (int i = i0; i < i1; ++i) {
        const int c = min(max(cached_lens[i], 0), row_slots), n = new_lens[i];
        const int had = page_of(p, c + (p.page_size - 1));
        const bool fits = n > 0 && n <= row_slots - c;
        mine.tokens += max(n, 0);
        mine.pages += fits ? page_of(p, c + n - 1) + 1 - had : 0;
        mine.ended += n < 0 ? had : 0;
    }
    PlanSums incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const PlanSums y = plan_shfl_up(incl, o);
        if (lane >= o)
            incl = plan_add(incl, y);
    }
    if (lane == 31)
        warp_sums[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        PlanSums w = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const PlanSums y = plan_shfl_up(w, o);
            if (lane >= o)
                w = plan_add(w, y);
        }
        warp_sums[lane] = w;
    }
    __syncthreads();
    const PlanSums before = warp > 0 ? warp_sums[warp - 1] : PlanSums{0, 0, 0};
    const PlanSums total = warp_sums[31];
    PlanSums run{before.tokens + incl.tokens - mine.tokens, before.pages + incl.pages - mine.pages,
                 before.ended + incl.ended - mine.ended};
    int taken = 0, refused = 0;
    for (int i = i0; i < i1; ++i) {
        const int c = min(max(cached_lens[i], 0), row_slots), n = new_lens[i];
        const int had = page_of(p, c + (p.page_size - 1));
        const bool fits = n > 0 && n <= row_slots - c;
        run.tokens += max(n, 0);
        const int need = fits ? page_of(p, c + n - 1) + 1 - had : 0;
        run.pages += need;
        run.ended += n < 0 ? had : 0;
        const bool pages = run.pages <= free_pages || (p.room && need == 0);
        const bool ok = fits && pages && run.tokens <= p.max_tokens;
        stop[i] = saturated(run.tokens);
        upto[i] = saturated(run.pages);
        gone[i] = saturated(run.ended);
        held[i] = ok ? (unsigned)c | kPlanAdmitted : n < 0 ? 0u : (unsigned)c;
        if (ok && need > 0)
            taken = (int)run.pages;
        refused += n > 0 && !ok;
    }
    if (taken > 0)
        atomicMax(&s_taken, taken);
    if (refused > 0)
        atomicAdd(&s_refused, refused);
    cg::this_cluster().sync();  // every CTA has read the lengths and the state
    taken = s_taken;
    const auto place = [&](long long i) {
        const long long r = i % p.num_pages;
        return (int)(r < 0 ? r + p.num_pages : r);
    };
    const int first = place(head), last = place(tail);
    const int back = (int)min(total.ended, (long long)(p.num_pages - free_pages));
    // requests
    for (int i = all; i < p.seqs; i += kPlanCtas * kPlanThreads) {
        const int start = i > 0 ? stop[i - 1] : 0, c = (int)(held[i] & kPlanHeld);
        query_start[i] = start;
        seq_lens[i] = held[i] & kPlanAdmitted ? c + stop[i] - start : c;
    }
    // tokens
#pragma unroll 2
    for (unsigned u = all; u < (unsigned)p.max_tokens; u += kPlanCtas * kPlanThreads) {  // the last step may pass 2^31
        const int t = (int)u, i = first_above(stop, p.seqs, t);
        int slot = -1, pos = 0;
        if (i < p.seqs && (held[i] & kPlanAdmitted)) {
            const int c = (int)(held[i] & kPlanHeld);
            const int had = page_of(p, c + (p.page_size - 1));
            pos = c + t - (i > 0 ? stop[i - 1] : 0);
            const int at = page_of(p, pos);
            const int page = at < had ? table[(size_t)i * p.table_stride + at]
                                      : ring[ring_index(first, (i > 0 ? upto[i - 1] : 0) + (at - had), p.num_pages)];
            if (page >= 0 && page < p.num_pages)
                slot = page * p.page_size + pos - at * p.page_size;
        }
        slots[t] = slot;
        positions[t] = pos;
    }
    // pages from the ring into the tables
    for (unsigned u = all; u < (unsigned)taken; u += kPlanCtas * kPlanThreads) {
        const int k = (int)u, i = first_above(upto, p.seqs, k);
        const int had = page_of(p, (int)(held[i] & kPlanHeld) + (p.page_size - 1));
        table[(size_t)i * p.table_stride + had + k - (i > 0 ? upto[i - 1] : 0)] = ring[ring_index(first, k, p.num_pages)];
    }
    // pages of ended requests into the ring
    for (unsigned u = all; u < (unsigned)back; u += kPlanCtas * kPlanThreads) {
        const int k = (int)u, i = first_above(gone, p.seqs, k);
        ring[ring_index(last, k, p.num_pages)] = table[(size_t)i * p.table_stride + k - (i > 0 ? gone[i - 1] : 0)];
    }
    if (all == 0) {
        query_start[p.seqs] = saturated(total.tokens);
        state_out[0] = head + taken;
        state_out[1] = tail + back;
        state_out[2] = s_refused;
        state_out[3] = total.tokens;
    }
}

// ---- rotary frequencies ----------------------------------------------------------------------------
__global__ void k_rope_frequencies(int pairs, double base, double freq_scale, double ext_factor, double attn_factor,
                                   double corr0, double corr1, const float* ff, double* table)
{
    pdl_wait();
    pdl_trigger();
    for (int j = threadIdx.x; j < pairs; j += blockDim.x) {
        double f = pow(base, -2.0 * j / (2.0 * pairs));
        if (ff)
            f /= (double)ff[j];
        double mix = 0.0;
        if (ext_factor != 0.0) {
            const double y = (j - corr0) / fmax(0.001, corr1 - corr0);
            mix = (1.0 - fmin(1.0, fmax(0.0, y))) * ext_factor;
        }
        table[j] = f * (freq_scale * (1.0 - mix) + mix);
    }
    if (threadIdx.x == 0)
        table[pairs] = ext_factor != 0.0 ? attn_factor * (1.0 + 0.1 * log(1.0 / freq_scale)) : attn_factor;
}

// ---- rotary positions + append -----------------------------------------------------------------------

template <typename KV>
__device__ __forceinline__ KV pool_round(float v);
template <>
__device__ __forceinline__ float pool_round<float>(float v)
{
    return v;
}
template <>
__device__ __forceinline__ __half pool_round<__half>(float v)
{
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_fp8_e4m3 pool_round<__nv_fp8_e4m3>(float v)
{
    __nv_fp8_e4m3 r;
    r.__x = __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);  // nearest even, NaN stays NaN
    return r;
}

template <typename KV>
__device__ __forceinline__ void pool_store4(KV* dst, float4 v);
template <>
__device__ __forceinline__ void pool_store4<float>(float* dst, float4 v)
{
    *reinterpret_cast<float4*>(dst) = v;
}
template <>
__device__ __forceinline__ void pool_store4<__half>(__half* dst, float4 v)
{
    const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
}
template <>
__device__ __forceinline__ void pool_store4<__nv_fp8_e4m3>(__nv_fp8_e4m3* dst, float4 v)
{
    const unsigned a = __nv_cvt_float2_to_fp8x2(make_float2(v.x, v.y), __NV_SATFINITE, __NV_E4M3);
    const unsigned b = __nv_cvt_float2_to_fp8x2(make_float2(v.z, v.w), __NV_SATFINITE, __NV_E4M3);
    *reinterpret_cast<unsigned*>(dst) = a | b << 16;
}

// x / scale rounded to F32. For F16 and e4m3 pools as a product in float64 with the scale's reciprocal, which gives the
// same F32: a quotient of two F32 that is not on a border between F32 values is 2^-49 of itself or more away from it, and the
// product is off by 2^-52 at most. The division takes 4% more (6001 tokens into an e4m3 pool, timed in turn).
struct PoolScale {
    float scale;
    double inverse;
    explicit PoolScale(float s) : scale(s), inverse(1.0 / s) {}
    PoolScale() {}
    template <typename KV>
    __device__ __forceinline__ float down(float x) const
    {
        if (sizeof(KV) < 4)
            return __double2float_rn(__dmul_rn((double)x, inverse));
        return scale == 1.0f ? x : __fdiv_rn(x, scale);
    }
    template <typename KV>
    __device__ __forceinline__ float4 down4(float4 v) const
    {
        return make_float4(down<KV>(v.x), down<KV>(v.y), down<KV>(v.z), down<KV>(v.w));
    }
};

struct AppendDev {
    PagedDev c;
    PoolScale k, v;
    int page_shift;  // log2(page_size), or -1
    int mode, n_dims, n_offs;
    long long stride_q, stride_k, stride_v, stride_q_out;
    int has_q;
};

// (a, b) turned by the angle of cosine c and sine s, in float64, rounded once.
__device__ __forceinline__ void turn(float& a, float& b, double c, double s)
{
    const double x = a, y = b;
    a = __double2float_rn(__dsub_rn(__dmul_rn(x, c), __dmul_rn(y, s)));
    b = __double2float_rn(__dadd_rn(__dmul_rn(x, s), __dmul_rn(y, c)));
}

// One CTA per token. The angles are formed once per token, in float64 as k_kv_append forms them, and shared by its
// heads. V4: a thread's unit is two float4 of a row - four pairs, or eight channels that pass unchanged, or eight
// channels of v, the second float4 half a range behind the first so that neighbours' accesses join up - all loaded
// before the angles are waited for; else a unit is one pair. Bound by the bytes
// (q twice, k and v once, the pools' rows): 6001 tokens of 32/8 heads of 128 into an e4m3 pool, 259 MB, take 43.9 us (5.9
// TB/s, 0.90 of the copy rate); the float64 rotation costs 2 us of it. Eight CTAs of four warps on an SM keep loads, turns and
// stores of different tokens going side by side: four of eight warps take 46.8 us, and a CTA that takes several tokens
// with the next one's loads under way more (63 us in registers, 97 us through shared memory): CTAs of one token are
// dealt out as SMs come free.
constexpr int kAppendThreads = 128;

template <typename KV, bool V4>
__global__ void __launch_bounds__(kAppendThreads, 8) k_paged_append(AppendDev p, const float* q, const float* k, const float* v,
                                                                 const int32_t* positions, const int32_t* slots,
                                                                 const double* freqs, float* q_out, KV* k_pool,
                                                                 KV* v_pool)
{
    __shared__ __align__(16) double cs[128];  // cos of pair j, then sin
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.x, tid = threadIdx.x;
    const int slot = slots[t];
    if (slot < 0 || slot >= p.c.page_size * p.c.num_pages)
        return;
    const int half = p.n_dims / 2, hd = p.c.head_dim;
    const int page = p.page_shift >= 0 ? slot >> p.page_shift : slot / p.c.page_size, at = slot - page * p.c.page_size;
    const long long row = page * p.c.page_stride + at * p.c.slot_stride;
    const int heads = p.has_q ? p.c.heads : 0;
    const auto angles = [&]() {
        for (int j = tid; j < half; j += kAppendThreads) {
            const double size = freqs[half];
            double s, c;
            sincos((double)positions[t] * freqs[j], &s, &c);
            cs[j] = c * size;
            cs[half + j] = s * size;
        }
    };
    if constexpr (V4) {
        const int shift = __ffs(hd) - 4, per_head = hd / 8, turned = p.n_dims / 8;  // units; hd is a power of two
        const int qk = (heads + p.c.kv_heads) * per_head, all = qk + p.c.kv_heads * per_head;
        constexpr int U = 3;  // a thread's units at a time
        bool formed = false;
        // so that head h of the CTA's heads (q's, k's, v's) is h * hd behind its row
        const float* q_row = q + t * p.stride_q;
        const float* k_row = k + t * p.stride_k - heads * hd;
        const float* v_row = v + t * p.stride_v - (heads + p.c.kv_heads) * hd;
        float* q_out_row = q_out + t * p.stride_q_out;
#pragma unroll 1
        for (int base = tid; base - tid < all; base += U * kAppendThreads) {
            float4 x[U][2];
            int d0[U], d1[U];  // the float4s' channels
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int e = base + i * kAppendThreads;
                if (e < all) {
                    const int h = e >> shift, u = e & (per_head - 1);
                    if (e >= qk) {
                        d0[i] = 4 * u, d1[i] = d0[i] + hd / 2;
                    } else if (u < turned) {
                        d0[i] = p.n_offs + 4 * u, d1[i] = d0[i] + half;
                    } else {
                        d0[i] = 4 * (u - turned), d1[i] = d0[i] + (hd - p.n_dims) / 2;
                        d0[i] += d0[i] < p.n_offs ? 0 : p.n_dims;
                        d1[i] += d1[i] < p.n_offs ? 0 : p.n_dims;
                    }
                    const float* src = (e >= qk ? v_row : h < heads ? q_row : k_row) + (h << (shift + 3));
                    x[i][0] = *reinterpret_cast<const float4*>(src + d0[i]);
                    x[i][1] = *reinterpret_cast<const float4*>(src + d1[i]);
                }
            }
            if (!formed) {
                angles();
                __syncthreads();
                formed = true;
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int e = base + i * kAppendThreads;
                if (e < all) {
                    const int h = e >> shift, u = e & (per_head - 1);
                    if (e < qk && u < turned) {
                        // the pairs in a row: 4 u .. 4 u + 3, or 2 u, 2 u + 1 and those half / 2 behind them
                        const bool neox = p.mode == MUYO_ROPE_NEOX;
                        const int at = neox ? 4 * u : 2 * u, next = neox ? at + 2 : at + half / 2;
                        const double2 c0 = *reinterpret_cast<const double2*>(cs + at);
                        const double2 c1 = *reinterpret_cast<const double2*>(cs + next);
                        const double2 s0 = *reinterpret_cast<const double2*>(cs + half + at);
                        const double2 s1 = *reinterpret_cast<const double2*>(cs + half + next);
                        if (neox) {
                            turn(x[i][0].x, x[i][1].x, c0.x, s0.x);
                            turn(x[i][0].y, x[i][1].y, c0.y, s0.y);
                            turn(x[i][0].z, x[i][1].z, c1.x, s1.x);
                            turn(x[i][0].w, x[i][1].w, c1.y, s1.y);
                        } else {
                            turn(x[i][0].x, x[i][0].y, c0.x, s0.x);
                            turn(x[i][0].z, x[i][0].w, c0.y, s0.y);
                            turn(x[i][1].x, x[i][1].y, c1.x, s1.x);
                            turn(x[i][1].z, x[i][1].w, c1.y, s1.y);
                        }
                    }
                    if (h < heads) {
                        float* y = q_out_row + (h << (shift + 3));
                        *reinterpret_cast<float4*>(y + d0[i]) = x[i][0];
                        *reinterpret_cast<float4*>(y + d1[i]) = x[i][1];
                    } else {
                        const bool is_v = e >= qk;
                        KV* y = (is_v ? v_pool : k_pool) + row + (h - heads - (is_v ? p.c.kv_heads : 0)) * p.c.head_stride;
                        const PoolScale scale = is_v ? p.v : p.k;
                        pool_store4<KV>(y + d0[i], scale.down4<KV>(x[i][0]));
                        pool_store4<KV>(y + d1[i], scale.down4<KV>(x[i][1]));
                    }
                }
            }
        }
    } else {
        angles();
        __syncthreads();
        const int pairs = hd / 2;
        for (int e = tid; e < (heads + p.c.kv_heads) * pairs; e += kAppendThreads) {
            const int h = e / pairs, i = e - h * pairs;
            // pair i of the head: the turned pairs first, then the channels that pass unchanged by twos
            int j0, j1;
            if (i < half) {
                j0 = p.n_offs + (p.mode == MUYO_ROPE_NEOX ? i : 2 * i);
                j1 = p.mode == MUYO_ROPE_NEOX ? j0 + half : j0 + 1;
            } else {
                j0 = 2 * (i - half);
                j0 = j0 < p.n_offs ? j0 : j0 + p.n_dims;
                j1 = j0 + 1;
            }
            const float* x = h < heads ? q + t * p.stride_q + (long long)h * hd
                                       : k + t * p.stride_k + (long long)(h - heads) * hd;
            float y0 = x[j0], y1 = x[j1];
            if (i < half)
                turn(y0, y1, cs[i], cs[half + i]);
            if (h < heads) {
                float* y = q_out + t * p.stride_q_out + (long long)h * hd;
                y[j0] = y0;
                y[j1] = y1;
            } else {
                KV* y = k_pool + row + (h - heads) * p.c.head_stride;
                y[j0] = pool_round<KV>(p.k.down<KV>(y0));
                y[j1] = pool_round<KV>(p.k.down<KV>(y1));
            }
        }
        for (int e = tid; e < p.c.kv_heads * hd; e += kAppendThreads) {
            const int h = e / hd, d = e - h * hd;
            v_pool[row + h * p.c.head_stride + d] = pool_round<KV>(p.v.down<KV>(v[t * p.stride_v + e]));
        }
    }
}

}  // namespace muyo

using namespace muyo;

extern "C" int muyo_cuda_paged_plan(const MuyoPagedPlanParams* p, const int32_t* cached_lens, const int32_t* new_lens,
                                    int32_t* block_table, int32_t* free_ring, const int64_t* state, int32_t* seq_lens,
                                    int32_t* query_start, int32_t* positions, int32_t* slots, int64_t* state_out,
                                    void* stream)
{
    clear_error();
    MUYO_REQUIRE(p, "paged_plan: null parameter block");
    MUYO_REQUIRE(p->seqs > 0, "paged_plan: seqs must be positive");
    if (p->seqs > (uint32_t)kPlanMaxSeqs) {
        set_error("paged_plan: %u requests exceed %d", p->seqs, kPlanMaxSeqs);
        return MUYO_EUNSUPPORTED;
    }
    MUYO_REQUIRE(p->page_size > 0 && p->num_pages > 0 && p->table_stride > 0,
                 "paged_plan: page_size, num_pages and table_stride must be positive");
    MUYO_REQUIRE((uint64_t)p->page_size * p->num_pages <= (uint64_t)INT_MAX,
                 "paged_plan: %u pages of %u slots exceed INT32_MAX slots", p->num_pages, p->page_size);
    MUYO_REQUIRE((uint64_t)p->page_size * p->table_stride <= (uint64_t)1 << 30,
                 "paged_plan: a row of %u pages of %u slots exceeds 2^30 slots", p->table_stride, p->page_size);
    MUYO_REQUIRE(p->max_tokens < (uint32_t)INT_MAX, "paged_plan: max_tokens %u is not below INT32_MAX", p->max_tokens);
    MUYO_REQUIRE(cached_lens && new_lens && block_table && free_ring && state && seq_lens && query_start && state_out,
                 "paged_plan: null buffer");
    MUYO_REQUIRE(p->max_tokens == 0 || (positions && slots), "paged_plan: positions and slots are needed with max_tokens");
    MUYO_REQUIRE(aligned_to(state, 8) && aligned_to(state_out, 8), "paged_plan: state must be 8-byte aligned");
    MUYO_REQUIRE((p->flags & ~MUYO_PLAN_ROOM) == 0, "paged_plan: unknown flags 0x%x", p->flags);
    const PlanDev d{(int)p->seqs, (int)p->page_size, (int)p->num_pages, (int)p->table_stride, (int)p->max_tokens,
                    page_shift_of((int)p->page_size), (p->flags & MUYO_PLAN_ROOM) != 0};
    const size_t smem = (size_t)p->seqs * 4 * sizeof(int);
    static std::atomic<unsigned long long> allowed{0};
    // for every size: the limit without it, 48 KB, holds for static and dynamic shared memory together
    MUYO_CUDA_TRY(allow_smem(k_paged_plan, (size_t)kPlanMaxSeqs * 4 * sizeof(int), allowed));
    MUYO_CUDA_TRY(launch_kernel(k_paged_plan, dim3(kPlanCtas), dim3(kPlanThreads), smem, as_stream(stream), true, d, cached_lens,
                                new_lens, block_table, free_ring, state, seq_lens, query_start, positions, slots, state_out));
    MUYO_LAUNCH_CHECK();
    return MUYO_OK;
}

extern "C" int muyo_cuda_rope_frequencies(const MuyoRopeParams* p, const float* freq_factors, double* table, void* stream)
{
    clear_error();
    MUYO_REQUIRE(p && table, "rope_frequencies: null parameter block or table");
    MUYO_REQUIRE(p->n_dims > 0 && p->n_dims % 2 == 0 && p->n_dims <= (uint32_t)INT_MAX,
                 "rope_frequencies: n_dims %u must be positive and even", p->n_dims);
    MUYO_REQUIRE(p->freq_base > 0.0f && std::isfinite(p->freq_base), "rope_frequencies: freq_base must be positive");
    MUYO_REQUIRE(p->ext_factor == 0.0f || p->freq_scale > 0.0f, "rope_frequencies: freq_scale must be positive with ext_factor");
    MUYO_REQUIRE(!p->has_ff || freq_factors, "rope_frequencies: has_ff without freq_factors");
    MUYO_REQUIRE(aligned_to(table, 8), "rope_frequencies: table must be 8-byte aligned");
    MUYO_CUDA_TRY(launch_kernel(k_rope_frequencies, dim3(1), dim3(64), 0, as_stream(stream), true, (int)(p->n_dims / 2),
                                (double)p->freq_base, (double)p->freq_scale, (double)p->ext_factor, (double)p->attn_factor,
                                (double)p->corr_dims[0], (double)p->corr_dims[1], p->has_ff ? freq_factors : nullptr, table));
    MUYO_LAUNCH_CHECK();
    return MUYO_OK;
}

template <typename KV>
static int launch_append(const AppendDev& d, int tokens, const float* q, const float* k, const float* v,
                         const int32_t* positions, const int32_t* slots, const double* freqs, float* q_out, void* k_pool,
                         void* v_pool, void* stream)
{
    // units of two float4 need four pairs at a time and channels that pass by fours
    const auto kernel = d.n_dims % 8 == 0 && d.n_offs % 4 == 0 ? k_paged_append<KV, true> : k_paged_append<KV, false>;
    MUYO_CUDA_TRY(launch_kernel(kernel, dim3(tokens), dim3(kAppendThreads), 0, as_stream(stream), true, d, q, k, v, positions,
                                slots, freqs, q_out, static_cast<KV*>(k_pool), static_cast<KV*>(v_pool)));
    MUYO_LAUNCH_CHECK();
    return MUYO_OK;
}

extern "C" int muyo_cuda_paged_rope_append(const MuyoPagedAppendParams* p, const float* q, const float* k, const float* v,
                                           const int32_t* positions, const int32_t* slots, const double* freqs,
                                           float* q_out, void* k_pool, void* v_pool, void* stream)
{
    clear_error();
    MUYO_REQUIRE(p, "paged_rope_append: null parameter block");
    AppendDev d{};
    const int rc = paged_prepare(p->cache, "paged_rope_append", d.c);
    if (rc != MUYO_OK)
        return rc;
    MUYO_REQUIRE(p->rope_mode == MUYO_ROPE_NORMAL || p->rope_mode == MUYO_ROPE_NEOX, "paged_rope_append: rope mode %u",
                 p->rope_mode);
    MUYO_REQUIRE(p->n_dims % 2 == 0 && p->n_offs % 2 == 0 && p->n_dims <= p->cache.head_dim &&
                     p->n_offs <= p->cache.head_dim - p->n_dims,
                 "paged_rope_append: channels [%u, %u + %u) must be even bounds within head_dim %u", p->n_offs, p->n_offs,
                 p->n_dims, p->cache.head_dim);
    MUYO_REQUIRE(p->tokens <= (uint32_t)INT_MAX, "paged_rope_append: too many tokens");
    MUYO_REQUIRE(k && v && positions && slots && k_pool && v_pool, "paged_rope_append: null buffer");
    MUYO_REQUIRE(p->n_dims == 0 || freqs, "paged_rope_append: freqs are needed to turn %u channels", p->n_dims);
    MUYO_REQUIRE(!q || q_out, "paged_rope_append: q without q_out");
    MUYO_REQUIRE(aligned_to(freqs, 8), "paged_rope_append: freqs must be 8-byte aligned");
    MUYO_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) && aligned16(k_pool) && aligned16(v_pool),
                 "paged_rope_append: q, k, v, q_out and the pools must be 16-byte aligned");
    const uint32_t q_row = p->cache.heads * p->cache.head_dim, kv_row = p->cache.kv_heads * p->cache.head_dim;
    d.stride_q = p->stride_q ? p->stride_q : q_row;
    d.stride_k = p->stride_k ? p->stride_k : kv_row;
    d.stride_v = p->stride_v ? p->stride_v : kv_row;
    d.stride_q_out = p->stride_q_out ? p->stride_q_out : q_row;
    MUYO_REQUIRE(d.stride_q >= q_row && d.stride_q_out >= q_row && d.stride_k >= kv_row && d.stride_v >= kv_row,
                 "paged_rope_append: a row stride is below its row (%u, %u)", q_row, kv_row);
    MUYO_REQUIRE((d.stride_q | d.stride_k | d.stride_v | d.stride_q_out) % 4 == 0,
                 "paged_rope_append: row strides must be multiples of 4");
    MUYO_REQUIRE(q != q_out || !q || d.stride_q == d.stride_q_out, "paged_rope_append: q in place needs equal strides");
    d.k = PoolScale(d.c.k_scale), d.v = PoolScale(d.c.v_scale);
    d.page_shift = page_shift_of(d.c.page_size);
    d.mode = (int)p->rope_mode, d.n_dims = (int)p->n_dims, d.n_offs = (int)p->n_offs, d.has_q = q != nullptr;
    if (p->tokens == 0)
        return MUYO_OK;
    const int T = (int)p->tokens;
    switch (p->cache.kv_dtype) {
        case MUYO_KV_F32: return launch_append<float>(d, T, q, k, v, positions, slots, freqs, q_out, k_pool, v_pool, stream);
        case MUYO_KV_F16: return launch_append<__half>(d, T, q, k, v, positions, slots, freqs, q_out, k_pool, v_pool, stream);
        default: return launch_append<__nv_fp8_e4m3>(d, T, q, k, v, positions, slots, freqs, q_out, k_pool, v_pool, stream);
    }
}
