// Attention of one new token per request over a paged key-value cache.
//
// o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = scale q . k_j, with the running maximum and sum of
// an online softmax. Every key and value is read once, for all query heads of its KV head, so the bound is
// the cache's bytes: 2 * keys * kv_heads * head_dim * sizeof(element).
//
// Work. The keys of a (request, KV head) are cut into tiles of KT keys (8 KB of keys and values, fewer for
// small heads); all tiles of the batch, in order, are dealt out evenly and contiguously to the warps of CTAs of
// four warps, as many as are on the SMs at once. The dealing is done on the device from seq_lens (a scan per CTA), so a
// captured graph stays right when lengths change, and no spread of lengths leaves warps idle: one request over
// 131071 keys and 200 requests over 60 to 2048 keys both keep every warp busy to within one tile. A warp that holds the
// whole of a segment (the tiles of one request and KV head) writes its output; pieces of segments cut by a warp's
// border are joined in shared memory by the CTA, those cut by a CTA's border by a second kernel from at most two
// partials per CTA (m, l, o).
//
// A warp copies its tiles with cp.async into a ring of its own (no block barriers) STAGES - 1 tiles ahead;
// the page numbers are fetched one tile further ahead. Rows are swizzled by 16-byte chunks so that the
// fragment reads below meet no bank conflicts at 128-byte rows and wider.
//
// Measured: 131071 keys of 32/8 heads of 128 in F16, 537 MB, 98 us (5.5 TB/s, 0.84 of the copy rate; the SMs of some
// GPCs stream 12% slower than the others, and even shares wait for them); 64 requests over 2000 to 16000 e4m3 keys,
// 901 MB, 175 us (5.1 TB/s, 0.78; the conversions' dependent chains with 8 warps on an SM - 12 warps with tiles of half
// the size take an eighth more); 200 requests over 60 to 2048 keys of 14/2 heads of 64 in F16, 60 MB, 23 us (start, joins and
// the second kernel are two thirds); one request over 1023 keys 8.8 us (two launches); 33 requests of 16 heads on one
// F32 head, windows of 4096 keys, 80 MB, 42 us (1009 instructions per tile of 8 keys; half of its 128 splits of
// F32 operands are of q, the same ones for each tile). With 9 to 16 heads of 128 per KV head 255 registers do not hold q's halves and the
// output: spills of 482 bytes a thread with e4m3, 142 with F16, 76 with F32 (36 with e4m3 and up to 8 heads). 64 requests over 2000 to
// 16000 keys of 32/2 heads of 128: e4m3 225 MB, 158 us (1.4 TB/s), F16 450 MB, 105 us (4.3 TB/s); of 16/2 heads 53 and 83 us.
//
// Products. mma.sync tiles of 16 rows x 8 keys (scores) and 16 rows x 8 channels (values). With at most 8 query
// heads per KV head the 16 rows are the heads' leading halves and, below them, their remainders: an F32
// operand x is split into two F16 (x = hi + lo, 22 bits; TF32 for an F32 cache), so one instruction makes both
// products and a lane adds its own rows g and g + 8 at the end. With 9 to 16 heads the two halves take an
// instruction each. q is brought near 2^14 by a power of two per head and the weights are formed as
// 2^(s - m + 15), so that neither half falls under F16's normal range. F16 and e4m3 caches enter exactly;
// F32 ones are split like q (the product of the two remainders is dropped for 9 to 16 heads only). Each
// tile's products start from zero and are added to the running sums in F32: the tensor core's own additions
// truncate, and long chains of them would drift. The channels' order in the contraction is free, so a
// lane reads 16 contiguous bytes of a key's row for four (two) steps, and the keys of a step
// are paired so that the scores' layout is the weights'. tcgen05 would hold 128 rows per tile for the 8 or 16 that one
// token has; at these sizes the mma.sync issue is far below the memory time.
#include <algorithm>

#include "paged.cuh"

namespace muyo {

constexpr int kPagedWarps = 4;
constexpr int kPagedThreads = 32 * kPagedWarps;
constexpr int kPagedTile = 4096;  // bytes of a tile's keys

struct PagedAttnDev {
    PagedDev c;
    int seqs, table_stride, window;
    int page_shift;  // log2(page_size), or -1
    int one_page;    // whether every tile lies inside one page
    long long stride_q, stride_out;
    float scale;  // softmax scale * k_scale
};

struct PagedDesc {
    int seq, kv_head, pieces, pad;
};

template <int T, int HD, bool WIDE>
struct PagedTile {
    static constexpr int ES = T == MUYO_KV_F32 ? 4 : T == MUYO_KV_F16 ? 2 : 1;
    static constexpr int RB = HD * ES;        // bytes of a row
    static constexpr int CPR = RB / 16;       // 16-byte chunks of a row
    static constexpr int KSTEP = T == MUYO_KV_F32 ? 8 : 16;
    // 4 KB of keys: half of that with three CTAs on an SM took 214 us where 4 KB took 190 (64 requests, e4m3). At most
    // 64 keys: a warp votes and masks two keys a lane.
    static constexpr int KT = kPagedTile / RB > 64 ? 64 : kPagedTile / RB < KSTEP ? KSTEP : kPagedTile / RB;  // keys of a tile
    static constexpr int STAGES = WIDE ? 2 : 3;  // WIDE: a third would leave shared memory for one CTA
    static constexpr int TILE = KT * RB;      // bytes of a tile's keys (or values)
    static constexpr int ROWS = WIDE ? 16 : 8;
    static constexpr int PART = ROWS * (HD + 2);  // floats of a partial: o [ROWS][HD], m, l
    static constexpr int CHB = RB / 4 < 16 ? RB / 4 : 16;  // bytes of a lane's K read
    static constexpr int EPC = CHB / ES;
    static constexpr int NCH = RB / (4 * CHB);
    static constexpr int KPS = T == MUYO_KV_F32 ? 2 : 4;   // a lane's channels per k-step
    static constexpr int NKS = NCH * EPC / KPS;            // k-steps of a row
    static constexpr int VPL = HD / 8;                     // a lane's channels of a value row
    static constexpr int VCHB = VPL * ES < 16 ? VPL * ES : 16;
    static constexpr int VE = VCHB / ES;
    static constexpr int NVC = VPL / VE;
    static constexpr int RING = STAGES * 2 * TILE;
    static_assert(KT % KSTEP == 0 && KT * CPR % 32 == 0, "tile shape");
    static_assert(RING >= PART * 4, "a drained ring holds a partial");
    static constexpr size_t SMEM = (size_t)kPagedWarps * (RING + PART * 4);
    // On an SM at once. Three where they fit; two of full tiles: twice the CTAs, half of them waiting for their turn,
    // took 108 us where one turn takes 99 (131071 keys) and 29 us where it takes 23 (200 requests).
    static constexpr int CTAS = SMEM <= 75 * 1024 ? 3 : 2;
};

template <int CPR>
__device__ __forceinline__ int k_chunk(int row, int ch)
{
    return CPR >= 8 ? ch ^ ((row & 1) << 2) : ch;
}

template <int CPR>
__device__ __forceinline__ int v_chunk(int row, int ch)
{
    return CPR >= 8 ? ch ^ (((row >> 1) & 3) << 1) : CPR == 4 ? ch ^ (((row >> 1) & 1) << 1) : ch;
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16 bytes, or 16 zero bytes when !valid.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool valid)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The first product of a sum: from zero.
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ void mma_tf32_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// (a, b) as F16 pairs: the leading halves and the remainders.
__device__ __forceinline__ void split_half2(float a, float b, uint32_t& hi, uint32_t& lo)
{
    hi = pack_half2(a, b);
    const float2 h = h2_to_f2(hi);
    lo = pack_half2(a - h.x, b - h.y);
}

// x as two TF32: rounded to 11 bits, and 11 bits of what is left, of either sign: 23 bits without a bias.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo)
{
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}

// Four e4m3 as F16 pairs, exactly: the two low bytes, the two high ones.
__device__ __forceinline__ void e4m3x4_half2(uint32_t v, uint32_t& low, uint32_t& high)
{
    asm("{.reg .b16 x, y; mov.b32 {x, y}, %2; cvt.rn.f16x2.e4m3x2 %0, x; cvt.rn.f16x2.e4m3x2 %1, y;}"
        : "=r"(low), "=r"(high)
        : "r"(v));
}

template <int BYTES>
struct Chunk {
    uint32_t w[BYTES < 4 ? 1 : BYTES / 4];
    __device__ __forceinline__ void load(uint32_t addr)
    {
        if constexpr (BYTES == 16)
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
        else if constexpr (BYTES == 8)
            asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
        else if constexpr (BYTES == 4)
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
        else
            asm volatile("{.reg .u16 t; ld.shared.u16 t, [%1]; cvt.u32.u16 %0, t;}" : "=r"(w[0]) : "r"(addr));
    }
};

// The keys that a request's token sees, in tiles: [t0, t1).
template <int KT>
struct PagedSpan {
    int n, begin, t0, t1;
    __device__ __forceinline__ PagedSpan() {}
    __device__ __forceinline__ PagedSpan(const PagedAttnDev& p, int len)
    {
        n = min(max(len, 0), p.table_stride * p.c.page_size);
        begin = p.window > 0 ? max(0, n - p.window) : 0;
        t0 = begin / KT;
        t1 = n > begin ? (n + KT - 1) / KT : t0;
    }
};

__device__ __forceinline__ float paged_lse(float m, float l)
{
    return l > 0.0f ? (m + log2f(l)) * 0.693147180559945f : -INFINITY;
}

// A tile of the batch: tile t of request s under KV head h.
template <int KT>
struct PagedCursor {
    int s, h, t;
    PagedSpan<KT> span;
    // Goes to the next tile, of which the caller knows; true at a segment's first.
    __device__ __forceinline__ bool next(const PagedAttnDev& p, const int32_t* lens)
    {
        if (++t < span.t1)
            return false;
        if (++h == p.c.kv_heads) {
            h = 0;
#pragma unroll 1
            do {
                span = PagedSpan<KT>(p, lens[++s]);
            } while (span.t1 == span.t0);
        }
        t = span.t0;
        return true;
    }
};

// Contiguous shares of `total` tiles for `workers` warps: the first `extra` get one more.
struct PagedShares {
    unsigned each, extra;
    __device__ __forceinline__ PagedShares(unsigned total, unsigned workers) : each(total / workers), extra(total % workers) {}
    __device__ __forceinline__ int begin(unsigned worker) const { return (int)(worker * each + min(worker, extra)); }
    __device__ __forceinline__ int worker_of(unsigned tile) const
    {
        const unsigned border = extra * (each + 1);
        return (int)(tile < border ? tile / (each + 1) : extra + (tile - border) / each);
    }
};

// Pieces of one segment that a CTA joins: bit w the first piece of warp w, bit kPagedWarps + w its last one.
struct PagedGroup {
    unsigned pieces;
    int seq, kv_head;
    int to;  // -1: complete; else the CTA's partial 0 (the segment came in) or 1 (it begins here)
};

template <int T, int HD, bool WIDE>
__global__ void __launch_bounds__(kPagedThreads, (PagedTile<T, HD, WIDE>::CTAS))
k_paged_attention(PagedAttnDev p, const float* q, const char* k_pool, const char* v_pool, const int32_t* table,
                  const int32_t* lens, float* out, float* lse, float* part, PagedDesc* descs)
{
    using C = PagedTile<T, HD, WIDE>;
    constexpr int KT = C::KT, HR = WIDE ? 2 : 1;  // HR: heads of a lane
    constexpr int W = kPagedWarps;
    extern __shared__ __align__(128) char paged_smem[];
    __shared__ unsigned long long s_mask[W][C::STAGES];
    __shared__ int s_sum[W];
    // the scan at first, the joins' rows and groups at the end (two CTAs' shared memory fits an SM to the byte)
    union Shared {
        int scan[kPagedThreads];
        struct {
            float2 rows[(W + 1) * C::ROWS];
            PagedGroup group[W + 1];
        } join;
    };
    __shared__ __align__(16) Shared s_u;
    static_assert(kPagedThreads == 128, "four shares per lane");
    __shared__ int s_first[W], s_last[W];  // open pieces: 0 none, 1 open at the end, 2 ends here
    __shared__ int s_seg[W][4];            // request and KV head of the first and the last piece
    __shared__ int s_open;                 // tiles of the CTA's last segment behind its range
    __shared__ int s_groups;
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, cq = lane & 3;

    // The batch's tiles, scanned over the threads' contiguous requests.
    const int per = (p.seqs + kPagedThreads - 1) / kPagedThreads;
    const int s_begin = min(tid * per, p.seqs), s_end = min(s_begin + per, p.seqs);
    int mine = 0, empty = 0;
#pragma unroll 1
    for (int s = s_begin; s < s_end; ++s) {
        const PagedSpan<KT> span(p, lens[s]);
        mine += (span.t1 - span.t0) * p.c.kv_heads;
        empty |= span.t1 == span.t0;
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o)
            incl += y;
    }
    if (lane == 31)
        s_sum[warp] = incl;
    if (tid < W)
        s_first[tid] = s_last[tid] = 0;
    if (tid == 0)
        s_open = 0;
    empty = __syncthreads_or(empty);
    int total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const int v = s_sum[w];
        incl += w < warp ? v : 0;
        total += v;
    }
    const int ctas = min((int)gridDim.x, (total + W - 1) / W);  // CTAs with work
    const PagedShares shares((unsigned)total, (unsigned)max(ctas, 1) * W);
    const int worker = blockIdx.x * W + warp;
    const bool idle = (int)blockIdx.x >= ctas;
    s_u.scan[tid] = incl;
    __syncthreads();
    if (empty) {  // requests without keys
#pragma unroll 1
        for (int s = blockIdx.x * W + warp; s < p.seqs; s += gridDim.x * W) {
            const PagedSpan<KT> span(p, lens[s]);
            if (span.t1 > span.t0)
                continue;
#pragma unroll 1
            for (int d = lane; d < p.c.heads * HD; d += 32)
                out[s * p.stride_out + d] = 0.0f;
            if (lse)
#pragma unroll 1
                for (int h = lane; h < p.c.heads; h += 32)
                    lse[(size_t)s * p.c.heads + h] = -INFINITY;
        }
    }
    if (idle) {
        if (tid == 0)
            descs[blockIdx.x] = PagedDesc{0, 0, 0, 0};
        return;
    }
    const int cta_end = shares.begin((blockIdx.x + 1) * W);
    const int u1 = shares.begin(worker + 1);
    int left = u1 - shares.begin(worker), ahead = left;  // tiles to work on, to copy
    PagedCursor<KT> cur;
    if (left > 0) {
        // the first thread whose requests reach past the warp's first tile
        const int u0 = u1 - left;
        const int4 mark = *reinterpret_cast<const int4*>(&s_u.scan[4 * lane]);
        const int share = __reduce_add_sync(0xffffffffu, (mark.x <= u0) + (mark.y <= u0) + (mark.z <= u0) + (mark.w <= u0));
        int rest = u0 - (share > 0 ? s_u.scan[share - 1] : 0), tiles;
        cur.s = share * per;
#pragma unroll 1
        for (;; ++cur.s) {
            cur.span = PagedSpan<KT>(p, lens[cur.s]);
            tiles = cur.span.t1 - cur.span.t0;
            if (rest < tiles * p.c.kv_heads)
                break;
            rest -= tiles * p.c.kv_heads;
        }
        cur.h = rest / tiles;
        cur.t = cur.span.t0 + rest - cur.h * tiles;
    }

    char* ring = paged_smem + (size_t)warp * C::RING;
    const uint32_t ring_at = smem_addr(ring);
    float* first_part = reinterpret_cast<float*>(paged_smem + (size_t)W * C::RING) + (size_t)warp * C::PART;

    // ---- copies ----
    // A tile inside one page (page_size a multiple of KT) has its rows slot_stride apart from one place on; else each
    // row's place comes from the lane that looked its page up.
    constexpr int RPI = 32 / C::CPR;  // rows of one copy instruction
    const int ch = lane % C::CPR, row0 = lane / C::CPR;
    const long long slot_bytes = p.c.slot_stride * C::ES;
    PagedCursor<KT> load = cur;
    int pages[(KT + 31) / 32];
    auto look_up = [&](bool begins) {
#pragma unroll
        for (int i = 0; i < (KT + 31) / 32; ++i) {
            const int key = p.one_page ? load.t * KT : load.t * KT + i * 32 + lane;
            const int at = p.page_shift >= 0 ? key >> p.page_shift : key / p.c.page_size;
            pages[i] = -1;
            if (p.one_page ? i == 0 : (KT % 32 == 0 || lane < KT) && key < load.span.n && key >= load.span.begin)
                pages[i] = table[(size_t)load.s * p.table_stride + at];
        }
        if (begins) {  // the segment's q into L1: behind the copies it would wait for them
            const float* qrow = q + load.s * p.stride_q + (long long)load.h * p.c.group * HD;
#pragma unroll 1
            for (int d = lane * 32; d < p.c.group * HD; d += 32 * 32) {
                float unused;
                asm volatile("ld.global.f32 %0, [%1];" : "=f"(unused) : "l"(qrow + d));
            }
        }
    };
    auto issue = [&](int stage) {
        const uint32_t kd = ring_at + stage * 2 * C::TILE, vd = kd + C::TILE;
        unsigned long long mask = 0;
        const int key0 = load.t * KT;
        if (p.one_page) {
            const bool ok = pages[0] >= 0 && pages[0] < p.c.num_pages;
            const int slot = p.page_shift >= 0 ? key0 & (p.c.page_size - 1) : key0 % p.c.page_size;
            const int lo = ok ? load.span.begin - key0 : KT, hi = load.span.n - key0;  // rows lo .. hi - 1 are seen
            long long o = ok ? (pages[0] * p.c.page_stride + load.h * p.c.head_stride + (slot + row0) * p.c.slot_stride) * C::ES
                             : 0;
            o += ch * 16;
#pragma unroll
            for (int i = 0; i < (KT + 31) / 32; ++i)
                mask |= (unsigned long long)__ballot_sync(0xffffffffu, i * 32 + lane >= lo && i * 32 + lane < min(hi, KT))
                        << (32 * i);
            const char *kp = k_pool + o, *vp = v_pool + o;
            if (lo <= 0 && hi >= KT) {
#pragma unroll
                for (int i = 0; i < KT * C::CPR / 32; ++i) {
                    const int row = i * RPI + row0;
                    copy16(kd + row * C::RB + k_chunk<C::CPR>(row, ch) * 16, kp, true);
                    copy16(vd + row * C::RB + v_chunk<C::CPR>(row, ch) * 16, vp, true);
                    kp += RPI * slot_bytes, vp += RPI * slot_bytes;
                }
            } else {
#pragma unroll 1
                for (int i = 0; i < KT * C::CPR / 32; ++i) {
                    const int row = i * RPI + row0;
                    const bool seen = row >= lo && row < hi;
                    copy16(kd + row * C::RB + k_chunk<C::CPR>(row, ch) * 16, seen ? kp : k_pool, seen);
                    copy16(vd + row * C::RB + v_chunk<C::CPR>(row, ch) * 16, seen ? vp : v_pool, seen);
                    kp += RPI * slot_bytes, vp += RPI * slot_bytes;
                }
            }
        } else {
            long long off[(KT + 31) / 32];
#pragma unroll
            for (int i = 0; i < (KT + 31) / 32; ++i) {
                const int key = key0 + i * 32 + lane;
                const int slot = p.page_shift >= 0 ? key & (p.c.page_size - 1) : key % p.c.page_size;
                const bool ok = pages[i] >= 0 && pages[i] < p.c.num_pages;
                off[i] = ok ? (pages[i] * p.c.page_stride + load.h * p.c.head_stride + slot * p.c.slot_stride) * C::ES : 0;
                mask |= (unsigned long long)__ballot_sync(0xffffffffu, ok) << (32 * i);
            }
#pragma unroll
            for (int i = 0; i < KT * C::CPR / 32; ++i) {
                const int row = i * RPI + row0;
                const long long o = __shfl_sync(0xffffffffu, off[i * RPI / 32], row & 31) + ch * 16;
                const bool seen = (mask >> row) & 1;
                copy16(kd + row * C::RB + k_chunk<C::CPR>(row, ch) * 16, k_pool + (seen ? o : 0), seen);
                copy16(vd + row * C::RB + v_chunk<C::CPR>(row, ch) * 16, v_pool + (seen ? o : 0), seen);
            }
        }
        if (lane == 0)
            s_mask[warp][stage] = mask;
        if (--ahead > 0)
            look_up(load.next(p, lens));
    };

    // ---- the segment at hand ----
    constexpr int NQ = T == MUYO_KV_F32 ? C::NKS * 2 * HR : C::NKS * 4 * HR;
    uint32_t qf[NQ];              // fragments (F32 cache: q itself)
    float qs[HR], m[HR], l[HR];   // m: reference of the weights, the running maximum - 15 rounded up
    float o[C::VPL][2 * HR];
    bool whole = false;           // this warp has the segment from its first tile on
    float raw[HR][C::NKS * C::KPS];
    auto load_q = [&]() {
        const float* qrow = q + cur.s * p.stride_q + (long long)cur.h * p.c.group * HD;
#pragma unroll
        for (int r = 0; r < HR; ++r) {
            const int head = g + 8 * r;
#pragma unroll
            for (int k = 0; k < C::NKS; ++k) {
                constexpr int SPC = C::EPC / C::KPS;  // steps of a chunk
                const int d = (4 * (k / SPC) + cq) * C::EPC + (k % SPC) * C::KPS;
#pragma unroll
                for (int e = 0; e < C::KPS; e += 2) {
                    const float2 x = head < p.c.group ? *reinterpret_cast<const float2*>(qrow + head * HD + d + e)
                                                      : make_float2(0.0f, 0.0f);
                    raw[r][k * C::KPS + e] = x.x;
                    raw[r][k * C::KPS + e + 1] = x.y;
                }
            }
        }
    };
    auto begin_segment = [&]() {
        whole = cur.t == cur.span.t0;
#pragma unroll
        for (int r = 0; r < HR; ++r) {
            const float(&v)[C::NKS * C::KPS] = raw[r];
            float most = 0.0f;
#pragma unroll
            for (int k = 0; k < C::NKS * C::KPS; ++k)
                most = fmaxf(most, fabsf(v[k]));
            qs[r] = p.scale * 1.4426950408889634f;
            if constexpr (T == MUYO_KV_F32) {
#pragma unroll
                for (int i = 0; i < C::NKS * 2; ++i)
                    qf[i * HR + r] = __float_as_uint(v[i]);
            } else {
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                // the exponent of 2^14 / most, by the bits; 0 and what is not finite stay as they are
                const int e = (int)((__float_as_uint(most) >> 23) & 255u);
                const int up = most > 0.0f && e < 255 ? min(126, 127 + 14 - e) : 0;
                const float by = __uint_as_float((unsigned)(127 + max(up, -126)) << 23);
                qs[r] *= __uint_as_float((unsigned)(127 - max(up, -126)) << 23);
#pragma unroll
                for (int k = 0; k < C::NKS; ++k) {
                    uint32_t h0, l0, h1, l1;
                    split_half2(v[4 * k] * by, v[4 * k + 1] * by, h0, l0);
                    split_half2(v[4 * k + 2] * by, v[4 * k + 3] * by, h1, l1);
                    if constexpr (WIDE) {  // [k][hi | lo][4]: rows g, g + 8 of each
                        qf[k * 8 + r] = h0, qf[k * 8 + 2 + r] = h1;
                        qf[k * 8 + 4 + r] = l0, qf[k * 8 + 6 + r] = l1;
                    } else {
                        qf[k * 4] = h0, qf[k * 4 + 1] = l0, qf[k * 4 + 2] = h1, qf[k * 4 + 3] = l1;
                    }
                }
            }
            m[r] = -INFINITY;
            l[r] = 0.0f;
        }
#pragma unroll
        for (int n = 0; n < C::VPL; ++n)
#pragma unroll
            for (int e = 0; e < 2 * HR; ++e)
                o[n][e] = 0.0f;
    };

    // A tile's products into the running sums: the two halves' rows added up, or a row's sums of each head.
    const auto add_tile = [](float(&on)[2 * HR], const float(&alpha)[HR], const float(&acc)[4]) {
        const float2 upper = make_float2(acc[0], acc[1]), lower = make_float2(acc[2], acc[3]);
        const float2 first = fma2(make_float2(on[0], on[1]), make_float2(alpha[0], alpha[0]), WIDE ? upper : add2(upper, lower));
        on[0] = first.x, on[1] = first.y;
        if constexpr (WIDE) {
            const float2 second = fma2(make_float2(on[2], on[3]), make_float2(alpha[1], alpha[1]), lower);
            on[2] = second.x, on[3] = second.y;
        }
    };
    auto tile = [&](int stage) {
        const uint32_t ks = ring_at + stage * 2 * C::TILE, vs = ks + C::TILE;
        const unsigned long long mask = s_mask[warp][stage];
        // scores: s[j][2 r + e] is head g + 8 r, key 8 j + 2 cq + e
        float s[KT / 8][2 * HR];
#pragma unroll
        for (int j = 0; j < KT / 8; ++j) {
            // An F32 cache's steps in turns by two sums, the products with the remainders apart: short chains.
            constexpr int S = T == MUYO_KV_F32 && C::NKS > 2 ? 2 : 1;
            float acc[4], accs[S][4], less[S][4], least[S][4];
            const int row = j * 8 + g;
#pragma unroll
            for (int i = 0; i < C::NCH; ++i) {
                Chunk<C::CHB> ch;
                const int byte = (4 * i + cq) * C::CHB;
                ch.load(ks + row * C::RB + k_chunk<C::CPR>(row, byte >> 4) * 16 + (byte & 15));
                constexpr int SPC = C::EPC / C::KPS;
#pragma unroll
                for (int j2 = 0; j2 < SPC; ++j2) {
                    const int k = i * SPC + j2;
                    if constexpr (T == MUYO_KV_F32) {
                        uint32_t bh[2], bl[2], ah[4], al[4];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            split_tf32(__uint_as_float(ch.w[2 * j2 + e]), bh[e], bl[e]);
#pragma unroll
                            for (int r = 0; r < HR; ++r)
                                split_tf32(__uint_as_float(qf[(k * 2 + e) * HR + r]), ah[2 * e + r], al[2 * e + r]);
                        }
                        if constexpr (WIDE) {
                            k < S ? mma_tf32_first(less[k % S], al, bh[0], bh[1]) : mma_tf32(less[k % S], al, bh[0], bh[1]);
                            k < S ? mma_tf32_first(least[k % S], ah, bl[0], bl[1]) : mma_tf32(least[k % S], ah, bl[0], bl[1]);
                            k < S ? mma_tf32_first(accs[k % S], ah, bh[0], bh[1]) : mma_tf32(accs[k % S], ah, bh[0], bh[1]);
                        } else {
                            const uint32_t a[4] = {ah[0], al[0], ah[2], al[2]};
                            k < S ? mma_tf32_first(less[k % S], a, bl[0], bl[1]) : mma_tf32(less[k % S], a, bl[0], bl[1]);
                            k < S ? mma_tf32_first(accs[k % S], a, bh[0], bh[1]) : mma_tf32(accs[k % S], a, bh[0], bh[1]);
                        }
                    } else {
                        uint32_t b0, b1;
                        if constexpr (T == MUYO_KV_F16) {
                            b0 = ch.w[2 * j2], b1 = ch.w[2 * j2 + 1];
                        } else {
                            e4m3x4_half2(ch.w[j2], b0, b1);
                        }
                        if constexpr (WIDE) {
                            const uint32_t lo[4] = {qf[k * 8 + 4], qf[k * 8 + 5], qf[k * 8 + 6], qf[k * 8 + 7]};
                            const uint32_t hi[4] = {qf[k * 8], qf[k * 8 + 1], qf[k * 8 + 2], qf[k * 8 + 3]};
                            k == 0 ? mma_f16_first(acc, lo, b0, b1) : mma_f16(acc, lo, b0, b1);
                            mma_f16(acc, hi, b0, b1);
                        } else {
                            const uint32_t a[4] = {qf[k * 4], qf[k * 4 + 1], qf[k * 4 + 2], qf[k * 4 + 3]};
                            k == 0 ? mma_f16_first(acc, a, b0, b1) : mma_f16(acc, a, b0, b1);
                        }
                    }
                }
            }
            if constexpr (T == MUYO_KV_F32) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float low = less[0][e];
                    acc[e] = accs[0][e];
                    if constexpr (S > 1)
                        low += less[1][e], acc[e] += accs[1][e];
                    if constexpr (WIDE) {
                        low += least[0][e];
                        if constexpr (S > 1)
                            low += least[1][e];
                    }
                    acc[e] += low;
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if constexpr (WIDE) {
                    s[j][e] = acc[e] * qs[0];
                    s[j][2 + e] = acc[2 + e] * qs[1];
                } else {
                    s[j][e] = (acc[e] + acc[2 + e]) * qs[0];
                }
            }
        }
        constexpr unsigned long long ALL = KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1;
        if (mask != ALL) {
#pragma unroll
            for (int j = 0; j < KT / 8; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (!((mask >> (8 * j + 2 * cq + e)) & 1)) {
#pragma unroll
                        for (int r = 0; r < HR; ++r)
                            s[j][2 * r + e] = -INFINITY;
                    }
        }
        float alpha[HR];
#pragma unroll
        for (int r = 0; r < HR; ++r) {
            float most = -INFINITY;
#pragma unroll
            for (int j = 0; j < KT / 8; ++j)
                most = fmaxf(most, fmaxf(s[j][2 * r], s[j][2 * r + 1]));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            // rounded up, so that no weight passes 2^15: from 2^24 on most - 15 is between two F32 values, and a weight of 2^16
            // has no F16 halves
            const float mn = fmaxf(m[r], __fsub_ru(most, 15.0f));
            const float ref = mn == -INFINITY ? 0.0f : mn;  // nothing seen yet: every weight is 2^-inf
            alpha[r] = ex2(m[r] - ref);
            m[r] = mn;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < KT / 8; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    s[j][2 * r + e] = ex2(s[j][2 * r + e] - ref);
                    sum += s[j][2 * r + e];
                }
            l[r] = fmaf(l[r], alpha[r], sum);
        }
        // values: o[n] is channel (8 ic + 2 cq + e) VE + n % VE of chunk ic = n / VE
        if constexpr (T == MUYO_KV_F32) {
            uint32_t wh[KT / 8][4], wl[KT / 8][4];
#pragma unroll
            for (int j = 0; j < KT / 8; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int r = 0; r < HR; ++r)
                        split_tf32(s[j][2 * r + e], wh[j][2 * e + r], wl[j][2 * e + r]);
#pragma unroll
            for (int ic = 0; ic < C::NVC; ++ic) {
                Chunk<C::VCHB> v[KT / 8][2];
                const int byte = (8 * ic + g) * C::VCHB;
#pragma unroll
                for (int j = 0; j < KT / 8; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int row = 8 * j + 2 * cq + e;
                        v[j][e].load(vs + row * C::RB + v_chunk<C::CPR>(row, byte >> 4) * 16 + (byte & 15));
                    }
#pragma unroll
                for (int n = 0; n < C::VE; ++n) {
                    float acc[4];
#pragma unroll
                    for (int j = 0; j < KT / 8; ++j) {
                        uint32_t bh[2], bl[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            split_tf32(__uint_as_float(v[j][e].w[n]), bh[e], bl[e]);
                        if constexpr (WIDE) {
                            j == 0 ? mma_tf32_first(acc, wl[j], bh[0], bh[1]) : mma_tf32(acc, wl[j], bh[0], bh[1]);
                            mma_tf32(acc, wh[j], bl[0], bl[1]);
                            mma_tf32(acc, wh[j], bh[0], bh[1]);
                        } else {
                            const uint32_t a[4] = {wh[j][0], wl[j][0], wh[j][2], wl[j][2]};
                            j == 0 ? mma_tf32_first(acc, a, bl[0], bl[1]) : mma_tf32(acc, a, bl[0], bl[1]);
                            mma_tf32(acc, a, bh[0], bh[1]);
                        }
                    }
                    float(&on)[2 * HR] = o[ic * C::VE + n];
                    add_tile(on, alpha, acc);
                }
            }
        } else {
            uint32_t w[KT / 16][WIDE ? 8 : 4];
#pragma unroll
            for (int j = 0; j < KT / 16; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {  // keys 16 j + 8 h + 2 cq + {0, 1}
                    if constexpr (WIDE) {
#pragma unroll
                        for (int r = 0; r < 2; ++r)
                            split_half2(s[2 * j + h][2 * r], s[2 * j + h][2 * r + 1], w[j][2 * h + r], w[j][4 + 2 * h + r]);
                    } else {
                        split_half2(s[2 * j + h][0], s[2 * j + h][1], w[j][2 * h], w[j][2 * h + 1]);
                    }
                }
#pragma unroll
            for (int ic = 0; ic < C::NVC; ++ic) {
                Chunk<C::VCHB> v[KT / 16][4];
                const int byte = (8 * ic + g) * C::VCHB;
#pragma unroll
                for (int j = 0; j < KT / 16; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int row = 16 * j + 8 * (e >> 1) + 2 * cq + (e & 1);
                        v[j][e].load(vs + row * C::RB + v_chunk<C::CPR>(row, byte >> 4) * 16 + (byte & 15));
                    }
#pragma unroll
                for (int n = 0; n < C::VE; n += 2) {  // two channels of both keys of a pair from one word of each
                    float acc[2][4];
#pragma unroll
                    for (int j = 0; j < KT / 16; ++j) {
                        uint32_t b[2][2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if constexpr (T == MUYO_KV_F16) {
                                const uint32_t x = v[j][2 * h].w[n >> 1], y = v[j][2 * h + 1].w[n >> 1];
                                b[0][h] = __byte_perm(x, y, 0x5410), b[1][h] = __byte_perm(x, y, 0x7632);
                            } else {
                                const uint32_t x = v[j][2 * h].w[n >> 2], y = v[j][2 * h + 1].w[n >> 2];
                                e4m3x4_half2(__byte_perm(x, y, n & 2 ? 0x7362 : 0x5140), b[0][h], b[1][h]);
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            if constexpr (WIDE) {
                                const uint32_t lo[4] = {w[j][4], w[j][5], w[j][6], w[j][7]};
                                const uint32_t hi[4] = {w[j][0], w[j][1], w[j][2], w[j][3]};
                                j == 0 ? mma_f16_first(acc[e], lo, b[e][0], b[e][1]) : mma_f16(acc[e], lo, b[e][0], b[e][1]);
                                mma_f16(acc[e], hi, b[e][0], b[e][1]);
                            } else {
                                const uint32_t a[4] = {w[j][0], w[j][1], w[j][2], w[j][3]};
                                j == 0 ? mma_f16_first(acc[e], a, b[e][0], b[e][1]) : mma_f16(acc[e], a, b[e][0], b[e][1]);
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float(&on)[2 * HR] = o[ic * C::VE + n + e];
                        add_tile(on, alpha, acc[e]);
                    }
                }
            }
        }
    };

    // Writes the segment's result: to `out` when it is complete, else as a partial.
    auto end_segment = [&](float* partial) {
        float* dst = partial ? partial : out + cur.s * p.stride_out + (long long)cur.h * p.c.group * HD;
#pragma unroll
        for (int r = 0; r < HR; ++r) {
            const int head = g + 8 * r;
            float L = l[r], by = 1.0f;
            L += __shfl_xor_sync(0xffffffffu, L, 1);
            L += __shfl_xor_sync(0xffffffffu, L, 2);
            if (head < p.c.group) {
                if (partial) {
                    if (cq == 0) {
                        partial[C::ROWS * HD + head] = m[r];
                        partial[C::ROWS * HD + C::ROWS + head] = L;
                    }
                } else {
                    by = L > 0.0f ? __fdiv_rn(p.c.v_scale, L) : 0.0f;
                    if (lse && cq == 0)
                        lse[(size_t)cur.s * p.c.heads + cur.h * p.c.group + head] = paged_lse(m[r], L);
                }
#pragma unroll
                for (int ic = 0; ic < C::NVC; ++ic)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float* at = dst + head * HD + (8 * ic + 2 * cq + e) * C::VE;
                        if constexpr (C::VE >= 4) {
#pragma unroll
                            for (int n = 0; n < C::VE; n += 4)
                                *reinterpret_cast<float4*>(at + n) =
                                    make_float4(o[ic * C::VE + n][2 * r + e] * by, o[ic * C::VE + n + 1][2 * r + e] * by,
                                                o[ic * C::VE + n + 2][2 * r + e] * by, o[ic * C::VE + n + 3][2 * r + e] * by);
                        } else {
#pragma unroll
                            for (int n = 0; n < C::VE; ++n)
                                at[n] = o[ic * C::VE + n][2 * r + e] * by;
                        }
                    }
            }
        }
    };

    if (left > 0) {
        load_q();  // before the copies, which it would wait for
        look_up(true);
        int stage = 0, into = 0;
        bool fresh = true;  // a segment begins with the next tile
#pragma unroll 1
        for (int step = 1 - C::STAGES; left > 0; ++step) {
            if (ahead > 0)
                issue(into);
            copies_commit();
            into = into + 1 == C::STAGES ? 0 : into + 1;
            if (step < 0)
                continue;
            if (fresh)
                begin_segment();
            copies_wait<C::STAGES - 1>();
            __syncwarp();
            tile(stage);
            __syncwarp();  // every lane is done with the stage before it is filled again
            stage = stage + 1 == C::STAGES ? 0 : stage + 1;
            --left;
            const bool ends = cur.t + 1 == cur.span.t1;
            if (ends || left == 0) {
                if (!(whole && ends) && lane == 0) {
                    const int k = whole ? 2 : 0;
                    s_seg[warp][k] = cur.s, s_seg[warp][k + 1] = cur.h;
                    (whole ? s_last : s_first)[warp] = ends ? 2 : 1;
                    if (!ends && u1 == cta_end)
                        s_open = cur.span.t1 - cur.t - 1;
                }
                // a piece that begins here and is open goes to the ring, which is drained then
                end_segment(whole && ends ? nullptr : whole ? reinterpret_cast<float*>(ring) : first_part);
            }
            fresh = ends;
            if (left > 0) {
                cur.next(p, lens);
                if (ends)
                    load_q();
            }
        }
    }
    __syncthreads();

    // ---- the CTA's join ----
    // A group is a piece that begins here (or comes in, to warp 0) and the first pieces of the warps behind it, up to the
    // one where the segment ends.
    if (warp == 0) {
        const int k = lane - 1, w = max(k, 0);  // lane 0: what comes in; lane w + 1: what begins in warp w
        const bool is = lane <= W && (k < 0 ? s_first[0] != 0 : s_last[min(w, W - 1)] != 0);
        const unsigned groups = __ballot_sync(0xffffffffu, is);
        bool open = false;
        if (is) {
            bool ended = k < 0 && s_first[0] == 2;
            unsigned pieces = 1u << (k < 0 ? 0 : W + w);
#pragma unroll
            for (int v = 1; v < W; ++v)
                if (v > w && !ended) {
                    pieces |= s_first[v] ? 1u << v : 0u;
                    ended = s_first[v] == 2;
                }
            open = k >= 0 && !ended;  // begun in this CTA and open behind it: one group at most
            s_u.join.group[__popc(groups & ((1u << lane) - 1))] =
                PagedGroup{pieces, s_seg[w][k < 0 ? 0 : 2], s_seg[w][k < 0 ? 1 : 3], k < 0 ? 0 : ended ? -1 : 1};
            if (open) {
                const int to = shares.worker_of((unsigned)(cta_end + s_open - 1)) / W;
                descs[blockIdx.x] = PagedDesc{s_seg[w][2], s_seg[w][3], to - (int)blockIdx.x + 1, 0};
            }
        }
        if (!__any_sync(0xffffffffu, open) && lane == 0)
            descs[blockIdx.x] = PagedDesc{0, 0, 0, 0};
        if (lane == 0)
            s_groups = __popc(groups);
    }
    __syncthreads();
    const int rows = s_groups * p.c.group;
    // The pieces' weights 2^(m - M), in place of m, by 2 W lanes per row; M and L by the first of them.
    auto piece_at = [&](int b) -> float* {
        return reinterpret_cast<float*>(b < W ? paged_smem + (size_t)W * C::RING + (size_t)b * C::PART * 4
                                              : paged_smem + (size_t)(b - W) * C::RING);
    };
    constexpr int LANES = 2 * W;  // of a row
    float* s_row = reinterpret_cast<float*>(s_u.join.rows);
#pragma unroll 1
    for (int i = tid / LANES; i < (rows + 32 / LANES - 1) / (32 / LANES) * (32 / LANES); i += kPagedThreads / LANES) {
        const int k = min(i, rows - 1) / p.c.group, r = min(i, rows - 1) % p.c.group, b = lane % LANES;
        const bool in = (s_u.join.group[k].pieces >> b) & 1;
        float* at = piece_at(b) + C::ROWS * HD + r;
        float m1 = in ? at[0] : -INFINITY, l1 = in ? at[C::ROWS] : 0.0f, M = m1;
#pragma unroll
        for (int o2 = LANES / 2; o2 > 0; o2 >>= 1)
            M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o2));
        const float w = l1 > 0.0f ? ex2(m1 - M) : 0.0f;
        float L = l1 * w;
#pragma unroll
        for (int o2 = LANES / 2; o2 > 0; o2 >>= 1)
            L += __shfl_xor_sync(0xffffffffu, L, o2);
        if (i < rows) {
            if (in)
                at[0] = w;
            if (b == 0) {
                s_row[2 * i] = M;
                s_row[2 * i + 1] = L;
            }
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < rows * (HD / 4); i += kPagedThreads) {
        const int row = i / (HD / 4), d = i % (HD / 4) * 4;
        const int k = row / p.c.group, r = row % p.c.group;
        const PagedGroup group = s_u.join.group[k];
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
        for (unsigned bits = group.pieces; bits; bits &= bits - 1) {
            const float* at = piece_at(__ffs(bits) - 1);
            const float w = at[C::ROWS * HD + r];
            const float4 x = *reinterpret_cast<const float4*>(at + r * HD + d);
            v.x = fmaf(w, x.x, v.x), v.y = fmaf(w, x.y, v.y), v.z = fmaf(w, x.z, v.z), v.w = fmaf(w, x.w, v.w);
        }
        const float M = s_row[2 * row], L = s_row[2 * row + 1];
        float* dst = part + ((size_t)blockIdx.x * 2 + group.to) * C::PART + r * HD;
        if (group.to < 0) {
            const int h = group.kv_head * p.c.group + r;
            const float by = L > 0.0f ? __fdiv_rn(p.c.v_scale, L) : 0.0f;
            v.x *= by, v.y *= by, v.z *= by, v.w *= by;
            dst = out + group.seq * p.stride_out + (long long)h * HD;
            if (lse && d == 0)
                lse[(size_t)group.seq * p.c.heads + h] = paged_lse(M, L);
        } else if (d == 0) {
            dst[C::ROWS * HD - r * HD + r] = M;
            dst[C::ROWS * HD - r * HD + C::ROWS + r] = L;
        }
        *reinterpret_cast<float4*>(dst + d) = v;
    }
}

// Joins the segment that begins in CTA blockIdx.x of the kernel above and ends in another: its last partial and the
// first ones of the CTAs behind it. Four channels of a row per thread; threads to spare share the pieces.
constexpr int kJoinThreads = 512;
constexpr int kJoinPieces = 480;  // one per CTA at most

template <int HD, int ROWS>
__global__ void __launch_bounds__(kJoinThreads) k_paged_join(PagedAttnDev p, const float* part, const PagedDesc* descs,
                                                             float* out, float* lse)
{
    constexpr int PART = ROWS * (HD + 2), Q = HD / 4;
    __shared__ float s_w[ROWS][kJoinPieces];
    __shared__ float s_L[ROWS];
    __shared__ float4 s_sum[kJoinThreads];
    pdl_wait();
    pdl_trigger();
    const PagedDesc d = descs[blockIdx.x];
    if (d.pieces == 0)
        return;
    const int tid = threadIdx.x, lane = tid & 31, G = p.c.group;
    auto piece = [&](int i) { return part + ((size_t)blockIdx.x + i) * 2 * PART + (i == 0 ? PART : 0); };
    const int items = G * Q, ways = items >= kJoinThreads ? 1 : kJoinThreads / items;
    const int way = tid / items, item = tid % items;
    if (tid >> 5 < G) {  // a warp per row: the pieces' weights
        const int r = tid >> 5;
        float M = -INFINITY, L = 0.0f;
#pragma unroll 1
        for (int i = lane; i < d.pieces; i += 32)
            M = fmaxf(M, piece(i)[ROWS * HD + r]);
        M = warp_max(M);
#pragma unroll 1
        for (int i = lane; i < d.pieces; i += 32) {
            const float* at = piece(i) + ROWS * HD + r;
            const float l = at[ROWS], w = l > 0.0f ? ex2(at[0] - M) : 0.0f;
            s_w[r][i] = w;
            L = fmaf(l, w, L);
        }
        L = warp_sum(L);
        if (lane == 0) {
            s_L[r] = L;
            if (lse)
                lse[(size_t)d.seq * p.c.heads + d.kv_head * G + r] = paged_lse(M, L);
        }
    }
    __syncthreads();
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (way < ways) {
#pragma unroll 8
        for (int i = way; i < d.pieces; i += ways) {
            const float w = s_w[item / Q][i];
            const float4 x = *reinterpret_cast<const float4*>(piece(i) + item * 4);
            v.x = fmaf(w, x.x, v.x), v.y = fmaf(w, x.y, v.y), v.z = fmaf(w, x.z, v.z), v.w = fmaf(w, x.w, v.w);
        }
    }
    s_sum[tid] = v;
    __syncthreads();
    if (tid < items) {
#pragma unroll 1
        for (int i = 1; i < ways; ++i) {
            const float4 x = s_sum[i * items + tid];
            v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
        }
        const int r = item / Q;
        const float by = s_L[r] > 0.0f ? __fdiv_rn(p.c.v_scale, s_L[r]) : 0.0f;
        *reinterpret_cast<float4*>(out + d.seq * p.stride_out + (long long)(d.kv_head * G + r) * HD + item % Q * 4) =
            make_float4(v.x * by, v.y * by, v.z * by, v.w * by);
    }
}

static int paged_attention_prepare(const MuyoPagedAttentionParams* p, PagedAttnDev& d)
{
    MUYO_REQUIRE(p, "paged_attention: null parameter block");
    const int rc = paged_prepare(p->cache, "paged_attention", d.c);
    if (rc != MUYO_OK)
        return rc;
    MUYO_REQUIRE(p->seqs > 0 && p->seqs <= 1u << 28, "paged_attention: seqs must be in [1, 2^28]");
    MUYO_REQUIRE(p->table_stride > 0 && (uint64_t)p->cache.page_size * p->table_stride <= (uint64_t)1 << 30,
                 "paged_attention: table_stride %u must be positive, and a row at most 2^30 slots", p->table_stride);
    MUYO_REQUIRE(p->window <= (uint32_t)INT_MAX, "paged_attention: window %u exceeds INT32_MAX", p->window);
    // scores are formed in powers of two
    MUYO_REQUIRE(std::isfinite(p->scale * d.c.k_scale * 1.4426950408889634f),
                 "paged_attention: scale and scale * k_scale must be at most 2^127");
    const uint32_t row = p->cache.heads * p->cache.head_dim;
    d.stride_q = p->stride_q ? p->stride_q : row;
    d.stride_out = p->stride_out ? p->stride_out : row;
    MUYO_REQUIRE(d.stride_q >= row && d.stride_out >= row, "paged_attention: a row stride is below the row of %u", row);
    MUYO_REQUIRE((d.stride_q | d.stride_out) % 4 == 0, "paged_attention: row strides must be multiples of 4");
    // tiles hold 8 keys or more; the kernel rounds their number up to whole CTAs
    const uint64_t tiles = ((uint64_t)p->cache.page_size * p->table_stride / 8 + 1) * p->cache.kv_heads;
    if (tiles > (uint64_t)(INT_MAX - kPagedWarps) / p->seqs) {
        set_error("paged_attention: %u requests of rows of %u pages are more than 2^31 - 5 tiles", p->seqs, p->table_stride);
        return MUYO_EUNSUPPORTED;
    }
    d.seqs = (int)p->seqs, d.table_stride = (int)p->table_stride, d.window = (int)p->window;
    d.scale = p->scale * d.c.k_scale;
    d.page_shift = page_shift_of(d.c.page_size);
    return MUYO_OK;
}

// CTAs at most: three per SM, fewer when the tables could not hold a tile per warp.
static int paged_attention_ctas(const PagedAttnDev& d, int per_sm)
{
    const long long tiles = ((long long)d.table_stride * d.c.page_size / 8 + 1) * d.c.kv_heads;
    const long long most = (tiles * d.seqs + kPagedWarps - 1) / kPagedWarps;
    return (int)std::min({most, (long long)sm_count() * per_sm, (long long)kJoinPieces});
}

static size_t paged_attention_parts(const PagedAttnDev& d)
{
    return (size_t)paged_attention_ctas(d, 3) * 2 * (d.c.group > 8 ? 16 : 8) * (d.c.head_dim + 2) * sizeof(float);
}

template <int T, int HD, bool WIDE>
static int launch_paged_attention(const PagedAttnDev& d, const float* q, const void* k, const void* v, const int32_t* table,
                                  const int32_t* lens, float* out, float* lse, void* ws, void* stream)
{
    using C = PagedTile<T, HD, WIDE>;
    auto kernel = k_paged_attention<T, HD, WIDE>;
    static std::atomic<unsigned long long> allowed{0};
    MUYO_CUDA_TRY(allow_smem(kernel, C::SMEM, allowed));
    const int ctas = paged_attention_ctas(d, C::CTAS);
    PagedAttnDev e = d;
    e.one_page = d.c.page_size % C::KT == 0;
    float* part = static_cast<float*>(ws);
    PagedDesc* descs = reinterpret_cast<PagedDesc*>(static_cast<char*>(ws) + paged_attention_parts(d));
    MUYO_CUDA_TRY(launch_kernel(kernel, dim3(ctas), dim3(kPagedThreads), C::SMEM, as_stream(stream), true, e, q,
                                static_cast<const char*>(k), static_cast<const char*>(v), table, lens, out, lse, part, descs));
    MUYO_LAUNCH_CHECK();
    MUYO_CUDA_TRY(launch_kernel(k_paged_join<HD, C::ROWS>, dim3(ctas), dim3(kJoinThreads), 0, as_stream(stream), true, d,
                                part, descs, out, lse));
    MUYO_LAUNCH_CHECK();
    return MUYO_OK;
}

template <int T>
static int launch_paged_attention_dim(const PagedAttnDev& d, const float* q, const void* k, const void* v,
                                      const int32_t* table, const int32_t* lens, float* out, float* lse, void* ws,
                                      void* stream)
{
#define MUYO_PAGED_DIM(HD)                                                                                      \
    return d.c.group > 8 ? launch_paged_attention<T, HD, true>(d, q, k, v, table, lens, out, lse, ws, stream)   \
                         : launch_paged_attention<T, HD, false>(d, q, k, v, table, lens, out, lse, ws, stream)
    switch (d.c.head_dim) {
        case 16: MUYO_PAGED_DIM(16);
        case 32: MUYO_PAGED_DIM(32);
        case 64: MUYO_PAGED_DIM(64);
        default: MUYO_PAGED_DIM(128);
    }
#undef MUYO_PAGED_DIM
}

}  // namespace muyo

using namespace muyo;

extern "C" size_t muyo_cuda_paged_attention_workspace_size(const MuyoPagedAttentionParams* p)
{
    PagedAttnDev d{};
    if (!p || paged_attention_prepare(p, d) != MUYO_OK)
        return 0;
    return paged_attention_parts(d) + (size_t)paged_attention_ctas(d, 3) * sizeof(PagedDesc);
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
            return launch_paged_attention_dim<MUYO_KV_F32>(d, q, k_pool, v_pool, block_table, seq_lens, out, lse, workspace,
                                                           stream);
        case MUYO_KV_F16:
            return launch_paged_attention_dim<MUYO_KV_F16>(d, q, k_pool, v_pool, block_table, seq_lens, out, lse, workspace,
                                                           stream);
        default:
            return launch_paged_attention_dim<MUYO_KV_F8>(d, q, k_pool, v_pool, block_table, seq_lens, out, lse, workspace,
                                                           stream);
    }
}
