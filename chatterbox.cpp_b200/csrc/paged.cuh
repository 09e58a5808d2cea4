// paged.cuh — the paged K/V cache with shared prefixes (t3b_op_kv_plan,
// t3b_op_kv_append, t3b_op_attention_shared, t3b_op_attention_shared_prompt):
// kernels and the C entry points.  Included by t3b_abi.cu.
#pragma once

#include <cuda_bf16.h>
#include <type_traits>

// Error word of the paged operators on each device (read and cleared by
// t3b_op_check).  Kernels name it directly, so a launch needs no address
// look-up and no allocation.
static __device__ unsigned g_paged_err;

// ---------------------------------------------------------------------------
// t3b_op_kv_plan: block tables, slots and positions of a step
// ---------------------------------------------------------------------------
#define PG_PLAN_T 1024
#define PG_PLAN_MAXN 8192
#define PG_PLAN_CLUSTER 8
#define PG_PLAN_ROWS 16384   // from this many rows on a kernel of its own fills them in

// exclusive prefix sums of two 64-bit values over the CTA; ta and tb get the sums
__device__ __forceinline__ void pg_scan2(unsigned long long & a, unsigned long long & b, unsigned long long (*red)[2],
                                         unsigned long long & ta, unsigned long long & tb) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    unsigned long long ia = a, ib = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long xa = __shfl_up_sync(0xffffffffu, ia, o), xb = __shfl_up_sync(0xffffffffu, ib, o);
        if (lane >= o) { ia += xa; ib += xb; }
    }
    __syncthreads();   // red is reused
    if (lane == 31) { red[w][0] = ia; red[w][1] = ib; }
    __syncthreads();
    const bool on = lane < (int) (blockDim.x >> 5);
    unsigned long long va = on ? red[lane][0] : 0ull, vb = on ? red[lane][1] : 0ull;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long xa = __shfl_up_sync(0xffffffffu, va, o), xb = __shfl_up_sync(0xffffffffu, vb, o);
        if (lane >= o) { va += xa; vb += xb; }
    }
    ta = __shfl_sync(0xffffffffu, va, 31);
    tb = __shfl_sync(0xffffffffu, vb, 31);
    const unsigned long long ba = __shfl_sync(0xffffffffu, va, (w + 31) & 31), bb = __shfl_sync(0xffffffffu, vb, (w + 31) & 31);
    a = (w ? ba : 0ull) + ia - a;
    b = (w ? bb : 0ull) + ib - b;
}

// last index i of the non-decreasing at[0 .. n) with at[i] <= x (at[0] = 0)
__device__ __forceinline__ int pg_find(const int * at, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (at[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

// Rows r0 .. r0 + E - 1 of the row maps: one bisection of s_row (n + 1 first
// rows) and, mostly, one page id for all of them.  start(i): the own tokens
// before the step; page(i, b): table entry b of request i.
template <int E, class Start, class Page>
__device__ __forceinline__ void pg_plan_rows(const t3b_kv_plan & p, int n, int nrow, int lg, int r0, const int * s_row, Start start, Page page) {
    int req[E], pos[E], slot[E];
    int i = r0 < nrow ? pg_find(s_row, n, r0) : 0, have = -1, id = -1, ln = r0 < nrow ? start(i) : 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int r = r0 + e;
        req[e] = pos[e] = slot[e] = -1;
        if (r >= nrow) continue;
        if (r >= s_row[i + 1]) {
            do ++i; while (r >= s_row[i + 1]);
            ln = start(i);
            have = -1;
        }
        req[e] = i;
        pos[e] = ln + (r - s_row[i]);
        const int blk = pos[e] >> lg;
        if (blk != have) {
            have = blk;
            id = page(i, blk);
            if (id < 0 || id > (0x7fffffff - (1 << lg) + 1) >> lg) {   // the slot would not fit 31 bits
                atomicOr(&g_paged_err, T3B_DEVERR_PAGE);
                id = -1;
            }
        }
        if (id >= 0) slot[e] = (id << lg) + (pos[e] & ((1 << lg) - 1));
    }
    if (((((uintptr_t) p.row_req) | ((uintptr_t) p.row_pos) | ((uintptr_t) p.slots)) & 15) == 0 && E == 4 && r0 + 4 <= p.rows_cap) {
        if (p.row_req) *(int4 *) (p.row_req + r0) = make_int4(req[0], req[E / 4], req[E / 2], req[E - 1]);
        if (p.row_pos) *(int4 *) (p.row_pos + r0) = make_int4(pos[0], pos[E / 4], pos[E / 2], pos[E - 1]);
        if (p.slots) *(int4 *) (p.slots + r0) = make_int4(slot[0], slot[E / 4], slot[E / 2], slot[E - 1]);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (r0 + e >= p.rows_cap) break;
            if (p.row_req) p.row_req[r0 + e] = req[e];
            if (p.row_pos) p.row_pos[r0 + e] = pos[e];
            if (p.slots) p.slots[r0 + e] = slot[e];
        }
    }
}

// The row maps of a large step, over the whole GPU, from what the plan kernel
// left: a step of 2048 requests and 200 000 rows took 18 us in one cluster and
// takes 12 so.
__global__ __launch_bounds__(256) void kv_plan_rows_kernel(t3b_kv_plan p) {
    extern __shared__ int pg_sm[];
    const int n = p.n, lg = __ffs(p.page_size) - 1;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int i = threadIdx.x; i <= n; i += 256) pg_sm[i] = __ldcg(p.row_start + i);
    __syncthreads();
    const int r0 = 4 * (blockIdx.x * 256 + threadIdx.x);
    if (r0 >= p.rows_cap) return;
    auto start = [&](int i) { return p.len_out ? __ldcg(p.len_out + i) - (pg_sm[i + 1] - pg_sm[i]) : __ldcg(p.len + i); };
    auto page = [&](int i, int blk) { return __ldcg(p.table + (size_t) i * p.max_blocks + blk); };
    pg_plan_rows<4>(p, n, pg_sm[n], lg, r0, pg_sm, start, page);
}

// who fills in the row maps: nobody (none is wanted), the plan kernel, or kv_plan_rows_kernel
enum class PgRowMaps { none, here, apart };

// One cluster.  Every CTA scans all requests (a few KB), so all of them know
// each request's first row, first new page and first returned page and come
// to the same verdict; the returned pages, the new pages and the rows are
// then flattened and shared out over the cluster's threads, each finding its
// request by bisection in shared memory.  A cluster barrier separates what
// reads the old state (lengths, n_free, the released rows of the table) from
// what overwrites it, which is what lets a slot be released and admitted in
// one step and the outputs be the inputs' own buffers.  Bound by latency: a
// launch, two trips to memory and the scan, 3.9 us for 64 requests (a graph
// node that does nothing takes 2).
__global__ __launch_bounds__(PG_PLAN_T, 1) void kv_plan_kernel(t3b_kv_plan p, PgRowMaps maps) {
    extern __shared__ int pg_sm[];
    __shared__ unsigned long long red[32][2];
    int * s_len = pg_sm, * s_take = s_len + p.n, * s_back = s_take + p.n, * s_row = s_back + p.n;   // s_row: n + 1
    const int tid = threadIdx.x, T = blockDim.x, n = p.n, P = p.page_size, lg = __ffs(P) - 1;
    unsigned rank, csize;
    if (maps == PgRowMaps::apart) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(csize));
    const long long cap = (long long) p.max_blocks * P;
    const int F = *p.n_free;
    unsigned long long rows = 0, pages = 0;   // pages: new ones in the low half, returned ones in the high
    int bad = 0;
    int ln_next = 0, ad_next = 0, rl_next = 0;
    if (tid < n) { ln_next = p.len[tid]; ad_next = p.add[tid]; if (p.release) rl_next = p.release[tid]; }
    for (int t0 = 0; t0 < n; t0 += T) {
        const int i = t0 + tid;
        int ln = ln_next, ad = ad_next, rl = rl_next;
        if (i + T < n) {                   // in flight during this tile's scan
            ln_next = p.len[i + T]; ad_next = p.add[i + T];
            if (p.release) rl_next = p.release[i + T];
        }
        if (i >= n) {
            ln = ad = rl = 0;
        } else {
            if (ln < 0 || ad < 0 || rl < 0 || (long long) ln + ad > cap || rl > cap || (rl > 0 && ln > 0)) {
                bad = 1; ln = ad = rl = 0;
            }
        }
        const unsigned take = (unsigned) (((ln + ad + P - 1) >> lg) - ((ln + P - 1) >> lg)), back = (unsigned) ((rl + P - 1) >> lg);
        unsigned long long a = (unsigned long long) ad, b = ((unsigned long long) back << 32) | take, ta, tb;
        pg_scan2(a, b, red, ta, tb);
        a += rows; b += pages;
        if (i < n) {
            s_len[i] = ln;
            s_row[i] = (int) min(a, 0x7fffffffull);
            s_take[i] = (int) (unsigned) b;
            s_back[i] = (int) (b >> 32);
        }
        rows += ta; pages += tb;
    }
    const int take_n = (int) (unsigned) pages, back_n = (int) (pages >> 32);
    const bool fits = F >= 0 && F <= p.free_cap && (long long) F + back_n <= p.free_cap && take_n <= F + back_n;
    const bool over = rows > (unsigned long long) p.rows_cap;
    bad = __syncthreads_or(bad);
    const bool ok = !bad && fits && !over;
    const int nrow = ok ? (int) rows : 0;
    if (tid == 0) s_row[n] = nrow;                 // read after the cluster's barrier
    const int me = (int) rank * T + tid, all = (int) csize * T;
    if (ok)   // returned pages, on top of the stack
        for (int k = me; k < back_n; k += all) {
            const int i = pg_find(s_back, n, k);
            p.free_pages[F + k] = p.table[(size_t) i * p.max_blocks + (k - s_back[i])];
        }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    const int top = F + back_n;
    if (ok)   // new pages
        for (int k = me; k < take_n; k += all) {
            const int i = pg_find(s_take, n, k);
            p.table[(size_t) i * p.max_blocks + ((s_len[i] + P - 1) >> lg) + (k - s_take[i])] = p.free_pages[top - 1 - k];
        }
    if (maps == PgRowMaps::here) {
        auto page = [&](int i, int blk) {
            const int held = (s_len[i] + P - 1) >> lg;
            return blk < held ? p.table[(size_t) i * p.max_blocks + blk] : p.free_pages[top - 1 - (s_take[i] + blk - held)];
        };
        auto start = [&](int i) { return s_len[i]; };
        if (p.rows_cap <= all) {                   // a thread for each: the shortest way
            if (me < p.rows_cap) pg_plan_rows<1>(p, n, nrow, lg, me, s_row, start, page);
        } else {
            for (int r0 = 4 * me; r0 < p.rows_cap; r0 += 4 * all) pg_plan_rows<4>(p, n, nrow, lg, r0, s_row, start, page);
        }
    }
    for (int i = me; i < n; i += all) {
        p.row_start[i] = ok ? s_row[i] : 0;
        if (p.len_out) {
            if (ok) p.len_out[i] = s_len[i] + s_row[i + 1] - s_row[i];
            else if (p.len_out != p.len) p.len_out[i] = p.len[i];
        }
    }
    if (me == 0) {
        p.row_start[n] = nrow;
        *p.n_free_out = ok ? top - take_n : F;
        if (!ok) atomicOr(&g_paged_err, (bad ? T3B_DEVERR_POS : 0u) | (fits ? 0u : T3B_DEVERR_FULL) | (over ? T3B_DEVERR_FULL : 0u));
    }
}

// ---------------------------------------------------------------------------
// t3b_op_kv_append: rows of K and V into their pages
// ---------------------------------------------------------------------------
struct PgAppendArgs {
    void * k, * v;
    long long page_stride;
    const void * ks, * vs;
    long long stride;
    const int * slots;
    int rows, n_slots, n_kv_head, page_log2, dim_log2;
};

template <class T> __device__ __forceinline__ T pg_from(float x);
template <> __device__ __forceinline__ __half pg_from<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 pg_from<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ float pg_from<float>(float x) { return x; }
__device__ __forceinline__ float pg_to(__half x) { return __half2float(x); }
__device__ __forceinline__ float pg_to(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float pg_to(float x) { return x; }

// eight elements of a source row as 16 bytes of the cache's type
template <class S, class T>
__device__ __forceinline__ uint4 pg_pack8(const S * src) {
    if (sizeof(S) == 2) return __ldg((const uint4 *) src);
    const float4 a = __ldg((const float4 *) src), b = __ldg((const float4 *) src + 1);
    union { T t[8]; uint4 u; } r;
    r.t[0] = pg_from<T>(a.x); r.t[1] = pg_from<T>(a.y); r.t[2] = pg_from<T>(a.z); r.t[3] = pg_from<T>(a.w);
    r.t[4] = pg_from<T>(b.x); r.t[5] = pg_from<T>(b.y); r.t[6] = pg_from<T>(b.z); r.t[7] = pg_from<T>(b.w);
    return r.u;
}

// A thread moves eight elements of K and the same eight of V, U times over.
// Bound by HBM.  U = 2 puts both pieces' loads in flight before the first
// store: 20001 rows of 8 x 128 bf16 26.0 to 26.4 us (6.2 to 6.3 TB/s, 0.95 to
// 0.97 of the copy rate) against 26.7 with one; a call that does not fill the GPU twice keeps one
// (128 rows of 16 x 64 f32: 2.1 us against 2.5).
template <class S, class T, int U>
__global__ __launch_bounds__(256) void kv_append_kernel(PgAppendArgs a) {
    const int wlog = a.dim_log2 - 3, per_row = a.n_kv_head << wlog;   // 16-byte chunks of a head / of a row
    const long long total = (long long) a.rows * per_row;
    const long long x0 = (long long) blockIdx.x * (256 * U) + threadIdx.x;
    uint4 kk[U], vv[U];
    long long dst[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long x = x0 + u * 256;
        dst[u] = -1;
        if (x >= total) continue;
        const int row = (int) (x / per_row), c = (int) (x - (long long) row * per_row);
        const int slot = __ldg(a.slots + row);
        if (slot < 0) continue;
        if (slot >= a.n_slots) { if (c == 0) atomicOr(&g_paged_err, T3B_DEVERR_PAGE); continue; }
        const int h = c >> wlog;
        const long long src = (long long) row * a.stride + ((long long) c << 3);
        dst[u] = (long long) (slot >> a.page_log2) * a.page_stride +
                 ((((long long) h << a.page_log2) + (slot & ((1 << a.page_log2) - 1))) << a.dim_log2) +
                 ((c & ((1 << wlog) - 1)) << 3);
        kk[u] = pg_pack8<S, T>((const S *) a.ks + src); vv[u] = pg_pack8<S, T>((const S *) a.vs + src);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (dst[u] >= 0) {
            *(uint4 *) ((T *) a.k + dst[u]) = kk[u];
            *(uint4 *) ((T *) a.v + dst[u]) = vv[u];
        }
}

// ---------------------------------------------------------------------------
// attention over shared prefixes and own pages
// ---------------------------------------------------------------------------
struct PgAttn {
    const void * k, * v;
    const void * q;
    void * out;
    long long page_stride, q_stride, out_stride;
    const int * len, * table, * row_start, * prefix_start, * prefix_len, * prefix_table;
    int n, rows, n_head, n_kv_head, group, page_log2, n_pages, max_blocks, n_prefix, prefix_max_blocks;
    float scale;
    bool pass;      // own keys are more than L2 holds: they pass through it
    float * part;   // own parts of a decode batch with prefixes: [n][n_head][D + 4] floats, (O, max, sum)
};

// the prefix whose range holds request i, or -1
__device__ __forceinline__ int pg_prefix_of(const PgAttn & a, int i) {
    int lo = 0, hi = a.n_prefix;   // prefix_start is non-decreasing: bisect for the last start <= i
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(a.prefix_start + mid) <= i) lo = mid + 1; else hi = mid;
    }
    if (lo == 0 || i >= __ldg(a.prefix_start + lo)) return -1;
    return lo - 1;
}

// One row and head by one warp, key by key in 32 bits: lane x ends with
// elements x * D / 32 .. of the output.  The tiled prompt kernel comes here
// for rows whose output is not finite: a NaN or infinity in the V of a later
// token that the row does not see meets a probability of zero in its tile.
// Rows that do see it come here too.  That is dear, about 1.4 us a key and warp:
// one NaN in the V of a shared prefix takes 8 chunks of 300 to 2000 tokens from
// 0.34 to 56 ms and 16 text prompts from 24 us to 4.4 ms.
template <class QT, class CT, int D>
__device__ __noinline__ void pg_row_slow(const PgAttn & a, const QT * q, int i, int px, int plen, int own, int kvh, float (&o)[D / 32]) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    float qv[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) { qv[e] = pg_to(q[lane * E + e]); o[e] = 0.0f; }
    for (int j = 0; j < plen + own; ++j) {
        const int t = j < plen ? j : j - plen;
        const int id = __ldg((j < plen ? a.prefix_table + (long long) px * a.prefix_max_blocks : a.table + (long long) i * a.max_blocks) +
                             (t >> a.page_log2));
        if ((unsigned) id >= (unsigned) a.n_pages) continue;
        const long long off = (long long) id * a.page_stride +
                              (((long long) kvh << a.page_log2) + (t & ((1 << a.page_log2) - 1))) * D + lane * E;
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) s = fmaf(qv[e], pg_to(((const CT *) a.k)[off + e]), s);
        s = warp_sum(s) * a.scale;
        // a NaN score is no maximum (fmaxf passes it over) but has to reach l and o, also before the first finite one
        const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.0f : expf(m - mn);
        const float p = s == -INFINITY ? 0.0f : expf(s - (mn == -INFINITY ? 0.0f : mn));
        l = l * c + p;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * c + p * pg_to(((const CT *) a.v)[off + e]);
        m = mn;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = l == 0.0f ? 0.0f : o[e] / l;
}

// ---- decode: one query token per request -----------------------------------
//
// Bound by HBM: each own key and value is read once and meets group (1 to 16)
// queries.  One CTA (or a cluster of them, each with a range of the keys) per
// (request, kv head); its four warps take 16-key tiles in turn, each with its
// own ring of cp.async stages, so no barrier stands between a tile's arrival
// and its use.  The arithmetic is mma.sync m16n8k16 with the group's queries
// as the 16 rows (there are too few of them for a 128-row tcgen05 tile):
// S = Q K^T comes out in the layout in which P enters P V, so the softmax
// stays in registers.  F32 queries take two rows, hi and lo, of 11 bits each
// (K and V are exact in f16), and so do their probabilities.
// The tensor cores cut their 32-bit sums off instead of rounding them, always
// towards zero: one accumulator over 8000 keys shrank F32 outputs by 2.2e-6 and
// left them 2.5e-6 off (2-norm).  So the MMAs of P V start from zero and each
// 16-key tile is added with rounding, its hi and lo rows to one sum (3.7e-7 at
// 64 dimensions, 4.3e-7 at 128).  That takes half the registers (16 bits x 128
// dimensions spilled 44 bytes before) and little time: 64 CFG streams 56.0 us
// before and 56.1 since, 256 short answers 53.8 and 53.2, 192 long requests
// 296.3 and 296.2, F32 groups of 16 heads 43.4 and 44.2.  Groups above 8 of
// 16-bit queries, whose outputs are rounded to 11 or 8 bits, keep
// the MMA's own sum, and round their probabilities to those bits once: both
// halves of a tile hold queries, and a lo part would take a second MMA.
//
// Four warps and 48 (64 dimensions) or 64 KB a CTA let four or three CTAs share
// an SM, with about 100 KB in flight: 192 requests of 500 to 4000 keys (f16, 8 x
// 128, prefix apart) run at 6.4 TB/s, 0.98 of the copy rate, in a short run and
// at 5.8 in a long one, under the power cap; 128 of 88 to 1088 (f32, 16 x 64) at
// 5.6 (5.2 with the call's cost), where a quarter of a CTA's 12 us goes to its
// first loads and its last join.  Two warps a CTA, deeper rings and a cluster
// for every unit were slower (58 us became 61 to 96), and so were CTAs that take
// over units which have not started (clusterlaunchcontrol), with the next
// unit's first keys under way during the join (56 became 63): they leave the
// SMs together at the end, where the tile kernel could have begun.
#define PD_WARPS 4
#define PD_TK 16                // keys of a tile
#define PD_LAZY 8.0f            // a row is rescaled when its maximum grew by 2^8 or more

template <class CT> struct PgBias { static constexpr float v = 0.0f; };
// f16 probabilities are held times 2^7: with the lazy maximum they stay below 2^15, and what
// falls under f16's normal range is 2^-21 of the largest or less
template <> struct PgBias<__half> { static constexpr float v = 7.0f; };

__device__ __forceinline__ float pg_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void pg_cp16(unsigned dst, const void * src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void pg_cp16(unsigned dst, const void * src, unsigned long long policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
}
__device__ __forceinline__ void pg_ldm4(unsigned (&r)[4], unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void pg_ldm4t(unsigned (&r)[4], unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <class CT>
__device__ __forceinline__ void pg_mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    if (std::is_same<CT, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two floats as a pair of the cache's type, the first in the low half
template <class CT> __device__ __forceinline__ unsigned pg_pack2(float x, float y);
template <> __device__ __forceinline__ unsigned pg_pack2<__half>(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *(const unsigned *) &h;
}
template <> __device__ __forceinline__ unsigned pg_pack2<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *(const unsigned *) &h;
}
// x and y as hi + lo pairs of f16: hi is x rounded, lo what that lost
__device__ __forceinline__ void pg_split2(float x, float y, unsigned & hi, unsigned & lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *(const unsigned *) &h;
    lo = *(const unsigned *) &l;
}
// the same for bf16
__device__ __forceinline__ void pg_split2_bf16(float x, float y, unsigned & hi, unsigned & lo) {
    hi = pg_pack2<__nv_bfloat16>(x, y);
    lo = pg_pack2<__nv_bfloat16>(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u));
}
// The power of two by which an F32 query row is divided before it is split:
// it brings the row's largest element to [2^8, 2^9), so that neither part
// leaves f16's range.  Zero and non-finite rows keep their values.
__device__ __forceinline__ int pg_row_exp(float mx) {
    if (!(mx > 0.0f) || mx > 3.0e38f) return 0;
    return max(-100, (int) ((__float_as_uint(mx) >> 23) & 255u) - 127 - 8);
}
__device__ __forceinline__ float pg_pow2(int e) { return __uint_as_float((unsigned) (e + 127) << 23); }   // -126 <= e <= 127

__device__ __forceinline__ void pg_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// float `p` of this CTA's shared memory, read from the cluster's CTA `rank`
__device__ __forceinline__ float pg_dsm(const float * p, unsigned rank) {
    unsigned a = (unsigned) __cvta_generic_to_shared(p), r;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(r) : "memory");
    return v;
}

// four floats like that, 16-byte aligned
__device__ __forceinline__ void pg_dsm4(float (&v)[4], const float * p, unsigned rank) {
    unsigned a = (unsigned) __cvta_generic_to_shared(p), r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(r) : "memory");
}
// four values, rounded to the row's type, in one store
__device__ __forceinline__ void pg_store4(float * p, const float (&v)[4]) { *(float4 *) p = make_float4(v[0], v[1], v[2], v[3]); }
template <class T> __device__ __forceinline__ void pg_store4(T * p, const float (&v)[4]) {
    *(uint2 *) p = make_uint2(pg_pack2<T>(v[0], v[1]), pg_pack2<T>(v[2], v[3]));
}

__host__ __device__ constexpr int pd_stages(int D) { return D == 64 ? 3 : 2; }
__host__ __device__ constexpr int pd_smem(int D) { return PD_WARPS * pd_stages(D) * 2 * PD_TK * D * 2; }

// grid = (splits, n_kv_head, n), clusters of `splits` CTAs, 128 threads
// MT: tiles of 16 rows; RH: their 8-row halves that hold queries of their own
// (F32: one; 16-bit: one up to 8 queries, then two).  With one, the other half
// takes the lo parts: F32's of the queries, and for every type those of the
// probabilities, which an MMA that runs anyway brings down from a rounding to
// 11 or 8 bits to one of 22 or 16.
template <class QT, class CT, int D, int MT, int RH>
__global__ __launch_bounds__(32 * PD_WARPS, MT == 1 ? (D == 64 ? 4 : 3) : 1) void attn_shared_decode_kernel(PgAttn a) {
    constexpr bool F32 = sizeof(QT) == 4;
    constexpr int RPM = 8 * RH;                    // queries of an M tile
    constexpr int NS = pd_stages(D), KS = D / 16, CH = D / 8;
    constexpr int TILE = PD_TK * D * 2;            // bytes of a K or a V tile
    constexpr float BIAS = PgBias<CT>::v;
    extern __shared__ __align__(128) unsigned char pd_sm[];
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    const int i = blockIdx.z, h = blockIdx.y, rank = blockIdx.x, nrank = gridDim.x, g = a.group;

    if (a.part) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // One trip to memory for the length, the prefix (up to 32 of them) and,
    // where the tile kernel has the prefix and no cluster splits the keys, the
    // pages of the warp's first tiles; another for the first keys.
    const int len = __ldg(a.len + i);
    int px = -1, plen = 0, early = -1;
    const bool first = nrank == 1 && (a.part || a.n_prefix == 0);
    if (first) {
        const int blk = ((w + (lane >> 1) * PD_WARPS) * PD_TK + (lane & 1) * 8) >> a.page_log2;
        if (blk < a.max_blocks) early = __ldg(a.table + (long long) i * a.max_blocks + blk);
    }
    unsigned qf[MT][KS][4];                        // queries as A fragments
    float2 qv[F32 ? MT : 1][KS][2];                // F32: as they come
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            if (F32) {
                const int r = mt * RPM + (lane >> 2);
                const float * q = (const float *) a.q + (long long) i * a.q_stride + (h * g + min(r, g - 1)) * D;
#pragma unroll
                for (int b = 0; b < 2; ++b) qv[mt][k][b] = *(const float2 *) (q + k * 16 + b * 8 + (lane & 3) * 2);
            } else {
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int r = mt * RPM + (lane >> 2) + (b & 1) * 8;
                    qf[mt][k][b] = (b & 1) < RH && r < g ? *(const unsigned *) ((const CT *) a.q + (long long) i * a.q_stride + (h * g + r) * D +
                                                                k * 16 + (b >> 1) * 8 + (lane & 3) * 2)
                                         : 0u;
                }
            }
        }
    if (a.n_prefix > 32) {
        px = pg_prefix_of(a, i);
        plen = px >= 0 ? __ldg(a.prefix_len + px) : 0;
    } else if (a.n_prefix > 0) {
        int beg = 0, end = 0, pl = 0;
        if (lane < a.n_prefix) {
            beg = __ldg(a.prefix_start + lane); end = __ldg(a.prefix_start + lane + 1); pl = __ldg(a.prefix_len + lane);
        }
        px = __ffs(__ballot_sync(0xffffffffu, beg <= i && i < end)) - 1;
        plen = px >= 0 ? __shfl_sync(0xffffffffu, pl, px) : 0;
    }
    if (len < 0 || len > (a.max_blocks << a.page_log2) || plen < 0 || plen > (a.prefix_max_blocks << a.page_log2)) {
        if (tid == 0) atomicOr(&g_paged_err, T3B_DEVERR_POS);
        if (a.part && rank == 0)                   // a negative sum: the tile kernel leaves the row as it is
            for (int q = tid; q < g; q += 32 * PD_WARPS) a.part[((long long) i * a.n_head + h * g + q) * (D + 4) + D + 1] = -1.0f;
        return;                                    // the whole cluster: it shares i
    }
    const int np = a.part ? 0 : (plen + PD_TK - 1) / PD_TK, total = np + (len + PD_TK - 1) / PD_TK;
    const int per = (total + nrank - 1) / nrank, t_beg = min(total, rank * per), t_end = min(total, t_beg + per);
    const int mine = t_end - t_beg > w ? (t_end - t_beg - w + PD_WARPS - 1) / PD_WARPS : 0;   // tiles of this warp

    // page ids of the warp's next 16 tiles, one per lane and 8-key half: tile
    // x's halves are lanes 2 (x % 16) and 2 (x % 16) + 1; -1 where no key is
    auto fetch_ids = [&](int x0, bool have) {
        const int x = x0 + (lane >> 1);
        int id = -1;
        if (x < mine) {
            const int t = t_beg + w + x * PD_WARPS;
            const bool pre = t < np;
            const int key = (pre ? t : t - np) * PD_TK + (lane & 1) * 8;
            if (key < (pre ? plen : len)) {
                id = have ? early
                          : __ldg((pre ? a.prefix_table + (long long) px * a.prefix_max_blocks : a.table + (long long) i * a.max_blocks) +
                                  (key >> a.page_log2));
                if ((unsigned) id >= (unsigned) a.n_pages) { atomicOr(&g_paged_err, T3B_DEVERR_PAGE); id = -1; }
            }
        }
        return id;
    };
    int ids = fetch_ids(0, first), ids_next = -1;

    const unsigned ring = (unsigned) __cvta_generic_to_shared(pd_sm) + w * NS * 2 * TILE;
    // keys that tile x's half holds (0 .. 8)
    auto half_keys = [&](int x, int half, int id) {
        const int t = t_beg + w + x * PD_WARPS;
        const int left = (t < np ? plen - t * PD_TK : len - (t - np) * PD_TK) - half * 8;
        return id < 0 ? 0 : min(8, left);
    };
    // lane's chunk of rows (lane / CH) + RPC c: where it lies in an 8-key half
    constexpr int RPC = 32 / CH, CPH = 8 / RPC;    // rows an instruction moves, instructions a half
    const int lrow = lane / CH, lch = lane % CH;
    unsigned spot[CPH];
#pragma unroll
    for (int c = 0; c < CPH; ++c) spot[c] = (c * RPC + lrow) * (D * 2) + ((lch ^ (c * RPC + lrow)) << 4);
    const long long lane_off = (((long long) h << a.page_log2) + lrow) * D + lch * 8;
    const int mask = (1 << a.page_log2) - 1;
    // Own keys that L2 could not hold anyway pass through it, which leaves the
    // tables, lengths, queries and prefixes there (64 CFG streams 57.7 -> 55.8
    // us); an unshared prefix is read again by the next request.
    unsigned long long once, again;
    asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(again));
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(once));
    if (!a.pass) once = again;
    auto issue = [&](int x, int my_ids, int slot) {   // tile x's K and V into a stage
        if (x < mine) {
            const int t = t_beg + w + x * PD_WARPS, key0 = (t < np ? t : t - np) * PD_TK;
            const unsigned st = ring + slot * 2 * TILE;
            const int left = (t < np ? plen : len) - key0;
            const unsigned long long policy = t < np ? again : once;
            int id[2];
            const CT * kp[2], * vp[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                id[b] = __shfl_sync(0xffffffffu, my_ids, 2 * (x & 15) + b);
                const long long off = (long long) max(id[b], 0) * a.page_stride + ((key0 + 8 * b) & mask) * D + lane_off;
                kp[b] = (const CT *) a.k + off; vp[b] = (const CT *) a.v + off;
            }
            if (left >= PD_TK && (id[0] | id[1]) >= 0) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int c = 0; c < CPH; ++c) {
                        pg_cp16(st + spot[c] + b * 8 * D * 2, kp[b] + c * RPC * D, policy);
                        pg_cp16(st + spot[c] + b * 8 * D * 2 + TILE, vp[b] + c * RPC * D, policy);
                    }
            } else {                               // keys past the end are zeros: 0 * NaN would stay
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int c = 0; c < CPH; ++c) {
                        const bool on = id[b] >= 0 && c * RPC + lrow + 8 * b < left;
                        pg_cp16(st + spot[c] + b * 8 * D * 2, on ? kp[b] + c * RPC * D : (const CT *) a.k, on);
                        pg_cp16(st + spot[c] + b * 8 * D * 2 + TILE, on ? vp[b] + c * RPC * D : (const CT *) a.v, on);
                    }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int x = 0; x < NS - 1; ++x) issue(x, ids, x);

    float sc[MT];                                  // what a score is multiplied by
    const float sl2 = a.scale * 1.4426950408889634f;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        if (F32) {
            float mx = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    float2 & v = qv[mt][k][b];
                    if (mt * RPM + (lane >> 2) >= g) v = make_float2(0.f, 0.f);
                    v.x *= sl2; v.y *= sl2;
                    mx = fmaxf(mx, fmaxf(fabsf(v.x), fabsf(v.y)));
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const int e = pg_row_exp(mx);
            const float f = pg_pow2(-e);
            sc[mt] = pg_pow2(e);
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int b = 0; b < 2; ++b) pg_split2(qv[mt][k][b].x * f, qv[mt][k][b].y * f, qf[mt][k][2 * b], qf[mt][k][2 * b + 1]);
        } else {
            sc[mt] = sl2;
        }
    }

    float o[MT][D / 8][2 * RH];                    // (RH == 1: hi and lo parts in one sum)
    float m[MT][RH], l[MT][RH];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int r = 0; r < RH; ++r) { m[mt][r] = -INFINITY; l[mt][r] = 0.0f; }
#pragma unroll
        for (int d = 0; d < D / 8; ++d)
#pragma unroll
            for (int e = 0; e < 2 * RH; ++e) o[mt][d][e] = 0.0f;
    }
    const int lr = lane & 7, mi = lane >> 3;       // ldmatrix: row of matrix mi
    int slot = 0, slot_in = NS - 1;                // stages of tiles x and x + NS - 1
    for (int x = 0; x < mine; ++x) {
        // stage x + NS - 1 is the one that tile x - 1 has left; its ids may be of the next batch
        const int xn = x + NS - 1;
        if ((x & 15) == 0) ids_next = fetch_ids(x + 16, false);
        issue(xn, (xn >> 4) == (x >> 4) ? ids : ids_next, slot_in);
        asm volatile("cp.async.wait_group %0;" ::"n"(NS - 1) : "memory");
        __syncwarp();
        const int n0 = half_keys(x, 0, __shfl_sync(0xffffffffu, ids, 2 * (x & 15)));
        const int n1 = half_keys(x, 1, __shfl_sync(0xffffffffu, ids, 2 * (x & 15) + 1));
        const unsigned st = ring + slot * 2 * TILE;
        float s[MT][2][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[mt][0][e] = s[mt][1][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            unsigned b[4];
            const int row = (mi >> 1) * 8 + lr, ch = k * 2 + (mi & 1);
            pg_ldm4(b, st + row * (D * 2) + ((ch ^ lr) << 4));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                pg_mma<CT>(s[mt][0], qf[mt][k], b[0], b[1]);
                pg_mma<CT>(s[mt][1], qf[mt][k], b[2], b[3]);
            }
        }
        unsigned p[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float z[2][2 * RH];                    // scores in units of log2: two keys for each half's row, twice
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < 2 * RH; ++e) z[nt][e] = (F32 ? s[mt][nt][e] + s[mt][nt][e + 2] : s[mt][nt][e]) * sc[mt];
            if (n0 + n1 < PD_TK) {
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int e = 0; e < 2 * RH; ++e)
                        if ((lane & 3) * 2 + (e & 1) >= (nt ? n1 : n0)) z[nt][e] = -INFINITY;
            }
            float top[RH];
            bool grow = false;
#pragma unroll
            for (int r = 0; r < RH; ++r) {
                float t = fmaxf(fmaxf(z[0][2 * r], z[0][2 * r + 1]), fmaxf(z[1][2 * r], z[1][2 * r + 1]));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
                top[r] = fmaxf(m[mt][r], t);
                grow |= top[r] > m[mt][r] + PD_LAZY;   // also from -inf
            }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int r = 0; r < RH; ++r) {
                    const float c = m[mt][r] == -INFINITY ? 0.0f : pg_exp2(m[mt][r] - top[r]);
                    m[mt][r] = top[r]; l[mt][r] *= c;
#pragma unroll
                    for (int d = 0; d < D / 8; ++d) { o[mt][d][2 * r] *= c; o[mt][d][2 * r + 1] *= c; }
                }
            }
#pragma unroll
            for (int r = 0; r < RH; ++r) {
                const float base = m[mt][r] == -INFINITY ? 0.0f : m[mt][r] - BIAS;
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    z[nt][2 * r] = pg_exp2(z[nt][2 * r] - base);
                    z[nt][2 * r + 1] = pg_exp2(z[nt][2 * r + 1] - base);
                    l[mt][r] += z[nt][2 * r] + z[nt][2 * r + 1];
                }
            }
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
                if (RH == 2) {
                    p[mt][2 * nt] = pg_pack2<CT>(z[nt][0], z[nt][1]);
                    p[mt][2 * nt + 1] = pg_pack2<CT>(z[nt][2 * RH - 2], z[nt][2 * RH - 1]);
                } else if (std::is_same<CT, __half>::value) {
                    pg_split2(z[nt][0], z[nt][1], p[mt][2 * nt], p[mt][2 * nt + 1]);
                } else {
                    pg_split2_bf16(z[nt][0], z[nt][1], p[mt][2 * nt], p[mt][2 * nt + 1]);
                }
            }
        }
#pragma unroll
        for (int d = 0; d < KS; ++d) {
            unsigned b[4];
            const int row = (mi & 1) * 8 + lr, ch = d * 2 + (mi >> 1);
            pg_ldm4t(b, st + TILE + row * (D * 2) + ((ch ^ lr) << 4));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    if constexpr (RH == 2) {
                        pg_mma<CT>(o[mt][2 * d + y], p[mt], b[2 * y], b[2 * y + 1]);
                    } else {                       // the tile's sum by itself, then added with rounding
                        float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        pg_mma<CT>(t, p[mt], b[2 * y], b[2 * y + 1]);
                        o[mt][2 * d + y][0] += t[0] + t[2]; o[mt][2 * d + y][1] += t[1] + t[3];
                    }
                }
            }
        }
        __syncwarp();
        if (++slot == NS) slot = 0;
        if (++slot_in == NS) slot_in = 0;
        if ((x & 15) == 15) ids = ids_next;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();

    // join the warps: each leaves (o, m, l) of the group's queries
    float * so = (float *) pd_sm;                  // [PD_WARPS][g][D]
    float * sm = so + PD_WARPS * g * D;            // [PD_WARPS][g]
    float * ss = sm + PD_WARPS * g;                // [PD_WARPS][g]
    float * co = ss + PD_WARPS * g;                // [g][D], the CTA's
    float * cm = co + g * D, * cl = cm + g;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < RH; ++r) {
            const int q = mt * RPM + (lane >> 2) + r * 8;
            l[mt][r] += __shfl_xor_sync(0xffffffffu, l[mt][r], 1);
            l[mt][r] += __shfl_xor_sync(0xffffffffu, l[mt][r], 2);
            if (q < g) {
#pragma unroll
                for (int d = 0; d < D / 8; ++d) {
                    *(float2 *) (so + (w * g + q) * D + d * 8 + (lane & 3) * 2) = make_float2(o[mt][d][2 * r], o[mt][d][2 * r + 1]);
                }
                if ((lane & 3) == 0) { sm[w * g + q] = m[mt][r]; ss[w * g + q] = l[mt][r]; }
            }
        }
    __syncthreads();
    // four elements a thread; an only CTA writes what it has, a cluster's
    // share the elements out once each has joined its warps
    constexpr int D4 = D / 4;
    QT * out = (QT *) a.out + (long long) i * a.out_stride + h * g * D;
    float * rec = a.part + ((long long) i * a.n_head + h * g) * (D + 4);
    auto finish = [&](int q, int c, float mx, float lv, float (&v)[4]) {
        if (a.part && px >= 0) {                   // the tile kernel adds the prefix's part
            pg_store4(rec + q * (D + 4) + c, v);
            if (c == 0) { rec[q * (D + 4) + D] = mx; rec[q * (D + 4) + D + 1] = lv; }
        } else {
            const float inv = lv == 0.0f ? 0.0f : 1.0f / lv;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= inv;
            pg_store4(out + q * D + c, v);
        }
    };
    for (int x = tid; x < g * D4; x += 32 * PD_WARPS) {
        const int q = x / D4, c = x % D4 * 4;
        float my[PD_WARPS], mx = -INFINITY, lv = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int y = 0; y < PD_WARPS; ++y) { my[y] = sm[y * g + q]; mx = fmaxf(mx, my[y]); }
#pragma unroll
        for (int y = 0; y < PD_WARPS; ++y) {
            const float f = my[y] == -INFINITY ? 0.0f : pg_exp2(my[y] - mx);
            const float4 u = *(const float4 *) (so + (y * g + q) * D + c);
            v[0] = fmaf(f, u.x, v[0]); v[1] = fmaf(f, u.y, v[1]); v[2] = fmaf(f, u.z, v[2]); v[3] = fmaf(f, u.w, v[3]);
            lv += f * ss[y * g + q];
        }
        if (nrank == 1) {
            finish(q, c, mx, lv, v);
        } else {
            pg_store4(co + q * D + c, v);
            if (c == 0) { cm[q] = mx; cl[q] = lv; }
        }
    }
    if (nrank == 1) return;
    pg_cluster_sync();
    for (int x = rank * 32 * PD_WARPS + tid; x < g * D4; x += nrank * 32 * PD_WARPS) {
        const int q = x / D4, c = x % D4 * 4;
        float my[8], ly[8], u[8][4], mx = -INFINITY, lv = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int y = 0; y < 8; ++y) {              // every CTA's in flight at once
            const int yy = min(y, nrank - 1);
            my[y] = y < nrank ? pg_dsm(cm + q, yy) : -INFINITY; ly[y] = pg_dsm(cl + q, yy);
            pg_dsm4(u[y], co + q * D + c, yy);
        }
#pragma unroll
        for (int y = 0; y < 8; ++y) mx = fmaxf(mx, my[y]);
#pragma unroll
        for (int y = 0; y < 8; ++y) {
            const float f = my[y] == -INFINITY ? 0.0f : pg_exp2(my[y] - mx);
            lv += f * ly[y];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = fmaf(f, u[y][e], v[e]);
        }
        finish(q, c, mx, lv, v);
    }
    pg_cluster_sync();                             // no CTA leaves while another reads its shared memory
}

// ---- many rows: tcgen05 tiles ------------------------------------------------
//
// 256 rows (token x head of the group) against 128-key tiles, for prompt
// chunks and for the prefix of a decode batch.  Compute-bound: 4 D operations
// per row and key.  Two 128-row tiles take turns: while the tensor cores work
// on one, eight warps (a thread per row) run the softmax of the other, so
// one K / V tile in shared memory serves 256 rows.
//
// A step of 256 x 128 (bf16, 128 dimensions) takes 3600 cycles: 32 MMAs of about
// 94 cycles (64 if shared memory fed them without a pause: an MMA of Q K^T reads
// 8 KB) and a softmax of 2500 per tile, half of it beside the other tile's.  Eight
// chunks of 300 to 2000 tokens (32 heads over 8) come to 860 TFLOP/s, 0.52 of
// the library GEMM's, in a short run and to 740 in a long one, 0.53 of what the
// GEMM keeps up under the power cap.  Measured and left: half of the exponentials as a
// polynomial on the FMA pipes (336 us became 366), P V and Q K^T interleaved by
// halves (339), output rows straight from registers (347).
//
// * Three loader warps bring K and V tiles into a ring in the 128-byte swizzle
//   (panels of 64 dimensions x 128 keys): a tile whose 128 keys are all there
//   by TMA, a box per page and panel; a ragged one by cp.async, 16 bytes at a
//   time, where the end (zero-filled: what lies behind it may be NaN) and absent
//   pages are a matter of each row's source address.  cp.async alone bounded
//   the loop: 1200 cycles to issue a 32 KB item, against a handful for TMA.
// * One thread issues the MMAs.  S = Q K^T (both K-major in shared memory) goes
//   to tensor memory; the softmax threads read it, write P over it, and P V
//   takes P from tensor memory and V as the MN-major operand.  MMAs of one
//   thread execute in issue order, so Q K^T of the next tile may follow P V
//   into the same columns.
// * O stays in tensor memory and is rescaled only when a row's maximum has
//   grown by 2^8 since the last time (as in the decode kernel).
// * F32 queries are two f16 parts, and so are their probabilities: two MMAs
//   into one accumulator, lo first: the tensor cores' sums are cut off, not
//   rounded, to 32 bits at every step, which costs least while they are small
//   (8000 keys x 128 dimensions 5.9e-7 off, 2-norm; hi first 1.0e-6).  Over 8000
//   keys in one accumulator that shrank O by 4.4e-6.  So F32 accumulates one
//   key tile at a time, and the softmax threads add the tiles; 16-bit outputs,
//   which are rounded by up to 2^-12 or 2^-9 in the end, keep the one sum.
// * 16-bit probabilities are rounded to the cache's type once, as they enter P V:
//   an error of the size of the output's own rounding (2-norm f16 2.9e-4 against
//   2.1e-4, bf16 2.3e-3 against 1.7e-3), where a lo part would double P V's
//   MMAs.  The row sum l is of the unrounded ones, in 32 bits.
// * The keys of a tile of rows may be split over a cluster (few rows, many
//   keys); its CTAs join their (O, max, sum) over distributed shared memory.
//
// Every wait has a limit (TF_SPIN polls); one that runs out ends the loops of
// its role, the others' waits run out in turn, and the call is reported.
#define PT_BN 128
#define PT_LOADERS 3
#define PT_PANEL (128 * 128)    // bytes of 128 rows x 64 elements

// NT: 128-row tiles of a CTA.  Warps 0 .. 4 NT - 1 softmax, then the MMA warp
// and three loaders: 384 threads of 168 registers, or 256 of 128 (two CTAs a
// SM), of which the softmax warps take 168 and leave the others 88.
__host__ __device__ constexpr int pt_threads(int NT) { return 128 * NT + 128; }
// (F32 x 128 dimensions has no NT = 2 and no room for a second CTA: tensor memory holds O twice, see below)
__host__ __device__ constexpr int pt_slots(int D, bool f32, int NT) { return NT == 1 && D == 128 && !f32 ? 2 : 4; }
__host__ __device__ constexpr int pt_tmem(int D, bool f32, int NT) { return NT == 2 || (f32 && D == 128) ? 512 : 256; }
__host__ __device__ constexpr int pt_q_bytes(int D, bool f32, int NT) { return NT * (f32 ? 2 : 1) * (D / 64) * PT_PANEL; }
// the epilogue's arrays lie over Q and the ring, which are larger
__host__ __device__ constexpr int pt_epilogue(int D, int NT) { return 128 * NT * ((D + 4) * 4 + 8 + 8 * 4 + 4 + 16 + 1); }
__host__ __device__ constexpr int pt_smem(int D, bool f32, int NT) {
    return 1024 + pt_q_bytes(D, f32, NT) + pt_slots(D, f32, NT) * (D / 64) * PT_PANEL;
}
static_assert(pt_smem(64, false, 1) >= 1024 + pt_epilogue(64, 1) && pt_smem(128, false, 1) >= 1024 + pt_epilogue(128, 1) &&
              pt_smem(64, false, 2) >= 1024 + pt_epilogue(64, 2) && pt_smem(128, false, 2) >= 1024 + pt_epilogue(128, 2), "epilogue");

#define PG_R8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define PG_W8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])
// 32 columns of this warp's 32 lanes (a row per thread); pg_tm_wait_ld before use
__device__ __forceinline__ void pg_tm_ld32(unsigned (&r)[32], unsigned addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : PG_R8(r, 0), PG_R8(r, 8), PG_R8(r, 16), PG_R8(r, 24) : "r"(addr) : "memory");
}
__device__ __forceinline__ void pg_tm_ld16(unsigned (&r)[16], unsigned addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : PG_R8(r, 0), PG_R8(r, 8) : "r"(addr) : "memory");
}
__device__ __forceinline__ void pg_tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pg_tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pg_tm_st16(const unsigned (&r)[16], unsigned addr) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(addr), PG_W8(r, 0), PG_W8(r, 8) : "memory");
}
__device__ __forceinline__ void pg_sts(unsigned addr, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// The MMA warp runs as a whole, so that descriptors and loop state stay in
// uniform registers, and `el` names the lane that issues.
__device__ __forceinline__ unsigned pg_elect() {
    unsigned el;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(el));
    return el;
}
__device__ __forceinline__ void pg_commit(unsigned bar, unsigned el) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(el) : "memory");
}
__device__ __forceinline__ bool pg_test(unsigned bar, unsigned parity) {
    unsigned done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done;
}
__device__ __forceinline__ void pg_arrive(unsigned bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Shared-memory descriptors: low word = address / 16 | leading offset / 16 <<
// 16, high word constant (8-row groups 1024 bytes apart, version 1, 128-byte
// swizzle; see tf_desc).  K-major operands have no leading offset; the
// MN-major V steps from panel to panel by it.
#define PT_DESC_HI ((1024u >> 4) | (1u << 14) | (2u << 29))
__device__ __forceinline__ void pg_mma_ss(unsigned d, unsigned a, unsigned b, unsigned idesc, unsigned acc, unsigned el) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "mov.b64 x, {%1, %6};\n\tmov.b64 y, {%2, %6};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}\n"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(el), "r"(PT_DESC_HI) : "memory");
}
__device__ __forceinline__ void pg_mma_ts(unsigned d, unsigned a, unsigned b, unsigned idesc, unsigned acc, unsigned el) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "mov.b64 y, {%2, %6};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}\n"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(el), "r"(PT_DESC_HI) : "memory");
}

// A tile of rows: rows lo .. of the `total` rows (token x head) of request i
// (prompt) or of prefix px's requests (its part of a decode batch), whose
// first token is row `row0` of q; lengths of the prefix (px < 0: none) and of
// the own keys (PARTIAL: none).
struct PgTile { int i, px, row0, total, lo, plen, len; };

// whether `cnt` rows from `beg` on are not among the call's `most`
__device__ __forceinline__ bool pg_range_wrong(int beg, int cnt, int most) { return beg < 0 || cnt < 0 || cnt > most - beg; }

// Reports row ranges that are out of range, wherever they are: a search for a
// tile ends at the tile's request and sees none behind it.  By T threads.
template <bool PARTIAL, int T>
__device__ void pg_check_ranges(const PgAttn & a, int tid) {
    const int n = PARTIAL ? a.n_prefix : a.n, most = PARTIAL ? a.n : a.rows;
    const int * start = PARTIAL ? a.prefix_start : a.row_start;
    bool bad = false;
#pragma unroll 4
    for (int x = tid; x < n; x += T) {
        const int beg = __ldg(start + x);
        bad |= pg_range_wrong(beg, __ldg(start + x + 1) - beg, most);
    }
    if (bad) atomicOr(&g_paged_err, T3B_DEVERR_POS);
}

// The z-th tile of ROWS rows over all requests (prompt) or prefixes, found by one
// warp; false past the last one.  Requests whose rows are out of range are
// passed over (pg_check_ranges reports them).  What the tile needs of its
// request is loaded beside the starts, and up to 32 prefixes beside those: one
// trip to memory for every 32 requests up to the tile's.
template <bool PARTIAL, int ROWS>
__device__ bool pg_find_tile(const PgAttn & a, int z, PgTile & t) {
    const int lane = threadIdx.x & 31, n = PARTIAL ? a.n_prefix : a.n;
    const int * start = PARTIAL ? a.prefix_start : a.row_start;
    const int * lens = PARTIAL ? a.prefix_len : a.len;
    const int most = PARTIAL ? a.n : a.rows;
    int pbeg = 0, pend = 0, pl = 0;
    if (!PARTIAL && lane < a.n_prefix && a.n_prefix <= 32) {
        pbeg = __ldg(a.prefix_start + lane); pend = __ldg(a.prefix_start + lane + 1); pl = __ldg(a.prefix_len + lane);
    }
    int before = 0;
    for (int b = 0; b < n; b += 32) {
        const int x = b + lane;
        int beg = 0, cnt = 0, ln = 0;
        if (x < n) {
            beg = __ldg(start + x); cnt = __ldg(start + x + 1) - beg; ln = __ldg(lens + x);
            if (pg_range_wrong(beg, cnt, most)) cnt = 0;
        }
        const int mine = (int) (((long long) cnt * a.group + ROWS - 1) / ROWS);
        int inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        const int sum = __shfl_sync(0xffffffffu, inc, 31);
        if (z < before + sum) {
            const int l = __ffs(__ballot_sync(0xffffffffu, z < before + inc)) - 1;
            t.i = t.px = b + l;
            t.row0 = __shfl_sync(0xffffffffu, beg, l);
            t.total = __shfl_sync(0xffffffffu, cnt, l) * a.group;
            t.lo = (z - before - __shfl_sync(0xffffffffu, inc - mine, l)) * ROWS;
            t.len = t.plen = __shfl_sync(0xffffffffu, ln, l);
            if (PARTIAL) {
                t.len = 0;
            } else if (a.n_prefix <= 32) {
                const unsigned in = __ballot_sync(0xffffffffu, pbeg <= t.i && t.i < pend);
                t.px = __ffs(in) - 1;
                t.plen = __shfl_sync(0xffffffffu, pl, max(0, t.px));
                if (!in) t.plen = 0;
            } else {
                t.px = pg_prefix_of(a, t.i);
                t.plen = t.px >= 0 ? __ldg(a.prefix_len + t.px) : 0;
            }
            return true;
        }
        before += sum;
    }
    return false;
}

// grid = tiles x kv heads x splits, clusters of `splits` CTAs, the last tiles
// (of a prompt, those with the most keys) first.  PARTIAL: the
// prefix keys for all of a decode batch's rows, joined with the own parts that
// the decode kernel left in the workspace; otherwise a prompt's rows over
// prefix and own keys.
template <class QT, class CT, int D, bool PARTIAL, int NT>
__global__ __launch_bounds__(pt_threads(NT), 3 - NT) void attn_shared_tile_kernel(const __grid_constant__ CUtensorMap mk,
                                                                         const __grid_constant__ CUtensorMap mv, PgAttn a) {
    constexpr bool F32 = sizeof(QT) == 4;
    constexpr int NP = D / 64, R = pt_slots(D, F32, NT), PARTS = F32 ? 2 : 1;
    constexpr int ROWS = 128 * NT, THREADS = pt_threads(NT), MMAW = 4 * NT;   // rows, threads, the MMA warp
    constexpr int TCOLS = pt_tmem(D, F32, NT);     // columns of tensor memory
    static_assert(!F32 || NT == 1, "no room for a sum of tiles");
    constexpr int SLOT = NP * PT_PANEL, QTILE = PARTS * SLOT;     // bytes
    constexpr float BIAS = PgBias<CT>::v;
    constexpr unsigned FMT = std::is_same<CT, __half>::value ? 0u : (1u << 7) | (1u << 10);
    constexpr unsigned ID_QK = (1u << 4) | FMT | ((unsigned) (PT_BN >> 3) << 17) | (8u << 24);
    constexpr unsigned ID_PV = (1u << 4) | FMT | (1u << 16) | ((unsigned) (D >> 3) << 17) | (8u << 24);   // B is MN-major
    extern __shared__ __align__(16) unsigned char pt_raw[];
    unsigned char * sm = pt_raw + ((1024u - ((unsigned) __cvta_generic_to_shared(pt_raw) & 1023u)) & 1023u);
    const unsigned smq = (unsigned) __cvta_generic_to_shared(sm), smr = smq + NT * QTILE;
    __shared__ __align__(8) unsigned long long bars[2 * R + 8];
    __shared__ __align__(16) unsigned char s_mask[4][16];      // keys present in 8-key groups, of the last four tiles
    __shared__ unsigned s_tmem;
    __shared__ PgTile s_tile;
    __shared__ int s_have, s_bad;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // the epilogue's arrays lie over Q and the ring: O, maxima, sums, the parts' weights, the rows' places in out and
    // in the own parts, marks
    float * so = (float *) sm, * s_m = so + ROWS * (D + 4), * s_l = s_m + ROWS, * s_w = s_l + ROWS;
    float * s_wo = s_w + 8 * ROWS;
    long long * s_off = (long long *) (s_wo + ROWS), * s_rec = s_off + ROWS;
    unsigned char * s_odd = (unsigned char *) (s_rec + ROWS);
    int rank, nrank;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(nrank));
    const int unit = blockIdx.x / nrank, h = unit % a.n_kv_head, g = a.group;
    const unsigned bar0 = (unsigned) __cvta_generic_to_shared(bars);
    auto full = [&](int s) { return bar0 + 8 * s; };
    auto empty = [&](int s) { return bar0 + 8 * (R + s); };
    auto s_full = [&](int t) { return bar0 + 8 * (2 * R + t); };
    auto p_full = [&](int t) { return bar0 + 8 * (2 * R + 2 + t); };
    auto p_half = [&](int t) { return bar0 + 8 * (2 * R + 4 + t); };
    const unsigned q_full = bar0 + 8 * (2 * R + 6), o_full = bar0 + 8 * (2 * R + 7);

    if (warp == 0) {
        PgTile t{};
        const bool have = pg_find_tile<PARTIAL, ROWS>(a, (int) (gridDim.x / nrank) / a.n_kv_head - 1 - unit / a.n_kv_head, t);
        if (lane == 0) { s_have = have; s_tile = t; s_bad = 0; }
    }
    if (blockIdx.x == 0 && (warp == 2 || warp == 3)) pg_check_ranges<PARTIAL, 64>(a, tid - 64);   // beside warp 0's search
    if (tid == 32) {
        for (int s = 0; s < R; ++s) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(full(s)), "n"(PT_LOADERS) : "memory");
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(empty(s)) : "memory");
        }
        for (int t = 0; t < 2; ++t) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(s_full(t)) : "memory");
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 128;" ::"r"(p_full(t)) : "memory");
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 128;" ::"r"(p_half(t)) : "memory");
        }
        asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(q_full), "n"(ROWS) : "memory");
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(o_full) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MMAW) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"((unsigned) __cvta_generic_to_shared(&s_tmem)), "n"(TCOLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tm = s_tmem;                    // S / P of tile x at 128 x, O at 128 NT + D x, F32's sum of tiles behind
    const PgTile t = s_tile;
    const int px = t.px, plen = t.plen, len = t.len, add = t.total / g;
    const bool wrong = plen < 0 || plen > (a.prefix_max_blocks << a.page_log2) ||
                       (!PARTIAL && (len < 0 || len > (a.max_blocks << a.page_log2) || add > len));
    if (!s_have || wrong) {                        // the whole cluster: it shares the tile
        if (s_have && tid == 0) atomicOr(&g_paged_err, T3B_DEVERR_POS);   // PARTIAL: the decode kernel leaves these requests alone too
        if (warp == MMAW) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "n"(TCOLS) : "memory");
        // The decode kernel let this grid start early, and what follows must find
        // rows without a prefix written: the grid cannot complete before the
        // decode kernel while one CTA waits for it, here or in the epilogue.
        // That is the last to start, tile 0's; the surplus ones start first and
        // would hold SMs that tiles need (192 long requests 296 us became 301).
        if (PARTIAL && unit == (int) (gridDim.x / nrank) - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    const int cnt = min(ROWS, t.total - t.lo), nt = cnt > 128 ? 2 : 1;   // rows, 128-row tiles
    // own keys that the tile's last row sees, key tiles of this CTA
    const int seen = PARTIAL ? 0 : len - add + (t.lo + cnt - 1) / g + 1;
    const int np = (plen + PT_BN - 1) / PT_BN, all = np + (seen + PT_BN - 1) / PT_BN;
    const int per = (all + nrank - 1) / nrank, kt0 = min(all, rank * per), nk = min(all, kt0 + per) - kt0;

    if (warp < MMAW) {
        // ---------------- softmax: thread = row ----------------
        if (NT == 1) asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
        const int x = warp >> 2, r = tid, row = t.lo + r;   // tile, row of the CTA, row of the request
        const int tok = row / g;
        const float sl2 = fabsf(a.scale) * 1.4426950408889634f;
        float sc = sl2;                            // what the row's scores are multiplied by
        if (x < nt) {
            // The warp stages its 32 rows, eight lanes to 64 elements: lane c
            // of a row's eight brings 16 bytes of each panel.
            constexpr int QB = 16 / (NP * PARTS) < 8 ? 16 / (NP * PARTS) : 8;
            const unsigned qd = smq + x * QTILE;
            const int c = lane & 7;
            const float cs = a.scale * 1.4426950408889634f;
            const unsigned flip = a.scale < 0.0f ? 0x80008000u : 0u;   // a negative scale is folded into q
#pragma unroll
            for (int b = 0; b < 8; b += QB) {      // QB rows of each lane group in flight, 16 loads
                float4 v[QB][NP][PARTS];           // F32: eight floats, else eight 16-bit values in [0]
#pragma unroll
                for (int k = 0; k < QB; ++k) {
                    const int rw = (r & ~31) + (b + k) * 4 + (lane >> 3), rq = t.lo + rw;
                    const QT * q = (const QT *) a.q + (long long) (t.row0 + rq / g) * a.q_stride + (h * g + rq % g) * D + c * 8;
#pragma unroll
                    for (int p = 0; p < NP; ++p)
#pragma unroll
                        for (int y = 0; y < PARTS; ++y)
                            v[k][p][y] = rw < cnt ? __ldg((const float4 *) (q + p * 64) + y) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int k = 0; k < QB; ++k) {
                    const int rr = ((r & ~31) + (b + k) * 4 + (lane >> 3)) & 127;
                    const unsigned off = rr * 128 + ((c ^ (rr & 7)) << 4);
                    if (F32) {
                        float mx = 0.0f;
#pragma unroll
                        for (int p = 0; p < NP; ++p)
#pragma unroll
                            for (int y = 0; y < PARTS; ++y) {
                                float4 & w = v[k][p][y];
                                w.x *= cs; w.y *= cs; w.z *= cs; w.w *= cs;
                                mx = fmaxf(fmaxf(fmaxf(mx, fabsf(w.x)), fmaxf(fabsf(w.y), fabsf(w.z))), fabsf(w.w));
                            }
#pragma unroll
                        for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                        const int ex = pg_row_exp(mx);
                        const float f = pg_pow2(-ex), back = pg_pow2(ex);
                        // the thread of row 4 (b + k) + y is lane 4 (b + k) + y; the row's scale is in lanes 8 y ..
                        const float mine = __shfl_sync(0xffffffffu, back, (lane & 3) * 8);
                        if ((lane >> 2) == b + k) sc = mine;
#pragma unroll
                        for (int p = 0; p < NP; ++p) {
                            const float4 u = v[k][p][0], w = v[k][p][PARTS - 1];
                            uint4 hi, lo;
                            pg_split2(u.x * f, u.y * f, hi.x, lo.x); pg_split2(u.z * f, u.w * f, hi.y, lo.y);
                            pg_split2(w.x * f, w.y * f, hi.z, lo.z); pg_split2(w.z * f, w.w * f, hi.w, lo.w);
                            pg_sts(qd + p * PT_PANEL + off, hi);
                            pg_sts(qd + SLOT + p * PT_PANEL + off, lo);
                        }
                    } else {
#pragma unroll
                        for (int p = 0; p < NP; ++p) {
                            const float4 u = v[k][p][0];
                            pg_sts(qd + p * PT_PANEL + off, make_uint4(__float_as_uint(u.x) ^ flip, __float_as_uint(u.y) ^ flip,
                                                                       __float_as_uint(u.z) ^ flip, __float_as_uint(u.w) ^ flip));
                        }
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        pg_arrive(q_full);

        float m = -INFINITY, l = 0.0f;
        bool ok = true;
        const unsigned lanes = tm + ((unsigned) ((warp & 3) * 32) << 16), ts = lanes + 128 * x, to = lanes + 128 * NT + D * x;
        const int lim_own = PARTIAL ? 0 : len - add + tok + 1;      // own keys that this row sees
        if (F32) {                                 // the sum of tiles
            const unsigned zero[16] = {};
#pragma unroll
            for (int c = 0; c < D; c += 16) pg_tm_st16(zero, to + D + c);
            pg_tm_wait_st();
        }
        if (x < nt) {
            for (int j = 0; j < nk; ++j) {
                ok = tf_wait(s_full(x), (unsigned) j & 1u);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const int kt = kt0 + j;
                const int left = kt < np ? PT_BN : lim_own - (kt - np) * PT_BN;   // keys of the tile before the causal limit
                if (F32 && j > 0)                  // the last tile's O is complete: add it to the sum
#pragma unroll 1
                    for (int c = 0; c < D; c += 16) {
                        unsigned w[16], v[16];
                        pg_tm_ld16(w, to + c);
                        pg_tm_ld16(v, to + D + c);
                        pg_tm_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) + __uint_as_float(v[e]));
                        pg_tm_st16(w, to + D + c);
                    }
                unsigned u[4][32];                 // the row's scores
#pragma unroll
                for (int c = 0; c < 4; ++c) pg_tm_ld32(u[c], ts + 32 * c);
                const uint4 here = *(const uint4 *) s_mask[kt & 3];
                pg_tm_wait_ld();
                const bool whole = (here.x & here.y & here.z & here.w) == 0xffffffffu && left >= PT_BN;
                if (!__all_sync(0xffffffffu, whole)) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int v = left - 32 * c;
                        const unsigned word = c == 0 ? here.x : c == 1 ? here.y : c == 2 ? here.z : here.w;
                        const unsigned msk = word & (v >= 32 ? 0xffffffffu : v <= 0 ? 0u : (1u << v) - 1u);
#pragma unroll
                        for (int e = 0; e < 32; ++e) if (!(msk >> e & 1u)) u[c][e] = 0xff800000u;
                    }
                }
                float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 32; ++e)
#pragma unroll
                    for (int c = 0; c < 4; ++c) tops[c] = fmaxf(tops[c], __uint_as_float(u[c][e]));
                const float top = fmaxf(m, fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * sc);   // sc > 0; -inf stays
                if (__any_sync(0xffffffffu, top > m + PD_LAZY)) {
                    const float f = m == -INFINITY ? 0.0f : pg_exp2(m - top);
                    m = top; l *= f;
                    if (j > 0)
#pragma unroll 1
                        for (int c = 0; c < D; c += 16) {
                            unsigned w[16];
                            const unsigned at = to + (F32 ? D : 0) + c;
                            if (F32) pg_tm_wait_st();
                            pg_tm_ld16(w, at);
                            pg_tm_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) * f);
                            pg_tm_st16(w, at);
                        }
                }
                const float base = m == -INFINITY ? 0.0f : m - BIAS;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float ls[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    unsigned hi[16], lo[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float p0 = pg_exp2(fmaf(__uint_as_float(u[c][2 * e]), sc, -base));
                        const float p1 = pg_exp2(fmaf(__uint_as_float(u[c][2 * e + 1]), sc, -base));
                        ls[2 * (e & 1)] += p0; ls[2 * (e & 1) + 1] += p1;
                        if (F32) pg_split2(p0, p1, hi[e], lo[e]);
                        else hi[e] = pg_pack2<CT>(p0, p1);
                    }
                    l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
                    // P lies over the columns of S: 16 per 32 keys, F32's lo parts right behind
                    pg_tm_st16(hi, ts + (F32 ? 32 : 16) * c);
                    if (F32) pg_tm_st16(lo, ts + 32 * c + 16);
                    if (c == 1) {                  // the first 64 keys' P V may begin
                        pg_tm_wait_st();
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        pg_arrive(p_half(x));
                    }
                }
                pg_tm_wait_st();
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                pg_arrive(p_full(x));
            }
            if (nk > 0 && ok) ok = tf_wait(o_full, 0u);
            ok = __all_sync(0xffffffffu, ok);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
        if (!ok) s_bad = 1;
        // (O, max, sum) of the row into shared memory, over Q and the ring:
        // o_full means that every MMA of the CTA has read them
        asm volatile("bar.sync 1, %0;" ::"n"(ROWS) : "memory");
        if (x < nt) {
            float big = 0.0f;                      // not finite if an element is not
#pragma unroll
            for (int c = 0; c < D; c += 32) {
                unsigned u[32];
                if (nk > 0) {
                    unsigned v[32];
                    pg_tm_ld32(u, to + c);
                    if (F32) pg_tm_ld32(v, to + D + c);
                    pg_tm_wait_ld();
                    if (F32)
#pragma unroll
                        for (int e = 0; e < 32; ++e) u[e] = __float_as_uint(__uint_as_float(u[e]) + __uint_as_float(v[e]));
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) u[e] = 0u;
                }
                if (!PARTIAL)
#pragma unroll
                    for (int e = 0; e < 32; ++e) big += fabsf(__uint_as_float(u[e])) * 0x1p-16f;   // (32-bit sums of 16-bit V stay in range)
#pragma unroll
                for (int e = 0; e < 32; e += 4)
                    *(uint4 *) (so + r * (D + 4) + c + e) = make_uint4(u[e], u[e + 1], u[e + 2], u[e + 3]);
            }
            s_m[r] = m; s_l[r] = big < INFINITY ? l : NAN;            // NaN: the row is worked out again at the end
            const long long qrow = t.row0 + tok;
            const int head = h * g + row % g;
            s_off[r] = qrow * a.out_stride + (long long) head * D;
            if (PARTIAL) s_rec[r] = (qrow * a.n_head + head) * (D + 4);
        }
        if (NT == 1) asm volatile("setmaxnreg.dec.sync.aligned.u32 128;");
    } else {
    if (NT == 1) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == MMAW) {
        // ---------------- MMA issue ----------------
        const unsigned el = pg_elect();
        // 14 bits of address: in a cluster, shared addresses carry the CTA's rank above them
        const unsigned qw = (smq >> 4) & 0x3fffu, rw = (smr >> 4) & 0x3fffu;
        const unsigned q0 = qw | (1u << 16), k0 = rw | (1u << 16), v0 = rw | ((unsigned) (PT_PANEL >> 4) << 16);
        auto qk = [&](int x, int slot) {            // S of tile x = Q K^T
            const unsigned qa = q0 + x * (QTILE >> 4), ka = k0 + slot * (SLOT >> 4);
#pragma unroll
            for (int part = PARTS - 1; part >= 0; --part)      // F32: the small lo parts first, before the sum is large
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const unsigned off = (k >> 2) * (PT_PANEL >> 4) + (k & 3) * 2;
                    pg_mma_ss(tm + 128 * x, qa + part * (SLOT >> 4) + off, ka + off, ID_QK, part < PARTS - 1 || k ? 1u : 0u, el);
                }
            pg_commit(s_full(x), el);
        };
        auto pv = [&](int x, int slot, unsigned acc, int half) {   // O of tile x += P V over half of the tile's keys
            const unsigned va = v0 + slot * (SLOT >> 4);
#pragma unroll
            for (int part = PARTS - 1; part >= 0; --part)
#pragma unroll
                for (int k = half * PT_BN / 32; k < (half + 1) * PT_BN / 32; ++k)
                    pg_mma_ts(tm + 128 * NT + D * x, tm + 128 * x + (F32 ? 32 * (k >> 1) + 16 * part + 8 * (k & 1) : 8 * k), va + k * 128,
                              ID_PV, half == 0 && k == 0 && part == PARTS - 1 ? acc : 1u, el);
        };
        bool ok = tf_wait(q_full, 0u);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (nk > 0 && ok) {
            ok = tf_wait(full(0), 0u);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (ok) {
                for (int x = 0; x < nt; ++x) qk(x, 0);
                pg_commit(empty(0), el);
            }
        }
        int sv = 1, pv_ph = 0;                      // slot of this tile's V and its phase; K of the next follows
        for (int j = 0; j < nk && ok; ++j) {
            const int sk = sv + 1 == R ? 0 : sv + 1, pk_ph = sv + 1 == R ? pv_ph ^ 1 : pv_ph;
            ok = tf_wait(full(sv), (unsigned) pv_ph);
            if (ok && j + 1 < nk) ok = tf_wait(full(sk), (unsigned) pk_ph);
            for (int x = 0; x < nt && ok; ++x) {
                ok = tf_wait(p_half(x), (unsigned) j & 1u);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                pv(x, sv, !F32 && j > 0, 0);
                ok = tf_wait(p_full(x), (unsigned) j & 1u);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                pv(x, sv, 1u, 1);
                if (x == nt - 1) pg_commit(empty(sv), el);
                if (j + 1 < nk) {
                    qk(x, sk);
                    if (x == nt - 1) pg_commit(empty(sk), el);
                }
            }
            sv = sk + 1 == R ? 0 : sk + 1; pv_ph = sk + 1 == R ? pk_ph ^ 1 : pk_ph;
        }
        pg_commit(o_full, el);
        if (!tf_wait(o_full, 0u) || !ok) s_bad = 1;                   // nothing is in flight when the CTA goes on
        __syncwarp();
    } else {
        // ---------------- loaders: every third group of 8 keys per warp ----------------
        const int lw = warp - MMAW - 1;
        const int items = 2 * nk;
        auto tile_keys = [&](int kt, int & key0, int & have) {        // first key of tile kt in its segment, keys from it on
            const bool pre = kt < np;
            key0 = (pre ? kt : kt - np) * PT_BN;
            have = (pre ? plen : seen) - key0;
            return pre;
        };
        auto fetch = [&](int kt) {                                    // lane x < 16: the page of keys 8 x ..
            int id = -1, key0, have;
            if (lane < 16 && kt < kt0 + nk) {
                const bool pre = tile_keys(kt, key0, have);
                const int k = lane * 8;
                if (k < have) {
                    id = __ldg((pre ? a.prefix_table + (long long) px * a.prefix_max_blocks : a.table + (long long) t.i * a.max_blocks) +
                               ((key0 + k) >> a.page_log2));
                    if ((unsigned) id >= (unsigned) a.n_pages) { atomicOr(&g_paged_err, T3B_DEVERR_PAGE); id = -1; }
                }
            }
            return id;
        };
        int done = 0;                                                 // items signalled
        auto signal_to = [&](int upto) {                              // their copies have been waited for
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            for (; done < upto; ++done) if (lane == 0) pg_arrive(full(done % R));
        };
        bool ok = true;
        int ids = fetch(kt0), ids_next = -1;
        for (int n = 0; n < items && ok; ++n) {
            const int kt = kt0 + (n >> 1), v = n & 1, s = n % R;
            if (!v) ids_next = fetch(kt + 1);
            if (n >= R) {
                const unsigned ph = (unsigned) (n / R - 1) & 1u;
                if (!__all_sync(0xffffffffu, pg_test(empty(s), ph))) {
                    // what is still in flight is waited for first: the MMAs may need it to free the slot
                    asm volatile("cp.async.wait_group 0;" ::: "memory");
                    signal_to(n);
                    ok = tf_wait(empty(s), ph);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                }
            }
            int key0, have;
            tile_keys(kt, key0, have);
            const CT * src = (const CT *) (v ? a.v : a.k);
            const unsigned slot = smr + s * SLOT;
            if (have >= PT_BN && (__ballot_sync(0xffffffffu, ids < 0) & 0xffffu) == 0u) {
                // a whole tile: boxes of a page's keys (at most 128) by TMA, one per lane of the first warp
                if (done < n) { asm volatile("cp.async.wait_group 0;" ::: "memory"); signal_to(n); }
                if (!v && lane < 16 && lane % PT_LOADERS == lw) s_mask[kt & 3][lane] = 0xffu;
                __syncwarp();
                if (lw == 0) {
                    const int br = min(1 << a.page_log2, PT_BN), k = lane / NP * br, p = lane % NP;
                    const int id = __shfl_sync(0xffffffffu, ids, (k >> 3) & 15);
                    if (lane == 0)
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full(s)), "r"((unsigned) SLOT) : "memory");
                    __syncwarp();
                    if (k < PT_BN)
                        asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                                     ::"r"(slot + p * PT_PANEL + k * 128), "l"(v ? &mv : &mk), "r"(p * 64),
                                       "r"((key0 + k) & ((1 << a.page_log2) - 1)), "r"(h), "r"(id), "r"(full(s)) : "memory");
                } else if (lane == 0) {
                    pg_arrive(full(s));
                }
                done = n + 1;
                if (v) ids = ids_next;
                continue;
            }
            if (!v && lane < 16 && lane % PT_LOADERS == lw)           // which keys of its groups are there
                s_mask[kt & 3][lane] = ids >= 0 ? (unsigned char) ((1u << min(8, max(0, have - lane * 8))) - 1u) : (unsigned char) 0;
#pragma unroll
            for (int gi = 0; gi < (16 + PT_LOADERS - 1) / PT_LOADERS; ++gi) {
                const int grp = gi * PT_LOADERS + lw;
                if (grp >= 16) break;
                const int id = __shfl_sync(0xffffffffu, ids, grp);
                const long long page = id >= 0 ? (long long) id * a.page_stride + ((long long) h << a.page_log2) * D : 0;
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const int krow = grp * 8 + y * 4 + (lane >> 3), c = lane & 7;
                    const bool on = id >= 0 && krow < have;
                    const CT * from = src + (on ? page + ((key0 + krow) & ((1 << a.page_log2) - 1)) * D + c * 8 : 0);
                    const unsigned d = slot + krow * 128 + ((c ^ (krow & 7)) << 4);
#pragma unroll
                    for (int p = 0; p < NP; ++p) pg_cp16(d + p * PT_PANEL, from + (on ? p * 64 : 0), on);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (v) ids = ids_next;
            if (n > done) {                                           // all but the newest item have arrived
                asm volatile("cp.async.wait_group 1;" ::: "memory");
                signal_to(n);
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (ok) signal_to(items);
        else {
            s_bad = 1;                                                // no copy is in flight when the CTA goes on
            for (int n = max(0, done - R); n < done; ++n) tf_wait(full(n % R), (unsigned) (n / R) & 1u);
        }
    }
    if (NT == 1) {
        __syncwarp();
        asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
    }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == MMAW) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "n"(TCOLS) : "memory");
    }
    if (s_bad && tid == 0) atomicOr(&g_paged_err, T3B_DEVERR_TIMEOUT);
    if (nrank > 1) pg_cluster_sync();

    // Join the cluster's parts (and a decode row's own part) and write, each
    // CTA an equal share of the rows: first the parts' weights, a thread per
    // row, then four elements per thread.
    const int share = (cnt + nrank - 1) / nrank, r_beg = min(cnt, rank * share), r_end = min(cnt, r_beg + share);
    if (PARTIAL) asm volatile("griddepcontrol.wait;" ::: "memory");   // the own parts are there
    if (tid < r_end - r_beg) {
        const int r = r_beg + tid;
        float mo = -INFINITY, lo = 0.0f;
        if (PARTIAL) { mo = __ldcg(a.part + s_rec[r] + D); lo = __ldcg(a.part + s_rec[r] + D + 1); }
        float mx = mo, lv = 0.0f, my[8], ly[8];    // every CTA's in flight at once
#pragma unroll
        for (int y = 0; y < 8; ++y) {
            my[y] = y < nrank ? pg_dsm(s_m + r, y) : -INFINITY;
            ly[y] = y < nrank ? pg_dsm(s_l + r, y) : 0.0f;
        }
#pragma unroll
        for (int y = 0; y < 8; ++y) mx = fmaxf(mx, my[y]);
#pragma unroll
        for (int y = 0; y < 8; ++y) {
            my[y] = my[y] == -INFINITY ? 0.0f : pg_exp2(my[y] - mx);
            lv += my[y] * ly[y];
        }
        const float wo = mo == -INFINITY ? 0.0f : pg_exp2(mo - mx);
        lv += wo * lo;
        const float inv = lv == 0.0f ? 0.0f : 1.0f / lv;
#pragma unroll
        for (int y = 0; y < 8; ++y) if (y < nrank) s_w[y * ROWS + tid] = my[y] * inv;
        if (!PARTIAL) s_odd[tid] = !(lv < INFINITY);
        if (PARTIAL) s_wo[tid] = lo < 0.0f ? -1.0f : wo * inv;        // -1: the request is refused
    }
    const bool odd = __syncthreads_or(!PARTIAL && tid < r_end - r_beg && s_odd[tid]);
    constexpr int C4 = D / 4;
    auto pieces = [&](auto ranks) {                // the parts' number at compile time: their loads in flight at once
        constexpr int N = decltype(ranks)::value;
#pragma unroll(N <= 2 ? 4 : 1)
        for (int x = tid; x < (r_end - r_beg) * C4; x += THREADS) {
            const int rr = x / C4, r = r_beg + rr, c = x % C4 * 4;
            if (!PARTIAL && s_odd[rr]) continue;   // (q may be out: the row's q is still needed)
            float v[4], u[N][4];
            float4 own;
            if (PARTIAL) own = __ldcg((const float4 *) (a.part + s_rec[r] + c));
#pragma unroll
            for (int y = 0; y < N; ++y) {
                if (N == 1) {
                    const float4 f = *(const float4 *) (so + r * (D + 4) + c);
                    u[y][0] = f.x; u[y][1] = f.y; u[y][2] = f.z; u[y][3] = f.w;
                } else {
                    pg_dsm4(u[y], so + r * (D + 4) + c, y);
                }
            }
#pragma unroll
            for (int y = 0; y < N; ++y) {
                const float w = s_w[y * ROWS + rr];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = y ? fmaf(w, u[y][e], v[e]) : w * u[y][e];
            }
            if (PARTIAL) {
                const float w = s_wo[rr];
                if (w > 0.0f) { v[0] = fmaf(w, own.x, v[0]); v[1] = fmaf(w, own.y, v[1]); v[2] = fmaf(w, own.z, v[2]); v[3] = fmaf(w, own.w, v[3]); }
                if (w != -1.0f) pg_store4((QT *) a.out + s_off[r] + c, v);
            } else {
                pg_store4((QT *) a.out + s_off[r] + c, v);
            }
        }
    };
    if (nrank == 1) pieces(std::integral_constant<int, 1>{});
    else if (nrank == 2) pieces(std::integral_constant<int, 2>{});
    else if (nrank == 4) pieces(std::integral_constant<int, 4>{});
    else pieces(std::integral_constant<int, 8>{});
    if (!PARTIAL && odd)                           // rows that are not finite again, by their keys one by one
        for (int rr = warp; rr < r_end - r_beg; rr += THREADS / 32) {
            if (!s_odd[rr]) continue;
            const int row = t.lo + r_beg + rr, tok = row / g;
            float sv[D / 32];
            pg_row_slow<QT, CT, D>(a, (const QT *) a.q + (long long) (t.row0 + tok) * a.q_stride + (h * g + row % g) * D, t.i, px, plen,
                                   len - add + tok + 1, h, sv);
            QT * out = (QT *) a.out + s_off[r_beg + rr] + lane * (D / 32);
#pragma unroll
            for (int e = 0; e < D / 32; ++e) out[e] = pg_from<QT>(sv[e]);
        }
    if (nrank > 1) pg_cluster_sync();              // no CTA leaves while another reads its shared memory
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
namespace {

bool pg_log2(int x, int lo, int hi, int * out) {
    for (int b = lo; b <= hi; ++b) if (x == 1 << b) { *out = b; return true; }
    return false;
}
bool pg_aligned(const void * p) { return (((uintptr_t) p) & 15) == 0; }

// what is wrong with a cache description, or NULL
const char * pg_cache_wrong(const t3b_paged_kv & c, bool pointers) {
    int lg;
    if (c.dtype != T3B_F16 && c.dtype != T3B_BF16) return "the cache's type is not T3B_F16 or T3B_BF16";
    if (!pg_log2(c.page_size, 3, 8, &lg)) return "page_size is not 8, 16, 32, 64, 128 or 256";
    if (c.head_dim != 64 && c.head_dim != 128) return "head_dim is not 64 or 128";
    if (c.n_pages <= 0 || c.n_kv_head <= 0 || (int64_t) c.n_pages * c.page_size > 0x7fffffffll || c.n_kv_head > 1024)
        return "n_pages or n_kv_head is out of range";
    const int64_t dense = (int64_t) c.n_kv_head * c.page_size * c.head_dim;
    if (c.page_stride && (c.page_stride < dense || c.page_stride % 8 || c.page_stride >= (int64_t) 1 << 39))
        return "page_stride is below a page's elements or not a multiple of 8";
    if (pointers && (!c.k || !c.v)) return "null cache";
    if (pointers && (!pg_aligned(c.k) || !pg_aligned(c.v))) return "K and V caches must be 16-byte aligned";
    return nullptr;
}
int64_t pg_page_stride(const t3b_paged_kv & c) {
    return c.page_stride ? c.page_stride : (int64_t) c.n_kv_head * c.page_size * c.head_dim;
}

// what is wrong with an attention call's sizes, or NULL
const char * pg_attn_wrong(const t3b_shared_attn & a, bool prompt, bool pointers) {
    if (const char * w = pg_cache_wrong(a.cache, pointers)) return w;
    if (!((a.dtype == T3B_F32 && a.cache.dtype == T3B_F16) || a.dtype == a.cache.dtype))
        return "q's type is neither the cache's nor T3B_F32 over an F16 cache";
    if (a.n_head <= 0 || a.n_head % a.cache.n_kv_head || a.n_head / a.cache.n_kv_head > 16)
        return "n_head is not 1 to 16 times n_kv_head";
    if (a.n <= 0 || a.n > 65535 || a.n_prefix < 0 || a.n_prefix > 65535 || a.rows < 0 || a.rows > 1 << 26) return "n, n_prefix or rows is out of range";
    if (a.max_blocks <= 0 || (int64_t) a.max_blocks * a.cache.page_size > 0x3fffffffll ||
        (a.n_prefix > 0 && (a.prefix_max_blocks <= 0 || (int64_t) a.prefix_max_blocks * a.cache.page_size > 0x3fffffffll)))
        return "max_blocks or prefix_max_blocks is out of range";
    if (!prompt && a.rows != a.n) return "rows is not n";
    if (!(a.scale > -INFINITY && a.scale < INFINITY)) return "scale is not finite";
    const int el = a.dtype == T3B_F32 ? 4 : 8;   // elements of 16 bytes
    const int64_t width = (int64_t) a.n_head * a.cache.head_dim;
    if (a.q_stride < width || a.out_stride < width || a.q_stride % el || a.out_stride % el || a.q_stride > (int64_t) 1 << 40 ||
        a.out_stride > (int64_t) 1 << 40)
        return "a row stride is below n_head * head_dim or not a multiple of 16 bytes";
    if (!pointers) return nullptr;
    if (!a.q || !a.out || !a.len || !a.table || (prompt && !a.row_start) ||
        (a.n_prefix > 0 && (!a.prefix_start || !a.prefix_len || !a.prefix_table))) return "null pointer";
    if (!pg_aligned(a.q) || !pg_aligned(a.out)) return "q and out must be 16-byte aligned";
    if (a.q == a.out && a.q_stride != a.out_stride) return "out is q with another stride";
    return nullptr;
}

// Whether a decode call computes its prefixes' attention once for the batch
// (the tile kernel after the decode kernel) or lets every request read its
// prefix through L2.  The host has no lengths, so this and the other rules of a
// launch (splits, what passes through L2) go by the room in the tables; the
// figures are of tables as wide as their longest request.  The tile kernel costs 6 to 8 us; what it saves is the
// prefix's K and V for all requests but one, at 5 to 8 TB/s.  Measured with own
// lengths around 300, us without / with it: 16 x 376 keys (25 MB, f32 x 64
// dimensions) 14 / 17, 32 x 376 (49 MB) 21 / 25 and (bf16, 8 x 128) 27 / 24,
// 16 x 1000 (66 MB) 19 / 18 and 27 / 20, 128 x 376 (197 MB) 53 / 43 and 61 / 49.
bool pg_shares(const t3b_shared_attn & a) {
    if (a.n_prefix == 0 || a.n <= a.n_prefix) return false;
    const double token = 4.0 * a.cache.n_kv_head * a.cache.head_dim;
    return (double) (a.n - a.n_prefix) * a.prefix_max_blocks * a.cache.page_size * token > 48e6;
}

size_t pg_workspace(const t3b_shared_attn & a, bool prompt) {
    return !prompt && pg_shares(a) ? (size_t) a.n * a.n_head * (a.cache.head_dim + 4) * sizeof(float) : 0;
}

PgAttn pg_args(const t3b_shared_attn & a, bool prompt) {
    PgAttn p{};
    p.k = a.cache.k; p.v = a.cache.v; p.q = a.q; p.out = a.out;
    p.page_stride = pg_page_stride(a.cache); p.q_stride = a.q_stride; p.out_stride = a.out_stride;
    p.len = a.len; p.table = a.table; p.row_start = prompt ? a.row_start : nullptr;
    p.prefix_start = a.prefix_start; p.prefix_len = a.prefix_len; p.prefix_table = a.prefix_table;
    p.n = a.n; p.rows = a.rows; p.n_head = a.n_head; p.n_kv_head = a.cache.n_kv_head; p.group = a.n_head / a.cache.n_kv_head;
    pg_log2(a.cache.page_size, 3, 8, &p.page_log2);
    p.n_pages = a.cache.n_pages; p.max_blocks = a.max_blocks; p.n_prefix = a.n_prefix;
    p.prefix_max_blocks = a.n_prefix > 0 ? a.prefix_max_blocks : 0;   // (not looked at without prefixes)
    p.pass = (double) a.n * a.max_blocks * a.cache.page_size * a.cache.n_kv_head * a.cache.head_dim * 4.0 > 64e6;
    p.part = pg_workspace(a, prompt) ? (float *) a.workspace : nullptr;
    p.scale = a.scale != 0.0f ? a.scale : 1.0f / sqrtf((float) a.cache.head_dim);
    return p;
}

// CTAs of a (request, kv head): enough that the grid fills the GPU about four
// times over, while each still has 256 keys
int pg_splits(const t3b_shared_attn & a) {
    const int64_t units = (int64_t) a.n * a.cache.n_kv_head;
    const int64_t keys = ((int64_t) a.max_blocks + (a.n_prefix > 0 && !pg_shares(a) ? a.prefix_max_blocks : 0)) * a.cache.page_size;
    int c = 1;
    while (c < 8 && units * c < 4 * 148 && keys > (int64_t) 256 * c) c *= 2;
    return c;
}

// Raises a kernel's dynamic shared memory limit on the current device.
template <class K> cudaError_t pg_allow_smem(K * kernel, int bytes) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <class QT, class CT, int D, int MT, int RH>
cudaError_t pg_launch_decode(const t3b_shared_attn & a, const PgAttn & p, cudaStream_t st) {
    const cudaError_t e = pg_allow_smem(attn_shared_decode_kernel<QT, CT, D, MT, RH>, pd_smem(D));
    if (e != cudaSuccess) return e;
    const unsigned c = (unsigned) pg_splits(a);
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = c; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(c, (unsigned) p.n_kv_head, (unsigned) p.n); cfg.blockDim = dim3(32 * PD_WARPS);
    cfg.dynamicSmemBytes = pd_smem(D); cfg.stream = st; cfg.attrs = at; cfg.numAttrs = c > 1;
    return cudaLaunchKernelEx(&cfg, attn_shared_decode_kernel<QT, CT, D, MT, RH>, p);
}

// The pages of K or V as a 4-D tensor [n_pages][n_kv_head][page][D], boxes of
// 64 elements x up to 128 keys in the 128-byte swizzle.  Both 16-bit types
// move as they are.
bool pg_map(CUtensorMap * map, const void * base, const t3b_paged_kv & c) {
    PFN_cuTensorMapEncodeTiled_v12000 enc = tf_encode();
    const cuuint64_t row = (cuuint64_t) c.head_dim * 2;
    const cuuint64_t dims[4] = {(cuuint64_t) c.head_dim, (cuuint64_t) c.page_size, (cuuint64_t) c.n_kv_head, (cuuint64_t) c.n_pages};
    const cuuint64_t strides[3] = {row, row * c.page_size, (cuuint64_t) pg_page_stride(c) * 2};
    const cuuint32_t box[4] = {64u, (cuuint32_t) std::min(c.page_size, PT_BN), 1u, 1u};
    const cuuint32_t es[4] = {1u, 1u, 1u, 1u};
    return enc && enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void *>(base), dims, strides, box, es,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class QT, class CT, int D, bool PARTIAL, int NT>
cudaError_t pg_launch_tiles_nt(const t3b_shared_attn & a, const PgAttn & p, cudaStream_t st) {
    constexpr int SMEM = pt_smem(D, sizeof(QT) == 4, NT), ROWS = 128 * NT;
    const cudaError_t e = pg_allow_smem(attn_shared_tile_kernel<QT, CT, D, PARTIAL, NT>, SMEM);
    if (e != cudaSuccess) return e;
    // each request (prefix) may end in a part-filled tile
    const int64_t parts = PARTIAL ? p.n_prefix : p.n, rows = PARTIAL ? p.n : p.rows;
    const int64_t tiles = std::min((rows * p.group + ROWS - 1) / ROWS + parts - 1, rows * p.group);
    // as many as there are if the rows are spread evenly: the others' CTAs leave at once
    const int64_t even = std::min(tiles, parts * ((rows * p.group + parts * ROWS - 1) / (parts * ROWS)));
    const int64_t keys = ((PARTIAL ? 0 : (int64_t) a.max_blocks) + (a.n_prefix > 0 ? a.prefix_max_blocks : 0)) * a.cache.page_size;
    if (tiles * p.n_kv_head > (1 << 27)) return cudaErrorInvalidConfiguration;
    int c = 1;
    while (c < 8 && even * p.n_kv_head * 2 * c <= (c < 4 ? 148 : 64) && ((PARTIAL && c < 4) || keys > (int64_t) 2 * PT_BN * c)) c *= 2;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned) c; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned) (tiles * c * p.n_kv_head)); cfg.blockDim = dim3(pt_threads(NT));
    cfg.dynamicSmemBytes = SMEM; cfg.stream = st; cfg.attrs = at; cfg.numAttrs = PARTIAL ? 2 : 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // PARTIAL: starts as the decode kernel's last CTAs run
    at[1].val.programmaticStreamSerializationAllowed = 1;
    CUtensorMap mk, mv;
    if (!pg_map(&mk, a.cache.k, a.cache) || !pg_map(&mv, a.cache.v, a.cache)) return cudaErrorInvalidValue;
    return cudaLaunchKernelEx(&cfg, attn_shared_tile_kernel<QT, CT, D, PARTIAL, NT>, mk, mv, p);
}

template <class QT, class CT, int D, bool PARTIAL>
cudaError_t pg_launch_tiles(const t3b_shared_attn & a, const PgAttn & p, cudaStream_t st) {
    // Two tiles a CTA halve the K / V traffic, which is what 128 dimensions ask
    // for; with 64 the exponentials bound the loop, and two small CTAs an SM
    // hide each other's first and last steps.  Measured, one tile against two:
    // 8 chunks of bf16 x 128 dimensions 368 / 337 us, 4 x 2000 rows of f16 x 64
    // dimensions 196 / 208; with at most 128 rows to a request the second
    // tile would be empty: 16 text prompts 23 / 34.
    if (D == 128 && sizeof(QT) == 2 && (PARTIAL ? (int64_t) p.n * p.group > (int64_t) 128 * p.n_prefix : (int64_t) p.rows * p.group > (int64_t) 128 * p.n))
        return pg_launch_tiles_nt<QT, CT, D, PARTIAL, D == 128 && sizeof(QT) == 2 ? 2 : 1>(a, p, st);
    return pg_launch_tiles_nt<QT, CT, D, PARTIAL, 1>(a, p, st);
}

template <class QT, class CT, int D>
cudaError_t pg_launch_attention(const t3b_shared_attn & a, const PgAttn & p, bool prompt, cudaStream_t st) {
    if (!prompt) {
        // an M tile has 16 rows: 8 F32 queries, or 16 of 16 bits (the second half left out where it has none)
        constexpr bool F32 = sizeof(QT) == 4;
        const cudaError_t e = p.group > 8 ? pg_launch_decode<QT, CT, D, F32 ? 2 : 1, F32 ? 1 : 2>(a, p, st)
                                          : pg_launch_decode<QT, CT, D, 1, 1>(a, p, st);
        return e != cudaSuccess || !p.part ? e : pg_launch_tiles<QT, CT, D, true>(a, p, st);
    }
    return pg_launch_tiles<QT, CT, D, false>(a, p, st);
}

template <class S, class T>
void pg_launch_append(int U, unsigned grid, cudaStream_t st, const PgAppendArgs & p) {
    if (U == 2) kv_append_kernel<S, T, 2><<<grid, 256, 0, st>>>(p);
    else kv_append_kernel<S, T, 1><<<grid, 256, 0, st>>>(p);
}

int pg_attention(const char * name, const t3b_shared_attn * a, bool prompt, void * cuda_stream) {
    if (!a) { set_err(nullptr, "%s: null argument", name); return T3B_ERR_ARG; }
    if (const char * w = pg_attn_wrong(*a, prompt, true)) { set_err(nullptr, "%s: %s", name, w); return T3B_ERR_ARG; }
    const size_t need = pg_workspace(*a, prompt);
    if (need && (!a->workspace || !pg_aligned(a->workspace) || a->workspace_bytes < need)) {
        set_err(nullptr, "%s: workspace must be 16-byte aligned and hold %zu bytes", name, need);
        return T3B_ERR_ARG;
    }
    if (a->rows == 0) return T3B_OK;
    cudaStream_t st = (cudaStream_t) cuda_stream;
    const PgAttn p = pg_args(*a, prompt);
    const bool wide = a->cache.head_dim == 128;
    cudaError_t e;
    if (a->dtype == T3B_F32)
        e = wide ? pg_launch_attention<float, __half, 128>(*a, p, prompt, st) : pg_launch_attention<float, __half, 64>(*a, p, prompt, st);
    else if (a->dtype == T3B_F16)
        e = wide ? pg_launch_attention<__half, __half, 128>(*a, p, prompt, st) : pg_launch_attention<__half, __half, 64>(*a, p, prompt, st);
    else
        e = wide ? pg_launch_attention<__nv_bfloat16, __nv_bfloat16, 128>(*a, p, prompt, st)
                 : pg_launch_attention<__nv_bfloat16, __nv_bfloat16, 64>(*a, p, prompt, st);
    if (e != cudaSuccess) { set_err(nullptr, "%s: %s", name, cudaGetErrorString(e)); (void) cudaGetLastError(); return T3B_ERR_CUDA; }
    return T3B_OK;
}

}  // namespace

extern "C" {

int t3b_op_kv_plan(const t3b_kv_plan * p, void * cuda_stream) {
    int lg;
    if (!p || !p->len || !p->add || !p->free_pages || !p->n_free || !p->n_free_out || !p->table || !p->row_start ||
        p->n <= 0 || p->n > PG_PLAN_MAXN || p->rows_cap < 0 || p->rows_cap > 1 << 30 || p->free_cap < 0 || p->max_blocks <= 0 ||
        !pg_log2(p->page_size, 3, 8, &lg) || (int64_t) p->max_blocks * p->page_size > 0x3fffffffll ||
        (int64_t) p->n * p->max_blocks > 0x3fffffffll) {
        set_err(nullptr, "t3b_op_kv_plan: bad args");
        return T3B_ERR_ARG;
    }
    const size_t smem = ((size_t) 4 * p->n + 1) * sizeof(int);
    if (smem > 40 * 1024 &&
        cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (4 * PG_PLAN_MAXN + 1) * (int) sizeof(int)) != cudaSuccess) {
        set_err(nullptr, "t3b_op_kv_plan: shared memory attribute");
        return T3B_ERR_CUDA;
    }
    // one CTA does for few requests and rows; eight cost 0.3 us more and take a larger step's work apart
    const int rows = p->row_req || p->row_pos || p->slots ? p->rows_cap : 0;   // that the maps hold
    const PgRowMaps maps = rows == 0 ? PgRowMaps::none : rows <= PG_PLAN_ROWS ? PgRowMaps::here : PgRowMaps::apart;
    const int most = std::max(p->n, rows);
    const unsigned threads = most <= 128 ? 128 : most <= 256 ? 256 : PG_PLAN_T;
    const unsigned c = p->n <= PG_PLAN_T && rows <= PG_PLAN_T ? 1 : PG_PLAN_CLUSTER;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = c; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(c); cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t) cuda_stream; cfg.attrs = at; cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kv_plan_kernel, *p, maps);
    if (e == cudaSuccess && maps == PgRowMaps::apart) {
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.gridDim = dim3((unsigned) ((rows + 1023) / 1024)); cfg.blockDim = dim3(256);
        cfg.dynamicSmemBytes = ((size_t) p->n + 1) * sizeof(int);
        e = cudaLaunchKernelEx(&cfg, kv_plan_rows_kernel, *p);
    }
    if (e != cudaSuccess) { set_err(nullptr, "t3b_op_kv_plan: %s", cudaGetErrorString(e)); (void) cudaGetLastError(); return T3B_ERR_CUDA; }
    return T3B_OK;
}

int t3b_op_kv_append(const t3b_kv_append * a, void * cuda_stream) {
    if (!a) { set_err(nullptr, "t3b_op_kv_append: null argument"); return T3B_ERR_ARG; }
    if (const char * w = pg_cache_wrong(a->cache, true)) { set_err(nullptr, "t3b_op_kv_append: %s", w); return T3B_ERR_ARG; }
    const t3b_paged_kv & c = a->cache;
    const int el = a->dtype == T3B_F32 ? 4 : 8;
    if (!a->k || !a->v || !a->slots || a->rows < 0 || (a->dtype != T3B_F32 && a->dtype != c.dtype) ||
        a->stride < (int64_t) c.n_kv_head * c.head_dim || a->stride % el || a->stride > (int64_t) 1 << 40 ||
        !pg_aligned(a->k) || !pg_aligned(a->v)) {
        set_err(nullptr, "t3b_op_kv_append: bad args (null pointer, type, stride or alignment)");
        return T3B_ERR_ARG;
    }
    if (a->rows == 0) return T3B_OK;
    PgAppendArgs p{};
    p.k = c.k; p.v = c.v; p.page_stride = pg_page_stride(c); p.ks = a->k; p.vs = a->v; p.stride = a->stride; p.slots = a->slots;
    p.rows = a->rows; p.n_slots = c.n_pages * c.page_size; p.n_kv_head = c.n_kv_head;
    pg_log2(c.page_size, 3, 8, &p.page_log2); pg_log2(c.head_dim, 6, 7, &p.dim_log2);
    const long long total = (long long) a->rows * c.n_kv_head * (c.head_dim / 8);
    const int U = total > 2ll * 148 * 2048 ? 2 : 1;
    if (total / (256 * U) >= 0x7fffffffll) { set_err(nullptr, "t3b_op_kv_append: too many rows"); return T3B_ERR_ARG; }
    const unsigned grid = (unsigned) ((total + 256 * U - 1) / (256 * U));
    cudaStream_t st = (cudaStream_t) cuda_stream;
    if (a->dtype != T3B_F32) pg_launch_append<__half, __half>(U, grid, st, p);   // 16-bit rows move as they are
    else if (c.dtype == T3B_F16) pg_launch_append<float, __half>(U, grid, st, p);
    else pg_launch_append<float, __nv_bfloat16>(U, grid, st, p);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) { set_err(nullptr, "t3b_op_kv_append: %s", cudaGetErrorString(e)); return T3B_ERR_CUDA; }
    return T3B_OK;
}

int t3b_op_attention_shared(const t3b_shared_attn * a, void * cuda_stream) {
    return pg_attention("t3b_op_attention_shared", a, false, cuda_stream);
}

int t3b_op_attention_shared_prompt(const t3b_shared_attn * a, void * cuda_stream) {
    return pg_attention("t3b_op_attention_shared_prompt", a, true, cuda_stream);
}

size_t t3b_op_attention_shared_workspace(const t3b_shared_attn * a) {
    if (!a || pg_attn_wrong(*a, true, false)) return 0;
    return std::max(pg_workspace(*a, true), a->rows == a->n ? pg_workspace(*a, false) : 0);
}

}  // extern "C"
