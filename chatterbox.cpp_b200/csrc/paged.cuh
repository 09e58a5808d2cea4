// paged.cuh — the paged K/V cache with shared prefixes (t3b_op_kv_plan,
// t3b_op_kv_append, t3b_op_attention_shared, t3b_op_attention_shared_prompt):
// kernels and the C entry points.  Included by t3b_abi.cu.
#pragma once

#include <cuda_bf16.h>

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

// exclusive prefix sums of two 64-bit values over the CTA; `tot` gets the sums
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
    unsigned long long va = red[lane][0], vb = red[lane][1];   // PG_PLAN_T / 32 = 32 warps
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

// One cluster.  Every CTA scans all requests (a few KB), so all of them know
// each request's first row, first new page and first returned page and come
// to the same verdict; the returned pages, the new pages and the rows are
// then flattened and shared out over the cluster's threads, each finding its
// request by bisection in shared memory.  A cluster barrier separates what
// reads the old state (lengths, n_free, the released rows of the table) from
// what overwrites it, which is what lets a slot be released and admitted in
// one step and the outputs be the inputs' own buffers.
__global__ __launch_bounds__(PG_PLAN_T, 1) void kv_plan_kernel(t3b_kv_plan p) {
    extern __shared__ int pg_sm[];
    __shared__ unsigned long long red[32][2];
    int * s_len = pg_sm, * s_row = s_len + p.n, * s_take = s_row + p.n, * s_back = s_take + p.n;
    const int tid = threadIdx.x, n = p.n, P = p.page_size;
    unsigned rank, csize;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(csize));
    const long long cap = (long long) p.max_blocks * P;
    const int F = *p.n_free;
    unsigned long long rows = 0, pages = 0;   // pages: new ones in the low half, returned ones in the high
    int bad = 0;
    for (int t0 = 0; t0 < n; t0 += PG_PLAN_T) {
        const int i = t0 + tid;
        int ln = 0, ad = 0, rl = 0;
        if (i < n) {
            ln = p.len[i]; ad = p.add[i]; rl = p.release ? p.release[i] : 0;
            if (ln < 0 || ad < 0 || rl < 0 || (long long) ln + ad > cap || rl > cap || (rl > 0 && ln > 0)) {
                bad = 1; ln = ad = rl = 0;
            }
        }
        const unsigned take = (unsigned) ((ln + ad + P - 1) / P - (ln + P - 1) / P), back = (unsigned) ((rl + P - 1) / P);
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
    const int me = (int) rank * PG_PLAN_T + tid, all = (int) csize * PG_PLAN_T;
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
            p.table[(size_t) i * p.max_blocks + (s_len[i] + P - 1) / P + (k - s_take[i])] = p.free_pages[top - 1 - k];
        }
    for (int r = me; r < p.rows_cap; r += all) {
        int req = -1, pos = -1, slot = -1;
        if (r < nrow) {
            req = pg_find(s_row, n, r);
            pos = s_len[req] + (r - s_row[req]);
            const int blk = pos / P, held = (s_len[req] + P - 1) / P;
            const int id = blk < held ? p.table[(size_t) req * p.max_blocks + blk]
                                      : p.free_pages[top - 1 - (s_take[req] + blk - held)];
            const bool sane = id >= 0 && id <= (0x7fffffff - P + 1) / P;   // the slot fits 31 bits
            slot = sane ? id * P + pos % P : -1;
            if (!sane) atomicOr(&g_paged_err, T3B_DEVERR_PAGE);
        }
        if (p.row_req) p.row_req[r] = req;
        if (p.row_pos) p.row_pos[r] = pos;
        if (p.slots) p.slots[r] = slot;
    }
    for (int i = me; i < n; i += all) {
        p.row_start[i] = ok ? s_row[i] : 0;
        if (p.len_out) {
            if (ok) p.len_out[i] = s_len[i] + (i + 1 < n ? s_row[i + 1] : nrow) - s_row[i];
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

// A thread moves eight elements of K and the same eight of V.
template <class S, class T>
__global__ __launch_bounds__(256) void kv_append_kernel(PgAppendArgs a) {
    const int wlog = a.dim_log2 - 3, per_row = a.n_kv_head << wlog;   // 16-byte chunks of a head / of a row
    const long long total = (long long) a.rows * per_row;
    for (long long x = (long long) blockIdx.x * blockDim.x + threadIdx.x; x < total; x += (long long) gridDim.x * blockDim.x) {
        const int row = (int) (x / per_row), c = (int) (x - (long long) row * per_row);
        const int slot = __ldg(a.slots + row);
        if (slot < 0) continue;
        if (slot >= a.n_slots) { if (c == 0) atomicOr(&g_paged_err, T3B_DEVERR_PAGE); continue; }
        const int h = c >> wlog;
        const long long src = (long long) row * a.stride + ((long long) c << 3);
        const long long dst = (long long) (slot >> a.page_log2) * a.page_stride +
                              ((((long long) h << a.page_log2) + (slot & ((1 << a.page_log2) - 1))) << a.dim_log2) +
                              ((c & ((1 << wlog) - 1)) << 3);
        const uint4 kk = pg_pack8<S, T>((const S *) a.ks + src), vv = pg_pack8<S, T>((const S *) a.vs + src);
        *(uint4 *) ((T *) a.k + dst) = kk;
        *(uint4 *) ((T *) a.v + dst) = vv;
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

// The plain form: one CTA per (row, head), its warps striding the keys, each
// lane holding D / 32 dimensions, every key's dot product added over the
// warp.
template <class T, class C, int D>
__global__ __launch_bounds__(128) void attn_shared_simple_kernel(PgAttn a) {
    constexpr int E = D / 32;
    __shared__ float sm_m[4], sm_l[4], sm_o[4][D];
    const int h = blockIdx.y, r = blockIdx.x, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int i = r, add = 1, at = 0;
    if (a.row_start) {
        if (r >= __ldg(a.row_start + a.n)) return;
        int lo = 0, hi = a.n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (__ldg(a.row_start + mid) <= r) lo = mid; else hi = mid;
        }
        i = lo;
        add = __ldg(a.row_start + i + 1) - __ldg(a.row_start + i);
        at = r - __ldg(a.row_start + i);
    }
    const int len = __ldg(a.len + i), px = pg_prefix_of(a, i);
    const int plen = px >= 0 ? __ldg(a.prefix_len + px) : 0;
    const bool one = a.row_start == nullptr;
    if (len < 0 || len > (a.max_blocks << a.page_log2) || plen < 0 || plen > (a.prefix_max_blocks << a.page_log2) ||
        (!one && (add <= 0 || add > len || at < 0))) {
        if (threadIdx.x == 0) atomicOr(&g_paged_err, T3B_DEVERR_POS);
        return;
    }
    const int own = one ? len : len - add + at + 1, total = plen + own;
    const int kvh = h / a.group;
    const T * q = (const T *) a.q + (long long) r * a.q_stride + h * D;
    float qv[E], o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) { qv[e] = pg_to(q[lane * E + e]); o[e] = 0.0f; }
    float m = -INFINITY, l = 0.0f;
    for (int j = w; j < total; j += 4) {
        const int t = j < plen ? j : j - plen;
        const int * tab = j < plen ? a.prefix_table + (long long) px * a.prefix_max_blocks : a.table + (long long) i * a.max_blocks;
        const int id = __ldg(tab + (t >> a.page_log2));
        if ((unsigned) id >= (unsigned) a.n_pages) { if (lane == 0) atomicOr(&g_paged_err, T3B_DEVERR_PAGE); continue; }
        const long long off = (long long) id * a.page_stride +
                              (((long long) kvh << a.page_log2) + (t & ((1 << a.page_log2) - 1))) * D + lane * E;
        const C * kp = (const C *) a.k + off, * vp = (const C *) a.v + off;
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) s = fmaf(qv[e], pg_to(kp[e]), s);
        s = warp_sum(s) * a.scale;
        const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.0f : expf(m - mn), p = expf(s - mn);
        l = l * c + p;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * c + p * pg_to(vp[e]);
        m = mn;
    }
    if (lane == 0) { sm_m[w] = m; sm_l[w] = l; }
#pragma unroll
    for (int e = 0; e < E; ++e) sm_o[w][lane * E + e] = o[e];
    __syncthreads();
    const float mx = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
    T * out = (T *) a.out + (long long) r * a.out_stride + h * D;
    for (int d = threadIdx.x; d < D; d += 128) {
        float ls = 0.0f, os = 0.0f;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const float c = sm_m[x] == -INFINITY ? 0.0f : expf(sm_m[x] - mx);
            ls += c * sm_l[x]; os += c * sm_o[x][d];
        }
        out[d] = pg_from<T>(ls > 0.0f ? os / ls : 0.0f);
    }
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
    if (c.page_stride && (c.page_stride < dense || c.page_stride % 8 || c.page_stride > (int64_t) 1 << 40))
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
    if (a.n <= 0 || a.n > 65535 || a.n_prefix < 0 || a.n_prefix > 65535 || a.rows < 0) return "n, n_prefix or rows is out of range";
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

size_t pg_workspace(const t3b_shared_attn & a, bool prompt) { (void) a; (void) prompt; return 0; }

PgAttn pg_args(const t3b_shared_attn & a, bool prompt) {
    PgAttn p{};
    p.k = a.cache.k; p.v = a.cache.v; p.q = a.q; p.out = a.out;
    p.page_stride = pg_page_stride(a.cache); p.q_stride = a.q_stride; p.out_stride = a.out_stride;
    p.len = a.len; p.table = a.table; p.row_start = prompt ? a.row_start : nullptr;
    p.prefix_start = a.prefix_start; p.prefix_len = a.prefix_len; p.prefix_table = a.prefix_table;
    p.n = a.n; p.rows = a.rows; p.n_head = a.n_head; p.n_kv_head = a.cache.n_kv_head; p.group = a.n_head / a.cache.n_kv_head;
    pg_log2(a.cache.page_size, 3, 8, &p.page_log2);
    p.n_pages = a.cache.n_pages; p.max_blocks = a.max_blocks; p.n_prefix = a.n_prefix; p.prefix_max_blocks = a.prefix_max_blocks;
    p.scale = a.scale != 0.0f ? a.scale : 1.0f / sqrtf((float) a.cache.head_dim);
    return p;
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
    const dim3 grid(a->rows, a->n_head);
    const int D = a->cache.head_dim;
    if (a->dtype == T3B_F32) {
        if (D == 64) attn_shared_simple_kernel<float, __half, 64><<<grid, 128, 0, st>>>(p);
        else attn_shared_simple_kernel<float, __half, 128><<<grid, 128, 0, st>>>(p);
    } else if (a->dtype == T3B_F16) {
        if (D == 64) attn_shared_simple_kernel<__half, __half, 64><<<grid, 128, 0, st>>>(p);
        else attn_shared_simple_kernel<__half, __half, 128><<<grid, 128, 0, st>>>(p);
    } else {
        if (D == 64) attn_shared_simple_kernel<__nv_bfloat16, __nv_bfloat16, 64><<<grid, 128, 0, st>>>(p);
        else attn_shared_simple_kernel<__nv_bfloat16, __nv_bfloat16, 128><<<grid, 128, 0, st>>>(p);
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) { set_err(nullptr, "%s: %s", name, cudaGetErrorString(e)); return T3B_ERR_CUDA; }
    return T3B_OK;
}

}  // namespace

extern "C" {

int t3b_op_kv_plan(const t3b_kv_plan * p, void * cuda_stream) {
    int lg;
    if (!p || !p->len || !p->add || !p->free_pages || !p->n_free || !p->n_free_out || !p->table || !p->row_start ||
        p->n <= 0 || p->n > PG_PLAN_MAXN || p->rows_cap < 0 || p->free_cap < 0 || p->max_blocks <= 0 ||
        !pg_log2(p->page_size, 3, 8, &lg) || (int64_t) p->max_blocks * p->page_size > 0x3fffffffll ||
        (int64_t) p->n * p->max_blocks > 0x3fffffffll) {
        set_err(nullptr, "t3b_op_kv_plan: bad args");
        return T3B_ERR_ARG;
    }
    const size_t smem = (size_t) 4 * p->n * sizeof(int);
    if (smem > 40 * 1024 &&
        cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * PG_PLAN_MAXN * (int) sizeof(int)) != cudaSuccess) {
        set_err(nullptr, "t3b_op_kv_plan: shared memory attribute");
        return T3B_ERR_CUDA;
    }
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = PG_PLAN_CLUSTER; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(PG_PLAN_CLUSTER); cfg.blockDim = dim3(PG_PLAN_T); cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t) cuda_stream; cfg.attrs = at; cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kv_plan_kernel, *p);
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
    const unsigned grid = (unsigned) std::min<long long>((total + 255) / 256, 1 << 20);
    cudaStream_t st = (cudaStream_t) cuda_stream;
    if (a->dtype != T3B_F32) kv_append_kernel<__half, __half><<<grid, 256, 0, st>>>(p);   // 16-bit rows move as they are
    else if (c.dtype == T3B_F16) kv_append_kernel<float, __half><<<grid, 256, 0, st>>>(p);
    else kv_append_kernel<float, __nv_bfloat16><<<grid, 256, 0, st>>>(p);
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
