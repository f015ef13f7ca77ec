// pages.hip — pages of a key/value cache for gfx950: truncate / free, fork, reserve (with copy of a shared last page), append, commit of
// an accepted draft, compaction (include/whisper_amd.h, wx_cache_*).
//
// All bookkeeping lives in device memory and is done by kernels, so that a drafted decode loop needs no host round trip and can be
// captured.  Two kinds of kernels: small ones over tables and counts (latency: one or two launches each), and copies of rows, which
// are 16 B a lane over memory that is contiguous per (layer, page, head).  Counts of users are integers: the order of the atomics
// does not matter.  Page numbers read from a table are checked against the pool before they address anything.
#include "common.h"

namespace wx {

constexpr int PG_MAX_SEQS = 8192;
constexpr int PG_NT = 1024;            // workgroup of the bookkeeping scans

// (small: a launch costs the host 2.6 us with 8 bytes of arguments, 3.3 with 320)
struct PageArgs {
    wx_cache c;
    const int32_t *seqs, *list, *path;   // list: sources (fork), lengths (truncate), tokens (reserve), counts (append, commit)
    int32_t* out;                        // status of every entry; compaction: number of live pages
    int n, n_extra, n_nodes;
    int per_group;                       // layers a workgroup
    int es;                              // bytes an element
};
struct AppendArgs {
    PageArgs a;
    const char *rk, *rv;
    int64_t ks[4], vs[4];
    int layer0, n_layers;
};

// ---- work buffer: one part for each purpose (include/whisper_amd.h: never kept between calls) ---------------------------------
__host__ __device__ static inline int64_t pad4(int64_t x) { return (x + 3) & ~(int64_t)3; }
__host__ __device__ static inline int32_t* w_pairs(const wx_cache& c) { return c.d_work; }                                  // [max_seqs][4]
__host__ __device__ static inline int32_t* w_need(const wx_cache& c) { return c.d_work + 4 * (int64_t)c.max_seqs; }         // [max_seqs][4]
__host__ __device__ static inline int32_t* w_free(const wx_cache& c) { return c.d_work + 8 * (int64_t)c.max_seqs; }         // [n_pages]
__host__ __device__ static inline int32_t* w_from(const wx_cache& c) { return w_free(c) + pad4(c.n_pages); }                // [n_pages]
__host__ __device__ static inline int32_t* w_map(const wx_cache& c) { return w_from(c) + pad4(c.n_pages); }                 // [n_pages]
__host__ __device__ static inline int32_t* w_count(const wx_cache& c) { return w_map(c) + pad4(c.n_pages); }                // [4]
__host__ __device__ static inline int32_t* w_rows(const wx_cache& c) { return w_count(c) + 4; }                             // [max_seqs][max_pages + 2]

static int64_t work_ints(const wx_cache& c) {
    return 8 * (int64_t)c.max_seqs + 3 * pad4(c.n_pages) + 4 + (int64_t)c.max_seqs * ((int64_t)c.max_pages + 2);
}

const char* cache_fault(const wx_cache* c) {
    if (!c) return "null cache";
    if (!c->d_k || !c->d_v || !c->d_table || !c->d_refs || !c->d_lens || !c->d_held || !c->d_work) return "null buffer in the cache";
    if (c->n_layer < 1 || c->n_pages < 1 || c->n_kv_head < 1 || c->max_seqs < 1 || c->max_pages < 1) return "bad cache dimensions";
    if (c->max_seqs > PG_MAX_SEQS) return "max_seqs must be at most 8192";
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128 && c->page_size != 256)
        return "page_size must be 16, 32, 64, 128 or 256";
    if (c->head_dim != 64 && c->head_dim != 128) return "head_dim must be 64 or 128";
    if (c->precision != WX_PREC_F32 && c->precision != WX_PREC_BF16) return "bad precision";
    if (c->n_kv_head > 4096 || c->n_layer > 4096 || c->n_pages > 0x3fffffff || (int64_t)c->max_pages * c->page_size > 0x3fffffff || (int64_t)c->max_seqs * c->max_pages > 0x7fffffff)
        return "cache dimensions too large";
    if (((uintptr_t)c->d_k | (uintptr_t)c->d_v | (uintptr_t)c->d_refs | (uintptr_t)c->d_work) & 15) return "cache buffers must be 16-byte aligned";
    return nullptr;
}

// one workgroup: whether seqs[i] is in range and not in the list before i (every thread gets the answer)
__device__ __forceinline__ bool entry_ok(const int32_t* seqs, int i, int max_seqs) {
    const int s = seqs[i];
    int twin = 0;
    for (int j = threadIdx.x; j < i; j += blockDim.x) twin |= seqs[j] == s;
    twin = __syncthreads_or(twin);
    return s >= 0 && s < max_seqs && !twin;
}
__device__ __forceinline__ void unref(const wx_cache& c, int page) { if ((unsigned)page < (unsigned)c.n_pages) atomicSub(&c.d_refs[page], 1); }

// ---- truncate / free ------------------------------------------------------------------------------------------------------------
// One workgroup an entry (its pages' counts are independent).  Latency: 4 us for 60 entries.
__global__ __launch_bounds__(128) void cache_truncate_kernel(PageArgs a) {
    const wx_cache& c = a.c;
    const int i = blockIdx.x;
    bool ok = entry_ok(a.seqs, i, c.max_seqs);
    const int s = a.seqs[i];
    int len = 0, held = 0, want = 0;
    if (ok) { len = c.d_lens[s]; held = min(c.d_held[s], c.max_pages); want = a.list ? a.list[i] : 0; ok = want >= 0 && want <= len; }
    __syncthreads();
    if (threadIdx.x == 0 && a.out) a.out[i] = ok ? WX_OK : WX_ERR_INVALID;
    if (!ok) return;
    const int keep = (want + c.page_size - 1) / c.page_size;
    int32_t* row = c.d_table + (int64_t)s * c.max_pages;
    for (int p = keep + threadIdx.x; p < held; p += blockDim.x) { unref(c, row[p]); row[p] = -1; }
    if (threadIdx.x == 0) { c.d_lens[s] = want; c.d_held[s] = min(held, keep); }
}

// ---- fork: all sources are read (and their pages counted up) before any destination is written -----------------------------------
__global__ __launch_bounds__(128) void cache_fork_read_kernel(PageArgs a) {
    const wx_cache& c = a.c;
    const int i = blockIdx.x, src = a.list[i];
    const bool ok = entry_ok(a.seqs, i, c.max_seqs) && src >= 0 && src < c.max_seqs;
    int32_t* to = w_rows(c) + (int64_t)i * (c.max_pages + 2);
    if (!ok) { if (threadIdx.x == 0) to[0] = -1; return; }
    const int len = c.d_lens[src], keep = min((len + c.page_size - 1) / c.page_size, min(c.d_held[src], c.max_pages));
    if (threadIdx.x == 0) { to[0] = len; to[1] = keep; }
    const int32_t* row = c.d_table + (int64_t)src * c.max_pages;
    for (int p = threadIdx.x; p < keep; p += blockDim.x) {
        const int page = row[p];
        to[2 + p] = page;
        if ((unsigned)page < (unsigned)c.n_pages) atomicAdd(&c.d_refs[page], 1);
    }
}
__global__ __launch_bounds__(128) void cache_fork_write_kernel(PageArgs a) {
    const wx_cache& c = a.c;
    const int i = blockIdx.x;
    const int32_t* from = w_rows(c) + (int64_t)i * (c.max_pages + 2);
    const int len = from[0];
    if (threadIdx.x == 0 && a.out) a.out[i] = len < 0 ? WX_ERR_INVALID : WX_OK;
    if (len < 0) return;
    const int s = a.seqs[i], keep = from[1], held = min(c.d_held[s], c.max_pages);
    __syncthreads();
    int32_t* row = c.d_table + (int64_t)s * c.max_pages;
    for (int p = threadIdx.x; p < max(held, keep); p += blockDim.x) {
        if (p < held) unref(c, row[p]);
        row[p] = p < keep ? from[2 + p] : -1;
    }
    if (threadIdx.x == 0) { c.d_lens[s] = len; c.d_held[s] = keep; }
}

// The same in one launch, by one workgroup that keeps what it read in LDS: lists of up to FK_ENTRIES x tables of up to FK_CELLS cells.
// Latency: 4.6 us for 15 entries of 13 pages, 9.1 us for 60 of 28 (the launch it saves costs 4 to 5 us and 3 us of the host's time; above the
// limits the tables no longer fit one workgroup's LDS).
constexpr int FK_ENTRIES = 512, FK_CELLS = 8192;
__global__ __launch_bounds__(1024) void cache_fork_small_kernel(PageArgs a) {
    __shared__ int cells[FK_CELLS], s_len[FK_ENTRIES], s_keep[FK_ENTRIES], s_held[FK_ENTRIES];
    const wx_cache& c = a.c;
    const int tid = threadIdx.x, MP = c.max_pages, n = a.n;
    for (int i = tid; i < n; i += 1024) {
        const int d = a.seqs[i], src = a.list[i];
        bool ok = d >= 0 && d < c.max_seqs && src >= 0 && src < c.max_seqs;
        for (int j = 0; j < i; ++j) ok &= a.seqs[j] != d;
        const int len = ok ? c.d_lens[src] : -1;
        s_len[i] = len;
        s_keep[i] = len < 0 ? 0 : min((len + c.page_size - 1) / c.page_size, min(c.d_held[src], MP));
        s_held[i] = len < 0 ? 0 : min(c.d_held[d], MP);
        if (a.out) a.out[i] = len < 0 ? WX_ERR_INVALID : WX_OK;
    }
    __syncthreads();
    for (int u = tid; u < n * MP; u += 1024) {
        const int i = u / MP, q = u % MP;
        int page = -1;
        if (q < s_keep[i]) {
            page = c.d_table[(int64_t)a.list[i] * MP + q];
            if ((unsigned)page < (unsigned)c.n_pages) atomicAdd(&c.d_refs[page], 1);
        }
        cells[u] = page;
    }
    __syncthreads();
    for (int u = tid; u < n * MP; u += 1024) {
        const int i = u / MP, q = u % MP;
        if (s_len[i] < 0 || q >= max(s_held[i], s_keep[i])) continue;
        int32_t* cell = c.d_table + (int64_t)a.seqs[i] * MP + q;
        if (q < s_held[i]) unref(c, *cell);
        *cell = cells[u];
    }
    for (int i = tid; i < n; i += 1024) if (s_len[i] >= 0) { c.d_lens[a.seqs[i]] = s_len[i]; c.d_held[a.seqs[i]] = s_keep[i]; }
}

// inclusive sum over a workgroup of PG_NT threads; *total = the sum of all
__device__ __forceinline__ int block_scan(int v, int* sh, int* total) {
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) { const int u = __shfl_up(v, off); if (lane >= off) v += u; }
    __syncthreads();
    if (lane == 63) sh[wid] = v;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < PG_NT / 64; ++w) { const int x = sh[w]; if (w < wid) before += x; all += x; }
    *total = all;
    return v + before;
}

// ---- reserve: one workgroup does the bookkeeping of all entries, then a launch copies the shared last pages ------------------------
// Pages are given out in the order of the list, lowest first, which is a sum over all entries: one workgroup, 6.3 us for 15 entries, 9.5 for 60
// on 560 pages (latency).  The copy: 12 x 5 children of large-v3's size, 32 layers x 20 heads of 64: 97 MB in 17 us, 5.7 TB/s.
__global__ __launch_bounds__(PG_NT) void cache_reserve_kernel(PageArgs a) {
    __shared__ int sh[PG_NT / 64], owner[PG_MAX_SEQS];
    const wx_cache& c = a.c;
    const int tid = threadIdx.x, PS = c.page_size;
    int32_t *need_l = w_need(c), *free_l = w_free(c), *pairs = w_pairs(c);
    for (int i = tid; i < a.n; i += PG_NT) { const int s = a.seqs[i]; if (s >= 0 && s < c.max_seqs) owner[s] = 0x7fffffff; }
    __syncthreads();
    for (int i = tid; i < a.n; i += PG_NT) { const int s = a.seqs[i]; if (s >= 0 && s < c.max_seqs) atomicMin(&owner[s], i); }
    __syncthreads();
    // what every entry needs, and the sum of what the entries up to it need
    int sum = 0;
    for (int i0 = 0; i0 < a.n; i0 += PG_NT) {
        const int i = i0 + tid;
        int need = 0, copy = 0, st = WX_ERR_INVALID;
        if (i < a.n) {
            const int s = a.seqs[i], extra = a.list ? a.list[i] : a.n_extra;
            if (s >= 0 && s < c.max_seqs && owner[s] == i && extra >= 0) {
                const int len = c.d_lens[s], held = c.d_held[s];
                const int64_t want = ((int64_t)len + extra + PS - 1) / PS;
                st = len < 0 || held < 0 || held > c.max_pages ? WX_ERR_INVALID : WX_OK;
                if (st == WX_OK && want > c.max_pages) st = WX_ERR_NOMEM;
                if (st == WX_OK) {
                    if (extra > 0 && len % PS && len / PS < held) {
                        const int p = c.d_table[(int64_t)s * c.max_pages + len / PS];
                        copy = (unsigned)p < (unsigned)c.n_pages && c.d_refs[p] > 1;
                    }
                    need = copy + max(0, (int)want - held);
                }
            }
        }
        int all;
        const int upto = sum + block_scan(need, sh, &all);
        sum += all;
        if (i < a.n) { need_l[4 * i] = upto - need; need_l[4 * i + 1] = need; need_l[4 * i + 2] = copy; need_l[4 * i + 3] = st; }
    }
    // the lowest free pages, in order, as many as are needed
    int found = 0;
    for (int p0 = 0; p0 < c.n_pages && found < sum; p0 += 4 * PG_NT) {
        const int p = p0 + 4 * tid;
        int f[4], k = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) { f[j] = p + j < c.n_pages && c.d_refs[p + j] == 0; k += f[j]; }
        int all;
        int at = found + block_scan(k, sh, &all) - k;
#pragma unroll
        for (int j = 0; j < 4; ++j) if (f[j]) { if (at < sum) free_l[at] = p + j; ++at; }
        found += all;
    }
    __syncthreads();
    // a wave an entry: table columns, counts, and the pair of pages to copy
    const int lane = tid & 63;
    for (int i = tid >> 6; i < a.n; i += PG_NT / 64) {
        const int first = need_l[4 * i], need = need_l[4 * i + 1], copy = need_l[4 * i + 2];
        int st = need_l[4 * i + 3];
        if (st == WX_OK && need > 0 && first + need > found) st = WX_ERR_NOMEM;
        const bool go = st == WX_OK && need > 0;
        if (lane == 0) {
            if (a.out) a.out[i] = st;
            pairs[4 * i] = -1;
        }
        if (!go) continue;
        const int s = a.seqs[i], len = c.d_lens[s], held = c.d_held[s], fresh = need - copy;
        int32_t* row = c.d_table + (int64_t)s * c.max_pages;
        if (copy && lane == 0) {
            const int was = row[len / PS], now = free_l[first];
            row[len / PS] = now;
            c.d_refs[now] = 1;
            atomicSub(&c.d_refs[was], 1);
            pairs[4 * i] = was; pairs[4 * i + 1] = now; pairs[4 * i + 2] = len % PS;
        }
        for (int j = lane; j < fresh; j += 64) {
            const int now = free_l[first + copy + j];
            row[held + j] = now;
            c.d_refs[now] = 1;
        }
        if (lane == 0 && fresh > 0) c.d_held[s] = held + fresh;
    }
}
// grid (entry, layer, keys / values): the committed rows of the page, every head
__global__ __launch_bounds__(256) void cache_copy_tail_kernel(PageArgs a) {
    const wx_cache& c = a.c;
    const int32_t* pair = w_pairs(c) + 4 * (int64_t)blockIdx.x;
    const int from = pair[0];
    if (from < 0) return;
    const int to = pair[1], fill = pair[2];
    const int64_t row_b = (int64_t)c.head_dim * a.es, head_b = row_b * c.page_size, page_b = head_b * c.n_kv_head;
    char* pool = (char*)(blockIdx.z ? c.d_v : c.d_k) + (int64_t)blockIdx.y * c.n_pages * page_b;
    const int per = (int)(fill * row_b / 16);                        // 16-byte units a head
    for (int u = threadIdx.x; u < per * c.n_kv_head; u += 256) {
        const int64_t off = (u / per) * head_b + (int64_t)(u % per) * 16;
        *reinterpret_cast<i32x4*>(pool + to * page_b + off) = *reinterpret_cast<const i32x4*>(pool + from * page_b + off);
    }
}

// ---- append: grid (entry, group of AP_NODES nodes, group of layers) -------------------------------------------------------------------
// The entry is checked and its places are looked up once for all layers of the group; a thread then takes its 16 bytes of keys and of
// values through the layers, two layers' loads at a time.  Bound by the copy: 64 x 16 rows (769 there), 32 layers x 20 heads of 64: 252 MB in
// 52 us, 4.8 TB/s; 16 x 24 rows, 4 layers: 7 us (latency).
constexpr int AP_NODES = 4;
__global__ __launch_bounds__(256) void cache_append_kernel(AppendArgs b) {
    __shared__ int64_t place[AP_NODES];
    const PageArgs& a = b.a;
    const wx_cache& c = a.c;
    const int i = blockIdx.x, j0 = blockIdx.y * AP_NODES, tid = threadIdx.x;
    const int l0 = blockIdx.z * a.per_group, l1 = min(b.n_layers, l0 + a.per_group);
    const int64_t row_b = (int64_t)c.head_dim * a.es, head_b = row_b * c.page_size, page_b = head_b * c.n_kv_head, layer_b = page_b * c.n_pages;
    const int per = (int)(row_b / 16), heads = c.n_kv_head;
    const int64_t kstep = b.ks[0] * a.es, vstep = b.vs[0] * a.es;
    auto k_at = [&](int u) { const int x = u % per, h = (u / per) % heads, j = u / (per * heads); return b.rk + (l0 * b.ks[0] + i * b.ks[1] + (j0 + j) * b.ks[2] + h * b.ks[3]) * a.es + x * 16; };
    auto v_at = [&](int u) { const int x = u % per, h = (u / per) % heads, j = u / (per * heads); return b.rv + (l0 * b.vs[0] + i * b.vs[1] + (j0 + j) * b.vs[2] + h * b.vs[3]) * a.es + x * 16; };
    // the thread's first rows are on their way while the entry is looked up
    i32x4 k0 = {0, 0, 0, 0}, v0 = k0, k1 = k0, v1 = k0;
    auto load = [&](const char* k, const char* v, bool two) {
        k0 = *reinterpret_cast<const i32x4*>(k); v0 = *reinterpret_cast<const i32x4*>(v);
        if (two) { k1 = *reinterpret_cast<const i32x4*>(k + kstep); v1 = *reinterpret_cast<const i32x4*>(v + vstep); }
    };
    const int s = a.seqs[i], count = a.list ? min(a.list[i], a.n_nodes) : a.n_nodes, nodes = min(AP_NODES, count - j0);
    if (tid < nodes * heads * per) load(k_at(tid), v_at(tid), l0 + 1 < l1);
    int bad = 0;
    for (int j = tid; j < i; j += 256) bad |= a.seqs[j] == s;
    if (j0 >= count || s < 0 || s >= c.max_seqs) return;
    const int len = c.d_lens[s], held = min(c.d_held[s], c.max_pages);
    if (len < 0 || (int64_t)len + count > (int64_t)held * c.page_size) return;
    const int32_t* row = c.d_table + (int64_t)s * c.max_pages;
    if (tid < nodes) {
        const int t = len + j0 + tid;
        place[tid] = row[t / c.page_size] * page_b + (t % c.page_size) * row_b;                  // (used if the pages are found right)
    }
    for (int q = len / c.page_size + tid; q <= (len + count - 1) / c.page_size; q += 256) {
        const int page = row[q];
        if ((unsigned)page >= (unsigned)c.n_pages || c.d_refs[page] != 1) bad = 1;
    }
    if (__syncthreads_or(bad)) return;
    for (int u = tid; u < nodes * heads * per; u += 256) {
        const char *k = k_at(u), *v = v_at(u);
        const int64_t to = (b.layer0 + l0) * layer_b + place[u / (per * heads)] + (u / per) % heads * head_b + u % per * 16;
        char *kt = (char*)c.d_k + to, *vt = (char*)c.d_v + to;
        if (u != tid) load(k, v, l0 + 1 < l1);
        for (int l = l0; l < l1; l += 2) {
            const bool two = l + 1 < l1;
            *reinterpret_cast<i32x4*>(kt) = k0; *reinterpret_cast<i32x4*>(vt) = v0;
            if (two) { *reinterpret_cast<i32x4*>(kt + layer_b) = k1; *reinterpret_cast<i32x4*>(vt + layer_b) = v1; }
            k += 2 * kstep; v += 2 * vstep; kt += 2 * layer_b; vt += 2 * layer_b;
            if (l + 2 < l1) load(k, v, l + 3 < l1);
        }
    }
}

// ---- commit ------------------------------------------------------------------------------------------------------------------------
// Whether entry i's path may be followed (every thread of the workgroup); *taken = its length, *stay = how many of its first blockDim.x rows
// stay where they are.  What depends on no other load is asked for first: list, count and path; then lengths; pages; their users.
__device__ __forceinline__ bool commit_ok(const PageArgs& a, int i, int* taken, int* stay) {
    const wx_cache& c = a.c;
    const int tid = threadIdx.x, nt = blockDim.x;
    const int32_t* path = a.path + (int64_t)i * a.n_nodes;
    const int s = a.seqs[i], k = a.list[i];
    const int mine = tid < a.n_nodes ? path[tid] : 0, before = tid > 0 && tid < a.n_nodes ? path[tid - 1] : -1;
    int bad = 0;
    for (int j = tid; j < i; j += nt) bad |= a.seqs[j] == s;
    *taken = k;
    if (s < 0 || s >= c.max_seqs || k < 0 || k > a.n_nodes) return false;
    const int len = c.d_lens[s], held = min(c.d_held[s], c.max_pages), last = k > 0 ? path[k - 1] : 0;
    bad |= tid < k && (mine < 0 || mine <= before);
    for (int j = tid + nt; j < k; j += nt) bad |= path[j] < 0 || path[j] <= path[j - 1];
    if (k > 0) {
        if (len < 0 || last < 0 || (int64_t)len + last + 1 > (int64_t)held * c.page_size) bad = 1;
        else {
            const int32_t* row = c.d_table + (int64_t)s * c.max_pages;
            for (int q = len / c.page_size + tid; q <= (len + last) / c.page_size; q += nt) {
                const int page = row[q];
                if ((unsigned)page >= (unsigned)c.n_pages || c.d_refs[page] != 1) bad = 1;
            }
        }
    }
    *stay = __syncthreads_count(tid < k && mine == tid);             // a path ascends: the first ones
    return !__syncthreads_or(bad);
}
// grid (entry, group of layers): a thread takes 16 bytes of a head's rows of one layer, keys or values, down the whole path.  path[k] >= k
// and ascends, so a row that is overwritten was read before by the same thread (eight rows are read before they are written); rows that
// stay (path[k] == k) are not touched.  Where one group holds all layers, the workgroup sets the length itself (saves a launch: 4.7 us).
// 64 entries, 32 layers x 20 heads of 64, 241 rows taken: 38 MB in 13 us; 16 entries, 4 layers: 8.6 us (latency).
constexpr int CM_ROWS = 64;                                          // moves looked up at a time
__global__ __launch_bounds__(256) void cache_commit_rows_kernel(PageArgs a) {
    __shared__ int64_t from[CM_ROWS], to[CM_ROWS];
    const wx_cache& c = a.c;
    const int i = blockIdx.x;
    int taken, k0;
    const bool ok = commit_ok(a, i, &taken, &k0);
    const bool all = gridDim.y == 1;
    if (all && threadIdx.x == 0 && a.out) a.out[i] = ok ? WX_OK : WX_ERR_INVALID;
    if (!ok) return;
    const int s = a.seqs[i], len = c.d_lens[s];
    const int32_t* path = a.path + (int64_t)i * a.n_nodes;
    const int32_t* row = c.d_table + (int64_t)s * c.max_pages;
    const int64_t row_b = (int64_t)c.head_dim * a.es, head_b = row_b * c.page_size, page_b = head_b * c.n_kv_head, layer_b = page_b * c.n_pages;
    const int per = (int)(row_b / 16), cols = c.n_kv_head * per, l0 = blockIdx.y * a.per_group, layers = min(c.n_layer, l0 + a.per_group) - l0;
    if (k0 == blockDim.x) while (k0 < taken && path[k0] == k0) ++k0;  // (uniform)
    for (; k0 < taken; k0 += CM_ROWS) {
        const int moves = min(CM_ROWS, taken - k0);
        __syncthreads();
        for (int k = threadIdx.x; k < moves; k += 256) {
            const int f = len + path[k0 + k], t = len + k0 + k;
            from[k] = row[f / c.page_size] * page_b + (f % c.page_size) * row_b;
            to[k] = row[t / c.page_size] * page_b + (t % c.page_size) * row_b;
        }
        __syncthreads();
        for (int u = threadIdx.x; u < cols * layers * 2; u += 256) {
            const int col = u % cols, w = u / cols;                  // w: layer, keys / values
            char* pool = (char*)(w & 1 ? c.d_v : c.d_k) + (l0 + (w >> 1)) * layer_b + (col / per) * head_b + (col % per) * 16;
            for (int k = 0; k < moves; k += 8) {
                i32x4 x[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) x[q] = *reinterpret_cast<const i32x4*>(pool + from[min(k + q, moves - 1)]);
#pragma unroll
                for (int q = 0; q < 8; ++q) if (k + q < moves) *reinterpret_cast<i32x4*>(pool + to[k + q]) = x[q];
            }
        }
    }
    if (all) {
        __syncthreads();
        if (threadIdx.x == 0) c.d_lens[s] = len + taken;
    }
}
__global__ __launch_bounds__(64) void cache_commit_len_kernel(PageArgs a) {
    const int i = blockIdx.x;
    int taken, stay;
    const bool ok = commit_ok(a, i, &taken, &stay);
    __syncthreads();
    if (threadIdx.x == 0) {
        if (a.out) a.out[i] = ok ? WX_OK : WX_ERR_INVALID;
        if (ok) a.c.d_lens[a.seqs[i]] += taken;
    }
}

// ---- compaction ----------------------------------------------------------------------------------------------------------------------
// The plan pairs the i-th live page behind the n_live-th place with the i-th hole before it (5.6 us for 1024 pages), the move copies whole pages,
// the table kernel renames them.  Bound by the copy: 247 pages of large-v3's size: 1295 MB in 257 us, 5.0 TB/s.
__global__ __launch_bounds__(PG_NT) void cache_compact_plan_kernel(PageArgs a) {
    __shared__ int sh[PG_NT / 64];
    const wx_cache& c = a.c;
    const int tid = threadIdx.x;
    int32_t *hole = w_free(c), *from = w_from(c), *map = w_map(c);
    int live = 0;
    for (int p0 = 0; p0 < c.n_pages; p0 += PG_NT) {
        int all;
        (void)block_scan(p0 + tid < c.n_pages && c.d_refs[p0 + tid] > 0, sh, &all);
        live += all;
    }
    int holes = 0, moves = 0;
    for (int p0 = 0; p0 < c.n_pages; p0 += PG_NT) {
        const int p = p0 + tid;
        const bool in = p < c.n_pages, used = in && c.d_refs[p] > 0;
        const int is_hole = in && !used && p < live, is_move = used && p >= live;
        int all_h, all_m;
        const int h = holes + block_scan(is_hole, sh, &all_h) - 1, m = moves + block_scan(is_move, sh, &all_m) - 1;
        if (is_hole) hole[h] = p;
        if (is_move) from[m] = p;
        if (in) map[p] = p;
        holes += all_h; moves += all_m;
    }
    __syncthreads();
    for (int i = tid; i < moves; i += PG_NT) {                        // as many holes as moves
        map[from[i]] = hole[i];
        c.d_refs[hole[i]] = c.d_refs[from[i]];
        c.d_refs[from[i]] = 0;
    }
    if (tid == 0) { *w_count(c) = moves; if (a.out) *a.out = live; }
}
// grid (any number, layer, keys / values): whole pages
__global__ __launch_bounds__(256) void cache_compact_move_kernel(PageArgs a) {
    const wx_cache& c = a.c;
    const int moves = *w_count(c);
    const int64_t page_b = (int64_t)c.head_dim * a.es * c.page_size * c.n_kv_head;
    char* pool = (char*)(blockIdx.z ? c.d_v : c.d_k) + (int64_t)blockIdx.y * c.n_pages * page_b;
    for (int m = blockIdx.x; m < moves; m += gridDim.x) {
        const char* from = pool + w_from(c)[m] * page_b;
        char* to = pool + w_free(c)[m] * page_b;
        for (int64_t u = threadIdx.x * 16; u < page_b; u += 256 * 16) *reinterpret_cast<i32x4*>(to + u) = *reinterpret_cast<const i32x4*>(from + u);
    }
}
__global__ __launch_bounds__(256) void cache_compact_table_kernel(PageArgs a) {
    const wx_cache& c = a.c;
    const int64_t all = (int64_t)c.max_seqs * c.max_pages;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int p = c.d_table[i];
        if ((unsigned)p < (unsigned)c.n_pages) { const int q = w_map(c)[p]; if (q != p) c.d_table[i] = q; }
    }
}

static PageArgs page_args(const wx_cache* c, const int32_t* seqs, int n, int32_t* status) {
    PageArgs a{};
    a.c = *c; a.seqs = seqs; a.n = n; a.out = status;
    a.es = c->precision == WX_PREC_F32 ? 4 : 2;
    return a;
}

}  // namespace wx

using namespace wx;

#define PG_CHECK(c) do { if (const char* _m = cache_fault(c)) return set_error(WX_ERR_INVALID, _m); } while (0)
#define PG_LIST(c, p, n) do { if ((n) < 0 || (n) > (c)->max_seqs || ((n) > 0 && !(p))) return set_error(WX_ERR_INVALID, "bad list of sequence slots (0 <= n <= max_seqs)"); } while (0)
#define PG_DONE() do { const hipError_t _e = hipGetLastError(); if (_e != hipSuccess) return set_error(WX_ERR_HIP, hipGetErrorString(_e)); return WX_OK; } while (0)

extern "C" {

int64_t wx_cache_work_ints(const wx_cache* c) {
    if (!c || c->n_pages < 1 || c->max_seqs < 1 || c->max_pages < 1) return set_error(WX_ERR_INVALID, "bad cache dimensions");
    return work_ints(*c);
}

int wx_cache_truncate(const wx_cache* c, const int32_t* d_seqs, const int32_t* d_lens, int32_t n, int32_t* d_status, void* stream) {
    PG_CHECK(c); PG_LIST(c, d_seqs, n);
    if (n == 0) return WX_OK;
    OnDevice on(c->device);
    PageArgs a = page_args(c, d_seqs, n, d_status);
    a.list = d_lens;
    hipLaunchKernelGGL(cache_truncate_kernel, dim3(n), dim3(128), 0, (hipStream_t)stream, a);
    PG_DONE();
}

int wx_cache_fork(const wx_cache* c, const int32_t* d_dst, const int32_t* d_src, int32_t n, int32_t* d_status, void* stream) {
    PG_CHECK(c); PG_LIST(c, d_dst, n);
    if (n == 0) return WX_OK;
    if (!d_src) return set_error(WX_ERR_INVALID, "null list of sources");
    OnDevice on(c->device);
    PageArgs a = page_args(c, d_dst, n, d_status);
    a.list = d_src;
    if (n <= FK_ENTRIES && (int64_t)n * c->max_pages <= FK_CELLS) {
        hipLaunchKernelGGL(cache_fork_small_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, a);
        PG_DONE();
    }
    hipLaunchKernelGGL(cache_fork_read_kernel, dim3(n), dim3(128), 0, (hipStream_t)stream, a);
    hipLaunchKernelGGL(cache_fork_write_kernel, dim3(n), dim3(128), 0, (hipStream_t)stream, a);
    PG_DONE();
}

int wx_cache_reserve(const wx_cache* c, const int32_t* d_seqs, const int32_t* d_extra, int32_t extra, int32_t n, int32_t* d_status, void* stream) {
    PG_CHECK(c); PG_LIST(c, d_seqs, n);
    if (!d_extra && extra < 0) return set_error(WX_ERR_INVALID, "extra must be >= 0");
    if (n == 0) return WX_OK;
    OnDevice on(c->device);
    PageArgs a = page_args(c, d_seqs, n, d_status);
    a.list = d_extra; a.n_extra = extra;
    hipLaunchKernelGGL(cache_reserve_kernel, dim3(1), dim3(PG_NT), 0, (hipStream_t)stream, a);
    hipLaunchKernelGGL(cache_copy_tail_kernel, dim3(n, c->n_layer, 2), dim3(256), 0, (hipStream_t)stream, a);
    PG_DONE();
}

int wx_cache_append(const wx_cache* c, const int32_t* d_seqs, const int32_t* d_counts, int32_t n, int32_t n_nodes, int32_t layer0, int32_t n_layers,
                    const void* d_k, const int64_t* k_strides, const void* d_v, const int64_t* v_strides, void* stream) {
    PG_CHECK(c); PG_LIST(c, d_seqs, n);
    if (layer0 < 0 || n_layers < 1 || (int64_t)layer0 + n_layers > c->n_layer) return set_error(WX_ERR_INVALID, "bad layer range");
    if (n_nodes < 0 || n_nodes > 65536) return set_error(WX_ERR_INVALID, "n_nodes must be 0 .. 65536");
    if (n == 0 || n_nodes == 0) return WX_OK;
    if (!d_k || !d_v || !k_strides || !v_strides) return set_error(WX_ERR_INVALID, "null rows");
    AppendArgs b{};
    PageArgs& a = b.a;
    a = page_args(c, d_seqs, n, nullptr);
    const int unit = 16 / a.es;
    for (int i = 0; i < 4; ++i) {
        b.ks[i] = k_strides[i]; b.vs[i] = v_strides[i];
        if (b.ks[i] < 0 || b.vs[i] < 0 || b.ks[i] % unit || b.vs[i] % unit) return set_error(WX_ERR_INVALID, "row strides must be >= 0 and multiples of 16 bytes");
    }
    if (((uintptr_t)d_k | (uintptr_t)d_v) & 15) return set_error(WX_ERR_INVALID, "rows must be 16-byte aligned");
    OnDevice on(c->device);
    a.list = d_counts; a.n_nodes = n_nodes; b.layer0 = layer0; b.n_layers = n_layers; b.rk = (const char*)d_k; b.rv = (const char*)d_v;
    // as many layers a workgroup as leave 2048 workgroups (8 on every CU): the look-up is paid once for them
    const int groups = (n_nodes + AP_NODES - 1) / AP_NODES;
    const int64_t z = (2048 + (int64_t)n * groups - 1) / ((int64_t)n * groups);
    a.per_group = (int)((n_layers + z - 1) / z);
    hipLaunchKernelGGL(cache_append_kernel, dim3(n, groups, (n_layers + a.per_group - 1) / a.per_group), dim3(256), 0, (hipStream_t)stream, b);
    PG_DONE();
}

int wx_cache_commit(const wx_cache* c, const int32_t* d_seqs, const int32_t* d_path, const int32_t* d_counts, int32_t n, int32_t n_nodes,
                    int32_t* d_status, void* stream) {
    PG_CHECK(c); PG_LIST(c, d_seqs, n);
    if (n_nodes < 0 || n_nodes > 65536) return set_error(WX_ERR_INVALID, "n_nodes must be 0 .. 65536");
    if (n == 0) return WX_OK;
    if (!d_counts || (n_nodes > 0 && !d_path)) return set_error(WX_ERR_INVALID, "null path or counts");
    OnDevice on(c->device);
    PageArgs a = page_args(c, d_seqs, n, d_status);
    a.path = d_path; a.list = d_counts; a.n_nodes = n_nodes;
    // one workgroup an entry where a token's rows of all layers are at most 32 KiB: no second launch for the lengths
    const int64_t token_b = 2 * (int64_t)c->n_layer * c->n_kv_head * c->head_dim * a.es;
    const int64_t y = token_b <= 32768 ? 1 : (1024 + n - 1) / n;
    a.per_group = (int)((c->n_layer + y - 1) / y);
    const int groups = (c->n_layer + a.per_group - 1) / a.per_group;
    hipLaunchKernelGGL(cache_commit_rows_kernel, dim3(n, groups), dim3(256), 0, (hipStream_t)stream, a);
    if (groups > 1) hipLaunchKernelGGL(cache_commit_len_kernel, dim3(n), dim3(64), 0, (hipStream_t)stream, a);
    PG_DONE();
}

int wx_cache_compact(const wx_cache* c, int32_t* d_n_live, void* stream) {
    PG_CHECK(c);
    OnDevice on(c->device);
    PageArgs a = page_args(c, nullptr, 0, nullptr);
    a.out = d_n_live;
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(cache_compact_plan_kernel, dim3(1), dim3(PG_NT), 0, st, a);
    const int64_t cells = (int64_t)c->max_seqs * c->max_pages;
    hipLaunchKernelGGL(cache_compact_move_kernel, dim3(c->n_pages < 512 ? c->n_pages : 512, c->n_layer, 2), dim3(256), 0, st, a);
    hipLaunchKernelGGL(cache_compact_table_kernel, dim3((unsigned)(cells / 256 + 1 < 2048 ? cells / 256 + 1 : 2048)), dim3(256), 0, st, a);
    PG_DONE();
}

}  // extern "C"
