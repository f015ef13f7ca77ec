// tree.hip — attention of drafted tokens over a paged cache, and greedy verification of the draft (include/whisper_amd.h,
// wx_tree_attention, wx_tree_verify).
//
//   o_i = sum_j p_ij v_j,   p_i = softmax_j(scale q_i . k_j),   j over the committed tokens, node i and its ancestors
//   pick_i = arg max_x logit_i[x],   log p(pick_i) = -log sum_x exp(logit_i[x] - max)
#include "common.h"

namespace wx {

constexpr int TR_NODES = 64;              // nodes a sequence: one bit each of a mask
constexpr float TR_LOG2E = 1.4426950408889634f;

// What an entry of the call is: 0 = its rows are 0 (padding), 1 = attend, 2 = refused (NaN).  Every thread of the workgroup; the same
// answer in every workgroup and in the append launch (cache_append_kernel).
__device__ __forceinline__ int tree_entry(const wx_cache& c, const wx_tree_attn& a, int i, int* len, int* count) {
    const int s = a.d_seqs[i];
    *len = 0;
    *count = a.d_counts ? min(max(a.d_counts[i], 0), a.n_nodes) : a.n_nodes;
    if (s == -1) return 0;
    int bad = s < 0 || s >= c.max_seqs;
    if (!bad) {
        const int l = c.d_lens[s], held = min(c.d_held[s], c.max_pages);
        *len = l;
        bad = l < 0 || (int64_t)l + *count > (int64_t)held * c.page_size;
        if (!bad) {
            const int32_t* row = c.d_table + (int64_t)s * c.max_pages;
            const int first_own = a.d_kn ? l / c.page_size : 0x7fffffff;
            for (int p = threadIdx.x; p * c.page_size < l + *count; p += blockDim.x) {
                const int page = row[p];
                if ((unsigned)page >= (unsigned)c.n_pages || (p >= first_own && c.d_refs[page] != 1)) bad = 1;
            }
        }
        if (a.d_kn) for (int j = threadIdx.x; j < i; j += blockDim.x) bad |= a.d_seqs[j] == s;
    }
    return __syncthreads_or(bad) ? 2 : 1;
}

// bit j of the result, on lane i of a wave: node j is node i or one of its ancestors.  *bad: node i hangs on a parent out of range.
// Doubling: after k steps a lane knows 2^k ancestors and jumps that far.
__device__ __forceinline__ uint64_t tree_mask(const int32_t* parents, int lane, int n_nodes, bool* bad) {
    int up = lane - 1;
    if (lane < n_nodes && parents) up = parents[lane];
    bool wrong = up < -1 || up >= lane;
    if (wrong) up = -1;
    uint64_t m = 1ull << lane;
#pragma unroll
    for (int k = 0; k < 6; ++k) {
        const int at = up < 0 ? lane : up;
        const uint32_t lo = __shfl((uint32_t)m, at), hi = __shfl((uint32_t)(m >> 32), at);
        const int next = __shfl(up, at);
        const bool w = __shfl((int)wrong, at);
        if (up >= 0) { m |= (uint64_t)hi << 32 | lo; up = next; wrong |= w; }
    }
    *bad = wrong;
    return m;
}

template <typename T> __device__ __forceinline__ void load_f32(const T* p, float* out);      // 16 bytes
template <> __device__ __forceinline__ void load_f32<float>(const float* p, float* out) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = v[j];
}
template <> __device__ __forceinline__ void load_f32<bf16>(const bf16* p, float* out) {
    const bf16x8 v = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = (float)v[j];
}

// One workgroup a (node, query head, sequence): every thread takes every 256th token with a running maximum, sum and output of its own.
template <typename T, int D>
__global__ __launch_bounds__(256) void tree_attention_kernel(wx_cache c, wx_tree_attn a) {
    constexpr int E = 16 / sizeof(T);
    __shared__ float sq[D], red[256], so[4][D];
    __shared__ uint64_t s_mask;
    __shared__ int s_bad;
    const int node = blockIdx.x, h = blockIdx.y, i = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
    int len, count;
    int what = tree_entry(c, a, i, &len, &count);
    if (tid < 64) {
        bool bad;
        const uint64_t m = tree_mask(a.d_parents ? a.d_parents + (int64_t)i * a.n_nodes : nullptr, lane, a.n_nodes, &bad);
        if (tid == node) { s_mask = m; s_bad = bad; }
    }
    T* out = reinterpret_cast<T*>(a.d_out) + i * a.o_seq + node * a.o_node + h * a.o_head;
    __syncthreads();
    if (node >= count && what == 1) what = 0;
    if (what == 1 && s_bad) what = 2;
    if (what != 1) {
        for (int x = tid; x < D; x += 256) out[x] = (T)(what == 2 ? __builtin_nanf("") : 0.f);
        return;
    }
    const T* q = reinterpret_cast<const T*>(a.d_q) + i * a.q_seq + node * a.q_node + h * a.q_head;
    for (int x = tid; x < D; x += 256) sq[x] = (float)q[x] * a.scale;
    __syncthreads();
    const uint64_t mask = s_mask;
    const int kh = h / (a.n_head / c.n_kv_head), PS = c.page_size;
    const int32_t* row = c.d_table + (int64_t)a.d_seqs[i] * c.max_pages;
    const int64_t page_e = (int64_t)c.n_kv_head * PS * D, layer_e = (int64_t)a.layer * c.n_pages * page_e;
    const T* K = reinterpret_cast<const T*>(c.d_k) + layer_e + (int64_t)kh * PS * D;
    const T* V = reinterpret_cast<const T*>(c.d_v) + layer_e + (int64_t)kh * PS * D;
    float m = -INFINITY, l = 0.f, o[D];
#pragma unroll
    for (int x = 0; x < D; ++x) o[x] = 0.f;
    for (int t = tid; t < len + count; t += 256) {
        if (t >= len && !((mask >> (t - len)) & 1)) continue;
        const int64_t off = row[t / PS] * page_e + (int64_t)(t % PS) * D;
        float s = 0.f;
#pragma unroll
        for (int x = 0; x < D; x += E) {
            float v[E];
            load_f32(K + off + x, v);
#pragma unroll
            for (int j = 0; j < E; ++j) s = fmaf(sq[x + j], v[j], s);
        }
        const float mn = fmaxf(m, s), al = m == -INFINITY ? 0.f : expf(m - mn), p = expf(s - mn);
        m = mn; l = l * al + p;
#pragma unroll
        for (int x = 0; x < D; x += E) {
            float v[E];
            load_f32(V + off + x, v);
#pragma unroll
            for (int j = 0; j < E; ++j) o[x + j] = fmaf(p, v[j], o[x + j] * al);
        }
    }
    red[tid] = m;
    __syncthreads();
    float M = -INFINITY;
    for (int t = 0; t < 256; ++t) M = fmaxf(M, red[t]);
    const float f = m == -INFINITY ? 0.f : expf(m - M);
    __syncthreads();
    red[tid] = l * f;
    __syncthreads();
    float L = 0.f;
    for (int t = 0; t < 256; ++t) L += red[t];
    for (int x = 0; x < D; ++x) {
        float v = o[x] * f;
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off);
        if (lane == 0) so[tid >> 6][x] = v;
    }
    __syncthreads();
    for (int x = tid; x < D; x += 256) out[x] = (T)((so[0][x] + so[1][x] + so[2][x] + so[3][x]) / L);
}

// ---- verification ---------------------------------------------------------------------------------------------------------------------
struct Best { float m, s; int i; };       // largest logit, sum of exp(logit - m), its lowest id
__device__ __forceinline__ void best_add(Best& b, float v, int i) {
    if (!(v > -INFINITY)) return;                                     // masked, or NaN
    if (v > b.m) { b.s = b.s * __expf(b.m - v) + 1.f; b.m = v; b.i = i; }
    else if (v == b.m) { b.s += 1.f; b.i = min(b.i, i); }             // also where both are +infinity
    else b.s += __expf(v - b.m);
}
__device__ __forceinline__ Best best_merge(Best a, Best b) {
    if (a.m == b.m) return Best{a.m, a.s + b.s, min(a.i, b.i)};
    if (b.m > a.m) { const Best t = a; a = b; b = t; }
    a.s += b.s * __expf(b.m - a.m);                                   // b.m may be -infinity: + 0
    return a;
}
constexpr int VF_NT = 256;

// one workgroup a (part of the vocabulary, node, sequence): one pass over the logits
template <typename T>
__global__ __launch_bounds__(VF_NT) void tree_verify_scan_kernel(wx_tree_check a, int parts) {
    __shared__ Best sh[VF_NT / 64];
    const int part = blockIdx.x, node = blockIdx.y, i = blockIdx.z, tid = threadIdx.x;
    const int count = a.d_counts ? a.d_counts[i] : a.n_nodes;
    if (node >= count) return;
    const int per = (a.n_vocab + parts - 1) / parts, lo = part * per, hi = min(a.n_vocab, lo + per);
    const T* row = reinterpret_cast<const T*>(a.d_logits) + i * a.l_seq + node * a.l_node;
    Best b{-INFINITY, 0.f, 0x7fffffff};
    for (int x = lo + tid; x < hi; x += VF_NT) {
        if (a.d_suppress && a.d_suppress[x]) continue;
        best_add(b, (float)row[x], x);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        Best o;
        o.m = __shfl_xor(b.m, off); o.s = __shfl_xor(b.s, off); o.i = __shfl_xor(b.i, off);
        b = best_merge(b, o);
    }
    if ((tid & 63) == 0) sh[tid >> 6] = b;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < VF_NT / 64; ++w) b = best_merge(b, sh[w]);
        float* rec = reinterpret_cast<float*>(a.d_work) + (((int64_t)i * a.n_nodes + node) * parts + part) * 4;
        rec[0] = b.m; rec[1] = b.s; reinterpret_cast<int*>(rec)[2] = b.i;
    }
}

// one wave a sequence: lane j merges node j's parts, then the wave walks down the tree
__global__ __launch_bounds__(64) void tree_verify_walk_kernel(wx_tree_check a, int parts) {
    const int i = blockIdx.x, j = threadIdx.x;
    const int count = a.d_counts ? min(max(a.d_counts[i], 0), a.n_nodes) : a.n_nodes;
    int pick = -1, token = -1, up = -1;
    float lp = 0.f;
    if (j < count) {
        Best b{-INFINITY, 0.f, 0x7fffffff};
        const float* rec = reinterpret_cast<const float*>(a.d_work) + ((int64_t)i * a.n_nodes + j) * parts * 4;
        for (int p = 0; p < parts; ++p) b = best_merge(b, Best{rec[4 * p], rec[4 * p + 1], reinterpret_cast<const int*>(rec)[4 * p + 2]});
        pick = b.m > -INFINITY ? b.i : -1;
        lp = b.m > -INFINITY ? -logf(b.s) : -INFINITY;
        token = a.d_tokens[(int64_t)i * a.n_nodes + j];
        up = a.d_parents ? a.d_parents[(int64_t)i * a.n_nodes + j] : j - 1;
    }
    const int64_t at = (int64_t)i * a.n_nodes + j;
    int cur = 0, n = 0, mine = -1, next = -1;
    while (n < count) {                                              // every turn moves to a later node
        if (j == n) mine = cur;
        ++n;
        next = __shfl(pick, cur);
        const uint64_t fit = __ballot(j < count && j > cur && up == cur && token == next && next >= 0);
        if (!fit) break;
        cur = __ffsll((unsigned long long)fit) - 1;
    }
    if (j < a.n_nodes) { a.d_pick[at] = pick; a.d_logprob[at] = lp; a.d_path[at] = mine; }
    if (j == 0) { a.d_n_accept[i] = n; a.d_next[i] = next; }
}

// enough workgroups to fill the chip where rows are few, and at least 2048 ids each
static int verify_parts(const wx_tree_check& a) {
    const int64_t rows = (int64_t)a.n * a.n_nodes;
    int64_t p = rows > 0 ? 1024 / rows : 1;
    if (p > a.n_vocab / 2048) p = a.n_vocab / 2048;
    return p < 1 ? 1 : (int)p;
}
static const char* verify_fault(const wx_tree_check* a) {
    if (!a) return "null argument";
    if (a->n < 0 || a->n > 65535) return "n must be 0 .. 65535";
    if (a->n_nodes < 1 || a->n_nodes > TR_NODES) return "n_nodes must be 1 .. 64";
    if (a->n_vocab < 1) return "n_vocab must be >= 1";
    if (a->precision != WX_PREC_F32 && a->precision != WX_PREC_BF16) return "bad precision";
    return nullptr;
}
static const char* tree_fault(const wx_cache* c, const wx_tree_attn* a) {
    if (const char* m = cache_fault(c)) return m;
    if (!a) return "null argument";
    if (a->n < 0 || a->n > 8192) return "n must be 0 .. 8192";
    if (a->n_nodes < 1 || a->n_nodes > TR_NODES) return "n_nodes must be 1 .. 64";
    if (a->layer < 0 || a->layer >= c->n_layer) return "no such layer";
    if (a->n_head < c->n_kv_head || a->n_head % c->n_kv_head || a->n_head / c->n_kv_head > 16) return "n_head must be 1 .. 16 times n_kv_head";
    if (a->split_tokens < 0) return "split_tokens must be >= 0";
    return nullptr;
}

}  // namespace wx

using namespace wx;

extern "C" {

int64_t wx_tree_attention_work_bytes(const wx_cache* c, const wx_tree_attn* a) {
    if (const char* m = tree_fault(c, a)) return set_error(WX_ERR_INVALID, m);
    return 0;
}

int wx_tree_attention(const wx_cache* c, const wx_tree_attn* a, void* stream) {
    if (const char* m = tree_fault(c, a)) return set_error(WX_ERR_INVALID, m);
    if (a->n == 0) return WX_OK;
    if (!a->d_seqs || !a->d_q || !a->d_out) return set_error(WX_ERR_INVALID, "null buffer");
    if (!a->d_kn != !a->d_vn) return set_error(WX_ERR_INVALID, "new keys and new values come together");
    const int unit = c->precision == WX_PREC_F32 ? 4 : 8;
    const int64_t strides[] = {a->q_seq, a->q_node, a->q_head, a->o_seq, a->o_node, a->o_head, a->d_kn ? a->kn_seq : 0, a->d_kn ? a->kn_node : 0,
                               a->d_kn ? a->kn_head : 0, a->d_kn ? a->vn_seq : 0, a->d_kn ? a->vn_node : 0, a->d_kn ? a->vn_head : 0};
    for (int64_t s : strides) if (s < 0 || s % unit) return set_error(WX_ERR_INVALID, "strides must be >= 0 and multiples of 16 bytes");
    if (((uintptr_t)a->d_q | (uintptr_t)a->d_out | (uintptr_t)a->d_kn | (uintptr_t)a->d_vn) & 15) return set_error(WX_ERR_INVALID, "rows must be 16-byte aligned");
    OnDevice on(c->device);
    hipStream_t st = (hipStream_t)stream;
    if (a->d_kn) {
        const int64_t ks[4] = {0, a->kn_seq, a->kn_node, a->kn_head}, vs[4] = {0, a->vn_seq, a->vn_node, a->vn_head};
        const int r = wx_cache_append(c, a->d_seqs, a->d_counts, a->n, a->n_nodes, a->layer, 1, a->d_kn, ks, a->d_vn, vs, stream);
        if (r) return r;
    }
    const dim3 grid(a->n_nodes, a->n_head, a->n), block(256);
    if (c->precision == WX_PREC_F32) {
        if (c->head_dim == 64) hipLaunchKernelGGL((tree_attention_kernel<float, 64>), grid, block, 0, st, *c, *a);
        else hipLaunchKernelGGL((tree_attention_kernel<float, 128>), grid, block, 0, st, *c, *a);
    } else {
        if (c->head_dim == 64) hipLaunchKernelGGL((tree_attention_kernel<bf16, 64>), grid, block, 0, st, *c, *a);
        else hipLaunchKernelGGL((tree_attention_kernel<bf16, 128>), grid, block, 0, st, *c, *a);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? WX_OK : set_error(WX_ERR_HIP, hipGetErrorString(e));
}

int64_t wx_tree_verify_work_bytes(const wx_tree_check* a) {
    if (const char* m = verify_fault(a)) return set_error(WX_ERR_INVALID, m);
    return (int64_t)a->n * a->n_nodes * verify_parts(*a) * 16;
}

int wx_tree_verify(const wx_tree_check* a, void* stream) {
    if (const char* m = verify_fault(a)) return set_error(WX_ERR_INVALID, m);
    if (a->n == 0) return WX_OK;
    if (!a->d_logits || !a->d_tokens || !a->d_pick || !a->d_logprob || !a->d_path || !a->d_n_accept || !a->d_next || !a->d_work)
        return set_error(WX_ERR_INVALID, "null buffer");
    if (a->l_seq < 0 || a->l_node < 0) return set_error(WX_ERR_INVALID, "strides must be >= 0");
    if (a->work_bytes < wx_tree_verify_work_bytes(a) || ((uintptr_t)a->d_work & 15)) return set_error(WX_ERR_INVALID, "work buffer too small or not 16-byte aligned");
    OnDevice on(a->device);
    hipStream_t st = (hipStream_t)stream;
    const int parts = verify_parts(*a);
    const dim3 grid(parts, a->n_nodes, a->n);
    if (a->precision == WX_PREC_F32) hipLaunchKernelGGL(tree_verify_scan_kernel<float>, grid, dim3(VF_NT), 0, st, *a, parts);
    else hipLaunchKernelGGL(tree_verify_scan_kernel<bf16>, grid, dim3(VF_NT), 0, st, *a, parts);
    hipLaunchKernelGGL(tree_verify_walk_kernel, dim3(a->n), dim3(64), 0, st, *a, parts);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? WX_OK : set_error(WX_ERR_HIP, hipGetErrorString(e));
}

}  // extern "C"
