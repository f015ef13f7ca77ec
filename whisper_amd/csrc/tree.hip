// tree.hip — attention of drafted tokens over a paged cache, and greedy verification of the draft (include/whisper_amd.h,
// wx_tree_attention, wx_tree_verify).
//
//   o_i = sum_j p_ij v_j,   p_i = softmax_j(scale q_i . k_j),   j over the committed tokens, node i and its ancestors
//   pick_i = arg max_x logit_i[x],   log p(pick_i) = -log sum_x exp(logit_i[x] - max)
#include "common.h"

#include <atomic>

namespace wx {

constexpr int TR_NODES = 64;              // nodes a sequence: one bit each of a mask
constexpr float TR_LOG2E = 1.4426950408889634f;

// How the work on a batch is cut.  A sequence has ceil(len / KT) tiles of committed tokens and `tree_tiles` behind them.  For every
// key / value head and block of rows, `takers` workgroups take equal shares of all sequences' tiles in a row (fewer takers where a
// share would fall below `least` tiles, or `least_few` with up to `few` takers), so that ragged lengths leave no workgroup behind: one may
// end a sequence, do some whole ones and begin another.  The part of a sequence that taker w does is piece w + i of the part buffer (w or i
// grows by one from piece to piece, so the numbers are distinct).  With `per` > 0 a sequence is cut into pieces of at most `per` tiles
// instead, one for each workgroup; with `single`, where no sequence can be longer than 512 tokens, a workgroup does one whole sequence.
// Equal shares against one sequence a workgroup, cut at equal lengths (8 sequences of 40000-131072 tokens): 967 us against 1272.
struct TreePlan {
    int row_blocks;          // workgroups over the rows (nodes x query heads of a key / value head)
    int tree_tiles, per, least, takers, least_few, few;
    int single;              // (the kernels' ONE)
    int shift;               // log2 of the page size
    int slots;               // workgroups for each key / value head and block of rows
    int pieces;              // ... and places for their parts
    int rows;                // rows a workgroup
    int merge_rows;          // rows a workgroup of the merge (a power of two); the rest of its threads share their pieces
    float* part;             // [pieces][n_kv_head][row_blocks][rows][D + 2]: output, maximum (NaN: refused) and sum (sequences in more than one piece)
};

__device__ __forceinline__ int tree_tiles_of(const wx_cache& c, const wx_tree_attn& a, const TreePlan& p, int i, int kt) {
    const int s = a.d_seqs[i];
    const int len = s >= 0 && s < c.max_seqs ? min(max(c.d_lens[s], 0), c.max_pages << p.shift) : 0;
    return (len + kt - 1) / kt + p.tree_tiles;
}
// the share that tile x of `all` falls to (share w: tiles w * all / takers and up)
__device__ __forceinline__ int tree_taker(int64_t x, int64_t all, int takers) { return (int)(((x + 1) * takers - 1) / all); }

// One wave, all lanes alike: tiles of the whole batch, and how many takers they are for.
__device__ __forceinline__ int64_t tree_all(const wx_cache& c, const wx_tree_attn& a, const TreePlan& p, int kt, int lane, int* takers) {
    int64_t all = 0;
    for (int i = lane; i < a.n; i += 64) all += tree_tiles_of(c, a, p, i, kt);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) all += __shfl_xor(all, off);
    *takers = (int)max((int64_t)1, min((int64_t)p.takers, max(all / p.least, min((int64_t)p.few, all / p.least_few))));
    return all;
}

struct TreeArgs { wx_cache c; wx_tree_attn a; TreePlan p; };
// The arguments anew for every job: kept over the loop of jobs, they take the scalar registers and spill into vector registers.
#define TREE_ARGS(ka) \
    const __attribute__((address_space(4))) TreeArgs* ka##_p = (const __attribute__((address_space(4))) TreeArgs*)__builtin_amdgcn_kernarg_segment_ptr(); \
    asm volatile("" : "+s"(ka##_p)); \
    const wx_cache& c = ((const TreeArgs*)ka##_p)->c; \
    const wx_tree_attn& a = ((const TreeArgs*)ka##_p)->a; \
    const TreePlan& p = ((const TreeArgs*)ka##_p)->p

// So is the thread's number: addresses that follow from it would be kept over the loop of jobs as well, 20 to 30 vector registers of them, and
// push some to scratch memory.
#define TREE_THREAD(tid) \
    int tid = threadIdx.x; \
    asm volatile("" : "+v"(tid))

// What a workgroup has to do now: sequence entry i, key / value head, block of rows, tiles [t0, t1) of the sequence's n_pre + tree_tiles.
struct TreeJob {
    int ok;                  // 0: the rows are 0 (padding, no nodes), 1: attend, 2: refused (NaN), -1: nothing (any more)
    int i, kh, rb, piece, whole, seq, len, count, n_pre, t0, t1, last;
    int w, takers;           // shares
    int64_t all, start, x0, x1;   // tiles of the batch; first tile of sequence i among them; the share
};

__device__ __forceinline__ void tree_fill(const wx_cache& c, const wx_tree_attn& a, const TreePlan& p, int kt, TreeJob& t) {
    t.ok = 1;
    t.seq = a.d_seqs[t.i];
    t.count = a.d_counts ? min(max(a.d_counts[t.i], 0), a.n_nodes) : a.n_nodes;
    t.len = 0; t.n_pre = 0;
    if (t.seq == -1) t.ok = 0;
    else if (t.seq < 0 || t.seq >= c.max_seqs) t.ok = 2;
    else {
        t.len = c.d_lens[t.seq];
        if (t.len < 0 || (int64_t)t.len + t.count > (int64_t)min(c.d_held[t.seq], c.max_pages) << p.shift) t.ok = 2;
        else if (t.count == 0) t.ok = 0;
        t.n_pre = (min(max(t.len, 0), c.max_pages << p.shift) + kt - 1) / kt;
    }
}

// The first job of a workgroup (first = true) or the next of its share; *sh is the same on every thread afterwards.
template <int KT>
__device__ __forceinline__ bool tree_next(const wx_cache& c, const wx_tree_attn& a, const TreePlan& p, TreeJob* sh, TreeJob& j, bool first) {
    const int tid = threadIdx.x, lane = tid & 63;
    if (!first && p.per) return false;
    __syncthreads();                                               // the job before is done with *sh and the other shared arrays
    if (tid < 64) {
        TreeJob t;
        if (first) {
            // XCD-aware: consecutive workgroups go to different XCDs, so the row blocks that read the same keys are 8 apart, on one L2
            const int lin = blockIdx.x, y = lin / 8, w = (y / p.row_blocks) * 8 + lin % 8;
            t.kh = w % c.n_kv_head; t.rb = y % p.row_blocks; t.w = w / c.n_kv_head; t.whole = 1; t.piece = 0; t.i = t.w; t.takers = 0;
            t.all = t.start = t.x0 = t.x1 = 0;
            t.ok = t.w < p.slots ? 1 : -1;
            if (t.ok == 1) {
                if (p.per) {                                       // piece number t.w, counted through the sequences
                    int before = 0;
                    t.ok = -1;
                    for (int i0 = 0; i0 < a.n && t.ok < 0; i0 += 64) {
                        const int i = i0 + lane, mine = i < a.n ? (tree_tiles_of(c, a, p, i, KT) + p.per - 1) / p.per : 0;
                        int upto = mine;
#pragma unroll
                        for (int off = 1; off < 64; off <<= 1) { const int u = __shfl_up(upto, off); if (lane >= off) upto += u; }
                        const uint64_t past = __ballot(before + upto > t.w);
                        if (past) {
                            const int at = __ffsll((unsigned long long)past) - 1, pieces = __shfl(mine, at);
                            t.ok = 1; t.i = i0 + at; t.whole = pieces == 1; t.piece = t.w;
                            const int q = t.w - (before + __shfl(upto, at) - pieces);
                            t.x0 = (int64_t)q * p.per; t.x1 = t.x0 + p.per;
                        }
                        before += __shfl(upto, 63);
                    }
                } else {                                           // share number t.w: the sequence of its first tile
                    t.all = tree_all(c, a, p, KT, lane, &t.takers);
                    if (t.w >= t.takers) t.ok = -1;
                    t.x0 = t.w * t.all / t.takers; t.x1 = (t.w + (int64_t)1) * t.all / t.takers;
                    for (int i0 = 0; i0 < a.n && t.ok == 1; i0 += 64) {
                        const int i = i0 + lane;
                        int64_t upto = i < a.n ? tree_tiles_of(c, a, p, i, KT) : 0;
                        const int64_t mine = upto;
#pragma unroll
                        for (int off = 1; off < 64; off <<= 1) { const int64_t u = __shfl_up(upto, off); if (lane >= off) upto += u; }
                        const uint64_t past = __ballot(t.start + upto > t.x0);
                        if (past) {
                            const int at = __ffsll((unsigned long long)past) - 1;
                            t.i = i0 + at;
                            t.start += __shfl(upto - mine, at);
                            break;
                        }
                        t.start += __shfl(upto, 63);
                    }
                }
            }
        } else {
            t = *sh;
            t.start += t.n_pre + p.tree_tiles;
            t.i += 1;
            t.ok = t.i < a.n && t.start < t.x1 ? 1 : -1;
        }
        if (t.ok == 1) {
            tree_fill(c, a, p, KT, t);
            const int tiles = t.n_pre + p.tree_tiles;
            if (p.per) { t.t0 = (int)t.x0; t.t1 = (int)min(t.x1, (int64_t)tiles); }
            else {
                t.t0 = (int)max((int64_t)0, t.x0 - t.start); t.t1 = (int)min((int64_t)tiles, t.x1 - t.start);
                t.whole = tree_taker(t.start, t.all, t.takers) == tree_taker(t.start + tiles - 1, t.all, t.takers);
                t.piece = t.w + t.i;
            }
            t.last = t.t1 == tiles;
        }
        if (tid == 0) *sh = t;
    }
    __syncthreads();
    j = *sh;
    if (j.ok < 0) return false;
    return true;
}
// A job's numbers are alike on every lane: in scalar registers (read back from LDS they would take a vector register each, and every loop
// over them a mask).
__device__ __forceinline__ void tree_uniform(TreeJob& t) {
#define UNI(x) t.x = __builtin_amdgcn_readfirstlane(t.x)
    UNI(ok); UNI(i); UNI(kh); UNI(rb); UNI(piece); UNI(whole); UNI(seq); UNI(len); UNI(count); UNI(n_pre); UNI(t0); UNI(t1); UNI(last);
#undef UNI
}
// The one job of a workgroup that does one whole sequence, or (solo >= 0) of its wave `solo`: no search, and nothing waits for another wave.
template <int KT>
__device__ __forceinline__ bool tree_whole(const wx_cache& c, const wx_tree_attn& a, const TreePlan& p, TreeJob& t, int solo) {
    const int lin = blockIdx.x, y = lin / 8, w = solo < 0 ? (y / p.row_blocks) * 8 + lin % 8 : (4 * lin + solo) / p.row_blocks;     // (as tree_next)
    t.kh = w % c.n_kv_head; t.rb = (solo < 0 ? y : 4 * lin + solo) % p.row_blocks; t.i = t.w = w / c.n_kv_head; t.whole = 1; t.piece = 0; t.takers = 0; t.last = 1;
    t.all = t.start = t.x0 = t.x1 = 0;
    if (t.w >= p.slots) return false;
    tree_fill(c, a, p, KT, t);
    t.t0 = 0; t.t1 = t.n_pre + p.tree_tiles;
    return true;
}
// A job's second look, by all threads that work on it, each with its share of it: whether a page of the piece's tiles is none of the
// pool's, a page of the draft's rows is not this slot's alone although they are to be written, or an appending call names the slot
// before.  What comes of it is needed at the end only (nothing is written before, and page_ok() keeps the reads inside the pool), so that
// its loads overlap the work.
__device__ __forceinline__ int tree_bad(const wx_cache& c, const wx_tree_attn& a, const TreePlan& p, const TreeJob& j, int kt, int me, int threads) {
    int bad = 0;
    const int32_t* row = c.d_table + (int64_t)j.seq * c.max_pages;
    const int upto = j.t1 > j.n_pre ? j.len + j.count : min(j.len, j.t1 * kt);
    const int own = a.d_kn && j.last ? j.len >> p.shift : 0x7fffffff;
    for (int q = (min(j.t0 * kt, j.len) >> p.shift) + me; q << p.shift < upto; q += threads) {
        const int page = row[q];
        if ((unsigned)page >= (unsigned)c.n_pages || (q >= own && c.d_refs[page] != 1)) bad = 1;
    }
    if (a.d_kn) for (int k = me; k < j.i; k += threads) bad |= a.d_seqs[k] == j.seq;
    return bad;
}
__device__ __forceinline__ int page_ok(const wx_cache& c, int page) { return (unsigned)page < (unsigned)c.n_pages ? page : 0; }

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


typedef __attribute__((ext_vector_type(4))) short i16x4;
typedef __attribute__((ext_vector_type(8))) short i16x8;

// ---- what differs between the element types -----------------------------------------------------------------------------------
// Both keep the QUERY ROW on the matrix instruction's column (lane & 15 = r, lane >> 4 = g):
//   S^T[key][row] = K Q^T    A = 16 keys x 64 bytes of a row (lane (g, r): bytes 16 g of key r), B = the query rows the same way
//   O^T[d][row] += V^T P^T   B = the S^T accumulator in place (lane (g, r) holds keys 4 g + 0..3 of row r), A = V^T out of LDS
// so the running maximum, sum and rescale factor of a row sit on the lanes that hold its scores and outputs, and P never moves.
template <typename T> struct Elem;
template <> struct Elem<bf16> {
    typedef bf16x8 Frag;
    static __device__ __forceinline__ f32x4 qk(Frag k, Frag q, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q, c, 0, 0, 0); }
    static __device__ __forceinline__ bool odd(Frag v) {                        // holds an infinity or a NaN
        const i32x4 b = __builtin_bit_cast(i32x4, v);
        bool o = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) o |= (b[j] & 0x7f800000) == 0x7f800000 || (b[j] & 0x7f80) == 0x7f80;
        return o;
    }
    static constexpr int PAD = 32;                                            // bytes behind a V row in LDS: the transposing reads hit every bank once
};
template <> struct Elem<float> {
    typedef f32x4 Frag;
    static __device__ __forceinline__ f32x4 qk(Frag k, Frag q, f32x4 c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(k[j], q[j], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ bool odd(Frag v) {
        const i32x4 b = __builtin_bit_cast(i32x4, v);
        bool o = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) o |= (b[j] & 0x7f800000) == 0x7f800000;
        return o;
    }
    static constexpr int PAD = 16;
};
template <typename F> __device__ __forceinline__ F finite_only(F v) {
#pragma unroll
    for (int j = 0; j < (int)(16 / sizeof(v[0])); ++j) { const float x = (float)v[j]; if (!(fabsf(x) < INFINITY)) v[j] = 0; }
    return v;
}

// The state of RT x 16 rows on a wave: maximum and (this lane's share of the) sum of every row, output.
template <int D, int RT> struct RowState {
    float m[RT], l[RT];
    f32x4 o[D / 16][RT];
    __device__ __forceinline__ void init() {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            m[t] = -INFINITY; l[t] = 0.f;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) o[d][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    // scores -> probabilities (in place); c = |scale| log2 e.  A tile that is masked altogether leaves the state alone.
    template <int NS> __device__ __forceinline__ void softmax(f32x4 (&s)[NS][RT], float c) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            float mt = s[0][t][0];
#pragma unroll
            for (int k = 0; k < NS; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) mt = fmaxf(mt, s[k][t][j]);
            mt = fmaxf(mt, __shfl_xor(mt, 16));
            mt = fmaxf(mt, __shfl_xor(mt, 32));
            const float mn = fmaxf(m[t], mt), base = mn == -INFINITY ? 0.f : mn * c;
            // 1 while the maximum stands: m c - base is the rounding of base, and its power, tile after tile, would weigh early keys by another
            // factor than late ones (16384 tokens in one piece, f32: 1.1e-5 off, 1.2e-6 without)
            const float alpha = mn == m[t] ? 1.f : __builtin_amdgcn_exp2f((m[t] - mn) * c);       // m = -infinity: 0
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < NS; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) { s[k][t][j] = __builtin_amdgcn_exp2f(fmaf(s[k][t][j], c, -base)); sum += s[k][t][j]; }
            l[t] = fmaf(l[t], alpha, sum);
            m[t] = mn;
            if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {                      // rare after the first tiles
#pragma unroll
                for (int d = 0; d < D / 16; ++d) o[d][t] *= alpha;
            }
        }
    }
    // o += V^T P^T for NS x 16 keys; vb: their rows in LDS, VROW bytes each
    template <int NS, int VROW> __device__ __forceinline__ void add(const f32x4 (&p)[NS][RT], const char* vb, int g, int r, bf16) {
#pragma unroll
        for (int h = 0; h < NS / 2; ++h) {
            bf16x8 pf[RT], pl[RT];
#pragma unroll
            for (int t = 0; t < RT; ++t) split_probs(p[2 * h][t], p[2 * h + 1][t], pf[t], pl[t]);
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
                // lane (g, r) receives V[32 h + 16 u + 4 g + j][16 d + r], j = 0..3, for u = 0, 1
                const char* p0 = vb + (32 * h + 4 * g + (r >> 2)) * VROW + (16 * d + 4 * (r & 3)) * 2;
                const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(p0));
                const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(p0 + 16 * VROW));
                const bf16x8 vf = __builtin_bit_cast(bf16x8, (i16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    o[d][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[t], o[d][t], 0, 0, 0);
                    o[d][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pl[t], o[d][t], 0, 0, 0);
                }
            }
            if (RT > 1) __builtin_amdgcn_sched_barrier(0);                         // the other half is split when this one is done with: registers
        }
    }
    template <int NS, int VROW> __device__ __forceinline__ void add(const f32x4 (&p)[NS][RT], const char* vb, int g, int r, float) {
#pragma unroll
        for (int k = 0; k < NS; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float* row = reinterpret_cast<const float*>(vb + (16 * k + 4 * g + j) * VROW) + r;
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                    const float v = row[16 * d];
#pragma unroll
                    for (int t = 0; t < RT; ++t) o[d][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, p[k][t][j], o[d][t], 0, 0, 0);
                }
            }
    }
};

// Rows of a sequence's drafted nodes: given with the call, or in the cache behind the committed tokens.
template <typename T, int D>
__device__ __forceinline__ const T* node_row(const wx_cache& c, const wx_tree_attn& a, const TreePlan& p, const TreeJob& j, const int32_t* table, int64_t head_off,
                                             int64_t page_e, bool keys, int node) {
    if (a.d_kn)
        return keys ? reinterpret_cast<const T*>(a.d_kn) + j.i * a.kn_seq + node * a.kn_node + j.kh * a.kn_head
                    : reinterpret_cast<const T*>(a.d_vn) + j.i * a.vn_seq + node * a.vn_node + j.kh * a.vn_head;
    const int t = j.len + node;
    return reinterpret_cast<const T*>(keys ? c.d_k : c.d_v) + head_off + page_ok(c, table[t >> p.shift]) * page_e + (int64_t)(t & (c.page_size - 1)) * D;
}

// The rare end of a tile of drafted rows whose values hold infinities or NaN: the matrix product ran on 0 in their place (0 x NaN would
// reach the rows that do not attend them); what they give to the rows that do is added here.
template <typename T, int D, int RT, int NS>
__device__ __forceinline__ void add_odd_values(const wx_cache& c, const wx_tree_attn& a, const TreePlan& p, const TreeJob& j, const int32_t* table, int64_t head_off,
                                            int64_t page_e, int node0, const f32x4 (&pr)[NS][RT], const uint64_t (&mask)[RT], RowState<D, RT>& st, int g, int r) {
    for (int k = 0; k < NS * 16 && node0 + k < j.count; ++k) {
        const T* row = node_row<T, D>(c, a, p, j, table, head_off, page_e, false, node0 + k);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            float x = 0.f;
#pragma unroll
            for (int kk = 0; kk < NS; ++kk)
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) if (kk == k / 16 && jj == k % 4) x = pr[kk][t][jj];
            x = __shfl(x, ((k % 16) / 4) * 16 + r);
            const bool seen = (mask[t] >> (node0 + k)) & 1;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) {
                    const float v = (float)row[16 * d + 4 * g + jj];
                    if (seen && !(fabsf(v) < INFINITY)) st.o[d][t][jj] = fmaf(x, v, st.o[d][t][jj]);
                }
                __builtin_amdgcn_sched_barrier(0);                                 // rare: no registers for its sake
            }
        }
    }
}

// drafted rows -> the cache (one workgroup a sequence and head does it): 16 bytes a thread, the first of them loaded ahead
template <typename T, int D>
__device__ __forceinline__ i32x4 append_load(const wx_cache& c, const wx_tree_attn& a, const TreeJob& j, int u) {
    constexpr int E = 16 / sizeof(T), PER = D / E;
    const int x = u % PER, node = (u / PER) % j.count;
    const T* row = u < j.count * PER ? reinterpret_cast<const T*>(a.d_kn) + j.i * a.kn_seq + node * a.kn_node + j.kh * a.kn_head
                                     : reinterpret_cast<const T*>(a.d_vn) + j.i * a.vn_seq + node * a.vn_node + j.kh * a.vn_head;
    return *reinterpret_cast<const i32x4*>(row + x * E);
}
template <typename T, int D>
__device__ __forceinline__ T* append_place(const wx_cache& c, const TreePlan& p, const TreeJob& j, const int32_t* table, int64_t head_off, int64_t page_e, int u) {
    constexpr int E = 16 / sizeof(T), PER = D / E;
    const int x = u % PER, node = (u / PER) % j.count, t = j.len + node;
    return reinterpret_cast<T*>(u < j.count * PER ? c.d_k : c.d_v) + head_off + page_ok(c, table[t >> p.shift]) * page_e + (int64_t)(t & (c.page_size - 1)) * D + x * E;
}
template <typename T, int D>
__device__ __forceinline__ void append_nodes(const wx_cache& c, const wx_tree_attn& a, const TreePlan& p, const TreeJob& j, const int32_t* table, int64_t head_off, int64_t page_e, int u0, int threads) {
    constexpr int PER = D * (int)sizeof(T) / 16;
    for (int u = u0; u < j.count * PER * 2; u += threads) *reinterpret_cast<i32x4*>(append_place<T, D>(c, p, j, table, head_off, page_e, u)) = append_load<T, D>(c, a, j, u);
}

template <typename T> __device__ __forceinline__ void store4(T* to, f32x4 v);
template <> __device__ __forceinline__ void store4<float>(float* to, f32x4 v) { *reinterpret_cast<f32x4*>(to) = v; }
template <> __device__ __forceinline__ void store4<bf16>(bf16* to, f32x4 v) {
    bf16x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (bf16)v[j];
    *reinterpret_cast<bf16x4*>(to) = o;
}

// ---- few rows: every wave has all rows of the workgroup and takes every fourth tile of keys -----------------------------------------
// Bound by the stream of keys and values.  A tile is 8 KiB of keys (straight into the matrix instruction's registers) and 8 KiB of
// values (through the wave's own LDS, for the transposing read); the next tile's 16 loads a lane are issued as soon as the scores of
// this one are taken, and no wave waits for another before the end, where the four states are merged through LDS.
// Kernel times on bf16, against one thread a key and head without matrix instructions: 16 x 24 rows, 20 heads of 64, 30-420 tokens: 268 us ->
// 16.6 us (24 MB; latency: four tiles a wave at most); 64 x 1 row, 200-447 tokens: 85 -> 30 us with SOLO (111 MB, 3.7 TB/s); 16 x 24 rows,
// 4000-16000 tokens, 20 heads of 64: 183 us (one launch and its merge).
// With three waves a SIMD instead of two the vector registers spill, 64 x 1 row take 33 us, and the cut form of that build gave wrong results (cause not
// established): no kernel here keeps vector registers in scratch memory.
// SOLO (whole sequences, jobs enough to fill the chip: tree_solo): every wave has a job of its own and takes all of its tiles, so
// that all jobs are under way at once and nothing is merged.
template <typename T, int D, int RT, bool ONE, bool SOLO = false>
__global__ __launch_bounds__(256, 2) void tree_attention_keys_kernel(TreeArgs) {
    static_assert(!SOLO || ONE, "a wave alone does one whole sequence");
    constexpr int STEP = SOLO ? 1 : 4, THREADS = SOLO ? 64 : 256;
    typedef typename Elem<T>::Frag Frag;
    constexpr int E = 16 / sizeof(T), KT = 8192 / (D * (int)sizeof(T)), NS = KT / 16, KS = D / (4 * E), CPR = D / E, NV = KT * CPR / 64;
    constexpr int VROW = D * (int)sizeof(T) + Elem<T>::PAD, VBYTES = KT * VROW, OROW = 68;
    constexpr int LDS = SOLO || 4 * VBYTES > 4 * RT * 16 * OROW * 4 ? 4 * VBYTES : 4 * RT * 16 * OROW * 4;
    __shared__ __attribute__((aligned(16))) char lds[LDS];
    __shared__ TreeJob s_job;
    __shared__ int s_wrong[64];
    __shared__ float s_m[4][RT * 16], s_l[4][RT * 16];
    TreeJob j;
    for (bool first = true;; first = false) {
    TREE_ARGS(ka);
    TREE_THREAD(tid);
    const int lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, r = lane & 15, me = SOLO ? lane : tid;
    if constexpr (ONE) { if (!first || !tree_whole<KT>(c, a, p, j, SOLO ? wid : -1)) break; }
    else if (!tree_next<KT>(c, a, p, &s_job, j, first)) break;
    tree_uniform(j);
    const int G = a.n_head / c.n_kv_head, rows = a.n_nodes * G, row0 = j.rb * RT * 16;
    int bad = 0;
    bool row_wrong[RT] = {};
    const bool writes = j.ok == 1 && a.d_kn && j.rb == 0 && j.last;
    i32x4 row0_part = {0, 0, 0, 0};
    T* place = nullptr;
    const int32_t* table = c.d_table + (int64_t)j.seq * c.max_pages;
    const int64_t page_e = (int64_t)c.n_kv_head * c.page_size * D, head_off = (int64_t)a.layer * c.n_pages * page_e + (int64_t)j.kh * c.page_size * D;
    RowState<D, RT> st;
    st.init();
    if (j.ok == 1) {
        Frag qf[RT][KS];
        const float sign = a.scale < 0.f ? -1.f : a.scale > 0.f ? 1.f : 0.f, cc = (a.scale == 0.f ? 1.f : fabsf(a.scale)) * TR_LOG2E;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int row = min(row0 + t * 16 + r, rows - 1), node = row / G;
            const T* q = reinterpret_cast<const T*>(a.d_q) + j.i * a.q_seq + node * a.q_node + (j.kh * G + row % G) * a.q_head;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                qf[t][ks] = *reinterpret_cast<const Frag*>(q + (ks * 4 + g) * E);
                if (sign != 1.f) {
#pragma unroll
                    for (int x = 0; x < E; ++x) qf[t][ks][x] = (T)((float)qf[t][ks][x] * sign);
                }
            }
        }
        const T* Kp = reinterpret_cast<const T*>(c.d_k) + head_off;
        const T* Vp = reinterpret_cast<const T*>(c.d_v) + head_off;
        char* vb = lds + wid * VBYTES;
        Frag kf[NS][KS], vr[NV];
        // a tile's pages: one for each 16 tokens, on lanes 0 .. NS-1
        auto load_ids = [&](int t) { return table[min(t * KT + 16 * min(lane, NS - 1), j.len - 1) >> p.shift]; };
        // (a scalar base for the page and a 32-bit lane offset inside it: a page of one head is at most 128 KiB)
        auto load_pre = [&](int t, int ids) {
            const int last = j.len - 1 - t * KT;                                  // >= 0
            ids = page_ok(c, ids);                                                // (here: looked at where it was loaded, it would be waited for there)
#pragma unroll
            for (int k = 0; k < NS; ++k) {
                const char* page = reinterpret_cast<const char*>(Kp + (int64_t)__builtin_amdgcn_readlane(ids, k) * page_e);
                const uint32_t off = (((t * KT + min(16 * k + r, last)) & (c.page_size - 1)) * D + g * E) * (uint32_t)sizeof(T);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) kf[k][ks] = *reinterpret_cast<const Frag*>(page + (off + ks * 64));
            }
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                constexpr int RPL = 64 / CPR;                                     // rows a load covers
                const char* page = reinterpret_cast<const char*>(Vp + (int64_t)__builtin_amdgcn_readlane(ids, v * RPL / 16) * page_e);
                const uint32_t off = (((t * KT + min(v * RPL + lane / CPR, last)) & (c.page_size - 1)) * D + (lane % CPR) * E) * (uint32_t)sizeof(T);
                vr[v] = *reinterpret_cast<const Frag*>(page + off);
            }
        };
        auto load_tree = [&](int node0) {                                         // (one address at a time in registers)
#pragma unroll
            for (int k = 0; k < NS; ++k) {
                const T* kr = node_row<T, D>(c, a, p, j, table, head_off, page_e, true, min(node0 + 16 * k + r, j.count - 1));
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) kf[k][ks] = *reinterpret_cast<const Frag*>(kr + (ks * 4 + g) * E);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                vr[v] = *reinterpret_cast<const Frag*>(node_row<T, D>(c, a, p, j, table, head_off, page_e, false, min(node0 + (v * 64 + lane) / CPR, j.count - 1)) + (lane % CPR) * E);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // rows of the tile from `live` on are no tokens: their values count as 0 (their scores are masked)
        auto stage = [&](int live) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int row = (v * 64 + lane) / CPR;
                Frag x = vr[v];
                if (row >= live) x = Frag{};
                *reinterpret_cast<Frag*>(vb + row * VROW + (lane % CPR) * 16) = x;
            }
            __builtin_amdgcn_wave_barrier();
        };
        auto scores = [&](f32x4 (&s)[NS][RT]) {
#pragma unroll
            for (int k = 0; k < NS; ++k)
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) x = Elem<T>::qk(kf[k][ks], qf[t][ks], x);
                    s[k][t] = x;
                }
        };
        // The drafted rows come first, the last wave's first tile: their places (where the call brings them) depend on no other load, so they are
        // on their way while the length and the pages are looked up.  Every lane has the mask of its node and takes those of its rows.
        bool wrong = a.d_parents && a.n_nodes == 1 && a.d_parents[j.i] != -1;
        const uint64_t own_mask = a.n_nodes == 1 ? 1 : tree_mask(a.d_parents ? a.d_parents + (int64_t)j.i * a.n_nodes : nullptr, lane, a.n_nodes, &wrong);
        if (!SOLO && wid == 0) s_wrong[lane] = wrong;
        uint64_t mask[RT];
#pragma unroll
        for (int q = 0; q < RT; ++q) {
            const int node = min(row0 + q * 16 + r, rows - 1) / G;
            mask[q] = (uint64_t)(uint32_t)__shfl((uint32_t)(own_mask >> 32), node) << 32 | (uint32_t)__shfl((uint32_t)own_mask, node);
            if constexpr (SOLO) row_wrong[q] = __shfl((int)wrong, node);
        }
        const int nt0 = ONE ? 0 : max(0, j.t0 - j.n_pre), nt1 = ONE ? p.tree_tiles : j.t1 - j.n_pre;
        for (int nt = nt0 + (SOLO ? 0 : 3 - wid); nt < nt1; nt += STEP) {
            const int node0 = nt * KT;
            if (node0 >= j.count) break;
            f32x4 s[NS][RT];
            load_tree(node0);
            bool odd = false;
#pragma unroll
            for (int v = 0; v < NV; ++v) odd |= Elem<T>::odd(vr[v]);
            const bool any_odd = __builtin_amdgcn_ballot_w64(odd) != 0;
            if (any_odd)
#pragma unroll
                for (int v = 0; v < NV; ++v) vr[v] = finite_only(vr[v]);
            stage(j.count - node0);
            scores(s);
#pragma unroll
            for (int k = 0; k < NS; ++k)
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int q = 0; q < RT; ++q) if (!((mask[q] >> (node0 + 16 * k + 4 * g + x)) & 1)) s[k][q][x] = -INFINITY;
            st.template softmax<NS>(s, cc);
            st.template add<NS, VROW>(s, vb, g, r, T());
            if (any_odd) add_odd_values<T, D, RT, NS>(c, a, p, j, table, head_off, page_e, node0, s, mask, st, g, r);
            __builtin_amdgcn_wave_barrier();
        }
        const int end = min(j.t1, j.n_pre);
        int t = j.t0 + (SOLO ? 0 : wid);
        if (writes && me < j.count * CPR * 2) { row0_part = append_load<T, D>(c, a, j, me); place = append_place<T, D>(c, p, j, table, head_off, page_e, me); }
        if (t >= end) bad = tree_bad(c, a, p, j, KT, me, THREADS);
        else {
            int ids = load_ids(t);
            load_pre(t, ids);
            ids = load_ids(min(t + STEP, j.n_pre - 1));
            bad = tree_bad(c, a, p, j, KT, me, THREADS);
            for (; t < end; t += STEP) {
                f32x4 s[NS][RT];
                const int live = j.len - t * KT;
                stage(live);
                scores(s);
                if (t + STEP < end) {
                    load_pre(t + STEP, ids);
                    ids = load_ids(min(t + 2 * STEP, j.n_pre - 1));
                }
                if (live < KT) {
                    asm volatile("");                                               // keep it a branch: as selects it costs every tile
#pragma unroll
                    for (int k = 0; k < NS; ++k)
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            if (16 * k + 4 * g + x >= live)
#pragma unroll
                                for (int q = 0; q < RT; ++q) s[k][q][x] = -INFINITY;
                }
                st.template softmax<NS>(s, cc);
                st.template add<NS, VROW>(s, vb, g, r, T());
                __builtin_amdgcn_wave_barrier();
            }
        }
    }
    if constexpr (SOLO) {
        if (__builtin_amdgcn_ballot_w64(bad != 0)) j.ok = 2;
        if (writes && j.ok == 1) {
            if (me < j.count * CPR * 2) *reinterpret_cast<i32x4*>(place) = row0_part;
            append_nodes<T, D>(c, a, p, j, table, head_off, page_e, me + THREADS, THREADS);
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            float l = st.l[t];
            l += __shfl_xor(l, 16);
            l += __shfl_xor(l, 32);
            const int at = row0 + t * 16 + r, node = at / G;
            if (at >= rows) continue;
            T* out = reinterpret_cast<T*>(a.d_out) + j.i * a.o_seq + node * a.o_node + (j.kh * G + at % G) * a.o_head + 4 * g;
            const int kind = j.ok == 1 ? node >= j.count ? 0 : row_wrong[t] ? 2 : 1 : j.ok;
            const float f = 1.f / l;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) store4<T>(out + 16 * d, kind == 1 ? st.o[d][t] * f : f32x4{1.f, 1.f, 1.f, 1.f} * (kind == 0 ? 0.f : __builtin_nanf("")));
        }
        break;
    }
    // ---- the four waves' states: factors first, then 64 columns of the outputs at a time ---------------------------------------------
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        float l = st.l[t];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (g == 0) { s_m[wid][t * 16 + r] = st.m[t]; s_l[wid][t * 16 + r] = l; }
    }
    if (__builtin_amdgcn_readfirstlane(__syncthreads_or(bad))) j.ok = 2;
    if (writes && j.ok == 1) {
        if (me < j.count * CPR * 2) *reinterpret_cast<i32x4*>(place) = row0_part;
        append_nodes<T, D>(c, a, p, j, table, head_off, page_e, me + THREADS, THREADS);
    }
    const bool whole = j.whole;
    float* part = whole ? nullptr : p.part + (((int64_t)j.piece * c.n_kv_head + j.kh) * p.row_blocks + j.rb) * (RT * 16) * (D + 2);
    const float cc = (a.scale == 0.f ? 1.f : fabsf(a.scale)) * TR_LOG2E;
    float f[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, s_m[w][t * 16 + r]);
        f[t] = st.m[t] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((st.m[t] - M) * cc);
    }
    float* o = reinterpret_cast<float*>(lds);
    for (int half = 0; half < D / 64; ++half) {
        if (half) __syncthreads();
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int hh = 0; hh < D / 64; ++hh)
                    if (hh == half) *reinterpret_cast<f32x4*>(o + ((wid * RT + t) * 16 + r) * OROW + 16 * d + 4 * g) = st.o[hh * 4 + d][t] * f[t];
        __syncthreads();
        for (int u = tid; u < RT * 16 * 16; u += 256) {
            const int row = u / 16, x = (u % 16) * 4, at = row0 + row;
            if (at >= rows) continue;
            f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) M = fmaxf(M, s_m[w][row]);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float m = s_m[w][row];
                if (m > -INFINITY || m != m || s_l[w][row] != 0.f) L += s_l[w][row] * (m == M ? 1.f : __builtin_amdgcn_exp2f((m - M) * cc));
                v += *reinterpret_cast<const f32x4*>(o + (w * RT * 16 + row) * OROW + x);
            }
            const int node = at / G;
            if (whole) {
                T* out = reinterpret_cast<T*>(a.d_out) + j.i * a.o_seq + node * a.o_node + (j.kh * G + at % G) * a.o_head + half * 64 + x;
                if (j.ok == 0 || (j.ok == 1 && node >= j.count)) v = f32x4{0.f, 0.f, 0.f, 0.f};
                else if (j.ok == 2 || s_wrong[node]) v = f32x4{1.f, 1.f, 1.f, 1.f} * __builtin_nanf("");
                else v *= 1.f / L;
                store4<T>(out, v);
            } else {
                float* to = part + (int64_t)row * (D + 2);
                *reinterpret_cast<f32x2*>(to + half * 64 + x) = f32x2{v[0], v[1]};
                *reinterpret_cast<f32x2*>(to + half * 64 + x + 2) = f32x2{v[2], v[3]};
                if (x == 0 && half == 0) { to[D] = j.ok == 2 ? __builtin_nanf("") : M; to[D + 1] = L; }
            }
        }
    }
    }
}

// ---- many rows (bf16): every wave has rows of its own, the workgroup shares the tiles of keys and values ------------------------------
// Eight waves, RT x 16 rows each (two waves on every SIMD of a CU).  Tiles of 64 keys go from HBM to LDS without registers
// (global_load_lds) into a ring of four, three tiles before their use; a wave-instruction writes 1 KiB of rows in a line, so the swizzle
// that the fragment reads need (16-byte chunk x of a row in slot x ^ (row mod chunks)) is applied to its lanes' source addresses.
// The softmax of a tile takes the vector pipe about as long as its products take the matrix pipe.  So waves 4-7 run half a tile
// behind waves 0-3, a barrier each half: while one wave of a SIMD does PV(t - 1) and QK(t), the other does the softmax of its tile.
// 8 x 64 nodes, 32 query heads on 8 of 128, 40000-131072 tokens (2.5 GB, 0.52 TFLOP, 0.78 with the second product of split_probs): 1005 us back to
// back (median of 15 replays; 1078 on average under the profiler), 0.78 PFLOP/s executed and 2.5 TB/s; with one product for the probabilities
// 760.  That form, step by step: keys and values through registers and all waves in step 967 us; to LDS directly, in two phases: 835; scalar
// addresses, loads issued in the softmax's half and waves without rows left out of the products: 760.  What is left, part by part (the others
// left out): the stream 467 us, the products with their LDS reads 720, products and softmax without the stream 960.  Splitting the
// probabilities with the products instead of with the softmax: 1020.  16 x 32 rows, 8000-16384 tokens, 8 heads of 128: 198 us, 4.0 TB/s.
//
// 16 bytes a lane from global memory (`from`, alike on the wave, + lane_off) to LDS address `to` + 16 x lane.  Written out because the
// compiler, which knows of the builtin's LDS write, waits for ALL loads before every transposing LDS read, whatever they write; the waits
// are the kernel's own.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"                            // m0 is named as changed on purpose
__device__ __forceinline__ void load_to_lds(const void* from, uint32_t lane_off, uint32_t to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(lane_off), "s"(from), "s"(to) : "m0", "memory");
}
#pragma clang diagnostic pop
constexpr int TRW = 8;                                                    // waves

template <int D, int RT, bool ONE>
__global__ __launch_bounds__(64 * TRW, 2) void tree_attention_rows_kernel(TreeArgs) {
    typedef bf16 T;
    typedef bf16x8 Frag;
    constexpr int KT = 64, NS = 4, KS = D / 32, CPR = D / 8, ROWB = D * 2, HALF = KT * ROWB, RING = 4;
    constexpr int RPW = KT / TRW, NL = RPW * CPR / 64, RPL = 64 / CPR;      // rows of a tile a wave brings, its loads for keys (values: as many), rows a load
    extern __shared__ __attribute__((aligned(1024))) char lds[];            // RING x (keys, values)
    __shared__ TreeJob s_job;
    __shared__ uint64_t s_mask[64];
    __shared__ int s_wrong[64], s_bad;
    TreeJob j;
    for (bool first = true;; first = false) {
    TREE_ARGS(ka);
    TREE_THREAD(tid);
    const int lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, r = lane & 15;
    const bool late = wid >= TRW / 2;
    if constexpr (ONE) { if (!first || !tree_whole<KT>(c, a, p, j, -1)) break; }
    else if (!tree_next<KT>(c, a, p, &s_job, j, first)) break;
    const int G = a.n_head / c.n_kv_head, rows = a.n_nodes * G, part_row0 = ((wid & 3) * 2 + (wid >> 2)) * 16 * RT, row0 = j.rb * TRW * 16 * RT + part_row0;
    if (wid == 0 && j.ok == 1) {
        bool wrong;
        const uint64_t m = tree_mask(a.d_parents ? a.d_parents + (int64_t)j.i * a.n_nodes : nullptr, lane, a.n_nodes, &wrong);
        s_mask[lane] = m; s_wrong[lane] = wrong;
    }
    if (tid == 0) { s_bad = 0; if (ONE) s_job = j; }
    __syncthreads();
    if (j.ok == 1 && tree_bad(c, a, p, j, KT, tid, 64 * TRW)) s_bad = 1;                          // (read behind later barriers)
    const int seq = __builtin_amdgcn_readfirstlane(j.seq), kh = __builtin_amdgcn_readfirstlane(j.kh), len = __builtin_amdgcn_readfirstlane(j.len);
    const int32_t* table = c.d_table + (int64_t)seq * c.max_pages;
    const int64_t page_e = (int64_t)c.n_kv_head * c.page_size * D, head_off = (int64_t)a.layer * c.n_pages * page_e + (int64_t)kh * c.page_size * D;
    RowState<D, RT> st;
    st.init();
    const float cc = (a.scale == 0.f ? 1.f : fabsf(a.scale)) * TR_LOG2E;
    if (j.ok == 1) {
        Frag qf[RT][KS];
        const float sign = a.scale < 0.f ? -1.f : a.scale > 0.f ? 1.f : 0.f;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int row = min(row0 + t * 16 + r, rows - 1), node = row / G;
            const T* q = reinterpret_cast<const T*>(a.d_q) + j.i * a.q_seq + node * a.q_node + (kh * G + row % G) * a.q_head;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                qf[t][ks] = *reinterpret_cast<const Frag*>(q + (ks * 4 + g) * 8);
                if (sign != 1.f) {
#pragma unroll
                    for (int x = 0; x < 8; ++x) qf[t][ks][x] = (T)((float)qf[t][ks][x] * sign);
                }
            }
        }
        const T* Kp = reinterpret_cast<const T*>(c.d_k) + head_off;
        const T* Vp = reinterpret_cast<const T*>(c.d_v) + head_off;
        const int t0 = __builtin_amdgcn_readfirstlane(j.t0), n_tiles = __builtin_amdgcn_readfirstlane(min(j.t1, j.n_pre)) - t0;
        const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds);
        // this wave's rows of a tile are on one page (RPW divides 16): the pages of 64 tiles, one a lane
        int pages = 0;
        auto page_of = [&](int t) {
            if ((t & 63) == 0) {
                pages = page_ok(c, table[min((t0 + min(t + lane, n_tiles - 1)) * KT + wid * RPW, len - 1) >> p.shift]);
                __builtin_amdgcn_s_waitcnt(0x0f70);                                // vmcnt(0): here, not by the compiler in every tile
            }
            return __builtin_amdgcn_readlane(pages, t & 63);
        };
        // no vector instructions but in the last tile: everything but the lane's place in the rows is alike on the wave
        uint32_t lane_off[NL];
#pragma unroll
        for (int x = 0; x < NL; ++x) {
            const int row = x * RPL + lane / CPR;
            lane_off[x] = row * ROWB + ((lane % CPR) ^ ((wid * RPW + row) & (CPR - 1))) * 16;
        }
        auto issue = [&](const T* pool, int half, int t, int page) {
            const int at = (t0 + t) * KT + wid * RPW, live = len - at;               // rows of this wave that are tokens
            const char* from = reinterpret_cast<const char*>(pool) + ((int64_t)page * page_e + (int64_t)(at & (c.page_size - 1)) * D) * 2;
            const uint32_t to = lds0 + (t & (RING - 1)) * 2 * HALF + half + wid * RPW * ROWB;
            if (live >= RPW) {
#pragma unroll
                for (int x = 0; x < NL; ++x) load_to_lds(from, lane_off[x], to + x * 1024);
            } else {                                                                // rows past the last token read it instead
                if (live <= 0) from = reinterpret_cast<const char*>(pool) + ((int64_t)page * page_e + (int64_t)((len - 1) & (c.page_size - 1)) * D) * 2;
                const int last = max(live, 1) - 1;
#pragma unroll
                for (int x = 0; x < NL; ++x) {
                    const int row = x * RPL + lane / CPR;
                    load_to_lds(from, lane_off[x] - (row - min(row, last)) * ROWB, to + x * 1024);
                }
            }
        };
        // Before QK(t) and PV(t - 1): this wave's loads of keys t and values t - 1 are done.  Issued behind them: keys t + 1, values t and, but by
        // the late waves, who wait half a tile before they issue, keys t + 2, values t + 1; at the end there are fewer, and all are waited for.
        auto landed = [&](int t) {
            if (t + 2 < n_tiles && (!late || t == 0)) {
                if constexpr (NL == 2) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
                else asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
            } else if (t + 2 < n_tiles) {
                if constexpr (NL == 2) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
                else asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
            } else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (t == n_tiles - 1) {                                                // the last tile's values are here too: rows past the last token count as 0
                const int live = len - (t0 + t) * KT;
                if (live < KT) {
                    char* vb = lds + (t & (RING - 1)) * 2 * HALF + HALF;
                    for (int u = lane; u < RPW * CPR; u += 64) {
                        const int row = wid * RPW + u / CPR;
                        if (row >= live) *reinterpret_cast<Frag*>(vb + row * ROWB + (u % CPR) * 16) = Frag{};
                    }
                }
            }
        };
        auto barrier = [&]() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); __builtin_amdgcn_sched_barrier(0); };
        // chunk 4 ks + g of key 16 k + r; chunk 2 d + (r & 3) / 2 of value row 32 h + 16 u + 4 g + r / 4
        const int kx = (g ^ (r & (CPR - 1))) << 4, vrow = 4 * g + (r >> 2), vx = ((((r & 3) >> 1) ^ (vrow & (CPR - 1))) << 4);
        // fragments of the next 16 keys (of the next 16 columns) are read while the matrix pipe works on these: the order is pinned, or the
        // compiler reads each right before its use and waits for LDS every time
        auto scores = [&](const char* kb, f32x4 (&s)[NS][RT]) {
            constexpr int AHEAD = 2;
            Frag kf[AHEAD + 1][KS];
            auto read = [&](int k) {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) kf[k % (AHEAD + 1)][ks] = *reinterpret_cast<const Frag*>(kb + (k * 16 + r) * ROWB + ((ks * 64) ^ kx));
                __builtin_amdgcn_sched_barrier(0);
            };
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) read(k);
#pragma unroll
            for (int k = 0; k < NS; ++k) {
                if (k + AHEAD < NS) read(k + AHEAD);
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) x = Elem<T>::qk(kf[k % (AHEAD + 1)][ks], qf[t][ks], x);
                    s[k][t] = x;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto pack = [&](const f32x4 (&s)[NS][RT], Frag (&pf)[RT][2], Frag (&pl)[RT][2]) {
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) split_probs(s[2 * h][t], s[2 * h + 1][t], pf[t][h], pl[t][h]);
        };
        auto add = [&](const char* vb, const Frag (&pf)[RT][2], const Frag (&pl)[RT][2]) {
            constexpr int AHEAD = 2;
            Frag vf[AHEAD + 1][2];
            auto read = [&](int d) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const char* p0 = vb + (32 * h + vrow) * ROWB + ((32 * d) ^ vx) + (r & 1) * 8;
                    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(p0));
                    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(p0 + 16 * ROWB));
                    vf[d % (AHEAD + 1)][h] = __builtin_bit_cast(Frag, (i16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                }
                __builtin_amdgcn_sched_barrier(0);
            };
#pragma unroll
            for (int d = 0; d < AHEAD; ++d) read(d);
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
                if (d + AHEAD < D / 16) read(d + AHEAD);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int t = 0; t < RT; ++t) st.o[d][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[d % (AHEAD + 1)][h], pf[t][h], st.o[d][t], 0, 0, 0);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int t = 0; t < RT; ++t) st.o[d][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[d % (AHEAD + 1)][h], pl[t][h], st.o[d][t], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        Frag pf[RT][2], pl[RT][2];
        const int count = __builtin_amdgcn_readfirstlane(j.count);
        if (n_tiles > 0) {
            __builtin_amdgcn_s_waitcnt(0);                                          // the counts below are of tiles' loads only (the builtin, so
            __builtin_amdgcn_sched_barrier(0);                                      // that the compiler does not wait for the queries in the loop)
            const int page0 = page_of(0), page1 = page_of(1);
            int page_v = page_of(2), page_k = page_of(3);                           // of tiles past the end: the last one's, not used
            issue(Kp, 0, 0, page0);
            if (n_tiles > 1) issue(Kp, 0, 1, page1);
            issue(Vp, HALF, 0, page0);
            if (n_tiles > 2) issue(Kp, 0, 2, page_v);
            if (n_tiles > 1) issue(Vp, HALF, 1, page1);
            landed(0);
            barrier();
            if (late) barrier();
            // Keys t + 3 take the place of keys t - 1, values t + 2 of values t - 2: the late waves read both last, two barriers ago for the
            // early waves, one for themselves.  Issued with the softmax and not before the products, which are the longer half.
            auto more = [&](int t) {
                if (t + 3 < n_tiles) issue(Kp, 0, t + 3, page_k);
                if (t + 2 < n_tiles) issue(Vp, HALF, t + 2, page_v);
                page_v = page_k;
                if (t + 4 < n_tiles) page_k = page_of(t + 4);
            };
            if (row0 < count * G) {
                for (int t = 0; t < n_tiles; ++t) {
                    if (t > 0) add(lds + ((t - 1) & (RING - 1)) * 2 * HALF + HALF, pf, pl);
                    f32x4 s[NS][RT];
                    scores(lds + (t & (RING - 1)) * 2 * HALF, s);
                    if (late && t + 1 < n_tiles) landed(t + 1);
                    barrier();
                    more(t);
                    const int live = len - (t0 + t) * KT;
                    if (live < KT) {
                        asm volatile("");                                           // keep it a branch: as selects it costs every tile
#pragma unroll
                        for (int k = 0; k < NS; ++k)
#pragma unroll
                            for (int x = 0; x < 4; ++x)
                                if (16 * k + 4 * g + x >= live)
#pragma unroll
                                    for (int q = 0; q < RT; ++q) s[k][q][x] = -INFINITY;
                    }
                    st.template softmax<NS>(s, cc);
                    pack(s, pf, pl);
                    if (!late && t + 1 < n_tiles) landed(t + 1);
                    barrier();
                }
                add(lds + ((n_tiles - 1) & (RING - 1)) * 2 * HALF + HALF, pf, pl);
            } else {                                                               // a wave of nodes that are not there only brings its rows
                for (int t = 0; t < n_tiles; ++t) {
                    if (late && t + 1 < n_tiles) landed(t + 1);
                    barrier();
                    more(t);
                    if (!late && t + 1 < n_tiles) landed(t + 1);
                    barrier();
                }
            }
            if (!late) barrier();
            __syncthreads();
        }
        j = s_job;                                                                 // not kept in registers over the loop
        if (j.t1 > j.n_pre) {                                                      // the drafted rows: one tile, through registers
            Frag rk[NL], rv[NL];
            int odd = 0;
#pragma unroll
            for (int x = 0; x < NL; ++x) {
                const int node = min(wid * RPW + x * RPL + lane / CPR, j.count - 1);
                rk[x] = *reinterpret_cast<const Frag*>(node_row<T, D>(c, a, p, j, table, head_off, page_e, true, node) + (lane % CPR) * 8);
                rv[x] = *reinterpret_cast<const Frag*>(node_row<T, D>(c, a, p, j, table, head_off, page_e, false, node) + (lane % CPR) * 8);
                odd |= Elem<T>::odd(rv[x]);
            }
            const bool any_odd = __syncthreads_or(odd);
#pragma unroll
            for (int x = 0; x < NL; ++x) {
                const int row = wid * RPW + x * RPL + lane / CPR, slot = ((lane % CPR) ^ (row & (CPR - 1))) << 4;
                if (any_odd) rv[x] = finite_only(rv[x]);
                *reinterpret_cast<Frag*>(lds + row * ROWB + slot) = rk[x];
                *reinterpret_cast<Frag*>(lds + HALF + row * ROWB + slot) = row < j.count ? rv[x] : Frag{};
            }
            __syncthreads();
            f32x4 s[NS][RT];
            scores(lds, s);
            uint64_t mask[RT];
#pragma unroll
            for (int t = 0; t < RT; ++t) mask[t] = s_mask[min(row0 + t * 16 + r, rows - 1) / G];
#pragma unroll
            for (int k = 0; k < NS; ++k)
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int q = 0; q < RT; ++q) if (!((mask[q] >> (16 * k + 4 * g + x)) & 1)) s[k][q][x] = -INFINITY;
            st.template softmax<NS>(s, cc);
            pack(s, pf, pl);
            add(lds + HALF, pf, pl);
            if (any_odd) add_odd_values<T, D, RT, NS>(c, a, p, j, table, head_off, page_e, 0, s, mask, st, g, r);
        }
    }
    __syncthreads();
    j = s_job;
    if (j.ok == 1 && s_bad) j.ok = 2;
    if (j.ok == 1 && a.d_kn && j.rb == 0 && j.last) append_nodes<T, D>(c, a, p, j, table, head_off, page_e, tid, 64 * TRW);
    const bool whole = j.whole;
    float* part = whole ? nullptr : p.part + (((int64_t)j.piece * c.n_kv_head + j.kh) * p.row_blocks + j.rb) * (TRW * 16 * RT) * (D + 2);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        float l = st.l[t];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        const int at = row0 + t * 16 + r;
        if (at >= rows) continue;
        const int node = at / G;
        if (whole) {
            T* out = reinterpret_cast<T*>(a.d_out) + j.i * a.o_seq + node * a.o_node + (j.kh * G + at % G) * a.o_head;
            const int kind = j.ok == 1 ? node >= j.count ? 0 : s_wrong[node] ? 2 : 1 : j.ok;
            const float f = 1.f / l;
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
                store4<T>(out + 16 * d + 4 * g, kind == 1 ? st.o[d][t] * f : f32x4{1.f, 1.f, 1.f, 1.f} * (kind == 0 ? 0.f : __builtin_nanf("")));
        } else {
            float* to = part + (int64_t)(part_row0 + t * 16 + r) * (D + 2);
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
                *reinterpret_cast<f32x2*>(to + 16 * d + 4 * g) = f32x2{st.o[d][t][0], st.o[d][t][1]};
                *reinterpret_cast<f32x2*>(to + 16 * d + 4 * g + 2) = f32x2{st.o[d][t][2], st.o[d][t][3]};
            }
            if (g == 0) { to[D] = j.ok == 2 ? __builtin_nanf("") : st.m[t]; to[D + 1] = l; }
        }
    }
    }
}

// ---- merge of the pieces of a sequence: grid (sequence, key / value head, merge_rows rows), D / 4 threads a row and group of pieces -----
//   M = max_p m_p,  o = sum_p exp(m_p - M) o_p / sum_p exp(m_p - M) l_p
// Reads every piece's 32-bit parts once: 8 x 64 nodes, 32 heads of 128, 40 pieces a sequence in 256 shares: 14 us.
template <typename T, int D, int KT>
__global__ __launch_bounds__(256) void tree_attention_merge_kernel(wx_cache c, wx_tree_attn a, TreePlan p) {
    __shared__ int s_first, s_pieces, s_wrong[64];
    const int i = blockIdx.x, kh = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int seq = a.d_seqs[i];
    if (tid < 64) {
        int pieces, at;
        if (p.per) {
            int before = 0;
            for (int x = lane; x < i; x += 64) before += (tree_tiles_of(c, a, p, x, KT) + p.per - 1) / p.per;
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) before += __shfl_xor(before, off);
            pieces = (tree_tiles_of(c, a, p, i, KT) + p.per - 1) / p.per; at = before;
        } else {
            int takers;
            const int64_t all = tree_all(c, a, p, KT, lane, &takers);
            int64_t before = 0;
            for (int x = lane; x < i; x += 64) before += tree_tiles_of(c, a, p, x, KT);
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) before += __shfl_xor(before, off);
            const int w = tree_taker(before, all, takers);
            pieces = tree_taker(before + tree_tiles_of(c, a, p, i, KT) - 1, all, takers) - w + 1; at = w + i;
        }
        bool wrong;
        (void)tree_mask(a.d_parents ? a.d_parents + (int64_t)i * a.n_nodes : nullptr, lane, a.n_nodes, &wrong);
        s_wrong[lane] = wrong;
        if (lane == 0) { s_first = at; s_pieces = pieces; }
    }
    __syncthreads();
    const int pieces = s_pieces, first = s_first;
    if (pieces <= 1) return;                                                        // written by the piece itself
    const int count = a.d_counts ? min(max(a.d_counts[i], 0), a.n_nodes) : a.n_nodes;
    const int G = a.n_head / c.n_kv_head, rows = a.n_nodes * G;
    const float cc = (a.scale == 0.f ? 1.f : fabsf(a.scale)) * TR_LOG2E;
    constexpr int TPR = D / 4, RPB = 256 / TPR;
    __shared__ f32x4 s_v[RPB][TPR];
    __shared__ float s_m[RPB], s_l[RPB];
    const int slot = tid / TPR, groups = RPB / p.merge_rows, group = slot / p.merge_rows;
    const int row = blockIdx.z * p.merge_rows + slot % p.merge_rows, x = (tid % TPR) * 4;
    const int64_t step = (int64_t)c.n_kv_head * p.row_blocks * p.rows * (D + 2);
    const float* part = p.part + ((((int64_t)first * c.n_kv_head + kh) * p.row_blocks + min(row, rows - 1) / p.rows) * p.rows + min(row, rows - 1) % p.rows) * (D + 2);
    // four pieces' loads at a time, one running maximum (a launch of this size is bound by the loads' latency)
    float M = -INFINITY, L = 0.f;
    bool refused = false;                                                           // by any piece: a maximum is never NaN otherwise
    f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int q0 = 4 * group; q0 < pieces; q0 += 4 * groups) {
        float m[4], l[4];
        f32x2 lo[4], hi[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float* from = part + min(q0 + q, pieces - 1) * step;
            m[q] = from[D]; l[q] = from[D + 1];
            lo[q] = *reinterpret_cast<const f32x2*>(from + x); hi[q] = *reinterpret_cast<const f32x2*>(from + x + 2);
        }
        float mn = M;
#pragma unroll
        for (int q = 0; q < 4; ++q) { mn = fmaxf(mn, m[q]); refused |= m[q] != m[q]; }
        const float old = M == mn ? 1.f : __builtin_amdgcn_exp2f((M - mn) * cc);
        M = mn;
        L *= old; v *= old;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (q0 + q < pieces) {
                const float f = m[q] == mn ? 1.f : __builtin_amdgcn_exp2f((m[q] - mn) * cc);
                L = fmaf(l[q], f, L);
                v += f32x4{lo[q][0], lo[q][1], hi[q][0], hi[q][1]} * f;
            }
    }
    if (groups > 1) {                                                               // the groups' parts, in order
        s_v[slot][tid % TPR] = v;
        if (x == 0) { s_m[slot] = refused ? __builtin_nanf("") : M; s_l[slot] = L; }
        __syncthreads();
        if (group > 0) return;
        for (int o = slot + p.merge_rows; o < RPB; o += p.merge_rows) {
            const float mo = s_m[o], mn = fmaxf(M, mo);
            refused |= mo != mo;
            const float fa = M == mn ? 1.f : __builtin_amdgcn_exp2f((M - mn) * cc), fb = mo == mn ? 1.f : __builtin_amdgcn_exp2f((mo - mn) * cc);
            M = mn;
            L = L * fa + s_l[o] * fb;
            v = v * fa + s_v[o][tid % TPR] * fb;
        }
    }
    if (row >= rows) return;
    const int node = row / G;
    T* out = reinterpret_cast<T*>(a.d_out) + i * a.o_seq + node * a.o_node + (kh * G + row % G) * a.o_head + x;
    const int kind = refused ? 2 : seq == -1 || node >= count ? 0 : s_wrong[node] ? 2 : 1;
    store4<T>(out, kind == 1 ? v * (1.f / L) : f32x4{1.f, 1.f, 1.f, 1.f} * (kind == 0 ? 0.f : __builtin_nanf("")));
}

// (more LDS than a launch has by default: asked for once per device, before the first launch there)
template <int D, int RT, bool ONE>
static hipError_t launch_rows(dim3 grid, int lds, hipStream_t st, const wx_cache& c, const wx_tree_attn& a, const TreePlan& p) {
    static std::atomic<uint64_t> asked{0};
    const uint64_t bit = 1ull << (c.device & 63);
    if (c.device > 63 || !(asked.load(std::memory_order_relaxed) & bit)) {
        const hipError_t e = hipFuncSetAttribute((const void*)tree_attention_rows_kernel<D, RT, ONE>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
        asked.fetch_or(bit, std::memory_order_relaxed);
    }
    hipLaunchKernelGGL((tree_attention_rows_kernel<D, RT, ONE>), grid, dim3(64 * TRW), lds, st, TreeArgs{c, a, p});
    return hipSuccess;
}

// Which kernel, and how the work is cut.
struct TreeForm { bool rows_form; int rt, rows, kt; };
static TreeForm tree_form(const wx_cache& c, const wx_tree_attn& a) {
    const int G = a.n_head / c.n_kv_head, rows = a.n_nodes * G, es = c.precision == WX_PREC_F32 ? 4 : 2;
    TreeForm f;
    // us with the keys shared / the rows shared, 16 sequences, 8 key / value heads.  Heads of 128, 30-420 tokens: 20 rows 17 / 24, 32 38 / 32, 64 59 /
    // 35; 4000-16000 tokens: 32 rows 155 / 163, 64 239 / 174, 256 764 / 315.  Heads of 64, whose tiles are half as large for the same barriers:
    // 4000-16000 tokens: 64 rows 98 / 193, 128 144 / 202, 192 199 / 208, 256 248 / 214; 30-420: 64 39 / 33, 128 51 / 37, 256 57 / 42.
    // With split_tokens the number of nodes must not matter (it is the widest sequence's): by the heads alone.  Heads of 128, 4 query heads: 1 node
    // 132 / 167, 8 171 / 213, 16 270 / 233, 64 973 / 441; 2: 1 133 / 165, 16 171 / 213, 32 272 / 233.
    f.rows_form = c.precision == WX_PREC_BF16 && (a.split_tokens > 0 ? c.head_dim == 128 && G >= 4 : rows > (c.head_dim == 128 ? 16 : 128));
    // 32 rows a wave (two row tiles for every fragment read) where they are there and the registers allow it
    f.rt = f.rows_form ? rows > 128 ? 2 : 1 : rows > 16 && c.head_dim == 64 ? 2 : 1;
    f.rows = f.rows_form ? 128 * f.rt : 16 * f.rt;
    f.kt = f.rows_form ? 64 : 8192 / (c.head_dim * es);
    return f;
}
static TreePlan tree_plan(const wx_cache& c, const wx_tree_attn& a, const TreeForm& f) {
    TreePlan p{};
    const int rows = a.n_nodes * (a.n_head / c.n_kv_head);
    p.row_blocks = (rows + f.rows - 1) / f.rows;
    p.rows = f.rows;
    p.tree_tiles = (a.n_nodes + f.kt - 1) / f.kt;
    while ((1 << p.shift) < c.page_size) ++p.shift;
    const int64_t most = ((int64_t)c.max_pages * c.page_size + f.kt - 1) / f.kt + p.tree_tiles;       // tiles of the longest sequence the tables hold
    const int64_t units = (int64_t)c.n_kv_head * p.row_blocks;
    // Shares of 512 tokens at least, but of 128 up to the first 256 workgroups, which leave compute units idle: one sequence of 40575 tokens,
    // 1 head of 64, f32: 37 us with 512, 23 with 128, 25 with 64; 7 sequences of up to 1912, 1 head of 128, f32: 39, 28, 26; 5 of up to 2283,
    // 20 heads of 128, bf16 (260 shares of 512): 28, 36.  Tables of up to 512 tokens are not cut at all: the second launch costs 5 us and the
    // pieces save less (1 x 430 tokens, 20 heads of 64: 12 us whole, 18 cut).
    p.least = 512 / f.kt + p.tree_tiles;
    p.least_few = 128 / f.kt + p.tree_tiles;
    p.few = (int)(units < 256 ? 256 / units : 1);
    // As many workgroups as run at once (one a compute unit that shares rows, two that share keys), never a few more, which would run alone at
    // the end: 3 sequences of up to 32792 tokens, 12 heads, 184 rows: 264 workgroups 240 us, 252 148 us; 16 x 24 rows, 20 heads of 64, 4000-16000
    // tokens: 512 workgroups 182 us, 768 203 us.  Where heads and row blocks do not divide that number nearly, four times as many smaller ones.
    const int64_t slots = f.rows_form ? 256 : 512;
    int64_t takers = slots / units;
    if (5 * takers * units < 4 * slots) takers = 4 * slots / units;
    p.takers = (int)(takers > 1 ? takers : 1);
    if (a.split_tokens > 0) {                                                       // at most 256 pieces a sequence, whatever n_nodes is
        const int64_t widest = most - p.tree_tiles + (TR_NODES + f.kt - 1) / f.kt;
        p.per = (int)(((int64_t)a.split_tokens + f.kt - 1) / f.kt);
        if (p.per < (widest + 255) / 256) p.per = (int)((widest + 255) / 256);
    }
    p.single = most <= (p.per ? p.per : 512 / f.kt + p.tree_tiles);
    p.slots = p.single ? a.n : p.per ? (int)(a.n * ((most + p.per - 1) / p.per)) : p.takers;
    p.pieces = p.single ? 0 : p.per ? p.slots : p.takers + a.n;
    // the merge: as few rows a workgroup (as many threads on a row's pieces) as leave it at most 2048 workgroups (6 sequences of up to 38255
    // tokens, 2 heads of 64, f32, shares of 128: 55 us so, 67 with every row's pieces on one group of threads); the order of the sum follows from
    // it, so with `per` it is taken for 8 sequences of 8 nodes whatever their number
    const int64_t merges = (int64_t)c.n_kv_head * (p.per ? 8 : a.n), merged = p.per ? 8 * (a.n_head / c.n_kv_head) : rows;
    p.merge_rows = 1024 / c.head_dim;
    while (p.merge_rows > 1 && merges * ((merged + p.merge_rows / 2 - 1) / (p.merge_rows / 2)) <= 2048) p.merge_rows /= 2;
    return p;
}
// Whether a wave alone takes a whole sequence (a key / value head, a block of rows): jobs enough to fill the chip without cutting them, and
// few tiles each.  us with four waves a job / one, 20 heads, 1 row: bf16, heads of 64, 200-447 tokens: 40 sequences 21.0 / 20.4, 64 30.6 / 29.4, 100
// 40.9 / 33.8, 200 89.5 / 70.5; 20-100 tokens: 40 15.2 / 12.2, 64 19.8 / 14.4, 200 53.9 / 27.4; f32, 64, 20-100: 26 15.2 / 16.9, 40 17.9 / 17.7, 200
// 64.6 / 40.5.  More tiles (bf16, heads of 128, 447 tokens: 15): 64 42.7 / 46.1, 100 68.0 / 62.9; 29 tiles (f32): 200 247 / 264.  More rows, bf16:
// 64 x 92 rows, 8 heads, 5-9 tokens 29.6 / 16.1, 64 x 24, 20 heads, 30-420 tokens 36.6 / 32.6; f32, whose products take longer: 40 x 24, 20 heads,
// 30-420 tokens 51 / 59.  With split_tokens a result must not depend on the number of sequences.
static bool tree_solo(const wx_cache& c, const wx_tree_attn& a, const TreeForm& f, const TreePlan& p) {
    const int rows = a.n_nodes * (a.n_head / c.n_kv_head);
    const int64_t jobs = (int64_t)a.n * c.n_kv_head * p.row_blocks, most = ((int64_t)c.max_pages * c.page_size + f.kt - 1) / f.kt + p.tree_tiles;
    return p.single && a.split_tokens == 0 && !f.rows_form && (c.precision == WX_PREC_BF16 || rows <= 16) && ((jobs >= 768 && most <= 9) || (jobs >= 2000 && most <= 16));
}
static int64_t tree_part_bytes(const wx_cache& c, const TreePlan& p) {
    return (int64_t)p.pieces * c.n_kv_head * p.row_blocks * p.rows * (c.head_dim + 2) * 4;
}

// ---- the decoder's input for drafted tokens: one workgroup a node ------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void tree_embed_kernel(const T* tok_emb, const T* pos_emb, wx_cache c, const int32_t* seqs, const int32_t* tokens, const int32_t* parents,
                                                         int n_nodes, float* x, int d, int n_tok, int n_pos) {
    const int i = blockIdx.x / n_nodes, j = blockIdx.x % n_nodes, s = seqs[i];
    int depth = j;
    if (parents) {
        depth = 0;
        for (int at = j, up = parents[(int64_t)i * n_nodes + j]; up >= 0 && up < at; ++depth) { at = up; up = parents[(int64_t)i * n_nodes + at]; }
    }
    int t = depth + (s >= 0 && s < c.max_seqs ? c.d_lens[s] : 0);
    if (t > n_pos - 1) t = n_pos - 1;
    if (t < 0) t = 0;
    int token = tokens[blockIdx.x];
    if ((unsigned)token >= (unsigned)n_tok) token = n_tok - 1;
    const T *te = tok_emb + (int64_t)token * d, *pe = pos_emb + (int64_t)t * d;
    for (int q = threadIdx.x; q < d; q += 256) x[(int64_t)blockIdx.x * d + q] = (float)te[q] + (float)pe[q];
}
int launch_tree_embed(const void* tok_emb, const void* pos_emb, int dt, const wx_cache& c, const int32_t* seqs, const int32_t* tokens, const int32_t* parents,
                      int n, int n_nodes, float* x, int d, hipStream_t st, int n_tok, int n_pos) {
    if (n < 1 || n_nodes < 1 || n_tok < 1 || n_pos < 1) return -1;
    if (dt == DT_F32) hipLaunchKernelGGL(tree_embed_kernel<float>, dim3(n * n_nodes), dim3(256), 0, st, (const float*)tok_emb, (const float*)pos_emb, c, seqs, tokens, parents, n_nodes, x, d, n_tok, n_pos);
    else hipLaunchKernelGGL(tree_embed_kernel<bf16>, dim3(n * n_nodes), dim3(256), 0, st, (const bf16*)tok_emb, (const bf16*)pos_emb, c, seqs, tokens, parents, n_nodes, x, d, n_tok, n_pos);
    return hipGetLastError() == hipSuccess ? 0 : -2;
}

// ---- verification ---------------------------------------------------------------------------------------------------------------------
struct Best { float m, s; int i; };       // largest logit, sum of exp(logit - m), its lowest id
__device__ __forceinline__ Best best_merge(Best a, Best b) {
    if (a.m == b.m) return Best{a.m, a.s + b.s, min(a.i, b.i)};
    if (b.m > a.m) { const Best t = a; a = b; b = t; }
    a.s += b.s * __builtin_amdgcn_exp2f((b.m - a.m) * TR_LOG2E);     // b.m may be -infinity: + 0
    return a;
}
// N values of ids i .. i + N - 1 (masked ones are -infinity).  The maximum of all of them comes first, so that the running sum is rescaled
// once for N ids, and seldom; v - m is rounded before it is scaled, or the rounding of m log2 e would shift every term.
template <int N>
__device__ __forceinline__ void best_add(Best& b, float (&v)[N], int i) {
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < N; ++j) { v[j] = fmaxf(v[j], -INFINITY); top = fmaxf(top, v[j]); }        // NaN counts as masked
    if (top > b.m) {
        b.s *= __builtin_amdgcn_exp2f((b.m - top) * TR_LOG2E);
        b.m = top;
#pragma unroll
        for (int j = N - 1; j >= 0; --j) if (v[j] == top) b.i = i + j;
    }
    if (b.m == INFINITY) {                                            // infinite logits share the probability
#pragma unroll
        for (int j = 0; j < N; ++j) b.s += v[j] == INFINITY ? 1.f : 0.f;
    } else if (b.m > -INFINITY) {
#pragma unroll
        for (int j = 0; j < N; ++j) b.s += __builtin_amdgcn_exp2f((v[j] - b.m) * TR_LOG2E);
    }
}
constexpr int VF_NT = 256, VF_U = 4;       // VF_U 16-byte loads a thread are in flight

// One workgroup a (part of the vocabulary, node, sequence): one pass over the logits, 16 bytes a lane, with the running maximum and sum.
// Bound by their stream: 64 x 16 nodes (795 there), 51866 ids, f32: 165 MB in 33 us, 5.0 TB/s (element by element: 146 us).
template <typename T>
__global__ __launch_bounds__(VF_NT) void tree_verify_scan_kernel(wx_tree_check a, int parts) {
    constexpr int E = 16 / sizeof(T);
    __shared__ Best sh[VF_NT / 64];
    const int part = blockIdx.x, node = blockIdx.y, i = blockIdx.z, tid = threadIdx.x;
    const int count = a.d_counts ? a.d_counts[i] : a.n_nodes;
    if (node >= count) return;
    const T* row = reinterpret_cast<const T*>(a.d_logits) + i * a.l_seq + node * a.l_node;
    // aligned 16-byte units of the row; the ids before the first and after the last (fewer than 16) go one by one, with part 0
    const int head = min(a.n_vocab, (int)(((16 - ((uintptr_t)row & 15)) & 15) / sizeof(T))), units = (a.n_vocab - head) / E;
    const int per = (units + parts - 1) / parts, lo = part * per, hi = min(units, lo + per);
    const uint8_t* sup = a.d_suppress;
    Best h{-INFINITY, 0.f, 0x7fffffff}, b = h;
    if (part == 0 && tid < a.n_vocab - units * E) {
        const int x = tid < head ? tid : units * E + tid;
        float v[1] = {sup && sup[x] ? -INFINITY : (float)row[x]};
        best_add<1>(h, v, x);
    }
    typedef __attribute__((ext_vector_type(E))) T Unit;
    for (int u0 = lo + tid; u0 < hi; u0 += VF_NT * VF_U) {
        Unit x[VF_U];
        uint32_t m[VF_U][E / 4];
#pragma unroll
        for (int k = 0; k < VF_U; ++k) {
            const int u = min(u0 + k * VF_NT, units - 1);
            x[k] = __builtin_nontemporal_load(reinterpret_cast<const Unit*>(row + head) + u);
            if (sup) __builtin_memcpy(m[k], sup + head + u * E, E);
            else __builtin_memset(m[k], 0, E);
        }
#pragma unroll
        for (int k = 0; k < VF_U; ++k) {
            if (u0 + k * VF_NT >= hi) break;
            float v[E];
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] = (float)x[k][j];
            uint32_t any = m[k][0];
            if constexpr (E == 8) any |= m[k][1];
            if (any) {
#pragma unroll
                for (int j = 0; j < E; ++j) if ((m[k][j / 4] >> (8 * (j % 4))) & 0xff) v[j] = -INFINITY;
            }
            best_add<E>(b, v, head + (u0 + k * VF_NT) * E);
        }
    }
    b = best_merge(b, h);
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
        reinterpret_cast<f32x4*>(a.d_work)[((int64_t)i * a.n_nodes + node) * parts + part] = f32x4{b.m, b.s, __builtin_bit_cast(float, b.i), 0.f};
    }
}

// one wave a sequence: lane j merges node j's parts, then the wave walks down the tree.  Latency: 4 us for 64 x 16 nodes (4 parts each), 6.6 us
// for 8 nodes in 26 parts
__global__ __launch_bounds__(64) void tree_verify_walk_kernel(wx_tree_check a, int parts) {
    const int i = blockIdx.x, j = threadIdx.x;
    const int count = a.d_counts ? min(max(a.d_counts[i], 0), a.n_nodes) : a.n_nodes;
    int pick = -1, token = -1, up = -1;
    float lp = 0.f;
    if (j < count) {
        Best b{-INFINITY, 0.f, 0x7fffffff};
        const f32x4* rec = reinterpret_cast<const f32x4*>(a.d_work) + ((int64_t)i * a.n_nodes + j) * parts;
#pragma unroll 8
        for (int p = 0; p < parts; ++p) { const f32x4 x = rec[p]; b = best_merge(b, Best{x[0], x[1], __builtin_bit_cast(int, (float)x[2])}); }
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
    return tree_part_bytes(*c, tree_plan(*c, *a, tree_form(*c, *a)));
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
    const TreeForm f = tree_form(*c, *a);
    TreePlan p = tree_plan(*c, *a, f);
    p.part = (float*)a->d_work;
    const int64_t need = tree_part_bytes(*c, p);
    if (need > 0 && (!a->d_work || a->work_bytes < need || ((uintptr_t)a->d_work & 15))) return set_error(WX_ERR_INVALID, "work buffer too small or not 16-byte aligned");
    const int64_t jobs = ((int64_t)p.slots * c->n_kv_head + 7) / 8 * 8 * p.row_blocks;
    if (jobs > 0x7fffff) return set_error(WX_ERR_INVALID, "too many pieces of work: fewer sequences, or larger split_tokens");
    const dim3 grid((unsigned)jobs), block(256);
    const bool f32 = c->precision == WX_PREC_F32, wide = c->head_dim == 128;
#define TREE_SOLO(T, D, RT) hipLaunchKernelGGL((tree_attention_keys_kernel<T, D, RT, true, true>), dim3((unsigned)((jobs + 3) / 4)), block, 0, st, TreeArgs{*c, *a, p})
#define TREE_KEYS(T, D, RT) do { if (p.single) hipLaunchKernelGGL((tree_attention_keys_kernel<T, D, RT, true>), grid, block, 0, st, TreeArgs{*c, *a, p}); \
                                 else hipLaunchKernelGGL((tree_attention_keys_kernel<T, D, RT, false>), grid, block, 0, st, TreeArgs{*c, *a, p}); } while (0)
#define TREE_ROWS(D, RT) do { const int lds = 4 * 2 * 64 * D * 2; \
                              const hipError_t le = p.single ? launch_rows<D, RT, true>(grid, lds, st, *c, *a, p) : launch_rows<D, RT, false>(grid, lds, st, *c, *a, p); \
                              if (le != hipSuccess) return set_error(WX_ERR_HIP, hipGetErrorString(le)); } while (0)
    if (f.rows_form) {
        if (wide) { if (f.rt == 2) TREE_ROWS(128, 2); else TREE_ROWS(128, 1); }
        else TREE_ROWS(64, 2);
    } else if (tree_solo(*c, *a, f, p)) {
        if (f32) { if (wide) TREE_SOLO(float, 128, 1); else TREE_SOLO(float, 64, 1); }
        else { if (wide) TREE_SOLO(bf16, 128, 1); else if (f.rt == 2) TREE_SOLO(bf16, 64, 2); else TREE_SOLO(bf16, 64, 1); }
    } else if (f32) {
        if (wide) TREE_KEYS(float, 128, 1);
        else { if (f.rt == 2) TREE_KEYS(float, 64, 2); else TREE_KEYS(float, 64, 1); }
    } else {
        if (wide) TREE_KEYS(bf16, 128, 1);
        else { if (f.rt == 2) TREE_KEYS(bf16, 64, 2); else TREE_KEYS(bf16, 64, 1); }
    }
    if (!p.single) {
        const int rows = a->n_nodes * (a->n_head / c->n_kv_head);
        const dim3 mg(a->n, c->n_kv_head, (rows + p.merge_rows - 1) / p.merge_rows);
        if (f32) {
            if (wide) hipLaunchKernelGGL((tree_attention_merge_kernel<float, 128, 16>), mg, block, 0, st, *c, *a, p);
            else hipLaunchKernelGGL((tree_attention_merge_kernel<float, 64, 32>), mg, block, 0, st, *c, *a, p);
        } else if (f.kt == 64) {
            if (wide) hipLaunchKernelGGL((tree_attention_merge_kernel<bf16, 128, 64>), mg, block, 0, st, *c, *a, p);
            else hipLaunchKernelGGL((tree_attention_merge_kernel<bf16, 64, 64>), mg, block, 0, st, *c, *a, p);
        } else hipLaunchKernelGGL((tree_attention_merge_kernel<bf16, 128, 32>), mg, block, 0, st, *c, *a, p);
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
