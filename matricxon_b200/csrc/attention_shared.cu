// Paged attention for a step whose sequences lie in groups with their first keys in common (a system prompt, one document
// and many questions): those keys are read once for all tokens of a group.
//
// Same mathematics and visibility rule as attention.cu (query at p sees key j iff j <= p and (window == 0 or j > p - window);
// scores q.k * scale, optionally capped; float softmax, with a sink in its denominator where the caller has one). The softmax
// of a (token, head) is cut into parts over disjoint keys, each with its maximum m_i, its sum l_i of exp(score - m_i) and its
// weighted values o_i, in float:
//   shared parts   the keys below lens[sequence], through the block table of the group's first sequence (under a window through
//                  another one's where that one has given the page up: shared_prefix.cuh). The rows of an MMA
//                  tile are (token, head) pairs of the whole group, whatever sequence a token is of;
//   own parts      the keys from there on, through the sequence's own table;
//   joined         m = max m_i, w_i = exp(m_i - m), out = sum w_i o_i / (sum w_i l_i + exp(sink - m)), rounded once.
// Which kernels: bfloat16 heads of 128 on pages of 16 or 32 take tcgen05 for the shared keys (attention_tc.cu), other
// bfloat16 heads of 64 and 128 mma.sync (attention_mma.cu), whose tiles of 16 or 64 rows also walk the own keys; everything
// else (float, other head sizes) the kernel below, tiles of sixteen rows on the FP32 cores.
// The two halves run at a time: the kernel of the shared keys waits for the queries and lets that of the own keys begin at
// once, beside it; that one ends only when the first has, so the join waits for both.
// Rows behind the last sequence's are read and written by nobody.
#include <math.h>

#include "common.cuh"
#include "shared_prefix.cuh"

namespace {

constexpr int SH_THREADS = 128;
constexpr int SH_WARPS = SH_THREADS / 32;
constexpr int SH_KEYS = 32;                // keys a chunk, one a lane
constexpr int SH_ROWS = 16;                // (token, head) rows a block
constexpr int SH_ROWS_PER_WARP = SH_ROWS / SH_WARPS;

struct SharedAttnParams {
    const void *q, *cache;
    float *part_o, *part_ml;
    const int *block_tables, *cu_q, *context_lens;
    int* status;
    long long n_pages;
    int q_stride, bt_stride, n_tokens, n_heads, n_kv_heads, group, head_dim, page_size, window, n_splits, part;
    float scale, softcap;
    SharedPrefixParams shared;
};

template <typename T> struct Vec16;        // 16 bytes of T
template <> struct Vec16<float> { static constexpr int E = 4; };
template <> struct Vec16<__nv_bfloat16> { static constexpr int E = 8; };

template <typename T>
__device__ __forceinline__ void unpack16(const uint4& raw, float* f);
template <>
__device__ __forceinline__ void unpack16<float>(const uint4& raw, float* f) {
    f[0] = __uint_as_float(raw.x); f[1] = __uint_as_float(raw.y);
    f[2] = __uint_as_float(raw.z); f[3] = __uint_as_float(raw.w);
}
template <>
__device__ __forceinline__ void unpack16<__nv_bfloat16>(const uint4& raw, float* f) {
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

// Sixteen bytes on their way to shared memory; zeros where `there` is false (nothing is read then).
__device__ __forceinline__ void copy16(void* dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"((unsigned)__cvta_generic_to_shared(dst)), "l"(src),
                 "r"(there ? 16 : 0)
                 : "memory");
}

// SHARED: a tile is sixteen (token, head) rows of a group, token-major. Otherwise up to sixteen heads of one token.
// Two stages: a chunk's keys [key][dim] and values [dim][key], as they lie in the pages, are on their way while the chunk
// before is computed on. Both are kept with their 16-byte pieces swizzled, so that 32 lanes on 32 keys (scores) and on 32
// dimensions (values) meet no bank twice.
template <typename T, int SLOTS, bool SHARED>
__global__ void __launch_bounds__(SH_THREADS)
shared_simt_kernel(const SharedAttnParams p) {
    constexpr int E = Vec16<T>::E;
    constexpr int RUNS = SH_KEYS / E;                         // 16-byte pieces of a dimension's values
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ int row_token[SH_ROWS], row_head[SH_ROWS], row_lo[SH_ROWS], row_hi[SH_ROWS];
    __shared__ float row_alpha[SH_ROWS], row_m[SH_ROWS], row_l[SH_ROWS];
    const int hd = p.head_dim, cpr = hd / E;                  // 16-byte pieces of a key
    const int swz_mask = (cpr % 8 == 0) ? 7 : (cpr % 4 == 0 ? 3 : (cpr % 2 == 0 ? 1 : 0));
    float* q_s = reinterpret_cast<float*>(smem_raw);          // [SH_ROWS][hd]
    float* p_s = q_s + SH_ROWS * hd;                          // [SH_ROWS][SH_KEYS]
    uint4* stages = reinterpret_cast<uint4*>(p_s + SH_ROWS * SH_KEYS);
    const int stage_pieces = SH_KEYS * cpr + hd * RUNS;       // keys, then values
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int kh = blockIdx.y, split = blockIdx.z;

    if (SHARED || !p.shared.beside) pdl_wait();
    pdl_trigger();
    int seq = 0, rows = 0, first_token = 0, first_row = 0;
    SharedPages group_pages;                                  // SHARED
    if (SHARED) {
        const GroupTile found = find_group_tile(p.shared, p.cu_q, blockIdx.x, SH_ROWS, p.group, lane);
        if (found.tokens <= 0) return;
        seq = found.seq; first_token = found.q_start; first_row = found.first;
        rows = min(SH_ROWS, found.tokens * p.group - first_row);
        group_pages = shared_pages_of(p.shared, found, p.block_tables, p.bt_stride, p.cu_q, p.context_lens, p.page_size, p.window);
    } else {
        const int parts = (p.group + SH_ROWS - 1) / SH_ROWS;
        first_token = blockIdx.x / parts;
        first_row = (blockIdx.x - first_token * parts) * SH_ROWS;
        rows = min(SH_ROWS, p.group - first_row);
        seq = first_token < p.cu_q[p.shared.n_seqs] ? p.shared.tok_seq[first_token] : -1;
        if (seq < 0 || seq >= p.shared.n_seqs) {
            wait_for_shared_keys();
            return;
        }
    }
    if (tid < rows) {
        const int r = first_row + tid, t = r / p.group;
        row_token[tid] = first_token + t;
        row_head[tid] = kh * p.group + r - t * p.group;
        if (SHARED) {
            const KeyRange range = shared_keys_of_token(p.shared, first_token + t, p.window);
            row_lo[tid] = range.first;
            row_hi[tid] = range.last;
        } else {
            const int position = p.shared.positions[first_token];
            row_lo[tid] = max(first_visible_key(position, p.window), p.shared.lens != nullptr ? p.shared.lens[seq] : 0);
            row_hi[tid] = position;
        }
    }
    __syncthreads();
    int lo = 0x7fffffff, hi = -1;                             // the keys that any row sees
    for (int r = 0; r < rows; ++r)
        if (row_lo[r] <= row_hi[r]) { lo = min(lo, row_lo[r]); hi = max(hi, row_hi[r]); }
    const int first_chunk = hi < lo ? 0 : lo / SH_KEYS, n_chunks = hi < lo ? 0 : hi / SH_KEYS + 1 - first_chunk;
    const int per_split = (n_chunks + p.n_splits - 1) / p.n_splits;
    const int c_begin = split * per_split, c_end = min(n_chunks, c_begin + per_split);

    const int* bt = p.block_tables + (size_t)seq * p.bt_stride;
    const T* cache = reinterpret_cast<const T*>(p.cache);
    const size_t head_stride = (size_t)p.page_size * hd;
    auto bring = [&](int c) {
        uint4* k_s = stages + (size_t)(c & 1) * stage_pieces;
        uint4* v_s = k_s + SH_KEYS * cpr;
        const int c0 = (first_chunk + c) * SH_KEYS;
        // a lane looks up a key's page, for the whole warp; a run of E keys lies inside a page
        const int key = c0 + lane, lp = key / p.page_size, offset = key - lp * p.page_size, run0 = key - key % E;
        int page = -1;
        if (run0 <= hi && run0 + E - 1 >= lo) {
            if (SHARED) page = shared_page(group_pages, lp);
            else if (lp < p.bt_stride) page = bt[lp];
            if (page < 0 || page >= p.n_pages) {
                if (key >= lo && key <= hi && !(SHARED && page == PAGE_UNSEEN)) atomicOr(p.status, MX_STATUS_BAD_PAGE);
                page = -1;
            }
        }
        // a warp a key
#pragma unroll
        for (int i = 0; i < SH_KEYS / SH_WARPS; ++i) {
            const int j = warp + i * SH_WARPS, pg = __shfl_sync(0xffffffffu, page, j), off = __shfl_sync(0xffffffffu, offset, j);
            const bool there = pg >= 0 && c0 + j >= lo && c0 + j <= hi;
            const T* from = cache + ((size_t)max(pg, 0) * 2 * p.n_kv_heads + kh) * head_stride + (size_t)off * hd;
            for (int piece = lane; piece < cpr; piece += 32)
                copy16(&k_s[j * cpr + (piece ^ (j & swz_mask))], there ? from + (size_t)piece * E : cache, there);
        }
        // a thread keeps to one run of keys and walks the dimensions
        const int run = tid % RUNS, pg = __shfl_sync(0xffffffffu, page, run * E), off = __shfl_sync(0xffffffffu, offset, run * E);
        const T* from = cache + ((size_t)max(pg, 0) * 2 * p.n_kv_heads + p.n_kv_heads + kh) * head_stride + off;
#pragma unroll 4
        for (int d = tid / RUNS; d < hd; d += SH_THREADS / RUNS)
            copy16(&v_s[d * RUNS + (run ^ (d & (RUNS - 1)))], pg >= 0 ? from + (size_t)d * p.page_size : cache, pg >= 0);
    };
    // the queries and the first keys set out together
    float query[SH_ROWS_PER_WARP][8];
#pragma unroll
    for (int i = 0; i < SH_ROWS_PER_WARP; ++i) {
        const int r = warp + i * SH_WARPS;
        const T* from = reinterpret_cast<const T*>(p.q) + (r < rows ? (size_t)row_token[r] * p.q_stride + (size_t)row_head[r] * hd : 0);
#pragma unroll
        for (int j = 0; j < 8; ++j) query[i][j] = r < rows && lane + 32 * j < hd ? to_float(from[lane + 32 * j]) : 0.f;
    }
    if (c_begin < c_end) bring(c_begin);
    asm volatile("cp.async.commit_group;\n" ::: "memory");

#pragma unroll
    for (int i = 0; i < SH_ROWS_PER_WARP; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (warp + i * SH_WARPS < rows && lane + 32 * j < hd) q_s[(warp + i * SH_WARPS) * hd + lane + 32 * j] = query[i][j];
    for (int i = rows * SH_KEYS + tid; i < SH_ROWS * SH_KEYS; i += SH_THREADS) p_s[i] = 0.f;
    if (tid < SH_ROWS) row_alpha[tid] = 1.f;
    float acc[SH_ROWS][SLOTS];
#pragma unroll
    for (int r = 0; r < SH_ROWS; ++r)
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) acc[r][s] = 0.f;
    float m_run[SH_ROWS_PER_WARP], l_run[SH_ROWS_PER_WARP];
#pragma unroll
    for (int i = 0; i < SH_ROWS_PER_WARP; ++i) { m_run[i] = -INFINITY; l_run[i] = 0.f; }

    for (int c = c_begin; c < c_end; ++c) {
        const int c0 = (first_chunk + c) * SH_KEYS;
        const uint4* k_s = stages + (size_t)(c & 1) * stage_pieces;
        uint4* v_s = const_cast<uint4*>(k_s) + SH_KEYS * cpr;
        if (c + 1 < c_end) bring(c + 1);
        asm volatile("cp.async.commit_group;\ncp.async.wait_group 1;\n" ::: "memory");
        __syncthreads();
        // ---- scores: a lane a key, this warp's rows are warp, warp + 4, ...
        float s[SH_ROWS_PER_WARP];
#pragma unroll
        for (int i = 0; i < SH_ROWS_PER_WARP; ++i) s[i] = 0.f;
#pragma unroll 4
        for (int piece = 0; piece < cpr; ++piece) {
            float kf[E];
            unpack16<T>(k_s[lane * cpr + (piece ^ (lane & swz_mask))], kf);
#pragma unroll
            for (int i = 0; i < SH_ROWS_PER_WARP; ++i) {
                const int r = warp + i * SH_WARPS;
                if (r < rows) {
                    const float4* qv = reinterpret_cast<const float4*>(q_s + r * hd + piece * E);
#pragma unroll
                    for (int e4 = 0; e4 < E / 4; ++e4) {
                        const float4 qq = qv[e4];
                        s[i] = fmaf(qq.x, kf[4 * e4 + 0], s[i]);
                        s[i] = fmaf(qq.y, kf[4 * e4 + 1], s[i]);
                        s[i] = fmaf(qq.z, kf[4 * e4 + 2], s[i]);
                        s[i] = fmaf(qq.w, kf[4 * e4 + 3], s[i]);
                    }
                }
            }
        }
        const int key = c0 + lane;
#pragma unroll
        for (int i = 0; i < SH_ROWS_PER_WARP; ++i) {
            const int r = warp + i * SH_WARPS;
            if (r < rows) {
                const bool valid = key >= row_lo[r] && key <= row_hi[r];
                float sv = s[i] * p.scale;
                if (p.softcap > 0.f) sv = p.softcap * tanhf(sv / p.softcap);
                sv = valid ? sv : -INFINITY;
                const float m_new = fmaxf(m_run[i], warp_max(sv));
                const float pj = valid ? expf(sv - m_new) : 0.f;
                const float alpha = m_run[i] == -INFINITY ? 0.f : expf(m_run[i] - m_new);
                l_run[i] = l_run[i] * alpha + warp_sum(pj);
                m_run[i] = m_new;
                p_s[r * SH_KEYS + lane] = pj;
                if (lane == 0) row_alpha[r] = alpha;
            }
        }
        if (c0 < lo || c0 + SH_KEYS - 1 > hi) {
            // slots that no row sees may hold anything (0 times NaN)
            T* v_t = reinterpret_cast<T*>(v_s);
            for (int d = warp; d < hd; d += SH_WARPS) {
                const int run = lane / E;
                if (c0 + lane < lo || c0 + lane > hi)
                    v_t[(size_t)(d * RUNS + (run ^ (d & (RUNS - 1)))) * E + lane % E] = from_float<T>(0.f);
            }
        }
        __syncthreads();
        // ---- weighted values: a thread a dimension (or two), all rows
#pragma unroll
        for (int slot = 0; slot < SLOTS; ++slot) {
            const int d = tid + slot * SH_THREADS;
            if (d < hd) {
#pragma unroll
                for (int r = 0; r < SH_ROWS; ++r) acc[r][slot] *= row_alpha[r];
#pragma unroll 2
                for (int run = 0; run < RUNS; ++run) {
                    float v[E];
                    unpack16<T>(v_s[d * RUNS + (run ^ (d & (RUNS - 1)))], v);
#pragma unroll
                    for (int r0 = 0; r0 < SH_ROWS; r0 += 4) {
                        if (r0 >= rows) break;               // rows of a started four that are none have weights of zero
#pragma unroll
                        for (int r = r0; r < r0 + 4; ++r) {
                            const float4* pp = reinterpret_cast<const float4*>(p_s + r * SH_KEYS + run * E);
#pragma unroll
                            for (int e4 = 0; e4 < E / 4; ++e4) {
                                const float4 w = pp[e4];
                                acc[r][slot] = fmaf(w.w, v[4 * e4 + 3], fmaf(w.z, v[4 * e4 + 2],
                                               fmaf(w.y, v[4 * e4 + 1], fmaf(w.x, v[4 * e4], acc[r][slot]))));
                            }
                        }
                    }
                }
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < SH_ROWS_PER_WARP; ++i) {
        const int r = warp + i * SH_WARPS;
        if (r < rows && lane == 0) { row_m[r] = m_run[i]; row_l[r] = l_run[i]; }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < SH_ROWS; ++r)
        if (r < rows) {
            const size_t base = ((size_t)row_token[r] * p.n_heads + row_head[r]) * p.shared.n_parts + p.part + split;
#pragma unroll
            for (int slot = 0; slot < SLOTS; ++slot) {
                const int d = tid + slot * SH_THREADS;
                if (d < hd) p.part_o[base * hd + d] = acc[r][slot];
            }
            if (tid == 0) { p.part_ml[base * 2] = row_m[r]; p.part_ml[base * 2 + 1] = row_l[r]; }
        }
    if (!SHARED) wait_for_shared_keys();
}

// The join: a warp a (token, head), four dimensions a lane. A token of no sequence is left alone. So is one whose parts nobody
// wrote, which is reported: a token that is not its sequence's (by the sequences' starts), whose sequence is not in one group
// (none, or groups that overlap), or that does not fit its sequence's narrow tile; where groups overlap so far that they have
// more tokens than there are, some tiles of the shared keys found no block, and all rows are. The lists are read before the
// wait: the kernels before this one have waited for what wrote them, and this one begins after that (from L2, where it is then).
constexpr int JOIN_WARPS = 4;
template <typename T>
__global__ void __launch_bounds__(JOIN_WARPS * 32)
shared_join_kernel(const float* part_o, const float* part_ml, T* out, int out_stride, const int* cu_q, const float* sink,
                   int n_heads, int head_dim, long long n_pairs, int tile_tokens, const SharedPrefixParams shared, int* status) {
    pdl_trigger();
    const long long pair = (long long)blockIdx.x * JOIN_WARPS + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const int token = (int)(min(pair, n_pairs - 1) / n_heads), head = (int)(pair - (long long)token * n_heads);
    const int rows = __ldcg(cu_q + shared.n_seqs), seq = __ldcg(shared.tok_seq + token);
    bool written = seq >= 0 && seq < shared.n_seqs;
    if (written) {
        const int start = __ldcg(cu_q + seq), end = __ldcg(cu_q + seq + 1);
        written = start >= 0 && token >= start && token < end && token - start < tile_tokens;
    }
    if (shared.n_shared_parts > 0) {
        auto start_of = [&](int g) { return min(max(__ldcg(shared.first + g), 0), shared.n_seqs); };
        bool rises = true;
        for (int g = threadIdx.x; g < shared.n_groups; g += JOIN_WARPS * 32) rises = rises && start_of(g) <= start_of(g + 1);
        if (__syncthreads_and(rises)) {
            written = written && seq >= start_of(0) && seq < start_of(shared.n_groups);
        } else {
            // groups that overlap, or a list that is filled up with anything that gives no group
            unsigned groups = 0, tokens = 0;           // (a lane's tokens stop counting where they are too many)
            for (int g = lane; g < shared.n_groups; g += 32) {
                const int first = start_of(g), end = start_of(g + 1);
                if (first >= end) continue;
                groups += seq >= first && seq < end;
                tokens = min(tokens + max(min(__ldcg(cu_q + end), shared.n_tokens) - max(__ldcg(cu_q + first), 0), 0), 0x7fffffffu);
            }
            const long long all = (long long)__reduce_add_sync(0xffffffffu, tokens & 0xffffu) + ((long long)__reduce_add_sync(0xffffffffu, tokens >> 16) << 16);
            written = written && __reduce_add_sync(0xffffffffu, groups) == 1u && all <= shared.n_tokens;
        }
    }
    pdl_wait();
    if (pair >= n_pairs) return;
    part_o = after_wait(part_o);
    part_ml = after_wait(part_ml);
    if (rows > shared.n_tokens && pair == 0 && lane == 0) atomicOr(status, MX_STATUS_BAD_STEP);
    if (token >= rows) return;
    if (!written) {
        if (lane == 0) atomicOr(status, MX_STATUS_BAD_STEP);
        return;
    }
    const size_t base = (size_t)pair * shared.n_parts;
    float m = -INFINITY;
    for (int s = lane; s < shared.n_parts; s += 32) m = fmaxf(m, part_ml[(base + s) * 2]);
    m = warp_max(m);
    float total = 0.f;
    float4 o[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    for (int s0 = 0; s0 < shared.n_parts; s0 += 32) {
        const int s = s0 + lane;
        const float2 ml = s < shared.n_parts ? *reinterpret_cast<const float2*>(part_ml + (base + s) * 2) : make_float2(-INFINITY, 0.f);
        const float weight = ml.x == -INFINITY ? 0.f : expf(ml.x - m);
        total += warp_sum(ml.y * weight);
        for (int j = 0; j < min(32, shared.n_parts - s0); ++j) {
            const float w = __shfl_sync(0xffffffffu, weight, j);
            if (w == 0.f) continue;                // a part without keys has values nobody wrote
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int d = 4 * lane + 128 * i;
                if (d < head_dim) {
                    const float4 v = *reinterpret_cast<const float4*>(part_o + (base + s0 + j) * head_dim + d);
                    o[i].x = fmaf(v.x, w, o[i].x); o[i].y = fmaf(v.y, w, o[i].y);
                    o[i].z = fmaf(v.z, w, o[i].z); o[i].w = fmaf(v.w, w, o[i].w);
                }
            }
        }
    }
    if (sink) total += expf(sink[head] - m);
    const float inv = 1.f / total;
    T* dst = out + (size_t)token * out_stride + (size_t)head * head_dim;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int d = 4 * lane + 128 * i;
        if (d < head_dim) {
            dst[d] = from_float<T>(o[i].x * inv); dst[d + 1] = from_float<T>(o[i].y * inv);
            dst[d + 2] = from_float<T>(o[i].z * inv); dst[d + 3] = from_float<T>(o[i].w * inv);
        }
    }
}

template <typename T, int SLOTS, bool SHARED>
int launch_simt(const SharedAttnParams& p, unsigned n_tiles, cudaStream_t stream) {
    const size_t smem = (size_t)SH_ROWS * p.head_dim * 4 + SH_ROWS * SH_KEYS * 4 + 4 * (size_t)SH_KEYS * p.head_dim * sizeof(T);
    if (smem > 47 * 1024 && cudaFuncSetAttribute(shared_simt_kernel<T, SLOTS, SHARED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 (int)smem) != cudaSuccess)
        MX_REFUSE("attention over shared keys: cannot reserve %zu bytes of shared memory", smem);
    const dim3 grid(n_tiles, p.n_kv_heads, p.n_splits);
    const cudaError_t e = !SHARED && p.shared.beside
                              ? mx_launch_beside(shared_simt_kernel<T, SLOTS, SHARED>, grid, dim3(SH_THREADS), smem, stream, p)
                              : mx_launch_chained(shared_simt_kernel<T, SLOTS, SHARED>, grid, dim3(SH_THREADS), smem, stream, p);
    if (e != cudaSuccess) {
        mx_set_error("attention over shared keys: launch failed: %s", cudaGetErrorString(e));
        return (int)e;
    }
    return MX_OK;
}

template <typename T>
int launch_join(const SharedAttnParams& p, T* out, int out_stride, const float* sink, int tile_tokens, cudaStream_t stream) {
    const long long pairs = (long long)p.n_tokens * p.n_heads;
    const cudaError_t e = mx_launch_beside(shared_join_kernel<T>, dim3((unsigned)((pairs + JOIN_WARPS - 1) / JOIN_WARPS)),
                                           dim3(JOIN_WARPS * 32), 0, stream, (const float*)p.part_o, (const float*)p.part_ml, out, out_stride,
                                           p.cu_q, sink, p.n_heads, p.head_dim, pairs, tile_tokens, p.shared, p.status);
    if (e != cudaSuccess) {
        mx_set_error("attention over shared keys: launch failed: %s", cudaGetErrorString(e));
        return (int)e;
    }
    return MX_OK;
}

// How the launch is cut up. tcgen05 tiles, mma tiles or the FP32 cores (`path` 2, 1, 0), the most tiles there can be of either
// kind, and into how many parts the shared and the own keys of a tile are dealt out.
struct SharedPlan {
    int path, shared_tiles, own_tiles, shared_parts, own_parts;
    bool narrow;
};

// The number of parts, at most 32, that `blocks` blocks of `chunks` chunks each are cut into. `start`: what a block costs beside
// its chunks, in chunks. `uneven`: the blocks' chunks differ, up to that many; they then go on one after another, half as long
// on the average.
int best_parts(long long blocks, int chunks, int room, int start, int uneven) {
    int best = 1;
    long long least = 0;
    for (int parts = 1; parts <= 32 && parts <= chunks; ++parts) {
        const int each = (chunks + parts - 1) / parts;
        const long long rounds = (blocks * parts + room - 1) / room;
        const long long cost = uneven ? blocks * parts * (each / 2 + start) / room + each + start : rounds * (each + start);
        if (parts == 1 || cost < least) { best = parts; least = cost; }
    }
    return best;
}

// Parts of the shared keys on tcgen05, a block an SM. The own keys' blocks, which are bound by memory, find no room beside one of
// these, so the parts also say how many SMs are left to them while these run: the two should end together. Of 128 requests on
// 32,768 shared keys and up to 2,048 own ones (32 tiles of heads) 1, 2, 3, 4 and 8 parts took 320, 164, 182, 189 and 199 us; of 32
// on 2,048 and 3,000 under a window (12) 2, 4, 8 and 11 took 37, 40, 44 and 45. As measured there, a tile of 128 keys takes 1.15 us,
// a block's start and end four of them, an SM takes 2.7 chunks of 32 own keys a us and the memory 330.
int balanced_parts(long long blocks, int chunks, int n_sm, double own_work, double join_us) {
    int best = 1;
    double least = 0.0;
    for (int parts = 1; parts <= 32 && parts <= chunks; ++parts) {
        const long long rounds = (blocks * parts + n_sm - 1) / n_sm;
        const double busy = 1.15 * rounds * ((chunks + parts - 1) / parts + 4), left = rounds == 1 ? (double)(n_sm - blocks * parts) : 0.0;
        const double memory = 330.0 * n_sm / 148.0, beside = busy * (2.7 * left < memory ? 2.7 * left : memory);
        const double time = busy + (own_work > beside ? (own_work - beside) / memory : 0.0) + join_us * parts;
        if (parts == 1 || time < least) { best = parts; least = time; }
    }
    return best;
}

SharedPlan make_plan(int dtype, int head_dim, int page_size, bool aligned, int n_tokens, int n_heads, int n_kv_heads, int n_seqs,
                     int n_groups, int max_q_len, int max_shared_len, int max_own_len, int n_sm) {
    SharedPlan plan;
    const int group = n_heads / n_kv_heads;
    const bool mma = dtype == MX_DTYPE_BF16 && aligned && (head_dim == 64 || head_dim == 128) &&
                     (page_size == 8 || page_size == 16 || page_size == 32);
    const bool tc = mma && head_dim == 128 && page_size != 8 && group <= 128;
    plan.path = tc ? 2 : (mma ? 1 : 0);
    const long long rows = (long long)n_tokens * group;
    plan.narrow = mma && (long long)max_q_len * group <= 16;
    const int shared_rows = tc ? 128 / group * group : (mma ? 64 : SH_ROWS);
    plan.shared_tiles = (int)min(rows / shared_rows + n_groups, rows);
    plan.own_tiles = mma ? (plan.narrow ? n_seqs : (int)min(rows / 64 + n_seqs, rows)) : n_tokens * ((group + SH_ROWS - 1) / SH_ROWS);
    // Parts: blocks run in rounds of as many as fit the GPU (narrow tiles two an SM, the others but tcgen05 three), and a round
    // takes as long as a block's chunks and its start. The number of parts with the shortest rounds is taken; the tiles of a
    // group each end in the middle of one, so there may be a tile a group more.
    const int shared_chunks = (max(max_shared_len, 1) + (tc ? 127 : 31)) / (tc ? 128 : 32), own_chunks = max(max_own_len, 1) / 32 + 1;
    const long long shared_blocks = (rows + shared_rows - 1) / shared_rows * n_kv_heads, own_blocks = (long long)plan.own_tiles * n_kv_heads;
    const int own_unit = plan.narrow ? 3 : (mma ? 2 : 1);       // chunks that a block takes at a time
    plan.own_parts = best_parts(own_blocks, (own_chunks + own_unit - 1) / own_unit, plan.narrow ? 2 * n_sm : 3 * n_sm, 3, 1);
    // the join reads and writes a part's values, float, at some 5 TB/s; own lengths are taken to be half the longest
    const double join_us = (double)n_tokens * n_heads * head_dim * 8.0 / 5e6, own_work = (double)own_blocks * own_chunks / 2.0;
    plan.shared_parts = max_shared_len <= 0 ? 0
                        : tc ? balanced_parts(shared_blocks, shared_chunks, n_sm, own_work, join_us)
                             : best_parts(shared_blocks, shared_chunks, 3 * n_sm, 8, 0);
    return plan;
}

bool rows_aligned(const void* q, int q_stride, const void* cache) {
    return q_stride % 8 == 0 && ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache)) & 15) == 0;
}

}  // namespace

int mx_attention_tc_shared(const void* q, int q_stride, const void* cache, long long n_pages, int page_size,
                           const int* block_tables, int bt_stride, const int* cu_q, const int* context_lens, int n_tokens,
                           int n_heads, int n_kv_heads, int window, float scale, float softcap, int n_tiles, int n_splits, float* part_o, float* part_ml,
                           const SharedPrefixParams& shared, int* status, cudaStream_t stream);
int mx_attention_mma_shared(const void* q, int q_stride, const void* cache, long long n_pages, int page_size,
                            const int* block_tables, int bt_stride, const int* cu_q, const int* context_lens, int n_heads,
                            int n_kv_heads, int head_dim, int window, float scale, float softcap, bool shared_keys, bool narrow,
                            int n_tiles, int n_splits, int part, float* part_o, float* part_ml,
                            const SharedPrefixParams& shared, int* status, cudaStream_t stream);

// Bytes of scratch of mx_paged_attention_shared with the same arguments: the parts' values, maxima and sums. `aligned`: the
// query rows and the pages start on 16 bytes.
extern "C" long long mx_attention_shared_scratch(int dtype, int aligned, int page_size, int n_seqs, int n_groups, int n_tokens,
                                                 int n_heads, int n_kv_heads, int head_dim, int max_q_len, int max_shared_len,
                                                 int max_own_len, int n_sm) {
    if (n_tokens <= 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0 || head_dim <= 0 || n_sm <= 0) return 0;
    const SharedPlan plan = make_plan(dtype, head_dim, page_size, aligned != 0, n_tokens, n_heads, n_kv_heads, n_seqs, n_groups,
                                      max_q_len, max_shared_len, max_own_len, n_sm);
    return (long long)n_tokens * n_heads * (plan.shared_parts + plan.own_parts) * (head_dim + 2) * (long long)sizeof(float);
}

// max_q_len: no sequence brings more tokens. max_shared_len and max_own_len size the parts alone: smaller numbers than the true
// ones cost time, not results (with max_shared_len 0 every key is read through its sequence's own table).
extern "C" int mx_paged_attention_shared(const void* q, int dtype, int q_stride, const void* cache, long long n_pages,
                                         int page_size, const int* block_tables, int bt_stride, const int* cu_q,
                                         const int* context_lens, const int* tok_seq, const int* positions, const int* first,
                                         const int* lens, int n_seqs, int n_groups, int n_tokens, int n_heads, int n_kv_heads,
                                         int head_dim, int window, float scale, float softcap, const float* sink, void* out,
                                         int out_stride, int max_q_len, int max_shared_len, int max_own_len, int n_sm,
                                         float* scratch, int* status, cudaStream_t stream) {
    if (n_tokens <= 0 || n_seqs <= 0) return MX_OK;
    if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0)
        MX_REFUSE("attention: %d heads are not a multiple of %d kv heads", n_heads, n_kv_heads);
    if (head_dim % 16 != 0 || head_dim < 16 || head_dim > 256)
        MX_REFUSE("attention: head_dim %d is not a multiple of 16 in [16, 256]", head_dim);
    if (page_size <= 0 || page_size % 8 != 0) MX_REFUSE("attention: page size %d is not a positive multiple of 8", page_size);
    if (n_kv_heads > 65535) MX_REFUSE("attention: %d kv heads exceed the grid", n_kv_heads);
    if (max_q_len <= 0 || max_shared_len < 0 || max_own_len < 0 || n_sm <= 0)
        MX_REFUSE("attention over shared keys: bounds of %d tokens, %d and %d keys", max_q_len, max_shared_len, max_own_len);
    if ((long long)n_tokens * n_heads > 0x7fffffffLL) MX_REFUSE("attention over shared keys: %d tokens of %d heads", n_tokens, n_heads);
    if (n_pages * 2 * n_kv_heads > 0x7fffffffLL) MX_REFUSE("attention over shared keys: %lld pages are too many", n_pages);
    if (reinterpret_cast<uintptr_t>(cache) % 16 != 0) MX_REFUSE("attention over shared keys needs 16-byte aligned pages");
    if (scratch == nullptr || status == nullptr) MX_REFUSE("attention over shared keys needs scratch memory and a status word");
    const SharedPlan plan = make_plan(dtype, head_dim, page_size, rows_aligned(q, q_stride, cache), n_tokens, n_heads, n_kv_heads,
                                      n_seqs, n_groups, max_q_len, max_shared_len, max_own_len, n_sm);
    SharedAttnParams p;
    p.q = q; p.cache = cache; p.block_tables = block_tables; p.cu_q = cu_q; p.context_lens = context_lens; p.status = status; p.n_pages = n_pages;
    p.q_stride = q_stride; p.bt_stride = bt_stride; p.n_tokens = n_tokens; p.n_heads = n_heads; p.n_kv_heads = n_kv_heads;
    p.group = n_heads / n_kv_heads; p.head_dim = head_dim; p.page_size = page_size; p.window = window; p.scale = scale;
    p.softcap = softcap;
    p.shared.first = first; p.shared.lens = lens; p.shared.tok_seq = tok_seq; p.shared.positions = positions;
    p.shared.n_groups = n_groups; p.shared.n_seqs = n_seqs; p.shared.n_tokens = n_tokens; p.shared.n_shared_parts = plan.shared_parts;
    p.shared.n_parts = plan.shared_parts + plan.own_parts;
    p.shared.beside = 0;
    if (plan.shared_parts == 0) p.shared.lens = nullptr;
    p.part_o = scratch;
    p.part_ml = scratch + (size_t)n_tokens * n_heads * p.shared.n_parts * head_dim;
    int rc = MX_OK;
    if (plan.shared_parts > 0) {
        if (plan.path == 2) {
            rc = mx_attention_tc_shared(q, q_stride, cache, n_pages, page_size, block_tables, bt_stride, cu_q, context_lens,
                                        n_tokens, n_heads, n_kv_heads, window, scale, softcap, plan.shared_tiles, plan.shared_parts,
                                        p.part_o, p.part_ml, p.shared, status, stream);
        } else if (plan.path == 1) {
            rc = mx_attention_mma_shared(q, q_stride, cache, n_pages, page_size, block_tables, bt_stride, cu_q, context_lens,
                                         n_heads, n_kv_heads, head_dim, window, scale, softcap, true, false, plan.shared_tiles,
                                         plan.shared_parts, 0, p.part_o, p.part_ml, p.shared, status, stream);
        } else {
            p.n_splits = plan.shared_parts;
            p.part = 0;
            if (dtype == MX_DTYPE_F32)
                rc = head_dim > SH_THREADS ? launch_simt<float, 2, true>(p, plan.shared_tiles, stream)
                                           : launch_simt<float, 1, true>(p, plan.shared_tiles, stream);
            else
                rc = head_dim > SH_THREADS ? launch_simt<__nv_bfloat16, 2, true>(p, plan.shared_tiles, stream)
                                           : launch_simt<__nv_bfloat16, 1, true>(p, plan.shared_tiles, stream);
        }
        if (rc != MX_OK) return rc;
        p.shared.beside = 1;
    }
    if (plan.path > 0) {
        rc = mx_attention_mma_shared(q, q_stride, cache, n_pages, page_size, block_tables, bt_stride, cu_q, context_lens, n_heads,
                                     n_kv_heads, head_dim, window, scale, softcap, false, plan.narrow, plan.own_tiles, plan.own_parts,
                                     plan.shared_parts, p.part_o, p.part_ml, p.shared, status, stream);
    } else {
        p.n_splits = plan.own_parts;
        p.part = plan.shared_parts;
        if (dtype == MX_DTYPE_F32)
            rc = head_dim > SH_THREADS ? launch_simt<float, 2, false>(p, plan.own_tiles, stream)
                                       : launch_simt<float, 1, false>(p, plan.own_tiles, stream);
        else
            rc = head_dim > SH_THREADS ? launch_simt<__nv_bfloat16, 2, false>(p, plan.own_tiles, stream)
                                       : launch_simt<__nv_bfloat16, 1, false>(p, plan.own_tiles, stream);
    }
    if (rc != MX_OK) return rc;
    // tokens of a sequence that its tile of the own keys has room for
    const int tile_tokens = plan.narrow ? 16 / p.group : 0x7fffffff;
    if (dtype == MX_DTYPE_F32) return launch_join<float>(p, (float*)out, out_stride, sink, tile_tokens, stream);
    return launch_join<__nv_bfloat16>(p, (__nv_bfloat16*)out, out_stride, sink, tile_tokens, stream);
}
