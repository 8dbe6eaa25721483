// The metadata of one step, laid out on the GPU from the requests' lengths: positions, sequence numbers and cache slots of
// its token rows, where each sequence's rows begin, and the block tables its attention reads.
//
// Sequence s brings q[s] tokens after context[s] cached ones. Its pages stand in row rows[s] of `tables`, which live on the
// device from step to step. With pages of P positions it holds have = ceil(context / P) pages and takes
// need = ceil((context + q) / P) - have more from `free_pages`, in the order of the sequences:
//   cu_q = running sum of q, base = running sum of need
//   page(s, k) = tables[shared_rows[s]][k]       k < shared_pages[s]: read through another request's row (where that request
//                                                takes its page k in this very step, that page: the row is being written then)
//                tables[rows[s]][k]              k < have
//                free_pages[base[s] + k - have]  k < have + need; also stored in tables[rows[s]][k]
//   row cu_q[s] + i: position context + i, slot page(position / P) * P + position % P
// Entries of the step's block table beyond the last page are -1, and so are those that no query of this step or a later one
// sees (first_visible_key(context) and the kept first positions, the rule by which the cache manager gives pages back).
// Rows of the buffers behind the last token get position 0, sequence -1, slot -1. Nothing that the results depend on is
// changed (lengths, free pages), so a step can be laid out twice.
//
// Every block adds up all sequences' lengths for itself (a sequence a thread, 8 to 20 bytes each out of L2), which spares a
// second launch or a wait between blocks; it then lays out its few sequences. On the way it notes for each row what its sequence
// holds (of more than 4,096 rows, a bit): where two meet, the sequences are compared one by one, and those whose row an earlier
// one has bring nothing, take nothing and are reported. Whoever reads pages through another row finds there how many of them are
// in the row before this step (looked up by a pass over all sequences instead: 5.2 and 12.5 us where these take 4.4 and 10.9, 64
// sequences and 1,024). A step that does not fit (more rows than the
// buffers hold, more pages than there are, a length out of range) sets MX_STATUS_BAD_STEP and every block leaves an empty step:
// all -1, nothing taken, `tables` as they were.
// The launch after this one must not begin early: attention kernels read tables and lengths before they wait for what ran
// before them, so this kernel never lets its successor start (no pdl_trigger).
#include "common.cuh"

namespace {

constexpr int ST_THREADS = 512;
constexpr int ST_OWN = 64;              // sequences a block lays out, at most
constexpr int ST_AHEAD = 8;
constexpr int ST_SLICE = 16384;         // block-table entries of a sequence that one block writes
// Notes on rows: word r says 1 + the pages held by the sequence of row r (ST_IDLE: one that brings nothing), 0 if there is none; of
// more rows, row r is bit r / ST_MARKS % 32 of word r % ST_MARKS.
constexpr int ST_MARKS = 4096;
constexpr unsigned ST_IDLE = 0x7fffffffu;

struct StepTablesParams {
    const int *q_lens, *context_lens, *rows, *shared_rows, *shared_pages, *free_pages, *n_free;
    int* tables;
    int *positions, *tok_seq, *cu_q, *slots, *block_tables, *taken, *status;
    int n_seqs, n_tokens, n_rows, width, page_size, n_pages, n_free_most, window, keep_first, per_block;
};

struct Sequence {
    int q, context, row, shared_row, shared;      // shared: pages
    int have, need, seen_from;                    // pages held, taken, and the first one that the next query needs
    bool fits;                                    // its numbers are possible
};

__device__ __forceinline__ Sequence read_sequence(const StepTablesParams& p, int s) {
    Sequence v;
    v.q = p.q_lens[s];
    v.context = p.context_lens[s];
    v.row = p.rows ? p.rows[s] : s;
    v.shared_row = p.shared_rows ? p.shared_rows[s] : -1;
    v.shared = v.shared_row >= 0 ? p.shared_pages[s] : 0;
    const long long most = min((long long)p.width * p.page_size, 0x7fffffffLL);
    v.fits = v.q >= 0 && v.context >= 0 && v.row >= -1 && v.row < p.n_rows && v.shared_row < p.n_rows &&
             (long long)v.context + v.q <= most && (v.row >= 0 || v.q == 0) && v.shared >= 0 &&
             (long long)v.shared * p.page_size <= v.context;
    if (!v.fits || v.row < 0) {
        v.q = v.context = v.shared = 0;
        v.row = v.shared_row = -1;
    }
    // (sums of two numbers below 2^31 and a page fit 32 bits without a sign)
    v.have = (int)(((unsigned)v.context + (unsigned)p.page_size - 1u) / (unsigned)p.page_size);
    v.need = (int)(((unsigned)v.context + (unsigned)v.q + (unsigned)p.page_size - 1u) / (unsigned)p.page_size) - v.have;
    v.seen_from = (int)((unsigned)first_visible_key(v.context, p.window) / (unsigned)p.page_size);
    return v;
}

// What sequences bring and take: all of them, and those before a block's own.
struct StepSums {
    long long q_all;
    int q_before, need_before, need_all;                     // (before: wrong only where the step does not fit anyway)
    bool none_again;
};

__device__ __forceinline__ void add_sequence(StepSums& sums, const Sequence& v, int s, int first, int last, Sequence* own) {
    sums.q_all += v.q;
    sums.need_all += v.need;
    if (s < first) { sums.q_before += v.q; sums.need_before += v.need; }
    else if (s < last) own[s - first] = v;
}

// Whether an earlier sequence has the row of sequence s (a warp reads the rows before its sequences together, a place for all lanes).
__device__ __forceinline__ bool row_again(const StepTablesParams& p, int s, int row) {
    if (p.rows == nullptr || row < 0) return false;
    for (int earlier = 0; earlier < s; ++earlier)
        if (p.rows[earlier] == row) return true;
    return false;
}

// The two passes that a step seldom needs are functions of their own, out of every step's way (8 sequences: 4.4 us in line, 4.2 so).

// A thread's share of the sums, where a sequence whose row an earlier one has is one of nothing.
__device__ __noinline__ StepSums sums_without_repeated(const StepTablesParams& p, int first, int last, Sequence* own) {
    StepSums sums = {0, 0, 0, 0, true};
    for (int s = threadIdx.x; s < p.n_seqs; s += ST_THREADS) {
        Sequence v = read_sequence(p, s);
        if (row_again(p, s, v.row)) {
            v.q = v.context = v.shared = v.have = v.need = v.seen_from = 0;
            v.row = v.shared_row = -1;
            sums.none_again = false;
        }
        add_sequence(sums, v, s, first, last, own);
    }
    return sums;
}

// Of a sequence that reads pages through another row: the sequence of that row in this step, how many of the shared pages it
// holds, how many more it takes, and where those begin.
struct Leader {
    int seq, have, need, page;
};

// For a block's sequences whose shared pages are not all in the leader's row before this step (as far as noted).
__device__ __noinline__ void find_leaders(const StepTablesParams& p, const Sequence* own, Leader* leader, int n, bool some_again) {
    const int tid = threadIdx.x;
    for (int s = tid; s < p.n_seqs; s += ST_THREADS) {
        const int row = p.rows ? p.rows[s] : s;
        for (int i = 0; i < n; ++i)
            if (own[i].shared > leader[i].have && own[i].shared_row == row) atomicMin(&leader[i].seq, s);
    }
    __syncthreads();
    if (tid < n) {
        leader[tid].have = own[tid].shared;                  // not in the step, or idle: its row as it is
        if (leader[tid].seq < p.n_seqs) {
            const Sequence v = read_sequence(p, leader[tid].seq);
            if (v.q > 0) leader[tid].have = min(v.have, own[tid].shared);
            leader[tid].need = v.need;
        }
    }
    __syncthreads();
    for (int i = 0; i < n; ++i) {
        if (own[i].shared <= leader[i].have || leader[i].need == 0) continue;
        int before = 0;
        for (int s = tid; s < leader[i].seq; s += ST_THREADS) {
            const Sequence v = read_sequence(p, s);
            if (v.need > 0 && !(some_again && row_again(p, s, v.row))) before += v.need;
        }
        before = (int)__reduce_add_sync(0xffffffffu, (unsigned)before);
        if ((tid & 31) == 0) atomicAdd(&leader[i].page, before);
    }
    __syncthreads();
}

__global__ void __launch_bounds__(ST_THREADS) step_tables_kernel(const __grid_constant__ StepTablesParams p) {
    __shared__ long long warp_total[ST_THREADS / 32];
    __shared__ int warp_sums[3][ST_THREADS / 32];
    __shared__ unsigned marks[ST_MARKS];
    __shared__ Sequence own[ST_OWN];
    __shared__ int own_row[ST_OWN], own_page[ST_OWN];
    __shared__ Leader leader[ST_OWN];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first = blockIdx.x * p.per_block, last = min(p.n_seqs, first + p.per_block);
    const bool noted = p.n_rows <= ST_MARKS;
    for (int i = tid; i < min(p.n_rows, ST_MARKS); i += ST_THREADS) marks[i] = 0u;
    pdl_wait();

    // ---- what all sequences bring and take, and what those before this block's do
    const int n_free = min(*p.n_free, p.n_free_most);
    StepSums sums = {0, 0, 0, 0, true};
    // the threads' sums; every thread gets them, and whether all of them say `fine`
    auto add_up = [&](bool fine) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sums.q_all += __shfl_xor_sync(0xffffffffu, sums.q_all, o);
        sums.q_before = (int)__reduce_add_sync(0xffffffffu, (unsigned)sums.q_before);
        sums.need_before = (int)__reduce_add_sync(0xffffffffu, (unsigned)sums.need_before);
        sums.need_all = (int)__reduce_add_sync(0xffffffffu, (unsigned)sums.need_all);
        if (lane == 0) {
            warp_total[warp] = sums.q_all;
            warp_sums[0][warp] = sums.q_before; warp_sums[1][warp] = sums.need_before; warp_sums[2][warp] = sums.need_all;
        }
        const bool all_fine = __syncthreads_and(fine);
        sums = {0, 0, 0, 0, true};
#pragma unroll
        for (int w = 0; w < ST_THREADS / 32; ++w) {
            sums.q_all += warp_total[w];
            sums.q_before += warp_sums[0][w]; sums.need_before += warp_sums[1][w]; sums.need_all += warp_sums[2][w];
        }
        return all_fine;
    };
    bool fits = true, met = false;
    Sequence next = {};
    if (tid < p.n_seqs) next = read_sequence(p, tid);
    __syncthreads();                                         // no row is noted
    for (int s = tid; s < p.n_seqs; s += ST_THREADS) {
        const Sequence v = next;
        if (s + ST_THREADS < p.n_seqs) next = read_sequence(p, s + ST_THREADS);
        fits = fits && v.fits;
        add_sequence(sums, v, s, first, last, own);
        if (v.row >= 0) {
            const unsigned bit = 1u << (v.row / ST_MARKS & 31);
            const unsigned old = noted ? atomicExch(&marks[v.row], v.q > 0 ? 1u + v.have : ST_IDLE) : atomicOr(&marks[v.row % ST_MARKS], bit) & bit;
            met = met || old != 0u;
        }
    }
    bool all_fit = add_up(fits && !met), some_again = false;
    if (!all_fit) {
        // something is wrong, or two rows met; `fits` goes on alone
        __syncthreads();                                     // everybody has read the sums
        sums = sums_without_repeated(p, first, last, own);
        some_again = !add_up(sums.none_again);
        all_fit = __syncthreads_and(fits);
        if (some_again && blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) atomicOr(p.status, MX_STATUS_BAD_STEP);
    }
    const bool possible = all_fit && sums.q_all <= p.n_tokens && sums.need_all <= n_free;
    const int total = possible ? (int)sums.q_all : 0;
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) {
        p.cu_q[0] = 0;
        *p.taken = possible ? sums.need_all : 0;
        if (!possible) atomicOr(p.status, MX_STATUS_BAD_STEP);
    }

    // ---- this block's sequences: where each one's rows and new pages begin, then their tables' entries, all in one row
    const int mine_n = last - first;
    bool missing = false;
    if (tid < mine_n) {
        int rows_before = sums.q_before, pages_before = sums.need_before;
        for (int i = 0; i < tid; ++i) { rows_before += own[i].q; pages_before += own[i].need; }
        own_row[tid] = rows_before;
        own_page[tid] = pages_before;
        // (nothing is known of more rows, and of two sequences' row not which one noted it)
        const unsigned mark = !noted || some_again ? 1u : marks[max(own[tid].shared_row, 0)];
        const int shared = own[tid].shared, have = mark != 0u ? min(shared, (int)mark - 1) : shared;
        leader[tid] = Leader{0x7fffffff, have, 0, 0};
        missing = shared > have;
        if (blockIdx.y == 0) p.cu_q[first + tid + 1] = possible ? rows_before + own[tid].q : 0;
    }
    // shared pages that are not in the leader's row before this step: one that takes pages now stores them there meanwhile
    if (__syncthreads_or(missing) && possible) find_leaders(p, own, leader, mine_n, some_again);
    // pages that nobody sees any more lie between the kept ones and the first that the next query needs
    const int kept = p.window > 0 ? (p.keep_first + p.page_size - 1) / p.page_size : 0;
    const int k_begin = blockIdx.y * ST_SLICE, k_end = min(p.width, k_begin + ST_SLICE);
    bool bad_page = false;
    for (int i = 0; i < mine_n; ++i) {
        const Sequence v = own[i];
        const bool there = possible && v.row >= 0;
        const int end = there ? min(k_end, v.have + v.need) : 0;
        int* out = p.block_tables + (size_t)(first + i) * p.width;
        int* row = p.tables + (size_t)max(v.row, 0) * p.width;
        const int* shared = p.tables + (size_t)max(v.shared_row, 0) * p.width;
        const int* fresh = p.free_pages + own_page[i] - v.have;
        const int held = leader[i].have;          // shared pages from here on are not in the leader's row yet, or never: see below
        // eight entries a thread are asked for before one is written: the rows are read and written in one place
        for (int k0 = k_begin + tid; k0 < end; k0 += ST_AHEAD * ST_THREADS) {
            int page[ST_AHEAD];
#pragma unroll
            for (int u = 0; u < ST_AHEAD; ++u) {
                const int k = k0 + u * ST_THREADS;
                page[u] = k >= end ? -1 : (k >= v.have ? fresh[k] : (k >= v.shared ? row[k] : (k < held ? shared[k] : 0)));
            }
#pragma unroll
            for (int u = 0; u < ST_AHEAD; ++u) {
                const int k = k0 + u * ST_THREADS;
                if (k >= end) break;
                if (k >= v.have) row[k] = page[u];
                if (k >= kept && k < v.seen_from) page[u] = -1;
                else if (page[u] < 0 || page[u] >= p.n_pages) {
                    page[u] = -1;
                    bad_page = true;
                }
                out[k] = page[u];
            }
        }
#pragma unroll 8
        for (int k = max(k_begin, end) + tid; k < k_end; k += ST_THREADS) out[k] = -1;
        if (held < v.shared)                       // (each thread its own entries once more)
            for (int k = k_begin + tid; k < min(end, v.shared); k += ST_THREADS) {
                if (k < held || (k >= kept && k < v.seen_from)) continue;
                const int page = k < held + leader[i].need ? p.free_pages[leader[i].page + k - held] : -1;
                if (page < 0 || page >= p.n_pages) bad_page = true;
                out[k] = page >= 0 && page < p.n_pages ? page : -1;
            }
    }
    if (blockIdx.y == 0 && possible) {
        // their token rows, a warp a sequence of few (decoding requests), the block one of more
        auto token_rows = [&](int i, int r0, int step) {
            const Sequence& v = own[i];
            for (int r = r0; r < v.q; r += step) {
                const int position = v.context + r, k = (int)((unsigned)position / (unsigned)p.page_size);
                int slot = -1;
                const int page = k >= v.have ? p.free_pages[own_page[i] + k - v.have] : p.tables[(size_t)v.row * p.width + k];
                if (page >= 0 && page < p.n_pages) slot = page * p.page_size + position - k * p.page_size;
                else bad_page = true;
                const int t = own_row[i] + r;
                p.positions[t] = position;
                p.tok_seq[t] = first + i;
                p.slots[t] = slot;
            }
        };
        for (int i = warp; i < mine_n; i += ST_THREADS / 32)
            if (own[i].q <= 32) token_rows(i, lane, 32);
        for (int i = 0; i < mine_n; ++i)
            if (own[i].q > 32) token_rows(i, tid, ST_THREADS);
    }
    if (bad_page) atomicOr(p.status, MX_STATUS_BAD_PAGE);
    // ---- rows behind the last token
    if (blockIdx.y == 0)
        for (int t = total + blockIdx.x * ST_THREADS + tid; t < p.n_tokens; t += gridDim.x * ST_THREADS) {
            p.positions[t] = 0;
            p.tok_seq[t] = -1;
            p.slots[t] = -1;
        }
}

}  // namespace

extern "C" int mx_step_tables(const int* q_lens, const int* context_lens, const int* rows, int n_seqs, int* tables, int n_rows,
                              int width, const int* free_pages, int n_free_most, const int* n_free, int page_size,
                              long long n_pages, const int* shared_rows, const int* shared_pages, int window, int keep_first,
                              int* positions, int* tok_seq, int* cu_q, int* slots, int n_tokens, int* block_tables, int* taken,
                              int* status, cudaStream_t stream) {
    if (n_seqs <= 0) MX_REFUSE("step tables: a step of %d sequences", n_seqs);
    if (width <= 0 || n_rows <= 0 || n_tokens < 0) MX_REFUSE("step tables: %d rows of %d entries, %d tokens", n_rows, width, n_tokens);
    if (page_size <= 0) MX_REFUSE("step tables: pages of %d positions", page_size);
    if ((long long)n_seqs * width > 0x7fffffffLL || (long long)n_rows * width > 0x7fffffffffffLL) MX_REFUSE("step tables: %d tables of %d entries", n_seqs, width);
    if (n_pages <= 0 || n_pages * page_size > 0x7fffffffLL) MX_REFUSE("step tables: %lld pages of %d positions have no 32-bit slots", n_pages, page_size);
    if (keep_first < 0) MX_REFUSE("step tables: %d kept positions", keep_first);
    if ((shared_rows == nullptr) != (shared_pages == nullptr)) MX_REFUSE("step tables: shared rows and shared pages go together");
    StepTablesParams p;
    p.q_lens = q_lens; p.context_lens = context_lens; p.rows = rows; p.shared_rows = shared_rows; p.shared_pages = shared_pages;
    p.free_pages = free_pages; p.n_free = n_free; p.tables = tables; p.positions = positions; p.tok_seq = tok_seq; p.cu_q = cu_q;
    p.slots = slots; p.block_tables = block_tables; p.taken = taken; p.status = status;
    p.n_seqs = n_seqs; p.n_tokens = n_tokens; p.n_rows = n_rows; p.width = width; p.page_size = page_size; p.n_pages = (int)n_pages;
    p.n_free_most = n_free_most; p.window = window; p.keep_first = window > 0 ? keep_first : 0;
    // a block a sequence while that makes no more than two blocks an SM: more of them add up the lengths more often
    p.per_block = (n_seqs + 295) / 296;
    if (p.per_block > ST_OWN) MX_REFUSE("step tables: %d sequences, at most %d a step", n_seqs, 296 * ST_OWN);
    const dim3 grid((n_seqs + p.per_block - 1) / p.per_block, (width + ST_SLICE - 1) / ST_SLICE);
    if (grid.y > 65535) MX_REFUSE("step tables: tables of %d entries a row", width);
    const cudaError_t e = mx_launch_chained(step_tables_kernel, grid, dim3(ST_THREADS), 0, stream, p);
    if (e != cudaSuccess) {
        mx_set_error("step tables: launch failed: %s", cudaGetErrorString(e));
        return (int)e;
    }
    return MX_OK;
}
