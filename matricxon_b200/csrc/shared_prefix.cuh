// What the attention kernels know of sequences that have their first keys in common (attention_shared.cu).
//
// The step's sequences lie in groups one after another: group g holds sequences first[g] .. first[g + 1] - 1. Sequence s reads
// its keys below lens[s] through the block table of its group's first sequence, together with the rest of the group, and its
// keys from lens[s] on through its own. Under a window (or blocks) the first sequence may have given up pages that others of
// the group still see: those are read through the first one of these that has to hold them (shared_page).
#pragma once

#include "common.cuh"

struct SharedPrefixParams {
    const int* first;        // [n_groups + 1]
    const int* lens;         // [sequences]; null: nothing is shared, every key is read through the sequence's own table
    const int* tok_seq;      // [tokens]
    const int* positions;    // [tokens]
    int n_groups;
    int n_seqs;
    int n_tokens;            // rows that there are: sequences that bring more are cut off there (and reported by the join)
    int n_parts;             // parts of a token and head's softmax, those of the shared keys first
    int n_shared_parts;
    int beside;              // the kernel of the shared keys was launched just before this one, which begins beside it
};

// At the end of a block of the kernel of the own keys, which began beside that of the shared ones: the grid must not be done
// before the other is, since what comes next waits for this one. One block that waits is enough (with all of them waiting,
// those that are done hold the SMs of those that have not begun).
__device__ __forceinline__ void wait_for_shared_keys() {
    if ((blockIdx.x | blockIdx.y | blockIdx.z) == 0) pdl_wait();
}

struct KeyRange {
    int first, last;         // none: last < first
};

// The shared keys that a token's query sees.
__device__ __forceinline__ KeyRange shared_keys_of_token(const SharedPrefixParams& p, int token, int window) {
    const int position = p.positions[token], seq = p.tok_seq[token];
    KeyRange range;
    range.first = first_visible_key(position, window);
    range.last = seq >= 0 && seq < p.n_seqs ? min(position, p.lens[seq] - 1) : -1;
    return range;
}

// From the first key that any of `n` tokens sees to the last one; by a whole warp.
__device__ __forceinline__ KeyRange shared_keys_of_tokens(const SharedPrefixParams& p, int first, int n, int window, int lane) {
    int low = 0x7fffffff, high = -1;
    for (int i = lane; i < n; i += 32) {
        const KeyRange one = shared_keys_of_token(p, first + i, window);
        if (one.first <= one.last) {
            low = min(low, one.first);
            high = max(high, one.last);
        }
    }
    KeyRange range;
    range.first = __reduce_min_sync(0xffffffffu, low);
    range.last = __reduce_max_sync(0xffffffffu, high);
    return range;
}

struct GroupTile {
    int seq, end;            // the group's sequences: seq .. end - 1
    int q_start, tokens;     // the group's tokens; none: there is no such tile
    int first;               // where the tile starts among their rows
};

// Tile `tile` of the groups' rows (`rows` a token) cut into tiles of `per_tile` rows, group after group; by a whole warp. The lists live on the
// device, so a captured step may be replayed with other groups; a launch has blocks for the most tiles that there can be.
__device__ __forceinline__ GroupTile find_group_tile(const SharedPrefixParams& p, const int* cu_q, int tile, int per_tile, int rows, int lane) {
    GroupTile found = {0, 0, 0, 0, 0};
    int before = 0;
    for (int g0 = 0; g0 < p.n_groups; g0 += 32) {
        const int g = g0 + lane;
        int seq = 0, end = 0, start = 0, tokens = 0;
        if (g < p.n_groups) {
            seq = min(max(p.first[g], 0), p.n_seqs);
            end = min(max(p.first[g + 1], 0), p.n_seqs);
            start = min(max(cu_q[seq], 0), p.n_tokens);
            tokens = min(cu_q[end], p.n_tokens) - start;
        }
        const int tiles = tokens > 0 ? (tokens * rows + per_tile - 1) / per_tile : 0;
        int through = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, through, o);
            if (lane >= o) through += up;
        }
        const unsigned past = __ballot_sync(0xffffffffu, before + through > tile);
        if (past) {
            const int at = __ffs(past) - 1;
            found.seq = __shfl_sync(0xffffffffu, seq, at);
            found.end = __shfl_sync(0xffffffffu, end, at);
            found.q_start = __shfl_sync(0xffffffffu, start, at);
            found.tokens = __shfl_sync(0xffffffffu, tokens, at);
            found.first = (tile - before - __shfl_sync(0xffffffffu, through - tiles, at)) * per_tile;
            return found;
        }
        before += __shfl_sync(0xffffffffu, through, 31);
    }
    return found;
}

// Where a page of a group's shared keys is looked up.
struct SharedPages {
    const int *block_tables, *cu_q, *context_lens, *lens;
    int bt_stride, page_size, window, seq, end;       // sequences seq .. end - 1
};
constexpr int PAGE_UNSEEN = -2;                       // no page, and no query of the group sees a key of it

__device__ __forceinline__ SharedPages shared_pages_of(const SharedPrefixParams& p, const GroupTile& group, const int* block_tables,
                                                       int bt_stride, const int* cu_q, const int* context_lens, int page_size, int window) {
    return SharedPages{block_tables, cu_q, context_lens, p.lens, bt_stride, page_size, window, group.seq, group.end};
}

// A page that the group's first sequence has no entry for. That is in order where it sees none of the page's keys any more.
// The page is then that of the first sequence that sees one and shares the whole page (of a page that its shared keys fill in
// part it has a copy of its own, whose first slots nobody fills). -1: there is no such sequence, though the page is seen.
// A sequence's lengths are two loads at one place for a whole warp, so a warp walks a group of 128 in a few us; only groups
// whose first sequence has moved on come here.
static __device__ __forceinline__ int shared_page_of_others(const SharedPages& g, int lp) {
    const long long begin = (long long)lp * g.page_size, last = begin + g.page_size - 1;
    bool seen = false;
    for (int s = g.seq; s < g.end; ++s) {
        const int context = g.context_lens[s], tokens = g.cu_q[s + 1] - g.cu_q[s], shared = g.lens[s];
        const int low = first_visible_key(context, g.window), high = min(context + tokens, shared) - 1;
        if (tokens <= 0 || low > last || high < begin || high < low) continue;
        if (s == g.seq) return -1;
        seen = true;
        if (last < shared) return lp < g.bt_stride ? max(g.block_tables[(size_t)s * g.bt_stride + lp], -1) : -1;
    }
    return seen ? -1 : PAGE_UNSEEN;
}

__device__ __forceinline__ int shared_page(const SharedPages& g, int lp) {
    const int page = lp < g.bt_stride ? g.block_tables[(size_t)g.seq * g.bt_stride + lp] : -1;
    return page >= 0 ? page : shared_page_of_others(g, lp);
}

// The same over the sequences' own (token, head) rows, tiles of `rows` rows of `group` a token: (sequence, first row).
struct SequenceTile {
    int seq, row;            // seq < 0: there is no such tile
};
__device__ __forceinline__ SequenceTile find_sequence_tile(const SharedPrefixParams& p, const int* cu_q, int tile, int rows, int group, int lane) {
    int before = 0;
    for (int s0 = 0; s0 < p.n_seqs; s0 += 32) {
        const int s = s0 + lane;
        const int mine = s < p.n_seqs ? max(0, min(cu_q[s + 1], p.n_tokens) - max(cu_q[s], 0)) * group : 0;
        const int tiles = (mine + rows - 1) / rows;
        int through = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, through, o);
            if (lane >= o) through += up;
        }
        const unsigned past = __ballot_sync(0xffffffffu, before + through > tile);
        if (past) {
            const int at = __ffs(past) - 1;
            return SequenceTile{s0 + at, (tile - before - __shfl_sync(0xffffffffu, through - tiles, at)) * rows};
        }
        before += __shfl_sync(0xffffffffu, through, 31);
    }
    return SequenceTile{-1, 0};
}

// A launch whose kernel may begin before the one before it has ended, in a captured step or not: for kernels launched one
// after another by one call, of which the first has waited for all that came before.
template <typename... KArgs, typename... Args>
static inline cudaError_t mx_launch_beside(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                                           Args... args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = block;
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attribute;
    config.numAttrs = 1;
    mx_count_launch();
    return cudaLaunchKernelEx(&config, kernel, KArgs(args)...);
}
