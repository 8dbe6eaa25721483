// What the attention kernels know of sequences that have their first keys in common (attention_shared.cu).
//
// The step's sequences lie in groups one after another: group g holds sequences first[g] .. first[g + 1] - 1. Sequence s reads
// its keys below lens[s] through the block table of its group's first sequence, together with the rest of the group, and its
// keys from lens[s] on through its own.
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
    int seq;                 // the group's first sequence
    int q_start, tokens;     // the group's tokens; none: there is no such tile
    int first;               // where the tile starts among their rows
};

// Tile `tile` of the groups' rows (`rows` a token) cut into tiles of `per_tile` rows, group after group; by a whole warp. The lists live on the
// device, so a captured step may be replayed with other groups; a launch has blocks for the most tiles that there can be.
__device__ __forceinline__ GroupTile find_group_tile(const SharedPrefixParams& p, const int* cu_q, int tile, int per_tile, int rows, int lane) {
    GroupTile found = {0, 0, 0, 0};
    int before = 0;
    for (int g0 = 0; g0 < p.n_groups; g0 += 32) {
        const int g = g0 + lane;
        int seq = 0, start = 0, tokens = 0;
        if (g < p.n_groups) {
            seq = min(max(p.first[g], 0), p.n_seqs);
            start = min(cu_q[seq], p.n_tokens);
            tokens = min(cu_q[min(max(p.first[g + 1], 0), p.n_seqs)], p.n_tokens) - start;
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
            found.q_start = __shfl_sync(0xffffffffu, start, at);
            found.tokens = __shfl_sync(0xffffffffu, tokens, at);
            found.first = (tile - before - __shfl_sync(0xffffffffu, through - tiles, at)) * per_tile;
            return found;
        }
        before += __shfl_sync(0xffffffffu, through, 31);
    }
    return found;
}

// The same over the sequences' own (token, head) rows, tiles of `rows` rows of `group` a token: (sequence, first row).
struct SequenceTile {
    int seq, row;            // seq < 0: there is no such tile
};
__device__ __forceinline__ SequenceTile find_sequence_tile(const SharedPrefixParams& p, const int* cu_q, int tile, int rows, int group, int lane) {
    int before = 0;
    for (int s0 = 0; s0 < p.n_seqs; s0 += 32) {
        const int s = s0 + lane;
        const int mine = s < p.n_seqs ? max(0, min(cu_q[s + 1], p.n_tokens) - cu_q[s]) * group : 0;
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
