// What a row's next scores lose and gain before a token is drawn: penalties for tokens it has generated, biases, and a mask of
// the tokens it may take.
//
// With c the number of times that token v stands among the row's generated ids (and the pending one):
//   y = c > 0 ? (x > 0 ? x / repeat : x * repeat) : x          the repeat penalty, as the sampler has it (sampling.cu)
//   y = y - (frequency * c + (c > 0 ? presence : 0)) + bias[v]
//   y = allowed[v] ? y : -infinity
// in float, from float or bfloat16 scores. An id outside the vocabulary counts for nothing; of a token with two biases the
// later one holds; a row without a mask (mask_rows < 0) may take every token.
//
// A block owns a stretch of one row's vocabulary. It first writes the scores as the mask leaves them, which is bound by memory:
// fours as 16-byte accesses wherever the rows of both sides lie alike (stretches are counted from the 16-byte boundary before
// the row, so odd vocabularies do); a four is asked for a turn before it is written, its mask a turn before that, and not
// at all if the mask shuts it out. Nothing in that loop may branch on a score: a look at each score's count there made it three
// times as long. Then the block counts, in shared memory, how often each token of its stretch stands in the row's list, and
// deals with each of them once, in what it has just written: of the threads that have one of a token's places the first to
// take its count does so. Integer atomics: the order in which threads come does not matter. The biases come last, the largest
// place in the list among a token's biases says which one holds. What a phase reads it asks for eight at a time.
// Where a row has many blocks and a long list, a kernel beside deals the ids out to the stretches first, so that each is looked
// at once, not by every block of the row.
// Offsets live on the device, where a captured call may find others than those it was captured with: a row's part of a list is
// what lies inside the list. Offsets that fall (parts of rows that overlap) have no place each in the dealt ids; every block
// then reads its row's list.
// 256 rows of 131,071 scores, a third of them allowed, with 6,144 ids each: 90 us (a copy of the scores takes 47), 121 with every
// block reading the whole list, 92 with a kernel after this one that gathers each row's list in a hash table. What is left
// above the copy are the atomics: shared memory takes some 0.75 lanes of them a cycle and SM, whatever words they go to.
#include <math.h>

#include "common.cuh"
#include "shared_prefix.cuh"

namespace {

constexpr int AL_THREADS = 256, AL_FOURS = 2;        // fours of scores a thread has on their way
constexpr int AL_TURN = 4 * AL_FOURS * AL_THREADS;
constexpr int AL_AHEAD = 8;                          // ids a thread asks for at a time
constexpr int DEAL_THREADS = 512;
constexpr int DEAL_BLOCKS = 1024;                    // stretches of a row that ids are dealt out to, at most

struct AdjustParams {
    const void* logits;
    float* out;
    long long row_stride, out_stride;
    int vocab, mask_width, n_masks;
    long long n_ids, n_biases;                       // sizes of the lists of all rows
    const int *token_offsets, *token_ids, *bias_offsets, *bias_ids, *mask_words, *mask_rows, *pending;
    const float *repeat, *presence, *frequency, *bias_values;
    int stretch;                                     // scores of a block
    int *dealt, *dealt_from;                         // ids by stretch, and where each stretch's begin [rows][blocks + 1]; or null
};

__device__ __forceinline__ const unsigned* mask_of(const AdjustParams& p, int row) {
    if (p.mask_words == nullptr) return nullptr;
    const int at = p.mask_rows ? p.mask_rows[row] : row;
    return at >= 0 && at < p.n_masks ? reinterpret_cast<const unsigned*>(p.mask_words) + (size_t)at * p.mask_width : nullptr;
}

// Where a row's part of a list of `size` begins, and how long it is.
struct Part {
    int first, count;
};
__device__ __forceinline__ int within(int offset, long long size) { return (int)min(max((long long)offset, 0LL), size); }
__device__ __forceinline__ Part part_of(const int* offsets, int row, long long size) {
    if (offsets == nullptr) return Part{0, 0};
    const int first = within(offsets[row], size);
    return Part{first, max(within(offsets[row + 1], size) - first, 0)};
}

__device__ __forceinline__ void load_four(const float* from, float* x) {
    const float4 v = *reinterpret_cast<const float4*>(from);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
__device__ __forceinline__ void load_four(const __nv_bfloat16* from, float* x) {
    const uint2 v = *reinterpret_cast<const uint2*>(from);
    x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xffff0000u);
    x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xffff0000u);
}

// Tokens are counted from the 16-byte boundary before the row's first one: place j is token j - shift.
__device__ __forceinline__ int shift_of(const AdjustParams& p, int row) {
    return (int)(reinterpret_cast<uintptr_t>(p.out + (size_t)row * p.out_stride) >> 2 & 3);
}

// A row's ids (and the pending one) sorted by stretch, in any order within one: counted, then put in place. A block a row.
__global__ void __launch_bounds__(DEAL_THREADS) deal_ids_kernel(const AdjustParams p, int n_blocks) {
    __shared__ int count[DEAL_BLOCKS];
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
    pdl_wait();
    pdl_trigger();                                    // the scores' kernel begins beside this one
    const Part list = part_of(p.token_offsets, row, p.n_ids);
    const int first = list.first, pending = p.pending ? p.pending[row] : -1, shift = shift_of(p, row);
    const int n = list.count + 1, log_stretch = 31 - __clz(p.stretch);       // a power of two
    // the stretches of ids k0 + tid, + DEAL_THREADS, ... (-1: none)
    auto ahead = [&](int k0, int* id, int* to) {
#pragma unroll
        for (int e = 0; e < AL_AHEAD; ++e) {
            const int k = k0 + e * DEAL_THREADS + tid;
            id[e] = k >= n ? -1 : (k == n - 1 ? pending : p.token_ids[first + k]);
        }
#pragma unroll
        for (int e = 0; e < AL_AHEAD; ++e) to[e] = id[e] >= 0 && id[e] < p.vocab ? (id[e] + shift) >> log_stretch : -1;
    };
    int id[AL_AHEAD], to[AL_AHEAD];
    ahead(0, id, to);
    for (int i = tid; i < n_blocks; i += DEAL_THREADS) count[i] = 0;
    bool falls = false;
    for (int i = tid; i < (int)gridDim.x; i += DEAL_THREADS)
        falls = falls || within(p.token_offsets[i + 1], p.n_ids) < within(p.token_offsets[i], p.n_ids);
    if (__syncthreads_or(falls)) {
        if (tid == 0) p.dealt_from[(size_t)row * (n_blocks + 1)] = -1;        // nothing is dealt out
        return;
    }
    for (int k0 = 0; k0 < n; k0 += AL_AHEAD * DEAL_THREADS) {
        if (k0 > 0) ahead(k0, id, to);
#pragma unroll
        for (int e = 0; e < AL_AHEAD; ++e)
            if (to[e] >= 0) atomicAdd(&count[to[e]], 1);
    }
    __syncthreads();
    if (tid < 32) {
        int before = 0;
        for (int i0 = 0; i0 < n_blocks; i0 += 32) {
            const int i = i0 + lane, mine = i < n_blocks ? count[i] : 0;
            int through = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, through, o);
                if (lane >= o) through += up;
            }
            if (i < n_blocks) {
                count[i] = before + through - mine;
                p.dealt_from[(size_t)row * (n_blocks + 1) + i] = before + through - mine;
            }
            before += __shfl_sync(0xffffffffu, through, 31);
        }
        if (lane == 0) p.dealt_from[(size_t)row * (n_blocks + 1) + n_blocks] = before;
    }
    __syncthreads();
    int* dealt = p.dealt + (size_t)first + row;       // behind the lists before this one, and a pending id each
    for (int k0 = 0; k0 < n; k0 += AL_AHEAD * DEAL_THREADS) {
        ahead(k0, id, to);
#pragma unroll
        for (int e = 0; e < AL_AHEAD; ++e)
            if (to[e] >= 0) dealt[atomicAdd(&count[to[e]], 1)] = id[e];
    }
}

template <typename T>
__global__ void __launch_bounds__(AL_THREADS, 5) adjust_logits_kernel(const AdjustParams p) {
    extern __shared__ __align__(16) int words[];      // a word a token of the stretch
    const int row = blockIdx.y, tid = threadIdx.x;
    if (p.dealt == nullptr) pdl_wait();               // the kernel before this one has waited otherwise
    const T* src = reinterpret_cast<const T*>(p.logits) + (size_t)row * p.row_stride;
    float* dst = p.out + (size_t)row * p.out_stride;
    const unsigned* mask = mask_of(p, row);
    const int shift = shift_of(p, row);
    const bool alike = (reinterpret_cast<uintptr_t>(src - shift) & (4 * sizeof(T) - 1)) == 0;
    const int begin = (int)min((long long)blockIdx.x * p.stretch, (long long)p.vocab + shift);
    const int end = min(begin + p.stretch, p.vocab + shift);
    // The fours that lie wholly in the row: places from `low` to `high`. What is left, up to three tokens at either end of the
    // row, is done one by one.
    const int row_low = (shift + 3) & ~3, row_high = (p.vocab + shift) & ~3;
    const int low = max(begin, row_low), high = min(end, row_high);
    auto takes = [&](int v) { return mask == nullptr || (mask[v >> 5] >> (v & 31) & 1u); };
    // which tokens of the four at place j the row may take (a bit each), and their scores if there are any
    auto bits_at = [&](int j) -> unsigned {
        if (j >= high) return 0u;
        if (mask == nullptr) return 15u;
        const int v = j - shift;
        const unsigned* word = mask + (v >> 5);
        // the four lies in two words only where the row is shifted against the mask
        const unsigned more = shift != 0 && (v & 31) > 28 ? word[1] : 0u;
        return __funnelshift_r(word[0], more, v & 31) & 15u;
    };
    auto load = [&](int j, unsigned allowed, float* x) {
        if (allowed == 0) return;
        const T* from = src + (j - shift);
        if (alike) {
            load_four(from, x);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = to_float(from[e]);
        }
    };
    float next[AL_FOURS][4];
    unsigned next_bits[AL_FOURS], later_bits[AL_FOURS];
#pragma unroll
    for (int u = 0; u < AL_FOURS; ++u) next_bits[u] = bits_at(low + 4 * (tid + u * AL_THREADS));
#pragma unroll
    for (int u = 0; u < AL_FOURS; ++u) {
        load(low + 4 * (tid + u * AL_THREADS), next_bits[u], next[u]);
        later_bits[u] = bits_at(low + 4 * (tid + u * AL_THREADS) + AL_TURN);
    }
    for (int j0 = low + 4 * tid; j0 < high; j0 += AL_TURN) {
        float x[AL_FOURS][4];
        unsigned allowed[AL_FOURS];
#pragma unroll
        for (int u = 0; u < AL_FOURS; ++u) {
            allowed[u] = next_bits[u];
            next_bits[u] = later_bits[u];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[u][e] = next[u][e];
        }
#pragma unroll
        for (int u = 0; u < AL_FOURS; ++u) {
            load(j0 + 4 * u * AL_THREADS + AL_TURN, next_bits[u], next[u]);
            later_bits[u] = bits_at(j0 + 4 * u * AL_THREADS + 2 * AL_TURN);
        }
#pragma unroll
        for (int u = 0; u < AL_FOURS; ++u) {
            const int j = j0 + 4 * u * AL_THREADS;
            if (j >= high) break;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[u][e] = allowed[u] >> e & 1u ? x[u][e] : -INFINITY;
            *reinterpret_cast<float4*>(dst + j - shift) = make_float4(x[u][0], x[u][1], x[u][2], x[u][3]);
        }
    }
    // the tokens before the first four (threads 0 to 3) and behind the last (4 to 7)
    if (tid < 8) {
        const int j = tid < 4 ? tid : row_high + tid - 4, v = j - shift;
        if (j >= begin && j < end && v >= 0 && (tid < 4 ? j < row_low : j >= row_low))
            dst[v] = takes(v) ? to_float(src[v]) : -INFINITY;
    }
    if (p.token_offsets == nullptr && p.pending == nullptr && p.bias_offsets == nullptr) return;

    // ---- the listed tokens
    const float repeat = p.repeat ? p.repeat[row] : 1.f, presence = p.presence ? p.presence[row] : 0.f;
    const float frequency = p.frequency ? p.frequency[row] : 0.f;
    const Part biases = part_of(p.bias_offsets, row, p.n_biases);
    const unsigned to_place = (unsigned)(shift - begin), n = (unsigned)(end - begin);
    const Part list = part_of(p.token_offsets, row, p.n_ids);
    const int* ids = p.token_ids + list.first;
    int n_ids = list.count, pending = p.pending ? p.pending[row] : -1;
    if (p.dealt != nullptr) {
        pdl_wait();                                   // the ids have been dealt out
        const int* from = after_wait(p.dealt_from) + (size_t)row * (gridDim.x + 1);
        const int dealt = from[0], before = from[blockIdx.x], behind = from[blockIdx.x + 1];
        if (dealt >= 0) {
            n_ids = behind - before;
            ids = after_wait(p.dealt) + (size_t)list.first + row + before;
            pending = -1;                             // among them
        }
    }
    // places in the stretch of ids k0 + tid, + AL_THREADS, ... of a list (n or more: elsewhere)
    auto ahead = [&](const int* list, int count, int last_id, int k0, unsigned* at) {
        int id[AL_AHEAD];
#pragma unroll
        for (int e = 0; e < AL_AHEAD; ++e) {
            const int k = k0 + e * AL_THREADS + tid;
            id[e] = k < count ? list[k] : (k == count ? last_id : -1);
        }
#pragma unroll
        for (int e = 0; e < AL_AHEAD; ++e) at[e] = id[e] >= 0 ? (unsigned)id[e] + to_place : n;
    };
    unsigned at[AL_AHEAD];
    if (n_ids > 0 || pending >= 0) {
        ahead(ids, n_ids, pending, 0, at);
        for (int i = tid; i < (int)(n + 3) / 4; i += AL_THREADS) reinterpret_cast<int4*>(words)[i] = make_int4(0, 0, 0, 0);
        __syncthreads();
        for (int k0 = 0; k0 <= n_ids; k0 += AL_AHEAD * AL_THREADS) {
            if (k0 > 0) ahead(ids, n_ids, pending, k0, at);
#pragma unroll
            for (int e = 0; e < AL_AHEAD; ++e)
                if (at[e] < n) atomicAdd(&words[at[e]], 1);
        }
        __syncthreads();                              // the counts are whole, the scores written
        for (int k0 = 0; k0 <= n_ids; k0 += AL_AHEAD * AL_THREADS) {
            if (n_ids >= AL_AHEAD * AL_THREADS) ahead(ids, n_ids, pending, k0, at);
            int c[AL_AHEAD];
            float x[AL_AHEAD];
#pragma unroll
            for (int e = 0; e < AL_AHEAD; ++e) c[e] = at[e] < n ? atomicExch(&words[at[e]], 0) : 0;
#pragma unroll
            for (int e = 0; e < AL_AHEAD; ++e) x[e] = c[e] > 0 ? dst[(int)(at[e] - to_place)] : 0.f;
#pragma unroll
            for (int e = 0; e < AL_AHEAD; ++e) {
                const int v = (int)(at[e] - to_place);
                if (c[e] > 0 && takes(v)) {
                    const float y = x[e] > 0.f ? x[e] / repeat : x[e] * repeat;
                    dst[v] = y - (frequency * (float)c[e] + presence);
                }
            }
        }
    }
    if (biases.count > 0) {
        const int bias_first = biases.first, n_biases = biases.count;
        ahead(p.bias_ids + bias_first, n_biases, -1, 0, at);
        bool here = n_biases > AL_AHEAD * AL_THREADS;
#pragma unroll
        for (int e = 0; e < AL_AHEAD; ++e) here = here || at[e] < n;
        if (__syncthreads_or(here)) {
            // three rounds over the biases of this stretch: the words' start, the largest place, the sum
            for (int round = 0; round < 3; ++round) {
                for (int k0 = 0; k0 < n_biases; k0 += AL_AHEAD * AL_THREADS) {
                    if (n_biases > AL_AHEAD * AL_THREADS) ahead(p.bias_ids + bias_first, n_biases, -1, k0, at);
#pragma unroll
                    for (int e = 0; e < AL_AHEAD; ++e) {
                        const int k = k0 + e * AL_THREADS + tid;
                        if (at[e] >= n) continue;
                        if (round == 0) words[at[e]] = -1;
                        else if (round == 1) atomicMax(&words[at[e]], k);
                        else if (words[at[e]] == k && takes((int)(at[e] - to_place))) dst[(int)(at[e] - to_place)] += p.bias_values[bias_first + k];
                    }
                }
                __syncthreads();
            }
        }
    }
}

// Scores of a block, a power of two: a turn while that makes no more than some eight blocks an SM, else four turns (32 KB of counts).
int stretch_of(int n_rows, int vocab) { return (long long)n_rows * vocab <= 8LL * 148 * AL_TURN ? AL_TURN : 4 * AL_TURN; }

long long blocks_of(int n_rows, int vocab) { return ((long long)vocab + 3 + stretch_of(n_rows, vocab) - 1) / stretch_of(n_rows, vocab); }

// Whether ids are dealt out first: where every block reading its row's whole list would look at more of them than at a quarter
// of its scores.
bool deals(long long n_ids, int n_rows, int vocab) {
    const long long n_blocks = blocks_of(n_rows, vocab);
    return n_blocks <= DEAL_BLOCKS && n_ids / n_rows * n_blocks > vocab / 4;
}

template <typename T>
int launch_adjust(const AdjustParams& p, int n_rows, int n_blocks, size_t smem, cudaStream_t stream) {
    const dim3 grid(n_blocks, n_rows);
    const cudaError_t e = p.dealt != nullptr ? mx_launch_beside(adjust_logits_kernel<T>, grid, dim3(AL_THREADS), smem, stream, p)
                                             : mx_launch_chained(adjust_logits_kernel<T>, grid, dim3(AL_THREADS), smem, stream, p);
    if (e != cudaSuccess) {
        mx_set_error("adjust logits: launch failed: %s", cudaGetErrorString(e));
        return (int)e;
    }
    return MX_OK;
}

}  // namespace

// Bytes of scratch of mx_adjust_logits with the same arguments: the ids by stretch, and where each stretch's begin.
extern "C" long long mx_adjust_logits_scratch(long long n_ids, int n_rows, int vocab) {
    if (n_rows <= 0 || vocab <= 0 || !deals(n_ids, n_rows, vocab)) return 0;
    return 4 * (n_ids + n_rows + n_rows * (blocks_of(n_rows, vocab) + 1));
}

// n_ids, n_biases: how many there are of all rows together (the sizes of token_ids and bias_ids).
extern "C" int mx_adjust_logits(const void* logits, int dtype, long long row_stride, float* out, long long out_stride, int n_rows,
                                int vocab, const int* token_offsets, const int* token_ids, long long n_ids, const float* repeat,
                                const float* presence, const float* frequency, const int* bias_offsets, const int* bias_ids,
                                const float* bias_values, long long n_biases, const int* mask_words, int n_masks, int mask_width,
                                const int* mask_rows, const int* pending, int* scratch, cudaStream_t stream) {
    if (n_rows <= 0) return MX_OK;
    if (n_rows > 65535) MX_REFUSE("adjust logits: %d rows exceed the grid", n_rows);
    if (vocab <= 0 || vocab > 0x7fffffff - 65536) MX_REFUSE("adjust logits: vocabulary of %d", vocab);
    if (mask_words != nullptr && (long long)mask_width * 32 < vocab) MX_REFUSE("adjust logits: masks of %d words for %d tokens", mask_width, vocab);
    AdjustParams p;
    p.logits = logits; p.out = out; p.row_stride = row_stride; p.out_stride = out_stride; p.vocab = vocab;
    p.mask_width = mask_width; p.n_masks = mask_words ? n_masks : 0; p.token_offsets = token_offsets; p.token_ids = token_ids;
    p.bias_offsets = bias_offsets; p.bias_ids = bias_ids; p.mask_words = mask_words; p.mask_rows = mask_rows; p.pending = pending;
    p.repeat = repeat; p.presence = presence; p.frequency = frequency; p.bias_values = bias_values;
    p.n_ids = n_ids; p.n_biases = n_biases;
    p.stretch = stretch_of(n_rows, vocab);
    p.dealt = p.dealt_from = nullptr;
    const int n_blocks = (int)blocks_of(n_rows, vocab);
    if (deals(n_ids, n_rows, vocab)) {
        if (scratch == nullptr) MX_REFUSE("adjust logits: long lists need scratch memory");
        p.dealt = scratch;
        p.dealt_from = scratch + n_ids + n_rows;
        const cudaError_t e = mx_launch_chained(deal_ids_kernel, dim3(n_rows), dim3(DEAL_THREADS), 0, stream, p, n_blocks);
        if (e != cudaSuccess) {
            mx_set_error("adjust logits: launch failed: %s", cudaGetErrorString(e));
            return (int)e;
        }
    }
    const bool listed = token_offsets != nullptr || pending != nullptr || bias_offsets != nullptr;
    const size_t smem = listed ? (size_t)p.stretch * 4 : 0;
    return dtype == MX_DTYPE_F32 ? launch_adjust<float>(p, n_rows, n_blocks, smem, stream)
                                 : launch_adjust<__nv_bfloat16>(p, n_rows, n_blocks, smem, stream);
}
