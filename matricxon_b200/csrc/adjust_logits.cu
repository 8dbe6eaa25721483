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
// A block owns a stretch of one row's vocabulary. It keeps, in shared memory, a word a token of its stretch: the count, and
// which entry of the bias list is the token's (largest index first). The row's ids are read whole by each of the row's blocks,
// which needs no sorting, no scratch memory and no second launch; integer atomics in shared memory make the counts
// independent of the order. Scores that the mask shuts out are not read.
#include <math.h>

#include "common.cuh"

namespace {

constexpr int AL_THREADS = 256;

struct AdjustParams {
    const void* logits;
    float* out;
    long long row_stride, out_stride;
    int vocab, stretch, mask_width, n_masks;
    const int *token_offsets, *token_ids, *bias_offsets, *bias_ids, *mask_words, *mask_rows, *pending;
    const float *repeat, *presence, *frequency, *bias_values;
};

template <typename T>
__global__ void __launch_bounds__(AL_THREADS) adjust_logits_kernel(const AdjustParams p) {
    extern __shared__ int words[];
    const int row = blockIdx.y, tid = threadIdx.x;
    const int begin = blockIdx.x * p.stretch, n = min(p.stretch, p.vocab - begin);
    pdl_trigger();
    pdl_wait();
    int* counts = words;
    int* bias_at = words + p.stretch;
    const int first = p.token_offsets ? p.token_offsets[row] : 0, last = p.token_offsets ? p.token_offsets[row + 1] : 0;
    const int pending = p.pending ? p.pending[row] : -1;
    const int bias_first = p.bias_offsets ? p.bias_offsets[row] : 0, bias_last = p.bias_offsets ? p.bias_offsets[row + 1] : 0;
    const int mask_row = p.mask_rows ? p.mask_rows[row] : (p.mask_words ? row : -1);
    const bool counted = last > first || pending >= 0, biased = bias_last > bias_first;
    const int* mask = mask_row >= 0 && mask_row < p.n_masks ? p.mask_words + (size_t)mask_row * p.mask_width : nullptr;
    if (counted)
        for (int i = tid; i < n; i += AL_THREADS) counts[i] = 0;
    if (biased)
        for (int i = tid; i < n; i += AL_THREADS) bias_at[i] = -1;
    if (counted || biased) __syncthreads();
    if (counted) {
        for (int j = first + tid; j < last; j += AL_THREADS) {
            const unsigned at = (unsigned)(p.token_ids[j] - begin);
            if (at < (unsigned)n) atomicAdd(&counts[at], 1);
        }
        if (tid == 0 && pending >= begin && pending < begin + n) atomicAdd(&counts[pending - begin], 1);
    }
    if (biased)
        for (int j = bias_first + tid; j < bias_last; j += AL_THREADS) {
            const unsigned at = (unsigned)(p.bias_ids[j] - begin);
            if (at < (unsigned)n) atomicMax(&bias_at[at], j);
        }
    if (counted || biased) __syncthreads();
    const float repeat = p.repeat ? p.repeat[row] : 1.f, presence = p.presence ? p.presence[row] : 0.f;
    const float frequency = p.frequency ? p.frequency[row] : 0.f;
    const T* src = reinterpret_cast<const T*>(p.logits) + (size_t)row * p.row_stride + begin;
    float* dst = p.out + (size_t)row * p.out_stride + begin;
#pragma unroll 4
    for (int i = tid; i < n; i += AL_THREADS) {
        const int v = begin + i;
        const bool allowed = mask == nullptr || ((unsigned)mask[v >> 5] >> (v & 31) & 1u);
        float x = allowed ? to_float(src[i]) : -INFINITY;
        if (allowed) {
            const int c = counted ? counts[i] : 0;
            if (c > 0) {
                x = x > 0.f ? x / repeat : x * repeat;
                x -= frequency * (float)c + presence;
            }
            if (biased && bias_at[i] >= 0) x += p.bias_values[bias_at[i]];
        }
        dst[i] = x;
    }
}

template <typename T>
int launch_adjust(const AdjustParams& p, int n_rows, cudaStream_t stream) {
    const size_t smem = (size_t)p.stretch * 8;
    const dim3 grid((p.vocab + p.stretch - 1) / p.stretch, n_rows);
    const cudaError_t e = mx_launch_chained(adjust_logits_kernel<T>, grid, dim3(AL_THREADS), smem, stream, p);
    if (e != cudaSuccess) {
        mx_set_error("adjust logits: launch failed: %s", cudaGetErrorString(e));
        return (int)e;
    }
    return MX_OK;
}

}  // namespace

extern "C" int mx_adjust_logits(const void* logits, int dtype, long long row_stride, float* out, long long out_stride, int n_rows,
                                int vocab, const int* token_offsets, const int* token_ids, const float* repeat,
                                const float* presence, const float* frequency, const int* bias_offsets, const int* bias_ids,
                                const float* bias_values, const int* mask_words, int n_masks, int mask_width,
                                const int* mask_rows, const int* pending, cudaStream_t stream) {
    if (n_rows <= 0) return MX_OK;
    if (n_rows > 65535) MX_REFUSE("adjust logits: %d rows exceed the grid", n_rows);
    if (vocab <= 0) MX_REFUSE("adjust logits: vocabulary of %d", vocab);
    if (mask_words != nullptr && (long long)mask_width * 32 < vocab) MX_REFUSE("adjust logits: masks of %d words for %d tokens", mask_width, vocab);
    AdjustParams p;
    p.logits = logits; p.out = out; p.row_stride = row_stride; p.out_stride = out_stride; p.vocab = vocab;
    p.mask_width = mask_width; p.n_masks = mask_words ? n_masks : 0; p.token_offsets = token_offsets; p.token_ids = token_ids;
    p.bias_offsets = bias_offsets; p.bias_ids = bias_ids; p.mask_words = mask_words; p.mask_rows = mask_rows; p.pending = pending;
    p.repeat = repeat; p.presence = presence; p.frequency = frequency; p.bias_values = bias_values;
    p.stretch = 4096;
    return dtype == MX_DTYPE_F32 ? launch_adjust<float>(p, n_rows, stream) : launch_adjust<__nv_bfloat16>(p, n_rows, stream);
}
