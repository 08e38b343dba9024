// dgnn_adjust_logits: penalties for repeated tokens, biases and masks, one pass over the logits.
//
// A workgroup owns a chunk of one row's vocabulary.  It counts the row's history into LDS -- only the tokens of its chunk, by integer
// atomics, whose order does not show -- and then reads, adjusts and writes its logits once.
#include "ops_device.h"

namespace dgnn {
namespace ops {
namespace {

constexpr int kChunk = 4096;
constexpr unsigned kPrompt = 0x80000000u;       // the token occurs in the given part; the bits below count the answer part

template <typename T, typename O, typename H>
__global__ __launch_bounds__(256)
void logits_kernel(dgnn_logits_args a, int64_t chunks)
{
    __shared__ unsigned seen[kChunk];
    for (int64_t item = blockIdx.x; item < a.b * chunks; item += gridDim.x) {
        const int64_t i = item / chunks, v0 = item % chunks * kChunk;
        const int n = (int)(a.v - v0 < kChunk ? a.v - v0 : kChunk);
        float repetition = 1.0f, presence = 0.0f, frequency = 0.0f;
        if (a.history) {
            repetition = a.repetition ? a.repetition[i] : a.repetition_all;
            presence = a.presence ? a.presence[i] : a.presence_all;
            frequency = a.frequency ? a.frequency[i] : a.frequency_all;
            int64_t length = a.lengths ? a.lengths[i] : a.t;
            length = length < 0 ? 0 : length > a.t ? a.t : length;
            const int64_t prompt = a.prompt_lengths ? a.prompt_lengths[i] : 0;
            __syncthreads();
            for (int e = threadIdx.x; e < n; e += 256) seen[e] = 0;
            __syncthreads();
            const H* const history = static_cast<const H*>(a.history) + i * a.ld_history;
            for (int64_t e = threadIdx.x; e < length; e += 256) {
                const int64_t at = (int64_t)history[e] - v0;
                if (at >= 0 && at < n) {
                    if (e < prompt) atomicOr(&seen[at], kPrompt);
                    else atomicAdd(&seen[at], 1u);
                }
            }
            __syncthreads();
        }
        for (int e = threadIdx.x; e < n; e += 256) {
            const int64_t v = v0 + e;
            float l = (float)static_cast<const T*>(a.logits)[i * a.ld_logits + v];
            if (a.history && seen[e]) {
                l = l > 0.0f ? l / repetition : l * repetition;
                const unsigned count = seen[e] & ~kPrompt;
                if (count) l = l - frequency * (float)count - presence;
            }
            if (a.bias) l += load_either<T>(a.bias, i * a.ld_bias + v, a.bias_type == DGNN_F32);
            if (a.mask && !(a.mask[i * a.ld_mask + (v >> 5)] >> (v & 31) & 1)) l = -INFINITY;
            static_cast<O*>(a.out)[i * a.ld_out + v] = (O)l;
        }
    }
}

template <typename T, typename O>
hipError_t launch_typed(const dgnn_logits_args& a, hipStream_t stream)
{
    const int64_t chunks = (a.v + kChunk - 1) / kChunk, items = a.b * chunks;
    const dim3 grid((unsigned)(items < kMaxGrid ? items : kMaxGrid));
    if (a.history_type == DGNN_I64) return launch(logits_kernel<T, O, int64_t>, grid, dim3(256), stream, a, chunks);
    return launch(logits_kernel<T, O, int32_t>, grid, dim3(256), stream, a, chunks);
}

}  // namespace

hipError_t launch_adjust_logits(const dgnn_logits_args& a, hipStream_t stream)
{
    switch (a.type) {
    case DGNN_F16: return a.out_type == DGNN_F32 ? launch_typed<f16, float>(a, stream) : launch_typed<f16, f16>(a, stream);
    case DGNN_BF16: return a.out_type == DGNN_F32 ? launch_typed<bf16, float>(a, stream) : launch_typed<bf16, bf16>(a, stream);
    default: return launch_typed<float, float>(a, stream);
    }
}

}  // namespace ops
}  // namespace dgnn
