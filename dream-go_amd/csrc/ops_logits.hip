// dgnn_adjust_logits: penalties for repeated tokens, biases and masks, one pass over the logits.
//
// A workgroup owns a chunk of one row's vocabulary.  Its logits, bias and mask are asked for first; while they are on their way it counts the
// row's history into LDS -- the tokens of its chunk only, by integer atomics, whose order does not show -- and then adjusts and writes what it
// has.  Memory bounds it as long as a history is short beside the vocabulary: every chunk reads the whole history (out of the L2), so chunks are as
// large as LDS allows two of on a compute unit, and smaller only where that leaves units idle.
#include "ops_device.h"

namespace dgnn {
namespace ops {
namespace {

constexpr int kMaxChunk = 16384, kMinChunk = 1024;      // tokens; 4 bytes of LDS each
constexpr int kEach = 2;                                // vectors of eight tokens that a thread holds at a time
constexpr unsigned kPrompt = 0x80000000u;               // the token occurs in the given part; the bits below count the answer part

template <typename T>
__device__ __forceinline__ vec<float, 8> load_eight(const T* p)
{
    return __builtin_convertvector(load_vec<T, 8>(p), vec<float, 8>);
}

// HISTORY: H is the type of its tokens.
template <typename T, typename O, typename H, bool HISTORY>
__global__ __launch_bounds__(1024)
void logits_kernel(dgnn_logits_args a, int chunk, int chunks)
{
    extern __shared__ __attribute__((aligned(16))) unsigned seen[];             // [chunk] with HISTORY
    const bool bias_is_float = a.bias_type == DGNN_F32;
    for (int64_t i = blockIdx.y; i < a.b; i += gridDim.y)
        for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
            const int64_t v0 = (int64_t)c * chunk;
            const int n = (int)(a.v - v0 < chunk ? a.v - v0 : chunk);
            const T* const logits = static_cast<const T*>(a.logits) + i * a.ld_logits + v0;
            const uint8_t* const mask = a.mask ? reinterpret_cast<const uint8_t*>(a.mask + i * a.ld_mask) + (v0 >> 3) : nullptr;
            const char* const bias = a.bias ? static_cast<const char*>(a.bias) + (i * a.ld_bias + v0) * (bias_is_float ? 4 : (int)sizeof(T)) : nullptr;
            O* const out = static_cast<O*>(a.out) + i * a.ld_out + v0;
            vec<T, 8> held[kEach];
            vec<float, 8> shift[kEach];
            unsigned allowed[kEach];
            const auto fetch = [&](int base) {
#pragma unroll
                for (int q = 0; q < kEach; ++q) {
                    const int e = base + (q * (int)blockDim.x + (int)threadIdx.x) * 8;
                    held[q] = vec<T, 8>{};
                    shift[q] = vec<float, 8>{};
                    allowed[q] = 0xff;
                    if (e + 8 <= n) {
                        held[q] = load_vec<T, 8>(logits + e);
                        if (bias) shift[q] = bias_is_float ? load_eight(reinterpret_cast<const float*>(bias) + e) : load_eight(reinterpret_cast<const T*>(bias) + e);
                        if (mask) allowed[q] = mask[e >> 3];
                    }
                }
            };
            fetch(0);

            float repetition = 1.0f, inverse = 1.0f, presence = 0.0f, frequency = 0.0f;
            if constexpr (HISTORY) {
                repetition = a.repetition ? a.repetition[i] : a.repetition_all;
                inverse = 1.0f / repetition;
                presence = a.presence ? a.presence[i] : a.presence_all;
                frequency = a.frequency ? a.frequency[i] : a.frequency_all;
                const int t = (int)a.t;
                int length = a.lengths ? a.lengths[i] : t, prompt = a.prompt_lengths ? a.prompt_lengths[i] : 0;
                length = length < 0 ? 0 : length > t ? t : length;
                __syncthreads();                                               // (seen of the chunk before)
                for (int e = threadIdx.x * 4; e < chunk; e += blockDim.x * 4) *reinterpret_cast<vec<unsigned, 4>*>(seen + e) = vec<unsigned, 4>{};
                __syncthreads();
                const H* const history = static_cast<const H*>(a.history) + i * a.ld_history;
                const auto note = [&](H token, int e) {
                    const int64_t at = (int64_t)token - v0;
                    if ((uint64_t)at < (uint64_t)n) {
                        if (e < prompt) atomicOr(&seen[at], kPrompt);
                        else atomicAdd(&seen[at], 1u);
                    }
                };
                const int whole = length & ~3;
                for (int e = threadIdx.x * 4; e < whole; e += blockDim.x * 4) {
                    const vec<H, 4> four = load_vec<H, 4>(history + e);
#pragma unroll
                    for (int r = 0; r < 4; ++r) note(four[r], e + r);
                }
                if (whole + (int)threadIdx.x < length) note(history[whole + threadIdx.x], whole + threadIdx.x);
                __syncthreads();
            }
            // l, with `count` as the history left it
            const auto adjust = [&](float l, unsigned count, float add, bool keep) {
                if constexpr (HISTORY) {
                    const unsigned answered = count & ~kPrompt;
                    const float p = l * (l > 0.0f ? inverse : repetition);
                    l = count ? p : l;
                    l = l - frequency * (float)answered - (answered ? presence : 0.0f);
                }
                return keep ? l + add : -INFINITY;
            };
            for (int base = 0; base < n; base += kEach * 8 * blockDim.x) {
                if (base > 0) fetch(base);
#pragma unroll
                for (int q = 0; q < kEach; ++q) {
                    const int e = base + (q * (int)blockDim.x + (int)threadIdx.x) * 8;
                    if (e + 8 <= n) {
                        vec<unsigned, 4> counts[2] = {};
                        if constexpr (HISTORY) {
                            counts[0] = *reinterpret_cast<const vec<unsigned, 4>*>(seen + e);
                            counts[1] = *reinterpret_cast<const vec<unsigned, 4>*>(seen + e + 4);
                        }
                        vec<O, 8> to;
#pragma unroll
                        for (int r = 0; r < 8; ++r) to[r] = (O)adjust((float)held[q][r], counts[r >> 2][r & 3], shift[q][r], allowed[q] >> r & 1);
                        store_vec<O, 8>(out + e, to);
                    } else {
                        for (int r = e; r < n; ++r) {
                            const float add = bias ? load_either<T>(bias, r, bias_is_float) : 0.0f;
                            out[r] = (O)adjust((float)logits[r], HISTORY ? seen[r] : 0u, add, !mask || (mask[r >> 3] >> (r & 7) & 1));
                        }
                    }
                }
            }
        }
}

int power_of_two(int64_t v)
{
    int p = 1;
    while (p < v) p *= 2;
    return p;
}

template <typename T, typename O>
hipError_t launch_typed(const dgnn_logits_args& a, hipStream_t stream)
{
    const bool history = a.history && a.t > 0;
    // two workgroups for every unit where there are tokens for that; threads for the chunk's vectors, and for a history that is longer
    int chunk = kMaxChunk;
    while (chunk > kMinChunk && a.b * ((a.v + chunk - 1) / chunk) < 512) chunk /= 2;
    int threads = power_of_two(history && a.t / 8 > chunk / (8 * kEach) ? a.t / 8 : chunk / (8 * kEach));
    threads = threads < 64 ? 64 : threads > 1024 ? 1024 : threads;
    const int chunks = (int)((a.v + chunk - 1) / chunk);
    const dim3 grid((unsigned)(chunks < (1 << 20) ? chunks : 1 << 20), (unsigned)(a.b < 65535 ? a.b : 65535));
    if (!history) return launch(logits_kernel<T, O, int32_t, false>, grid, dim3(threads), stream, a, chunk, chunks);
    const size_t shared = chunk * sizeof(unsigned);
    if (a.history_type == DGNN_I64) return launch_shared(logits_kernel<T, O, int64_t, true>, grid, dim3(threads), shared, stream, a, chunk, chunks);
    return launch_shared(logits_kernel<T, O, int32_t, true>, grid, dim3(threads), shared, stream, a, chunk, chunks);
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
