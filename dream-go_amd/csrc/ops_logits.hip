// dgnn_adjust_logits: penalties for repeated tokens, biases and masks, one pass over the logits.
//
// A workgroup owns a chunk of one row's vocabulary.  Its logits and mask are asked for first; while they are on their way it counts the row's
// history into LDS -- the tokens of its chunk only, by integer atomics, whose order does not show -- and then adjusts and writes what it
// has.  Memory bounds it as long as a history is short beside the vocabulary: every chunk reads the whole history (out of the L2), so chunks are as
// large as LDS allows two of on a compute unit, and smaller only where that leaves units idle.  256 rows of 131072 bf16 logits with 8192 tokens of
// history each: 40.3 us, 3.65 TB/s; 32 of 50257 fp32: 7.25 us; one of 362: 4.8, of which a launch is 2.5.
#include "ops_device.h"

namespace dgnn {
namespace ops {
namespace {

constexpr int kMaxChunk = 16384, kMinChunk = 1024;      // tokens; 4 bytes of LDS each
constexpr int kMaxThreads = 1024, kEach = 2;            // vectors of eight tokens that a thread holds
static_assert(kMaxThreads * kEach * 8 >= kMaxChunk, "a workgroup holds its chunk");

// What is counted of a token: how often it occurs in the given part, above, and in the answer part, below.  A history of fewer than 65536 tokens
// fits sixteen bits each, and one kind of atomic does; with LONG one bit says that the given part has it at all.
constexpr unsigned kLongHistory = 65536;
template <bool LONG> constexpr unsigned kPrompt = LONG ? 0x80000000u : 0x10000u;
template <bool LONG> constexpr unsigned kAnswers = kPrompt<LONG> - 1;

template <typename T>
__device__ __forceinline__ vec<float, 8> load_eight(const T* p)
{
    return __builtin_convertvector(load_vec<T, 8>(p), vec<float, 8>);
}

// The kernel's arguments, read anew: kept from one phase to the next, they and what is made of them are more scalars than there are, and each that
// is put aside takes vector instructions to fetch.
typedef const __attribute__((address_space(4))) dgnn_logits_args* Arguments;
__device__ __forceinline__ Arguments again(Arguments a)
{
    asm volatile("" : "+s"(a));
    return a;
}

// A row's part of a chunk, as pointers.
template <typename T, typename O>
struct Chunk {
    const T* logits;
    O* out;
    const uint8_t* mask;
    const char* bias;
    bool bias_is_float;
    __device__ __forceinline__ Chunk(Arguments a, int64_t i, int64_t v0)
        : logits(static_cast<const T*>(a->logits) + i * a->ld_logits + v0), out(static_cast<O*>(a->out) + i * a->ld_out + v0),
          mask(a->mask ? reinterpret_cast<const uint8_t*>(a->mask + i * a->ld_mask) + (v0 >> 3) : nullptr), bias(nullptr), bias_is_float(a->bias_type == DGNN_F32)
    {
        if (a->bias) bias = static_cast<const char*>(a->bias) + (i * a->ld_bias + v0) * (bias_is_float ? 4 : (int)sizeof(T));
    }
};

// HISTORY: H is the type of its tokens.
template <typename T, typename O, typename H, bool HISTORY, bool LONG>
__global__ __launch_bounds__(kMaxThreads, 8)            // two workgroups on a unit: one counts while the other writes
void logits_kernel(dgnn_logits_args, int chunk, int chunks)
{
    const Arguments args = (Arguments)__builtin_amdgcn_kernarg_segment_ptr();   // (the first parameter)
    extern __shared__ __attribute__((aligned(16))) unsigned seen[];             // [chunk] with HISTORY
    for (int64_t i = blockIdx.y; i < args->b; i += gridDim.y)
        for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
            const int64_t v0 = (int64_t)c * chunk;
            const int64_t left = again(args)->v - v0;
            const int n = left < chunk ? (int)left : chunk;
            vec<T, 8> held[kEach];
            unsigned allowed[kEach];
            {
                const Chunk<T, O> at(again(args), i, v0);
#pragma unroll
                for (int q = 0; q < kEach; ++q) {
                    const int e = (q * (int)blockDim.x + (int)threadIdx.x) * 8;
                    held[q] = vec<T, 8>{};
                    allowed[q] = 0xff;
                    if (e + 8 <= n) {
                        held[q] = load_vec<T, 8>(at.logits + e);
                        if (at.mask) allowed[q] = at.mask[e >> 3];
                    }
                }
            }

            float repetition = 1.0f, mantissa = 1.0f, inverse = 1.0f, presence = 0.0f, frequency = 0.0f;     // repetition: mantissa 2^-exponent
            int exponent = 0;
            if constexpr (HISTORY) {
                const Arguments a = again(args);
                const int t = (int)a->t, wanted = a->lengths ? a->lengths[i] : t, given = a->prompt_lengths ? a->prompt_lengths[i] : 0;
                const unsigned length = wanted < 0 ? 0 : wanted > t ? t : wanted, prompt = given < 0 ? 0 : given;     // (counting past either stays in 32 bits)
                __syncthreads();                                               // (seen of the chunk before)
                for (int e = threadIdx.x * 4; e < chunk; e += blockDim.x * 4) *reinterpret_cast<vec<unsigned, 4>*>(seen + e) = vec<unsigned, 4>{};
                __syncthreads();
                const H* const history = static_cast<const H*>(a->history) + i * a->ld_history;
                const auto note = [&](H token, unsigned e) {
                    typedef std::make_unsigned_t<H> Unsigned;
                    const Unsigned at = (Unsigned)token - (Unsigned)v0;            // (a token in front of the chunk becomes a large number)
                    if (LONG && e < prompt) {
                        if (at < (Unsigned)n) atomicOr(&seen[at], kPrompt<LONG>);
                    } else {
                        const unsigned one = e < prompt ? kPrompt<LONG> : 1u;
                        if (at < (Unsigned)n) atomicAdd(&seen[at], one);
                    }
                };
                const unsigned whole = length & ~3u;
                for (unsigned e = threadIdx.x * 4; e < whole; e += blockDim.x * 4) {
                    const vec<H, 4> four = load_vec<H, 4>(history + e);
#pragma unroll
                    for (int r = 0; r < 4; ++r) note(four[r], e + r);
                }
                if (whole + threadIdx.x < length) note(history[whole + threadIdx.x], whole + threadIdx.x);
                __syncthreads();
                const Arguments p = again(args);
                repetition = p->repetition ? p->repetition[i] : p->repetition_all;
                mantissa = 2.0f * __builtin_amdgcn_frexp_mantf(repetition);
                exponent = 1 - __builtin_amdgcn_frexp_expf(repetition);
                inverse = 1.0f / mantissa;
                presence = p->presence ? p->presence[i] : p->presence_all;
                frequency = p->frequency ? p->frequency[i] : p->frequency_all;
            }
            // l / repetition to the last bit: a quotient by the reciprocal, corrected by what the exact product with it leaves of l (fixup: where l is
            // infinite).  By a mantissa, so that the reciprocal is no matter of range.  256 rows of 131072 with it 40.3 us, with the compiler's division 42.8,
            // with the product alone, which is a step off now and then, 39.4.
            const auto divided = [&](float l) {
                float q = l * inverse;
                q = __builtin_fmaf(__builtin_fmaf(-q, mantissa, l), inverse, q);
                return __builtin_ldexpf(__builtin_amdgcn_div_fixupf(q, mantissa, l), exponent);
            };
            const auto penalize = [&](float l, unsigned count) {
                const unsigned answered = count & kAnswers<LONG>;
                const float p = (l > 0.0f ? divided(l) : l * repetition) - frequency * (float)answered;
                return count ? p - (answered ? presence : 0.0f) : l;
            };
            const Chunk<T, O> at(again(args), i, v0);
#pragma unroll
            for (int q = 0; q < kEach; ++q) {
                const int e = (q * (int)blockDim.x + (int)threadIdx.x) * 8;
                if (e + 8 <= n) {
                    vec<float, 8> l = __builtin_convertvector(held[q], vec<float, 8>);
                    if constexpr (HISTORY) {
                        const vec<unsigned, 8> counts = *reinterpret_cast<const vec<unsigned, 8>*>(seen + e);
#pragma unroll
                        for (int r = 0; r < 8; ++r)
                            if (__builtin_amdgcn_ballot_w64(counts[r] != 0)) l[r] = penalize(l[r], counts[r]);      // (most of a vocabulary is never seen)
                    }
                    if (at.bias) l += at.bias_is_float ? load_eight(reinterpret_cast<const float*>(at.bias) + e) : load_eight(reinterpret_cast<const T*>(at.bias) + e);
                    if (at.mask) {
#pragma unroll
                        for (int r = 0; r < 8; ++r) l[r] = allowed[q] & 1u << r ? l[r] : -INFINITY;
                    }
                    store_vec<O, 8>(at.out + e, __builtin_convertvector(l, vec<O, 8>));
                } else {
                    for (int r = e; r < n; ++r) {
                        float l = (float)at.logits[r];
                        if constexpr (HISTORY) l = penalize(l, seen[r]);
                        if (at.bias) l += load_either<T>(at.bias, r, at.bias_is_float);
                        at.out[r] = (O)(!at.mask || (at.mask[r >> 3] >> (r & 7) & 1) ? l : -INFINITY);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);          // (one vector after the other: together they take more registers than there are)
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
    // two workgroups for every unit where there are tokens for that; threads that hold the chunk's vectors, more for a history that is longer
    int chunk = kMaxChunk;
    while (chunk > kMinChunk && a.b * ((a.v + chunk - 1) / chunk) < 512) chunk /= 2;
    int threads = power_of_two(history && a.t / 8 > chunk / (8 * kEach) ? a.t / 8 : chunk / (8 * kEach));
    threads = threads < 64 ? 64 : threads > kMaxThreads ? kMaxThreads : threads;
    const int chunks = (int)((a.v + chunk - 1) / chunk);
    const dim3 grid((unsigned)(chunks < (1 << 20) ? chunks : 1 << 20), (unsigned)(a.b < 65535 ? a.b : 65535));
    if (!history) return launch(logits_kernel<T, O, int32_t, false, false>, grid, dim3(threads), stream, a, chunk, chunks);
    static_assert(kMaxChunk * sizeof(unsigned) <= kMaxShared / 2, "two workgroups on a unit");
    const size_t shared = chunk * sizeof(unsigned);
    const bool wide = a.history_type == DGNN_I64, many = a.t >= kLongHistory;
    if (many && wide) return launch_shared(logits_kernel<T, O, int64_t, true, true>, grid, dim3(threads), shared, stream, a, chunk, chunks);
    if (many) return launch_shared(logits_kernel<T, O, int32_t, true, true>, grid, dim3(threads), shared, stream, a, chunk, chunks);
    if (wide) return launch_shared(logits_kernel<T, O, int64_t, true, false>, grid, dim3(threads), shared, stream, a, chunk, chunks);
    return launch_shared(logits_kernel<T, O, int32_t, true, false>, grid, dim3(threads), shared, stream, a, chunk, chunks);
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
