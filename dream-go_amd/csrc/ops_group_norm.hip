// dgnn_group_norm: group norm over channels-last maps, the skip input and the activation applied on the way out.
#include "ops_device.h"

namespace dgnn {
namespace ops {
namespace {

__device__ float group_sum(float v, float* lds)
{
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}

// One workgroup per sample and group; the variance is the mean of squared differences from the mean, not a difference of sums.
template <typename T>
__global__ __launch_bounds__(256)
void group_norm_kernel(dgnn_group_norm_args a)
{
    __shared__ float lds[4];
    const int64_t per = a.c / a.groups, count = a.p * per;
    for (int64_t item = blockIdx.x; item < a.n * a.groups; item += gridDim.x) {
        const int64_t i = item / a.groups, c0 = item % a.groups * per;
        const T* const x = static_cast<const T*>(a.x) + i * a.x_n + c0;
        float sum = 0.0f;
        for (int64_t e = threadIdx.x; e < count; e += 256) sum += (float)x[e / per * a.x_p + e % per];
        const float mean = group_sum(sum, lds) / (float)count;
        float square = 0.0f;
        for (int64_t e = threadIdx.x; e < count; e += 256) {
            const float d = (float)x[e / per * a.x_p + e % per] - mean;
            square = __builtin_fmaf(d, d, square);
        }
        const float scale = 1.0f / sqrtf(group_sum(square, lds) / (float)count + a.eps);
        for (int64_t e = threadIdx.x; e < count; e += 256) {
            const int64_t q = e / per, c = c0 + e % per;
            float v = ((float)x[q * a.x_p + e % per] - mean) * scale;
            if (a.weight) v *= load_either<T>(a.weight, c, a.affine_type == DGNN_F32);
            if (a.bias) v += load_either<T>(a.bias, c, a.affine_type == DGNN_F32);
            if (a.z) v += (float)static_cast<const T*>(a.z)[i * a.z_n + q * a.z_p + c];
            static_cast<T*>(a.y)[i * a.y_n + q * a.y_p + c] = (T)activate(v, a.activation);
        }
    }
}

template <typename T>
hipError_t launch_typed(const dgnn_group_norm_args& a, hipStream_t stream)
{
    const int64_t items = a.n * a.groups;
    return launch(group_norm_kernel<T>, dim3((unsigned)(items < kMaxGrid ? items : kMaxGrid)), dim3(256), stream, a);
}

}  // namespace

int64_t group_norm_workspace(const dgnn_group_norm_args&) { return 0; }

hipError_t launch_group_norm(const dgnn_group_norm_args& a, hipStream_t stream)
{
    switch (a.type) {
    case DGNN_F16: return launch_typed<f16>(a, stream);
    case DGNN_BF16: return launch_typed<bf16>(a, stream);
    default: return launch_typed<float>(a, stream);
    }
}

}  // namespace ops
}  // namespace dgnn
