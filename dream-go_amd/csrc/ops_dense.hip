// dgnn_dense: y = act(alpha1 * x W^T + alpha2 * z + bias) on the matrix cores.
//
// The products are v_mfma_f32_16x16x32 with the ROWS OF W as the first operand and the rows of x as the second: D[i][j] then holds four
// consecutive outputs n of one row m in a lane's four registers, which is how y lies in memory.  Sums are fp32; alpha1, z, bias and the
// activation are applied in fp32 and the result is rounded once.
#include "ops_device.h"

namespace dgnn {
namespace ops {
namespace {

template <typename T>
__device__ __forceinline__ floatx4 mfma(vec<T, 8> a, vec<T, 8> b, floatx4 c)
{
    if constexpr (sizeof(T) == 2 && __is_same(T, f16)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// One output: everything behind the sum.
template <typename T, typename O>
__device__ __forceinline__ void finish(const dgnn_dense_args& a, int64_t m, int64_t n, float sum)
{
    float v = a.alpha1 * sum;
    if (a.z) v = __builtin_fmaf(a.alpha2, (float)static_cast<const O*>(a.z)[m * a.ldz + n], v);
    if (a.bias) v += load_either<T>(a.bias, n, a.bias_type == DGNN_F32);
    static_cast<O*>(a.y)[m * a.ldy + n] = (O)activate(v, a.activation);
}

// Eight elements of a row from column k on; zero at and beyond `k_end`.
template <typename T>
__device__ __forceinline__ vec<T, 8> load_row(const T* row, int64_t k, int64_t k_end)
{
    if (k + 8 <= k_end) return load_vec<T, 8>(row + k);
    vec<T, 8> v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = k + e < k_end ? row[k + e] : (T)0.0f;
    return v;
}

// 64 x 64 outputs per workgroup, 64 of k at a time through LDS, four waves of 32 x 32.
template <typename T, typename O>
__global__ __launch_bounds__(256)
void dense_kernel(dgnn_dense_args a, int64_t tiles_n, int64_t tiles)
{
    constexpr int kPitch = 72;                  // 64 + 8: rows start in different banks
    __shared__ __attribute__((aligned(16))) T lds[2][64 * kPitch];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T* const x = static_cast<const T*>(a.x);
    const T* const w = static_cast<const T*>(a.w);
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int64_t m0 = tile / tiles_n * 64, n0 = tile % tiles_n * 64;
        floatx4 acc[2][2] = {};
        for (int64_t k0 = 0; k0 < a.k; k0 += 64) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = (tid >> 3) + 32 * i, seg = (tid & 7) * 8;
                const int64_t n = n0 + row < a.n ? n0 + row : a.n - 1, m = m0 + row < a.m ? m0 + row : a.m - 1;
                *reinterpret_cast<vec<T, 8>*>(&lds[0][row * kPitch + seg]) = load_row<T>(w + n * a.ldw, k0 + seg, a.k);
                *reinterpret_cast<vec<T, 8>*>(&lds[1][row * kPitch + seg]) = load_row<T>(x + m * a.ldx, k0 + seg, a.k);
            }
            __syncthreads();
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                vec<T, 8> fw[2], fx[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    fw[i] = *reinterpret_cast<const vec<T, 8>*>(&lds[0][((wave & 1) * 32 + i * 16 + (lane & 15)) * kPitch + s * 32 + (lane >> 4) * 8]);
                    fx[i] = *reinterpret_cast<const vec<T, 8>*>(&lds[1][((wave >> 1) * 32 + i * 16 + (lane & 15)) * kPitch + s * 32 + (lane >> 4) * 8]);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = mfma<T>(fw[i], fx[j], acc[i][j]);
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int64_t n = n0 + (wave & 1) * 32 + i * 16 + (lane >> 4) * 4 + r, m = m0 + (wave >> 1) * 32 + j * 16 + (lane & 15);
                    if (m < a.m && n < a.n) finish<T, O>(a, m, n, acc[i][j][r]);
                }
    }
}

template <typename T, typename O>
hipError_t launch_typed(const dgnn_dense_args& a, hipStream_t stream)
{
    const int64_t tiles_n = (a.n + 63) / 64, tiles = tiles_n * ((a.m + 63) / 64);
    return launch(dense_kernel<T, O>, dim3((unsigned)(tiles < kMaxGrid ? tiles : kMaxGrid)), dim3(256), stream, a, tiles_n, tiles);
}

}  // namespace

hipError_t launch_dense(const dgnn_dense_args& a, hipStream_t stream)
{
    if (a.type == DGNN_F16) return a.out_type == DGNN_F32 ? launch_typed<f16, float>(a, stream) : launch_typed<f16, f16>(a, stream);
    return a.out_type == DGNN_F32 ? launch_typed<bf16, float>(a, stream) : launch_typed<bf16, bf16>(a, stream);
}

}  // namespace ops
}  // namespace dgnn
