// dgnn_group_norm: group norm over channels-last maps, the skip input and the activation applied on the way out.
//
// A workgroup owns a slab of channels of one sample -- whole groups, up to 64 sixteen-byte vectors -- and all positions, or a share of them.
// Threads are laid over (position, vector): a wave reads whole lines.  Mean and variance take two passes over values that are in REGISTERS:
// the variance is the mean of squared differences from the mean, never a difference of sums, and costs no second read.
//
//   one pass   a sample's slab fits the registers of a workgroup: read once, written once (the floor).  256 x 361 x 256 fp16 with skip and ReLU,
//              142 MB: kOnePassTime
//   two        it does not: a first kernel leaves (mean, sum of squares about it) of every share of the positions, a second joins those of its
//              groups -- both about the JOINT mean, in a fixed order -- and reads the maps again, mostly out of the last-level cache.
//
// Bound by memory on both ways; the activations are branch-free for that reason (ops_device.h).
#include "ops_device.h"

namespace dgnn {
namespace ops {
namespace {

constexpr int kMaxThreads = 1024, kMaxVectors = 64, kRegisters = 8;     // vectors of a row of a slab; vectors of a thread
constexpr int kMaxShares = 256;                                         // of a sample's positions

template <typename T> constexpr int width_of = 16 / (int)sizeof(T);     // elements of a vector

// How a call is cut up; the same for every workgroup.
struct Layout {
    int per;                // channels of a group
    int groups_per_slab;    // 1 where a group is wider than a slab: then `subs` slabs make a group
    int subs;
    int slabs;              // of a sample
    int lanes;              // threads side by side on a row: a power of two
    int threads;
    int64_t shares, share;  // of a sample's positions, positions of each
    int64_t pieces() const { return shares * subs; }
};

struct Slab {
    int c0, channels, g0, groups, sub;
};

__device__ __forceinline__ Slab slab_of(const Layout& l, int c, int groups, int vector, int s)
{
    Slab r;
    if (l.subs == 1) {
        r.g0 = s * l.groups_per_slab;
        r.groups = groups - r.g0 < l.groups_per_slab ? groups - r.g0 : l.groups_per_slab;
        r.c0 = r.g0 * l.per;
        r.channels = r.groups * l.per;
        r.sub = 0;
    } else {
        r.g0 = s / l.subs;
        r.groups = 1;
        r.sub = s % l.subs;
        r.c0 = r.g0 * l.per + r.sub * kMaxVectors * vector;
        const int left = l.per - r.sub * kMaxVectors * vector;
        r.channels = left < kMaxVectors * vector ? left : kMaxVectors * vector;
    }
    return r;
}

template <typename T, int V>
__device__ __forceinline__ void load_part(const T* p, int n, float (&v)[V])
{
    if (n >= V) {
        const vec<T, V> all = load_vec<T, V>(p);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (float)all[e];
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = e < n ? (float)p[e] : 0.0f;
    }
}

template <typename T, int V>
__device__ __forceinline__ void load_affine(const void* p, bool is_float, int c, int n, float otherwise, float (&v)[V])
{
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = otherwise;
    if (!p) return;
#pragma unroll
    for (int e = 0; e < V; ++e)
        if (e < n) v[e] = load_either<T>(p, c + e, is_float);
}

// Sums of `mine` (per channel of the thread's vector) over the threads of each group of the slab, to sums[group].
template <int V>
__device__ __forceinline__ void group_sums(const Layout& l, const Slab& s, const float (&mine)[V], float* scratch, float* sums)
{
    const int tid = threadIdx.x, rows = blockDim.x / l.lanes, waves = (blockDim.x + 63) >> 6;
    // a vector lies in one group, or (wide groups) the slab does: one number of each thread is enough
    const bool single = l.subs > 1 || l.per % V == 0;
    __syncthreads();                                            // (scratch and sums of the time before)
    if (single) {
        float all = mine[0];
#pragma unroll
        for (int e = 1; e < V; ++e) all += mine[e];
        scratch[tid] = all;
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) scratch[tid * V + e] = mine[e];
    }
    __syncthreads();
    const int pitch = single ? l.lanes : l.lanes * V;
    const int n = l.subs > 1 ? (s.channels + V - 1) / V : single ? l.per / V : l.per;
    for (int g = tid >> 6; g < s.groups; g += waves) {
        float sum = 0.0f;
        for (int e = tid & 63; e < rows * n; e += 64) {
            const int row = e / n;
            sum += scratch[row * pitch + g * n + (e - row * n)];
        }
        sum = wave_sum(sum);
        if ((tid & 63) == 0) sums[g] = sum;
    }
    __syncthreads();
}

// The group (of the slab) of each channel of the thread's vector.
template <int V>
__device__ __forceinline__ void per_channel(const Layout& l, int at, const float* of_group, float (&v)[V])
{
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = of_group[l.subs > 1 ? 0 : (at + e) / l.per];
}

template <typename T, int V>
__device__ __forceinline__ void finish(const dgnn_group_norm_args& a, int64_t i, int64_t q, int c, int n, float (&v)[V])
{
    if (a.z) {
        float z[V];
        load_part<T, V>(static_cast<const T*>(a.z) + i * a.z_n + q * a.z_p + c, n, z);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += z[e];
    }
    activate(v, a.activation);
    T* const y = static_cast<T*>(a.y) + i * a.y_n + q * a.y_p + c;
    if (n >= V) {
        vec<T, V> out;
#pragma unroll
        for (int e = 0; e < V; ++e) out[e] = (T)v[e];
        store_vec<T, V>(y, out);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < n) y[e] = (T)v[e];
    }
}

constexpr int kMaxGroups = kMaxVectors * 8;                     // of a slab

// R vectors per thread.
template <typename T, int R>
__global__ __launch_bounds__(kMaxThreads)
void one_pass_kernel(dgnn_group_norm_args a, Layout l)
{
    constexpr int V = width_of<T>;
    __shared__ float scratch[kMaxThreads * V], sums[kMaxGroups];
    const int lane = threadIdx.x & (l.lanes - 1), row = threadIdx.x / l.lanes, rows = blockDim.x / l.lanes;
    const int64_t items = a.n * l.slabs;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t i = item / l.slabs;
        const Slab s = slab_of(l, (int)a.c, (int)a.groups, V, (int)(item % l.slabs));
        const int at = lane * V, n = s.channels - at;           // n <= 0: this thread has no part of a row
        const T* const x = static_cast<const T*>(a.x) + i * a.x_n + s.c0 + at;
        vec<T, V> held[R];
        float sum[V] = {};
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t q = row + r * rows;
            held[r] = vec<T, V>{};
            if (q < a.p && n > 0) {
                if (n >= V) held[r] = load_vec<T, V>(x + q * a.x_p);
                else {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (e < n) held[r][e] = x[q * a.x_p + e];
                }
            }
        }
        float weight[V], bias[V];
        load_affine<T, V>(a.weight, a.affine_type == DGNN_F32, s.c0 + at, n, 1.0f, weight);
        load_affine<T, V>(a.bias, a.affine_type == DGNN_F32, s.c0 + at, n, 0.0f, bias);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < V; ++e) sum[e] += (float)held[r][e];
        const float count = (float)a.p * (float)l.per;
        float mean[V], scale[V];
        group_sums<V>(l, s, sum, scratch, sums);
        per_channel<V>(l, at < s.channels ? at : 0, sums, mean);
#pragma unroll
        for (int e = 0; e < V; ++e) mean[e] /= count, sum[e] = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (row + (int64_t)r * rows < a.p) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float d = (float)held[r][e] - mean[e];
                    sum[e] = e < n ? __builtin_fmaf(d, d, sum[e]) : 0.0f;
                }
            }
        group_sums<V>(l, s, sum, scratch, sums);
        per_channel<V>(l, at < s.channels ? at : 0, sums, scale);
#pragma unroll
        for (int e = 0; e < V; ++e) scale[e] = weight[e] / sqrtf(scale[e] / count + a.eps);
        if (n <= 0) continue;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t q = row + (int64_t)r * rows;
            if (q >= a.p) break;
            float v[V];
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = __builtin_fmaf((float)held[r][e] - mean[e], scale[e], bias[e]);
            finish<T, V>(a, i, q, s.c0 + at, n, v);
        }
    }
}

// What is known of some of a group's values.
struct Moments {
    float mean, squares;                                        // squares: sum of squared differences from the mean
};

// (mean, squares) of a share of the positions of a slab's groups, to moments[sample][group][share][sub].
template <typename T>
__global__ __launch_bounds__(kMaxThreads)
void moments_kernel(dgnn_group_norm_args a, Layout l, Moments* moments)
{
    constexpr int V = width_of<T>, R = kRegisters;
    __shared__ float scratch[kMaxThreads * V], sums[kMaxGroups];
    __shared__ Moments joint[kMaxGroups];
    const int lane = threadIdx.x & (l.lanes - 1), row = threadIdx.x / l.lanes, rows = blockDim.x / l.lanes;
    const int64_t items = a.n * l.shares * l.slabs;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t i = item / (l.shares * l.slabs), share = item / l.slabs % l.shares;
        const Slab s = slab_of(l, (int)a.c, (int)a.groups, V, (int)(item % l.slabs));
        const int at = lane * V, n = s.channels - at, per = l.subs > 1 ? s.channels : l.per;
        const int64_t begin = share * l.share, end = begin + l.share < a.p ? begin + l.share : a.p;
        const T* const x = static_cast<const T*>(a.x) + i * a.x_n + s.c0 + at;
        // as many positions as the registers hold at a time, joined as they come
        for (int64_t q0 = begin; q0 < end; q0 += R * rows) {
            vec<T, V> held[R];
            float sum[V] = {}, mean[V];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int64_t q = q0 + row + r * rows;
                held[r] = vec<T, V>{};
                if (q < end && n > 0) {
                    if (n >= V) held[r] = load_vec<T, V>(x + q * a.x_p);
                    else {
#pragma unroll
                        for (int e = 0; e < V; ++e)
                            if (e < n) held[r][e] = x[q * a.x_p + e];
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < V; ++e) sum[e] += (float)held[r][e];
            const int64_t here = end - q0 < R * rows ? end - q0 : R * rows;
            const float count = (float)here * (float)per;
            group_sums<V>(l, s, sum, scratch, sums);
            per_channel<V>(l, at < s.channels ? at : 0, sums, mean);
            const float first_mean = threadIdx.x < s.groups ? sums[threadIdx.x] / count : 0.0f;
#pragma unroll
            for (int e = 0; e < V; ++e) mean[e] /= count, sum[e] = 0.0f;
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (q0 + row + r * rows < end) {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float d = (float)held[r][e] - mean[e];
                        sum[e] = e < n ? __builtin_fmaf(d, d, sum[e]) : 0.0f;
                    }
                }
            group_sums<V>(l, s, sum, scratch, sums);
            if (threadIdx.x < s.groups) {
                Moments m{first_mean, sums[threadIdx.x]};
                if (q0 > begin) {
                    const Moments before = joint[threadIdx.x];
                    const float old = (float)(q0 - begin) * (float)per, d = m.mean - before.mean, part = count / (old + count);
                    m.squares = before.squares + m.squares + d * d * old * part;
                    m.mean = before.mean + d * part;
                }
                joint[threadIdx.x] = m;
            }
        }
        if (threadIdx.x < s.groups) moments[((i * a.groups + s.g0 + threadIdx.x) * l.shares + share) * l.subs + s.sub] = joint[threadIdx.x];
    }
}

template <typename T>
__global__ __launch_bounds__(kMaxThreads)
void apply_kernel(dgnn_group_norm_args a, Layout l, const Moments* moments)
{
    constexpr int V = width_of<T>;
    __shared__ Moments joint[kMaxGroups];
    const int lane = threadIdx.x & (l.lanes - 1), row = threadIdx.x / l.lanes, rows = blockDim.x / l.lanes, waves = (blockDim.x + 63) >> 6;
    const int64_t items = a.n * l.shares * l.slabs;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t i = item / (l.shares * l.slabs), share = item / l.slabs % l.shares;
        const Slab s = slab_of(l, (int)a.c, (int)a.groups, V, (int)(item % l.slabs));
        const int64_t begin = share * l.share, end = begin + l.share < a.p ? begin + l.share : a.p, pieces = l.shares * l.subs;
        __syncthreads();                                        // (joint of the time before)
        for (int g = threadIdx.x >> 6; g < s.groups; g += waves) {
            const Moments* const of = moments + (i * a.groups + s.g0 + g) * pieces;
            const auto count = [&](int64_t piece) {
                const int64_t first = piece / l.subs * l.share, left = a.p - first;
                const int from = (int)(piece % l.subs) * kMaxVectors * V, wide = l.per - from < kMaxVectors * V || l.subs == 1 ? l.per - from : kMaxVectors * V;
                return (float)(left < l.share ? left : l.share) * (float)wide;
            };
            const float all = (float)a.p * (float)l.per;
            float sum = 0.0f, squares = 0.0f;
            for (int64_t piece = threadIdx.x & 63; piece < pieces; piece += 64) sum = __builtin_fmaf(of[piece].mean, count(piece) / all, sum);
            const float mean = wave_sum(sum);
            for (int64_t piece = threadIdx.x & 63; piece < pieces; piece += 64) {
                const float d = of[piece].mean - mean;
                squares += __builtin_fmaf(d * d, count(piece), of[piece].squares);
            }
            squares = wave_sum(squares);
            if ((threadIdx.x & 63) == 0) joint[g] = Moments{mean, 1.0f / sqrtf(squares / all + a.eps)};
        }
        __syncthreads();
        const int at = lane * V, n = s.channels - at;
        if (n <= 0) continue;
        float mean[V], scale[V], bias[V];
        load_affine<T, V>(a.weight, a.affine_type == DGNN_F32, s.c0 + at, n, 1.0f, scale);
        load_affine<T, V>(a.bias, a.affine_type == DGNN_F32, s.c0 + at, n, 0.0f, bias);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int channel = at + e < s.channels ? at + e : at;
            const Moments m = joint[l.subs > 1 ? 0 : channel / l.per];
            mean[e] = m.mean;
            scale[e] *= m.squares;
        }
        const T* const x = static_cast<const T*>(a.x) + i * a.x_n + s.c0 + at;
        for (int64_t q = begin + row; q < end; q += rows) {
            float v[V];
            load_part<T, V>(x + q * a.x_p, n, v);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = __builtin_fmaf(v[e] - mean[e], scale[e], bias[e]);
            finish<T, V>(a, i, q, s.c0 + at, n, v);
        }
    }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int power_of_two(int64_t v)
{
    int p = 1;
    while (p < v) p *= 2;
    return p;
}

// One pass where a workgroup's registers hold a slab of a sample, two otherwise.
Layout make_layout(const dgnn_group_norm_args& a, int* registers)
{
    const int vector = a.type == DGNN_F32 ? 4 : 8;
    Layout l;
    l.per = (int)(a.c / a.groups);
    l.subs = (int)ceil_div(l.per, kMaxVectors * vector);
    l.shares = 1;
    l.share = a.p;
    // lines of 128 bytes where groups are narrow, fewer channels where that leaves compute units idle
    const int64_t wanted = 128 / (16 / vector);
    int64_t groups = l.subs > 1 ? 1 : wanted / l.per > 1 ? wanted / l.per : 1;
    if (groups > a.groups) groups = a.groups;
    while (groups > 1 && a.n * ceil_div(a.groups, groups) < 256) groups = (groups + 1) / 2;
    const auto cut = [&]() {
        l.groups_per_slab = (int)groups;
        l.slabs = (int)(l.subs > 1 ? a.groups * l.subs : ceil_div(a.groups, groups));
        l.lanes = power_of_two(l.subs > 1 ? kMaxVectors : ceil_div(groups * l.per, vector));
    };
    cut();
    // a slab that does not fit may fit when it is narrower, down to 32 bytes of a line
    while (l.subs == 1 && groups > 1 && groups * l.per > 2 * vector && a.p > (int64_t)kMaxThreads / l.lanes * kRegisters) {
        groups = (groups + 1) / 2;
        cut();
    }
    *registers = 0;
    if (l.subs == 1 && a.p <= (int64_t)kMaxThreads / l.lanes * kRegisters) {
        const int64_t vectors = a.p * l.lanes;
        int threads = 64;
        while (threads < kMaxThreads && vectors > threads * 4) threads *= 2;
        l.threads = threads;
        const int64_t each = ceil_div(a.p, threads / l.lanes);
        *registers = each <= 1 ? 1 : each <= 2 ? 2 : each <= 4 ? 4 : 8;
        return l;
    }
    groups = l.subs > 1 ? 1 : wanted / l.per > 1 ? wanted / l.per : 1;
    if (groups > a.groups) groups = a.groups;
    cut();
    l.threads = kMaxThreads;
    const int64_t rows = kMaxThreads / l.lanes, at_once = rows * kRegisters;
    // shares of what the registers hold, fewer and larger ones where there would be too many to join
    l.share = ceil_div(ceil_div(a.p, at_once), kMaxShares) * at_once;
    l.shares = ceil_div(a.p, l.share);
    return l;
}

template <typename T>
hipError_t launch_typed(const dgnn_group_norm_args& a, hipStream_t stream)
{
    int registers;
    const Layout l = make_layout(a, &registers);
    const int64_t items = a.n * l.slabs * l.shares;
    const dim3 grid((unsigned)(items < kMaxGrid ? items : kMaxGrid)), block(l.threads);
    switch (registers) {
    case 1: return launch(one_pass_kernel<T, 1>, grid, block, stream, a, l);
    case 2: return launch(one_pass_kernel<T, 2>, grid, block, stream, a, l);
    case 4: return launch(one_pass_kernel<T, 4>, grid, block, stream, a, l);
    case 8: return launch(one_pass_kernel<T, 8>, grid, block, stream, a, l);
    }
    Moments* const moments = static_cast<Moments*>(a.workspace);
    const hipError_t err = launch(moments_kernel<T>, grid, block, stream, a, l, moments);
    if (err != hipSuccess) return err;
    return launch(apply_kernel<T>, grid, block, stream, a, l, moments);
}

}  // namespace

int64_t group_norm_workspace(const dgnn_group_norm_args& a)
{
    int registers;
    const Layout l = make_layout(a, &registers);
    return registers ? 0 : a.n * a.groups * l.pieces() * (int64_t)sizeof(Moments);
}

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
