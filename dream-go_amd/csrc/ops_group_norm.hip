// dgnn_group_norm: group norm over channels-last maps, the skip input and the activation applied on the way out.
//
// A workgroup owns a slab of channels of one sample -- whole groups, up to 64 sixteen-byte vectors -- and all positions, or a share of them.
// Threads are laid over (position, vector), so that neighbours read what lies side by side.  Mean and variance take two passes over values that
// are in REGISTERS: the variance is the mean of squared differences from the mean, never a difference of sums, and costs no second read.
//
//   one pass   a sample's slab fits the registers of a workgroup: read once, written once, which is the floor
//   two        it does not: a first kernel leaves (mean, sum of squares about it) of every share of the positions, a second joins those of its
//              groups -- about their joint mean, in a fixed order -- and reads the maps again, mostly out of the last-level cache
//
// Bound by memory on both ways; the activations are branch-free for that reason (ops_device.h).
#include "ops_device.h"

namespace dgnn {
namespace ops {
namespace {

constexpr int kMaxThreads = 1024, kMaxVectors = 64, kRegisters = 8;     // vectors of a row of a slab; vectors of a thread
constexpr int kMaxGroups = kMaxVectors * 8;                             // of a slab
constexpr int kMaxShares = 256;                                         // of a sample's positions
constexpr int kUnitsWanted = 256;                                       // workgroups that give every compute unit one

template <typename T> constexpr int width_of = 16 / (int)sizeof(T);     // elements of a vector

// How a call is cut up; the same for every workgroup.
struct Layout {
    int per;                // channels of a group
    int groups_per_slab;    // 1 where a group is wider than a slab: then `subs` slabs make a group
    int subs;
    int slabs;              // of a sample
    int lanes, rows;        // vectors of a slab's row, rows that a workgroup's threads cover
    int threads;
    int shares;             // of a sample's positions
    int64_t share;          // positions of each
};

// The part of a slab that a thread works on.
struct Part {
    int g0, groups, sub;    // the slab's groups; which of a wide group's slabs it is
    int channels;           // of the slab
    int row;                // of the workgroup's rows; -1: this thread has no part
    int at, c, n;           // first channel in the slab and of all, channels (fewer than a vector at the end of a slab)
};

template <int V>
__device__ __forceinline__ Part part_of(const Layout& l, int groups, int slab)
{
    Part p;
    const int row = threadIdx.x / l.lanes, lane = threadIdx.x - row * l.lanes;
    int c0;
    if (l.subs == 1) {
        p.g0 = slab * l.groups_per_slab;
        p.groups = groups - p.g0 < l.groups_per_slab ? groups - p.g0 : l.groups_per_slab;
        p.sub = 0;
        p.channels = p.groups * l.per;
        c0 = p.g0 * l.per;
    } else {
        p.g0 = slab / l.subs;
        p.groups = 1;
        p.sub = slab - p.g0 * l.subs;
        const int first = p.sub * kMaxVectors * V;
        p.channels = l.per - first < kMaxVectors * V ? l.per - first : kMaxVectors * V;
        c0 = p.g0 * l.per + first;
    }
    p.at = lane * V;
    p.c = c0 + p.at;
    p.n = p.channels - p.at < V ? p.channels - p.at : V;
    p.row = row < l.rows && p.n > 0 ? row : -1;
    if (p.row < 0) p.at = p.n = 0, p.c = c0;
    return p;
}

template <typename T, int V>
__device__ __forceinline__ vec<T, V> load_part(const T* p, int n)
{
    if (n == V) return load_vec<T, V>(p);
    vec<T, V> v = {};
#pragma unroll
    for (int e = 0; e < V; ++e)
        if (e < n) v[e] = p[e];
    return v;
}

template <typename T, int V>
__device__ __forceinline__ void store_part(T* p, int n, const float (&v)[V])
{
    vec<T, V> out;
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = (T)v[e];
    if (n == V) return store_vec<T, V>(p, out);
#pragma unroll
    for (int e = 0; e < V; ++e)
        if (e < n) p[e] = out[e];
}

template <typename T, int V>
__device__ __forceinline__ void load_affine(const void* p, bool is_float, int c, int n, float otherwise, float (&v)[V])
{
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = otherwise;
    if (!p) return;
    if (is_float) {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < n) v[e] = static_cast<const float*>(p)[c + e];
    } else {
        const vec<T, V> all = load_part<T, V>(static_cast<const T*>(p) + c, n);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (float)all[e];
    }
}

// One number of every group of the slab for each channel of the thread's vector.
template <int V>
__device__ __forceinline__ void of_channels(const Layout& l, const Part& p, const float* of_group, float (&v)[V])
{
    if (l.subs > 1 || l.per % V == 0) {
        const float all = of_group[l.subs > 1 ? 0 : p.at / l.per];
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = all;
    } else {
        int g = p.at / l.per, left = l.per - p.at % l.per;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            v[e] = of_group[g < p.groups ? g : p.groups - 1];
            if (--left == 0) ++g, left = l.per;
        }
    }
}

// The sums of `mine` over the threads of each group of the slab, as `last` makes them, to out[group].  One barrier inside and one behind;
// `scratch` is not the one of the call before.
template <int V, typename Last>
__device__ __forceinline__ void group_sums(const Layout& l, const Part& p, const float (&mine)[V], float* scratch, float* out, Last last)
{
    // a vector lies in one group, or (wide groups) the slab does: one number of each thread is enough
    const bool single = l.subs > 1 || l.per % V == 0;
    if (single) {
        float all = mine[0];
#pragma unroll
        for (int e = 1; e < V; ++e) all += mine[e];
        scratch[threadIdx.x] = all;
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) scratch[threadIdx.x * V + e] = mine[e];
    }
    __syncthreads();
    const int waves = (int)(blockDim.x + 63) >> 6, lane = threadIdx.x & 63;
    const int pitch = single ? l.lanes : l.lanes * V, n = l.subs > 1 ? l.lanes : single ? l.per / V : l.per;
    const int down = 64 / n, across = 64 - down * n;            // 64 numbers on
    for (int g = threadIdx.x >> 6; g < p.groups; g += waves) {
        float sum = 0.0f;
        int row = lane / n, column = lane - row * n;
        while (row < l.rows) {
            sum += scratch[row * pitch + g * n + column];
            row += down;
            column += across;
            if (column >= n) column -= n, ++row;
        }
        sum = wave_sum(sum);
        if (lane == 0) out[g] = last(sum);
    }
    __syncthreads();
}

// The values as they came: without it the compiler keeps them as fp32 as well, from one use to the next, and runs out of registers.
template <typename V>
__device__ __forceinline__ void as_loaded(V& v) { asm volatile("" : "+v"(v)); }

// R vectors per thread.
template <typename T, int R, bool SKIP>
__global__ __launch_bounds__(R == kRegisters ? kMaxThreads / 2 : kMaxThreads)
void one_pass_kernel(dgnn_group_norm_args a, Layout l)
{
    constexpr int V = width_of<T>;
    __shared__ float scratch[2][kMaxThreads * V], means[kMaxGroups], scales[kMaxGroups];
    const float inverse = 1.0f / ((float)a.p * (float)l.per);
    for (int64_t i = blockIdx.z; i < a.n; i += gridDim.z)
        for (int slab = blockIdx.x; slab < l.slabs; slab += gridDim.x) {
            const Part p = part_of<V>(l, (int)a.groups, slab);
            const int here = p.row < 0 || p.row >= a.p ? 0 : (int)(a.p - 1 - p.row) / l.rows + 1;    // positions of this thread
            const T* x = static_cast<const T*>(a.x) + i * a.x_n + p.row * a.x_p + p.c;
            vec<T, V> held[R], skip[SKIP ? R : 1];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                held[r] = r < here ? load_part<T, V>(x, p.n) : vec<T, V>{};
                x += l.rows * a.x_p;
            }
            if constexpr (SKIP) {
                const T* z = static_cast<const T*>(a.z) + i * a.z_n + p.row * a.z_p + p.c;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    skip[r] = r < here ? load_part<T, V>(z, p.n) : vec<T, V>{};
                    z += l.rows * a.z_p;
                }
            }
            float weight[V], bias[V], sum[V] = {}, mean[V], scale[V];
            load_affine<T, V>(a.weight, a.affine_type == DGNN_F32, p.c, p.n, 1.0f, weight);
            load_affine<T, V>(a.bias, a.affine_type == DGNN_F32, p.c, p.n, 0.0f, bias);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < V; ++e) sum[e] += (float)held[r][e];
            group_sums<V>(l, p, sum, scratch[0], means, [&](float s) { return s * inverse; });
            of_channels<V>(l, p, means, mean);
#pragma unroll
            for (int r = 0; r < R; ++r) as_loaded(held[r]);
#pragma unroll
            for (int e = 0; e < V; ++e) sum[e] = 0.0f;
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (r < here) {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float d = (float)held[r][e] - mean[e];
                        sum[e] = __builtin_fmaf(d, d, sum[e]);
                    }
                }
#pragma unroll
            for (int e = 0; e < V; ++e) sum[e] = e < p.n ? sum[e] : 0.0f;
            group_sums<V>(l, p, sum, scratch[1], scales, [&](float s) { return 1.0f / sqrtf(__builtin_fmaf(s, inverse, a.eps)); });
            of_channels<V>(l, p, scales, scale);
#pragma unroll
            for (int e = 0; e < V; ++e) scale[e] *= weight[e];
#pragma unroll
            for (int r = 0; r < R; ++r) as_loaded(held[r]);
            T* y = static_cast<T*>(a.y) + i * a.y_n + p.row * a.y_p + p.c;
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (r < here) {
                    float v[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        v[e] = __builtin_fmaf((float)held[r][e] - mean[e], scale[e], bias[e]);
                        if constexpr (SKIP) v[e] += (float)skip[r][e];
                    }
                    activate(v, a.activation);
                    store_part<T, V>(y, p.n, v);
                    y += l.rows * a.y_p;
                }
        }
}

// What is known of some of a group's values.
struct Moments {
    float mean, squares;                                        // squares: sum of squared differences from the mean
};

// (mean, squares) of a share of the positions of a slab's groups, to moments[sample][group][share][sub].  Every thread joins what it reads as it
// comes, channel by channel; the threads of a group are joined at the end.
template <typename T>
__global__ __launch_bounds__(kMaxThreads)
void moments_kernel(dgnn_group_norm_args a, Layout l, Moments* moments)
{
    constexpr int V = width_of<T>, R = kRegisters;
    __shared__ float scratch[2][kMaxThreads * V], means[kMaxGroups], squares[kMaxGroups];
    const int64_t begin = blockIdx.y * l.share, end = begin + l.share < a.p ? begin + l.share : a.p;
    for (int64_t i = blockIdx.z; i < a.n; i += gridDim.z)
        for (int slab = blockIdx.x; slab < l.slabs; slab += gridDim.x) {
            const Part p = part_of<V>(l, (int)a.groups, slab);
            const float inverse = 1.0f / ((float)(end - begin) * (float)(l.subs > 1 ? p.channels : l.per));
            float mean[V] = {}, square[V] = {}, count = 0.0f;
            if (p.row >= 0)
                for (int64_t q = begin + p.row; q < end; q += R * l.rows) {
                    const T* x = static_cast<const T*>(a.x) + i * a.x_n + q * a.x_p + p.c;
                    const int here = end - q > (R - 1) * l.rows ? R : (int)(end - 1 - q) / l.rows + 1;
                    vec<T, V> held[R];
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        held[r] = r < here ? load_part<T, V>(x, p.n) : vec<T, V>{};
                        x += l.rows * a.x_p;
                    }
                    const float each = 1.0f / (float)here, all = count + (float)here, part = (float)here / all, between = count * part;
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        float s = 0.0f, m2 = 0.0f;
#pragma unroll
                        for (int r = 0; r < R; ++r) s += (float)held[r][e];
                        const float m = s * each;
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            const float d = r < here ? (float)held[r][e] - m : 0.0f;
                            m2 = __builtin_fmaf(d, d, m2);
                        }
                        const float d = m - mean[e];
                        mean[e] = __builtin_fmaf(d, part, mean[e]);
                        square[e] += __builtin_fmaf(d * d, between, m2);
                    }
                    count = all;
                }
            float mine[V], joint[V];
#pragma unroll
            for (int e = 0; e < V; ++e) mine[e] = e < p.n ? mean[e] * count : 0.0f;
            group_sums<V>(l, p, mine, scratch[0], means, [&](float s) { return s * inverse; });
            of_channels<V>(l, p, means, joint);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = mean[e] - joint[e];
                mine[e] = e < p.n ? __builtin_fmaf(d * d, count, square[e]) : 0.0f;
            }
            group_sums<V>(l, p, mine, scratch[1], squares, [&](float s) { return s; });
            for (int g = threadIdx.x; g < p.groups; g += blockDim.x)
                moments[((i * a.groups + p.g0 + g) * l.shares + blockIdx.y) * l.subs + p.sub] = Moments{means[g], squares[g]};
            __syncthreads();                                    // (means and squares are the next slab's)
        }
}

template <typename T, bool SKIP>
__global__ __launch_bounds__(kMaxThreads)
void apply_kernel(dgnn_group_norm_args a, Layout l, const Moments* moments)
{
    constexpr int V = width_of<T>, R = kRegisters / 2;
    __shared__ float means[kMaxGroups], scales[kMaxGroups];
    const int64_t begin = blockIdx.y * l.share, end = begin + l.share < a.p ? begin + l.share : a.p;
    const int pieces = l.shares * l.subs, waves = (int)(blockDim.x + 63) >> 6;
    const float inverse = 1.0f / ((float)a.p * (float)l.per);
    for (int64_t i = blockIdx.z; i < a.n; i += gridDim.z)
        for (int slab = blockIdx.x; slab < l.slabs; slab += gridDim.x) {
            const Part p = part_of<V>(l, (int)a.groups, slab);
            for (int g = threadIdx.x >> 6; g < p.groups; g += waves) {
                const Moments* const of = moments + (i * a.groups + p.g0 + g) * pieces;
                const auto count = [&](int piece) {
                    const int share = piece / l.subs, from = (piece - share * l.subs) * kMaxVectors * V;
                    const int64_t left = a.p - share * l.share;
                    const int wide = l.subs == 1 || l.per - from < kMaxVectors * V ? l.per - from : kMaxVectors * V;
                    return (float)(left < l.share ? left : l.share) * (float)wide;
                };
                float sum = 0.0f, squares = 0.0f;
                for (int piece = threadIdx.x & 63; piece < pieces; piece += 64) sum = __builtin_fmaf(of[piece].mean, count(piece), sum);
                const float mean = wave_sum(sum) * inverse;
                for (int piece = threadIdx.x & 63; piece < pieces; piece += 64) {
                    const float d = of[piece].mean - mean;
                    squares += __builtin_fmaf(d * d, count(piece), of[piece].squares);
                }
                squares = wave_sum(squares);
                if ((threadIdx.x & 63) == 0) means[g] = mean, scales[g] = 1.0f / sqrtf(__builtin_fmaf(squares, inverse, a.eps));
            }
            __syncthreads();
            float weight[V], bias[V], mean[V], scale[V];
            load_affine<T, V>(a.weight, a.affine_type == DGNN_F32, p.c, p.n, 1.0f, weight);
            load_affine<T, V>(a.bias, a.affine_type == DGNN_F32, p.c, p.n, 0.0f, bias);
            of_channels<V>(l, p, means, mean);
            of_channels<V>(l, p, scales, scale);
#pragma unroll
            for (int e = 0; e < V; ++e) scale[e] *= weight[e];
            __syncthreads();                                    // (means and scales are the next slab's)
            if (p.row < 0) continue;
            for (int64_t q = begin + p.row; q < end; q += R * l.rows) {
                const T* x = static_cast<const T*>(a.x) + i * a.x_n + q * a.x_p + p.c;
                const T* z = SKIP ? static_cast<const T*>(a.z) + i * a.z_n + q * a.z_p + p.c : nullptr;
                T* y = static_cast<T*>(a.y) + i * a.y_n + q * a.y_p + p.c;
                const int here = end - q > (R - 1) * l.rows ? R : (int)(end - 1 - q) / l.rows + 1;
                vec<T, V> held[R], skip[SKIP ? R : 1];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    held[r] = r < here ? load_part<T, V>(x, p.n) : vec<T, V>{};
                    x += l.rows * a.x_p;
                    if constexpr (SKIP) {
                        skip[r] = r < here ? load_part<T, V>(z, p.n) : vec<T, V>{};
                        z += l.rows * a.z_p;
                    }
                }
#pragma unroll
                for (int r = 0; r < R; ++r)
                    if (r < here) {
                        float v[V];
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            v[e] = __builtin_fmaf((float)held[r][e] - mean[e], scale[e], bias[e]);
                            if constexpr (SKIP) v[e] += (float)skip[r][e];
                        }
                        activate(v, a.activation);
                        store_part<T, V>(y, p.n, v);
                        y += l.rows * a.y_p;
                    }
            }
        }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Groups that make lines of 128 bytes where that is possible within a slab, as few as that takes; otherwise about a line.
int64_t groups_of_whole_lines(int64_t per, int64_t groups, int64_t vector)
{
    const int64_t line = vector * 8;
    int64_t g = 1;
    while (g * per % line != 0 && g < line) g *= 2;
    if (g * per % line == 0 && g <= groups && g * per <= kMaxVectors * vector) return g;
    if (groups * per <= kMaxVectors * vector) return groups;
    return line / per > 1 ? line / per : 1;
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
    int64_t groups = l.subs > 1 ? 1 : groups_of_whole_lines(l.per, a.groups, vector);
    const int64_t whole = groups;
    const auto cut = [&]() {
        l.groups_per_slab = (int)groups;
        l.slabs = (int)(l.subs > 1 ? a.groups * l.subs : ceil_div(a.groups, groups));
        l.lanes = (int)(l.subs > 1 ? kMaxVectors : ceil_div(groups * l.per, vector));
    };
    cut();
    // rows that a workgroup holds: 512 threads of eight vectors each, or 1024 of four
    const auto held = [&]() { return (int64_t)(kMaxThreads / 2 / l.lanes) * kRegisters; };
    *registers = 0;
    if (l.subs == 1) {
        // narrower slabs where these leave compute units idle, or do not fit and two vectors of a line would
        while (groups > 1 && a.n * l.slabs < kUnitsWanted) groups = (groups + 1) / 2, cut();
        while (groups > 1 && groups * l.per > 2 * vector && a.p > held()) groups = (groups + 1) / 2, cut();
        if (a.p <= held()) {
            // many vectors to a thread where there are enough workgroups for several on a unit, few where a call is one trip through the chip
            const int wanted = a.n * l.slabs >= 2 * kUnitsWanted ? kRegisters : 2;
            l.threads = 64;
            while (l.threads < kMaxThreads / (wanted == kRegisters ? 2 : 1) && (l.threads < l.lanes || (int64_t)(l.threads / l.lanes) * wanted < a.p)) l.threads *= 2;
            l.rows = l.threads / l.lanes;
            const int64_t each = ceil_div(a.p, l.rows);
            *registers = each <= 2 ? 2 : each <= 4 ? 4 : 8;
            return l;
        }
        groups = whole;
        cut();
    }
    l.threads = kMaxThreads;
    l.rows = l.threads / l.lanes;
    // shares enough for two workgroups on every unit, of whole trips through the registers
    const int64_t trip = (int64_t)l.rows * kRegisters, trips = ceil_div(a.p, trip);
    int64_t shares = ceil_div(2 * kUnitsWanted, a.n * l.slabs);
    shares = shares > kMaxShares ? kMaxShares : shares > trips ? trips : shares;
    l.share = ceil_div(trips, shares) * trip;
    l.shares = (int)ceil_div(a.p, l.share);
    return l;
}

template <typename T>
hipError_t launch_typed(const dgnn_group_norm_args& a, hipStream_t stream)
{
    int registers;
    const Layout l = make_layout(a, &registers);
    const dim3 grid((unsigned)(l.slabs < 65536 ? l.slabs : 65536), (unsigned)l.shares, (unsigned)(a.n < 32768 ? a.n : 32768)), block(l.threads);
    switch (registers) {
    case 2: return a.z ? launch(one_pass_kernel<T, 2, true>, grid, block, stream, a, l) : launch(one_pass_kernel<T, 2, false>, grid, block, stream, a, l);
    case 4: return a.z ? launch(one_pass_kernel<T, 4, true>, grid, block, stream, a, l) : launch(one_pass_kernel<T, 4, false>, grid, block, stream, a, l);
    case 8: return a.z ? launch(one_pass_kernel<T, 8, true>, grid, block, stream, a, l) : launch(one_pass_kernel<T, 8, false>, grid, block, stream, a, l);
    }
    Moments* const moments = static_cast<Moments*>(a.workspace);
    const hipError_t err = launch(moments_kernel<T>, grid, block, stream, a, l, moments);
    if (err != hipSuccess) return err;
    const Moments* const done = moments;
    return a.z ? launch(apply_kernel<T, true>, grid, block, stream, a, l, done) : launch(apply_kernel<T, false>, grid, block, stream, a, l, done);
}

}  // namespace

int64_t group_norm_workspace(const dgnn_group_norm_args& a)
{
    int registers;
    const Layout l = make_layout(a, &registers);
    return registers ? 0 : a.n * a.groups * l.shares * l.subs * (int64_t)sizeof(Moments);
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
