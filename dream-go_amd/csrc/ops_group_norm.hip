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
    int back;               // how far back a whole vector has to begin to end inside the row
};

template <int V>
__device__ __forceinline__ Part part_of(const Layout& l, int channels, int groups, int slab)
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
    p.back = p.c + V <= channels ? 0 : p.c + V - channels;
    return p;
}

// The vector `n` elements on: element e of what is returned is element e + n, n < V.
template <typename T, int V>
__device__ __forceinline__ vec<T, V> moved_down(vec<T, V> v, int n)
{
    typedef vec<unsigned, 4> Words;
    Words w = __builtin_bit_cast(Words, v);
    const unsigned bytes = n * sizeof(T) & 3;
    if (n * (int)sizeof(T) & 8) w = Words{w[2], w[3], 0, 0};
    if (n * (int)sizeof(T) & 4) w = Words{w[1], w[2], w[3], 0};
    if (bytes) w = Words{__builtin_amdgcn_alignbyte(w[1], w[0], bytes), __builtin_amdgcn_alignbyte(w[2], w[1], bytes), __builtin_amdgcn_alignbyte(w[3], w[2], bytes), w[3] >> bytes * 8};
    return __builtin_bit_cast(vec<T, V>, w);
}

// The thread's part of `here` rows (R at most), `step` elements apart; zeros behind a part's end and for the other rows.  All loads first, then
// what makes them parts: the loads of a thread are on their way at once.  TINY: no row is as long as a vector.
template <typename T, int R, int V, bool TINY>
__device__ __forceinline__ void load_rows(const T* p, int64_t step, int here, const Part& part, vec<T, V> (&held)[R])
{
    if constexpr (TINY) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int e = 0; e < V; ++e) held[r][e] = r < here && e < part.n ? p[e] : (T)0.0f;
            p += step;
        }
        return;
    }
    p -= part.back;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        held[r] = r < here ? load_vec<T, V>(p) : vec<T, V>{};
        p += step;
    }
    if (part.n < V) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (part.back > 0) held[r] = moved_down<T, V>(held[r], part.back);
#pragma unroll
            for (int e = 0; e < V; ++e) held[r][e] = e < part.n ? held[r][e] : (T)0.0f;
        }
    }
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
__device__ __forceinline__ void load_affine(const void* from, bool is_float, const Part& p, float otherwise, float (&v)[V])
{
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = otherwise;
    if (!from || p.n <= 0) return;
    if (p.back == 0) {                                          // (of the channels behind the part nothing is used)
        if (is_float) {
            const vec<float, V> all = load_vec<float, V>(static_cast<const float*>(from) + p.c);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = all[e];
        } else {
            const vec<T, V> all = load_vec<T, V>(static_cast<const T*>(from) + p.c);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = (float)all[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < p.n) v[e] = load_either<T>(from, p.c + e, is_float);
    }
}

// One number of every group of the slab for each channel of the thread's vector.
template <int V>
__device__ __forceinline__ void of_channels(const Layout& l, const Part& p, const float* of_group, float (&v)[V])
{
    if (l.groups_per_slab == 1 || l.per % V == 0) {
        const float all = of_group[l.groups_per_slab == 1 ? 0 : p.at / l.per];
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
__device__ __forceinline__ void group_sums(const Layout& l, const Part& p, float (&mine)[V], float* scratch, float* out, Last last)
{
    // a vector, or the whole slab, lies in one group: one number of each thread is enough
    const bool single = l.groups_per_slab == 1 || l.per % V == 0;
    // rows of a power of two are added up within each wave first
    const bool even = (l.lanes & (l.lanes - 1)) == 0 && l.lanes <= 64;
    const int waves = (int)(blockDim.x + 63) >> 6, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int mine_at = even ? wave * l.lanes + lane : threadIdx.x;
    if (single) {
        float all[1] = {mine[0]};
#pragma unroll
        for (int e = 1; e < V; ++e) all[0] += mine[e];
        if (even) periodic_sums(all, l.lanes);
        if (!even || lane < l.lanes) scratch[mine_at] = all[0];
    } else {
        if (even) periodic_sums(mine, l.lanes);
        if (!even || lane < l.lanes) {
#pragma unroll
            for (int e = 0; e < V; ++e) scratch[mine_at * V + e] = mine[e];
        }
    }
    __syncthreads();
    const int rows = even ? waves : l.rows, pitch = single ? l.lanes : l.lanes * V, n = l.groups_per_slab == 1 ? l.lanes : single ? l.per / V : l.per;
    const int down = 64 / n, across = 64 - down * n;            // 64 numbers on (n is 512 at most: down may be 0)
    for (int g = wave; g < p.groups; g += waves) {
        const float* const of = scratch + g * n;
        float sum = 0.0f;
        int row = lane / n, column = lane - row * n;
        while (row < rows) {
            float four[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                four[q] = row < rows ? of[row * pitch + column] : 0.0f;
                row += down;
                column += across;
                if (column >= n) column -= n, ++row;
            }
            sum += (four[0] + four[1]) + (four[2] + four[3]);
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
template <typename T, int R, Kind K, bool SKIP, bool TINY>
__global__ __launch_bounds__(R == kRegisters ? kMaxThreads / 2 : kMaxThreads, 4)
void one_pass_kernel(dgnn_group_norm_args a, Layout l)
{
    constexpr int V = width_of<T>;
    __shared__ float scratch[2][kMaxThreads * V], means[kMaxGroups], scales[kMaxGroups];
    const float inverse = 1.0f / ((float)a.p * (float)l.per);
    for (int64_t i = blockIdx.z; i < a.n; i += gridDim.z)
        for (int slab = blockIdx.x; slab < l.slabs; slab += gridDim.x) {
            const Part p = part_of<V>(l, (int)a.c, (int)a.groups, slab);
            const int here = p.row < 0 || p.row >= a.p ? 0 : (int)(a.p - 1 - p.row) / l.rows + 1;    // positions of this thread
            const T* const x = static_cast<const T*>(a.x) + i * a.x_n + p.row * a.x_p + p.c;
            vec<T, V> held[R], skip[SKIP ? R : 1];
            load_rows<T, R, V, TINY>(x, l.rows * a.x_p, here, p, held);
            if constexpr (SKIP) load_rows<T, R, V, TINY>(static_cast<const T*>(a.z) + i * a.z_n + p.row * a.z_p + p.c, l.rows * a.z_p, here, p, skip);
            float weight[V], bias[V], sum[V] = {}, mean[V], scale[V];
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
            load_affine<T, V>(a.weight, a.affine_type == DGNN_F32, p, 1.0f, weight);
            load_affine<T, V>(a.bias, a.affine_type == DGNN_F32, p, 0.0f, bias);
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
                    activate_kind<K>(v, a.activation);
                    store_part<T, V>(y, p.n, v);
                    y += l.rows * a.y_p;
                }
        }
}

// What is known of some of a group's values.
struct Moments {
    float mean, squares;                                        // squares: sum of squared differences from the mean
};

// (mean, squares) of a share of the positions of a slab's groups, to moments[sample][group][share][sub].
//
// Each thread sums, channel by channel, the differences of its rows from its FIRST row and their squares: four operations a value, where a second
// look at the values would take six, and this kernel is bound by them as much as by memory.  The shift is one of the n values it is taken from, so
// n (mean - shift)^2 is less than n times the sum of squares about the mean, whatever the values are: n times a rounding is all that the
// difference `square - sum^2 / n` can lose.  The threads of a group are then joined about their common mean.
template <typename T, bool TINY>
__global__ __launch_bounds__(kMaxThreads / 2, 4)
void moments_kernel(dgnn_group_norm_args a, Layout l, Moments* moments)
{
    constexpr int V = width_of<T>, R = kRegisters;
    __shared__ float scratch[2][kMaxThreads / 2 * V], means[kMaxGroups], squares[kMaxGroups];
    const int64_t begin = blockIdx.y * l.share, end = begin + l.share < a.p ? begin + l.share : a.p;
    for (int64_t i = blockIdx.z; i < a.n; i += gridDim.z)
        for (int slab = blockIdx.x; slab < l.slabs; slab += gridDim.x) {
            const Part p = part_of<V>(l, (int)a.c, (int)a.groups, slab);
            const float inverse = 1.0f / ((float)(end - begin) * (float)(l.subs > 1 ? p.channels : l.per));
            const int rows = (int)(end - begin), here = p.row < 0 || p.row >= rows ? 0 : (rows - 1 - p.row) / l.rows + 1;
            float shift[V] = {}, sum[V] = {}, square[V] = {};
            if (here > 0) {
                const int64_t step = l.rows * a.x_p;
                const T* x = static_cast<const T*>(a.x) + i * a.x_n + (begin + p.row) * a.x_p + p.c;
                vec<T, V> first[1];
                load_rows<T, 1, V, TINY>(x, step, 1, p, first);
#pragma unroll
                for (int e = 0; e < V; ++e) shift[e] = (float)first[0][e];
                int done = 0;
                for (; done + R <= here; done += R) {
                    vec<T, V> held[R];
                    load_rows<T, R, V, TINY>(x, step, R, p, held);
                    x += R * step;
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            const float d = (float)held[r][e] - shift[e];
                            sum[e] += d;
                            square[e] = __builtin_fmaf(d, d, square[e]);
                        }
                }
                if (done < here) {
                    vec<T, V> held[R];
                    load_rows<T, R, V, TINY>(x, step, here - done, p, held);
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        if (done + r < here) {
#pragma unroll
                            for (int e = 0; e < V; ++e) {
                                const float d = (float)held[r][e] - shift[e];
                                sum[e] += d;
                                square[e] = __builtin_fmaf(d, d, square[e]);
                            }
                        }
                }
            }
            const float count = (float)here, each = here > 0 ? 1.0f / count : 0.0f;
            float mean[V], mine[V], joint[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float about = sum[e] * each;
                square[e] = __builtin_fmaf(-about, sum[e], square[e]);
                square[e] = square[e] < 0.0f ? 0.0f : square[e];       // (a NaN stays)
                mean[e] = shift[e] + about;
                mine[e] = e < p.n ? mean[e] * count : 0.0f;
            }
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

template <typename T, Kind K, bool SKIP, bool TINY>
__global__ __launch_bounds__(kMaxThreads / 2, 4)
void apply_kernel(dgnn_group_norm_args a, Layout l, const Moments* moments)
{
    constexpr int V = width_of<T>, R = 2;
    __shared__ float means[kMaxGroups], scales[kMaxGroups];
    const int64_t begin = blockIdx.y * l.share, end = begin + l.share < a.p ? begin + l.share : a.p;
    const int pieces = l.shares * l.subs, waves = (int)(blockDim.x + 63) >> 6;
    const float inverse = 1.0f / ((float)a.p * (float)l.per);
    for (int64_t i = blockIdx.z; i < a.n; i += gridDim.z)
        for (int slab = blockIdx.x; slab < l.slabs; slab += gridDim.x) {
            const Part p = part_of<V>(l, (int)a.c, (int)a.groups, slab);
            for (int g = threadIdx.x >> 6; g < p.groups; g += waves) {
                const Moments* const of = moments + (i * a.groups + p.g0 + g) * pieces;
                const auto count = [&](int piece) {
                    const int share = piece / l.subs, from = (piece - share * l.subs) * kMaxVectors * V;
                    const int64_t left = a.p - share * l.share;
                    const int wide = l.subs == 1 || l.per - from < kMaxVectors * V ? l.per - from : kMaxVectors * V;
                    return (float)(left < l.share ? left : l.share) * (float)wide;
                };
                // four of a lane's pieces at a time, asked for together; up to 256 pieces are still there for the second sum
                Moments m[4];
                float c[4], sum = 0.0f, squares = 0.0f;
                const auto fetch = [&](int base) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int piece = base + q * 64 + (threadIdx.x & 63);
                        m[q] = piece < pieces ? of[piece] : Moments{0.0f, 0.0f};
                        c[q] = piece < pieces ? count(piece) : 0.0f;
                    }
                };
                for (int base = 0; base < pieces; base += 256) {
                    fetch(base);
#pragma unroll
                    for (int q = 0; q < 4; ++q) sum = __builtin_fmaf(m[q].mean, c[q], sum);
                }
                const float mean = wave_sum(sum) * inverse;
                for (int base = 0; base < pieces; base += 256) {
                    if (pieces > 256) fetch(base);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float d = m[q].mean - mean;
                        squares += __builtin_fmaf(d * d, c[q], m[q].squares);
                    }
                }
                squares = wave_sum(squares);
                if ((threadIdx.x & 63) == 0) means[g] = mean, scales[g] = 1.0f / sqrtf(__builtin_fmaf(squares, inverse, a.eps));
            }
            __syncthreads();
            float weight[V], bias[V], mean[V], scale[V];
            load_affine<T, V>(a.weight, a.affine_type == DGNN_F32, p, 1.0f, weight);
            load_affine<T, V>(a.bias, a.affine_type == DGNN_F32, p, 0.0f, bias);
            of_channels<V>(l, p, means, mean);
            of_channels<V>(l, p, scales, scale);
#pragma unroll
            for (int e = 0; e < V; ++e) scale[e] *= weight[e];
            __syncthreads();                                    // (means and scales are the next slab's)
            if (p.row < 0) continue;
            for (int64_t q = begin + p.row; q < end; q += R * l.rows) {
                const T* const x = static_cast<const T*>(a.x) + i * a.x_n + q * a.x_p + p.c;
                T* y = static_cast<T*>(a.y) + i * a.y_n + q * a.y_p + p.c;
                const int here = end - q > (R - 1) * l.rows ? R : (int)(end - 1 - q) / l.rows + 1;
                vec<T, V> held[R], skip[SKIP ? R : 1];
                load_rows<T, R, V, TINY>(x, l.rows * a.x_p, here, p, held);
                if constexpr (SKIP) load_rows<T, R, V, TINY>(static_cast<const T*>(a.z) + i * a.z_n + q * a.z_p + p.c, l.rows * a.z_p, here, p, skip);
#pragma unroll
                for (int r = 0; r < R; ++r)
                    if (r < here) {
                        float v[V];
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            v[e] = __builtin_fmaf((float)held[r][e] - mean[e], scale[e], bias[e]);
                            if constexpr (SKIP) v[e] += (float)skip[r][e];
                        }
                        activate_kind<K>(v, a.activation);
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
    constexpr int kThreads = kMaxThreads / 2;                   // (1024 of four vectors hold what 512 of eight do)
    const int vector = a.type == DGNN_F32 ? 4 : 8;
    Layout l;
    l.per = (int)(a.c / a.groups);
    l.shares = 1;
    l.share = a.p;
    int64_t groups;
    const auto cut = [&](int64_t g, int subs) {
        groups = g;
        l.subs = subs;
        l.groups_per_slab = (int)groups;
        l.slabs = (int)(subs > 1 ? a.groups * subs : ceil_div(a.groups, groups));
        l.lanes = (int)(subs > 1 ? kMaxVectors : ceil_div(groups * l.per, vector));
    };
    const auto held = [&]() { return (int64_t)(kThreads / l.lanes) * kRegisters; };
    cut(groups_of_whole_lines(l.per, a.groups, vector), 1);
    const int64_t whole = groups;
    *registers = 0;
    // narrower slabs where these leave compute units idle, or do not fit and two vectors of a line would
    while (groups > 1 && a.n * l.slabs < kUnitsWanted) cut((groups + 1) / 2, 1);
    while (groups > 1 && groups * l.per > 2 * vector && a.p > held()) cut((groups + 1) / 2, 1);
    if (a.p <= held()) {
        // as many vectors to a thread as give every unit 1024 of them: few where a call is one trip through the chip
        const int64_t each_unit = a.n * l.slabs * l.lanes * a.p / (kUnitsWanted * kMaxThreads);
        const int wanted = each_unit >= 6 ? kRegisters : each_unit >= 3 ? 4 : 2, most = wanted == kRegisters ? kThreads : kMaxThreads;
        l.threads = 64;
        while (l.threads < most && (l.threads < l.lanes || (int64_t)(l.threads / l.lanes) * wanted < a.p)) l.threads *= 2;
        l.rows = l.threads / l.lanes;
        const int64_t each = ceil_div(a.p, l.rows);
        *registers = each <= 2 ? 2 : each <= 4 ? 4 : 8;
        return l;
    }
    const int subs = (int)ceil_div(l.per, kMaxVectors * vector);
    cut(subs > 1 ? 1 : whole, subs);
    l.threads = kThreads;
    l.rows = l.threads / l.lanes;
    // shares enough for two workgroups on every unit
    int64_t shares = ceil_div(2 * kUnitsWanted, a.n * l.slabs);
    if (shares > kMaxShares) shares = kMaxShares;
    l.share = ceil_div(ceil_div(a.p, shares), l.rows) * l.rows;
    l.shares = (int)ceil_div(a.p, l.share);
    return l;
}

template <typename T, Kind K, bool SKIP, bool TINY>
hipError_t launch_kind(const dgnn_group_norm_args& a, hipStream_t stream)
{
    int registers;
    const Layout l = make_layout(a, &registers);
    const dim3 grid((unsigned)(l.slabs < 65536 ? l.slabs : 65536), (unsigned)l.shares, (unsigned)(a.n < 32768 ? a.n : 32768)), block(l.threads);
    if (registers == 2) return launch(one_pass_kernel<T, 2, K, SKIP, TINY>, grid, block, stream, a, l);
    if (registers == 4) return launch(one_pass_kernel<T, 4, K, SKIP, TINY>, grid, block, stream, a, l);
    if (registers == 8) return launch(one_pass_kernel<T, 8, K, SKIP, TINY>, grid, block, stream, a, l);
    Moments* const moments = static_cast<Moments*>(a.workspace);
    const hipError_t err = launch(moments_kernel<T, TINY>, grid, block, stream, a, l, moments);
    return err != hipSuccess ? err : launch(apply_kernel<T, K, SKIP, TINY>, grid, block, stream, a, l, static_cast<const Moments*>(moments));
}

template <typename T, bool SKIP>
hipError_t launch_skip(const dgnn_group_norm_args& a, hipStream_t stream)
{
    if (a.c < width_of<T>) return launch_kind<T, kAny, SKIP, true>(a, stream);
    if (a.activation == DGNN_ACT_IDENTITY || a.activation == DGNN_ACT_RELU) return launch_kind<T, kPlain, SKIP, false>(a, stream);
    if (a.activation == DGNN_ACT_SILU) return launch_kind<T, kSilu, SKIP, false>(a, stream);
    return launch_kind<T, kAny, SKIP, false>(a, stream);
}

template <typename T>
hipError_t launch_type(const dgnn_group_norm_args& a, hipStream_t stream)
{
    return a.z ? launch_skip<T, true>(a, stream) : launch_skip<T, false>(a, stream);
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
    case DGNN_F16: return launch_type<f16>(a, stream);
    case DGNN_BF16: return launch_type<bf16>(a, stream);
    default: return launch_type<float>(a, stream);
    }
}

}  // namespace ops
}  // namespace dgnn
