// dgnn_group_norm: group norm over channels-last maps, the skip input and the activation applied on the way out.
//
// A workgroup owns a slab of channels of one sample -- whole groups, up to 64 sixteen-byte vectors -- and all positions, or a share of them.
// Threads are laid over (position, vector), so that neighbours read what lies side by side.
//
//   one pass   a sample's slab fits the registers of a workgroup: read once, written once, which is the floor.  Mean and variance are two passes over
//              values that are in registers: the variance is the mean of squared differences from the mean and costs no second read
//   two        it does not: a first kernel leaves (mean, sum of squares about it) of every share of the positions, gathered eight rows at a time
//              about the mean of the rows before (moments_kernel says what that loses); a second joins those of its groups -- about their joint
//              mean, in a fixed order -- and reads the maps again, mostly out of the last-level cache
//
// Large maps are bound by memory on both ways; the activations are branch-free for that reason (ops_device.h).  256 maps of 361 x 256 fp16 with a
// skip (142 MB) take 32.5 us in one pass, 4.4 TB/s; 8 maps of 16384 x 320 bf16 with SiLU (168 MB, its input read twice) 58 us in two, 2.9 TB/s
// of what has to move.  Small ones are bound by the chain of waits and by what a thread does beside its values: one map of 361 x 64 takes 5.9 us, of
// which an empty kernel's launch is about 2.5, and 13 of 1021 x 90 fp32 12.9.  Kernels are made for what a call's sizes promise (Shape) because of the latter: vectors of one
// group each need one sum where others need eight, whole ones no masks (one map of 361 x 256: 5.8 us, 6.4 without the distinction; 383 maps of
// 15 x 128: 10.7 us, 20.6 -- that one because LDS is now asked for as needed, not for the largest workgroup).
#include "ops_device.h"

namespace dgnn {
namespace ops {
namespace {

constexpr int kMaxThreads = 1024, kMaxVectors = 64, kRegisters = 8;     // vectors of a row of a slab; vectors of a thread
constexpr int kMaxGroups = kMaxVectors * 8;                             // of a slab
constexpr int kMaxShares = 256;                                         // of a sample's positions, where these are not more than
constexpr int kSerialRows = 2048;                                       // a thread adds up one after the other
constexpr int kUnitsWanted = 256;                                       // workgroups that give every compute unit one

template <typename T> constexpr int width_of = 16 / (int)sizeof(T);     // elements of a vector

// What a call's sizes promise its kernels: vectors of one group each; whole vectors; nothing; rows shorter than a vector.
enum Shape { kAligned, kWhole, kRagged, kTiny };

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
    int scratch;            // floats that group_sums needs
};

// The part of a slab that a thread works on.
struct Part {
    int g0, groups, sub;    // the slab's groups; which of a wide group's slabs it is
    int channels;           // of the slab
    int row;                // of the workgroup's rows; -1: this thread has no part
    int at, c, n;           // first channel in the slab and of all, channels (fewer than a vector at the end of a slab)
    int back;               // how far back a whole vector has to begin to end inside the row
};

template <Shape S, int V>
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
    p.n = p.channels - p.at < V ? p.channels - p.at : V;
    p.row = row < l.rows && p.n > 0 ? row : -1;
    if (p.row < 0) p.at = p.n = 0;
    p.c = c0 + p.at;
    p.back = S <= kWhole ? 0 : overhang(p.c, V, channels);
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
// what makes them parts: the loads of a thread are on their way at once.
template <Shape S, typename T, int R, int V>
__device__ __forceinline__ void load_rows(const T* p, int64_t step, int here, const Part& part, vec<T, V> (&held)[R])
{
    if constexpr (S == kTiny) {
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
    if (S == kRagged && part.n < V) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (part.back > 0) held[r] = moved_down<T, V>(held[r], part.back);
#pragma unroll
            for (int e = 0; e < V; ++e) held[r][e] = e < part.n ? held[r][e] : (T)0.0f;
        }
    }
}

template <Shape S, typename T, int V>
__device__ __forceinline__ void store_part(T* p, int n, const float (&v)[V])
{
    vec<T, V> out;
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = (T)v[e];
    if (S <= kWhole || n == V) return store_vec<T, V>(p, out);
#pragma unroll
    for (int e = 0; e < V; ++e)
        if (e < n) p[e] = out[e];
}

template <Shape S, typename T, int V>
__device__ __forceinline__ void load_affine(const void* from, bool is_float, const Part& p, float otherwise, float (&v)[V])
{
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = otherwise;
    if (!from || p.n <= 0) return;
    if (S <= kWhole || p.back == 0) {                                          // (of the channels behind the part nothing is used)
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
template <Shape S, int V>
__device__ __forceinline__ void of_channels(const Layout& l, const Part& p, const float* of_group, float (&v)[V])
{
    if (S == kAligned || (S != kWhole && l.groups_per_slab == 1)) {
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
template <Shape S, int V, typename Last>
__device__ __forceinline__ void group_sums(const Layout& l, const Part& p, float (&mine)[V], float* scratch, float* out, Last last)
{
    // a vector, or the whole slab, lies in one group: one number of each thread is enough
    const bool single = S == kAligned || (S != kWhole && l.groups_per_slab == 1);
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
template <Shape S, typename T, int R, Kind K, bool SKIP>
__global__ __launch_bounds__(R == kRegisters ? kMaxThreads / 2 : kMaxThreads, 4)
void one_pass_kernel(dgnn_group_norm_args a, Layout l)
{
    constexpr int V = width_of<T>;
    extern __shared__ float scratch[];
    float* const means = scratch + 2 * l.scratch;
    float* const scales = means + l.groups_per_slab;
    const float inverse = 1.0f / ((float)a.p * (float)l.per);
    for (int64_t i = blockIdx.z; i < a.n; i += gridDim.z)
        for (int slab = blockIdx.x; slab < l.slabs; slab += gridDim.x) {
            const Part p = part_of<S, V>(l, (int)a.c, (int)a.groups, slab);
            const int here = p.row < 0 || p.row >= a.p ? 0 : (int)(a.p - 1 - p.row) / l.rows + 1;    // positions of this thread
            const T* const x = static_cast<const T*>(a.x) + i * a.x_n + p.row * a.x_p + p.c;
            vec<T, V> held[R], skip[SKIP ? R : 1];
            load_rows<S, T, R, V>(x, l.rows * a.x_p, here, p, held);
            if constexpr (SKIP) load_rows<S, T, R, V>(static_cast<const T*>(a.z) + i * a.z_n + p.row * a.z_p + p.c, l.rows * a.z_p, here, p, skip);
            float weight[V], bias[V], sum[V] = {}, mean[V], scale[V];
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < V; ++e) sum[e] += (float)held[r][e];
            group_sums<S, V>(l, p, sum, scratch, means, [&](float s) { return s * inverse; });
            of_channels<S, V>(l, p, means, mean);
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
            group_sums<S, V>(l, p, sum, scratch + l.scratch, scales, [&](float s) { return 1.0f / sqrtf(__builtin_fmaf(s, inverse, a.eps)); });
            load_affine<S, T, V>(a.weight, a.affine_type == DGNN_F32, p, 1.0f, weight);
            load_affine<S, T, V>(a.bias, a.affine_type == DGNN_F32, p, 0.0f, bias);
            of_channels<S, V>(l, p, scales, scale);
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
                    activate_kind<K, T>(v, a.activation);
                    store_part<S, T, V>(y, p.n, v);
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
// Each thread takes its rows by eights and sums, channel by channel, their differences from the mean of the rows BEFORE them (the first eight: from
// its first row) and the squares of those: four operations a value, where a second look at the values would take six, and this kernel is bound by them
// as much as by memory.  With s and q the two sums, m the mean of n - 8 rows and n those with the eight, the rows join as
//   mean = m + s / n,   squares about it += q - s^2 / n,
// in which s^2 / n is at most half of q (s^2 <= 8 q, n >= 16): a difference that loses one bit at most, whatever the rows are.  For the first eight
// the shift is one of the values themselves, 8 (mean - shift)^2 is at most eight times the sum of squares about the mean, and the difference loses
// a few.  No sum runs over more than kSerialRows / 8 joins (make_layout), each of them a few half steps of fp32.  The threads of a group are then
// joined about their common mean.
template <Shape S, typename T>
__global__ __launch_bounds__(kMaxThreads / 2, 4)
void moments_kernel(dgnn_group_norm_args a, Layout l, Moments* moments)
{
    constexpr int V = width_of<T>, R = kRegisters;
    extern __shared__ float scratch[];
    float* const means = scratch + 2 * l.scratch;
    float* const squares = means + l.groups_per_slab;
    const int64_t begin = blockIdx.y * l.share, end = begin + l.share < a.p ? begin + l.share : a.p;
    for (int64_t i = blockIdx.z; i < a.n; i += gridDim.z)
        for (int slab = blockIdx.x; slab < l.slabs; slab += gridDim.x) {
            const Part p = part_of<S, V>(l, (int)a.c, (int)a.groups, slab);
            const float inverse = 1.0f / ((float)(end - begin) * (float)(l.subs > 1 ? p.channels : l.per));
            const int rows = (int)(end - begin), here = p.row < 0 || p.row >= rows ? 0 : (rows - 1 - p.row) / l.rows + 1;
            float mean[V] = {}, squared[V] = {};
            if (here > 0) {
                const int64_t step = l.rows * a.x_p;
                const T* x = static_cast<const T*>(a.x) + i * a.x_n + (begin + p.row) * a.x_p + p.c;
                for (int done = 0; done < here; done += R) {
                    const int now = here - done < R ? here - done : R;
                    vec<T, V> held[R];
                    load_rows<S, T, R, V>(x, step, now, p, held);
                    x += R * step;
                    if (done == 0) {
#pragma unroll
                        for (int e = 0; e < V; ++e) mean[e] = (float)held[0][e];
                    }
                    float sum[V] = {}, square[V] = {};
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        if (r < now) {
#pragma unroll
                            for (int e = 0; e < V; ++e) {
                                const float d = (float)held[r][e] - mean[e];
                                sum[e] += d;
                                square[e] = __builtin_fmaf(d, d, square[e]);
                            }
                        }
                    const float each = rcp((float)(done + now));
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float moved = sum[e] * each, more = __builtin_fmaf(-moved, sum[e], square[e]);
                        mean[e] += moved;
                        squared[e] += more < 0.0f ? 0.0f : more;       // (a NaN stays)
                    }
                }
            }
            const float count = (float)here;
            float mine[V], joint[V];
#pragma unroll
            for (int e = 0; e < V; ++e) mine[e] = e < p.n ? mean[e] * count : 0.0f;
            group_sums<S, V>(l, p, mine, scratch, means, [&](float s) { return s * inverse; });
            of_channels<S, V>(l, p, means, joint);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = mean[e] - joint[e];
                mine[e] = e < p.n && here > 0 ? __builtin_fmaf(d * d, count, squared[e]) : 0.0f;      // (no row: d * d may be infinite, times 0 no number)
            }
            group_sums<S, V>(l, p, mine, scratch + l.scratch, squares, [&](float s) { return s; });
            for (int g = threadIdx.x; g < p.groups; g += blockDim.x)
                moments[((i * a.groups + p.g0 + g) * l.shares + blockIdx.y) * l.subs + p.sub] = Moments{means[g], squares[g]};
            __syncthreads();                                    // (means and squares are the next slab's)
        }
}

template <Shape S, typename T, Kind K, bool SKIP>
__global__ __launch_bounds__(kMaxThreads / 2, 4)
void apply_kernel(dgnn_group_norm_args a, Layout l, const Moments* moments)
{
    constexpr int V = width_of<T>, R = 2;
    __shared__ float means[kMaxGroups], scales[kMaxGroups];
    const int64_t begin = blockIdx.y * l.share, end = begin + l.share < a.p ? begin + l.share : a.p;
    constexpr int G = 2, Q = 4;
    const int pieces = l.shares * l.subs, waves = (int)(blockDim.x + 63) >> 6, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const auto count = [&](int piece) {                         // values of a piece
        int share = piece, wide = l.per;
        if (l.subs > 1) {
            share = piece / l.subs;
            const int from = (piece - share * l.subs) * kMaxVectors * V;
            wide = l.per - from < kMaxVectors * V ? l.per - from : kMaxVectors * V;
        }
        return (float)(share < l.shares - 1 ? l.share : a.p - (l.shares - 1) * l.share) * (float)wide;
    };
    const float inverse = 1.0f / ((float)a.p * (float)l.per);
    for (int64_t i = blockIdx.z; i < a.n; i += gridDim.z)
        for (int slab = blockIdx.x; slab < l.slabs; slab += gridDim.x) {
            const Part p = part_of<S, V>(l, (int)a.c, (int)a.groups, slab);
            // the first rows are on their way while the groups' moments are joined
            const int64_t x_step = l.rows * a.x_p, z_step = SKIP ? l.rows * a.z_p : 0;
            int64_t q = p.row < 0 ? end : begin + p.row;
            const T* x = static_cast<const T*>(a.x) + i * a.x_n + (begin + p.row) * a.x_p + p.c;
            const T* z = SKIP ? static_cast<const T*>(a.z) + i * a.z_n + (begin + p.row) * a.z_p + p.c : nullptr;
            int here;
            vec<T, V> held[R], skip[SKIP ? R : 1];
            const auto load = [&]() {
                here = end - q > (R - 1) * l.rows ? R : (int)(end - 1 - q) / l.rows + 1;
                load_rows<S, T, R, V>(x, x_step, here, p, held);
                x += R * x_step;
                if constexpr (SKIP) {
                    load_rows<S, T, R, V>(z, z_step, here, p, skip);
                    z += R * z_step;
                }
            };
            if (q < end) load();
            float weight[V], bias[V], of_mean[V], scale[V];
            load_affine<S, T, V>(a.weight, a.affine_type == DGNN_F32, p, 1.0f, weight);
            load_affine<S, T, V>(a.bias, a.affine_type == DGNN_F32, p, 0.0f, bias);
            // A wave joins two groups at once, so that what it waits for is asked for together; up to 256 pieces of each are still there for
            // the second sum.  A lane behind the last piece reads that one and takes nothing of it.
            for (int first = wave; first < p.groups; first += G * waves) {
                const Moments* of[G];
                Moments m[G][Q];
                float mean[G] = {}, squares[G] = {};
#pragma unroll
                for (int k = 0; k < G; ++k) of[k] = moments + (i * a.groups + p.g0 + first + k * waves) * pieces;
                const int groups = (p.groups - first + waves - 1) / waves;      // of this wave, from here on
                const auto fetch = [&](int base) {
#pragma unroll
                    for (int q = 0; q < Q; ++q)
                        if (base + q * 64 < pieces) {
                            const int at = base + q * 64 + lane < pieces ? base + q * 64 + lane : pieces - 1;
#pragma unroll
                            for (int k = 0; k < G; ++k)
                                if (k < groups) m[k][q] = of[k][at];
                        }
                };
                for (int base = 0; base < pieces; base += Q * 64) {
                    fetch(base);
#pragma unroll
                    for (int q = 0; q < Q; ++q)
                        if (base + q * 64 < pieces) {
                            const bool is = base + q * 64 + lane < pieces;
                            const float c = count(base + q * 64 + lane);
#pragma unroll
                            for (int k = 0; k < G; ++k)
                                if (k < groups) mean[k] = is ? __builtin_fmaf(m[k][q].mean, c, mean[k]) : mean[k];
                        }
                }
#pragma unroll
                for (int k = 0; k < G; ++k)
                    if (k < groups) mean[k] = wave_sum(mean[k]) * inverse;
                for (int base = 0; base < pieces; base += Q * 64) {
                    if (pieces > Q * 64) fetch(base);
#pragma unroll
                    for (int q = 0; q < Q; ++q)
                        if (base + q * 64 < pieces) {
                            const bool is = base + q * 64 + lane < pieces;
                            const float c = count(base + q * 64 + lane);
#pragma unroll
                            for (int k = 0; k < G; ++k)
                                if (k < groups) {
                                    const float d = m[k][q].mean - mean[k];
                                    squares[k] = is ? squares[k] + __builtin_fmaf(d * d, c, m[k][q].squares) : squares[k];
                                }
                        }
                }
#pragma unroll
                for (int k = 0; k < G; ++k)
                    if (k < groups) {
                        const float all = wave_sum(squares[k]);
                        if (lane == 0) means[first + k * waves] = mean[k], scales[first + k * waves] = 1.0f / sqrtf(__builtin_fmaf(all, inverse, a.eps));
                    }
            }
            __syncthreads();
            of_channels<S, V>(l, p, means, of_mean);
            of_channels<S, V>(l, p, scales, scale);
#pragma unroll
            for (int e = 0; e < V; ++e) scale[e] *= weight[e];
            __syncthreads();                                    // (means and scales are the next slab's)
            T* y = static_cast<T*>(a.y) + i * a.y_n + (begin + p.row) * a.y_p + p.c;
            while (q < end) {
#pragma unroll
                for (int r = 0; r < R; ++r)
                    if (r < here) {
                        float v[V];
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            v[e] = __builtin_fmaf((float)held[r][e] - of_mean[e], scale[e], bias[e]);
                            if constexpr (SKIP) v[e] += (float)skip[r][e];
                        }
                        activate_kind<K, T>(v, a.activation);
                        store_part<S, T, V>(y, p.n, v);
                        y += l.rows * a.y_p;
                    }
                q += R * l.rows;
                if (q < end) load();
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

int vector_of(const dgnn_group_norm_args& a) { return a.type == DGNN_F32 ? 4 : 8; }

Shape shape_of(const dgnn_group_norm_args& a, const Layout& l)
{
    const int vector = vector_of(a);
    if (a.c < vector) return kTiny;
    if (l.per % vector == 0) return kAligned;
    return a.c % vector == 0 && l.per * l.groups_per_slab % vector == 0 && l.subs == 1 ? kWhole : kRagged;
}

// What group_sums needs: a number, or one for each channel, from every thread, or from every one of a wave's row.
int scratch_of(const dgnn_group_norm_args& a, const Layout& l)
{
    const bool single = l.groups_per_slab == 1 || l.per % vector_of(a) == 0, even = (l.lanes & (l.lanes - 1)) == 0 && l.lanes <= 64;
    return (even ? (l.threads + 63) / 64 * l.lanes : l.threads) * (single ? 1 : vector_of(a));
}

// One pass where a workgroup's registers hold a slab of a sample, two otherwise.
Layout make_layout(const dgnn_group_norm_args& a, int* registers)
{
    constexpr int kThreads = kMaxThreads / 2;                   // (1024 of four vectors hold what 512 of eight do)
    const int vector = vector_of(a);
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
    const auto may_halve = [&]() {
        const int64_t now = groups * l.per, half = (groups + 1) / 2 * l.per;
        return (half % vector == 0 || now % vector != 0) && (half >= 2 * vector || a.p <= 1024);
    };
    cut(groups_of_whole_lines(l.per, a.groups, vector), 1);
    const int64_t whole = groups;
    *registers = 0;
    // Narrower slabs where these leave more than a quarter of the units idle, or do not fit and two vectors of a line would.  Not slabs whose rows
    // end inside a vector where they do not yet (107 maps of 632 x 80, groups of ten: 16 us, 23 so), and single vectors of a line for short maps
    // only: every workgroup fetches the whole line (2 maps of 4096 x 256: 18 us so, 12 in two passes; 114 of 1120 x 32: 11.4 us with two
    // vectors for 228 workgroups, 18.6 with one for 456).
    while (groups > 1 && a.n * l.slabs < kUnitsWanted * 3 / 4 && may_halve()) cut((groups + 1) / 2, 1);
    while (groups > 1 && groups * l.per > 2 * vector && a.p > held()) cut((groups + 1) / 2, 1);
    if (a.p <= held()) {
        // Eight vectors to a thread where the chip has about three or more for each of its threads (256 maps of 361 x 256: 32 us, 41 with four), two
        // where a call is one trip through it (one map: 5.8, 6.7 with eight) -- unless the groups end inside vectors: what such a thread does
        // beside its vectors is several times theirs (32 maps of 400 x 80, groups of ten: 8.7 us, 12 with two)
        const int64_t each_unit = a.n * l.slabs * l.lanes * a.p / (kUnitsWanted * kMaxThreads);
        const int wanted = each_unit >= 3 || shape_of(a, l) == kWhole ? kRegisters : 2, most = wanted == kRegisters ? kThreads : kMaxThreads;
        l.threads = 64;
        while (l.threads < most && (l.threads < l.lanes || (int64_t)(l.threads / l.lanes) * wanted < a.p)) l.threads *= 2;
        l.rows = l.threads / l.lanes;
        const int64_t each = ceil_div(a.p, l.rows);
        *registers = each <= 2 ? 2 : each <= 4 ? 4 : 8;
        l.scratch = scratch_of(a, l);
        return l;
    }
    const int subs = (int)ceil_div(l.per, kMaxVectors * vector);
    cut(subs > 1 ? 1 : whole, subs);
    l.threads = kThreads;
    l.rows = l.threads / l.lanes;
    // shares enough for two workgroups on every unit; for one where that would leave a thread fewer rows than it loads at once, and mostly at work on
    // what is the same for any number of rows
    int64_t shares = ceil_div(2 * kUnitsWanted, a.n * l.slabs);
    if (shares * kRegisters * l.rows > a.p) shares = ceil_div(kUnitsWanted, a.n * l.slabs);
    if (shares > kMaxShares) shares = kMaxShares;
    // and as many as keep a thread's rows few.  (At most 2^37 elements a sample: fewer than 40000, whatever the lanes)
    const int64_t least = ceil_div(a.p, (int64_t)kSerialRows * l.rows);
    if (shares < least) shares = least;
    l.share = ceil_div(ceil_div(a.p, shares), l.rows) * l.rows;
    l.shares = (int)ceil_div(a.p, l.share);
    l.scratch = scratch_of(a, l);
    return l;
}

template <Shape S, typename T, Kind K, bool SKIP>
hipError_t launch_kind(const dgnn_group_norm_args& a, const Layout& l, int registers, hipStream_t stream)
{
    const dim3 grid((unsigned)(l.slabs < 65536 ? l.slabs : 65536), (unsigned)l.shares, (unsigned)(a.n < 32768 ? a.n : 32768)), block(l.threads);
    // (up to 66048 bytes: 1024 threads with a number for each of eight channels, twice, where 64 groups end inside vectors)
    static_assert(2 * (kMaxThreads * 8 + kMaxGroups) * sizeof(float) <= kMaxShared, "what a compute unit has");
    const size_t shared = 2 * (size_t)(l.scratch + l.groups_per_slab) * sizeof(float);
    if (registers == 2) return launch_shared(one_pass_kernel<S, T, 2, K, SKIP>, grid, block, shared, stream, a, l);
    if (registers == 4) return launch_shared(one_pass_kernel<S, T, 4, K, SKIP>, grid, block, shared, stream, a, l);
    if (registers == 8) return launch_shared(one_pass_kernel<S, T, 8, K, SKIP>, grid, block, shared, stream, a, l);
    Moments* const moments = static_cast<Moments*>(a.workspace);
    const hipError_t err = launch_shared(moments_kernel<S, T>, grid, block, shared, stream, a, l, moments);
    return err != hipSuccess ? err : launch(apply_kernel<S, T, K, SKIP>, grid, block, stream, a, l, static_cast<const Moments*>(moments));
}

template <Shape S, typename T, bool SKIP>
hipError_t launch_shape(const dgnn_group_norm_args& a, const Layout& l, int registers, hipStream_t stream)
{
    if (a.activation == DGNN_ACT_IDENTITY || a.activation == DGNN_ACT_RELU) return launch_kind<S, T, kPlain, SKIP>(a, l, registers, stream);
    if (a.activation == DGNN_ACT_SILU) return launch_kind<S, T, kSilu, SKIP>(a, l, registers, stream);
    return launch_kind<S, T, kAny, SKIP>(a, l, registers, stream);
}

template <typename T, bool SKIP>
hipError_t launch_skip(const dgnn_group_norm_args& a, hipStream_t stream)
{
    int registers;
    const Layout l = make_layout(a, &registers);
    switch (shape_of(a, l)) {
    case kAligned: return launch_shape<kAligned, T, SKIP>(a, l, registers, stream);
    case kWhole: return launch_shape<kWhole, T, SKIP>(a, l, registers, stream);
    case kRagged: return launch_kind<kRagged, T, kAny, SKIP>(a, l, registers, stream);
    default: return launch_kind<kTiny, T, kAny, SKIP>(a, l, registers, stream);
    }
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
