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
    if constexpr (__is_same(T, f16)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The same with the sums tied to the accumulator half of the register file.  With all 256 of them in use the compiler's own choice moves sums
// back and forth between the halves (five moves per product); tied, it has none to make.  It does not see a matrix instruction in here:
// settle() before anything else reads the sums.
template <typename T>
__device__ __forceinline__ void mfma_tied(vec<T, 8> a, vec<T, 8> b, floatx4& c)
{
    if constexpr (__is_same(T, f16)) asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    else asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void settle() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

// Everything asked for has arrived; the builtin, so that the compiler knows too.
__device__ __forceinline__ void wait_all()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);         // vmcnt(0) expcnt(7) lgkmcnt(0)
    asm volatile("" ::: "memory");
}

// Up to eight neighbouring outputs of row m, from column n on: everything behind the sums.
template <typename T, typename O>
__device__ __forceinline__ void finish_as(const dgnn_dense_args& a, int64_t m, int64_t n, float (&v)[8])
{
    const O* const z = a.z ? static_cast<const O*>(a.z) + m * a.ldz + n : nullptr;
    O* const y = static_cast<O*>(a.y) + m * a.ldy + n;
    const bool bias_is_float = a.bias_type == DGNN_F32;
    if (n + 8 <= a.n) {
        if (z) {
            const vec<O, 8> s = load_vec<O, 8>(z);
#pragma unroll
            for (int r = 0; r < 8; ++r) v[r] = __builtin_fmaf(a.alpha2, (float)s[r], v[r]);
        }
        if (a.bias) {
            if (bias_is_float) {
                const vec<float, 8> s = load_vec<float, 8>(static_cast<const float*>(a.bias) + n);
#pragma unroll
                for (int r = 0; r < 8; ++r) v[r] += s[r];
            } else {
                const vec<T, 8> s = load_vec<T, 8>(static_cast<const T*>(a.bias) + n);
#pragma unroll
                for (int r = 0; r < 8; ++r) v[r] += (float)s[r];
            }
        }
        activate(v, a.activation);
        vec<O, 8> out;
#pragma unroll
        for (int r = 0; r < 8; ++r) out[r] = (O)v[r];
        store_vec<O, 8>(y, out);
    } else {
        const int left = (int)(a.n - n);
#pragma unroll
        for (int r = 0; r < 7; ++r) {
            if (r >= left) continue;
            if (z) v[r] = __builtin_fmaf(a.alpha2, (float)z[r], v[r]);
            if (a.bias) v[r] += load_either<T>(a.bias, n + r, bias_is_float);
        }
        activate(v, a.activation);
#pragma unroll
        for (int r = 0; r < 7; ++r)
            if (r < left) y[r] = (O)v[r];
    }
}

template <typename T>
__device__ __forceinline__ void finish(const dgnn_dense_args& a, int64_t m, int64_t n, float (&v)[8])
{
    if (m >= a.m || n >= a.n) return;
    if (a.out_type == DGNN_F32) finish_as<T, float>(a, m, n, v);
    else finish_as<T, T>(a, m, n, v);
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

// 16 bytes per lane from `base` + the lane's offset into 1 KiB of LDS, past the registers.
template <typename T>
__device__ __forceinline__ void dma_row(const char* base, unsigned offset, T* lds)
{
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(base + offset), (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// ---- tiles through LDS ------------------------------------------------------------------------------------------------------------
//
// WN x WM waves, each FN x FM fragments of 16 x 16 outputs; 64 of k at a time, double buffered.  A row's 64 elements are 128 bytes of LDS,
// its eight 16-byte segments stored at position segment ^ (row / 2 % 8): the sixteen lanes that one ds_read_b128 cycle serves (0-3, 12-15,
// 20-27 and the like: two segments, eight rows each) then fall into sixteen different 16-byte columns of the 64 banks.
//
// A tile is two steps of k = 32.  While the products of one step run, the fragments of the next are read, so a wave never waits for the read
// it has just asked for; the buffer of a tile is free once its second step has been read, i.e. at the one barrier in the middle of each tile,
// and is filled again two tiles ahead: a load has a whole tile's products to arrive.
//   DMA    rows whose address and stride are multiples of 16 bytes go from memory into LDS without passing through registers
//   else   the same pipeline with loads into registers (unaligned, but as wide) and ds_writes one tile later
// What is left of k behind the last whole tile (masked, element by element) comes FIRST: it is the one tile that is always written through registers.
template <typename T, int FN, int FM, int WN, int WM, bool DMA>
struct Tile {
    static constexpr int kWaves = WN * WM, kThreads = kWaves * 64;
    static constexpr int BN = WN * FN * 16, BM = WM * FM * 16, BK = 64;
    static constexpr int kRows = BN + BM;
    static constexpr int kLoads = kRows / 8 / kWaves;           // 1 KiB pieces (8 rows) per wave and tile: first those of W, then those of x
    static constexpr int kLoadsW = BN / 8 / kWaves;
    static_assert(BN / 8 % kWaves == 0 && BM / 8 % kWaves == 0, "whole pieces");
    static constexpr int kReads = FN + FM, kProducts = FN * FM;
    static constexpr bool kTied = FN * FM >= 32;
    typedef vec<T, 8> Frag;

    struct Frags { Frag w[FN], x[FM]; };

    const dgnn_dense_args& a;
    T* const lds;                                               // [2][kRows][64]
    int lane;
    const int wave;
    const int64_t m0, n0;
    const char* base_w;
    const char* base_x;
    int last_w, last_x;                                         // the last row of the tile's W (x) that is there
    int read_w, read_x;                                         // elements: this lane's row of fragment 0, and its segment of step 0 and 1
    int seg[2];
    vec<T, 8> staged[DMA ? 1 : kLoads];

    __device__ __forceinline__ Tile(const dgnn_dense_args& args, T* memory, int64_t m, int64_t n)
        : a(args), lds(memory), lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), m0(m), n0(n)
    {
        base_w = static_cast<const char*>(a.w) + n0 * a.ldw * 2;
        base_x = static_cast<const char*>(a.x) + m0 * a.ldx * 2;
        last_w = (int)(a.n - n0 < BN ? a.n - n0 : BN) - 1;
        last_x = (int)(a.m - m0 < BM ? a.m - m0 : BM) - 1;
        const int r = lane & 15;
        read_w = ((wave % WN) * FN * 16 + r) * BK;
        read_x = (BN + (wave / WN) * FM * 16 + r) * BK;
#pragma unroll
        for (int s = 0; s < 2; ++s) seg[s] = ((s * 4 + (lane >> 4)) ^ (r >> 1 & 7)) * 8;
    }

    // Piece j of this wave: which row of the tile's W (x) this lane fetches -- beyond the last row that one again, its outputs are never stored --
    // and which of its segments.
    __device__ __forceinline__ int piece(int j) const { return j < kLoadsW ? wave * kLoadsW + j : BN / 8 + wave * (kLoads - kLoadsW) + j - kLoadsW; }
    __device__ __forceinline__ int row_of(int j) const
    {
        const int row = (j < kLoadsW ? piece(j) : piece(j) - BN / 8) * 8 + (lane >> 3), last = j < kLoadsW ? last_w : last_x;
        return row < last ? row : last;
    }
    __device__ __forceinline__ int segment_of(int j) const { return (lane & 7) ^ ((piece(j) * 4 + (lane >> 4)) & 7); }

    __device__ __forceinline__ const T* source(int j, int64_t k) const
    {
        return reinterpret_cast<const T*>(j < kLoadsW ? base_w : base_x) + row_of(j) * (j < kLoadsW ? a.ldw : a.ldx) + k;
    }
    __device__ __forceinline__ void write(int j, int buffer, Frag v)
    {
        *reinterpret_cast<Frag*>(lds + buffer * kRows * BK + piece(j) * 8 * BK + lane * 8) = v;
    }
    // the ragged piece of k, through registers
    __device__ __forceinline__ void load_ragged(int buffer, int64_t k)
    {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) write(j, buffer, load_row<T>(source(j, 0), k + segment_of(j) * 8, a.k));
    }
    // Piece j of the tile whose first column is at `w` (`x`) in the tile's first row.  The offset of a row is a 24-bit product, formed anew each time:
    // kept, the offsets of all pieces would be more registers than the sums leave.
    __device__ __forceinline__ void load(int j, int buffer, const char* w, const char* x)
    {
        if constexpr (DMA) {
            const unsigned offset = __umul24(row_of(j), (unsigned)(j < kLoadsW ? a.ldw : a.ldx) * 2) + segment_of(j) * 16;
            dma_row(j < kLoadsW ? w : x, offset, lds + buffer * kRows * BK + piece(j) * 8 * BK);
        } else {
            const T* const row = reinterpret_cast<const T*>(j < kLoadsW ? w : x) + row_of(j) * (j < kLoadsW ? a.ldw : a.ldx);
            staged[j] = load_vec<T, 8>(row + segment_of(j) * 8);
        }
    }
    __device__ __forceinline__ void read(int r, int buffer, int step, Frags& f) const
    {
        // in the order of their first use: w 0, every x, the other w
        const T* const at = lds + buffer * kRows * BK + seg[step];
        if (r >= 1 && r <= FM) f.x[r - 1] = *reinterpret_cast<const Frag*>(at + read_x + (r - 1) * 16 * BK);
        else f.w[r == 0 ? 0 : r - FM] = *reinterpret_cast<const Frag*>(at + read_w + (r == 0 ? 0 : r - FM) * 16 * BK);
    }

    // The products of one step; beside them the fragments of the next step are read and, with LOAD, the tile two ahead is asked for.  Nothing in
    // here branches: the compiler keeps the sums and the fragments where they are.
    template <bool LOAD>
    __device__ __forceinline__ void step(floatx4 (&acc)[FN][FM], const Frags& f, Frags& next, int read_buffer, int read_step, int load_buffer, const char* w, const char* x)
    {
        constexpr int kGroups = kReads, kReadGroups = kGroups * 3 / 4;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
#pragma unroll
            for (int p = g * kProducts / kGroups; p < (g + 1) * kProducts / kGroups; ++p)
                if constexpr (kTied) mfma_tied<T>(f.w[p / FM], f.x[p % FM], acc[p / FM][p % FM]);
                else acc[p / FM][p % FM] = mfma<T>(f.w[p / FM], f.x[p % FM], acc[p / FM][p % FM]);
            if constexpr (LOAD) {
#pragma unroll
                for (int j = g * kLoads / kGroups; j < (g + 1) * kLoads / kGroups; ++j) load(j, load_buffer, w, x);
            }
            if (g < kReadGroups) {
#pragma unroll
                for (int r = g * kReads / kReadGroups; r < (g + 1) * kReads / kReadGroups; ++r) read(r, read_buffer, read_step, next);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // Tile t, whose first fragments are in f0; leaves those of tile t + 1 there (behind the last tile: whatever the buffer holds).
    template <bool LOAD>
    __device__ __forceinline__ void tile(floatx4 (&acc)[FN][FM], Frags& f0, Frags& f1, int t, int k)
    {
        const int b = t & 1;
        step<false>(acc, f0, f1, b, 1, 0, nullptr, nullptr);
        if constexpr (!DMA) {
            if (t > 0) {
#pragma unroll
                for (int j = 0; j < kLoads; ++j) write(j, b ^ 1, staged[j]);
            }
        }
        wait_all();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const char *w = base_w + (int64_t)k * 2, *x = base_x + (int64_t)k * 2;
        asm volatile("" : "+s"(w), "+s"(x), "+v"(lane));        // (otherwise every piece's address is kept in registers and counted up)
        step<LOAD>(acc, f1, f0, b ^ 1, 0, b, w, x);
    }

    __device__ __forceinline__ void run(floatx4 (&acc)[FN][FM])
    {
        const int whole = (int)(a.k / BK), ragged = a.k % BK ? 1 : 0, tiles = whole + ragged;
        if (tiles == 0) return;
        // tile t starts at column first + t * 64, the ragged one (t = 0) at the end of the row
        const int first = ragged ? -BK : 0;
        __syncthreads();                                        // (the LDS of the tile before)
        if (ragged) load_ragged(0, (int64_t)whole * BK);
        else fill(0, 0);
        if (tiles > 1) fill(1, first + BK);
        wait_all();
        __syncthreads();
        Frags f0, f1;
#pragma unroll
        for (int r = 0; r < kReads; ++r) read(r, 0, 0, f0);
        int t = 0;
        for (; t + 2 < tiles; ++t) tile<true>(acc, f0, f1, t, first + (t + 2) * BK);
        for (; t < tiles; ++t) tile<false>(acc, f0, f1, t, 0);
        if constexpr (kTied) settle();
    }

    // a whole tile, at once (before the loop)
    __device__ __forceinline__ void fill(int buffer, int k)
    {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            load(j, buffer, base_w + (int64_t)k * 2, base_x + (int64_t)k * 2);
            if constexpr (!DMA) write(j, buffer, staged[j]);
        }
    }

    // The outputs pass through LDS, 16 rows of the wave's columns at a time, so that each row is written in whole lines.
    __device__ __forceinline__ void store(const floatx4 (&acc)[FN][FM])
    {
        constexpr int kColumns = FN * 16, kPitch = kColumns + 4;        // (16 bytes on: the rows of a fragment start in different banks)
        static_assert(kWaves * 16 * kPitch * sizeof(float) <= 2 * kRows * BK * sizeof(T), "fits the tiles' LDS");
        float* const mine = reinterpret_cast<float*>(lds) + wave * 16 * kPitch;
        __syncthreads();                                        // every wave has read its last fragments
#pragma unroll 1
        for (int j = 0; j < FM; ++j) {
#pragma unroll
            for (int q = 0; q < FM; ++q)
                if (q == j) {
#pragma unroll
                    for (int i = 0; i < FN; ++i)
                        *reinterpret_cast<floatx4*>(mine + (lane & 15) * kPitch + i * 16 + (lane >> 4) * 4) = acc[i][q] * a.alpha1;
                }
            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
            for (int e = lane * 8; e < 16 * kColumns; e += 64 * 8) {
                const int row = e / kColumns, column = e % kColumns;
                float v[8];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const floatx4 part = *reinterpret_cast<const floatx4*>(mine + row * kPitch + column + h * 4);
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[h * 4 + r] = part[r];
                }
                finish<T>(a, m0 + ((wave / WN) * FM + j) * 16 + row, n0 + (wave % WN) * FN * 16 + column, v);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
};

// Tiles in the order in which they are handed out.  Workgroup i runs on die i % 8, each die with an L2 of its own: every die takes a
// contiguous eighth of the tiles, and those run down strips of kStrip rows of tiles, so that what runs at one time on a die shares rows of
// x and W.
constexpr int kDies = 8;
constexpr int kStrip = 8;
__device__ __forceinline__ void place(int64_t i, int64_t tiles_m, int64_t tiles_n, int64_t& tm, int64_t& tn)
{
    const int64_t tiles = tiles_m * tiles_n, die = i % kDies, each = tiles / kDies, more = tiles % kDies;
    i = die * each + (die < more ? die : more) + i / kDies;
    const int64_t strip = i / (kStrip * tiles_n), in = i % (kStrip * tiles_n);
    const int64_t height = tiles_m - strip * kStrip < kStrip ? tiles_m - strip * kStrip : kStrip;
    tm = strip * kStrip + in % height;
    tn = in / height;
}

template <typename T, int FN, int FM, int WN, int WM, bool DMA>
__global__ __launch_bounds__(WN * WM * 64, FN * FM > 32 ? 1 : 2)
void dense_tile_kernel(dgnn_dense_args a, int64_t tiles_m, int64_t tiles_n)
{
    typedef Tile<T, FN, FM, WN, WM, DMA> Work;
    __shared__ __attribute__((aligned(1024))) T lds[2 * Work::kRows * Work::BK];
    for (int64_t i = blockIdx.x; i < tiles_m * tiles_n; i += gridDim.x) {
        int64_t tm, tn;
        place(i, tiles_m, tiles_n, tm, tn);
        Work work(a, lds, tm * Work::BM, tn * Work::BN);
        floatx4 acc[FN][FM] = {};
        work.run(acc);
        work.store(acc);
    }
}

template <typename T, int FN, int FM, int WN, int WM, bool DMA>
hipError_t launch_tiles(const dgnn_dense_args& a, hipStream_t stream)
{
    typedef Tile<T, FN, FM, WN, WM, DMA> Work;
    const int64_t tiles_m = (a.m + Work::BM - 1) / Work::BM, tiles_n = (a.n + Work::BN - 1) / Work::BN, tiles = tiles_m * tiles_n;
    return launch(dense_tile_kernel<T, FN, FM, WN, WM, DMA>, dim3((unsigned)(tiles < kMaxGrid ? tiles : kMaxGrid)), dim3(Work::kThreads), stream, a, tiles_m, tiles_n);
}

bool sixteen(const void* p, int64_t stride, int64_t rows) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows <= 1 || stride % 8 == 0); }

template <typename T>
hipError_t launch_typed(const dgnn_dense_args& a, hipStream_t stream)
{
    // an offset inside a tile's 256 rows is 32 bits
    const bool dma = sixteen(a.x, a.ldx, a.m) && sixteen(a.w, a.ldw, a.n) && a.ldx < 1 << 22 && a.ldw < 1 << 22;
    if (!dma) return launch_tiles<T, 4, 4, 2, 2, false>(a, stream);
    const int64_t big = ((a.m + 255) / 256) * ((a.n + 255) / 256);
    if (big >= 192) return launch_tiles<T, 4, 8, 4, 2, true>(a, stream);
    const int64_t mid = ((a.m + 127) / 128) * ((a.n + 127) / 128);
    if (mid >= 128) return launch_tiles<T, 4, 4, 2, 2, true>(a, stream);
    return launch_tiles<T, 2, 2, 2, 2, true>(a, stream);
}

}  // namespace

hipError_t launch_dense(const dgnn_dense_args& a, hipStream_t stream)
{
    return a.type == DGNN_F16 ? launch_typed<f16>(a, stream) : launch_typed<bf16>(a, stream);
}

}  // namespace ops
}  // namespace dgnn
