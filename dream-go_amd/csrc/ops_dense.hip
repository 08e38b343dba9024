// dgnn_dense: y = act(alpha1 * x W^T + alpha2 * z + bias) on the matrix cores.
//
// The products are v_mfma_f32_16x16x32 with the ROWS OF W as the first operand and the rows of x as the second: D[i][j] then holds four
// consecutive outputs n of one row m in a lane's four registers, which is how y lies in memory.  Sums are fp32; alpha1, z, bias and the
// activation are applied in fp32 and the result is rounded once.
//
// Measured: 8192 x 16384 -> 4096 bf16 with a skip 868 us, 1267 TFLOP/s (bound by the matrix pipe under its power limit); 16 x 4096 -> 16384 26 us
// (31 with the weights out of every cache: HBM, 4.3 TB/s); 1021 x 2027 -> 1531, where no row is aligned, 28 us, 9 of them the copies (then bound by a
// unit's path to the L2); 256 x 2888 -> 362 fp16 10.8 us and one row of it 6.9 (chains of waits);
// 2048 x 4096 -> 4096 74 us, 928 TFLOP/s, and 512 rows of it 26.6 (tiles that do not come out even on 256 units).
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

// Every LDS operation of the wave is done and at most N of its loads are still on their way; the builtin, so that the compiler knows too.
template <int N>
__device__ __forceinline__ void wait_for_all_but()
{
    static_assert(N < 64, "the counter has six bits");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | 0x0070 | (N >> 4) << 14);             // vmcnt(N) expcnt(7) lgkmcnt(0)
    asm volatile("" ::: "memory");
}

// Up to eight neighbouring outputs of row m, from column n on: everything behind the sums.
template <typename T, typename O>
__device__ __forceinline__ void finish_as(const dgnn_dense_args& a, int64_t m, int64_t n, float (&v)[8])
{
#pragma unroll
    for (int r = 0; r < 8; ++r) v[r] *= a.alpha1;
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
        activate<O>(v, a.activation);
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
        activate<O>(v, a.activation);
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

// The sums of one share of k, as they are: dense_join_kernel finishes them.
__device__ __forceinline__ void keep(const dgnn_dense_args& a, float* part, int64_t m, int64_t n, const float (&v)[8])
{
    if (m >= a.m || n >= a.n) return;
    float* const to = part + m * a.n + n;
    if (n + 8 <= a.n) {
        vec<float, 8> all;
#pragma unroll
        for (int r = 0; r < 8; ++r) all[r] = v[r];
        store_vec<float, 8>(to, all);
    } else {
#pragma unroll
        for (int r = 0; r < 7; ++r)
            if (n + r < a.n) to[r] = v[r];
    }
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
// WN x WM waves, each FN x FM fragments of 16 x 16 outputs; 64 of k at a time in a ring of S tiles.  A row's 64 elements are 128 bytes of LDS,
// its eight 16-byte segments stored at position segment ^ (row / 2 % 8): the sixteen lanes that one ds_read_b128 cycle serves (0-3, 12-15,
// 20-27 and the like: two segments, eight rows each) then fall into sixteen different 16-byte columns of the 64 banks.
//
// A tile is two steps of k = 32.  While the products of one step run, the fragments of the next are read, so a wave never waits for the read
// it has just asked for; the buffer of a tile is free once its second step has been read, i.e. at the one barrier in the middle of each tile,
// and is filled again S tiles ahead: a load has S - 1 tiles' products to arrive, and is waited for by count.
// KG crews of waves share the columns of k tile by tile, each with a ring of its own, and add their sums up in the end: one crew does not ask for as
// much as a compute unit's path to the L2 carries (32 x 32 outputs: 43 bytes a nanosecond, four crews 52).
//
// Rows go from memory into LDS without passing through registers: their addresses and strides are multiples of 16 bytes (dense_pack_kernel sees
// to it where the caller's are not).  What is left of k behind the last whole tile (masked, element by element) comes FIRST: it is the one tile
// that is written through registers.
template <typename T, int FN, int FM, int WN, int WM, int S, int KG>
struct Tile {
    static constexpr int kWaves = WN * WM, kThreads = kWaves * KG * 64;         // waves of one crew
    static constexpr int BN = WN * FN * 16, BM = WM * FM * 16, BK = 64;
    static constexpr int kRows = BN + BM;
    static constexpr int kPieces = kRows / 8, kPiecesW = BN / 8;                // 1 KiB pieces (8 rows): first those of W, then those of x
    static constexpr bool kEven = kPiecesW % kWaves == 0 && kPieces % kWaves == 0;
    static constexpr int kLoads = (kPieces + kWaves - 1) / kWaves, kLoadsW = kEven ? kPiecesW / kWaves : 0;
    static constexpr int kReads = FN + FM, kProducts = FN * FM;
    static constexpr bool kTied = FN * FM >= 32;
    static constexpr int kLdsBytes = KG * S * kRows * BK * 2;
    static constexpr int kPerUnit = 160 * 1024 / kLdsBytes < 2 ? 1 : 2;         // workgroups on a compute unit at a time
    static_assert(S >= 2 && (S - 2) * kLoads < 64, "loads in flight are counted");
    typedef vec<T, 8> Frag;

    struct Frags { Frag w[FN], x[FM]; };

    const dgnn_dense_args& a;
    T* const lds;                                               // [S][kRows][64]
    int lane;
    const int crew, wave;                                       // the wave's number in its crew
    const int64_t m0, n0;
    const int columns;                                          // of k, from `begin` on
    const char* base_w;
    const char* base_x;
    int last_w, last_x;                                         // the last row of the tile's W (x) that is there
    int read_w, read_x;                                         // elements: this lane's row of fragment 0, and its segment of step 0 and 1
    int seg[2];

    __device__ __forceinline__ Tile(const dgnn_dense_args& args, T* memory, int64_t m, int64_t n, int64_t begin, int64_t end)
        : a(args), lds(memory + __builtin_amdgcn_readfirstlane(threadIdx.x / (kWaves * 64)) * S * kRows * BK), lane(threadIdx.x & 63),
          crew(__builtin_amdgcn_readfirstlane(threadIdx.x / (kWaves * 64))), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % kWaves), m0(m), n0(n), columns((int)(end - begin))
    {
        base_w = static_cast<const char*>(a.w) + (n0 * a.ldw + begin) * 2;
        base_x = static_cast<const char*>(a.x) + (m0 * a.ldx + begin) * 2;
        last_w = (int)(a.n - n0 < BN ? a.n - n0 : BN) - 1;
        last_x = (int)(a.m - m0 < BM ? a.m - m0 : BM) - 1;
        const int r = lane & 15;
        read_w = ((wave % WN) * FN * 16 + r) * BK;
        read_x = (BN + (wave / WN) * FM * 16 + r) * BK;
#pragma unroll
        for (int s = 0; s < 2; ++s) seg[s] = ((s * 4 + (lane >> 4)) ^ (r >> 1 & 7)) * 8;
    }

    // Piece j of this wave: which row of the tile's W (x) this lane fetches -- beyond the last row that one again, its outputs are never stored --
    // and which of its segments.  Where the pieces do not divide evenly the last one is fetched more than once, by every wave alike many loads.
    __device__ __forceinline__ int piece(int j) const
    {
        if constexpr (kEven) return j < kLoadsW ? wave * kLoadsW + j : kPiecesW + wave * (kLoads - kLoadsW) + j - kLoadsW;
        else return wave * kLoads + j < kPieces ? wave * kLoads + j : kPieces - 1;
    }
    __device__ __forceinline__ bool of_w(int j) const
    {
        if constexpr (kEven) return j < kLoadsW;
        else return piece(j) < kPiecesW;
    }
    __device__ __forceinline__ int row_of(int j) const
    {
        const int row = (of_w(j) ? piece(j) : piece(j) - kPiecesW) * 8 + (lane >> 3), last = of_w(j) ? last_w : last_x;
        return row < last ? row : last;
    }
    __device__ __forceinline__ int segment_of(int j) const { return (lane & 7) ^ ((piece(j) * 4 + (lane >> 4)) & 7); }

    __device__ __forceinline__ const T* source(int j) const
    {
        return reinterpret_cast<const T*>(of_w(j) ? base_w : base_x) + row_of(j) * (of_w(j) ? a.ldw : a.ldx);
    }
    __device__ __forceinline__ void write(int j, int buffer, Frag v)
    {
        *reinterpret_cast<Frag*>(lds + buffer * kRows * BK + piece(j) * 8 * BK + lane * 8) = v;
    }
    // the ragged piece of k, through registers
    __device__ __forceinline__ void load_ragged(int buffer, int k)
    {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) write(j, buffer, load_row<T>(source(j), k + segment_of(j) * 8, columns));
    }
    // Piece j of the tile whose first column is at `w` (`x`) in the tile's first row.  The offset of a row is a 24-bit product, formed anew each time:
    // kept, the offsets of all pieces would be more registers than the sums leave.
    __device__ __forceinline__ void load(int j, int buffer, const char* w, const char* x)
    {
        const unsigned offset = __umul24(row_of(j), (unsigned)(of_w(j) ? a.ldw : a.ldx) * 2) + segment_of(j) * 16;
        dma_row(of_w(j) ? w : x, offset, lds + buffer * kRows * BK + piece(j) * 8 * BK);
    }
    __device__ __forceinline__ void read(int r, int buffer, int step, Frags& f) const
    {
        // in the order of their first use: w 0, every x, the other w
        const T* const at = lds + buffer * kRows * BK + seg[step];
        if (r >= 1 && r <= FM) f.x[r - 1] = *reinterpret_cast<const Frag*>(at + read_x + (r - 1) * 16 * BK);
        else f.w[r == 0 ? 0 : r - FM] = *reinterpret_cast<const Frag*>(at + read_w + (r == 0 ? 0 : r - FM) * 16 * BK);
    }

    // The products of one step; beside them the fragments of the next step are read and, with LOAD, the tile S ahead is asked for.  Nothing in
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

    // Waits until at most `tiles` tiles (N at most) are on their way to LDS.
    template <int N>
    __device__ __forceinline__ static void wait_for_all_but_tiles(int tiles)
    {
        if constexpr (N == 0) wait_for_all_but<0>();
        else if (tiles >= N) wait_for_all_but<N * kLoads>();
        else wait_for_all_but_tiles<N - 1>(tiles);
    }

    // The tile in buffer b, whose first fragments are in f0; leaves those of the next tile there (behind the last tile: whatever the buffer holds).
    // With LOAD the tile that starts at column k takes its place.  `ahead` tiles may be on their way when the next one is needed.
    template <bool LOAD>
    __device__ __forceinline__ void tile(floatx4 (&acc)[FN][FM], Frags& f0, Frags& f1, int b, int ahead, int k)
    {
        const int next = b + 1 == S ? 0 : b + 1;
        step<false>(acc, f0, f1, b, 1, 0, nullptr, nullptr);
        if constexpr (LOAD) wait_for_all_but<(S - 2) * kLoads>();
        else wait_for_all_but_tiles<S - 2>(ahead);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const char *w = base_w + (int64_t)k * 2, *x = base_x + (int64_t)k * 2;
        asm volatile("" : "+s"(w), "+s"(x), "+v"(lane));        // (otherwise every piece's address is kept in registers and counted up)
        step<LOAD>(acc, f1, f0, next, 0, b, w, x);
    }

    __device__ __forceinline__ void run(floatx4 (&acc)[FN][FM])
    {
        const int whole = columns / BK, more = columns % BK ? 1 : 0, all = whole + more;
        if (all == 0) return;
        // tile t of this crew starts at column first + t * KG * 64; the ragged one, the first of all, at the end of the row
        const int ragged = KG == 1 || crew == 0 ? more : 0, first = (crew - more) * BK, tiles = (all - crew + KG - 1) / KG, turns = (all + KG - 1) / KG;
        const int filled = tiles < S ? tiles : S;
        __syncthreads();                                        // (the LDS of the tile before)
        for (int t = ragged; t < filled; ++t)
#pragma unroll
            for (int j = 0; j < kLoads; ++j) load(j, t, base_w + (int64_t)(first + t * KG * BK) * 2, base_x + (int64_t)(first + t * KG * BK) * 2);
        if (ragged) load_ragged(0, whole * BK);
        wait_for_all_but_tiles<S - 2>(ragged || filled < S ? 0 : S - 2);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        Frags f0, f1;
#pragma unroll
        for (int r = 0; r < kReads; ++r) read(r, 0, 0, f0);     // (a crew without a tile reads what LDS holds, and uses none of it)
        int t = 0, b = 0;
        for (; t + S < tiles; ++t) {
            tile<true>(acc, f0, f1, b, 0, first + (t + S) * KG * BK);
            b = b + 1 == S ? 0 : b + 1;
        }
        for (; t < tiles; ++t) {
            tile<false>(acc, f0, f1, b, tiles - t - 2, 0);
            b = b + 1 == S ? 0 : b + 1;
        }
        if constexpr (kTied) settle();
        if constexpr (KG > 1) {
            for (; t < turns; ++t) __builtin_amdgcn_s_barrier();        // (one barrier in every crew's every turn)
            join_crews(acc);
        }
    }

    // The first crew's sums and the others', in their order.
    __device__ __forceinline__ void join_crews(floatx4 (&acc)[FN][FM])
    {
        static_assert((KG - 1) * kWaves * kProducts * 1024 <= kLdsBytes, "fits the tiles' LDS");
        floatx4* const place = reinterpret_cast<floatx4*>(lds - crew * S * kRows * BK) + wave * kProducts * 64 + lane;
        __syncthreads();
        if (crew > 0) {
#pragma unroll
            for (int p = 0; p < kProducts; ++p) place[((crew - 1) * kWaves * kProducts + p) * 64] = acc[p / FM][p % FM];
        }
        __syncthreads();
        if (crew == 0) {
#pragma unroll 1
            for (int g = 0; g < KG - 1; ++g)
#pragma unroll
                for (int p = 0; p < kProducts; ++p) acc[p / FM][p % FM] += place[(g * kWaves * kProducts + p) * 64];
        }
    }

    // The outputs pass through LDS, 16 rows of the wave's columns at a time, so that each row is written in whole lines.
    // `part`: where to put the bare sums ([m][n]) instead of finished outputs.
    __device__ __forceinline__ void store(const floatx4 (&acc)[FN][FM], float* part)
    {
        constexpr int kColumns = FN * 16, kPitch = kColumns + 4;        // (16 bytes on: the rows of a fragment start in different banks)
        static_assert(kWaves * 16 * kPitch * sizeof(float) <= S * kRows * BK * sizeof(T), "fits the tiles' LDS");
        float* const mine = reinterpret_cast<float*>(lds) + wave * 16 * kPitch;
        __syncthreads();                                        // every wave has read its last fragments
        if (crew > 0) return;
#pragma unroll 1
        for (int j = 0; j < FM; ++j) {
#pragma unroll
            for (int q = 0; q < FM; ++q)
                if (q == j) {
#pragma unroll
                    for (int i = 0; i < FN; ++i)
                        *reinterpret_cast<floatx4*>(mine + (lane & 15) * kPitch + i * 16 + (lane >> 4) * 4) = acc[i][q];
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
                const int64_t m = m0 + ((wave / WN) * FM + j) * 16 + row, n = n0 + (wave % WN) * FN * 16 + column;
                if (part) keep(a, part, m, n, v);
                else finish<T>(a, m, n, v);
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

// `splits` shares of k, of `share` columns (a multiple of 64) each; with more than one, the sums go to `parts`.
template <typename T, int FN, int FM, int WN, int WM, int S, int KG>
__global__ __launch_bounds__(WN * WM * KG * 64, (WN * WM * KG * Tile<T, FN, FM, WN, WM, S, KG>::kPerUnit + 3) / 4)
void dense_tile_kernel(dgnn_dense_args a, int64_t tiles_m, int64_t tiles_n, int64_t splits, int64_t share, float* parts)
{
    typedef Tile<T, FN, FM, WN, WM, S, KG> Work;
    __shared__ __attribute__((aligned(1024))) T lds[KG * S * Work::kRows * Work::BK];
    const int64_t tiles = tiles_m * tiles_n;
    for (int64_t i = blockIdx.x; i < tiles * splits; i += gridDim.x) {
        const int64_t split = i / tiles, begin = split * share;
        int64_t tm, tn;
        place(i % tiles, tiles_m, tiles_n, tm, tn);
        Work work(a, lds, tm * Work::BM, tn * Work::BN, begin, begin + share < a.k ? begin + share : a.k);
        floatx4 acc[FN][FM] = {};
        work.run(acc);
        work.store(acc, parts ? parts + split * a.m * a.n : nullptr);
    }
}

// The shares' sums, in their order, and everything behind them.  Eight columns a thread; the sums of four shares are asked for at a time.
template <typename T>
__global__ __launch_bounds__(256)
void dense_join_kernel(dgnn_dense_args a, int splits, int lanes, const float* parts)
{
    const int lane = threadIdx.x & (lanes - 1), down = 256 / lanes;
    const int64_t plane = a.m * a.n;
    for (int64_t m = (int64_t)blockIdx.x * down + threadIdx.x / lanes; m < a.m; m += (int64_t)gridDim.x * down)
        for (int64_t n = lane * 8; n < a.n; n += lanes * 8) {
            const float* const from = parts + m * a.n + n;
            float v[8] = {};
            for (int s = 0; s < splits; s += 4) {
                vec<float, 8> four[4];                                         // (behind a row's end: the next one's, and used for nothing)
#pragma unroll
                for (int q = 0; q < 4; ++q) four[q] = s + q < splits ? load_vec<float, 8>(from + (s + q) * plane) : vec<float, 8>{};
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int r = 0; r < 8; ++r) v[r] += four[q][r];
            }
            finish<T>(a, m, n, v);
        }
}

// Rows of any alignment -> rows that start at multiples of 16 bytes, zero behind their end.  Sixteen-bit types alone, so their bits.
struct Packing {
    const uint16_t* from;
    uint16_t* to;
    int64_t rows, ld;
};
__global__ __launch_bounds__(256)
void dense_pack_kernel(Packing w, Packing x, int64_t k, int64_t pitch, int lanes)
{
    const int lane = threadIdx.x & (lanes - 1), down = 256 / lanes;
    for (int64_t row = (int64_t)blockIdx.x * down + threadIdx.x / lanes; row < w.rows + x.rows; row += (int64_t)gridDim.x * down) {
        const bool of_w = row < w.rows;
        const int64_t r = of_w ? row : row - w.rows;
        const uint16_t* const from = (of_w ? w.from : x.from) + r * (of_w ? w.ld : x.ld);
        uint16_t* const to = (of_w ? w.to : x.to) + r * pitch;
        for (int64_t column = lane * 8; column < pitch; column += lanes * 8) *reinterpret_cast<vec<uint16_t, 8>*>(to + column) = load_row<uint16_t>(from, column, k);
    }
}

// ---- few rows on one side: fragments straight from memory -------------------------------------------------------------------------
//
// Where one of the operands has few rows, or both are small, there is little to share through LDS: a workgroup owns 16 x 16 outputs, its waves
// share the columns of k in contiguous pieces and fetch the fragments they multiply, and their sums meet in LDS, in order.  Rows need no alignment.
// Bound by what a unit's L1 passes on: 28 GB/s a unit at 16 x 8192 x 512 (18 us on 32 units); at 1 x 4096 x 16384 by HBM, 4.9 TB/s (27.5 us with the
// weights out of every cache).  A wave with fewer than kUnroll steps takes them one by one, each load waited for before the next: 1 x 2888 x 362, six steps
// a wave, spends most of its 6.9 us so.
constexpr int kDirectWaves = 16;
template <typename T>
__global__ __launch_bounds__(kDirectWaves * 64)
void dense_direct_kernel(dgnn_dense_args a, int64_t tiles_n, int64_t tiles)
{
    constexpr int kPitch = 20, kUnroll = 8;
    __shared__ __attribute__((aligned(16))) float partial[kDirectWaves][16][kPitch];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int steps = (int)((a.k + 31) / 32), whole = (int)(a.k / 32), each = (steps + waves - 1) / waves;
    const int begin = wave * each, end = begin + each < steps ? begin + each : steps, full = end < whole ? end : whole;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int64_t m0 = tile / tiles_n * 16, n0 = tile % tiles_n * 16;
        // (beyond the last row: that one again, its outputs are not stored)
        const int64_t n = n0 + (lane & 15), m = m0 + (lane & 15);
        const T* const w = static_cast<const T*>(a.w) + (n < a.n ? n : a.n - 1) * a.ldw + (lane >> 4) * 8;
        const T* const x = static_cast<const T*>(a.x) + (m < a.m ? m : a.m - 1) * a.ldx + (lane >> 4) * 8;
        floatx4 acc = {};
        int s = begin;
        for (; s + kUnroll <= full; s += kUnroll) {
            vec<T, 8> fw[kUnroll], fx[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                fw[u] = load_vec<T, 8>(w + (int64_t)(s + u) * 32);
                fx[u] = load_vec<T, 8>(x + (int64_t)(s + u) * 32);
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) acc = mfma<T>(fw[u], fx[u], acc);
        }
        for (; s < end; ++s) {
            const int64_t left = a.k - (int64_t)s * 32 - (lane >> 4) * 8;
            acc = mfma<T>(load_row<T>(w + (int64_t)s * 32, 0, left), load_row<T>(x + (int64_t)s * 32, 0, left), acc);
        }
        __syncthreads();                                                       // (the sums of the tile before)
        *reinterpret_cast<floatx4*>(&partial[wave][lane & 15][(lane >> 4) * 4]) = acc;
        __syncthreads();
        for (int e = threadIdx.x; e < 32; e += blockDim.x) {
            const int row = e >> 1, column = (e & 1) * 8;
            float v[8] = {};
            for (int g = 0; g < waves; ++g)
#pragma unroll
                for (int r = 0; r < 8; ++r) v[r] += partial[g][row][column + r];
            finish<T>(a, m0 + row, n0 + column, v);
        }
    }
}

// ---- which form a call takes ---------------------------------------------------------------------------------------------------------
//
// A call is priced in every form it could take and takes the cheapest.  The prices are measured (microseconds, bf16): one tile of 64 columns
// of k where a compute unit holds one workgroup, the same where it holds two, and what a workgroup takes besides (first loads, outputs).  What
// the forms cost beside each other at the sizes where they change places (m, k, n; operands not in the caches):
//    1 x 4096 x 16384 (m, k, n)   direct 27.5 (4.9 TB/s)   16 x 64: 31.2   32 x 32: 34.4
//   16 x 4096 x 16384             direct 39.7   16 x 64: 31.2 (4.3 TB/s)   32 x 32: 35.5
//    1 x 2888 x 362               direct  6.2   32 x 32:  8.0   64 x 64: 8.5 (shares of k)
//  256 x 2888 x 362               32 x 32: 12.8   four crews: 11.4   64 x 64: 12.7   64 x 128: 14.8
// 1024 x 4096 x 1024              64 x 64: 19.4   two crews: 17.0   64 x 128: 19.7   128 x 128: 24.0
//  512 x 4096 x 4096              64 x 64: 35.8   64 x 128: 31.7   128 x 128: 32.7   256 x 256: 45.4
// 4096 x 4096 x 1024              64 x 64: 62.4   64 x 128: 59.0   128 x 128: 42.4   256 x 256: 61.1
// 4096 x 1024 x 4096              64 x 128: 74.8   128 x 128: 53.9   256 x 256: 38.7
struct Form {
    int bm, bn, per_unit;
    double alone, crowded, fixed;
};
constexpr Form kForms[] = {
    {16, 64, 2, 0.27, 0.40, 2.5},
    {64, 16, 2, 0.27, 0.40, 2.5},
    {32, 32, 2, 0.19, 0.29, 3.2},
    {64, 64, 2, 0.30, 0.49, 3.8},
    {64, 128, 1, 0.47, 0.47, 4.0},
    {128, 128, 1, 0.60, 0.60, 4.5},
    {256, 256, 1, 1.72, 1.72, 12.0},
    {32, 32, 1, 0.145, 0.145, 4.6},         // four crews
    {64, 64, 1, 0.215, 0.215, 4.6},         // two
};
constexpr int kNumForms = sizeof(kForms) / sizeof(kForms[0]), kDirect = -1;
constexpr double kUnits = 256;
constexpr int64_t kMaxSplits = 16;
// One launch more: what it takes on the device and, where calls follow each other closely, the host.
constexpr double kLaunch = 5.0;

struct Plan {
    int form = kDirect;
    int64_t splits = 1, share = 0;          // shares of k, columns of each
    bool pack_w = false, pack_x = false;    // rows are copied to where they can be fetched 16 bytes at a time
    int64_t pitch = 0;                      // of packed rows
    int64_t bytes_w = 0, bytes_x = 0, bytes_parts = 0;
    int64_t workspace() const { return bytes_w + bytes_x + bytes_parts; }
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// Rows the DMA can fetch: 16-byte aligned, and offsets inside a tile's 256 rows in 24 x 24 bits.
bool fetchable(const void* p, int64_t stride, int64_t rows) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows <= 1 || (stride % 8 == 0 && stride < 1 << 22)); }

Plan make_plan(const dgnn_dense_args& a)
{
    Plan best;
    const int64_t tiles_k = ceil_div(a.k, 64);
    const bool ready_w = fetchable(a.w, a.ldw, a.n), ready_x = fetchable(a.x, a.ldx, a.m);
    // fragments straight from memory: bound by what a unit's L1 passes on; rows that are not there cost nothing, unaligned ones nearly twice
    const double few = (double)(a.m < a.n ? a.m : a.n), tiles = (double)ceil_div(a.m, 16) * (double)ceil_div(a.n, 16);
    const double bytes = ((double)a.m + (double)a.n) * (double)a.k * 2;
    double price = (tiles > kUnits ? tiles / kUnits : 1.0) * (double)tiles_k * (0.08 + 0.066 * (few < 16 ? few : 16) / 16) * (ready_w && ready_x ? 1.0 : 1.9);
    price = (price > bytes / 5.0e6 ? price : bytes / 5.0e6) + 3.0;
    if (a.k == 0) return best;
    double packing = 0.0;
    const int64_t pitch = round_up(a.k, 64);
    if (!ready_w || !ready_x) {
        if (pitch >= 1 << 22) return best;
        packing = kLaunch + (double)((ready_w ? 0 : a.n) + (ready_x ? 0 : a.m)) * (double)pitch * 4 / 4.0e6;
    }
    for (int f = 0; f < kNumForms; ++f) {
        const Form& form = kForms[f];
        const double count = (double)ceil_div(a.m, form.bm) * (double)ceil_div(a.n, form.bn);
        // shares of k where they give idle units something to do, of 256 columns at least
        int64_t most = 1;
        if (count * 2 <= kUnits * form.per_unit && a.k >= 512) {
            most = (int64_t)(kUnits * form.per_unit / count);
            most = most > a.k / 256 ? a.k / 256 : most;
            most = most > kMaxSplits ? kMaxSplits : most;
        }
        for (int64_t splits = 1; splits <= most; splits = splits < 4 ? splits + 1 : splits + 2) {
            const int64_t share = round_up(ceil_div(a.k, splits), 64);
            if (ceil_div(a.k, share) != splits) continue;
            const double all = count * (double)splits, slots = kUnits * form.per_unit, rounds = (double)(int64_t)((all + slots - 1) / slots);
            // (the units that hold two workgroups slow down those alone)
            const double full = all >= slots ? 1.0 : all <= kUnits ? 0.0 : (all - kUnits) / (slots - kUnits);
            const double each = (double)(share / 64) * (form.alone + (form.crowded - form.alone) * full) + form.fixed;
            const double join = splits > 1 ? kLaunch + (double)splits * (double)a.m * (double)a.n * 8 / 3.0e6 : 0.0;
            const double work = rounds * each, cost = (work > bytes / 4.4e6 ? work : bytes / 4.4e6) + join + packing;
            if (cost >= price) continue;
            price = cost;
            best.form = f;
            best.splits = splits;
            best.share = share;
        }
    }
    if (best.form == kDirect) return best;
    best.pack_w = !ready_w;
    best.pack_x = !ready_x;
    best.pitch = pitch;
    best.bytes_w = best.pack_w ? round_up(a.n * pitch * 2, 256) : 0;
    best.bytes_x = best.pack_x ? round_up(a.m * pitch * 2, 256) : 0;
    best.bytes_parts = best.splits > 1 ? best.splits * a.m * a.n * 4 + 32 : 0;      // (the last row is read by eights)
    return best;
}

template <typename T, int FN, int FM, int WN, int WM, int S, int KG>
hipError_t launch_tiles(const dgnn_dense_args& a, const Plan& plan, float* parts, hipStream_t stream)
{
    typedef Tile<T, FN, FM, WN, WM, S, KG> Work;
    const int64_t tiles_m = ceil_div(a.m, Work::BM), tiles_n = ceil_div(a.n, Work::BN), all = tiles_m * tiles_n * plan.splits;
    return launch(dense_tile_kernel<T, FN, FM, WN, WM, S, KG>, dim3((unsigned)(all < kMaxGrid ? all : kMaxGrid)), dim3(Work::kThreads), stream,
                  a, tiles_m, tiles_n, plan.splits, plan.share, parts);
}

// Threads side by side on a row of `columns`, eight to each: a power of two, a workgroup at most.
int lanes_for(int64_t columns)
{
    int lanes = 1;
    while (lanes < 256 && lanes * 8 < columns) lanes *= 2;
    return lanes;
}

template <typename T>
hipError_t launch_direct(const dgnn_dense_args& a, hipStream_t stream)
{
    const int64_t tiles_n = ceil_div(a.n, 16), tiles = ceil_div(a.m, 16) * tiles_n, steps = ceil_div(a.k, 32);
    int waves = 16;                                             // as many as give every unit sixteen, and each a few steps of its own
    while (waves > 4 && (tiles * waves > 4096 || waves * 4 > steps)) waves /= 2;
    return launch(dense_direct_kernel<T>, dim3((unsigned)(tiles < kMaxGrid ? tiles : kMaxGrid)), dim3(waves * 64), stream, a, tiles_n, tiles);
}

template <typename T>
hipError_t launch_typed(dgnn_dense_args a, hipStream_t stream)
{
    const Plan plan = make_plan(a);
    if (plan.form == kDirect) return launch_direct<T>(a, stream);
    char* const memory = static_cast<char*>(a.workspace);
    float* const parts = plan.splits > 1 ? reinterpret_cast<float*>(memory + plan.bytes_w + plan.bytes_x) : nullptr;
    if (plan.pack_w || plan.pack_x) {
        const Packing w{static_cast<const uint16_t*>(a.w), reinterpret_cast<uint16_t*>(memory), plan.pack_w ? a.n : 0, a.ldw};
        const Packing x{static_cast<const uint16_t*>(a.x), reinterpret_cast<uint16_t*>(memory + plan.bytes_w), plan.pack_x ? a.m : 0, a.ldx};
        const int lanes = lanes_for(plan.pitch);
        const int64_t blocks = ceil_div(w.rows + x.rows, 256 / lanes);
        const hipError_t err = launch(dense_pack_kernel, dim3((unsigned)(blocks < kMaxGrid ? blocks : kMaxGrid)), dim3(256), stream, w, x, a.k, plan.pitch, lanes);
        if (err != hipSuccess) return err;
        if (plan.pack_w) { a.w = w.to; a.ldw = plan.pitch; }
        if (plan.pack_x) { a.x = x.to; a.ldx = plan.pitch; }
        if (plan.pack_w && plan.pack_x) a.k = plan.pitch;       // the zeros behind the rows are as good as the rows' end
    }
    hipError_t err = hipErrorInvalidValue;
    switch (plan.form) {
    case 0: err = launch_tiles<T, 1, 1, 4, 1, 8, 1>(a, plan, parts, stream); break;
    case 1: err = launch_tiles<T, 1, 1, 1, 4, 8, 1>(a, plan, parts, stream); break;
    case 2: err = launch_tiles<T, 1, 1, 2, 2, 8, 1>(a, plan, parts, stream); break;
    case 3: err = launch_tiles<T, 2, 2, 2, 2, 4, 1>(a, plan, parts, stream); break;
    case 4: err = launch_tiles<T, 4, 2, 2, 2, 4, 1>(a, plan, parts, stream); break;
    case 5: err = launch_tiles<T, 4, 2, 2, 4, 4, 1>(a, plan, parts, stream); break;
    case 6: err = launch_tiles<T, 4, 8, 4, 2, 2, 1>(a, plan, parts, stream); break;
    case 7: err = launch_tiles<T, 1, 1, 2, 2, 4, 4>(a, plan, parts, stream); break;
    case 8: err = launch_tiles<T, 2, 2, 2, 2, 4, 2>(a, plan, parts, stream); break;
    }
    if (err != hipSuccess || !parts) return err;
    const int lanes = lanes_for(a.n);
    const int64_t blocks = ceil_div(a.m, 256 / lanes);
    return launch(dense_join_kernel<T>, dim3((unsigned)(blocks < kMaxGrid ? blocks : kMaxGrid)), dim3(256), stream, a, (int)plan.splits, lanes, parts);
}

}  // namespace

int64_t dense_workspace(const dgnn_dense_args& a) { return make_plan(a).workspace(); }

hipError_t launch_dense(const dgnn_dense_args& a, hipStream_t stream)
{
    return a.type == DGNN_F16 ? launch_typed<f16>(a, stream) : launch_typed<bf16>(a, stream);
}

}  // namespace ops
}  // namespace dgnn
