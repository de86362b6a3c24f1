// Linear layers on gfx950: a matrix product with bias, activation and residual in its epilogue, dense or with one weight
// matrix per modality over rows sorted by modality, and its gradients.
//
//   z = x W^T + b,  y = act(z) + residual             act: none, relu, gelu (erf), silu
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz
//
// Types float, bfloat16, half; sums are float.  z is kept for the backward pass in the layers' type when there is an
// activation: one rounding, half a step of the type relative to z, and act' is taken at that point (it adds 3 % to the error of dx and
// dW).  dz is rounded once to that type, the one the matrix cores multiply (dx and dW are off by sqrt 2 times their own rounding); db
// is the sum of dz before that rounding.  (In 32 bits z would move 270 MB more and dz 400, of the 1.9 GB that 32 768 rows of
// 2048 -> 2048 move forward and back.)
#include "linear_kernel.h"

// One or two matrices laid out anew with rows that start where the LDS loads want them (a 16-bit row of odd length starts on 2
// bytes, their unit is 4): rows of `cols` elements, from ld to ldo apart, eight elements a thread.  Short of large ones a launch
// (2614 x 97 and 201 x 97 halves: 4.9 us).
template <typename T>
struct LinCopy {
    const T *from;
    T *to;
    int64_t rows, ld, ldo;
    int cols;
};
template <typename T>
__global__ __launch_bounds__(256) void k_linear_relayout(LinCopy<T> p, LinCopy<T> q, int64_t first_blocks) {
    const bool second = blockIdx.x >= first_blocks;
    const LinCopy<T> &m = second ? q : p;
    const int64_t block = second ? blockIdx.x - first_blocks : blockIdx.x, blocks = second ? gridDim.x - first_blocks : first_blocks;
    const uint32_t per = (uint32_t)(m.cols + 7) / 8;
    // a block takes a run of rows, so that the division stays in 32 bits
    const int64_t run = (m.rows + blocks - 1) / blocks, r0 = block * run;
    const int64_t mine = m.rows - r0 < run ? m.rows - r0 : run;
    if (mine <= 0) return;
    typedef typename LinLoose<T, 8>::type loose;
    for (uint32_t i = threadIdx.x; i < (uint32_t)mine * per; i += 256) {
        const uint32_t r = i / per, c = lin_piece_at((i - r * per) * 8, m.cols, 8);
        const T *from = m.from + (r0 + r) * m.ld + c;
        T *to = m.to + (r0 + r) * m.ldo + c;
        if (m.cols >= 8) *reinterpret_cast<loose *>(to) = *reinterpret_cast<const loose *>(from);
        else
            for (int e = 0; e < m.cols; ++e) to[e] = from[e];
    }
}

// dz = g * act'(z), 16 bytes a thread.  HBM-bound: g and z are read (once, past the caches), dz is written for the products that
// follow (73 568 x 512 floats 68 us, 6.6 TB/s).  Rows of dz may lie further apart than those of g and z (ldo).
template <typename T>
__global__ __launch_bounds__(256) void k_linear_act_grad(const T *__restrict__ g, const T *__restrict__ z, int64_t rows, int cols,
                                                         int act, const int32_t *offsets, int n_sets, T *__restrict__ dz,
                                                         int64_t ldo) {
    constexpr int N = 16 / (int)sizeof(T);
    typedef typename LinLoose<T, N>::type loose;
    if (offsets != nullptr) {
        const int64_t end = offsets[n_sets];
        rows = end < rows ? (end < 0 ? 0 : end) : rows;
    }
    auto one = [&](const loose &gv, const loose &zv, T *to) {
        float v[N];
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = to_f32(gv[e]) * lin_slope(to_f32(zv[e]), act);
        lin_store<T, N>(to, v);
    };
    if (ldo == cols) {  // one long row
        const int64_t n = rows * cols;
        for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * N; i < n; i += (int64_t)gridDim.x * 256 * N) {
            if (i + N <= n) {
                one(__builtin_nontemporal_load(reinterpret_cast<const loose *>(g + i)),
                    __builtin_nontemporal_load(reinterpret_cast<const loose *>(z + i)), dz + i);
            } else {
                for (int64_t e = i; e < n; ++e) dz[e] = from_f32<T>(to_f32(g[e]) * lin_slope(to_f32(z[e]), act));
            }
        }
        return;
    }
    const uint32_t per = (uint32_t)(cols + N - 1) / N;
    const int64_t run = (rows + gridDim.x - 1) / gridDim.x, r0 = blockIdx.x * run;
    const int64_t mine = rows - r0 < run ? rows - r0 : run;
    if (mine <= 0) return;
    for (uint32_t i = threadIdx.x; i < (uint32_t)mine * per; i += 256) {
        const uint32_t r = i / per, c = lin_piece_at((i - r * per) * N, cols, N);
        const int64_t at = (r0 + r) * cols + c;
        T *to = dz + (r0 + r) * ldo + c;
        if (cols >= N) {
            one(__builtin_nontemporal_load(reinterpret_cast<const loose *>(g + at)),
                __builtin_nontemporal_load(reinterpret_cast<const loose *>(z + at)), to);
        } else {
            for (int e = 0; e < cols; ++e)
                to[e] = from_f32<T>(to_f32(g[at + e]) * lin_slope(to_f32(z[at + e]), act));
        }
    }
}

// The same with db: a workgroup has 1 << bits rows of a set (of the matrix, if there is one) and 64 pieces of columns at most; a thread
// keeps one piece's eight columns and goes down its rows, the threads of a piece are added through LDS in a fixed order.  16-bit types
// with gelu or silu only: elsewhere dz is exact in its type and the weight gradient sums it by the way.  Bound like the above, and by
// the search for the set: 32 768 x 2048 bfloat16 74 us (65 without db), 143 760 x 256 over 400 sets 49 (37).
struct LinSums {
    float *partial;  // [parts][cols rounded up to 4]: the sums of sets that have more than one piece
    void *out;       // db [n_sets][cols]
    int bits;
    int64_t parts;   // room for so many
};
constexpr int SUMS_PIECES = 64;
template <typename T, int ACT>
__global__ __launch_bounds__(256) void k_linear_act_grad_sums(const T *__restrict__ g, const T *__restrict__ z, int64_t rows, int cols,
                                                              const int32_t *offsets, int n_sets, T *__restrict__ dz, int64_t ldo,
                                                              LinSums b) {
    constexpr int N = 16 / (int)sizeof(T), AT_ONCE = 4;
    typedef typename LinLoose<T, N>::type loose;
    __shared__ f32x4v sums[2][256];
    const int tid = threadIdx.x;
    LinPiece p{0, lin_pieces(rows, b.bits, 1), (int64_t)blockIdx.x, 0, rows, 0};
    if (offsets != nullptr) {
        if (!lin_find<true>(offsets, n_sets, n_sets - 1, rows, b.bits, 1, blockIdx.x, &p)) return;
    } else if (p.index >= p.count) {
        return;
    }
    const int per = (cols + N - 1) / N, first = (int)blockIdx.y * SUMS_PIECES, pieces = per - first < SUMS_PIECES ? per - first : SUMS_PIECES;
    const int groups = 256 / pieces, group = tid / pieces, x = first + tid % pieces;
    const int c = (int)lin_piece_at((uint32_t)x * N, cols, N);
    const int n = cols < N ? cols : N, again = x * N - c;  // what the piece before has too
    const int64_t lo = p.lo + (p.index << b.bits), end = p.hi - lo < (1ll << b.bits) ? p.hi : lo + (1ll << b.bits);
    float sum[N];
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] = 0.f;
    if (group < groups) {
        for (int64_t r0 = lo + group; r0 < end; r0 += groups * AT_ONCE) {
            loose gv[AT_ONCE], zv[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const int64_t r = r0 + u * groups < end ? r0 + u * groups : r0, at = r * cols + c;
                if (n == N) {
                    gv[u] = __builtin_nontemporal_load(reinterpret_cast<const loose *>(g + at));
                    zv[u] = __builtin_nontemporal_load(reinterpret_cast<const loose *>(z + at));
                } else {
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        gv[u][e] = e < n ? g[at + e] : (T)0.f;
                        zv[u][e] = e < n ? z[at + e] : (T)0.f;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const int64_t r = r0 + u * groups;
                if (r >= end) break;
                float v[N];
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    v[e] = to_f32(gv[u][e]) * lin_slope(to_f32(zv[u][e]), ACT);
                    sum[e] += v[e];
                }
                T *to = dz + r * ldo + c;
                if (n == N) lin_store<T, N>(to, v);
                else {
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        if (e < n) to[e] = from_f32<T>(v[e]);
                }
            }
        }
    }
    static_assert(N == 8, "two quads a piece");
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[q][tid][e] = sum[q * 4 + e];
    int most = 1;
    while (most < groups) most *= 2;
    for (int half = most / 2; half > 0; half /= 2) {
        __syncthreads();
        if (group < half && group + half < groups) {
            sums[0][tid] += sums[0][tid + half * pieces];
            sums[1][tid] += sums[1][tid + half * pieces];
        }
    }
    if (group != 0) return;
    const int64_t part = p.split_at + p.index, ld = (cols + 3) / 4 * 4;
    if (p.count > 1 && part >= b.parts) return;  // offsets that overlap: more parts than there can be
    for (int e = again; e < n; ++e) {
        const float v = sums[e >> 2][tid][e & 3];
        if (p.count > 1) b.partial[part * ld + c + e] = v;
        else reinterpret_cast<T *>(b.out)[(int64_t)p.set * cols + c + e] = from_f32<T>(v);
    }
}

// The parts of a cut weight gradient, or of a bias gradient, added in a fixed order: G groups of parts side by side, then the groups.
// A workgroup takes 1024 / G of a set's n elements; sets in one part are done already.
struct LinJoin {
    const float *partial;  // [parts][ld]
    void *out;             // [n_sets][n]
    int64_t n, ld;
    int bits;
    int64_t parts;
};
template <typename T, int G>
__device__ __forceinline__ void lin_join(const LinJoin &j, const int32_t *offsets, int n_sets, int64_t rows, unsigned block, f32x4v *sums) {
    constexpr int E = 256 / G;  // threads of a group, four elements each
    const int mine = threadIdx.x % E, group = threadIdx.x / E, set = blockIdx.y;
    int64_t first = 0;
    int count = lin_pieces(rows, j.bits, 1);
    if (offsets != nullptr) {
        int64_t lo, hi;
        lin_bounds(offsets, set, n_sets, rows, &lo, &hi);
        count = lin_pieces(hi - lo, j.bits, 1);
        if (count <= 1) return;
        first = lin_parts_before(offsets, n_sets, set, rows, j.bits);
    }
    if (count <= 1 || first + count > j.parts) return;
    const int64_t i0 = ((int64_t)block * E + mine) * 4;
    f32x4v s = {0.f, 0.f, 0.f, 0.f};
    if (i0 + 4 <= j.ld && j.ld % 4 == 0) {
        const float *at = j.partial + first * j.ld + i0;
#pragma unroll 4
        for (int p = group; p < count; p += G) s += *reinterpret_cast<const f32x4v *>(at + p * j.ld);
    } else {
        for (int e = 0; e < 4; ++e) {
            if (i0 + e >= j.n) break;
            const float *at = j.partial + first * j.ld + i0 + e;
            for (int p = group; p < count; p += G) s[e] += at[p * j.ld];
        }
    }
    if constexpr (G > 1) {
        sums[threadIdx.x] = s;
        for (int half = G / 2; half > 0; half /= 2) {
            __syncthreads();
            if (group < half) sums[threadIdx.x] += sums[threadIdx.x + half * E];
        }
        if (group != 0) return;
        s = sums[mine];
    }
    for (int e = 0; e < 4; ++e)
        if (i0 + e < j.n) reinterpret_cast<T *>(j.out)[set * j.n + i0 + e] = from_f32<T>(s[e]);
}
// the weight gradient's workgroups, then the bias gradient's (BG groups)
template <typename T, int G, int BG>
__global__ __launch_bounds__(256) void k_linear_join(LinJoin weight, LinJoin bias, const int32_t *offsets, int n_sets, int64_t rows,
                                                     unsigned weight_blocks) {
    __shared__ f32x4v sums[256];
    if (blockIdx.x < weight_blocks) lin_join<T, G>(weight, offsets, n_sets, rows, blockIdx.x, sums);
    else lin_join<T, BG>(bias, offsets, n_sets, rows, blockIdx.x - weight_blocks, sums);
}

// rows behind the last set have no gradient: out = g there is none, g elsewhere
template <typename T>
__global__ __launch_bounds__(256) void k_linear_mask_rows(const T *__restrict__ g, int64_t rows, int cols, const int32_t *offsets,
                                                          int n_sets, T *__restrict__ out) {
    int64_t end = offsets[n_sets];
    end = end < 0 ? 0 : (end < rows ? end : rows);
    const int64_t n = rows * cols, held = end * cols;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
        out[i] = i < held ? g[i] : (T)0.f;
}

namespace {

int elem_size(int dtype) { return dtype == MTP_FLOAT ? 4 : 2; }
int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
unsigned grid_for(int64_t items) {
    const int64_t b = (items + 255) / 256;
    return (unsigned)(b < 1 ? 1 : (b > 256 * 16 ? 256 * 16 : b));
}

// Tiles of 16 rows that k_linear_few works on at a time, 0: the product is too much for it.  Microseconds, few / tiles: bfloat16
// 64 rows of 2048 x 2048 10.8 / 16.9, 512 of 512 x 512 7.5 / 7.2, 256 of 2048 x 2048 33 / 17; float 64 of 2048 x 2048 18.8 / 50
// (two row tiles 16.6), 256 of 2048 x 2048 64 / 51.  One matrix per modality: 64 rows over 200 of 512 x 128 7.9 / 12.3,
// 2000 rows over 200 of 256 x 96 13.6 / 8.8.
int few_rows(int64_t rows, int in, int out, bool grouped, bool half) {
    const int64_t products = rows * in * out;
    if (rows > 512 || products > (half ? 1ll << 28 : 1ll << 29)) return 0;
    return !grouped && products >= 1ll << 28 ? 2 : 1;
}

// rows of a 16-bit operand have to start on 4 bytes; a row distance beyond 2^20 elements would leave the loads' 32-bit offsets
bool needs_relayout(int dtype, const void *p, int64_t ld) {
    return ld > (1 << 20) || (elem_size(dtype) == 2 && (ld % 2 != 0 || (uintptr_t)p % 4 != 0));
}
int64_t relayout_bytes(int dtype, const void *p, int64_t ld, int64_t rows, int64_t cols) {
    return needs_relayout(dtype, p, ld) ? round_up(rows * round_up(cols, 8) * elem_size(dtype), 256) : 0;
}

// blocks for a copy of rows x cols: some eight pieces of eight elements a thread, a run of rows each
int64_t copy_blocks(int64_t rows, int cols) {
    const int64_t b = (rows * ((cols + 7) / 8) + 2047) / 2048;
    return b < 1 ? 1 : (b > 65536 ? 65536 : (b > rows && rows > 0 ? rows : b));
}
// the two operands of a product, where they need it
template <typename T>
int relayout(const void **a, int64_t *lda, int64_t a_rows, int a_cols, const void **b, int64_t *ldb, int64_t b_rows, int b_cols,
             char **ws, hipStream_t s) {
    const int dtype = sizeof(T) == 4 ? MTP_FLOAT : MTP_BFLOAT16;
    LinCopy<T> c[2];
    int n = 0;
    auto take = [&](const void **p, int64_t *ld, int64_t rows, int cols) {
        const int64_t bytes = relayout_bytes(dtype, *p, *ld, rows, cols);
        if (bytes == 0) return;
        c[n++] = LinCopy<T>{reinterpret_cast<const T *>(*p), reinterpret_cast<T *>(*ws), rows, *ld, round_up(cols, 8), cols};
        *p = *ws;
        *ld = round_up(cols, 8);
        *ws += bytes;
    };
    take(a, lda, a_rows, a_cols);
    take(b, ldb, b_rows, b_cols);
    if (n == 0) return MTP_OK;
    const int64_t first = copy_blocks(c[0].rows, c[0].cols), second = n == 2 ? copy_blocks(c[1].rows, c[1].cols) : 0;
    hipLaunchKernelGGL(k_linear_relayout<T>, dim3((unsigned)(first + second)), dim3(256), 0, s, c[0], c[n - 1], first);
    MTP_LAUNCH_CHECK();
    return MTP_OK;
}

// Which tile: columns x rows of the output a workgroup owns.  Measured on the card, microseconds of one product:
//   TILE_32x128   few columns (143 760 rows, 256 -> 24, bfloat16: 20, 24 with 64x64, 29 with 128x128), few tiles in all
//                 (1024 rows, 256 -> 200: 5.1, 6.9 with 128x128), float with up to 96 columns (73 568 rows, 512 -> 96: 72,
//                 82 with 96x128, 113 with 128x128)
//   TILE_64x64    few tiles and few rows; weight gradients of float (8192 rows, 512 x 512: 65, 75 with 128x64)
//   TILE_64x128   up to 64 columns (300 000 rows, 96 -> 64: 18, 25 with 128x64)
//   TILE_96x128   up to 96 columns of 16-bit types (143 760 rows, 256 -> 96: 30, 31 with 128x64, 37 with 32x128)
//   TILE_128x64   most others: three workgroups a CU (143 760 rows, 96 -> 256 with gelu: 62, 67 with 128x128)
//   TILE_128x128  input and weight gradients of 16-bit types, whose products are longer than their way out (143 760 rows,
//                 24 -> 256: 33, 37 with 128x64); long sums forward that give each CU two (2048 rows, 4096 -> 4096: 75, 126;
//                 8192 rows, 1024 -> 1024 with gelu: 28, 34; but 2048 rows, 2048 -> 2048: 31, 29; 8192 rows, 512 -> 512: 16.1, 15.6)
//   TILE_256x256  long sums of 16-bit types that fill the card with such tiles (32 768 rows, 2048 -> 2048: 247, 318 with
//                 128x128): half the LDS traffic a product; weight gradients with 2048 rows for each of 256 workgroups (32 768 rows,
//                 2048 x 2048: 256, 299 with 128x128; 1024 x 1024: 82, 84; 4096 rows, 2048 x 2048: 54, 51)
enum LinTileShape { TILE_32x128, TILE_64x64, TILE_64x128, TILE_96x128, TILE_128x64, TILE_128x128, TILE_256x256 };

int64_t tiles_of(int64_t rows, int64_t cols, int bc, int br) { return ((rows + br - 1) / br) * ((cols + bc - 1) / bc); }

LinTileShape pick_tile(int mode, bool half, int64_t rows, int cols, int64_t k, int n_sets) {
    if (mode == MTP_LINEAR_GRAD_WEIGHT) {  // rows, cols: of the gradient
        if (!half) return cols <= 96 ? TILE_32x128 : TILE_64x64;
        if (cols <= 32) return TILE_32x128;
        if (rows <= 64) return cols <= 64 ? TILE_64x64 : TILE_128x64;
        if (cols <= 64) return TILE_64x128;
        if (cols <= 96) return TILE_96x128;
        const int64_t big = tiles_of(rows, cols, 256, 256);
        if (n_sets == 1 && k * big >= 512 * 1024 && 4ll * rows * cols >= 3 * big * 256 * 256) return TILE_256x256;
        return tiles_of(rows, cols, 128, 128) >= 64 ? TILE_128x128 : TILE_128x64;
    }
    if (cols <= 32) return TILE_32x128;
    const int64_t least = n_sets > 1 ? (int64_t)n_sets * ((cols + 63) / 64) : 0;  // each set has a tile of its own
    if (tiles_of(rows, cols, 64, 64) + least < 512) return rows < 128 || n_sets > 1 ? TILE_64x64 : TILE_32x128;
    if (cols <= 64) return TILE_64x128;
    if (cols <= 96) return half ? TILE_96x128 : TILE_32x128;
    if (half && n_sets == 1 && k >= 512 && tiles_of(rows, cols, 256, 256) >= 192) return TILE_256x256;
    if (half && (mode == MTP_LINEAR_GRAD_INPUT || (k >= 512 && tiles_of(rows, cols, 128, 128) >= 512))) return TILE_128x128;
    return TILE_128x64;
}

// Rows of x that one workgroup of the weight gradient sums, as a power of two.
// One matrix: a part of L rows takes about 8 ns a row (23 in float), and rows / L parts of in x out floats are written and read again at
// some 5 bytes a picosecond; the sum of both is least around L^2 = rows in out / 5000 (/ 15 000), and flat towards longer parts, of
// which fewer share the card.  2614 rows, 96 x 200 fp16: 9.4 us with parts of 256 rows, 14.4 of 1024; 20 000 rows, 512 x 512 bfloat16:
// 29 of 1024, 44 of 256; 73 568 rows, 512 x 512 float 327 of 2048, 363 of 512, 353 of 4096.  256 x 256 tiles, one a CU: one part for
// each (32 768 rows, 2048 x 2048: 256 us, 282 with two, 2048 rows, 4096 x 4096: 65 us, 102 with two).
// Many: sets differ in size by a factor of ten and the longest one is what the others wait for, but parts have to be written and added
// (143 760 rows over 400, 96 -> 256: 36 us with parts of 2048, 40 of 1024, 47 of 512; 52 280 rows over 200: 23 us of 1024, 29 of 2048).
int part_bits_for(int64_t rows, int in, int out, int n_sets, bool half) {
    int bits = 6;
    if (n_sets == 1) {
        if (pick_tile(MTP_LINEAR_GRAD_WEIGHT, half, out, in, rows, 1) == TILE_256x256) {
            while (bits < 30 && ((int64_t)256 << bits) < rows * tiles_of(out, in, 256, 256)) ++bits;
            return bits;
        }
        const double least = (double)rows * in * out / (half ? 2500 : 6700);
        while ((double)((int64_t)1 << bits) * (double)((int64_t)1 << bits) < least) ++bits;
        return bits;
    }
    bits = half ? 10 : 9;
    while (bits < 30 && ((int64_t)160 << bits) < rows * tiles_of(out, in, in <= 64 ? 64 : 128, out <= 64 ? 64 : 128)) ++bits;
    return bits;
}
// parts of the sets that have more than one: such a set has more rows than `part`, so fewer parts than twice its rows / part
int64_t most_parts(int64_t rows, int n_sets, int bits) {
    if (n_sets == 1) return rows <= (int64_t)1 << bits ? 0 : (rows + ((int64_t)1 << bits) - 1) >> bits;
    return (2 * rows) >> bits;
}

// db summed beside dz: 16-bit types whose slope is not 0 or 1
bool sums_beside(int dtype, int act) { return elem_size(dtype) == 2 && (act == LIN_GELU || act == LIN_SILU); }
int sums_tiles(int out) { return ((out + 7) / 8 + SUMS_PIECES - 1) / SUMS_PIECES; }  // of columns
// rows of one workgroup there, as a power of two: two rows a thread at least, and some 2000 workgroups (143 760 x 256 over 400 sets: up
// to 2560 of them 49 us, 1280 52, 640 63, 5120 52; 32 768 x 2048 with its join 91, 90, 96, 99)
int sum_bits_for(int64_t rows, int out) {
    const int per = (out + 7) / 8, pieces = per < SUMS_PIECES ? per : SUMS_PIECES;
    int bits = 4;
    while ((1 << bits) < 2 * (256 / pieces)) ++bits;
    while (bits < 30 && (rows >> bits) * sums_tiles(out) > 2560) ++bits;
    return bits;
}
int64_t sums_bytes(int64_t rows, int out, int n_sets) { return most_parts(rows, n_sets, sum_bits_for(rows, out)) * round_up(out, 4) * 4; }
template <typename T>
int launch_sums(const void *g, const void *pre, int64_t rows, int out, int act, const int32_t *offsets, int n_sets, void *dz, int64_t lddz,
                const LinSums &b, hipStream_t s) {
    const int64_t pieces = offsets == nullptr ? lin_pieces(rows, b.bits, 1) : (rows >> b.bits) + n_sets;
    const dim3 grid((unsigned)pieces, (unsigned)sums_tiles(out));
    if (act == LIN_GELU)
        hipLaunchKernelGGL((k_linear_act_grad_sums<T, LIN_GELU>), grid, dim3(256), 0, s, reinterpret_cast<const T *>(g),
                           reinterpret_cast<const T *>(pre), rows, out, offsets, n_sets, reinterpret_cast<T *>(dz), lddz, b);
    else
        hipLaunchKernelGGL((k_linear_act_grad_sums<T, LIN_SILU>), grid, dim3(256), 0, s, reinterpret_cast<const T *>(g),
                           reinterpret_cast<const T *>(pre), rows, out, offsets, n_sets, reinterpret_cast<T *>(dz), lddz, b);
    MTP_LAUNCH_CHECK();
    return MTP_OK;
}

// Up to so many workgroups the two products of a backward pass share a launch, in tiles that leave room for each other on a CU; in
// launches of their own they have tiles of their own size.  Both products, microseconds in one launch / in two:
//   bfloat16 2614 rows, 96 -> 200 8.4 / 13.7, 20 000 rows, 96 -> 200 15.7 / 19.9, 4096 rows, 1024 -> 1024 42 / 46; 30 000 rows,
//   200 -> 200 32.2 / 32.5 (over the limit)
//   float 2614 rows, 96 -> 200 13.5 / 19.1, 40 000 rows, 64 -> 64 22 / 31, 20 000 rows, 96 -> 96 24 / 23, 8000 rows, 512 -> 512 88 / 85
//   sets, of whose tiles many are empty: bfloat16 5000 rows over 100, 200 -> 200 15.5 / 19.3 (2372 workgroups), 20 000 over 300,
//   256 -> 24 17.8 / 19.6 (2300), 52 280 over 200, 96 -> 256 29.3 / 28.1 (3032)
int64_t both_blocks(int n_sets, bool half) { return n_sets > 1 ? 2560 : half ? 2048 : 1024; }

// Outputs larger than this leave past the caches (what is kept for the backward pass always does): 73 568 x 512 floats with gelu
// and a residual 139 -> 135 us for what is kept, 119 for both.
constexpr int64_t AWAY_BYTES = 64ll << 20;

// a's tiles of BC columns x BR rows, and the workgroups of NT threads for them
template <typename T, int MODE, int BC, int BR, int NT>
int set_tiles(LinArgs *a, int64_t *blocks) {
    a->col_tiles = (a->cols + BC - 1) / BC;
    if (MODE == LIN_GRAD_WEIGHT) {
        a->row_tiles = (a->out_rows + BR - 1) / BR;
        // of sets at most so many
        const int64_t pieces = a->offsets == nullptr ? lin_pieces(a->rows, a->part_bits, 1) : (a->rows >> a->part_bits) + a->n_sets;
        *blocks = a->row_tiles * a->col_tiles * pieces;
    } else {
        // a set's last tile may be ragged, and so may the one behind the last set; each has a row
        a->row_tiles = a->offsets == nullptr ? (a->rows + BR - 1) / BR : (a->rows + (int64_t)(a->n_sets + 1) * (BR - 1)) / BR;
        if (a->row_tiles > a->rows) a->row_tiles = a->rows;
        *blocks = a->row_tiles * a->col_tiles;
        a->away = a->rows * a->cols * (int64_t)sizeof(T) > AWAY_BYTES;
    }
    MTP_REQUIRE(*blocks * NT <= 0xffffffffll, "mtp_linear: %lld workgroups are too many", (long long)*blocks);
    a->tiles = (uint32_t)*blocks;
    if (MODE != LIN_GRAD_WEIGHT && a->offsets != nullptr && a->n_sets < 512) {  // as many workgroups as have a place
        int cus = 0;
        const int rc = mtp_device_cu_count(&cus);
        if (rc != MTP_OK) return rc;
        const int64_t places = (int64_t)cus * lin_waves(BC, BR, NT) * 256 / NT;
        if (*blocks > places) *blocks = places;
    }
    return MTP_OK;
}

template <typename T, int MODE, int BC, int BR, int WC, int WR>
int launch_tile(LinArgs a, hipStream_t s) {
    constexpr int NT = 64 * (BC / WC) * (BR / WR);
    constexpr int LDS = 2 * (BC + BR) * 128;
    int64_t blocks;
    const int rc = set_tiles<T, MODE, BC, BR, NT>(&a, &blocks);
    if (rc != MTP_OK || blocks == 0) return rc;
    MTP_SET_MAX_LDS_ONCE((k_linear_tile<T, MODE, BC, BR, WC, WR>), LDS);
    hipLaunchKernelGGL((k_linear_tile<T, MODE, BC, BR, WC, WR>), dim3((unsigned)blocks), dim3(NT), LDS, s, a);
    MTP_LAUNCH_CHECK();
    return MTP_OK;
}

// Both products of a backward pass in one launch, if they are small; *done says whether.
template <typename T, int BC, int BR>
int launch_both(LinArgs input, LinArgs weight, bool *done, hipStream_t s) {
    constexpr int LDS = 2 * (BC + BR > 128 ? BC + BR : 128) * 128;
    int64_t input_blocks, weight_blocks;
    int rc = set_tiles<T, LIN_GRAD_INPUT, BC, BR, 256>(&input, &input_blocks);
    if (rc == MTP_OK) rc = set_tiles<T, LIN_GRAD_WEIGHT, 64, 64, 256>(&weight, &weight_blocks);
    *done = rc == MTP_OK && input_blocks + weight_blocks <= both_blocks(input.n_sets, sizeof(T) == 2);
    if (!*done) return rc;
    MTP_SET_MAX_LDS_ONCE((k_linear_both<T, BC, BR>), LDS);
    hipLaunchKernelGGL((k_linear_both<T, BC, BR>), dim3((unsigned)(input_blocks + weight_blocks)), dim3(256), LDS, s, input, weight,
                       (uint32_t)input_blocks);
    MTP_LAUNCH_CHECK();
    return MTP_OK;
}

template <typename T, int MODE>
int launch_product(const LinArgs &a, hipStream_t s) {
    const bool half = sizeof(T) == 2;
    switch (pick_tile(MODE, half, MODE == LIN_GRAD_WEIGHT ? a.out_rows : a.rows, a.cols, a.k, a.n_sets)) {
        case TILE_32x128: return launch_tile<T, MODE, 32, 128, 32, 32>(a, s);
        case TILE_64x64: return launch_tile<T, MODE, 64, 64, 32, 32>(a, s);
        case TILE_64x128: return launch_tile<T, MODE, 64, 128, 32, 64>(a, s);
        case TILE_128x64: return launch_tile<T, MODE, 128, 64, 64, 32>(a, s);
        case TILE_96x128:
            if constexpr (sizeof(T) == 2) return launch_tile<T, MODE, 96, 128, 96, 32>(a, s);
        case TILE_128x128:
            if constexpr (sizeof(T) == 2) return launch_tile<T, MODE, 128, 128, 64, 64>(a, s);
        case TILE_256x256:
            if constexpr (sizeof(T) == 2) return launch_tile<T, MODE, 256, 256, 128, 64>(a, s);
    }
    mtp_set_error("mtp_linear: no kernel of this shape");
    return MTP_E_ARG;
}

// Few rows (of each set): see k_linear_few.  RT tiles of 16 rows share a reading of W.
template <typename T, int RT>
int launch_few(LinArgs a, hipStream_t s) {
    a.col_tiles = (a.cols + 15) / 16;
    a.row_tiles = a.offsets == nullptr ? (a.rows + 16 * RT - 1) / (16 * RT)
                                       : (a.rows + (int64_t)(a.n_sets + 1) * (16 * RT - 1)) / (16 * RT);
    const int64_t most = a.offsets == nullptr ? a.row_tiles : a.row_tiles < a.rows ? a.row_tiles : a.rows;  // a tile has a row
    const int64_t blocks = most * a.col_tiles;
    MTP_REQUIRE(blocks * 256 <= 0xffffffffll, "mtp_linear: %lld workgroups are too many", (long long)blocks);
    hipLaunchKernelGGL((k_linear_few<T, RT>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    MTP_LAUNCH_CHECK();
    return MTP_OK;
}

int check_sizes(const char *who, int dtype, int64_t rows, int in, int out, const int32_t *offsets, int n_sets) {
    MTP_REQUIRE(dtype == MTP_FLOAT || dtype == MTP_BFLOAT16 || dtype == MTP_HALF, "%s: unknown type %d", who, dtype);
    MTP_REQUIRE(rows >= 0 && rows <= 0x7fffffff && in >= 1 && out >= 1 && in <= 65536 && out <= 65536,
                "%s: bad shape rows=%lld in=%d out=%d", who, (long long)rows, in, out);
    MTP_REQUIRE(n_sets >= 1 && n_sets <= 65535 && (offsets != nullptr || n_sets == 1), "%s: bad number of sets %d", who, n_sets);
    return MTP_OK;
}

template <typename T>
int forward(const void *x, int64_t rows, int in, int64_t ldx, const void *w, int out, const void *bias, int act,
            const void *residual, int64_t ldr, const int32_t *offsets, int n_sets, void *y, void *pre, char *ws, hipStream_t s) {
    int64_t ldw = in;
    const int few = few_rows(rows, in, out, n_sets > 1, sizeof(T) == 2);
    if (few == 0) {
        const int rc = relayout<T>(&x, &ldx, rows, in, &w, &ldw, (int64_t)n_sets * out, in, &ws, s);
        if (rc != MTP_OK) return rc;
    }
    LinArgs a{};
    a.P = LinOperand{w, ldw, (int64_t)out * ldw};
    a.Q = LinOperand{x, ldx, 0};
    a.rows = rows;
    a.cols = out;
    a.k = in;
    a.offsets = offsets;
    a.n_sets = n_sets;
    a.bias = bias;
    a.residual = residual;
    a.ld_res = ldr;
    a.act = act;
    a.out = y;
    a.pre = pre;
    if (few == 1) return launch_few<T, 1>(a, s);
    if (few == 2) return launch_few<T, 2>(a, s);
    return launch_product<T, LIN_FORWARD>(a, s);
}

// where the parts of a backward pass lie in the workspace, one behind the other: dz, the bias gradient's parts where it is summed beside
// dz, the weights and x with rows as the products load them, the weight gradient's parts
struct BackwardPlan {
    int64_t lddz, dz_bytes, w_bytes, x_bytes, parts_bytes, sums_bytes;
    int64_t total() const { return dz_bytes + w_bytes + x_bytes + parts_bytes + sums_bytes; }
};
BackwardPlan plan_backward(int dtype, int64_t rows, int in, int out, int n_sets, int act, const void *g, const void *w,
                           int64_t ldw, const void *x, int64_t ldx, bool want_x, bool want_w) {
    BackwardPlan p{};
    if (act == LIN_NONE) {
        p.lddz = out;
        p.dz_bytes = relayout_bytes(dtype, g, out, rows, out);
    } else {  // dz has rows of its own, so they can start where the loads want them
        p.lddz = elem_size(dtype) == 2 && out % 2 != 0 ? round_up(out, 8) : out;
        p.dz_bytes = round_up(rows * p.lddz * elem_size(dtype), 256);
    }
    if (want_x && rows > 0) p.w_bytes = relayout_bytes(dtype, w, ldw, (int64_t)n_sets * out, in);
    if (want_w) {
        p.x_bytes = relayout_bytes(dtype, x, ldx, rows, in);
        p.parts_bytes = most_parts(rows, n_sets, part_bits_for(rows, in, out, n_sets, elem_size(dtype) == 2)) * out * (in + 1) * 4;
        if (sums_beside(dtype, act)) p.sums_bytes = round_up(sums_bytes(rows, out, n_sets), 256);
    }
    return p;
}

LinArgs input_args(const void *dz, int64_t rows, int out, int64_t lddz, const void *w, int in, int64_t ldw, const int32_t *offsets,
                   int n_sets, void *dx) {
    LinArgs a{};
    a.P = LinOperand{w, ldw, (int64_t)out * ldw};
    a.Q = LinOperand{dz, lddz, 0};
    a.rows = rows;
    a.cols = in;
    a.k = out;
    a.offsets = offsets;
    a.n_sets = n_sets;
    a.out = dx;
    return a;
}
LinArgs weight_args(bool half, const void *dz, int64_t rows, int out, int64_t lddz, const void *x, int in, int64_t ldx,
                    const int32_t *offsets, int n_sets, void *dw, void *db, char *ws) {
    LinArgs a{};
    a.P = LinOperand{x, ldx, 0};
    a.Q = LinOperand{dz, lddz, 0};
    a.rows = rows;
    a.cols = in;
    a.out_rows = out;
    a.offsets = offsets;
    a.n_sets = n_sets;
    a.k = (int)rows;
    a.part_bits = part_bits_for(rows, in, out, n_sets, half);
    a.parts = most_parts(rows, n_sets, a.part_bits);
    a.out = dw;
    a.bias_out = db;
    a.partial = reinterpret_cast<float *>(ws);
    a.partial_bias = a.partial + a.parts * out * in;
    return a;
}
// the parts of the weight gradient and of the bias gradient (`b`, where it was summed beside dz), if there are any
template <typename T>
int join_parts(const LinArgs &a, const LinSums &b, hipStream_t s) {
    const int64_t n = (int64_t)a.out_rows * a.cols;
    const LinJoin weight{a.partial, a.out, n, n, a.part_bits, a.parts};
    const LinJoin bias = a.bias_out != nullptr ? LinJoin{a.partial_bias, a.bias_out, a.out_rows, a.out_rows, a.part_bits, a.parts}
                                               : LinJoin{b.partial, b.out, a.out_rows, round_up(a.out_rows, 4), b.bits, b.parts};
    // a matrix has few biases and many parts of them, a set has few
    const int bias_each = a.n_sets > 1 ? 256 : 32, each = a.n_sets > 1 || a.parts < 8 ? 1024 : a.parts < 32 ? 256 : 64;  // of a workgroup
    const unsigned bias_blocks = bias.out != nullptr && bias.parts > 0 ? (unsigned)((bias.n + bias_each - 1) / bias_each) : 0;
    const unsigned blocks = weight.parts == 0 ? 0 : (unsigned)((weight.n + each - 1) / each);
    if (blocks + bias_blocks == 0) return MTP_OK;
    const dim3 grid(blocks + bias_blocks, (unsigned)a.n_sets);
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, weight, bias, a.offsets, a.n_sets, a.rows, blocks); };
    if (a.n_sets > 1) launch(k_linear_join<T, 1, 4>);
    else if (each == 64) launch(k_linear_join<T, 16, 32>);
    else if (each == 256) launch(k_linear_join<T, 4, 32>);
    else launch(k_linear_join<T, 1, 32>);
    MTP_LAUNCH_CHECK();
    return MTP_OK;
}

template <typename T>
int grad_input(const void *dz, int64_t rows, int out, int64_t lddz, const void *w, int in, const int32_t *offsets, int n_sets,
               void *dx, char *ws, hipStream_t s) {
    int64_t ldw = in;
    const int rc = relayout<T>(&dz, &lddz, rows, out, &w, &ldw, (int64_t)n_sets * out, in, &ws, s);
    if (rc != MTP_OK) return rc;
    return launch_product<T, LIN_GRAD_INPUT>(input_args(dz, rows, out, lddz, w, in, ldw, offsets, n_sets, dx), s);
}

template <typename T>
int grad_weight(const void *dz, int64_t rows, int out, int64_t lddz, const void *x, int in, int64_t ldx, const int32_t *offsets,
                int n_sets, void *dw, void *db, char *ws, hipStream_t s) {
    int rc = relayout<T>(&dz, &lddz, rows, out, &x, &ldx, rows, in, &ws, s);
    if (rc != MTP_OK) return rc;
    const LinArgs a = weight_args(sizeof(T) == 2, dz, rows, out, lddz, x, in, ldx, offsets, n_sets, dw, db, ws);
    rc = launch_product<T, LIN_GRAD_WEIGHT>(a, s);
    return rc != MTP_OK ? rc : join_parts<T>(a, LinSums{}, s);
}

// both from operands that need no new layout; db NULL: not wanted, or summed beside dz (`sums`)
template <typename T>
int grad_both(const void *dz, int64_t rows, int out, int64_t lddz, const void *w, int64_t ldw, const void *x, int in, int64_t ldx,
              const int32_t *offsets, int n_sets, void *dx, void *dw, void *db, const LinSums &sums, char *ws, hipStream_t s) {
    const LinArgs input = input_args(dz, rows, out, lddz, w, in, ldw, offsets, n_sets, dx);
    const LinArgs weight = weight_args(sizeof(T) == 2, dz, rows, out, lddz, x, in, ldx, offsets, n_sets, dw, db, ws);
    bool done = false;
    int rc = MTP_OK;
    if (dx != nullptr && dw != nullptr && rows > 0) {
        rc = n_sets > 1 || rows < 128 ? launch_both<T, 64, 64>(input, weight, &done, s) : launch_both<T, 32, 128>(input, weight, &done, s);
        if (rc != MTP_OK) return rc;
    }
    if (!done) {
        if (dx != nullptr && rows > 0) rc = launch_product<T, LIN_GRAD_INPUT>(input, s);
        if (rc == MTP_OK && dw != nullptr) rc = launch_product<T, LIN_GRAD_WEIGHT>(weight, s);
        if (rc != MTP_OK) return rc;
    }
    return dw != nullptr ? join_parts<T>(weight, sums, s) : rc;
}

}  // namespace

#define MTP_BY_TYPE(dtype, call)                              \
    ((dtype) == MTP_FLOAT ? call<float> : (dtype) == MTP_BFLOAT16 ? call<__bf16> : call<_Float16>)

extern "C" int64_t mtp_linear_workspace_bytes(int dtype, int step, int64_t rows, int in, int out, int n_sets, const void *a,
                                              int64_t lda, const void *b, int64_t ldb) {
    if (rows < 0 || in < 1 || out < 1 || n_sets < 1) return 0;
    const int64_t w_rows = (int64_t)n_sets * out;
    if (step == MTP_LINEAR_FORWARD && few_rows(rows, in, out, n_sets > 1, elem_size(dtype) == 2) != 0) return 0;
    if (step == MTP_LINEAR_FORWARD) return relayout_bytes(dtype, a, lda, rows, in) + relayout_bytes(dtype, b, in, w_rows, in);
    if (step == MTP_LINEAR_GRAD_INPUT) return relayout_bytes(dtype, a, lda, rows, out) + relayout_bytes(dtype, b, in, w_rows, in);
    int64_t n = relayout_bytes(dtype, a, lda, rows, out) + relayout_bytes(dtype, b, ldb, rows, in);
    return n + most_parts(rows, n_sets, part_bits_for(rows, in, out, n_sets, elem_size(dtype) == 2)) * out * (in + 1) * 4;
}

extern "C" int mtp_linear_rows_aligned(int dtype, const void *x, int64_t ld) { return !needs_relayout(dtype, x, ld); }

extern "C" int mtp_linear(int dtype, const void *x, int64_t rows, int in, int64_t ldx, const void *w, int out, const void *bias,
                          int act, const void *residual, int64_t ldr, const int32_t *offsets, int n_sets, void *y, void *pre,
                          void *ws, size_t ws_bytes, void *stream) {
    int rc = check_sizes("mtp_linear", dtype, rows, in, out, offsets, n_sets);
    if (rc != MTP_OK) return rc;
    MTP_REQUIRE(act >= LIN_NONE && act <= LIN_SILU, "mtp_linear: unknown activation %d", act);
    MTP_REQUIRE(ldx >= in && (residual == nullptr || ldr >= out), "mtp_linear: row distance below the row's length");
    if (rows == 0) return MTP_OK;
    MTP_REQUIRE(x && w && y, "mtp_linear: null pointer");
    const int64_t need = mtp_linear_workspace_bytes(dtype, MTP_LINEAR_FORWARD, rows, in, out, n_sets, x, ldx, w, in);
    if ((int64_t)ws_bytes < need || (need > 0 && (ws == nullptr || (uintptr_t)ws % 16 != 0))) {
        mtp_set_error("mtp_linear: workspace of %zu bytes, needs %lld on a 16-byte boundary", ws_bytes, (long long)need);
        return MTP_E_WORKSPACE;
    }
    return MTP_BY_TYPE(dtype, forward)(x, rows, in, ldx, w, out, bias, act, residual, ldr, offsets, n_sets, y, pre,
                                       reinterpret_cast<char *>(ws), mtp_stream(stream));
}

extern "C" int mtp_linear_act_grad(int dtype, const void *g, const void *pre, int64_t rows, int out, int act,
                                   const int32_t *offsets, int n_sets, void *dz, int64_t lddz, void *stream) {
    int rc = check_sizes("mtp_linear_act_grad", dtype, rows, 1, out, offsets, n_sets);
    if (rc != MTP_OK) return rc;
    MTP_REQUIRE(act >= LIN_NONE && act <= LIN_SILU, "mtp_linear_act_grad: unknown activation %d", act);
    MTP_REQUIRE(lddz >= out, "mtp_linear_act_grad: row distance below the row's length");
    if (rows == 0) return MTP_OK;
    MTP_REQUIRE(g && pre && dz, "mtp_linear_act_grad: null pointer");
    hipStream_t s = mtp_stream(stream);
    int64_t blocks = (rows * out + 256 * 16 - 1) / (256 * 16);
    if (lddz != out && blocks > rows) blocks = rows;
    const dim3 grid((unsigned)(blocks < 1 ? 1 : blocks > 65536 ? 65536 : blocks));
    if (dtype == MTP_FLOAT)
        hipLaunchKernelGGL(k_linear_act_grad<float>, grid, dim3(256), 0, s, (const float *)g, (const float *)pre, rows, out, act,
                           offsets, n_sets, (float *)dz, lddz);
    else if (dtype == MTP_BFLOAT16)
        hipLaunchKernelGGL(k_linear_act_grad<__bf16>, grid, dim3(256), 0, s, (const __bf16 *)g, (const __bf16 *)pre, rows, out,
                           act, offsets, n_sets, (__bf16 *)dz, lddz);
    else
        hipLaunchKernelGGL(k_linear_act_grad<_Float16>, grid, dim3(256), 0, s, (const _Float16 *)g, (const _Float16 *)pre, rows,
                           out, act, offsets, n_sets, (_Float16 *)dz, lddz);
    MTP_LAUNCH_CHECK();
    return MTP_OK;
}

extern "C" int mtp_linear_mask_rows(int dtype, const void *g, int64_t rows, int out, const int32_t *offsets, int n_sets, void *dst,
                                    void *stream) {
    int rc = check_sizes("mtp_linear_mask_rows", dtype, rows, 1, out, offsets, n_sets);
    if (rc != MTP_OK) return rc;
    if (rows == 0) return MTP_OK;
    MTP_REQUIRE(g && dst && offsets, "mtp_linear_mask_rows: null pointer");
    hipStream_t s = mtp_stream(stream);
    const dim3 grid(grid_for(rows * out));
    if (dtype == MTP_FLOAT)
        hipLaunchKernelGGL(k_linear_mask_rows<float>, grid, dim3(256), 0, s, (const float *)g, rows, out, offsets, n_sets,
                           (float *)dst);
    else  // the other two types are moved as they are
        hipLaunchKernelGGL(k_linear_mask_rows<_Float16>, grid, dim3(256), 0, s, (const _Float16 *)g, rows, out, offsets, n_sets,
                           (_Float16 *)dst);
    MTP_LAUNCH_CHECK();
    return MTP_OK;
}

extern "C" int mtp_linear_grad_input(int dtype, const void *dz, int64_t rows, int out, int64_t lddz, const void *w, int in,
                                     const int32_t *offsets, int n_sets, void *dx, void *ws, size_t ws_bytes, void *stream) {
    int rc = check_sizes("mtp_linear_grad_input", dtype, rows, in, out, offsets, n_sets);
    if (rc != MTP_OK) return rc;
    MTP_REQUIRE(lddz >= out, "mtp_linear_grad_input: row distance below the row's length");
    if (rows == 0) return MTP_OK;
    MTP_REQUIRE(dz && w && dx, "mtp_linear_grad_input: null pointer");
    const int64_t need = mtp_linear_workspace_bytes(dtype, MTP_LINEAR_GRAD_INPUT, rows, in, out, n_sets, dz, lddz, w, in);
    if ((int64_t)ws_bytes < need || (need > 0 && (ws == nullptr || (uintptr_t)ws % 16 != 0))) {
        mtp_set_error("mtp_linear_grad_input: workspace of %zu bytes, needs %lld on a 16-byte boundary", ws_bytes, (long long)need);
        return MTP_E_WORKSPACE;
    }
    return MTP_BY_TYPE(dtype, grad_input)(dz, rows, out, lddz, w, in, offsets, n_sets, dx, reinterpret_cast<char *>(ws),
                                          mtp_stream(stream));
}

extern "C" int mtp_linear_grad_weight(int dtype, const void *dz, int64_t rows, int out, int64_t lddz, const void *x, int in,
                                      int64_t ldx, const int32_t *offsets, int n_sets, void *dw, void *db, void *ws,
                                      size_t ws_bytes, void *stream) {
    int rc = check_sizes("mtp_linear_grad_weight", dtype, rows, in, out, offsets, n_sets);
    if (rc != MTP_OK) return rc;
    MTP_REQUIRE(lddz >= out && ldx >= in, "mtp_linear_grad_weight: row distance below the row's length");
    MTP_REQUIRE(dw && (rows == 0 || (dz && x)), "mtp_linear_grad_weight: null pointer");
    const int64_t need = mtp_linear_workspace_bytes(dtype, MTP_LINEAR_GRAD_WEIGHT, rows, in, out, n_sets, dz, lddz, x, ldx);
    if ((int64_t)ws_bytes < need || (need > 0 && (ws == nullptr || (uintptr_t)ws % 16 != 0))) {
        mtp_set_error("mtp_linear_grad_weight: workspace of %zu bytes, needs %lld on a 16-byte boundary", ws_bytes, (long long)need);
        return MTP_E_WORKSPACE;
    }
    return MTP_BY_TYPE(dtype, grad_weight)(dz, rows, out, lddz, x, in, ldx, offsets, n_sets, dw, db,
                                           reinterpret_cast<char *>(ws), mtp_stream(stream));
}

extern "C" int64_t mtp_linear_backward_workspace_bytes(int dtype, int64_t rows, int in, int out, int n_sets, int act, const void *g,
                                                       const void *w, int64_t ldw, const void *x, int64_t ldx, int want_x,
                                                       int want_w) {
    if (rows < 0 || in < 1 || out < 1 || n_sets < 1) return 0;
    return plan_backward(dtype, rows, in, out, n_sets, act, g, w, ldw, x, ldx, want_x != 0, want_w != 0).total();
}

extern "C" int mtp_linear_backward(int dtype, const void *g, const void *pre, int act, const void *x, int64_t rows, int in,
                                   int64_t ldx, const void *w, int out, int64_t ldw, const int32_t *offsets, int n_sets, void *dx,
                                   void *dw, void *db, void *ws, size_t ws_bytes, void *stream) {
    int rc = check_sizes("mtp_linear_backward", dtype, rows, in, out, offsets, n_sets);
    if (rc != MTP_OK) return rc;
    MTP_REQUIRE(dx || dw, "mtp_linear_backward: nothing is asked for");
    MTP_REQUIRE(db == nullptr || dw != nullptr, "mtp_linear_backward: the bias' gradient comes with the weight's");
    const BackwardPlan p = plan_backward(dtype, rows, in, out, n_sets, act, g, w, ldw, x, ldx, dx != nullptr, dw != nullptr);
    if ((int64_t)ws_bytes < p.total() || (p.total() > 0 && (ws == nullptr || (uintptr_t)ws % 16 != 0))) {
        mtp_set_error("mtp_linear_backward: workspace of %zu bytes, needs %lld on a 16-byte boundary", ws_bytes, (long long)p.total());
        return MTP_E_WORKSPACE;
    }
    MTP_REQUIRE(rows == 0 || (g && (act == LIN_NONE || pre) && (dx == nullptr || w) && (dw == nullptr || x)),
                "mtp_linear_backward: null pointer");
    MTP_REQUIRE(ldx >= in && ldw >= in, "mtp_linear_backward: row distance below the row's length");
    char *at = reinterpret_cast<char *>(ws);
    const void *dz = g;
    int64_t lddz = p.lddz;
    hipStream_t s = mtp_stream(stream);
    LinSums sums{};
    if (act != LIN_NONE) {
        if (db != nullptr && rows > 0 && sums_beside(dtype, act)) {
            const int bits = sum_bits_for(rows, out);
            sums = LinSums{reinterpret_cast<float *>(at + p.dz_bytes), db, bits, most_parts(rows, n_sets, bits)};
            db = nullptr;
            rc = dtype == MTP_BFLOAT16 ? launch_sums<__bf16>(g, pre, rows, out, act, offsets, n_sets, ws, lddz, sums, s)
                                       : launch_sums<_Float16>(g, pre, rows, out, act, offsets, n_sets, ws, lddz, sums, s);
        } else {
            rc = mtp_linear_act_grad(dtype, g, pre, rows, out, act, offsets, n_sets, ws, lddz, stream);
        }
        if (rc != MTP_OK) return rc;
        dz = ws;
        at += p.dz_bytes + p.sums_bytes;
    } else if (p.dz_bytes > 0) {  // both products read it
        const void *none = nullptr;
        int64_t ld = 0;
        rc = MTP_BY_TYPE(dtype, relayout)(&dz, &lddz, rows, out, &none, &ld, 0, 0, &at, s);
        if (rc != MTP_OK) return rc;
    }
    if (p.w_bytes + p.x_bytes > 0) {  // in one launch
        rc = MTP_BY_TYPE(dtype, relayout)(&w, &ldw, p.w_bytes > 0 ? (int64_t)n_sets * out : 0, in, &x, &ldx, p.x_bytes > 0 ? rows : 0, in,
                                          &at, s);
        if (rc != MTP_OK) return rc;
    }
    return MTP_BY_TYPE(dtype, grad_both)(dz, rows, out, lddz, w, ldw, x, in, ldx, offsets, n_sets, dx, dw, db, sums, at, s);
}
