// The tiled product of the linear layers (included by linear.hip).
//
//   out[r][c] = sum_k Q(r, k) P(c, k)
//
// P runs along the contiguous axis of the output, Q along its rows.  Forward: P = W, Q = x; input gradient: P = W taken
// along its rows, Q = dz; weight gradient: P = x, Q = dz, the sum running over the tokens.  Each operand is either "KC"
// (the summed index is contiguous in memory) or "RC" (the output's index is).
//
// One workgroup owns a BC x BR tile.  Tiles of 128 bytes of k (64 halves or 32 floats) go from memory straight into LDS,
// 16 bytes a lane, into one of two buffers while the other feeds the matrix cores.  The loads are buffer loads: what lies
// behind the operand's last element arrives as zero, so ragged rows and ragged sums need no code in the loop.  A KC row
// whose length is no multiple of 16 bytes has its last piece cleared in LDS before it is used.
//
// LDS layouts (16-byte pieces; 64 banks of 4 bytes):
//   KC: row i holds its 8 pieces at p ^ ((i >> 1) & 7): the 16 rows that one step of a ds_read_b128 touches fall on 16
//       different pieces of the 256-byte bank line.
//   RC: k row after k row; 16-bit operands are read with the transposing ds_read_b64_tr_b16 (a group of 16 lanes reads four
//       k rows of 16 columns), pieces placed at p ^ 4 * (row bits) so that the four rows fall on different banks; floats
//       are read one by one, the two lane halves (k and k + 4) on different halves of the bank line.
#pragma once
#include <type_traits>

#include "mtp_internal.h"

typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef float f32x16v __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8v __attribute__((ext_vector_type(8)));
typedef short s16x4v __attribute__((ext_vector_type(4)));
typedef short s16x8v __attribute__((ext_vector_type(8)));
typedef int i32x4v __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    return (float)v;
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    return (T)v;  // round to nearest even
}

// LDS-DMA of 16 bytes a lane: LDS destination = uniform byte address + lane * 16, source = buffer + voff, zero where voff is
// outside the buffer.  Inline asm so that the compiler does not wait for it in front of the next ds_read; the caller waits
// (dma_wait_all) before the barrier that publishes the tile.  M0 is kept.
__device__ __forceinline__ void buffer_lds16(i32x4v rsrc, unsigned voff, unsigned lds_uniform) {
    unsigned keep;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %3\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %1, %2, 0 offen lds\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(keep)
        : "v"(voff), "s"(rsrc), "s"(lds_uniform)
        : "memory");
}
__device__ __forceinline__ void dma_wait_all() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// until at most N of this wave's loads are in flight (they land in their order)
template <int N>
__device__ __forceinline__ void dma_wait() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Buffer descriptor of [p, p + bytes), raw; p and bytes are the same in every lane.
__device__ __forceinline__ i32x4v make_rsrc(const void *p, int64_t bytes) {
    // the range check works on 4 bytes: a last lone half has to be inside (its neighbour is in the same aligned 4 bytes)
    const uint64_t a = (uint64_t)(uintptr_t)p;
    const int64_t n = bytes <= 0 ? 0 : (bytes > 0x7ffffffc ? 0x7ffffffc : (bytes + 3) & ~(int64_t)3);
    i32x4v r;
    r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
    r[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)((a >> 32) & 0xffff));
    r[2] = __builtin_amdgcn_readfirstlane((int)n);
    r[3] = 0x00020000;
    return r;
}

// One operand: the matrix, its leading dimension, and how many of its elements count.
struct LinOperand {
    const void *base;
    int64_t ld;     // elements from row to row
    int64_t group;  // elements from one set to the next (weights), 0 where all sets share the matrix
};

constexpr unsigned LIN_OUTSIDE = 0x80000000u;  // a buffer offset that no descriptor above reaches

// Loads and reads R x 128 bytes of one operand.  SZ: element size.
template <typename T, bool KC, int R, int NT>
struct LinTile {
    static constexpr int SZ = sizeof(T);
    static constexpr int EPC = 16 / SZ;             // elements per piece
    static constexpr int BK = 128 / SZ;             // k per tile
    static constexpr int PIECES = R * 8;            // the same for both layouts
    static constexpr int PER = PIECES / NT;         // pieces per thread
    static constexpr int RB = R * SZ;               // RC: bytes of a k row
    static constexpr int CPR = RB / 16;             // RC: pieces of a k row
    static_assert(PIECES % NT == 0, "tile");

    // RC: what is added to a piece's place in its k row
    static __device__ __forceinline__ int twist(int k) {
        if constexpr (SZ == 4) return RB % 256 == 0 ? 8 * ((k >> 2) & 1) : 0;
        else if constexpr (RB % 128 == 64) return 0;  // four rows fall on four different quarters of the bank line by themselves
        else if constexpr (RB == 128) return 4 * ((k >> 1) & 1);
        else return 4 * (k & 3);
    }

    unsigned voff[PER];
    int piece_k[KC ? PER : 1];  // KC: first k of the piece

    __device__ __forceinline__ void init(int64_t ld, int tid) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int q = i * NT + tid;
            if constexpr (KC) {
                const int row = q >> 3, p = (q & 7) ^ ((row >> 1) & 7);
                voff[i] = (unsigned)(row * (int)ld * SZ + p * 16);
                piece_k[i] = p * EPC;
            } else {
                const int k = q / CPR, p = (q % CPR) ^ twist(k);
                voff[i] = (unsigned)(k * (int)ld * SZ + p * 16);
            }
        }
    }
    // k_left: how much of the summed axis this and the later tiles hold
    __device__ __forceinline__ void load(i32x4v rsrc, int64_t k_left, unsigned lds, int wave) const {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            unsigned v = voff[i];
            if constexpr (KC) v = piece_k[i] < k_left ? v : LIN_OUTSIDE;
            buffer_lds16(rsrc, v, lds + (unsigned)((i * NT + wave * 64) * 16));
        }
    }
    // KC, last tile, k_left no multiple of a piece: the elements behind the end of each row become zero
    static __device__ __forceinline__ void clear_tail(char *lds, int k_left, int tid) {
        const int p = k_left / EPC, e0 = k_left % EPC;
        for (int row = tid; row < R; row += NT) {
            T *at = reinterpret_cast<T *>(lds + row * 128 + (p ^ ((row >> 1) & 7)) * 16);
            for (int e = e0; e < EPC; ++e) at[e] = (T)0.f;
        }
    }
};

template <typename T>
struct LinMfma;
template <>
struct LinMfma<__bf16> {
    typedef bf16x8v frag;
    static __device__ __forceinline__ f32x16v mul(frag p, frag q, f32x16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(p, q, c, 0, 0, 0);
    }
    static __device__ __forceinline__ frag ones() {
        frag f;
        for (int i = 0; i < 8; ++i) f[i] = (__bf16)1.f;
        return f;
    }
};
template <>
struct LinMfma<_Float16> {
    typedef f16x8v frag;
    static __device__ __forceinline__ f32x16v mul(frag p, frag q, f32x16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(p, q, c, 0, 0, 0);
    }
    static __device__ __forceinline__ frag ones() {
        frag f;
        for (int i = 0; i < 8; ++i) f[i] = (_Float16)1.f;
        return f;
    }
};
// float: a "fragment" is the four floats a lane half holds of eight consecutive k; four matrix instructions consume it
template <>
struct LinMfma<float> {
    typedef f32x4v frag;
    static __device__ __forceinline__ f32x16v mul(frag p, frag q, f32x16v c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(p[e], q[e], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ frag ones() { return frag{1.f, 1.f, 1.f, 1.f}; }
};

// Reads the 32-row fragments of one operand out of an LDS tile.  A tile holds 128 bytes of k = STEPS fragments (of 16 halves
// or 8 floats).
template <typename T, bool KC, int R>
struct LinReader {
    static constexpr int SZ = sizeof(T);
    static constexpr int STEPS = 4;
    static constexpr int RB = R * SZ;
    typedef typename LinMfma<T>::frag frag;
    const char *at;  // this lane's place for fragment row 0 of the wave
    int k_off[STEPS];
    int lane_, col0_;

    // row0: first row of the wave within the tile (a multiple of 32)
    __device__ __forceinline__ void init(int row0, int lane) {
        const int i = lane & 31, h = lane >> 5;
        lane_ = lane;
        col0_ = row0;
        if constexpr (KC) {
#pragma unroll
            for (int s = 0; s < STEPS; ++s) k_off[s] = (row0 + i) * 128 + (((s * 2 + h) ^ ((i >> 1) & 7)) * 16);
        }
    }
    __device__ __forceinline__ frag read(const char *lds, int f, int s) const {
        if constexpr (KC) {
            return *reinterpret_cast<const frag *>(lds + k_off[s] + f * 32 * 128);
        } else if constexpr (SZ == 2) {
            const int g = lane_ >> 4, i = lane_ & 15;
            const int col = col0_ + f * 32 + 16 * (g & 1) + 4 * (i & 3);
            const int kr = i >> 2;
            const int piece = (col >> 3) ^ LinTile<T, false, R, 64>::twist(kr);
            const char *p = lds + (s * 16 + 8 * (g >> 1) + kr) * RB + piece * 16 + (col & 7) * 2;
            typedef __attribute__((address_space(3))) s16x4v lds_s4;
            const s16x4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)p);
            const s16x4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(p + 4 * RB));
            s16x8v v;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = lo[e];
                v[4 + e] = hi[e];
            }
            return __builtin_bit_cast(frag, v);
        } else {
            const int i = lane_ & 31, h = lane_ >> 5;
            const int col = col0_ + f * 32 + i;
            const int piece = (col >> 2) ^ LinTile<T, false, R, 64>::twist(4 * h);
            const char *p = lds + (s * 8 + 4 * h) * RB + piece * 16 + (col & 3) * 4;
            frag v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const float *>(p + e * RB);
            return v;
        }
    }
};

// ---- sets (experts): rows [offsets[e], offsets[e+1]) belong to set e ----
__device__ __forceinline__ void lin_bounds(const int32_t *offsets, int e, int n_sets, int64_t rows, int64_t *lo, int64_t *hi) {
    // what the caller hands over is kept inside the matrix whatever it says
    int64_t a = offsets[e], b = e < n_sets ? (int64_t)offsets[e + 1] : rows;
    a = a < 0 ? 0 : (a > rows ? rows : a);
    b = b < a ? a : (b > rows ? rows : b);
    *lo = a;
    *hi = b;
}

constexpr int lin_log2(int v) { return v <= 1 ? 0 : 1 + lin_log2(v / 2); }

// prefix sum over the 64 lanes
__device__ __forceinline__ int lin_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8: within 16 lanes
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // lane 15 to the second 16, lane 47 to the fourth
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // lane 31 to the upper 32
    return v;
}

// What a set's rows are cut into, pieces of 1 << part_bits rows: row tiles, or the weight gradient's parts, one at least (a set
// without rows has a gradient of zero).
__host__ __device__ __forceinline__ int lin_pieces(int64_t len, int part_bits, int least) {
    const int n = (int)(((uint32_t)len + (1u << part_bits) - 1) >> part_bits);
    return n < least ? least : n;
}

struct LinPiece {
    int set, count;     // the set and the number of its pieces
    int64_t index;      // which of them
    int64_t lo, hi;     // the set's rows
    int64_t split_at;   // CUT: pieces of sets with more than one piece before this set
};

// Eight neighbouring sets a lane, 512 a wave: the numbers of pieces of the sets from e0 + 8 * lane on (0 beyond `last`).
__device__ __forceinline__ void lin_count(const int32_t *offsets, int n_sets, int last, int64_t rows, int part_bits, int least, int e0,
                                          int (&lo)[8], int (&len)[8], int (&n)[8]) {
    const int first = e0 + (int)(threadIdx.x & 63) * 8;
    int at[9];
#pragma unroll
    for (int u = 0; u < 9; ++u) at[u] = offsets[first + u < n_sets ? first + u : n_sets];  // all on their way at once
    const int top = (int)rows;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const int a = min(max(at[u], 0), top);
        const int b = first + u < n_sets ? min(max(at[u + 1], a), top) : top;
        lo[u] = a;
        len[u] = b - a;
        n[u] = first + u <= last ? lin_pieces(b - a, part_bits, least) : 0;
    }
}

// The sets as a wave sees them, 512 at a time: each lane its eight and the pieces up to and in them.
template <bool CUT>
struct LinSets {
    int lo[8], len[8], n[8], mine, upto, many, many_upto;

    __device__ __forceinline__ void look(const int32_t *offsets, int n_sets, int last, int64_t rows, int part_bits, int least, int e0) {
        lin_count(offsets, n_sets, last, rows, part_bits, least, e0, lo, len, n);
        mine = many = 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            mine += n[u];
            if (CUT) many += n[u] > 1 ? n[u] : 0;
        }
        upto = lin_scan(mine);
        many_upto = CUT ? lin_scan(many) : 0;
    }
    // piece `want` of these 512 (e0: the first of them): the lane that has it, then its counts one by one
    __device__ __forceinline__ bool find(int64_t want, int e0, int64_t split_before, LinPiece *out) const {
        const uint64_t hit = __ballot(want >= upto - mine && want < upto);
        if (hit == 0) return false;
        const int src = __builtin_ctzll(hit);
        int at = __builtin_amdgcn_readlane(upto - mine, src), split_at = CUT ? __builtin_amdgcn_readlane(many_upto - many, src) : 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int c = __builtin_amdgcn_readlane(n[u], src);
            if (want < at + c) {
                out->set = e0 + src * 8 + u;
                out->count = c;
                out->index = want - at;
                out->lo = __builtin_amdgcn_readlane(lo[u], src);
                out->hi = out->lo + __builtin_amdgcn_readlane(len[u], src);
                out->split_at = split_before + split_at;
                return true;
            }
            at += c;
            if (CUT) split_at += c > 1 ? c : 0;
        }
        return false;
    }
};

// Piece number `piece`, counted set after set (`last`: number of the last set; the rows behind the sets are "set" n_sets).  Every
// wave finds it for itself.
template <bool CUT>
__device__ __forceinline__ bool lin_find(const int32_t *offsets, int n_sets, int last, int64_t rows, int part_bits, int least,
                                         int64_t piece, LinPiece *out) {
    int64_t before = 0, split_before = 0;
    for (int e0 = 0; e0 <= last; e0 += 512) {
        LinSets<CUT> sets;
        sets.look(offsets, n_sets, last, rows, part_bits, least, e0);
        if (sets.find(piece - before, e0, split_before, out)) return true;
        before += __builtin_amdgcn_readlane(sets.upto, 63);
        if (CUT) split_before += __builtin_amdgcn_readlane(sets.many_upto, 63);
    }
    return false;
}

// The piece behind `p`: the next of its set, or the first of the next set that has rows (the rows behind the sets are "set" n_sets).
__device__ __forceinline__ void lin_next(const int32_t *offsets, int n_sets, int64_t rows, int part_bits, LinPiece *p) {
    if (++p->index < p->count) return;
    p->index = 0;
    const int top = (int)rows;
    do {
        ++p->set;
        if (p->set > n_sets) return;  // not while pieces are left
        const int lo = min(max(offsets[p->set], 0), top);
        const int hi = p->set < n_sets ? min(max(offsets[p->set + 1], lo), top) : top;
        p->lo = lo;
        p->hi = hi;
        p->count = lin_pieces(hi - lo, part_bits, 0);
    } while (p->count == 0);
}

// parts of the sets before `set` that are cut into more than one
__device__ __forceinline__ int64_t lin_parts_before(const int32_t *offsets, int n_sets, int set, int64_t rows, int part_bits) {
    int64_t before = 0;
    for (int e0 = 0; e0 < set; e0 += 512) {
        int lo[8], len[8], n[8], many = 0;
        lin_count(offsets, n_sets, set - 1, rows, part_bits, 1, e0, lo, len, n);
#pragma unroll
        for (int u = 0; u < 8; ++u) many += n[u] > 1 ? n[u] : 0;
        before += __builtin_amdgcn_readlane(lin_scan(many), 63);
    }
    return before;
}

enum { LIN_NONE = 0, LIN_RELU = 1, LIN_GELU = 2, LIN_SILU = 3 };

// 0.5 erfc(|z| / sqrt 2) = 0.5 exp(-z^2 / 2) t P(t), t = 1 / (1 + 0.4 |z| / sqrt 2): the form of Hastings' approximations
// (Abramowitz and Stegun 7.1.26), P of degree 5 fitted here to 3e-8; evaluated in float it is off by at most 2e-7.  *e
// receives exp(-z^2 / 2), which the slope needs too.
__device__ __forceinline__ float lin_gauss_tail(float z, float *e) {
    *e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
    const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(z), 0.28284271247461901f, 1.f));
    float p = fmaf(t, -0.20033471286296844f, 0.7094687819480896f);
    p = fmaf(t, p, -0.37145283818244934f);
    p = fmaf(t, p, 0.46873366832733154f);
    p = fmaf(t, p, 0.16163088381290436f);
    p = fmaf(t, p, 0.23195423185825348f);
    return 0.5f * *e * t * p;
}
// the standard normal distribution function
__device__ __forceinline__ float lin_gauss(float z, float *e) {
    const float tail = lin_gauss_tail(z, e);
    return z < 0.f ? tail : 1.f - tail;
}
__device__ __forceinline__ float lin_sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
}

__device__ __forceinline__ float lin_act(float z, int act) {
    if (act == LIN_RELU) return z > 0.f ? z : (z != z ? z : 0.f);
    if (act == LIN_GELU) {
        float e;
        return z * lin_gauss(z, &e);
    }
    if (act == LIN_SILU) return z * lin_sigmoid(z);
    return z;
}
__device__ __forceinline__ float lin_slope(float z, int act) {
    if (act == LIN_RELU) return z > 0.f ? 1.f : (z != z ? z : 0.f);
    if (act == LIN_GELU) {
        float e;
        const float c = lin_gauss(z, &e);
        return fmaf(z * 0.39894228040143268f, e, c);
    }
    if (act == LIN_SILU) {
        const float q = lin_sigmoid(z);
        return q * fmaf(z, 1.f - q, 1.f);
    }
    return 1.f;
}

struct LinArgs {
    LinOperand P, Q;
    int64_t rows;      // rows of x
    int cols, k;       // contiguous size of the output; length of the summed axis (forward, input gradient)
    const int32_t *offsets;  // [n_sets + 1] or NULL
    int n_sets;
    int64_t row_tiles;
    uint32_t tiles;    // workgroups' worth of work in all, at most
    int col_tiles;
    int out_rows, part_bits;  // weight gradient: rows of the output; a workgroup sums 1 << part_bits rows of x
    const void *bias;
    const void *residual;
    int64_t ld_res;
    int act;
    void *out;
    void *pre;
    void *bias_out;
    float *partial;  // weight gradient: the sums of sets that are cut into parts, [parts][out_rows][cols], ...
    float *partial_bias;  // ... and [parts][out_rows]
    int64_t parts;        // room for so many
    int away;             // the output is more than the caches hold: past them
};

// N consecutive elements at any address an element can have (the card reads and writes 16 bytes wherever they start)
template <typename T, int N>
struct LinLoose {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T>
struct LinLoose<T, 1> {
    typedef T type;
};
// where a row's piece starts: the last one moves back so that it ends with the row, and says some of the one before it again (a
// thread that went through an incomplete piece by elements would hold its wave up)
__device__ __forceinline__ uint32_t lin_piece_at(uint32_t c, int cols, int n) {
    return (int)c + n <= cols ? c : cols >= n ? (uint32_t)(cols - n) : 0;
}
template <typename T, int N>
__device__ __forceinline__ typename LinLoose<T, N>::type lin_pack(const float *v) {
    typename LinLoose<T, N>::type w;
    if constexpr (N == 1) w = from_f32<T>(v[0]);
    else {
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = from_f32<T>(v[e]);
    }
    return w;
}
template <typename T, int N>
__device__ __forceinline__ void lin_store(T *p, const float *v) {
    *reinterpret_cast<typename LinLoose<T, N>::type *>(p) = lin_pack<T, N>(v);
}
// the same past the caches: what is not read again soon
template <typename T, int N>
__device__ __forceinline__ void lin_store_away(T *p, const float *v) {
    __builtin_nontemporal_store(lin_pack<T, N>(v), reinterpret_cast<typename LinLoose<T, N>::type *>(p));
}
template <typename T, int N>
__device__ __forceinline__ void lin_unpack(const typename LinLoose<T, N>::type &w, float *v) {
    if constexpr (N == 1) v[0] = to_f32(w);
    else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = to_f32(w[e]);
    }
}
template <typename T, int N>
__device__ __forceinline__ void lin_load(const T *p, float *v) {
    lin_unpack<T, N>(*reinterpret_cast<const typename LinLoose<T, N>::type *>(p), v);
}
// Consecutive workgroups go to different XCDs in turn: each XCD gets one contiguous run of tiles, so that the tiles that share
// an operand meet in one L2.
__device__ __forceinline__ uint32_t lin_xcd_order(uint32_t id, uint32_t n) {
    const uint32_t per = n / 8;
    return id < per * 8 ? (id % 8) * per + id / 8 : id;
}

// a piece's place in a row of `pieces` may be twisted by these bits of the row's number
constexpr int lin_twist_mask(int pieces) { return (pieces & -pieces) < 32 ? (pieces & -pieces) - 1 : 31; }
// the largest power of two that is at most `room` and `rows`
constexpr int lin_pass_rows(int room, int rows) {
    int n = 1;
    while (n * 2 <= room && n * 2 <= rows) n *= 2;
    return n;
}

enum { LIN_FORWARD = 0, LIN_GRAD_INPUT = 1, LIN_GRAD_WEIGHT = 2 };

// A tile's rows on their way out of LDS, N columns (16 bytes) a thread; U is the type they leave in.  Up to four rows are on their
// way at a time (two where there are many: 256 x 256 tiles with everything 335 us, 388 with four).  The thread that has a row's
// last, incomplete piece takes it element by element.
template <typename T, typename U, int MODE, int BC, int ER, int NT>
__device__ __forceinline__ void lin_leave(const LinArgs &a, const float *z, const float *bias, U *to, int64_t r0, int64_t row_end,
                                          int64_t c0, int tid) {
    constexpr int N = 16 / (int)sizeof(U), ITEMS = BC / N, STEP = NT / ITEMS;  // STEP: rows that the workgroup takes at a time
    constexpr int PM = lin_twist_mask(BC / 4), AT_ONCE = ER / STEP < 1 ? 1 : ER / STEP <= 4 ? ER / STEP : 2;
    const int item = tid % ITEMS;
    const int64_t col = c0 + item * N;
    if (col >= a.cols || tid >= ITEMS * STEP) return;
    const int n = (int)(a.cols - col < N ? a.cols - col : N);
    const int rows = (int)(row_end - r0 < ER ? row_end - r0 : ER);
    const bool away = MODE != LIN_GRAD_WEIGHT && a.away;
    for (int row0 = tid / ITEMS; row0 < rows; row0 += STEP * AT_ONCE) {
        float v[AT_ONCE][N], res[AT_ONCE][N];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int row = row0 + u * STEP < rows ? row0 + u * STEP : row0;
#pragma unroll
            for (int q = 0; q < N / 4; ++q) {
                const f32x4v w = *reinterpret_cast<const f32x4v *>(z + row * BC + (((item * (N / 4) + q) ^ (row & PM)) << 2));
#pragma unroll
                for (int e = 0; e < 4; ++e) v[u][q * 4 + e] = w[e];
            }
            if constexpr (MODE == LIN_FORWARD) {
                if (a.residual != nullptr) {
                    const T *from = reinterpret_cast<const T *>(a.residual) + (r0 + row) * a.ld_res + col;
                    if (n == N) lin_load<T, N>(from, res[u]);
                    else {
#pragma unroll
                        for (int e = 0; e < N; ++e) res[u][e] = e < n ? to_f32(from[e]) : 0.f;
                    }
                }
            }
        }
        auto leave = [&](auto *first, bool past) {
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                if (row0 + u * STEP >= rows) continue;
                auto *at = first + (r0 + row0 + u * STEP) * a.cols + col;
                typedef std::remove_reference_t<decltype(*at)> V;
                if (n < N) {
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        if (e < n) at[e] = from_f32<V>(v[u][e]);
                } else if (past) {
                    lin_store_away<V, N>(at, v[u]);
                } else {
                    lin_store<V, N>(at, v[u]);
                }
            }
        };
        if constexpr (MODE == LIN_FORWARD) {
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
                for (int e = 0; e < N; ++e) v[u][e] += bias[e];
            if (a.pre != nullptr) leave(reinterpret_cast<T *>(a.pre), true);
            auto bend = [&](auto kind) {
#pragma unroll
                for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
                    for (int e = 0; e < N; ++e) v[u][e] = lin_act(v[u][e], decltype(kind)::value);
            };
            if (a.act == LIN_GELU) bend(std::integral_constant<int, LIN_GELU>{});
            else if (a.act == LIN_SILU) bend(std::integral_constant<int, LIN_SILU>{});
            else if (a.act == LIN_RELU) bend(std::integral_constant<int, LIN_RELU>{});
            if (a.residual != nullptr) {
#pragma unroll
                for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
                    for (int e = 0; e < N; ++e) v[u][e] += res[u][e];
            }
        }
        leave(to, away);
    }
}
// the bias of the columns that lin_leave gives this thread
template <typename T, int BC>
__device__ __forceinline__ void lin_bias(const LinArgs &a, int set, int64_t c0, int tid, float *bias) {
    constexpr int N = 16 / (int)sizeof(T);
    const int64_t col = c0 + tid % (BC / N) * N;
#pragma unroll
    for (int e = 0; e < N; ++e) bias[e] = 0.f;
    if (a.bias == nullptr) return;
    const T *b = reinterpret_cast<const T *>(a.bias) + (int64_t)set * a.cols;
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (col + e < a.cols) bias[e] = to_f32(b[col + e]);
}

// waves a SIMD that a tile's 2 * (BC + BR) * 128 bytes of LDS leave room for (160 KB a CU): what the registers have to allow
constexpr int lin_waves(int bc, int br, int threads) {
    const int groups = 160 * 1024 / (2 * (bc + br) * 128);
    const int waves = groups * threads / 256;
    return waves < 1 ? 1 : waves > 4 ? 4 : waves;
}

// A wave owns WC x WR of the BC x BR tile as 32 x 32 fragments: 32x32x16 matrix instructions for the 16-bit types, 32x32x2 for float.
// What bounds it depends on the sizes.  Long sums, bfloat16, 32 768 rows of 2048 -> 2048 in 256 x 256 tiles: forward 248 us
// (1.11 PFLOP/s; a library product 1.13 to 1.46), 330 with gelu, the kept z and a residual, as nothing covers a single workgroup's
// way out; input gradient 235; weight gradient 245 with its join, as the transposing reads run at half the rate of the others.  The
// matrix cores are busy for half of the time; leaving the LDS loads out would take a fifth off, fragments read one step ahead
// nothing.  Short sums: the way out (143 760 rows over 400 sets, 96 -> 256 bfloat16: 46 us, 68 with gelu and the kept z, which are
// some 25 vector instructions an element and 74 MB).  float: the matrix cores (73 568 rows, 512 -> 96: 71 us, 102 TFLOP/s; 153 in a
// large library product).
template <typename T, int MODE, int BC, int BR, int WC, int WR>
__device__ __forceinline__ void lin_tile(const LinArgs &a, uint32_t block, uint32_t blocks, char *smem) {
    constexpr int NT = 64 * (BC / WC) * (BR / WR);
    constexpr bool PKC = MODE == LIN_FORWARD, QKC = MODE != LIN_GRAD_WEIGHT;
    constexpr int SZ = sizeof(T), BK = 128 / SZ;
    constexpr int FC = WC / 32, FR = WR / 32;
    constexpr int P_BYTES = BC * 128, STAGE = (BC + BR) * 128;
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wc = wave % (BC / WC), wr = wave / (BC / WC);

    // How many tiles there are of up to 511 sets is known here only.  Forward and input gradient: a workgroup takes several that follow
    // each other, so that it looks the sets up once (143 760 rows over 400, 96 -> 256: 1.5 of the 6 us that a tile took were that).
    // Weight gradient: a run of them for each XCD (numbered over the whole grid the last XCD would have the empty ones).
    uint32_t left = 1, id = block;
    int ct = 0;
    LinPiece p{0, 1, 0, 0, a.rows, 0};
    if (a.offsets != nullptr && a.n_sets < 512) {
        constexpr bool WEIGHT = MODE == LIN_GRAD_WEIGHT;
        LinSets<WEIGHT> sets;
        sets.look(a.offsets, a.n_sets, WEIGHT ? a.n_sets - 1 : a.n_sets, a.rows, WEIGHT ? a.part_bits : lin_log2(BR), WEIGHT ? 1 : 0, 0);
        const uint32_t most = (uint32_t)__builtin_amdgcn_readlane(sets.upto, 63) * (uint32_t)a.col_tiles *
                              (WEIGHT ? (uint32_t)a.row_tiles : 1u);
        const uint32_t tiles = most < a.tiles ? most : a.tiles;
        if (WEIGHT) {
            if (id >= tiles) return;
            id = lin_xcd_order(id, tiles);
        } else {
            id = lin_xcd_order(id, blocks);
            const uint32_t per = tiles / blocks, more = tiles % blocks;
            const uint32_t first = id * per + id * more / blocks;
            left = (id + 1) * per + (id + 1) * more / blocks - first;
            id = first;
        }
        ct = (int)(id % (uint32_t)a.col_tiles);
        id /= (uint32_t)a.col_tiles;
        const uint32_t at = WEIGHT ? id / (uint32_t)a.row_tiles : id;
        if (left == 0 || !sets.find(at, 0, 0, &p)) return;
    } else {
        if (a.offsets == nullptr) id = lin_xcd_order(id, a.tiles);
        ct = (int)(id % (uint32_t)a.col_tiles);
        id /= (uint32_t)a.col_tiles;
        if (a.offsets == nullptr) {
            if (MODE != LIN_GRAD_WEIGHT) p.index = id;
            else {
                p.count = lin_pieces(a.rows, a.part_bits, 1);
                p.index = id / (uint32_t)a.row_tiles;
            }
        } else if (MODE == LIN_GRAD_WEIGHT ? !lin_find<true>(a.offsets, a.n_sets, a.n_sets - 1, a.rows, a.part_bits, 1,
                                                             id / (uint32_t)a.row_tiles, &p)
                                           : !lin_find<false>(a.offsets, a.n_sets, a.n_sets, a.rows, lin_log2(BR), 0, id, &p)) {
            return;
        }
    }
    for (bool again = false; left > 0; --left, again = true) {
        int tid_here = tid;
        asm volatile("" : "+v"(tid_here));  // what follows from it is found anew for each tile: there are no registers to keep it in
        if (again) {
            __syncthreads();  // the last tile has left LDS
            if (++ct == (int)a.col_tiles) {
                ct = 0;
                lin_next(a.offsets, a.n_sets, a.rows, lin_log2(BR), &p);
                if (p.set > a.n_sets) return;
            }
        }
        int64_t row0 = 0, row_end = 0, k_lo = 0, k_len = a.k, part_at = -1;
        const int64_t c0 = (int64_t)ct * BC;
        if constexpr (MODE == LIN_GRAD_WEIGHT) {
            row0 = (int64_t)(id % (uint32_t)a.row_tiles) * BR;
            row_end = a.out_rows;
            k_lo = p.lo + (p.index << a.part_bits);
            k_len = p.hi - k_lo < (1 << a.part_bits) ? p.hi - k_lo : (int64_t)1 << a.part_bits;
            if (p.count > 1) {
                part_at = p.split_at + p.index;
                if (part_at >= a.parts) return;  // offsets that overlap: more parts than there can be
            }
        } else {
            row0 = p.lo + p.index * BR;
            row_end = p.hi;
        }
        const int set = p.set;
        T *out = reinterpret_cast<T *>(a.out);
        if (MODE != LIN_GRAD_WEIGHT && set == a.n_sets) {  // rows behind the last set
            for (int i = tid; i < BR * BC; i += NT) {
                const int64_t r = row0 + i / BC, c = c0 + i % BC;
                if (r < row_end && c < a.cols) {
                    out[r * a.cols + c] = (T)0.f;
                    if (MODE == LIN_FORWARD && a.pre != nullptr) reinterpret_cast<T *>(a.pre)[r * a.cols + c] = (T)0.f;
                }
            }
            continue;
        }

        // operand windows: first element, bytes to the last element that counts, bytes per step along k
        const T *p_at = reinterpret_cast<const T *>(a.P.base) + set * a.P.group;
        const T *q_at = reinterpret_cast<const T *>(a.Q.base) + set * a.Q.group;
        int64_t p_left, q_left, p_step, q_step;
        if constexpr (PKC) {
            const int64_t n = a.cols - c0 < BC ? a.cols - c0 : BC;
            p_at += c0 * a.P.ld;
            p_left = ((n - 1) * a.P.ld + k_len) * SZ;
            p_step = 128;
        } else {
            p_at += k_lo * a.P.ld + c0;
            p_left = k_len > 0 ? ((k_len - 1) * a.P.ld + a.cols - c0) * SZ : 0;
            p_step = (int64_t)BK * a.P.ld * SZ;
        }
        const int64_t n_rows = row_end - row0 < BR ? row_end - row0 : BR;
        if constexpr (QKC) {
            q_at += row0 * a.Q.ld;
            q_left = ((n_rows - 1) * a.Q.ld + k_len) * SZ;
            q_step = 128;
        } else {
            q_at += k_lo * a.Q.ld + row0;
            q_left = k_len > 0 ? ((k_len - 1) * a.Q.ld + row_end - row0) * SZ : 0;
            q_step = (int64_t)BK * a.Q.ld * SZ;
        }
        LinTile<T, PKC, BC, NT> tp;
        LinTile<T, QKC, BR, NT> tq;
        tp.init(a.P.ld, tid_here);
        tq.init(a.Q.ld, tid_here);
        LinReader<T, PKC, BC> rp;
        LinReader<T, QKC, BR> rq;
        rp.init(wc * WC, tid_here & 63);
        rq.init(wr * WR, tid_here & 63);
        f32x16v acc[FC][FR];
        f32x16v acc_ones[MODE == LIN_GRAD_WEIGHT ? FR : 1];
#pragma unroll
        for (int c = 0; c < FC; ++c)
#pragma unroll
            for (int r = 0; r < FR; ++r)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[c][r][e] = 0.f;
        const bool sum_q = MODE == LIN_GRAD_WEIGHT && a.bias_out != nullptr && ct == 0 && wc == 0;
        if constexpr (MODE == LIN_GRAD_WEIGHT) {
#pragma unroll
            for (int r = 0; r < FR; ++r)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc_ones[r][e] = 0.f;
        }

        const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)smem;
        const int64_t n_steps = (k_len + BK - 1) / BK;
        int64_t k_left = k_len;
        auto fetch_p = [&](int buf) {
            const unsigned l = __builtin_amdgcn_readfirstlane(lds0 + (unsigned)(buf * STAGE));
            tp.load(make_rsrc(p_at, p_left), k_left, l, wave);
            p_at = reinterpret_cast<const T *>(reinterpret_cast<const char *>(p_at) + p_step);
            p_left -= p_step;
        };
        auto fetch_q = [&](int buf) {
            const unsigned l = __builtin_amdgcn_readfirstlane(lds0 + (unsigned)(buf * STAGE));
            tq.load(make_rsrc(q_at, q_left), k_left, l + P_BYTES, wave);
            q_at = reinterpret_cast<const T *>(reinterpret_cast<const char *>(q_at) + q_step);
            q_left -= q_step;
            k_left -= BK;
        };
        auto fetch = [&](int buf) {
            fetch_p(buf);
            fetch_q(buf);
        };
        // Big tiles have one workgroup a CU: its loads are sent in two halves, between products, as eight in a row keep a wave from
        // its products until they have been taken (32 768 rows, 2048 -> 2048: input gradient 257 -> 250 us, weight gradient 365 -> 340;
        // 128x128 tiles, two a CU, 314 -> 326).
        constexpr bool HALVES = BC == 256;
        // both buffers are on their way before the first is used; later tiles are fetched one ahead
        constexpr int IN_FLIGHT = LinTile<T, PKC, BC, NT>::PER + LinTile<T, QKC, BR, NT>::PER;
        if (n_steps > 0) fetch(0);
        if (n_steps > 1) fetch(1);
        for (int64_t t = 0; t < n_steps; ++t) {
            if (t == 0 && n_steps > 1) dma_wait<IN_FLIGHT>();
            else dma_wait_all();
            __syncthreads();  // tile t has landed for every wave, and nobody reads the other buffer any more
            const bool more = t > 0 && t + 1 < n_steps;
            if (more) {
                if constexpr (HALVES) fetch_p((int)((t + 1) & 1));
                else fetch((int)((t + 1) & 1));
            }
            char *buf = smem + (t & 1) * STAGE;
            const int64_t left = k_len - t * BK;
            if constexpr (PKC || QKC) {
                if (left < BK && left % (16 / SZ) != 0) {
                    if constexpr (PKC) LinTile<T, true, BC, NT>::clear_tail(buf, (int)left, tid);
                    if constexpr (QKC) LinTile<T, true, BR, NT>::clear_tail(buf + P_BYTES, (int)left, tid);
                    __syncthreads();
                }
            }
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                if (HALVES && s == 1 && more) fetch_q((int)((t + 1) & 1));
                typename LinMfma<T>::frag fp[FC], fq[FR];
#pragma unroll
                for (int c = 0; c < FC; ++c) fp[c] = rp.read(buf, c, s);
#pragma unroll
                for (int r = 0; r < FR; ++r) fq[r] = rq.read(buf + P_BYTES, r, s);
#pragma unroll
                for (int c = 0; c < FC; ++c)
#pragma unroll
                    for (int r = 0; r < FR; ++r) acc[c][r] = LinMfma<T>::mul(fp[c], fq[r], acc[c][r]);
                if constexpr (MODE == LIN_GRAD_WEIGHT) {
                    if (sum_q) {
#pragma unroll
                        for (int r = 0; r < FR; ++r) {
                            if constexpr (SZ == 4) {  // a matrix instruction would cost as much as one of the product's
#pragma unroll
                                for (int e = 0; e < 4; ++e) acc_ones[r][0] += fq[r][e];
                            } else {
                                acc_ones[r] = LinMfma<T>::mul(LinMfma<T>::ones(), fq[r], acc_ones[r]);
                            }
                        }
                    }
                }
            }
        }

        // ---- epilogue ----
        // lane (i, h) holds row i of a fragment, columns 8 g + 4 h + 0..3 for g = 0..3: stored from there a wave would touch 32 rows
        // with 16 bytes each.  The sums go through LDS (as floats, pieces of 16 bytes placed at p ^ row so that neither side
        // conflicts), and whole rows of the tile leave in 16-byte pieces; bias, activation and residual are applied on the way.
        asm volatile("" : "+v"(tid_here));
        const int lane_here = tid_here & 63, i = lane_here & 31, h = lane_here >> 5;
        constexpr int ER = lin_pass_rows(2 * STAGE / (BC * 4), BR);  // rows per pass
        constexpr int PM = lin_twist_mask(BC / 4);
        static_assert(BR % ER == 0 && ER % WR == 0, "a wave's rows are in one pass");
        float *z = reinterpret_cast<float *>(smem);
        const bool to_partial = MODE == LIN_GRAD_WEIGHT && part_at >= 0;
        float bias[16 / SZ];
        if constexpr (MODE == LIN_FORWARD) lin_bias<T, BC>(a, set, c0, tid_here, bias);
        for (int p0 = 0; p0 < BR; p0 += ER) {
            __syncthreads();
            if (wr * WR >= p0 && wr * WR < p0 + ER) {
#pragma unroll
                for (int c = 0; c < FC; ++c)
#pragma unroll
                    for (int r = 0; r < FR; ++r)
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const int row = wr * WR - p0 + r * 32 + i;
                            const int piece = (wc * WC + c * 32 + 8 * g + 4 * h) >> 2;
                            f32x4v v;
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] = acc[c][r][4 * g + e];
                            *reinterpret_cast<f32x4v *>(z + row * BC + ((piece ^ (row & PM)) << 2)) = v;
                        }
            }
            __syncthreads();
            const int64_t r0 = row0 + p0;
            if (to_partial) {
                float *part = a.partial + part_at * a.out_rows * a.cols;
                lin_leave<T, float, MODE, BC, ER, NT>(a, z, bias, part, r0, row_end, c0, tid_here);
            } else {
                T *to = out + (MODE == LIN_GRAD_WEIGHT ? (int64_t)set * a.out_rows * a.cols : 0);
                lin_leave<T, T, MODE, BC, ER, NT>(a, z, bias, to, r0, row_end, c0, tid_here);
            }
        }
        if constexpr (MODE == LIN_GRAD_WEIGHT && SZ == 4) {  // the two halves of a wave hold different k
            if (sum_q) {
#pragma unroll
                for (int r = 0; r < FR; ++r) acc_ones[r][0] += __shfl_xor(acc_ones[r][0], 32);
            }
        }
        if constexpr (MODE == LIN_GRAD_WEIGHT) {
            if (sum_q && h == 0) {
#pragma unroll
                for (int r = 0; r < FR; ++r) {
                    const int64_t row = row0 + wr * WR + r * 32 + i;
                    if (row < row_end) {
                        if (part_at >= 0) a.partial_bias[part_at * a.out_rows + row] = acc_ones[r][0];
                        else reinterpret_cast<T *>(a.bias_out)[(int64_t)set * a.out_rows + row] = from_f32<T>(acc_ones[r][0]);
                    }
                }
            }
        }
    }
}

template <typename T, int MODE, int BC, int BR, int WC, int WR>
__global__ __launch_bounds__(64 * (BC / WC) * (BR / WR), lin_waves(BC, BR, 64 * (BC / WC) * (BR / WR))) void k_linear_tile(LinArgs a) {
    extern __shared__ __attribute__((aligned(16))) char tile_lds[];  // 2 * (BC + BR) * 128
    lin_tile<T, MODE, BC, BR, WC, WR>(a, blockIdx.x, gridDim.x, tile_lds);
}

// Both products of a small backward pass side by side: `input_blocks` workgroups for the input gradient (BC x BR tiles), the others for
// the weight gradient (64 x 64).
template <typename T, int BC, int BR>
__global__ __launch_bounds__(256, 4) void k_linear_both(LinArgs input, LinArgs weight, uint32_t input_blocks) {
    extern __shared__ __attribute__((aligned(16))) char both_lds[];
    static_assert((BC / 32) * (BR / 32) == 4, "four waves");
    if (blockIdx.x < input_blocks) lin_tile<T, LIN_GRAD_INPUT, BC, BR, 32, 32>(input, blockIdx.x, input_blocks, both_lds);
    else lin_tile<T, LIN_GRAD_WEIGHT, 64, 64, 32, 32>(weight, blockIdx.x - input_blocks, gridDim.x - input_blocks, both_lds);
}

// ---- few rows ----
// Up to 16 * RT rows of x against 16 columns of the output: W is read once, straight from memory into the operands of the 16 x 16
// matrix instructions (a lane holds 16 bytes of k of one row of W and of x), the four waves share the sum over k and are
// added through LDS.  What bounds it is reading W: each wave has UNROLL pieces of it in flight (64 rows of 2048 x 2048 bfloat16
// 10.8 us; one row of 1024 x 1024 is a launch, 4.7 us).
template <typename T>
struct LinMfma16;
template <>
struct LinMfma16<__bf16> {
    static __device__ __forceinline__ f32x4v mul(bf16x8v p, bf16x8v q, f32x4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(p, q, c, 0, 0, 0);
    }
};
template <>
struct LinMfma16<_Float16> {
    static __device__ __forceinline__ f32x4v mul(f16x8v p, f16x8v q, f32x4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(p, q, c, 0, 0, 0);
    }
};
template <>
struct LinMfma16<float> {
    static __device__ __forceinline__ f32x4v mul(f32x4v p, f32x4v q, f32x4v c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(p[e], q[e], c, 0, 0, 0);
        return c;
    }
};

// 16 bytes of a row; rows need the alignment of their elements only
template <typename T>
__device__ __forceinline__ typename LinMfma<T>::frag lin_piece(const T *at) {
    constexpr int N = 16 / sizeof(T);
    typedef T loose __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    return *reinterpret_cast<const loose *>(at);
}
// the same from k0 on, elements from k on are zero
template <typename T>
__device__ __forceinline__ typename LinMfma<T>::frag lin_piece_to(const T *row, int k0, int k) {
    constexpr int N = 16 / sizeof(T);
    if (k0 + N <= k) return lin_piece<T>(row + k0);
    typename LinMfma<T>::frag f;
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = k0 + e < k ? row[k0 + e] : (T)0.f;
    return f;
}

template <typename T, int RT>
__global__ __launch_bounds__(256) void k_linear_few(LinArgs a) {
    constexpr int N = 16 / (int)sizeof(T), STEP = 4 * N, UNROLL = RT == 1 ? 4 : 2;  // k of a step: four lane groups
    typedef typename LinMfma<T>::frag frag;
    __shared__ f32x4v sums[3][RT][64];
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t ct = blockIdx.x % (uint32_t)a.col_tiles, id = blockIdx.x / (uint32_t)a.col_tiles;
    const int64_t c0 = (int64_t)ct * 16;
    int64_t row0 = 0, row_end = a.rows;
    int set = 0;
    if (a.offsets != nullptr) {
        LinPiece p;
        if (!lin_find<false>(a.offsets, a.n_sets, a.n_sets, a.rows, lin_log2(16 * RT), 0, id, &p)) return;
        set = p.set;
        row0 = p.lo + p.index * (16 * RT);
        row_end = p.hi;
    } else {
        row0 = (int64_t)id * (16 * RT);
    }
    T *out = reinterpret_cast<T *>(a.out);
    if (set == a.n_sets) {  // rows behind the last set
        const int64_t r = row0 + tid / 16, c = c0 + tid % 16;
        for (int64_t x = r; x < row_end && x < row0 + 16 * RT; x += 16)
            if (c < a.cols) {
                out[x * a.cols + c] = (T)0.f;
                if (a.pre != nullptr) reinterpret_cast<T *>(a.pre)[x * a.cols + c] = (T)0.f;
            }
        return;
    }
    const int k = a.k, steps = (k + STEP - 1) / STEP;
    const int64_t wc = c0 + i < a.cols ? c0 + i : a.cols - 1;  // rows and columns that are not there are computed and dropped
    const T *w = reinterpret_cast<const T *>(a.P.base) + set * a.P.group + wc * a.P.ld;
    const T *x[RT];
    f32x4v acc[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int64_t at = row0 + r * 16 + i < row_end ? row0 + r * 16 + i : row_end - 1;
        x[r] = reinterpret_cast<const T *>(a.Q.base) + at * a.Q.ld;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[r][e] = 0.f;
    }
    // wave w takes the steps w, w + 4, ...; the last one may reach beyond k
    const int whole = k / STEP;
    int s0 = wave;
    for (; s0 + 4 * (UNROLL - 1) < whole; s0 += 4 * UNROLL) {
        frag fw[UNROLL], fx[UNROLL][RT];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int k0 = (s0 + 4 * u) * STEP + g * N;
            fw[u] = lin_piece<T>(w + k0);
#pragma unroll
            for (int r = 0; r < RT; ++r) fx[u][r] = lin_piece<T>(x[r] + k0);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int r = 0; r < RT; ++r) acc[r] = LinMfma16<T>::mul(fw[u], fx[u][r], acc[r]);
    }
    for (; s0 < steps; s0 += 4) {
        const int k0 = s0 * STEP + g * N;
        const frag fw = lin_piece_to<T>(w, k0, k);
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[r] = LinMfma16<T>::mul(fw, lin_piece_to<T>(x[r], k0, k), acc[r]);
    }
    if (wave > 0) {
#pragma unroll
        for (int r = 0; r < RT; ++r) sums[wave - 1][r][lane] = acc[r];
    }
    __syncthreads();
    if (wave > 0) return;
    // lane (i, g): row i, columns 4 g to 4 g + 3
    const int64_t col = c0 + 4 * g;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        f32x4v v = acc[r];
#pragma unroll
        for (int o = 0; o < 3; ++o) v += sums[o][r][lane];
        const int64_t row = row0 + r * 16 + i;
        if (row >= row_end) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (col + e >= a.cols) break;
            const int64_t at = row * a.cols + col + e;
            float z = v[e];
            if (a.bias != nullptr) z += to_f32(reinterpret_cast<const T *>(a.bias)[(int64_t)set * a.cols + col + e]);
            if (a.pre != nullptr) reinterpret_cast<T *>(a.pre)[at] = from_f32<T>(z);
            z = lin_act(z, a.act);
            if (a.residual != nullptr) z += to_f32(reinterpret_cast<const T *>(a.residual)[row * a.ld_res + col + e]);
            out[at] = from_f32<T>(z);
        }
    }
}
